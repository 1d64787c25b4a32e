"""Layer norm, dropout, label sampling and input gradients at the ends of what they accept, without a GPU."""
import pytest
import torch


def test_sizes_beyond_32_bits_are_counted_in_64():
    """Workspaces of as many rows as a 32-bit count wraps around for: never less than for fewer rows."""
    from tensornetworksfork_amd import _lib
    L = _lib.lib()
    for rows in ((1 << 31) - 1, 1 << 31, (1 << 31) + 1, 1 << 32, (1 << 32) + 5, 3 << 31):
        for dtype in range(4):
            assert L.ttk_sample_ws_bytes(dtype, rows, 9000) == L.ttk_sample_ws_bytes(dtype, 1 << 20, 9000) > 0
            for cols in (3, 40, 600, 5000, 16000, 20000):
                assert L.ttk_layer_norm_backward_ws_bytes(dtype, rows, cols) >= L.ttk_layer_norm_backward_ws_bytes(dtype, 1 << 20, cols) > 0
