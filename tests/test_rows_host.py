"""Layer norm, dropout and sampling without a GPU: what the entry points refuse, and the oracles of the GPU tests."""
import numpy as np
import pytest
import torch

from tests import _row_oracles as R


def test_host_tensors_are_refused():
    from tensornetworksfork_amd import _lib, ops
    from tensornetworksfork_amd.models.tensor_train import sample_labels
    from tensornetworksfork_amd.tensor.norm import Dropout, LayerNorm, dropout, layer_norm
    x, u = torch.zeros(3, 4), torch.zeros(3)
    for f in (lambda: ops.layer_norm(x), lambda: ops.layer_norm_backward(x, x, u, u), lambda: ops.dropout(x, 0.5, 1),
              lambda: ops.sample(x, u), lambda: layer_norm(x), lambda: dropout(x, 0.5, 1), lambda: sample_labels(x, u),
              lambda: LayerNorm(4)(x), lambda: Dropout(0.5)(x), lambda: ops.layer_norm(None), lambda: ops.sample([1.0], u)):
        with pytest.raises(_lib.TTKError):
            f()
    assert Dropout(0.5).eval()(x) is x and Dropout(0.0)(x) is x


def test_library_refuses_bad_arguments_before_any_launch():
    from tensornetworksfork_amd import _lib
    L = _lib.lib()
    P = 4096          # never read: every call below is refused on the host
    ln = lambda **k: L.ttk_layer_norm(*{**dict(dt=1, wdt=1, x=P, ld=4, w=P, b=P, y=P, m=P, r=P, rows=2, cols=4, eps=0.1, p=0.0,  # noqa: E731
                                               seed=0, off=0, offd=None, st=None), **k}.values())
    bw = lambda **k: L.ttk_layer_norm_backward(*{**dict(dt=1, wdt=1, dy=P, lddy=4, x=P, ld=4, w=P, m=P, r=P, dx=P, dw=P, db=P,  # noqa: E731
                                                        rows=2, cols=4, p=0.0, seed=0, off=0, offd=None, ws=P, n=1 << 20,
                                                        st=None), **k}.values())
    dr = lambda **k: L.ttk_dropout(*{**dict(dt=1, x=P, y=P, n=4, p=0.5, seed=0, off=0, offd=None, st=None), **k}.values())  # noqa: E731
    sm = lambda **k: L.ttk_sample(*{**dict(dt=1, z=P, ld=4, u=P, f64=0, t=None, ta=1.0, k=None, ka=0, p=None, pa=1.0, m=None,  # noqa: E731
                                           ma=0.0, out=P, rows=2, V=4, ws=None, n=0, st=None), **k}.values())
    nan = float("nan")
    for k in (dict(x=None), dict(y=None), dict(m=None), dict(r=None), dict(rows=0), dict(cols=0), dict(ld=-1), dict(eps=-1.0),
              dict(eps=nan), dict(dt=4), dict(dt=0, wdt=1), dict(dt=1, wdt=2), dict(dt=-1, wdt=-1), dict(p=1.5), dict(p=nan), dict(off=-1)):
        assert ln(**k) == -1, k
    for k in (dict(dy=None), dict(x=None), dict(m=None), dict(r=None), dict(rows=0), dict(cols=0), dict(lddy=-1), dict(dt=2, wdt=3),
              dict(p=-0.1), dict(off=-5)):
        assert bw(**k) == -1, k
    assert bw(ws=None) == -2 and bw(n=8) == -2
    for k in (dict(x=None), dict(y=None), dict(n=0), dict(dt=7), dict(p=2.0), dict(off=-1)):
        assert dr(**k) == -1, k
    for k in (dict(z=None), dict(u=None), dict(out=None), dict(rows=0), dict(V=0), dict(ld=-2), dict(dt=9), dict(V=(1 << 30) + 1)):
        assert sm(**k) == -1, k
    need = L.ttk_sample_ws_bytes(1, 2, 9000)
    assert need > 0 and sm(V=9000) == -2 and sm(V=9000, ws=P, n=need - 1) == -2
    assert sm(V=9000, ws=P + 4, n=need) == -1 and bw(ws=P + 4) == -1      # (workspaces are aligned to 8 bytes)
    assert L.ttk_sample_ws_bytes(1, 7, 8192) == 0 and L.ttk_sample_ws_bytes(4, 7, 9) == -1 and L.ttk_sample_ws_bytes(1, 0, 9) == -1
    assert L.ttk_layer_norm_backward_ws_bytes(1, 0, 4) == -1 and L.ttk_layer_norm_backward_ws_bytes(9, 4, 4) == -1
    assert L.ttk_layer_norm_backward_ws_bytes(1, 5, 7) >= 2 * 7 * 4


def test_rows_view():
    from tensornetworksfork_amd import _lib, ops
    t = torch.zeros(6, 10)
    assert ops.rows_view(t) == (6, 10, 10) and ops.rows_view(t[:, 2:5]) == (6, 3, 10) and ops.rows_view(t[0]) == (1, 10, 10)
    assert ops.rows_view(t[::2]) == (3, 10, 20) and ops.rows_view(t[:1].expand(4, 10)) == (4, 10, 0)
    assert ops.rows_view(torch.zeros(2, 3, 4)) == (6, 4, 4) and ops.rows_view(torch.zeros(2, 3, 5)[..., :4]) == (6, 4, 5)
    assert ops.rows_view(torch.zeros(5, 1)[:, :1]) == (5, 1, 1) and ops.rows_view(t[:, 3:4]) == (6, 1, 10)
    assert ops.rows_view(torch.zeros(2, 1, 4)) == (2, 4, 4) and ops.rows_view(torch.zeros(0, 4))[0] == 0
    for bad in (t.t(), torch.zeros(2, 3, 4).transpose(0, 1), torch.zeros(3, 0), torch.zeros(())):
        with pytest.raises(_lib.TTKError):
            ops.rows_view(bad)


def test_philox_oracle_known_answer():
    """The generator's published answer for counter 0, key 0."""
    w = R.philox(np.zeros(1, np.uint64), np.zeros(1, np.uint64), 0)[0]
    assert [int(v) for v in w] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    m = R.keep_mask(4000, 0.25, 7, 3)
    assert torch.equal(m[5:], R.keep_mask(3995, 0.25, 7, 8)) and 0.7 < float(m.double().mean()) < 0.8


def test_sampling_oracle():
    z = np.array([1.0, 3.0, 2.0, 3.0])
    assert R.sample_row(z, 0.0, T=0.0)[0] == 1
    assert R.sample_row(z, 0.0, k=1)[0] == 1 and R.sample_row(z, 0.99, k=2)[0] == 3
    assert R.sample_row(z, 0.99, P=0.3)[0] == 1                      # the first of the two largest alone holds 0.39
    assert R.sample_row(z, 0.999, M=0.9)[0] == 3 and R.sample_row(z, 0.0, M=0.9)[0] == 1
    assert R.sample_row(np.full(3, -np.inf), 0.5)[0] == -1 and R.sample_row(np.array([np.nan, 0.0]), 0.0)[0] == 1


def test_estimators_refuse_and_keep_their_defaults():
    from tensornetworksfork_amd.models.tensor_train import TensorTrainRegressor
    from tensornetworksfork_amd.models.tnml import TNMLRegressor
    for cls in (TensorTrainRegressor, TNMLRegressor):
        e = cls()
        assert e.layer_norm is False and e.dropout == 0.0
        with pytest.raises(ValueError):
            cls(dropout=1.0)
        with pytest.raises(ValueError):
            e.sample(np.zeros((2, 3)))
