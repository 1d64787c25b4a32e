"""Layer norm, dropout and label sampling at the borders of their kernels' layouts: every row length at which a layout begins or
ends, rows that start at any alignment, memory around the operands, cuts that the short lists do not hold."""
import numpy as np
import pytest
import torch

from tests import _row_oracles as R
from tests import test_norm_gpu as N
from tests import test_sample_gpu as S

gpu = pytest.mark.gpu
F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _float32_default():
    """Other tests of the process may have left float64 as torch's default."""
    old = torch.get_default_dtype()
    torch.set_default_dtype(F32)
    yield
    torch.set_default_dtype(old)


# whole and incomplete last vectors on both sides of every layout of 8 to 1024 lanes, for elements of 8, 4 and 2 bytes
COLS = [9, 15, 20, 24, 25, 30, 48, 61, 72, 100, 120, 131, 200, 256, 301, 500, 513, 777, 1024, 1500, 2047, 2300, 4096, 4100, 6001, 8000, 12001,
        16383]


@gpu
@pytest.mark.parametrize("dtype,wdtype", N.TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_layouts(cols, dtype, wdtype):
    from tensornetworksfork_amd import ops
    dev = N._dev()
    rows, p, seed, offset = 37, 0.375, 99, 3          # (scale 1.6: not a power of two; rows that no workgroup divides)
    x, dy, w, b = N._make(rows, cols, dtype, wdtype, cols)
    X, DY, W, B = x.to(dev), dy.to(dev), w.to(dev), b.to(dev)
    y, mean, rstd = ops.layer_norm(X, W, B, 1e-5)
    N._check_forward(y, mean, rstd, x, w, b, 1e-5, dtype)
    N._check_backward(ops.layer_norm_backward(DY, X, mean, rstd, W), dy, x, mean, rstd, w, dtype, wdtype)
    keep = R.keep_mask(rows * cols, p, seed, offset).reshape(rows, cols)
    y, mean, rstd = ops.layer_norm(X, W, B, 1e-5, p, seed, offset)
    N._check_forward(y, mean, rstd, x, w, b, 1e-5, dtype, 1 / (1 - p), keep)
    got = ops.layer_norm_backward(DY, X, mean, rstd, W, p, seed, offset)
    g = torch.where(keep, dy.double() / (1 - p), torch.zeros_like(dy, dtype=F64))
    N._check_backward(got, g, x, mean, rstd, w, dtype, wdtype)
    # what stands where the mask drops does not matter
    other = ops.layer_norm_backward(torch.where(keep.to(dev), DY, torch.full_like(DY, float("nan"))), X, mean, rstd, W, p, seed, offset)
    assert all(torch.equal(a, b) for a, b in zip(got, other))


def _guarded(n, dtype, dev, front=5, behind=70):
    """n elements of memory between sentinels -> (the elements, a check that nothing around them was written)."""
    size = torch.empty(0, dtype=dtype).element_size()
    raw = torch.full(((front + n + behind) * size,), 0xA5, dtype=torch.uint8, device=dev)
    t = raw.view(dtype)[front:front + n]

    def untouched():
        return bool((raw[:front * size] == 0xA5).all()) and bool((raw[(front + n) * size:] == 0xA5).all())
    return t, untouched


@gpu
@pytest.mark.parametrize("dtype", [F64, F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (5, 7), (67, 17), (65, 24), (9, 31), (33, 33), (35, 60), (17, 100), (7, 250), (5, 500),
                                       (3, 1021), (3, 2050), (3, 4090), (2, 6003), (3, 10007), (2, 16390), (2, 40001)])
def test_memory_around_the_operands(rows, cols, dtype):
    """Rows between NaNs come out as they do by themselves, and nothing around the outputs is written."""
    from tensornetworksfork_amd import _lib, ops
    dev = N._dev()
    lib, code, st = _lib.lib(), ops.ROW_TYPES[dtype], torch.cuda.current_stream(dev).cuda_stream
    g = torch.Generator().manual_seed(cols)
    n, stat = rows * cols, F64 if dtype == F64 else F32

    def inside(values):
        big = torch.full((values.numel() + 80,), float("nan"), dtype=dtype, device=dev)
        big[3:3 + values.numel()] = values.reshape(-1)
        return big[3:3 + values.numel()]
    X, DY = (torch.randn(rows, cols, generator=g).to(dtype).to(dev) for _ in range(2))
    W, B = (torch.randn(cols, generator=g).to(dtype).to(dev) for _ in range(2))
    x, dy, w, b = inside(X), inside(DY), inside(W), inside(B)
    y, y_ok = _guarded(n, dtype, dev)
    mean, mean_ok = _guarded(rows, stat, dev)
    rstd, rstd_ok = _guarded(rows, stat, dev)
    assert lib.ttk_layer_norm(code, code, x.data_ptr(), cols, w.data_ptr(), b.data_ptr(), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                              rows, cols, 1e-5, 0.25, 7, 1, None, st) == 0
    ref = ops.layer_norm(X, W, B, 1e-5, 0.25, 7, 1)
    assert torch.equal(y.reshape(rows, cols), ref[0]) and torch.equal(mean, ref[1]) and torch.equal(rstd, ref[2])
    assert y_ok() and mean_ok() and rstd_ok()
    dx, dx_ok = _guarded(n, dtype, dev)
    dw, dw_ok = _guarded(cols, dtype, dev)
    db, db_ok = _guarded(cols, dtype, dev)
    need = lib.ttk_layer_norm_backward_ws_bytes(code, rows, cols)
    ws, ws_ok = _guarded(need, torch.uint8, dev, front=256)
    assert lib.ttk_layer_norm_backward(code, code, dy.data_ptr(), cols, x.data_ptr(), cols, w.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                       dx.data_ptr(), dw.data_ptr(), db.data_ptr(), rows, cols, 0.25, 7, 1, None, ws.data_ptr(), need, st) == 0
    ref = ops.layer_norm_backward(DY, X, ref[1], ref[2], W, 0.25, 7, 1)
    assert torch.equal(dx.reshape(rows, cols), ref[0]) and torch.equal(dw, ref[1]) and torch.equal(db, ref[2])
    assert dx_ok() and dw_ok() and db_ok() and ws_ok()
    y, y_ok = _guarded(n, dtype, dev)
    assert lib.ttk_dropout(code, x.data_ptr(), y.data_ptr(), n, 0.25, 7, 2, None, st) == 0
    assert torch.equal(y.reshape(rows, cols), ops.dropout(X, 0.25, 7, 2)) and y_ok()


@gpu
@pytest.mark.parametrize("dtype", [F64, F32, BF16, F16])
@pytest.mark.parametrize("V", [1, 16, 18, 64, 65, 128, 129, 256, 257, 512, 513, 1023, 1500, 2048, 2050, 4095, 4097, 6001, 8191, 8193, 20011])
def test_sample_at_any_alignment(V, dtype):
    """Rows between NaNs and +inf, which would be drawn; nothing around the labels is written."""
    from tensornetworksfork_amd import _lib, ops
    dev = N._dev()
    lib, code, st = _lib.lib(), ops.ROW_TYPES[dtype], torch.cuda.current_stream(dev).cuda_stream
    g = torch.Generator().manual_seed(V)
    rows = 5
    for shift, ld in ((1, V), (2, V + 3), (3, V + 8)):
        z = (2.5 * torch.randn(rows, V, generator=g)).to(dtype)
        wide = torch.full((rows + 2, ld), float("inf"), dtype=dtype)
        wide.view(-1)[shift:shift + rows * ld].reshape(rows, ld)[:, :V] = z
        flat = wide.to(dev).view(-1)
        for c in S.CUTS:
            u = torch.rand(rows, generator=g)
            U = u.to(dev)
            label, ok = _guarded(rows, torch.int64, dev)
            need = lib.ttk_sample_ws_bytes(code, rows, V)
            ws, ws_ok = _guarded(max(need, 1), torch.uint8, dev, front=256)
            kw = S._kw(c)
            assert lib.ttk_sample(code, flat.data_ptr() + shift * z.element_size(), ld, U.data_ptr(), 0, None, kw["temperature"], None, kw["top_k"],
                                  None, kw["top_p"], None, kw["min_p"], label.data_ptr(), rows, V, ws.data_ptr() if need else None, need, st) == 0
            S._check(z, u, label.cpu(), c, least=0.4)
            assert ok() and ws_ok()


@gpu
@pytest.mark.parametrize("dtype,V", [(F64, 12001), (F32, 100003), (BF16, 131072), (F16, 9001), (F32, 6000)])
def test_top_k_of_every_size(dtype, V):
    """From one element to all but one: bounds by few groups, by many, and rows whose list would not hold them."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    g = torch.Generator().manual_seed(V)
    z = (2.0 * torch.randn(2, V, generator=g, dtype=F64)).to(dtype)
    Z = z.to(dev)
    for k in (1, 100, 170, 171, 341, 342, 776, 777, 1000, 1016, 1017, 2500, 2800, 3440, 3500, 5000, V // 2, V - 1):
        if k >= V:
            continue
        for c in (dict(k=k), dict(k=k, P=0.9, M=1e-4)):
            u = torch.rand(2, generator=g, dtype=F64)
            S._check(z, u, ops.sample(Z, u.to(dev), **S._kw(c)).cpu(), c, least=0.5)


@gpu
@pytest.mark.parametrize("dtype", [F64, F32, BF16])
def test_cuts_inside_thousands_of_equal_logits(dtype):
    """Whole-number weights: a cut that takes part of a run takes its lowest indices, whatever the run's length."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    V, run = 30011, 12000
    z = torch.full((3, V), -float("inf"), dtype=dtype)
    g = torch.Generator().manual_seed(0)
    at = torch.randperm(V, generator=g)[:run].sort().values
    z[0, at] = 1.0                                        # 12000 equal ones
    z[1, at] = 1.0
    z[1, at[5::7]] = 500.0                                # a seventh of them far above
    z[2] = 0.0                                            # all equal
    top = at[5::7]
    Z = z.to(dev)
    for uu in (0.0, 0.25, 0.5, 0.999):
        U = torch.full((3,), uu, dtype=F64, device=dev)
        for k in (9000, 11999, 3, 100):
            got = ops.sample(Z, U, top_k=k).cpu()
            assert int(got[0]) == int(at[int(uu * k)]) and int(got[2]) == int(uu * k)
            n = min(k, top.numel())
            # (at u = 0 the first kept element is drawn however little it weighs: e^-499 of the ones top-k keeps as well)
            assert int(got[1]) == int(at[0] if uu == 0 and k > n else top[int(uu * n)])
        for P in (0.5, 0.25, 0.75):
            got = ops.sample(Z, U, top_p=P).cpu()
            assert int(got[0]) == int(at[int(uu * (P * run))])
            assert int(got[2]) == int(uu * np.ceil(P * V))
            assert int(got[1]) == int(top[int(uu * np.ceil(P * top.numel()))])


@gpu
@pytest.mark.parametrize("V", [3000, 9001])
def test_more_rows_than_share_a_workspace(V):
    from tensornetworksfork_amd import ops
    dev = N._dev()
    g = torch.Generator().manual_seed(V)
    rows = 1100
    z = 2.0 * torch.randn(rows, V, generator=g)
    u = torch.rand(rows, generator=g)
    K = torch.tensor([0, 20, 900, 4000, 0], dtype=torch.int32).repeat(rows // 5)
    P = torch.tensor([0.9, 1.0, 0.8, 1.0, 1.0]).repeat(rows // 5)
    got = ops.sample(z.to(dev), u.to(dev), top_k=K.to(dev), top_p=P.to(dev)).cpu()
    at = torch.cat([torch.arange(0, 15), torch.arange(500, 530), torch.arange(1010, 1040), torch.arange(rows - 15, rows)])
    cuts = [dict(k=int(K[i]) if int(K[i]) < V else 0, P=float(P[i])) for i in at]
    S._check(z[at], u[at], got[at], cuts)


@gpu
@pytest.mark.parametrize("V", [12, 500, 3001, 20011])
def test_top_p_of_its_own_for_every_row_and_no_top_k(V):
    """Shares of zero and below keep one element, shares of one and above all, also where no top-k was asked for."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    g = torch.Generator().manual_seed(V)
    z = 2.0 * torch.randn(8, V, generator=g) - 40.0
    u = torch.rand(8, generator=g)
    P = torch.tensor([0.0, -1.0, 0.5, 1.0, 2.0, 0.9, float("nan"), 0.0])
    for _ in range(2):
        torch.full((1 << 22,), 255, dtype=torch.uint8, device=dev)      # (what a workspace may hold before the call)
        got = ops.sample(z.to(dev), u.to(dev), top_p=P.to(dev)).cpu()
        S._check(z, u, got, [dict(k=1) if float(p) <= 0 else dict(P=float(p)) if float(p) < 1 else dict() for p in P])


@gpu
@pytest.mark.parametrize("V", [40, 2000, 20011])
def test_extreme_temperatures_and_shares(V):
    """Flat and needle-like distributions, float64 rows whose logits span the whole range, shares next to 0 and 1."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    g = torch.Generator().manual_seed(V)
    z = torch.randn(6, V, generator=g, dtype=F64)
    z[1] *= 1e300
    z[2] *= 1e-300
    z[3] = torch.where(z[3] > 0, torch.tensor(1.7e308, dtype=F64), torch.tensor(-1.7e308, dtype=F64))      # (differences overflow)
    z[4] = torch.linspace(-1, 1, V, dtype=F64)
    for c in (dict(T=1e300), dict(T=1e-300), dict(T=1e300, P=0.3037), dict(T=1e9, k=V // 2, P=0.999), dict(T=3.0, P=1 - 1e-6), dict(P=1e-300),
              dict(T=50.0, M=0.9)):
        u = torch.rand(6, generator=g, dtype=F64)
        got = ops.sample(z.to(dev), u.to(dev), **S._kw(c)).cpu()
        # (0.999 of 1000 almost equal weights ends between two elements to within 1e-12: rows that the comparison leaves out)
        S._check(z, u, got, c, least=0.1 if c.get("k") else 0.5)


@gpu
@pytest.mark.parametrize("V,kw", [(40000, dict(top_p=0.95)), (40000, dict(temperature=0.0)), (40000, dict()), (9001, dict(top_k=3000, top_p=0.9)),
                                  (4000, dict(top_p=0.9)), (1500, dict(top_k=10, min_p=0.01))])
def test_graph_replays_of_every_path(V, kw):
    from tensornetworksfork_amd import ops
    dev = N._dev()
    g = torch.Generator(device=dev).manual_seed(1)
    z = torch.randn(7, V, generator=g, device=dev)
    u = torch.rand(7, generator=g, device=dev)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        ops.sample(z, u, **kw)
    torch.cuda.current_stream(dev).wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):                                    # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.sample(z, u, **kw))
        graphs.append(graph)
    for turn in range(4):
        u.uniform_(generator=g)
        z.normal_(generator=g)
        ref = ops.sample(z, u, **kw)
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[turn % 2], ref), turn
        graphs[1 - turn % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[1 - turn % 2], ref), turn


@gpu
def test_two_streams_at_once():
    """Calls on two streams, none waiting for the other, have workspaces of their own."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    g = torch.Generator(device=dev).manual_seed(3)
    z = [torch.randn(300, 30011, generator=g, device=dev) for _ in range(2)]
    u = torch.rand(300, generator=g, device=dev)
    x = [torch.randn(5000, 300, generator=g, device=dev) for _ in range(2)]
    w = torch.randn(300, generator=g, device=dev)

    def both(i):
        _, mean, rstd = ops.layer_norm(x[i], w, w)
        return (ops.sample(z[i], u, top_p=0.9), ops.sample(z[i], u, top_k=40), *ops.layer_norm_backward(x[1 - i], x[i], mean, rstd, w, 0.1, 5))
    ref = [both(0), both(1)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = [None, None]
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = both(i)
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(ref[i], got[i]):
                assert torch.equal(a, b)
