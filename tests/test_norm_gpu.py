"""Layer norm and dropout (csrc/ttk_norm.hip) against 64-bit restatements, at the sizes, strides, types and masks where
they can go wrong.  Tolerances count roundings: `u` is half a step of the arithmetic (2^-24, float64 rows 2^-53), the last
rounding to the element type is half a step of that type."""
import itertools

import pytest
import torch

from tests import _row_oracles as R

gpu = pytest.mark.gpu
F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16
TYPES = [(F64, F64), (F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)]
# one column and one row; both sides of every row length at which the kernels change their layout; odd ones between
SHAPES = [(1, 1), (3, 1), (1, 2), (5, 3), (70, 7), (1000, 8), (129, 16), (260, 17), (513, 31), (64, 32), (65, 33), (1, 64),
          (300, 65), (33, 128), (9, 129), (40, 255), (7, 257), (1, 512), (21, 784), (6, 1025), (5, 2048), (3, 2049), (2, 4097),
          (19, 5120), (3, 8193), (700, 10007), (2, 16384), (2, 16385), (1, 32769), (3, 70001)]


@pytest.fixture(autouse=True)
def _float32_default():
    """Other tests of the process may have left float64 as torch's default."""
    old = torch.get_default_dtype()
    torch.set_default_dtype(F32)
    yield
    torch.set_default_dtype(old)


def _dev():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    return torch.device("cuda:0")


def _make(rows, cols, dtype, wdtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g, dtype=F64) * 1.5 + 0.5 * torch.randn(rows, 1, generator=g, dtype=F64)).to(dtype)
    dy = torch.randn(rows, cols, generator=g, dtype=F64).to(dtype)
    w = (1 + 0.3 * torch.randn(cols, generator=g, dtype=F64)).to(wdtype)
    b = (0.2 * torch.randn(cols, generator=g, dtype=F64)).to(wdtype)
    return x, dy, w, b


def _depth(n):
    """Additions a term of a sum of n values can pass through: at most 80 in a row in one lane (longer rows are split over
    more lanes), 16 across the lanes and waves."""
    return min(n, 80) + 16


def _check_forward(y, mean, rstd, x, w, b, eps, dtype, scale=1.0, keep=None):
    ry, rmean, rrstd, h = R.norm_forward(x, w, b, eps)
    u, D = R.unit(dtype), _depth(x.shape[-1])
    xa = x.double().abs().mean(dim=-1, keepdim=True)
    dmean = (D + 2) * u * xa                                  # the mean's error
    # rstd: the sum of squares (D + 4 roundings), the mean's error (second order), the square root and the quotient
    drel = (D + 8) * u + (dmean * rrstd) ** 2
    assert bool(((mean.cpu().double().unsqueeze(-1) - rmean).abs() <= dmean + R.tiny(mean.dtype)).all())
    assert bool(((rstd.cpu().double().unsqueeze(-1) - rrstd).abs() <= drel * rrstd + R.tiny(rstd.dtype)).all())
    wa = torch.ones_like(h) if w is None else w.double().abs()
    tol = h.abs() * wa * (drel + 4 * u) + dmean * rrstd * wa + 2 * u * ry.abs()
    if keep is not None:
        ry, tol = torch.where(keep, ry * scale, torch.zeros_like(ry)), torch.where(keep, (tol + 2 * u * ry.abs()) * scale,
                                                                                     torch.zeros_like(ry))
    tol = tol + R.half_step(dtype) * (ry.abs() + tol) + R.tiny(dtype)
    if keep is not None:
        assert bool((y.cpu()[~keep] == 0).all())
    err = (y.cpu().double() - ry).abs()
    assert bool((err <= tol).all()), (err - tol).max()


def _check_backward(got, dy, x, mean, rstd, w, dtype, wdtype):
    """dy: the gradient behind the mask (what the oracle sums), as exact 64-bit values."""
    dx, dw, db = got
    m, r = mean.cpu().double().unsqueeze(-1), rstd.cpu().double().unsqueeze(-1)
    rdx, rdw, rdb, h, a = R.norm_backward(dy, x, m, r, w)
    u, D = R.unit(dtype), _depth(x.shape[-1])
    # h: subtraction, product (2 roundings); a: mask and product (2); the two means: D and D + 4 roundings of their terms
    c1, c2 = a.abs().mean(-1, keepdim=True), (a * h).abs().mean(-1, keepdim=True)
    tol = r * u * (6 * a.abs() + (D + 6) * c1 + h.abs() * (D + 14) * c2)
    if dx is not None:
        t = tol + R.half_step(dtype) * (rdx.abs() + tol) + R.tiny(dtype)
        err = (dx.cpu().double() - rdx).abs()
        assert bool((err <= t).all()), (err - t).max()
    # column sums: at most 512 terms in a row in one lane, 16 across lanes and partials, 64-bit sums of the partials
    rows = x.numel() // x.shape[-1]
    lead = tuple(range(x.ndim - 1))
    C = min(rows, 512) + 16
    g = dy.double()
    for out, ref, mag in ((dw, rdw, (g * h).abs().sum(lead)), (db, rdb, g.abs().sum(lead))):
        if out is not None:
            t = u * (C + 6) * mag
            t = t + R.half_step(wdtype) * (ref.abs() + t) + R.tiny(wdtype)
            err = (out.cpu().double() - ref).abs()
            assert bool((err <= t).all()), (err - t).max()


@gpu
@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layer_norm(rows, cols, dtype, wdtype):
    from tensornetworksfork_amd import ops
    dev = _dev()
    x, dy, w, b = _make(rows, cols, dtype, wdtype, 11)
    X, DY, W, B = x.to(dev), dy.to(dev), w.to(dev), b.to(dev)
    y, mean, rstd = ops.layer_norm(X, W, B, 1e-5)
    assert y.dtype == dtype and mean.dtype == (F64 if dtype == F64 else F32)
    _check_forward(y, mean, rstd, x, w, b, 1e-5, dtype)
    _check_backward(ops.layer_norm_backward(DY, X, mean, rstd, W), dy, x, mean, rstd, w, dtype, wdtype)
    # with dropout as the epilogue: the same mask forwards and backwards, from an odd element on
    p, seed, off = 0.3, (5 << 33) + 7, 4099
    keep = R.keep_mask(rows * cols, p, seed, off).reshape(rows, cols)
    y, mean, rstd = ops.layer_norm(X, W, B, 1e-5, p=p, seed=seed, offset=off)
    _check_forward(y, mean, rstd, x, w, b, 1e-5, dtype, scale=1 / (1 - p), keep=keep)
    g = torch.where(keep, dy.double() / (1 - p), torch.zeros_like(dy, dtype=F64))
    _check_backward(ops.layer_norm_backward(DY, X, mean, rstd, W, p=p, seed=seed, offset=off), g, x, mean, rstd, w, dtype, wdtype)


@gpu
@pytest.mark.parametrize("rows,cols", [(40, 6), (33, 17), (25, 130), (11, 1000), (5, 4099), (3, 70000)])
@pytest.mark.parametrize("dtype", [F64, F32, BF16])
def test_weights_absent_and_gradients_not_wanted(rows, cols, dtype):
    from tensornetworksfork_amd import ops
    dev = _dev()
    x, dy, w, b = _make(rows, cols, dtype, dtype, 3)
    X, DY = x.to(dev), dy.to(dev)
    for ww, bb in ((None, None), (w, None), (None, b)):
        W, B = (None if t is None else t.to(dev) for t in (ww, bb))
        y, mean, rstd = ops.layer_norm(X, W, B, 1e-3)
        _check_forward(y, mean, rstd, x, ww, bb, 1e-3, dtype)
        for need in itertools.product((True, False), repeat=3):
            got = ops.layer_norm_backward(DY, X, mean, rstd, W, need=need)
            assert [t is not None for t in got] == list(need)
            _check_backward(got, dy, x, mean, rstd, ww, dtype, dtype)


@gpu
@pytest.mark.parametrize("cols", [5, 17, 40, 600, 3000])
@pytest.mark.parametrize("dtype", [F64, F32, F16])
def test_row_distances(cols, dtype):
    """Column ranges of wider matrices (with and without a shifted start), one row broadcast to many, three axes."""
    from tensornetworksfork_amd import ops
    dev = _dev()
    rows = 37
    wide, dwide, w, b = _make(rows, cols + 11, dtype, dtype, 8)
    w, b = w[:cols].contiguous(), b[:cols].contiguous()
    Wd, DWd, W, B = wide.to(dev), dwide.to(dev), w.to(dev), b.to(dev)
    for s in (0, 3):
        X, DY = Wd[:, s:s + cols], DWd[:, s + 1:s + 1 + cols]
        y, mean, rstd = ops.layer_norm(X, W, B)
        assert y.is_contiguous()
        _check_forward(y, mean, rstd, wide[:, s:s + cols], w, b, 1e-5, dtype)
        _check_backward(ops.layer_norm_backward(DY, X, mean, rstd, W), dwide[:, s + 1:s + 1 + cols], wide[:, s:s + cols], mean,
                        rstd, w, dtype, dtype)
    one = Wd[:1, :cols].expand(rows, cols)
    y, mean, rstd = ops.layer_norm(one, W, B)
    _check_forward(y, mean, rstd, wide[:1, :cols].expand(rows, cols), w, b, 1e-5, dtype)
    _check_backward(ops.layer_norm_backward(DWd[:, :cols], one, mean, rstd, W), dwide[:, :cols],
                    wide[:1, :cols].expand(rows, cols), mean, rstd, w, dtype, dtype)
    x3 = wide[:36, :cols].contiguous().reshape(4, 9, cols)
    y, mean, rstd = ops.layer_norm(x3.to(dev), W, B)
    assert y.shape == x3.shape and mean.shape == (4, 9)
    _check_forward(y, mean, rstd, x3, w, b, 1e-5, dtype)


@gpu
@pytest.mark.parametrize("cols", [4, 17, 100, 2000])
def test_rows_that_are_not_numbers_stay_by_themselves(cols):
    """NaN and infinities spoil their own row and, through the column sums, every dw they enter; nothing else."""
    from tensornetworksfork_amd import ops
    dev = _dev()
    x, dy, w, b = _make(130, cols, F32, F32, 21)
    x[3, 1] = float("nan")
    x[77, 0] = float("inf")
    x[78] = 2.5                                    # a constant row: variance 0
    ok = torch.ones(130, dtype=torch.bool)
    ok[3] = ok[77] = False
    X, DY, W, B = x.to(dev), dy.to(dev), w.to(dev), b.to(dev)
    y, mean, rstd = ops.layer_norm(X, W, B)
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[77]).all())
    _check_forward(y.cpu()[ok], mean.cpu()[ok], rstd.cpu()[ok], x[ok], w, b, 1e-5, F32)
    dx, dw, db = ops.layer_norm_backward(DY, X, mean, rstd, W)
    assert bool(torch.isnan(dw).all()) and bool(torch.isfinite(db).all())
    _check_backward((dx.cpu()[ok], None, None), dy[ok], x[ok], mean.cpu()[ok], rstd.cpu()[ok], w, F32, F32)


@gpu
def test_whole_numbers_come_out_exactly():
    """Rows of +-1 with mean 0 and eps 0: mean 0, rstd 1, y = x w + b and the column sums are whole numbers."""
    from tensornetworksfork_amd import ops
    dev = _dev()
    for cols in (2, 16, 64, 1024, 8192):
        x = torch.ones(301, cols)
        x[:, ::2] = -1
        y, mean, rstd = ops.layer_norm(x.to(dev), eps=0.0)
        assert torch.equal(y.cpu(), x) and bool((mean == 0).all()) and bool((rstd == 1).all())
        dx, dw, db = ops.layer_norm_backward(torch.ones_like(x).to(dev), x.to(dev), mean, rstd)
        assert torch.equal(dw.cpu(), 301 * x[0]) and bool((db == 301).all()) and bool((dx == 0).all())


@gpu
@pytest.mark.parametrize("dtype", [F64, F32, BF16, F16])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 63, 1000, 2049, 100003])
def test_dropout(n, dtype):
    from tensornetworksfork_amd import ops
    dev = _dev()
    g = torch.Generator().manual_seed(n)
    base = torch.randn(n + 1, generator=g, dtype=F64).to(dtype)
    for p, seed, off in ((0.0, 1, 0), (0.25, 0, 0), (0.5, (1 << 64) - 1, 1), (0.9, 12345, (1 << 34) - 2), (0.1, 3, (1 << 62) + 3),
                         (1e-9, 3, 7), (1 - 1e-12, 3, 7), (1.0, 3, 0)):
        for x in (base[:n], base[1:]):             # (the second starts off any vector's alignment)
            y = ops.dropout(base.to(dev)[:n] if x.data_ptr() == base.data_ptr() else base.to(dev)[1:], p, seed, off)
            ref = R.dropout(x, p, seed, off)
            assert torch.equal(y.cpu() == 0, (ref == 0) | (ref.abs() < R.tiny(dtype))), (n, p)
            u = R.unit(dtype)
            with_max = ref.abs() <= torch.finfo(dtype).max
            err = (y.cpu().double() - ref).abs()[with_max]
            tol = (2 * u + R.half_step(dtype)) * 1.001 * ref.abs()[with_max] + R.tiny(dtype)
            assert bool((err <= tol).all())


@gpu
def test_dropout_mask_is_a_function_of_seed_and_element():
    """A shard draws its part of the whole set's mask; the fraction kept is 1 - p; other seeds draw other masks; what is
    dropped is 0 whatever it held."""
    from tensornetworksfork_amd import ops
    dev = _dev()
    n = 1 << 20
    x = torch.ones(n, device=dev)
    whole = ops.dropout(x, 0.3, 9, 0)
    for a, b in ((0, 7), (7, 1001), (1001, n)):
        assert torch.equal(ops.dropout(x[a:b].contiguous(), 0.3, 9, a), whole[a:b])
    kept = float((whole != 0).double().mean())
    assert abs(kept - 0.7) < 6 * (0.21 / n) ** 0.5            # six standard deviations of n draws
    assert 0.3 < float(((ops.dropout(x, 0.3, 10, 0) != 0) == (whole != 0)).double().mean()) < 0.7
    bad = torch.where(whole == 0, torch.full_like(x, float("nan")), x)
    assert torch.equal(ops.dropout(bad, 0.3, 9, 0), whole)
    # the epilogue of the norm draws the same mask
    y, _, _ = ops.layer_norm(torch.randn(1 << 10, 1 << 10, device=dev), bias=torch.full((1 << 10,), 100.0, device=dev), p=0.3, seed=9)
    assert torch.equal(y.reshape(-1) != 0, whole != 0)


@gpu
def test_empty_rows_and_one_element():
    from tensornetworksfork_amd import ops
    dev = _dev()
    x = torch.zeros(0, 5, device=dev)
    y, mean, rstd = ops.layer_norm(x)
    assert y.shape == (0, 5) and mean.shape == (0,)
    dx, dw, db = ops.layer_norm_backward(x, x, mean, rstd)
    assert dx.shape == (0, 5) and bool((dw == 0).all()) and bool((db == 0).all())
    assert ops.dropout(torch.zeros(0, device=dev), 0.5, 1).numel() == 0
    y, mean, rstd = ops.layer_norm(torch.tensor([4.0], device=dev))
    assert mean.shape == () and float(y) == 0.0 and float(mean) == 4.0


@gpu
@pytest.mark.parametrize("p", [0.0, 0.4])
@pytest.mark.parametrize("cols", [6, 40, 1030])
def test_gradients_against_differences(p, cols):
    """float64 gradients of sum(y v) through autograd against central differences (error ~ h^2 |f'''| / 6 + 2^-53 |f| / h:
    h = 1e-5, relative to gradients of order 1)."""
    from tensornetworksfork_amd.tensor.norm import dropout, layer_norm
    dev = _dev()
    x, v, w, b = (t.to(dev) for t in _make(3, cols, F64, F64, 5))

    def f(x, w, b):
        return (layer_norm(x, w, b, p=p, seed=4, offset=3) * v).sum() + (dropout(x, p, 5) * v).sum()
    args = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(f(*args), args)
    h = 1e-5
    for i, t in enumerate((x, w, b)):
        flat = t.reshape(-1)
        for j in list(range(0, flat.numel(), max(1, flat.numel() // 7))):
            old = flat[j].item()
            vals = []
            for s in (h, -h):
                flat[j] = old + s
                vals.append(float(f(x, w, b)))
            flat[j] = old
            num = (vals[0] - vals[1]) / (2 * h)
            assert abs(num - float(grads[i].reshape(-1)[j])) < 1e-6 * max(1.0, abs(num)), (i, j)


@gpu
def test_autograd_of_broadcast_and_strided_inputs():
    from tensornetworksfork_amd.tensor.norm import LayerNorm, layer_norm
    dev = _dev()
    x, dy, w, b = (t.to(dev) for t in _make(40, 24, F32, F32, 2))
    row = x[:1].clone().requires_grad_(True)
    wd = w.clone().requires_grad_(True)
    y = layer_norm(row.expand(40, 24), wd, b)
    gr, gw = torch.autograd.grad(y, (row, wd), dy)
    _, mean, rstd, _ = R.norm_forward(x[:1].cpu().expand(40, 24))
    rdx, rdw, _, _, _ = R.norm_backward(dy.cpu(), x[:1].cpu().expand(40, 24), mean, rstd, w.cpu())
    assert (gr.cpu().double() - rdx.sum(0, keepdim=True)).abs().max() < 1e-4      # 40 float32 gradients of order 1 to 10
    assert (gw.cpu().double() - rdw).abs().max() < 1e-4
    # a transposed input is copied, a gradient broadcast from a sum too
    xt = x.t().contiguous().t().requires_grad_(True)
    g1, = torch.autograd.grad(layer_norm(xt, w, b).sum(), xt)
    xc = x.clone().requires_grad_(True)
    g2, = torch.autograd.grad(layer_norm(xc, w, b), xc, torch.ones_like(x))
    assert torch.equal(g1, g2)
    # the module: parameters get gradients, evaluation drops nothing, every training pass draws new elements
    ln = LayerNorm(24, p=0.5, seed=3, device=dev)
    a1, a2 = ln(x), ln(x)
    assert not torch.equal(a1 == 0, a2 == 0) and ln.offset == 2 * x.numel()
    a1.sum().backward()
    assert ln.weight.grad is not None and ln.bias.grad is not None
    ln.eval()
    assert bool((ln(x) != 0).all()) and ln.offset == 2 * x.numel()
    # gradients of gradients are refused
    xg = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(layer_norm(xg, w, b).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@gpu
def test_other_streams_and_repeated_calls_give_the_same_bits():
    from tensornetworksfork_amd import ops
    dev = _dev()
    x, dy, w, b = (t.to(dev) for t in _make(3000, 333, BF16, F32, 6))
    first = None
    streams = [torch.cuda.current_stream(dev)] + [torch.cuda.Stream(dev) for _ in range(2)]
    for s in streams * 2:
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            y, mean, rstd = ops.layer_norm(x, w, b, p=0.2, seed=1)
            out = (y, mean, rstd) + ops.layer_norm_backward(dy, x, mean, rstd, w, p=0.2, seed=1)
        torch.cuda.synchronize()
        if first is None:
            first = out
        assert all(torch.equal(a, c) for a, c in zip(first, out))


@gpu
def test_graph_replays_follow_the_offset_tensor():
    """Forward and backward captured once: every replay equals the eager calls at the offset the device holds then."""
    from tensornetworksfork_amd import ops
    dev = _dev()
    x, dy, w, b = (t.to(dev) for t in _make(200, 50, F32, F32, 6))
    off = torch.zeros(1, dtype=torch.int64, device=dev)

    def step():
        y, mean, rstd = ops.layer_norm(x, w, b, p=0.3, seed=2, offset=off)
        return (y,) + ops.layer_norm_backward(dy, x, mean, rstd, w, p=0.3, seed=2, offset=off) + (ops.dropout(x, 0.3, 2, off),)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream(dev).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        off.fill_(10007 * turn)
        x.mul_(1.0 + 0.01 * turn)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        y, mean, rstd = ops.layer_norm(x, w, b, p=0.3, seed=2, offset=10007 * turn)
        ref = (y,) + ops.layer_norm_backward(dy, x, mean, rstd, w, p=0.3, seed=2, offset=10007 * turn) \
            + (ops.dropout(x, 0.3, 2, 10007 * turn),)
        assert all(torch.equal(a, c) for a, c in zip(got, ref)), turn


@gpu
def test_refusals_on_the_device():
    from tensornetworksfork_amd import _lib, ops
    from tensornetworksfork_amd.tensor.norm import LayerNorm
    dev = _dev()
    x = torch.zeros(4, 6, device=dev)
    _, mean, rstd = ops.layer_norm(x)
    bad = [lambda: ops.layer_norm(x, torch.ones(5, device=dev)), lambda: ops.layer_norm(x, torch.ones(6, device=dev, dtype=F64)),
           lambda: ops.layer_norm(x, torch.ones(6)), lambda: ops.layer_norm(x.t()), lambda: ops.layer_norm(x.int()),
           lambda: ops.layer_norm(x.bfloat16(), torch.ones(6, device=dev), torch.ones(6, device=dev).bfloat16()),
           lambda: ops.layer_norm(x, eps=-1.0), lambda: ops.layer_norm(x, eps=float("nan")),
           lambda: ops.layer_norm(x, p=1.5), lambda: ops.layer_norm(x, p=0.5, offset=torch.zeros(2, dtype=torch.int64, device=dev)),
           lambda: ops.layer_norm(x[:, :0]), lambda: ops.layer_norm(x[0, 0]),
           lambda: ops.layer_norm(torch.zeros(2, 3, 4, device=dev).transpose(0, 1)),
           lambda: ops.layer_norm_backward(x.double(), x, mean, rstd), lambda: ops.layer_norm_backward(x[:2], x, mean, rstd),
           lambda: ops.layer_norm_backward(x, x, mean[:2], rstd), lambda: ops.layer_norm_backward(x, x, mean.double(), rstd),
           lambda: ops.layer_norm_backward(x, x, mean, rstd, wdtype=F64),
           lambda: ops.dropout(x.t(), 0.5, 1), lambda: ops.dropout(x, float("nan"), 1), lambda: ops.dropout(x, 0.5, -1),
           lambda: ops.dropout(x, 0.5, 1 << 64), lambda: ops.dropout(x, 0.5, 1, -4), lambda: ops.dropout(x.int(), 0.5, 1),
           lambda: LayerNorm(5).to(dev)(x)]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.TTKError):
            f()
            raise AssertionError(i)
    # one byte of workspace short: refused before anything is written
    lib = _lib.lib()
    n = int(lib.ttk_layer_norm_backward_ws_bytes(1, 4, 6))
    ws = torch.full((n,), 7, dtype=torch.uint8, device=dev)
    dw = torch.full((6,), 5.0, device=dev)
    rc = lib.ttk_layer_norm_backward(1, 1, x.data_ptr(), 6, x.data_ptr(), 6, None, mean.data_ptr(), rstd.data_ptr(), None,
                                     dw.data_ptr(), None, 4, 6, 0.0, 0, 0, None, ws.data_ptr(), n - 1, None)
    torch.cuda.synchronize()
    assert rc == -2 and bool((ws == 7).all()) and bool((dw == 5).all())
