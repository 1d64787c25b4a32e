"""Layer norm, dropout and label sampling at the ends of what their entry points accept: rows of millions of columns and up to
2^31 - 1, sums over millions of rows, constant rows, columns behind a row, temperatures without bounds, weights far below the
largest, lists that hold just what top-k asks for."""
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


@gpu
@pytest.mark.parametrize("dtype,V,k,rows", [(F32, 131072, 300, 65), (F32, 100003, 1000, 70), (BF16, 131072, 300, 66), (F16, 50000, 700, 65),
                                            (F64, 20011, 300, 65), (F32, 131072, 300, 1)])
def test_top_k_alone_of_a_list_that_holds_just_as_many(dtype, V, k, rows):
    """k leaders in groups of their own over a background that weighs about as much: what top-k drops is never drawn."""
    from tensornetworksfork_amd import ops
    dev = S._dev()
    g = torch.Generator().manual_seed(V + k)
    z = torch.zeros(rows, V)
    at = torch.arange(k) * (V // k)
    z[:, at] = float(np.log(V / k))                       # (as much as the background together, before it is cut)
    z[rows // 2:, at] += 0.25 * torch.randint(0, 4, (rows - rows // 2, k), generator=g)
    z = z.to(dtype)
    Z, leaders = z.to(dev), set(at.tolist())
    K = torch.full((rows,), k, dtype=torch.int32)
    K[1::3] = k - 1
    K[2::3] = k + 1
    for top_k in (k, K.to(dev)):
        u = torch.rand(rows, generator=g, dtype=F64)
        got = ops.sample(Z, u.to(dev), top_k=top_k).cpu()
        if top_k is not K and isinstance(top_k, int):
            assert set(got.tolist()) <= leaders
        S._check(z, u, got, [dict(k=int(n)) for n in (K if top_k is not k else [k] * rows)], least=0.95)
    # min-p above the list's smallest weights, in the same draw
    u = torch.rand(rows, generator=g, dtype=F64)
    S._check(z, u, ops.sample(Z, u.to(dev), top_k=k, min_p=0.7).cpu(), dict(k=k, M=0.7), least=0.95)


@gpu
@pytest.mark.parametrize("dtype", [F64, F32, BF16])
@pytest.mark.parametrize("V", [3, 12, 40, 500, 3000, 8192, 8193, 40000])
def test_temperatures_without_bounds(V, dtype):
    """An infinite temperature makes every logit above -inf weigh the same, also where min-p asks for the largest weight; so does
    one so large that exp((z - m) / T) is 1 in 64 bits."""
    from tensornetworksfork_amd import ops
    dev = S._dev()
    MAX = np.finfo(np.float64).max                        # (what the oracle takes an infinite temperature for: -inf / inf is no number)
    g = torch.Generator().manual_seed(V)
    z = (2.0 * torch.randn(12, V, generator=g, dtype=F64)).to(dtype)
    z[3, ::2] = -float("inf")
    z[4] = -float("inf")
    z[5, V // 2] = float("inf")
    T = torch.full((12,), float("inf"), dtype=F64)
    T[6:9] = 1e300
    T[9] = 1.7e308
    T[10] = 1.0
    T[11] = 1e25
    u = torch.rand(12, generator=g, dtype=F64)
    for dt in (F64, F32):
        t = T.to(dt)                                      # (1e300 is infinite in float32)
        for P in (1.0, 0.30371):
            for M in (0.0, 0.5, 1.0):
                c = dict(temperature=t.to(dev), top_p=P, min_p=torch.full((12,), M, dtype=dt, device=dev))
                got = ops.sample(z.to(dev), u.to(dt).to(dev), **c).cpu()
                assert int(got[4]) == -1 and int(got[5]) == V // 2
                S._check(z, u.to(dt), got, [dict(T=min(float(x), MAX), P=P, M=M) for x in t], least=0.9)
        K = torch.full((12,), max(1, V // 3), dtype=torch.int32, device=dev)
        got = ops.sample(z.to(dev), u.to(dt).to(dev), temperature=t.to(dev), top_k=K, min_p=torch.ones(12, dtype=dt, device=dev)).cpu()
        S._check(z, u.to(dt), got, [dict(T=min(float(x), MAX), k=max(1, V // 3), M=1.0) for x in t], least=0.9)


@gpu
def test_column_sums_of_2_28_columns():
    """A launch counts its threads in 32 bits: the sum over the partials walks more columns than one launch of a thread each."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    cols = (1 << 28) + 8256
    x = ((torch.arange(1001, device=dev) % 13) - 6.0).repeat(cols // 1001 + 1)[:cols]
    dy = ((torch.arange(1003, device=dev) % 5) - 2.0).repeat(cols // 1003 + 1)[:cols]
    mean, rstd = torch.full((3,), 1.0, device=dev), torch.full((3,), 0.5, device=dev)
    _, dw, db = ops.layer_norm_backward(dy[None].expand(3, cols), x[None].expand(3, cols), mean, rstd, need=(False, True, True))
    assert torch.equal(db, 3 * dy) and torch.equal(dw, 3 * dy * (x - 1) * 0.5)
    del x, dy, dw, db
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("cols", [(1 << 30) + 8, (1 << 31) - 1])
def test_column_sums_of_rows_beyond_2_30_columns(cols):
    """One row broadcast to three: dw = 3 dy h, db = 3 dy, exact in float32 for these values (small whole numbers and halves)."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    reps = cols // 1001 + 1
    x = ((torch.arange(1001, device=dev) % 13) - 6.0).to(BF16).repeat(reps)[:cols]
    dy = ((torch.arange(1003, device=dev) % 5) - 2.0).to(BF16).repeat(reps)[:cols]
    mean = torch.full((3,), 1.0, device=dev)
    rstd = torch.full((3,), 0.5, device=dev)
    dx, dw, db = ops.layer_norm_backward(dy[None].expand(3, cols), x[None].expand(3, cols), mean, rstd, need=(False, True, True))
    assert dx is None
    step = 1 << 28
    for a in range(0, cols, step):
        g = dy[a:a + step].float()
        assert torch.equal(db[a:a + step].float(), 3 * g)
        # (bfloat16 holds 3 dy (x - 1) / 2 where it has at most 8 significant bits: |3 * 2 * 7 / 2| = 21 in steps of 1 / 2)
        assert torch.equal(dw[a:a + step].float(), 3 * g * (x[a:a + step].float() - 1) * 0.5)
    del x, dy, dw, db, g
    torch.cuda.empty_cache()


@gpu
def test_a_row_of_as_many_columns_as_are_accepted():
    """2^31 - 1 columns of +-1 and one 0: mean 0, rstd 1 to rounding; y = x, and dx = dy - x mean(dy x) for dy = x is 0."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    cols = (1 << 31) - 1
    x = torch.ones(cols, dtype=BF16, device=dev)
    x[::2] = -1
    x[cols // 2] = 0
    n = float(cols)
    s = -1.0 - float(1 - 2 * (1 - (cols // 2) % 2))       # (one -1 more than there are +1, and the one set to 0)
    y, mean, rstd = ops.layer_norm(x[None], eps=0.0)
    assert abs(float(mean) - s / n) <= 2 * R.U32 * abs(s / n) + 1e-12
    assert abs(float(rstd) - (n / (n - 1)) ** 0.5) <= 8 * R.U32
    step = 1 << 28
    for a in range(0, cols, step):
        assert torch.equal(y[0, a:a + step].float().round(), x[a:a + step].float())
    dx, dw, db = ops.layer_norm_backward(x[None], x[None], mean, rstd)
    for a in range(0, cols, step):
        # (x - 0 - x (1 - 1 / n) in float32, of which 1 / n is below half a step)
        assert float(dx[0, a:a + step].float().abs().max()) <= 16 * R.U32
        assert torch.equal(db[a:a + step], x[a:a + step])
        assert torch.equal(dw[a:a + step].float(), x[a:a + step].float().square())
    del x, y, dx, dw, db
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("V,rows", [(3, (1 << 32) + 70), (17, (1 << 26) + 5), (1000, (1 << 26) + 5), (1025, (1 << 25) + 3), (2049, (1 << 24) + 3),
                                    (4097, (1 << 23) + 3)])
def test_more_rows_than_a_launch_counts_threads_for(V, rows):
    """One row of equal logits broadcast to many: the label is floor(u V), exact in 64 bits; parameters of their own at the end."""
    from tensornetworksfork_amd import ops
    dev = S._dev()
    pattern = torch.rand(1000003, generator=torch.Generator().manual_seed(V)).to(dev)
    u = pattern.repeat(rows // pattern.numel() + 1)[:rows]
    Z = torch.full((1, V), 0.5, dtype=BF16, device=dev).expand(rows, V)
    if V == 3:
        got = ops.sample(Z, u)
    else:
        P = torch.ones(rows, device=dev)
        K = torch.zeros(rows, dtype=torch.int32, device=dev)
        P[-2], K[-1] = 0.5, 2
        got = ops.sample(Z, u, top_k=K, top_p=P)
        # the last two rows keep ceil(V / 2) elements and two
        for i, n in ((rows - 2, (V + 1) // 2), (rows - 1, 2)):
            assert int(got[i]) == int(np.floor(float(u[i]) * n))
        got, u = got[:-2], u[:-2]
    step = 1 << 28
    for a in range(0, got.numel(), step):
        assert torch.equal(got[a:a + step], (u[a:a + step].double() * V).floor().long())
    del got, u, Z
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("dtype,wdtype", N.TYPES)
@pytest.mark.parametrize("cols", [7, 24, 33, 48, 100, 333, 784, 1000, 1500, 2300, 5120, 6001, 10007, 16383, 20011])
def test_constant_rows_are_zero(cols, dtype, wdtype):
    """Rows of one whole number: their sums are exact (below 2^24), so the mean is the number itself and y is 0, whatever the
    layout; a constant gradient has no part that the norm passes on."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    values = [255.0, 1000.0, 3.0, -7.0] if cols < 16000 else [255.0, 3.0, -7.0, 11.0]
    x = torch.tensor(values, dtype=F64)[:, None].expand(4, cols).to(dtype).contiguous().to(dev)
    assert max(abs(float(v)) for v in x[:, 0]) * cols < 1 << 24
    w = torch.full((cols,), 3.0, dtype=wdtype, device=dev)
    for ww in (None, w):
        y, mean, rstd = ops.layer_norm(x, ww)
        assert bool((y == 0).all()) and torch.equal(mean, x[:, 0].to(mean.dtype))
        dy = torch.tensor([3.0, 255.0, -7.0, 1.0], dtype=F64)[:, None].expand(4, cols).to(dtype).contiguous().to(dev)
        dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, ww, wdtype=wdtype)
        assert bool((dx == 0).all()) and bool((dw == 0).all()) and bool((db == 252).all())


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [200003, 3000001])
def test_sums_of_millions_of_columns(cols, dtype):
    """Terms of one sign, of which a running float32 sum loses a part at every step."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    g = torch.Generator().manual_seed(cols)
    x = torch.full((3, cols), 1.0 / 3, dtype=F64)
    x[1] = 0.7 + 0.2 * torch.rand(cols, generator=g, dtype=F64)
    x[2] += torch.where(torch.arange(cols) % 2 == 0, 0.3, -0.1).to(F64)
    dy = torch.full((3, cols), 0.1, dtype=F64)
    dy[1] = 0.1 + 0.2 * torch.rand(cols, generator=g, dtype=F64)
    x, dy = x.to(dtype), dy.to(dtype)
    y, mean, rstd = ops.layer_norm(x.to(dev), eps=1e-5)
    N._check_forward(y, mean, rstd, x, None, None, 1e-5, dtype)
    N._check_backward(ops.layer_norm_backward(dy.to(dev), x.to(dev), mean, rstd), dy, x, mean, rstd, None, dtype, dtype)


@gpu
@pytest.mark.parametrize("dtype", [F64, F32, BF16])
@pytest.mark.parametrize("cols", [5, 33, 100, 129, 300, 784, 1001, 2300, 5000, 6001, 10007, 16383])
def test_what_stands_behind_a_row_stays_out_of_its_sums(cols, dtype):
    """Lanes behind the row's end hold 0, which lies -mean rstd (beyond the type's range here) from the mean."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    c, eps = (2.0 ** 1000, 1e-300) if dtype == F64 else (2.0 ** 80, 1e-36)
    g = torch.Generator().manual_seed(cols)
    x = torch.full((9, cols), c, dtype=dtype)
    dy = torch.randn(9, cols, generator=g, dtype=F64).to(dtype)
    w = (1 + 0.3 * torch.randn(cols, generator=g, dtype=F64)).to(dtype)
    y, mean, rstd = ops.layer_norm(x.to(dev), eps=eps)
    assert bool((y == 0).all()) and bool((mean.double() == c).all())
    for p in (0.0, 0.3):
        keep = R.keep_mask(x.numel(), p, 5, 3).reshape(x.shape)
        gm = torch.where(keep, dy.double() / (1 - p), torch.zeros_like(dy, dtype=F64))
        got = ops.layer_norm_backward(dy.to(dev), x.to(dev), mean, rstd, w.to(dev), p=p, seed=5, offset=3)
        assert bool((got[1] == 0).all())
        m, r = mean.cpu().double().unsqueeze(-1), rstd.cpu().double().unsqueeze(-1)
        dx, _, db, _, a = R.norm_backward(gm, x, m, r, w)
        with_max = dx.abs() <= torch.finfo(dtype).max
        u, D = R.unit(dtype), N._depth(cols)
        tol = r * u * (6 * a.abs() + (D + 6) * a.abs().mean(-1, keepdim=True))
        tol = tol + R.half_step(dtype) * (dx.abs() + tol) + R.tiny(dtype)
        assert bool((((got[0].cpu().double() - dx).abs() <= tol) | ~with_max).all())


@gpu
@pytest.mark.parametrize("dtype,cols,rows", [(F32, 4100, 1 << 22), (BF16, 9000, 1 << 21), (F32, 300, 1 << 24), (F16, 20, 1 << 26), (F32, 784, 1 << 23)])
def test_column_sums_of_millions_of_rows(dtype, cols, rows):
    """The same gradient in every row, of which a running float32 sum loses a part at every step (one row in memory, broadcast)."""
    from tensornetworksfork_amd import ops
    dev = N._dev()
    dy = torch.full((1, cols), 1.0 / 3, dtype=F64).to(dtype)
    x = torch.full((1, cols), 1.0, dtype=dtype)
    x[:, ::2] = -1.0
    X, DY = (t.to(dev).expand(rows, cols) for t in (x, dy))
    mean, rstd = torch.full((rows,), 0.25, device=dev), torch.full((rows,), 0.7, device=dev)
    dx, dw, db = ops.layer_norm_backward(DY, X, mean, rstd, need=(False, True, True), wdtype=F32 if dtype != F32 else None)
    g, h = dy[0].double(), (x[0].double() - 0.25) * float(torch.tensor(0.7))
    # 512 terms in a row in one lane, 16 across lanes and partials, 6 in a term; one rounding at the end
    tol = (512 + 16 + 6 + 1) * R.U32
    assert bool(((db.cpu().double() / rows - g).abs() <= tol * g.abs()).all())
    assert bool(((dw.cpu().double() / rows - g * h).abs() <= tol * (g * h).abs()).all())


@gpu
def test_top_p_where_the_tail_weighs_little_and_is_long():
    """One leader and 2^26 - 1 equal logits of 2^-37 of its weight, together 2^-11: the border of top-p lies among them."""
    from tensornetworksfork_amd import ops
    dev = S._dev()
    V = 1 << 26
    w = 2.0 ** -37
    z = torch.full((1, V), -37.0, dtype=BF16, device=dev)
    z[0, 12345] = 0.0
    T = float(1 / np.log(2.0))                            # weights 2^z, to a rounding of the exponent (37 2^-52)
    total = 1 + (V - 1) * w
    for P, u in ((1 - 2.0 ** -13, 0.99985), (0.99995, 1 - 2.0 ** -13), (0.9997, 0.9999)):
        target = P * total
        kept = int(np.ceil((target - 1) / w))             # elements of the tail
        assert kept > 1 << 20
        t = u * (1 + kept * w)
        got = int(ops.sample(z, torch.tensor([u], dtype=F64, device=dev), temperature=T, top_p=P)[0])
        # by index: 12345 of the tail, the leader, the rest of the tail
        want = 12345 + (t - 12345 * w - 1) / w + 1 if t > 12345 * w + 1 else 12345
        # one element for the whole numbers `kept` and the label each, one for the roundings: sums near 1 round at 2^-53, which is
        # 2^-16 of an element, some thousand times
        assert want > 12346 and abs(got - want) <= 3


@gpu
@pytest.mark.parametrize("V", [1 << 24, 20011])
def test_light_elements_of_a_list_keep_their_weights(V):
    """A leader and 899 (399) elements of 2^-38.5 of its weight, some 2^-29 of it together: u near 1 draws one of them."""
    from tensornetworksfork_amd import ops
    dev = S._dev()
    rows, k = 65, 900 if V > 1 << 20 else 400
    z = torch.full((1, V), -float("inf"))
    at = torch.arange(k) * (V // k)
    z[0, at] = -38.5 * float(np.log(2.0))
    z[0, 0] = 0.0
    w = float(np.exp(float(z[0, at[1]])))
    Z = z.to(dev).expand(rows, V)
    u = 1 - torch.linspace(0.1, 0.9, rows, dtype=F64) * (k - 1) * w
    got = ops.sample(Z, u.to(dev), top_k=k).cpu()
    t = u.numpy() * (1 + (k - 1) * w)
    want = 1 + np.floor((t - 1) / w)
    # a list's weights are multiples of 2^-48 of the largest, half a unit off at most: k 2^-49 / w = k 2^-10.5 elements; sums
    # near 1 round at 2^-53, a hundred of them are 2^-7 of an element
    assert np.all(np.abs(got.numpy() / (V // k) - want) <= k * 2.0 ** -10.5 + 1)


@gpu
@pytest.mark.parametrize("dtype", [F64, F32, BF16])
@pytest.mark.parametrize("V", [10, 60, 1000, 8192, 8193, 50000])
def test_the_first_kept_element_is_drawn_at_zero(V, dtype):
    """u = 0 draws the first kept element whose weight is above 0 in 64 bits, however little that is: on every path, down to the
    smallest numbers there are (2^-1074)."""
    from tensornetworksfork_amd import ops
    dev = S._dev()
    for depth in (10.0, 20.0, 45.0, 60.0, 500.0, 692.0, 700.0, 720.0, 738.0, 760.0):
        g = torch.Generator().manual_seed(V)
        z = torch.randn(67, V, generator=g, dtype=F64)
        z[:, 2:] += 5.0
        z[:, 0] = -900.0
        z[:, 1] = z[:, 2:].max(dim=1).values.to(dtype).double() - depth
        z = z.to(dtype)
        u = torch.zeros(67, dtype=F64, device=dev)
        first = 1 if depth < 744 else 2
        Z = z.to(dev)
        for kw in (dict(), dict(top_k=V - 1)) + ((dict(top_p=1 - 1e-12),) if depth < 11 else ()):
            assert bool((ops.sample(Z, u, **kw) == first).all()), (depth, kw)
        if V > 300:
            # a list of 300: its lightest element is the first by index
            y = torch.full_like(Z, -float("inf"))
            y[:, 1] = Z[:, 1]
            y[:, V - 299:] = Z[:, V - 299:]
            y[:, V - 1] = Z[:, 2:].max(dim=1).values
            for kw in (dict(top_k=300), dict(top_k=V // 2), dict(top_k=300, top_p=1 - 2.0 ** -53)):
                want = 1 if depth < 744 and (kw.get("top_p", 1.0) == 1.0 or depth < 35) else V - 299
                assert bool((ops.sample(y, u, **kw) == want).all()), (depth, kw)


@gpu
@pytest.mark.parametrize("V", [12, 40, 3000, 8193, 20011])
def test_differences_that_overflow_weigh_nothing(V):
    """float64 logits further apart than the largest number: (z - m) / T is -inf in 64 bits whatever T is."""
    from tensornetworksfork_amd import ops
    dev = S._dev()
    MAX = np.finfo(np.float64).max
    g = torch.Generator().manual_seed(V)
    z = torch.where(torch.rand(8, V, generator=g) > 0.5, 1.0, -1.0).to(F64) * 1.7e308
    z[1, 3] = -0.9e307                                    # (one that does not overflow)
    z[2] *= 0.5                                           # (none does)
    z[3] = -1.7e308
    z[3, V // 2] = 1.7e308
    Z = z.to(dev)
    for T in (1e305, 1e306, 1e307, 1.7e308, float("inf")):
        t = torch.full((8,), T, dtype=F64, device=dev)
        for c in (dict(), dict(P=0.30371), dict(k=max(2, V // 3)), dict(k=2, P=0.6), dict(M=0.25)):
            u = torch.rand(8, generator=g, dtype=F64)
            got = ops.sample(Z, u.to(dev), **{**S._kw(c), "temperature": t}).cpu()
            S._check(z, u, got, dict(c, T=min(T, MAX)), least=0.85)


@gpu
def test_layers_on_the_device_tell_what_has_a_gradient():
    """A float32 train has an input gradient (against differences of a multilinear function: exact but for rounding); a CPD
    network has none and says so; the values are those of an unrecorded pass either way."""
    from tensornetworksfork_amd.tensor.layers import CPDLayer, TensorTrainLayer
    dev = S._dev()
    layer = TensorTrainLayer(3, 4, 5, output_shape=2, seed=3, dtype=F32).to(dev)
    x = torch.randn(8, 5, generator=torch.Generator().manual_seed(2)).to(dev)
    xs = [x.clone().requires_grad_(True), x * 0.5, x + 1.0]
    y = layer(xs)
    with torch.no_grad():
        assert torch.equal(layer([t.detach() for t in xs]), y)
    dy = torch.linspace(-1, 1, y.numel(), dtype=y.dtype, device=dev).reshape(y.shape)
    got, = torch.autograd.grad(y, xs[0], dy)
    assert got.dtype == F32 and got.shape == x.shape
    # linear in each site's input: sum_j got[s, j] x[s, j] = sum_c dy[s, c] y[s, c]
    a, b = (got.double() * x.double()).sum(1), (dy.double() * y.detach().double()).sum(1)
    size = (got.double() * x.double()).abs().sum(1) + (dy.double() * y.detach().double()).abs().sum(1)
    # float64 arithmetic on float32 nodes, and the gradient rounded to float32: half a step a term
    assert bool(((a - b).abs() <= 4 * R.U32 * size).all())
    cpd = CPDLayer(3, 4, 5, output_shape=2, seed=1).to(dev)
    plain = cpd(x.double())
    with pytest.warns(UserWarning, match="gradient"):
        z = cpd(x.double().requires_grad_(True))
    assert not z.requires_grad and torch.equal(z, plain)


@gpu
@pytest.mark.parametrize("rows,cols", [((1 << 31) + 3, 20), (1 << 25, 5000), ((1 << 28) + 1, 300)])
def test_one_row_broadcast_to_more_than_memory_holds(rows, cols):
    """Whole numbers: every partial sum is exact however many rows a lane adds, and the workspace stays bounded."""
    from tensornetworksfork_amd import _lib, ops
    dev = N._dev()
    assert _lib.lib().ttk_layer_norm_backward_ws_bytes(1, rows, cols) <= 5 << 28
    x = (torch.arange(cols) % 3 - 1.0).to(dev)
    dy = (torch.arange(cols) % 2 + 1.0).to(dev)
    mean, rstd = torch.zeros(rows, device=dev), torch.ones(rows, device=dev)
    _, dw, db = ops.layer_norm_backward(dy.expand(rows, cols), x.expand(rows, cols), mean, rstd, need=(False, True, True))
    assert torch.equal(db.double(), (rows * dy.double()).float().double())
    assert torch.equal(dw.double(), (rows * (dy * x).double()).float().double())
    del mean, rstd
    torch.cuda.empty_cache()
