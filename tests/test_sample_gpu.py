"""Label sampling (csrc/ttk_sample.hip) against a 64-bit restatement.  Labels are compared for equality; a row whose
decisions lie closer to a border than the roundings of the sums they compare (MARGIN, relative: 2^20 terms of 2^-53, the
weights rounded to 2^-42 of the largest at worst) is left out, which random rows hardly ever are."""
import numpy as np
import pytest
import torch

from tests import _row_oracles as R

gpu = pytest.mark.gpu
F64, F32, BF16, F16 = torch.float64, torch.float32, torch.bfloat16, torch.float16
MARGIN = 1e-9
# both sides of every row length at which the kernels change, and odd ones
SIZES = [1, 2, 3, 10, 15, 16, 17, 63, 64, 65, 100, 255, 1000, 1024, 1025, 2049, 5003, 8192, 30011, 65536, 100003]
CUTS = [dict(), dict(T=0.6), dict(k=1), dict(k=7), dict(P=0.9), dict(P=0.2, T=1.7), dict(M=0.05), dict(k=50, P=0.8, M=0.01),
        dict(k=1000, T=2.5), dict(T=0.0), dict(P=1e-12), dict(k=600, P=0.97, T=1.3), dict(M=1.0), dict(P=0.999, T=0.2)]


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


def _kw(c):
    return dict(temperature=c.get("T", 1.0), top_k=c.get("k", 0), top_p=c.get("P", 1.0), min_p=c.get("M", 0.0))


def _check(z, u, got, cuts, least=0.9):
    """cuts: one dict for all rows or one a row"""
    z64, u64 = z.double().cpu().numpy(), u.double().cpu().numpy()
    rows = z64.shape[0]
    compared = 0
    for i in range(rows):
        c = cuts if isinstance(cuts, dict) else cuts[i]
        ref, margin = R.sample_row(z64[i], float(u64[i]), **c)
        if margin < MARGIN:
            continue
        compared += 1
        assert int(got[i]) == ref, (i, c, int(got[i]), ref, margin)
    assert compared >= least * rows, (compared, rows)


@gpu
@pytest.mark.parametrize("dtype", [F64, F32, BF16, F16])
@pytest.mark.parametrize("V", SIZES)
def test_sample(V, dtype):
    from tensornetworksfork_amd import ops
    dev = _dev()
    rows = 3 if V > 20000 else 9
    g = torch.Generator().manual_seed(V)
    z = (2.5 * torch.randn(rows, V, generator=g, dtype=F64)).to(dtype)
    for n, c in enumerate(CUTS):
        u = torch.rand(rows, generator=g, dtype=F64 if n % 2 else F32)
        got = ops.sample(z.to(dev), u.to(dev), **_kw(c)).cpu()
        assert got.dtype == torch.int64
        _check(z, u, got, c, least=0.5)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [10, 33, 700, 4096, 40000])
def test_ties_go_to_the_lowest_index(V, dtype):
    """Few distinct logits: cuts fall inside runs of equal elements, and every weight is a power of two (exact sums)."""
    from tensornetworksfork_amd import ops
    dev = _dev()
    g = torch.Generator().manual_seed(V)
    z = torch.randint(0, 3, (6, V), generator=g).to(dtype)
    z[0] = 0.25                                           # all equal
    z[1, :] = -1.0
    z[1, V // 2] = 3.0
    z[2] = torch.where(z[2] > 1, torch.zeros(()), -0.0).to(dtype)      # +0 and -0 are equal
    # temperature 1 / ln 2: weights 2^(z - m) up to a rounding of the exponent
    for k, P in ((0, 1.0), (1, 1.0), (3, 1.0), (V // 2 + 1, 1.0), (0, 0.5), (0, 0.75), (V // 3 + 1, 0.5), (2, 0.6)):
        for uu in (0.0, 0.25, 0.499, 0.75, 0.999):
            u = torch.full((6,), uu, dtype=F64)
            got = ops.sample(z.to(dev), u.to(dev), top_k=k, top_p=P).cpu()
            _check(z, u, got, dict(k=k, P=P), least=0.3)
    # all equal, arithmetic exact: the first ceil(P k) elements are kept, the draw is floor(u n)
    for k, P, uu in ((0, 0.5, 0.5), (0, 0.25, 0.0), (8, 0.5, 0.75), (0, 1.0, 0.5)):
        n = V if k == 0 else min(k, V)
        n = int(np.ceil(P * n))
        got = ops.sample(z[:1].to(dev), torch.tensor([uu], dtype=F64, device=dev), top_k=k, top_p=P)
        assert int(got[0]) == int(np.floor(uu * n))


@gpu
@pytest.mark.parametrize("V", [5, 16, 40, 1000, 3000, 70000])
def test_masked_and_infinite_logits(V):
    from tensornetworksfork_amd import ops
    dev = _dev()
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(F32).min
    g = torch.Generator().manual_seed(V)
    z = torch.randn(10, V, generator=g)
    z[0] = -inf                                           # nothing left
    z[1] = nan
    z[2] = -inf
    z[2, V - 1] = -3.0                                    # one element left, the last
    z[3] = low                                            # masked by the lowest value: all equal
    z[4] = low
    z[4, 2] = 0.0
    z[5, 1] = inf                                         # +inf takes all
    z[5, V - 1] = inf
    z[6, ::2] = -inf                                      # half masked
    z[7, 1::2] = nan
    z[8] = torch.where(torch.arange(V) < 3, torch.tensor(5.0), torch.tensor(-inf))
    for dtype in (F64, F32, BF16, F16):
        zd = z.to(dtype)
        for c in (dict(), dict(k=4), dict(P=0.7), dict(k=3, P=0.5, M=0.1), dict(M=0.3), dict(T=0.0), dict(k=V), dict(T=1e-30), dict(P=0.999999)):
            for uu in (0.0, 0.3, 0.62, 0.999):
                u = torch.full((10,), uu, dtype=F64)
                got = ops.sample(zd.to(dev), u.to(dev), **_kw(c)).cpu()
                assert int(got[0]) == -1 and int(got[1]) == -1
                assert int(got[2]) == V - 1
                assert int(got[5]) in (1, V - 1)
                _check(zd, u, got, c, least=0.5)


@gpu
def test_random_numbers_at_the_ends():
    from tensornetworksfork_amd import ops
    dev = _dev()
    for V in (3, 50, 5000, 60000):
        g = torch.Generator().manual_seed(V)
        z = torch.randn(8, V, generator=g, dtype=F64)
        z[:, 0] = -float("inf")
        z[1] -= 600.0 * torch.rand(V, generator=g, dtype=F64)
        u = torch.tensor([0.0, 0.0, 1.0, 1.5, -1.0, float("nan"), 1 - 2.0 ** -53, 2.0 ** -60], dtype=F64)
        for c in (dict(), dict(k=5), dict(P=0.5), dict(M=0.2)):
            got = ops.sample(z.to(dev), u.to(dev), **_kw(c)).cpu()
            for i in range(8):
                uu = float(u[i])
                uu = 0.0 if not uu > 0 else uu
                ref, margin = R.sample_row(z[i].numpy(), uu, **c)
                if 0 < uu < 1 - 1e-9 and margin < MARGIN:
                    continue
                assert int(got[i]) == ref, (V, i, c)


@gpu
@pytest.mark.parametrize("V", [12, 300, 20000])
def test_parameters_of_their_own_for_every_row(V):
    from tensornetworksfork_amd import ops
    dev = _dev()
    rows = 64
    g = torch.Generator().manual_seed(V)
    z = 2.0 * torch.randn(rows, V, generator=g)
    for dt in (F32, F64):
        T = torch.tensor([0.0, 0.7, 1.0, -1.0, 2.0, float("nan"), 0.3, 1.0]).repeat(rows // 8).to(dt)
        K = torch.tensor([0, 1, 5, -2, 40, 0, V, 1 << 30], dtype=torch.int32).repeat(rows // 8).flip(0)
        P = torch.tensor([1.0, 0.9, 0.5, 2.0, 0.0, -1.0, float("nan"), 0.99]).repeat_interleave(rows // 8).to(dt)
        M = torch.tensor([0.0, 0.1, 2.0, -1.0, float("nan"), 0.01, 0.0, 0.0]).repeat_interleave(rows // 8).flip(0).to(dt)
        u = torch.rand(rows, generator=g, dtype=dt)
        got = ops.sample(z.to(dev), u.to(dev), T.to(dev), K.to(dev), P.to(dev), M.to(dev)).cpu()
        cuts = []
        for i in range(rows):
            t, k, p, m = float(T[i]), int(K[i]), float(P[i]), float(M[i])
            cuts.append(dict(T=t if t > 0 else 0.0, k=k if 0 < k < V else 0, P=p if p < 1 else 1.0, M=m if m > 0 else 0.0))
        _check(z, u, got, cuts, least=0.9)


@gpu
def test_frequencies_follow_the_distribution():
    from tensornetworksfork_amd import ops
    dev = _dev()
    n = 1 << 16
    p = torch.tensor([0.1, 0.2, 0.3, 0.4], dtype=F64)
    z = p.log().expand(n, 4)
    g = torch.Generator().manual_seed(0)
    got = ops.sample(z.to(dev).contiguous(), torch.rand(n, generator=g, dtype=F64).to(dev)).cpu()
    f = torch.bincount(got, minlength=4).double() / n
    assert bool(((f - p).abs() < 6 * (p * (1 - p) / n).sqrt()).all())          # six standard deviations
    got = ops.sample(z.to(dev).contiguous(), torch.rand(n, generator=g, dtype=F64).to(dev), top_k=2).cpu()
    assert set(got.tolist()) == {2, 3}


@gpu
def test_row_distances_shapes_and_streams():
    from tensornetworksfork_amd import ops
    dev = _dev()
    g = torch.Generator().manual_seed(4)
    for V in (9, 500, 9001):
        wide = torch.randn(6, V + 5, generator=g)
        u = torch.rand(6, generator=g)
        Z = wide.to(dev)[:, 3:3 + V]
        _check(wide[:, 3:3 + V], u, ops.sample(Z, u.to(dev), top_p=0.9).cpu(), dict(P=0.9))
        one = wide.to(dev)[:1, :V].expand(6, V)
        _check(wide[:1, :V].expand(6, V), u, ops.sample(one, u.to(dev), top_k=3).cpu(), dict(k=3))
        z3 = wide[:, :V].contiguous().reshape(2, 3, V)
        u3 = u.reshape(2, 3)
        ref = ops.sample(z3.to(dev), u3.to(dev), top_p=0.8, top_k=100)
        assert ref.shape == (2, 3)
        s = torch.cuda.Stream(dev)
        Zs, us = z3.to(dev), u3.to(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            again = ops.sample(Zs, us, top_p=0.8, top_k=100)
        torch.cuda.synchronize()
        assert torch.equal(ref, again)
    assert ops.sample(torch.zeros(0, 4, device=dev), torch.zeros(0, device=dev)).shape == (0,)
    assert ops.sample(torch.tensor([0.0, 9.0], device=dev), torch.tensor(0.5, device=dev)).shape == ()


@gpu
@pytest.mark.parametrize("rows,V", [(4, 11), (5, 700), (3, 50000)])
def test_graph_replays(rows, V):
    from tensornetworksfork_amd import ops
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(1)
    z = torch.randn(rows, V, generator=g, device=dev)
    u = torch.rand(rows, generator=g, device=dev)
    kw = dict(temperature=0.9, top_k=min(V, 400), top_p=0.95, min_p=0.001)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        ops.sample(z, u, **kw)
    torch.cuda.current_stream(dev).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample(z, u, **kw)
    for turn in range(4):
        u.uniform_(generator=g)
        z.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, ops.sample(z, u, **kw)), turn


@gpu
def test_refusals_on_the_device():
    from tensornetworksfork_amd import _lib, ops
    dev = _dev()
    z, u = torch.zeros(4, 6, device=dev), torch.zeros(4, device=dev)
    bad = [lambda: ops.sample(z, u[:3]), lambda: ops.sample(z, u.cpu()), lambda: ops.sample(z, u.half()), lambda: ops.sample(z.int(), u),
           lambda: ops.sample(z.t(), torch.zeros(6, device=dev)), lambda: ops.sample(z, u, temperature=-1.0),
           lambda: ops.sample(z, u, temperature=float("nan")), lambda: ops.sample(z, u, temperature=float("inf")),
           lambda: ops.sample(z, u, top_k=-1), lambda: ops.sample(z, u, top_k=1.5), lambda: ops.sample(z, u, top_p=0.0),
           lambda: ops.sample(z, u, top_p=1.5), lambda: ops.sample(z, u, min_p=-0.1), lambda: ops.sample(z, u, min_p=1.1),
           lambda: ops.sample(z, u, top_p=u.double()), lambda: ops.sample(z, u, top_k=u), lambda: ops.sample(z, u, temperature=u[:2]),
           lambda: ops.sample(z[:, :0], u)]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.TTKError):
            f()
            raise AssertionError(i)
