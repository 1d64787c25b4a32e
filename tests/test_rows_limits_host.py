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


def _stub_kernels(monkeypatch):
    """The rows' kernels replaced by what passes the values on: which graph autograd records is the host's matter."""
    from tensornetworksfork_amd import ops
    monkeypatch.setattr(ops, "layer_norm", lambda x, *a, stats=True, **k: (x.detach().clone(), x[..., 0].detach(), x[..., 0].detach()))
    monkeypatch.setattr(ops, "dropout", lambda x, *a, **k: x.detach().clone())


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A dual tensor requires no gradient: without a look at its tangent the result would carry none, in silence."""
    import torch.autograd.forward_ad as fw
    from tensornetworksfork_amd import _lib
    from tensornetworksfork_amd.tensor.norm import Dropout, LayerNorm, dropout, layer_norm
    _stub_kernels(monkeypatch)
    x, w, v = torch.randn(3, 4), torch.randn(4), torch.randn(4)
    calls = [lambda a, b, c: layer_norm(a, b, c), lambda a, b, c: layer_norm(x, b, c), lambda a, b, c: layer_norm(x, w, c),
             lambda a, b, c: dropout(a, 0.5, 1), lambda a, b, c: LayerNorm(4)(a), lambda a, b, c: Dropout(0.5)(a),
             lambda a, b, c: layer_norm(a.t(), None, None), lambda a, b, c: layer_norm(a.clone().requires_grad_(True), b, c)]
    for f in calls:
        assert f(x, w, v) is not None
        with fw.dual_level():
            dual = [fw.make_dual(t, torch.ones_like(t)) for t in (x, w, v)]
            with pytest.raises(_lib.TTKError):
                f(*dual)
            with torch.no_grad(), pytest.raises(_lib.TTKError):
                f(*dual)
            f(x, w, v)                                    # tensors without a tangent pass at any level
    with pytest.raises(_lib.TTKError):
        torch.func.jvp(lambda a: layer_norm(a, w, v), (x,), (x,))


def test_rows_a_lane_adds_are_bounded():
    """The backward pass leaves a partial row of sums for every 480 rows of a lane or fewer: the workspace grows with the rows, as
    far as rows and gradients fit the memory of a GPU (288 GB); rows that are one row broadcast may be more, but not the workspace."""
    from tensornetworksfork_amd import _lib
    L = _lib.lib()
    for dtype in range(4):
        size = 8 if dtype == 0 else 4
        for cols in (1, 8, 20, 32, 33, 100, 784, 1500, 5000, 12000, 16000):
            if dtype == 0 and cols > 8192:
                continue                                  # (rows the registers do not hold: added in 64 bits, however many)
            held = 288 * 10 ** 9 // (2 * cols * (8, 4, 2, 2)[dtype])
            for rows in (1, 1000, 1 << 20, min(1 << 24, held), held, 1 << 31, 1 << 36):
                need = L.ttk_layer_norm_backward_ws_bytes(dtype, rows, cols)
                parts = need // (2 * cols * size)
                assert 0 < need <= 5 << 28
                if rows <= held:
                    assert parts * 256 * 480 >= rows      # (256 lanes a workgroup, each with a row of its own, at most)
                    if cols >= 5000:
                        assert parts * 480 >= rows        # (a workgroup a row)


@pytest.fixture
def cpu_kernels(monkeypatch):
    from tests import _kernel_standins
    _kernel_standins.install(monkeypatch)
    old = torch.get_default_dtype()
    torch.set_default_dtype(torch.float64)
    yield
    torch.set_default_dtype(old)


def _train(seed=3, S=9, p=4, C=2):
    from tensornetworksfork_amd.tensor.layers import TensorTrainLayer
    layer = TensorTrainLayer(3, 4, p, output_shape=C, seed=seed)
    return layer, torch.randn(S, p, generator=torch.Generator().manual_seed(seed))


def _plain(layer, xs):
    a, b, c = (n.tensor for n in layer.tensor_network.main_nodes)
    p = xs[0].shape[1]
    y = torch.einsum("cpl,sp->scl", a.reshape(-1, p, a.shape[-1]), xs[0])
    y = torch.einsum("scl,lpr,sp->scr", y, b.reshape(-1, p, b.shape[-1]), xs[1])
    return torch.einsum("scl,lp,sp->sc", y, c.reshape(-1, p), xs[2])


def test_recorded_passes_leave_the_cached_data_sets_alone(cpu_kernels):
    """A sweep keeps the environments of its data sets; passes on inputs that require a gradient must not push them out."""
    layer, x = _train()
    eng = layer.tensor_network._engine
    sets = [x, x.clone(), x.clone()]
    for t in sets:
        layer(t)
    kept = list(eng.datasets)
    assert len(kept) == 3
    for i in range(5):
        y = layer((x + i).requires_grad_(True))
        assert y.requires_grad
    assert len(eng.datasets) == 3 and all(a is b for a, b in zip(eng.datasets, kept))


def test_recorded_passes_of_one_input_share_their_environments(cpu_kernels, monkeypatch):
    """As unrecorded passes do; an input that changed in place since, or another one, gets its own."""
    layer, x = _train()
    eng = layer.tensor_network._engine
    made, make = [], eng.make_data
    monkeypatch.setattr(eng, "make_data", lambda *a, **k: made.append(1) or make(*a, **k))
    leaf = x.clone().requires_grad_(True)
    for _ in range(3):
        y = layer(leaf)
        g, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert len(made) == 1
    with torch.no_grad():
        leaf.mul_(2.0)
    y2 = layer(leaf)
    assert len(made) == 2 and torch.allclose(y2, _plain(layer, [2 * x] * 3).reshape(y2.shape), rtol=1e-12)
    assert torch.allclose(layer([leaf] * 3), y2, rtol=1e-12)
    layer.tensor_network.main_nodes[1].tensor.mul_(3.0)
    assert torch.allclose(layer(leaf), 3 * y2, rtol=1e-12)
    ref_in = leaf.detach().clone().requires_grad_(True)
    ref, = torch.autograd.grad(_plain(layer, [ref_in] * 3).sum(), ref_in)
    y = layer(leaf)
    got, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.allclose(got, ref, rtol=1e-10)
    # the pass before last still has its own data when another input has taken its place
    one, two = x.clone().requires_grad_(True), (x + 1).requires_grad_(True)
    y1, y2 = layer(one), layer(two)
    got, = torch.autograd.grad(y1, one, torch.ones_like(y1))
    ref_in = x.clone().requires_grad_(True)
    ref, = torch.autograd.grad(_plain(layer, [ref_in] * 3).sum(), ref_in)
    assert torch.allclose(got, ref, rtol=1e-10)


def test_recorded_passes_do_not_keep_their_inputs_graph_alive(cpu_kernels):
    import gc
    import weakref
    layer, x = _train()
    h = x.clone().requires_grad_(True) * 2.0
    y = layer(h)
    ref = weakref.ref(h)
    del h, y
    gc.collect()
    assert ref() is None


def test_input_gradient_with_labels_in_another_order(cpu_kernels):
    """The output's labels may be asked for in any order; the gradient follows them."""
    layer, x = _train(C=3)
    g = torch.Generator().manual_seed(1)
    plain = layer(x)
    ref_in = x.clone().requires_grad_(True)
    ref = _plain(layer, [ref_in] * 3)
    assert torch.allclose(plain, ref, rtol=1e-12) and list(layer.labels) == ["s", "c1"]
    for order in ((0, 1), (1, 0)):
        layer.labels = [("s", "c1")[i] for i in order]
        leaf = x.clone().requires_grad_(True)
        y = layer(leaf)
        assert y.requires_grad and torch.equal(y.detach(), plain.permute(order))
        dy = torch.randn(y.shape, generator=g)
        got, = torch.autograd.grad(y, leaf, dy)
        want, = torch.autograd.grad(ref.permute(order), ref_in, dy, retain_graph=True)
        assert torch.allclose(got, want, rtol=1e-10, atol=1e-12)


def test_networks_without_an_input_gradient_say_so(cpu_kernels, monkeypatch):
    """Their outputs stay what they were, without a gradient: a warning tells who asked for one."""
    import warnings

    import torch.autograd.forward_ad as fw
    from tensornetworksfork_amd.tensor.layers import CPDLayer, TensorTrainLayer
    nets = [CPDLayer(3, 4, 5, output_shape=2, seed=1), TensorTrainLayer(3, 4, 5, output_shape=(2, 3), seed=1)]
    train = TensorTrainLayer(3, 4, 5, output_shape=2, seed=1)
    x = torch.randn(6, 5)
    for net in nets + [train]:      # (kernels are nothing autograd sees: the stand-ins, which are torch operations, would be)
        def closed(*args, predict=net.tensor_network._predict):
            with torch.no_grad():
                return fw.unpack_dual(predict(*args)).primal.clone()
        monkeypatch.setattr(net.tensor_network, "_predict", closed)
    for net in nets:
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            plain = net(x)
            with torch.no_grad():
                net(x.clone().requires_grad_(True))
        with pytest.warns(UserWarning, match="gradient"):
            y = net(x.clone().requires_grad_(True))
        assert not y.requires_grad and torch.equal(y, plain)
    for net in nets + [train]:
        with fw.dual_level(), pytest.warns(UserWarning, match="derivative"):
            net(fw.make_dual(x, torch.ones_like(x)))


def test_estimators_saved_before_the_front_end_work():
    """An estimator pickled when it had neither layer norm nor dropout takes rows as it did."""
    import pickle

    from tensornetworksfork_amd.models.tensor_train import TensorTrainRegressor
    from tensornetworksfork_amd.models.tnml import TNMLRegressor
    for cls in (TensorTrainRegressor, TNMLRegressor):
        e = cls(seed=3)
        state = {k: v for k, v in e.__dict__.items() if k not in ("layer_norm", "dropout", "_dropout_offset")}
        assert len(state) == len(e.__dict__) - 3
        old = cls.__new__(cls)
        old.__setstate__(state)
        old = pickle.loads(pickle.dumps(old))
        x = torch.randn(4, 3)
        assert old._normalise(x) is x and old._drop(x) is x
        assert (old.layer_norm, old.dropout) == (False, 0.0)


def test_layers_are_saved_and_copied_after_a_recorded_pass(cpu_kernels):
    import copy
    import pickle
    layer, x = _train()
    want = layer(x)
    h = x.clone().requires_grad_(True) * 2.0
    for t in (x.clone().requires_grad_(True), h):
        layer(t)
        for other in (pickle.loads(pickle.dumps(layer)), copy.deepcopy(layer)):
            assert torch.equal(other(x), want)
            leaf = x.clone().requires_grad_(True)
            y = other(leaf)
            got, = torch.autograd.grad(y, leaf, torch.ones_like(y))
            y = layer(leaf)
            assert torch.equal(got, torch.autograd.grad(y, leaf, torch.ones_like(y))[0])
    # one that was saved before there was such a place
    old = copy.deepcopy(layer)
    old.tensor_network._engine.__dict__.pop("recorded", None)
    assert old(x.clone().requires_grad_(True)).requires_grad and torch.equal(old(x), want)
