"""GPU: root-mean-square normalisation with the residual's addition (F.rms_norm, nn.RMSNorm; dfhip_rms_norm_forward /
_backward) against the formula in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, half a step of fp32, relative):
  h   = the rounded sum: equal to NumPy's float32 addition;
  y   = h r w: the rounding of h in the numerator and through r, of r to fp32 and two products: 5 u |y|;
  dx  = r (g - n c) + add, c = mean(g n): g, n carry one and two roundings; c a sum of depth `deep` (at most 64 terms a thread
        and 12 exchanges, or width / 256 + 12 for rows read twice): u r (8 |g| + |n| (deep + 8) mean|g n|) + u |dx| of the last
        addition;
  dw  = a sum over the rows, a team's rows (at most rows / 512), up to 16 teams, up to 2048 partial rows as 16 sums of 128: depth
        rows / 512 + 163, each term two roundings."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _want(x, r, w, eps, dy, dh):
    x64 = x.astype(np.float64)
    h = x64 if r is None else x64 + r.astype(np.float64)
    D = x.shape[-1]
    inv = 1.0 / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    n = h * inv
    w64 = np.ones(D) if w is None else w.astype(np.float64)
    y = n * w64
    g = dy.astype(np.float64) * w64
    c = (g * n).mean(-1, keepdims=True)
    dx = inv * (g - n * c) + (0.0 if dh is None else dh.astype(np.float64))
    dw = (dy.astype(np.float64) * n).reshape(-1, D).sum(0)
    deep = 76 + D // 256
    rows = x.size // D
    tol_dx = U * (inv * (8 * np.abs(g) + np.abs(n) * (deep + 8) * np.abs(g * n).mean(-1, keepdims=True)) + 2 * np.abs(dx)
                  + (0.0 if dh is None else np.abs(dh)))
    tol_dw = U * (rows // 512 + 165) * np.abs(dy.astype(np.float64) * n).reshape(-1, D).sum(0)
    return y, dx, dw, 5 * U * np.abs(y) + 1e-37, tol_dx + 1e-37, tol_dw + 1e-37


def _upstream(dev, y, h, dy, dh):
    """a scalar whose gradient at y is dy (and at h, dh)"""
    from deepflows_amd import tensor
    from deepflows_amd.tensor import Tensor
    loss = tensor.sum(y * Tensor(dy, device=dev))
    if dh is not None:
        loss = loss + tensor.sum(h * Tensor(dh, device=dev))
    return loss.reshape(1)


def _within(got, want, tol, what):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, what
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.abs(got - want)[bad].max():.3e} against {tol[bad].min():.3e}"


def _case(dev, shape, residual, affine, seed=0, eps=1e-6, scale=1.0):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    rng = np.random.default_rng(seed)
    D = shape[-1]
    x = (scale * rng.standard_normal(shape)).astype(np.float32)
    r = (2 * scale * rng.standard_normal(shape)).astype(np.float32) if residual else None
    w = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32) if affine else None
    dy = rng.standard_normal(shape).astype(np.float32)
    dh = rng.standard_normal(shape).astype(np.float32) if residual else None
    xt = Tensor(x, device=dev, requires_grad=True)
    rt = Tensor(r, device=dev, requires_grad=True) if residual else None
    wt = Tensor(w, device=dev, requires_grad=True) if affine else None
    out = F.rms_norm(xt, wt, eps, residual=rt)
    y, h = out if residual else (out, None)
    got_y = y.numpy()
    if residual:
        assert np.array_equal(h.numpy(), x + r)
    _upstream(dev, y, h, dy, dh).backward()
    wy, wdx, wdw, ty, tdx, tdw = _want(x, r, w, eps, dy, dh)
    _within(got_y, wy, ty, "y")
    _within(xt.grad.numpy(), wdx, tdx, "dx")
    if residual:
        assert np.array_equal(rt.grad.numpy(), xt.grad.numpy())
    if affine:
        _within(wt.grad.numpy(), wdw, tdw, "dw")
    Graph.free_graph_all()


@pytest.mark.parametrize("width", [1, 2, 7, 16, 127, 128, 132, 512, 513, 1000, 1024, 1531, 2048, 4100, 8191, 16384, 16385, 20000,
                                   33001])
@pytest.mark.parametrize("rows", [1, 5, 37])
def test_values_and_gradients(hip_device, rows, width):
    _case(hip_device, (rows, width), residual=True, affine=True, seed=width)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("shape", [(64,), (3, 5, 200), (2, 3, 4, 33)])
def test_any_number_of_axes(hip_device, shape, residual, affine):
    _case(hip_device, shape, residual, affine, seed=len(shape))


@pytest.mark.parametrize("rows,width", [(9001, 16), (9001, 57), (40007, 24), (4500, 300), (2500, 1001), (1300, 1536), (600, 9999), (700, 17000)])
def test_more_rows_than_workgroups(hip_device, rows, width):
    _case(hip_device, (rows, width), residual=True, affine=True, seed=rows)


@pytest.mark.parametrize("scale", [1e-18, 1e18, 3e37])
def test_squares_beyond_the_range_of_a_float(hip_device, scale):
    """eps = 0: the mean of the squares is held in double, so neither it nor its root leaves the range"""
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(3)
    x = (scale * rng.uniform(0.5, 2.0, (4, 250))).astype(np.float32)
    y = F.rms_norm(Tensor(x, device=hip_device), None, 0.0).numpy()
    want = x.astype(np.float64) / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True))
    _within(y, want, 5 * U * np.abs(want), "y")


def test_a_row_of_zeros_and_rows_that_are_not_finite(hip_device):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 300)).astype(np.float32)
    x[1] = 0.0
    x[3, 7] = np.nan
    x[4, 9] = np.inf
    y = F.rms_norm(Tensor(x, device=hip_device), None, 1e-6).numpy()
    assert np.all(y[1] == 0.0) and np.all(np.isnan(y[3]))
    assert np.isnan(y[4, 9]) and np.all(y[4, :9] == 0.0)           # inf * 0, x / inf
    for i in (0, 2, 5):
        want = x[i].astype(np.float64) / np.sqrt((x[i].astype(np.float64) ** 2).mean() + 1e-6)
        _within(y[i], want, 5 * U * np.abs(want), f"row {i}")


def test_no_rows(hip_device):
    from deepflows_amd.backend_selection import BackendTensor
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    x = Tensor(BackendTensor.make((0, 8), device=hip_device))
    assert tuple(F.rms_norm(x, None).shape) == (0, 8)


def test_a_transposed_view(hip_device):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(5)
    a = rng.standard_normal((40, 12)).astype(np.float32)
    r = rng.standard_normal((12, 40)).astype(np.float32)
    y, h = F.rms_norm(Tensor(a, device=hip_device).transpose(), None, 1e-6, residual=Tensor(r, device=hip_device))
    assert np.array_equal(h.numpy(), a.T + r)
    s = (a.T + r).astype(np.float64)
    want = s / np.sqrt((s * s).mean(-1, keepdims=True) + 1e-6)
    _within(y.numpy(), want, 5 * U * np.abs(want), "y")


def test_the_input_as_its_own_residual(hip_device):
    from deepflows_amd import tensor
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(6)
    x = rng.standard_normal((5, 96)).astype(np.float32)
    dy = rng.standard_normal((5, 96)).astype(np.float32)
    xt = Tensor(x, device=hip_device, requires_grad=True)
    y, h = F.rms_norm(xt, None, 1e-6, residual=xt)
    tensor.sum(y * Tensor(dy, device=hip_device)).reshape(1).backward()
    _, dx, _, _, tol, _ = _want(2 * x, None, None, 1e-6, dy, None)
    _within(xt.grad.numpy(), 2 * dx, 2 * tol + U * np.abs(2 * dx), "dx")


def test_only_the_weight_needs_a_gradient_and_its_place_is_given(hip_device):
    """a parameter's slice of a gradient bucket (not 16-byte aligned) receives the gradient"""
    from deepflows_amd import nn, tensor
    from deepflows_amd.backend_selection import BackendTensor
    from deepflows_amd.parallel import _ArrayView
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(7)
    x = rng.standard_normal((19, 64)).astype(np.float32)
    dy = rng.standard_normal((19, 64)).astype(np.float32)
    norm = nn.RMSNorm(64, device=hip_device)
    flat = BackendTensor.make((67,), device=hip_device)
    flat.fill(7.0)
    norm.weight.grad_slot = BackendTensor.make((64,), device=hip_device, handle=_ArrayView(flat._handle, 1, 64))
    y = norm(Tensor(x, device=hip_device))
    tensor.sum(y * Tensor(dy, device=hip_device)).reshape(1).backward()
    assert norm.weight.grad is norm.weight.grad_slot
    _, _, dw, _, _, tol = _want(x, None, np.ones(64, np.float32), 1e-6, dy, None)
    _within(flat.numpy()[1:65], dw, tol, "dw")
    assert np.all(flat.numpy()[[0, 65, 66]] == 7.0)


def test_two_sweeps_over_a_retained_graph(hip_device):
    from deepflows_amd import tensor
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    rng = np.random.default_rng(8)
    x = Tensor(rng.standard_normal((4, 32)).astype(np.float32), device=hip_device, requires_grad=True)
    w = Tensor(rng.standard_normal(32).astype(np.float32), device=hip_device, requires_grad=True)
    y, h = F.rms_norm(x, w, 1e-6, residual=x * 0.5)
    loss = tensor.sum(y * y) + tensor.sum(h * h)
    loss = loss.reshape(1)
    loss.backward(retain_graph=True)
    first = x.grad.numpy().copy(), w.grad.numpy().copy()
    x.grad = w.grad = None
    loss.backward()
    assert np.array_equal(x.grad.numpy(), first[0]) and np.array_equal(w.grad.numpy(), first[1])
    Graph.free_graph_all()


def test_gradients_against_differences(hip_device):
    from deepflows_amd import tensor
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    rng = np.random.default_rng(9)
    x, r, w = (rng.standard_normal(s).astype(np.float32) for s in ((3, 20), (3, 20), (20,)))
    c, d = rng.standard_normal((3, 20)), rng.standard_normal((3, 20))

    def value(x, r, w):
        h = x + r
        return ((h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-3) * w) * c + h * d).sum()

    ts = [Tensor(a, device=hip_device, requires_grad=True) for a in (x, r, w)]
    y, h = F.rms_norm(ts[0], ts[2], 1e-3, residual=ts[1])
    (tensor.sum(y * Tensor(c, device=hip_device)) + tensor.sum(h * Tensor(d, device=hip_device))).reshape(1).backward()
    args = [a.astype(np.float64) for a in (x, r, w)]
    for k in range(3):
        got = ts[k].grad.numpy()
        for _ in range(6):
            at = tuple(int(rng.integers(0, s)) for s in args[k].shape)
            step = 1e-5
            up = [a.copy() for a in args]; up[k][at] += step
            dn = [a.copy() for a in args]; dn[k][at] -= step
            slope = (value(*up) - value(*dn)) / (2 * step)
            # (central differences in 64 bits: 1e-9 of their own; the gradient's values are of order 1-10, fp32)
            assert abs(got[at] - slope) <= 2e-6 * max(1.0, abs(slope)) * 10
    Graph.free_graph_all()


def test_refusals(hip_device):
    from deepflows_amd import nn
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    x = Tensor(np.ones((3, 8), np.float32), device=hip_device)
    w9 = Tensor(np.ones(9, np.float32), device=hip_device)
    with pytest.raises(ValueError):
        F.rms_norm(x, w9)
    with pytest.raises(ValueError):
        F.rms_norm(x, None, residual=Tensor(np.ones((3, 9), np.float32), device=hip_device))
    with pytest.raises(ValueError):
        F.rms_norm(x, None, eps=-1.0)
    with pytest.raises(ValueError):
        F.rms_norm(w9, w9)
    with pytest.raises(ValueError):
        nn.RMSNorm(9, device=hip_device)(x)
    mod = hip_device.mod
    a = x.data._handle
    with pytest.raises(ValueError):
        mod.rms_norm_forward(a, None, None, a, None, None, 3, 0, 1e-6)
    with pytest.raises(ValueError):
        mod.rms_norm_forward(a, a, None, a, None, None, 3, 8, 1e-6)      # a residual, and no place for the sum
    with pytest.raises(ValueError):
        mod.rms_norm_backward(a, a, a, None, None, None, None, 3, 8)


def test_inside_a_captured_graph(hip_device):
    """a captured forward and backward pass, replayed on changed inputs, beside the eager one bit for bit"""
    from deepflows_amd import tensor
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    mod = hip_device.mod
    rng = np.random.default_rng(10)
    x = Tensor(rng.standard_normal((37, 257)).astype(np.float32), device=hip_device, requires_grad=True)
    r = Tensor(rng.standard_normal((37, 257)).astype(np.float32), device=hip_device, requires_grad=True)
    w = Tensor(rng.standard_normal(257).astype(np.float32), device=hip_device, requires_grad=True)

    def step():
        x.grad = r.grad = w.grad = None
        y, h = F.rms_norm(x, w, 1e-6, residual=r)
        tensor.sum(y * y * 0.5 + h).reshape(1).backward()
        return y, h, x.grad, w.grad

    step()
    mod.capture_begin()
    got = step()
    graph = mod.capture_end(keep=got)
    for k in range(3):
        mod.from_numpy(rng.standard_normal((37, 257)).astype(np.float32), x.data._handle)
        graph.replay()
        replayed = [t.numpy().copy() for t in got]
        eager = [t.numpy().copy() for t in step()]
        for a, b in zip(replayed, eager):
            assert np.array_equal(a, b)
    graph.destroy()
    Graph.free_graph_all()


def test_more_rows_than_one_launch_holds(hip_device):
    """2^28 + 5 rows of one element: sixteen threads a row would be a launch of more than 2^32 threads.  The rows differ at the places
    where one launch could end and the next begin; y = x w / sqrt(x^2 + eps), dx = w dy (1 - y^2 / w^2) / sqrt(x^2 + eps)."""
    from deepflows_amd import tensor
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    rows, eps = (1 << 28) + 5, 1.0
    places = [(k << 24) - 3 for k in range(1, 17)] + [0, rows - 6]
    xd = hip_device.full((rows, 1), 2.0)
    value = {}
    for k, at in enumerate(places):
        for j in range(6):
            value[at + j] = 0.25 * (1 + k) - 0.125 * j
            xd[at + j:at + j + 1, :] = value[at + j]
    x = Tensor(xd, requires_grad=True)
    w = Tensor(np.array([3.0], np.float32), device=hip_device, requires_grad=True)
    y = F.rms_norm(x, w, eps)
    yd = y.data

    class Rest(tensor.UnaryOperator):
        def forward(self, x):
            return hip_device.full((1,), 0.0)

        def grad_fn(self, node, grad):
            return hip_device.full((rows, 1), 1.0)

    Rest(y).backward()
    middle = 12345678
    value[middle] = 2.0
    for at in places + [middle]:
        n = 1 if at == middle else 6
        v = np.array([value[at + j] for j in range(n)], np.float64)
        inv = 1 / np.sqrt(v * v + eps)
        _within(yd[at:at + n, :].compact().numpy()[:, 0], 3 * v * inv, 5 * U * np.abs(3 * v * inv) + 1e-37, f"y from {at}")
        want = 3 * inv * (1 - (v * inv) ** 2)
        # (g - n c with c = g n: both terms up to 3 inv, eight roundings)
        _within(x.grad[at:at + n, :].compact().numpy()[:, 0], want, 24 * U * inv * (1 + (v * inv) ** 2), f"dx from {at}")
    Graph.free_graph_all()
