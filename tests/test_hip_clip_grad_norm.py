"""GPU: the norm over all gradients and clipping (optim.clip_grad_norm_; dfhip_clip_grad_norm) against 64 bits.

Tolerances (u = 2^-24): the norm is summed in double and rounded once: 1.01 u; the factor is rounded once and multiplied in once:
2.02 u of an element."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _params(dev, arrays):
    from deepflows_amd import nn
    from deepflows_amd.tensor import Tensor
    out = []
    for a in arrays:
        p = nn.Parameter(Tensor(np.zeros(a.shape, np.float32), device=dev))
        p.grad = Tensor(a, device=dev).data
        out.append(p)
    return out


def _check(arrays, params, total, max_norm, kind, scale=1.0):
    flat = np.concatenate([a.reshape(-1).astype(np.float64) for a in arrays])
    want = (np.sqrt((flat ** 2).sum()) if kind == 2 else np.abs(flat).max()) * scale
    got = float(total.numpy()[0])
    assert tuple(total.shape) == (1,)
    assert abs(got - want) <= 1.01 * U * want + 1e-45, (got, want)
    coef = min(1.0, max_norm / (want + 1e-6))
    for a, p in zip(arrays, params):
        g = p.grad.numpy().astype(np.float64)
        assert g.shape == a.shape
        assert np.all(np.abs(g - a * coef) <= 2.02 * U * np.abs(a * coef) + 1e-44)


SETS = {
    "one element": [(1,)],
    "odd sizes": [(3,), (1, 5), (4097,), (7, 11), (2, 3, 5), (8191,)],
    "a perceptron": [(784, 256), (1, 256), (256, 10), (1, 10)],
    "sixty-four": [(k + 1,) for k in range(64)],
    "more than one launch holds": [(3 * k + 1,) for k in range(150)],
    "several shares a tensor": [(3000, 4000), (100,), (1 << 22,)],
}


@pytest.mark.parametrize("kind", [2, math.inf])
@pytest.mark.parametrize("max_norm", [0.0, 0.7, 1e9, math.inf])
@pytest.mark.parametrize("name", list(SETS))
def test_norm_and_scaled_gradients(hip_device, name, max_norm, kind):
    from deepflows_amd import optim
    rng = np.random.default_rng(len(name))
    arrays = [(rng.standard_normal(s) * 10.0 ** rng.integers(-3, 2)).astype(np.float32) for s in SETS[name]]
    params = _params(hip_device, arrays)
    held = [p.grad for p in params]
    total = optim.clip_grad_norm_(params, max_norm, norm_type=kind)
    _check(arrays, params, total, max_norm, kind)
    for a, g in zip(arrays, held):                          # the arrays that were there are as they were
        assert np.array_equal(g.numpy(), a)


def test_the_optimizers_factor_enters_the_norm(hip_device):
    from deepflows_amd import optim
    a = [np.arange(1, 9, dtype=np.float32)]
    params = _params(hip_device, a)
    _check(a, params, optim.clip_grad_norm_(params, 1.0, grad_scale=0.25), 1.0, 2, scale=0.25)


@pytest.mark.parametrize("value", [1e-30, 1e30])
def test_squares_beyond_the_range_of_a_float(hip_device, value):
    from deepflows_amd import optim
    a = [np.full((1000,), value, np.float32), np.full((17,), -value, np.float32)]
    params = _params(hip_device, a)
    _check(a, params, optim.clip_grad_norm_(params, 2.0), 2.0, 2)


def test_unaligned_and_strided_gradients(hip_device):
    from deepflows_amd import nn, optim
    from deepflows_amd.backend_selection import BackendTensor
    from deepflows_amd.parallel import _ArrayView
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(1)
    flat = rng.standard_normal(40001).astype(np.float32)
    m = rng.standard_normal((30, 50)).astype(np.float32)
    ft, mt = Tensor(flat, device=hip_device).data, Tensor(m, device=hip_device).data
    params = _params(hip_device, [np.zeros(40000, np.float32), np.zeros((50, 30), np.float32)])
    params[0].grad = BackendTensor.make((40000,), device=hip_device, handle=_ArrayView(ft._handle, 1, 40000))
    params[1].grad = mt.transpose()
    arrays = [flat[1:], m.T]
    _check(arrays, params, optim.clip_grad_norm_(params, 3.0), 3.0, 2)


def test_a_gradient_two_parameters_share_and_one_listed_twice(hip_device):
    from deepflows_amd import optim
    a = np.array([3.0, 4.0], np.float32)
    params = _params(hip_device, [a, a])
    params[1].grad = params[0].grad
    total = optim.clip_grad_norm_(params + [params[0]], 1.0)
    _check([a, a], params, total, 1.0, 2)


def test_parameters_without_gradients(hip_device):
    from deepflows_amd import optim
    params = _params(hip_device, [np.ones(3, np.float32), np.ones(4, np.float32)])
    params[0].grad = None
    total = optim.clip_grad_norm_(params, 1.0)
    assert params[0].grad is None and abs(float(total.numpy()[0]) - 2.0) <= 1e-6
    params[1].grad = None
    assert float(optim.clip_grad_norm_(params, 1.0).numpy()[0]) == 0.0


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("kind", [2, math.inf])
def test_gradients_that_are_not_finite(hip_device, bad, kind):
    from deepflows_amd import optim
    a = [np.ones(5000, np.float32), np.ones(70, np.float32)]
    a[0][4321] = bad
    params = _params(hip_device, a)
    with pytest.raises(RuntimeError):
        optim.clip_grad_norm_(params, 1.0, norm_type=kind, error_if_nonfinite=True)
    assert np.array_equal(params[1].grad.numpy(), a[1])     # (refused: nothing was scaled)
    total = float(optim.clip_grad_norm_(params, 1.0, norm_type=kind).numpy()[0])
    if np.isnan(bad):
        assert math.isnan(total) and all(np.all(np.isnan(p.grad.numpy())) for p in params)
    else:
        assert total == math.inf and np.all(params[1].grad.numpy() == 0.0) and np.isnan(params[0].grad.numpy()[4321])


def test_refusals(hip_device):
    from deepflows_amd import optim
    params = _params(hip_device, [np.ones(3, np.float32)])
    for kw in ({"max_norm": -1.0}, {"max_norm": math.nan}, {"max_norm": 1.0, "norm_type": 1.0},
               {"max_norm": 1.0, "grad_scale": -1.0}, {"max_norm": 1.0, "grad_scale": math.inf}):
        with pytest.raises(ValueError):
            optim.clip_grad_norm_(params, **kw)
    mod = hip_device.mod
    mod.capture_begin()
    try:
        with pytest.raises(RuntimeError):
            optim.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    finally:
        mod.capture_end().destroy()


def test_two_captured_graphs_and_eager_calls(hip_device):
    """two graphs captured one after the other (each with scratch memory of its own), replayed in turn with eager calls in
    between: every result is the eager call's"""
    from deepflows_amd import optim
    from deepflows_amd.tensor import Tensor
    mod = hip_device.mod
    rng = np.random.default_rng(2)
    sets = [[(300, 500), (77,)], [(65, 33), (9,), (1 << 20,)]]
    made = []
    for shapes in sets:
        params = _params(hip_device, [np.zeros(s, np.float32) for s in shapes])
        ins = [p.grad for p in params]
        mod.capture_begin()
        total = optim.clip_grad_norm_(params, 0.5)
        outs = [p.grad for p in params]
        made.append((ins, outs, total, mod.capture_end(keep=(ins, outs, total)), params))
    for _ in range(3):
        fresh = [[rng.standard_normal(s).astype(np.float32) for s in shapes] for shapes in sets]
        for (ins, _, _, _, _), arrays in zip(made, fresh):
            for t, a in zip(ins, arrays):
                mod.from_numpy(a, t._handle)
        for m in made:
            m[3].replay()
        for (ins, outs, total, _, params), arrays in zip(made, fresh):
            for p, t in zip(params, ins):
                p.grad = t
            eager = optim.clip_grad_norm_(params, 0.5)
            assert np.array_equal(eager.numpy(), total.numpy())
            for p, o in zip(params, outs):
                assert np.array_equal(p.grad.numpy(), o.numpy())
    for m in made:
        m[3].destroy()
