"""CPU: F.rms_norm, nn.RMSNorm and optim.clip_grad_norm_ on the NumPy oracle device (their compositions over the device
primitives), and what they refuse."""
import math

import numpy as np
import pytest

from conftest import assert_close


def test_rms_norm_composition(cpu_oracle):
    from deepflows_amd import nn, tensor
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(0)
    x, r, c = (rng.standard_normal((4, 10)).astype(np.float32) for _ in range(3))
    norm = nn.RMSNorm(10, eps=1e-3, device=cpu_oracle)
    xt = Tensor(x, device=cpu_oracle, requires_grad=True)
    y, h = norm(xt, Tensor(r, device=cpu_oracle))
    s = (x + r).astype(np.float64)
    inv = 1 / np.sqrt((s * s).mean(-1, keepdims=True) + 1e-3)
    assert_close(h.numpy(), x + r, 1e-7)
    assert_close(y.numpy(), s * inv, 1e-6)
    (tensor.sum(y * Tensor(c, device=cpu_oracle))).reshape(1).backward()
    assert_close(xt.grad.numpy(), inv * (c - s * inv * (c * s * inv).mean(-1, keepdims=True)), 1e-5)
    assert_close(norm.weight.grad.numpy(), (c * s * inv).sum(0), 1e-5)
    assert "weight" in norm.state_dict()


def test_rms_norm_refusals(cpu_oracle):
    from deepflows_amd import nn
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    x = Tensor(np.ones((3, 8), np.float32), device=cpu_oracle)
    with pytest.raises(ValueError):
        F.rms_norm(x, Tensor(np.ones(7, np.float32), device=cpu_oracle))
    with pytest.raises(ValueError):
        F.rms_norm(x, None, eps=float("nan"))
    with pytest.raises(ValueError):
        F.rms_norm(x, None, residual=Tensor(np.ones((2, 8), np.float32), device=cpu_oracle))
    with pytest.raises(ValueError):
        nn.RMSNorm(0, device=cpu_oracle)


def _params(dev, arrays):
    from deepflows_amd import nn
    from deepflows_amd.tensor import Tensor
    out = []
    for a in arrays:
        p = nn.Parameter(Tensor(np.zeros(a.shape), device=dev))
        p.grad = Tensor(a, device=dev).data
        out.append(p)
    return out


@pytest.mark.parametrize("kind", [2, math.inf])
def test_clip_composition(cpu_oracle, kind):
    from deepflows_amd import optim
    rng = np.random.default_rng(1)
    arrays = [rng.standard_normal(s).astype(np.float32) for s in ((3, 4), (1, 7), (5,))]
    params = _params(cpu_oracle, arrays)
    total = optim.clip_grad_norm_(params, 0.5, norm_type=kind, grad_scale=0.5)
    flat = np.concatenate([a.reshape(-1) for a in arrays]).astype(np.float64)
    want = 0.5 * (np.sqrt((flat ** 2).sum()) if kind == 2 else np.abs(flat).max())
    assert_close(total.numpy(), [want], 1e-6)
    for a, p in zip(arrays, params):
        assert_close(p.grad.numpy(), a * min(1.0, 0.5 / (want + 1e-6)), 1e-6)


def test_clip_refusals(cpu_oracle):
    from deepflows_amd import optim
    params = _params(cpu_oracle, [np.ones(3, np.float32)])
    for kw in ({"max_norm": -1.0}, {"max_norm": 1.0, "norm_type": 3.0}, {"max_norm": 1.0, "grad_scale": -0.1}):
        with pytest.raises(ValueError):
            optim.clip_grad_norm_(params, **kw)
    params[0].grad.fill(np.inf)
    with pytest.raises(RuntimeError):
        optim.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)


@pytest.mark.parametrize("smoothing", [0.0, 0.2])
def test_linear_cross_entropy_composition(cpu_oracle, smoothing):
    from deepflows_amd import nn
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(2)
    x, t = rng.standard_normal((6, 5)).astype(np.float32), np.array([0, 6, -100, 3, 3, -100], np.float32)
    fc = nn.Linear(5, 7, device=cpu_oracle)
    xt = Tensor(x, device=cpu_oracle, requires_grad=True)
    loss = nn.LinearCrossEntropyLoss(fc, label_smoothing=smoothing)(xt, Tensor(t, device=cpu_oracle))
    l = x.astype(np.float64) @ fc.weight.numpy() + fc.bias.numpy()
    lp = l - l.max(1, keepdims=True)
    lp -= np.log(np.exp(lp).sum(1, keepdims=True))
    q = np.full((6, 7), smoothing / 7)
    q[np.arange(6), np.where(t < 0, 0, t).astype(int)] += 1 - smoothing
    q[t < 0] = 0
    assert_close(loss.numpy(), [-(lp * q).sum() / 4], 1e-6)
    loss.backward()
    dl = np.where((t < 0)[:, None], 0, np.exp(lp) - q) / 4
    assert_close(xt.grad.numpy(), dl @ fc.weight.numpy().T, 1e-5)
    assert_close(fc.weight.grad.numpy(), x.T @ dl, 1e-5)
    assert_close(fc.bias.grad.numpy(), dl.sum(0, keepdims=True), 1e-5)


def test_linear_cross_entropy_refusals(cpu_oracle):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    new = lambda *s: Tensor(np.zeros(s, np.float32), device=cpu_oracle)
    x, w, b, t = new(4, 3), new(3, 5), new(1, 5), new(4)
    for args, kw in [((x, new(4, 5), b, t), {}), ((x, w, new(1, 4), t), {}), ((x, w, b, new(4, 5)), {}),
                     ((x, w, b, t), {"reduction": "none"}), ((x, w, b, t), {"label_smoothing": -0.1}),
                     ((x, w, b, Tensor(np.full(4, 5.0), device=cpu_oracle)), {}),
                     ((x, w, b, Tensor(np.full(4, 0.5), device=cpu_oracle)), {})]:
        with pytest.raises(ValueError):
            F.linear_cross_entropy(*args, **kw)


@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38])
def test_rows_that_are_not_counted_may_hold_anything(cpu_oracle, bad):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(4)
    x, w = rng.standard_normal((5, 6)).astype(np.float32), rng.standard_normal((6, 9)).astype(np.float32)
    t = np.array([3, -100, 8, -100, 0], np.float32)
    results = []
    for fill in (0.0, bad):
        y = np.where(t[:, None] == -100, np.float32(fill), x)
        ts = [Tensor(a, device=cpu_oracle, requires_grad=True) for a in (y, w)]
        loss = F.linear_cross_entropy(*ts, None, Tensor(t, device=cpu_oracle))
        loss.backward()
        results.append([loss.numpy()] + [p.grad.numpy() for p in ts])
    for a, b in zip(*results):
        assert np.all(np.isfinite(a)) and np.array_equal(a, b)
    assert not results[1][1][t == -100].any()


def test_a_clipped_training_step_of_two_ranks(cpu_oracle):
    """the summed gradients of two ranks with grad_scale = 1/2 are clipped as their mean is"""
    from deepflows_amd import nn, optim, workloads
    from deepflows_amd.tensor import Tensor
    rng = np.random.default_rng(3)
    x, y = rng.standard_normal((5, 12)).astype(np.float32), np.eye(4, dtype=np.float32)[rng.integers(0, 4, 5)]
    finals = []
    for double in (False, True):
        np.random.seed(1)
        model = workloads.MLP((12, 16, 4), device=cpu_oracle)
        opt = optim.SGD(model.parameters(), lr=0.5)

        def sync():
            if double:
                opt.grad_scale = 0.5
                for p in opt.params:
                    p.grad = p.grad * 2.0

        workloads.train_step(model, nn.CrossEntropyLoss(), opt, Tensor(x, device=cpu_oracle), Tensor(y, device=cpu_oracle),
                             sync=sync, max_grad_norm=0.01)
        finals.append([p.numpy() for p in opt.params])
    for a, b in zip(*finals):
        assert_close(a, b, 1e-6)


def test_two_gloo_ranks_clip_the_mean_of_their_gradients(tmp_path):
    """three steps through the gradient bucket, whose slices the clipped windows replace: the ranks agree bit for bit, and with one
    process that clips the averaged gradients itself"""
    import json
    import os
    import subprocess
    import sys

    import test_data_parallel as dp
    from conftest import ROOT
    adam, plain = "optim.Adam(model.parameters(), lr=1e-2, weight_decay=5e-4)", "sync=bucket.sync if world > 1 else None"
    assert adam in dp.WORKER and plain in dp.WORKER
    script = tmp_path / "worker.py"
    script.write_text(dp.WORKER.replace(adam, "optim.SGD(model.parameters(), lr=0.5)").replace(plain, plain + ", max_grad_norm=0.1"))
    env = dict(os.environ, DF_ROOT=ROOT, DF_OUT=str(tmp_path), MASTER_ADDR="127.0.0.1")
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
                        "--master-port", str(31500 + os.getpid() % 2000), str(script)], env=env, capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    outs = [json.load(open(tmp_path / f"rank{k}.json")) for k in range(2)]
    for a, b in zip(outs[0]["params"], outs[1]["params"]):
        assert np.array_equal(np.array(a), np.array(b))

    from deepflows_amd import backend_api, nn, workloads
    from deepflows_amd.tensor import Graph, Tensor
    from oracle.numpy_device import NumpyDevice
    dev = backend_api.register_device("cpu", NumpyDevice())
    try:
        np.random.seed(0)
        model = workloads.MLP((12, 16, 4), device=dev)
        params = [p.numpy().astype(np.float64) for p in model.parameters()]
        rngs, clipped = [np.random.default_rng(100 + r) for r in range(2)], 0
        for _ in range(3):
            mean = 0.0
            for rng in rngs:
                x = rng.standard_normal((8, 12)).astype(np.float32)
                y = np.eye(4, dtype=np.float32)[rng.integers(0, 4, 8)]
                for p, a in zip(model.parameters(), params):
                    p.data, p.grad = Tensor(a.astype(np.float32), device=dev).data, None
                nn.CrossEntropyLoss()(model(Tensor(x, device=dev)), Tensor(y, device=dev)).backward()
                mean = mean + 0.5 * np.concatenate([p.grad.numpy().reshape(-1) for p in model.parameters()]).astype(np.float64)
                Graph.free_graph()
            norm = np.sqrt((mean ** 2).sum())
            clipped += norm > 0.1
            mean, at = mean * min(1.0, 0.1 / (norm + 1e-6)), 0
            for k, a in enumerate(params):
                params[k] = a - 0.5 * mean[at:at + a.size].reshape(a.shape)
                at += a.size
        assert clipped == 3
        for a, want in zip(outs[0]["params"], params):
            assert_close(np.array(a), want, 1e-5)
    finally:
        backend_api.unregister_device("cpu")


@pytest.mark.parametrize("magnitude", [1e30, 1e-30, 3e38, 1e-44])
def test_clip_of_magnitudes_whose_squares_no_float_holds(cpu_oracle, magnitude):
    """the norm is held in double: 2 roundings (it and the factor) and the product's, u = 2^-24 each"""
    from deepflows_amd import optim
    rng = np.random.default_rng(6)
    arrays = [(magnitude * rng.uniform(0.25, 1.0, s)).astype(np.float32) for s in ((3, 4), (7,))]
    params = _params(cpu_oracle, arrays)
    norm = math.sqrt(sum(float((a.astype(np.float64) ** 2).sum()) for a in arrays))
    most = 0.5 * norm
    total = optim.clip_grad_norm_(params, most, error_if_nonfinite=norm < 3.4e38)
    want = np.float32(norm) if norm < 3.4e38 else np.inf
    assert abs(float(total.numpy()[0]) - want) <= 2 ** -23 * want + 2 ** -149 or float(total.numpy()[0]) == want
    for a, p in zip(arrays, params):
        expected = a.astype(np.float64) * min(1.0, most / (norm + 1e-6))
        assert np.all(np.abs(p.grad.numpy() - expected) <= 2 ** -22 * np.abs(expected) + 2 ** -149)


def test_operands_without_an_axis_are_refused(cpu_oracle):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    new = lambda *s: Tensor(np.zeros(s, np.float32), device=cpu_oracle)
    with pytest.raises(ValueError):
        F.rms_norm(new(3, 1), new())
    with pytest.raises(ValueError):
        F.rms_norm(new(), None)
    with pytest.raises(ValueError):
        F.linear_cross_entropy(new(4, 3), new(3, 1), new(), new(4))
    with pytest.raises(ValueError):
        F.linear_cross_entropy(new(4, 3), new(3, 1), None, new())
