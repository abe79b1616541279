"""GPU: the norm, the vocabulary loss and the clipping as they are used together: a residual network whose last norm feeds a head
with many classes, its gradients clipped, its parameters updated -- eagerly, captured, through the epoch loop.

Against the oracle (the same step in 64 bits, NumPy): 1e-4 relative of the largest value, the framework's bound for
whole steps; captured steps against eager ones: bit for bit."""
import numpy as np
import pytest

from conftest import assert_close

pytestmark = pytest.mark.gpu

V, D, K = 1503, 72, 40


def _build(dev, seed=3):
    from deepflows_amd import nn

    class Network(nn.Module):
        def __init__(self):
            super().__init__()
            self.fc0, self.fc1 = nn.Linear(K, D, device=dev), nn.Linear(D, D, device=dev)
            self.norm0, self.norm1 = nn.RMSNorm(D, device=dev), nn.RMSNorm(D, device=dev)

        def forward(self, x):
            h = self.fc0(x)
            y = nn.functional.relu(self.fc1(self.norm0(h)))
            return self.norm1(y, h)[0]

    np.random.seed(seed)
    net = Network()
    head = nn.Linear(D, V, device=dev)
    return net, nn.LinearCrossEntropyLoss(head, label_smoothing=0.1), list(net.parameters()) + list(head.parameters())


def _batches(n, rows):
    rng = np.random.default_rng(11)
    out = []
    for _ in range(n):
        t = rng.integers(0, V, rows).astype(np.float32)
        t[rng.random(rows) < 0.2] = -100
        out.append((rng.standard_normal((rows, K)).astype(np.float32), t))
    return out


def _norm(h, g):
    r = 1.0 / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6)
    return h * r * g, r


def _norm_gradient(dy, h, g, r):
    """(dh, dg) of y = h r g"""
    n = h * r
    return r * (dy * g - n * (dy * g * n).mean(-1, keepdims=True)), (dy * n).sum(0)


def _loss_and_gradients(ps, x, t):
    w0, b0, w1, b1, g0, g1, wh, bh = ps
    h = x @ w0 + b0
    y0, r0 = _norm(h, g0)
    z = y0 @ w1 + b1
    h1 = np.maximum(z, 0.0) + h
    y1, r1 = _norm(h1, g1)
    l = y1 @ wh + bh
    l = l - l.max(1, keepdims=True)
    logp = l - np.log(np.exp(l).sum(1, keepdims=True))
    counted = t != -100
    q = np.full(l.shape, 0.1 / V)
    q[np.arange(len(t)), np.where(counted, t, 0).astype(int)] += 0.9
    q[~counted] = 0.0
    n = counted.sum()
    dl = (np.exp(logp) * counted[:, None] - q) / n
    dh1, dg1 = _norm_gradient(dl @ wh.T, h1, g1, r1)
    dz = dh1 * (z > 0)
    dh0, dg0 = _norm_gradient(dz @ w1.T, h, g0, r0)
    dh = dh0 + dh1
    return -(q * logp).sum() / n, [x.T @ dh, dh.sum(0), y0.T @ dz, dz.sum(0), dg0, dg1, y1.T @ dl, dl.sum(0)]


def _oracle(arrays, batches, max_norm, lr):
    """the same steps in 64 bits: (losses, norms, parameters)"""
    ps = [a.astype(np.float64) for a in arrays]
    losses, norms = [], []
    for x, t in batches:
        loss, grads = _loss_and_gradients(ps, x.astype(np.float64), t)
        total = np.sqrt(sum((g * g).sum() for g in grads))
        scale = min(1.0, max_norm / (total + 1e-6))
        ps = [p - lr * scale * g.reshape(p.shape) for p, g in zip(ps, grads)]
        losses.append(loss)
        norms.append(total)
    return losses, norms, ps


def test_steps_against_the_oracle(hip_device):
    from deepflows_amd import optim
    from deepflows_amd.tensor import Graph, Tensor
    net, crit, params = _build(hip_device)
    opt = optim.SGD(params, lr=0.5)
    named = [net.fc0.weight, net.fc0.bias, net.fc1.weight, net.fc1.bias, net.norm0.weight, net.norm1.weight,
             crit.linear.weight, crit.linear.bias]
    batches = _batches(3, 50)
    want = _oracle([p.numpy() for p in named], batches, 0.2, 0.5)
    losses, norms = [], []
    for x, t in batches:
        loss = crit(net(Tensor(x, device=hip_device)), Tensor(t, device=hip_device))
        opt.zero_grad()
        loss.backward()
        norms.append(float(optim.clip_grad_norm_(opt.params, 0.2).numpy()[0]))
        opt.step()
        losses.append(float(loss.numpy()[0]))
        Graph.free_graph()
    assert min(want[1]) > 0.2                                  # (the clipping does something)
    assert_close(losses, want[0], 1e-4, "losses")
    assert_close(norms, want[1], 1e-4, "norms")
    for p, w in zip(named, want[2]):
        assert_close(p.numpy(), w, 1e-4, "parameter")


@pytest.mark.parametrize("kind", ["SGD", "Adam"])
@pytest.mark.parametrize("steps_per_graph", [1, 2])
def test_captured_steps_equal_eager_ones(hip_device, kind, steps_per_graph):
    from deepflows_amd import optim, workloads
    from deepflows_amd.graph_step import CapturedTrainStep
    from deepflows_amd.tensor import Graph, Tensor
    batches = _batches(4, 37)
    make = (lambda p: optim.SGD(p, lr=0.3, momentum=0.9)) if kind == "SGD" else (lambda p: optim.Adam(p, lr=1e-2))

    net, crit, params = _build(hip_device)
    opt = make(params)
    want = []
    for x, t in batches:
        loss, _ = workloads.train_step(net, crit, opt, Tensor(x, device=hip_device), Tensor(t, device=hip_device), max_grad_norm=0.3)
        want.append(float(loss.numpy()[0]))
        Graph.free_graph()
    want_params = [p.numpy().copy() for p in params]
    Graph.free_graph_all()

    net, crit, params = _build(hip_device)
    opt = make(params)
    xs = [Tensor(batches[0][0], device=hip_device) for _ in range(steps_per_graph)]
    ts = [Tensor(batches[0][1], device=hip_device) for _ in range(steps_per_graph)]
    step = CapturedTrainStep(net, crit, opt, xs if steps_per_graph > 1 else xs[0], ts if steps_per_graph > 1 else ts[0],
                             steps_per_graph=steps_per_graph, max_grad_norm=0.3)
    got = []
    for k, (x, t) in enumerate(batches):
        if k % steps_per_graph == 0:
            for j in range(steps_per_graph):
                hip_device.mod.from_numpy(batches[k + j][0], xs[j].data._handle)
                hip_device.mod.from_numpy(batches[k + j][1], ts[j].data._handle)
        got.append(float(step.replay().numpy()[0]))
    last = slice(steps_per_graph - 1, None, steps_per_graph)    # (the loss of a graph's last step is what a replay shows)
    assert got[last] == want[last]
    assert float(step.grad_norm.numpy()[0]) > 0.0
    for p, w in zip(params, want_params):
        assert np.array_equal(p.numpy(), w)
    step.destroy()
    Graph.free_graph_all()


def test_a_changed_gradient_factor_is_refused(hip_device):
    from deepflows_amd import optim
    from deepflows_amd.graph_step import CapturedTrainStep
    from deepflows_amd.tensor import Graph, Tensor
    net, crit, params = _build(hip_device)
    opt = optim.SGD(params, lr=0.1)
    x, t = _batches(1, 8)[0]
    step = CapturedTrainStep(net, crit, opt, Tensor(x, device=hip_device), Tensor(t, device=hip_device), max_grad_norm=1.0)
    step.replay()
    opt.grad_scale = 0.5
    with pytest.raises(RuntimeError):
        step.replay()
    step.destroy()
    Graph.free_graph_all()


def test_gradient_bucket_clipping_and_the_optimizers_factor(hip_device):
    """gradients that live in a data-parallel bucket (its slices begin at any element), summed over two ranks' worth by hand"""
    from deepflows_amd import optim, parallel
    from deepflows_amd.tensor import Graph, Tensor

    class TwoTimes(parallel.Communicator):
        exchanges, world = True, 2

        def allreduce_sum(self, flat, overlap=False):
            flat.device.mod.axpy(flat._handle, (flat * 1.0)._handle, 1.0)
            return flat

    net, crit, params = _build(hip_device)
    x, t = _batches(1, 20)[0]
    xt, tt = Tensor(x, device=hip_device), Tensor(t, device=hip_device)
    crit(net(xt), tt).backward()
    plain = np.concatenate([p.grad.numpy().reshape(-1) for p in params]).astype(np.float64)
    Graph.free_graph()
    for p in params:
        p.grad = None
    bucket = parallel.GradientBucket(params, TwoTimes())
    crit(net(xt), tt).backward()
    bucket.sync()
    total = float(optim.clip_grad_norm_(params, 0.1, grad_scale=0.5).numpy()[0])
    want = np.sqrt((plain ** 2).sum())
    assert abs(total - want) <= 1e-6 * want
    got = np.concatenate([p.grad.numpy().reshape(-1) for p in params])
    assert_close(got, 2 * plain * min(1.0, 0.1 / (want + 1e-6)), 1e-6)
    bucket.release()
    Graph.free_graph_all()


def test_the_epoch_loop_clips(hip_device):
    """full batches through the captured step and a ragged one eagerly: the parameters of the plain loop, bit for bit"""
    from deepflows_amd import nn, optim, workloads
    from deepflows_amd.tensor import Graph
    from deepflows_amd.utils.data import data_loader
    from deepflows_amd.utils.train_loop import EpochTrainer
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((40, 3, 32, 32)) * 0.8).astype(np.float32)
    y = rng.integers(0, 10, 40)
    finals = []
    for capture in (True, False):
        np.random.seed(3)
        model = workloads.ResNet18(10, device=hip_device, register_blocks=True)
        opt = optim.Adam(model.parameters(), lr=1e-3)
        trainer = EpochTrainer(model, nn.CrossEntropyLoss(), opt, hip_device, capture=capture, max_grad_norm=0.05)
        np.random.seed(9)
        losses = trainer.run_epoch(data_loader(x, y, 16, shuffle=True), 0, 2)
        finals.append((losses, [p.numpy().copy() for p in opt.params]))
        trainer.destroy()
        Graph.free_graph_all()
    assert np.array_equal(finals[0][0], finals[1][0])
    for a, b in zip(finals[0][1], finals[1][1]):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("inside", [True, False])
def test_a_captured_step_clips_behind_the_exchange(hip_device, inside):
    """the gradients of a bucket, clipped in the captured graph or eagerly behind its replays: the eager steps' parameters"""
    from deepflows_amd import optim, parallel, workloads
    from deepflows_amd.graph_step import CapturedTrainStep
    from deepflows_amd.tensor import Graph, Tensor

    class Doubling(parallel.Communicator):
        exchanges, world = True, 2

        def allreduce_sum(self, flat, overlap=False):
            flat.device.mod.axpy(flat._handle, (flat * 1.0)._handle, 1.0)
            return flat

    batches, runs = _batches(4, 30), []
    for captured in (False, True):
        net, crit, params = _build(hip_device)
        opt = optim.SGD(params, lr=0.3, momentum=0.9)
        opt.grad_scale = 0.5
        bucket = parallel.GradientBucket(opt.params, Doubling())
        x, t = (Tensor(a, device=hip_device) for a in batches[0])
        step = None
        if captured:
            step = CapturedTrainStep(net, crit, opt, x, t, sync=bucket.sync, capture_exchange=inside, max_grad_norm=0.2)
            assert step.exchange_captured == inside
        norms = []
        for bx, bt in batches:
            hip_device.mod.from_numpy(bx, x.data._handle)
            hip_device.mod.from_numpy(bt, t.data._handle)
            if captured:
                step.replay()
                norms.append(float(step.grad_norm.numpy()[0]))
            else:
                workloads.train_step(net, crit, opt, x, t, sync=bucket.sync, max_grad_norm=0.2)
                Graph.free_graph()
        assert all(n > 0.2 for n in norms)
        runs.append([p.numpy().copy() for p in params])
        if step is not None:
            step.destroy()
        bucket.release()
        Graph.free_graph_all()
    for a, b in zip(*runs):
        assert np.array_equal(a, b)


def test_a_negative_norm_is_refused_before_anything_is_captured(hip_device):
    from deepflows_amd import optim
    from deepflows_amd.graph_step import CapturedTrainStep
    from deepflows_amd.tensor import Graph, Tensor
    net, crit, params = _build(hip_device)
    x, t = (Tensor(a, device=hip_device) for a in _batches(1, 8)[0])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            CapturedTrainStep(net, crit, optim.SGD(params, lr=0.1), x, t, max_grad_norm=bad)
    Graph.free_graph_all()


def test_the_overlapped_exchange_clips(hip_device):
    """both halves of the gradients on their way when the clipping begins: the eager step's parameters, bit for bit.  (One rank
    without a collective: what is checked is that the clipping sees the gradients of both graphs.)"""
    from deepflows_amd import nn, optim, parallel, workloads
    from deepflows_amd.graph_step import OverlappedCapturedTrainStep
    from deepflows_amd.tensor import Graph, Tensor

    class Alone(parallel.Communicator):
        exchanges = True

        def allreduce_sum(self, flat, overlap=False):
            return flat

    rng = np.random.default_rng(3)
    xs = Tensor(rng.standard_normal((32, 3, 32, 32)).astype(np.float32), device=hip_device)
    ys = Tensor(np.eye(10, dtype=np.float32)[rng.integers(0, 10, 32)], device=hip_device)
    crit, comm, runs = nn.CrossEntropyLoss(), Alone(), []
    for overlapped in (False, True):
        np.random.seed(1)
        m = workloads.ResNet18(device=hip_device, register_blocks=True)
        o = optim.Adam(workloads.all_block_parameters(m), lr=1e-3)
        bucket = parallel.GradientBucket(o.params, comm)
        for _ in range(1 if overlapped else 4):
            workloads.train_step(m, crit, o, xs, ys, sync=bucket.sync, max_grad_norm=0.1)
            Graph.free_graph()
        if overlapped:
            late, early = workloads.late_and_early_parameters(m, o.params)
            step = OverlappedCapturedTrainStep(m, crit, o, xs, ys, parallel.GradientBucket(late, comm),
                                               parallel.GradientBucket(early, comm), max_grad_norm=0.1)
            for _ in range(3):
                step.replay()
        runs.append([p.numpy().copy() for p in o.params])
        Graph.free_graph_all()
    for a, b in zip(*runs):
        assert np.array_equal(a, b)


def test_a_changed_norm_of_a_captured_step_is_refused(hip_device):
    from deepflows_amd import optim
    from deepflows_amd.graph_step import CapturedTrainStep
    from deepflows_amd.tensor import Graph, Tensor
    net, crit, params = _build(hip_device)
    x, t = (Tensor(a, device=hip_device) for a in _batches(1, 8)[0])
    for first, second in ((1.0, 2.0), (1.0, None), (None, 1.0)):
        step = CapturedTrainStep(net, crit, optim.SGD(params, lr=0.1), x, t, max_grad_norm=first)
        step.replay()
        step.max_grad_norm = second
        with pytest.raises(RuntimeError):
            step.replay()
        step.max_grad_norm = first
        step.replay()
        step.destroy()
    Graph.free_graph_all()


def test_the_epoch_loop_clips_to_the_norm_it_has_now(hip_device):
    """another norm for the second epoch and none for the third, captured and eagerly: the same losses and parameters, bit for bit"""
    from deepflows_amd import nn, optim, workloads
    from deepflows_amd.tensor import Graph
    from deepflows_amd.utils.data import data_loader
    from deepflows_amd.utils.train_loop import EpochTrainer
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((40, 3, 32, 32)) * 0.8).astype(np.float32)
    y = rng.integers(0, 10, 40)
    finals = []
    for capture in (True, False):
        np.random.seed(4)
        model = workloads.ResNet18(10, device=hip_device, register_blocks=True)
        opt = optim.SGD(model.parameters(), lr=0.1)
        trainer = EpochTrainer(model, nn.CrossEntropyLoss(), opt, hip_device, capture=capture, max_grad_norm=0.05)
        losses = []
        for epoch, norm in enumerate((0.05, 0.5, None)):
            trainer.max_grad_norm = norm
            np.random.seed(9 + epoch)
            losses.append(trainer.run_epoch(data_loader(x, y, 16, shuffle=True), epoch, 3))
        finals.append((losses, [p.numpy().copy() for p in opt.params]))
        trainer.destroy()
        Graph.free_graph_all()
    for a, b in zip(*[f[0] for f in finals]):
        assert np.array_equal(a, b)
    for a, b in zip(*[f[1] for f in finals]):
        assert np.array_equal(a, b)


def test_a_step_that_clips_behind_its_graph_follows_both_settings(hip_device):
    """the exchange outside the graph, and the clipping behind it: another norm or factor between replays is what the eager step does"""
    from deepflows_amd import optim, parallel, workloads
    from deepflows_amd.graph_step import CapturedTrainStep
    from deepflows_amd.tensor import Graph, Tensor

    class Same(parallel.Communicator):
        exchanges = True

        def allreduce_sum(self, flat, overlap=False):
            return flat

    batches, runs = _batches(3, 24), []
    for captured in (False, True):
        net, crit, params = _build(hip_device)
        opt = optim.SGD(params, lr=0.3)
        bucket = parallel.GradientBucket(opt.params, Same())
        x, t = (Tensor(a, device=hip_device) for a in batches[0])
        step = None
        if captured:
            step = CapturedTrainStep(net, crit, opt, x, t, sync=bucket.sync, capture_exchange=False, max_grad_norm=0.2)
        for (bx, bt), norm, factor in zip(batches, (0.2, 0.1, 0.4), (1.0, 0.5, 2.0)):
            hip_device.mod.from_numpy(bx, x.data._handle)
            hip_device.mod.from_numpy(bt, t.data._handle)
            opt.grad_scale = factor
            if captured:
                step.max_grad_norm = norm
                step.replay()
            else:
                workloads.train_step(net, crit, opt, x, t, sync=bucket.sync, max_grad_norm=norm)
                Graph.free_graph()
        runs.append([p.numpy().copy() for p in params])
        if step is not None:
            step.destroy()
        bucket.release()
        Graph.free_graph_all()
    for a, b in zip(*runs):
        assert np.array_equal(a, b)
