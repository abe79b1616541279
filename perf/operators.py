"""Cases that measure the operators around the last layers of a network with many classes, and what they are checked against.

Three operators, each with its gradient where it has one:

    linear_cross_entropy   loss = cross-entropy(x . W + b, class indices), d loss / dx, dW, db; the logits are not an output
    rms_norm               h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight over the last axis, and the way back
    clip_grad_norm_        the norm over all gradients of a network, and the gradients scaled down to `max_norm`

`run` computes a case in its plain form, elementary torch operations in 32 bits, or -- with `own` set -- through this package's
functions; `exact` computes it in 64 bits from the definitions.  Everything is fp32, the framework's only type; class indices
come as the whole numbers a 32-bit float holds exactly, as every array of the framework does.
"""
import math

import torch

own = False

IGNORED = -100


# ---- the cases -----------------------------------------------------------------------------------------------------------
def _loss(name, rows, width, classes, smoothing=0.0, ignored=0.0, bias=True, train=True):
    return {"name": name, "op": "loss", "rows": rows, "width": width, "classes": classes, "smoothing": smoothing,
            "ignored": ignored, "bias": bias, "train": train}


def _norm(name, rows, width, residual=True, train=True):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "residual": residual, "train": train}


def _clip(name, network, scale, max_norm, kind="2"):
    return {"name": name, "op": "clip", "network": network, "scale": scale, "max_norm": max_norm, "kind": kind}


def listed():
    return [
        # a small batch of a classifier with a thousand classes: every launch counts
        _loss("loss 64x256x1000", 64, 256, 1000),
        # an odd vocabulary, smoothed targets, a padded batch (one row in ten is not counted)
        _loss("loss 509x512x10007", 509, 512, 10007, smoothing=0.05, ignored=0.1),
        # an ordinary training step over a vocabulary
        _loss("loss 2048x768x32000", 2048, 768, 32000, ignored=0.02, bias=False),
        # a large one: the logits alone would be 1.6 GB
        _loss("loss 8192x1024x50001", 8192, 1024, 50001, smoothing=0.1),
        # the loss of held-out data: no gradients
        _loss("loss 1500x1024x30011 eval", 1500, 1024, 30011, train=False),
        # one short sequence through a narrow layer: every launch counts
        _norm("norm 33x512", 33, 512),
        # a batch of an ordinary width
        _norm("norm 4096x1024", 4096, 1024),
        # many rows of a wide layer: 268 MB an array
        _norm("norm 16384x4096", 16384, 4096),
        # rows of an odd width, no residual, no gradients: an evaluation pass
        _norm("norm 2500x1531 eval", 2500, 1531, residual=False, train=False),
        # the four arrays of the 784-256-10 perceptron
        _clip("clip perceptron", "mlp", 1, 1.0),
        # the 62 arrays of the CIFAR ResNet-18
        _clip("clip resnet18", "resnet", 1, 5.0),
        # 48 arrays of a network with large layers, 0.4 G elements
        _clip("clip 0.4 G", "layers", 2048, 1.0),
    ]


def _spread(rng, low, high):
    """a whole number between low and high, spread over its logarithm"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "norm", "clip"])
    if kind == "loss":
        width, classes = _spread(rng, 16, 2048), _spread(rng, 10, 100000)
        most = min(8192, max(1, 8192 * 1024 * 50001 // (width * classes)))
        rows = _spread(rng, 1, most)
        return {k: v for k, v in _loss("", rows, width, classes, smoothing=rng.choice([0.0, 0.05, 0.1]),
                                       ignored=rng.choice([0.0, 0.0, 0.2]), bias=rng.random() < 0.7,
                                       train=rng.random() < 0.8).items() if k != "name"}
    if kind == "norm":
        width = _spread(rng, 8, 16384)
        rows = _spread(rng, 1, max(1, (1 << 26) // width))
        return {k: v for k, v in _norm("", rows, width, residual=rng.random() < 0.7, train=rng.random() < 0.8).items()
                if k != "name"}
    network = rng.choice(["mlp", "resnet", "layers", "layers"])
    scale = {"mlp": _spread(rng, 2, 64), "resnet": _spread(rng, 2, 11), "layers": _spread(rng, 5, 2048)}[network]
    return {k: v for k, v in _clip("", network, scale, rng.choice([0.5, 1.0, 5.0, 1e6]), rng.choice(["2", "2", "inf"])).items()
            if k != "name"}


def _shapes(case):
    """the shapes of the gradients of a `clip` case"""
    s = case["scale"]
    if case["network"] == "mlp":
        return [(784, 256 * s), (1, 256 * s), (256 * s, 10), (1, 10)]
    if case["network"] == "resnet":                # (channels 32 / 64 / 128 / 256, two blocks a stage, as the CIFAR script's model)
        out, cin = [(32 * s, 3, 3, 3), (1, 32 * s, 1, 1), (1, 32 * s, 1, 1)], 32 * s
        for stage, c in enumerate((32 * s, 64 * s, 128 * s, 256 * s)):
            for block in range(2):
                out += [(c, cin, 3, 3), (1, c, 1, 1), (1, c, 1, 1), (c, c, 3, 3), (1, c, 1, 1), (1, c, 1, 1)]
                if block == 0 and stage > 0:
                    out += [(c, cin, 1, 1), (1, c, 1, 1), (1, c, 1, 1)]
                cin = c
        return out + [(256 * s, 10), (1, 10)]
    out = []                                       # (eight layers of a width: two products, their biases, two norms)
    for _ in range(8):
        out += [(s, 4 * s), (1, 4 * s), (4 * s, s), (1, s), (s,), (s, 4 * s)]
    return out


def _counts(case):
    return [math.prod(s) for s in _shapes(case)]


# ---- inputs --------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def rand(*shape):
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)

    s = {"case": case}
    if case["op"] == "loss":
        n, d, v = case["rows"], case["width"], case["classes"]
        s["x"] = rand(n, d)
        s["w"] = rand(d, v) * (1.5 / math.sqrt(d))
        s["b"] = rand(1, v) if case["bias"] else None
        # (a few classes are much more frequent than the others, as in text)
        u = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)
        t = (float(v) ** u).long().clamp_(1, v) - 1
        out = torch.rand(n, generator=gen, device=dev) < case["ignored"]
        out[0] = False
        s["target"] = torch.where(out, torch.full_like(t, IGNORED), t)
        names = ["x", "w", "b"]
        if own:
            s["target"] = s["target"].float()
            names.append("target")
    elif case["op"] == "norm":
        n, d = case["rows"], case["width"]
        s["x"], s["w"] = rand(n, d), 1 + 0.1 * rand(d)
        s["r"] = 2 * rand(n, d) if case["residual"] else None
        if case["train"]:
            s["dy"] = rand(n, d)
            s["dh"] = rand(n, d) if case["residual"] else None
        names = ["x", "w", "r", "dy", "dh"]
    else:
        s["grads"] = [rand(*shape) * 10.0 ** (-(k % 3)) for k, shape in enumerate(_shapes(case))]
        names = ["grads"]
    if own:
        # the same memory as arrays of the framework, which is what a program of its user has in hand
        s["own"] = {k: [_array(t) for t in s[k]] if isinstance(s[k], list) else _array(s[k])
                    for k in names if s.get(k) is not None}
        if case["op"] == "clip":
            s["own"]["params"] = _parameters(s["own"]["grads"])
    return s


def run(state):
    case = state["case"]
    if own:
        return {"loss": _own_loss, "norm": _own_norm, "clip": _own_clip}[case["op"]](case, state["own"])
    return {"loss": _plain_loss, "norm": _plain_norm, "clip": _plain_clip}[case["op"]](case, state)


# ---- plain forms ---------------------------------------------------------------------------------------------------------
def _plain_loss(case, s):
    x, w, b, t = s["x"], s["w"], s["b"], s["target"]
    n, v, eps = case["rows"], case["classes"], case["smoothing"]
    counted = t != IGNORED
    place = torch.where(counted, t, torch.zeros_like(t)).unsqueeze(1)
    count = counted.sum().clamp(min=1).float()
    logits = x @ w
    if b is not None:
        logits += b
    logits -= logits.max(dim=1, keepdim=True).values
    e = torch.exp(logits)
    z = e.sum(dim=1, keepdim=True)
    row = torch.log(z) - (1.0 - eps) * logits.gather(1, place)
    if eps:
        row = row - eps * (logits.sum(dim=1, keepdim=True) / v)
    row = row.squeeze(1) * counted
    loss = (row.sum() / count).reshape(1)
    if not case["train"]:
        return [loss]
    dl = e.div_(z)
    if eps:
        dl -= eps / v
    dl.scatter_add_(1, place, torch.full((n, 1), eps - 1.0, device=dl.device))
    dl *= (counted / count).unsqueeze(1)
    out = [loss, dl @ w.T, x.T @ dl]
    return out + [dl.sum(dim=0, keepdim=True)] if b is not None else out


NORM_EPS = 1e-6


def _plain_norm(case, s):
    x, w, r = s["x"], s["w"], s["r"]
    h = x + r if r is not None else x
    rs = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + NORM_EPS)
    nh = h * rs
    y = nh * w
    out = [y, h] if r is not None else [y]
    if not case["train"]:
        return out
    g = s["dy"] * w
    c = (g * nh).mean(dim=1, keepdim=True)
    dx = rs * (g - nh * c)
    if r is not None:
        dx = dx + s["dh"]
    return out + [dx, (s["dy"] * nh).sum(dim=0)]


def _plain_clip(case, s):
    if case["kind"] == "inf":
        total = torch.stack([g.abs().max() for g in s["grads"]]).max()
    else:
        total = torch.sqrt(torch.stack([(g * g).sum() for g in s["grads"]]).sum())
    scale = torch.clamp(case["max_norm"] / (total + 1e-6), max=1.0)
    return [total.reshape(1)] + [g * scale for g in s["grads"]]


# ---- the framework's operators -------------------------------------------------------------------------------------------
class _Shared:
    """memory of a torch tensor as a flat array of the framework (what its own arrays offer: ptr and size)"""
    __slots__ = ("ptr", "size", "_keep")

    def __init__(self, t):
        self.ptr, self.size, self._keep = t.data_ptr(), t.numel(), t


class _Shown:
    """an array of the framework as torch takes it, without a copy"""
    __slots__ = ("__cuda_array_interface__", "_keep")

    def __init__(self, a):
        a = a.compact()
        self._keep = a
        self.__cuda_array_interface__ = {"shape": tuple(int(v) for v in a.shape), "typestr": "<f4", "version": 2,
                                         "data": (a._handle.ptr, False), "strides": None}


class _Results(list):
    """arrays of the framework; whoever goes through them gets torch tensors over the same memory"""

    def __iter__(self):
        return (torch.as_tensor(_Shown(a), device="cuda") for a in list.__iter__(self))


def _array(t):
    from deepflows_amd import backend_api
    from deepflows_amd.backend_selection import BackendTensor
    t = t.contiguous()
    return BackendTensor.make(tuple(t.shape), device=backend_api.Device("hip"), handle=_Shared(t))


def _parameters(grads):
    from deepflows_amd import nn
    from deepflows_amd.tensor import Tensor
    return [nn.Parameter(Tensor(g)) for g in grads]


def _leaf(a, train):
    from deepflows_amd.tensor import Tensor
    return Tensor(a, device=a.device, requires_grad=train) if a is not None else None


def _own_loss(case, s):
    from deepflows_amd.autograd import no_grad
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph
    train = case["train"]
    x, w, b, t = _leaf(s["x"], train), _leaf(s["w"], train), _leaf(s.get("b"), train), _leaf(s["target"], False)
    if not train:
        with no_grad():
            return _Results([F.linear_cross_entropy(x, w, b, t, label_smoothing=case["smoothing"]).data])
    loss = F.linear_cross_entropy(x, w, b, t, label_smoothing=case["smoothing"])
    loss.backward()
    Graph.free_graph_all()
    return _Results([loss.data] + [p.grad for p in (x, w, b) if p is not None])


def _own_norm(case, s):
    from deepflows_amd.autograd import no_grad
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph
    train = case["train"]
    x, w, r = _leaf(s["x"], train), _leaf(s["w"], train), _leaf(s.get("r"), train)
    if not train:
        with no_grad():
            y = F.rms_norm(x, w, NORM_EPS, residual=r)
        return _Results([y.data] if r is None else [v.data for v in y])
    y = F.rms_norm(x, w, NORM_EPS, residual=r)
    y, h = y if r is not None else (y, None)
    _rest(y, h, s["dy"], s.get("dh")).backward()
    Graph.free_graph_all()
    return _Results([y.data] + ([h.data] if h is not None else []) + [x.grad, w.grad])


def _rest(y, h, dy, dh):
    """the rest of a network: a node of the tape that takes y (and h) in and hands the given gradients back"""
    from deepflows_amd.backend_selection import BackendTensor
    from deepflows_amd import tensor

    class One(tensor.UnaryOperator):
        def forward(self, x):
            return BackendTensor.make((1,), device=x.device)

        def grad_fn(self, node, grad):
            return dy

    class Two(tensor.BinaryOperator):
        def forward(self, x, y):
            return BackendTensor.make((1,), device=x.device)

        def grad_fn(self, node, grad):
            return dy if node is self.parents[0] else dh

    return One(y) if h is None else Two(y, h)


def _own_clip(case, s):
    from deepflows_amd import optim
    for p, g in zip(s["params"], s["grads"]):
        p.grad = g
    total = optim.clip_grad_norm_(s["params"], case["max_norm"], norm_type=float(case["kind"]))
    return _Results([total.data] + [p.grad for p in s["params"]])


# ---- 64 bits -------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "loss":
        return _exact_loss(case, s)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    if case["kind"] == "inf":
        total = max(float(g.abs().max()) for g in s["grads"])
    else:
        total = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in s["grads"]))
    scale = min(1.0, case["max_norm"] / (total + 1e-6))
    return [torch.tensor([total], dtype=torch.float64)] + [g.double() * scale for g in s["grads"]]


def _exact_loss(case, s):
    """-sum_j q_j log p_j averaged over the counted rows, and its derivatives, a block of rows at a time"""
    x, w, t = s["x"].double(), s["w"].double(), s["target"]
    v, eps = case["classes"], case["smoothing"]
    b = s["b"].double() if s["b"] is not None else torch.zeros(1, v, dtype=torch.float64, device=x.device)
    count = max(1, int((t != IGNORED).sum()))
    loss = torch.zeros((), dtype=torch.float64, device=x.device)
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    for i in range(0, case["rows"], 2048):
        keep = torch.nonzero(t[i:i + 2048] != IGNORED).flatten()
        if keep.numel() == 0:
            continue
        xi, ti = x[i:i + 2048][keep], t[i:i + 2048][keep]
        log_p = torch.addmm(b, xi, w)
        log_p = log_p - torch.logsumexp(log_p, dim=1, keepdim=True)
        q = torch.full_like(log_p, eps / v)
        q[torch.arange(len(ti), device=x.device), ti] += 1.0 - eps
        loss = loss - (q * log_p).sum() / count
        if case["train"]:
            d = (log_p.exp() - q) / count
            dx[i:i + 2048].index_copy_(0, keep, d @ w.t())
            dw += xi.t() @ d
            db += d.sum(dim=0, keepdim=True)
    out = [loss.reshape(1)]
    if case["train"]:
        out += [dx, dw] + ([db] if s["b"] is not None else [])
    return out


def _exact_norm(case, s):
    """y_i = w_i h_i / R with R^2 = mean(h^2) + eps; dy_i / dh_j = w_i (delta_ij / R - h_i h_j / (width R^3))"""
    h = s["x"].double()
    if s["r"] is not None:
        h = h + s["r"].double()
    w, width = s["w"].double(), case["width"]
    big = torch.sqrt(h.square().sum(dim=1, keepdim=True) / width + NORM_EPS)
    out = [h / big * w] + ([h] if s["r"] is not None else [])
    if not case["train"]:
        return out
    dy = s["dy"].double()
    along = torch.linalg.vecdot(dy * w, h).unsqueeze(1)
    dh = dy * w / big - h * along / (width * big ** 3)
    if s["r"] is not None:
        dh = dh + s["dh"].double()
    return out + [dh, torch.linalg.vecdot(dy, h / big, dim=0)]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "loss":
        n, d, v = case["rows"], case["width"], case["classes"]
        arrays = n * d + d * v + (v if case["bias"] else 0)
        return {"bytes": 4 * (arrays * (2 if case["train"] else 1) + n + 1), "flops": (6 if case["train"] else 2) * n * d * v}
    if case["op"] == "norm":
        n, d = case["rows"], case["width"]
        arrays = 2 + (2 if case["residual"] else 0) + ((2 + (1 if case["residual"] else 0)) if case["train"] else 0)
        return {"bytes": 4 * (arrays * n * d + d * (2 if case["train"] else 1)),
                "flops": n * d * (12 if case["train"] else 4)}
    n = sum(_counts(case))
    return {"bytes": 4 * (2 * n + 1), "flops": 3 * n}
