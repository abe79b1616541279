"""GPU: cross entropy of a linear layer over many classes without its logits (F.linear_cross_entropy,
nn.LinearCrossEntropyLoss; dfhip_linear_ce_forward) against the definition in 64 bits.

Tolerances, from the arithmetic (u = 2^-24).  A product of K terms a b is formed from operands that carry at most 2^-22 relative
each (or a floor of 2^-39 of the array's largest magnitude A, B) and summed in fp32 in at most 3 K roundings, independent of each
other: |error| <= (12 + 6 sqrt(3 K)) u sum|a b| + 2^-38 (A sum|b| + B sum|a|), six standard deviations.
Few rows are multiplied in fp32 as they are: operands without an error, K roundings, inside the same bound.
  E   = the largest such error of a row's logits, plus u |l| for the bias;
  row loss: the log-sum-exp and the target's logit move by at most E each, the sums over V (depth V / 256 + 20) and the last
        operations add u (V / 256 + 40) (1 + |lse - l_t|), the smoothing term another E + u (V/256 + 20) mean|l - m|;
  dl  = p - q: p (2 E + (V / 256 + 40) u), 4 u for the subtractions from values up to 1, 2^-22 |dl| + 2^-38 for its operand form;
  dx, dW, db: the product's own error plus the sum of |other operand| times dl's error."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _product_error(a, b):
    """bound on the error of a . b (64-bit copies of fp32 operands), elementwise"""
    K = a.shape[1]
    aa, bb = np.abs(a), np.abs(b)
    fl = 2.0 ** -38 * (aa.max(initial=0.0) * bb.sum(0)[None, :] + bb.max(initial=0.0) * aa.sum(1)[:, None])
    return (12 + 6 * np.sqrt(3 * K)) * U * (aa @ bb) + fl


def _reference(x, w, b, t, mean=True, ignore=-100, e=0.0):
    x, w = x.astype(np.float64), w.astype(np.float64)
    N, V = x.shape[0], w.shape[1]
    l = x @ w
    E = _product_error(x, w)
    if b is not None:
        l = l + b.astype(np.float64).reshape(1, -1)
    E = (E + U * np.where(np.isfinite(l), np.abs(l), 0.0)).max(1, keepdims=True)
    counted = (t != ignore)
    m = l.max(1, keepdims=True)
    p = np.exp(l - m)
    z = p.sum(1, keepdims=True)
    lse = np.log(z) + m
    p = p / z
    q = np.full((N, V), e / V)
    at = np.where(counted, t, 0).astype(np.int64)
    q[np.arange(N), at] += 1 - e
    lt = l[np.arange(N), at][:, None]
    row = lse - (1 - e) * lt - (e * l.mean(1, keepdims=True) if e else 0.0)
    trow = 3 * E + U * (V / 256 + 60) * (1 + np.abs(lse - lt)) + (U * (V / 256 + 30) * np.abs(l - m).mean(1, keepdims=True) if e else 0.0)
    count = max(1, int(counted.sum())) if mean else 1
    keep = counted[:, None].astype(np.float64)
    loss = float((row * keep).sum() / count)
    tloss = float((trow * keep).sum() / count) + U * (N / 256 + 12) * float((np.abs(row) * keep).sum() / count) + 1e-30
    dl = (p - q) * keep
    td = (p * (2 * E + (V / 256 + 40) * U) + 4 * U * (p + q) + 2.0 ** -22 * np.abs(dl) + 2.0 ** -38) * keep
    dx, dw, db = dl @ w.T / count, x.T @ dl / count, dl.sum(0) / count
    tdx = (_product_error(dl, w.T) + td @ np.abs(w).T) / count + 4 * U * np.abs(dx)
    tdw = (_product_error(x.T, dl) + np.abs(x).T @ td) / count + 4 * U * np.abs(dw)
    tdb = (td.sum(0) + (N / 64 + 30) * U * np.abs(dl).sum(0)) / count + 4 * U * np.abs(db)
    tiny = 1e-30
    return (loss, tloss), (dx, tdx + tiny), (dw, tdw + tiny), (db, tdb + tiny)


def _within(got, want, tol, what):
    got = np.asarray(got, np.float64).reshape(np.shape(want))
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} off; worst {np.abs(got - want)[bad].max():.3e} "
                           f"against {np.asarray(tol)[bad].min() if np.ndim(tol) else tol:.3e}")


def _data(N, D, V, seed, ignored=0.0, ignore=-100, bias=True):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((N, D)).astype(np.float32)
    w = (rng.standard_normal((D, V)) * 1.5 / np.sqrt(D)).astype(np.float32)
    b = rng.standard_normal((1, V)).astype(np.float32) if bias else None
    t = rng.integers(0, V, N).astype(np.float32)
    t[rng.random(N) < ignored] = ignore
    return x, w, b, t


def _run(dev, x, w, b, t, scale=None, **kw):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    xt, wt = Tensor(x, device=dev, requires_grad=True), Tensor(w, device=dev, requires_grad=True)
    bt = Tensor(b, device=dev, requires_grad=True) if b is not None else None
    loss = F.linear_cross_entropy(xt, wt, bt, Tensor(t, device=dev), **kw)
    assert tuple(loss.shape) == (1,)
    value = float(loss.numpy()[0])
    (loss if scale is None else loss * scale).backward()
    out = value, xt.grad.numpy(), wt.grad.numpy(), (bt.grad.numpy() if b is not None else None)
    Graph.free_graph_all()
    return out


def _check(dev, x, w, b, t, scale=None, **kw):
    got = _run(dev, x, w, b, t, scale, **kw)
    ref = _reference(x, w, b, t, kw.get("reduction", "mean") == "mean", kw.get("ignore_index", -100), kw.get("label_smoothing", 0.0))
    s = 1.0 if scale is None else abs(scale)
    _within(got[0], ref[0][0], ref[0][1], "loss")
    for g, (want, tol), what in zip(got[1:], ref[1:], ("dx", "dw", "db")):
        if g is not None:
            _within(g, (scale or 1.0) * want, s * tol + 2 * U * s * np.abs(want), what)


SHAPES = [(1, 1, 1), (1, 1, 2), (3, 5, 7), (1, 64, 1000), (2, 33, 31), (31, 32, 33), (64, 256, 1000), (130, 100, 257), (257, 129, 511),
          (300, 48, 4099), (65, 300, 640), (1000, 17, 129), (33, 1031, 77), (512, 512, 512), (640, 256, 2100), (7, 40, 20011)]


@pytest.mark.parametrize("N,D,V", SHAPES)
def test_values_and_gradients(hip_device, N, D, V):
    _check(hip_device, *_data(N, D, V, N + D + V))


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("ignore", [-100, 3])
def test_smoothing_reductions_and_rows_that_are_not_counted(hip_device, reduction, smoothing, ignore):
    x, w, b, t = _data(150, 70, 333, 5, ignored=0.3, ignore=ignore)
    _check(hip_device, x, w, b, t, reduction=reduction, label_smoothing=smoothing, ignore_index=ignore)


# few rows go another way (the fp32 matrix cores, W as it is): one to 64 rows, 32- and 128-column tiles, classes and widths that
# end inside a tile, a step, a window
FEW = [(1, 8, 4), (1, 300, 1003), (2, 7, 5), (5, 37, 33), (8, 64, 127), (9, 65, 129), (20, 129, 1000), (32, 8, 4097), (32, 515, 700),
       (33, 100, 500), (64, 256, 1000), (50, 70, 4), (64, 512, 2001), (47, 33, 50001), (3, 16, 32641), (17, 45, 33003), (32, 130, 50001), (1, 2100, 32770)]


@pytest.mark.parametrize("N,D,V", FEW)
def test_few_rows(hip_device, N, D, V):
    _check(hip_device, *_data(N, D, V, N + D + V, ignored=0.2 if N > 4 else 0.0, bias=D % 2 == 1), label_smoothing=0.1 if V % 2 else 0.0)


@pytest.mark.parametrize("D", [700, 1100])
def test_33_to_64_rows_of_a_large_product(hip_device, D):
    _check(hip_device, *_data(45, D, 48001, 25, ignored=0.1), label_smoothing=0.1)


@pytest.mark.parametrize("N,D,V", [(1, 90, 700), (40, 65, 50001), (64, 700, 5001), (30, 40, 33001), (100, 700, 48001),
                                   (70, 8, 3), (130, 100, 257), (300, 64, 4099), (700, 520, 9001), (70, 2000, 300), (257, 33, 64)])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_evaluation_keeps_no_logits(hip_device, N, D, V, smoothing):
    from deepflows_amd.autograd import no_grad
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    x, w, b, t = _data(N, D, V, 26, ignored=0.3 if N > 1 else 0.0)
    with no_grad():
        loss = F.linear_cross_entropy(*[Tensor(a, device=hip_device) for a in (x, w, b, t)], label_smoothing=smoothing)
    ref = _reference(x, w, b, t, e=smoothing)
    _within(float(loss.numpy()[0]), ref[0][0], ref[0][1], "loss")


@pytest.mark.parametrize("N", [12, 90])
@pytest.mark.parametrize("V", [300, 33000])
def test_masked_runs_of_classes(hip_device, N, V):
    """a bias that takes out whole column tiles, the first and the last among them"""
    from deepflows_amd.autograd import no_grad
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    x, w, b, t = _data(N, 40, V, 27)
    out = np.zeros(V, bool)
    out[:200] = out[-40:] = out[210::5] = True
    t[:] = np.nonzero(~out)[0][t.astype(int) % int((~out).sum())]
    ref = _reference(x, w[:, ~out], b[:, ~out], np.searchsorted(np.nonzero(~out)[0], t).astype(np.float32))
    for low in (-np.inf, np.finfo(np.float32).min):
        c = b.copy()
        c[0, out] = low
        loss, dx, dw, db = _run(hip_device, x, w, c, t)
        _within(loss, ref[0][0], ref[0][1], "loss")
        _within(dx, ref[1][0], 2 * ref[1][1], "dx")
        _within(dw[:, ~out], ref[2][0], 2 * ref[2][1], "dw")
        assert not dw[:, out].any() and not db[0, out].any()
        with no_grad():
            _within(float(F.linear_cross_entropy(*[Tensor(a, device=hip_device) for a in (x, w, c, t)]).numpy()[0]), *ref[0], "loss")


@pytest.mark.parametrize("V", [90, 33000])
def test_few_rows_that_are_not_finite_or_not_counted(hip_device, V):
    x, w, b, t = _data(21, 30, V, 28)
    t[5] = t[20] = -100
    clean = _run(hip_device, np.where(t[:, None] == -100, np.float32(0), x), w, b, t)
    for bad in (np.nan, np.inf, 3e38):
        y = x.copy()
        y[t == -100] = bad
        for a, c in zip(_run(hip_device, y, w, b, t), clean):
            assert np.array_equal(a, c)
        y = x.copy()
        y[11, 3] = bad if bad != 3e38 else -np.inf
        loss, dx, _, _ = _run(hip_device, y, w, b, t)
        assert np.isnan(loss) and np.all(np.isnan(dx[11])) and np.all(np.isfinite(np.delete(dx, 11, 0)[t[np.arange(21) != 11] != -100]))
    for bad in (float(V), -1.0, 2.5, np.nan):
        u = t.copy()
        u[17] = bad
        loss, dx, dw, db = _run(hip_device, x, w, b, u)
        assert np.isnan(loss) and np.all(np.isnan(dx[17])) and np.all(np.isnan(dw)) and np.all(np.isnan(db))
        assert np.all(np.isfinite(np.delete(dx, 17, axis=0)))
    t[:] = -100
    loss, dx, dw, db = _run(hip_device, x, w, b, t)
    assert loss == 0.0 and not dx.any() and not dw.any() and not db.any()


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("N,D,V", [(9, 48, 210), (25, 33, 33003)])
def test_one_gradient_of_few_rows_at_a_time(hip_device, which, N, D, V):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    x, w, b, t = _data(N, D, V, 29)
    ts = [Tensor(a, device=hip_device, requires_grad=k == which) for k, a in enumerate((x, w, b))]
    F.linear_cross_entropy(*ts, Tensor(t, device=hip_device)).backward()
    want, tol = _reference(x, w, b, t)[1 + which]
    _within(ts[which].grad.numpy(), want, tol, "gradient")
    assert all(ts[k].grad is None for k in range(3) if k != which)
    Graph.free_graph_all()


def test_without_a_bias(hip_device):
    _check(hip_device, *_data(90, 64, 700, 6, bias=False))


@pytest.mark.parametrize("scale", [0.5, -3.0])
def test_an_upstream_gradient_other_than_one(hip_device, scale):
    _check(hip_device, *_data(50, 40, 300, 7), scale=scale)


def test_no_row_is_counted(hip_device):
    x, w, b, t = _data(20, 16, 50, 8)
    t[:] = -100
    loss, dx, dw, db = _run(hip_device, x, w, b, t)
    assert loss == 0.0 and not dx.any() and not dw.any() and not db.any()


def test_rows_that_are_not_counted_leave_their_inputs_alone(hip_device):
    """what stands in a row that is not counted does not matter for the others, nor does it reach its own gradient"""
    x, w, b, t = _data(70, 32, 200, 9, ignored=0.4)
    first = _run(hip_device, x, w, b, t)
    y = x.copy()
    y[t == -100] *= 3.0
    second = _run(hip_device, y, w, b, t)
    ref = _reference(x, w, b, t)
    _within(second[0], ref[0][0], 2 * ref[0][1], "loss")
    assert not second[1][t == -100].any() and not first[1][t == -100].any()
    for g, (want, tol) in zip(second[1:], ref[1:]):
        _within(g, want, 4 * tol, "gradient")


@pytest.mark.parametrize("D", [32, 37, 2100])
@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38, -1e30])
def test_padding_may_hold_anything(hip_device, D, bad):
    """values that are not finite, or so large that the counted rows would vanish beside them, in rows that are not counted"""
    x, w, b, t = _data(70, D, 200, 24, ignored=0.4)
    clean = _run(hip_device, np.where(t[:, None] == -100, np.float32(0), x), w, b, t)
    y = x.copy()
    y[t == -100] = bad
    for a, c in zip(_run(hip_device, y, w, b, t), clean):
        assert np.array_equal(a, c)
    ref = _reference(np.where(t[:, None] == -100, np.float32(0), x), w, b, t)
    _within(clean[0], ref[0][0], ref[0][1], "loss")


def test_bad_targets_show(hip_device):
    x, w, b, t = _data(40, 24, 100, 10)
    for bad in (100.0, -1.0, 2.5, np.nan, np.inf, 1e9):
        u = t.copy()
        u[17] = bad
        loss, dx, dw, db = _run(hip_device, x, w, b, u)
        assert np.isnan(loss) and np.all(np.isnan(dx[17])) and np.all(np.isnan(dw)) and np.all(np.isnan(db))
        assert np.all(np.isfinite(np.delete(dx, 17, axis=0)))


def test_classes_masked_by_the_bias(hip_device):
    """a bias of -inf, or of the type's lowest value, takes a class out: probability 0, gradient 0"""
    x, w, b, t = _data(60, 48, 300, 11)
    out = np.zeros(300, bool)
    out[5::7] = True
    t = np.array([v if not out[int(v)] else 0.0 for v in t], np.float32)
    ref = _reference(x, w[:, ~out], b[:, ~out], np.searchsorted(np.nonzero(~out)[0], t).astype(np.float32))
    for low in (-np.inf, np.finfo(np.float32).min):
        c = b.copy()
        c[0, out] = low
        loss, dx, dw, db = _run(hip_device, x, w, c, t)
        _within(loss, ref[0][0], ref[0][1], "loss")
        _within(dx, ref[1][0], 2 * ref[1][1], "dx")
        _within(dw[:, ~out], ref[2][0], 2 * ref[2][1], "dw")
        assert not dw[:, out].any() and not db[0, out].any()


def test_a_row_that_is_not_finite_stays_in_its_row(hip_device):
    x, w, b, t = _data(45, 30, 90, 12)
    for bad in (np.nan, np.inf):
        y = x.copy()
        y[11, 3] = bad
        loss, dx, _, _ = _run(hip_device, y, w, b, t, reduction="sum")
        assert np.isnan(loss) and np.all(np.isnan(dx[11]))
        ref = _reference(np.delete(x, 11, 0), w, b, np.delete(t, 11), mean=False)
        _within(np.delete(dx, 11, 0), ref[1][0], 2 * ref[1][1], "dx")


@pytest.mark.parametrize("sx,sw", [(1e-15, 1e15), (1e12, 1e-12), (1e-30, 1.0), (1.0, 1e-30), (0.0, 1.0), (1.0, 0.0)])
def test_operands_of_any_magnitude(hip_device, sx, sw):
    x, w, b, t = _data(40, 60, 130, 13)
    _check(hip_device, (x * np.float32(sx)), (w * np.float32(sw)), b, t)


@pytest.mark.parametrize("factor", [1.0, 3.0, 300.0, 1e6])
@pytest.mark.parametrize("place", [0, 1, 5 * 64 + 1024, 16777215])
def test_a_large_weight_whose_largest_element_is_one_of_many(hip_device, factor, place):
    """16.8 M weights, whose scale is found from a sample: single elements that it holds, or does not, far above the others"""
    x, w, b, t = _data(140, 512, 32769, 32)
    w.reshape(-1)[place] = np.abs(w).max() * np.float32(factor)
    _check(hip_device, x, w, b, t)


def test_large_logits(hip_device):
    """probabilities of 0 and 1 to the last bit"""
    x, w, b, t = _data(64, 50, 400, 14)
    _check(hip_device, 20 * x, 5 * w, b, t)


def test_strided_operands_and_a_flat_bias(hip_device):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    x, w, b, t = _data(33, 20, 60, 15)
    dev = hip_device
    loss = F.linear_cross_entropy(Tensor(np.ascontiguousarray(x.T), device=dev).transpose(),
                                  Tensor(np.ascontiguousarray(w.T), device=dev).transpose(), Tensor(b.reshape(-1), device=dev),
                                  Tensor(t, device=dev))
    ref = _reference(x, w, b, t)
    _within(float(loss.numpy()[0]), ref[0][0], ref[0][1], "loss")


@pytest.mark.parametrize("which", [0, 1, 2])
def test_one_gradient_at_a_time(hip_device, which):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    x, w, b, t = _data(80, 48, 210, 16)
    ts = [Tensor(a, device=hip_device, requires_grad=k == which) for k, a in enumerate((x, w, b))]
    F.linear_cross_entropy(*ts, Tensor(t, device=hip_device)).backward()
    want, tol = _reference(x, w, b, t)[1 + which]
    _within(ts[which].grad.numpy(), want, tol, "gradient")
    assert all(ts[k].grad is None for k in range(3) if k != which)
    Graph.free_graph_all()


def test_evaluation_and_training_agree(hip_device):
    from deepflows_amd import nn
    from deepflows_amd.autograd import no_grad
    from deepflows_amd.tensor import Graph, Tensor
    x, w, b, t = _data(100, 64, 900, 17, ignored=0.2)
    fc = nn.Linear(64, 900, device=hip_device)
    fc.weight.data, fc.bias.data = Tensor(w, device=hip_device).data, Tensor(b, device=hip_device).data
    crit = nn.LinearCrossEntropyLoss(fc, label_smoothing=0.05)
    xt, tt = Tensor(x, device=hip_device), Tensor(t, device=hip_device)
    train = crit(xt, tt)
    with no_grad():
        held_out = crit(xt, tt)
    ref = _reference(x, w, b, t, e=0.05)
    for v in (train, held_out):
        _within(float(v.numpy()[0]), ref[0][0], ref[0][1], "loss")
    Graph.free_graph_all()


def test_many_classes_in_a_ragged_last_tile(hip_device):
    """a class count whose last tiles are ragged, in 140 M logits"""
    _check(hip_device, *_data(1400, 20, 100003, 18, ignored=0.1), label_smoothing=0.1)


def test_more_rows_than_one_piece_of_logits_holds(hip_device):
    """600 M logits are two pieces (of at most 2 GiB each): the second one adds to the first one's dW and db.  The rows are 60
    different ones, 100 times each in any order, so that the 60 rows' loss, dW and db are theirs too, and dx a hundredth.  dW's
    bound grows with the root of the rows (10 times), db's N / 64 + 30 and the loss's N / 256 + 12 by less (4 and 3 times)."""
    x, w, b, t = _data(60, 20, 100003, 22, ignored=0.1)
    order = np.random.default_rng(23).permutation(np.repeat(np.arange(60), 100))
    got = _run(hip_device, x[order], w, b, t[order], label_smoothing=0.1)
    (loss, tloss), (dx, tdx), (dw, tdw), (db, tdb) = _reference(x, w, b, t, e=0.1)
    _within(got[0], loss, 3 * tloss, "loss")
    _within(got[1], dx[order] / 100, tdx[order] / 100 + 4 * U * np.abs(dx[order]) / 100, "dx")
    _within(got[2], dw, 10 * tdw, "dw")
    _within(got[3], db, 4 * tdb, "db")


def test_evaluation_of_bad_targets_and_rows(hip_device):
    from deepflows_amd.autograd import no_grad
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    for N in (20, 100):
        x, w, b, t = _data(N, 24, 400, 31, ignored=0.2)
        def value(x, t):
            with no_grad():
                return float(F.linear_cross_entropy(*[Tensor(a, device=hip_device) for a in (x, w, b, t)]).numpy()[0])
        for bad in (400.0, -1.0, 2.5, np.nan, np.inf, 1e9):
            u = t.copy()
            u[7] = bad
            assert np.isnan(value(x, u))
        y = x.copy()
        y[t == -100] = np.nan
        assert value(y, t) == value(x, t)
        y[np.nonzero(t != -100)[0][0], 3] = np.nan
        assert np.isnan(value(y, t))
        assert value(x, np.full_like(t, -100)) == 0.0


def test_no_rows(hip_device):
    from deepflows_amd.backend_selection import BackendTensor
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    w = Tensor(np.ones((4, 6), np.float32), device=hip_device, requires_grad=True)
    b = Tensor(np.ones((1, 6), np.float32), device=hip_device, requires_grad=True)
    loss = F.linear_cross_entropy(Tensor(BackendTensor.make((0, 4), device=hip_device)), w, b,
                                  Tensor(BackendTensor.make((0,), device=hip_device)))
    loss.backward()
    assert float(loss.numpy()[0]) == 0.0 and not w.grad.numpy().any() and not b.grad.numpy().any()
    Graph.free_graph_all()


def test_gradients_against_differences(hip_device):
    rng = np.random.default_rng(19)
    x, w, b, t = _data(6, 9, 14, 19)
    _, dx, dw, db = _run(hip_device, x, w, b, t, label_smoothing=0.2)

    def value(x, w, b):
        return _reference(x, w, b, t, e=0.2)[0][0]

    args = [a.astype(np.float64) for a in (x, w, b)]
    for k, got in enumerate((dx, dw, db)):
        for _ in range(6):
            at = tuple(int(rng.integers(0, s)) for s in args[k].shape)
            up, dn = [a.copy() for a in args], [a.copy() for a in args]
            up[k][at] += 1e-5
            dn[k][at] -= 1e-5
            slope = (value(*up) - value(*dn)) / 2e-5
            # (differences in 64 bits: 1e-10; fp32 values of at most order 1 with sums of 14 and 9 terms: 64 u)
            assert abs(got[at] - slope) <= 64 * U * (1 + abs(slope))


def test_two_sweeps_over_a_retained_graph_and_a_held_gradient(hip_device):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    x, w, b, t = _data(30, 20, 50, 20)
    ts = [Tensor(a, device=hip_device, requires_grad=True) for a in (x, w, b)]
    loss = F.linear_cross_entropy(*ts, Tensor(t, device=hip_device))
    loss.backward(retain_graph=True)
    first = [p.grad.numpy().copy() for p in ts]
    loss.backward()                                            # (added to what the leaves hold)
    for p, g in zip(ts, first):
        assert np.array_equal(p.grad.numpy(), 2 * g)
    Graph.free_graph_all()


def test_inside_a_captured_graph(hip_device):
    """graphs over different shapes captured one after the other, replayed in turn on changed inputs with eager calls between"""
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    mod = hip_device.mod
    made = []
    for k, (N, D, V) in enumerate([(96, 64, 1500), (40, 100, 333), (16, 100, 2003)]):
        x, w, b, t = _data(N, D, V, 30 + k, ignored=0.2)
        leaves = [Tensor(a, device=hip_device, requires_grad=True) for a in (x, w, b)]
        tt = Tensor(t, device=hip_device)

        def step(leaves=leaves, tt=tt):
            for p in leaves:
                p.grad = None
            loss = F.linear_cross_entropy(*leaves, tt, label_smoothing=0.1)
            loss.backward()
            return [loss.data] + [p.grad for p in leaves]

        step()
        mod.capture_begin()
        got = step()
        made.append((leaves, tt, step, got, mod.capture_end(keep=got), (N, D, V)))
    for r in range(3):
        for k, (leaves, tt, step, got, graph, shape) in enumerate(made):
            x, w, b, t = _data(*shape, 100 + 10 * r + k, ignored=0.1)
            for p, a in zip(leaves + [tt], (x, w, b, t)):
                mod.from_numpy(a, p.data._handle)
        for m in made:
            m[4].replay()
        replayed = [[g.numpy().copy() for g in m[3]] for m in made]
        for m, rep in zip(made, replayed):
            for a, c in zip(rep, m[2]()):
                assert np.array_equal(a, c.numpy())
    for m in made:
        m[4].destroy()
    Graph.free_graph_all()


def test_a_captured_large_weight_whose_scale_moves(hip_device):
    """replays over weights that need the second conversion, and again over ones that do not"""
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    mod = hip_device.mod
    x, w, b, t = _data(70, 512, 32801, 33)
    leaves = [Tensor(a, device=hip_device, requires_grad=True) for a in (x, w, b)]
    tt = Tensor(t, device=hip_device)

    def step():
        for p in leaves:
            p.grad = None
        loss = F.linear_cross_entropy(*leaves, tt)
        loss.backward()
        return [loss.data] + [p.grad for p in leaves]

    step()
    mod.capture_begin()
    got = step()
    graph = mod.capture_end(keep=got)
    for factor in (1.0, 1000.0, 1.0, 50.0):
        v = w.copy()
        v[3, 777] = np.abs(w).max() * np.float32(factor)
        mod.from_numpy(v, leaves[1].data._handle)
        graph.replay()
        replayed = [g.numpy().copy() for g in got]
        for a, c in zip(replayed, step()):
            assert np.array_equal(a, c.numpy())
        ref = _reference(x, v, b, t)
        _within(float(replayed[0][0]), ref[0][0], ref[0][1], "loss")
        _within(replayed[1], ref[1][0], ref[1][1], "dx")
    graph.destroy()
    Graph.free_graph_all()


def test_refusals(hip_device):
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    x, w, b, t = (Tensor(a, device=hip_device) for a in _data(8, 6, 10, 21))
    bad = lambda shape: Tensor(np.zeros(shape, np.float32), device=hip_device)
    for args, kw in [((x, bad((7, 10)), b, t), {}), ((x, w, bad((1, 9)), t), {}), ((x, w, b, bad((7,))), {}),
                     ((x, w, b, bad((8, 10))), {}), ((bad((2, 4, 6)), w, b, t), {}), ((x, w, b, t), {"reduction": "none"}),
                     ((x, w, b, t), {"label_smoothing": 1.5}), ((x, w, b, t), {"label_smoothing": float("nan")}),
                     ((x, w, b, t), {"ignore_index": 0.5})]:
        with pytest.raises(ValueError):
            F.linear_cross_entropy(*args, **kw)
    s = bad((6, 6))
    with pytest.raises(ValueError):
        F.linear_cross_entropy(s, s, None, bad((6,)))
    mod = hip_device.mod
    h = lambda v: v.data._handle
    one = bad((1,))
    for rows, width, classes, ign, sm in [(-1, 6, 10, -100, 0.0), (8, 0, 10, -100, 0.0), (8, 6, 0, -100, 0.0),
                                          (8, 6, (1 << 24) + 1, -100, 0.0), (8, 6, 10, 1 << 25, 0.0), (8, 6, 10, -100, -0.1)]:
        with pytest.raises(ValueError):
            mod.linear_ce_forward(h(x), h(w), None, h(t), h(one), None, None, None, rows, width, classes, ign, sm, True)


def _sparse_weight(D, V, seed):
    x, _, b, t = _data(70, D, V, seed)
    return x, np.zeros((D, V), np.float32), b, t, np.random.default_rng(seed + 1)


@pytest.mark.parametrize("magnitude", [1.0, 1e-5, 1e-10])
@pytest.mark.parametrize("piece", [0, 1, 7, 15, 5 * 16 + 9])
def test_a_large_weight_that_is_zero_but_for_a_few_elements(hip_device, magnitude, piece):
    """16.8 M weights, 64 neighbours of which are not zero: whichever elements a scale is sampled from, most of these pieces are not
    among them.  (The bounds are relative to the weight's magnitude: dx is as small as it is.)"""
    x, w, b, t, rng = _sparse_weight(512, 32768, 40)
    w.reshape(-1)[piece * 64:piece * 64 + 64] = magnitude * rng.uniform(0.5, 1.0, 64)
    _check(hip_device, x, w, b, t)


@pytest.mark.parametrize("V", [32768, 49152])
@pytest.mark.parametrize("magnitude", [1e-4, 1e-6])
def test_a_large_weight_of_few_columns(hip_device, V, magnitude):
    """a head that starts at zero and some of whose classes are filled in, at numbers of classes that are multiples of 16 384"""
    x, w, b, t, rng = _sparse_weight(512, V, 42)
    w[:, 64:128] = magnitude * rng.standard_normal((512, 64))
    _check(hip_device, x, w, b, t)


def test_a_captured_large_weight_that_comes_and_goes(hip_device):
    """replays over weights that are zero at most places, everywhere, and nowhere"""
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    mod = hip_device.mod
    x, w, b, t, rng = _sparse_weight(512, 32768, 44)
    leaves = [Tensor(a, device=hip_device, requires_grad=True) for a in (x, w, b)]
    tt = Tensor(t, device=hip_device)

    def step():
        for p in leaves:
            p.grad = None
        loss = F.linear_cross_entropy(*leaves, tt)
        loss.backward()
        return [loss.data] + [p.grad for p in leaves]

    step()
    mod.capture_begin()
    got = step()
    graph = mod.capture_end(keep=got)
    block, full = w.copy(), (0.05 * rng.standard_normal(w.shape)).astype(np.float32)
    block[7, 512:576] = 1e-6 * rng.standard_normal(64)
    for v in (block, full, w, block):
        mod.from_numpy(v, leaves[1].data._handle)
        graph.replay()
        replayed = [g.numpy().copy() for g in got]
        for a, c in zip(replayed, step()):
            assert np.array_equal(a, c.numpy())
        ref = _reference(x, v, b, t)
        _within(float(replayed[0][0]), ref[0][0], ref[0][1], "loss")
        _within(replayed[1], ref[1][0], ref[1][1], "dx")
        _within(replayed[2], ref[2][0], ref[2][1], "dw")
    graph.destroy()
    Graph.free_graph_all()


@pytest.mark.parametrize("log2", [7, 19, 21])
@pytest.mark.parametrize("train", [True, False])
def test_the_mean_of_equal_rows_is_a_row(hip_device, train, log2):
    """2^k equal rows have one row's loss: their sum is exact in double, 2^-k is too, so what is left is one rounding of a number that
    needs none.  (The row's own rounding cancels: 128 rows of the same inputs, by the same products, say what it is.)"""
    from deepflows_amd.autograd import no_grad
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Graph, Tensor
    _, w, b, _ = _data(1, 4, 9, 45)

    def value(N):
        x, t = np.tile(np.array([[0.3, -1.2, 0.7, 0.1]], np.float32), (N, 1)), np.full(N, 3.0, np.float32)
        leaves = [Tensor(a, device=hip_device, requires_grad=train) for a in (x, w, b)]
        if train:
            loss = F.linear_cross_entropy(*leaves, Tensor(t, device=hip_device))
        else:
            with no_grad():
                loss = F.linear_cross_entropy(*leaves, Tensor(t, device=hip_device))
        out = loss.numpy()[0]
        Graph.free_graph_all()
        return out

    one = value(128)
    want = _reference(np.array([[0.3, -1.2, 0.7, 0.1]], np.float32), w, b, np.array([3.0], np.float32))[0]
    _within(float(one), *want, "loss")
    assert value(1 << log2) == one


@pytest.mark.parametrize("N", [12, 45, 90])
@pytest.mark.parametrize("V", [2, 9, 300, 33000, 60001])
def test_smoothing_over_several_classes_of_the_lowest_value(hip_device, N, V):
    """Masked classes of the type's lowest value and a smoothed target: the loss is e / V times their sum, large but finite although
    the sum itself is no float.  Its terms have one sign: each a rounding, their sum V / 256 + 40, a few for the rest."""
    from deepflows_amd.autograd import no_grad
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    x, w, b, t = _data(N, 40, V, 46)
    low = np.finfo(np.float32).min
    out = np.zeros(V, bool)
    out[1::3] = True
    if V > 1000:
        out[200:500] = True                                    # whole runs of classes
    t[:] = np.nonzero(~out)[0][t.astype(int) % int((~out).sum())]
    b[0, out] = low
    want = _reference(x, w, b, t, e=0.1)[0][0]
    assert np.isfinite(np.float32(want))
    tol = (V / 256 + 60) * U * want
    _within(_run(hip_device, x, w, b, t, label_smoothing=0.1)[0], want, tol, "loss")
    with no_grad():
        loss = F.linear_cross_entropy(*[Tensor(a, device=hip_device) for a in (x, w, b, t)], label_smoothing=0.1)
    _within(float(loss.numpy()[0]), want, tol, "loss alone")


# ---- small elements beside large ones --------------------------------------------------------------------------------------------
# The two halves of an operand carry 2^-23 of it down to 2^-28 of the array's largest magnitude A, and an absolute 2^-49 A below
# (dl, whose scale is fixed: 2^-51).  A product's bound is the one above with those floors, times two:
#   |error| <= (12 + 6 sqrt(3 K)) u sum|a b| + 2^-48 (A sum|b| + B sum|a|).
def _fine_product_error(a, b):
    K = a.shape[1]
    aa, bb = np.abs(a), np.abs(b)
    fl = 2.0 ** -48 * (aa.max(initial=0.0) * bb.sum(0)[None, :] + bb.max(initial=0.0) * aa.sum(1)[:, None])
    return (12 + 6 * np.sqrt(3 * K)) * U * (aa @ bb) + fl


def _fine_gradients(x, w, b, t):
    """the gradients of the mean and their bounds"""
    x, w = x.astype(np.float64), w.astype(np.float64)
    N, V = x.shape[0], w.shape[1]
    l = x @ w + b.astype(np.float64).reshape(1, -1)
    # (one error of a row's largest logits moves all its probabilities; a logit's own moves its own)
    E = _fine_product_error(x, w) + U * np.abs(l)
    p = np.exp(l - l.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    # (the exponential's argument l - m is rounded: u |l - m|)
    tp = p * (E + (E * p).sum(1, keepdims=True) + U * np.abs(l - l.max(1, keepdims=True)) + (V / 256 + 40) * U)
    dl = p.copy()
    dl[np.arange(N), t.astype(int)] -= 1.0
    td = tp + 2.0 ** -22 * np.abs(dl) + 2.0 ** -50
    td[np.arange(N), t.astype(int)] += 4 * U
    dx, dw, db = dl @ w.T / N, x.T @ dl / N, dl.sum(0) / N
    return ((dx, (_fine_product_error(dl, w.T) + td @ np.abs(w).T) / N + 4 * U * np.abs(dx)),
            (dw, (_fine_product_error(x.T, dl) + np.abs(x).T @ td) / N + 4 * U * np.abs(dw)),
            (db, (td.sum(0) + (N / 64 + 30) * U * np.abs(dl).sum(0)) / N + 4 * U * np.abs(db)))


@pytest.mark.parametrize("N,D,V", [(100, 24, 700), (300, 130, 4001), (700, 64, 60000)])
def test_classes_that_are_hardly_ever_likely(hip_device, N, D, V):
    """probabilities from 1e-2 to 1e-13 side by side: every class's column of dW and element of db is as good as its own magnitude asks"""
    x, w, b, t = _data(N, D, V, 47)
    b -= np.array([0.0, 10.0, 16.0, 22.0, 26.0], np.float32)[np.arange(V) % 5]
    t -= t % 5                                                 # (targets among the likely ones: the others' columns are as small as p)
    got = _run(hip_device, 0.25 * x, w, b, t)
    for g, (want, tol), what in zip(got[1:], _fine_gradients(np.float32(0.25) * x, w, b, t), ("dx", "dw", "db")):
        _within(g, want, tol, what)


@pytest.mark.parametrize("small", [2.0 ** -12, 2.0 ** -20, 2.0 ** -26])
def test_features_of_different_magnitudes(hip_device, small):
    """columns of x far below the others: their rows of dW; rows of W far below the others: their columns of dx"""
    x, w, b, t = _data(200, 96, 900, 48)
    x[:, 1::3] *= np.float32(small)
    w[2::3] *= np.float32(small)
    got = _run(hip_device, x, w, b, t)
    for g, (want, tol), what in zip(got[1:], _fine_gradients(x, w, b, t), ("dx", "dw", "db")):
        _within(g, want, tol, what)


@pytest.mark.parametrize("large", [2.0 ** 10, 2.0 ** 20, 2.0 ** 30])
def test_a_row_far_above_the_others(hip_device, large):
    """one row's magnitude does not cost the others their logits: the gradients of the rows of an ordinary batch beside it.  (Its own
    loss is so large that the mean says nothing of theirs: dx does.)"""
    x, w, b, t = _data(150, 48, 500, 49)
    x[17] *= np.float32(large)
    got = _run(hip_device, x, w, b, t)
    want, tol = _fine_gradients(x, w, b, t)[0]
    _within(np.delete(got[1], 17, 0), np.delete(want, 17, 0), np.delete(tol, 17, 0), "dx")


@pytest.mark.parametrize("N", [65, 100, 128])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_evaluation_of_65_to_128_rows_over_a_very_large_weight(hip_device, N, smoothing):
    """140 M weights, 1 000 different columns of them with a bias each: the bound of `_reference`"""
    from deepflows_amd.autograd import no_grad
    from deepflows_amd.nn import functional as F
    from deepflows_amd.tensor import Tensor
    D, V, e = 1401, 100003, smoothing
    x, w0, _, _ = _data(N, D, 1000, 50)
    _, _, b, t = _data(N, 1, V, 51, ignored=0.2)
    wide = lambda a: np.tile(a, (1, V // 1000 + 1))[:, :V]
    x64, w64 = x.astype(np.float64), w0.astype(np.float64)
    l = wide(x64 @ w64) + b.astype(np.float64)
    E = (wide(_product_error(x64, w64)) + U * np.abs(l)).max(1)
    m = l.max(1)
    lse = np.log(np.exp(l - m[:, None]).sum(1)) + m
    counted = t != -100
    lt = l[np.arange(N), np.where(counted, t, 0).astype(int)]
    row = lse - (1 - e) * lt - e * l.mean(1)
    trow = 3 * E + U * (V / 256 + 60) * (1 + np.abs(lse - lt)) + e * U * (V / 256 + 30) * np.abs(l - m[:, None]).mean(1)
    want, tol = row[counted].mean(), trow[counted].mean() + 14 * U * np.abs(row[counted]).mean()
    x[~counted] = np.nan
    with no_grad():
        loss = F.linear_cross_entropy(*[Tensor(a, device=hip_device) for a in (x, wide(w0), b, t)], label_smoothing=e)
    _within(float(loss.numpy()[0]), want, tol, "loss")


@pytest.mark.parametrize("N,D,V", [(8328, 183, 7929), (1858, 1542, 4233), (2239, 438, 14704), (2776, 1197, 5054), (6144, 180, 100003)])
def test_the_largest_tiles_of_the_gradient_products(hip_device, N, D, V):
    """Gradient products by 256 x 128 tiles: both with a last round that is cut along the reduction, neither, one each, and two pieces
    of the logits.  The rows are 60 different ones in any order: their loss, dW and db are theirs times their share.  dW's bound grows
    with the root of the rows, db's with N / 64 + 30, the loss's not (it is added up in double)."""
    x, w, b, t = _data(60, D, V, 52, ignored=0.1)
    order = np.random.default_rng(53).permutation(np.tile(np.arange(60), N // 60 + 1)[:N])
    share = np.bincount(order, minlength=60).astype(np.float64)
    got = _run(hip_device, x[order], w, b, t[order], label_smoothing=0.1)
    counted = t != -100
    total = share[counted].sum()
    _, (dx, tdx), (_, tdw), (_, tdb) = _reference(x, w, b, t, mean=False, e=0.1)
    x64, l = x.astype(np.float64), x.astype(np.float64) @ w.astype(np.float64) + b.astype(np.float64)
    lse = np.log(np.exp(l - l.max(1, keepdims=True)).sum(1)) + l.max(1)
    place = np.where(counted, t, 0).astype(int)
    row = (lse - 0.9 * l[np.arange(60), place] - 0.1 * l.mean(1)) * counted
    E = (_product_error(x64, w.astype(np.float64)) + U * np.abs(l)).max(1)
    trow = 3 * E + U * (V / 256 + 60) * (1 + np.abs(lse - l[np.arange(60), place])) \
        + U * (V / 256 + 30) * np.abs(l - l.max(1, keepdims=True)).mean(1)
    _within(got[0], (share * row).sum() / total, (share * trow * counted).sum() / total + 14 * U * np.abs(share * row).sum() / total, "loss")
    _within(got[1], dx[order] / total, tdx[order] / total + 4 * U * np.abs(dx[order]) / total, "dx")
    dl = np.exp(l - lse[:, None])
    dl -= 0.1 / V
    dl[np.arange(60), place] -= 0.9
    dl *= (counted * share / total)[:, None]
    most = share.max()                                         # (a row's share differs by one)
    _within(got[2], x64.T @ dl, np.sqrt(N / 60) * tdw * most / total, "dw")
    _within(got[3], dl.sum(0, keepdims=True), (N / 64 + 30) / 30 * tdb * most / total, "db")
