"""Losses of the language-model head: cross entropy and distillation on hidden states without the logits, distillation on
logits.  Values and gradients against a float64 restatement, refusals, and the calls that go together."""
import ctypes
from ctypes import byref, c_size_t, c_void_p

import numpy as np
import pytest

from gradtuity_b200 import _lib
from gradtuity_b200.tensor import Storage, Tensor

# Relative Frobenius error of gradients.  3xtf32 / fp32: the bar of this repository for products as exact as 32-bit sums
# (1e-5).  tf32: operands are rounded by half a step of 2^-11 relative, so a logit of size |z| built of independent terms is
# off by 2^-12 sqrt(2/3) |z| (rms), which is the relative error of p; the tests keep |z| (rms) under 3, G and the other
# operand are rounded again: (3 + 1) 2^-12 sqrt(2/3) = 8e-4, times 4 for the spread between inputs.
TOL = {"3xtf32": 1e-5, "fp32": 1e-5, "tf32": 3.2e-3}
# Absolute error of a row's loss: |z| and log s below 16 in 32 bits (a few steps of 2^-21), or the logits' error in tf32.
LOSS_TOL = {"3xtf32": 1e-5, "fp32": 1e-5, "tf32": 1e-2}


def rel(got, want):
    scale = np.linalg.norm(want)
    return np.linalg.norm(got.astype(np.float64) - want) / scale if scale else np.abs(got).max()


def dense_targets(M, V, ids, teacher, T):
    """(target distribution (M, V), rows that count) in float64."""
    q = np.zeros((M, V))
    counted = np.zeros(M, bool)
    for t in range(M):
        used = [(int(i), float(v)) for i, v in zip(ids[t], teacher[t]) if i >= 0 and v > -np.inf]
        if not used:
            continue
        counted[t] = True
        v = np.array([u[1] for u in used]) / T
        e = np.exp(v - v.max())
        for (i, _), p in zip(used, e / e.sum()):
            q[t, i] += p
    return q, counted


def entropy_of(M, ids, teacher, T):
    """sum of q log q over the entries (an id that comes twice is two entries)."""
    out = np.zeros(M)
    for t in range(M):
        v = np.array([float(v) for i, v in zip(ids[t], teacher[t]) if i >= 0 and v > -np.inf]) / T
        if len(v):
            lp = v - v.max()
            lp = lp - np.log(np.exp(lp).sum())
            p = np.exp(lp)
            out[t] = np.sum(np.where(p > 0, p * lp, 0.0))
    return out


def oracle(logits, q, counted, entropy, T, reduction, upstream=None):
    """(loss or losses, d loss / d logits) in float64; upstream: per row for 'none'."""
    z = logits / T
    m = z.max(1, keepdims=True)
    lse = m + np.log(np.exp(z - m).sum(1, keepdims=True))
    with np.errstate(invalid="ignore"):
        row = T * T * (entropy - np.where(q > 0, q * (z - lse), 0.0).sum(1)) * counted
    row = np.where(counted, row, 0.0)
    g = T * (np.exp(z - lse) - q) * counted[:, None]
    g[~counted] = 0.0
    n = max(1, int(counted.sum()))
    if reduction == "none":
        return row, g * (np.ones(len(row)) if upstream is None else upstream)[:, None]
    if reduction == "mean":
        return row.sum() / n, g / n
    return row.sum(), g


def hard(M, V, targets, ignore=-100):
    q = np.zeros((M, V))
    counted = targets != ignore
    q[np.nonzero(counted)[0], targets[counted].astype(int)] = 1.0
    return q, counted


def hidden(rng, M, V, E, spread=2.0):
    w = (rng.standard_normal((V, E)) * spread / np.sqrt(E)).astype(np.float32)
    x = rng.standard_normal((M, E)).astype(np.float32)
    return x, w


def teacher_of(rng, M, V, K, ragged=True, duplicates=False):
    ids = np.stack([rng.integers(0, V, K) if duplicates or K > V else rng.permutation(V)[:K] for _ in range(M)]).astype(np.float32)
    t = (rng.standard_normal((M, K)) * 3).astype(np.float32)
    if ragged:
        for r in range(M):
            n = rng.integers(0, K + 1)
            ids[r, n:] = -1
            t[r, n:] = np.nan
    return ids, t


def run_linear(x, w, make, upstream=None, need=("x", "w")):
    """loss, dx, dw of make(xt, wt); upstream: per-row factors applied before the sum."""
    xt, wt = Tensor.from_numpy(x, requires_grad="x" in need), Tensor.from_numpy(w, requires_grad="w" in need)
    loss = make(xt, wt)
    value = loss.numpy()
    if loss.numel > 1 or upstream is not None:
        up = np.ones(loss.numel, np.float32) if upstream is None else upstream
        loss.mul(Tensor.from_numpy(up.astype(np.float32))).sum().backward()
    else:
        loss.backward()
    assert _lib.device_status() == 0
    return value, (xt.grad.numpy() if "x" in need else None), (wt.grad.numpy() if "w" in need else None)


# ---- refusals (no GPU) ----------------------------------------------------------------------------

def fake(*shape):
    """A tensor without memory: the checks of the arguments come before any use of it."""
    return Tensor._wrap(Storage(0, 0, owns=False), shape)


@pytest.mark.parametrize("call, match", [
    (lambda: fake(4).linear_cross_entropy(fake(9, 4), fake(4)), "requires 2D input"),
    (lambda: fake(4, 8).linear_cross_entropy(fake(8), fake(4)), "weight must be 2D"),
    (lambda: fake(4, 8).linear_cross_entropy(fake(9, 7), fake(4)), "!= weight last dim 7"),
    (lambda: fake(4, 8).linear_cross_entropy(fake(9, 8), fake(5)), "batch size mismatch"),
    (lambda: fake(4, 8).linear_cross_entropy(fake(9, 8), fake(4, 1)), "expects 1D targets"),
    (lambda: fake(4, 8).linear_cross_entropy(fake(9, 8), fake(4), reduction="max"), "reduction must be"),
    (lambda: fake(4, 8).linear_cross_entropy(fake(9, 8), fake(4), precision="bf16"), "precision must be one of"),
    (lambda: fake(4, 8).linear_topk_distillation(fake(9, 8), fake(4, 2), fake(4, 3)), "one \\(rows, top\\) shape"),
    (lambda: fake(4, 8).linear_topk_distillation(fake(9, 8), fake(5, 2), fake(5, 2)), "batch size mismatch"),
    (lambda: fake(4, 8).linear_topk_distillation(fake(9, 8), fake(4), fake(4)), "one \\(rows, top\\) shape"),
    (lambda: fake(4, 8).linear_topk_distillation(fake(9, 8), fake(4, 2), fake(4, 2), temperature=0.0), "temperature must be"),
    (lambda: fake(4, 8).linear_topk_distillation(fake(9, 8), fake(4, 1025), fake(4, 1025)), "at most 1024"),
    (lambda: fake(4, 2, 2).topk_distillation(fake(4, 2), fake(4, 2)), "expects 2D logits"),
    (lambda: fake(4, 9).topk_distillation(fake(4, 2), fake(4, 2), temperature=float("inf")), "temperature must be"),
    (lambda: fake(4, 9).topk_distillation(fake(4, 2), fake(4, 2), temperature=float("nan")), "temperature must be"),
    (lambda: fake(4, 9).topk_distillation(fake(4, 2), fake(4, 2), temperature=1e-7), "temperature must be"),
    (lambda: fake(4, 9).topk_distillation(fake(4, 2), fake(4, 2), temperature=-2.0), "temperature must be"),
    (lambda: fake(4, 9).topk_distillation(fake(3, 2), fake(3, 2)), "batch size mismatch"),
    (lambda: fake(4, 9).topk_distillation(fake(4, 2), fake(4, 2), reduction="avg"), "reduction must be"),
])
def test_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_entry_points_refuse_a_null_context():
    lib = _lib.load_library()
    n = c_size_t(0)
    bad = _lib.GT_ERR_INVALID_ARG
    assert lib.gt_linear_loss_sizes(None, 1, 1, 1, 1, 0, byref(n), byref(n)) == bad
    assert lib.gt_linear_cross_entropy(None, None, None, None, None, None, None, 1, 1, 1, -100.0, 1, 0) == bad
    assert lib.gt_linear_topk_distillation(None, None, None, None, None, None, None, None, 1, 1, 1, 1, 1.0, 1, 0) == bad
    assert lib.gt_linear_loss_backward(None, None, None, None, None, None, None, None, 1, 1, 1, 1, 1.0, 1, 0, 0, 0) == bad
    assert lib.gt_topk_distillation_sizes(None, 1, 1, 1, byref(n)) == bad
    assert lib.gt_topk_distillation(None, None, None, None, 1, None, 1, None, None, 1, 1, 1, 1.0, 1) == bad
    assert lib.gt_topk_distillation_backward(None, None, 1, None, None, 1, None, 1, 1, 1, 1.0, 1, 0) == bad


@pytest.mark.gpu
def test_entry_points_refuse_bad_sizes(gt):
    lib, ctx = gt.load_library(), gt.context()
    a, b = c_size_t(0), c_size_t(0)
    for M, V, E, K in [(0, 5, 5, 1), (5, 0, 5, 1), (5, 5, 0, 1), (5, 5, 5, 0), (5, 1 << 24, 5, 1), (5, 5000, 5, 1025), (1 << 31, 5, 5, 1)]:
        assert lib.gt_linear_loss_sizes(ctx, M, V, E, K, 0, byref(a), byref(b)) == gt.GT_ERR_INVALID_ARG
    assert lib.gt_linear_loss_sizes(ctx, 5, 5, 5, 1, 3, byref(a), byref(b)) == gt.GT_ERR_INVALID_ARG
    p = c_void_p(256)          # never read: the call is refused first
    assert lib.gt_linear_cross_entropy(ctx, p, p, p, p, p, p, 5, 5, 5, -100.0, 3, 0) == gt.GT_ERR_INVALID_ARG
    assert lib.gt_linear_topk_distillation(ctx, p, p, p, p, p, p, p, 5, 5, 5, 1, ctypes.c_float(-1.0), 1, 0) == gt.GT_ERR_INVALID_ARG
    assert lib.gt_topk_distillation(ctx, p, p, None, 0, p, 4, p, p, 5, 5, 1, 1.0, 1) == gt.GT_ERR_INVALID_ARG       # pitch below the row length
    assert lib.gt_topk_distillation(ctx, p, p, p, 4, p, 5, p, p, 5, 5, 1, 1.0, 1) == gt.GT_ERR_INVALID_ARG
    assert lib.gt_topk_distillation(ctx, p, p, p, 5, p, 5, p, p, 5, 5, 1, 1.0, 0) == gt.GT_ERR_INVALID_ARG          # gradient of 'none'
    assert lib.gt_linear_cross_entropy(ctx, p, p, p, p, p, p, 5, 5, 5, -100.0, 1, 7) == gt.GT_ERR_INVALID_ARG


# ---- values and gradients -------------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 7, 3), (3, 2, 64), (2, 257, 65), (48, 500, 64), (129, 1000, 100), (300, 5003, 203), (257, 70001, 33), (520, 300, 768),
         (64, 4096, 128), (1, 30011, 96), (17, 3001, 130),
         # few rows: every number of columns a lane and of warps beside each other
         (1, 2003, 768), (1, 900, 1024), (1, 515, 300), (1, 100, 600), (4, 1501, 700), (3, 333, 200), (2, 40, 1000), (16, 1200, 1000), (5, 700, 520),
         (9, 401, 260), (64, 130, 900), (33, 290, 33),
         # two pieces of the vocabulary, the second ragged, and dx in shares
         (1100, 33001, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["3xtf32", "tf32", "fp32"])
@pytest.mark.parametrize("M, V, E", SIZES)
def test_linear_cross_entropy(gt, M, V, E, precision):
    rng = np.random.default_rng([M, V, E])
    x, w = hidden(rng, M, V, E)
    targets = rng.integers(0, V, M).astype(np.float32)
    if M > 2:
        targets[rng.random(M) < 0.3] = -100
    targets[0], targets[-1] = V - 1, 0
    q, counted = hard(M, V, targets)
    logits = x.astype(np.float64) @ w.astype(np.float64).T
    want, g = oracle(logits, q, counted, np.zeros(M), 1.0, "mean")
    loss, dx, dw = run_linear(x, w, lambda a, b: a.linear_cross_entropy(b, Tensor.from_numpy(targets), precision=precision))
    assert abs(loss[0] - want) < LOSS_TOL[precision]
    if V > 1:
        assert rel(dx, g @ w) < TOL[precision] and rel(dw, g.T @ x) < TOL[precision]
    else:
        assert not dx.any() and not dw.any()          # one word: p = 1 = q


@pytest.mark.gpu
@pytest.mark.parametrize("M, V, E, K, T, reduction, duplicates", [
    (1, 5, 3, 1, 1.0, "mean", False), (4, 6, 8, 6, 2.0, "sum", False), (33, 700, 64, 17, 0.5, "mean", True), (300, 5003, 203, 32, 2.0, "none", False),
    (130, 70001, 40, 100, 4.0, "mean", False), (9, 3000, 96, 1024, 1.5, "none", True), (257, 300, 128, 33, 1.0, "mean", True)])
@pytest.mark.parametrize("precision", ["3xtf32", "tf32"])
def test_linear_topk_distillation(gt, M, V, E, K, T, reduction, duplicates, precision):
    rng = np.random.default_rng([M, V, E, K])
    x, w = hidden(rng, M, V, E)
    ids, teacher = teacher_of(rng, M, V, K, ragged=True, duplicates=duplicates)
    q, counted = dense_targets(M, V, ids, teacher, T)
    up = (rng.standard_normal(M).astype(np.float32)) if reduction == "none" else None
    logits = x.astype(np.float64) @ w.astype(np.float64).T
    want, g = oracle(logits, q, counted, entropy_of(M, ids, teacher, T), T, reduction, up)
    loss, dx, dw = run_linear(x, w, lambda a, b: a.linear_topk_distillation(b, Tensor.from_numpy(ids), Tensor.from_numpy(teacher), temperature=T,
                                                                            reduction=reduction, precision=precision), up)
    assert np.abs(loss - want).max() < LOSS_TOL[precision] * max(1, T * T) * (M if reduction == "sum" else 1)
    if counted.any():
        # G = p - q cancels where the student has learned its teacher: the error is that of p and q, not of their difference
        assert rel(dx, g @ w) < 2 * TOL[precision] and rel(dw, g.T @ x) < 2 * TOL[precision]


@pytest.mark.gpu
@pytest.mark.parametrize("B, C, K, T, reduction, duplicates", [
    (1, 1, 1, 1.0, "mean", False), (1, 3, 2, 2.0, "none", False), (16, 1000, 5, 1.0, "mean", False), (300, 50257, 32, 2.0, "mean", False),
    (37, 32003, 100, 0.7, "sum", True), (1001, 4099, 64, 3.0, "none", True), (5, 60007, 1024, 1.0, "mean", False), (200, 4096, 7, 1.0, "mean", True),
    (7, 777, 777, 5.0, "mean", False), (150, 56001, 31, 1.0, "none", False)])
def test_topk_distillation(gt, B, C, K, T, reduction, duplicates):
    rng = np.random.default_rng([B, C, K])
    logits = (rng.standard_normal((B, C)) * 2.5).astype(np.float32)
    ids, teacher = teacher_of(rng, B, C, K, ragged=B > 1, duplicates=duplicates)
    q, counted = dense_targets(B, C, ids, teacher, T)
    up = rng.standard_normal(B).astype(np.float32) if reduction == "none" else None
    want, g = oracle(logits.astype(np.float64), q, counted, entropy_of(B, ids, teacher, T), T, reduction, up)
    xt = Tensor.from_numpy(logits, requires_grad=True)
    loss = xt.topk_distillation(Tensor.from_numpy(ids), Tensor.from_numpy(teacher), temperature=T, reduction=reduction)
    value = loss.numpy()
    (loss if up is None else loss.mul(Tensor.from_numpy(up)).sum()).backward()
    assert _lib.device_status() == 0
    assert np.abs(value - want).max() < 1e-5 * max(1, T * T) * (B if reduction == "sum" else 1)
    # every step in 32 bits: a few roundings of 2^-24 and the exponential's, far below 2e-6
    if C > 1:
        assert rel(xt.grad.numpy(), g) < 2e-6
    else:
        assert not xt.grad.numpy().any()


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["linear_cross_entropy", "linear_topk_distillation", "topk_distillation"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("M, V, E", [(33, 300, 40), (1, 300, 40), (200, 4500, 40), (1500, 300, 300)])
def test_rows_that_do_not_count(gt, op, reduction, M, V, E):
    """All rows without a target: loss 0 and gradients that are written, as zeros; masked places may hold anything."""
    rng = np.random.default_rng(5)
    x, w = hidden(rng, M, V, E)
    xt, wt = Tensor.from_numpy(x, requires_grad=True), Tensor.from_numpy(w, requires_grad=True)
    ids = np.full((M, 4), -1, np.float32)
    teacher = np.full((M, 4), np.inf, np.float32)
    ids[:, 1], teacher[:, 1] = 3, -np.inf
    ids[:, 2], teacher[:, 2] = 5, np.nan
    ti, tt = Tensor.from_numpy(ids), Tensor.from_numpy(teacher)
    if op == "linear_cross_entropy":
        loss = xt.linear_cross_entropy(wt, Tensor.from_numpy(np.full(M, 7, np.float32)), ignore_index=7, reduction=reduction)
    elif op == "linear_topk_distillation":
        loss = xt.linear_topk_distillation(wt, ti, tt, reduction=reduction)
    else:
        xt = Tensor.from_numpy(rng.standard_normal((M, V)).astype(np.float32), requires_grad=True)
        loss = xt.topk_distillation(ti, tt, reduction=reduction)
    assert not loss.numpy().any()
    (loss.sum() if reduction == "none" else loss).backward()
    assert _lib.device_status() == 0
    assert not xt.grad.numpy().any()
    if op != "topk_distillation":
        assert not wt.grad.numpy().any()


@pytest.mark.gpu
def test_lowest_values_infinities_and_nan(gt):
    """Masks made with the type's lowest value or -inf, in the student's logits and in the teacher's."""
    low = np.finfo(np.float32).min
    logits = np.array([[1.0, 2.0, -np.inf, 0.5], [low, 3.0, low, 1.0], [0.0, 0.0, 0.0, -np.inf], [2.0, 1.0, 0.0, -1.0]], np.float32)
    ids = np.array([[0, 1], [1, 3], [0, 2], [3, 0]], np.float32)
    teacher = np.array([[0.0, 1.0], [low, low], [low, 2.0], [5.0, -np.inf]], np.float32)
    for T in (1.0, 2.0, 0.5):
        q = np.zeros((4, 4))
        q[0, 0], q[0, 1] = 1 / (1 + np.exp(1 / T)), 1 / (1 + np.exp(-1 / T))
        q[1, 1] = q[1, 3] = 0.5
        q[2, 2] = 1.0
        q[3, 3] = 1.0
        ent = np.array([np.sum(q[0, :2] * np.log(q[0, :2])), np.log(0.5), 0.0, 0.0])
        z = np.maximum(logits.astype(np.float64) / T, -1e30)          # exp of either is 0
        want, g = oracle(z * T, q, np.ones(4, bool), ent, T, "mean")
        xt = Tensor.from_numpy(logits, requires_grad=True)
        loss = xt.topk_distillation(Tensor.from_numpy(ids), Tensor.from_numpy(teacher), temperature=T)
        assert loss.item() == pytest.approx(want, rel=2e-6)
        loss.backward()
        assert np.abs(xt.grad.numpy() - g).max() < 1e-6
    # a student that gives a teacher's word no probability: the loss is infinite, the gradient is not
    xt = Tensor.from_numpy(logits[:1], requires_grad=True)
    loss = xt.topk_distillation(Tensor([[2.0]]), Tensor([[1.0]]))
    assert loss.item() == np.inf
    loss.backward()
    p = np.exp(logits[0].astype(np.float64)) / np.exp(logits[0].astype(np.float64)).sum()
    assert np.abs(xt.grad.numpy()[0] - (p - [0, 0, 1, 0])).max() < 1e-6
    # a NaN among a row's logits makes that row's loss NaN, and no other row's
    bad = logits.copy()
    bad[1, 0] = np.nan
    rows = Tensor.from_numpy(bad).topk_distillation(Tensor.from_numpy(ids), Tensor.from_numpy(teacher), reduction="none").numpy()
    assert np.isnan(rows[1]) and np.isfinite(rows[[0, 2, 3]]).all()


@pytest.mark.gpu
def test_linear_nan_and_large_values_stay_in_their_rows(gt):
    rng = np.random.default_rng(8)
    M, V, E = 140, 900, 72
    x, w = hidden(rng, M, V, E)
    x[3, 5] = np.nan
    x[7] *= 1e4                                     # logits of 1e4: one word takes the whole row
    x[9] = 0.0                                      # all logits equal
    x[11] *= 1e-30
    targets = rng.integers(0, V, M).astype(np.float32)
    rows = Tensor.from_numpy(x).linear_cross_entropy(Tensor.from_numpy(w), Tensor.from_numpy(targets), reduction="none", precision="3xtf32").numpy()
    logits = x.astype(np.float64) @ w.astype(np.float64).T
    q, counted = hard(M, V, targets)
    want, _ = oracle(logits, q, counted, np.zeros(M), 1.0, "none")
    ok = np.arange(M) != 3
    assert np.isnan(rows[3])
    assert np.abs(rows[ok] - want[ok]).max() < 1e-5 * np.abs(want[ok]).max()
    assert rows[9] == pytest.approx(np.log(V), abs=1e-5) and rows[11] == pytest.approx(np.log(V), abs=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-18, 1e-3, 1e3, 1e12])
def test_linear_scales_far_from_one(gt, scale):
    """x large and w small by the same factor (or the other way round): the logits are ordinary, the operands are not."""
    rng = np.random.default_rng(9)
    M, V, E = 200, 1500, 96
    x, w = hidden(rng, M, V, E)
    x, w = (x * np.float32(scale)).astype(np.float32), (w / np.float32(scale)).astype(np.float32)
    targets = rng.integers(0, V, M).astype(np.float32)
    logits = x.astype(np.float64) @ w.astype(np.float64).T
    want, g = oracle(logits, *hard(M, V, targets), np.zeros(M), 1.0, "mean")
    loss, dx, dw = run_linear(x, w, lambda a, b: a.linear_cross_entropy(b, Tensor.from_numpy(targets), precision="3xtf32"))
    assert abs(loss[0] - want) < 1e-5
    assert rel(dx, g @ w) < 1e-5 and rel(dw, g.T @ x) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 300, 1e9, np.nan])
def test_ids_outside_the_vocabulary_are_reported(gt, bad):
    rng = np.random.default_rng(1)
    x, w = hidden(rng, 5, 300, 16)
    targets = np.array([1, 2, bad, 4, 5], np.float32)
    loss = Tensor.from_numpy(x).linear_cross_entropy(Tensor.from_numpy(w), Tensor.from_numpy(targets), reduction="none").numpy()
    with pytest.raises(RuntimeError, match="invalid argument"):
        _lib.device_status()
    assert loss[2] == 0.0 and loss[0] > 0.0                       # left out, the others untouched
    if not bad < 0:
        ids = np.array([[0, 1], [bad, 2], [2, 3], [3, 4], [4, 5]], np.float32)
        Tensor.from_numpy(x @ w.T).topk_distillation(Tensor.from_numpy(ids), Tensor.from_numpy(np.zeros((5, 2), np.float32)))
        with pytest.raises(RuntimeError, match="invalid argument"):
            _lib.device_status()
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("need", [("x",), ("w",)])
def test_one_gradient_alone(gt, need):
    rng = np.random.default_rng(2)
    M, V, E = 150, 1203, 56
    x, w = hidden(rng, M, V, E)
    targets = rng.integers(0, V, M).astype(np.float32)
    _, g = oracle(x.astype(np.float64) @ w.astype(np.float64).T, *hard(M, V, targets), np.zeros(M), 1.0, "sum")
    _, dx, dw = run_linear(x, w, lambda a, b: a.linear_cross_entropy(b, Tensor.from_numpy(targets), reduction="sum", precision="3xtf32"), need=need)
    if "x" in need:
        assert rel(dx, g @ w) < 1e-5
    else:
        assert rel(dw, g.T @ x) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("M, V, E", [(70, 2000, 64), (5, 2000, 64), (300, 70001, 48)])
def test_gradients_accumulate_and_scale(gt, M, V, E):
    """Existing gradients are added to; an upstream gradient other than 1; x and w used twice."""
    rng = np.random.default_rng(3)
    x, w = hidden(rng, M, V, E)
    targets = rng.integers(0, V, M).astype(np.float32)
    _, g = oracle(x.astype(np.float64) @ w.astype(np.float64).T, *hard(M, V, targets), np.zeros(M), 1.0, "mean")
    xt, wt, tt = Tensor.from_numpy(x, requires_grad=True), Tensor.from_numpy(w, requires_grad=True), Tensor.from_numpy(targets)
    xt.grad, wt.grad = Tensor.from_numpy(np.ones_like(x)), Tensor.from_numpy(np.ones_like(w))
    a = xt.linear_cross_entropy(wt, tt, precision="3xtf32")
    b = xt.linear_cross_entropy(wt, tt, precision="3xtf32")
    a.scale(0.25).add(b.scale(-2.0)).backward()
    assert rel(xt.grad.numpy(), 1.0 - 1.75 * (g @ w)) < 1e-5
    assert rel(wt.grad.numpy(), 1.0 - 1.75 * (g.T @ x)) < 1e-5
    # logits with a gradient in place already
    lt = Tensor.from_numpy((x @ w.T), requires_grad=True)
    lt.grad = Tensor.from_numpy(np.ones((M, V), np.float32))
    ids = Tensor.from_numpy(targets[:, None].copy())
    lt.topk_distillation(ids, Tensor.from_numpy(np.zeros((M, 1), np.float32))).scale(3.0).backward()
    _, g32 = oracle((x @ w.T).astype(np.float64), *hard(M, V, targets), np.zeros(M), 1.0, "mean")
    assert rel(lt.grad.numpy(), 1.0 + 3.0 * g32) < 2e-6


@pytest.mark.gpu
def test_losses_in_flight_do_not_share_memory(gt):
    """Two forward passes of different sizes before either backward, backward in the other order, and bit-equal repeats."""
    rng = np.random.default_rng(4)
    made = []
    for M, V, E in [(90, 3000, 64), (33, 5001, 80)]:
        x, w = hidden(rng, M, V, E)
        made.append((x, w, rng.integers(0, V, M).astype(np.float32)))

    def forward(i):
        x, w, t = made[i]
        xt, wt = Tensor.from_numpy(x, requires_grad=True), Tensor.from_numpy(w, requires_grad=True)
        return xt, wt, xt.linear_cross_entropy(wt, Tensor.from_numpy(t), precision="3xtf32")

    def result(f):
        f[2].backward()
        return f[2].numpy(), f[0].grad.numpy(), f[1].grad.numpy()

    alone = [result(forward(i)) for i in (0, 1)]
    a, b = forward(0), forward(1)
    rb, ra = result(b), result(a)
    for got, want in ((ra, alone[0]), (rb, alone[1])):
        for p, q in zip(got, want):
            assert np.array_equal(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("M, V, E", [(4, 9000, 96), (60, 2000, 200), (300, 30001, 100), (1100, 33001, 40), (700, 5000, 513)])
def test_repeats_are_equal_to_the_bit(gt, M, V, E):
    """Units of work are handed out as they come, sums are taken in a fixed order: the same call gives the same bits."""
    rng = np.random.default_rng([M, V])
    x, w = hidden(rng, M, V, E)
    ids, teacher = teacher_of(rng, M, V, 9)
    ti, tt = Tensor.from_numpy(ids), Tensor.from_numpy(teacher)
    runs = [run_linear(x, w, lambda a, b: a.linear_topk_distillation(b, ti, tt, temperature=2.0, precision="3xtf32")) for _ in range(4)]
    for run in runs[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(run, runs[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("M, V, E, K", [(1, 900, 96, 3), (12, 2000, 96, 1), (300, 5003, 104, 1), (300, 5003, 104, 7), (1100, 33001, 40, 5)])
def test_captured_and_replayed(gt, M, V, E, K):
    """Forward and backward of a linear loss, and a distillation of given logits with its gradient, captured from the context's
    stream and replayed on other inputs in the same buffers: the bits of the calls made one by one."""
    import torch

    lib, ctx = gt.load_library(), gt.context()
    stream = torch.cuda.ExternalStream(lib.gt_ctx_stream(ctx))
    mean, prec, T = gt.REDUCTIONS["mean"], gt.PREC_TF32X3, 1.0 if K == 1 else 1.5
    n_saved, n_scratch, n_given = c_size_t(0), c_size_t(0), c_size_t(0)
    gt.check(lib.gt_linear_loss_sizes(ctx, M, V, E, K, prec, byref(n_saved), byref(n_scratch)), "sizes")
    gt.check(lib.gt_topk_distillation_sizes(ctx, M, V, K, byref(n_given)), "sizes")

    def new(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    x, w, ids, teacher, logits = new(M, E), new(V, E), new(M, K), new(M, K), new(M, V)
    loss, dx, dw, loss_given, dlogits, one = new(1), new(M, E), new(V, E), new(1), new(M, V), torch.ones(1, device="cuda")
    saved, scratch, given = (new(n.value, dtype=torch.uint8) for n in (n_saved, n_scratch, n_given))

    def run():
        p = lambda t: c_void_p(t.data_ptr())          # noqa: E731
        if K == 1:
            gt.check(lib.gt_linear_cross_entropy(ctx, p(loss), p(saved), p(scratch), p(x), p(w), p(ids), M, V, E, -1.0, mean, prec), "forward")
        else:
            gt.check(lib.gt_linear_topk_distillation(ctx, p(loss), p(saved), p(scratch), p(x), p(w), p(ids), p(teacher), M, V, E, K, T, mean, prec),
                     "forward")
        gt.check(lib.gt_linear_loss_backward(ctx, p(dx), p(dw), p(saved), p(scratch), p(x), p(w), p(one), M, V, E, K, T, mean, prec, 0, 0), "backward")
        gt.check(lib.gt_topk_distillation(ctx, p(loss_given), p(given), p(dlogits), V, p(logits), V, p(ids), p(teacher), M, V, K, T, mean), "given")

    def fill(seed):
        rng = np.random.default_rng([M, V, K, seed])
        hx, hw = hidden(rng, M, V, E)
        hi, ht = teacher_of(rng, M, V, K, ragged=False)
        if M > 1:
            hi[seed] = -1.0                           # a row without a target, another one each time
        for t, a in ((x, hx), (w, hw), (ids, hi), (teacher, ht), (logits, rng.standard_normal((M, V)).astype(np.float32))):
            t.copy_(torch.from_numpy(a))
        torch.cuda.synchronize()

    def results():
        torch.cuda.synchronize()
        return [t.clone().cpu().numpy() for t in (loss, dx, dw, loss_given, dlogits)]

    want = []
    for seed in (1, 2):
        fill(seed)
        run()
        want.append(results())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run()
    for seed in (1, 2, 1):
        fill(seed)
        for t in (loss, dx, dw, loss_given, dlogits):
            t.fill_(np.nan)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        for got, wanted in zip(results(), want[seed - 1]):
            assert np.array_equal(got, wanted)
    gt.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("M, V, E", [(8192, 12800, 64), (2500, 40000, 130)])
def test_many_pieces_against_the_path_through_the_logits(gt, monkeypatch, M, V, E):
    """Several pieces of the vocabulary, dx of each added to the last: against linear_tied and cross_entropy, whose products are
    3xTF32 (5e-6 off); a third of the rows is left out."""
    monkeypatch.setenv("GRADTUITY_GEMM_PRECISION", "3xtf32")
    rng = np.random.default_rng(21)
    x, w = hidden(rng, M, V, E)
    targets = rng.integers(0, V, M).astype(np.float32)
    out = rng.random(M) < 0.33
    labels = np.where(out, -100, targets).astype(np.float32)
    loss, dx, dw = run_linear(x, w, lambda a, b: a.linear_cross_entropy(b, Tensor.from_numpy(labels)))
    xt, wt = Tensor.from_numpy(x[~out], requires_grad=True), Tensor.from_numpy(w, requires_grad=True)
    want = xt.linear_tied(wt).cross_entropy(Tensor.from_numpy(targets[~out]))
    assert loss[0] == pytest.approx(want.item(), rel=1e-5)
    want.backward()
    assert not dx[out].any()
    assert rel(dx[~out], xt.grad.numpy().astype(np.float64)) < 2e-5 and rel(dw, wt.grad.numpy().astype(np.float64)) < 2e-5


@pytest.mark.gpu
@pytest.mark.parametrize("M, V, E", [(1, 700, 64), (12, 700, 64), (150, 1200, 72)])
def test_rows_left_out_hold_garbage(gt, M, V, E):
    """Padding rows of NaN and infinities: no trace in the loss or dw, dx 0 there, or what it was when gradients accumulate."""
    rng = np.random.default_rng([22, M])
    x, w = hidden(rng, M, V, E)
    targets = rng.integers(0, V, M).astype(np.float32)
    out = rng.random(M) < 0.5
    out[0] = True
    targets[out] = -1
    logits = np.where(out[:, None], 0.0, x.astype(np.float64)) @ w.astype(np.float64).T
    want, g = oracle(logits, *hard(M, V, targets, -1), np.zeros(M), 1.0, "mean")
    x[out] = np.where(rng.random((int(out.sum()), E)) < 0.5, np.nan, np.inf)
    xt, wt = Tensor.from_numpy(x, requires_grad=True), Tensor.from_numpy(w, requires_grad=True)
    for times in (1, 2):
        loss = xt.linear_cross_entropy(wt, Tensor.from_numpy(targets), ignore_index=-1, precision="3xtf32")
        assert abs(loss.item() - want) < 1e-5
        loss.backward()
        clean = np.where(out[:, None], 0.0, x)
        dx = xt.grad.numpy()
        assert not dx[out].any()
        assert rel(dx, times * (g @ w)) < 1e-5 and rel(wt.grad.numpy(), times * (g.T @ clean)) < 1e-5
    assert _lib.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("V, E", [(30, 24), (300, 70)])
def test_one_tensor_as_input_and_weight(gt, V, E):
    rng = np.random.default_rng(23)
    w = (rng.standard_normal((V, E)) / np.sqrt(E)).astype(np.float32)
    targets = rng.integers(0, V, V).astype(np.float32)
    _, g = oracle(w.astype(np.float64) @ w.astype(np.float64).T, *hard(V, V, targets), np.zeros(V), 1.0, "mean")
    wt = Tensor.from_numpy(w, requires_grad=True)
    wt.linear_cross_entropy(wt, Tensor.from_numpy(targets), precision="3xtf32").backward()
    assert rel(wt.grad.numpy(), g @ w + g.T @ w) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("first", ["cross_entropy", "distillation"])
@pytest.mark.parametrize("B, C", [(40, 30001), (9, 500)])
def test_two_losses_of_the_same_logits(gt, first, B, C):
    """Both prepare the logits' gradient in their forward pass; one is taken over, the other added."""
    rng = np.random.default_rng(24)
    z = (rng.standard_normal((B, C)) * 2).astype(np.float32)
    targets = rng.integers(0, C, B).astype(np.float32)
    ids, teacher = teacher_of(rng, B, C, 6)
    q, counted = dense_targets(B, C, ids, teacher, 2.0)
    a, ga = oracle(z.astype(np.float64), *hard(B, C, targets), np.zeros(B), 1.0, "mean")
    b, gb = oracle(z.astype(np.float64), q, counted, entropy_of(B, ids, teacher, 2.0), 2.0, "mean")
    zt = Tensor.from_numpy(z, requires_grad=True)
    losses = [zt.cross_entropy(Tensor.from_numpy(targets)), zt.topk_distillation(Tensor.from_numpy(ids), Tensor.from_numpy(teacher), temperature=2.0)]
    if first == "distillation":
        losses.reverse()
    total = losses[0].add(losses[1])
    assert total.item() == pytest.approx(a + b, rel=1e-5)
    total.backward()
    assert rel(zt.grad.numpy(), ga + gb) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["linear_cross_entropy", "linear_topk_distillation", "topk_distillation"])
def test_gradients_against_differences(gt, op):
    """Central differences of the 32-bit loss along random directions: a loss of about 5 is exact to 5 2^-22, which the
    quotient divides by 2 h; the third-order term adds a multiple of h^2."""
    rng = np.random.default_rng(6)
    M, V, E, T = 24, 400, 32, 1.5
    x, w = hidden(rng, M, V, E, spread=1.0)
    logits = (x @ w.T).astype(np.float32)
    ids, teacher = teacher_of(rng, M, V, 6)
    ti, tt = Tensor.from_numpy(ids), Tensor.from_numpy(teacher)
    targets = Tensor.from_numpy(rng.integers(0, V, M).astype(np.float32))

    def value(arrays, grad=False):
        ts = [Tensor.from_numpy(a, requires_grad=grad) for a in arrays]
        if op == "linear_cross_entropy":
            loss = ts[0].linear_cross_entropy(ts[1], targets, precision="3xtf32")
        elif op == "linear_topk_distillation":
            loss = ts[0].linear_topk_distillation(ts[1], ti, tt, temperature=T, precision="3xtf32")
        else:
            loss = ts[0].topk_distillation(ti, tt, temperature=T)
        if not grad:
            return loss.item()
        loss.backward()
        return [t.grad.numpy().astype(np.float64) for t in ts]

    arrays = [logits] if op == "topk_distillation" else [x, w]
    grads = value(arrays, grad=True)
    for i, a in enumerate(arrays):
        for _ in range(3):
            d = rng.standard_normal(a.shape).astype(np.float32)
            h = 2.0 ** -5 if i == 0 else 2.0 ** -7
            shifted = [[(b + s * h * d).astype(np.float32) if j == i else b for j, b in enumerate(arrays)] for s in (1, -1)]
            quotient = (value(shifted[0]) - value(shifted[1])) / (2 * h)
            slope = float((grads[i] * d).sum())
            # a loss of about 5 in 32 bits, over 2 h, and the third derivative's h^2 / 6
            assert abs(quotient - slope) < 5 * 2.0 ** -22 / (2 * h) + h * h * max(1.0, abs(slope)) * 6


@pytest.mark.gpu
@pytest.mark.parametrize("C", [50257, 1003])
def test_distillation_of_padded_logits(gt, C):
    """Logits from linear_tied with padded rows: read in place, the gradient padded the same way."""
    rng = np.random.default_rng(12)
    M, E = 100, 64
    x, w = hidden(rng, M, C, E)
    ids, teacher = teacher_of(rng, M, C, 12)
    xt, wt = Tensor.from_numpy(x, requires_grad=True), Tensor.from_numpy(w, requires_grad=True)
    logits = xt.linear_tied(wt)
    padded = logits._pitch is not None
    assert padded == (C == 50257)
    z = logits.detach().numpy().astype(np.float64)
    loss = logits.topk_distillation(Tensor.from_numpy(ids), Tensor.from_numpy(teacher), temperature=2.0)
    q, counted = dense_targets(M, C, ids, teacher, 2.0)
    want, g = oracle(z, q, counted, entropy_of(M, ids, teacher, 2.0), 2.0, "mean")
    assert loss.item() == pytest.approx(want, rel=2e-6)
    loss.backward()
    assert rel(xt.grad.numpy(), g @ w) < 3.2e-3 and rel(wt.grad.numpy(), g.T @ x) < 3.2e-3       # the products are the default, tf32


# ---- together -------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_gpt2_trained_with_both_losses(gt, monkeypatch):
    """A small GPT-2 (tied head): its losses without logits and their gradients equal the ones through the logits, and a
    student's step mixes both."""
    from gradtuity_b200.gpt2.model import GPT2Small
    from gradtuity_b200.optim import AdamW

    monkeypatch.setenv("GRADTUITY_GEMM_PRECISION", "3xtf32")
    rng = np.random.default_rng(13)
    V, S, B = 333, 40, 2
    model = GPT2Small(vocab_size=V, n_positions=S, n_embd=64, n_layer=2, n_head=2, embd_pdrop=0.0, attn_pdrop=0.0, resid_pdrop=0.0)
    ids = Tensor.from_numpy(rng.integers(0, V, (B, S)).astype(np.float32))
    labels = Tensor.from_numpy(rng.integers(0, V, B * S).astype(np.float32))
    top_ids, top = teacher_of(rng, B * S, V, 7)
    ti, tt = Tensor.from_numpy(top_ids), Tensor.from_numpy(top)
    params = model.parameters()

    def step(loss):
        model.zero_grad()
        loss.backward()
        assert _lib.device_status() == 0
        return loss.item(), [p.grad.numpy() for p in params]

    full = lambda: model(ids).view((B * S, V))
    for a, b in ((model.loss(ids, labels), full().cross_entropy(labels)),
                 (model.distillation_loss(ids, ti, tt, temperature=2.0), full().topk_distillation(ti, tt, temperature=2.0))):
        la, ga = step(a)
        lb, gb = step(b)
        assert la == pytest.approx(lb, abs=1e-5)
        for p, u, v in zip(params, ga, gb):
            # the gradient of bk is a sum that cancels to nothing: measured against the largest gradient
            scale = max(np.linalg.norm(v), 1e-3 * max(np.linalg.norm(w) for w in gb))
            assert np.linalg.norm(u - v) < 5e-5 * scale
    opt = AdamW(params, lr=1e-3)
    mixed = model.loss(ids, labels).scale(0.5).add(model.distillation_loss(ids, ti, tt, temperature=2.0).scale(0.5))
    before = [p.numpy() for p in params]
    opt.zero_grad()
    mixed.backward()
    opt.step()
    assert _lib.device_status() == 0
    assert all(np.isfinite(p.numpy()).all() for p in params)
    assert any((p.numpy() != b).any() for p, b in zip(params, before))


@pytest.mark.gpu
def test_train_step_without_logits(gt, monkeypatch):
    """The training step's option gives the step's loss and the same updated parameters, up to the products' rounding."""
    from gradtuity_b200.gpt2.train import build_model, synthetic_batch, train_step
    from gradtuity_b200.optim import AdamW

    monkeypatch.setenv("GRADTUITY_GEMM_PRECISION", "3xtf32")
    ids, labels = synthetic_batch(0, 0, 2, 32, 301)
    losses, grads = [], []
    for keep in (True, False):
        model = build_model(vocab_size=301, seq_len=32, n_embd=64, n_layer=1, n_head=1)
        params = model.parameters()
        loss = train_step(model, AdamW(params, lr=1e-3), params, Tensor.from_numpy(ids), Tensor.from_numpy(labels), keep_logits=keep)
        assert _lib.device_status() == 0
        losses.append(loss.item())
        grads.append([p.grad.numpy() for p in params])
    assert losses[0] == pytest.approx(losses[1], abs=1e-5)
    largest = max(np.linalg.norm(g) for g in grads[0])
    for a, b in zip(*grads):
        assert np.linalg.norm(a - b) < 5e-5 * max(np.linalg.norm(a), 1e-3 * largest)
