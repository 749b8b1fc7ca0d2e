"""Scores and their gradient where logits are far from 0: classes masked by finite numbers, rows filled with one, rows whose maximum is large.

Tolerances, with u = 2^-24 (half a step of 32 bits), n classes and t_j = v_j - max v, s = sum e^t_j:
  an exponential: exp_of and exp2_of (ex2.approx.ftz.f32) are off by 2 steps of the result, and by u |t| for the rounding of their argument;
    1.2 |t| 2u covers base e, where the argument is rounded as a product. Long rows sum 2^(x L - M) with M = max L rounded: where the
    maximum is between -2^16 and 2^17, M is off by 2^17 L u < 2^-6, which the row's result takes back; elsewhere they are summed in base e.
  s: S = (2 + 1.2 ln n) 2u of itself, since E|t| <= ln n under p, and 4 sqrt(n / 32 + 8) u for adding n terms (a thread adds n / 32 at most).
  log s: B = S + 2u (1 + ln n).   log_sum = max + log s: B + u |log_sum|.   log p = t - log s: B + 2u |log p|, whatever the maximum.
  entropy = log s - E t: S (3 + 2 ln n) + 4u, whatever the maximum.
  gradient: p from log p = v - log_sum is off by what log_sum was rounded by, u |log_sum|, as long as |log_sum| is below FAR (64, and 1024
    for 16 bits: a sixteenth of their half step); beyond that it is computed again from the row, so that min(|log_sum|, FAR) u counts.
    p below 2^-126 counts as 0 (exp_of has no numbers below the normal ones), and a result there is rounded to them: 2^-125 (1 + |bracket|), the
    bracket being what multiplies p.
  results of 16 bits: half a step more.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
FAR = {torch.float32: 64.0, torch.float16: 1024.0, torch.bfloat16: 1024.0}
CLASSES = [5, 33, 300, 600, 1000, 2055, 4096, 9001, 70001]  # a thread, lanes, a warp, blocks, and clusters for few rows


@pytest.fixture(scope="module")
def answers():
    from visualmesh_b200 import answers
    return answers


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def near(got, want, tolerance):
    """Equal where want is not finite, else within tolerance."""
    fine = torch.isfinite(want)
    got = got.double()
    assert bool(((got == want) | (torch.isnan(got) & torch.isnan(want)) | fine).all()), "values that are not finite differ"
    off = torch.where(fine, (got - want).abs() - tolerance, torch.zeros_like(want))
    assert bool((off <= 0).all()), f"off by {float((got - want).abs()[fine].max()):.3g}, {float(off.max()):.3g} more than allowed"


def sum_error(n):
    return (2 + 1.2 * math.log(n)) * 2 * U + 4 * math.sqrt(n / 32 + 8) * U


def reference(x, labels, top):
    v = x.double()
    m = v.amax(1, keepdim=True)
    e = torch.exp(v - m)
    log_s = e.sum(1, keepdim=True).log()
    log_p = (v - m) - log_s
    p = torch.exp(log_p)
    entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(1)
    order = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :top]
    return log_p, p, log_p.gather(1, labels[:, None])[:, 0], entropy, (m + log_s)[:, 0], order


def check(answers, x, labels, top):
    """All scores of rows that have a distribution."""
    n = x.shape[1]
    got = answers.scores(x, labels, top)
    log_p, _, log_prob, entropy, log_sum, order = reference(x, labels, top)
    base = sum_error(n) + 2 * U * (1 + math.log(n))
    near(got.log_sum, log_sum, base + U * log_sum.abs())
    near(got.entropy, entropy, sum_error(n) * (3 + 2 * math.log(n)) + 4 * U)
    near(got.log_prob, log_prob, base + 2 * U * log_prob.abs().nan_to_num(0, 0, 0))
    if top:
        assert torch.equal(got.top_index.long(), order)
        best = log_p.gather(1, order)
        near(got.top_log_prob, best, base + 2 * U * best.abs().nan_to_num(0, 0, 0))
    return got


def masked_rows(rows, classes, dtype, value, seed):
    """Rows with a few allowed classes in every place of a row: in front, behind, a range in the middle, scattered, a masked range in front or behind, one alone."""
    q = generator(seed)
    x = (torch.randn((rows, classes), device="cuda", generator=q) * 3).to(dtype)
    kept = torch.zeros((rows, classes), dtype=torch.bool, device="cuda")
    few = min(8, max(1, classes // 2))
    for r in range(rows):
        kind = r % 7
        if kind == 0: kept[r, :few] = True
        elif kind == 1: kept[r, classes - few:] = True
        elif kind == 2: kept[r, classes // 2:classes // 2 + few] = True
        elif kind == 3: kept[r, torch.randperm(classes, device="cuda", generator=q)[:few]] = True
        elif kind == 4: kept[r, classes // 3:] = True
        elif kind == 5: kept[r, :classes - classes // 3] = True
        else: kept[r, classes - 1 - r % classes] = True
    labels = kept.int().argmax(1)
    return x.masked_fill(~kept, value), labels


def values_of(dtype):
    return [-1e4, -6e4] + ([] if dtype == torch.float16 else [-1e9, -1e10, -1e15, -1e20, -1e30, -1e35, -1e37, -5e37, -1e38])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_scores_of_classes_masked_by_finite_numbers(answers, classes, dtype):
    for rows in (3, 350):
        if rows * classes > 4_000_000:
            rows = 60
        for value in values_of(dtype):
            x, labels = masked_rows(rows, classes, dtype, value, classes)
            for top in (0, min(5, classes)):
                check(answers, x, labels, top)


def filled_rows(classes, dtype):
    """Rows of one value, and rows around one that may be far from 0."""
    values = [-1e4, -6e4, 6e4, 1e3]
    if dtype != torch.float16:
        values += [-7e4, 1e5, 2e5, -1e6, 1e6, -1e9, 1e9, -1e10, 1e10, -6e9, 6e9, -1e20, 1e20, -1e30, 1e30, -1e36, 1e36, -9e36, 9e36, -2e37, 2e37]
    values += [torch.finfo(dtype).min, torch.finfo(dtype).max]
    offset = torch.tensor(values, dtype=torch.float64, device="cuda")
    near_by = torch.randn((len(values), classes), device="cuda", dtype=torch.float64, generator=generator(classes)).clamp(-5, 5)
    limit = torch.finfo(dtype).max
    around = (offset[:, None] + near_by).clamp(-limit, limit)
    apart = (offset[:, None] * (1 + 2.0**-9 * near_by)).clamp(-limit, limit)  # neighbours of the type, far apart as logits
    return torch.cat([offset[:, None].expand(-1, classes), around, apart]).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", CLASSES)
def test_scores_of_rows_far_from_zero(answers, classes, dtype):
    x = filled_rows(classes, dtype)
    labels = torch.arange(x.shape[0], device="cuda") % classes
    for rows, chosen in ((x, labels), (x[:2], labels[:2]), (x.repeat(6, 1), labels.repeat(6))):
        for top in (0, min(5, classes)):
            check(answers, rows, chosen, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [5, 300, 1000, 1025, 2055, 9001, 70001])
def test_gradient_of_rows_with_a_clear_maximum_far_from_zero(answers, classes, dtype):
    """One class is all of the distribution (the others are masked, or some thousands below): log_sum is that logit, p is 1 there and 0 elsewhere, and
    the entropy 0 but for 4u."""
    values = [1e3, -1e3, 6e4, -6e4] + ([] if dtype == torch.float16 else [3e5, -3e5, 1e6, -1e6, 2e10, -2e10, 1e20, -1e20, 1e36, -1e36])
    rows = 2 * len(values)
    x = torch.tensor(values, dtype=torch.float64, device="cuda").repeat(2)[:, None].expand(rows, classes).clone()
    x[:len(values)] -= x[:len(values)].abs() * 0.25 + 300
    x[len(values):] = -math.inf
    winner = (torch.arange(rows, device="cuda") * 37 + classes // 2) % classes
    x.scatter_(1, winner[:, None], torch.tensor(values, dtype=torch.float64, device="cuda").repeat(2)[:, None])
    x = torch.where(x == -math.inf, x, x.clamp(min=torch.finfo(dtype).min)).to(dtype)
    q = generator(classes)
    d_l, d_e, d_s = (torch.randn(rows, device="cuda", generator=q) for _ in range(3))
    labels = (winner + torch.arange(rows, device="cuda") % 2) % classes  # every other label is another class
    got = answers.scores(x, labels)
    assert torch.equal(got.log_sum, x.gather(1, winner[:, None])[:, 0].float()) and bool((got.entropy.abs() <= 4 * U).all())
    dx = answers.scores_backward(x, got, labels, d_l, d_e, d_s)
    want = torch.zeros((rows, classes), dtype=torch.float64, device="cuda")
    want.scatter_add_(1, winner[:, None], (d_s - d_l).double()[:, None])
    there = torch.isfinite(x.gather(1, labels[:, None])[:, 0].float())  # a masked label's gradient is 0
    want.scatter_add_(1, labels[:, None], torch.where(there, d_l, torch.zeros_like(d_l)).double()[:, None])
    step = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    size = (d_s.abs() + d_l.abs() + d_e.abs()).double()[:, None]
    near(dx, want, want.abs() * step + torch.where(want != 0, 8 * U * size, torch.zeros_like(want)))


def check_gradient(answers, x, labels, grads):
    d_l, d_e, d_s = (d.double()[:, None] for d in grads)
    classes, dtype = x.shape[1], x.dtype
    got = answers.scores(x, labels)
    dx = answers.scores_backward(x, got, labels, *grads)
    log_p, p, _, entropy, log_sum, _ = reference(x, labels, 0)
    lp = torch.where(p > 0, log_p, torch.zeros_like(log_p))
    at = torch.zeros_like(p).scatter_(1, labels[:, None], 1.0)
    bracket = d_s - d_l - d_e * (lp + entropy[:, None])
    want = p * bracket + at * d_l
    base = sum_error(classes) + 2 * U * (1 + math.log(classes)) + U * log_sum.abs().clamp(max=FAR[dtype])[:, None]
    of_entropy = sum_error(classes) * (3 + 2 * math.log(classes)) + 4 * U
    error = p * (bracket.abs() * (base + 2.4 * U * lp.abs() + 8 * U) + d_e.abs() * (base + of_entropy + 2 * U * lp.abs()) + 4 * U * (d_s.abs() + d_l.abs() + d_e.abs() * (lp.abs() + entropy[:, None])))
    error += at * d_l.abs() * 2 * U
    if dtype != torch.float32:
        error += want.abs().clamp(min=torch.finfo(dtype).tiny) * torch.finfo(dtype).eps / 2
    near(dx, want, error + 2.0**-125 * (1 + bracket.abs()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [3, 5, 8, 16, 33, 100, 300, 700, 1024, 1025, 2055, 9001, 70001])
def test_gradient_of_rows_far_from_zero(answers, classes, dtype):
    """Wherever a row lies, its gradient is that of its distribution: a row of the type's lowest value has 1 / n for every class."""
    x = filled_rows(classes, dtype)
    labels = torch.arange(x.shape[0], device="cuda") % classes
    grads = [torch.randn(x.shape[0], device="cuda", generator=generator(classes + k)) for k in range(3)]
    check_gradient(answers, x, labels, grads)
    check_gradient(answers, x.repeat(7, 1), labels.repeat(7), [d.repeat(7) for d in grads])
    wide = torch.full((x.shape[0], classes + 3), math.nan, dtype=dtype, device="cuda")
    wide[:, 1:classes + 1] = x
    check_gradient(answers, wide[:, 1:classes + 1], labels, grads)  # rows that begin inside a piece


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [5, 33, 300, 1000, 2055, 9001, 70001])
def test_gradient_of_classes_masked_by_finite_numbers(answers, classes, dtype):
    for value in values_of(dtype):
        x, labels = masked_rows(21, classes, dtype, value, classes)
        grads = [torch.randn(x.shape[0], device="cuda", generator=generator(classes + k)) for k in range(3)]
        check_gradient(answers, x, labels, grads)
