"""The operators on answers against plain implementations in 64 bits.

Tolerances, with u = 2^-24 (half a step of 32 bits) and ulp = 2u:
  exponentials: __expf(t) is off by (2 + 1.17 |t|) ulp of itself, the division behind the factors of the recurrence by 2 ulp more.
  sums of scores: sum e^t with t <= 0 is off by (2 + 1.17 E|t|) ulp, E|t| <= ln n under p, and by what adding n terms rounds, taken as random:
    4 sqrt(n / 32 + 8) u (a thread adds n / 32 terms at most). So log_sum is off by S = (2 + 1.2 ln n) 2u + 4 sqrt(n / 32 + 8) u, plus u of
    itself, of the largest value and of v; entropy = log s - E t multiplies S by 1 + 2 (1 + ln n) at most. v = log p adds an ulp of v.
  recurrence: with e = (4 + 1.2 max |g|) 2u for a factor, its product and sum and the doubling of what a split over time adds, the error E_t
    and the majorant M_t of |h_t| obey E_t = f_t E_(t-1) + e M_t, M_t = f_t M_(t-1) + u_t |x_t|; the gradient's the same backwards.
  results of 16 bits: half a step more, eps / 2 of the value, or of the smallest normal value below it.
"""
import math

import pytest
import torch

from visualmesh_b200 import abi

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def answers():
    from visualmesh_b200 import answers
    return answers


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def half_step(v, dtype):
    """What rounding v to dtype may be off by."""
    if dtype == torch.float32:
        return torch.zeros_like(v)
    return v.abs().clamp(min=torch.finfo(dtype).tiny) * (torch.finfo(dtype).eps / 2)


def near(got, want, tolerance):
    """Equal where want is not finite, else within tolerance. What rounds beyond got's largest number (half a step, eps / 4 of it) is infinite there."""
    kind = torch.finfo(got.dtype)
    limit, sign = kind.max * (1 + kind.eps / 4), torch.sign(want)
    got = got.double()
    beyond = want.abs() > limit
    beyond |= (want.abs() + tolerance > limit) & (got == sign * math.inf)  # either is right
    want = torch.where(beyond, sign * math.inf, want)
    fine = torch.isfinite(want)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want)) | (beyond & (got.abs() + tolerance > limit) & (torch.sign(got) == sign))
    off = torch.where(fine, (got - want).abs() - tolerance, torch.zeros_like(want))
    assert bool((same | fine).all()), "values that are not finite differ"
    assert bool((off <= 0).all()), f"off by {float(((got - want).abs())[fine].max()):.3g}, {float(off[fine].max()):.3g} more than allowed"


# ---- scores ----------------------------------------------------------------------------------------------------------------

def reference_scores(x, labels, top, probabilities):
    v = x.double()
    if probabilities:
        v = torch.log(v)
    m = v.max(1, keepdim=True).values
    none = (m == -math.inf)[:, 0]
    bad = ~(m < math.inf)[:, 0]
    shift = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    e = torch.exp(v - shift)
    s = e.sum(1, keepdim=True)
    log_sum = torch.where(none, -math.inf, torch.where(bad, math.nan, (shift + s.log())[:, 0]))
    # from the difference: 64 bits do not hold log n beside the lowest value of 32 bits
    log_p = torch.where((v == -math.inf) & ~bad[:, None], -math.inf, torch.where(bad[:, None], math.nan, v - shift - s.log()))
    p = torch.exp(log_p)
    entropy = -torch.where(p > 0, p * log_p, torch.where(torch.isnan(p), p, torch.zeros_like(p))).sum(1)
    entropy = torch.where(none, 0.0, entropy)
    rows, classes = x.shape
    log_prob = None
    if labels is not None:
        inside = (labels >= 0) & (labels < classes)
        log_prob = log_p.gather(1, labels.long().clamp(0, classes - 1)[:, None])[:, 0]
        log_prob = torch.where(inside, log_prob, torch.where(labels == -1, 0.0, math.nan))
    key = torch.where(torch.isnan(x.double()), math.inf, x.double())
    # NaN first, then the largest, ties by index: two stable sorts
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    nan_last = torch.isnan(x).gather(1, order).logical_not().to(torch.int32)
    order = order.gather(1, torch.sort(nan_last, dim=1, stable=True).indices)[:, :top]
    return v, log_p, p, log_prob, entropy, log_sum, log_p.gather(1, order), order


def sum_error(n):
    return (2 + 1.2 * math.log(n)) * 2 * U + 4 * math.sqrt(n / 32 + 8) * U


def check_scores(answers, x, labels, top, probabilities=False):
    got = answers.scores(x, labels, top, probabilities)
    v, log_p, p, log_prob, entropy, log_sum, top_log_prob, order = reference_scores(x, labels, top, probabilities)
    n = x.shape[1]
    size = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(1)
    base = sum_error(n) + 2 * U * (size + log_sum.abs().nan_to_num(0, 0, 0)) + (4 * U * size if probabilities else 0)
    near(got.log_sum, log_sum, base)
    near(got.entropy, entropy, sum_error(n) * (3 + 2 * math.log(n)) + 4 * U + (8 * U if probabilities else 0))
    if labels is None:
        assert got.log_prob is None
    else:
        near(got.log_prob, log_prob, base + 2 * U * log_prob.abs().nan_to_num(0, 0, 0))
    if top:
        assert torch.equal(got.top_index.long(), order)
        near(got.top_log_prob, top_log_prob, base[:, None] + 2 * U * top_log_prob.abs().nan_to_num(0, 0, 0))
    else:
        assert got.top_index is None and got.top_log_prob is None
    return got


def reference_scores_grad(x, labels, d_log_prob, d_entropy, d_log_sum, probabilities):
    """(gradient, what it may be off by but for its rounding)"""
    rows, classes = x.shape
    v, log_p, p, _, entropy, log_sum, _, _ = reference_scores(x, None, 0, probabilities)
    zero = torch.zeros(rows, dtype=torch.float64, device=x.device)
    d_s, d_e = (zero if d is None else d.double() for d in (d_log_sum, d_entropy))
    d_l, at = zero, None
    if d_log_prob is not None:
        d_l = torch.where(labels == -1, 0.0, torch.where((labels >= 0) & (labels < classes), d_log_prob.double(), math.nan))
        at = torch.zeros_like(v)
        inside = (labels >= 0) & (labels < classes)
        at[inside, labels[inside].long()] = 1.0
    masked = v == -math.inf
    lp = torch.where(masked, 0.0, log_p)
    bracket = d_s[:, None] - d_l[:, None] - d_e[:, None] * (lp + entropy[:, None])
    weight = 1 / x.double().sum(1, keepdim=True) if probabilities else p
    dx = bracket * weight
    size = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(1, keepdim=True)
    base = sum_error(classes) + 4 * U * (size + log_sum.abs().nan_to_num(0, 0, 0)[:, None]) + 4 * U * lp.abs()
    error = (d_s.abs() + d_l.abs())[:, None] * weight * (base + 8 * U)
    error += weight * d_e.abs()[:, None] * ((lp + entropy[:, None]).abs() * (base + 8 * U) + base + sum_error(classes) * (3 + 2 * math.log(classes)) + 8 * U)
    if at is not None:
        part = torch.where(at > 0, d_l[:, None] / (x.double() if probabilities else 1.0), torch.zeros_like(at))
        dx = dx + part
        error += part.abs() * 4 * U
    return torch.where(masked, 0.0, dx), torch.where(masked, 0.0, error).nan_to_num(0, 0, 0)


def check_scores_grad(answers, x, labels, got, d_log_prob, d_entropy, d_log_sum, probabilities=False):
    dx = answers.scores_backward(x, got, labels, d_log_prob, d_entropy, d_log_sum, probabilities)
    want, error = reference_scores_grad(x, labels, d_log_prob, d_entropy, d_log_sum, probabilities)
    assert dx.dtype == x.dtype
    near(dx, want, error + half_step(want, x.dtype) + 1e-37)
    return dx


def answers_of(rows, classes, dtype, seed, probabilities=False):
    q = generator(seed)
    x = torch.randn((rows, classes), device="cuda", generator=q) * 2
    labels = torch.randint(0, classes, (rows,), device="cuda", generator=q)
    x.scatter_add_(1, labels[:, None], torch.rand((rows, 1), device="cuda", generator=q) * 6)
    if probabilities:
        x = torch.softmax(x, 1)
    labels[::7] = -1
    grads = [torch.randn(rows, device="cuda", generator=q) for _ in range(3)]
    return x.to(dtype), labels, grads


SIZES = [(1, 1), (3, 2), (1000, 3), (4, 4), (259, 5), (2049, 8), (64, 16), (70, 17), (70, 31), (65, 32), (33, 33), (9, 63), (10, 64), (11, 65), (5, 257), (3, 1000), (300, 1024), (7, 4099),
         (149, 8192), (2, 50021), (1, 131072), (3, 200003)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes", SIZES)
def test_scores(answers, rows, classes, dtype):
    x, labels, grads = answers_of(rows, classes, dtype, rows + classes)
    for top in sorted({0, 1, min(5, classes), min(32, classes)}):
        got = check_scores(answers, x, labels, top)
    check_scores_grad(answers, x, labels, got, *grads)
    check_scores_grad(answers, x, None, got, None, grads[1], None)
    check_scores_grad(answers, x, labels, got, grads[0], None, None)
    check_scores(answers, x, None, 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes", [(1, 1), (3, 2), (5000, 3), (257, 5), (1031, 13), (40, 33), (5, 300), (2, 5003)])
def test_scores_of_probabilities(answers, rows, classes, dtype):
    x, labels, grads = answers_of(rows, classes, dtype, rows + classes, True)
    got = check_scores(answers, x, labels.int(), min(3, classes), True)
    check_scores_grad(answers, x, labels.int(), got, *grads, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes", [(80001, 9), (60007, 16), (30001, 21), (30001, 32), (20003, 50), (20003, 64), (9001, 100), (5003, 128), (9001, 24), (4001, 200), (1300, 300), (5003, 300), (2501, 512), (320, 2400), (40, 33000), (1500, 2055), (400, 9000), (1200, 8300)])
def test_scores_of_many_rows(answers, rows, classes, dtype):
    """Rows one after another for the same lanes, and blocks of every size."""
    x, labels, grads = answers_of(rows, classes, dtype, rows)
    for top in (0, 1, 5):
        got = check_scores(answers, x, labels, top)
    check_scores_grad(answers, x, labels, got, *grads)
    p = torch.softmax(x.float(), 1).to(dtype)
    got = check_scores(answers, p, labels, 3, True)
    check_scores_grad(answers, p, labels, got, *grads, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [2, 3, 7, 32, 40, 500, 9001, 70001])
def test_scores_masks_and_special_values(answers, classes, dtype):
    x, labels, grads = answers_of(24, classes, dtype, classes)
    lowest, largest = torch.finfo(dtype).min, torch.finfo(dtype).max
    x[0] = -math.inf                      # nothing is left
    x[1, 1:] = -math.inf                  # one class is left
    x[2] = lowest                         # masked by the type's lowest value, all of it
    x[3, 1:] = lowest
    x[4, 0], x[4, 1:] = largest, lowest
    x[5, classes // 2] = math.nan
    x[6, classes - 1] = math.inf
    x[7] = math.inf
    x[8] = math.nan
    x[9] = 1.5                            # ties
    x[10] = 0.0
    x[10, ::2] = -0.0
    x[11, 0] = -math.inf
    x[12, :] = -math.inf
    x[12, classes - 1] = lowest
    x[13] = largest
    x[14, 0], x[14, 1] = math.nan, math.inf
    x[15, 0], x[15, 1] = -math.inf, math.nan
    x[16, : classes - 1] = -math.inf
    labels[:20] = torch.arange(20, device="cuda") % classes
    labels[17], labels[18], labels[19] = classes, -2, -1
    labels[20] = 2**40 + 1
    for top in (1, min(classes, 6)):
        got = check_scores(answers, x, labels, top)
    check_scores_grad(answers, x, labels, got, *grads)
    labels[20] = -1
    for wide in (labels, labels.int()):
        got = check_scores(answers, x, wide, min(classes, 2))
        check_scores_grad(answers, x, wide, got, *grads)


@pytest.mark.parametrize("classes", [2, 5, 33, 3000])
def test_scores_of_probabilities_that_are_none(answers, classes):
    x, labels, grads = answers_of(12, classes, torch.float32, classes, True)
    x[0] = 0.0
    x[1, 0] = 0.0
    x[2, 1:], x[2, 0] = 0.0, 1.0
    x[3, 0] = -0.25
    x[4, classes - 1] = math.nan
    x[5, 0] = math.inf
    x[6] *= 2.5                           # not normalised: it is made so
    x[7] = 2.0**-140                      # below the normal numbers
    labels[:8] = 0
    got = check_scores(answers, x, labels, 2, True)
    large = answers.scores(torch.tensor([[2.0**90] * classes, [2.0**97] + [1.0] * (classes - 1)], device="cuda"), labels[:2], 2, True)
    near(large.entropy[:1], torch.tensor([math.log(classes) if classes <= 64 else math.nan], dtype=torch.float64, device="cuda"), sum_error(classes) * (3 + 2 * math.log(classes)) + 2 * U * math.log(2.0**90 * classes))
    assert bool(torch.isnan(large.entropy[1])) and bool(torch.isnan(large.log_sum[1])) and bool(torch.isnan(large.log_prob[1])) and large.top_index[1].tolist() == [0, 1]
    # gradients of rows with a distribution; 2^-140 has an inverse that 32 bits cannot hold
    keep = torch.tensor([0, 1, 2, 6, 8, 9, 10, 11], device="cuda")
    part = answers.Scores(None, got.entropy[keep].contiguous(), got.log_sum[keep].contiguous(), None, None)
    check_scores_grad(answers, x[keep].contiguous(), labels[keep].contiguous(), part, *(g[keep].contiguous() for g in grads), True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes,gap,offset", [(3, 2, 1), (5, 0, 3), (16, 1, 0), (64, 8, 8), (257, 3, 5), (1024, 8, 1), (4096, 16, 8), (20000, 1, 1)])
def test_scores_of_rows_with_gaps(answers, classes, gap, offset, dtype):
    """Row strides and addresses that no vector load fits, and what lies between the rows left alone."""
    rows = 37
    wide, labels, grads = answers_of(rows, classes + gap, dtype, classes)
    flat = torch.full((rows * (classes + gap) + offset + 8,), math.nan, dtype=dtype, device="cuda")
    x = flat[offset:offset + rows * (classes + gap)].view(rows, classes + gap)[:, :classes]
    x.copy_(wide[:, :classes])
    labels = labels.clamp(max=classes - 1)
    got = check_scores(answers, x, labels, 2)
    check_scores_grad(answers, x, labels, got, *grads)
    # the same row for all of them
    same = x[:1].expand(rows, classes)
    got = check_scores(answers, same, labels, 2)
    check_scores_grad(answers, same, labels, got, *grads)
    # a gradient written between other values, by the C entry point
    into = torch.full((rows, classes + 9), 7.0, dtype=dtype, device="cuda")
    dx = answers.scores_backward(x, got, labels, *grads)
    got = answers.scores(x, labels)
    kind = {torch.float32: abi.VM_F32, torch.float16: abi.VM_F16, torch.bfloat16: abi.VM_BF16}[dtype]
    abi.check(abi.load().vm_scores_backward(-1, x.data_ptr(), kind, rows, classes, x.stride(0), abi.VM_LABELS_64, labels.data_ptr(), got.entropy.data_ptr(), got.log_sum.data_ptr(),
                                            grads[0].data_ptr(), grads[1].data_ptr(), grads[2].data_ptr(), into.data_ptr() + 4 * dtype.itemsize, classes + 9,
                                            torch.cuda.current_stream().cuda_stream))
    assert torch.equal(into[:, 4:4 + classes], answers.scores_backward(x, got, labels, *grads))
    assert bool((into[:, :4] == 7).all()) and bool((into[:, 4 + classes:] == 7).all()) and dx.shape == x.shape


def test_scores_in_ascending_order(answers):
    """Every value displaces one of the best so far."""
    x = torch.arange(60000, device="cuda", dtype=torch.float32).view(4, -1) / 4096
    check_scores(answers, x, torch.zeros(4, dtype=torch.int32, device="cuda"), 32)
    check_scores(answers, x.flip(1).contiguous(), None, 32)
    check_scores(answers, torch.zeros((3, 40000), device="cuda", dtype=torch.float16), None, 32)


@pytest.mark.parametrize("probabilities", [False, True])
def test_scores_gradient_against_differences(answers, probabilities):
    """Central differences of the definition in 64 bits: their own error, h^2 / 6 of the third derivative, is below 1e-7 at h = 1e-4."""
    x, labels, (d_l, d_e, d_s) = answers_of(6, 5, torch.float32, 3, probabilities)
    x = x.clamp(min=0.05) if probabilities else x * 0.3
    labels = torch.tensor([0, 1, 4, -1, 2, 3], device="cuda")

    def loss(v):
        _, _, _, log_prob, entropy, log_sum, _, _ = reference_scores(v, labels, 0, probabilities)
        return (d_l.double() * log_prob + d_e.double() * entropy + d_s.double() * log_sum).sum(0)

    dx = answers.scores_backward(x, answers.scores(x, labels, probabilities=probabilities), labels, d_l, d_e, d_s, probabilities)
    h = 1e-4 if not probabilities else 1e-5
    for r in range(6):
        for c in range(5):
            step = torch.zeros((6, 5), dtype=torch.float64, device="cuda")
            step[r, c] = h
            want = float((loss(x.double() + step) - loss(x.double() - step)) / (2 * h))
            assert abs(float(dx[r, c]) - want) <= 1e-5 * (1 + abs(want))


def test_scores_of_more_elements_than_32_bits_count(answers):
    rows, classes = 70001, 32768 + 11
    x = torch.zeros((rows, classes), dtype=torch.float16, device="cuda")
    x[-3:] = torch.randn((3, classes), device="cuda", generator=generator(1)).half()
    labels = torch.randint(0, classes, (rows,), device="cuda", generator=generator(2))
    got = answers.scores(x, labels, 3)
    # how a row is split between blocks depends on how many there are, so the last rows are held to 64 bits and not to another call's digits
    _, _, _, log_prob, entropy, log_sum, top_log_prob, order = reference_scores(x[-3:], labels[-3:], 3, False)
    base = sum_error(classes) + 2 * U * 32
    assert torch.equal(got.top_index[-3:].long(), order)
    near(got.log_sum[-3:], log_sum, base)
    near(got.log_prob[-3:], log_prob, base + 2 * U * log_prob.abs())
    near(got.top_log_prob[-3:], top_log_prob, base + 2 * U * top_log_prob.abs())
    near(got.entropy[-3:], entropy, sum_error(classes) * (3 + 2 * math.log(classes)) + 4 * U)
    assert bool((got.log_sum[:-3] - math.log(classes)).abs().max() < sum_error(classes) + 32 * U)
    d = torch.full((rows,), -1.0, device="cuda")
    dx = answers.scores_backward(x, got, labels, d)
    want, error = reference_scores_grad(x[-3:], labels[-3:], d[-3:], None, None, False)
    near(dx[-3:], want, error + half_step(want, x.dtype))


# ---- recurrence --------------------------------------------------------------------------------------------------------------

def factors(g):
    f = 1 / (1 + torch.exp(-g))
    return f, 1 / (1 + torch.exp(g))


def times(a, b):
    return torch.where(a == 0, torch.zeros_like(b), a * b)


def recurrence(f, v, first):
    """All h_t = f_t h_(t-1) + v_t from h_(-1) = first, a factor of 0 dropping what it multiplies; by doubling: the composition of steps is one of their kind."""
    v = torch.cat([(v[:, :1] + times(f[:, :1], first[:, None])), v[:, 1:]], 1)
    step = 1
    while step < f.shape[1]:
        v = torch.cat([v[:, :step], v[:, step:] + times(f[:, step:], v[:, :-step])], 1)
        f = torch.cat([f[:, :step], times(f[:, step:], f[:, :-step])], 1)
        step *= 2
    return v


def reference_scan(x, g, h0, lengths, dy=None, d_last=None):
    """Values and what they may be off by (but for their rounding): y, last, states, and with gradients dx, d_gate, d_h0"""
    x, g = x.double(), g.double()
    batch, steps, channels = x.shape
    f, u = factors(g)
    widest = torch.where(torch.isfinite(g), g.abs(), torch.zeros_like(g))
    e = (4 + 1.2 * (float(widest.max()) if g.numel() else 0.0)) * 2 * U * 2
    first = torch.zeros((batch, channels), dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    on = torch.ones((batch, steps, 1), dtype=torch.bool, device=x.device)
    if lengths is not None:
        on = (torch.arange(steps, device=x.device)[None, :] < lengths[:, None])[:, :, None]
    zero = torch.zeros_like(x)
    f, u = torch.where(on, f, 1.0), torch.where(on, u, 0.0)
    h = recurrence(f, times(u, x), first)
    m = recurrence(f, times(u, x.abs()), first.abs())
    error = recurrence(f, torch.where(on, e * m, zero), torch.zeros_like(first))
    end = lambda v, start: v[:, -1] if steps else start
    before, before_m, before_e = (torch.cat([start[:, None], v], 1)[:, :steps] for v, start in ((h, first), (m, first.abs()), (error, torch.zeros_like(first))))
    keep = abi.VM_GATED_KEEP
    out = [(torch.where(on, h, zero), torch.where(on, error, zero)), (end(h, first), end(error, torch.zeros_like(first))), (before[:, ::keep], before_e[:, ::keep])]
    if dy is None and d_last is None:
        return out
    dy = torch.where(on, zero if dy is None else dy.double(), zero)
    last = torch.zeros_like(first) if d_last is None else d_last.double()
    if steps == 0:
        return out + [(zero, zero), (zero, zero), (last, torch.zeros_like(last))]
    # backwards: c_t = f_t dy_t + f_t c_(t+1), from c_T = last
    back = lambda v, start: recurrence(f.flip(1), v.flip(1), start).flip(1)
    later = lambda v, start: torch.cat([v[:, 1:], start[:, None]], 1)
    c, c_m = back(times(f, dy), last), back(times(f, dy.abs()), last.abs())
    total, total_m = dy + later(c, last), dy.abs() + later(c_m, last.abs())
    # a total is off by what the carry behind it is, and e of its majorant; the carry by f of that, and e of its own
    c_e = back(torch.where(on, times(f, e * total_m) + e * c_m, zero), torch.zeros_like(last))
    total_e = later(c_e, torch.zeros_like(last)) + e * total_m
    fu, reach = f * u, before_m + x.abs()
    return out + [(times(u, total), times(u, total_e + e * total_m)),
                  (times(fu, (before - x) * total), times(fu, (before_e + e * reach) * total_m + reach * (total_e + 2 * e * total_m))),
                  (c[:, 0], c_e[:, 0])]


def check_scan(answers, x, g, h0=None, lengths=None, dy=None, d_last=None):
    got = answers.gated_scan(x, g, h0, lengths, keep=True)
    want = reference_scan(x, g, h0, lengths, dy, d_last)
    have = [got.y, got.last, got.states]
    if dy is not None or d_last is not None:
        have += list(answers.gated_scan_backward(x, g, got.states, dy, d_last, lengths))
    for name, value, (right, error) in zip(("y", "last", "states", "dx", "d_gate", "d_h0"), have, want):
        assert value.shape == right.shape, name
        assert value.dtype == (x.dtype if name in ("y", "dx", "d_gate") else torch.float32), name
        near(value, right, error.nan_to_num(0, 0, 0) + half_step(right, value.dtype) + 1e-37)
    plain = answers.gated_scan(x, g, h0, lengths)
    assert plain.states is None and same(plain.y, got.y) and same(plain.last, got.last)
    return got, have[3:]


def same(a, b):
    return a.dtype == b.dtype and torch.equal(a.nan_to_num(12345.0), b.nan_to_num(12345.0)) and torch.equal(torch.isnan(a), torch.isnan(b))


def sequences(batch, steps, channels, dtype, seed):
    q = generator(seed)
    shape = (batch, steps, channels)
    x, dy = (torch.randn(shape, device="cuda", generator=q).to(dtype) for _ in range(2))
    g = (torch.randn(shape, device="cuda", generator=q) * 1.5 + 2).to(dtype)
    h0, d_last = (torch.randn((batch, channels), device="cuda", generator=q) for _ in range(2))
    return x, g, h0, dy, d_last


SCANS = [(1, 1, 1), (2, 0, 3), (1, 2, 64), (3, 63, 5), (2, 64, 8), (2, 65, 33), (1, 127, 1), (1, 257, 96), (5, 33, 40), (1, 1000, 130), (2, 511, 512), (3, 300, 515), (1, 1500, 16), (2, 700, 7),
         (1, 129, 4096), (1, 40, 20011), (40, 12, 1), (700, 70, 3)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,steps,channels", SCANS)
def test_scan(answers, batch, steps, channels, dtype):
    x, g, h0, dy, d_last = sequences(batch, steps, channels, dtype, steps + channels)
    check_scan(answers, x, g, h0, None, dy, d_last)
    check_scan(answers, x, g, None, None, dy, None)
    lengths = torch.randint(0, steps + 1, (batch,), device="cuda", generator=generator(batch)).to(torch.int32)
    lengths[0] = steps
    lengths[-1] = steps // 2
    check_scan(answers, x, g, h0, lengths, dy, d_last)
    check_scan(answers, x, g, h0, None, None, d_last)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,steps,channels", [(1, 20000, 16), (1, 9001, 3), (2, 5000, 64), (1, 4097, 512)])
def test_scan_of_long_sequences(answers, batch, steps, channels, dtype):
    """Long enough to be split over time."""
    x, g, h0, dy, d_last = sequences(batch, steps, channels, dtype, steps)
    lengths = torch.tensor([steps - 77, 0][:batch], dtype=torch.int32, device="cuda")
    check_scan(answers, x, g, h0, None, dy, d_last)
    check_scan(answers, x, g, h0, lengths, dy, d_last)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,steps,channels", [(1, 70, 76001), (30000, 67, 3), (2, 66, 40002), (1, 64, 20003), (9000, 17, 4), (2, 33, 9002), (3, 1, 8000), (5, 8, 16384), (1, 0, 20000)])
def test_scan_of_many_sequences(answers, batch, steps, channels, dtype):
    """Enough for a thread each, where they are single elements; states are kept twice."""
    x, g, h0, dy, d_last = sequences(batch, steps, channels, dtype, 3)
    g[:, steps // 5:steps // 5 + 1] = -math.inf
    lengths = torch.randint(0, steps + 1, (batch,), device="cuda", generator=generator(batch)).to(torch.int32)
    check_scan(answers, x, g, h0, None, dy, d_last)
    check_scan(answers, x, g, None, lengths, dy, None)
    beside = [torch.empty(batch * channels + 1, device="cuda")[1:].view(batch, channels).copy_(v) for v in (h0, d_last)]  # no vector load fits them
    check_scan(answers, x, g, beside[0], lengths, None, beside[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("steps,channels", [(50, 8), (200, 3), (3000, 24), (9000, 6), (60, 80001), (50, 20002), (300, 76000)])
def test_scan_gates_that_drop(answers, steps, channels, dtype):
    """-inf drops the past, +inf the present, whatever is there; a gate of NaN drops nothing."""
    x, g, h0, dy, d_last = sequences(1, steps, channels, dtype, steps)
    g[:, 3] = math.inf
    x[:, 3, 0], x[:, 3, 1], x[:, 3, 2] = math.nan, math.inf, -math.inf
    g[:, steps // 2] = -math.inf
    h0[0, 0], h0[0, 1] = math.inf, math.nan
    g[0, 0, 0] = g[0, 0, 1] = -math.inf
    x[:, steps // 2 - 1, 2] = math.inf
    g[:, steps - 1] = math.inf
    big = 3e4
    g[0, 7, 0], g[0, 8, 0] = big, -big
    dy[0, steps // 2 - 2, 2] = 0.0
    got = answers.gated_scan(x, g, h0, keep=True)
    want = reference_scan(x, g, h0, None)
    near(got.y, want[0][0], want[0][1].nan_to_num(0, 0, 0) + half_step(want[0][0], dtype) + 1e-37)
    near(got.last, want[1][0], want[1][1].nan_to_num(0, 0, 0))
    # finite values everywhere but where a gate drops them: finite gradients
    x[:, steps // 2 - 1, 2] = 0.5
    g[0, 8, 0] = 0.5
    got = check_scan(answers, x, g, h0, None, dy, d_last)
    assert bool(torch.isfinite(got[1][0]).all()) and bool(torch.isfinite(got[1][1]).all())
    g[0, 9, 0] = math.nan
    y = answers.gated_scan(x, g, h0).y
    assert bool(torch.isnan(y[0, 9:steps // 2, 0]).all()) and not bool(torch.isnan(y[0, steps // 2:, 0]).any())


def test_scan_lengths_are_clamped(answers):
    x, g, h0, dy, d_last = sequences(4, 70, 9, torch.float32, 5)
    odd = torch.tensor([-5, 2**30, 70, -2**31], dtype=torch.int32, device="cuda")
    clamped = odd.clamp(0, 70)
    for a, b in zip(answers.gated_scan(x, g, h0, odd, keep=True), answers.gated_scan(x, g, h0, clamped, keep=True)):
        assert torch.equal(a, b)
    states = answers.gated_scan(x, g, h0, odd, keep=True).states
    for a, b in zip(answers.gated_scan_backward(x, g, states, dy, d_last, odd), answers.gated_scan_backward(x, g, states, dy, d_last, clamped)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,steps,channels", [(3, 90, 16), (2, 2500, 24)])
def test_scan_of_other_layouts(answers, batch, steps, channels, dtype):
    """Whatever the strides, the numbers are those of dense copies: transposed, padded, off their alignment, repeated."""
    x, g, h0, dy, d_last = sequences(batch, steps, channels, dtype, 11)
    dense = check_scan(answers, x, g, h0, None, dy, d_last)

    def layouts(v):
        yield v.transpose(0, 1).contiguous().transpose(0, 1)
        yield v.transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.full((batch, steps, channels + 3), math.nan, dtype=dtype, device="cuda")
        wide[:, :, 1:channels + 1] = v
        yield wide[:, :, 1:channels + 1]
        padded = torch.full((batch, steps, channels * 2), math.nan, dtype=dtype, device="cuda")
        padded[:, :, ::2] = v
        yield padded[:, :, ::2]

    for a, b, c in zip(layouts(x), layouts(g), layouts(dy)):
        got = answers.gated_scan(a, b, h0, keep=True)
        grads = answers.gated_scan_backward(a, b, got.states, c, d_last)
        for have, want in zip(list(got) + list(grads), list(dense[0]) + list(dense[1])):
            error = 1e-5 * (1 + want.double().abs()) + 2 * half_step(want.double(), want.dtype)
            near(have, want.double(), error)
    # a gate for all channels of a step, one for a channel at all steps, one for all; a row of x for all steps
    for gate in (g[:, :, :1].expand(x.shape), g[:1, :1].expand(x.shape), g[:1, :1, :1].expand(x.shape)):
        check_scan(answers, x, gate, h0, None, dy, d_last)
    check_scan(answers, x[:, :1].expand(x.shape), g, h0, None, dy[:, :, :1].expand(x.shape), d_last)


def test_scan_nodes_by_steps_by_classes(answers):
    """Frames of nodes with a few classes and one gate for a node: batch and channels far apart in memory."""
    frames, nodes, classes = 30, 501, 3
    x, g, _, dy, _ = sequences(frames, nodes, classes, torch.float32, 2)
    h0 = torch.rand((nodes, classes), device="cuda")
    by_node = lambda v: v.transpose(0, 1)
    check_scan(answers, by_node(x), by_node(g[:, :, :1].expand(x.shape)), h0, None, by_node(dy), None)


def test_scan_gradient_against_differences(answers):
    """Central differences of the definition in 64 bits, h = 1e-4: their own error is below 1e-7."""
    x, g, h0, dy, d_last = sequences(2, 5, 2, torch.float32, 7)

    def loss(x, g, h0):
        y, last, _ = (v for v, _ in reference_scan(x, g, h0, None))
        return float((dy.double() * y).sum() + (d_last.double() * last).sum())

    got = answers.gated_scan(x, g, h0, keep=True)
    have = answers.gated_scan_backward(x, g, got.states, dy, d_last)
    values = [v.double() for v in (x, g, h0)]
    for k in range(3):
        flat = have[k].flatten()
        for i in range(flat.numel()):
            step = torch.zeros_like(values[k])
            step.view(-1)[i] = 1e-4
            up, down = list(values), list(values)
            up[k], down[k] = values[k] + step, values[k] - step
            want = (loss(*up) - loss(*down)) / 2e-4
            assert abs(float(flat[i]) - want) <= 1e-5 * (1 + abs(want))


def test_scan_offsets_beyond_32_bits(answers):
    """Rows 2^30 elements apart: the third begins behind 2^31."""
    step = 2**30
    flat = torch.zeros(2 * step + 4096, dtype=torch.float16, device="cuda")
    x, g, h0, dy, d_last = sequences(1, 3, 40, torch.float16, 3)
    far = torch.as_strided(flat, (1, 3, 40), (1, step, 1))
    far.copy_(x)
    want = answers.gated_scan(x, g, h0, keep=True)
    got = answers.gated_scan(far, g, h0, keep=True)
    assert torch.equal(got.y, want.y) and torch.equal(got.last, want.last)
    for a, b in zip(answers.gated_scan_backward(far, g, want.states, dy, d_last), answers.gated_scan_backward(x, g, want.states, dy, d_last)):
        assert torch.equal(a, b)


# ---- steps -------------------------------------------------------------------------------------------------------------------

def check_step(answers, state, x, g, index):
    slots, channels = state.shape
    rows = x.shape[0]
    f, u = factors(g.double())
    e = (6 + 1.2 * float(torch.where(torch.isfinite(g), g.abs(), torch.zeros_like(g)).max())) * 2 * U
    names = list(range(rows)) if index is None else index.tolist()
    want, taken = state.double().clone(), set()
    y, error = torch.zeros_like(f), torch.zeros_like(f)
    table_error = torch.zeros_like(want)
    for r, slot in enumerate(names):
        if not 0 <= slot < slots or slot in taken:
            continue
        taken.add(slot)
        y[r] = times(f[r], want[slot]) + times(u[r], x[r].double())
        error[r] = e * (times(f[r], want[slot].abs()) + times(u[r], x[r].double().abs()))
        want[slot], table_error[slot] = y[r], error[r]
    before = state.clone()
    got = answers.gated_step(state, x, g, index)
    assert got.dtype == x.dtype
    near(got, y, error + half_step(y, x.dtype) + 1e-37)
    near(state, want, table_error + 1e-37)
    left = [s for s in range(slots) if s not in taken]
    assert torch.equal(state[left], before[left])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,slots,channels", [(1, 1, 1), (1, 9, 4096), (3, 3, 7), (64, 100, 64), (65, 70, 33), (300, 1000, 3), (250, 1000, 5), (900, 1000, 96), (1500, 1501, 2), (2500, 9000, 5), (5, 6, 20000)])
def test_step(answers, rows, slots, channels, dtype):
    q = generator(rows)
    state = torch.randn((slots, channels), device="cuda", generator=q)
    x, g = ((torch.randn((rows, channels), device="cuda", generator=q) * 2).to(dtype) for _ in range(2))
    check_step(answers, state, x, g, None)
    index = torch.randperm(slots, device="cuda", generator=q)[:rows].int()
    check_step(answers, state, x, g, index)
    index[::5] = -1
    index[1::9] = slots
    index[2::11] = -2**31
    check_step(answers, state, x, g, index)
    g[::3], g[1::3] = math.inf, -math.inf
    check_step(answers, state, x, g, index)


@pytest.mark.parametrize("channels", [6, 64])
@pytest.mark.parametrize("rows", [2, 40, 256, 257, 700, 1025, 3000])
def test_step_of_a_slot_named_twice(answers, rows, channels):
    """The first row that names a slot advances it, each time the same."""
    q = generator(rows)
    x, g = (torch.randn((rows, channels), device="cuda", generator=q) for _ in range(2))
    index = torch.randint(0, 1 + rows // 3, (rows,), device="cuda", generator=q).int()
    for _ in range(3):
        check_step(answers, torch.ones((rows, channels), device="cuda"), x, g, index)
    check_step(answers, torch.ones((rows, channels), device="cuda"), x, g, torch.full_like(index, rows - 1))
    none = torch.empty((0, channels), device="cuda")
    assert not bool(answers.gated_step(none, x, g, index).any())


@pytest.mark.parametrize("dtype", TYPES)
def test_step_of_other_layouts(answers, dtype):
    q = generator(4)
    table = torch.randn((50, 24), device="cuda", generator=q)
    x = torch.randn((24, 40), device="cuda", generator=q).to(dtype)
    index = torch.randperm(50, device="cuda", generator=q)[:20].int()
    check_step(answers, table[:, 1:22], x[3:24, 10:30].t(), x[0, :1].expand(20, 21), index)
    check_step(answers, table[::2, :16], x[:20, 8:24], x[:20, 8:24], (index // 2).contiguous())
    out = torch.full((20, 30), 7.0, dtype=dtype, device="cuda")
    y = answers.gated_step(table[:, :16].clone(), x[:20, 8:24], x[:20, :16], index)
    again = answers.gated_step(table[:, :16].clone(), x[:20, 8:24], x[:20, :16], index, out=out[:, 5:21])
    assert torch.equal(again, y) and bool((out[:, :5] == 7).all()) and bool((out[:, 21:] == 7).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_steps_follow_the_scan(answers, dtype):
    x, g, h0, _, _ = sequences(6, 40, 24, dtype, 1)
    scan = answers.gated_scan(x, g, h0)
    state = torch.zeros((9, 24), device="cuda")
    index = torch.tensor([8, 2, 0, 5, 7, 1], dtype=torch.int32, device="cuda")
    state[index.long()] = h0
    for t in range(40):
        y = answers.gated_step(state, x[:, t], g[:, t], index)
        near(y, scan.y[:, t].double(), 2e-5 + 2 * half_step(scan.y[:, t].double(), dtype))
    near(state[index.long()], scan.last.double(), 2e-5)


# ---- how they are called -----------------------------------------------------------------------------------------------------

def test_refusals_of_tensors(answers):
    x = torch.zeros((4, 8), device="cuda")
    s = torch.zeros((2, 5, 8), device="cuda")
    labels = torch.zeros(4, dtype=torch.int64, device="cuda")
    got = answers.scores(x, labels)
    states = answers.gated_scan(s, s, keep=True).states
    bad = [
        lambda: answers.scores(x.double()), lambda: answers.scores(x[0]), lambda: answers.scores(x.t()[:, ::2].t().t()), lambda: answers.scores(x, labels.short()),
        lambda: answers.scores(x, labels[:3]), lambda: answers.scores(x, labels.cpu()), lambda: answers.scores(x, top=9), lambda: answers.scores(x, top=-1),
        lambda: answers.scores(torch.zeros((4, 0), device="cuda")), lambda: answers.scores(x.clone().requires_grad_()),
        lambda: answers.scores(x, torch.zeros(8, dtype=torch.int64, device="cuda")[::2]),
        lambda: answers.scores_backward(x, got, None, x[:, 0].contiguous()), lambda: answers.scores_backward(x, got, labels, x[:, 0]),
        lambda: answers.scores_backward(x, got, labels, torch.zeros(4, dtype=torch.float64, device="cuda")),
        lambda: answers.gated_scan(s, s.half()), lambda: answers.gated_scan(s, s[:1]), lambda: answers.gated_scan(s, s.cpu()), lambda: answers.gated_scan(x, x),
        lambda: answers.gated_scan(s, s, torch.zeros((2, 8), device="cuda").half()), lambda: answers.gated_scan(s, s, torch.zeros((8, 2), device="cuda").t()),
        lambda: answers.gated_scan(s, s, None, torch.zeros(2, dtype=torch.int64, device="cuda")), lambda: answers.gated_scan(s, s.clone().requires_grad_()),
        lambda: answers.gated_scan_backward(s, s, states[:, :, :7]), lambda: answers.gated_scan_backward(s, s, states, s[:, :4]),
        lambda: answers.gated_step(x.half(), x, x), lambda: answers.gated_step(x[:2], x, x), lambda: answers.gated_step(x.t().contiguous().t(), x, x),
        lambda: answers.gated_step(x, x, x, labels), lambda: answers.gated_step(x[:, :7], x, x), lambda: answers.gated_step(x[:1].expand(4, 8), x, x),
        lambda: answers.gated_step(x, x.clone(), x.clone(), out=x.half()), lambda: answers.gated_step(x, x.clone(), x.clone(), out=x[:1].expand(4, 8)),
    ]
    for call in bad:
        with pytest.raises(abi.VisualMeshError):
            call()
    with torch.no_grad():
        answers.scores(x.clone().requires_grad_())


def everything(answers, x, labels, s, g, long, table, index, few):
    """Every operator, in launches of every kind: rows of lanes, blocks and clusters, sequences whole, in clusters and in parts, both kinds of steps."""
    out = []
    for rows, n in ((x, 300), (x[:, :77], 300), (x[:3], 3)):
        got = answers.scores(rows, labels[:n], 3)
        out += list(got) + [answers.scores_backward(rows, got, labels[:n], got.log_prob, got.entropy)]
    for a, b in ((s, g), (long, long)):
        scan = answers.gated_scan(a, b, keep=True)
        out += list(scan) + list(answers.gated_scan_backward(a, b, scan.states, scan.y, scan.last))
    rows = s.view(-1, 8)[:1800]
    out += [answers.gated_step(table, rows, rows, index), answers.gated_step(table, rows[:40], rows[:40], few), table]
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graphs_streams_and_devices(answers, dtype):
    """A captured run replayed on new inputs, two graphs at once, and calls on a stream of their own give what a plain call gives."""
    def inputs(seed):
        x, labels, _ = answers_of(300, 16411, dtype, seed)
        labels = labels % 77
        s, g, _, _, _ = sequences(2, 3000, 24, dtype, seed)
        long = sequences(1, 9100, 16, dtype, seed)[0]
        table = torch.ones((2000, 8), device="cuda")
        index = torch.randint(-1, 2000, (1800,), device="cuda", generator=generator(seed)).int()
        return [x, labels, s, g, long, table, index, index[:40].clone()]

    plain = {seed: [v.clone() for v in everything(answers, *inputs(seed))] for seed in (1, 2)}
    graphs = []
    for _ in range(2):
        held, graph = inputs(9), torch.cuda.CUDAGraph()
        everything(answers, *held)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = everything(answers, *held)
        graphs.append((held, graph, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for round in range(3):
        for k, (held, graph, out) in enumerate(graphs):
            for a, b in zip(held, inputs(1 + (k + round) % 2)):
                a.copy_(b)
        torch.cuda.synchronize()
        for stream, (_, graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for k, (_, _, out) in enumerate(graphs):
            for a, b in zip(out, plain[1 + (k + round) % 2]):
                assert torch.equal(a, b)
    held = [inputs(1), inputs(2)]
    torch.cuda.synchronize()
    outs = []
    for stream, h in zip(streams, held):
        with torch.cuda.stream(stream):
            outs.append(everything(answers, *h))
    torch.cuda.synchronize()
    for seed in (1, 2):
        for a, b in zip(outs[seed - 1], plain[seed]):
            assert torch.equal(a, b)
    assert torch.cuda.current_device() == 0


# ---- together, on what the engine answers --------------------------------------------------------------------------------------

def test_a_stream_of_frames_is_filtered_scored_and_learned_from(answers):
    import golden_io as G
    from visualmesh_b200.engine import Engine, FrameInput, Mesh, VisualMeshError
    from visualmesh_b200 import workloads as W

    case = G.Case("ring6_equisolid_rgba")
    mesh = Mesh.from_arrays(case.rays, case.nbrs, case.bsp)
    engine = Engine(case.network, device=0)
    fr = case.frames[0]
    images = [W.random_bytes(31 + f, fr["image"].size).reshape(fr["image"].shape) for f in range(5)]
    frames = [FrameInput(mesh, fr["Hoc"], case.lens, image, case.format) for image in images]
    host = [engine.run_batch(frames).frame(f) for f in range(5)]
    classes = engine.n_classes
    result = engine.run_batch(frames, results_on_device=True)
    held = result.tensors()
    x = held["classifications"]
    n = host[0].global_indices.shape[0]
    assert x.shape == (5 * (n + 1), classes)
    for f in range(5):
        assert bool((x[f * (n + 1):(f + 1) * (n + 1)].cpu() == torch.from_numpy(host[f].classifications)).all())
        assert bool((held["global_indices"][f * n:(f + 1) * n].cpu() == torch.from_numpy(host[f].global_indices)).all())
        assert bool((held["pixel_coordinates"][f * n:(f + 1) * n].cpu() == torch.from_numpy(host[f].pixel_coordinates)).all())
        assert bool((held["neighbourhood"][f * (n + 1):(f + 1) * (n + 1)].cpu() == torch.from_numpy(host[f].neighbourhood)).all())

    # how sure the network is of every node
    labels = torch.randint(-1, classes, (x.shape[0],), device="cuda", generator=generator(5))
    got = result.scores(labels, top=classes)
    v, log_p, p, log_prob, entropy, log_sum, top_log_prob, order = reference_scores(x, labels, classes, True)
    size = float(v.abs().amax())
    near(got.log_prob, log_prob, sum_error(classes) + 8 * U * (1 + size))
    near(got.entropy, entropy, sum_error(classes) * (3 + 2 * math.log(classes)) + 12 * U)
    assert torch.equal(got.top_index.long(), order)

    # filtered over time, by node and as sequences: a gate for every class
    gate = torch.randn(classes, device="cuda", generator=generator(6))
    prior = torch.full((mesh.n_nodes, classes), 1.0 / classes, device="cuda")
    state = prior.clone()
    y = result.advance(state, gate).view(5, n + 1, classes)
    scan = result.filtered(gate, torch.full((n + 1, classes), 1.0 / classes, device="cuda"), keep=True)
    assert scan.y.shape == (1, 5, (n + 1) * classes)
    near(y[:, :n], scan.y.view(5, n + 1, classes)[:, :n].double(), 1e-6)
    assert bool((y[:, n] == 0).all())
    nodes = torch.from_numpy(host[0].global_indices).cuda().long()
    near(state[nodes], scan.last.view(n + 1, classes)[:n].double(), 1e-6)
    off = torch.ones(mesh.n_nodes, dtype=torch.bool, device="cuda")
    off[nodes] = False
    assert torch.equal(state[off], prior[off])

    # the gradient of the mean log probability of the labels, through the filter to its gates, against differences in 64 bits
    def loss(gate):
        y = reference_scan(x.view(1, 5, -1), gate.expand(5, n + 1, classes).reshape(1, 5, -1),
                           torch.full((1, (n + 1) * classes), 1.0 / classes, device="cuda"), None)[0][0].view(-1, classes)
        return float(reference_scores(y, labels, 0, True)[3].mean())

    filtered = scan.y.view(-1, classes)
    scored = answers.scores(filtered, labels, probabilities=True)
    d = torch.full((x.shape[0],), 1.0 / x.shape[0], device="cuda")
    dy = answers.scores_backward(filtered, scored, labels, d_log_prob=d, probabilities=True)
    wide = gate.expand(5, n + 1, classes).reshape(1, 5, -1)
    _, d_gate, _ = answers.gated_scan_backward(x.view(wide.shape), wide, scan.states, dy.view(wide.shape))
    d_gate = d_gate.view(-1, classes).double().sum(0)
    for c in range(classes):
        h = torch.zeros(classes, dtype=torch.float64, device="cuda")
        h[c] = 1e-4
        want = (loss(gate.double() + h) - loss(gate.double() - h)) / 2e-4
        assert abs(float(d_gate[c]) - want) <= 2e-5 * (1 + abs(want))

    with pytest.raises(VisualMeshError):
        engine.run_batch(frames[:1]).scores()
    projector = Engine(None, device=0)
    with pytest.raises(VisualMeshError):
        projector.run_batch([FrameInput(mesh, fr["Hoc"], case.lens)], results_on_device=True).scores()
    projector.close()
    if len(case.frames) > 1:
        other = [frames[0], FrameInput(mesh, case.frames[1]["Hoc"], case.lens, case.frames[1]["image"], case.format)]
        moved = engine.run_batch(other, results_on_device=True)
        if moved.offsets[1] * 2 != moved.offsets[2]:
            with pytest.raises(VisualMeshError):
                moved.filtered(gate)
    engine.close()


def test_tensors_of_a_batch_hold_on_to_its_engine(answers):
    import gc

    import golden_io as G
    from visualmesh_b200.engine import Engine, FrameInput, Mesh

    case = G.Case("ring6_equisolid_rgba")
    mesh = Mesh.from_arrays(case.rays, case.nbrs, case.bsp)
    fr = case.frames[0]

    def held():
        engine = Engine(case.network, device=0)
        frames = [FrameInput(mesh, fr["Hoc"], case.lens, fr["image"], case.format)] * 2
        want = engine.run_batch(frames).frame(1).classifications
        return want, engine.run_batch(frames, results_on_device=True).tensors()["classifications"]

    want, x = held()
    gc.collect()
    assert bool((x[want.shape[0]:].cpu() == torch.from_numpy(want)).all())
    got = answers.scores(x, probabilities=True)
    assert bool(torch.isfinite(got.entropy).all())
