"""The gated recurrence with states and values of any size: what a factor of 32 bits can hold of them, and nothing more, is lost.

Tolerances, with u = 2^-24: the half of a gate times log2 e is off by |g| u in the exponent (its product and its constant), ex2.approx by 2^-22.5
of its result, both doubled by the square; with the square's own rounding, the sum, the reciprocal (2u) and the product behind it a factor is off by
(11 + 2 |g|) u of itself as long as it is a normal number, and by 2^-149 more below. |g| counts up to 104, where the factor is 0 in 32 bits. A step's
product and sum round by 2u, and of the joining of runs of steps it has less than 3u (a tile of 64 steps and more is joined in some thirteen
products). With e_t = (20 + 2.4 |g_t|) u for a step the error E_t of h_t obeys
E_t = f_t E_(t-1) + e_t M_t with the majorant M_t = f_t M_(t-1) + u_t |x_t|, and the gradient's the same backwards. The factor of a run of steps
may be a number below the normal ones, off by 2^-149 for each of 64 products (the steps of a thread, the threads of a block, the tiles):
2^-143 of the largest state or sum of gradients in all.
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


def near(got, want, tolerance, name=""):
    """Equal where want is not finite, else within tolerance; infinite only where that reaches beyond got's largest number."""
    kind = torch.finfo(got.dtype)
    limit, got = kind.max * (1 + kind.eps / 4), got.double()
    fine = torch.isfinite(want)
    beyond = ((got == math.inf) & (want + tolerance > limit)) | ((got == -math.inf) & (want - tolerance < -limit))
    assert bool((fine | (got == want) | (torch.isnan(got) & torch.isnan(want))).all()), f"{name}: values that are not finite differ"
    off = torch.where(fine & ~beyond, (got - want).abs() - tolerance, torch.zeros_like(want))
    assert bool((off <= 0).all()), f"{name}: off by {float((got - want).abs()[fine & ~beyond].max()):.3g}, {float(off.max()):.3g} more than allowed"


def rounding(v, dtype):
    return v.abs() * 0 if dtype == torch.float32 else v.abs().clamp(min=torch.finfo(dtype).tiny) * (torch.finfo(dtype).eps / 2)


def times(a, b):
    return torch.where(a == 0, torch.zeros_like(b), a * b)


def factors(g):
    """In 64 bits, and 0 where 32 bits have nothing: below half of 2^-149."""
    f, u = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    return (torch.where(v < 2.0**-150, torch.zeros_like(v), v) for v in (f, u))


def reference(x, g, h0, dy=None, d_last=None):
    """(value, what it may be off by but for its rounding) of y, last, states, dx, d_gate, d_h0, step by step."""
    x, g, h = x.double(), g.double(), h0.double()
    batch, steps, channels = x.shape
    f, u = factors(g)
    e = 2 * (10 + 1.2 * g.abs().clamp(max=104)) * U
    m, err = h.abs(), torch.zeros_like(h)
    largest = torch.maximum(m, torch.where(u == 0, 0.0, x.abs()).amax(1)).nan_to_num(0, 0, 0) * 2.0**-143
    ys, errs, before, before_m, before_e = [], [], [], [], []
    for t in range(steps):
        before.append(h), before_m.append(m), before_e.append(err)
        h = times(f[:, t], h) + times(u[:, t], x[:, t])
        m = times(f[:, t], m) + times(u[:, t], x[:, t].abs())
        err = times(f[:, t], err) + e[:, t] * m + largest
        ys.append(h), errs.append(err)
    stack = lambda v: torch.stack(v, 1)
    before, before_m, before_e = stack(before), stack(before_m), stack(before_e)
    keep = abi.VM_GATED_KEEP
    out = [(stack(ys), stack(errs)), (h, err), (before[:, ::keep], before_e[:, ::keep])]
    if dy is None:
        return out
    dy, c = dy.double(), d_last.double()
    c_m, c_e = c.abs(), torch.zeros_like(c)
    most = (dy.abs().amax(1) * steps + c_m) * 2.0**-143
    dx, dg, dx_e, dg_e = (torch.zeros_like(x) for _ in range(4))
    for t in reversed(range(steps)):
        total, total_m = dy[:, t] + c, dy[:, t].abs() + c_m
        total_e = c_e + e[:, t] * total_m
        fu, reach = f[:, t] * u[:, t], before_m[:, t] + x[:, t].abs()
        dx[:, t], dx_e[:, t] = times(u[:, t], total), times(u[:, t], total_e + e[:, t] * total_m) + most
        dg[:, t] = times(fu, (before[:, t] - x[:, t]) * total)
        dg_e[:, t] = times(fu, (before_e[:, t] + e[:, t] * reach) * total_m + reach * (total_e + 2 * e[:, t] * total_m)) + reach * 2.0**-148 * total_m
        c, c_m = times(f[:, t], total), times(f[:, t], total_m)
        c_e = times(f[:, t], total_e) + e[:, t] * c_m + most
    return out + [(dx, dx_e), (dg, dg_e), (c, c_e)]


def check(answers, x, g, h0, dy=None, d_last=None):
    got = answers.gated_scan(x, g, h0, keep=True)
    # many steps of few values are faster on the host
    want = reference(*(None if v is None else v.cpu() if x[:, 0].numel() < 1000 else v for v in (x, g, h0, dy, d_last)))
    want = [(right.cuda(), error.cuda()) for right, error in want]
    have = [got.y, got.last, got.states]
    if dy is not None:
        have += list(answers.gated_scan_backward(x, g, got.states, dy, d_last))
    for name, value, (right, error) in zip(("y", "last", "states", "dx", "d_gate", "d_h0"), have, want):
        near(value, right, error.nan_to_num(0, 0, 0) + rounding(right, value.dtype) + 1e-37, name)
    return have


def sequences(batch, steps, channels, dtype, seed):
    q = generator(seed)
    shape = (batch, steps, channels)
    x, dy = (torch.randn(shape, device="cuda", generator=q).to(dtype) for _ in range(2))
    g = (torch.randn(shape, device="cuda", generator=q) * 1.5 + 2).to(dtype)
    h0, d_last = (torch.randn((batch, channels), device="cuda", generator=q) for _ in range(2))
    return x, g, h0, dy, d_last


# in tiles of pieces and of single elements, in clusters, in parts, and a thread each
SIZES = [(1, 50, 8), (1, 200, 3), (3, 300, 40), (1, 1300, 24), (2, 2000, 130), (1, 9000, 6), (1, 60, 80001), (1, 50, 20002), (1, 300, 76000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,steps,channels", SIZES)
def test_gates_that_drop_what_is_not_finite(answers, batch, steps, channels, dtype):
    """-inf drops the past, +inf the present, whatever is there, and everything beside it keeps its digits."""
    x, g, h0, dy, d_last = sequences(batch, steps, channels, dtype, steps)
    half = steps // 2
    g[:, 3] = g[:, steps - 1] = math.inf
    g[:, half] = -math.inf
    x[:, 3, 0], x[:, 3, 1], x[:, 3, 2] = math.nan, math.inf, -math.inf
    h0[:, 0], h0[:, 1] = math.inf, math.nan
    g[:, 0, 0] = g[:, 0, 1] = -math.inf
    check(answers, x, g, h0, dy, d_last)
    x[:, half - 1, 2] = math.inf  # until the reset
    check(answers, x, g, h0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,steps,channels", SIZES)
def test_large_states_are_forgotten(answers, batch, steps, channels, dtype):
    """A state near the top of the range leaves nothing behind once its factor has fallen below what 32 bits hold of it."""
    x, g, h0, dy, d_last = sequences(batch, steps, channels, dtype, steps + 1)
    h0 *= 1e37
    h0[:, 0] = 3e38
    d_last *= 1e36
    g[:, 5:45:2] = -20.0
    g[:, steps - 12:steps - 2] = -25.0
    if dtype != torch.float16:
        x[:, steps // 2, 1] = 1e38
    check(answers, x, g, h0, dy * 0.5, d_last)
    # nothing to see, and gates that close slowly: what is left of the first state, alone
    g = torch.full_like(g, -6.0)
    x[:] = 0
    check(answers, x, g, h0, dy, d_last)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,steps,channels", SIZES)
def test_factors_below_the_normal_numbers(answers, batch, steps, channels, dtype):
    """A gate between -104 and 104 drops nothing: its factors are numbers of 32 bits, and an infinity goes on."""
    x, g, h0, dy, d_last = sequences(batch, steps, channels, dtype, steps + 2)
    gates = torch.tensor([-86.0, -88.0, -90.0, -95.0, -100.0, -103.0], device="cuda")
    at = torch.arange(4, min(steps - 2, 40), 5, device="cuda")
    g[:, at] = gates[at % 6][None, :, None].to(dtype).expand(batch, -1, channels)
    g[:, at + 1] = -gates[at % 6][None, :, None].to(dtype).expand(batch, -1, channels)
    if dtype != torch.float16:
        x[:, at + 1, 1] = 3e38  # masked by a gate that lets a little of it through
        x[:, at - 1, 2] = 1e38
    h0[:, 0] = math.inf
    x[:, 2, 1] = -math.inf
    check(answers, x, g, h0)
    h0[:, 0], x[:, 2, 1] = 3e38, 0.5
    check(answers, x, g, h0, dy, d_last)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(5, 7), (40, 64), (700, 3)])
def test_steps_with_factors_below_the_normal_numbers(answers, rows, channels, dtype):
    q = generator(rows)
    state = torch.randn((rows, channels), device="cuda", generator=q) * 1e38
    x = torch.randn((rows, channels), device="cuda", generator=q).to(dtype)
    g = torch.linspace(-103.5, 103.5, rows * channels, device="cuda").view(rows, channels).to(dtype)
    state[0, 0] = math.inf
    for index in (None, torch.randperm(rows, device="cuda", generator=q).int()):
        table = state.clone()
        rows_of = torch.arange(rows, device="cuda") if index is None else index.long()
        f, u = factors(g.double())
        want = times(f, state.double()[rows_of]) + times(u, x.double())
        error = 2 * (10 + 1.2 * g.double().abs()) * U * (times(f, state.double()[rows_of].abs()) + times(u, x.double().abs())) + 2.0**-148 * state.double()[rows_of].abs()
        y = answers.gated_step(table, x, g, index)
        near(y, want, error.nan_to_num(0, 0, 0) + rounding(want, dtype) + 1e-37)
        near(table[rows_of], want, error.nan_to_num(0, 0, 0) + 1e-37)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,steps,channels", SIZES)
def test_lowest_values_that_are_masked_beside_large_states(answers, batch, steps, channels, dtype):
    """What a gate of infinity drops has no part in a gradient, though its difference to the state is beyond the range."""
    x, g, h0, dy, d_last = sequences(batch, steps, channels, dtype, steps + 3)
    h0 = h0.abs() * 1e37 + 1e37
    at = torch.arange(2, 12, 3, device="cuda")
    g[:, at] = math.inf
    x[:, at] = torch.finfo(dtype).min
    g[:, 12] = -math.inf
    check(answers, x, g, h0, dy * 0.5, d_last)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,steps,channels", SIZES)
def test_values_at_both_ends_of_the_range(answers, batch, steps, channels, dtype):
    """States and values whose difference is beyond the range, inside a thread's steps too: what a factor of 0 drops is dropped, and a small one comes first."""
    x, g, h0, dy, d_last = sequences(batch, steps, channels, dtype, steps + 4)
    lowest = torch.finfo(dtype).min
    for at in (2, 9, 19, 27):
        x[:, at], g[:, at] = 3e37, 1.0                  # large for a while,
        x[:, at + 1], g[:, at + 1] = lowest, math.inf   # beside what is masked,
        x[:, at + 2], g[:, at + 2] = lowest, -math.inf  # until a new beginning with the lowest value,
        x[:, at + 3], g[:, at + 3] = 2e37, -20.0        # which is forgotten at once
        g[:, at + 4] = -math.inf
    check(answers, x, g, h0, dy * 0.1, d_last)
