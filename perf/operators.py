"""The operators on what a network answers, as cases that can be timed and compared: scores of answers (log probability of a label,
entropy, alternatives) with their gradient, and a gated recurrence over a sequence of answers with its gradient and its single step.

  "scores"        what is known of every row: log probability of its label, entropy, log of the sum, the `top` best classes
  "train_scores"  a step of training on labelled rows: log probability and entropy, then the gradient of the rows
  "scan"          h_t = f_t h_(t-1) + (1 - f_t) x_t with f = sigmoid(gate) over whole sequences
  "train_scan"    the same, then the gradients of x, of the gate and of the first state
  "step"          one step of it for rows that name their states in a table, which is updated in place
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _scores(name, op, rows, classes, type, top=0, probabilities=False, masked=False):
    return {"name": name, "op": op, "rows": rows, "classes": classes, "type": type, "top": top, "probabilities": probabilities, "masked": masked}


def _scan(name, op, batch, steps, channels, type, ragged=False):
    return {"name": name, "op": op, "batch": batch, "steps": steps, "channels": channels, "type": type, "ragged": ragged}


def _step(name, slots, rows, channels, type):
    return {"name": name, "op": "step", "slots": slots, "rows": rows, "channels": channels, "type": type}


def listed():
    return [
        # one frame's classified nodes (68,100 and the off-screen row, two classes) against its labels: the smallest call of a vision loop
        _scores("scores_frame", "scores", 68101, 2, "f32", 1, True),
        # a batch of 64 such frames of a three-class network, with the runner-up of every node
        _scores("scores_batch", "scores", 64 * 70001, 3, "f32", 2, True),
        # evaluation over a large vocabulary: 16-bit logits, some classes masked, the five best of each row
        _scores("scores_wide", "scores", 4099, 32771, "bf16", 5, False, True),
        # the answer of a few rows at a time (decoding): little to read, so latency and the split of a row count
        _scores("scores_few", "scores", 4, 131072, "f16", 20),
        # a training step on sixteen labelled frames of a five-class network, from the logits
        _scores("train_frames", "train_scores", 16 * 68101, 5, "f32"),
        # a training step over a large vocabulary
        _scores("train_wide", "train_scores", 2048, 50021, "bf16"),
        # the answers of a camera that stands still, 64 frames of 68,101 rows with three classes, filtered over time
        _scan("scan_frames", "scan", 1, 64, 68101 * 3, "f32"),
        # few channels over a very long sequence: work has to be split over time
        _scan("scan_long", "scan", 1, 65537, 64, "bf16"),
        # a training step over sequences of a wide layer: the largest
        _scan("train_sequences", "train_scan", 4, 4096, 2048, "bf16"),
        # padded sequences of odd sizes in 32 bits
        _scan("train_ragged", "train_scan", 3, 1021, 515, "f32", True),
        # serving: one new element for each of 64 sequences, whose states are anywhere in a table
        _step("step_rows", 512, 64, 2048, "bf16"),
        # the nodes that one frame shows, of a mesh of 121,083, three classes each
        _step("step_nodes", 121083, 68100, 3, "f32"),
    ]


def draw(rng):
    log = lambda lo, hi: int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))
    op = rng.choice(["scores", "scores", "train_scores", "scan", "scan", "train_scan", "step"])
    type = rng.choice(["f32", "f16", "bf16"])
    if op in ("scores", "train_scores"):
        most = 134_000_000 if op == "scores" else 100_000_000
        probabilities = rng.random() < 0.4
        if probabilities:
            classes, type = log(2, 64), "f32"
        else:
            classes = log(2, 131072)
        rows = log(1, max(1, min(4_000_000, most // classes)))
        top = min(classes, rng.choice([0, 1, 2, 3, 5, 8, 20])) if op == "scores" else 0
        case = _scores("", op, rows, classes, type, top, probabilities, not probabilities and classes > 8 and rng.random() < 0.4)
    elif op == "step":
        rows, channels = log(1, 60000), log(1, 4096)
        rows = max(1, min(rows, 30_000_000 // channels))
        case = _step("", rows + log(1, 2 * rows), rows, channels, type)
    else:
        batch, steps, channels = log(1, 8), log(1, 65536), log(1, 4096)
        steps = max(1, min(steps, 33_000_000 // (batch * channels)))
        case = _scan("", op, batch, steps, channels, type, rng.random() < 0.4)
    del case["name"]
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _random(shape, generator):
    return torch.randn(shape, device="cuda", generator=generator)


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]
    state = {"case": case}
    if case["op"] in ("scores", "train_scores"):
        rows, classes = case["rows"], case["classes"]
        labels = torch.randint(0, classes, (rows,), device="cuda", generator=generator)
        x = _random((rows, classes), generator).mul_(2.0)
        # a trained network is mostly right: its answer leans to the label
        x.scatter_add_(1, labels[:, None], torch.rand((rows, 1), device="cuda", generator=generator) * (2.0 + math.log(classes)))
        if case["masked"]:
            masked = torch.rand((1, classes), device="cuda", generator=generator) < 0.1
            masked = masked.expand(rows, classes).scatter(1, labels[:, None], False)
            x = x.masked_fill_(masked, -math.inf)
        if case["probabilities"]:
            x = torch.softmax(x, 1)
        state["x"] = x.to(kind)
        # rows without a label (off-screen rows, padding) are marked -1
        state["labels"] = torch.where(torch.rand(rows, device="cuda", generator=generator) < 0.05, -1, labels)
        if case["op"] == "train_scores":
            # gradients of a mean of weighted rows, and of an entropy that is kept up
            state["d_log_prob"] = -(0.5 + torch.rand(rows, device="cuda", generator=generator))
            state["d_entropy"] = -0.1 * torch.rand(rows, device="cuda", generator=generator)
        return state
    if case["op"] == "step":
        rows, slots, channels = case["rows"], case["slots"], case["channels"]
        state["table"] = _random((slots, channels), generator)
        state["x"] = _random((rows, channels), generator).to(kind)
        state["gate"] = (_random((rows, channels), generator) + 1.0).to(kind)
        index = torch.randperm(slots, device="cuda", generator=generator)[:rows].to(torch.int32)
        # a padded batch: rows that belong to no sequence
        state["index"] = torch.where(torch.rand(rows, device="cuda", generator=generator) < 0.03, -1, index)
        return state
    shape = (case["batch"], case["steps"], case["channels"])
    state["x"] = _random(shape, generator).to(kind)
    gate = _random(shape, generator).mul_(1.5).add_(2.0)
    chance = torch.rand(shape[:2], device="cuda", generator=generator)[:, :, None]
    # now and then a sequence begins anew, and now and then there is nothing to see
    gate = gate.masked_fill_(chance < 0.002, -math.inf).masked_fill_(chance > 0.99, math.inf)
    state["gate"] = gate.to(kind)
    state["h0"] = _random((shape[0], shape[2]), generator)
    state["lengths"] = None
    if case["ragged"]:
        state["lengths"] = torch.randint(0, shape[1] + 1, (shape[0],), device="cuda", generator=generator).to(torch.int32)
    if case["op"] == "train_scan":
        state["dy"] = _random(shape, generator).to(kind)
        state["d_last"] = _random((shape[0], shape[2]), generator)
    return state


# ---- plain forms ---------------------------------------------------------------------------------------------------------

def _distribution(x, probabilities):
    """log p and p of every class, the log of the sum"""
    v = x.float()
    if probabilities:
        v = torch.log(v)
    m = v.amax(1, keepdim=True)
    e = torch.exp(v - m)
    total = e.sum(1, keepdim=True)
    log_sum = m + torch.log(total)
    return v - log_sum, e / total, log_sum[:, 0]


def _of_labels(log_p, labels):
    picked = log_p.gather(1, labels.clamp(min=0)[:, None])[:, 0]
    return torch.where(labels < 0, torch.zeros_like(picked), picked)


def _entropy(log_p, p):
    return -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(1)


def _best(x, top):
    """Indices of the largest, ties to the lowest index: keys of the values' order above the columns'."""
    bits = (x.float() + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    columns = x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device)
    return torch.topk(order * 2**32 + columns, top, dim=1).indices


def _plain_scores(state):
    case, x = state["case"], state["x"]
    log_p, p, log_sum = _distribution(x, case["probabilities"])
    out = {"log_prob": _of_labels(log_p, state["labels"]), "entropy": _entropy(log_p, p)}
    if not case["probabilities"]:  # the sum of probabilities is one but for what they were rounded by
        out["log_sum"] = log_sum
    if case["top"]:
        best = _best(x, case["top"])
        out["top_log_prob"], out["top_index"] = log_p.gather(1, best), best.to(torch.int32)
    return out


def _plain_train_scores(state):
    case, x, labels = state["case"], state["x"], state["labels"]
    log_p, p, _ = _distribution(x, case["probabilities"])
    entropy = _entropy(log_p, p)
    d_label = torch.where(labels < 0, torch.zeros_like(entropy), state["d_log_prob"])
    inner = -d_label[:, None] - state["d_entropy"][:, None] * (log_p + entropy[:, None])
    at_label = labels.clamp(min=0)[:, None]
    if case["probabilities"]:
        v = x.float()
        dx = inner / v.sum(1, keepdim=True)
        dx = dx.scatter_add(1, at_label, d_label[:, None] / v.gather(1, at_label))
    else:
        dx = torch.where(p > 0, p * inner, torch.zeros_like(p)).scatter_add(1, at_label, d_label[:, None])
    return {"log_prob": _of_labels(log_p, labels), "entropy": entropy, "dx": dx.to(x.dtype)}


def _recurrence(f, v):
    """h_t = f_t h_(t-1) + v_t along dimension 1, by doubling"""
    step = 1
    while step < f.shape[1]:
        v = torch.cat([v[:, :step], v[:, step:] + f[:, step:] * v[:, :-step]], 1)
        f = torch.cat([f[:, :step], f[:, step:] * f[:, :-step]], 1)
        step *= 2
    return v


def _factors(state):
    g = state["gate"].float()
    f, u, valid = torch.sigmoid(g), torch.sigmoid(-g), None
    if state["lengths"] is not None:
        valid = (torch.arange(g.shape[1], device=g.device)[None, :] < state["lengths"][:, None])[:, :, None]
        f, u = torch.where(valid, f, torch.ones_like(f)), torch.where(valid, u, torch.zeros_like(u))
    return f, u, valid


def _plain_scan(state):
    x = state["x"].float()
    f, u, valid = _factors(state)
    v = u * x
    v[:, 0] += f[:, 0] * state["h0"]
    h = _recurrence(f, v)
    y = h if valid is None else torch.where(valid, h, torch.zeros_like(h))
    out = {"y": y.to(state["x"].dtype), "last": h[:, -1].clone()}
    if state["case"]["op"] == "scan":
        return out
    before = torch.cat([state["h0"][:, None], h[:, :-1]], 1)
    d = state["dy"].float()
    if valid is not None:
        d = torch.where(valid, d, torch.zeros_like(d))
    d[:, -1] += state["d_last"]
    after = torch.cat([f[:, 1:], torch.ones_like(f[:, :1])], 1)
    total = _recurrence(after.flip(1), d.flip(1)).flip(1)
    out["dx"] = (u * total).to(state["x"].dtype)
    out["d_gate"] = (f * u * (before - x) * total).to(state["x"].dtype)
    out["d_h0"] = f[:, 0] * total[:, 0]
    return out


def _plain_step(state):
    index, table = state["index"], state["table"]
    g = state["gate"].float()
    there = (index >= 0)[:, None]
    at = index.clamp(min=0).to(torch.int64)
    h = torch.sigmoid(g) * table[at] + torch.sigmoid(-g) * state["x"].float()
    y = torch.where(there, h, torch.zeros_like(h))
    rows = there[:, 0].nonzero()[:, 0]
    table[at[rows]] = h[rows]
    return {"y": y.to(state["x"].dtype), "table": table}


# ---- the framework's operators -------------------------------------------------------------------------------------------

def _own(state):
    from visualmesh_b200 import answers

    case, x = state["case"], state["x"]
    if case["op"] == "scores":
        got = answers.scores(x, state["labels"], top=case["top"], probabilities=case["probabilities"])
        out = {"log_prob": got.log_prob, "entropy": got.entropy}
        if not case["probabilities"]:
            out["log_sum"] = got.log_sum
        if case["top"]:
            out["top_log_prob"], out["top_index"] = got.top_log_prob, got.top_index
        return out
    if case["op"] == "train_scores":
        got = answers.scores(x, state["labels"], probabilities=case["probabilities"])
        dx = answers.scores_backward(x, got, state["labels"], d_log_prob=state["d_log_prob"], d_entropy=state["d_entropy"],
                                     probabilities=case["probabilities"])
        return {"log_prob": got.log_prob, "entropy": got.entropy, "dx": dx}
    if case["op"] == "step":
        return {"y": answers.gated_step(state["table"], x, state["gate"], state["index"]), "table": state["table"]}
    if case["op"] == "scan":
        got = answers.gated_scan(x, state["gate"], state["h0"], state["lengths"])
        return {"y": got.y, "last": got.last}
    got = answers.gated_scan(x, state["gate"], state["h0"], state["lengths"], keep=True)
    dx, d_gate, d_h0 = answers.gated_scan_backward(x, state["gate"], got.states, state["dy"], state["d_last"], state["lengths"])
    return {"y": got.y, "last": got.last, "dx": dx, "d_gate": d_gate, "d_h0": d_h0}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"scores": _plain_scores, "train_scores": _plain_train_scores, "step": _plain_step}.get(op, _plain_scan)(state)


def work(case):
    size = _BYTES[case["type"]]
    if case["op"] in ("scores", "train_scores"):
        rows, cells = case["rows"], case["rows"] * case["classes"]
        if case["op"] == "scores":
            # the rows and labels, three results a row and its alternatives; an exponential, its sum, its product with the logarithm
            return {"bytes": cells * size + rows * (8 + 12 + 8 * case["top"]), "flops": 6 * cells}
        # a training step has to read the rows before it knows their sums, and again (they need not stay on chip) for the gradients
        return {"bytes": 2 * cells * size + rows * (8 + 12 + 8), "flops": 12 * cells}
    if case["op"] == "step":
        cells = case["rows"] * case["channels"]
        return {"bytes": cells * (3 * size + 8) + 4 * case["rows"], "flops": 8 * cells}
    cells, ends = case["batch"] * case["steps"] * case["channels"], 8 * case["batch"] * case["channels"]
    if case["op"] == "scan":
        return {"bytes": 3 * size * cells + ends, "flops": 8 * cells}
    # x, gate and dy in; y, dx and the gate's gradient out
    return {"bytes": 6 * size * cells + 2 * ends, "flops": 24 * cells}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("scores", "train_scores"):
        v = state["x"].double()
        total = v.sum(1) if case["probabilities"] else None
        if case["probabilities"]:
            v = v.log()
        log_sum = torch.logsumexp(v, 1)
        log_p = v - log_sum[:, None]
        p = log_p.exp()
        seen = p > 0
        entropy = -(p * log_p.masked_fill(~seen, 0.0)).sum(1)
        labels = state["labels"]
        marked = labels >= 0
        row = torch.arange(case["rows"], device="cuda")[marked]
        log_prob = torch.zeros_like(entropy)
        log_prob[marked] = log_p[row, labels[marked]]
        out = {"log_prob": log_prob, "entropy": entropy}
        if case["op"] == "scores":
            if not case["probabilities"]:
                out["log_sum"] = log_sum
            if case["top"]:
                out["top_log_prob"], out["top_index"] = torch.topk(log_p, case["top"], 1).values, None
            return out
        d_label = state["d_log_prob"].double() * marked
        # d log p[label] / d v_j = [j = label] - p_j;  d H / d v_j = -p_j (log p_j + H)
        dv = -p * (d_label[:, None] + state["d_entropy"].double()[:, None] * (log_p.masked_fill(~seen, 0.0) + entropy[:, None]))
        dv[row, labels[marked]] += d_label[marked]
        out["dx"] = dv / state["x"].double() if total is not None else dv
        return out
    if case["op"] == "step":
        index = state["index"].to(torch.int64)
        f = 1.0 / (1.0 + torch.exp(-state["gate"].double()))
        table = state["table"].double()
        y = torch.zeros_like(f)
        rows = torch.nonzero(index >= 0).flatten()
        h = f[rows] * table[index[rows]] + (1.0 - f[rows]) * state["x"].double()[rows]
        y[rows], table[index[rows]] = h, h
        return {"y": y, "table": table}
    x, g, h = state["x"].double(), state["gate"].double(), state["h0"].double()
    f = 1.0 / (1.0 + torch.exp(-g))
    u = 1.0 / (1.0 + torch.exp(g))
    if state["lengths"] is not None:
        beyond = torch.arange(case["steps"], device="cuda")[None, :] >= state["lengths"][:, None]
        f[beyond], u[beyond] = 1.0, 0.0
    h_all = torch.empty_like(x)
    for t in range(case["steps"]):
        h = f[:, t] * h + u[:, t] * x[:, t]
        h_all[:, t] = h
    y = h_all.clone()
    if state["lengths"] is not None:
        y[beyond] = 0.0
    out = {"y": y, "last": h}
    if case["op"] == "scan":
        return out
    dy, carry = state["dy"].double(), state["d_last"].double()
    if state["lengths"] is not None:
        dy[beyond] = 0.0
    dx, d_gate = torch.empty_like(x), torch.empty_like(x)
    for t in reversed(range(case["steps"])):
        total = dy[:, t] + carry
        before = h_all[:, t - 1] if t else state["h0"].double()
        dx[:, t] = u[:, t] * total
        d_gate[:, t] = f[:, t] * u[:, t] * (before - x[:, t]) * total
        carry = f[:, t] * total
    out["dx"], out["d_gate"], out["d_h0"] = dx, d_gate, carry
    return out
