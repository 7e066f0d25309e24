"""Plain implementations of the experts' operators in 64 bits (CPU), by their definitions."""
import math

import torch


def route(logits, top_k, scoring="softmax", bias=None, groups=1, top_groups=None, group_score="max", renormalize=True, scale=1.0):
    """(weights float64 [T, k], experts int32 [T, k]); what cannot be chosen is -1 with weight 0."""
    T, E = logits.shape
    top_groups = groups if top_groups is None else top_groups
    weights = torch.zeros(T, top_k, dtype=torch.float64)
    experts = torch.full((T, top_k), -1, dtype=torch.int32)
    b = None if bias is None else bias.double().tolist()
    for t, row in enumerate(logits.double().tolist()):
        row = [v if v > -math.inf else -math.inf for v in row]  # NaN masks
        live = [e for e in range(E) if row[e] > -math.inf and (b is None or b[e] > -math.inf)]
        if scoring == "softmax":
            top = max(row)
            total = math.fsum(math.exp(v - top) for v in row if v > -math.inf)
            score = {e: math.exp(row[e] - top) / total for e in live}
        else:
            score = {e: 1.0 / (1.0 + math.exp(-row[e])) if row[e] > -700 else math.exp(row[e]) for e in live}
        choice = {e: row[e] if b is None else score[e] + b[e] for e in live}
        if groups > 1 and top_groups < groups:
            size = E // groups
            values = {}
            for e in live:
                values.setdefault(e // size, []).append(choice[e] if group_score == "max" or b is not None else score[e])
            n = 1 if group_score == "max" else 2
            value = {g: sum(sorted(v)[-n:]) for g, v in values.items()}
            kept = sorted(value, key=lambda g: (-value[g], g))[:top_groups]
            live = [e for e in live if e // size in kept]
        ids = sorted(live, key=lambda e: (-choice[e], e))[:top_k]
        w = [score[e] for e in ids]
        total = math.fsum(w) if renormalize else 1.0
        for j, e in enumerate(ids):
            experts[t, j] = e
            weights[t, j] = w[j] / total * scale
    return weights, experts


def group(experts, num_experts, first=0):
    flat = experts.reshape(-1).tolist()
    offsets, slots, places = [0], [], [-1] * len(flat)
    for e in range(first, first + num_experts):
        for i, v in enumerate(flat):
            if v == e:
                places[i] = len(slots)
                slots.append(i)
        offsets.append(len(slots))
    slots += [-1] * (len(flat) - len(slots))
    return (torch.tensor(offsets, dtype=torch.int32), torch.tensor(slots, dtype=torch.int32),
            torch.tensor(places, dtype=torch.int32).reshape(experts.shape))


def row_experts(offsets, rows):
    """Expert of every row, -1 behind the last."""
    out = torch.full((rows,), -1, dtype=torch.long)
    for e, (a, b) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
        out[a:b] = e
    return out


def product(x_q, w_q, x_scale, w_scale, offsets, slots=None, top_k=1):
    """(exact float64 [rows, N], the same with the kernel's three fp32 roundings)."""
    rows = x_q.shape[0] if slots is None else slots.numel()
    src = torch.arange(rows) if slots is None else slots.long().clamp_min(0) // top_k
    exact = torch.zeros(rows, w_q.shape[1], dtype=torch.float64)
    single = torch.zeros(rows, w_q.shape[1], dtype=torch.float32)
    of_row = row_experts(offsets, rows)
    for e in range(w_q.shape[0]):
        r = (of_row == e).nonzero()[:, 0]
        if r.numel():
            acc = x_q[src[r]].double() @ w_q[e].double().t()  # integers below 2^53
            exact[r] = acc * (x_scale[src[r]].double()[:, None] * w_scale[e].double()[None, :])
            single[r] = acc.float() * (x_scale[src[r]][:, None] * w_scale[e][None, :])
    return exact, single


def swiglu(v):
    """(gate, silu(gate) * up) of [rows, 2 N] in float64."""
    g, u = v.double().chunk(2, dim=1)
    return g, g * torch.sigmoid(g) * u


def combine(y, weights, places, add=None):
    """(exact, sum of the terms' magnitudes)."""
    out = torch.zeros(places.shape[0], y.shape[1], dtype=torch.float64) if add is None else add.double()
    size = out.abs()
    for j in range(places.shape[1]):
        p = places[:, j].long()
        term = torch.where((p >= 0)[:, None], weights[:, j, None].double() * y.double()[p.clamp_min(0)], torch.zeros(1, dtype=torch.float64))
        out, size = out + term, size + term.abs()
    return out, size
