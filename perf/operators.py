"""The operators of a mixture-of-experts layer with int8 weights, as a list of measurable cases.

A token's hidden vector is sent to `top_k` of the experts and comes back as the weighted sum of what they make of it.  The layer is five
operators in a row, and inference only, as everything in this package:

    route     logits [T, E] -> weights [T, k], experts [T, k]        which experts a token takes, and with which weight
    group     experts [T, k] -> offsets [E + 1], slots [T k], places [T, k]   the (token, choice) pairs in the order of their experts
    product   int8 rows times the int8 weight of each row's expert, scales per token and per output channel, bf16 out
    swiglu    the same with a gate half and an up half of the weight: silu(gate) * up, bf16 out
    combine   the weighted sum of a token's k rows, bf16 out
    layer     all of them with the per-token quantiser in front of either product: `Int8Experts`

Fields of a case (those that its kind has):
    kind                 one of the above
    T, E, k              tokens, experts of the router, experts per token
    ranks                the experts are split over this many ranks, of which this is the last; what the others hold is dropped here
    N, K                 product, swiglu: output channels (of the result) and input channels; combine: N; layer: hidden K, inner N
    gather               product, swiglu: rows are read where their tokens lie; else they lie in the order of the experts already
    logits               route: "bf16" | "fp32"
    scoring, bias, groups, top_groups, group_score, renormalize, scale    of the router
    add                  combine, layer: a tensor (the residual stream, a shared expert's result) is added to the sum
"""
from __future__ import annotations

import math
import statistics

import torch

own = False

_FLOP_LIMIT = 6 * 2048 * 2 * 14336 * 4096  # of the largest listed case
_BYTE_LIMIT = 1_450_000_000                # its bytes; weights and results stay below as well

_ROUTER = {"logits": "fp32", "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_score": "max",
           "renormalize": True, "scale": 1.0}


def listed():
    return [
        # The router of a decode batch: sixteen tokens, biased sigmoid scores, four of eight groups.  Launch latency.
        {"name": "route_decode16", "kind": "route", "T": 16, "E": 256, "k": 8, **_ROUTER, "logits": "bf16", "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_score": "top2", "scale": 2.5},
        # The same router over a whole batch of prompts.
        {"name": "route_prompts", "kind": "route", "T": 16384, "E": 256, "k": 8, **_ROUTER, "scoring": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_score": "top2", "scale": 2.5},
        # Grouping of an odd decode batch over an odd number of experts.
        {"name": "group_decode", "kind": "group", "T": 61, "E": 60, "k": 4, "ranks": 1},
        # Grouping of a batch of prompts on one of two ranks: half of the pairs are dropped.
        {"name": "group_prompts", "kind": "group", "T": 16384, "E": 256, "k": 8, "ranks": 2},
        # The second product of a prefill: rows already in the order of the experts.
        {"name": "product_prompts", "kind": "product", "T": 4096, "E": 64, "k": 8, "ranks": 1, "N": 4096, "K": 2048, "gather": False},
        # A short prompt, no size a whole number of tiles, output rows of odd length, on one of two ranks.
        {"name": "product_ragged", "kind": "product", "T": 777, "E": 20, "k": 3, "ranks": 2, "N": 2501, "K": 2832, "gather": True},
        # One token: eight of 128 experts' gate and up weights are read.
        {"name": "swiglu_decode1", "kind": "swiglu", "T": 1, "E": 128, "k": 8, "ranks": 1, "N": 2048, "K": 4096, "gather": True},
        # The first product of a prefill, rows gathered from their tokens.
        {"name": "swiglu_prompts", "kind": "swiglu", "T": 4096, "E": 64, "k": 8, "ranks": 1, "N": 2048, "K": 4096, "gather": True},
        # The sum behind a decode batch, onto the residual stream.
        {"name": "combine_decode", "kind": "combine", "T": 32, "E": 64, "k": 6, "ranks": 1, "N": 4096, "add": True},
        # The sum behind a batch of prompts of odd length.
        {"name": "combine_prompts", "kind": "combine", "T": 8191, "E": 128, "k": 8, "ranks": 1, "N": 4096, "add": False},
        # A decode batch through the whole layer: most experts are met by a token or two.
        {"name": "layer_decode16", "kind": "layer", "T": 16, "E": 64, "k": 8, "ranks": 1, "N": 1408, "K": 4096, "add": True, **_ROUTER, "logits": "bf16"},
        # Prompts through the whole layer, few large experts.
        {"name": "layer_prompts", "kind": "layer", "T": 2048, "E": 8, "k": 2, "ranks": 1, "N": 14336, "K": 4096, "add": True, **_ROUTER, "logits": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_router(rng, E, k):
    r = dict(_ROUTER, logits=rng.choice(["bf16", "fp32"]), scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
             renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), group_score=rng.choice(["max", "top2"]))
    groups = [n for n in (2, 4, 5, 8, 16) if E % n == 0 and E // n >= 2]
    if groups and rng.random() < 0.5:
        r["groups"] = rng.choice(groups)
        r["top_groups"] = rng.randint(-(-k * r["groups"] // E), r["groups"])
    return r


def draw(rng):
    while True:
        kind = rng.choice(["route", "group", "product", "swiglu", "combine", "layer"])
        E = rng.choice([8, 16, 20, 60, 64, 72, 128, 160, 256])
        c = {"kind": kind, "T": _log_int(rng, 1, 16384), "E": E, "k": rng.randint(1, min(8, E))}
        if kind == "route":
            c.update(_draw_router(rng, E, c["k"]))
            return c
        c["ranks"] = rng.choice([1, 1, 2, 4]) if E % 4 == 0 and kind != "layer" else 1
        if kind == "group":
            return c
        c["N"] = _log_int(rng, 256, 8192)
        if rng.random() < 0.7:
            c["N"] = max(128, c["N"] // 128 * 128)
        if kind == "combine":
            c["add"] = rng.random() < 0.5
        else:
            c["K"] = _log_int(rng, 256, 8192) // 16 * 16
        if kind in ("product", "swiglu"):
            c["gather"] = kind == "swiglu" or rng.random() < 0.5
        if kind == "layer":
            c["N"] = c["N"] // 16 * 16
            c.update(_draw_router(rng, E, c["k"]), add=rng.random() < 0.5)
        if "K" in c and E * c["K"] * c["N"] * {"product": 1, "swiglu": 2, "layer": 3}[kind] > _BYTE_LIMIT:
            continue
        if work(c)["flops"] <= _FLOP_LIMIT and work(c)["bytes"] <= _BYTE_LIMIT:
            return c


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------
def _popularity(E):
    """How much likelier some experts are than others, in logits: the quantiles of a Gaussian of width one half."""
    return [0.5 * statistics.NormalDist().inv_cdf((e + 0.5) / E) for e in range(E)]


def _held(case):
    """First expert of this rank, and how many it holds."""
    n = case["E"] // case["ranks"]
    return case["E"] - n, n


def _logits(case, gen):
    E = case["E"]
    pop = torch.tensor(_popularity(E), device="cuda")[torch.randperm(E, device="cuda", generator=gen)]
    return torch.randn(case["T"], E, device="cuda", generator=gen) + pop


def _experts(case, gen):
    """Distinct experts for every token: the largest of popularity plus noise."""
    u = torch.rand(case["T"], case["E"], device="cuda", generator=gen).clamp_(1e-7, 1 - 1e-7)
    pop = torch.tensor(_popularity(case["E"]), device="cuda")[torch.randperm(case["E"], device="cuda", generator=gen)]
    return (pop - torch.log(-torch.log(u))).topk(case["k"], dim=1).indices.to(torch.int32)


def _group(experts, first, held):
    """offsets, slots, places by a stable sort."""
    flat = experts.reshape(-1).long() - first
    key = torch.where((flat >= 0) & (flat < held), flat, held)
    order = torch.argsort(key, stable=True)
    offsets = torch.zeros(held + 1, dtype=torch.int32, device=flat.device)
    offsets[1:] = (key[:, None] == torch.arange(held, device=flat.device)).sum(0).cumsum(0)
    kept = torch.arange(flat.numel(), device=flat.device) < offsets[held]
    slots = torch.where(kept, order, -1).to(torch.int32)
    places = torch.empty_like(flat)
    places[order] = torch.where(kept, torch.arange(flat.numel(), device=flat.device), -1)
    return offsets, slots, places.to(torch.int32).reshape(experts.shape)


def _int8(gen, *shape):
    return torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)


def _scales(gen, *shape, top):
    return torch.rand(*shape, device="cuda", generator=gen) * top * 0.9 + top * 0.1


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, T, E, k = case["kind"], case["T"], case["E"], case["k"]
    if kind in ("route", "layer"):
        t = {"logits": _logits(case, gen).to(torch.bfloat16 if case["logits"] == "bf16" else torch.float32)}
        t["bias"] = torch.randn(E, device="cuda", generator=gen) * 0.1 if case["bias"] else None
        if kind == "route":
            return t
        K, N = case["K"], case["N"]
        t["x"] = torch.randn(T, K, device="cuda", generator=gen).to(torch.bfloat16)
        t["gate_up"], t["gate_up_scale"] = _int8(gen, E, 2 * N, K), _scales(gen, E, 2 * N, top=2.0 / (127 * math.sqrt(K)))
        t["down"], t["down_scale"] = _int8(gen, E, K, N), _scales(gen, E, K, top=2.0 / (127 * math.sqrt(N)))
        t["add"] = torch.randn(T, K, device="cuda", generator=gen).to(torch.bfloat16) if case["add"] else None
        return t
    first, held = _held(case)
    t = {"experts": _experts(case, gen)}
    if kind == "group":
        return t
    t["offsets"], slots, places = _group(t.pop("experts"), first, held)
    if kind == "combine":
        t["places"], t["y"] = places, torch.randn(T * k, case["N"], device="cuda", generator=gen).to(torch.bfloat16)
        w = torch.rand(T, k, device="cuda", generator=gen) + 0.05
        t["weights"] = w / w.sum(1, keepdim=True)
        t["add"] = torch.randn(T, case["N"], device="cuda", generator=gen).to(torch.bfloat16) if case["add"] else None
        return t
    N, K, rows = case["N"] * (2 if kind == "swiglu" else 1), case["K"], T if case["gather"] else T * k
    t["slots"] = slots if case["gather"] else None
    t["x_q"], t["x_scale"] = _int8(gen, rows, K), _scales(gen, rows, top=2.0 / 127)
    t["w_q"], t["w_scale"] = _int8(gen, held, N, K), _scales(gen, held, N, top=2.0 / (127 * math.sqrt(K)))
    return t


def _router_args(case):
    return {f: case[f] for f in ("scoring", "groups", "top_groups", "group_score", "renormalize", "scale")}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own and case["kind"] == "layer":
        import gemm_int8_b200 as g

        state["layer"] = g.Int8Experts(state["gate_up"], state["gate_up_scale"], state["down"], state["down_scale"], case["k"],
                                       bias=state["bias"], **_router_args(case))
    return state


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


def _run_own(s, case):
    import gemm_int8_b200 as g

    kind = case["kind"]
    if kind == "route":
        return g.route_experts(s["logits"], case["k"], bias=s["bias"], **_router_args(case))
    if kind == "group":
        first, held = _held(case)
        return g.group_by_expert(s["experts"], held, first)
    if kind == "product":
        return g.matmul_experts(s["x_q"], s["w_q"], s["x_scale"], s["w_scale"], s["offsets"], s["slots"], case["k"])
    if kind == "swiglu":
        return g.matmul_experts_swiglu(s["x_q"], s["w_q"], s["x_scale"], s["w_scale"], s["offsets"], s["slots"], case["k"])
    if kind == "combine":
        return g.combine_experts(s["y"], s["weights"], s["places"], s["add"])
    return s["layer"](s["x"], s["logits"], s["add"])


def _route(logits, bias, case):
    """The plain router.  Scores are compared in 64 bits, as two that differ may be equal in 32; without a bias the logits themselves
    are compared, of which the scores are increasing functions."""
    l = logits.double()
    if case["scoring"] == "softmax":
        e = torch.exp(l - l.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-l))
    choice = l if bias is None else score + bias.double()
    T, E, G = l.shape[0], l.shape[1], case["groups"]
    if G > 1:
        if case["group_score"] == "max":
            of_group = choice.reshape(T, G, E // G).amax(2)
        else:
            of_group = (score if bias is None else choice).reshape(T, G, E // G).sort(dim=2, descending=True).values[:, :, :2].sum(2)
        best = of_group.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros(T, G, dtype=torch.bool, device=l.device)
        kept[torch.arange(T, device=l.device)[:, None], best] = True
        choice = torch.where(kept.repeat_interleave(E // G, dim=1), choice, -math.inf)
    experts = choice.sort(dim=1, descending=True, stable=True).indices[:, :case["k"]]
    weights = score[torch.arange(T, device=l.device)[:, None], experts]
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    return weights * case["scale"], experts.to(torch.int32)


def _product(x_q, w_q, x_scale, w_scale, offsets, slots, k, dtype):
    """Rows times their experts' weights in `dtype`, zero behind the last expert's rows."""
    rows = x_q.shape[0] if slots is None else slots.numel()
    out = torch.zeros(rows, w_q.shape[1], dtype=dtype, device=x_q.device)
    ends = offsets.tolist()
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        if a < b:
            src = slice(a, b) if slots is None else slots[a:b].long() // k
            out[a:b] = (x_q[src].to(dtype) @ w_q[e].to(dtype).t()) * (x_scale[src].to(dtype)[:, None] * w_scale[e].to(dtype)[None, :])
    return out


def _silu_times(gate_up):
    gate, up = gate_up.chunk(2, dim=1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _combine(y, weights, places, add, dtype):
    out = torch.zeros(places.shape[0], y.shape[1], dtype=dtype, device=y.device) if add is None else add.to(dtype)
    for j in range(places.shape[1]):
        p = places[:, j].long()
        rows = y[p.clamp_min(0)].to(dtype) * weights[:, j, None].to(dtype)
        out = out + torch.where((p >= 0)[:, None], rows, torch.zeros_like(rows))
    return out


def _quantise(v):
    """Symmetric per-row int8: scale = largest magnitude / 127 (1 for a row of zeros), round half to even."""
    s = v.abs().amax(1) / 127.0
    s = torch.where(s > 0, s, torch.ones_like(s))
    return torch.round(v / s[:, None]).clamp(-127, 127).to(torch.int8), s


def _run_plain(s, case):
    kind, k, f32, bf16 = case["kind"], case["k"], torch.float32, torch.bfloat16
    if kind == "route":
        weights, experts = _route(s["logits"], s["bias"], case)
        return weights.float(), experts
    if kind == "group":
        return _group(s["experts"], *_held(case))
    if kind == "product":
        return _product(s["x_q"], s["w_q"], s["x_scale"], s["w_scale"], s["offsets"], s["slots"], k, f32).to(bf16)
    if kind == "swiglu":
        return _silu_times(_product(s["x_q"], s["w_q"], s["x_scale"], s["w_scale"], s["offsets"], s["slots"], k, f32)).to(bf16)
    if kind == "combine":
        return _combine(s["y"], s["weights"], s["places"], s["add"], f32).to(bf16)
    # the layer: its operators in a row, each with its result rounded to the type that it has between them
    weights, experts = _route(s["logits"], s["bias"], case)
    offsets, slots, places = _group(experts, 0, case["E"])
    x_q, x_scale = _quantise(s["x"].float())
    h = _silu_times(_product(x_q, s["gate_up"], x_scale, s["gate_up_scale"], offsets, slots, k, f32)).to(bf16)
    h_q, h_scale = _quantise(h.float())
    y = _product(h_q, s["down"], h_scale, s["down_scale"], offsets, None, k, f32).to(bf16)
    return _combine(y, weights.float(), places, s["add"], f32).to(bf16)


# --------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------
def _use(case):
    """(rows of this rank, its experts that have any), expected for tokens that choose by popularity."""
    _, held = _held(case)
    T, E, k = case["T"], case["E"], case["k"]
    p = [math.exp(v) for v in _popularity(E)]
    total = sum(p)
    met = sum(1.0 - (1.0 - min(1.0, k * v / total)) ** T for v in p)
    return T * k * held / E, max(1.0, met * held / E)


def work(case):
    kind, T, E, k = case["kind"], case["T"], case["E"], case["k"]
    if kind == "route":
        return {"bytes": T * E * (2 if case["logits"] == "bf16" else 4) + 8 * T * k + (4 * E if case["bias"] else 0), "flops": 4 * T * E}
    rows, met = _use(case)
    if kind == "group":
        return {"bytes": 12 * T * k + 4 * _held(case)[1], "flops": T * k}
    if kind == "combine":
        return {"bytes": int(2 * rows * case["N"] + 2 * T * case["N"] * (2 if case["add"] else 1) + 8 * T * k), "flops": int(2 * rows * case["N"])}
    N, K = case["N"], case["K"]
    if kind == "layer":
        ends = 2 * T * (2 * K + E + (K if case["add"] else 0)) + (2 * T * E if case["logits"] == "fp32" else 0)
        return {"bytes": int(met * 3 * N * K + met * 4 * (2 * N + K) + ends), "flops": int(6 * rows * N * K)}
    wide = 2 * N if kind == "swiglu" else N
    read = (min(T, rows) if case["gather"] else rows) * (K + 4)
    return {"bytes": int(met * wide * (K + 4) + read + 2 * T * k * N + 4 * rows * case["gather"]), "flops": int(2 * rows * wide * K)}


# --------------------------------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------------------------------
def _exact_route(t, case):
    """Token by token on the host: scores, groups and experts by Python's own sort of (-value, index)."""
    weights, chosen = [], []
    bias = None if t["bias"] is None else t["bias"].double().tolist()
    E, G, k = case["E"], case["groups"], case["k"]
    for row in t["logits"].double().tolist():
        if case["scoring"] == "softmax":
            top = max(row)
            e = [math.exp(v - top) for v in row]
            total = math.fsum(e)
            score = [v / total for v in e]
        else:
            score = [1.0 / (1.0 + math.exp(-v)) for v in row]
        key = row if bias is None else [a + b for a, b in zip(score, bias)]
        pool = range(E)
        if G > 1:
            size = E // G
            if case["group_score"] == "max":
                value = [max(key[g * size:(g + 1) * size]) for g in range(G)]
            else:
                value = [sum(sorted((score if bias is None else key)[g * size:(g + 1) * size])[-2:]) for g in range(G)]
            groups = sorted(range(G), key=lambda g: (-value[g], g))[:case["top_groups"]]
            pool = [e for g in groups for e in range(g * size, (g + 1) * size)]
        ids = sorted(pool, key=lambda e: (-key[e], e))[:k]
        w = [score[e] for e in ids]
        total = math.fsum(w) if case["renormalize"] else 1.0
        weights.append([v / total * case["scale"] for v in w])
        chosen.append(ids)
    return torch.tensor(weights, dtype=torch.float64, device="cuda"), torch.tensor(chosen, dtype=torch.int32, device="cuda")


def _exact_group(experts, first, held):
    """Buckets on the host."""
    flat = experts.reshape(-1).tolist()
    buckets = [[] for _ in range(held)]
    for slot, e in enumerate(flat):
        if first <= e < first + held:
            buckets[e - first].append(slot)
    offsets, slots, places = [0], [], [-1] * len(flat)
    for b in buckets:
        for slot in b:
            places[slot] = len(slots)
            slots.append(slot)
        offsets.append(len(slots))
    slots += [-1] * (len(flat) - len(slots))
    return tuple(torch.tensor(v, dtype=torch.int32, device="cuda") for v in (offsets, slots)) + (
        torch.tensor(places, dtype=torch.int32, device="cuda").reshape(experts.shape),)


def _exact_rows(x, w_q, w_scale, offsets, of_row):
    """Float64 rows (already scaled) times dequantised weights; `of_row`: which row of x a result's row reads."""
    out = torch.zeros(of_row.numel(), w_q.shape[1], dtype=torch.float64, device=x.device)
    ends = offsets.tolist()
    for e in range(w_q.shape[0]):
        a, b = ends[e], ends[e + 1]
        if b > a:
            w = w_q[e].double() * w_scale[e].double()[:, None]
            out[a:b] = torch.mm(x.index_select(0, of_row[a:b]), w.t())
    return out


def _exact_swiglu(v):
    half = v.shape[1] // 2
    return v[:, :half] * torch.sigmoid(v[:, :half]) * v[:, half:]


def _exact_rounded(v):
    """What per-row int8 quantisation leaves of v."""
    s = v.abs().amax(dim=1, keepdim=True) / 127.0
    s[s == 0] = 1.0
    return (v / s).round().clamp(-127, 127) * s


def exact(case, seed):
    t = _inputs(case, seed)
    kind, k = case["kind"], case["k"]
    if kind == "route":
        return _exact_route(t, case)
    if kind == "group":
        return _exact_group(t["experts"], *_held(case))
    if kind == "combine":
        held = torch.cat([t["y"].double(), torch.zeros(1, case["N"], dtype=torch.float64, device="cuda")])  # place -1 reads the zero row
        out = sum(t["weights"][:, j:j + 1].double() * held[t["places"][:, j].long()] for j in range(k))
        return out if t["add"] is None else out + t["add"].double()
    if kind == "layer":
        weights, experts = _exact_route(t, case)
        offsets, slots, places = _exact_group(experts, 0, case["E"])
        x = _exact_rounded(t["x"].double())
        h = _exact_swiglu(_exact_rows(x, t["gate_up"], t["gate_up_scale"], offsets, slots.long() // k))
        h = _exact_rounded(h.to(torch.bfloat16).double())  # what is quantised is the bf16 result of the first product
        y = _exact_rows(h, t["down"], t["down_scale"], offsets, torch.arange(h.shape[0], device="cuda"))
        out = (weights[:, :, None] * y[places.long()]).sum(dim=1)
        return out if t["add"] is None else out + t["add"].double()
    x = t["x_q"].double() * t["x_scale"].double()[:, None]
    of_row = torch.arange(x.shape[0], device="cuda") if t["slots"] is None else t["slots"].long().clamp_min(0) // k
    out = _exact_rows(x, t["w_q"], t["w_scale"], t["offsets"], of_row)
    return _exact_swiglu(out) if kind == "swiglu" else out
