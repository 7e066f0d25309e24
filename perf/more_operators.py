"""The operators around the products of a W8A8 feed-forward block, and the product in 8-bit floating point, as a list of measurable cases.

    norm      x [M, H] (+ residual) -> root-mean-square norm times a weight, in 8 bits with scales; and the sum, which is the next residual
    swiglu    gate and up halves [M, 2 H] -> silu(gate) * up, in 8 bits with scales
    product   e4m3 x e4m3 with a scale per token and 128 inputs, and one per 128 x 128 of the weight, bf16 out
    linear    the layer on it: activations quantised to e4m3 on the way, bias: `Fp8Linear`

Inference only, as everything in this package.  Fields of a case (those that its kind has):
    kind                 one of the above
    M                    tokens
    H                    norm, swiglu: features of the result
    N, K                 product, linear: output and input features
    x                    norm, swiglu, linear: type of the activations, "bf16" | "fp32"
    residual             norm: its type, or "none"
    weight               norm: type of the weight
    out                  norm, swiglu: "e4m3" (a scale per token and 128 features), "int8" (the same), "int8_token" (a scale per token)
    bias                 linear: a bf16 bias is added

What comes in 8 bits is returned with its scales: e4m3 tensors as they are (floats), int8 as the values that it stands for, rounded to bf16.
"""
from __future__ import annotations

import math

import torch

own = False

_EPS = 1e-5
_F8 = torch.float8_e4m3fn
_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_FLOP_LIMIT = 2 * 16384 * 57344 * 8192  # of the largest listed case
_BYTE_LIMIT = 1_500_000_000             # of a drawn one; weights stay below a third of it


def listed():
    return [
        # The norm in front of one token's gate and up product.  Launch latency.
        {"name": "norm_decode1", "kind": "norm", "M": 1, "H": 4096, "x": "bf16", "residual": "bf16", "weight": "bf16", "out": "e4m3"},
        # The same over a batch of prompts of a wide model.
        {"name": "norm_prompts", "kind": "norm", "M": 16384, "H": 8192, "x": "bf16", "residual": "bf16", "weight": "bf16", "out": "e4m3"},
        # An odd number of tokens in front of an int8 product with per-token scales, the residual stream kept in fp32.
        {"name": "norm_int8_stream32", "kind": "norm", "M": 8191, "H": 4096, "x": "bf16", "residual": "fp32", "weight": "fp32", "out": "int8_token"},
        # Between the products of a decode batch in int8 with per-token scales.
        {"name": "swiglu_decode16", "kind": "swiglu", "M": 16, "H": 14336, "x": "bf16", "out": "int8_token"},
        # Between the products of a batch of prompts.
        {"name": "swiglu_prompts", "kind": "swiglu", "M": 4096, "H": 14336, "x": "bf16", "out": "e4m3"},
        # fp32 products (partial sums of several ranks), a width that is no whole number of scale blocks.
        {"name": "swiglu_ragged32", "kind": "swiglu", "M": 777, "H": 6992, "x": "fp32", "out": "e4m3"},
        # A decode batch: the weights are streamed past sixteen tokens.
        {"name": "product_decode16", "kind": "product", "M": 16, "N": 8192, "K": 8192},
        # A short prompt, no size a whole number of tiles, output rows of odd length.
        {"name": "product_ragged", "kind": "product", "M": 777, "N": 5003, "K": 6992},
        # A large square.
        {"name": "product_square", "kind": "product", "M": 8192, "N": 8192, "K": 8192},
        # The first product of a large model's feed-forward block over a batch of prompts.
        {"name": "product_prompts", "kind": "product", "M": 16384, "N": 57344, "K": 8192},
        # One layer of a decode batch.
        {"name": "linear_decode4", "kind": "linear", "M": 4, "N": 14336, "K": 4096, "x": "bf16", "bias": True},
        # One layer of a prompt.
        {"name": "linear_prompt", "kind": "linear", "M": 2048, "N": 11008, "K": 4096, "x": "bf16", "bias": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _features(rng, lo, hi):
    """A multiple of 16, and of 128 in seven cases of ten."""
    n = _log_int(rng, lo, hi)
    return max(lo, n // 128 * 128 if rng.random() < 0.7 else n // 16 * 16)


def draw(rng):
    while True:
        kind = rng.choice(["norm", "swiglu", "product", "linear"])
        c = {"kind": kind, "M": _log_int(rng, 1, 16384)}
        if kind in ("norm", "swiglu"):
            c.update(H=_features(rng, 128, 16384 if kind == "norm" else 32768), x=rng.choice(["bf16", "bf16", "fp32"]),
                     out=rng.choice(["e4m3", "int8", "int8_token"]))
            if kind == "norm":
                c.update(residual=rng.choice(["none", "bf16", "fp32"]), weight=rng.choice(["bf16", "fp32"]))
        else:
            c.update(N=_log_int(rng, 64, 57344), K=_features(rng, 128, 28672))
            if rng.random() < 0.7:
                c["N"] = max(64, c["N"] // 128 * 128)
            if kind == "linear":
                c.update(x=rng.choice(["bf16", "bf16", "fp32"]), bias=rng.random() < 0.5)
            if c["N"] * c["K"] > _BYTE_LIMIT // 3:
                continue
        if work(c)["bytes"] <= _BYTE_LIMIT and work(c)["flops"] <= _FLOP_LIMIT:
            return c


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------
def _randn(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def _activations(gen, M, H):
    """Gaussian, one channel in a thousand twenty times as large; a few tokens of a longer batch are padding."""
    a = _randn(gen, M, H)
    a[:, torch.randperm(H, device="cuda", generator=gen)[: max(1, H // 1000)]] *= 20.0
    a[13::97] = 0.0
    return a


def _blocks(v):
    """v [R, C] -> [R, ceil(C / 128), 128], zeros behind the last column."""
    pad = -v.shape[1] % 128
    return torch.nn.functional.pad(v, (0, pad)).reshape(v.shape[0], -1, 128)


def _quantise_block(v):
    """Per row and 128 columns: e4m3 and scales (largest magnitude / 448; 1 for a block of zeros)."""
    b = _blocks(v)
    s = b.abs().amax(2) / 448.0
    s = torch.where(s > 0, s, torch.ones_like(s))
    return (b / s[:, :, None]).reshape(v.shape[0], -1)[:, : v.shape[1]].to(_F8), s


def _quantise_weight(w):
    """Per 128 x 128."""
    N, K = w.shape
    b = torch.nn.functional.pad(w, (0, -K % 128, 0, -N % 128)).reshape(-(-N // 128), 128, -(-K // 128), 128)
    s = b.abs().amax((1, 3)) / 448.0
    q = (b / s[:, None, :, None]).reshape(b.shape[0] * 128, -1)[:N, :K]
    return q.to(_F8).contiguous(), s


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, M = case["kind"], case["M"]
    if kind == "norm":
        H = case["H"]
        t = {"x": _activations(gen, M, H).to(_TYPES[case["x"]]), "weight": (1.0 + 0.2 * _randn(gen, H)).to(_TYPES[case["weight"]])}
        t["residual"] = None if case["residual"] == "none" else (2.0 * _activations(gen, M, H)).to(_TYPES[case["residual"]])
        return t
    if kind == "swiglu":
        return {"gate_up": (1.5 * _activations(gen, M, 2 * case["H"])).to(_TYPES[case["x"]])}
    N, K = case["N"], case["K"]
    t = {}
    t["w_q"], t["w_scale"] = _quantise_weight(_randn(gen, N, K) * 0.02)
    x = _activations(gen, M, K)
    if kind == "linear":
        t["x"] = x.to(_TYPES[case["x"]])
        t["bias"] = _randn(gen, N).to(torch.bfloat16) if case["bias"] else None
    else:
        t["x_q"], t["x_scale"] = _quantise_block(x)
        t["x_q"] = t["x_q"].contiguous()
    return t


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own and case["kind"] == "linear":
        import gemm_int8_b200 as g

        state["layer"] = g.Fp8Linear(state["w_q"], state["w_scale"], state["bias"])
    return state


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------
def _spread(s, columns):
    """Block scales [R, B] -> [R, columns]."""
    return s.repeat_interleave(128, dim=1)[:, :columns]


def _values(q, s):
    """What int8 with scales stands for, rounded once to bf16."""
    out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    if s.dim() == 1:
        return torch.mul(q, s[:, None], out=out)
    if q.shape[1] % 128:
        return torch.mul(q, _spread(s, q.shape[1]), out=out)
    torch.mul(q.view(*s.shape, 128), s[:, :, None], out=out.view(*s.shape, 128))
    return out


def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


def _run_own(s, case):
    import gemm_int8_b200 as g

    kind = case["kind"]
    if kind == "product":
        return g.matmul_blockwise_fp8(s["x_q"], s["w_q"], s["x_scale"], s["w_scale"])
    if kind == "linear":
        return s["layer"](s["x"])
    how = {"scales": "token" if case["out"] == "int8_token" else "block", "dtype": _F8 if case["out"] == "e4m3" else torch.int8}
    if kind == "swiglu":
        q, *rest = g.swiglu_quantize(s["gate_up"], **how)
    else:
        q, *rest = g.rms_norm_quantize(s["x"], s["weight"], s["residual"], _EPS, **how)
    return (q if case["out"] == "e4m3" else _values(q, rest[0]), *rest)


def _quantised(v, out):
    if out == "e4m3":
        return _quantise_block(v)
    b = _blocks(v) if out == "int8" else v
    s = b.abs().amax(-1) / 127.0
    s = torch.where(s > 0, s, torch.ones_like(s))
    q = torch.round(b / s[..., None]).clamp(-127, 127).to(torch.int8)
    return _values(q.reshape(v.shape[0], -1)[:, : v.shape[1]].contiguous(), s), s


def _product(x_q, w_q, x_scale, w_scale):
    w = w_q.float() * _spread(w_scale, w_q.shape[1]).repeat_interleave(128, dim=0)[: w_q.shape[0]]
    return (x_q.float() * _spread(x_scale, x_q.shape[1])) @ w.t()


def _run_plain(s, case):
    kind = case["kind"]
    if kind == "norm":
        h = s["x"].float()
        if s["residual"] is not None:
            h = h + s["residual"].float()
        v = h / torch.sqrt((h * h).mean(1, keepdim=True) + _EPS) * s["weight"].float()
        total = () if s["residual"] is None else (h.to(s["residual"].dtype),)
        return (*_quantised(v, case["out"]), *total)
    if kind == "swiglu":
        gate, up = s["gate_up"].float().chunk(2, dim=1)
        return _quantised(gate / (1.0 + torch.exp(-gate)) * up, case["out"])
    if kind == "product":
        return _product(s["x_q"], s["w_q"], s["x_scale"], s["w_scale"]).to(torch.bfloat16)
    x_q, x_scale = _quantise_block(s["x"].float())
    out = _product(x_q, s["w_q"], x_scale, s["w_scale"])
    if s["bias"] is not None:
        out = out + s["bias"].float()
    return out.to(torch.bfloat16)


# --------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------
def work(case):
    kind, M = case["kind"], case["M"]
    size = {"bf16": 2, "fp32": 4, "none": 0}
    if kind in ("norm", "swiglu"):
        H = case["H"]
        out = H + 4 * (1 if case["out"] == "int8_token" else -(-H // 128))
        if kind == "swiglu":
            return {"bytes": M * (2 * H * size[case["x"]] + out), "flops": 8 * M * H}
        return {"bytes": M * (H * (size[case["x"]] + 2 * size[case["residual"]]) + out) + H * size[case["weight"]], "flops": 8 * M * H}
    N, K = case["N"], case["K"]
    KB = -(-K // 128)
    x = M * K * size[case["x"]] if kind == "linear" else M * (K + 4 * KB)
    return {"bytes": x + N * K + 4 * -(-N // 128) * KB + 2 * M * N + (2 * N if case.get("bias") else 0), "flops": 2 * M * N * K}


# --------------------------------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------------------------------
def _round_e4m3(v):
    """Nearest number of three mantissa bits, exponents from -6 on (even in the middle)."""
    mantissa, exponent = torch.frexp(v.abs().clamp_min(2.0 ** -30))  # (mantissa in [0.5, 1))
    step = torch.ldexp(torch.ones_like(v), (exponent - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def _exact_scale(b, top):
    s = b.abs().amax(dim=-1, keepdim=True) / top
    s[s == 0] = 1.0
    return s


def _exact_block(v):
    """(e4m3 values [R, C], scales [R, B]) of v in 64 bits."""
    R, C = v.shape
    b = torch.zeros(R, -(-C // 128) * 128, dtype=torch.float64, device=v.device)
    b[:, :C] = v
    b = b.view(R, -1, 128)
    s = _exact_scale(b, 448.0)
    return _round_e4m3(b / s).view(R, -1)[:, :C], s[:, :, 0]


def _exact_quantised(v, out):
    if out == "e4m3":
        return _exact_block(v)
    if out == "int8_token":
        s = _exact_scale(v, 127.0)
        return (v / s).round() * s, s[:, 0]
    R, C = v.shape
    b = torch.zeros(R, -(-C // 128) * 128, dtype=torch.float64, device=v.device)
    b[:, :C] = v
    b = b.view(R, -1, 128)
    s = _exact_scale(b, 127.0)
    return ((b / s).round() * s).view(R, -1)[:, :C], s[:, :, 0]


def _exact_scaled(q, s, rows):
    """Values of a quantised operand, each scale over `rows` rows and 128 columns."""
    v = q.double()
    for j in range(s.shape[1]):
        v[:, 128 * j : 128 * (j + 1)] *= s[:, j].double().repeat_interleave(rows)[: v.shape[0], None]
    return v


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        h = t["x"].double()
        if t["residual"] is not None:
            h += t["residual"].double()
        norm = torch.linalg.vector_norm(h, dim=1, keepdim=True)
        v = t["weight"].double() * h * torch.rsqrt(norm ** 2 / h.shape[1] + _EPS)
        return (*_exact_quantised(v, case["out"]), *(() if t["residual"] is None else (h,)))
    if kind == "swiglu":
        gate, up = t["gate_up"].double().split(case["H"], dim=1)
        return _exact_quantised(gate * torch.sigmoid(gate) * up, case["out"])
    w = _exact_scaled(t["w_q"], t["w_scale"], 128)
    if kind == "product":
        return torch.mm(_exact_scaled(t["x_q"], t["x_scale"], 1), w.t())
    q, s = _exact_block(t["x"].double())
    out = torch.mm(_exact_scaled(q, s, 1), w.t())
    return out if t["bias"] is None else out + t["bias"].double()
