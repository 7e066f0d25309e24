"""Mixture-of-experts layer in W8A8: the router, the grouping by expert, the experts' products, the weighted sum, and the layer that runs them.

The reference has one dense product only; these are its counterparts where every token has experts of its own.  All steps take their
sizes from tensors on the device (how many rows an expert has is never read back), so a layer can be captured into a CUDA graph and replayed
with other tokens.  Inference only, as everything in this package.
"""
from __future__ import annotations

import torch

from . import quant

_NS = "gemm_int8_CUDA"
_ops = torch.ops.gemm_int8_CUDA
# (the overloads themselves: a call that looks for them first takes half a microsecond longer)
_route, _group, _matmul, _combine, _layer = (op.default for op in (_ops.route_experts, _ops.group_by_expert, _ops.int8_matmul_experts, _ops.combine_experts, _ops.int8_experts))
_SIGMOID = {"softmax": False, "sigmoid": True}
_TOP2 = {"max": False, "top2": True}


def _refuse(scoring, group_score):
    if scoring not in _SIGMOID:
        raise ValueError("scoring must be 'softmax' or 'sigmoid'") from None
    raise ValueError("group_score must be 'max' or 'top2'") from None


def route_experts(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
                  top_groups: int | None = None, group_score: str = "max", renormalize: bool = True, scale: float = 1.0):
    """The `top_k` experts of every token: logits [T, E] fp32/bf16 -> (weights fp32 [T, top_k], experts int32 [T, top_k]).

    ``score = softmax(logits)`` or ``sigmoid(logits)``; the choice is by ``score + bias`` (bias fp32 [E], for balance: it does not enter the
    weights), in descending order, the lower index first among equals.  groups > 1: the experts form that many equal runs, and only the
    top_groups of them with the best value (group_score "max": the largest choice, "top2": the sum of the two largest) keep theirs.
    ``weights = score of the chosen (/ their sum) * scale``.

    A logit (or bias) of -inf masks an expert, and so does NaN; a logit of +inf counts as the largest finite value of fp32, so that a softmax
    shares its weight among the infinite ones.  Where fewer than top_k experts are left, the remaining places hold expert -1 and weight 0,
    which the operators below skip.  Near ties are decided by the values in 64 bits, not by how fp32 rounds a score.  E <= 1024,
    top_k <= 32, groups <= 32.
    """
    try:
        sigmoid, top2 = _SIGMOID[scoring], _TOP2[group_score]
    except (KeyError, TypeError):
        _refuse(scoring, group_score)
    return _route(logits, bias, top_k, sigmoid, groups, groups if top_groups is None else top_groups, top2, renormalize, scale)


def group_by_expert(experts: torch.Tensor, num_experts: int, first_expert: int = 0):
    """Rows for the experts' products: experts int32 [T, top_k] -> (offsets int32 [num_experts + 1], slots int32 [T top_k], places int32 [T, top_k]).

    Rows offsets[e] .. offsets[e + 1] - 1 are those of expert first_expert + e, in the order of their pairs (token, choice).  slots holds the
    pair, token * top_k + choice, of each row (-1 behind the last one), places the row of each pair (-1 for an expert that is not one of
    the num_experts here: expert -1, or one of another rank's).
    """
    return _group(experts, num_experts, first_expert)


def _pairs(slots, top_k):
    if top_k is None:
        if slots is not None:
            raise ValueError("slots are pairs of a token and a choice: top_k must be given with them")
        return 1
    return top_k


def matmul_experts(x_q: torch.Tensor, w_q: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor,
                   slots: torch.Tensor | None = None, top_k: int | None = None) -> torch.Tensor:
    """`matmul_scaled` with a weight of its own for every group of rows -> bf16 [rows, N].

    ``out[p, n] = bf16( fp32(x_q[s] . w_q[e, n]) * (x_scale[s] * w_scale[e, n]) )`` for offsets[e] <= p < offsets[e + 1], where s is p or, with
    slots, the token slots[p] // top_k: rows are then read where the tokens lie, without a copy.  Rows in front of offsets[0] and from offsets[-1] on are zero.
    x_q int8 [rows or tokens, K], w_q int8 [E, N, K], x_scale fp32 [rows or tokens], w_scale fp32 [E, N]; K a multiple of 16.  top_k, the
    pairs of a token, has to be given with slots and means nothing without.
    """
    return _matmul(x_q, w_q, x_scale, w_scale, offsets, slots, _pairs(slots, top_k), False)


def matmul_experts_swiglu(x_q: torch.Tensor, w_q: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor,
                          slots: torch.Tensor | None = None, top_k: int | None = None) -> torch.Tensor:
    """`matmul_experts` for a weight [E, 2 N, K] of N gate rows and then N up rows -> bf16 [rows, N]: ``silu(gate) * up`` of the two products in
    fp32, rounded once."""
    return _matmul(x_q, w_q, x_scale, w_scale, offsets, slots, _pairs(slots, top_k), True)


def combine_experts(y: torch.Tensor, weights: torch.Tensor, places: torch.Tensor, add: torch.Tensor | None = None) -> torch.Tensor:
    """Weighted sum of every token's rows: ``out[t] = bf16( add[t] + sum_j weights[t, j] * y[places[t, j]] )`` in fp32, ascending j.

    y bf16 [rows, N], weights fp32 [T, top_k], places int32 [T, top_k] (negative: left out), add fp32 or bf16 [T, N] or None; top_k <= 32.
    """
    return _combine(y, weights, places, add)


# --------------------------------------------------------------------------------------------------
# fake (meta) kernels
# --------------------------------------------------------------------------------------------------
@torch.library.register_fake(f"{_NS}::route_experts")
def _(logits, bias, top_k, sigmoid, groups, top_groups, group_top2, renormalize, scale):
    torch._check(len(logits.shape) == 2, lambda: "logits must be a 2D tensor")
    shape = (logits.shape[0], top_k)
    return torch.empty(shape, device=logits.device, dtype=torch.float32), torch.empty(shape, device=logits.device, dtype=torch.int32)


@torch.library.register_fake(f"{_NS}::group_by_expert")
def _(experts, num_experts, first_expert):
    torch._check(len(experts.shape) == 2 and experts.dtype == torch.int32, lambda: "experts must be a 2D int32 tensor")
    return experts.new_empty(num_experts + 1), experts.new_empty(experts.shape[0] * experts.shape[1]), experts.new_empty(experts.shape)


@torch.library.register_fake(f"{_NS}::int8_matmul_experts")
def _(x, weight_q, x_scale, weight_scale, offsets, slots, top_k, swiglu):
    torch._check(len(x.shape) == 2 and len(weight_q.shape) == 3, lambda: "x must be a 2D and the weight a 3D tensor")
    torch._check(x.dtype == torch.int8 and weight_q.dtype == torch.int8, lambda: "x and the weight must be int8 tensors")
    torch._check(x.shape[1] == weight_q.shape[2], lambda: "x.shape[1] must be equal to weight_q.shape[2]")
    rows = x.shape[0] if slots is None else slots.shape[0]
    return torch.empty(rows, weight_q.shape[1] // 2 if swiglu else weight_q.shape[1], device=x.device, dtype=torch.bfloat16)


@torch.library.register_fake(f"{_NS}::combine_experts")
def _(y, weights, places, add):
    torch._check(len(y.shape) == 2 and len(weights.shape) == 2, lambda: "y and weights must be 2D tensors")
    return torch.empty(weights.shape[0], y.shape[1], device=y.device, dtype=torch.bfloat16)


@torch.library.register_fake(f"{_NS}::int8_experts")
def _(x, logits, bias, gate_up_q, gate_up_scale, down_q, down_scale, top_k, sigmoid, groups, top_groups, group_top2, renormalize, scale, first_expert, add):
    torch._check(len(x.shape) == 2 and len(logits.shape) == 2, lambda: "x and logits must be 2D tensors")
    return torch.empty(x.shape, device=x.device, dtype=torch.bfloat16)


# --------------------------------------------------------------------------------------------------
# layer
# --------------------------------------------------------------------------------------------------
def _quantize_experts(weight: torch.Tensor):
    """weight [E, N, K] -> (int8 [E, N, K], fp32 scales [E, N]), expert by expert."""
    q = torch.empty(weight.shape, dtype=torch.int8, device=weight.device)
    s = torch.empty(weight.shape[:2], dtype=torch.float32, device=weight.device)
    for e in range(weight.shape[0]):
        q[e], s[e] = quant.quantize_per_row(weight[e].detach().to(torch.float32))
    return q, s


class Int8Experts(torch.nn.Module):
    """The feed-forward block of a mixture of experts in W8A8: ``sum_j weight_j * down_e(silu(gate_e(x)) * up_e(x))`` over a token's experts.

    Weights are quantised once, per output channel; activations on the fly, per token.  The module holds experts first_expert ..
    first_expert + E - 1 of a router that may have more (the others' share of the sum is left to whoever holds them).

    gate_up_q int8 [E, 2 inner, hidden] (gate rows, then up rows), gate_up_scale fp32 [E, 2 inner], down_q int8 [E, hidden, inner],
    down_scale fp32 [E, hidden]; the other arguments are those of `route_experts`.  hidden and inner are multiples of 16.
    """

    def __init__(self, gate_up_q: torch.Tensor, gate_up_scale: torch.Tensor, down_q: torch.Tensor, down_scale: torch.Tensor, top_k: int, *,
                 scoring: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1, top_groups: int | None = None,
                 group_score: str = "max", renormalize: bool = True, scale: float = 1.0, first_expert: int = 0):
        super().__init__()
        if scoring not in _SIGMOID or group_score not in _TOP2:
            _refuse(scoring, group_score)
        self._router = (top_k, _SIGMOID[scoring], groups, groups if top_groups is None else top_groups, _TOP2[group_score], renormalize, float(scale))
        self.top_k = top_k
        self.first_expert = first_expert
        self.register_buffer("gate_up_q", gate_up_q.contiguous())
        self.register_buffer("gate_up_scale", gate_up_scale.contiguous())
        self.register_buffer("down_q", down_q.contiguous())
        self.register_buffer("down_scale", down_scale.contiguous())
        self.register_buffer("bias", bias)

    @classmethod
    def from_float(cls, gate_up: torch.Tensor, down: torch.Tensor, top_k: int, **router) -> "Int8Experts":
        """Quantises fp32/bf16 weights gate_up [E, 2 inner, hidden] and down [E, hidden, inner] once, on whatever device they live."""
        return cls(*_quantize_experts(gate_up), *_quantize_experts(down), top_k, **router)

    def forward(self, x: torch.Tensor, logits: torch.Tensor, add: torch.Tensor | None = None) -> torch.Tensor:
        """x [..., hidden], logits [..., experts of the router], add (the residual stream, a shared expert's result) [..., hidden] -> bf16 [..., hidden].

        x, logits and add are taken as they are in fp32 and bf16.  Of other types, fp16 activations go to bf16, as in `Int8Linear`, and everything
        else to fp32.
        """
        x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
        if x2.dtype not in (torch.float32, torch.bfloat16):
            x2 = x2.to(torch.bfloat16 if x2.dtype == torch.float16 else torch.float32)
        logits = logits.reshape(-1, logits.shape[-1])
        if logits.dtype not in (torch.float32, torch.bfloat16):
            logits = logits.to(torch.float32)
        if add is not None:
            add = add.reshape(x2.shape)
            if add.dtype not in (torch.float32, torch.bfloat16):
                add = add.to(torch.float32)
        out = _layer(x2, logits, self.bias, self.gate_up_q, self.gate_up_scale, self.down_q, self.down_scale, *self._router,
                                                    self.first_expert, add)
        return out if x.dim() == 2 else out.reshape(x.shape)
