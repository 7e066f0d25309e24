"""Operators around the products of a feed-forward (or attention) block in 8 bits, and the block-scaled product in 8-bit floating point.

A block in W8A8 is norm, product, activation, product; the norm and the activation produce what the products take, 8-bit values and their
scales, in one pass.  The reference has the product only.  Inference only, as everything in this package.

    q, s, stream = rms_norm_quantize(x, weight, stream)         # stream: the residual stream, onto which x is added first
    gate_up = matmul_blockwise(q, w1_q, s, w1_scale)
    q, s = swiglu_quantize(gate_up)
    x = matmul_blockwise(q, w2_q, s, w2_scale)
"""
from __future__ import annotations

import torch

_NS = "gemm_int8_CUDA"
_ops = torch.ops.gemm_int8_CUDA
# (the overloads themselves: a call that looks for them first takes half a microsecond longer)
_norm, _swiglu, _matmul = (op.default for op in (_ops.rms_norm_quantize, _ops.swiglu_quantize, _ops.fp8_matmul_blockwise))
_E4M3 = torch.float8_e4m3fn


def _refuse(scales, dtype):
    if scales not in ("block", "token"):
        raise ValueError("scales must be 'block' or 'token'")
    if dtype not in (torch.int8, _E4M3):
        raise ValueError("dtype must be torch.int8 or torch.float8_e4m3fn")
    raise ValueError("float8_e4m3fn has block scales, which matmul_blockwise_fp8 takes")


def _form(scales, dtype):
    """(blockwise, e4m3)"""
    if scales == "block":
        if dtype == torch.int8 or dtype == _E4M3:
            return True, dtype == _E4M3
    elif scales == "token" and dtype == torch.int8:
        return False, False
    _refuse(scales, dtype)


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6, *, scales: str = "block",
                      dtype: torch.dtype = torch.int8):
    """Root-mean-square norm in 8 bits: x [M, H] fp32/bf16 -> (q [M, H], scales), or with a residual -> (q, scales, x + residual).

    ``h = x + residual;  v = h / sqrt(mean(h^2) + eps) * weight`` in fp32, quantised as the package's quantisers do: scales="block" one scale per
    token and 128 columns (fp32 [M, ceil(H/128)], for `matmul_blockwise` and, with dtype=torch.float8_e4m3fn, `matmul_blockwise_fp8`),
    scales="token" one per token (fp32 [M], int8 only, for `matmul_scaled`).  The sum comes back in the residual's type; the norm is of the
    sum in fp32, before it is rounded to that type.  weight [H] and residual [M, H] are fp32 or bf16, each independently; H is a multiple of 16,
    at most 32768, and eps lies between 1e-20 and 1e20.  A NaN or infinity in a token makes the scales it reaches NaN or infinite.
    A token's results do not depend on the other tokens or their number.
    """
    blockwise, e4m3 = _form(scales, dtype)
    q, s, total = _norm(x, weight, residual, eps, blockwise, e4m3)
    return (q, s) if residual is None else (q, s, total)


def swiglu_quantize(gate_up: torch.Tensor, *, scales: str = "block", dtype: torch.dtype = torch.int8):
    """``silu(gate) * up`` in 8 bits: gate_up [M, 2 N] fp32/bf16 (N gate columns, then N up columns) -> (q [M, N], scales).

    In fp32, quantised once; scales and dtype as in `rms_norm_quantize`.  N is a multiple of 16 below 131072.
    """
    return _swiglu(gate_up, *_form(scales, dtype))


def matmul_blockwise_fp8(x_q: torch.Tensor, w_q: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor) -> torch.Tensor:
    """`matmul_blockwise` in 8-bit floating point -> bf16 [M, N].

    ``out[m, n] = bf16( sum_kb P[m, n, kb] * (x_scale[m, kb] * w_scale[n // 128, kb]) )`` where ``P`` is the fp32 dot product over the kb-th
    128-wide K block, accumulated in fp32 in ascending kb order (where few tiles have long sums, in up to eight ranges of K blocks whose sums are
    added up in order).  x_q (M, K) and w_q (N, K) float8_e4m3fn, x_scale (M, ceil(K/128)) and w_scale (ceil(N/128), ceil(K/128)) fp32; K a
    multiple of 16 below 131072.
    """
    return _matmul(x_q, w_q, x_scale, w_scale)


# --------------------------------------------------------------------------------------------------
# fake (meta) kernels
# --------------------------------------------------------------------------------------------------
def _fake_out8(like, rows, cols, blockwise, e4m3):
    s = (rows, (cols + 127) // 128) if blockwise else (rows,)
    return (torch.empty(rows, cols, device=like.device, dtype=_E4M3 if e4m3 else torch.int8), torch.empty(s, device=like.device, dtype=torch.float32))


@torch.library.register_fake(f"{_NS}::rms_norm_quantize")
def _(x, weight, residual, eps, blockwise, e4m3):
    torch._check(len(x.shape) == 2, lambda: "x must be a 2D tensor")
    total = torch.empty(0, device=x.device, dtype=x.dtype) if residual is None else torch.empty(x.shape, device=x.device, dtype=residual.dtype)
    return (*_fake_out8(x, x.shape[0], x.shape[1], blockwise, e4m3), total)


@torch.library.register_fake(f"{_NS}::swiglu_quantize")
def _(gate_up, blockwise, e4m3):
    torch._check(len(gate_up.shape) == 2, lambda: "gate_up must be a 2D tensor")
    return _fake_out8(gate_up, gate_up.shape[0], gate_up.shape[1] // 2, blockwise, e4m3)


@torch.library.register_fake(f"{_NS}::fp8_quantize_token_block")
def _(a):
    torch._check(len(a.shape) == 2, lambda: "a must be a 2D tensor")
    return _fake_out8(a, a.shape[0], a.shape[1], True, True)


@torch.library.register_fake(f"{_NS}::fp8_matmul_blockwise")
def _(x, y, A_scale, B_scale):
    torch._check(len(x.shape) == 2 and len(y.shape) == 2, lambda: "x and y must be 2D tensors")
    torch._check(x.dtype == _E4M3 and y.dtype == _E4M3, lambda: "x and y must be float8_e4m3fn tensors")
    torch._check(x.shape[1] == y.shape[1], lambda: "x.shape[1] must be equal to y.shape[1]")
    return torch.empty(x.shape[0], y.shape[0], device=x.device, dtype=torch.bfloat16)


@torch.library.register_fake(f"{_NS}::fp8_linear")
def _(x, weight_q, weight_scale, bias):
    torch._check(len(x.shape) == 2 and len(weight_q.shape) == 2, lambda: "x and weight_q must be 2D tensors")
    torch._check(weight_q.dtype == _E4M3, lambda: "weight_q must be a float8_e4m3fn tensor")
    torch._check(x.shape[1] == weight_q.shape[1], lambda: "x.shape[1] must be equal to weight_q.shape[1]")
    return torch.empty(x.shape[0], weight_q.shape[0], device=x.device, dtype=torch.bfloat16)
