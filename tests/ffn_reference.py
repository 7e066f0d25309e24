"""The operators of gemm_int8_b200.ffn in 64 bits, and how far fp32 arithmetic may be from them (test infrastructure)."""
import torch

F8 = torch.float8_e4m3fn
TOP = {torch.int8: 127.0, F8: 448.0}


def norm(x, weight, residual, eps):
    """(v, h) in 64 bits."""
    h = x.double() if residual is None else x.double() + residual.double()
    return h / (h.square().mean(1, keepdim=True) + eps).sqrt() * weight.double(), h


# h one rounding (2^-24); its square, a sum of at most 16 terms a thread and 10 levels of a tree, and the mean's division 28 roundings, of
# which the root halves the effect; rsqrtf 2 units in the last place (4 x 2^-24), two products: 1 + 14 + 4 + 2 + (eps) 1 = 22 of 2^-24.
NORM_REL = 2.0 ** -19


def swiglu(gate_up):
    """(v, bound of |fp32 v - v|) in 64 bits: __expf is off by 2 + 1.173 |g| units in the last place (CUDA's bound), 1 + e by half a unit, the quick
    division by two, the product with u by half a unit; a unit is at most 2^-23 of the value.  Below -88 the exponential overflows and v is zero."""
    g, u = gate_up.double().chunk(2, dim=1)
    v = g * torch.sigmoid(g) * u
    rel = (5.0 + 1.2 * g.abs()) * 2.0 ** -23
    return v, v.abs() * rel + torch.where(g < -80, v.abs(), torch.zeros_like(v)) + 2.0 ** -120


def blocks(v, fill=0.0):
    return torch.nn.functional.pad(v, (0, -v.shape[1] % 128), value=fill).reshape(v.shape[0], -1, 128)


def check_quantised(q, s, v, err, dtype, per_block):
    """q, s against the 64-bit values v, each known to +-err: the scale against the largest value, every q against its value over the scale that came."""
    assert q.dtype == dtype and s.dtype == torch.float32 and q.shape == v.shape
    top = TOP[dtype]
    if per_block:
        assert s.shape == (v.shape[0], -(-v.shape[1] // 128))
        amax, slack = blocks(v).abs().amax(2), blocks(err).amax(2)
        spread = s.double().repeat_interleave(128, 1)[:, : v.shape[1]]
    else:
        assert s.shape == (v.shape[0],)
        amax, slack = v.abs().amax(1), err.amax(1)
        spread = s.double()[:, None].expand_as(v)
    want = torch.where(amax > 0, amax / top, torch.ones_like(amax))
    ok = (s.double() - want).abs() <= slack / top + want * 2.0 ** -23
    # (values that all lie within their error of zero may be zeros, whose scale is 1: the rule jumps there)
    ok |= (s == 1.0) & (amax <= slack)
    assert bool(ok.all()), float(((s.double() - want).abs() / want)[~ok].max())
    t = v / spread
    if dtype == torch.int8:
        half = torch.full_like(t, 0.5)
    else:
        _, e = torch.frexp(t.abs().clamp_min(2.0 ** -30))
        half = torch.ldexp(torch.ones_like(t), (e - 1).clamp_min(-6) - 4)
    # (the quotient: one rounding; a value on the other side of a power of two by its error has the larger step)
    bad = (q.double() - t).abs() > half + 2 * err / spread + t.abs() * 2.0 ** -23
    assert not bool(bad.any()), (int(bad.sum()), q[bad][:4], t[bad][:4])


def spread_scales(s, columns):
    return s.double().repeat_interleave(128, dim=1)[:, :columns]


def product(x_q, w_q, x_scale, w_scale):
    """(out, bound of the fp32 result's error) in 64 bits: a block's dot product in fp32 in any order, truncating, 128 x 2^-23 of the sum of
    magnitudes; the scales' product and the chain over the blocks (KB + 1) x 2^-24 of it."""
    x = x_q.double() * spread_scales(x_scale, x_q.shape[1])
    w = w_q.double() * spread_scales(w_scale, w_q.shape[1]).repeat_interleave(128, dim=0)[: w_q.shape[0]]
    KB = x_scale.shape[1]
    return x @ w.t(), (x.abs() @ w.abs().t()) * (128 * 2.0 ** -23 + (KB + 1) * 2.0 ** -24)


def check_bf16(out, want, err):
    """A value known to +-err, rounded to bf16: half a step (2^-8 of the value)."""
    bad = (out.double() - want).abs() > want.abs() * 2.0 ** -8 + err * (1 + 2.0 ** -8)
    assert not bool(bad.any()), (int(bad.sum()), out[bad][:4], want[bad][:4])


def outliers(gen, M, H, dtype, device="cuda"):
    a = torch.randn(M, H, generator=gen, device=device)
    a[:, ::97] *= 20
    return a.to(dtype)
