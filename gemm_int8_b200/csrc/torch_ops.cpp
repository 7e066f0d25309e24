// CUDA implementations of the torch operators of the namespace gemm_int8_CUDA (their schemas and fake kernels are defined in
// Python): operand checks, allocation of the results, and one call into the C ABI on the current stream.
//
// The reference binds its operator in C++ as well (csrc/kernels/bindings.cpp:10-38).  What bounds a decode step is host
// time: with these bodies in Python, a linear layer of one token (4096 x 4096) took 25.4 us a call, with them here 12.2 us.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <torch/library.h>

#include <tuple>

#include "../../include/gemm_int8_b200.h"

// The torch and Python this library was compiled against; _build.py compares it with what is installed.
extern "C" {
extern const char gi8_torch_ops_built_for[];
const char gi8_torch_ops_built_for[] = GI8_BUILT_FOR;
}

namespace {

constexpr int64_t kBlock = 128;

int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

// A non-zero status of the C ABI becomes the package's Python exception, with its status code.
void check(int status)
{
    if (status == GI8_OK) return;
    const std::string message = gi8_last_error();
    pybind11::gil_scoped_acquire gil;
    pybind11::object type = pybind11::module_::import("gemm_int8_b200._lib").attr("GemmInt8Error");
    pybind11::object value = type(status, message);
    PyErr_SetObject(type.ptr(), value.ptr());
    throw pybind11::error_already_set();
}

struct Sizes {
    int64_t M, N, K;
};

// The reference checks contiguity, device type and same-GPU (bindings.cpp:15-20) and leaves dtype, rank and the K match
// to its fake kernel (gemm_int8/__init__.py:18-24); here the real kernel checks them all.
Sizes check_operands(const char* name, const at::Tensor& A, const at::Tensor& B)
{
    TORCH_CHECK(A.is_cuda() && B.is_cuda(), name, ": A and B must be CUDA tensors");
    TORCH_CHECK(A.device() == B.device(), name, ": A and B must be on the same GPU, got ", A.device(), " and ", B.device());
    TORCH_CHECK(A.scalar_type() == at::kChar && B.scalar_type() == at::kChar, name, ": A and B must be int8, got ", A.scalar_type(),
                " and ", B.scalar_type());
    TORCH_CHECK(A.dim() == 2 && B.dim() == 2, name, ": A and B must be 2-D");
    TORCH_CHECK(A.size(1) == B.size(1), name, ": A.shape[1] (", A.size(1), ") must equal B.shape[1] (", B.size(1), ")");
    TORCH_CHECK(A.is_contiguous() && B.is_contiguous(), name, ": A and B must be contiguous");
    return {A.size(0), B.size(0), A.size(1)};
}

void check_scale(const char* name, const char* what, const at::Tensor& t, at::IntArrayRef shape, const at::Device& device)
{
    TORCH_CHECK(t.device() == device, name, ": ", what, " must be on ", device, ", got ", t.device());
    TORCH_CHECK(t.scalar_type() == at::kFloat, name, ": ", what, " must be float32, got ", t.scalar_type());
    TORCH_CHECK(t.sizes() == shape, name, ": ", what, " must have shape ", shape, ", got ", t.sizes());
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// (straight from the allocator: a trip through the dispatcher costs half a microsecond more for each tensor)
at::Tensor new_tensor(at::IntArrayRef shape, at::ScalarType dtype, const at::Tensor& like)
{
    return at::detail::empty_cuda(shape, dtype, like.device(), std::nullopt);
}

const int8_t* i8(const at::Tensor& t) { return static_cast<const int8_t*>(t.data_ptr()); }
const float* f32(const at::Tensor& t) { return static_cast<const float*>(t.data_ptr()); }

at::Tensor int8_matmul(const at::Tensor& A, const at::Tensor& B, double alpha)
{
    const Sizes n = check_operands("int8_matmul", A, B);
    const c10::cuda::CUDAGuard guard(A.device());
    at::Tensor out = new_tensor({n.M, n.N}, at::kBFloat16, A);
    check(gi8_matmul(i8(A), i8(B), out.data_ptr(), n.M, n.N, n.K, static_cast<float>(alpha), stream_of(A)));
    return out;
}

at::Tensor int8_matmul_i32(const at::Tensor& A, const at::Tensor& B)
{
    const Sizes n = check_operands("int8_matmul_i32", A, B);
    const c10::cuda::CUDAGuard guard(A.device());
    at::Tensor out = new_tensor({n.M, n.N}, at::kInt, A);
    check(gi8_matmul_i32(i8(A), i8(B), static_cast<int32_t*>(out.data_ptr()), n.M, n.N, n.K, stream_of(A)));
    return out;
}

// Per-row scales: [R] or [R, 1].
at::Tensor row_scale(const char* name, const char* what, const at::Tensor& t, int64_t rows, const at::Device& device)
{
    const at::Tensor flat = t.dim() == 2 && t.size(1) == 1 ? t.reshape({-1}) : t;
    check_scale(name, what, flat, {rows}, device);
    return flat.contiguous();
}

at::Tensor int8_matmul_scaled(const at::Tensor& A, const at::Tensor& B, const at::Tensor& a_scale, const at::Tensor& b_scale)
{
    const char* name = "int8_matmul_scaled";
    const Sizes n = check_operands(name, A, B);
    const at::Tensor sa = row_scale(name, "a_scale", a_scale, n.M, A.device());
    const at::Tensor sb = row_scale(name, "b_scale", b_scale, n.N, A.device());
    const c10::cuda::CUDAGuard guard(A.device());
    at::Tensor out = new_tensor({n.M, n.N}, at::kBFloat16, A);
    // (only a forced scratch variant asks for a workspace)
    const int64_t bytes = gi8_matmul_scaled_workspace_bytes(n.M, n.N, n.K);
    at::Tensor ws;
    if (bytes > 0) ws = at::zeros({bytes}, at::TensorOptions().dtype(at::kByte).device(A.device()));
    check(gi8_matmul_scaled(i8(A), i8(B), f32(sa), f32(sb), out.data_ptr(), n.M, n.N, n.K, bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                            stream_of(A)));
    return out;
}

// Block scales [rows, cols] and their row stride; copied where the kernels could not walk them.
at::Tensor block_scale(const at::Tensor& t, int64_t& ld)
{
    const int64_t rows = t.size(0), cols = t.size(1);
    at::Tensor s = t.stride(1) != 1 && cols > 1 ? t.contiguous() : t;
    ld = rows > 1 ? s.stride(0) : cols;
    if (ld < cols) s = s.contiguous(), ld = cols;
    return s;
}

at::Tensor blockwise(const char* name, const at::Tensor& A, const at::Tensor& B, const at::Tensor& A_scale, const at::Tensor& B_scale,
                     bool as_f32)
{
    const Sizes n = check_operands(name, A, B);
    check_scale(name, "A_scale", A_scale, {n.M, blocks_of(n.K)}, A.device());
    check_scale(name, "B_scale", B_scale, {blocks_of(n.N), blocks_of(n.K)}, A.device());
    const c10::cuda::CUDAGuard guard(A.device());
    int64_t ld_sa, ld_sb;
    const at::Tensor sa = block_scale(A_scale, ld_sa), sb = block_scale(B_scale, ld_sb);
    at::Tensor out = new_tensor({n.M, n.N}, as_f32 ? at::kFloat : at::kBFloat16, A);
    if (as_f32)
        check(gi8_matmul_blockwise_f32(i8(A), i8(B), f32(sa), ld_sa, f32(sb), ld_sb, static_cast<float*>(out.data_ptr()), n.M, n.N, n.K,
                                       stream_of(A)));
    else
        check(gi8_matmul_blockwise(i8(A), i8(B), f32(sa), ld_sa, f32(sb), ld_sb, out.data_ptr(), n.M, n.N, n.K, stream_of(A)));
    return out;
}

at::Tensor int8_matmul_blockwise(const at::Tensor& A, const at::Tensor& B, const at::Tensor& A_scale, const at::Tensor& B_scale)
{
    return blockwise("int8_matmul_blockwise", A, B, A_scale, B_scale, false);
}

at::Tensor int8_matmul_blockwise_f32(const at::Tensor& A, const at::Tensor& B, const at::Tensor& A_scale, const at::Tensor& B_scale)
{
    return blockwise("int8_matmul_blockwise_f32", A, B, A_scale, B_scale, true);
}

// ------------------------------------------------------------------------------------------------ quantisers
void check_activations(const char* name, const at::Tensor& a)
{
    TORCH_CHECK(a.is_cuda(), name, ": input must be a CUDA tensor (the torch reference lives in gemm_int8_b200.quant)");
    TORCH_CHECK(a.dim() == 2, name, ": input must be 2-D [tokens, features]");
    TORCH_CHECK(a.scalar_type() == at::kFloat || a.scalar_type() == at::kBFloat16, name, ": input must be float32 or bfloat16, got ",
                a.scalar_type());
}

enum class Quantiser { kRow, kBlock, kHadamard };

std::tuple<at::Tensor, at::Tensor> quantise(const char* name, const at::Tensor& a, Quantiser kind, int64_t had)
{
    check_activations(name, a);
    const c10::cuda::CUDAGuard guard(a.device());
    const at::Tensor c = a.contiguous();
    const int64_t M = c.size(0), K = c.size(1);
    at::Tensor q = new_tensor({M, K}, at::kChar, c);
    at::Tensor s = kind == Quantiser::kRow ? new_tensor({M}, at::kFloat, c) : new_tensor({M, blocks_of(K)}, at::kFloat, c);
    const int dtype = c.scalar_type() == at::kFloat ? 0 : 1;
    int8_t* qp = static_cast<int8_t*>(q.data_ptr());
    float* sp = static_cast<float*>(s.data_ptr());
    if (kind == Quantiser::kRow) check(gi8_quantize_token(c.data_ptr(), dtype, qp, sp, M, K, stream_of(c)));
    else if (kind == Quantiser::kBlock) check(gi8_quantize_token_block(c.data_ptr(), dtype, qp, sp, M, K, stream_of(c)));
    else check(gi8_hadamard_quantize_token_block(c.data_ptr(), dtype, qp, sp, M, K, had, stream_of(c)));
    return {q, s};
}

std::tuple<at::Tensor, at::Tensor> quantize_token_block(const at::Tensor& a) { return quantise("quantize", a, Quantiser::kBlock, 0); }
std::tuple<at::Tensor, at::Tensor> quantize_token(const at::Tensor& a) { return quantise("quantize", a, Quantiser::kRow, 0); }
std::tuple<at::Tensor, at::Tensor> hadamard_quantize_token_block(const at::Tensor& a, int64_t block)
{
    return quantise("hadamard_quantize", a, Quantiser::kHadamard, block);
}

// ------------------------------------------------------------------------------------------------ linear layer
// Quantiser and product with one call into the library, which launches the second as a programmatic dependent of the
// first; the quantised activations live in one scratch tensor.  hadamard: rotation block, or none.
at::Tensor int8_linear(const at::Tensor& x, const at::Tensor& w, const at::Tensor& w_scale, const std::optional<at::Tensor>& bias, bool blocks,
                       std::optional<int64_t> hadamard)
{
    const char* name = "int8_linear";
    TORCH_CHECK(!hadamard.has_value() || *hadamard > 0, name, ": rotation block ", *hadamard);
    check_activations(name, x);
    TORCH_CHECK(w.device() == x.device(), name, ": the weight must be on ", x.device(), ", got ", w.device());
    TORCH_CHECK(w.scalar_type() == at::kChar && w.dim() == 2 && w.is_contiguous(), name, ": the weight must be a contiguous 2-D int8 tensor");
    TORCH_CHECK(x.size(1) == w.size(1), name, ": x has ", x.size(1), " features, the weight ", w.size(1));
    const int64_t M = x.size(0), N = w.size(0), K = x.size(1);
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor ws;
    int64_t ld = 0;
    if (blocks) {
        check_scale(name, "weight_scale", w_scale, {blocks_of(N), blocks_of(K)}, x.device());
        ws = block_scale(w_scale, ld);
    } else {
        ws = row_scale(name, "weight_scale", w_scale, N, x.device());
    }
    at::Tensor b;
    if (bias.has_value()) {
        TORCH_CHECK(bias->device() == x.device() && bias->dim() == 1 && bias->size(0) == N, name, ": bias must have shape [", N, "] on ", x.device());
        b = bias->to(at::kBFloat16).contiguous();
    }
    const at::Tensor c = x.contiguous();
    at::Tensor out = new_tensor({M, N}, at::kBFloat16, x);
    const int64_t q_bytes = (M * K + 255) / 256 * 256;
    at::Tensor scratch = new_tensor({q_bytes + 4 * M * (blocks ? blocks_of(K) : 1)}, at::kByte, x);
    uint8_t* q = static_cast<uint8_t*>(scratch.data_ptr());
    const int status = gi8_linear(c.data_ptr(), c.scalar_type() == at::kFloat ? 0 : 1, i8(w), f32(ws), ld, b.defined() ? b.data_ptr() : nullptr,
                                  blocks, hadamard.value_or(0), reinterpret_cast<int8_t*>(q), reinterpret_cast<float*>(q + q_bytes), out.data_ptr(), M, N, K,
                                  stream_of(x));
    if (status == GI8_ERR_WORKSPACE && !blocks) {  // a forced variant that the single call does not have
        auto [xq, xs] = quantize_token(c);
        out = int8_matmul_scaled(xq, w, xs, ws);
        return b.defined() ? out + b : out;
    }
    check(status);
    return out;
}

// ------------------------------------------------------------------------------------------------ experts
void check_vector(const char* name, const char* what, const at::Tensor& t, at::ScalarType dtype, at::IntArrayRef shape, const at::Device& device)
{
    TORCH_CHECK(t.device() == device, name, ": ", what, " must be on ", device, ", got ", t.device());
    TORCH_CHECK(t.scalar_type() == dtype, name, ": ", what, " must be ", dtype, ", got ", t.scalar_type());
    TORCH_CHECK(t.sizes() == shape, name, ": ", what, " must have shape ", shape, ", got ", t.sizes());
}

int float_type(const char* name, const char* what, const at::Tensor& t)
{
    TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name, ": ", what, " must be float32 or bfloat16, got ", t.scalar_type());
    return t.scalar_type() == at::kFloat ? 0 : 1;
}

// Contiguous, with a base that vectors of `bytes` can be read from.
at::Tensor aligned(const at::Tensor& t, uintptr_t bytes = 16)
{
    const at::Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % bytes ? c.clone() : c;
}

// What a sum starts from: fp32 or bf16, contiguous; undefined without one.
at::Tensor check_add(const char* name, const std::optional<at::Tensor>& add, at::IntArrayRef shape, const at::Device& device)
{
    if (!add.has_value()) return {};
    float_type(name, "add", *add);
    check_vector(name, "add", *add, add->scalar_type(), shape, device);
    return add->contiguous();
}

std::tuple<at::Tensor, at::Tensor> route_experts(const at::Tensor& logits, const std::optional<at::Tensor>& bias, int64_t top_k, bool sigmoid, int64_t groups,
                                                 int64_t top_groups, bool group_top2, bool renormalize, double scale)
{
    const char* name = "route_experts";
    TORCH_CHECK(logits.is_cuda(), name, ": logits must be a CUDA tensor");
    TORCH_CHECK(logits.dim() == 2, name, ": logits must be 2-D [tokens, experts]");
    const int dtype = float_type(name, "logits", logits);
    TORCH_CHECK(top_k >= 1 && top_k <= logits.size(1), name, ": top_k=", top_k, " of ", logits.size(1), " experts");
    const c10::cuda::CUDAGuard guard(logits.device());
    const at::Tensor l = logits.contiguous();
    at::Tensor b;
    if (bias.has_value()) {
        check_vector(name, "bias", *bias, at::kFloat, {l.size(1)}, l.device());
        b = bias->contiguous();
    }
    at::Tensor weights = new_tensor({l.size(0), top_k}, at::kFloat, l), experts = new_tensor({l.size(0), top_k}, at::kInt, l);
    check(gi8_route_experts(l.data_ptr(), dtype, b.defined() ? f32(b) : nullptr, static_cast<float*>(weights.data_ptr()), static_cast<int32_t*>(experts.data_ptr()),
                            l.size(0), l.size(1), top_k, sigmoid, groups, top_groups, group_top2, renormalize, static_cast<float>(scale), stream_of(l)));
    return {weights, experts};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> group_by_expert(const at::Tensor& experts, int64_t num_experts, int64_t first_expert)
{
    const char* name = "group_by_expert";
    TORCH_CHECK(experts.is_cuda() && experts.scalar_type() == at::kInt && experts.dim() == 2, name, ": experts must be a 2-D int32 CUDA tensor [tokens, top_k]");
    TORCH_CHECK(num_experts >= 1, name, ": num_experts=", num_experts);
    const c10::cuda::CUDAGuard guard(experts.device());
    const at::Tensor e = experts.contiguous();
    at::Tensor offsets = new_tensor({num_experts + 1}, at::kInt, e), slots = new_tensor({e.numel()}, at::kInt, e), places = new_tensor(e.sizes(), at::kInt, e);
    at::Tensor ws;
    const int64_t bytes = gi8_group_by_expert_workspace_bytes(e.numel(), num_experts);
    if (bytes > 0) ws = new_tensor({bytes}, at::kByte, e);
    check(gi8_group_by_expert(static_cast<const int32_t*>(e.data_ptr()), e.numel(), num_experts, first_expert, static_cast<int32_t*>(offsets.data_ptr()),
                              static_cast<int32_t*>(slots.data_ptr()), static_cast<int32_t*>(places.data_ptr()), bytes > 0 ? ws.data_ptr() : nullptr, bytes, stream_of(e)));
    return {offsets, slots, places};
}

at::Tensor int8_matmul_experts(const at::Tensor& x, const at::Tensor& w, const at::Tensor& x_scale, const at::Tensor& w_scale, const at::Tensor& offsets,
                               const std::optional<at::Tensor>& slots, int64_t top_k, bool swiglu)
{
    const char* name = "int8_matmul_experts";
    TORCH_CHECK(x.is_cuda(), name, ": x must be a CUDA tensor");
    TORCH_CHECK(w.device() == x.device(), name, ": the weight must be on ", x.device(), ", got ", w.device());
    TORCH_CHECK(x.scalar_type() == at::kChar && w.scalar_type() == at::kChar, name, ": x and the weight must be int8");
    TORCH_CHECK(x.dim() == 2 && w.dim() == 3, name, ": x must be 2-D [rows, K] and the weight 3-D [experts, N, K]");
    TORCH_CHECK(x.size(1) == w.size(2), name, ": x has ", x.size(1), " features, the weight ", w.size(2));
    TORCH_CHECK(x.is_contiguous() && w.is_contiguous(), name, ": x and the weight must be contiguous");
    TORCH_CHECK(!swiglu || w.size(1) % 2 == 0, name, ": gate and up rows must be the two halves of the weight, got ", w.size(1), " rows");
    TORCH_CHECK(top_k >= 1, name, ": top_k=", top_k);
    const int64_t E = w.size(0), N = swiglu ? w.size(1) / 2 : w.size(1), K = x.size(1);
    const at::Tensor sx = row_scale(name, "x_scale", x_scale, x.size(0), x.device());
    check_scale(name, "w_scale", w_scale, {E, w.size(1)}, x.device());
    check_vector(name, "offsets", offsets, at::kInt, {E + 1}, x.device());
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor sw = w_scale.contiguous(), off = offsets.contiguous();
    at::Tensor sl;
    int64_t rows = x.size(0);
    if (slots.has_value()) {
        check_vector(name, "slots", *slots, at::kInt, {slots->numel()}, x.device());
        sl = slots->contiguous();
        rows = sl.numel();
    }
    at::Tensor out = new_tensor({rows, N}, at::kBFloat16, x);
    // (an empty list of pairs has no data, and is not the absence of one)
    if (rows == 0) return out;
    check(gi8_matmul_experts(i8(x), i8(w), f32(sx), f32(sw), static_cast<const int32_t*>(off.data_ptr()),
                             sl.defined() ? static_cast<const int32_t*>(sl.data_ptr()) : nullptr, top_k, out.data_ptr(), rows, x.size(0), E, N, K, swiglu, stream_of(x)));
    return out;
}

at::Tensor combine_experts(const at::Tensor& y, const at::Tensor& weights, const at::Tensor& places, const std::optional<at::Tensor>& add)
{
    const char* name = "combine_experts";
    TORCH_CHECK(y.is_cuda() && y.scalar_type() == at::kBFloat16 && y.dim() == 2, name, ": y must be a 2-D bfloat16 CUDA tensor [rows, N]");
    TORCH_CHECK(weights.dim() == 2, name, ": weights must be 2-D [tokens, top_k]");
    check_vector(name, "weights", weights, at::kFloat, weights.sizes(), y.device());
    check_vector(name, "places", places, at::kInt, weights.sizes(), y.device());
    const int64_t T = weights.size(0), N = y.size(1);
    const c10::cuda::CUDAGuard guard(y.device());
    const at::Tensor yc = y.contiguous(), wc = weights.contiguous(), pc = places.contiguous();
    const at::Tensor ac = check_add(name, add, {T, N}, y.device());
    at::Tensor out = new_tensor({T, N}, at::kBFloat16, y);
    const int32_t* places_p = static_cast<const int32_t*>(pc.data_ptr());
    if (ac.defined() && ac.scalar_type() == at::kFloat)
        check(gi8_combine_experts_add_f32(yc.data_ptr(), f32(wc), places_p, f32(ac), out.data_ptr(), T, weights.size(1), yc.size(0), N, stream_of(y)));
    else
        check(gi8_combine_experts(yc.data_ptr(), f32(wc), places_p, ac.defined() ? ac.data_ptr() : nullptr, out.data_ptr(), T, weights.size(1), yc.size(0), N, stream_of(y)));
    return out;
}

at::Tensor int8_experts(const at::Tensor& x, const at::Tensor& logits, const std::optional<at::Tensor>& bias, const at::Tensor& gate_up,
                        const at::Tensor& gate_up_scale, const at::Tensor& down, const at::Tensor& down_scale, int64_t top_k, bool sigmoid, int64_t groups,
                        int64_t top_groups, bool group_top2, bool renormalize, double scale, int64_t first_expert, const std::optional<at::Tensor>& add)
{
    const char* name = "int8_experts";
    check_activations(name, x);
    TORCH_CHECK(logits.device() == x.device() && logits.dim() == 2 && logits.size(0) == x.size(0), name, ": logits must have shape [", x.size(0), ", experts] on ", x.device());
    const int logits_dtype = float_type(name, "logits", logits);
    TORCH_CHECK(gate_up.device() == x.device() && gate_up.scalar_type() == at::kChar && gate_up.dim() == 3 && gate_up.is_contiguous() && gate_up.size(1) % 2 == 0 &&
                    gate_up.size(2) == x.size(1),
                name, ": gate_up must be a contiguous int8 tensor [experts, 2 inner, ", x.size(1), "] on ", x.device());
    const int64_t T = x.size(0), H = x.size(1), I = gate_up.size(1) / 2, E = gate_up.size(0);
    check_vector(name, "down", down, at::kChar, {E, H, I}, x.device());
    TORCH_CHECK(down.is_contiguous(), name, ": down must be contiguous");
    check_scale(name, "gate_up_scale", gate_up_scale, {E, 2 * I}, x.device());
    check_scale(name, "down_scale", down_scale, {E, H}, x.device());
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor xc = aligned(x), lc = logits.contiguous(), gs = gate_up_scale.contiguous(), ds = down_scale.contiguous();
    at::Tensor b;
    if (bias.has_value()) {
        check_vector(name, "bias", *bias, at::kFloat, {logits.size(1)}, x.device());
        b = bias->contiguous();
    }
    const at::Tensor ac = check_add(name, add, {T, H}, x.device());
    at::Tensor out = new_tensor({T, H}, at::kBFloat16, x);
    at::Tensor scratch = new_tensor({gi8_experts_scratch_bytes(T, H, I, E, top_k)}, at::kByte, x);
    auto run = [&](auto entry, auto* add_p) {
        check(entry(xc.data_ptr(), xc.scalar_type() == at::kFloat ? 0 : 1, lc.data_ptr(), logits_dtype, b.defined() ? f32(b) : nullptr, i8(gate_up), f32(gs), i8(down), f32(ds),
                    add_p, out.data_ptr(), scratch.data_ptr(), scratch.numel(), T, H, I, logits.size(1), E, first_expert, top_k, sigmoid, groups, top_groups, group_top2,
                    renormalize, static_cast<float>(scale), stream_of(x)));
    };
    if (ac.defined() && ac.scalar_type() == at::kFloat) run(gi8_experts_add_f32, f32(ac));
    else run(gi8_experts, ac.defined() ? ac.data_ptr() : nullptr);
    return out;
}

}  // namespace

TORCH_LIBRARY_IMPL(gemm_int8_CUDA, CUDA, m)
{
    m.impl("int8_matmul", &int8_matmul);
    m.impl("int8_matmul_i32", &int8_matmul_i32);
    m.impl("int8_matmul_scaled", &int8_matmul_scaled);
    m.impl("int8_matmul_blockwise", &int8_matmul_blockwise);
    m.impl("int8_matmul_blockwise_f32", &int8_matmul_blockwise_f32);
    m.impl("quantize_token_block", &quantize_token_block);
    m.impl("quantize_token", &quantize_token);
    m.impl("hadamard_quantize_token_block", &hadamard_quantize_token_block);
    m.impl("int8_linear", &int8_linear);
    m.impl("route_experts", &route_experts);
    m.impl("group_by_expert", &group_by_expert);
    m.impl("int8_matmul_experts", &int8_matmul_experts);
    m.impl("combine_experts", &combine_experts);
    m.impl("int8_experts", &int8_experts);
}
