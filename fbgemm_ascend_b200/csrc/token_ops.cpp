// PyTorch operator registrations of the token tables: lookup of scaled rows with its gradient, 4-bit rows with group
// scales, and products with them.  They have no upstream counterpart, so they live under `tbe_b200`.  Implemented by
// the C ABI of libtbe_b200.so; no host synchronisation and no CPU fallback, like torch_ops.cpp.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <optional>
#include <vector>

#include "tbe_b200.h"

namespace {

using at::Tensor;
using torch::autograd::variable_list;

tbe_b200_stream_t current_stream() { return reinterpret_cast<tbe_b200_stream_t>(c10::cuda::getCurrentCUDAStream().stream()); }

void check_status(int rc, const char* op)
{
    TORCH_CHECK(rc == TBE_B200_OK, op, " failed (status ", rc, "): ", tbe_b200_last_error());
}

void check_cuda(const Tensor& t, const char* op, const char* name)
{
    TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a CUDA tensor; this library has no CPU path");
}

int element_type(const Tensor& t, const char* op, const char* name)
{
    switch (t.scalar_type()) {
        case at::kFloat: return TBE_B200_FP32;
        case at::kHalf: return TBE_B200_FP16;
        case at::kBFloat16: return TBE_B200_BF16;
        default: TORCH_CHECK(false, op, ": ", name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
    }
}

at::ScalarType scalar_type_of(int64_t output_dtype, const char* op)
{
    switch (output_dtype) {
        case TBE_B200_FP32: return at::kFloat;
        case TBE_B200_FP16: return at::kHalf;
        case TBE_B200_BF16: return at::kBFloat16;
        default: TORCH_CHECK(false, op, ": unsupported output_dtype: ", output_dtype, ". Supported: 0(FP32), 1(FP16), 5(BF16)");
    }
}

void check_tokens(const Tensor& tokens, const Tensor& beside, const char* op)
{
    check_cuda(tokens, op, "tokens");
    TORCH_CHECK(tokens.scalar_type() == at::kInt || tokens.scalar_type() == at::kLong, op, ": tokens must be int32 or int64");
    TORCH_CHECK(tokens.device() == beside.device(), op, ": tokens are on ", tokens.device(), ", the rows on ", beside.device());
}

int bits_of(const Tensor& tokens) { return tokens.scalar_type() == at::kInt ? 32 : 64; }

std::vector<int64_t> with_dim(const Tensor& tokens, int64_t D)
{
    std::vector<int64_t> s = tokens.sizes().vec();
    s.push_back(D);
    return s;
}

// A matrix whose rows the kernels can walk: neighbouring elements next to one another, rows at least D apart.
Tensor as_matrix(const Tensor& t)
{
    const bool fine = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
    return fine ? t : t.contiguous();
}

int64_t row_stride(const Tensor& m) { return m.size(0) <= 1 ? m.size(1) : m.stride(0); }

// -1: no padding row.  Negative numbers count from the end, as in torch's own embedding.
int64_t padding_row(std::optional<int64_t> padding_idx, int64_t rows, const char* op)
{
    if (!padding_idx) return -1;
    TORCH_CHECK(*padding_idx >= -rows && *padding_idx < rows, op, ": padding_idx ", *padding_idx, " is no row of a table of ", rows);
    return *padding_idx < 0 ? *padding_idx + rows : *padding_idx;
}

// The operator of that name from the keys below autograd on, for tensors that are wrapped, or made of zeros alone, too.
template <typename Signature, typename... Args>
auto call_below(const c10::TypedOperatorHandle<Signature>& op, Args&&... args)
{
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(std::forward<Args>(args)...);
}

template <typename Signature>
c10::TypedOperatorHandle<Signature> operator_of(const char* name, Signature*)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

// Whether forward-mode differentiation goes through `t`.
bool has_tangent(const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }

bool differentiated(const Tensor& t) { return (at::GradMode::is_enabled() && t.requires_grad()) || has_tangent(t); }

// ---- lookup and gradient ----------------------------------------------------------------------------------------

Tensor token_embedding_cuda(const Tensor& weight, const Tensor& tokens, double scale, std::optional<int64_t> padding_idx,
                            std::optional<int64_t> output_dtype)
{
    const char* op = "token_embedding";
    check_cuda(weight, op, "weight");
    TORCH_CHECK(weight.dim() == 2, op, ": weight must be a matrix [num_embeddings, D]");
    const int wt = element_type(weight, op, "weight");
    check_tokens(tokens, weight, op);
    padding_row(padding_idx, weight.size(0), op);     // of no effect on the lookup itself
    const c10::cuda::CUDAGuard guard(weight.device());
    const Tensor w = as_matrix(weight), t = tokens.contiguous();
    const int64_t D = w.size(1), out_type = output_dtype.value_or(wt);
    Tensor out = at::empty(with_dim(t, D), w.options().dtype(scalar_type_of(out_type, op)));
    check_status(tbe_b200_token_embedding(w.data_ptr(), wt, w.size(0), D, row_stride(w), t.data_ptr(), bits_of(t), t.numel(), static_cast<float>(scale),
                                          out.data_ptr(), static_cast<int32_t>(out_type), D, nullptr, current_stream()), op);
    return out;
}

// Gradient rows [tokens..., D] as a matrix; rows that are all one (stride 0) are read as such.
Tensor grad_rows(const Tensor& grad, const Tensor& tokens, const char* op)
{
    TORCH_CHECK(grad.dim() == tokens.dim() + 1 && grad.sizes().slice(0, tokens.dim()) == tokens.sizes(), op, ": grad must be [", tokens.sizes(),
                ", D], got ", grad.sizes());
    const Tensor g = grad.reshape({tokens.numel(), grad.size(-1)});
    return g.size(1) <= 1 || g.stride(1) == 1 ? g : g.contiguous();
}

void run_grad(const Tensor& grad, const Tensor& tokens, double scale, int64_t padding, bool accumulate, Tensor& into, const char* op)
{
    const int gt = element_type(grad, op, "grad"), wt = element_type(into, op, "grad_weight");
    const Tensor g = grad_rows(grad, tokens, op), t = tokens.contiguous();
    const int64_t n = t.numel(), V = into.size(0), D = into.size(1);
    TORCH_CHECK(g.size(1) == D, op, ": grad has rows of ", g.size(1), " elements, the table of ", D);
    if (V == 0 || D == 0) return;
    const int64_t need = tbe_b200_token_embedding_grad_scratch_bytes(n, V, D);
    TORCH_CHECK(need >= 0, op, ": tokens and rows must be fewer than 2^31, D at most 2^20");
    Tensor scratch;
    if (need > 0) scratch = at::empty({need}, g.options().dtype(at::kByte));    // caching-allocator blocks are 512-byte aligned
    check_status(tbe_b200_token_embedding_grad(n ? g.data_ptr() : nullptr, gt, n > 1 ? g.stride(0) : D, n ? t.data_ptr() : nullptr, bits_of(t), n, V, D,
                                               static_cast<float>(scale), padding, accumulate, into.data_ptr(), wt, row_stride(into),
                                               need ? scratch.data_ptr() : nullptr, need, current_stream()), op);
}

Tensor token_embedding_grad_cuda(const Tensor& grad, const Tensor& tokens, int64_t num_embeddings, double scale, std::optional<int64_t> padding_idx,
                                 std::optional<int64_t> output_dtype)
{
    const char* op = "token_embedding_grad";
    check_cuda(grad, op, "grad");
    check_tokens(tokens, grad, op);
    TORCH_CHECK(num_embeddings >= 0, op, ": num_embeddings must not be negative, got ", num_embeddings);
    TORCH_CHECK(grad.dim() >= 1, op, ": grad must have at least one dimension");
    const int64_t padding = padding_row(padding_idx, num_embeddings, op);
    const int64_t out_type = output_dtype.value_or(element_type(grad, op, "grad"));
    const c10::cuda::CUDAGuard guard(grad.device());
    Tensor out = at::empty({num_embeddings, grad.size(-1)}, grad.options().dtype(scalar_type_of(out_type, op)));
    run_grad(grad, tokens, scale, padding, false, out, op);
    return out;
}

Tensor& token_embedding_grad_into_cuda(Tensor& grad_weight, const Tensor& grad, const Tensor& tokens, double scale, std::optional<int64_t> padding_idx)
{
    const char* op = "token_embedding_grad_";
    check_cuda(grad_weight, op, "grad_weight");
    check_cuda(grad, op, "grad");
    check_tokens(tokens, grad_weight, op);
    TORCH_CHECK(grad.device() == grad_weight.device(), op, ": grad is on ", grad.device(), ", grad_weight on ", grad_weight.device());
    TORCH_CHECK(grad_weight.dim() == 2, op, ": grad_weight must be a matrix [num_embeddings, D]");
    TORCH_CHECK((grad_weight.size(1) <= 1 || grad_weight.stride(1) == 1) && row_stride(grad_weight) >= grad_weight.size(1), op,
                ": rows of grad_weight must lie apart and their elements next to one another");
    at::assert_no_overlap(grad_weight, grad);
    at::assert_no_overlap(grad_weight, tokens);
    const c10::cuda::CUDAGuard guard(grad_weight.device());
    run_grad(grad, tokens, scale, padding_row(padding_idx, grad_weight.size(0), op), true, grad_weight, op);
    if (!grad_weight.is_inference()) grad_weight.unsafeGetTensorImpl()->bump_version();
    return grad_weight;
}

Tensor& token_embedding_grad_into_autograd(Tensor& grad_weight, const Tensor& grad, const Tensor& tokens, double scale, std::optional<int64_t> padding_idx)
{
    TORCH_CHECK(!differentiated(grad_weight) && !differentiated(grad),
                "token_embedding_grad_: adds in place without a graph; call it with detached tensors, or under torch.no_grad() without tangents");
    static const auto op = operator_of("tbe_b200::token_embedding_grad_", token_embedding_grad_into_cuda);
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(grad_weight, grad, tokens, scale, padding_idx);
}

// The lookup is linear in the table and its gradient linear in the rows: each is the other's backward, any number of times, and
// a tangent goes through them as the values do.
Tensor token_embedding_autograd(const Tensor& weight, const Tensor& tokens, double scale, std::optional<int64_t> padding_idx,
                                std::optional<int64_t> output_dtype);
Tensor token_embedding_grad_autograd(const Tensor& grad, const Tensor& tokens, int64_t num_embeddings, double scale,
                                     std::optional<int64_t> padding_idx, std::optional<int64_t> output_dtype);

int64_t type_number(const Tensor& t) { return t.scalar_type() == at::kFloat ? TBE_B200_FP32 : t.scalar_type() == at::kHalf ? TBE_B200_FP16 : TBE_B200_BF16; }

class TokenEmbeddingFunction : public torch::autograd::Function<TokenEmbeddingFunction> {
public:
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& weight, const Tensor& tokens, double scale,
                          std::optional<int64_t> padding_idx, std::optional<int64_t> output_dtype)
    {
        at::AutoDispatchBelowADInplaceOrView g;
        Tensor out = token_embedding_cuda(weight, tokens, scale, padding_idx, output_dtype);
        ctx->save_for_backward({tokens});
        ctx->saved_data["rows"] = weight.size(0);
        ctx->saved_data["type"] = type_number(weight);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding_row(padding_idx, weight.size(0), "token_embedding");
        return out;
    }
    static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grad)
    {
        const int64_t padding = ctx->saved_data["padding"].toInt();
        Tensor g = token_embedding_grad_autograd(grad[0], ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
                                                 ctx->saved_data["scale"].toDouble(), padding < 0 ? std::nullopt : std::make_optional(padding),
                                                 ctx->saved_data["type"].toInt());
        return {g, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

class TokenEmbeddingGradFunction : public torch::autograd::Function<TokenEmbeddingGradFunction> {
public:
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& grad, const Tensor& tokens, int64_t num_embeddings, double scale,
                          std::optional<int64_t> padding_idx, std::optional<int64_t> output_dtype)
    {
        at::AutoDispatchBelowADInplaceOrView g;
        Tensor out = token_embedding_grad_cuda(grad, tokens, num_embeddings, scale, padding_idx, output_dtype);
        ctx->save_for_backward({tokens});
        ctx->saved_data["type"] = type_number(grad);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding_row(padding_idx, num_embeddings, "token_embedding_grad");
        return out;
    }
    // d(out) of a token's row, zeros for the tokens that took no part (padding included: it is made -1 here).
    static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grad)
    {
        Tensor tokens = ctx->get_saved_variables()[0];
        const int64_t padding = ctx->saved_data["padding"].toInt();
        if (padding >= 0) tokens = tokens.masked_fill(tokens.eq(padding), -1);
        Tensor g = token_embedding_autograd(grad[0], tokens, ctx->saved_data["scale"].toDouble(), std::nullopt, ctx->saved_data["type"].toInt());
        return {g, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// A leaf keeps one node that adds up its gradient, bound to the stream it was made on, for as long as any graph over the
// leaf lives.  Captured from another stream, a backward pass would make that stream (the default one, which no capture can
// join) wait for the capture, and the process would not survive it: refused here, before anything is recorded.
void check_capture(const Tensor& t, const char* op)
{
    if (!t.is_leaf() || !t.is_cuda()) return;
    const c10::cuda::CUDAGuard guard(t.device());
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) return;
    const auto stream = node->stream();
    TORCH_CHECK(!stream || *stream != c10::cuda::getDefaultCUDAStream(t.device().index()).unwrap(), op,
                ": a graph made outside this capture, on the default stream, still holds the table's gradient; release it (and the outputs "
                "that hold it) before capturing a training step, or run it on a side stream");
}

Tensor token_embedding_autograd(const Tensor& weight, const Tensor& tokens, double scale, std::optional<int64_t> padding_idx,
                                std::optional<int64_t> output_dtype)
{
    static const auto op = operator_of("tbe_b200::token_embedding", token_embedding_cuda);
    if (has_tangent(weight)) {
        Tensor out = token_embedding_autograd(weight._fw_primal(0), tokens, scale, padding_idx, output_dtype);
        out._set_fw_grad(op.call(weight._fw_grad(0), tokens, scale, padding_idx, type_number(out)), /*level=*/0, /*is_inplace_op=*/false);
        return out;
    }
    if (!(at::GradMode::is_enabled() && weight.requires_grad())) return call_below(op, weight, tokens, scale, padding_idx, output_dtype);
    check_capture(weight, "token_embedding");
    return TokenEmbeddingFunction::apply(weight, tokens, scale, padding_idx, output_dtype);
}

Tensor token_embedding_grad_autograd(const Tensor& grad, const Tensor& tokens, int64_t num_embeddings, double scale,
                                     std::optional<int64_t> padding_idx, std::optional<int64_t> output_dtype)
{
    static const auto op = operator_of("tbe_b200::token_embedding_grad", token_embedding_grad_cuda);
    if (has_tangent(grad)) {
        Tensor out = token_embedding_grad_autograd(grad._fw_primal(0), tokens, num_embeddings, scale, padding_idx, output_dtype);
        out._set_fw_grad(op.call(grad._fw_grad(0), tokens, num_embeddings, scale, padding_idx, type_number(out)), /*level=*/0, /*is_inplace_op=*/false);
        return out;
    }
    if (!(at::GradMode::is_enabled() && grad.requires_grad())) return call_below(op, grad, tokens, num_embeddings, scale, padding_idx, output_dtype);
    check_capture(grad, "token_embedding_grad");
    return TokenEmbeddingGradFunction::apply(grad, tokens, num_embeddings, scale, padding_idx, output_dtype);
}

// ---- 4-bit rows with group scales ----------------------------------------------------------------------------------

int64_t row_bytes_of(int64_t D, int64_t group_size) { return (D / 2 + 4 * ((D + group_size - 1) / group_size) + 15) / 16 * 16; }

void check_group(const char* op, int64_t D, int64_t group_size)
{
    TORCH_CHECK(group_size == 32 || group_size == 64 || group_size == 128 || group_size == 256, op, ": group_size must be 32, 64, 128 or 256, got ", group_size);
    TORCH_CHECK(D > 0 && D <= 0x7fffffff && D % 8 == 0, op, ": rows must have a positive multiple of 8 elements, got ", D);
}

Tensor checked_rows(const Tensor& rows, int64_t D, int64_t group_size, const char* op)
{
    check_cuda(rows, op, "rows");
    TORCH_CHECK(rows.scalar_type() == at::kByte && rows.dim() == 2, op, ": rows must be a uint8 matrix");
    check_group(op, D, group_size);
    TORCH_CHECK(rows.size(1) == row_bytes_of(D, group_size), op, ": rows of ", D, " elements in groups of ", group_size, " have ",
                row_bytes_of(D, group_size), " bytes, got ", rows.size(1));
    return rows.contiguous();
}

void check_no_grad(const Tensor& t, const char* op, const char* name)
{
    TORCH_CHECK(!differentiated(t), op, ": has no gradient; call it with a detached ", name, ", or under torch.no_grad() without tangents");
}

Tensor quantize_to_group_rows(const Tensor& input, int64_t group_size)
{
    const char* op = "quantize_to_group_rows";
    check_cuda(input, op, "input");
    TORCH_CHECK(input.dim() == 2, op, ": input must be a matrix");
    const int it = element_type(input, op, "input");
    check_group(op, input.size(1), group_size);
    const c10::cuda::CUDAGuard guard(input.device());
    const Tensor x = as_matrix(input);
    const int64_t D = x.size(1), bytes = row_bytes_of(D, group_size);
    Tensor out = at::empty({x.size(0), bytes}, x.options().dtype(at::kByte));
    check_status(tbe_b200_quantize_to_group_rows(x.data_ptr(), it, row_stride(x), x.size(0), D, static_cast<int32_t>(group_size), bytes,
                                                 out.data_ptr<uint8_t>(), current_stream()), op);
    return out;
}

Tensor quantize_to_group_rows_autograd(const Tensor& input, int64_t group_size)
{
    check_no_grad(input, "quantize_to_group_rows", "input");
    static const auto op = operator_of("tbe_b200::quantize_to_group_rows", quantize_to_group_rows);
    return call_below(op, input, group_size);
}

Tensor read_group_rows(const Tensor& rows, const Tensor* tokens, int64_t D, int64_t group_size, double scale, int64_t output_dtype, const char* op)
{
    const Tensor r = checked_rows(rows, D, group_size, op);
    const at::ScalarType type = scalar_type_of(output_dtype, op);
    const c10::cuda::CUDAGuard guard(rows.device());
    Tensor t;
    if (tokens) t = tokens->contiguous();
    const int64_t n = tokens ? t.numel() : r.size(0);
    Tensor out = at::empty(tokens ? with_dim(t, D) : std::vector<int64_t>{n, D}, r.options().dtype(type));
    if (n == 0) return out;
    check_status(tbe_b200_group_row_embedding(r.data_ptr<uint8_t>(), r.size(0), r.size(1), D, static_cast<int32_t>(group_size),
                                              tokens ? t.data_ptr() : nullptr, tokens ? bits_of(t) : 64, n, static_cast<float>(scale), out.data_ptr(),
                                              static_cast<int32_t>(output_dtype), D, nullptr, current_stream()), op);
    return out;
}

Tensor group_rows_to_float(const Tensor& rows, int64_t D, int64_t group_size, int64_t output_dtype)
{
    return read_group_rows(rows, nullptr, D, group_size, 1.0, output_dtype, "group_rows_to_float");
}

Tensor group_row_embedding(const Tensor& rows, const Tensor& tokens, int64_t D, int64_t group_size, double scale, int64_t output_dtype)
{
    check_tokens(tokens, rows, "group_row_embedding");
    return read_group_rows(rows, &tokens, D, group_size, scale, output_dtype, "group_row_embedding");
}

Tensor group_row_linear(const Tensor& input, const Tensor& rows, int64_t group_size, const std::optional<Tensor>& bias,
                        std::optional<int64_t> output_dtype)
{
    const char* op = "group_row_linear";
    check_cuda(input, op, "input");
    TORCH_CHECK(input.dim() >= 1, op, ": input must have at least one dimension");
    const int64_t D = input.size(-1);
    const int it = element_type(input, op, "input");
    const Tensor r = checked_rows(rows, D, group_size, op);
    TORCH_CHECK(rows.device() == input.device(), op, ": input is on ", input.device(), ", the rows on ", rows.device());
    const int64_t N = r.size(0), out_type = output_dtype.value_or(it);
    const at::ScalarType type = scalar_type_of(out_type, op);
    const c10::cuda::CUDAGuard guard(input.device());
    Tensor b;
    if (bias && bias->defined()) {
        check_cuda(*bias, op, "bias");
        element_type(*bias, op, "bias");
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N && bias->device() == input.device(), op, ": bias must have one entry per row, on the rows' device");
        b = bias->contiguous();
    }
    Tensor x = as_matrix(input.reshape({D ? input.numel() / D : 0, D}));
    if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 || (x.size(0) > 1 && x.stride(0) % 8)) x = x.clone(at::MemoryFormat::Contiguous);
    const int64_t m = x.size(0);
    std::vector<int64_t> shape = input.sizes().vec();
    shape.back() = N;
    Tensor out = at::empty(shape, x.options().dtype(type));
    if (m == 0 || N == 0) return out;
    const int64_t need = tbe_b200_group_row_linear_scratch_bytes(m, D, static_cast<int32_t>(group_size), it);
    TORCH_CHECK(need >= 0, op, ": at most 2^19 vectors of at most 2^20 elements");
    Tensor scratch;
    if (need > 0) scratch = at::empty({need}, x.options().dtype(at::kByte));
    check_status(tbe_b200_group_row_linear(x.data_ptr(), it, row_stride(x), m, r.data_ptr<uint8_t>(), N, r.size(1), D, static_cast<int32_t>(group_size),
                                           b.defined() ? b.data_ptr() : nullptr, b.defined() ? element_type(b, op, "bias") : 0, out.data_ptr(),
                                           static_cast<int32_t>(out_type), N, nullptr, need > 0 ? scratch.data_ptr() : nullptr, need, current_stream()), op);
    return out;
}

Tensor group_row_linear_autograd(const Tensor& input, const Tensor& rows, int64_t group_size, const std::optional<Tensor>& bias,
                                 std::optional<int64_t> output_dtype)
{
    check_no_grad(input, "group_row_linear", "input");
    if (bias && bias->defined()) check_no_grad(*bias, "group_row_linear", "bias");
    static const auto op = operator_of("tbe_b200::group_row_linear", group_row_linear);
    return call_below(op, input, rows, group_size, bias, output_dtype);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(tbe_b200, m)
{
    m.def("token_embedding(Tensor weight, Tensor tokens, float scale=1.0, int? padding_idx=None, int? output_dtype=None) -> Tensor");
    m.def("token_embedding_grad(Tensor grad, Tensor tokens, int num_embeddings, float scale=1.0, int? padding_idx=None, "
          "int? output_dtype=None) -> Tensor");
    m.def("token_embedding_grad_(Tensor(a!) grad_weight, Tensor grad, Tensor tokens, float scale=1.0, int? padding_idx=None) -> Tensor(a!)");
    m.def("quantize_to_group_rows(Tensor input, int group_size) -> Tensor");
    m.def("group_rows_to_float(Tensor rows, int D, int group_size, int output_dtype=0) -> Tensor");
    m.def("group_row_embedding(Tensor rows, Tensor tokens, int D, int group_size, float scale=1.0, int output_dtype=5) -> Tensor");
    m.def("group_row_linear(Tensor input, Tensor rows, int group_size, Tensor? bias=None, int? output_dtype=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(tbe_b200, CUDA, m)
{
    m.impl("token_embedding", TORCH_FN(token_embedding_cuda));
    m.impl("token_embedding_grad", TORCH_FN(token_embedding_grad_cuda));
    m.impl("token_embedding_grad_", TORCH_FN(token_embedding_grad_into_cuda));
    m.impl("quantize_to_group_rows", TORCH_FN(quantize_to_group_rows));
    m.impl("group_rows_to_float", TORCH_FN(group_rows_to_float));
    m.impl("group_row_embedding", TORCH_FN(group_row_embedding));
    m.impl("group_row_linear", TORCH_FN(group_row_linear));
}

TORCH_LIBRARY_IMPL(tbe_b200, AutogradCUDA, m)
{
    m.impl("token_embedding", TORCH_FN(token_embedding_autograd));
    m.impl("token_embedding_grad", TORCH_FN(token_embedding_grad_autograd));
    m.impl("token_embedding_grad_", TORCH_FN(token_embedding_grad_into_autograd));
    m.impl("quantize_to_group_rows", TORCH_FN(quantize_to_group_rows_autograd));
    m.impl("group_row_linear", TORCH_FN(group_row_linear_autograd));
}
