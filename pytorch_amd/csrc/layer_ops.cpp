// torch.ops.npu.*: what a decoder layer needs between its quantised projections - the residual's addition with the norm behind
// it, and rotary positions.
//
// Named and registered like the operators of npu_ops.cpp (keys CUDA(=HIP) and Meta, no CPU kernel); the C ABI behind them is
// in include/mi355_quant.h.
#include <torch/library.h>

#include "npu_ops.h"

namespace {

int type_code(at::ScalarType t) { return t == at::kBFloat16 ? MI355_DTYPE_BF16 : t == at::kHalf ? MI355_DTYPE_FP16 : MI355_DTYPE_FP32; }
bool act_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

// ---------------------------------------------------------------- npu_add_rms_norm, npu_add_rms_norm_dynamic_quant

using Three = std::tuple<Tensor, Tensor, Tensor>;

void norm_check(const char *op, const Tensor &x1, const Tensor *x2, const Tensor &gamma, double epsilon)
{
    TORCH_CHECK(act_type(x1.scalar_type()), op, ": x1 must be bfloat16 or float16, got ", x1.scalar_type());
    TORCH_CHECK(x1.dim() >= 1 && x1.size(-1) > 0, op, ": x1 must have a last dimension that is not empty, got ", x1.sizes());
    if (x2) {
        TORCH_CHECK(x2->scalar_type() == x1.scalar_type(), op, ": x1 and x2 must have the same dtype, got ", x1.scalar_type(), " and ", x2->scalar_type());
        TORCH_CHECK(x2->sizes() == x1.sizes(), op, ": x1 and x2 must have the same shape, got ", x1.sizes(), " and ", x2->sizes());
    }
    TORCH_CHECK(gamma.scalar_type() == x1.scalar_type() || gamma.scalar_type() == at::kFloat, op, ": gamma must be float32 or have the dtype of x1, got ",
                gamma.scalar_type());
    TORCH_CHECK(gamma.dim() == 1 && gamma.size(0) == x1.size(-1), op, ": gamma must have shape [", x1.size(-1), "], got ", gamma.sizes());
    TORCH_CHECK(epsilon >= 0, op, ": epsilon must not be negative, got ", epsilon);
}

// y, rstd [..., 1] or scale [...], and x1 + x2 (without x2: no elements)
Three norm_alloc(Alloc how, const Tensor &x1, const Tensor *x2, bool int8)
{
    at::DimVector stat(x1.sizes());
    if (int8) stat.pop_back();
    else stat.back() = 1;
    return {new_empty(how, x1, x1.sizes(), int8 ? at::kChar : x1.scalar_type()), new_empty(how, x1, stat, at::kFloat),
            new_empty(how, x1, x2 ? x1.sizes() : at::IntArrayRef{0}, x1.scalar_type())};
}

// Rows with one stride between them: a two-dimensional view with unit inner stride as it is, else packed
Tensor as_rows(const Tensor &t, int64_t &stride)
{
    const int64_t cols = t.size(-1);
    stride = cols;
    if (t.dim() == 2 && (t.stride(1) == 1 || cols == 1) && t.stride(0) >= cols) {
        stride = t.stride(0);
        return t;
    }
    return packed(t);
}

Three norm_hip(const char *op, const Tensor &x1, const optional<Tensor> &x2_, const Tensor &gamma, double epsilon, bool int8)
{
    const Tensor *x2 = opt(x2_);
    norm_check(op, x1, x2, gamma, epsilon);
    check_same_device(op, {&x1, x2, &gamma});
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x1.device());
    Three out = norm_alloc(kLaunch, x1, x2, int8);
    auto &[y, stat, x] = out;
    if (x1.numel() == 0) return out;
    int64_t s1, s2 = 0;
    const Tensor a = as_rows(x1, s1), b = x2 ? as_rows(*x2, s2) : Tensor(), g = packed(gamma);
    const int64_t cols = x1.size(-1), rows = x1.numel() / cols;
    const void *const pb = x2 ? b.data_ptr() : nullptr;
    void *const px = x2 ? x.data_ptr() : nullptr;
    const int type = type_code(x1.scalar_type()), gamma_type = type_code(g.scalar_type());
    check_status(int8 ? mi355_add_rms_norm_dynamic_quant(a.data_ptr(), pb, type, g.data_ptr(), gamma_type, y.data_ptr<int8_t>(), stat.data_ptr<float>(),
                                                         px, rows, cols, s1, s2, (float)epsilon, stream_of(x1))
                      : mi355_add_rms_norm(a.data_ptr(), pb, type, g.data_ptr(), gamma_type, y.data_ptr(), stat.data_ptr<float>(), px, rows, cols, s1, s2,
                                           (float)epsilon, stream_of(x1)),
                 op);
    return out;
}

Three norm_meta(const char *op, const Tensor &x1, const optional<Tensor> &x2, const Tensor &gamma, double epsilon, bool int8)
{
    norm_check(op, x1, opt(x2), gamma, epsilon);
    return norm_alloc(kMeta, x1, opt(x2), int8);
}

Three add_rms_norm_hip(const Tensor &x1, const optional<Tensor> &x2, const Tensor &gamma, double epsilon)
{
    return norm_hip("npu_add_rms_norm", x1, x2, gamma, epsilon, false);
}
Three add_rms_norm_meta(const Tensor &x1, const optional<Tensor> &x2, const Tensor &gamma, double epsilon)
{
    return norm_meta("npu_add_rms_norm", x1, x2, gamma, epsilon, false);
}
Three add_rms_norm_dynamic_quant_hip(const Tensor &x1, const optional<Tensor> &x2, const Tensor &gamma, double epsilon)
{
    return norm_hip("npu_add_rms_norm_dynamic_quant", x1, x2, gamma, epsilon, true);
}
Three add_rms_norm_dynamic_quant_meta(const Tensor &x1, const optional<Tensor> &x2, const Tensor &gamma, double epsilon)
{
    return norm_meta("npu_add_rms_norm_dynamic_quant", x1, x2, gamma, epsilon, true);
}

// ---------------------------------------------------------------- npu_mrope

using Two = std::tuple<Tensor, Tensor>;

void mrope_check(const Tensor &positions, const Tensor &query, const Tensor &key, const Tensor &table, int64_t head_size,
                 at::OptionalIntArrayRef sections, c10::string_view mode)
{
    const char *op = "npu_mrope";
    TORCH_CHECK(head_size > 0 && head_size <= 65536, op, ": head_size must be between 1 and 65536, got ", head_size);
    TORCH_CHECK(act_type(query.scalar_type()) && key.scalar_type() == query.scalar_type(), op,
                ": query and key must both be bfloat16 or both float16, got ", query.scalar_type(), " and ", key.scalar_type());
    const int64_t tokens = query.dim() >= 1 ? query.size(0) : 0;
    for (const Tensor *t : {&query, &key}) {
        const char *name = t == &query ? "query" : "key";
        TORCH_CHECK((t->dim() == 2 && t->size(1) % head_size == 0) || (t->dim() == 3 && t->size(2) == head_size), op, ": ", name,
                    " must have shape [tokens, heads * ", head_size, "] or [tokens, heads, ", head_size, "], got ", t->sizes());
        TORCH_CHECK(t->size(0) == tokens, op, ": query and key must have the same number of tokens, got ", tokens, " and ", t->size(0));
        TORCH_CHECK((t->dim() == 2 ? t->size(1) / head_size : t->size(1)) <= 65535, op, ": at most 65535 heads, got ", t->sizes());
    }
    TORCH_CHECK(table.scalar_type() == query.scalar_type() || table.scalar_type() == at::kFloat, op,
                ": cos_sin_cache must be float32 or have the dtype of query, got ", table.scalar_type());
    TORCH_CHECK(table.dim() == 2 && table.size(1) >= 2 && table.size(1) % 2 == 0 && table.size(1) <= head_size, op,
                ": cos_sin_cache must have shape [positions, rotary_dim] with an even rotary_dim of at most ", head_size, ", got ", table.sizes());
    TORCH_CHECK(mode == "half" || mode == "interleave", op, ": rotary_mode must be 'half' or 'interleave', got '", mode, "'");
    TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, op, ": positions must be int32 or int64, got ",
                positions.scalar_type());
    if (!sections.has_value()) {
        TORCH_CHECK(positions.dim() == 1 && positions.size(0) == tokens, op, ": positions must have shape [", tokens, "], got ", positions.sizes(),
                    " (with several axes mrope_section says how the frequencies are shared)");
        return;
    }
    const int64_t axes = (int64_t)sections->size();
    TORCH_CHECK(axes >= 1 && axes <= 4, op, ": mrope_section must name between 1 and 4 axes, got ", axes);
    int64_t sum = 0;
    for (const int64_t n : *sections) {
        TORCH_CHECK(n >= 0 && n <= head_size, op, ": a section of mrope_section must be between 0 and half of rotary_dim, got ", n);
        sum += n;
    }
    TORCH_CHECK(sum == table.size(1) / 2, op, ": mrope_section must add up to half of rotary_dim, ", table.size(1) / 2, ", got ", sum);
    TORCH_CHECK(positions.dim() == 2 && positions.size(0) == axes && positions.size(1) == tokens, op, ": positions must have shape [", axes, ", ", tokens,
                "], got ", positions.sizes());
}

Two mrope_alloc(Alloc how, const Tensor &query, const Tensor &key)
{
    return {new_empty(how, query, query.sizes(), query.scalar_type()), new_empty(how, key, key.sizes(), key.scalar_type())};
}

Two mrope_hip(const Tensor &positions, const Tensor &query, const Tensor &key, const Tensor &cos_sin_cache, int64_t head_size,
              at::OptionalIntArrayRef mrope_section, c10::string_view rotary_mode)
{
    const char *op = "npu_mrope";
    mrope_check(positions, query, key, cos_sin_cache, head_size, mrope_section, rotary_mode);
    check_same_device(op, {&positions, &query, &key, &cos_sin_cache});
    c10::hip::HIPGuardMasqueradingAsCUDA guard(query.device());
    Two out = mrope_alloc(kLaunch, query, key);
    const int64_t tokens = query.size(0);
    if (tokens == 0 || query.numel() + key.numel() == 0) return out;
    const auto inner = [](const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous(); };
    const Tensor q = inner(query), k = inner(key), table = inner(cos_sin_cache);
    const auto heads = [&](const Tensor &t) { return t.dim() == 2 ? t.size(1) / head_size : t.size(1); };
    const int64_t q_stride[2] = {q.stride(0), q.dim() == 2 ? head_size : q.stride(1)}, k_stride[2] = {k.stride(0), k.dim() == 2 ? head_size : k.stride(1)};
    const int64_t axes = mrope_section.has_value() ? (int64_t)mrope_section->size() : 1;
    check_status(mi355_mrope(positions.data_ptr(), positions.scalar_type() == at::kLong ? MI355_DTYPE_INT64 : MI355_DTYPE_INT32,
                             positions.dim() == 2 ? positions.stride(0) : 0, positions.stride(-1), axes, axes > 1 ? mrope_section->data() : nullptr,
                             q.data_ptr(), q_stride, heads(q), k.data_ptr(), k_stride, heads(k), type_code(q.scalar_type()), table.data_ptr(),
                             type_code(table.scalar_type()), table.stride(0), table.size(0), tokens, head_size, table.size(1), rotary_mode == "interleave",
                             std::get<0>(out).data_ptr(), std::get<1>(out).data_ptr(), stream_of(query)),
                 op);
    return out;
}

Two mrope_meta(const Tensor &positions, const Tensor &query, const Tensor &key, const Tensor &cos_sin_cache, int64_t head_size,
               at::OptionalIntArrayRef mrope_section, c10::string_view rotary_mode)
{
    mrope_check(positions, query, key, cos_sin_cache, head_size, mrope_section, rotary_mode);
    return mrope_alloc(kMeta, query, key);
}

} // namespace

TORCH_LIBRARY_FRAGMENT(npu, m)
{
    m.def("npu_add_rms_norm(Tensor x1, Tensor? x2, Tensor gamma, float epsilon=1e-06) -> (Tensor, Tensor, Tensor)");
    m.def("npu_add_rms_norm_dynamic_quant(Tensor x1, Tensor? x2, Tensor gamma, *, float epsilon=1e-06) -> (Tensor, Tensor, Tensor)");
    m.def("npu_mrope(Tensor positions, Tensor query, Tensor key, Tensor cos_sin_cache, int head_size, *, int[]? mrope_section=None, "
          "str rotary_mode='half') -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(npu, CUDA, m)
{
    m.impl("npu_add_rms_norm", TORCH_FN(add_rms_norm_hip));
    m.impl("npu_add_rms_norm_dynamic_quant", TORCH_FN(add_rms_norm_dynamic_quant_hip));
    m.impl("npu_mrope", TORCH_FN(mrope_hip));
}

TORCH_LIBRARY_IMPL(npu, Meta, m)
{
    m.impl("npu_add_rms_norm", TORCH_FN(add_rms_norm_meta));
    m.impl("npu_add_rms_norm_dynamic_quant", TORCH_FN(add_rms_norm_dynamic_quant_meta));
    m.impl("npu_mrope", TORCH_FN(mrope_meta));
}
