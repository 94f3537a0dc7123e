// torch.ops.npu.npu_paged_*: the paged key-value cache's operators.
//
// Named and registered like the operators of npu_ops.cpp (keys CUDA(=HIP) and Meta, no CPU kernel); the C ABI behind them is
// the paged section of include/mi355_quant.h.
#include <ATen/MemoryOverlap.h>
#include <torch/library.h>

#include <cmath>

#include "npu_ops.h"

namespace {

int act_code(at::ScalarType t) { return t == at::kBFloat16 ? MI355_DTYPE_BF16 : MI355_DTYPE_FP16; }
bool act_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool index_type(at::ScalarType t) { return t == at::kInt || t == at::kLong; }
bool inner_contiguous(const Tensor &t) { return t.stride(-1) == 1 || t.size(-1) <= 1; }

// Scales and offsets of a cache of codes; none for 16 bits, no offsets for int8.
struct Params {
    const Tensor *ks, *vs, *ko, *vo;
    Params(const optional<Tensor> &key_scale, const optional<Tensor> &value_scale, const optional<Tensor> &key_offset, const optional<Tensor> &value_offset)
        : ks(opt(key_scale)), vs(opt(value_scale)), ko(opt(key_offset)), vo(opt(value_offset))
    {
    }
};

bool int4(const Tensor &cache) { return cache.scalar_type() == at::kInt; }               // words of eight codes
bool codes(const Tensor &cache) { return cache.scalar_type() == at::kChar || int4(cache); }
int64_t head_dim(const Tensor &cache) { return int4(cache) ? cache.size(3) * 8 : cache.size(3); }

// Shapes, types and strides of a cache; `written`: its tensors are updated in place.
void check_cache(const char *op, const Tensor &k, const Tensor &v, const Params &p, bool written)
{
    TORCH_CHECK(k.dim() == 4, op, ": key_cache must have shape [num_blocks, block_size, kv_heads, head_dim], got ", k.sizes());
    TORCH_CHECK(v.sizes() == k.sizes(), op, ": key_cache and value_cache must have the same shape, got ", k.sizes(), " and ", v.sizes());
    TORCH_CHECK(act_type(k.scalar_type()) || codes(k), op, ": the cache must be bfloat16, float16 or int8, or int32 words of eight 4-bit codes, got ",
                k.scalar_type());
    TORCH_CHECK(v.scalar_type() == k.scalar_type(), op, ": key_cache and value_cache must have the same dtype, got ", k.scalar_type(), " and ",
                v.scalar_type());
    TORCH_CHECK(k.numel() > 0, op, ": the cache is empty: ", k.sizes());
    TORCH_CHECK(k.size(0) <= 0x7fffffff / k.size(1), op, ": num_blocks * block_size must be below 2^31");
    TORCH_CHECK(inner_contiguous(k) && inner_contiguous(v), op, ": the last dimension of key_cache and value_cache must be contiguous");
    const auto check = [&](const Tensor *t, const char *names) {
        TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 3 && t->sizes() == k.sizes().slice(0, 3), op, ": ", names, " must be float32 of shape ",
                    k.sizes().slice(0, 3), ", got ", t->scalar_type(), " ", t->sizes());
    };
    if (codes(k)) {
        if (int4(k)) TORCH_CHECK(p.ks && p.vs && p.ko && p.vo, op, ": a 4-bit cache needs key_scale, value_scale, key_offset and value_offset");
        TORCH_CHECK(p.ks && p.vs, op, ": an int8 cache needs key_scale and value_scale");
        for (const Tensor *t : {p.ks, p.vs}) check(t, "key_scale and value_scale");
    } else {
        TORCH_CHECK(!p.ks && !p.vs, op, ": key_scale and value_scale belong to an int8 cache or a 4-bit one, this one is ", k.scalar_type());
    }
    if (int4(k))
        for (const Tensor *t : {p.ko, p.vo}) check(t, "key_offset and value_offset");
    else
        TORCH_CHECK(!p.ko && !p.vo, op, ": key_offset and value_offset belong to a 4-bit cache, this one is ", k.scalar_type());
    if (!written) return;
    for (const Tensor *t : {&k, &v, p.ks, p.vs, p.ko, p.vo})
        TORCH_CHECK(!t || at::has_internal_overlap(*t) != at::MemOverlap::Yes, op, ": elements of the cache share memory; it cannot be written");
}

mi355_paged_cache describe(const Tensor &k, const Tensor &v, const Params &p)
{
    const auto data = [](const Tensor *t) { return t ? t->data_ptr<float>() : nullptr; };
    mi355_paged_cache c = {};
    c.key = k.data_ptr();
    c.value = v.data_ptr();
    c.key_scale = data(p.ks);
    c.value_scale = data(p.vs);
    c.key_offset = data(p.ko);
    c.value_offset = data(p.vo);
    c.dtype = int4(k) ? MI355_DTYPE_INT4 : codes(k) ? MI355_DTYPE_INT8 : act_code(k.scalar_type());
    c.num_blocks = k.size(0);
    c.block_size = k.size(1);
    c.kv_heads = k.size(2);
    c.head_dim = head_dim(k);
    for (int i = 0; i < 3; i++) {
        c.key_stride[i] = k.stride(i);
        c.value_stride[i] = v.stride(i);
        c.key_scale_stride[i] = p.ks ? p.ks->stride(i) : 0;
        c.value_scale_stride[i] = p.vs ? p.vs->stride(i) : 0;
        c.key_offset_stride[i] = p.ko ? p.ko->stride(i) : 0;
        c.value_offset_stride[i] = p.vo ? p.vo->stride(i) : 0;
    }
    return c;
}

void check_slots(const char *op, const Tensor &slots)
{
    TORCH_CHECK(index_type(slots.scalar_type()) && slots.dim() == 1, op, ": slots must be int32 or int64 of shape [tokens], got ", slots.scalar_type(),
                " ", slots.sizes());
}

// the table and the lengths as the kernels take them: int32, what does not fit still beyond every block and length
Tensor as_int(const Tensor &t)
{
    Tensor i = t.scalar_type() == at::kInt ? t : t.clamp(-1, 0x7fffffff).to(at::kInt);
    return i.dim() == 1 ? packed(i) : inner_contiguous(i) ? i : i.contiguous();
}

// (the number of positions that the table can hold)
int64_t check_table(const char *op, const Tensor &k, const Tensor &table, const Tensor &lens, int64_t batch)
{
    TORCH_CHECK(index_type(table.scalar_type()) && table.dim() == 2 && (batch < 0 || table.size(0) == batch), op,
                ": block_table must be int32 or int64 of shape [batch, blocks]", ", got ", table.scalar_type(), " ", table.sizes());
    TORCH_CHECK(index_type(lens.scalar_type()) && lens.dim() == 1 && lens.size(0) == table.size(0), op,
                ": context_lens must be int32 or int64 of shape [", table.size(0), "], got ", lens.scalar_type(), " ", lens.sizes());
    TORCH_CHECK(table.size(1) <= 0x7fffff00 / k.size(1), op, ": a block_table of ", table.size(1), " blocks holds more than 2^31 positions");
    return table.size(1) * k.size(1);
}

// ---------------------------------------------------------------- npu_paged_cache_write

void write_check(const Tensor &key, const Tensor &value, const Tensor &kc, const Tensor &vc, const Tensor &slots, const Params &p)
{
    const char *op = "npu_paged_cache_write";
    check_cache(op, kc, vc, p, true);
    check_slots(op, slots);
    TORCH_CHECK(act_type(key.scalar_type()) && value.scalar_type() == key.scalar_type(), op,
                ": key and value must both be bfloat16 or both float16, got ", key.scalar_type(), " and ", value.scalar_type());
    TORCH_CHECK(codes(kc) || kc.scalar_type() == key.scalar_type(), op, ": the cache is ", kc.scalar_type(), ", key and value are ",
                key.scalar_type());
    TORCH_CHECK(key.dim() == 3 && key.size(0) == slots.size(0) && key.size(1) == kc.size(2) && key.size(2) == head_dim(kc), op,
                ": key must have shape [", slots.size(0), ", ", kc.size(2), ", ", head_dim(kc), "], got ", key.sizes());
    TORCH_CHECK(value.sizes() == key.sizes(), op, ": key and value must have the same shape, got ", key.sizes(), " and ", value.sizes());
}

void write_meta(const Tensor &key, const Tensor &value, const Tensor &key_cache, const Tensor &value_cache, const Tensor &slots,
                const optional<Tensor> &key_scale, const optional<Tensor> &value_scale, const optional<Tensor> &key_offset, const optional<Tensor> &value_offset)
{
    write_check(key, value, key_cache, value_cache, slots, {key_scale, value_scale, key_offset, value_offset});
}

void write_hip(const Tensor &key, const Tensor &value, const Tensor &key_cache, const Tensor &value_cache, const Tensor &slots,
               const optional<Tensor> &key_scale, const optional<Tensor> &value_scale, const optional<Tensor> &key_offset, const optional<Tensor> &value_offset)
{
    const Params p(key_scale, value_scale, key_offset, value_offset);
    write_check(key, value, key_cache, value_cache, slots, p);
    check_same_device("npu_paged_cache_write", {&key, &value, &key_cache, &value_cache, &slots, p.ks, p.vs, p.ko, p.vo});
    if (slots.size(0) == 0) return;
    c10::hip::HIPGuardMasqueradingAsCUDA guard(key_cache.device());
    const Tensor k = inner_contiguous(key) ? key : key.contiguous(), v = inner_contiguous(value) ? value : value.contiguous(), at = packed(slots);
    const mi355_paged_cache c = describe(key_cache, value_cache, p);
    const int64_t k_stride[2] = {k.stride(0), k.stride(1)}, v_stride[2] = {v.stride(0), v.stride(1)};
    check_status(mi355_paged_cache_write(&c, k.data_ptr(), k_stride, v.data_ptr(), v_stride, act_code(k.scalar_type()), at.data_ptr(),
                                         at.scalar_type() == at::kLong ? MI355_DTYPE_INT64 : MI355_DTYPE_INT32, at.size(0), stream_of(key_cache)),
                 "npu_paged_cache_write");
}

// ---------------------------------------------------------------- npu_paged_cache_read

std::tuple<Tensor, Tensor> read_alloc(Alloc how, const Tensor &kc, const Tensor &vc, const Tensor &slots, const Params &p,
                                      optional<at::ScalarType> dtype)
{
    const char *op = "npu_paged_cache_read";
    check_cache(op, kc, vc, p, false);
    check_slots(op, slots);
    const at::ScalarType type = dtype.has_value() ? *dtype : codes(kc) ? at::kBFloat16 : kc.scalar_type();
    TORCH_CHECK(act_type(type) && (codes(kc) || kc.scalar_type() == type), op, ": dtype must be ",
                codes(kc) ? "torch.bfloat16 or torch.float16" : "that of the cache", ", got ", type);
    const int64_t shape[3] = {slots.size(0), kc.size(2), head_dim(kc)};
    return {new_empty(how, kc, shape, type), new_empty(how, kc, shape, type)};
}

std::tuple<Tensor, Tensor> read_meta(const Tensor &key_cache, const Tensor &value_cache, const Tensor &slots, const optional<Tensor> &key_scale,
                                     const optional<Tensor> &value_scale, optional<at::ScalarType> dtype, const optional<Tensor> &key_offset, const optional<Tensor> &value_offset)
{
    return read_alloc(kMeta, key_cache, value_cache, slots, {key_scale, value_scale, key_offset, value_offset}, dtype);
}

std::tuple<Tensor, Tensor> read_hip(const Tensor &key_cache, const Tensor &value_cache, const Tensor &slots, const optional<Tensor> &key_scale,
                                    const optional<Tensor> &value_scale, optional<at::ScalarType> dtype, const optional<Tensor> &key_offset, const optional<Tensor> &value_offset)
{
    const Params p(key_scale, value_scale, key_offset, value_offset);
    check_same_device("npu_paged_cache_read", {&key_cache, &value_cache, &slots, p.ks, p.vs, p.ko, p.vo});
    c10::hip::HIPGuardMasqueradingAsCUDA guard(key_cache.device());
    auto [k, v] = read_alloc(kLaunch, key_cache, value_cache, slots, p, dtype);
    if (slots.size(0) == 0) return {k, v};
    const Tensor at = packed(slots);
    const mi355_paged_cache c = describe(key_cache, value_cache, p);
    const int64_t stride[2] = {k.stride(0), k.stride(1)};
    check_status(mi355_paged_cache_read(&c, k.data_ptr(), stride, v.data_ptr(), stride, act_code(k.scalar_type()), at.data_ptr(),
                                        at.scalar_type() == at::kLong ? MI355_DTYPE_INT64 : MI355_DTYPE_INT32, at.size(0), stream_of(key_cache)),
                 "npu_paged_cache_read");
    return {k, v};
}

// ---------------------------------------------------------------- npu_paged_decode_attention

std::tuple<Tensor, Tensor> attention_alloc(Alloc how, const Tensor &q, const Tensor &kc, const Tensor &vc, const Tensor &table, const Tensor &lens,
                                           const Params &p, const Tensor *mask, const Tensor *sums, bool lse)
{
    const char *op = "npu_paged_decode_attention";
    check_cache(op, kc, vc, p, false);
    TORCH_CHECK(act_type(q.scalar_type()), op, ": query must be bfloat16 or float16, got ", q.scalar_type());
    TORCH_CHECK(codes(kc) || kc.scalar_type() == q.scalar_type(), op, ": the cache is ", kc.scalar_type(), ", query is ",
                q.scalar_type());
    TORCH_CHECK(q.dim() == 3 && q.size(2) == head_dim(kc), op, ": query must have shape [batch, heads, ", head_dim(kc), "], got ", q.sizes());
    TORCH_CHECK(q.size(1) > 0 && q.size(1) % kc.size(2) == 0, op, ": the ", q.size(1), " heads of query are not a multiple of the cache's ", kc.size(2));
    TORCH_CHECK(q.size(2) <= 256, op, ": head_dim must be at most 256, got ", q.size(2));
    TORCH_CHECK(q.size(1) <= 65535, op, ": at most 65535 heads, got ", q.size(1));
    const int64_t capacity = check_table(op, kc, table, lens, q.size(0));
    if (mask)
        TORCH_CHECK(mask->scalar_type() == at::kBool && mask->dim() == 2 && mask->size(0) == q.size(0) && mask->size(1) == capacity, op,
                    ": atten_mask must be bool of shape [", q.size(0), ", ", capacity, "], got ", mask->scalar_type(), " ", mask->sizes());
    if (sums) {
        TORCH_CHECK(sums->scalar_type() == at::kFloat && sums->dim() == 3 && sums->size(0) == q.size(0) && sums->size(1) == kc.size(2) &&
                        sums->size(2) == capacity,
                    op, ": attn_sums must be float32 of shape [", q.size(0), ", ", kc.size(2), ", ", capacity, "], got ", sums->scalar_type(), " ",
                    sums->sizes());
        TORCH_CHECK(inner_contiguous(*sums), op, ": the last dimension of attn_sums must be contiguous");
        TORCH_CHECK(at::has_internal_overlap(*sums) != at::MemOverlap::Yes, op, ": elements of attn_sums share memory; it cannot be updated");
    }
    return {new_empty(how, q, q.sizes(), q.scalar_type()), new_empty(how, q, lse ? q.sizes().slice(0, 2) : at::IntArrayRef{0}, at::kFloat)};
}

std::tuple<Tensor, Tensor> attention_meta(const Tensor &query, const Tensor &key_cache, const Tensor &value_cache, const Tensor &block_table,
                                          const Tensor &context_lens, const optional<Tensor> &key_scale, const optional<Tensor> &value_scale,
                                          optional<double>, const optional<Tensor> &atten_mask, const optional<Tensor> &attn_sums, bool softmax_lse,
                                          const optional<Tensor> &key_offset, const optional<Tensor> &value_offset)
{
    return attention_alloc(kMeta, query, key_cache, value_cache, block_table, context_lens, {key_scale, value_scale, key_offset, value_offset},
                           opt(atten_mask), opt(attn_sums), softmax_lse);
}

std::tuple<Tensor, Tensor> attention_hip(const Tensor &query, const Tensor &key_cache, const Tensor &value_cache, const Tensor &block_table,
                                         const Tensor &context_lens, const optional<Tensor> &key_scale, const optional<Tensor> &value_scale,
                                         optional<double> scale_value, const optional<Tensor> &atten_mask, const optional<Tensor> &attn_sums,
                                         bool softmax_lse, const optional<Tensor> &key_offset, const optional<Tensor> &value_offset)
{
    const char *op = "npu_paged_decode_attention";
    const Params p(key_scale, value_scale, key_offset, value_offset);
    const Tensor *mask = opt(atten_mask), *sums = opt(attn_sums);
    check_same_device(op, {&query, &key_cache, &value_cache, &block_table, &context_lens, p.ks, p.vs, p.ko, p.vo, mask, sums});
    c10::hip::HIPGuardMasqueradingAsCUDA guard(query.device());
    auto [out, lse] = attention_alloc(kLaunch, query, key_cache, value_cache, block_table, context_lens, p, mask, sums, softmax_lse);
    const int64_t batch = query.size(0), heads = query.size(1), kv_heads = key_cache.size(2);
    if (batch == 0) return {out, lse};
    const Tensor q = inner_contiguous(query) ? query : query.contiguous(), table = as_int(block_table), lens = as_int(context_lens);
    const Tensor hidden = !mask || inner_contiguous(*mask) ? (mask ? *mask : Tensor()) : mask->contiguous();
    const mi355_paged_cache c = describe(key_cache, value_cache, p);
    const size_t bytes = mi355_paged_decode_attention_workspace(batch, heads, kv_heads, q.size(2), table.size(1), key_cache.size(1), sums != nullptr);
    const Workspace ws = mi355_ops::workspace(q, bytes, sums != nullptr);
    const double scale = scale_value.has_value() ? *scale_value : 1.0 / std::sqrt((double)q.size(2));
    check_status(mi355_paged_decode_attention(&c, q.data_ptr(), act_code(q.scalar_type()), q.stride(0), q.stride(1), out.data_ptr(),
                                              softmax_lse ? lse.data_ptr<float>() : nullptr, batch, heads, table.data_ptr<int32_t>(), table.stride(0),
                                              table.size(1), lens.data_ptr<int32_t>(), (float)scale,
                                              mask ? reinterpret_cast<const uint8_t *>(hidden.data_ptr()) : nullptr, mask ? hidden.stride(0) : 0,
                                              sums ? sums->data_ptr<float>() : nullptr, sums ? sums->stride(0) : 0, sums ? sums->stride(1) : 0,
                                              ws.memory.data_ptr(), bytes, stream_of(query)),
                 op);
    return {out, lse};
}

// ---------------------------------------------------------------- npu_paged_cache_evict

std::tuple<Tensor, Tensor, Tensor> evict_alloc(Alloc how, const Tensor &kc, const Tensor &vc, const Tensor &table, const Tensor &lens,
                                               const Tensor &sums, const Tensor &positions, int64_t keep, int64_t recent, const Params &p)
{
    const char *op = "npu_paged_cache_evict";
    check_cache(op, kc, vc, p, true);
    const int64_t capacity = check_table(op, kc, table, lens, -1);
    const int64_t shape[3] = {table.size(0), kc.size(2), capacity};
    TORCH_CHECK(sums.scalar_type() == at::kFloat && sums.sizes() == at::IntArrayRef(shape), op, ": attn_sums must be float32 of shape ",
                at::IntArrayRef(shape), ", got ", sums.scalar_type(), " ", sums.sizes());
    TORCH_CHECK(positions.scalar_type() == at::kInt && positions.sizes() == at::IntArrayRef(shape), op, ": positions must be int32 of shape ",
                at::IntArrayRef(shape), ", got ", positions.scalar_type(), " ", positions.sizes());
    TORCH_CHECK(keep >= 0 && recent >= 0 && recent <= keep, op, ": keep and recent must satisfy 0 <= recent <= keep, got keep ", keep, ", recent ", recent);
    return {new_empty(how, kc, {table.size(0)}, at::kInt), new_empty(how, kc, shape, at::kFloat), new_empty(how, kc, shape, at::kInt)};
}

std::tuple<Tensor, Tensor, Tensor> evict_meta(const Tensor &key_cache, const Tensor &value_cache, const Tensor &block_table, const Tensor &context_lens,
                                              const Tensor &attn_sums, const Tensor &positions, int64_t keep, int64_t recent,
                                              const optional<Tensor> &key_scale, const optional<Tensor> &value_scale,
                                              const optional<Tensor> &key_offset, const optional<Tensor> &value_offset)
{
    return evict_alloc(kMeta, key_cache, value_cache, block_table, context_lens, attn_sums, positions, keep, recent,
                       {key_scale, value_scale, key_offset, value_offset});
}

std::tuple<Tensor, Tensor, Tensor> evict_hip(const Tensor &key_cache, const Tensor &value_cache, const Tensor &block_table, const Tensor &context_lens,
                                             const Tensor &attn_sums, const Tensor &positions, int64_t keep, int64_t recent,
                                             const optional<Tensor> &key_scale, const optional<Tensor> &value_scale,
                                             const optional<Tensor> &key_offset, const optional<Tensor> &value_offset)
{
    const char *op = "npu_paged_cache_evict";
    const Params p(key_scale, value_scale, key_offset, value_offset);
    check_same_device(op, {&key_cache, &value_cache, &block_table, &context_lens, &attn_sums, &positions, p.ks, p.vs, p.ko, p.vo});
    c10::hip::HIPGuardMasqueradingAsCUDA guard(key_cache.device());
    auto [new_lens, new_sums, new_positions] = evict_alloc(kLaunch, key_cache, value_cache, block_table, context_lens, attn_sums, positions, keep, recent, p);
    const int64_t batch = block_table.size(0);
    if (batch == 0) return {new_lens, new_sums, new_positions};
    const Tensor table = as_int(block_table), lens = as_int(context_lens);
    const Tensor sums = inner_contiguous(attn_sums) ? attn_sums : attn_sums.contiguous(), pos = inner_contiguous(positions) ? positions : positions.contiguous();
    const mi355_paged_cache c = describe(key_cache, value_cache, p);
    const size_t bytes = mi355_paged_cache_evict_workspace(batch, key_cache.size(2), table.size(1), key_cache.size(1), keep);
    // behind the zero area of the stream's workspace: 0.35 us less on the host than memory of its own
    const Workspace ws = mi355_ops::workspace(key_cache, MI355_WORKSPACE_ZERO_BYTES + bytes, true);
    check_status(mi355_paged_cache_evict(&c, table.data_ptr<int32_t>(), table.stride(0), table.size(1), lens.data_ptr<int32_t>(), batch,
                                         sums.data_ptr<float>(), sums.stride(0), sums.stride(1), pos.data_ptr<int32_t>(), pos.stride(0), pos.stride(1),
                                         keep, recent, new_lens.data_ptr<int32_t>(), new_sums.data_ptr<float>(), new_positions.data_ptr<int32_t>(),
                                         static_cast<char *>(ws.memory.data_ptr()) + MI355_WORKSPACE_ZERO_BYTES, bytes, stream_of(key_cache)),
                 op);
    return {new_lens, new_sums, new_positions};
}

} // namespace

TORCH_LIBRARY_FRAGMENT(npu, m)
{
    m.def("npu_paged_cache_write(Tensor key, Tensor value, Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor slots, *, "
          "Tensor(c!)? key_scale=None, Tensor(d!)? value_scale=None, Tensor(e!)? key_offset=None, Tensor(f!)? value_offset=None) -> ()");
    m.def("npu_paged_cache_read(Tensor key_cache, Tensor value_cache, Tensor slots, *, Tensor? key_scale=None, Tensor? value_scale=None, "
          "ScalarType? dtype=None, Tensor? key_offset=None, Tensor? value_offset=None) -> (Tensor, Tensor)");
    m.def("npu_paged_decode_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor context_lens, *, "
          "Tensor? key_scale=None, Tensor? value_scale=None, float? scale_value=None, Tensor? atten_mask=None, Tensor(a!)? attn_sums=None, "
          "bool softmax_lse=False, Tensor? key_offset=None, Tensor? value_offset=None) -> (Tensor, Tensor)");
    m.def("npu_paged_cache_evict(Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor block_table, Tensor context_lens, Tensor attn_sums, "
          "Tensor positions, int keep, int recent, *, Tensor(c!)? key_scale=None, Tensor(d!)? value_scale=None, "
          "Tensor(e!)? key_offset=None, Tensor(f!)? value_offset=None) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(npu, CUDA, m)
{
    m.impl("npu_paged_cache_write", TORCH_FN(write_hip));
    m.impl("npu_paged_cache_read", TORCH_FN(read_hip));
    m.impl("npu_paged_decode_attention", TORCH_FN(attention_hip));
    m.impl("npu_paged_cache_evict", TORCH_FN(evict_hip));
}

TORCH_LIBRARY_IMPL(npu, Meta, m)
{
    m.impl("npu_paged_cache_write", TORCH_FN(write_meta));
    m.impl("npu_paged_cache_read", TORCH_FN(read_meta));
    m.impl("npu_paged_decode_attention", TORCH_FN(attention_meta));
    m.impl("npu_paged_cache_evict", TORCH_FN(evict_meta));
}
