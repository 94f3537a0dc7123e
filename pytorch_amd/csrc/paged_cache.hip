// npu_paged_cache_write and npu_paged_cache_read for gfx950: rows of head_dim elements between [tokens, heads, dim] tensors
// and the slots of a paged cache, as they are or as int8 codes with one float32 scale per row.
//
// Per row and plane (keys, values), with float32 arithmetic rounded operation by operation:
//   write int8   scale = max_d |x_d| / 127,  code_d = rint_half_even(x_d / scale)      (npu_dynamic_quant's rule)
//   read  int8   x_d = round(code_d * scale)
// Both only move bytes.  A row is handled by a group of 8, 16 or 32 lanes with 8 elements each, so the maximum of a row takes
// three to five lane exchanges and no barrier, and a wavefront's loads cover whole rows.
#include "paged_cache.h"
#include "weight_quant_common.h"

namespace mi355 {
namespace {

struct RowArgs {
    PagedCache cache;
    uint16_t *plane[2];                // key, value: [tokens, heads, dim]
    int64_t tok[2], head[2];           // their element strides
    const void *slot_ids;
    int slots64;                       // slot ids are int64, else int32
    FastDiv heads;
    uint32_t rows;                     // tokens * heads
};

__device__ __forceinline__ int64_t load_slot(const RowArgs &a, uint32_t t)
{
    return a.slots64 ? static_cast<const int64_t *>(a.slot_ids)[t] : (int64_t) static_cast<const int32_t *>(a.slot_ids)[t];
}

__device__ __forceinline__ float cvt16(uint16_t h, int fp16) { return fp16 ? act_1<1>(h) : act_1<0>(h); }

// largest |x| of eight 16-bit values, on the bit patterns
__device__ __forceinline__ uint32_t absmax8(u32x4 v)
{
    typedef uint16_t us2 __attribute__((ext_vector_type(2)));
    us2 m = __builtin_elementwise_max(__builtin_bit_cast(us2, v.x & 0x7fff7fffu), __builtin_bit_cast(us2, v.y & 0x7fff7fffu));
    m = __builtin_elementwise_max(m, __builtin_elementwise_max(__builtin_bit_cast(us2, v.z & 0x7fff7fffu), __builtin_bit_cast(us2, v.w & 0x7fff7fffu)));
    return m[0] > m[1] ? m[0] : m[1];
}

// x / scale rounded to the nearest integer.  For the significands of 16-bit x, a scale that is such a value over 127 and a
// scale in [2^-60, 2^60], one correction of x * (1 / scale) gives the correctly rounded quotient (checked exhaustively for
// npu_dynamic_quant); adding 1.5 * 2^23 rounds it, and the low byte of the sum's pattern is the code.
struct RowQuant {
    float scale, r;
    bool zero, fast;
    __device__ explicit RowQuant(float amax) : scale(amax / 127.0f), r(1.0f / scale), zero(!(amax > 0.0f)), fast(scale >= 0x1p-60f && scale <= 0x1p60f) {}
    __device__ __forceinline__ uint32_t operator()(float x) const
    {
        if (zero) return 0;
        if (fast) {
            const float q0 = x * r;
            return __float_as_uint(__builtin_fmaf(__builtin_fmaf(-scale, q0, x), r, q0) + 12582912.0f);
        }
        float q = __builtin_rintf(x / scale);
        q = q > 127.0f ? 127.0f : q;
        q = q < -127.0f ? -127.0f : q;               // NaN falls through both tests and converts to 0
        return (uint32_t)(int)q;
    }
};

// GL lanes per row, eight elements per lane: rows that start on 16-byte boundaries, dim % 8 == 0 and <= 8 GL.
// QUANT: int8 cache; FP16: the 16-bit type (read by the conversions alone).
template <int GL, bool QUANT, bool FP16>
__global__ __launch_bounds__(256) void paged_write_kernel(RowArgs a)
{
    const int plane = blockIdx.y, lane = threadIdx.x % GL;
    const uint32_t row = blockIdx.x * (256 / GL) + threadIdx.x / GL;
    const uint32_t t = div_by(row, a.heads), h = row - t * a.heads.d;
    if (row >= a.rows) return;                                   // whole groups of GL lanes leave together
    const int64_t slot = load_slot(a, t);
    const bool mine = lane * 8 < a.cache.dim;
    u32x4 v = u32x4{0, 0, 0, 0};
    if (mine) v = *reinterpret_cast<const u32x4 *>(a.plane[plane] + t * a.tok[plane] + h * a.head[plane] + lane * 8);
    if (slot < 0 || slot >= a.cache.slots) return;
    const PagedArray &to = plane ? a.cache.value : a.cache.key;
    char *dst = to.base + a.cache.offset(to, (uint32_t)slot, (int)h);
    if constexpr (!QUANT) {
        if (mine) *reinterpret_cast<u32x4 *>(dst + lane * 16) = v;
    } else {
        uint32_t m = absmax8(v);
#pragma unroll
        for (int off = GL / 2; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, GL));
        const RowQuant q(act_1<FP16>((uint16_t)m));
        if (mine) {
            u32x2 o;
            o.x = pack4(q(act_lo<FP16>(v.x)), q(act_hi<FP16>(v.x)), q(act_lo<FP16>(v.y)), q(act_hi<FP16>(v.y)));
            o.y = pack4(q(act_lo<FP16>(v.z)), q(act_hi<FP16>(v.z)), q(act_lo<FP16>(v.w)), q(act_hi<FP16>(v.w)));
            *reinterpret_cast<u32x2 *>(dst + lane * 8) = o;
        }
        if (lane == 0) {
            const PagedArray &s = plane ? a.cache.value_scale : a.cache.key_scale;
            *reinterpret_cast<float *>(s.base + a.cache.offset(s, (uint32_t)slot, (int)h)) = q.scale;
        }
    }
}

// Any width, alignment and strides: one wavefront per row, element by element.
template <bool QUANT>
__global__ __launch_bounds__(256) void paged_write_any_kernel(RowArgs a, int fp16)
{
    const int plane = blockIdx.y, lane = threadIdx.x % 64;
    const uint32_t row = blockIdx.x * 4 + threadIdx.x / 64;
    if (row >= a.rows) return;
    const uint32_t t = div_by(row, a.heads), h = row - t * a.heads.d;
    const int64_t slot = load_slot(a, t);
    if (slot < 0 || slot >= a.cache.slots) return;
    const uint16_t *x = a.plane[plane] + t * a.tok[plane] + h * a.head[plane];
    const PagedArray &to = plane ? a.cache.value : a.cache.key;
    char *dst = to.base + a.cache.offset(to, (uint32_t)slot, (int)h);
    if constexpr (!QUANT) {
        for (int d = lane; d < a.cache.dim; d += 64) reinterpret_cast<uint16_t *>(dst)[d] = x[d];
    } else {
        uint32_t m = 0;
        for (int d = lane; d < a.cache.dim; d += 64) m = max(m, (uint32_t)(x[d] & 0x7fffu));
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
        const RowQuant q(cvt16((uint16_t)m, fp16));
        for (int d = lane; d < a.cache.dim; d += 64) dst[d] = (char)(q(cvt16(x[d], fp16)) & 0xffu);
        if (lane == 0) {
            const PagedArray &s = plane ? a.cache.value_scale : a.cache.key_scale;
            *reinterpret_cast<float *>(s.base + a.cache.offset(s, (uint32_t)slot, (int)h)) = q.scale;
        }
    }
}

template <int GL, bool QUANT, bool FP16>
__global__ __launch_bounds__(256) void paged_read_kernel(RowArgs a)
{
    const int plane = blockIdx.y, lane = threadIdx.x % GL;
    const uint32_t row = blockIdx.x * (256 / GL) + threadIdx.x / GL;
    const uint32_t t = div_by(row, a.heads), h = row - t * a.heads.d;
    if (row >= a.rows || lane * 8 >= a.cache.dim) return;
    const int64_t slot = load_slot(a, t);
    u32x4 v = u32x4{0, 0, 0, 0};
    if (slot >= 0 && slot < a.cache.slots) {
        const PagedArray &from = plane ? a.cache.value : a.cache.key;
        const char *src = from.base + a.cache.offset(from, (uint32_t)slot, (int)h);
        if constexpr (!QUANT) {
            v = *reinterpret_cast<const u32x4 *>(src + lane * 16);
        } else {
            const PagedArray &s = plane ? a.cache.value_scale : a.cache.key_scale;
            const float scale = *reinterpret_cast<const float *>(s.base + a.cache.offset(s, (uint32_t)slot, (int)h));
            const u32x2 c = *reinterpret_cast<const u32x2 *>(src + lane * 8);
            v.x = pack_act2<FP16>(sbyte_f32(c.x, 0) * scale, sbyte_f32(c.x, 1) * scale);
            v.y = pack_act2<FP16>(sbyte_f32(c.x, 2) * scale, sbyte_f32(c.x, 3) * scale);
            v.z = pack_act2<FP16>(sbyte_f32(c.y, 0) * scale, sbyte_f32(c.y, 1) * scale);
            v.w = pack_act2<FP16>(sbyte_f32(c.y, 2) * scale, sbyte_f32(c.y, 3) * scale);
        }
    }
    *reinterpret_cast<u32x4 *>(a.plane[plane] + t * a.tok[plane] + h * a.head[plane] + lane * 8) = v;
}

template <bool QUANT>
__global__ __launch_bounds__(256) void paged_read_any_kernel(RowArgs a, int fp16)
{
    const int plane = blockIdx.y, lane = threadIdx.x % 64;
    const uint32_t row = blockIdx.x * 4 + threadIdx.x / 64;
    if (row >= a.rows) return;
    const uint32_t t = div_by(row, a.heads), h = row - t * a.heads.d;
    const int64_t slot = load_slot(a, t);
    uint16_t *y = a.plane[plane] + t * a.tok[plane] + h * a.head[plane];
    const bool there = slot >= 0 && slot < a.cache.slots;
    const PagedArray &from = plane ? a.cache.value : a.cache.key;
    const PagedArray &s = plane ? a.cache.value_scale : a.cache.key_scale;
    const char *src = there ? from.base + a.cache.offset(from, (uint32_t)slot, (int)h) : nullptr;
    const float scale = QUANT && there ? *reinterpret_cast<const float *>(s.base + a.cache.offset(s, (uint32_t)slot, (int)h)) : 0.0f;
    for (int d = lane; d < a.cache.dim; d += 64) {
        uint16_t o = 0;
        if (there) {
            if constexpr (QUANT) {
                const float f = (float)(int8_t)src[d] * scale;
                o = fp16 ? (uint16_t)pack_act2<1>(f, 0.0f) : (uint16_t)pack_act2<0>(f, 0.0f);
            } else {
                o = reinterpret_cast<const uint16_t *>(src)[d];
            }
        }
        y[d] = o;
    }
}

template <bool WRITE, int GL>
void launch_rows(const RowArgs &a, bool quant, bool fp16, dim3 grid, hipStream_t s)
{
    if constexpr (WRITE) {
        if (!quant) hipLaunchKernelGGL((paged_write_kernel<GL, false, false>), grid, dim3(256), 0, s, a);
        else if (fp16) hipLaunchKernelGGL((paged_write_kernel<GL, true, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((paged_write_kernel<GL, true, false>), grid, dim3(256), 0, s, a);
    } else {
        if (!quant) hipLaunchKernelGGL((paged_read_kernel<GL, false, false>), grid, dim3(256), 0, s, a);
        else if (fp16) hipLaunchKernelGGL((paged_read_kernel<GL, true, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((paged_read_kernel<GL, true, false>), grid, dim3(256), 0, s, a);
    }
}

template <bool WRITE>
int move_rows(const mi355_paged_cache *cache, int dtype, void *key, const int64_t *key_stride, void *value, const int64_t *value_stride,
              const void *slots, int slots_dtype, int64_t tokens, void *stream)
{
    RowArgs a;
    if (const int st = open_cache(cache, &a.cache); st != MI355_OK) return st;
    const bool quant = cache->dtype == MI355_DTYPE_INT8;
    if (tokens < 0 || (dtype != MI355_DTYPE_BF16 && dtype != MI355_DTYPE_FP16) || (!quant && cache->dtype != dtype)) return MI355_ERR_BAD_ARGUMENT;
    if (slots_dtype != MI355_DTYPE_INT32 && slots_dtype != MI355_DTYPE_INT64) return MI355_ERR_BAD_ARGUMENT;
    if (tokens == 0) return MI355_OK;
    if (!key || !value || !slots || !key_stride || !value_stride) return MI355_ERR_BAD_ARGUMENT;
    if (tokens > 0x7fffffff / cache->kv_heads) return MI355_ERR_UNSUPPORTED;
    if (!aligned(key, 2) || !aligned(value, 2) || !aligned(slots, slots_dtype == MI355_DTYPE_INT64 ? 8 : 4)) return MI355_ERR_ALIGNMENT;
    a.plane[0] = static_cast<uint16_t *>(key);
    a.plane[1] = static_cast<uint16_t *>(value);
    bool vec = a.cache.dim % 8 == 0 && a.cache.dim <= 256;
    const int64_t *strides[2] = {key_stride, value_stride};
    for (int i = 0; i < 2; i++) {
        a.tok[i] = strides[i][0];
        a.head[i] = strides[i][1];
        vec = vec && aligned(a.plane[i], 16) && a.tok[i] % 8 == 0 && a.head[i] % 8 == 0 && rows_aligned(i ? a.cache.value : a.cache.key, quant ? 8 : 16);
    }
    a.slot_ids = slots;
    a.slots64 = slots_dtype == MI355_DTYPE_INT64;
    a.heads = fast_div((uint32_t)cache->kv_heads);
    a.rows = (uint32_t)(tokens * cache->kv_heads);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool fp16 = dtype == MI355_DTYPE_FP16;
    const auto grid = [&](int per) { return dim3((a.rows + per - 1) / per, 2); };
    if (!vec) {
        if constexpr (WRITE) {
            if (quant) hipLaunchKernelGGL(paged_write_any_kernel<true>, grid(4), dim3(256), 0, s, a, fp16);
            else hipLaunchKernelGGL(paged_write_any_kernel<false>, grid(4), dim3(256), 0, s, a, fp16);
        } else {
            if (quant) hipLaunchKernelGGL(paged_read_any_kernel<true>, grid(4), dim3(256), 0, s, a, fp16);
            else hipLaunchKernelGGL(paged_read_any_kernel<false>, grid(4), dim3(256), 0, s, a, fp16);
        }
    } else if (a.cache.dim <= 64) {
        launch_rows<WRITE, 8>(a, quant, fp16, grid(32), s);
    } else if (a.cache.dim <= 128) {
        launch_rows<WRITE, 16>(a, quant, fp16, grid(16), s);
    } else {
        launch_rows<WRITE, 32>(a, quant, fp16, grid(8), s);
    }
    return check_launch();
}

} // namespace
} // namespace mi355

extern "C" int mi355_paged_cache_write(const mi355_paged_cache *cache, const void *key, const int64_t *key_stride, const void *value,
                                       const int64_t *value_stride, int dtype, const void *slots, int slots_dtype, int64_t tokens, void *stream)
{
    return mi355::move_rows<true>(cache, dtype, const_cast<void *>(key), key_stride, const_cast<void *>(value), value_stride, slots, slots_dtype,
                                  tokens, stream);
}

extern "C" int mi355_paged_cache_read(const mi355_paged_cache *cache, void *key, const int64_t *key_stride, void *value,
                                      const int64_t *value_stride, int dtype, const void *slots, int slots_dtype, int64_t tokens, void *stream)
{
    return mi355::move_rows<false>(cache, dtype, key, key_stride, value, value_stride, slots, slots_dtype, tokens, stream);
}
