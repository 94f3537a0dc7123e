// npu_paged_cache_write and npu_paged_cache_read for gfx950: rows of head_dim elements between [tokens, heads, dim] tensors
// and the slots of a paged cache, as they are or as int8 codes with one float32 scale per row.
//
// Per row and plane (keys, values), with float32 arithmetic rounded operation by operation:
//   write int8   scale = max_d |x_d| / 127,  code_d = rint_half_even(x_d / scale)      (npu_dynamic_quant's rule)
//   read  int8   x_d = round(code_d * scale)
// Both only move bytes.  A row is handled by a group of 8, 16 or 32 lanes with 8 elements each, so the maximum of a row takes
// three to five lane exchanges and no barrier, and a wavefront's loads cover whole rows.
//
// Measured, 8 heads of 128: 64 tokens written in 2.8 us, 2047 read in 3.8 us (16.8 MB; both the latency of a launch and of three
// dependent trips to memory); 8192 bf16 tokens to int8 13.3 us, 51 MB, 3.8 TB/s, bound by the instructions of the quantisation
// and of the addresses; 32768 int8 tokens to fp16 31.3 us, 204 MB, 6.5 TB/s, bound by memory.
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
    FastDiv parts;                     // groups of heads of a token: heads / N
    uint32_t tokens, groups;           // groups = tokens, rounded up to the run, * parts
    int run;                           // log2 of the tokens of one head that follow each other
};

// Groups of N heads of a token are numbered so that neighbours lie side by side in the cache: the heads of a token, or 16
// tokens of the same heads.
__device__ __forceinline__ void group_at(const RowArgs &a, uint32_t group, uint32_t &t, uint32_t &part)
{
    const uint32_t q = group >> a.run, block = div_by(q, a.parts);
    part = q - block * a.parts.d;
    t = (block << a.run) + (group & ((1u << a.run) - 1));
}

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

// GL lanes per row, eight elements per lane: rows that start on 16-byte boundaries, dim % 8 == 0 and <= 8 GL.  N heads of a
// token per group of lanes: slot and addresses are worked out once (they were half of the instructions, and the int8 writer
// is bound by those), the rows requested together.  QUANT: int8 cache; FP16: the 16-bit type (for the conversions alone).
template <int GL, int N, bool QUANT, bool FP16>
__global__ __launch_bounds__(256) void paged_write_kernel(RowArgs a)
{
    const int plane = blockIdx.y, lane = threadIdx.x % GL;
    const uint32_t group = blockIdx.x * (256 / GL) + threadIdx.x / GL;
    uint32_t t, part;
    group_at(a, group, t, part);
    if (group >= a.groups || t >= a.tokens) return;              // whole groups of lanes leave together
    const bool mine = lane * 8 < a.cache.dim;
    const PagedArray &to = plane ? a.cache.value : a.cache.key, &sc = plane ? a.cache.value_scale : a.cache.key_scale;
    const int64_t slot = load_slot(a, t);
    const uint16_t *src = a.plane[plane] + t * a.tok[plane] + (part * N) * a.head[plane] + lane * 8;
    u32x4 v[N];
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = mine ? *reinterpret_cast<const u32x4 *>(src + i * a.head[plane]) : u32x4{0, 0, 0, 0};
    if (slot < 0 || slot >= a.cache.slots) return;
    char *dst = to.base + a.cache.offset(to, (uint32_t)slot, (int)(part * N)) + lane * (QUANT ? 8 : 16);
    char *scale = QUANT ? sc.base + a.cache.offset(sc, (uint32_t)slot, (int)(part * N)) : nullptr;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if constexpr (!QUANT) {
            if (mine) *reinterpret_cast<u32x4 *>(dst + i * to.head) = v[i];
        } else {
            uint32_t m = absmax8(v[i]);
#pragma unroll
            for (int off = GL / 2; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, GL));
            const RowQuant q(act_1<FP16>((uint16_t)m));
            u32x2 o;
            o.x = pack4(q(act_lo<FP16>(v[i].x)), q(act_hi<FP16>(v[i].x)), q(act_lo<FP16>(v[i].y)), q(act_hi<FP16>(v[i].y)));
            o.y = pack4(q(act_lo<FP16>(v[i].z)), q(act_hi<FP16>(v[i].z)), q(act_lo<FP16>(v[i].w)), q(act_hi<FP16>(v[i].w)));
            if (mine) *reinterpret_cast<u32x2 *>(dst + i * to.head) = o;
            if (lane == 0) *reinterpret_cast<float *>(scale + i * sc.head) = q.scale;
        }
    }
}

// Any width, alignment and strides: one wavefront per row, element by element, each a trip of its own.
template <bool QUANT>
__global__ __launch_bounds__(256) void paged_write_any_kernel(RowArgs a, int fp16)
{
    const int plane = blockIdx.y, lane = threadIdx.x % 64;
    const uint32_t row = blockIdx.x * 4 + threadIdx.x / 64;
    uint32_t t, h;
    group_at(a, row, t, h);
    if (row >= a.groups || t >= a.tokens) return;
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

template <int GL, int N, bool QUANT, bool FP16>
__global__ __launch_bounds__(256) void paged_read_kernel(RowArgs a)
{
    const int plane = blockIdx.y, lane = threadIdx.x % GL;
    const uint32_t group = blockIdx.x * (256 / GL) + threadIdx.x / GL;
    uint32_t t, part;
    group_at(a, group, t, part);
    if (group >= a.groups || t >= a.tokens || lane * 8 >= a.cache.dim) return;
    const PagedArray &from = plane ? a.cache.value : a.cache.key, &sc = plane ? a.cache.value_scale : a.cache.key_scale;
    const int64_t slot = load_slot(a, t);
    u32x4 v[N] = {};
    if (slot >= 0 && slot < a.cache.slots) {
        const char *src = from.base + a.cache.offset(from, (uint32_t)slot, (int)(part * N)) + lane * (QUANT ? 8 : 16);
        if constexpr (QUANT) {
            const char *at = sc.base + a.cache.offset(sc, (uint32_t)slot, (int)(part * N));
            u32x2 c[N];
            float scale[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                c[i] = *reinterpret_cast<const u32x2 *>(src + i * from.head);
                scale[i] = *reinterpret_cast<const float *>(at + i * sc.head);
            }
#pragma unroll
            for (int i = 0; i < N; i++) {
                v[i].x = pack_act2<FP16>(sbyte_f32(c[i].x, 0) * scale[i], sbyte_f32(c[i].x, 1) * scale[i]);
                v[i].y = pack_act2<FP16>(sbyte_f32(c[i].x, 2) * scale[i], sbyte_f32(c[i].x, 3) * scale[i]);
                v[i].z = pack_act2<FP16>(sbyte_f32(c[i].y, 0) * scale[i], sbyte_f32(c[i].y, 1) * scale[i]);
                v[i].w = pack_act2<FP16>(sbyte_f32(c[i].y, 2) * scale[i], sbyte_f32(c[i].y, 3) * scale[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = *reinterpret_cast<const u32x4 *>(src + i * from.head);
        }
    }
    uint16_t *dst = a.plane[plane] + t * a.tok[plane] + (part * N) * a.head[plane] + lane * 8;
#pragma unroll
    for (int i = 0; i < N; i++) __builtin_nontemporal_store(v[i], reinterpret_cast<u32x4 *>(dst + i * a.head[plane]));
}

template <bool QUANT>
__global__ __launch_bounds__(256) void paged_read_any_kernel(RowArgs a, int fp16)
{
    const int plane = blockIdx.y, lane = threadIdx.x % 64;
    const uint32_t row = blockIdx.x * 4 + threadIdx.x / 64;
    uint32_t t, h;
    group_at(a, row, t, h);
    if (row >= a.groups || t >= a.tokens) return;
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

// Groups of n heads (a divisor of the heads); RowArgs is complete after it.
void number_groups(RowArgs &a, int n)
{
    const uint32_t parts = (uint32_t)(a.cache.heads / n);
    a.parts = fast_div(parts);
    a.groups = ((a.tokens + (1u << a.run) - 1) >> a.run << a.run) * parts;
}

template <bool WRITE, int GL, int N>
void launch_rows(RowArgs &a, bool quant, bool fp16, hipStream_t s)
{
    number_groups(a, N);
    const dim3 grid((a.groups + 256 / GL - 1) / (256 / GL), 2);
    if constexpr (WRITE) {
        if (!quant) hipLaunchKernelGGL((paged_write_kernel<GL, N, false, false>), grid, dim3(256), 0, s, a);
        else if (fp16) hipLaunchKernelGGL((paged_write_kernel<GL, N, true, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((paged_write_kernel<GL, N, true, false>), grid, dim3(256), 0, s, a);
    } else {
        if (!quant) hipLaunchKernelGGL((paged_read_kernel<GL, N, false, false>), grid, dim3(256), 0, s, a);
        else if (fp16) hipLaunchKernelGGL((paged_read_kernel<GL, N, true, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((paged_read_kernel<GL, N, true, false>), grid, dim3(256), 0, s, a);
    }
}
template <bool WRITE, int GL>
void launch_rows(RowArgs &a, bool quant, bool fp16, hipStream_t s)
{
    // One row per group of lanes while that leaves the card short of workgroups.  Beyond: 8192 tokens to int8, 8 heads of 128,
    // 14.3 us with one row per group, 13.2 with two, 13.9 with four; 32768 tokens from int8 33.6, 31.3 and 31.2.
    const bool many = (int64_t)a.tokens * a.cache.heads * 2 / (256 / GL) >= kNumCU * 16;
    if (many && !WRITE && a.cache.heads % 4 == 0) launch_rows<WRITE, GL, 4>(a, quant, fp16, s);
    else if (many && a.cache.heads % 2 == 0) launch_rows<WRITE, GL, 2>(a, quant, fp16, s);
    else launch_rows<WRITE, GL, 1>(a, quant, fp16, s);
}

template <bool WRITE>
void launch_tokens(RowArgs &a, bool vec, bool quant, bool fp16, hipStream_t s)
{
    if (!vec) {
        number_groups(a, 1);
        const dim3 grid((a.groups + 3) / 4, 2);
        if constexpr (WRITE) {
            if (quant) hipLaunchKernelGGL(paged_write_any_kernel<true>, grid, dim3(256), 0, s, a, fp16);
            else hipLaunchKernelGGL(paged_write_any_kernel<false>, grid, dim3(256), 0, s, a, fp16);
        } else {
            if (quant) hipLaunchKernelGGL(paged_read_any_kernel<true>, grid, dim3(256), 0, s, a, fp16);
            else hipLaunchKernelGGL(paged_read_any_kernel<false>, grid, dim3(256), 0, s, a, fp16);
        }
    } else if (a.cache.dim <= 64) {
        launch_rows<WRITE, 8>(a, quant, fp16, s);
    } else if (a.cache.dim <= 128) {
        launch_rows<WRITE, 16>(a, quant, fp16, s);
    } else {
        launch_rows<WRITE, 32>(a, quant, fp16, s);
    }
}

// Rows of one launch at most: the threads of a grid, up to 64 for a row, are numbered in 32 bits (beyond, the grid wraps without
// an error), and a token has up to 65535 rows.
constexpr int64_t kRowsPerLaunch = (int64_t)1 << 25;

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
    if (tokens > 0x7fffff00 / cache->kv_heads - 16) return MI355_ERR_UNSUPPORTED;
    const int id_bytes = slots_dtype == MI355_DTYPE_INT64 ? 8 : 4;
    if (!aligned(key, 2) || !aligned(value, 2) || !aligned(slots, id_bytes)) return MI355_ERR_ALIGNMENT;
    uint16_t *const plane[2] = {static_cast<uint16_t *>(key), static_cast<uint16_t *>(value)};
    bool vec = a.cache.dim % 8 == 0 && a.cache.dim <= 256;
    const int64_t *strides[2] = {key_stride, value_stride};
    for (int i = 0; i < 2; i++) {
        a.tok[i] = strides[i][0];
        a.head[i] = strides[i][1];
        vec = vec && aligned(plane[i], 16) && a.tok[i] % 8 == 0 && a.head[i] % 8 == 0 && rows_aligned(i ? a.cache.value : a.cache.key, quant ? 8 : 16);
    }
    a.slots64 = slots_dtype == MI355_DTYPE_INT64;
    a.run = a.cache.key.token < a.cache.key.head ? 4 : 0;
    const int64_t most = kRowsPerLaunch / cache->kv_heads;
    for (int64_t t0 = 0; t0 < tokens; t0 += most) {
        for (int i = 0; i < 2; i++) a.plane[i] = plane[i] + t0 * a.tok[i];
        a.slot_ids = static_cast<const char *>(slots) + t0 * id_bytes;
        a.tokens = (uint32_t)(tokens - t0 < most ? tokens - t0 : most);
        launch_tokens<WRITE>(a, vec, quant, dtype == MI355_DTYPE_FP16, static_cast<hipStream_t>(stream));
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
