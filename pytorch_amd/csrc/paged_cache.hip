// npu_paged_cache_write and npu_paged_cache_read for gfx950: rows of head_dim elements between [tokens, heads, dim] tensors
// and the slots of a paged cache, as they are, as int8 codes with one float32 scale per row, or as int4 codes, eight to a word,
// with one scale and one offset.
//
// Per row and plane (keys, values), with float32 arithmetic rounded operation by operation:
//   write int8   scale = max_d |x_d| / 127,  code_d = rint_half_even(x_d / scale)      (npu_dynamic_quant's rule)
//   read  int8   x_d = round(code_d * scale)
//   write int4   lo, hi = min_d, max_d x_d; scale = (hi - lo) / 15; offset = lo / scale + 8
//                code_d = rint_half_even((x_d - lo) * 15 / (hi - lo)) - 8: a value between two codes is told exactly as long as x_d - lo
//                has 20 bits;  hi - lo <= 2^-120: scale 1, offset lo, codes 0
//   read  int4   x_d = round((code_d + offset) * scale)
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

// (x - lo) * 15 / (hi - lo), rounded to the nearest integer, of a row between lo and hi.  With r = 1 / (hi - lo) correctly rounded,
// one correction of t * r by its residual gives one of the two floats next to the quotient, and by Markstein's theorem a second
// one the correctly rounded quotient, where nothing leaves the normal range: for hi - lo in [2^-60, 2^60] only quotients below 2^-40
// do, which round to 0 either way.  The sum with 1.5 * 2^23 rounds, ties to even; its low bits are the number, 0 to 15.
struct RowQuant4 {
    float lo, span;
    bool flat, finite, fast;
    __device__ RowQuant4(float lo_, float hi) : lo(lo_), span(hi - lo_)
    {
        flat = span <= 0x1p-120f;
        finite = span <= 0x1p124f;                           // 15 times it is a number (false for NaN)
        fast = span >= 0x1p-60f && span <= 0x1p60f;
    }
    // span / 15: for every significand the product with 1 / 15, corrected once, is the correctly rounded quotient (checked exhaustively)
    __device__ __forceinline__ float scale() const
    {
        const float c = 1.0f / 15.0f, q = span * c;
        return flat ? 1.0f : finite ? __builtin_fmaf(__builtin_fmaf(-15.0f, q, span), c, q) : NAN;
    }
    // `quotient` = lo / scale()
    __device__ __forceinline__ float offset(float quotient) const { return flat ? lo : quotient + 8.0f; }
    // codes of eight elements in a word; r = 1 / span
    template <bool FP16>
    __device__ __forceinline__ uint32_t word(u32x4 v, float r) const
    {
        uint32_t w = 0;
        if (fast) {
            constexpr uint32_t kOne = 0x4b400000u;           // 1.5 * 2^23, which eight shifted sums leave in the word three times
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float t = ((i % 2 ? act_hi<FP16>(v[i / 2]) : act_lo<FP16>(v[i / 2])) - lo) * 15.0f;
                float q = t * r;
                q = __builtin_fmaf(__builtin_fmaf(-span, q, t), r, q);
                q = __builtin_fmaf(__builtin_fmaf(-span, q, t), r, q);
                w += __float_as_uint(q + 12582912.0f) << (4 * i);
            }
            w -= kOne + (kOne << 4) + (kOne << 8);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float t = ((i % 2 ? act_hi<FP16>(v[i / 2]) : act_lo<FP16>(v[i / 2])) - lo) * 15.0f;
                w |= (flat ? 8u : finite ? (uint32_t)(int)__builtin_rintf(t / span) & 15u : 0u) << (4 * i);
            }
        }
        return w ^ 0x88888888u;                              // u - 8 in two's complement
    }
};
// 16-bit values as integers in their order (and back: its own inverse); NaN lies beyond the infinities
__device__ __forceinline__ uint32_t order16(uint32_t two)
{
    typedef int16_t ss2 __attribute__((ext_vector_type(2)));
    const ss2 x = __builtin_bit_cast(ss2, two);
    return two ^ (__builtin_bit_cast(uint32_t, x >> (int16_t)15) & 0x7fff7fffu);
}
__device__ __forceinline__ uint32_t max16(uint32_t x, uint32_t y)
{
    typedef int16_t ss2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ss2, x), __builtin_bit_cast(ss2, y)));
}
// [largest, largest of the complements] of eight values, in the low and the high half
__device__ __forceinline__ uint32_t range8(u32x4 v)
{
    const uint32_t a = order16(v.x), b = order16(v.y), c = order16(v.z), d = order16(v.w);
    const uint32_t top = max16(max16(a, b), max16(c, d)), low = max16(max16(~a, ~b), max16(~c, ~d));
    return max16(__builtin_amdgcn_perm(low, top, 0x05040100u), __builtin_amdgcn_perm(low, top, 0x07060302u));
}
constexpr uint32_t kNoRange = 0x80008000u;                   // of no values: below everything
template <bool FP16>
__device__ __forceinline__ RowQuant4 quant_of(uint32_t range)
{
    return RowQuant4(act_1<FP16>((uint16_t)order16(~range >> 16)), act_1<FP16>((uint16_t)order16(range & 0xffffu)));
}
// the lane of another place among the four, eight, 16 (32) neighbours
template <int CTRL>
__device__ __forceinline__ uint32_t lane_of_four(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
// range over GL lanes, in all of them: neighbours, pairs, mirrored fours, mirrored eights, rows of 16
template <int GL>
__device__ __forceinline__ uint32_t over_row(uint32_t v)
{
    v = max16(v, lane_of_four<0xb1>(v));
    v = max16(v, lane_of_four<0x4e>(v));
    v = max16(v, lane_of_four<0x141>(v));
    if constexpr (GL >= 16) v = max16(v, lane_of_four<0x140>(v));
    if constexpr (GL >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max16(r[0], r[1]);
    }
    return v;
}
__device__ __forceinline__ float nibble_f32(uint32_t w, int i) { return (float)((int32_t)(w << (28 - 4 * i)) >> 28); }

// GL lanes per row, eight elements per lane: rows that start on 16-byte boundaries, dim % 8 == 0 and <= 8 GL.  N heads of a
// token per group of lanes: slot and addresses are worked out once (they were half of the instructions, and the int8 writer
// is bound by those), the rows requested together.  BITS: of the cache's elements; FP16: the 16-bit type (for the conversions alone).
template <int GL, int N, int BITS, bool FP16>
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
    char *dst = to.base + a.cache.offset(to, (uint32_t)slot, (int)(part * N)) + lane * BITS;
    char *scale = BITS < 16 ? sc.base + a.cache.offset(sc, (uint32_t)slot, (int)(part * N)) : nullptr;
    const PagedArray &of = plane ? a.cache.value_offset : a.cache.key_offset;
    char *offset = BITS == 4 ? of.base + a.cache.offset(of, (uint32_t)slot, (int)(part * N)) : nullptr;
    if constexpr (BITS == 4) {
        // Lanes 0 and 1 (of four) divide 1 by the rows' spans, lanes 2 and 3 their least values by their scales: one division, an exact
        // one is eleven instructions, for up to four.
        static_assert(N <= 2, "a lane for each quotient");
        uint32_t range[N];
#pragma unroll
        for (int i = 0; i < N; i++) range[i] = over_row<GL>(mine ? range8(v[i]) : kNoRange);
        const RowQuant4 first = quant_of<FP16>(range[0]), second = quant_of<FP16>(range[N - 1]), &own = lane & 1 ? second : first;
        const float own_scale = own.scale(), quotient = (lane & 2 ? own.lo : 1.0f) / (lane & 2 ? own_scale : own.span);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float r = __uint_as_float(i ? lane_of_four<0x55>(__float_as_uint(quotient)) : lane_of_four<0x00>(__float_as_uint(quotient)));
            const uint32_t word = (i ? second : first).template word<FP16>(v[i], r);
            if (mine) *reinterpret_cast<uint32_t *>(dst + i * to.head) = word;
        }
        if (lane >= 2 && lane < 2 + N) {
            *reinterpret_cast<float *>(scale + (lane - 2) * sc.head) = own_scale;
            *reinterpret_cast<float *>(offset + (lane - 2) * of.head) = own.offset(quotient);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        if constexpr (BITS == 16) {
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
template <int BITS>
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
    if constexpr (BITS == 16) {
        for (int d = lane; d < a.cache.dim; d += 64) reinterpret_cast<uint16_t *>(dst)[d] = x[d];
    } else if constexpr (BITS == 4) {
        uint32_t range = kNoRange;
        for (int d = lane; d < a.cache.dim; d += 64) {
            const uint32_t o = order16(x[d]) & 0xffffu;
            range = max16(range, o | ~o << 16);
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) range = max16(range, (uint32_t)__shfl_xor((int)range, off, 64));
        const RowQuant4 q = fp16 ? quant_of<true>(range) : quant_of<false>(range);
        const float r = 1.0f / q.span, scale = q.scale();
        for (int w = lane; w < a.cache.dim / 8; w += 64) {
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = x[8 * w + 2 * i] | (uint32_t)x[8 * w + 2 * i + 1] << 16;
            reinterpret_cast<uint32_t *>(dst)[w] = fp16 ? q.word<true>(v, r) : q.word<false>(v, r);
        }
        if (lane == 0) {
            const PagedArray &s = plane ? a.cache.value_scale : a.cache.key_scale, &o = plane ? a.cache.value_offset : a.cache.key_offset;
            *reinterpret_cast<float *>(s.base + a.cache.offset(s, (uint32_t)slot, (int)h)) = scale;
            *reinterpret_cast<float *>(o.base + a.cache.offset(o, (uint32_t)slot, (int)h)) = q.offset(q.lo / scale);
        }
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

template <int GL, int N, int BITS, bool FP16>
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
        const char *src = from.base + a.cache.offset(from, (uint32_t)slot, (int)(part * N)) + lane * BITS;
        if constexpr (BITS == 4) {
            const PagedArray &of = plane ? a.cache.value_offset : a.cache.key_offset;
            const char *at = sc.base + a.cache.offset(sc, (uint32_t)slot, (int)(part * N)), *at_of = of.base + a.cache.offset(of, (uint32_t)slot, (int)(part * N));
            uint32_t w[N];
            float scale[N], offset[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                w[i] = *reinterpret_cast<const uint32_t *>(src + i * from.head);
                scale[i] = *reinterpret_cast<const float *>(at + i * sc.head);
                offset[i] = *reinterpret_cast<const float *>(at_of + i * of.head);
            }
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    v[i][k] = pack_act2<FP16>((nibble_f32(w[i], 2 * k) + offset[i]) * scale[i], (nibble_f32(w[i], 2 * k + 1) + offset[i]) * scale[i]);
        } else if constexpr (BITS == 8) {
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

template <int BITS>
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
    const float scale = BITS < 16 && there ? *reinterpret_cast<const float *>(s.base + a.cache.offset(s, (uint32_t)slot, (int)h)) : 0.0f;
    const PagedArray &of = plane ? a.cache.value_offset : a.cache.key_offset;
    const float offset = BITS == 4 && there ? *reinterpret_cast<const float *>(of.base + a.cache.offset(of, (uint32_t)slot, (int)h)) : 0.0f;
    for (int d = lane; d < a.cache.dim; d += 64) {
        uint16_t o = 0;
        if (there) {
            if constexpr (BITS < 16) {
                const float f = BITS == 4 ? (nibble_f32(reinterpret_cast<const uint32_t *>(src)[d / 8], d % 8) + offset) * scale : (float)(int8_t)src[d] * scale;
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
void launch_rows(RowArgs &a, int bits, bool fp16, hipStream_t s)
{
    number_groups(a, N);
    const dim3 grid((a.groups + 256 / GL - 1) / (256 / GL), 2);
    const auto with = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    if constexpr (WRITE) {
        if (bits == 16) with(paged_write_kernel<GL, N, 16, false>);
        else if (bits == 8) fp16 ? with(paged_write_kernel<GL, N, 8, true>) : with(paged_write_kernel<GL, N, 8, false>);
        else fp16 ? with(paged_write_kernel<GL, N, 4, true>) : with(paged_write_kernel<GL, N, 4, false>);
    } else {
        if (bits == 16) with(paged_read_kernel<GL, N, 16, false>);
        else if (bits == 8) fp16 ? with(paged_read_kernel<GL, N, 8, true>) : with(paged_read_kernel<GL, N, 8, false>);
        else fp16 ? with(paged_read_kernel<GL, N, 4, true>) : with(paged_read_kernel<GL, N, 4, false>);
    }
}
template <bool WRITE, int GL>
void launch_rows(RowArgs &a, int bits, bool fp16, hipStream_t s)
{
    // One row per group of lanes while that leaves the card short of workgroups.  Beyond: 8192 tokens to int8, 8 heads of 128,
    // 14.3 us with one row per group, 13.2 with two, 13.9 with four; 32768 tokens from int8 33.6, 31.3 and 31.2.  8192 tokens to int4
    // (43 MB) 15.6 us with one row, 14.5 with two; from int4 8.6 with four.
    const bool many = (int64_t)a.tokens * a.cache.heads * 2 / (256 / GL) >= kNumCU * 16;
    if constexpr (!WRITE)
        if (many && a.cache.heads % 4 == 0) return launch_rows<WRITE, GL, 4>(a, bits, fp16, s);
    if (many && a.cache.heads % 2 == 0) launch_rows<WRITE, GL, 2>(a, bits, fp16, s);
    else launch_rows<WRITE, GL, 1>(a, bits, fp16, s);
}

template <bool WRITE>
void launch_tokens(RowArgs &a, bool vec, int bits, bool fp16, hipStream_t s)
{
    if (!vec) {
        number_groups(a, 1);
        const dim3 grid((a.groups + 3) / 4, 2);
        const auto with = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, fp16); };
        if constexpr (WRITE) bits == 16 ? with(paged_write_any_kernel<16>) : bits == 8 ? with(paged_write_any_kernel<8>) : with(paged_write_any_kernel<4>);
        else bits == 16 ? with(paged_read_any_kernel<16>) : bits == 8 ? with(paged_read_any_kernel<8>) : with(paged_read_any_kernel<4>);
    } else if (a.cache.dim <= 64) {
        launch_rows<WRITE, 8>(a, bits, fp16, s);
    } else if (a.cache.dim <= 128) {
        launch_rows<WRITE, 16>(a, bits, fp16, s);
    } else {
        launch_rows<WRITE, 32>(a, bits, fp16, s);
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
    const int bits = cache_bits(cache->dtype);
    if (tokens < 0 || (dtype != MI355_DTYPE_BF16 && dtype != MI355_DTYPE_FP16) || (bits == 16 && cache->dtype != dtype)) return MI355_ERR_BAD_ARGUMENT;
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
        vec = vec && aligned(plane[i], 16) && a.tok[i] % 8 == 0 && a.head[i] % 8 == 0 && rows_aligned(i ? a.cache.value : a.cache.key, bits);
    }
    a.slots64 = slots_dtype == MI355_DTYPE_INT64;
    a.run = a.cache.key.token < a.cache.key.head ? 4 : 0;
    const int64_t most = kRowsPerLaunch / cache->kv_heads;
    for (int64_t t0 = 0; t0 < tokens; t0 += most) {
        for (int i = 0; i < 2; i++) a.plane[i] = plane[i] + t0 * a.tok[i];
        a.slot_ids = static_cast<const char *>(slots) + t0 * id_bytes;
        a.tokens = (uint32_t)(tokens - t0 < most ? tokens - t0 : most);
        launch_tokens<WRITE>(a, vec, bits, dtype == MI355_DTYPE_FP16, static_cast<hipStream_t>(stream));
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
