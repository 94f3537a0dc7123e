// npu_mrope for gfx950: rotary positions on one or several axes, for the queries and keys of a fused projection in one launch.
//
// The first R of a head's D elements are R / 2 pairs - (i, i + R / 2), or (2 i, 2 i + 1) interleaved -, one for each frequency
// f; with the position p of the token on the axis that f belongs to, in float32, every operation rounded by itself:
//   a' = a * cos[p][f] - b * sin[p][f]     b' = b * cos[p][f] + a * sin[p][f]
// and one rounding to 16 bits.  The other D - R elements are copied.  Cosines and sines come from a table [positions][R], the
// cosines first.  A position outside the table counts as cos = sin = 0.
//
// Bound by memory: every element is read and written once.  A thread takes eight frequencies (two pieces of 16 bytes), or four, of one head
// of a token; neighbouring threads take neighbouring pieces, then neighbouring heads.  The heads of a token share its cosines and sines,
// which the caches hand out: with two or four heads a thread the table is read less, and 32767 tokens on three axes, 32 + 8 heads of
// 128, 689 MB, take 115 or 124 us, not 110 (6.2 TB/s), 64 tokens 3.8 or 5.1, not 3.0 (the launch and a trip to memory for the
// positions, one for the table and one for the heads).
#include "paged_cache.h"
#include "weight_quant_common.h"

namespace mi355 {
namespace {

constexpr int kAxes = 4;

struct RopeArgs {
    const uint16_t *in[2];             // query, key: [tokens, heads, dim]
    uint16_t *out[2];                  // the same, contiguous
    int64_t tok[2], head[2];           // elements between tokens and heads of the inputs
    int heads[2];
    const void *table;
    int64_t table_stride, positions;   // elements between rows; rows
    const void *pos;
    int64_t pos_axis, pos_tok;
    int pos64, axes, end[kAxes];       // frequencies of the axes up to and with this one
    int dim, half;                     // half = R / 2
    int interleaved;
    uint32_t tokens, units;            // units = tokens * rows * pieces
    FastDiv pieces, rows;              // pieces of a head; heads of a token, queries first
};

__device__ __forceinline__ int64_t position(const RopeArgs &a, uint32_t token, int axis)
{
    const int64_t at = axis * a.pos_axis + token * a.pos_tok;
    return a.pos64 ? static_cast<const int64_t *>(a.pos)[at] : (int64_t) static_cast<const int32_t *>(a.pos)[at];
}
__device__ __forceinline__ int axis_of(const RopeArgs &a, int f)
{
    int axis = 0;
#pragma unroll
    for (int i = 0; i < kAxes - 1; i++) axis += i + 1 < a.axes && f >= a.end[i];
    return axis;
}

// TABLE: type of the cosines and sines: 0 bf16, 1 fp16, 2 float32
template <int TABLE>
__device__ __forceinline__ float table_1(const RopeArgs &a, int64_t at)
{
    if constexpr (TABLE == 2) return static_cast<const float *>(a.table)[at];
    else return act_1<TABLE>(static_cast<const uint16_t *>(a.table)[at]);
}
template <int TABLE, int W>
__device__ __forceinline__ void table_piece(const RopeArgs &a, int64_t at, float (&to)[W])
{
    if constexpr (TABLE == 2) {
        const f32x4 *p = reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.table) + at);
#pragma unroll
        for (int k = 0; k < W / 4; k++) {
            const f32x4 v = p[k];
#pragma unroll
            for (int i = 0; i < 4; i++) to[4 * k + i] = v[i];
        }
    } else {
        typedef uint32_t piece __attribute__((ext_vector_type(W / 2)));
        const piece v = *reinterpret_cast<const piece *>(static_cast<const uint16_t *>(a.table) + at);
#pragma unroll
        for (int i = 0; i < W / 2; i++) to[2 * i] = act_lo<TABLE>(v[i]), to[2 * i + 1] = act_hi<TABLE>(v[i]);
    }
}
// cosines and sines of W frequencies from f on at position p
template <int TABLE, int W>
__device__ __forceinline__ void turns_at(const RopeArgs &a, int64_t p, int f, float (&c)[W], float (&s)[W])
{
#pragma unroll
    for (int i = 0; i < W; i++) c[i] = s[i] = 0.0f;
    if (p < 0 || p >= a.positions) return;
    table_piece<TABLE>(a, p * a.table_stride + f, c);
    table_piece<TABLE>(a, p * a.table_stride + a.half + f, s);
}
// one value of cosine and sine
template <int TABLE>
__device__ __forceinline__ void turn_of(const RopeArgs &a, uint32_t token, int f, float &c, float &s)
{
    const int64_t p = position(a, token, axis_of(a, f));
    const bool there = p >= 0 && p < a.positions;
    c = there ? table_1<TABLE>(a, p * a.table_stride + f) : 0.0f;
    s = there ? table_1<TABLE>(a, p * a.table_stride + a.half + f) : 0.0f;
}

// Pairs (x[i], y[i]) of W frequencies, packed in two pieces of W elements
template <bool FP16, bool INTERLEAVED, int W, class Piece>
__device__ __forceinline__ void turn(Piece &x, Piece &y, const float (&c)[W], const float (&s)[W])
{
#pragma unroll
    for (int i = 0; i < W / 2; i++) {
        if constexpr (INTERLEAVED) {
            const auto pair = [&](uint32_t w, float c, float s) {
                const float p = act_lo<FP16>(w), q = act_hi<FP16>(w);
                return pack_act2<FP16>(p * c - q * s, q * c + p * s);
            };
            x[i] = pair(x[i], c[i], s[i]);
            y[i] = pair(y[i], c[W / 2 + i], s[W / 2 + i]);
        } else {
            const float p0 = act_lo<FP16>(x[i]), p1 = act_hi<FP16>(x[i]), q0 = act_lo<FP16>(y[i]), q1 = act_hi<FP16>(y[i]);
            const float c0 = c[2 * i], c1 = c[2 * i + 1], s0 = s[2 * i], s1 = s[2 * i + 1];
            x[i] = pack_act2<FP16>(p0 * c0 - q0 * s0, p1 * c1 - q1 * s1);
            y[i] = pack_act2<FP16>(q0 * c0 + p0 * s0, q1 * c1 + p1 * s1);
        }
    }
}

// W frequencies a thread, 8 or 4: rows on boundaries of 2 W bytes, half a multiple of W and dim of 2 W.  SPLIT: an axis may end inside the W
// frequencies, which two axes share then as a rule.  The results are not kept in the caches (32767 tokens: 110 us, 117
// kept); what is read may be there, from the projection (4096 tokens: 14.2 us, 17.5 past the caches).
template <int W, bool FP16, int TABLE, bool INTERLEAVED, bool SPLIT>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a)
{
    typedef uint32_t piece_t __attribute__((ext_vector_type(W / 2)));
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit >= a.units) return;
    const uint32_t rest = div_by(unit, a.pieces), piece = unit - rest * a.pieces.d;
    const uint32_t token = div_by(rest, a.rows), row = rest - token * a.rows.d;
    const int turned = a.half / W, f = (int)piece * W, which = (int)row >= a.heads[0], head = (int)row - (which ? a.heads[0] : 0);
    const bool copied = (int)piece >= turned;
    // first elements of the two pieces
    const int e0 = copied || INTERLEAVED ? (int)piece * 2 * W : f, e1 = copied || INTERLEAVED ? e0 + W : a.half + f;

    const uint16_t *from = a.in[which] + token * a.tok[which] + head * a.head[which];
    piece_t x = *reinterpret_cast<const piece_t *>(from + e0), y = *reinterpret_cast<const piece_t *>(from + e1);
    if (!copied) {
        float c[W], s[W];
        const int axis = axis_of(a, f), last = SPLIT ? axis_of(a, f + W - 1) : axis;
        const int64_t here = position(a, token, axis), there = SPLIT ? position(a, token, last) : here;
        turns_at<TABLE>(a, here, f, c, s);
        if (SPLIT && last != axis) {
            float lc[W], ls[W];
            turns_at<TABLE>(a, there, f, lc, ls);
#pragma unroll
            for (int i = 1; i < W; i++) {
                const int of = axis_of(a, f + i);
                if (of == last) c[i] = lc[i], s[i] = ls[i];
                else if (of != axis) turn_of<TABLE>(a, token, f + i, c[i], s[i]);
            }
        }
        turn<FP16, INTERLEAVED>(x, y, c, s);
    }
    uint16_t *to = a.out[which] + ((int64_t)token * a.heads[which] + head) * a.dim;
    __builtin_nontemporal_store(x, reinterpret_cast<piece_t *>(to + e0));
    __builtin_nontemporal_store(y, reinterpret_cast<piece_t *>(to + e1));
}

// Any width, alignment and strides: a thread per pair or copied element.  pieces = half + (dim - R).
template <int TABLE>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs a, int fp16)
{
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    if (unit >= a.units) return;
    const uint32_t rest = div_by(unit, a.pieces);
    const int piece = (int)(unit - rest * a.pieces.d);
    const uint32_t token = div_by(rest, a.rows);
    int head = (int)(rest - token * a.rows.d);
    const int which = head >= a.heads[0];
    head -= which ? a.heads[0] : 0;
    const uint16_t *row = a.in[which] + token * a.tok[which] + head * a.head[which];
    uint16_t *out = a.out[which] + ((int64_t)token * a.heads[which] + head) * a.dim;
    if (piece >= a.half) {
        out[a.half + piece] = row[a.half + piece];
        return;
    }
    const int e0 = a.interleaved ? 2 * piece : piece, e1 = a.interleaved ? e0 + 1 : a.half + piece;
    float c, s;
    turn_of<TABLE>(a, token, piece, c, s);
    const float p = fp16 ? act_1<1>(row[e0]) : act_1<0>(row[e0]), q = fp16 ? act_1<1>(row[e1]) : act_1<0>(row[e1]);
    const float x = p * c - q * s, y = q * c + p * s;
    const uint32_t w = fp16 ? pack_act2<1>(x, y) : pack_act2<0>(x, y);
    out[e0] = (uint16_t)w;
    out[e1] = (uint16_t)(w >> 16);
}

template <int W, bool FP16, int TABLE>
void launch_rope(const RopeArgs &a, bool split, unsigned blocks, hipStream_t s)
{
    const dim3 grid(blocks), block(256);
    const auto with = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, a); };
    if constexpr (W < 8)
        if (split) return a.interleaved ? with(rope_kernel<W, FP16, TABLE, true, true>) : with(rope_kernel<W, FP16, TABLE, false, true>);
    a.interleaved ? with(rope_kernel<W, FP16, TABLE, true, false>) : with(rope_kernel<W, FP16, TABLE, false, false>);
}
template <int W>
void launch_rope(const RopeArgs &a, bool fp16, int table, bool split, unsigned blocks, hipStream_t s)
{
    if (table == MI355_DTYPE_FP32) {
        if (fp16) launch_rope<W, true, 2>(a, split, blocks, s);
        else launch_rope<W, false, 2>(a, split, blocks, s);
    } else if (fp16) {
        launch_rope<W, true, 1>(a, split, blocks, s);
    } else {
        launch_rope<W, false, 0>(a, split, blocks, s);
    }
}

// Threads of one launch at most: they are numbered in 31 bits.
constexpr int64_t kUnitsPerLaunch = (int64_t)1 << 30;

} // namespace
} // namespace mi355

extern "C" int mi355_mrope(const void *positions, int positions_dtype, int64_t positions_stride_axis, int64_t positions_stride_token, int64_t axes,
                           const int64_t *sections, const void *query, const int64_t *query_stride, int64_t heads, const void *key,
                           const int64_t *key_stride, int64_t kv_heads, int dtype, const void *cos_sin, int cos_sin_dtype, int64_t cos_sin_stride,
                           int64_t max_positions, int64_t tokens, int64_t head_dim, int64_t rotary_dim, int interleaved, void *query_out,
                           void *key_out, void *stream)
{
    using namespace mi355;
    const bool fp16 = dtype == MI355_DTYPE_FP16;
    if (tokens < 0 || heads < 0 || kv_heads < 0 || max_positions < 0 || axes < 1 || (axes > 1 && !sections)) return MI355_ERR_BAD_ARGUMENT;
    if (rotary_dim < 2 || rotary_dim % 2 || head_dim < rotary_dim || (dtype != MI355_DTYPE_BF16 && !fp16)) return MI355_ERR_BAD_ARGUMENT;
    if (cos_sin_dtype != dtype && cos_sin_dtype != MI355_DTYPE_FP32) return MI355_ERR_BAD_ARGUMENT;
    if (positions_dtype != MI355_DTYPE_INT32 && positions_dtype != MI355_DTYPE_INT64) return MI355_ERR_BAD_ARGUMENT;
    if (axes > kAxes || heads > 65535 || kv_heads > 65535 || head_dim > 65536) return MI355_ERR_UNSUPPORTED;
    RopeArgs a;
    a.half = (int)(rotary_dim / 2);
    int64_t odd = 0;                                             // an axis ends inside w frequencies if it has a bit below w
    int64_t end = 0;
    for (int i = 0; i < kAxes; i++) {
        if (axes > 1 && i < axes) {
            if (sections[i] < 0 || sections[i] > a.half) return MI355_ERR_BAD_ARGUMENT;
            end += sections[i];
            odd |= end;
        } else if (axes == 1) {
            end = a.half;
        }
        a.end[i] = (int)end;
    }
    if (end != a.half) return MI355_ERR_BAD_ARGUMENT;
    if (tokens == 0 || heads + kv_heads == 0) return MI355_OK;
    if (!positions || (max_positions > 0 && !cos_sin) || (heads > 0 && (!query || !query_stride || !query_out)) ||
        (kv_heads > 0 && (!key || !key_stride || !key_out)))
        return MI355_ERR_BAD_ARGUMENT;
    const int table_bytes = cos_sin_dtype == MI355_DTYPE_FP32 ? 4 : 2, pos_bytes = positions_dtype == MI355_DTYPE_INT64 ? 8 : 4;
    if (!aligned(query, 2) || !aligned(key, 2) || !aligned(query_out, 2) || !aligned(key_out, 2) || !aligned(cos_sin, (size_t)table_bytes) ||
        !aligned(positions, (size_t)pos_bytes))
        return MI355_ERR_ALIGNMENT;
    a.heads[0] = (int)heads, a.heads[1] = (int)kv_heads;
    const void *const in[2] = {query, key};
    void *const out[2] = {query_out, key_out};
    const int64_t *const stride[2] = {query_stride, key_stride};
    for (int i = 0; i < 2; i++) {
        const bool any = a.heads[i] > 0;
        a.tok[i] = any ? stride[i][0] : 0, a.head[i] = any ? stride[i][1] : 0;
    }
    // What the frequencies of a thread have to be a multiple of, and the addresses and strides of two pieces with them
    const auto fits = [&](int w) {
        const int64_t table_piece = w * table_bytes < 16 ? w * table_bytes : 16;
        bool fit = rotary_dim % (2 * w) == 0 && head_dim % (2 * w) == 0 && aligned(cos_sin, (size_t)table_piece) && cos_sin_stride * table_bytes % table_piece == 0;
        for (int i = 0; i < 2; i++)
            fit = fit && (a.heads[i] == 0 || (aligned(in[i], 2 * w) && aligned(out[i], 2 * w) && a.tok[i] % w == 0 && a.head[i] % w == 0));
        return fit;
    };
    a.table = cos_sin;
    a.table_stride = cos_sin_stride;
    a.positions = max_positions;
    a.pos64 = positions_dtype == MI355_DTYPE_INT64;
    a.pos_axis = positions_stride_axis;
    a.pos_tok = positions_stride_token;
    a.axes = (int)axes;
    a.dim = (int)head_dim;
    a.interleaved = interleaved != 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    // Frequencies of a thread: eight, or four, also where an axis ends inside eight (16384 tokens of 40 heads of 128 on axes of 5, 7 and 52
    // frequencies, 344 MB: 75 us, 88 with eight, though 83 and 70 where heads are 64 wide and the table has 16 bits; heads of 80, 40 of them
    // turned, 77 us, one by one 308)
    const int w = fits(8) && odd % 8 == 0 ? 8 : fits(4) ? 4 : 1;
    const bool split = odd % w != 0;
    const int64_t all = heads + kv_heads, pieces = w > 1 ? head_dim / (2 * w) : a.half + (head_dim - rotary_dim);
    a.pieces = fast_div((uint32_t)pieces);
    a.rows = fast_div((uint32_t)all);
    const int64_t most = kUnitsPerLaunch / (all * pieces) > 0 ? kUnitsPerLaunch / (all * pieces) : 1;
    if (all * pieces > 0x7fffff00) return MI355_ERR_UNSUPPORTED;
    for (int64_t t0 = 0; t0 < tokens; t0 += most) {
        a.tokens = (uint32_t)(tokens - t0 < most ? tokens - t0 : most);
        a.units = (uint32_t)(a.tokens * all * pieces);
        a.pos = static_cast<const char *>(positions) + t0 * positions_stride_token * pos_bytes;
        for (int i = 0; i < 2; i++) {
            a.in[i] = static_cast<const uint16_t *>(in[i]) + t0 * a.tok[i];
            a.out[i] = static_cast<uint16_t *>(out[i]) + t0 * a.heads[i] * head_dim;
        }
        const unsigned blocks = (a.units + 255) / 256;
        if (w == 8) launch_rope<8>(a, fp16, cos_sin_dtype, split, blocks, s);
        else if (w == 4) launch_rope<4>(a, fp16, cos_sin_dtype, split, blocks, s);
        else if (cos_sin_dtype == MI355_DTYPE_FP32) hipLaunchKernelGGL(rope_any_kernel<2>, dim3(blocks), dim3(256), 0, s, a, fp16);
        else if (fp16) hipLaunchKernelGGL(rope_any_kernel<1>, dim3(blocks), dim3(256), 0, s, a, 1);
        else hipLaunchKernelGGL(rope_any_kernel<0>, dim3(blocks), dim3(256), 0, s, a, 0);
    }
    return check_launch();
}
