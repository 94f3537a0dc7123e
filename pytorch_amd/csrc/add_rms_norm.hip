// npu_add_rms_norm and npu_add_rms_norm_dynamic_quant for gfx950: the residual's addition, the root-mean-square norm of the
// sum and, for the W8A8 projections, its symmetric int8 quantisation per row, in one pass over memory.
//
// Per row of N elements, in float32, every operation rounded by itself:
//   s = x1 + x2 (x1 alone without a residual)     rstd = 1 / sqrt(sum s^2 / N + epsilon)     x = round16(s)
//   16 bits  y = round16((s * rstd) * gamma)
//   int8     u = s * gamma     step = max |u| / 127     code = rint_half_even(u / step)     scale = step * rstd
// rstd is one positive factor of a whole row, so it cancels in the codes: they are those of u, do not depend on the order in
// which squares are added, and the sum and the maximum are reduced together, behind one barrier.
//
// One row per workgroup (per wavefront or per 16 lanes, where rows are short), held in registers from its only load to its only store.
//
// Bound by memory where rows are many: 8191 rows of 8192 to int8, 470 MB, in 80 us, 5.9 TB/s; 2047 of 5128 in 16 bits, 84 MB, in 15.0 us,
// 5.6 TB/s.  Few rows are bound by the launch and one trip to memory and back: one row of 4096 to int8 in 2.9 us, 64 of 8192 in 3.8.
#include "common.h"
#include "weight_quant_common.h"

namespace mi355 {
namespace {

struct NormArgs {
    const uint16_t *x1, *x2;                 // x2: or null
    const void *gamma;
    void *y;                                 // [rows, cols] 16-bit or int8
    float *stat;                             // rstd or scale, [rows]; rstd may be null
    uint16_t *sum;                           // [rows, cols], with x2
    int64_t rows, x1_stride, x2_stride;
    int cols, gamma32;
    int once;                                // the inputs are more than the caches hold
    float epsilon;
};

// Eight consecutive elements, of which n (1 to 8) exist; ANY: from any address, else 16-byte aligned and whole, ONCE: past the caches.
template <bool ANY, bool ONCE = false>
__device__ __forceinline__ u32x4 load8(const uint16_t *p, int n)
{
    if constexpr (!ANY && ONCE) {
        return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
    } else if constexpr (!ANY) {
        return *reinterpret_cast<const u32x4 *>(p);
    } else {
        typedef u32x4 anywhere __attribute__((aligned(2)));
        if (n >= 8) return *reinterpret_cast<const anywhere *>(p);
        u32x4 v = {0, 0, 0, 0};
        for (int i = 0; i < n; i++) {
            const uint32_t w = (uint32_t)p[i] << (16 * (i & 1));
            v.x |= i / 2 == 0 ? w : 0, v.y |= i / 2 == 1 ? w : 0, v.z |= i / 2 == 2 ? w : 0, v.w |= i / 2 == 3 ? w : 0;
        }
        return v;
    }
}
template <bool ANY>
__device__ __forceinline__ void store8(uint16_t *p, u32x4 v, int n)
{
    if constexpr (!ANY) {
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(p));
    } else {
        typedef u32x4 anywhere __attribute__((aligned(2)));
        if (n >= 8) {
            *reinterpret_cast<anywhere *>(p) = v;
            return;
        }
        for (int i = 0; i < n; i++) p[i] = (uint16_t)((i < 4 ? (i < 2 ? v.x : v.y) : (i < 6 ? v.z : v.w)) >> (16 * (i & 1)));
    }
}
template <bool ANY>
__device__ __forceinline__ void store_codes(int8_t *p, u32x2 v, int n)
{
    if constexpr (!ANY) {
        __builtin_nontemporal_store(v, reinterpret_cast<u32x2 *>(p));
    } else {
        typedef u32x2 anywhere __attribute__((aligned(1)));
        if (n >= 8) {
            *reinterpret_cast<anywhere *>(p) = v;
            return;
        }
        for (int i = 0; i < n; i++) p[i] = (int8_t)((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
    }
}

template <bool FP16>
__device__ __forceinline__ void widen(u32x4 v, float (&f)[8])
{
#pragma unroll
    for (int i = 0; i < 4; i++) f[2 * i] = act_lo<FP16>(v[i]), f[2 * i + 1] = act_hi<FP16>(v[i]);
}
template <bool FP16>
__device__ __forceinline__ u32x4 narrow(const float (&f)[8])
{
    return u32x4{pack_act2<FP16>(f[0], f[1]), pack_act2<FP16>(f[2], f[3]), pack_act2<FP16>(f[4], f[5]), pack_act2<FP16>(f[6], f[7])};
}
// gamma of eight columns, of which n exist
template <bool ANY, bool FP16>
__device__ __forceinline__ void load_gamma(const NormArgs &a, int col, int n, float (&g)[8])
{
    if (a.gamma32) {
        const float *p = static_cast<const float *>(a.gamma) + col;
        if (!ANY || n >= 8) {
            typedef f32x4 anywhere __attribute__((aligned(4)));
            const f32x4 lo = *reinterpret_cast<const anywhere *>(p), hi = *reinterpret_cast<const anywhere *>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) g[i] = lo[i], g[i + 4] = hi[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) g[i] = i < n ? p[i] : 0.0f;
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(a.gamma) + col;
        widen<FP16>(ANY ? load8<true>(p, n) : *reinterpret_cast<const u32x4 *>(p), g);
    }
}

// Sum and largest bit pattern over the 64 lanes of a wavefront, in all of them: shifts within rows of 16 lanes, then the rows'
// last lanes handed on.  The sum is that of neighbours, pairs, fours and eights in a row, then (row 3 + row 2) + (row 1 + row 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t shifted(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ void reduce_step(float &sum, uint32_t &top)
{
    sum += __uint_as_float(shifted<CTRL, ROWS>(__float_as_uint(sum)));
    top = max(top, shifted<CTRL, ROWS>(top));
}
__device__ __forceinline__ void reduce_wave(float &sum, uint32_t &top)
{
    reduce_step<0x111, 0xf>(sum, top);           // row_shr:1, 2, 4, 8
    reduce_step<0x112, 0xf>(sum, top);
    reduce_step<0x114, 0xf>(sum, top);
    reduce_step<0x118, 0xf>(sum, top);
    reduce_step<0x142, 0xa>(sum, top);           // row_bcast:15 into rows 1 and 3
    reduce_step<0x143, 0xc>(sum, top);           // row_bcast:31 into rows 2 and 3
    sum = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(sum), 63));
    top = (uint32_t)__builtin_amdgcn_readlane((int)top, 63);
}
// over 16 lanes, in all of them: neighbours, pairs, mirrored fours, mirrored eights, so the same sum as that of a wavefront's row
__device__ __forceinline__ void reduce_16(float &sum, uint32_t &top)
{
    reduce_step<0xb1, 0xf>(sum, top);
    reduce_step<0x4e, 0xf>(sum, top);
    reduce_step<0x141, 0xf>(sum, top);
    reduce_step<0x140, 0xf>(sum, top);
}
// the same over the threads of a row: 16 lanes, a wavefront, or the wavefronts of a workgroup
template <int TPR>
__device__ __forceinline__ void reduce_row(float &sum, uint32_t &top, float (&sums)[16], uint32_t (&tops)[16])
{
    constexpr int WAVES = TPR / 64;
    if constexpr (TPR == 16) reduce_16(sum, top);
    else reduce_wave(sum, top);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum, tops[threadIdx.x >> 6] = top;
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) sum += sums[w], top = max(top, tops[w]);
    }
}

// u / step, rounded to an integer, for |u| <= 127 * step.  With r = 1 / step correctly rounded, one correction of u * r by its
// residual gives one of the two floats next to the quotient, and by Markstein's theorem a second one the correctly rounded
// quotient, where nothing leaves the normal range: for a step in [2^-60, 2^60] only quotients below 2^-40 do, which round to 0
// either way.  The sum with 1.5 * 2^23 is rounded to an integer, ties to even, whose low byte is the code.
struct Codes {
    float step, r;
    bool none, safe;
    __device__ explicit Codes(float top) : step(top / 127.0f), r(1.0f / step), none(!(top > 0.0f)), safe(step >= 0x1p-60f && step <= 0x1p60f) {}
    __device__ __forceinline__ u32x2 operator()(const float (&u)[8]) const
    {
        uint32_t c[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (safe) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float q = u[i] * r;
                q = __builtin_fmaf(__builtin_fmaf(-step, q, u[i]), r, q);
                q = __builtin_fmaf(__builtin_fmaf(-step, q, u[i]), r, q);
                c[i] = __float_as_uint(q + 12582912.0f);
            }
        } else if (!none) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float q = __builtin_rintf(u[i] / step);
                q = q > 127.0f ? 127.0f : q;
                q = q < -127.0f ? -127.0f : q;                   // NaN falls through both tests and converts to 0
                c[i] = (uint32_t)(int)q;
            }
        }
        return u32x2{pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7])};
    }
};

__device__ __forceinline__ float rstd_of(float sum, const NormArgs &a) { return 1.0f / sqrtf(sum / (float)a.cols + a.epsilon); }

// s of eight columns, and their part of the sum of squares
template <bool FP16>
__device__ __forceinline__ void add8(const NormArgs &a, u32x4 v1, u32x4 v2, float (&s)[8], float &sum)
{
    widen<FP16>(v1, s);
    if (a.x2) {
        float t[8];
        widen<FP16>(v2, t);
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] = s[i] + t[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) sum = __builtin_fmaf(s[i], s[i], sum);
}

// TPR threads of a workgroup of BLOCK per row, VPT pieces of eight columns each.
template <int BLOCK, int TPR, int VPT, bool INT8, bool FP16, bool ANY>
__global__ __launch_bounds__(BLOCK) void norm_rows_kernel(NormArgs a)
{
    static_assert(TPR == 16 || TPR == 64 || TPR == BLOCK, "a row belongs to 16 lanes, a wavefront or the workgroup");
    __shared__ float sums[16];
    __shared__ uint32_t tops[16];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (BLOCK / TPR) + threadIdx.x / TPR;
    if (row >= a.rows) return;                                   // all threads of a row, and no barrier follows if those are not the workgroup
    const uint16_t *x1 = a.x1 + row * a.x1_stride, *x2 = a.x2 + row * a.x2_stride;

    u32x4 v1[VPT], v2[VPT];
    const auto load = [&](auto eight) {
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int col = (t + i * TPR) * 8;
            v1[i] = v2[i] = u32x4{0, 0, 0, 0};
            if (col < a.cols) {
                v1[i] = eight(x1 + col, a.cols - col);
                if (a.x2) v2[i] = eight(x2 + col, a.cols - col);
            }
        }
    };
    if (!ANY && a.once) load([](const uint16_t *p, int n) { return load8<ANY, true>(p, n); });
    else load([](const uint16_t *p, int n) { return load8<ANY>(p, n); });
    // 16 lanes of four pieces add the squares of a row as a wavefront of one piece a lane does, a row of 16 lanes for each piece, so that a
    // row's scale does not depend on the number of rows, which chooses between them (12 more additions: 8191 rows of 512 7.35 and 7.31 us)
    constexpr bool AS_WAVE = TPR == 16 && VPT == 4;
    float s[VPT][8], g[VPT][8], sums_of[AS_WAVE ? VPT : 1] = {};
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int col = (t + i * TPR) * 8;
        if (col < a.cols) {
            load_gamma<ANY, FP16>(a, col, a.cols - col, g[i]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) g[i][k] = 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int col = (t + i * TPR) * 8;
        add8<FP16>(a, v1[i], v2[i], s[i], sums_of[AS_WAVE ? i : 0]);
        if (a.x2 && col < a.cols) store8<ANY>(a.sum + row * a.cols + col, narrow<FP16>(s[i]), a.cols - col);
        if constexpr (INT8) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                s[i][k] = s[i][k] * g[i][k];
                top = max(top, __float_as_uint(s[i][k]) & 0x7fffffffu);
            }
        }
    }
    if constexpr (AS_WAVE) {
        uint32_t unused = 0;
        reduce_16(sums_of[0], top);
#pragma unroll
        for (int i = 1; i < VPT; i++) reduce_16(sums_of[i], unused);
        sums_of[0] = (sums_of[3] + sums_of[2]) + (sums_of[1] + sums_of[0]);
    } else {
        reduce_row<TPR>(sums_of[0], top, sums, tops);
    }
    const float rstd = rstd_of(sums_of[0], a);
    if constexpr (INT8) {
        const Codes codes(__uint_as_float(top));
        if (t == 0) a.stat[row] = codes.step * rstd;
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int col = (t + i * TPR) * 8;
            if (col < a.cols) store_codes<ANY>(static_cast<int8_t *>(a.y) + row * a.cols + col, codes(s[i]), a.cols - col);
        }
    } else {
        if (t == 0 && a.stat) a.stat[row] = rstd;
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int col = (t + i * TPR) * 8;
#pragma unroll
            for (int k = 0; k < 8; k++) s[i][k] = (s[i][k] * rstd) * g[i][k];
            if (col < a.cols) store8<ANY>(static_cast<uint16_t *>(a.y) + row * a.cols + col, narrow<FP16>(s[i]), a.cols - col);
        }
    }
}

// Rows longer than registers hold: read again for the second half, from the caches as a rule.
template <bool INT8, bool FP16>
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs a)
{
    __shared__ float sums[16];
    __shared__ uint32_t tops[16];
    const int64_t row = blockIdx.x;
    const uint16_t *x1 = a.x1 + row * a.x1_stride, *x2 = a.x2 + row * a.x2_stride;
    float sum = 0.0f;
    uint32_t top = 0;
    const auto piece = [&](int col, float (&s)[8], float (&g)[8], float &sum) {
        const u32x4 v1 = load8<true>(x1 + col, a.cols - col), v2 = a.x2 ? load8<true>(x2 + col, a.cols - col) : u32x4{0, 0, 0, 0};
        load_gamma<true, FP16>(a, col, a.cols - col, g);
        add8<FP16>(a, v1, v2, s, sum);
    };
    for (int64_t at = (int64_t)threadIdx.x * 8; at < a.cols; at += 1024 * 8) {
        float s[8], g[8];
        piece((int)at, s, g, sum);
#pragma unroll
        for (int k = 0; k < 8; k++) top = max(top, __float_as_uint(s[k] * g[k]) & 0x7fffffffu);
    }
    reduce_row<1024>(sum, top, sums, tops);
    const float rstd = rstd_of(sum, a);
    const Codes codes(__uint_as_float(top));
    if (threadIdx.x == 0 && a.stat) a.stat[row] = INT8 ? codes.step * rstd : rstd;
    for (int64_t at = (int64_t)threadIdx.x * 8; at < a.cols; at += 1024 * 8) {
        const int col = (int)at, n = a.cols - col;
        float s[8], g[8], unused = 0.0f;
        piece(col, s, g, unused);
        if (a.x2) store8<true>(a.sum + row * a.cols + col, narrow<FP16>(s), n);
#pragma unroll
        for (int k = 0; k < 8; k++) s[k] = INT8 ? s[k] * g[k] : (s[k] * rstd) * g[k];
        if constexpr (INT8) store_codes<true>(static_cast<int8_t *>(a.y) + row * a.cols + col, codes(s), n);
        else store8<true>(static_cast<uint16_t *>(a.y) + row * a.cols + col, narrow<FP16>(s), n);
    }
}

template <int BLOCK, int TPR, int VPT, bool INT8, bool FP16>
void launch_rows(const NormArgs &a, bool any, hipStream_t s)
{
    const dim3 grid((unsigned)((a.rows + BLOCK / TPR - 1) / (BLOCK / TPR)));
    if (any) hipLaunchKernelGGL((norm_rows_kernel<BLOCK, TPR, VPT, INT8, FP16, true>), grid, dim3(BLOCK), 0, s, a);
    else hipLaunchKernelGGL((norm_rows_kernel<BLOCK, TPR, VPT, INT8, FP16, false>), grid, dim3(BLOCK), 0, s, a);
}

template <bool INT8, bool FP16>
void launch_norm(const NormArgs &a, bool any, hipStream_t s)
{
    // Two pieces a thread from 1025 columns on, as long as a workgroup has the threads: 64 rows of 8192 take 5.0 us with four pieces for 256
    // threads, 3.9 with two for 512, 3.8 with one for 1024; 8191 rows to int8 85, 82 and 87; one row of 4096 3.1 us with two for 256 or one for 512.
    const int pieces = (a.cols - 1) / 8 + 1;
    // Up to 256 columns 16 lanes a row: a wavefront's lanes would idle, and a row's divisions count for it alone (20000 rows of 72 7.7 and 4.4 us, to
    // int8 15.4 and 6.5; 64 of 64 2.9 and 2.2; 1000 of 200 2.8 and 3.2).  Up to 512 they need four pieces a thread, which pays for many
    // rows to int8 (8191 of 512 9.6 and 7.9 us, of 300 11.2 and 8.9; in 16 bits 6.9 and 7.7; 1000 of 512 3.8 and 5.1).
    if (pieces <= 16) launch_rows<256, 16, 1, INT8, FP16>(a, any, s);
    else if (pieces <= 32) launch_rows<256, 16, 2, INT8, FP16>(a, any, s);
    else if (pieces <= 64 && INT8 && a.rows >= 4096) {
        if constexpr (INT8) launch_rows<256, 16, 4, INT8, FP16>(a, any, s);
    } else if (pieces <= 64) launch_rows<256, 64, 1, INT8, FP16>(a, any, s);
    else if (pieces <= 256) launch_rows<256, 256, 1, INT8, FP16>(a, any, s);
    else if (pieces <= 512) launch_rows<256, 256, 2, INT8, FP16>(a, any, s);
    else if (pieces <= 1024) launch_rows<512, 512, 2, INT8, FP16>(a, any, s);
    else if (pieces <= 2048) launch_rows<1024, 1024, 2, INT8, FP16>(a, any, s);
    else if (pieces <= 4096) launch_rows<1024, 1024, 4, INT8, FP16>(a, any, s);
    else hipLaunchKernelGGL((norm_long_kernel<INT8, FP16>), dim3((unsigned)a.rows), dim3(1024), 0, s, a);
}

// Rows of one launch at most: the threads of a grid are numbered in 32 bits (beyond, it wraps without an error).
constexpr int64_t kRowsPerLaunch = (int64_t)1 << 21;

template <bool INT8>
int add_rms_norm(const void *x1, const void *x2, int dtype, const void *gamma, int gamma_dtype, void *y, float *stat, void *x, int64_t rows,
                 int64_t cols, int64_t x1_stride, int64_t x2_stride, float epsilon, void *stream)
{
    const bool fp16 = dtype == MI355_DTYPE_FP16;
    if (rows < 0 || cols < 0 || (dtype != MI355_DTYPE_BF16 && !fp16) || (gamma_dtype != dtype && gamma_dtype != MI355_DTYPE_FP32) || !(epsilon >= 0.0f))
        return MI355_ERR_BAD_ARGUMENT;
    if (rows == 0 || cols == 0) return MI355_OK;
    if (!x1 || !gamma || !y || (x2 != nullptr) != (x != nullptr) || (INT8 && !stat)) return MI355_ERR_BAD_ARGUMENT;
    if (cols > 0x7ffffff0) return MI355_ERR_UNSUPPORTED;
    if (!aligned(x1, 2) || !aligned(x2, 2) || !aligned(x, 2) || !aligned(gamma, gamma_dtype == MI355_DTYPE_FP32 ? 4 : 2) || !aligned(y, INT8 ? 1 : 2) ||
        !aligned(stat, 4))
        return MI355_ERR_ALIGNMENT;
    NormArgs a;
    a.gamma = gamma;
    a.gamma32 = gamma_dtype == MI355_DTYPE_FP32;
    a.x1_stride = x1_stride;
    a.x2_stride = x2 ? x2_stride : 0;
    a.cols = (int)cols;
    a.epsilon = epsilon;
    const bool any = cols % 8 || x1_stride % 8 || a.x2_stride % 8 || !aligned(x1, 16) || !aligned(x2, 16) || !aligned(x, 16) || !aligned(gamma, 16) ||
                     !aligned(y, INT8 ? 8 : 16);
    // Inputs that fit into the Infinity Cache may still be there, from the operators that wrote them (2047 rows of 5128: 15.0 us, 17.0 past
    // the caches; 8192 of 2048, 67 MB: 22.4 and 25); larger ones only drive each other out (8192 of 4096, 134 MB: 50 us, 48 past the
    // caches; 8191 of 8192 to int8 85 and 82; all of them 2 to 4 us less since the loads of a row stand together).
    a.once = rows * cols * (x2 ? 4 : 2) > (int64_t)96 << 20;
    for (int64_t r0 = 0; r0 < rows; r0 += kRowsPerLaunch) {
        a.rows = rows - r0 < kRowsPerLaunch ? rows - r0 : kRowsPerLaunch;
        a.x1 = static_cast<const uint16_t *>(x1) + r0 * x1_stride;
        a.x2 = x2 ? static_cast<const uint16_t *>(x2) + r0 * x2_stride : nullptr;
        a.y = static_cast<char *>(y) + r0 * cols * (INT8 ? 1 : 2);
        a.stat = stat ? stat + r0 : nullptr;
        a.sum = x ? static_cast<uint16_t *>(x) + r0 * cols : nullptr;
        if (fp16) launch_norm<INT8, true>(a, any, static_cast<hipStream_t>(stream));
        else launch_norm<INT8, false>(a, any, static_cast<hipStream_t>(stream));
    }
    return check_launch();
}

} // namespace
} // namespace mi355

extern "C" int mi355_add_rms_norm(const void *x1, const void *x2, int dtype, const void *gamma, int gamma_dtype, void *y, float *rstd, void *x,
                                  int64_t rows, int64_t cols, int64_t x1_stride, int64_t x2_stride, float epsilon, void *stream)
{
    return mi355::add_rms_norm<false>(x1, x2, dtype, gamma, gamma_dtype, y, rstd, x, rows, cols, x1_stride, x2_stride, epsilon, stream);
}

extern "C" int mi355_add_rms_norm_dynamic_quant(const void *x1, const void *x2, int dtype, const void *gamma, int gamma_dtype, int8_t *y, float *scale,
                                                void *x, int64_t rows, int64_t cols, int64_t x1_stride, int64_t x2_stride, float epsilon, void *stream)
{
    return mi355::add_rms_norm<true>(x1, x2, dtype, gamma, gamma_dtype, y, scale, x, rows, cols, x1_stride, x2_stride, epsilon, stream);
}
