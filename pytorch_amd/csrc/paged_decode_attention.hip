// npu_paged_decode_attention for gfx950: one new token per sequence against the tokens of a paged key-value cache.
//
// Per sequence b and query head h (key/value head h / group), over the positions j that are seen:
//   z_j = scale * log2(e) * sum_d q_d k_jd      m = max z_j      l = sum_j 2^(z_j - m)
//   out_d = sum_j 2^(z_j - m) v_jd / l          lse = (m + log2 l) / log2(e)
// Every cached byte is read once and used for `group` heads, so the bound is the cache's bytes over the memory's rate.
//
// One wavefront takes 32 positions at a time and keeps running (m, l, out) for up to 16 heads:
//   scores   C[position][head] = K[position][d] Q[d][head]: MFMA 16x16x32, keys as the first operand straight from memory
//            (a lane holds 8 consecutive d of one position), the heads' queries as the second, in registers for good.
//            A lane ends up with 4 consecutive positions (of each half of the 32) of ONE head, so the statistics of a head
//            are per-lane scalars: one maximum over 8 registers and two lane exchanges.
//   outputs  C[d][head] = V^T[d][position] P[position][head]: the lane's 8 probabilities already are the second operand,
//            if the positions are numbered lane group by lane group; the first operand needs, for one d, the same 8
//            positions side by side, so a lane loads 8 (4) consecutive d of its 8 positions' rows - whole cache lines - and
//            transposes 2x2 blocks of 16-bit values with one byte permute per register.
// Nothing passes through LDS but the sums of the four wavefronts of a workgroup when they finish a stretch of positions.
//
// int8 caches: codes become 16-bit numbers exactly; the scale of a position's keys multiplies its score, the scale of its
// values multiplies its probability, in float32.
//
// Work is dealt out on the device, because the lengths are known only there: the positions of every (sequence, head) pair
// are cut into units of 128, all units are numbered, and every workgroup takes the same number of consecutive ones.  A pair
// that lies within one workgroup is finished there; of a pair that is cut, every workgroup leaves (sums, m, l) in the
// workspace and the join kernel adds them in order.
#include "paged_cache.h"
#include "weight_quant_common.h"

namespace mi355 {
namespace {

constexpr int kUnit = 128;                   // positions per unit: 32 for each wavefront of a workgroup
constexpr int kHeads = 16;                   // query heads of one tile
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

struct AttnArgs {
    PagedCache cache;
    const uint16_t *q;
    int64_t q_batch, q_head;                 // elements
    uint16_t *out;
    float *lse;                              // [batch, heads] or null
    const int32_t *table, *lens;
    int64_t table_stride;
    const uint8_t *mask;
    int64_t mask_stride;
    float *part;                             // [workgroups][2][rows][DP]
    float *part_ml;                          // [workgroups][2][kHeads][2]: maximum, sum
    float *scores;                           // [batch * heads][score_pitch] z_j, or null
    float *lse2;                             // [batch * heads] m + log2 l, with scores
    float *sums;
    int64_t score_pitch, sums_batch, sums_head;
    int batch, heads, group, rows, tiles, pairs, workgroups;    // pairs = key/value heads * tiles, of one sequence
    int capacity;                            // max_blocks * block_size
    float scale2;                            // scale * log2(e)
    int vec;                                 // rows are read in 16-byte (int8: up to 16-byte) pieces
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform64(int64_t v)
{
    return (int64_t)(((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32) | (uint32_t)uniform((int)v));
}

// What sums over a maximum `m` count for under the maximum `top`.  Nothing seen yet: m = -infinity, sums 0 - or NaN, from NaN
// scores, which the product with 0 keeps.
__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top); }

__device__ __forceinline__ int length_of(const AttnArgs &a, int b) { return min(max(a.lens[b], 0), a.capacity); }
__device__ __forceinline__ uint32_t units_of(int len) { return ((uint32_t)len + kUnit - 1) / kUnit; }

// The numbering of units: sequence by sequence, in it pair by pair.  `before(b)`: units of one pair in the sequences before
// b; total: in all.  Thread t of 256 counts a run of consecutive sequences.
struct Numbering {
    uint32_t run_before, run_sum, total;
    int run, first;                          // sequences per thread, the thread's first

    __device__ Numbering(const AttnArgs &a, uint32_t *lds /* 4 */)
    {
        run = (a.batch + 255) / 256;
        first = threadIdx.x * run;
        run_sum = 0;
        for (int i = 0; i < run && first + i < a.batch; i++) run_sum += units_of(length_of(a, first + i));
        uint32_t scan = run_sum;
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)scan, off, 64);
            if (lane >= off) scan += o;
        }
        if (lane == 63) lds[threadIdx.x >> 6] = scan;
        __syncthreads();
        run_before = scan - run_sum;
        total = 0;
        for (int w = 0; w < 4; w++) {
            if (w < (int)(threadIdx.x >> 6)) run_before += lds[w];
            total += lds[w];
        }
        total = (uint32_t)uniform((int)total);
    }
};

__device__ __forceinline__ int64_t share_of(const AttnArgs &a, int64_t all) { return (all + a.workgroups - 1) / a.workgroups; }

// Eight (four) 16-bit values or bytes from any address: what the vector loads do for aligned rows.
template <int BYTES>
__device__ __forceinline__ void load_piece(uint32_t *to, const char *from, bool vec, int valid_bytes)
{
    if (valid_bytes >= BYTES && vec) {
        __builtin_memcpy(to, __builtin_assume_aligned(from, BYTES), BYTES);
        return;
    }
#pragma unroll
    for (int w = 0; w < BYTES / 4; w++) {
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (w * 4 + i < valid_bytes) v |= (uint32_t)(uint8_t)from[w * 4 + i] << (8 * i);
        to[w] = v;
    }
}

template <int W>
__device__ __forceinline__ void buffer_load(uint32_t (&to)[W], __amdgpu_buffer_rsrc_t rsrc, uint32_t offset)
{
    if constexpr (W == 4) {
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, offset, 0, 0);
        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
    } else if constexpr (W == 2) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rsrc, offset, 0, 0);
        to[0] = v.x, to[1] = v.y;
    } else {
        to[0] = __builtin_amdgcn_raw_buffer_load_b32(rsrc, offset, 0, 0);
    }
}

// DP: head_dim rounded up to 64, 128 or 256.  QT: type of q and out (0 bf16, 1 fp16).  UNI: the 16 positions of a half tile
// lie in one block at a small stride, so that addresses are one scalar descriptor per half and per-lane constants.
template <int DP, bool QUANT, int QT, bool UNI>
struct Tile {
    static constexpr int ES = QUANT ? 1 : 2;
    static constexpr int NCH = DP / 32;                          // chunks of 32 d, one MFMA each
    static constexpr int KL = QUANT ? NCH / 2 : NCH;             // 16-byte loads of a key row per lane
    static constexpr int PE = DP >= 128 ? 8 : 4;                 // consecutive d of a value row per lane and piece
    static constexpr int NP = DP / (16 * PE);
    static constexpr int VW = PE * ES / 4;                       // registers of a piece

    uint32_t k[2][KL][4];
    uint32_t v[2][4][NP][VW];
    float ks[2][4], vs[2][4];
    int valid_rows[2];                                           // UNI
    uint32_t valid;                                              // bit 4 s + r: position s * 16 + lane group * 4 + r is seen
};

template <int DP, bool QUANT, int QT, bool UNI>
__global__ __launch_bounds__(256) void paged_decode_kernel(AttnArgs a)
{
    using T = Tile<DP, QUANT, QT, UNI>;
    constexpr int PT = QUANT ? 0 : QT;                           // type of the probabilities and value images
    // fp16 probabilities are 2^14 times as large, so that ones down to 2^-38 of the largest keep their place
    constexpr float kShift = PT == 1 ? 14.0f : 0.0f;
    constexpr int RP = 128 + 4;                                  // row pitch of the sums in LDS, 4 words past a bank cycle
    __shared__ float red[4][kHeads][RP];
    __shared__ float ml[4][kHeads][2];
    __shared__ int where[4];
    __shared__ uint32_t scan[4];

    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int D = a.cache.dim;
    int64_t x, x_end;
    int b, pair, unit, units;
    {
        const Numbering n(a, scan);
        const int64_t all = (int64_t)n.total * a.pairs, share = share_of(a, all);
        x = (int64_t)blockIdx.x * share;
        x_end = min(x + share, all);
        if (x >= all) return;
        const uint32_t y = (uint32_t)((uint64_t)x / (uint32_t)a.pairs);
        if (y >= n.run_before && y - n.run_before < n.run_sum) {           // one thread
            uint32_t before = n.run_before;
            int i = n.first;
            for (;; i++) {
                const uint32_t u = units_of(length_of(a, i));
                if (y - before < u) break;
                before += u;
            }
            const uint32_t u = units_of(length_of(a, i));
            const uint64_t in = (uint64_t)x - (uint64_t)before * (uint32_t)a.pairs;
            where[0] = i;
            where[1] = (int)(in / u);
            where[2] = (int)(in % u);
        }
        __syncthreads();
        b = uniform(where[0]), pair = uniform(where[1]), unit = uniform(where[2]);
    }
    int slot = 0;
    const int64_t kstep = a.cache.key.token, vstep = a.cache.value.token;
    uint32_t koff[T::KL], voff[4][T::NP];
    if constexpr (UNI) {
#pragma unroll
        for (int c = 0; c < T::KL; c++) {
            const int d = QUANT ? c * 64 + g * 16 : c * 32 + g * 8;
            koff[c] = d < D ? (uint32_t)(col * kstep) + d * T::ES : kOutOfRange;
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int h = 0; h < T::NP; h++) {
                const int d = h * 128 + col * T::PE;
                voff[j][h] = d < D ? (uint32_t)((g * 4 + j) * vstep) + d * T::ES : kOutOfRange;
            }
    }

    while (x < x_end) {
        int len = uniform(length_of(a, b));
        units = (int)units_of(len);
        while (units == 0) {                                     // the sequence is over: the next one that has positions
            b++;
            len = uniform(length_of(a, b));
            units = (int)units_of(len);
        }
        const int last = (int)min((int64_t)units, unit + (x_end - x));     // units [unit, last) of this pair
        const int kvh = pair / a.tiles, head0 = kvh * a.group + (pair % a.tiles) * kHeads;
        const int rows = min(kHeads, (kvh + 1) * a.group - head0);
        const int end = min(len, last * kUnit);

        u32x4 q[T::NCH];
        {
            const uint16_t *row = a.q + b * a.q_batch + (head0 + min(col, rows - 1)) * a.q_head;
#pragma unroll
            for (int c = 0; c < T::NCH; c++) {
                const int d = QUANT ? (c / 2) * 64 + g * 16 + (c % 2) * 8 : c * 32 + g * 8;
                uint32_t w[4];
                load_piece<16>(w, reinterpret_cast<const char *>(row + d), a.vec, col < rows ? 2 * (D - d) : 0);
                q[c] = u32x4{w[0], w[1], w[2], w[3]};
            }
        }
        float m = -INFINITY, l = 0.0f;
        f32x4 acc[T::NP][T::PE] = {};

        const int32_t *table = a.table + b * a.table_stride;
        const int64_t khead = kvh * a.cache.key.head, vhead = kvh * a.cache.value.head;

        T t;
        uint32_t lane_slot[2];                                   // !UNI: slot of position s * 16 + col, or ~0
        // where the tile's rows are
        const auto place = [&](int tile, int64_t (&kb)[2], int64_t (&vb)[2], int64_t (&sb)[2]) {
            (void)sb;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const int key0 = tile * 32 + s * 16;
                if constexpr (UNI) {
                    int n = min(max(end - key0, 0), 16);
                    const uint32_t block = div_by((uint32_t)key0, a.cache.page);
                    const uint32_t off = (uint32_t)key0 - block * a.cache.page.d;
                    int id = n > 0 ? table[block] : 0;
                    if ((uint32_t)id >= (uint32_t)a.cache.num_blocks) n = 0, id = 0;
                    t.valid_rows[s] = uniform(n);
                    kb[s] = uniform64(id * a.cache.key.block + off * kstep + khead);
                    vb[s] = uniform64(id * a.cache.value.block + off * vstep + vhead);
                    lane_slot[s] = (uint32_t)uniform((int)((uint32_t)id * a.cache.page.d + off));
                } else {
                    const int key = key0 + col;
                    const uint32_t block = div_by((uint32_t)key, a.cache.page);
                    const int id = key < end ? table[block] : -1;
                    lane_slot[s] = (uint32_t)id < (uint32_t)a.cache.num_blocks ? (uint32_t)id * a.cache.page.d + ((uint32_t)key - block * a.cache.page.d) : ~0u;
                }
            }
        };
        const auto load_k = [&](const int64_t (&kb)[2]) {
#pragma unroll
            for (int s = 0; s < 2; s++) {
                if constexpr (UNI) {
                    const int n = t.valid_rows[s];
                    const __amdgpu_buffer_rsrc_t r = make_rsrc(a.cache.key.base + kb[s], n > 0 ? (uint32_t)((n - 1) * kstep) + D * T::ES : 0);
#pragma unroll
                    for (int c = 0; c < T::KL; c++) buffer_load<4>(t.k[s][c], r, koff[c]);
                } else {
                    const uint32_t sl = lane_slot[s];
                    const char *row = a.cache.key.base + (sl == ~0u ? 0 : a.cache.offset(a.cache.key, sl, kvh));
#pragma unroll
                    for (int c = 0; c < T::KL; c++) {
                        const int d = QUANT ? c * 64 + g * 16 : c * 32 + g * 8;
                        load_piece<16>(t.k[s][c], row + d * T::ES, a.vec, sl == ~0u ? 0 : (D - d) * T::ES);
                    }
                }
            }
        };
        const auto load_v = [&](const int64_t (&vb)[2]) {
#pragma unroll
            for (int s = 0; s < 2; s++) {
                if constexpr (UNI) {
                    const int n = t.valid_rows[s];
                    const __amdgpu_buffer_rsrc_t r = make_rsrc(a.cache.value.base + vb[s], n > 0 ? (uint32_t)((n - 1) * vstep) + D * T::ES : 0);
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int h = 0; h < T::NP; h++) buffer_load<T::VW>(t.v[s][j][h], r, voff[j][h]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t sl = (uint32_t)__shfl((int)lane_slot[s], g * 4 + j, 64);
                        const char *row = a.cache.value.base + (sl == ~0u ? 0 : a.cache.offset(a.cache.value, sl, kvh));
#pragma unroll
                        for (int h = 0; h < T::NP; h++) {
                            const int d = h * 128 + col * T::PE;
                            load_piece<T::VW * 4>(t.v[s][j][h], row + d * T::ES, a.vec, sl == ~0u ? 0 : (D - d) * T::ES);
                        }
                    }
                }
            }
        };
        // which positions are seen, and their scales
        const auto load_seen = [&](int tile) {
            t.valid = 0;
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = g * 4 + r, key = tile * 32 + s * 16 + i;
                    bool seen;
                    uint32_t sl;
                    if constexpr (UNI) {
                        seen = i < t.valid_rows[s];
                        sl = lane_slot[s] + i;
                    } else {
                        sl = (uint32_t)__shfl((int)lane_slot[s], i, 64);
                        seen = sl != ~0u;
                    }
                    if constexpr (QUANT) {
                        t.ks[s][r] = seen ? *reinterpret_cast<const float *>(a.cache.key_scale.base + a.cache.offset(a.cache.key_scale, sl, kvh)) : 0.0f;
                        t.vs[s][r] = seen ? *reinterpret_cast<const float *>(a.cache.value_scale.base + a.cache.offset(a.cache.value_scale, sl, kvh)) : 0.0f;
                    }
                    if (a.mask && seen) seen = a.mask[b * a.mask_stride + key] == 0;
                    t.valid |= (uint32_t)seen << (4 * s + r);
                }
        };

        const int t_end = (end + 31) / 32;
        for (int tile = unit * 4 + wave; tile < t_end; tile += 4) {
            int64_t kb[2], vb[2], sb[2];
            place(tile, kb, vb, sb);
            load_k(kb);
            load_v(vb);
            load_seen(tile);
            f32x4 z[2] = {};
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int c = 0; c < T::NCH; c++) {
                    u32x4 image;
                    if constexpr (QUANT) {
                        const u32x2 lo = sbytes_act4<QT>(t.k[s][c / 2][(c % 2) * 2]), hi = sbytes_act4<QT>(t.k[s][c / 2][(c % 2) * 2 + 1]);
                        image = u32x4{lo.x, lo.y, hi.x, hi.y};
                    } else {
                        image = u32x4{t.k[s][c][0], t.k[s][c][1], t.k[s][c][2], t.k[s][c][3]};
                    }
                    z[s] = mfma_act<QT>(image, q[c], z[s]);
                }
            float top = -INFINITY;
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    z[s][r] = QUANT ? z[s][r] * (a.scale2 * t.ks[s][r]) : z[s][r] * a.scale2;
                    if (!((t.valid >> (4 * s + r)) & 1)) z[s][r] = -INFINITY;
                    top = fmaxf(top, z[s][r]);
                }
            if (a.scores && col < rows) {
                float *to = a.scores + ((int64_t)b * a.heads + head0 + col) * a.score_pitch + tile * 32 + g * 4;
#pragma unroll
                for (int s = 0; s < 2; s++)
                    if (tile * 32 + s * 16 + g * 4 < end) *reinterpret_cast<f32x4 *>(to + s * 16) = z[s];
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (__any(top > m)) {
                const float higher = fmaxf(m, top);
                const float f = weight_of(m, higher);
                m = higher;
                l *= f;
#pragma unroll
                for (int h = 0; h < T::NP; h++)
#pragma unroll
                    for (int i = 0; i < T::PE; i++) acc[h][i] *= f;
            }
            const float base = m == -INFINITY ? 0.0f : m - kShift;
            float p[8];
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    p[4 * s + r] = __builtin_amdgcn_exp2f(z[s][r] - base);
                    l += p[4 * s + r];
                }
            // a value that is not seen must not turn 0 * NaN into NaN
            if (!__all(t.valid == 0xffu)) {
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t keep = (t.valid >> (4 * s + j)) & 1 ? ~0u : 0u;
#pragma unroll
                        for (int h = 0; h < T::NP; h++)
#pragma unroll
                            for (int w = 0; w < T::VW; w++) t.v[s][j][h][w] &= keep;
                        if constexpr (QUANT) t.vs[s][j] = keep ? t.vs[s][j] : 0.0f;
                    }
            }
            u32x4 ph, pl;
            if constexpr (QUANT) {
                // probabilities times value scales in two bf16 terms: 16 significant bits of any magnitude
                float hi[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    p[i] *= t.vs[i / 4][i % 4];
                    hi[i] = bf16_1(f32_to_bf16(p[i]));
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    ph[i] = pack_bf16x2(hi[2 * i], hi[2 * i + 1]);
                    pl[i] = pack_bf16x2(p[2 * i] - hi[2 * i], p[2 * i + 1] - hi[2 * i + 1]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) ph[i] = pack_act2<PT>(p[2 * i], p[2 * i + 1]);
            }
#pragma unroll
            for (int h = 0; h < T::NP; h++)
#pragma unroll
                for (int i = 0; i < T::PE; i++) {
                    u32x4 image;
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const int s = w / 2, j = (w % 2) * 2;
                        if constexpr (QUANT)
                            image[w] = pack_bf16x2(sbyte_f32(t.v[s][j][h][i / 4], i % 4), sbyte_f32(t.v[s][j + 1][h][i / 4], i % 4));
                        else
                            image[w] = __builtin_amdgcn_perm(t.v[s][j + 1][h][i / 2], t.v[s][j][h][i / 2], i % 2 ? 0x07060302u : 0x05040100u);
                    }
                    acc[h][i] = mfma_act<PT>(image, ph, acc[h][i]);
                    if constexpr (QUANT) acc[h][i] = mfma_act<PT>(image, pl, acc[h][i]);
                }
        }

        // the four wavefronts' sums on a common maximum
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (g == 0) ml[wave][col][0] = m, ml[wave][col][1] = l;
        __syncthreads();
        const float top = fmaxf(fmaxf(ml[0][col][0], ml[1][col][0]), fmaxf(ml[2][col][0], ml[3][col][0]));
        const float f = weight_of(m, top);
        const bool whole = unit == 0 && last == units;
        const int64_t part_at = ((int64_t)blockIdx.x * 2 + slot) * a.rows;
#pragma unroll
        for (int h = 0; h < T::NP; h++) {
            if (h) __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int i = 0; i < T::PE; i += 4)
                    *reinterpret_cast<f32x4 *>(&red[wave][col][(g * 4 + r) * T::PE + i]) =
                        f32x4{acc[h][i][r] * f, acc[h][i + 1][r] * f, acc[h][i + 2][r] * f, acc[h][i + 3][r] * f};
            __syncthreads();
            constexpr int QPR = 16 * T::PE / 4;                  // quads of a row
            for (int e = threadIdx.x; e < rows * QPR; e += 256) {
                const int row = e / QPR, d = (e % QPR) * 4;
                f32x4 sum = *reinterpret_cast<const f32x4 *>(&red[0][row][d]);
#pragma unroll
                for (int w = 1; w < 4; w++) sum += *reinterpret_cast<const f32x4 *>(&red[w][row][d]);
                if (whole) {
                    const float rt = fmaxf(fmaxf(ml[0][row][0], ml[1][row][0]), fmaxf(ml[2][row][0], ml[3][row][0]));
                    float total = 0.0f;
#pragma unroll
                    for (int w = 0; w < 4; w++) total += ml[w][row][1] * weight_of(ml[w][row][0], rt);
                    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
                    uint16_t *o = a.out + ((int64_t)b * a.heads + head0 + row) * D + h * 128 + d;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (h * 128 + d + i < D) o[i] = (uint16_t)pack_act2<QT>(sum[i] * inv, 0.0f);
                } else {
                    *reinterpret_cast<f32x4 *>(a.part + (part_at + row) * DP + h * 128 + d) = sum;
                }
            }
        }
        if (wave == 0 && g == 0 && col < rows) {
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) total += ml[w][col][1] * weight_of(ml[w][col][0], top);
            if (whole) {
                const float lse2 = total == 0.0f ? -INFINITY : top + (__builtin_amdgcn_logf(total) - kShift);
                const int64_t at = (int64_t)b * a.heads + head0 + col;
                if (a.lse) a.lse[at] = lse2 * kLn2;
                if (a.lse2) a.lse2[at] = lse2;
            } else {
                float *to = a.part_ml + (((int64_t)blockIdx.x * 2 + slot) * kHeads + col) * 2;
                to[0] = top;
                to[1] = total;
            }
        }
        __syncthreads();                                         // ml and red are free again
        slot = 1;
        x += last - unit;
        unit = 0;
        if (last == units && ++pair == a.pairs) pair = 0, b++;
    }
}

// One workgroup per (sequence, pair): nothing to do for a pair that one workgroup finished; zeros where there are no
// positions; else the partial sums of the workgroups that met in it, in their order.
template <int DP, int QT>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(AttnArgs a, float shift)
{
    __shared__ uint32_t scan[4];
    __shared__ uint32_t mine;
    const int b = blockIdx.x / a.pairs, pair = blockIdx.x % a.pairs;
    const Numbering n(a, scan);
    if (b >= n.first && b < n.first + n.run) {
        uint32_t before = n.run_before;
        for (int i = n.first; i < b; i++) before += units_of(length_of(a, i));
        mine = before;
    }
    __syncthreads();
    const int units = (int)units_of(length_of(a, b));
    const int kvh = pair / a.tiles, head0 = kvh * a.group + (pair % a.tiles) * kHeads;
    const int rows = min(kHeads, (kvh + 1) * a.group - head0);
    const int64_t all = (int64_t)n.total * a.pairs, share = max(share_of(a, all), (int64_t)1);
    const int64_t x0 = (int64_t)mine * a.pairs + (int64_t)pair * units;
    const int w0 = (int)(x0 / share), w1 = units ? (int)((x0 + units - 1) / share) : w0;
    if (units && w0 == w1) return;
    const int D = a.cache.dim;
    const auto slot_of = [&](int w) { return w * share >= x0 ? 0 : 1; };
    for (int e = threadIdx.x; e < rows * (DP / 4); e += 256) {
        const int row = e / (DP / 4), d = (e % (DP / 4)) * 4;
        float top = -INFINITY;
        if (units)
            for (int w = w0; w <= w1; w++) top = fmaxf(top, a.part_ml[(((int64_t)w * 2 + slot_of(w)) * kHeads + row) * 2]);
        f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
        float total = 0.0f;
        if (units)
            for (int w = w0; w <= w1; w++) {
                const int64_t at = (int64_t)w * 2 + slot_of(w);
                const float mw = a.part_ml[(at * kHeads + row) * 2], lw = a.part_ml[(at * kHeads + row) * 2 + 1];
                const float f = weight_of(mw, top);
                total += lw * f;
                const f32x4 v = *reinterpret_cast<const f32x4 *>(a.part + (at * a.rows + row) * DP + d);
                sum += v * f;
            }
        const int64_t at = (int64_t)b * a.heads + head0 + row;
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (d + i < D) a.out[at * D + d + i] = (uint16_t)pack_act2<QT>(sum[i] * inv, 0.0f);
        if (d == 0) {
            const float lse2 = total == 0.0f ? -INFINITY : top + (__builtin_amdgcn_logf(total) - shift);
            if (a.lse) a.lse[at] = lse2 * kLn2;
            if (a.lse2) a.lse2[at] = lse2;
        }
    }
}

// attn_sums[b, kv head, j] += sum over the kv head's query heads of 2^(z_j - lse2), in the heads' order.  Four positions per
// thread; what was hidden has z = -infinity.
__global__ __launch_bounds__(256) void paged_sums_kernel(AttnArgs a)
{
    const int b = blockIdx.z, kvh = blockIdx.y;
    const int len = length_of(a, b);
    for (int64_t j = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; j < len; j += (int64_t)gridDim.x * 1024) {
        f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int h = 0; h < a.group; h++) {
            const int64_t at = (int64_t)b * a.heads + kvh * a.group + h;
            const float lse2 = a.lse2[at];
            const f32x4 z = *reinterpret_cast<const f32x4 *>(a.scores + at * a.score_pitch + j);
#pragma unroll
            for (int i = 0; i < 4; i++) sum[i] += z[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(z[i] - lse2);
        }
        float *to = a.sums + b * a.sums_batch + kvh * a.sums_head + j;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (j + i < len) to[i] += sum[i];
    }
}

struct AttnSizes {
    int64_t rows, tiles, pairs, units, workgroups, dp, score_pitch;
    size_t part, part_ml, lse2, scores, bytes;                    // offsets in the workspace, and its size
};

constexpr size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// false: outside what the kernels number in 32 bits
bool plan_attention(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_blocks, int64_t block_size, bool sums,
                    AttnSizes *p)
{
    if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || head_dim > 256 || max_blocks < 0 || block_size < 1)
        return false;
    if (max_blocks > 0x7fffff00 / block_size || batch > 0x7fffffff / heads || heads > 0xffff) return false;
    const int64_t group = heads / kv_heads, capacity = max_blocks * block_size;
    p->rows = group < kHeads ? group : kHeads;
    p->tiles = (group + kHeads - 1) / kHeads;
    p->pairs = kv_heads * p->tiles;
    p->units = (capacity + kUnit - 1) / kUnit;
    if (p->units && batch > 0x7fffffff / p->units) return false;
    p->dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    const int64_t most = batch * p->units;
    p->workgroups = 768;
    if (most < p->workgroups && most * p->pairs < p->workgroups) p->workgroups = most * p->pairs > 0 ? most * p->pairs : 1;
    p->score_pitch = (capacity + 3) / 4 * 4;
    size_t at = 0;
    const auto take = [&](size_t bytes) { const size_t o = at; at += round256(bytes); return o; };
    p->part = take((size_t)(p->workgroups * 2 * p->rows * p->dp) * 4);
    p->part_ml = take((size_t)(p->workgroups * 2 * kHeads * 2) * 4);
    p->lse2 = take(sums ? (size_t)(batch * heads) * 4 : 0);
    p->scores = take(sums ? (size_t)(batch * heads) * (size_t)p->score_pitch * 4 : 0);
    p->bytes = at;
    return true;
}

template <int DP, bool QUANT, int QT>
void launch_attention(const AttnArgs &a, bool uni, hipStream_t s)
{
    if (uni) hipLaunchKernelGGL((paged_decode_kernel<DP, QUANT, QT, true>), dim3(a.workgroups), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((paged_decode_kernel<DP, QUANT, QT, false>), dim3(a.workgroups), dim3(256), 0, s, a);
    hipLaunchKernelGGL((paged_decode_join_kernel<DP, QT>), dim3((unsigned)(a.batch * a.pairs)), dim3(256), 0, s, a, QUANT || QT == 0 ? 0.0f : 14.0f);
}

template <int DP>
void launch_attention(const AttnArgs &a, bool quant, bool fp16, bool uni, hipStream_t s)
{
    if (quant) {
        if (fp16) launch_attention<DP, true, 1>(a, uni, s);
        else launch_attention<DP, true, 0>(a, uni, s);
    } else {
        if (fp16) launch_attention<DP, false, 1>(a, uni, s);
        else launch_attention<DP, false, 0>(a, uni, s);
    }
}

} // namespace
} // namespace mi355

extern "C" size_t mi355_paged_decode_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                         int64_t max_blocks, int64_t block_size, int with_sums)
{
    mi355::AttnSizes p;
    return mi355::plan_attention(batch, heads, kv_heads, head_dim, max_blocks, block_size, with_sums != 0, &p) ? p.bytes : 0;
}

extern "C" int mi355_paged_decode_attention(const mi355_paged_cache *cache, const void *q, int q_dtype, int64_t q_stride_batch,
                                            int64_t q_stride_head, void *out, float *lse, int64_t batch, int64_t heads,
                                            const int32_t *block_table, int64_t table_stride, int64_t max_blocks,
                                            const int32_t *context_lens, float scale, const uint8_t *mask, int64_t mask_stride,
                                            float *attn_sums, int64_t sums_stride_batch, int64_t sums_stride_head, void *workspace,
                                            size_t workspace_bytes, void *stream)
{
    using namespace mi355;
    AttnArgs a;
    if (const int st = open_cache(cache, &a.cache); st != MI355_OK) return st;
    const bool quant = cache->dtype == MI355_DTYPE_INT8, fp16 = q_dtype == MI355_DTYPE_FP16;
    if (batch < 0 || heads < 1 || heads % cache->kv_heads || max_blocks < 0 || (q_dtype != MI355_DTYPE_BF16 && !fp16) ||
        (!quant && cache->dtype != q_dtype))
        return MI355_ERR_BAD_ARGUMENT;
    if (batch == 0) return MI355_OK;
    if (!q || !out || !context_lens || (max_blocks > 0 && !block_table)) return MI355_ERR_BAD_ARGUMENT;
    AttnSizes p;
    if (!plan_attention(batch, heads, cache->kv_heads, cache->head_dim, max_blocks, cache->block_size, attn_sums != nullptr, &p)) return MI355_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < p.bytes) return MI355_ERR_WORKSPACE;
    if (!aligned(workspace, 16) || !aligned(q, 2) || !aligned(out, 2) || !aligned(lse, 4) || !aligned(block_table, 4) || !aligned(context_lens, 4) ||
        !aligned(attn_sums, 4))
        return MI355_ERR_ALIGNMENT;
    if (batch * p.pairs > 0x7fffffff || batch > 65535 * 32) return MI355_ERR_UNSUPPORTED;
    a.q = static_cast<const uint16_t *>(q);
    a.q_batch = q_stride_batch;
    a.q_head = q_stride_head;
    a.out = static_cast<uint16_t *>(out);
    a.lse = lse;
    a.table = block_table;
    a.table_stride = table_stride;
    a.lens = context_lens;
    a.mask = mask;
    a.mask_stride = mask_stride;
    char *ws = static_cast<char *>(workspace);
    a.part = reinterpret_cast<float *>(ws + p.part);
    a.part_ml = reinterpret_cast<float *>(ws + p.part_ml);
    a.scores = attn_sums ? reinterpret_cast<float *>(ws + p.scores) : nullptr;
    a.lse2 = attn_sums ? reinterpret_cast<float *>(ws + p.lse2) : nullptr;
    a.sums = attn_sums;
    a.score_pitch = p.score_pitch;
    a.sums_batch = sums_stride_batch;
    a.sums_head = sums_stride_head;
    a.batch = (int)batch;
    a.heads = (int)heads;
    a.group = (int)(heads / cache->kv_heads);
    a.rows = (int)p.rows;
    a.tiles = (int)p.tiles;
    a.pairs = (int)p.pairs;
    a.workgroups = (int)p.workgroups;
    a.capacity = (int)(max_blocks * cache->block_size);
    a.scale2 = scale * kLog2e;
    const int es = quant ? 1 : 2;
    // pieces of 16 bytes: rows and q on 16-byte boundaries, and no piece reaching past a row's end
    a.vec = cache->head_dim * es % 16 == 0 && rows_aligned(a.cache.key, 16) && rows_aligned(a.cache.value, 16) && aligned(q, 16) &&
            q_stride_batch % 8 == 0 && q_stride_head % 8 == 0;
    const int64_t reach = (int64_t)1 << 26;                       // 16 rows stay within a 31-bit offset
    const bool uni = a.vec && cache->block_size % 16 == 0 && a.cache.key.token < reach && a.cache.value.token < reach;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.dp == 64) launch_attention<64>(a, quant, fp16, uni, s);
    else if (p.dp == 128) launch_attention<128>(a, quant, fp16, uni, s);
    else launch_attention<256>(a, quant, fp16, uni, s);
    if (attn_sums && a.capacity > 0) {
        const int64_t chunks = (a.capacity + 1023) / 1024;
        for (int64_t b0 = 0; b0 < batch; b0 += 65535) {           // a grid's third dimension has 16 bits
            AttnArgs c = a;
            c.batch = (int)(batch - b0 < 65535 ? batch - b0 : 65535);
            c.lens += b0;
            c.scores += b0 * heads * p.score_pitch;
            c.lse2 += b0 * heads;
            c.sums += b0 * sums_stride_batch;
            hipLaunchKernelGGL(paged_sums_kernel, dim3((unsigned)(chunks < 64 ? chunks : 64), (unsigned)cache->kv_heads, (unsigned)c.batch), dim3(256), 0, s, c);
        }
    }
    return check_launch();
}
