// npu_paged_decode_attention for gfx950: one new token per sequence against the tokens of a paged key-value cache.
//
// Per sequence b and query head h (key/value head h / group), over the positions j that are seen:
//   z_j = scale * log2(e) * sum_d q_d k_jd      m = max z_j      l = sum_j 2^(z_j - m)
//   out_d = sum_j 2^(z_j - m) v_jd / l          lse = (m + log2 l) / log2(e)
// Every cached byte is read once for up to 16 query heads of its key/value head (a larger group reads it once for each 16), so
// the bound is the cache's bytes over the memory's rate.
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
// Scores, maxima, l and out are float32.  The second product takes 16-bit operands, so probabilities are rounded once, to the
// values' own type: 2^-8 of each in bf16, 2^-11 in fp16, which is what the values themselves carry, and l sums them unrounded.
// Against probabilities kept in float32 the outputs' error grows from 0.0017 to 0.0018 of their norm for 37 bf16 positions, and by
// less over more of them; the rounding of out to its own type makes the rest.  Products with value scales, on int8 caches, whose
// values are exact, keep two bf16 terms, 2^-16.
//
// Work is dealt out on the device, because the lengths are known only there: the positions of every (sequence, head) pair
// are cut into halves of a tile, 16 positions of one block (fewer at a block's end), eight halves make a unit, and a pair
// of more units than the card's fair share is cut into equal pieces of at most that.  A workgroup takes a piece at a time; a
// pair of one piece is finished there, else the workgroup leaves (sums, m, l) in the workspace, and the last one to arrive adds
// them in their order.
//
// Bound by memory, at 5.5 to 5.9 TB/s where the work is long (32 sequences of 8192, 1.07 GB, in 188 us), behind about 12 us that
// do not depend on it: the launch, two trips to memory for lengths and blocks, the first rows, and at the end the four
// wavefronts' sums, their trip through the workspace and the addition.  With 32 query heads on 8 heads of 128: 32 sequences of up to 4095 tokens
// (280 MB) 62 us, one of 131071 (537 MB) 104 us, int8, 64 of up to 8192 (563 MB) 120 us, one of 37 6.5 us.
#include "paged_cache.h"
#include "weight_quant_common.h"

namespace mi355 {
namespace {

constexpr int kHalf = 16;                    // positions of half a tile: rows of one MFMA operand
constexpr int kUnit = 8;                     // halves per unit: a tile of two for each wavefront of a workgroup
constexpr int kHeads = 16;                   // query heads of one tile
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
constexpr uint32_t kDealt = 64;              // pieces that are dealt to the XCDs at once
constexpr int kSC1 = 16;                     // cache-policy bit: agent scope, past the caches of one XCD

// Workgroups of a compute unit that the work is cut for, no more than their registers allow: one wavefront's keys, values and
// sums are 2 rows of 16 tokens and 16 rows of outputs, 139 to 168 registers for heads of 65 to 128, where three fit.  Rows of 512
// bytes take more than 256 (16-bit heads of 256, one sequence of 65000, 532 MB: 99 us with one workgroup and no spills, 190 with
// two that spill).  A piece more or fewer for each leaves compute units waiting for the last (heads of 128, 32 sequences of up to
// 4095, 280 MB: 62 us for 768 pieces, 66 for 512, 64 for 1024, 68 for 1536).  Heads of up to 64 take 103 to 124 registers, of
// which four would fit; they are cut for three like the others.
constexpr int resident(int dp, bool quant) { return dp < 256 ? 3 : quant ? 2 : 1; }

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
    uint32_t *arrived;                       // [2][cut pieces] zero before and after
    float *part;                             // [cut pieces][rows][DP]
    float *part_ml;                          // [cut pieces][kHeads][2]: maximum, sum
    float *scores;                           // [batch * heads][score_pitch] z_j, or null
    float *lse2;                             // [batch * heads] m + log2 l, with scores
    float *sums;
    int64_t score_pitch, sums_batch, sums_head;
    FastDiv by_pairs, by_shares;
    FastDiv span, halves;                    // positions that are cut into halves together (a block, or 16), and their halves
    int batch, heads, group, rows, tiles, pairs, shares;        // pairs = key/value heads * tiles, of one sequence
    int capacity, max_blocks;                // capacity = max_blocks * block_size
    uint32_t part_bytes, part_ml_bytes;
    float scale2;                            // scale * log2(e)
    int together;                            // the heads of a token share cache lines
};

// The kernel's arguments where the launch put them, in constant memory.  A kernel of several phases would otherwise load every
// field that a later phase needs at the start, and spill a hundred scalar registers; behind args_now() they are read again.
// What such a pointer leads to has to be named global memory (at()), since the compiler no longer sees where it came from.
typedef const __attribute__((address_space(4))) AttnArgs *Args;
__device__ __forceinline__ Args args_now()
{
    auto p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}
// The thread's number, out of the compiler's sight for the same reason: what is derived from it is derived where it is used
// and not kept in vector registers through the phases before.
__device__ __forceinline__ int thread_now()
{
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}
template <class T>
using Global = __attribute__((address_space(1))) T;
template <class T>
__device__ __forceinline__ Global<T> *at(T *p) { return (Global<T> *)p; }
__device__ __forceinline__ uint32_t divide(uint32_t n, const __attribute__((address_space(4))) FastDiv &f)
{
    return (uint32_t)(((uint64_t)n * f.mul) >> f.shift);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ int64_t uniform(int64_t v) { return (int64_t)(((uint64_t)uniform((uint32_t)(v >> 32)) << 32) | uniform((uint32_t)v)); }
// read-only words through the scalar cache
__device__ __forceinline__ int scalar_load(const int32_t *p) { return *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)p; }

// What sums over a maximum `m` count for under the maximum `top`.  Nothing seen yet: m = -infinity, sums 0 - or NaN, from NaN
// scores, which the product with 0 keeps.
__device__ __forceinline__ float weight_of(float m, float top) { return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top); }

__device__ __forceinline__ int clamp_len(Args a, int len) { return min(max(len, 0), a->capacity); }
__device__ __forceinline__ uint32_t halves_of(Args a, int len)
{
    const uint32_t whole = divide((uint32_t)len, a->span);
    return whole * a->halves.d + ((uint32_t)len - whole * a->span.d + kHalf - 1) / kHalf;
}
__device__ __forceinline__ uint32_t units_of(Args a, int len) { return (halves_of(a, len) + kUnit - 1) / kUnit; }

// How the work is cut up, and the numbering of the pieces: sequence by sequence, in it pair by pair, or the
// pairs of a stretch together.  Every wavefront counts for itself, lane i a run of consecutive sequences; no barrier, no LDS.
struct Pieces {
    uint32_t share;                          // units of a piece at most
    uint32_t before, count, total;           // pieces of one pair: in the runs before this lane's, in it, in all
    uint32_t cut_before;                     // those of pairs with several pieces, before this lane's run
    int run, len;                            // sequences per lane; the length of the first
    bool empty;                              // there is a sequence without positions

    __device__ uint32_t of(uint32_t units) const { return (units + share - 1) / share; }
    __device__ explicit Pieces(Args a)
    {
        const int lane = threadIdx.x & 63, batch = a->batch;
        run = (batch + 63) / 64;
        const int first = lane * run, end = min(first + run, batch);
        len = first < batch ? clamp_len(a, at(a->lens)[first]) : 0;
        const uint32_t mine = units_of(a, len);
        uint32_t sum = mine;
        bool none = first < batch && mine == 0;
        for (int i = first + 1; i < end; i++) {
            const uint32_t units = units_of(a, clamp_len(a, at(a->lens)[i]));
            none = none || units == 0;
            sum += units;
        }
        empty = __any(none);
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)scan_lanes(sum, Add()), 63) * (uint32_t)a->pairs;
        share = max(divide(all + a->shares - 1, a->by_shares), 1u);
        count = of(mine);
        uint32_t cut = count > 1 ? count : 0;
        for (int i = first + 1; i < end; i++) {
            const uint32_t pieces = of(units_of(a, clamp_len(a, at(a->lens)[i])));
            count += pieces;
            cut += pieces > 1 ? pieces : 0;
        }
        const uint32_t scan = scan_lanes(count, Add());
        before = scan - count;
        total = (uint32_t)__builtin_amdgcn_readlane((int)scan, 63);
        cut_before = scan_lanes(cut, Add()) - cut;
    }
    // the sequence that holds piece y of one pair: its length and pieces, and how many (of them cut) come before it
    __device__ void find(Args a, uint32_t y, int &b, int &length, uint32_t &pieces, uint32_t &pieces_before, uint32_t &cut_pieces_before) const
    {
        const int lane = __builtin_ctzll(__ballot(y >= before && y - before < count));
        b = lane * run;
        pieces_before = (uint32_t)__builtin_amdgcn_readlane((int)before, lane);
        cut_pieces_before = (uint32_t)__builtin_amdgcn_readlane((int)cut_before, lane);
        length = __builtin_amdgcn_readlane(len, lane);
        pieces = uniform(of(units_of(a, length)));
        while (y - pieces_before >= pieces) {
            pieces_before += pieces;
            cut_pieces_before += pieces > 1 ? pieces : 0;
            length = clamp_len(a, scalar_load(a->lens + ++b));
            pieces = uniform(of(units_of(a, length)));
        }
    }
};

// BYTES of a row from any address, of which `valid` belong to the row; the rest is zero and not read.
template <int BYTES>
__device__ __forceinline__ void load_piece(uint32_t *to, const Global<char> *from, int valid)
{
    if (valid >= BYTES) {
        typedef uint32_t piece __attribute__((ext_vector_type(BYTES / 4)));
        typedef piece anywhere __attribute__((aligned(1)));
        const piece v = *(const Global<anywhere> *)from;
        __builtin_memcpy(to, &v, BYTES);
        return;
    }
    uint64_t low = 0, high = 0;
#pragma unroll 1
    for (int i = 0; i < valid; i++) (i < 8 ? low : high) |= (uint64_t)(uint8_t)from[i] << (8 * (i & 7));
#pragma unroll
    for (int w = 0; w < BYTES / 4; w++) to[w] = (uint32_t)((w < 2 ? low : high) >> (32 * (w & 1)));
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

// Over the four lanes that differ in their group of 16, in all of them: exchanges of neighbouring groups, then of halves.
template <class Op>
__device__ __forceinline__ float over_groups(float v, Op op)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(h[0]), __uint_as_float(h[1]));
}

// How the rows of half a tile are addressed.
//   kRows   lane by lane: any block size, stride, width and alignment
//   kBlock  the half lies in one block: a scalar descriptor that ends with the half's last row, constant lane offsets; rows in
//           16-byte pieces.  Rows behind the end read as zero without traffic, so the loop needs no edge code.
//   kBlockAlike  int8, as kBlock; keys and values lie alike, so that one offset serves both, and so do the scales, those of four
//           tokens of a head in 16 aligned bytes (64 sequences of up to 8192, 8 heads of 128: 123.4 us, 124.5 as kBlock; 32 of up
//           to 4095, 8 heads of 64: 24.8 and 25.4.  16-bit caches have no scales and gain nothing)
//   kBlockMask  as kBlock, with a mask, whose bytes are read four at a time
// 32 sequences of up to 4095, 8 heads of 128, blocks of 16: 62.9 us as kBlock, 74.4 as kRows; 16 masked ones, 32 heads of 80,
// blocks of 24: 28.6 as kBlockMask, 36.4 as kRows; int8, 64 of up to 8192: 219.9 as kRows.  A short half wastes its operand's
// rows, so kBlock loses with small blocks: 66.2 and 74.8 us for blocks of 8, 79.8 and 75 for 5, 84.9 and 75.4 for 4.
enum Addressing { kRows, kBlock, kBlockAlike, kBlockMask };

// DP: head_dim rounded up to 64, 128 or 256.  QT: type of q and out (0 bf16, 1 fp16).
template <int DP, bool QUANT, int QT, Addressing AD>
struct Decode {
    static constexpr int ES = QUANT ? 1 : 2;
    static constexpr int NCH = DP / 32;                          // chunks of 32 d, one MFMA each
    static constexpr int KL = QUANT ? NCH / 2 : NCH;             // 16-byte loads of a key row per lane
    static constexpr int PE = DP >= 128 ? 8 : 4;                 // consecutive d of a value row per lane and piece
    static constexpr int NP = DP / (16 * PE);
    static constexpr int VW = PE * ES / 4;                       // registers of a piece
    static constexpr int PT = QUANT ? 0 : QT;                    // type of the probabilities and of the values' images
    // fp16 probabilities are 2^14 times as large, so that ones down to 2^-38 of the largest keep their place
    static constexpr float kShift = PT == 1 ? 14.0f : 0.0f;

    // where the two halves of a tile are
    struct Place {
        int n[2], key[2], id[2];                                 // positions seen from the half's first one on, that one, its block
        uint32_t off[2];                                         // and its token within the block
    };

    const Args a;
    const int wave, col, g, D;
    uint32_t koff[KL], voff[4][NP], soff[2][4];                  // lane offsets of key pieces, value pieces, scales
    uint32_t k[2][KL][4], v[2][4][NP][VW], hidden[2];
    float ks[2][4], vs[2][4];
    uint32_t lane_slot[2], v_slot[2];                            // kRows: slot of position 16 s + col of the tile, or ~0
    u32x4 q[NCH];
    f32x4 acc[NP][PE];
    float m, l;

    // of the pair that is being worked on
    int b, kvh, len, half_end;
    const int32_t *table;
    const char *kbase, *vbase, *ksbase, *vsbase;
    uint64_t start[2], scale_start[2];                           // kBlockAlike: of the tile whose keys were requested last
    uint32_t reach[2];

    __device__ explicit Decode(Args args)
        : Decode(args, thread_now())
    {
    }
    __device__ __forceinline__ Decode(Args args, int thread) : a(args), wave(uniform(thread >> 6)), col(thread & 15), g((thread & 63) >> 4), D(args->cache.dim)
    {
        if constexpr (AD != kRows) {
#pragma unroll
            for (int c = 0; c < KL; c++) {
                const int d = first_d(c);
                koff[c] = d < D ? (uint32_t)col * (uint32_t)a->cache.key.token + d * ES : kOutOfRange;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int h = 0; h < NP; h++) {
                    const int d = h * 128 + col * PE;
                    voff[j][h] = d < D ? (uint32_t)(g * 4 + j) * (uint32_t)a->cache.value.token + d * ES : kOutOfRange;
                }
                if constexpr (QUANT) {
                    soff[0][j] = (uint32_t)(g * 4 + j) * (uint32_t)a->cache.key_scale.token;
                    soff[1][j] = (uint32_t)(g * 4 + j) * (uint32_t)a->cache.value_scale.token;
                }
            }
        }
    }

    using ArgArray = const __attribute__((address_space(4))) PagedArray;
    __device__ __forceinline__ int64_t offset(ArgArray &x, uint32_t slot) const
    {
        const uint32_t block = divide(slot, a->cache.page);
        return block * x.block + (int64_t)(slot - block * a->cache.page.d) * x.token + kvh * x.head;
    }
    // first d of the lane's key piece c; an int8 piece serves the chunks 2c and 2c + 1
    __device__ __forceinline__ int first_d(int c) const { return QUANT ? c * 64 + g * 16 : c * 32 + g * 8; }

    __device__ __forceinline__ void begin(int b_, int kvh_, int head0, int rows, int len_, int half_end_)
    {
        b = b_, kvh = kvh_, len = len_, half_end = half_end_;
        table = a->table + b * a->table_stride;
        kbase = a->cache.key.base + kvh * a->cache.key.head;
        vbase = a->cache.value.base + kvh * a->cache.value.head;
        if constexpr (QUANT) ksbase = a->cache.key_scale.base + kvh * a->cache.key_scale.head, vsbase = a->cache.value_scale.base + kvh * a->cache.value_scale.head;
        const uint16_t *row = a->q + b * a->q_batch + (head0 + min(col, rows - 1)) * a->q_head;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const int d = QUANT ? first_d(c / 2) + (c % 2) * 8 : first_d(c);
            uint32_t w[4];
            load_piece<16>(w, (const Global<char> *)(row + d), col < rows ? 2 * (D - d) : 0);
            q[c] = u32x4{w[0], w[1], w[2], w[3]};
        }
        m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int h = 0; h < NP; h++)
#pragma unroll
            for (int i = 0; i < PE; i++) acc[h][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    __device__ __forceinline__ Place place(int tile) const
    {
        Place p;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const uint32_t half = uniform((uint32_t)tile * 2 + s);
            const uint32_t span = divide(half, a->halves);
            p.off[s] = (half - span * a->halves.d) * kHalf;
            p.key[s] = (int)(span * a->span.d + p.off[s]);
            const int n = min(min(kHalf, (int)(a->span.d - p.off[s])), len - p.key[s]);
            p.n[s] = uniform((int)half < half_end ? max(n, 0) : 0);
            p.id[s] = AD != kRows ? scalar_load(table + min(span, (uint32_t)a->max_blocks - 1)) : 0;
        }
        return p;
    }
    // a block that the table does not name holds nothing
    __device__ __forceinline__ void settle(Place &p) const
    {
        if constexpr (AD != kRows) {
#pragma unroll
            for (int s = 0; s < 2; s++)
                if ((uint32_t)p.id[s] >= (uint32_t)a->cache.num_blocks) p.n[s] = 0, p.id[s] = 0;
        }
    }
    // where half s begins within an array, and how far its rows reach
    __device__ __forceinline__ uint64_t start_of(ArgArray &x, const Place &p, int s) const
    {
        return (uint64_t)(uint32_t)p.id[s] * (uint32_t)x.block + p.off[s] * (uint32_t)x.token;
    }
    __device__ __forceinline__ uint32_t reach_of(ArgArray &x, const Place &p, int s, int row_bytes) const
    {
        return uniform(p.n[s] > 0 ? (uint32_t)(p.n[s] - 1) * (uint32_t)x.token + row_bytes : 0);
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const char *base, uint64_t start, uint32_t reach) const
    {
        return make_rsrc((const char *)uniform((int64_t)((uint64_t)base + start)), reach);
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const char *base, ArgArray &x, const Place &p, int s, int row_bytes) const
    {
        return rows_at(base, start_of(x, p, s), reach_of(x, p, s, row_bytes));
    }
    // positions of the tile, their keys, key scales and mask bytes
    __device__ __forceinline__ void load_keys(const Place &p)
    {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            if constexpr (AD != kRows) {
                if constexpr (AD == kBlockAlike) {
                    start[s] = start_of(a->cache.key, p, s), reach[s] = reach_of(a->cache.key, p, s, D * ES);
                    scale_start[s] = start_of(a->cache.key_scale, p, s);
                }
                const __amdgpu_buffer_rsrc_t r = AD == kBlockAlike ? rows_at(kbase, start[s], reach[s]) : rows_of(kbase, a->cache.key, p, s, D * ES);
#pragma unroll
                for (int c = 0; c < KL; c++) buffer_load<4>(k[s][c], r, koff[c]);
                if constexpr (QUANT) load_scales(ks[s], ksbase, a->cache.key_scale, p, s, soff[0]);
            } else {
                const int key = p.key[s] + col;
                const uint32_t block = divide((uint32_t)key, a->cache.page);
                const int id = col < p.n[s] ? at(table)[block] : -1;
                bool there = (uint32_t)id < (uint32_t)a->cache.num_blocks;
                if (a->mask && there) there = at(a->mask)[b * a->mask_stride + key] == 0;
                lane_slot[s] = there ? (uint32_t)id * a->cache.page.d + ((uint32_t)key - block * a->cache.page.d) : ~0u;
                const Global<char> *row = at(a->cache.key.base) + (there ? offset(a->cache.key, lane_slot[s]) : 0);
#pragma unroll
                for (int c = 0; c < KL; c++) load_piece<16>(k[s][c], row + first_d(c) * ES, there ? (D - first_d(c)) * ES : 0);
                if constexpr (QUANT) {
                    const float mine = there ? *(const Global<float> *)(at(a->cache.key_scale.base) + offset(a->cache.key_scale, lane_slot[s])) : 0.0f;
#pragma unroll
                    for (int r = 0; r < 4; r++) ks[s][r] = __shfl(mine, g * 4 + r, 64);
                }
            }
            if constexpr (AD == kBlockMask) {                    // from any byte (the host: blocks of a multiple of 4 tokens)
                const uint64_t first = (uint64_t)a->mask + (uint64_t)(b * a->mask_stride) + (uint32_t)p.key[s];
                const __amdgpu_buffer_rsrc_t r = make_rsrc((const void *)uniform((int64_t)first), (uint32_t)(p.n[s] + 3) & ~3u);
                hidden[s] = __builtin_amdgcn_raw_buffer_load_b32(r, g * 4, 0, 0);
            }
        }
    }
    __device__ __forceinline__ void load_scales(float (&to)[4], const char *base, ArgArray &x, const Place &p, int s, const uint32_t (&off)[4]) const
    {
        // (alike: the four scales of a lane group, or none; of those behind the end nothing is used)
        const __amdgpu_buffer_rsrc_t r = AD == kBlockAlike ? rows_at(base, scale_start[s], (uint32_t)(p.n[s] + 3 & ~3) * 4) : rows_of(base, x, p, s, 4);
        if constexpr (AD == kBlockAlike) {
            const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(r, g * 16, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) to[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) to[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, off[i], 0, 0));
        }
    }
    __device__ __forceinline__ void load_values(const Place &p)
    {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            if constexpr (AD != kRows) {
                const __amdgpu_buffer_rsrc_t r = AD == kBlockAlike ? rows_at(vbase, start[s], reach[s]) : rows_of(vbase, a->cache.value, p, s, D * ES);
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int h = 0; h < NP; h++) buffer_load<VW>(v[s][j][h], r, voff[j][h]);
                if constexpr (QUANT) load_scales(vs[s], vsbase, a->cache.value_scale, p, s, soff[1]);
            } else {
                const int64_t mine = lane_slot[s] == ~0u ? -1 : offset(a->cache.value, lane_slot[s]);
                if constexpr (QUANT) {
                    const float scale = mine >= 0 ? *(const Global<float> *)(at(a->cache.value_scale.base) + offset(a->cache.value_scale, lane_slot[s])) : 0.0f;
#pragma unroll
                    for (int r = 0; r < 4; r++) vs[s][r] = __shfl(scale, g * 4 + r, 64);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int64_t from = __shfl(mine, g * 4 + j, 64);
                    const Global<char> *row = at(a->cache.value.base) + (from < 0 ? 0 : from);
#pragma unroll
                    for (int h = 0; h < NP; h++) {
                        const int d = h * 128 + col * PE;
                        load_piece<VW * 4>(v[s][j][h], row + d * ES, from < 0 ? 0 : (D - d) * ES);
                    }
                }
            }
        }
    }
    // bit 4 s + r: position 16 s + 4 g + r of the tile is seen
    __device__ __forceinline__ uint32_t seen(const Place &p) const
    {
        uint32_t bits = 0;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            uint32_t four;
            if constexpr (AD != kRows) {
                four = (1u << min(max(p.n[s] - g * 4, 0), 4)) - 1;
                if constexpr (AD == kBlockMask) {
                    // a mask byte that is not 0 leaves bit 7 of its sum with 0x7f set, or has it itself
                    const uint32_t set = (((hidden[s] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | hidden[s]) & 0x80808080u;
                    four &= ~((set * 0x00204081u) >> 28);
                }
            } else {
                four = 0;
#pragma unroll
                for (int r = 0; r < 4; r++) four |= (uint32_t)(__shfl((int)lane_slot[s], g * 4 + r, 64) != -1) << r;
            }
            bits |= four << (4 * s);
        }
        return bits;
    }

    // z_j of the tile's positions
    __device__ __forceinline__ void score(const Place &p, uint32_t valid, f32x4 (&z)[2]) const
    {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            z[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NCH; c++) {
                u32x4 image;
                if constexpr (QUANT) {
                    const u32x2 lo = sbytes_act4<QT>(k[s][c / 2][(c % 2) * 2]), hi = sbytes_act4<QT>(k[s][c / 2][(c % 2) * 2 + 1]);
                    image = u32x4{lo.x, lo.y, hi.x, hi.y};
                } else {
                    image = u32x4{k[s][c][0], k[s][c][1], k[s][c][2], k[s][c][3]};
                }
                z[s] = mfma_act<QT>(image, q[c], z[s]);
            }
        }
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                z[s][r] = QUANT ? z[s][r] * (a->scale2 * ks[s][r]) : z[s][r] * a->scale2;
            }
        if (!full(p)) {
            no_select();
#pragma unroll
            for (int i = 0; i < 8; i++) z[i / 4][i % 4] = (valid >> i) & 1 ? z[i / 4][i % 4] : -INFINITY;
        }
    }
    // keeps a uniform branch a branch: the edge cases would cost selects in every tile
    __device__ static __forceinline__ void no_select() { asm volatile(""); }
    // every position of the tile is seen, known without a look at the lanes
    __device__ __forceinline__ bool full(const Place &p) const { return AD != kRows && AD != kBlockMask && p.n[0] + p.n[1] == 2 * kHalf; }
    __device__ __forceinline__ void store_scores(const Place &p, const f32x4 (&z)[2], int head0, int rows) const
    {
        if (col >= rows) return;
        Global<float> *to = at(a->scores) + ((int64_t)b * a->heads + head0 + col) * a->score_pitch + g * 4;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int n = AD != kRows ? min(kHalf, (int)(a->span.d - p.off[s])) : kHalf;        // a block's places, seen or not
            const int left = (p.key[s] < len ? min(n, len - p.key[s]) : 0) - g * 4;
            if (left <= 0) continue;
            if (a->span.d % 4 == 0) {
                *(Global<f32x4> *)(to + p.key[s]) = z[s];
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (r < left) to[p.key[s] + r] = z[s][r];
            }
        }
    }
    // probabilities under the running maximum, and what they weigh
    __device__ __forceinline__ void add(const Place &place, uint32_t valid, const f32x4 (&z)[2], u32x4 &ph, u32x4 &pl)
    {
        float top = fmaxf(fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[0][2], z[0][3])), fmaxf(fmaxf(z[1][0], z[1][1]), fmaxf(z[1][2], z[1][3])));
        top = over_groups(top, [](float x, float y) { return fmaxf(x, y); });
        if (__any(top > m)) {
            const float higher = fmaxf(m, top), f = weight_of(m, higher);
            m = higher;
            l *= f;
#pragma unroll
            for (int h = 0; h < NP; h++)
#pragma unroll
                for (int i = 0; i < PE; i++) acc[h][i] *= f;
        }
        const float base = m == -INFINITY ? 0.0f : m - kShift;
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            p[i] = __builtin_amdgcn_exp2f(z[i / 4][i % 4] - base);
            l += p[i];
        }
        if constexpr (QUANT) {
            // probabilities times value scales in two bf16 terms: 16 significant bits of any magnitude (one term would be 2^-8 of
            // each, where the codes are exact)
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = p[i] * vs[i / 4][i % 4];
            if (!full(place)) {                                  // (a scale that is not seen may be anything)
                no_select();
#pragma unroll
                for (int i = 0; i < 8; i++) p[i] = (valid >> i) & 1 ? p[i] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                ph[i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
                pl[i] = pack_bf16x2(p[2 * i] - bf16_lo(ph[i]), p[2 * i + 1] - bf16_hi(ph[i]));
            }
        } else {
            // one term, as precise as the values
#pragma unroll
            for (int i = 0; i < 4; i++) ph[i] = pack_act2<PT>(p[2 * i], p[2 * i + 1]);
        }
    }
    __device__ __forceinline__ void weigh(const Place &place, uint32_t valid, const u32x4 &ph, const u32x4 &pl)
    {
        if constexpr (!QUANT) {
            // a value that is not seen must not turn 0 * NaN into NaN (codes are always finite)
            if (!full(place)) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t keep = (valid >> i) & 1 ? ~0u : 0u;
#pragma unroll
                    for (int h = 0; h < NP; h++)
#pragma unroll
                        for (int w = 0; w < VW; w++) v[i / 4][i % 4][h][w] &= keep;
                }
            }
        }
#pragma unroll
        for (int h = 0; h < NP; h++)
#pragma unroll
            for (int i = 0; i < PE; i++) {
                u32x4 image;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const int s = w / 2, j = (w % 2) * 2;
                    if constexpr (QUANT)
                        image[w] = pack_bf16x2(sbyte_f32(v[s][j][h][i / 4], i % 4), sbyte_f32(v[s][j + 1][h][i / 4], i % 4));
                    else
                        image[w] = __builtin_amdgcn_perm(v[s][j + 1][h][i / 2], v[s][j][h][i / 2], i % 2 ? 0x07060302u : 0x05040100u);
                }
                acc[h][i] = mfma_act<PT>(image, ph, acc[h][i]);
                if constexpr (QUANT) acc[h][i] = mfma_act<PT>(image, pl, acc[h][i]);
            }
    }

    // The wavefront's tiles of this stretch.  The next tile's keys are requested as soon as this one's scores are out of the
    // registers, its values as soon as this one's are, so about a tile is always on the way.
    __device__ __forceinline__ void run(int tile, int tile_end, int head0, int rows)
    {
        Place cur = place(tile);
        settle(cur);
        load_keys(cur);
        __builtin_amdgcn_sched_barrier(0);
        load_values(cur);
        __builtin_amdgcn_sched_barrier(0);
        Place next = place(tile + 4);
        for (; tile < tile_end; tile += 4) {
            uint32_t valid = 0xff;
            if (!full(cur)) {
                no_select();
                valid = seen(cur);
            }
            f32x4 z[2];
            score(cur, valid, z);
            if (a->scores) store_scores(cur, z, head0, rows);
            settle(next);
            if constexpr (AD != kRows) load_keys(next);
            __builtin_amdgcn_sched_barrier(0);                   // requests stay in this order, so that a wait for one leaves the later ones out
            u32x4 ph, pl;
            add(cur, valid, z, ph, pl);
            weigh(cur, valid, ph, pl);
            if constexpr (AD == kRows) load_keys(next);          // the slots of this tile's values are no longer needed
            load_values(next);
            __builtin_amdgcn_sched_barrier(0);
            cur = next;
            next = place(tile + 8);
        }
    }
};

template <int QT>
__device__ __forceinline__ void store_out(Args a, int64_t row, int d, f32x4 v)
{
    const int D = a->cache.dim;
    Global<uint16_t> *o = at(a->out) + row * D + d;
    const u32x2 w = {pack_act2<QT>(v[0], v[1]), pack_act2<QT>(v[2], v[3])};
    if (d + 4 <= D) {
        typedef u32x2 anywhere __attribute__((aligned(2)));
        *(Global<anywhere> *)o = w;
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (d + i < D) o[i] = (uint16_t)(w[i / 2] >> (16 * (i % 2)));
    }
}
__device__ __forceinline__ void store_lse(Args a, int64_t row, float m, float l, float shift)
{
    const float lse2 = l == 0.0f ? -INFINITY : m + (__builtin_amdgcn_logf(l) - shift);
    if (a->lse) at(a->lse)[row] = lse2 * kLn2;
    if (a->lse2) at(a->lse2)[row] = lse2;
}

// Sums of one stretch of positions over the 16 query heads: what a workgroup has in LDS, what it leaves in the workspace and
// what comes of adding those.
template <int DP>
struct Sums {
    static constexpr int RP = (DP > 128 ? DP : 128) + 4;         // row pitch, 4 words past a bank cycle
    float (*row)[RP];
    float (*ml)[2];                                              // maximum, sum of probabilities
    __device__ __forceinline__ f32x4 &quad(int r, int d) const { return *reinterpret_cast<f32x4 *>(&row[r][d]); }
};
__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_of(Args a) { return make_rsrc(a->part, a->part_bytes); }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_ml_of(Args a) { return make_rsrc(a->part_ml, a->part_ml_bytes); }

// Leaves the sums in the workspace, as those of cut piece `place`, written through to where every XCD sees them.
template <int DP>
__device__ void publish(Args a, const Sums<DP> &own, uint32_t place, int rows)
{
    const __amdgpu_buffer_rsrc_t part = part_of(a);
    const int thread = thread_now();
    for (int e = thread; e < rows * (DP / 4); e += 256) {
        const int r = e / (DP / 4), d = (e % (DP / 4)) * 4;
        buffer_store_b128<kSC1>(__builtin_bit_cast(u32x4, own.quad(r, d)), part, ((place * (uint32_t)a->rows + r) * DP + d) * 4, 0);
    }
    if (thread < rows) {
        const u32x2 w = {__float_as_uint(own.ml[thread][0]), __float_as_uint(own.ml[thread][1])};
        __builtin_amdgcn_raw_buffer_store_b64(w, part_ml_of(a), (place * kHeads + thread) * 8, 0, kSC1);
    }
}
template <int DP, int QT>
__device__ void finish(Args a, const Sums<DP> &own, int64_t out_row, int rows, float shift)
{
    const int thread = thread_now();
    for (int e = thread; e < rows * (DP / 4); e += 256) {
        const int r = e / (DP / 4), d = (e % (DP / 4)) * 4;
        const float l = own.ml[r][1], inv = l == 0.0f ? 0.0f : 1.0f / l;
        store_out<QT>(a, out_row + r, d, own.quad(r, d) * inv);
    }
    if (thread < rows) store_lse(a, out_row + thread, own.ml[thread][0], own.ml[thread][1], shift);
}

// Over the 16 lanes of a row of lanes, in all of them.
template <int CTRL>
__device__ __forceinline__ float from_lane(float v, float outside)
{
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(outside), (int)__float_as_uint(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float row_max(float v)
{
    v = fmaxf(v, from_lane<0x111>(v, -INFINITY));                // row_shr:1, 2, 4, 8: the last lane has it
    v = fmaxf(v, from_lane<0x112>(v, -INFINITY));
    v = fmaxf(v, from_lane<0x114>(v, -INFINITY));
    v = fmaxf(v, from_lane<0x118>(v, -INFINITY));
    return __shfl(v, 15, 16);
}
__device__ __forceinline__ float row_sum(float v)
{
    v += from_lane<0x111>(v, 0.0f);
    v += from_lane<0x112>(v, 0.0f);
    v += from_lane<0x114>(v, 0.0f);
    v += from_lane<0x118>(v, 0.0f);
    return __shfl(v, 15, 16);
}

// Adds the sums of n cut pieces, first, first + step, ..., in this order, into `own`, which already holds those of number
// `mine`.  A thread adds one quad, eight partials in flight; where there are fewer quads than threads, several share the
// partials of a quad.  What the partials weigh is worked out meanwhile, 16 lanes to a head.
constexpr int kFlight = 8;
constexpr int kJoin = 64;                                        // sums of one call at most
constexpr size_t kJoinLds = (kJoin * kHeads + 256 * 4) * sizeof(float);
template <int DP>
__device__ void join(Args a, const Sums<DP> &own, int mine, uint32_t first, uint32_t step, int n, int rows, float *lds)
{
    constexpr int QPR = DP / 4;
    const int thread = thread_now();
    const uint32_t row_bytes = DP * 4, place_bytes = (uint32_t)a->rows * row_bytes;
    const auto place = [&](int i) { return first + (uint32_t)i * step; };
    // ends with the last of them: a request for number n or a later one reads zeros
    const __amdgpu_buffer_rsrc_t part = make_rsrc(a->part, uniform((place(n - 1) + 1) * place_bytes));
    const __amdgpu_buffer_rsrc_t mls = make_rsrc(a->part_ml, uniform((place(n - 1) + 1) * kHeads * 8));
    float(*weight)[kHeads] = reinterpret_cast<float(*)[kHeads]>(lds);
    f32x4 *shared = reinterpret_cast<f32x4 *>(lds + kJoin * kHeads);
    int threads = QPR;                                           // of all quads, a power of two
    while (threads < rows * QPR && threads < 256) threads *= 2;
    const int split = 256 / threads, part_no = thread / threads;
#pragma unroll 1
    for (int e0 = 0; e0 < rows * QPR; e0 += threads) {
        const int e = e0 + (thread & (threads - 1)), row = min(e / QPR, rows - 1), d = (e % QPR) * 4;
        f32x4 v[kFlight];
        const auto request = [&](int i0) {
            const uint32_t from = (uint32_t)row * row_bytes + d * 4;
#pragma unroll
            for (int k = 0; k < kFlight; k++)
                v[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(part, place(i0 + k * split) * place_bytes + from, 0, kSC1));
        };
        request(part_no);
        if (e0 == 0) {
            const int r = thread / 16, lane = thread % 16;
            float m[kJoin / 16], l[kJoin / 16], top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kJoin / 16; k++) {
                const int i = lane + 16 * k;
                const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(mls, (place(i) * kHeads + r) * 8, 0, kSC1);
                m[k] = i < n ? __uint_as_float(w.x) : -INFINITY, l[k] = __uint_as_float(w.y);
                if (i == mine) m[k] = own.ml[r][0], l[k] = own.ml[r][1];
                top = fmaxf(top, m[k]);
            }
            top = row_max(top);
#pragma unroll
            for (int k = 0; k < kJoin / 16; k++) {
                const float f = weight_of(m[k], top);
                weight[lane + 16 * k][r] = f;                    // 0 behind the last one
                sum += l[k] * f;
            }
            sum = row_sum(sum);
            if (lane == 0) own.ml[r][0] = top, own.ml[r][1] = sum;          // (this row's lanes have read it)
            __syncthreads();
        }
        const f32x4 here = own.quad(row, d);
        f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int i0 = part_no; i0 < n; i0 += kFlight * split) {
            if (i0 != part_no) request(i0);
#pragma unroll
            for (int k = 0; k < kFlight; k++) {
                const int i = i0 + k * split;
                const float f = weight[min(i, kJoin - 1)][row];
#pragma unroll
                for (int c = 0; c < 4; c++) sum[c] = __builtin_fmaf(i == mine ? here[c] : v[k][c], f, sum[c]);
            }
        }
        if (split > 1) {                                         // (one round: every quad has its threads)
            shared[thread] = sum;
            __syncthreads();
            if (part_no) continue;
            for (int k = 1; k < split; k++) sum += shared[thread + k * threads];
        }
        if (e < rows * QPR) own.quad(row, d) = sum;
    }
    __syncthreads();
}

// Says that this workgroup's sums are in the workspace; true for the last of `n` to say so.  The counter is 0 again then.
__device__ __forceinline__ bool arrive(Global<uint32_t> *counter, int n, int *lds)
{
    wait_vmcnt<0>();                                             // they have reached the coherence point
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t old = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *lds = old == (uint32_t)(n - 1);
        if (*lds) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);     // for the next launch
    }
    __syncthreads();
    return uniform(*lds) != 0;
}

template <int DP, bool QUANT, int QT, Addressing AD>
__global__ __launch_bounds__(256, resident(DP, QUANT)) void paged_decode_kernel(AttnArgs)
{
    using W = Decode<DP, QUANT, QT, AD>;
    constexpr int RP = 128 + 4;                                  // row pitch of a wavefront's sums in LDS
    __shared__ float red[4][kHeads][RP];
    __shared__ float ml[4][kHeads][2];
    __shared__ float all_wide[W::NP > 1 ? kHeads : 1][Sums<DP>::RP];     // the workgroup's sums: the first wavefront's place, if they fit
    __shared__ float all_ml[kHeads][2];
    __shared__ int counted[2];
    static_assert(W::NP > 1 || Sums<DP>::RP == RP, "the workgroup's sums lie where a wavefront's were");
    static_assert(sizeof(red) - sizeof(red[0]) >= kJoinLds, "join works behind the workgroup's sums");
    __shared__ int last_here;

    const Pieces pieces = [] {
        const Args a = args_now();
        uint32_t lines = 0;                                      // the arguments' cache lines, for the phases that follow
#pragma unroll
        for (size_t i = 0; i < sizeof(AttnArgs); i += 64) lines |= *(const __attribute__((address_space(4))) uint32_t *)((const __attribute__((address_space(4))) char *)a + i);
        const Pieces p(a);
        asm volatile("" ::"s"(lines));
        return p;
    }();
    const uint32_t all_pieces = uniform(pieces.total * (uint32_t)args_now()->pairs);

    for (uint32_t turn = blockIdx.x; turn < (all_pieces + kDealt - 1) / kDealt * kDealt; turn += gridDim.x) {
        // Consecutive workgroups go to the eight XCDs in turn; together: eight heads of the same tokens to one of them
        const uint32_t piece = args_now()->together ? (turn & ~(kDealt - 1)) | ((turn & 7) << 3) | ((turn >> 3) & 7) : turn;
        if (piece >= all_pieces) continue;
        int b, head0, rows, n, number;                           // piece `number` of the pair's n
        uint32_t first_cut;                                      // the pair's first cut piece
        float l, m;
        f32x4 acc[W::NP][W::PE];
        {
            const Args a = args_now();
            W w(a);
            int len;
            uint32_t count, before, cut_before;
            const uint32_t of_one = divide(piece, a->by_pairs);
            pieces.find(a, of_one, b, len, count, before, cut_before);
            b = uniform(b), len = uniform(len), n = uniform((int)count);
            uint32_t pair = piece - of_one * (uint32_t)a->pairs;
            number = uniform((int)(of_one - before));
            if (!a->together && n > 1) {
                const uint32_t in = piece - before * (uint32_t)a->pairs;
                pair = uniform(in / count), number = uniform((int)(in - pair * count));
            }
            first_cut = cut_before * (uint32_t)a->pairs + pair * count;
            const int kvh = (int)pair / a->tiles, halves = (int)halves_of(a, len), units = (halves + kUnit - 1) / kUnit;
            head0 = kvh * a->group + ((int)pair - kvh * a->tiles) * kHeads;
            rows = min(kHeads, (kvh + 1) * a->group - head0);
            // the first units % n pieces have one more unit
            const int each = n == 1 ? units : uniform(units / n), more = units - each * n;
            const int unit = number * each + min(number, more), end = unit + each + (number < more ? 1 : 0);
            w.begin(b, kvh, head0, rows, len, min(halves, end * kUnit));
            w.run(unit * (kUnit / 2) + w.wave, end * (kUnit / 2), head0, rows);
            l = w.l, m = w.m;
#pragma unroll
            for (int h = 0; h < W::NP; h++)
#pragma unroll
                for (int i = 0; i < W::PE; i++) acc[h][i] = w.acc[h][i];
        }

        const Args a = args_now();
        const int64_t out_row = (int64_t)b * a->heads + head0;
        Global<uint32_t> *arrived = at(a->arrived);
        // Of a pair that is cut, the last of its workgroups to arrive adds everybody's sums.  Where those are more than 64 KiB, groups
        // of about the root of their number are added first, so that no workgroup has many to read (one sequence of 8000, 16
        // query heads each: 19.5 us, 25.7 without groups; with 4 heads each and 4000 tokens 11.9 us at once, 13.8 in groups).  The
        // counter of a group is its first piece's, that of the groups lies behind all of these.
        int size = n;
        if (n >= kJoin || n * rows * (DP / 4) > 512 * kFlight) {
            size = 8;
            while (size * size < n) size += 4;
        }
        const int group = number / size, groups = (n + size - 1) / size, members = min(size, n - group * size);
        const uint32_t first = first_cut + group * size, behind = 2 * (uint32_t)a->shares;
        uint32_t seen = 0;                                       // how many have arrived: requested here, looked at behind what follows
        if (n > 1 && threadIdx.x < 2)
            seen = __hip_atomic_load(arrived + (threadIdx.x ? behind + first_cut : first), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

        // the four wavefronts' sums on a common maximum
        const int thread = thread_now(), lane = thread & 63, wave = thread >> 6, col = lane & 15, g = lane >> 4;
        const Sums<DP> own = {W::NP > 1 ? all_wide : reinterpret_cast<float (*)[Sums<DP>::RP]>(red[0]), all_ml};
        l = over_groups(l, [](float x, float y) { return x + y; });
        if (g == 0) ml[wave][col][0] = m, ml[wave][col][1] = l;
        __syncthreads();
        const float top = fmaxf(fmaxf(ml[0][col][0], ml[1][col][0]), fmaxf(ml[2][col][0], ml[3][col][0]));
        const float f = weight_of(m, top);
        if (thread < kHeads) {
            float total = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) total += ml[i][col][1] * weight_of(ml[i][col][0], top);
            all_ml[col][0] = top, all_ml[col][1] = total;
        }
#pragma unroll
        for (int h = 0; h < W::NP; h++) {
            if (h) __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int i = 0; i < W::PE; i += 4)
                    *reinterpret_cast<f32x4 *>(&red[wave][col][(g * 4 + r) * W::PE + i]) =
                        f32x4{acc[h][i][r] * f, acc[h][i + 1][r] * f, acc[h][i + 2][r] * f, acc[h][i + 3][r] * f};
            __syncthreads();
            constexpr int QPR = 16 * W::PE / 4;                  // quads of a row
            for (int e = thread; e < rows * QPR; e += 256) {
                const int row = e / QPR, d = (e % QPR) * 4;
                f32x4 sum = *reinterpret_cast<const f32x4 *>(&red[0][row][d]);
#pragma unroll
                for (int i = 1; i < 4; i++) sum += *reinterpret_cast<const f32x4 *>(&red[i][row][d]);
                own.quad(row, h * 128 + d) = sum;
            }
        }
        if (thread < 2) counted[thread] = (int)seen;
        __syncthreads();

        bool done = true;
        const auto last_of = [&](Global<uint32_t> *counter, int of, int seen, uint32_t place) {
            if (of == 1) return true;
            if (seen == of - 1) {                                // everybody else was there already: nobody waits for these sums
                if (thread == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                return true;
            }
            publish<DP>(a, own, place, rows);
            return arrive(counter, of, &last_here);
        };
        const int seen0 = uniform(counted[0]), seen1 = uniform(counted[1]);
#pragma unroll 1
        for (int level = 0; level < 2 && done; level++) {        // within the group, among the groups
            const int of = level ? groups : members;
            done = last_of(arrived + (level ? behind + first_cut : first), of, level ? seen1 : seen0, first + (level ? 0 : number - group * size));
            if (done && of > 1)
                join<DP>(a, own, level ? group : number - group * size, level ? first_cut : first, level ? (uint32_t)size : 1u, of, rows, &red[1][0][0]);
        }
        if (done) finish<DP, QT>(args_now(), own, out_row, rows, W::kShift);
        __syncthreads();                                         // ml and red are free again
    }

    if (!pieces.empty) return;
    const Args a = args_now();
    for (int e = blockIdx.x; e < a->batch; e += gridDim.x) {
        if (clamp_len(a, scalar_load(a->lens + e)) != 0) continue;
        for (int i = threadIdx.x; i < a->heads * a->cache.dim; i += 256) at(a->out)[(int64_t)e * a->heads * a->cache.dim + i] = 0;
        for (int i = threadIdx.x; i < a->heads; i += 256)
            if (a->lse) at(a->lse)[(int64_t)e * a->heads + i] = -INFINITY;
    }
}

// attn_sums[b, kv head, j] += sum over the kv head's query heads of 2^(z_j - lse2), in the heads' order.  Four positions per
// thread, four heads requested at once; what was hidden has z = -infinity.  Bound by latency: 16 sequences of 4097, 32 heads on
// 8, 12.6 MB in 5.2 us (5.8 with one head at a time).
__global__ __launch_bounds__(256) void paged_sums_kernel(AttnArgs a)
{
    const int b = blockIdx.z, kvh = blockIdx.y;
    const int len = min(max(a.lens[b], 0), a.capacity);
    const int64_t first = (int64_t)b * a.heads + kvh * a.group;
    for (int64_t j = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; j < len; j += (int64_t)gridDim.x * 1024) {
        float *to = a.sums + b * a.sums_batch + kvh * a.sums_head + j;
        float old[4];
#pragma unroll
        for (int i = 0; i < 4; i++) old[i] = to[min((int64_t)i, len - 1 - j)];
        f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int h0 = 0; h0 < a.group; h0 += 4) {
            f32x4 z[4];
            float lse2[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int64_t at = first + min(h0 + k, a.group - 1);
                lse2[k] = a.lse2[at];
                z[k] = *reinterpret_cast<const f32x4 *>(a.scores + at * a.score_pitch + j);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) sum[i] += h0 + k >= a.group || z[k][i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(z[k][i] - lse2[k]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (j + i < len) to[i] = old[i] + sum[i];
    }
}

struct AttnSizes {
    int64_t rows, tiles, pairs, units, shares, workgroups, dp, score_pitch;
    size_t part, part_ml, lse2, scores, bytes;                    // offsets in the workspace, and its size
    uint32_t part_bytes, part_ml_bytes;
};

constexpr size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// false: outside what the kernels number in 32 bits
bool plan_attention(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_blocks, int64_t block_size, bool quant,
                    bool sums, AttnSizes *p)
{
    if (batch < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 || head_dim > 256 || max_blocks < 0 || block_size < 1)
        return false;
    if (max_blocks > 0x7fffff00 / block_size || batch > 0x7fffffff / heads || heads > 0xffff) return false;
    const int64_t group = heads / kv_heads, capacity = max_blocks * block_size;
    p->rows = group < kHeads ? group : kHeads;
    p->tiles = (group + kHeads - 1) / kHeads;
    p->pairs = kv_heads * p->tiles;
    // halves per position at most: one for each block's remainder beside its sixteens
    const int64_t halves = capacity / kHalf + max_blocks + 1;
    p->units = (halves + kUnit - 1) / kUnit;
    if (batch * p->pairs > 0x7ffff000 / p->units) return false;
    p->dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    // Pieces: as many as the card holds workgroups at once, and up to one more for every pair, whose last piece is smaller.
    p->shares = kNumCU * resident((int)p->dp, quant);
    const int64_t pieces = batch * p->pairs * p->units < p->shares ? batch * p->pairs * p->units : p->shares + batch * p->pairs;
    p->workgroups = pieces < 2048 ? (pieces + kDealt - 1) / kDealt * kDealt : 2048;
    p->score_pitch = (capacity + 3) / 4 * 4;
    size_t at = MI355_WORKSPACE_ZERO_BYTES;                       // the arrival counters lie at its start
    const auto take = [&](size_t bytes) { const size_t o = at; at += round256(bytes); return o; };
    // of pairs that are cut there are fewer than twice as many pieces as shares: a pair of u units, u more than a share of s, has
    // fewer than u / s + 1 < 2 u / s
    const int64_t reserved = kNumCU * resident((int)p->dp, true);    // (the query of the size knows no type)
    p->part_bytes = (uint32_t)(reserved * 2 * p->rows * p->dp * 4);
    p->part_ml_bytes = (uint32_t)(reserved * 2 * kHeads * 2 * 4);
    p->part = take(p->part_bytes);
    p->part_ml = take(p->part_ml_bytes);
    p->lse2 = take(sums ? (size_t)(batch * heads) * 4 : 0);
    p->scores = take(sums ? (size_t)(batch * heads) * (size_t)p->score_pitch * 4 : 0);
    p->bytes = at;
    return true;
}
static_assert(resident(256, false) <= resident(256, true), "the workspace's size");
static_assert(kNumCU * 3 * 4 * sizeof(uint32_t) <= kWorkspaceCounterBytes, "arrival counters");
static_assert(kNumCU * 3 <= (kJoin / 2) * (kJoin / 2), "groups of pieces, and members of a group");

template <int DP, bool QUANT, int QT>
void launch_attention(const AttnArgs &a, Addressing ad, unsigned workgroups, hipStream_t s)
{
    const dim3 grid(workgroups), block(256);
    if (ad == kRows) hipLaunchKernelGGL((paged_decode_kernel<DP, QUANT, QT, kRows>), grid, block, 0, s, a);
    else if (ad == kBlockMask) hipLaunchKernelGGL((paged_decode_kernel<DP, QUANT, QT, kBlockMask>), grid, block, 0, s, a);
    else if (ad == kBlock) hipLaunchKernelGGL((paged_decode_kernel<DP, QUANT, QT, kBlock>), grid, block, 0, s, a);
    else if constexpr (QUANT) hipLaunchKernelGGL((paged_decode_kernel<DP, QUANT, QT, kBlockAlike>), grid, block, 0, s, a);
}

template <int DP>
void launch_attention(const AttnArgs &a, bool quant, bool fp16, Addressing ad, unsigned workgroups, hipStream_t s)
{
    if (quant) {
        if (fp16) launch_attention<DP, true, 1>(a, ad, workgroups, s);
        else launch_attention<DP, true, 0>(a, ad, workgroups, s);
    } else {
        if (fp16) launch_attention<DP, false, 1>(a, ad, workgroups, s);
        else launch_attention<DP, false, 0>(a, ad, workgroups, s);
    }
}

} // namespace
} // namespace mi355

extern "C" size_t mi355_paged_decode_attention_workspace(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                         int64_t max_blocks, int64_t block_size, int with_sums)
{
    mi355::AttnSizes p;
    return mi355::plan_attention(batch, heads, kv_heads, head_dim, max_blocks, block_size, true, with_sums != 0, &p) ? p.bytes : 0;
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
    if (!plan_attention(batch, heads, cache->kv_heads, cache->head_dim, max_blocks, cache->block_size, quant, attn_sums != nullptr, &p)) return MI355_ERR_UNSUPPORTED;
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
    a.arrived = reinterpret_cast<uint32_t *>(ws);
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
    a.shares = (int)p.shares;
    a.by_pairs = fast_div((uint32_t)p.pairs);
    a.by_shares = fast_div((uint32_t)p.shares);
    a.capacity = (int)(max_blocks * cache->block_size);
    a.max_blocks = (int)max_blocks;
    a.part_bytes = p.part_bytes;
    a.part_ml_bytes = p.part_ml_bytes;
    a.scale2 = scale * kLog2e;
    const int es = quant ? 1 : 2;
    // pieces of 16 bytes: rows on 16-byte boundaries, and no piece reaching past a row's end
    const bool pieces = cache->head_dim * es % 16 == 0 && rows_aligned(a.cache.key, 16) && rows_aligned(a.cache.value, 16);
    // Halves that lie in one block: block by block, the last half of a block may be short, so blocks of fewer than 8 tokens
    // would leave most of a tile empty.  Offsets within a block have 31 bits, a block's own offset is a 32 x 32-bit product.
    const PagedArray *const arrays[] = {&a.cache.key, &a.cache.value, &a.cache.key_scale, &a.cache.value_scale};
    bool blocks = pieces && cache->block_size >= 8 && (!mask || cache->block_size % 4 == 0), scales = cache->block_size % 4 == 0;
    for (int i = 0; i < (quant ? 4 : 2); i++) {
        const PagedArray &x = *arrays[i];
        blocks = blocks && x.block >= 0 && x.block <= 0xffffffffll && x.token >= 0 && x.token <= 0x7fffffff / (cache->block_size + 16);
        if (i >= 2) scales = scales && x.token == 4 && aligned(x.base, 16) && x.block % 16 == 0 && x.head % 16 == 0;
    }
    const auto alike = [](const PagedArray &x, const PagedArray &y) { return x.block == y.block && x.token == y.token && x.head == y.head; };
    const bool same = quant && scales && alike(a.cache.key, a.cache.value) && alike(a.cache.key_scale, a.cache.value_scale);
    const Addressing ad = !blocks ? kRows : mask ? kBlockMask : same ? kBlockAlike : kBlock;
    // Rows of several heads in a cache line, with other heads' rows of the same token: work on them at the same time and on one XCD,
    // so that the line comes once (16 sequences of up to 1001 tokens, 32 heads of 80: 32.4 -> 28.6 us; int8, 32 sequences of up to
    // 4095, 8 heads of 64: 34.5 -> 26.2 us).  Where heads have lines of their own, that would make the workgroups ask the same
    // memory channels at the same time (32 of up to 4095, 8 heads of 128: 68 us, against 62).
    const auto shared = [](const PagedArray &x) { return x.head % 128 != 0 && x.head < x.token; };
    a.together = shared(a.cache.key) || shared(a.cache.value);
    a.span = ad != kRows ? a.cache.page : fast_div(kHalf);
    a.halves = fast_div((a.span.d + kHalf - 1) / kHalf);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.dp == 64) launch_attention<64>(a, quant, fp16, ad, (unsigned)p.workgroups, s);
    else if (p.dp == 128) launch_attention<128>(a, quant, fp16, ad, (unsigned)p.workgroups, s);
    else launch_attention<256>(a, quant, fp16, ad, (unsigned)p.workgroups, s);
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
