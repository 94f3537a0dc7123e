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
// int4 caches: the image of a code c is c + 24 = 16 + u, its four bits u = c + 8 placed as the top mantissa bits of 16.0: one
// three-input instruction for two codes, where a conversion would take five.  A value is (c + offset) * scale = (image + offset - 24)
// * scale, so the second addend, the same for a whole row, is left to float32:
//   z_j += scale_j (offset_j - 24) sum_d q_d, the sum once per head       out_d += sum_j P_j (offset_j - 24), P_j = 2^(z_j - m) scale_j
//
// Scores, maxima, l and out are float32.  The second product takes 16-bit operands, so probabilities are rounded once, to the
// values' own type: 2^-8 of each in bf16, 2^-11 in fp16, which is what the values themselves carry, and l sums them unrounded.
// Against probabilities kept in float32 the outputs' error grows from 0.0017 to 0.0018 of their norm for 37 bf16 positions, and by
// less over more of them; the rounding of out to its own type makes the rest.  Products with value scales, on int8 caches, whose
// values are exact, keep two bf16 terms, 2^-16; int4 caches as int8 ones.
//
// Work is dealt out on the device, because the lengths are known only there: the positions of every (sequence, head) pair
// are cut into halves of a tile, 16 positions of one block (fewer at a block's end), eight halves make a unit, and a pair
// of more units than the card's fair share is cut into equal pieces of at most that.  A workgroup takes a piece at a time; a
// pair of one piece is finished there, else the workgroup leaves (sums, m, l) in the workspace, and the last one to arrive adds
// them in their order.  (int4: Ranges.)
//
// Bound by memory, at 5.5 to 5.9 TB/s where the work is long (32 sequences of 8192, 1.07 GB, in 188 us), behind about 12 us that
// do not depend on it: the launch, two trips to memory for lengths and blocks, the first rows, and at the end the four
// wavefronts' sums, their trip through the workspace and the addition.  With 32 query heads on 8 heads of 128: 32 sequences of up to 4095 tokens
// (280 MB) 62 us, one of 131071 (537 MB) 104 us, int8, 64 of up to 8192 (563 MB) 120 us, one of 37 6.5 us.  int4: 32 of up to 4095 (78 MB)
// 25.7 us, 64 of up to 8192 (308 MB) 62 to 65 us, one of 131071 (151 MB) 40 us, one of 37 7.2 us; 64 of up to 8192 with attn_sums 92.6 us.
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
// int4, Decode4: halves of a step of a workgroup; its workgroups of a compute unit (119 or 120 registers for heads of up to 64, 137 to 143
// of 65 to 128, 207 to 209 for wider ones); what the start and the end of a range cost, in halves (dense, 32 sequences of up to 4095, 78 MB: 25.7
// us with 24, 27.2 with 16, 26.4 with 30, 28.8 with 8, 27.1 with 40, 27.2 with 64; 64 of up to 8192, 308 MB: 64 to 65, with 8 71, with 40 and 64 67); and
// the addition of a sequence's pieces (a step is 1.5 us where work is short, the addition 2.8; 128 of 300 with 16, whole in two rounds, 22.1 us,
// with 8, dense, 27.1)
constexpr int kStep = 8;
constexpr int resident4(int dp) { return dp < 256 ? 3 : 2; }
constexpr uint32_t kStart = 24, kCut = 16;
// what removes the bias of int4 images, offset - 24, is computed with the offsets
constexpr float kBias4 = 24.0f;

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
    FastDiv by_pairs, by_shares, by_ranges;
    uint32_t ranges;                         // int4: ranges of a pair at most
    FastDiv span, halves;                    // positions that are cut into halves together (a block, or 16), and their halves
    int batch, heads, group, rows, tiles, pairs, shares;        // pairs = key/value heads * tiles, of one sequence
    int capacity, max_blocks;                // capacity = max_blocks * block_size
    uint32_t part_bytes, part_ml_bytes;
    float scale2;                            // scale * log2(e)
    int together;                            // the heads of a token share cache lines
    int regular;                             // int4: no mask, blocks of a multiple of 16, parameters of a head's tokens side by side
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
//   kPlain  int4: Decode4, which has the conditions
enum Addressing { kRows, kBlock, kBlockAlike, kBlockMask, kPlain };

// The images of an int4 word's codes i and i + 4: its bits 4 i and 16 + 4 i on, as the top mantissa bits of 16.0, the sign bit turned.
template <int ACT>
__device__ __forceinline__ uint32_t image4(uint32_t w, int i)
{
    constexpr int place = ACT == 0 ? 3 : 6;
    constexpr uint32_t mask = ACT == 0 ? 0x00780078u : 0x03c003c0u, one = ACT == 0 ? 0x41804180u | 0x00400040u : 0x4c004c00u | 0x02000200u;
    return bit_blend(4 * i > place ? w >> (4 * i - place) : w << (place - 4 * i), mask, one);
}

// DP: head_dim rounded up to 64, 128 or 256.  BITS: of the cache's elements.  QT: type of q and out (0 bf16, 1 fp16).
template <int DP, int BITS, int QT, Addressing AD>
struct Decode {
    static constexpr bool QUANT = BITS < 16;
    static constexpr int NCH = DP / 32;                          // chunks of 32 d, one MFMA each
    static constexpr int KL = QUANT ? NCH / 2 : NCH;             // loads of a key row per lane
    static constexpr int KW = BITS == 4 ? 2 : 4;                 // and their registers
    static constexpr int PE = DP >= 128 ? 8 : 4;                 // consecutive d of a value row per lane and piece
    static constexpr int NP = DP / (16 * PE);
    static constexpr int VW = BITS == 4 ? 1 : PE * BITS / 32;    // registers of a piece (int4, PE 4: a word that two lanes share)
    static constexpr int PARAMS = BITS == 4 ? 4 : 2;             // arrays of scales and offsets, as they lie in PagedCache
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
    uint32_t koff[KL], voff[4][NP], soff[PARAMS][4];             // lane offsets of key pieces, value pieces, scales, offsets
    uint32_t k[2][KL][KW], v[2][4][NP][VW], hidden[2];
    float ks[2][4], vs[2][4], ko[2][4], vo[2][4];
    uint32_t lane_slot[2], v_slot[2];                            // kRows: slot of position 16 s + col of the tile, or ~0
    u32x4 q[NCH];
    f32x4 acc[NP][PE];
    float m, l;
    float qsum, osum;                                            // int4: sum of the head's query; the lane's sum of P_j (offset_j - 24)

    // of the pair that is being worked on
    int b, kvh, len, half_end;
    const int32_t *table;
    const char *kbase, *vbase, *ksbase, *vsbase, *kobase, *vobase;
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
                koff[c] = d < D ? (uint32_t)col * (uint32_t)a->cache.key.token + bytes(d) : kOutOfRange;
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int h = 0; h < NP; h++) {
                    const int d = value_d(h);
                    voff[j][h] = d < D ? (uint32_t)(g * 4 + j) * (uint32_t)a->cache.value.token + bytes(d) : kOutOfRange;
                }
                if constexpr (QUANT) {
                    soff[0][j] = (uint32_t)(g * 4 + j) * (uint32_t)a->cache.key_scale.token;
                    soff[1][j] = (uint32_t)(g * 4 + j) * (uint32_t)a->cache.value_scale.token;
                }
                if constexpr (BITS == 4) {
                    soff[PARAMS - 2][j] = (uint32_t)(g * 4 + j) * (uint32_t)a->cache.key_offset.token;
                    soff[PARAMS - 1][j] = (uint32_t)(g * 4 + j) * (uint32_t)a->cache.value_offset.token;
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
    __device__ static __forceinline__ int bytes(int d) { return BITS == 4 ? d / 2 : d * (BITS / 8); }
    // first d of the lane's value piece h (int4: of its word)
    __device__ __forceinline__ int value_d(int h) const { return h * 128 + (BITS == 4 && PE == 4 ? col / 2 * 8 : col * PE); }
    // first d of the lane's key piece c; a piece of codes serves the chunks 2c and 2c + 1
    __device__ __forceinline__ int first_d(int c) const { return QUANT ? c * 64 + g * 16 : c * 32 + g * 8; }

    __device__ __forceinline__ void begin(int b_, int kvh_, int head0, int rows, int len_, int half_end_)
    {
        b = b_, kvh = kvh_, len = len_, half_end = half_end_;
        table = a->table + b * a->table_stride;
        kbase = a->cache.key.base + kvh * a->cache.key.head;
        vbase = a->cache.value.base + kvh * a->cache.value.head;
        if constexpr (QUANT) ksbase = a->cache.key_scale.base + kvh * a->cache.key_scale.head, vsbase = a->cache.value_scale.base + kvh * a->cache.value_scale.head;
        if constexpr (BITS == 4) kobase = a->cache.key_offset.base + kvh * a->cache.key_offset.head, vobase = a->cache.value_offset.base + kvh * a->cache.value_offset.head;
        const uint16_t *row = a->q + b * a->q_batch + (head0 + min(col, rows - 1)) * a->q_head;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const int d = QUANT ? first_d(c / 2) + (c % 2) * 8 : first_d(c);
            uint32_t w[4];
            load_piece<16>(w, (const Global<char> *)(row + d), col < rows ? 2 * (D - d) : 0);
            q[c] = u32x4{w[0], w[1], w[2], w[3]};
        }
        if constexpr (BITS == 4) {
            qsum = osum = 0.0f;
#pragma unroll
            for (int c = 0; c < NCH; c++) {
#pragma unroll
                for (int i = 0; i < 4; i++) qsum += act_lo<QT>(q[c][i]) + act_hi<QT>(q[c][i]);
                // in the order of image4: (d, d + 4)
                const u32x4 w = q[c];
                q[c] = u32x4{__builtin_amdgcn_perm(w.z, w.x, 0x05040100u), __builtin_amdgcn_perm(w.z, w.x, 0x07060302u),
                             __builtin_amdgcn_perm(w.w, w.y, 0x05040100u), __builtin_amdgcn_perm(w.w, w.y, 0x07060302u)};
            }
            qsum = over_groups(qsum, [](float x, float y) { return x + y; });
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
                    start[s] = start_of(a->cache.key, p, s), reach[s] = reach_of(a->cache.key, p, s, bytes(D));
                    scale_start[s] = start_of(a->cache.key_scale, p, s);
                }
                const __amdgpu_buffer_rsrc_t r = AD == kBlockAlike ? rows_at(kbase, start[s], reach[s]) : rows_of(kbase, a->cache.key, p, s, bytes(D));
#pragma unroll
                for (int c = 0; c < KL; c++) buffer_load<KW>(k[s][c], r, koff[c]);
                if constexpr (QUANT) load_scales(ks[s], ksbase, a->cache.key_scale, p, s, soff[0]);
                if constexpr (BITS == 4) load_scales(ko[s], kobase, a->cache.key_offset, p, s, soff[PARAMS - 2]);
            } else {
                const int key = p.key[s] + col;
                const uint32_t block = divide((uint32_t)key, a->cache.page);
                const int id = col < p.n[s] ? at(table)[block] : -1;
                bool there = (uint32_t)id < (uint32_t)a->cache.num_blocks;
                if (a->mask && there) there = at(a->mask)[b * a->mask_stride + key] == 0;
                lane_slot[s] = there ? (uint32_t)id * a->cache.page.d + ((uint32_t)key - block * a->cache.page.d) : ~0u;
                const Global<char> *row = at(a->cache.key.base) + (there ? offset(a->cache.key, lane_slot[s]) : 0);
#pragma unroll
                for (int c = 0; c < KL; c++) load_piece<KW * 4>(k[s][c], row + bytes(first_d(c)), there ? bytes(D - first_d(c)) : 0);
                if constexpr (QUANT) spread(ks[s], a->cache.key_scale, there, lane_slot[s]);
                if constexpr (BITS == 4) spread(ko[s], a->cache.key_offset, there, lane_slot[s]);
            }
            if constexpr (AD == kBlockMask) {                    // from any byte (the host: blocks of a multiple of 4 tokens)
                const uint64_t first = (uint64_t)a->mask + (uint64_t)(b * a->mask_stride) + (uint32_t)p.key[s];
                const __amdgpu_buffer_rsrc_t r = make_rsrc((const void *)uniform((int64_t)first), (uint32_t)(p.n[s] + 3) & ~3u);
                hidden[s] = __builtin_amdgcn_raw_buffer_load_b32(r, g * 4, 0, 0);
            }
        }
    }
    // kRows: each lane of the 16 loads the parameter of its slot; a lane gets those of its group's four positions
    __device__ __forceinline__ void spread(float (&to)[4], ArgArray &x, bool there, uint32_t slot) const
    {
        const float mine = there ? *(const Global<float> *)(at(x.base) + offset(x, slot)) : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; r++) to[r] = __shfl(mine, g * 4 + r, 64);
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
                const __amdgpu_buffer_rsrc_t r = AD == kBlockAlike ? rows_at(vbase, start[s], reach[s]) : rows_of(vbase, a->cache.value, p, s, bytes(D));
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int h = 0; h < NP; h++) buffer_load<VW>(v[s][j][h], r, voff[j][h]);
                if constexpr (QUANT) load_scales(vs[s], vsbase, a->cache.value_scale, p, s, soff[1]);
                if constexpr (BITS == 4) load_scales(vo[s], vobase, a->cache.value_offset, p, s, soff[PARAMS - 1]);
            } else {
                const int64_t mine = lane_slot[s] == ~0u ? -1 : offset(a->cache.value, lane_slot[s]);
                if constexpr (QUANT) spread(vs[s], a->cache.value_scale, mine >= 0, lane_slot[s]);
                if constexpr (BITS == 4) spread(vo[s], a->cache.value_offset, mine >= 0, lane_slot[s]);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int64_t from = __shfl(mine, g * 4 + j, 64);
                    const Global<char> *row = at(a->cache.value.base) + (from < 0 ? 0 : from);
#pragma unroll
                    for (int h = 0; h < NP; h++) {
                        const int d = value_d(h);
                        load_piece<VW * 4>(v[s][j][h], row + bytes(d), from < 0 ? 0 : bytes(D - d));
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
                if constexpr (BITS == 4) {
                    const uint32_t w = k[s][c / 2][c % 2];
                    image = u32x4{image4<QT>(w, 0), image4<QT>(w, 1), image4<QT>(w, 2), image4<QT>(w, 3)};
                } else if constexpr (QUANT) {
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
                if constexpr (BITS == 4) z[s][r] = __builtin_fmaf(ko[s][r] - kBias4, qsum, z[s][r]);
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
            if constexpr (BITS == 4) osum *= f;
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
                if constexpr (BITS == 4) {
#pragma unroll
                    for (int i = 0; i < 8; i++) vo[i / 4][i % 4] = (valid >> i) & 1 ? vo[i / 4][i % 4] : 0.0f;
                }
            }
            if constexpr (BITS == 4) {
#pragma unroll
                for (int i = 0; i < 8; i++) osum = __builtin_fmaf(p[i], vo[i / 4][i % 4] - kBias4, osum);
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
                    if constexpr (BITS == 4) {
                        // the low or the high half of the words of two positions; codes i % 4 of their halves
                        const uint32_t half = PE == 4 ? (col & 1 ? 0x07060302u : 0x05040100u) : i < 4 ? 0x05040100u : 0x07060302u;
                        image[w] = image4<PT>(__builtin_amdgcn_perm(v[s][j + 1][h][0], v[s][j][h][0], half), i % 4);
                    } else if constexpr (QUANT)
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
        if constexpr (BITS == 4) {
            osum = over_groups(osum, [](float x, float y) { return x + y; });
#pragma unroll
            for (int h = 0; h < NP; h++)
#pragma unroll
                for (int i = 0; i < PE; i++) acc[h][i] += osum;
        }
    }
};

// int4, where keys and values lie alike, and scales and offsets, in blocks of 8 tokens and more, so that every half of a tile lies in one
// block.  A row is 72 bytes of memory for as much arithmetic as one of 256 in 16 bits, so it is instructions that Decode runs short
// of, not memory or matrix cycles, and this is about their number:
//   the bias of the key images is what the first MFMA's sum starts from; that of the value images is taken off at the end, with the
//   sum of the rounded products P_j scale_j that two more MFMAs keep, so it cancels exactly, and the two bf16 terms, 2^-16 of P_j scale_j,
//   count for the code alone.  (With one term, 2^-8, 64 sequences of up to 8192 take 60 to 63 us, not 62 to 65, but an output whose code and offset
//   cancel is off by up to 2^-5 of the scale, and over 37 positions outputs by 0.0023 of their norm, not by the 0.0017 of their own rounding)
//   exponents are taken from a number m that is raised only where a score is more than kSlack above it, so the look at all lanes
//   of a head is left out as a rule; sums stay below 2^kSlack of what they would be, far from the end of float32
//   scales and offsets come one position to a lane and are handed round through LDS: one load where Decode has four
// Against Decode, 8 heads of 128: 32 sequences of up to 4095 25.7 and 34.0 us, 64 of up to 8192 65 and 92, one of 131071 40.1 and 45.8,
// one of 37 7.3 and 7.0; 64 of up to 8192, heads of 64 51 and 61, of 80 65 and 95; 32 of them, of 256 66 and 89.
//   kTogether  a token's heads share cache lines, and other workgroups want what this one leaves
//   kAlone     heads have lines of their own, which nobody else wants, and requests are marked so (64 of up to 8192: 66.1 us, 71.8 unmarked; heads
//              of 64 51.0 and 52.0, of 80 65.1 and 67.5; one of 131071 39.5 and 42.3) - but rows of 65 bytes and more come in two requests for the
//              same line, which the mark makes two trips (heads of 256: 66.9 us marked and 65.7; 32 of up to 4095, token by token, 49 and 41)
//   kAny       a mask, blocks of other than a multiple of 16 tokens, scales and offsets that do not lie token by token.  What that takes would cost the
//              others 3 to 10 of a hundred.  Masked, 64 of up to 8192 81 us, 95 with Decode, 32 of up to 4095 29.5 and 34.8, 8 of up to 500 11.2 and
//              10.5; blocks of 24, 32 of up to 4095 33 and 40, 4 of 1000 12.8 and 12.3
enum Kind { kAlone, kTogether, kAny };
template <int DP, int QT, Kind KIND>
struct Decode4 {
    static constexpr int NCH = DP / 32, KL = NCH / 2, PE = DP >= 128 ? 8 : 4, NP = DP / (16 * PE);
    static constexpr float kShift = 0.0f, kSlack = 8.0f, kNone = -3.402823466e38f;
    static constexpr int HS = kStep / 4;                         // halves of a step of a wavefront: a tile
    static constexpr int kOnce = KIND == kAlone && DP < 256 ? 2 : 0;             // cache-policy bit: not temporal

    struct Place {                                               // of a step's halves
        int n[HS], key[HS], off[HS], id[HS];                     // positions that are there, the first of them, its token within its block, its block
    };

    const Args a;
    const int wave, col, g, D;
    const bool wide;
    uint32_t koff[KL], voff[4][NP];
    uint32_t k[HS][KL][2], v[HS][4][NP];
    float param[4];                                              // of position `lane` of the step: key scale, offset, value scale, offset
    bool hidden;                                                 // and what the mask says of it
    float *const lds;                                            // [4][64], of the whole step: key scale times scale2, key offset, value scale, value
                                                                 // offset times value scale
    u32x4 q[NCH];
    f32x4 acc[NP][PE], bias;
    float m, l, qsum, osum;

    int len, half_end;
    const int32_t *table;
    const uint8_t *mask;
    const char *kbase, *vbase;
    const char *ksbase, *kobase, *vsbase, *vobase;

    __device__ Decode4(Args args, float *own) : Decode4(args, thread_now(), own) {}
    __device__ __forceinline__ Decode4(Args args, int thread, float *own)
        : a(args), wave(uniform(thread >> 6)), col(thread & 15), g((thread & 63) >> 4), D(args->cache.dim), wide(args->cache.dim % 32 == 0), lds(own)
    {
#pragma unroll
        for (int c = 0; c < KL; c++) {
            const int d = first_d(c);
            koff[c] = d < D ? (uint32_t)col * (uint32_t)a->cache.key.token + d / 2 : kOutOfRange;
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int h = 0; h < NP; h++) {
                const int d = h * 128 + (PE == 4 ? col / 2 * 8 : col * PE);
                voff[j][h] = d < D ? (uint32_t)(g * 4 + j) * (uint32_t)a->cache.key.token + d / 2 : kOutOfRange;
            }
    }

    // first d of the lane's key piece c, 16 codes: from DP 128 on pieces 2 i and 2 i + 1 lie side by side
    __device__ __forceinline__ int first_d(int c) const { return KL >= 2 ? c / 2 * 128 + g * 32 + c % 2 * 16 : g * 16; }

    __device__ __forceinline__ void begin(int b, int kvh, int head0, int rows, int len_, int half_end_)
    {
        len = len_, half_end = half_end_;
        table = a->table + b * a->table_stride;
        if constexpr (KIND == kAny) {
            mask = a->mask ? a->mask + b * a->mask_stride : nullptr;
            hidden = false;
        }
        kbase = a->cache.key.base + kvh * a->cache.key.head;
        vbase = a->cache.value.base + kvh * a->cache.value.head;
        ksbase = a->cache.key_scale.base + kvh * a->cache.key_scale.head;
        kobase = a->cache.key_offset.base + kvh * a->cache.key_offset.head;
        vsbase = a->cache.value_scale.base + kvh * a->cache.value_scale.head;
        vobase = a->cache.value_offset.base + kvh * a->cache.value_offset.head;
        const uint16_t *row = a->q + b * a->q_batch + (head0 + min(col, rows - 1)) * a->q_head;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const int d = first_d(c / 2) + c % 2 * 8;            // (D is a multiple of 16: a piece exists as a whole or not at all)
            typedef u32x4 anywhere __attribute__((aligned(2)));
            q[c] = u32x4{0, 0, 0, 0};
            if (col < rows && d < D) q[c] = *(const Global<anywhere> *)(row + d);
        }
        osum = 0.0f;
        m = kNone, l = 0.0f;
        bias = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < NP; h++)
#pragma unroll
            for (int i = 0; i < PE; i++) acc[h][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // the query in the order of image4, (d, d + 4), and its sum
    __device__ __forceinline__ void order_query()
    {
        qsum = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const u32x4 w = q[c];
#pragma unroll
            for (int i = 0; i < 4; i++) qsum += act_lo<QT>(w[i]) + act_hi<QT>(w[i]);
            q[c] = u32x4{__builtin_amdgcn_perm(w.z, w.x, 0x05040100u), __builtin_amdgcn_perm(w.z, w.x, 0x07060302u),
                         __builtin_amdgcn_perm(w.w, w.y, 0x05040100u), __builtin_amdgcn_perm(w.w, w.y, 0x07060302u)};
        }
        qsum = over_groups(qsum, [](float x, float y) { return x + y; });
    }
    // the first position of half `half`, at token `off` of the sequence's block `span`, and how many tokens of it the block has
    __device__ __forceinline__ int key_of(int half, uint32_t span, int off) const { return KIND == kAny ? (int)(span * a->span.d) + off : half * kHalf; }
    __device__ __forceinline__ int in_block(const Place &p, int s) const { return KIND == kAny ? min((int)a->span.d - p.off[s], kHalf) : kHalf; }
    __device__ __forceinline__ Place place(int first) const
    {
        Place p;
        const uint32_t half = uniform((uint32_t)first), span = divide(half, a->halves);
        const int off = (int)(half - span * a->halves.d) * kHalf;
        if (a->halves.d % HS == 0) {                             // (a piece begins at a multiple of HS halves)
            const int id = scalar_load(table + min(span, (uint32_t)a->max_blocks - 1));
#pragma unroll
            for (int s = 0; s < HS; s++) p.off[s] = off + s * kHalf, p.key[s] = key_of(first + s, span, p.off[s]), p.id[s] = id;
        } else {
#pragma unroll
            for (int s = 0; s < HS; s++) {
                const uint32_t span_s = s ? divide(half + s, a->halves) : span;
                p.off[s] = s ? (int)(half + s - span_s * a->halves.d) * kHalf : off;
                p.key[s] = key_of(first + s, span_s, p.off[s]);
                p.id[s] = scalar_load(table + min(span_s, (uint32_t)a->max_blocks - 1));
            }
        }
#pragma unroll
        for (int s = 0; s < HS; s++)
            p.n[s] = KIND == kAny ? first + s < half_end ? min(max(len - p.key[s], 0), in_block(p, s)) : 0
                                  : min(max(min(len, half_end * kHalf) - p.key[s], 0), kHalf);
        return p;
    }
    // a block that the table does not name holds nothing
    __device__ __forceinline__ void settle(Place &p) const
    {
        if (a->halves.d % HS == 0) {
            if ((uint32_t)p.id[0] >= (uint32_t)a->cache.num_blocks)
#pragma unroll
                for (int s = 0; s < HS; s++) p.n[s] = 0, p.id[s] = 0;
        } else {
#pragma unroll
            for (int s = 0; s < HS; s++)
                if ((uint32_t)p.id[s] >= (uint32_t)a->cache.num_blocks) p.n[s] = 0, p.id[s] = 0;
        }
    }
    __device__ __forceinline__ uint64_t start_of(const Place &p, int s) const
    {
        return (uint64_t)(uint32_t)p.id[s] * (uint32_t)a->cache.key.block + (uint32_t)p.off[s] * (uint32_t)a->cache.key.token;
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const char *base, const Place &p, int s) const
    {
        const uint32_t reach = p.n[s] > 0 ? (uint32_t)(p.n[s] - 1) * (uint32_t)a->cache.key.token + D / 2 : 0;
        return make_rsrc((const char *)((uint64_t)base + start_of(p, s)), reach);
    }
    // f(descriptor, scalar offset, half): where the halves' rows are - from the first one's on, if they are whole and of one block
    template <class F>
    __device__ __forceinline__ void each_half(const char *base, const Place &p, F f) const
    {
        if (full(p) && a->halves.d % HS == 0) {
            const __amdgpu_buffer_rsrc_t r = make_rsrc((const char *)((uint64_t)base + start_of(p, 0)), 0x7fffffffu);
#pragma unroll
            for (int s = 0; s < HS; s++) f(r, (uint32_t)(s * kHalf) * (uint32_t)a->cache.key.token, s);
        } else {
#pragma unroll
            for (int s = 0; s < HS; s++) f(rows_of(base, p, s), 0, s);
        }
    }
    // (those of a half that ends early lie in its block; of one that the block ends the last ones are read twice)
    __device__ __forceinline__ void load_params(const Place &p)
    {
        const uint32_t token = KIND == kAny ? (uint32_t)a->cache.key_scale.token : 4;
        uint32_t start = 0;
        int n = 0, key = 0;
#pragma unroll
        for (int s = 0; s < HS; s++) {
            const uint32_t of_half = (uint32_t)p.id[s] * (uint32_t)a->cache.key_scale.block + (uint32_t)p.off[s] * token;
            const bool here = s == 0 || g == s;                  // (the groups behind the last half have the first one's)
            start = here ? of_half : start;
            n = here ? p.n[s] : n;
            key = here ? p.key[s] : key;
        }
        start += (uint32_t)(KIND == kAny ? min(col, max(n - 1, 0)) : col) * token;
        param[0] = *(const Global<float> *)(at(ksbase) + start);
        param[1] = *(const Global<float> *)(at(kobase) + start);
        param[2] = *(const Global<float> *)(at(vsbase) + start);
        param[3] = *(const Global<float> *)(at(vobase) + start);
        if constexpr (KIND == kAny)
            if (mask) hidden = col < n && at(mask)[key + col] != 0;
    }
    // (a row of D % 32 == 0 is whole pieces of 16 bytes, of which a lane takes one)
    __device__ __forceinline__ void load_keys(const Place &p)
    {
        each_half(kbase, p, [&](__amdgpu_buffer_rsrc_t r, uint32_t offset, int s) {
            if constexpr (KL >= 2) {
                if (wide) {
#pragma unroll
                    for (int c = 0; c < KL; c += 2) {
                        const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(r, koff[c], offset, kOnce);
                        k[s][c][0] = w.x, k[s][c][1] = w.y, k[s][c + 1][0] = w.z, k[s][c + 1][1] = w.w;
                    }
                    return;
                }
            }
#pragma unroll
            for (int c = 0; c < KL; c++) {
                const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(r, koff[c], offset, kOnce);
                k[s][c][0] = w.x, k[s][c][1] = w.y;
            }
        });
    }
    __device__ __forceinline__ void load_values(const Place &p)
    {
        each_half(vbase, p, [&](__amdgpu_buffer_rsrc_t r, uint32_t offset, int s) {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int h = 0; h < NP; h++) v[s][j][h] = __builtin_amdgcn_raw_buffer_load_b32(r, voff[j][h], offset, kOnce);
        });
    }
    // parameter i of the lane's four positions of half s
    __device__ __forceinline__ f32x4 four(int i, int s) const { return *reinterpret_cast<const f32x4 *>(lds + i * 64 + s * 16 + g * 4); }
    // bit 4 s + r: position 4 g + r of half s is seen
    __device__ __forceinline__ uint32_t seen(const Place &p) const
    {
        uint32_t bits = 0;
#pragma unroll
        for (int s = 0; s < HS; s++) bits |= ((1u << min(max(p.n[s] - g * 4, 0), 4)) - 1) << (4 * s);
        return bits;
    }
    __device__ static __forceinline__ bool full(const Place &p) { return p.n[0] + p.n[1] == HS * kHalf; }
    __device__ static __forceinline__ void no_select() { asm volatile(""); }
    // (of fmaxf the compiler would make two instructions for each, for signalling NaNs)
    __device__ static __forceinline__ float max3(float x, float y, float z)
    {
        float r;
        asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
        return r;
    }

    // z_j over its factor, four(0)
    __device__ __forceinline__ void score(f32x4 (&z)[HS]) const
    {
        const float less = -kBias4 * qsum;
#pragma unroll
        for (int s = 0; s < HS; s++) {
            z[s] = f32x4{less, less, less, less};
#pragma unroll
            for (int i = 0; i < NCH; i++) {
                const uint32_t w = k[s][i / 2][i % 2];
                z[s] = mfma_act<QT>(u32x4{image4<QT>(w, 0), image4<QT>(w, 1), image4<QT>(w, 2), image4<QT>(w, 3)}, q[i], z[s]);
            }
        }
#pragma unroll
        for (int s = 0; s < HS; s++) {
            const f32x4 ko = four(1, s);
#pragma unroll
            for (int r = 0; r < 4; r++) z[s][r] = __builtin_fmaf(ko[r], qsum, z[s][r]);
        }
    }
    __device__ __forceinline__ void store_scores(const Place &p, const f32x4 (&z)[HS], uint32_t valid, int b, int head0, int rows, int first) const
    {
        if (col >= rows) return;
        Global<float> *to = at(a->scores) + ((int64_t)b * a->heads + head0 + col) * a->score_pitch + g * 4;
#pragma unroll
        for (int s = 0; s < HS; s++) {
            if (first + s >= half_end || g * 4 >= min(len - p.key[s], in_block(p, s))) continue;       // (positions are stored in fours)
            const f32x4 t = four(0, s);
            f32x4 w;
#pragma unroll
            for (int r = 0; r < 4; r++) w[r] = (valid >> (4 * s + r)) & 1 ? z[s][r] * t[r] : -INFINITY;
            *(Global<f32x4> *)(to + p.key[s]) = w;
        }
    }
    // probabilities times value scales
    __device__ __forceinline__ void add(bool whole, uint32_t valid, const f32x4 (&z)[HS], u32x4 (&terms)[2])
    {
        constexpr int N = HS * 4;
        float e[N];
        const auto exponents = [&] {
#pragma unroll
            for (int s = 0; s < HS; s++) {
                const f32x4 t = four(0, s);
#pragma unroll
                for (int r = 0; r < 4; r++) e[4 * s + r] = __builtin_fmaf(z[s][r], t[r], -m);
            }
            if (!whole) {
                no_select();
#pragma unroll
                for (int i = 0; i < N; i++) e[i] = (valid >> i) & 1 ? e[i] : -INFINITY;
            }
        };
        exponents();
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; i += 2) top = max3(top, e[i], e[i + 1]);
        if (__any(top > kSlack)) {
            top = -INFINITY;
#pragma unroll
            for (int s = 0; s < HS; s++) {
                const f32x4 t = four(0, s);
#pragma unroll
                for (int r = 0; r < 4; r++) top = fmaxf(top, (valid >> (4 * s + r)) & 1 ? z[s][r] * t[r] : -INFINITY);
            }
            top = over_groups(top, [](float x, float y) { return fmaxf(x, y); });
            const float higher = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - higher);
            m = higher;
            l *= f;
            osum *= f;
            bias *= f;
#pragma unroll
            for (int h = 0; h < NP; h++)
#pragma unroll
                for (int i = 0; i < PE; i++) acc[h][i] *= f;
            exponents();
        }
#pragma unroll
        for (int s = 0; s < HS; s++) {
            f32x4 vs = four(2, s), vo = four(3, s);
            float p[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                p[r] = __builtin_amdgcn_exp2f(e[4 * s + r]);
                l += p[r];
            }
            if (!whole) {                                        // (a scale and an offset that are not seen may be anything)
                no_select();
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    vs[r] = (valid >> (4 * s + r)) & 1 ? vs[r] : 0.0f;
                    vo[r] = (valid >> (4 * s + r)) & 1 ? vo[r] : 0.0f;
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                osum = __builtin_fmaf(p[r], vo[r], osum);
                p[r] = p[r] * vs[r];
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int to = s * 2 + i;
                terms[0][to] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
                terms[1][to] = pack_bf16x2(p[2 * i] - bf16_lo(terms[0][to]), p[2 * i + 1] - bf16_hi(terms[0][to]));
            }
        }
    }
    __device__ __forceinline__ void weigh(const u32x4 (&terms)[2])
    {
#pragma unroll
        for (int n = 0; n < 2; n++) bias = mfma_act<0>(u32x4{kOnes2<0>, kOnes2<0>, kOnes2<0>, kOnes2<0>}, terms[n], bias);
#pragma unroll
        for (int h = 0; h < NP; h++) {
            uint32_t pairs[4][2];                                // the low and the high halves of the words of two positions
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const uint32_t x = v[w / 2][w % 2 * 2][h], y = v[w / 2][w % 2 * 2 + 1][h];
                pairs[w][0] = __builtin_amdgcn_perm(y, x, PE == 4 && col & 1 ? 0x07060302u : 0x05040100u);
                pairs[w][1] = PE == 4 ? 0 : __builtin_amdgcn_perm(y, x, 0x07060302u);
            }
#pragma unroll
            for (int i = 0; i < PE; i++) {
                const u32x4 image = {image4<0>(pairs[0][i / 4], i % 4), image4<0>(pairs[1][i / 4], i % 4), image4<0>(pairs[2][i / 4], i % 4),
                                     image4<0>(pairs[3][i / 4], i % 4)};
#pragma unroll
                for (int n = 0; n < 2; n++) acc[h][i] = mfma_act<0>(image, terms[n], acc[h][i]);
            }
        }
    }

    // Wavefronts that have come less far go first: those of a compute unit then end together (64 sequences of up to 8192: 65.1 us, 68.6
    // without; 32 of up to 4095 25.7 and 27.0).
    __device__ static __forceinline__ void set_priority(int quarters)
    {
        if (quarters == 3) __builtin_amdgcn_s_setprio(3);
        else if (quarters == 2) __builtin_amdgcn_s_setprio(2);
        else if (quarters == 1) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
    }

    // The wavefront's steps of the halves from `from` to half_end, requested as in Decode::run.  A step's parameters come one to a lane
    // and are handed round through LDS, so that a step ahead of them is four registers.
    __device__ __forceinline__ void run(int from, int b, int head0, int rows)
    {
        int first = from + wave * HS;
        const int end = half_end;
        Place cur = place(first);
        settle(cur);
        load_keys(cur);
        load_params(cur);
        __builtin_amdgcn_sched_barrier(0);
        load_values(cur);
        __builtin_amdgcn_sched_barrier(0);
        order_query();
        Place next = place(first + 4 * HS);
        int behind = 4, quarter_end = from;                      // quarters that are not done
        for (; first < end; first += 4 * HS) {
            if (first >= quarter_end) {
                quarter_end += (end - from) / 4;
                set_priority(--behind);
            }
            uint32_t valid = (1u << (4 * HS)) - 1;
            bool whole = full(cur);
            if (!whole) {
                no_select();
                valid = seen(cur);
            }
            if (KIND == kAny && mask) {
                const uint32_t out = (uint32_t)__ballot(hidden) >> (g * 4);
                valid &= ~((out & 15) | (out >> 16 & 15) << 4);
                whole = whole && !__any(hidden);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) lds[i * 64 + g * 16 + col] = i == 0 ? param[0] * a->scale2 : i == 3 ? param[3] * param[2] : param[i];
            __builtin_amdgcn_wave_barrier();                     // (a wavefront's LDS accesses are done in their order)
            f32x4 z[HS];
            score(z);
            if (a->scores) store_scores(cur, z, valid, b, head0, rows, first);
            settle(next);
            load_keys(next);
            load_params(next);
            __builtin_amdgcn_sched_barrier(0);
            u32x4 terms[2];
            add(whole, valid, z, terms);
            weigh(terms);
            __builtin_amdgcn_wave_barrier();
            load_values(next);
            __builtin_amdgcn_sched_barrier(0);
            cur = next;
            next = place(first + 8 * HS);
        }
        osum = __builtin_fmaf(-kBias4, bias[0], over_groups(osum, [](float x, float y) { return x + y; }));
#pragma unroll
        for (int h = 0; h < NP; h++)
#pragma unroll
            for (int i = 0; i < PE; i++) acc[h][i] += osum;
        m = m == kNone ? -INFINITY : m;                          // nothing seen: sums of 0 - or NaN, from NaN scores
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

// Adds the sums of n cut pieces at place(0), place(1), ..., ascending, in this order, into `own`, which already holds those of number
// `mine`.  A thread adds one quad, eight partials in flight; where there are fewer quads than threads, several share the
// partials of a quad.  What the partials weigh is worked out meanwhile, 16 lanes to a head.
constexpr int kFlight = 8;
constexpr int kJoin = 64;                                        // sums of one call at most
constexpr size_t kJoinLds = (kJoin * kHeads + 256 * 4) * sizeof(float);
template <int DP, class Place>
__device__ void join(Args a, const Sums<DP> &own, int mine, Place place, int n, int rows, float *lds)
{
    constexpr int QPR = DP / 4;
    const int thread = thread_now();
    const uint32_t row_bytes = DP * 4, place_bytes = (uint32_t)a->rows * row_bytes;
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

// What the wavefronts of a workgroup share.
template <int DP>
struct Shared {
    static constexpr int RP = 128 + 4;                           // row pitch of a wavefront's sums
    static constexpr int NP = DP / 128 ? DP / 128 : 1;           // pieces of 128 (or 64) outputs
    alignas(16) float red[4][kHeads][RP];
    alignas(16) float ml[4][kHeads][2];
    alignas(16) float all_wide[NP > 1 ? kHeads : 1][Sums<DP>::RP];           // the workgroup's sums: the first wavefront's place, if they fit
    alignas(16) float all_ml[kHeads][2];
    int counted[2];
    int last_here;
    static_assert(NP > 1 || Sums<DP>::RP == RP, "the workgroup's sums lie where a wavefront's were");
    static_assert(sizeof(red) - sizeof(red[0]) >= kJoinLds, "join works behind the workgroup's sums");
};

// The end of a piece, number `number` of n of a pair, with the sums of this workgroup's four wavefronts; place(i): where piece i's
// sums lie in the workspace.
template <int DP, int QT, int NP, int PE, class Place>
__device__ __forceinline__ void end_piece(Shared<DP> &lds, const f32x4 (&acc)[NP][PE], float l, float m, int64_t out_row, int rows, int n, int number, Place place,
                                          float shift)
{
    const Args a = args_now();
    Global<uint32_t> *arrived = at(a->arrived);
    // Of a pair that is cut, the last of its workgroups to arrive adds everybody's sums.  Where those are more than 64 KiB, groups
    // of about the root of their number are added first, so that no workgroup has many to read (one sequence of 8000, 16
    // query heads each: 19.5 us, 25.7 without groups; with 4 heads each and 4000 tokens 11.9 us at once, 13.8 in groups).  The
    // counter of a group is its first piece's, that of the groups lies behind all of these.
    int size = n, group = 0, groups = 1;
    if (n >= kJoin || n * rows * (DP / 4) > 512 * kFlight) {
        size = 8;
        while (size * size < n) size += 4;
        group = uniform(number / size), groups = uniform((n + size - 1) / size);
    }
    const int members = min(size, n - group * size);
    const uint32_t whole = place(0), first = place(group * size), behind = 2 * (uint32_t)a->shares;
    uint32_t seen = 0;                                       // how many have arrived: requested here, looked at behind what follows
    if (n > 1 && threadIdx.x < 2)
        seen = __hip_atomic_load(arrived + (threadIdx.x ? behind + whole : first), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

    // the four wavefronts' sums on a common maximum
    const int thread = thread_now(), lane = thread & 63, wave = thread >> 6, col = lane & 15, g = lane >> 4;
    const Sums<DP> own = {NP > 1 ? lds.all_wide : reinterpret_cast<float (*)[Sums<DP>::RP]>(lds.red[0]), lds.all_ml};
    l = over_groups(l, [](float x, float y) { return x + y; });
    if (g == 0) lds.ml[wave][col][0] = m, lds.ml[wave][col][1] = l;
    __syncthreads();
    const float top = fmaxf(fmaxf(lds.ml[0][col][0], lds.ml[1][col][0]), fmaxf(lds.ml[2][col][0], lds.ml[3][col][0]));
    const float f = weight_of(m, top);
    if (thread < kHeads) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) total += lds.ml[i][col][1] * weight_of(lds.ml[i][col][0], top);
        lds.all_ml[col][0] = top, lds.all_ml[col][1] = total;
    }
#pragma unroll
    for (int h = 0; h < NP; h++) {
        if (h) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int i = 0; i < PE; i += 4)
                *reinterpret_cast<f32x4 *>(&lds.red[wave][col][(g * 4 + r) * PE + i]) =
                    f32x4{acc[h][i][r] * f, acc[h][i + 1][r] * f, acc[h][i + 2][r] * f, acc[h][i + 3][r] * f};
        __syncthreads();
        constexpr int QPR = 16 * PE / 4;                  // quads of a row
        for (int e = thread; e < rows * QPR; e += 256) {
            const int row = e / QPR, d = (e % QPR) * 4;
            f32x4 sum = *reinterpret_cast<const f32x4 *>(&lds.red[0][row][d]);
#pragma unroll
            for (int i = 1; i < 4; i++) sum += *reinterpret_cast<const f32x4 *>(&lds.red[i][row][d]);
            own.quad(row, h * 128 + d) = sum;
        }
    }
    if (thread < 2) lds.counted[thread] = (int)seen;
    __syncthreads();

    bool done = true;
    const auto last_of = [&](Global<uint32_t> *counter, int of, int seen, uint32_t place) {
        if (of == 1) return true;
        if (seen == of - 1) {                                // everybody else was there already: nobody waits for these sums
            if (thread == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            return true;
        }
        publish<DP>(a, own, place, rows);
        return arrive(counter, of, &lds.last_here);
    };
    const int seen0 = uniform(lds.counted[0]), seen1 = uniform(lds.counted[1]);
#pragma unroll 1
    for (int level = 0; level < 2 && done; level++) {        // within the group, among the groups
        const int of = level ? groups : members;
        done = last_of(arrived + (level ? behind + whole : first), of, level ? seen1 : seen0, level ? first : place(number));
        const int from = level ? 0 : group * size, step = level ? size : 1;
        if (done && of > 1) join<DP>(a, own, level ? group : number - from, [&](int i) { return place(from + i * step); }, of, rows, &lds.red[1][0][0]);
    }
    if (done) finish<DP, QT>(args_now(), own, out_row, rows, shift);
    __syncthreads();                                             // ml and red are free again
}

// outputs of the sequences without positions
__device__ __forceinline__ void clear_empty()
{
    const Args a = args_now();
    for (int e = blockIdx.x; e < a->batch; e += gridDim.x) {
        if (clamp_len(a, scalar_load(a->lens + e)) != 0) continue;
        for (int i = threadIdx.x; i < a->heads * a->cache.dim; i += 256) at(a->out)[(int64_t)e * a->heads * a->cache.dim + i] = 0;
        for (int i = threadIdx.x; i < a->heads; i += 256)
            if (a->lse) at(a->lse)[(int64_t)e * a->heads + i] = -INFINITY;
    }
}

template <int DP, int QT, class W>
__device__ __forceinline__ void decode_pieces()
{
    __shared__ Shared<DP> lds;
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
            const int kvh = a->tiles == 1 ? (int)pair : uniform((int)pair / a->tiles), halves = (int)halves_of(a, len), units = (halves + kUnit - 1) / kUnit;
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

        end_piece<DP, QT>(lds, acc, l, m, (int64_t)b * args_now()->heads + head0, rows, n, number, [&](int i) { return first_cut + (uint32_t)i; }, W::kShift);
    }

    if (pieces.empty) clear_empty();
}

// How Decode4's work is cut up: the sequences, one after the other, into ranges of `share` halves, the same for every pair.  A
// workgroup takes one range of one pair; a sequence's pieces are the ranges that it touches.  There are `ranges` workgroups for a pair at once,
// the start and the end of a range cost as much as kStart halves, and the addition of a sequence's pieces as much as kCut.  Taken is the least of
//   whole   every sequence a range of its own, in rounds if there are more than `ranges`
//   cut     every sequence into pieces of its own of `share` halves, no longer than the average range, at most `ranges` in all
//   dense   kStart and the halves of a sequence behind those of the one before, so that a range may end one and begin the next
// What is short takes as long as its longest piece: 64 sequences of up to 100, 8 heads of 128, 9.0 us, 17.1 dense, 8 of up to 600 10.7 and 12.3, one of
// 1200 10.6 and 12.0.  What is long and cut evenly leaves the last pieces to run alone: 32 of up to 4095, with one bf16 term for the weights, 26.3 us
// dense, 27.3 in pieces of its sequences in one round, 33.9 in Pieces, which are more than fit at once.
struct Ranges {
    uint32_t share, count, before, mine, total;      // halves of a range; ranges at most; halves in the runs before this lane's, in it, in all
    int run, len;                            // sequences per lane; the length of the first
    bool dense, empty;                       // there is a sequence without positions

    __device__ explicit Ranges(Args a)
    {
        const int lane = threadIdx.x & 63, batch = a->batch;
        run = (batch + 63) / 64;
        const int first = lane * run, end = min(first + run, batch);
        len = first < batch ? clamp_len(a, at(a->lens)[first]) : 0;
        const uint32_t own = halves_of(a, len);
        const auto others = [&](auto f) {                        // halves of the lane's other sequences
            for (int i = first + 1; i < end; i++) f(halves_of(a, clamp_len(a, at(a->lens)[i])));
        };
        uint32_t halves = own, units = units_in(own), longest = units, there = own > 0;
        bool none = first < batch && own == 0;
        others([&](uint32_t h) { halves += h, units += units_in(h), longest = max(longest, units_in(h)), there += h > 0, none = none || h == 0; });
        empty = __any(none);
        const uint32_t ranges = a->ranges, sequences = run == 1 ? (uint32_t)__builtin_popcountll(__ballot(there)) : over_lanes(there, Add());
        const uint32_t steps = over_lanes(units, Add());
        uint32_t chosen = kStep, most = ranges, cost = units * kStep;
        bool close = false;
        if (sequences <= ranges && !__any(longest > 2)) {        // whole: two steps take less than an addition
            if (__any(longest > 1)) chosen = 2 * kStep;
            cost = there * chosen;
            most = sequences;
        } else if (steps > ranges) {                             // (else cut into single steps)
            const uint32_t all = over_lanes(halves, Add()), tallest = over_lanes(longest, Max());
            const uint32_t average = max(divide(all + sequences * kStart + ranges - 1, a->by_ranges), (uint32_t)kStep);
            // pieces of u units, no longer than the average range, or, where that is short, taking no more steps (4 sequences of 4000, 8 heads:
            // 15.7 us, 17.2 dense)
            uint32_t u = average <= 2 * kStep ? units_in(average) : average / kStep;
            bool cut = false;
            if (run == 1) {
                const auto pieces = [units](uint32_t u) { return over_lanes((units + u - 1) / u, Add()); };
                while (u > 1 && pieces(u) <= ranges) u--, cut = true;
                u += cut;
            } else if (sequences < ranges) {                     // (as many pieces as units / u and one more for each sequence)
                cut = steps <= (uint64_t)u * (ranges - sequences);
            }
            const uint32_t rounds = divide(sequences + ranges - 1, a->by_ranges);
            const bool whole = (uint64_t)rounds * (kStart + tallest * kStep) < kStart + kCut + (cut ? u * kStep : average);
            close = !whole && !cut;
            chosen = whole ? tallest * kStep : cut ? u * kStep : average;
            most = whole ? sequences : ranges;
            cost = cost_of(own, close, chosen);
            others([&](uint32_t h) { cost += cost_of(h, close, chosen); });
        }
        dense = close, share = chosen, count = most, mine = cost;
        const uint32_t scan = scan_lanes(mine, Add());
        before = scan - mine;
        total = (uint32_t)__builtin_amdgcn_readlane((int)scan, 63);
    }
    __device__ static uint32_t units_in(uint32_t halves) { return (halves + kStep - 1) / kStep; }
    template <class Op>
    __device__ static uint32_t over_lanes(uint32_t v, Op op) { return (uint32_t)__builtin_amdgcn_readlane((int)scan_lanes(v, op), 63); }
    __device__ uint32_t start() const { return dense ? kStart : 0; }
    __device__ static uint32_t cost_of(uint32_t halves, bool dense, uint32_t share)
    {
        return dense ? halves ? halves + kStart : 0 : (halves + share - 1) / share * share;
    }
    // the sequence that holds y, its length, and what comes before it
    __device__ void find(Args a, uint32_t y, int &b, int &length, uint32_t &start) const
    {
        const int lane = __builtin_ctzll(__ballot(y >= before && y - before < mine));
        b = lane * run;
        start = (uint32_t)__builtin_amdgcn_readlane((int)before, lane);
        length = __builtin_amdgcn_readlane(len, lane);
        if (run == 1) return;
        uint32_t cost = cost_of(halves_of(a, length), dense, share);
        while (y - start >= cost) {
            start += cost;
            length = clamp_len(a, scalar_load(a->lens + ++b));
            cost = cost_of(halves_of(a, length), dense, share);
        }
    }
};

template <int DP, int QT, Kind KIND>
__global__ __launch_bounds__(256, resident4(DP)) void paged_decode4_kernel(AttnArgs)
{
    using W = Decode4<DP, QT, KIND>;
    __shared__ Shared<DP> lds;
    static_assert(sizeof(lds.red[0]) >= 4 * 64 * sizeof(float), "a wavefront's parameters lie where its sums will be");
    const Ranges ranges = [] {
        const Args a = args_now();
        uint32_t lines = 0;                                      // the arguments' cache lines, for the phases that follow
#pragma unroll
        for (size_t i = 0; i < sizeof(AttnArgs); i += 64) lines |= *(const __attribute__((address_space(4))) uint32_t *)((const __attribute__((address_space(4))) char *)a + i);
        const Ranges r(a);
        asm volatile("" ::"s"(lines));
        return r;
    }();
    const uint32_t share = uniform(ranges.share), total = uniform(ranges.total), count = uniform(ranges.count), pairs = (uint32_t)args_now()->pairs;
    const uint32_t all = count * pairs;

    for (uint32_t turn = blockIdx.x; turn < (all + kDealt - 1) / kDealt * kDealt; turn += gridDim.x) {
        // together: the pairs of a range side by side, eight of them on one XCD
        const bool together = KIND == kAny ? args_now()->together : KIND == kTogether;
        const uint32_t piece = together ? (turn & ~(kDealt - 1)) | ((turn & 7) << 3) | ((turn >> 3) & 7) : turn;
        uint32_t range, pair;
        if (together) {
            range = divide(piece, args_now()->by_pairs);
            pair = piece - range * pairs;
        } else {
            pair = count == args_now()->ranges ? divide(piece, args_now()->by_ranges) : uniform(piece / count);
            range = piece - pair * count;
        }
        if (piece >= all || range * share >= total) continue;
        const uint32_t range_end = min(range * share + share, total);
        uint32_t from = range * share, start;
        int b, len;
        ranges.find(args_now(), from, b, len, start);
        b = uniform(b), len = uniform(len), start = uniform(start);
#pragma unroll 1
        for (;;) {
            int head0, rows, n, number;
            float l, m;
            f32x4 acc[W::NP][W::PE];
            // dense: a sequence's first kStart are its cost alone, its halves follow; it is cut at multiples of a step of a wavefront
            const uint32_t halves = uniform(halves_of(args_now(), len)), begin = start + ranges.start();
            const auto cut = [&](uint32_t at) { return begin + min(at > begin ? (at - begin + W::HS - 1) / W::HS * W::HS : 0, halves); };
            const uint32_t to = cut(range_end);
            from = cut(from);
            // the ranges that hold the first and the last of its steps: this one as a rule, and divisions take a while
            const uint32_t last = begin + (halves - 1) / W::HS * W::HS;
            const uint32_t first_range = begin >= range * share ? range : uniform(begin / share), last_range = last < range_end ? range : uniform(last / share);
            if (from < to) {
                {
                    const Args a = args_now();
                    W w(a, &lds.red[uniform(thread_now() >> 6)][0][0]);
                    const int kvh = a->tiles == 1 ? (int)pair : uniform((int)pair / a->tiles);
                    head0 = kvh * a->group + ((int)pair - kvh * a->tiles) * kHeads;
                    rows = min(kHeads, (kvh + 1) * a->group - head0);
                    n = (int)(last_range - first_range + 1), number = (int)(range - first_range);
                    w.begin(b, kvh, head0, rows, len, (int)(to - begin));
                    w.run((int)(from - begin), b, head0, rows);
                    l = w.l, m = w.m;
#pragma unroll
                    for (int h = 0; h < W::NP; h++)
#pragma unroll
                        for (int i = 0; i < W::PE; i++) acc[h][i] = w.acc[h][i];
                }
                // Dense: a range has a piece that goes on in the next one, and one that came from the range before and ends here, at most.
                // Pair by pair, so that the arrivals of different pairs count in cache lines of their own (one sequence of 9353, 32 heads: 20 us,
                // 29 with the pairs' counters side by side; one of 131071, 8 heads: 38.9 and 40.2)
                const uint32_t places = pair * args_now()->ranges * 2 + first_range * 2;
                const auto place = [&](int i) { return places + (uint32_t)(i * 2 + (i < n - 1 ? 1 : 0)); };
                end_piece<DP, QT>(lds, acc, l, m, (int64_t)b * args_now()->heads + head0, rows, n, number, place, W::kShift);
            }
            if (!ranges.dense || begin + halves >= range_end) break;
            from = start = begin + halves;
            do len = uniform(clamp_len(args_now(), scalar_load(args_now()->lens + ++b)));
            while (len == 0);                                    // (there are halves left, so a sequence with some follows)
        }
    }
    if (ranges.empty) clear_empty();
}

template <int DP, int BITS, int QT, Addressing AD>
__global__ __launch_bounds__(256, resident(DP, BITS < 16)) void paged_decode_kernel(AttnArgs)
{
    decode_pieces<DP, QT, Decode<DP, BITS, QT, AD>>();
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
static_assert(resident4(128) <= resident(128, true) && resident4(256) <= resident(256, true), "a range leaves two sums at most");
static_assert(kNumCU * 3 * 4 * sizeof(uint32_t) <= kWorkspaceCounterBytes, "arrival counters");
static_assert(kNumCU * 3 <= (kJoin / 2) * (kJoin / 2), "groups of pieces, and members of a group");

template <int DP, int BITS, int QT>
void launch_attention(const AttnArgs &a, Addressing ad, unsigned workgroups, hipStream_t s)
{
    const dim3 grid(workgroups), block(256);
    if (ad == kRows) hipLaunchKernelGGL((paged_decode_kernel<DP, BITS, QT, kRows>), grid, block, 0, s, a);
    else if (ad == kBlockMask) hipLaunchKernelGGL((paged_decode_kernel<DP, BITS, QT, kBlockMask>), grid, block, 0, s, a);
    else if (ad == kBlock) hipLaunchKernelGGL((paged_decode_kernel<DP, BITS, QT, kBlock>), grid, block, 0, s, a);
    else if constexpr (BITS < 16) hipLaunchKernelGGL((paged_decode_kernel<DP, BITS, QT, kBlockAlike>), grid, block, 0, s, a);
}

template <int DP, int QT>
void launch_attention4(const AttnArgs &a, Addressing ad, unsigned workgroups, hipStream_t s)
{
    const dim3 grid(workgroups), block(256);
    if (ad == kPlain && !a.regular) hipLaunchKernelGGL((paged_decode4_kernel<DP, QT, kAny>), grid, block, 0, s, a);
    else if (ad == kPlain && a.together) hipLaunchKernelGGL((paged_decode4_kernel<DP, QT, kTogether>), grid, block, 0, s, a);
    else if (ad == kPlain) hipLaunchKernelGGL((paged_decode4_kernel<DP, QT, kAlone>), grid, block, 0, s, a);
    else if (ad == kRows) hipLaunchKernelGGL((paged_decode_kernel<DP, 4, QT, kRows>), grid, block, 0, s, a);
    else if (ad == kBlockMask) hipLaunchKernelGGL((paged_decode_kernel<DP, 4, QT, kBlockMask>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((paged_decode_kernel<DP, 4, QT, kBlock>), grid, block, 0, s, a);
}

template <int DP>
void launch_attention(const AttnArgs &a, int bits, bool fp16, Addressing ad, unsigned workgroups, hipStream_t s)
{
    if (bits == 4) {
        if (fp16) launch_attention4<DP, 1>(a, ad, workgroups, s);
        else launch_attention4<DP, 0>(a, ad, workgroups, s);
    } else if (bits == 8) {
        if (fp16) launch_attention<DP, 8, 1>(a, ad, workgroups, s);
        else launch_attention<DP, 8, 0>(a, ad, workgroups, s);
    } else {
        if (fp16) launch_attention<DP, 16, 1>(a, ad, workgroups, s);
        else launch_attention<DP, 16, 0>(a, ad, workgroups, s);
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
    const int bits = cache_bits(cache->dtype);
    const bool quant = bits < 16, fp16 = q_dtype == MI355_DTYPE_FP16;
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
    // pieces of 16 bytes (int4: 8, in words): rows on 16-byte boundaries, and no piece reaching past a row's end
    const int piece = bits == 4 ? 8 : 16, line = bits == 4 ? 4 : 16;
    const bool pieces = cache->head_dim * bits / 8 % piece == 0 && rows_aligned(a.cache.key, line) && rows_aligned(a.cache.value, line);
    // Halves that lie in one block: block by block, the last half of a block may be short, so blocks of fewer than 8 tokens
    // would leave most of a tile empty.  Offsets within a block have 31 bits, a block's own offset is a 32 x 32-bit product.
    const PagedArray *const arrays[] = {&a.cache.key, &a.cache.value, &a.cache.key_scale, &a.cache.value_scale, &a.cache.key_offset, &a.cache.value_offset};
    bool blocks = pieces && cache->block_size >= 8, scales = cache->block_size % 4 == 0;
    for (int i = 0; i < (bits == 4 ? 6 : quant ? 4 : 2); i++) {
        const PagedArray &x = *arrays[i];
        blocks = blocks && x.block >= 0 && x.block <= 0xffffffffll && x.token >= 0 && x.token <= 0x7fffffff / (cache->block_size + 16);
        if (i >= 2) scales = scales && x.token == 4 && aligned(x.base, 16) && x.block % 16 == 0 && x.head % 16 == 0;
    }
    const auto alike = [](const PagedArray &x, const PagedArray &y) { return x.block == y.block && x.token == y.token && x.head == y.head; };
    const bool same = quant && alike(a.cache.key, a.cache.value) && alike(a.cache.key_scale, a.cache.value_scale);
    // Decode4: offsets into a whole array of parameters have 32 bits, and so do the halves of all sequences; a few steps behind the
    // last position still have a number in 31
    const PagedArray &par = a.cache.key_scale;
    const int64_t halves = max_blocks * ((cache->block_size + kHalf - 1) / kHalf);       // of a sequence at most
    const bool plain = bits == 4 && same && alike(par, a.cache.key_offset) && alike(par, a.cache.value_offset) && par.block >= 0 && par.token >= 0 &&
                       par.block <= 0xffffffffll / cache->num_blocks && par.block * cache->num_blocks + par.token * cache->block_size <= 0xffffffffll &&
                       (!attn_sums || cache->block_size % 4 == 0) && a.capacity < 0x7fff0000 && batch * (halves + kStart) < 0x7fff0000;
    const Addressing ad = !blocks ? kRows : plain ? kPlain : mask ? (cache->block_size % 4 == 0 ? kBlockMask : kRows) : same && scales && bits == 8 ? kBlockAlike : kBlock;
    // Rows of several heads in a cache line, with other heads' rows of the same token: work on them at the same time and on one XCD,
    // so that the line comes once (16 sequences of up to 1001 tokens, 32 heads of 80: 32.4 -> 28.6 us; int8, 32 sequences of up to
    // 4095, 8 heads of 64: 34.5 -> 26.2 us).  Where heads have lines of their own, that would make the workgroups ask the same
    // memory channels at the same time (32 of up to 4095, 8 heads of 128: 68 us, against 62).
    const auto shared = [](const PagedArray &x) { return x.head % 128 != 0 && x.head < x.token; };
    a.together = shared(a.cache.key) || shared(a.cache.value);
    a.span = ad != kRows ? a.cache.page : fast_div(kHalf);
    a.halves = fast_div((a.span.d + kHalf - 1) / kHalf);
    a.regular = !mask && cache->block_size % 16 == 0 && par.token == 4;
    if (ad == kPlain) {
        a.shares = kNumCU * resident4((int)p.dp);
        // as many as the card holds, or as full sequences have steps
        const int64_t most = batch * ((halves + kStep - 1) / kStep), fit = a.shares / p.pairs;
        a.ranges = (uint32_t)(fit < 1 || most < 1 ? 1 : fit < most ? fit : most);
        a.by_ranges = fast_div(a.ranges);
        const int64_t pieces = a.ranges * p.pairs;
        p.workgroups = pieces < 2048 ? (pieces + kDealt - 1) / kDealt * kDealt : 2048;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p.dp == 64) launch_attention<64>(a, bits, fp16, ad, (unsigned)p.workgroups, s);
    else if (p.dp == 128) launch_attention<128>(a, bits, fp16, ad, (unsigned)p.workgroups, s);
    else launch_attention<256>(a, bits, fp16, ad, (unsigned)p.workgroups, s);
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
