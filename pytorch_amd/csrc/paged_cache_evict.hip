// npu_paged_cache_evict for gfx950: sequences that outgrew their budget keep the newest tokens and those with the largest
// summed attention weights, each key/value head its own.
//
// Per (sequence, head) with n > keep a token's worth is a 32-bit key that orders like (recent, sum): all ones for the recent
// ones, else the sum's bits with the sign flipped into place, 0 for NaN.  The keep-th largest key is found digit by digit
// (histograms of 11, 11 and 10 bits); among tokens with exactly that key the lowest places stay.  Kept tokens behind place
// `keep` then fill the holes before it, both in ascending order: the fewest rows move, sources and destinations are disjoint,
// so all of them move at once, in place.
//
// One workgroup of 1024 threads chooses for one (sequence, head).  Thread t holds the places t, t + 1024, ...: their sums,
// positions and keys stay in its registers over the three digits, up to 17 rounds; at 33 rounds (99 words) 86 registers spill to
// scratch, still faster than reading again; rows of more rounds are read again for each digit.  Ranks in the order of the places
// come from ballots, counted per wavefront and 1024 places, and one scan over those counts.  Bound by latency: a dozen
// barriers, three trips to memory, and 0.6 us per 1024 places.  All of that also runs for a row with one token too many, where
// the least worth alone would do.  One token over a budget of 4096, 128 rows of 128 elements:
// 7.7 us in one launch, of 16384 17.7.  64 rows of 8192 places halved: 12 us, and 15.7 for the moves of 62 MB, 4.0 TB/s.
#include "paged_cache.h"

namespace mi355 {
namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;

struct EvictArgs {
    PagedCache cache;
    const int32_t *table, *lens, *positions;
    const float *sums;
    int64_t table_stride, sums_batch, sums_head, positions_batch, positions_head;
    int32_t *new_lens, *new_positions;
    float *new_sums;
    int32_t *count;                              // [batch * heads] moves
    int32_t *moves;                              // [batch * heads][2 * most]: count places that tokens go to, then those they leave
    int64_t most, recent;
    int keep, capacity;
};

// sums as unsigned numbers in their order, NaN lowest; -0 counts as 0
__device__ __forceinline__ uint32_t worth_of(float sum, int pos, int64_t oldest)
{
    if (pos > oldest) return ~0u;
    if (sum != sum) return 0;
    const uint32_t u = __float_as_uint(sum + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Scan over the workgroup, 16 wavefronts: what the threads before this one make together; `all` gets everybody's.  `lds`: one
// word per wavefront, free again after the next barrier.
static_assert(kSelectWaves == 16, "one row of lanes holds a word of every wavefront");
template <class Op>
__device__ __forceinline__ uint32_t scan_threads(uint32_t v, uint32_t *lds, uint32_t &all, Op op)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const uint32_t scan = scan_lanes(v, op);
    if (lane == 63) lds[wave] = scan;
    __syncthreads();
    const uint32_t waves = scan_row(lds[lane & 15], op);
    all = (uint32_t)__builtin_amdgcn_readlane((int)waves, 15);
    const uint32_t others = wave ? (uint32_t)__builtin_amdgcn_readlane((int)waves, wave - 1) : 0;
    const uint32_t left_lane = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)scan, 0x138, 0xf, 0xf, false);       // wave_shr:1
    return op(others, left_lane);
}

// Moves rows of keys and values (and their scales and offsets) within one (sequence, head), W bytes per access: pieces first,
// first + step, ... of all of them.  per_row = pieces of a row of keys, then of the row of values.  BITS: of the cache's elements
// (looked up while it runs, what a row carries cost every eviction 0.3 to 0.4 us, and 6 of a hundred where 64 heads move 15000 rows each).
template <int W, int BITS>
__device__ __forceinline__ void move_pieces(const EvictArgs &a, int row, uint32_t count, uint32_t first, uint32_t step, const FastDiv &per_row)
{
    typedef uint32_t word __attribute__((ext_vector_type(W >= 4 ? W / 4 : 1)));
    const int b = row / a.cache.heads, head = row % a.cache.heads;
    const int32_t *to = a.moves + (int64_t)row * 2 * a.most, *from = to + count;
    const int32_t *table = a.table + b * a.table_stride;
    const uint32_t pieces = per_row.d / 2, all = count * per_row.d;      // below 2^31: the host checks
    for (uint32_t e = first; e < all; e += step) {
        const uint32_t r = div_by(e, per_row), piece = e - r * per_row.d;
        const uint32_t dst = (uint32_t)to[r], src = (uint32_t)from[r];
        const uint32_t dst_block = div_by(dst, a.cache.page), src_block = div_by(src, a.cache.page);
        const int dst_id = table[dst_block], src_id = table[src_block];
        if ((uint32_t)dst_id >= (uint32_t)a.cache.num_blocks || (uint32_t)src_id >= (uint32_t)a.cache.num_blocks) continue;
        const uint32_t dst_slot = (uint32_t)dst_id * a.cache.page.d + (dst - dst_block * a.cache.page.d);
        const uint32_t src_slot = (uint32_t)src_id * a.cache.page.d + (src - src_block * a.cache.page.d);
        const bool value = piece >= pieces;
        const PagedArray &x = value ? a.cache.value : a.cache.key;
        const uint32_t at = (value ? piece - pieces : piece) * W;
        char *d = x.base + a.cache.offset(x, dst_slot, head) + at;
        const char *s = x.base + a.cache.offset(x, src_slot, head) + at;
        if constexpr (W >= 4) *reinterpret_cast<word *>(d) = *reinterpret_cast<const word *>(s);
        else if constexpr (W == 2) *reinterpret_cast<uint16_t *>(d) = *reinterpret_cast<const uint16_t *>(s);
        else *d = *s;
        if (BITS < 16 && at == 0) {
            const auto move = [&](const PagedArray &one) {
                *reinterpret_cast<float *>(one.base + a.cache.offset(one, dst_slot, head)) =
                    *reinterpret_cast<const float *>(one.base + a.cache.offset(one, src_slot, head));
            };
            move(value ? a.cache.value_scale : a.cache.key_scale);
            if constexpr (BITS == 4) move(value ? a.cache.value_offset : a.cache.key_offset);
        }
    }
}

// KPT: rounds of 1024 places whose keys are held, KPT * 1024 >= capacity; 0: any number, read again for every digit (64 rows of
// 16000 places halved: 52 us held, 82 read again; of 32000, held in part in scratch, 114 and 157).
// W: bytes per access of the moves that this kernel makes itself; 0: it leaves them to paged_move_kernel.
template <int KPT, int W, int BITS>
__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(EvictArgs a, FastDiv per_row)
{
    // places per scan of the counts below: 64 rounds with one count per thread
    constexpr int kBatch = KPT ? KPT : 64;
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t found[3];
    __shared__ uint32_t wave_top[kSelectWaves], wave_sum[kSelectWaves];
    __shared__ uint32_t count[kBatch * kSelectWaves];           // per round and wavefront: the ballot's ones, then those before

    const int row = blockIdx.x, b = row / a.cache.heads, head = row % a.cache.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *sums = a.sums + b * a.sums_batch + head * a.sums_head;
    const int32_t *pos = a.positions + b * a.positions_batch + head * a.positions_head;
    float *new_sums = a.new_sums + (int64_t)row * a.capacity;
    int32_t *new_pos = a.new_positions + (int64_t)row * a.capacity;
    constexpr int kHeld = KPT ? KPT : 1;
    float sum[kHeld];
    int32_t at[kHeld];
    uint32_t key[kHeld];
    if constexpr (KPT > 0) {                                    // requested before the length is known
#pragma unroll
        for (int j = 0; j < KPT; j++) {
            const int i = min(j * kSelectThreads + tid, a.capacity - 1);
            sum[j] = i >= 0 ? sums[i] : 0.0f, at[j] = i >= 0 ? pos[i] : 0;
        }
    }
    const int n = min(max(a.lens[b], 0), a.capacity);
    const int stay = min(n, a.keep);
    if (head == 0 && tid == 0) a.new_lens[b] = stay;
    if (n <= a.keep || a.keep == 0) {
        for (int i = tid; i < a.capacity; i += kSelectThreads) new_sums[i] = i < stay ? sums[i] : 0.0f, new_pos[i] = i < stay ? pos[i] : -1;
        if (tid == 0) a.count[row] = 0;
        return;
    }
    for (int i = stay + tid; i < a.capacity; i += kSelectThreads) new_sums[i] = 0.0f, new_pos[i] = -1;
    hist[tid] = 0, hist[tid + 1024] = 0;
    int newest = INT32_MIN;
    if constexpr (KPT > 0) {
#pragma unroll
        for (int j = 0; j < KPT; j++) newest = j * kSelectThreads + tid < n ? max(newest, at[j]) : newest;
    } else {
        for (int i = tid; i < n; i += kSelectThreads) newest = max(newest, pos[i]);
    }
    uint32_t top;                                               // positions as unsigned numbers in their order
    scan_threads((uint32_t)newest ^ 0x80000000u, wave_top, top, Max());
    newest = (int)(top ^ 0x80000000u);
    const int64_t oldest = (int64_t)newest - a.recent;
#pragma unroll
    for (int j = 0; j < KPT; j++) key[j] = worth_of(sum[j], at[j], oldest);
    const int rounds = KPT ? KPT : (n + kSelectThreads - 1) / kSelectThreads;
    // calls each(j, place, key) for the thread's places, rounds [j0, j1)
    const auto walk = [&](int j0, int j1, auto &&each) {
        if constexpr (KPT > 0) {
#pragma unroll
            for (int j = 0; j < KPT; j++) each(j, j * kSelectThreads + tid, key[j]);
        } else {
            for (int j = j0; j < j1; j++) {
                const int i = j * kSelectThreads + tid;
                each(j, i, i < n ? worth_of(sums[i], pos[i], oldest) : 0u);
            }
        }
    };

    uint32_t prefix = 0, left = (uint32_t)a.keep, all;          // the left-th largest among the keys that start with prefix
#pragma unroll
    for (int digit = 0; digit < 3; digit++) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, above = digit == 2 ? 10 : 21;
        const uint32_t mask = digit == 2 ? 1023 : 2047;
        walk(0, rounds, [&](int, int i, uint32_t k) {
            if (i < n && (digit == 0 || (k >> above) == (prefix >> above))) {
                // a wavefront of equal digits counts as one: equal sums, all 0 after a prefill, would wait for each other
                const uint32_t d = (k >> shift) & mask, d0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)d);
                const uint64_t same = __ballot(d == d0);
                if (__ballot(d != d0)) atomicAdd(&hist[d], 1u);
                else if (lane == __builtin_ctzll(same)) atomicAdd(&hist[d], (uint32_t)__popcll(same));
            }
        });
        __syncthreads();
        const uint32_t c0 = hist[2047 - 2 * tid], c1 = hist[2046 - 2 * tid];       // thread 0 has the largest digits
        const uint32_t before = scan_threads(c0 + c1, wave_sum, all, Add());
        if (before < left && left <= before + c0 + c1) {                           // one thread
            const bool second = left > before + c0;
            found[0] = 2047 - 2 * tid - second;
            found[1] = left - before - (second ? c0 : 0);
            found[2] = second ? c1 : c0;
        }
        hist[2047 - 2 * tid] = 0, hist[2046 - 2 * tid] = 0;                        // nobody else's
        __syncthreads();
        prefix |= found[0] << shift;
        left = found[1];
    }
    const bool some = found[2] > left;                          // of the tokens with exactly the last key only some stay

    // Counts, per round and wavefront, become the ones before; every thread of the workgroup calls it with its part.
    const auto before_each = [&](uint32_t carry) {
        __syncthreads();
        const uint32_t mine = tid < kBatch * kSelectWaves ? count[tid] : 0;        // (kBatch * kSelectWaves <= 1024)
        const uint32_t before = scan_threads(mine, wave_sum, all, Add());
        if (tid < kBatch * kSelectWaves) count[tid] = carry + before;
        __syncthreads();
    };
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    // the holes, then as many fills
    int32_t *list = a.moves + (int64_t)row * 2 * a.most;
    uint32_t ties = 0, ranks = 0;                               // before the batch of rounds
    for (int j0 = 0; j0 < rounds; j0 += kBatch) {
        const int j1 = min(j0 + kBatch, rounds);
        uint64_t stays = 0;                                     // one bit per round
        static_assert(kBatch <= 64, "one bit per round");
        if (some) {
            walk(j0, j1, [&](int j, int i, uint32_t k) {
                const uint64_t tie = __ballot(i < n && k == prefix);
                if (lane == 0) count[(j - j0) * kSelectWaves + wave] = (uint32_t)__popcll(tie);
            });
            if (tid >= (j1 - j0) * kSelectWaves && tid < kBatch * kSelectWaves) count[tid] = 0;
            before_each(ties);
            ties += all;
        }
        walk(j0, j1, [&](int j, int i, uint32_t k) {
            bool kept = k > prefix || (k == prefix && !some);
            if (some) {
                const bool tie = i < n && k == prefix;
                const uint32_t rank = count[(j - j0) * kSelectWaves + wave] + (uint32_t)__popcll(__ballot(tie) & below);
                kept = kept || (tie && rank < left);
            }
            stays |= (uint64_t)(kept && i < n) << (j - j0);
        });
        if (some) __syncthreads();                              // the counts are used again
        // a hole before `keep`, a fill behind it: holes come before all fills
        const auto moves = [&](int i, int j) { return i < n && ((stays >> (j - j0)) & 1) == (uint64_t)(i >= a.keep); };
        for (int j = j0; j < j1; j++) {
            const uint64_t m = __ballot(moves(j * kSelectThreads + tid, j));
            if (lane == 0) count[(j - j0) * kSelectWaves + wave] = (uint32_t)__popcll(m);
        }
        if (tid >= (j1 - j0) * kSelectWaves && tid < kBatch * kSelectWaves) count[tid] = 0;
        before_each(ranks);
        ranks += all;
        walk(j0, j1, [&](int j, int i, uint32_t) {
            const bool move = moves(i, j);
            const uint64_t m = __ballot(move);
            if (move) {
                list[count[(j - j0) * kSelectWaves + wave] + (uint32_t)__popcll(m & below)] = i;
            } else if (i < a.keep) {
                new_sums[i] = KPT ? sum[KPT ? j : 0] : sums[i];
                new_pos[i] = KPT ? at[KPT ? j : 0] : pos[i];
            }
        });
        __syncthreads();
    }
    const uint32_t holes = ranks / 2;
    for (uint32_t r = tid; r < holes; r += kSelectThreads) {
        const int place = list[r], src = list[holes + r];
        new_sums[place] = sums[src];
        new_pos[place] = pos[src];
    }
    if constexpr (W > 0) move_pieces<W, BITS>(a, row, holes, tid, kSelectThreads, per_row);
    else if (tid == 0) a.count[row] = (int32_t)holes;
}

template <int W, int BITS>
__global__ __launch_bounds__(256) void paged_move_kernel(EvictArgs a, FastDiv per_row)
{
    move_pieces<W, BITS>(a, blockIdx.y, (uint32_t)a.count[blockIdx.y], blockIdx.x * 256 + threadIdx.x, gridDim.x * 256, per_row);
}

// A workgroup that chooses moves its rows itself where there can be few: up to this many bytes of keys.  (128 heads, rows of 256
// bytes, 16 moves 9.7 us against 11.9 with a second launch, 64 moves 11.7 and 13.3, 256 moves 17.4 and 17.6; 512 heads, 64 moves
// 22.5 and 22.9, 128 moves 33.7 and 31.5.)
constexpr int64_t kMovedBySelect = 16384;
template <int BITS>
constexpr int kNarrow = BITS == 4 ? 4 : BITS / 8;

// `wide`: rows in pieces of 16 bytes, else element by element (4 bits: word by word)
template <int KPT, int BITS>
void launch_select(const EvictArgs &a, unsigned rows, bool here, bool wide, const FastDiv &per_row, hipStream_t s)
{
    const dim3 grid(rows), block(kSelectThreads);
    if (!here) hipLaunchKernelGGL((paged_select_kernel<KPT, 0, 16>), grid, block, 0, s, a, per_row);
    else if (wide) hipLaunchKernelGGL((paged_select_kernel<KPT, 16, BITS>), grid, block, 0, s, a, per_row);
    else hipLaunchKernelGGL((paged_select_kernel<KPT, kNarrow<BITS>, BITS>), grid, block, 0, s, a, per_row);
}
// Rounds in steps of 2^k + 1: budgets are powers of two as a rule, and a cache that is kept at one has a block or two more.  A
// round too many costs 0.2 to 0.6 us (one token over 8192: 11.9 us in 9 rounds, 15.1 in 16, 24 where nothing is held).
template <int BITS>
void launch_select(const EvictArgs &a, unsigned rows, bool here, bool wide, const FastDiv &per_row, hipStream_t s)
{
    if (a.capacity <= 2 * kSelectThreads) launch_select<2, BITS>(a, rows, here, wide, per_row, s);
    else if (a.capacity <= 3 * kSelectThreads) launch_select<3, BITS>(a, rows, here, wide, per_row, s);
    else if (a.capacity <= 5 * kSelectThreads) launch_select<5, BITS>(a, rows, here, wide, per_row, s);
    else if (a.capacity <= 9 * kSelectThreads) launch_select<9, BITS>(a, rows, here, wide, per_row, s);
    else if (a.capacity <= 17 * kSelectThreads) launch_select<17, BITS>(a, rows, here, wide, per_row, s);
    else if (a.capacity <= 33 * kSelectThreads) launch_select<33, BITS>(a, rows, here, wide, per_row, s);
    else launch_select<0, BITS>(a, rows, here, wide, per_row, s);
}
template <int BITS>
void launch_evict(const EvictArgs &a, unsigned rows, bool here, bool wide, const FastDiv &per_row, hipStream_t s)
{
    launch_select<BITS>(a, rows, here, wide, per_row, s);
    if (here) return;
    const int64_t chunks = (a.most * per_row.d + 255) / 256;
    const dim3 grid((unsigned)(chunks < 64 ? chunks : 64), rows);
    if (wide) hipLaunchKernelGGL((paged_move_kernel<16, BITS>), grid, dim3(256), 0, s, a, per_row);
    else hipLaunchKernelGGL((paged_move_kernel<kNarrow<BITS>, BITS>), grid, dim3(256), 0, s, a, per_row);
}

// moves of one row at most
int64_t most_moves(int64_t capacity, int64_t keep) { return capacity > keep ? (keep < capacity - keep ? keep : capacity - keep) : 0; }

size_t evict_bytes(int64_t rows, int64_t most) { return (size_t)((rows * 4 + 255) / 256 * 256) + (size_t)rows * 2 * (size_t)most * 4; }

} // namespace
} // namespace mi355

extern "C" size_t mi355_paged_cache_evict_workspace(int64_t batch, int64_t kv_heads, int64_t max_blocks, int64_t block_size, int64_t keep)
{
    if (batch < 1 || kv_heads < 1 || max_blocks < 0 || block_size < 1 || keep < 0 || max_blocks > 0x7fffff00 / block_size) return 0;
    return mi355::evict_bytes(batch * kv_heads, mi355::most_moves(max_blocks * block_size, keep));
}

extern "C" int mi355_paged_cache_evict(const mi355_paged_cache *cache, const int32_t *block_table, int64_t table_stride, int64_t max_blocks,
                                       const int32_t *context_lens, int64_t batch, const float *sums, int64_t sums_stride_batch,
                                       int64_t sums_stride_head, const int32_t *positions, int64_t positions_stride_batch,
                                       int64_t positions_stride_head, int64_t keep, int64_t recent, int32_t *new_lens, float *new_sums,
                                       int32_t *new_positions, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace mi355;
    EvictArgs a;
    if (const int st = open_cache(cache, &a.cache); st != MI355_OK) return st;
    if (batch < 0 || max_blocks < 0 || keep < 0 || recent < 0 || recent > keep) return MI355_ERR_BAD_ARGUMENT;
    if (batch == 0) return MI355_OK;
    if (max_blocks > 0x7fffff00 / cache->block_size || batch > 0x7fffffff / cache->kv_heads) return MI355_ERR_UNSUPPORTED;
    if (!context_lens || !new_lens || (max_blocks > 0 && (!block_table || !sums || !positions || !new_sums || !new_positions))) return MI355_ERR_BAD_ARGUMENT;
    const int64_t capacity = max_blocks * cache->block_size, rows = batch * cache->kv_heads;
    a.most = most_moves(capacity, keep);
    if (a.most > 0x7fffffff / (cache->head_dim * 4)) return MI355_ERR_UNSUPPORTED;       // pieces of a row's moves are counted in 31 bits
    if (!workspace || workspace_bytes < evict_bytes(rows, a.most)) return MI355_ERR_WORKSPACE;
    const void *const words[] = {workspace, block_table, context_lens, sums, positions, new_lens, new_sums, new_positions};
    for (const void *p : words)
        if (!aligned(p, p == workspace ? 16 : 4)) return MI355_ERR_ALIGNMENT;
    a.table = block_table;
    a.table_stride = table_stride;
    a.lens = context_lens;
    a.sums = sums;
    a.sums_batch = sums_stride_batch;
    a.sums_head = sums_stride_head;
    a.positions = positions;
    a.positions_batch = positions_stride_batch;
    a.positions_head = positions_stride_head;
    a.new_lens = new_lens;
    a.new_sums = new_sums;
    a.new_positions = new_positions;
    a.capacity = (int)capacity;
    a.keep = (int)(keep < capacity ? keep : capacity);
    a.recent = recent;
    a.count = static_cast<int32_t *>(workspace);
    a.moves = reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + (rows * 4 + 255) / 256 * 256);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int bits = cache_bits(cache->dtype), elem = cache_elem_bytes(cache->dtype), bytes = (int)(cache->head_dim * bits / 8);
    const bool wide = bytes % 16 == 0 && rows_aligned(a.cache.key, 16) && rows_aligned(a.cache.value, 16);
    const FastDiv per_row = fast_div((uint32_t)(bytes / (wide ? 16 : elem)) * 2);
    const bool here = a.most * bytes <= kMovedBySelect;
    // Rows are a grid's second dimension (16 bits) for the moves, and 1024 threads each (32 bits in all; beyond, a grid wraps
    // without an error) for the choice: more of them go sequence by sequence into several launches.
    const int64_t sequences = (here ? (int64_t)1 << 21 : 65535) / cache->kv_heads;
    for (int64_t b0 = 0; b0 < batch; b0 += sequences) {
        const int64_t n = (batch - b0 < sequences ? batch - b0 : sequences) * cache->kv_heads, r0 = b0 * cache->kv_heads;
        EvictArgs c = a;
        c.table += b0 * table_stride;
        c.lens += b0;
        c.sums += b0 * sums_stride_batch;
        c.positions += b0 * positions_stride_batch;
        c.new_lens += b0;
        c.new_sums += r0 * capacity;
        c.new_positions += r0 * capacity;
        c.count += r0;
        c.moves += r0 * 2 * a.most;
        if (bits == 16) launch_evict<16>(c, (unsigned)n, here, wide, per_row, s);
        else if (bits == 8) launch_evict<8>(c, (unsigned)n, here, wide, per_row, s);
        else launch_evict<4>(c, (unsigned)n, here, wide, per_row, s);
    }
    return check_launch();
}
