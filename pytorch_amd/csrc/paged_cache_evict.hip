// npu_paged_cache_evict for gfx950: sequences that outgrew their budget keep the newest tokens and those with the largest
// summed attention weights, each key/value head its own.
//
// Per (sequence, head) with n > keep tokens a token's worth is a 32-bit key that orders like (recent, sum): all ones for the
// recent ones, else the sum's bits with the sign flipped into place, 0 for NaN.  The keep-th largest key is found digit by
// digit (four histograms of 8 bits); among tokens with exactly that key the lowest places stay.  Kept tokens behind place
// `keep` then fill the holes before it, both in ascending order: the fewest rows move, sources and destinations are disjoint,
// so all of them move at once, in place.
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
    int32_t *moves;                              // [batch * heads][2][most]: places to, places from
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

__global__ __launch_bounds__(kSelectThreads) void paged_select_kernel(EvictArgs a)
{
    __shared__ uint32_t hist[256];
    __shared__ uint32_t found[2];
    __shared__ int wave_top[kSelectWaves];
    __shared__ uint32_t wave_count[3][kSelectWaves];

    const int row = blockIdx.x, b = row / a.cache.heads, head = row % a.cache.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = min(max(a.lens[b], 0), a.capacity);
    const float *sums = a.sums + b * a.sums_batch + head * a.sums_head;
    const int32_t *pos = a.positions + b * a.positions_batch + head * a.positions_head;
    float *new_sums = a.new_sums + (int64_t)row * a.capacity;
    int32_t *new_pos = a.new_positions + (int64_t)row * a.capacity;
    const int stay = min(n, a.keep);
    if (head == 0 && tid == 0) a.new_lens[b] = stay;
    for (int i = stay + tid; i < a.capacity; i += kSelectThreads) new_sums[i] = 0.0f, new_pos[i] = -1;
    if (n <= a.keep || a.keep == 0) {
        for (int i = tid; i < stay; i += kSelectThreads) new_sums[i] = sums[i], new_pos[i] = pos[i];
        if (tid == 0) a.count[row] = 0;
        return;
    }

    int newest = INT32_MIN;
    for (int i = tid; i < n; i += kSelectThreads) newest = max(newest, pos[i]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) newest = max(newest, __shfl_xor(newest, off, 64));
    if (lane == 0) wave_top[wave] = newest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelectWaves; w++) newest = max(newest, wave_top[w]);
    const int64_t oldest = (int64_t)newest - a.recent;

    uint32_t prefix = 0, left = (uint32_t)a.keep;              // the left-th largest among the keys that start with prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kSelectThreads) {
            const uint32_t key = worth_of(sums[i], pos[i], oldest);
            if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (wave == 0) {                                        // four digits per lane, lane 0 the largest ones
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = hist[255 - (lane * 4 + i)], sum += c[i];
            uint32_t scan = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t o = (uint32_t)__shfl_up((int)scan, off, 64);
                if (lane >= off) scan += o;
            }
            uint32_t before = scan - sum;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (before < left && left <= before + c[i]) {   // one lane, one digit
                    found[0] = 255 - (lane * 4 + i);
                    found[1] = left - before;
                }
                before += c[i];
            }
        }
        __syncthreads();
        prefix |= found[0] << shift;
        left = found[1];
    }

    // in the order of the places: which of the tokens with exactly the last key stay, the holes and what fills them
    int32_t *to = a.moves + (int64_t)row * 2 * a.most, *from = to + a.most;
    uint32_t ties = 0, holes = 0, fills = 0;
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    for (int base = 0; base < n; base += kSelectThreads) {
        const int i = base + tid;
        const uint32_t key = i < n ? worth_of(sums[i], pos[i], oldest) : 0;
        const bool tie = i < n && key == prefix;
        const uint64_t tie_mask = __ballot(tie);
        if (lane == 0) wave_count[0][wave] = (uint32_t)__popcll(tie_mask);
        __syncthreads();
        uint32_t rank = ties + (uint32_t)__popcll(tie_mask & below);
        for (int w = 0; w < kSelectWaves; w++) {
            if (w < wave) rank += wave_count[0][w];
            ties += wave_count[0][w];
        }
        const bool kept = i < n && (key > prefix || (tie && rank < left));
        const bool hole = i < n && i < a.keep && !kept, fill = kept && i >= a.keep;
        const uint64_t hole_mask = __ballot(hole), fill_mask = __ballot(fill);
        if (lane == 0) wave_count[1][wave] = (uint32_t)__popcll(hole_mask), wave_count[2][wave] = (uint32_t)__popcll(fill_mask);
        __syncthreads();
        uint32_t hole_rank = holes + (uint32_t)__popcll(hole_mask & below), fill_rank = fills + (uint32_t)__popcll(fill_mask & below);
        for (int w = 0; w < kSelectWaves; w++) {
            if (w < wave) hole_rank += wave_count[1][w], fill_rank += wave_count[2][w];
            holes += wave_count[1][w];
            fills += wave_count[2][w];
        }
        if (hole) to[hole_rank] = i;
        if (fill) from[fill_rank] = i;
        if (kept && i < a.keep) new_sums[i] = sums[i], new_pos[i] = pos[i];
    }
    __syncthreads();
    for (uint32_t i = tid; i < holes; i += kSelectThreads) {
        new_sums[to[i]] = sums[from[i]];
        new_pos[to[i]] = pos[from[i]];
    }
    if (tid == 0) a.count[row] = (int32_t)holes;
}

// Rows of keys and values, W bytes per access: 16 where every row starts on 16 bytes and has a multiple of them.
template <int W>
__global__ __launch_bounds__(256) void paged_move_kernel(EvictArgs a, int elem, int pieces, FastDiv per_row)
{
    typedef uint32_t word __attribute__((ext_vector_type(W >= 4 ? W / 4 : 1)));
    const int row = blockIdx.y, b = row / a.cache.heads, head = row % a.cache.heads;
    const int count = a.count[row];
    const int32_t *to = a.moves + (int64_t)row * 2 * a.most, *from = to + a.most;
    const int32_t *table = a.table + b * a.table_stride;
    const uint32_t all = (uint32_t)count * (uint32_t)pieces * 2;         // below 2^31: the host checks
    for (uint32_t e = blockIdx.x * 256 + threadIdx.x; e < all; e += gridDim.x * 256) {
        const uint32_t r = div_by(e, per_row), piece = e - r * per_row.d;   // per_row = pieces of keys, then of values
        const uint32_t dst = (uint32_t)to[r], src = (uint32_t)from[r];
        const uint32_t dst_block = div_by(dst, a.cache.page), src_block = div_by(src, a.cache.page);
        const int dst_id = table[dst_block], src_id = table[src_block];
        if ((uint32_t)dst_id >= (uint32_t)a.cache.num_blocks || (uint32_t)src_id >= (uint32_t)a.cache.num_blocks) continue;
        const uint32_t dst_slot = (uint32_t)dst_id * a.cache.page.d + (dst - dst_block * a.cache.page.d);
        const uint32_t src_slot = (uint32_t)src_id * a.cache.page.d + (src - src_block * a.cache.page.d);
        const bool value = piece >= (uint32_t)pieces;
        const PagedArray &x = value ? a.cache.value : a.cache.key;
        const uint32_t at = (value ? piece - pieces : piece) * W;
        char *d = x.base + a.cache.offset(x, dst_slot, head) + at;
        const char *s = x.base + a.cache.offset(x, src_slot, head) + at;
        if constexpr (W >= 4) *reinterpret_cast<word *>(d) = *reinterpret_cast<const word *>(s);
        else if constexpr (W == 2) *reinterpret_cast<uint16_t *>(d) = *reinterpret_cast<const uint16_t *>(s);
        else *d = *s;
        if (elem == 1 && at == 0) {
            const PagedArray &sc = value ? a.cache.value_scale : a.cache.key_scale;
            *reinterpret_cast<float *>(sc.base + a.cache.offset(sc, dst_slot, head)) =
                *reinterpret_cast<const float *>(sc.base + a.cache.offset(sc, src_slot, head));
        }
    }
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
    hipLaunchKernelGGL(paged_select_kernel, dim3((unsigned)rows), dim3(kSelectThreads), 0, s, a);
    if (a.most > 0) {
        const int elem = cache_elem_bytes(cache->dtype), bytes = (int)cache->head_dim * elem;
        const bool wide = bytes % 16 == 0 && rows_aligned(a.cache.key, 16) && rows_aligned(a.cache.value, 16);
        const int width = wide ? 16 : elem, pieces = bytes / width;
        const int64_t most = (a.most * pieces * 2 + 255) / 256;
        const dim3 grid((unsigned)(most < 64 ? most : 64), 1);
        for (int64_t r0 = 0; r0 < rows; r0 += 65535 / cache->kv_heads * cache->kv_heads) {   // a grid's second dimension has 16 bits
            EvictArgs c = a;
            const int64_t n = 65535 / cache->kv_heads * cache->kv_heads;
            c.count += r0;
            c.moves += r0 * 2 * a.most;
            c.table += r0 / cache->kv_heads * table_stride;
            const dim3 g(grid.x, (unsigned)(rows - r0 < n ? rows - r0 : n));
            const FastDiv per_row = fast_div((uint32_t)pieces * 2);
            if (wide) hipLaunchKernelGGL(paged_move_kernel<16>, g, dim3(256), 0, s, c, elem, pieces, per_row);
            else if (elem == 2) hipLaunchKernelGGL(paged_move_kernel<2>, g, dim3(256), 0, s, c, elem, pieces, per_row);
            else hipLaunchKernelGGL(paged_move_kernel<1>, g, dim3(256), 0, s, c, elem, pieces, per_row);
        }
    }
    return check_launch();
}
