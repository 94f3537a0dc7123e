// Addressing of the paged key-value cache (mi355_paged_cache): shared by the kernels that write, read, attend to and evict
// from it.
#pragma once
#include "common.h"

namespace mi355 {

// n / d for 0 <= n < 2^31 and a divisor known to the host: with l = ceil(log2 d) and m = ceil(2^(31 + l) / d), which is below
// 2^32, (n * m) >> (31 + l) is the quotient (the error n * (m d - 2^(31 + l)) / (d 2^(31 + l)) stays below 1 / d).
struct FastDiv {
    uint32_t d = 1, mul = 0x80000000u, shift = 31;
};
inline FastDiv fast_div(uint32_t d)
{
    FastDiv f;
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) l++;
    f.d = d;
    f.shift = 31 + l;
    f.mul = (uint32_t)((((uint64_t)1 << f.shift) + d - 1) / d);
    return f;
}
__host__ __device__ inline uint32_t div_by(uint32_t n, const FastDiv &f) { return (uint32_t)(((uint64_t)n * f.mul) >> f.shift); }

// One of the four arrays of a cache; strides in bytes.
struct PagedArray {
    char *base;
    int64_t block, token, head;
};
struct PagedCache {
    PagedArray key, value, key_scale, value_scale;
    FastDiv page;
    int num_blocks, heads, dim;
    int slots;                      // num_blocks * block_size

    __device__ __forceinline__ int64_t offset(const PagedArray &a, uint32_t slot, int head) const
    {
        const uint32_t block = div_by(slot, page);
        return block * a.block + (int64_t)(slot - block * page.d) * a.token + head * a.head;
    }
};

inline int cache_elem_bytes(int dtype) { return dtype == MI355_DTYPE_INT8 ? 1 : 2; }

// Checks a descriptor and translates it; MI355_OK or the status to return.
inline int open_cache(const mi355_paged_cache *c, PagedCache *out)
{
    if (!c || !c->key || !c->value || c->num_blocks < 1 || c->block_size < 1 || c->kv_heads < 1 || c->head_dim < 1) return MI355_ERR_BAD_ARGUMENT;
    const bool quantised = c->dtype == MI355_DTYPE_INT8;
    if (!quantised && c->dtype != MI355_DTYPE_BF16 && c->dtype != MI355_DTYPE_FP16) return MI355_ERR_BAD_ARGUMENT;
    if (quantised != (c->key_scale != nullptr) || quantised != (c->value_scale != nullptr)) return MI355_ERR_BAD_ARGUMENT;
    constexpr int64_t kMost = 0x7fffffff;                  // slots are numbered in 31 bits; byte offsets have 64
    if (c->block_size > kMost || c->num_blocks > kMost / c->block_size || c->kv_heads > 65535 || c->head_dim > 65536) return MI355_ERR_UNSUPPORTED;
    const int size = cache_elem_bytes(c->dtype);
    if (!aligned(c->key, size) || !aligned(c->value, size) || (quantised && (!aligned(c->key_scale, 4) || !aligned(c->value_scale, 4))))
        return MI355_ERR_ALIGNMENT;
    const auto array = [](void *p, const int64_t *stride, int64_t bytes) {
        return PagedArray{static_cast<char *>(p), p ? stride[0] * bytes : 0, p ? stride[1] * bytes : 0, p ? stride[2] * bytes : 0};
    };
    out->key = array(c->key, c->key_stride, size);
    out->value = array(c->value, c->value_stride, size);
    out->key_scale = array(c->key_scale, c->key_scale_stride, 4);
    out->value_scale = array(c->value_scale, c->value_scale_stride, 4);
    out->page = fast_div((uint32_t)c->block_size);
    out->num_blocks = (int)c->num_blocks;
    out->heads = (int)c->kv_heads;
    out->dim = (int)c->head_dim;
    out->slots = (int)(c->num_blocks * c->block_size);
    return MI355_OK;
}

// Whether every row of the array starts on a multiple of `a` bytes.
inline bool rows_aligned(const PagedArray &x, int64_t a)
{
    return aligned(x.base, (size_t)a) && x.block % a == 0 && x.token % a == 0 && x.head % a == 0;
}

// Inclusive scans over the lanes of a wavefront: shifts within rows of 16 lanes, then the rows' last lanes handed on.  What a
// lane gets from outside its row is the identity 0.
struct Add {
    __device__ uint32_t operator()(uint32_t x, uint32_t y) const { return x + y; }
};
struct Max {
    __device__ uint32_t operator()(uint32_t x, uint32_t y) const { return max(x, y); }
};
template <int CTRL, int ROWS, class Op>
__device__ __forceinline__ uint32_t take(uint32_t v, Op op)
{
    return op(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false));
}
template <class Op>
__device__ __forceinline__ uint32_t scan_row(uint32_t v, Op op)
{
    v = take<0x111, 0xf>(v, op);                 // row_shr:1
    v = take<0x112, 0xf>(v, op);
    v = take<0x114, 0xf>(v, op);
    return take<0x118, 0xf>(v, op);
}
template <class Op>
__device__ __forceinline__ uint32_t scan_lanes(uint32_t v, Op op)
{
    v = take<0x142, 0xa>(scan_row(v, op), op);   // row_bcast:15 into rows 1 and 3
    return take<0x143, 0xc>(v, op);              // row_bcast:31 into rows 2 and 3
}

} // namespace mi355
