// A cache of keys and values in pages: as the kernels see it, and what both entry points check of its description.
#pragma once
#include <hip/hip_runtime.h>
#include <cmath>
#include "attention.hpp"
#include "attention_desc.hpp"

namespace sddmm {

enum { kHeldOwn = 0, kHeldI8 = 1, kHeldE4m3 = 2 };  // in the operands' type, or in codes

// (strides in bytes)
struct CacheArgs {
    char *k, *v;
    float *k_scale, *v_scale;
    const int32_t *table;
    int64_t k_head, v_head, table_row;
    uint32_t k_page, k_row, v_page, v_row;
    int32_t n_pages, page_shift, block_shift, n_kv_heads;

    // row `at` of a page of one head (a page's rows lie within 2^32 bytes)
    __device__ __forceinline__ char *k_at(int page, int kv, int at) const { return k + kv * k_head + ((uint64_t)(uint32_t)page * k_page + (uint32_t)at * k_row); }
    __device__ __forceinline__ char *v_at(int page, int kv, int at) const { return v + kv * v_head + ((uint64_t)(uint32_t)page * v_page + (uint32_t)at * v_row); }

    // the entry at `i` of sequence s, held to the pages that exist
    __device__ __forceinline__ int page(int s, int i) const { return min(max(table[s * table_row + i], 0), n_pages - 1); }
    // the scale of the token `at` of a page, in k_scale or v_scale
    __device__ __forceinline__ int64_t scale_at(int page, int kv, int at) const
    {
        return (((int64_t)page * n_kv_heads + kv) << (page_shift - block_shift)) + (at >> block_shift);
    }
};

inline int held_as(const sddmm_attention_desc &d, const sddmm_cache_desc &c) { return c.type == SDDMM_TYPE_I8 ? kHeldI8 : c.type == SDDMM_TYPE_E4M3 ? kHeldE4m3 : kHeldOwn; }
inline int log2_of(int64_t x) { return 63 - __builtin_clzll((uint64_t)x); }

// `d` has been checked.
inline int check_cache(const char *who, const sddmm_attention_desc &d, const sddmm_cache_desc *p)
{
    if (!p) return fail(SDDMM_ERR_ARG, "%s: NULL description of the cache", who);
    const sddmm_cache_desc &c = *p;
    if (c.type != d.type && c.type != SDDMM_TYPE_I8 && c.type != SDDMM_TYPE_E4M3) return fail(SDDMM_ERR_ARG, "%s: a cache of type %d for operands of type %d", who, c.type, d.type);
    auto power = [](int64_t x) { return x > 0 && (x & (x - 1)) == 0; };
    if (!power(c.page_len) || c.page_len < 16 || c.page_len > 65536) return fail(SDDMM_ERR_ARG, "%s: page_len = %d is no power of two from 16 to 65536", who, c.page_len);
    const bool codes = c.type != d.type;
    if (codes && (!power(c.block_len) || c.block_len > 64 || c.block_len > c.page_len))
        return fail(SDDMM_ERR_ARG, "%s: block_len = %d is no power of two up to 64 and page_len", who, c.block_len);
    if (d.shared_len || d.k_ptr) return fail(SDDMM_ERR_ARG, "%s: a cache in pages goes without shared_len and k_ptr", who);
    if (c.n_pages < 0 || c.n_pages > INT32_MAX) return fail(SDDMM_ERR_RANGE, "%s: n_pages must be 0 .. 2^31 - 1", who);
    const int64_t e = codes ? 1 : element(d.type), piece = 16 / e;
    for (int64_t row : {c.k_row, c.v_row})
        if (row < d.head_dim || row >= ((int64_t)1 << 23) / e || row % piece) return fail(SDDMM_ERR_ARG, "%s: rows of the cache must be multiples of 16 bytes apart, from head_dim to 2^23 bytes", who);
    for (int64_t s : {c.k_page, c.v_page, c.k_head, c.v_head})
        if (s < 0 || s > ((int64_t)1 << 40) || s % piece) return fail(SDDMM_ERR_ARG, "%s: strides of pages and heads must be multiples of 16 bytes", who);
    for (int64_t bytes : {c.k_page * e, c.v_page * e, c.k_row * e * c.page_len, c.v_row * e * c.page_len})
        if (bytes > UINT32_MAX) return fail(SDDMM_ERR_RANGE, "%s: pages 2^32 bytes apart, or rows of a page", who);
    if (c.table_row < div_up(d.max_k, c.page_len)) return fail(SDDMM_ERR_ARG, "%s: table_row = %lld is less than the pages of max_k tokens", who, (long long)c.table_row);
    if (!aligned({c.k, c.v})) return fail(SDDMM_ERR_ARG, "%s: pointers must be 16-byte aligned", who);
    if (((uintptr_t)c.k_scale | (uintptr_t)c.v_scale | (uintptr_t)c.table) & 3u) return fail(SDDMM_ERR_ARG, "%s: arrays of the description must be aligned to their elements", who);
    if (d.n_seq > 0 && d.max_k > 0 && c.n_pages > 0 && (!c.k || !c.v || !c.table || (codes && (!c.k_scale || !c.v_scale)))) return fail(SDDMM_ERR_ARG, "%s: NULL device pointer", who);
    return SDDMM_OK;
}

inline CacheArgs cache_arguments(const sddmm_attention_desc &d, const sddmm_cache_desc &c)
{
    const int64_t e = c.type == d.type ? element(d.type) : 1;
    CacheArgs a{};
    a.k = (char *)c.k, a.v = (char *)c.v, a.k_scale = c.k_scale, a.v_scale = c.v_scale, a.table = c.table;
    a.k_page = (uint32_t)(c.k_page * e), a.k_row = (uint32_t)(c.k_row * e), a.k_head = c.k_head * e, a.v_page = (uint32_t)(c.v_page * e), a.v_row = (uint32_t)(c.v_row * e), a.v_head = c.v_head * e;
    a.table_row = c.table_row;
    a.n_pages = (int32_t)c.n_pages, a.page_shift = log2_of(c.page_len), a.block_shift = c.type == d.type ? 0 : log2_of(c.block_len), a.n_kv_heads = d.n_kv_heads;
    return a;
}

}  // namespace sddmm
