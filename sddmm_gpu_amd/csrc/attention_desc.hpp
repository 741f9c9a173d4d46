// Descriptions of attention calls on the host: what all entry points check of them, and the kernels' arguments that follow from them.
#pragma once
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include "attention.hpp"
#include "internal.hpp"

namespace sddmm {

constexpr int64_t kMostRows = INT32_MAX;

inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

inline int element(int type) { return type == SDDMM_TYPE_F32 ? 4 : 2; }

inline bool strides_fit(const sddmm_attention_desc &d, int64_t seq, int64_t row, int64_t head, bool packed)
{
    const int64_t e = element(d.type), piece = 16 / e;
    return row >= d.head_dim && row < ((int64_t)1 << 23) / e && row % piece == 0 && head % piece == 0 && (packed || seq % piece == 0) &&
           head >= 0 && (packed || seq >= 0);
}

// Whether no two rows of an array that is written lie in each other's place (broadcast operands have strides of 0).
inline bool apart(const sddmm_attention_desc &d, int64_t seq, int64_t row, int64_t head, int64_t n_seq, int64_t n_rows, int64_t n_heads)
{
    std::pair<int64_t, int64_t> dims[3] = {{row, n_rows}, {head, n_heads}, {seq, n_seq}};
    if (n_seq == 0 || n_rows == 0) return true;
    std::sort(dims, dims + 3);
    int64_t extent = d.head_dim;
    for (const auto &[stride, n] : dims) {
        if (n <= 1) continue;
        if (stride < extent) return false;
        extent += (n - 1) * stride;
    }
    return true;
}

inline int check_desc(const char *who, const sddmm_attention_desc *p)
{
    if (!p) return fail(SDDMM_ERR_ARG, "%s: NULL description", who);
    const sddmm_attention_desc &d = *p;
    if (d.type != SDDMM_TYPE_F32 && d.type != SDDMM_TYPE_BF16 && d.type != SDDMM_TYPE_F16) return fail(SDDMM_ERR_ARG, "%s: unknown type %d", who, d.type);
    if (d.head_dim < 8 || d.head_dim > 128 || d.head_dim % 8)
        return fail(SDDMM_ERR_ARG, "%s: head_dim = %d is no multiple of 8 up to 128", who, d.head_dim);
    if (d.n_heads < 1 || d.n_kv_heads < 1 || d.n_heads % d.n_kv_heads || d.n_heads > 65536)
        return fail(SDDMM_ERR_ARG, "%s: %d query heads do not share %d key heads", who, d.n_heads, d.n_kv_heads);
    if (d.n_seq < 0 || d.max_q < 0 || d.max_k < 0 || d.shared_len < 0 || d.q_rows < 0 || d.k_rows < 0) return fail(SDDMM_ERR_ARG, "%s: negative size", who);
    if (d.window_left < -1 || d.window_right < -1) return fail(SDDMM_ERR_ARG, "%s: a window below -1", who);
    if (!std::isfinite(d.scale) || !(d.scale > 0.f)) return fail(SDDMM_ERR_ARG, "%s: scale must be finite and above 0", who);
    if (!std::isfinite(d.cap) || d.cap < 0.f) return fail(SDDMM_ERR_ARG, "%s: cap must be finite and not negative", who);
    if (d.cap > 0.f && !(d.scale / d.cap > 1e-15f && d.scale / d.cap < 1e15f && d.cap < 1e30f)) return fail(SDDMM_ERR_ARG, "%s: cap and scale are too far apart", who);
    if ((d.q_ptr && d.q_len) || (d.k_ptr && d.k_len)) return fail(SDDMM_ERR_ARG, "%s: lengths beside the pointers of packed sequences", who);
    if (!strides_fit(d, d.q_seq, d.q_row, d.q_head, d.q_ptr) || !strides_fit(d, d.k_seq, d.k_row, d.k_head, d.k_ptr) ||
        !strides_fit(d, d.v_seq, d.v_row, d.v_head, d.k_ptr) || !strides_fit(d, d.o_seq, d.o_row, d.o_head, d.q_ptr))
        return fail(SDDMM_ERR_ARG, "%s: strides must be multiples of 16 bytes, a row's from head_dim to 2^23 bytes", who);
    for (const void *p : {(const void *)d.q_ptr, (const void *)d.k_ptr, (const void *)d.q_len, (const void *)d.k_len, (const void *)d.prefix, (const void *)d.slopes})
        if ((uintptr_t)p & 3u) return fail(SDDMM_ERR_ARG, "%s: arrays of the description must be aligned to their elements", who);
    const int64_t rows = d.q_ptr ? d.q_rows : (int64_t)d.n_seq * d.max_q;
    if (rows > kMostRows || d.k_rows > kMostRows || (int64_t)d.shared_len + d.max_k > kMostRows / 2 || d.max_q > kMostRows / 2)
        return fail(SDDMM_ERR_RANGE, "%s: sizes beyond 32-bit positions", who);
    return SDDMM_OK;
}

// The description with the bounds that packed arrays give: no sequence has more rows or keys than all of them.  Tiles of a sequence then are at most those of the
// grid, and fit 32 bits as it does, whatever bound the caller names.
inline sddmm_attention_desc held(sddmm_attention_desc d)
{
    if (d.q_ptr) d.max_q = (int32_t)std::min<int64_t>(d.max_q, d.q_rows);
    if (d.k_ptr) d.max_k = (int32_t)std::min<int64_t>(d.max_k, d.k_rows);
    return d;
}

// Rows and keys of all sequences (0 where none can have any, whatever the arrays hold).
inline int64_t rows_of(const sddmm_attention_desc &d) { return d.n_seq == 0 || d.max_q == 0 ? 0 : d.q_ptr ? d.q_rows : (int64_t)d.n_seq * d.max_q; }
inline int64_t key_rows_of(const sddmm_attention_desc &d) { return d.n_seq == 0 || d.max_k == 0 ? 0 : d.k_ptr ? d.k_rows : (int64_t)d.n_seq * d.max_k; }

inline AttnArgs arguments(const sddmm_attention_desc &d)
{
    AttnArgs a{};
    a.q_seq = d.q_seq, a.q_row = d.q_row, a.q_head = d.q_head, a.k_seq = d.k_seq, a.k_row = d.k_row, a.k_head = d.k_head;
    a.v_seq = d.v_seq, a.v_row = d.v_row, a.v_head = d.v_head, a.o_seq = d.o_seq, a.o_row = d.o_row, a.o_head = d.o_head;
    a.q_ptr = d.q_ptr, a.k_ptr = d.k_ptr, a.q_len = d.q_len, a.k_len = d.k_len, a.prefix = d.prefix, a.slopes = d.slopes;
    a.rows = rows_of(d), a.key_rows = key_rows_of(d);
    a.head_dim = d.head_dim, a.n_heads = d.n_heads, a.n_kv_heads = d.n_kv_heads, a.group = d.n_heads / d.n_kv_heads;
    a.n_seq = d.n_seq, a.max_q = d.max_q, a.max_k = d.max_k, a.left = std::min(d.window_left, 1 << 30), a.right = std::min(d.window_right, 1 << 30),  // (positions are below)
    a.shared_len = d.shared_len;
    a.scale = d.scale, a.cap = d.cap;
    return a;
}

inline bool aligned(std::initializer_list<const void *> pointers)
{
    for (const void *p : pointers)
        if ((uintptr_t)p & 15u) return false;
    return true;
}

// Whether a result begins where an operand does (workgroups that are still to come read operands).
inline bool in_place_of(std::initializer_list<const void *> results, std::initializer_list<const void *> operands)
{
    for (const void *r : results)
        for (const void *o : operands)
            if (r && r == o) return true;
    return false;
}

}  // namespace sddmm
