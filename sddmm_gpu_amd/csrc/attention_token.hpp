// Dense attention for few rows (gfx950): the newest tokens of every sequence against a long cache.
#pragma once
#include "attention.hpp"
#include "attention_launch.hpp"

namespace sddmm {

// The (token, head) pairs that share a key head are the rows: one tile of 32 reads every key once.  Each wave works on keys of
// its own, every NW-th tile of 32 of the workgroup's piece, in LDS of its own and without a barrier, with statistics and sums of
// its own, which are joined at the end.  What bounds it is the rate at which the caches are read, so a wave always has half a tile
// under way: the next keys are requested when the scores are done, the next values when the products are (each 32 rows' worth: 8 KB at
// 128 bf16 elements, 32 to 64 KB a compute unit with one or two workgroups of four waves).  Most rows of the tile are empty where few heads share the
// keys; the matrix instructions are below a tenth of the time all the same.  P is rounded as in the kernel of whole tiles.
// 64 users of 284 to 8192 keys, 32 heads over 8 of 128, bf16: 205 us = 5.2 TB/s, a large copy's rate; one user, 1501 keys: 8.5 us for the chain of
// loads, and 4 to join 6 pieces.
template <class T, int DP, bool MOD, int NW>
struct TokenTile {
    static constexpr int KT = 32;
    typedef Tile<T, DP, KT> Keys;
    static constexpr int kLds = NW * 2 * Keys::kBytes;
    static __device__ __forceinline__ void run(const AttnArgs &a, int b, char (&memory)[kLds]);
};

template <class T, int DP, bool MOD, int NW>
__device__ __forceinline__ void TokenTile<T, DP, MOD, NW>::run(const AttnArgs &a, int b, char (&memory)[kLds])
{
    constexpr int DB = DP / 32;
    typedef typename Elem<T>::Vec8 Vec8;
    constexpr int kLoads = Keys::kBytes / 1024;
    auto &lds = *(char (*)[NW][2][Keys::kBytes])memory;
    __shared__ float2 ml[NW][32];
    static_assert(2 * Keys::kBytes >= 128 * DP);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
    const int kv = b % a.n_kv_heads;
    b /= a.n_kv_heads;
    const int split = b % a.n_split;
    b /= a.n_split;
    int s, tile;
    if (a.q_ptr && a.max_tiles > 1) {
        s = slot_sequence<false>(a.q_ptr, a.n_seq, a.group, kTokenRows, a.max_tiles, a.n_slots, b, tile);
        if (s < 0) return;
    } else {
        s = b % a.n_seq, tile = a.max_tiles - 1 - b / a.n_seq;
    }
    const Seq e = sequence(a, s);
    const int n_rows = e.nq * a.group, n_keys = e.nk;
    if (tile * kTokenRows >= n_rows) return;
    const int row = tile * kTokenRows + n;
    const bool there = row < n_rows;
    const int token = row / a.group, head = kv * a.group + row % a.group;
    const int shift = e.nk - e.nq, prefix = a.prefix ? max(a.prefix[s], a.shared_len) - a.shared_len : 0, pos = token + shift;
    const int lo = first_key(a, pos), hi = end_key(a, pos, prefix, n_keys);
    const int t0 = tile * kTokenRows / a.group, t1 = (min(n_rows, tile * kTokenRows + kTokenRows) - 1) / a.group;
    const int any_lo = first_key(a, t0 + shift), any_hi = end_key(a, t1 + shift, prefix, n_keys);
    const int full_lo = first_key(a, t1 + shift), full_hi = end_key(a, t0 + shift, prefix, n_keys);

    floatx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = zero16();
    const float scale = a.scale;
    Bend<T> bend;
    if constexpr (MOD) bend.init(scale, a.cap);
    const float unit = MOD ? 1.f : scale * kLog2e;
    const float slope = MOD && a.slopes && there ? a.slopes[head] * kLog2e : 0.f;
    float m = -INFINITY, sum = 0.f;

    const T *k = k_base<T>(a, a.k, e, s, kv), *v = v_base<T>(a, a.v, e, s, kv);
    const int n_tiles = any_hi > any_lo ? (any_hi - any_lo + KT - 1) / KT : 0;
    const int each = (n_tiles + a.n_split - 1) / a.n_split;
    const int first = split * each, last = min(n_tiles, first + each);
    const int row_bytes = a.head_dim * (int)sizeof(T);
    const uint32_t k_stride = (uint32_t)(a.k_row * sizeof(T)), v_stride = (uint32_t)(a.v_row * sizeof(T));
    char *kt = lds[wave][0], *vt = lds[wave][1];
    // (behind the last tile nothing is read, but the requests are made, so that the waits count the same)
    auto request = [&](char *to, const T *base, int64_t step, uint32_t stride, int t) {
        const int key = any_lo + t * KT;
        const bool more = t < last;
        Keys::template request<1>(to, (const char *)(base + (more ? key : 0) * step), stride, more ? n_keys - key : 0, row_bytes, 0, lane);
    };
    int t = first + wave;
    request(kt, k, a.k_row, k_stride, t);
    request(vt, v, a.v_row, v_stride, t);
    const T *q = q_base<T>(a, a.q, e, s, head) + (int64_t)token * a.q_row;
    Vec8 qf[DP / 16];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) qf[c] = global_operand<T>(q, there, 16 * c + 8 * h, a.head_dim);
    __builtin_amdgcn_s_waitcnt(0x0f70);  // the first tile and q: from here on only tiles are under way
    for (; t < last; t += NW) {
        const int key = any_lo + t * KT;
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
        floatx16 x = zero16();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) x = Elem<T>::mma(Keys::row_operand(kt, 0, c, lane), qf[c], x);
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(x) :: "memory");  // (all of the keys have been read)
        request(kt, k, a.k_row, k_stride, t + NW);

        if constexpr (MOD) {
            if (bend.cap > 0.f) {
                floatx16 y[1] = {x};
                bend.template apply<1, false>(y, y);
                x = y[0];
            } else {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] *= scale * kLog2e;
            }
            if (a.slopes) {
                const float at = (float)(pos - key - 4 * h);
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = fmaf(-slope, fabsf(at - (float)(8 * (r >> 2) + (r & 3))), x[r]);
            }
        }
        if (key < full_lo || key + KT > full_hi) {
            const int at = key + 4 * h - lo;
            const uint32_t span = there && hi > lo ? hi - lo : 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = (uint32_t)(at + 8 * (r >> 2) + (r & 3)) < span ? x[r] : -INFINITY;
        }
        float top = x[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, x[r]);
        const float raised = fmaxf(m, halves_max(top));
        if (__any(raised > m)) {
            const float by = raised == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - raised) * unit);
            m = raised;
            sum *= by;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= by;
        }
        const float base = m == -INFINITY ? 0.f : m * unit;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], unit, -base));
            sum += x[r];
        }
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const Vec8 p = operand<T>(x, c);
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = Elem<T>::mma(Keys::column_operand(vt, d, c, lane), p, o[d]);
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(o[d]) :: "memory");
        request(vt, v, a.v_row, v_stride, t + NW);
    }
    sum = halves_sum(sum);
    m = m == -INFINITY ? m : m * unit;

    // join the waves: [element of the lane / 4][lane] of 16 bytes for each wave
    __builtin_amdgcn_s_waitcnt(0x0070);
    floatx4 *mine = (floatx4 *)lds[wave][0];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[(4 * d + i) * 64 + lane] = floatx4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    if (h == 0) ml[wave][n] = make_float2(m, sum);
    __syncthreads();
    if (!there) return;
    float top = -INFINITY, total = 0.f, w[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) top = fmaxf(top, ml[i][n].x);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        w[i] = ml[i][n].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[i][n].x - top);
        total = fmaf(w[i], ml[i][n].y, total);
    }
    const bool parts = a.n_part > 1;
    const int64_t at = (e.lse0 + token) * a.n_heads + head, all = a.rows * a.n_heads, part = a.part0 + split;
    const float by = parts ? 1.f : total > 0.f || total != total ? 1.f / total : 0.f;
    T *to = (T *)o_base<T>(a, a.out, e, s, head) + (int64_t)token * a.o_row;
    float *to_part = a.part_o + (part * all + at) * a.head_dim;
#pragma unroll
    for (int j = 0; j < 4 * DB / NW; ++j) {
        const int piece = wave * (4 * DB / NW) + j, col = 8 * piece + 4 * h;
        floatx4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) y += ((const floatx4 *)lds[i][0])[piece * 64 + lane] * w[i];
        y *= by;
        if (col >= a.head_dim) continue;
        if (parts) *(floatx4 *)(to_part + col) = y;
        else *(typename Elem<T>::Vec4 *)(to + col) = __builtin_convertvector(y, typename Elem<T>::Vec4);
    }
    if (wave == 0 && h == 0) {
        if (parts) a.part_ml[part * all + at] = make_float2(top, total);
        else if (a.lse) a.lse[at] = (top + __builtin_amdgcn_logf(total)) * kLn2;
    }
}

}  // namespace sddmm
