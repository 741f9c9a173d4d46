// Dense attention, forward (gfx950): a tile of rows against tiles of keys.
#pragma once
#include "attention.hpp"
#include "attention_launch.hpp"

namespace sddmm {

constexpr int kWaves = 4;  // of a workgroup, 32 rows to each

// o_i = sum_j p_ij v_j / sum_j p_ij with p_ij = exp(s_ij - m_i), in one pass over the keys with a running maximum m_i.  A wave
// holds 32 rows: their q as operands, the sums of o turned (element of the head by row).  Per tile of keys, which the four
// waves share in LDS: S^T = K Q^T, so that a lane holds scores of one row only and the statistics need one exchange between the
// two halves of the wave; the probabilities are the second operand of O^T += V^T P^T as they lie.  The maximum is raised only
// when a row's exceeds it by more than 2^8: the sums stay far inside fp32, and the sums of o are rarely scaled.
// P is rounded to the element type (bf16: half a step is 2^-9 of the step's upper end, as for the output itself), its sum is not: the output is off by
// 0.0020 of its size where rounding it alone makes 0.0016; a second operand for what P loses would be a third product beside two.
//
// What bounds it: matrix and vector instructions about alike, each half of the time on long prompts, with the clock at 1.9 GHz under the power limit.
// 16,384 tokens, causal, 16 heads over 2 of 128, bf16: 1.00 ms = 1.10 PFLOP/s, where a large library product reaches 1.17; 8192 tokens, 16 heads of 128
// 0.29 to 0.33 ms by card (0.95; capped 0.36), of 64, fp16 0.18 ms (0.76); fp32, 4096 tokens, 16 heads of 64 0.29 ms = 118 TFLOP/s of 154.  LDS is read without conflicts.
//
// What the rows of a workgroup are: the rows of one query head (kRowsOfHead); the (token, head) pairs of the query heads that share
// a key head, for few tokens (kRowsPacked); the same pairs of all sequences, against the keys that all of them begin with
// (kRowsShared: each sequence's rows have positions, and so masks, of their own).
//
// RW: waves on rows of their own.  With 2 the others take the second half of every tile of keys for the same 64 rows, and the halves
// are joined at the end: twice the workgroups, where those of 128 rows are so few that the longest keeps the others waiting.
template <class T, int DP, bool MOD, int ROWS, int RW>
struct ForwardTile {
    static constexpr int KT = sizeof(T) == 2 || RW == 2 ? 64 : 32;
    typedef Tile<T, DP, KT> Keys;
    static constexpr int kLds = 4 * Keys::kBytes;
    static __device__ __forceinline__ void run(const AttnArgs &a, int b, char (&memory)[kLds]);
};

template <class T, int DP, bool MOD, int ROWS, int RW>
__device__ __forceinline__ void ForwardTile<T, DP, MOD, ROWS, RW>::run(const AttnArgs &a, int b, char (&memory)[kLds])
{
    constexpr int KB = KT / 32 / (kWaves / RW), DB = DP / 32, kRows = 32 * RW;
    // A wave that is at its softmax goes before another one of its SIMD that is at its products, so that one's vector instructions run beside the other's products; its
    // second products too, where scores are not bent (us, causal: 8192 tokens, 16 heads of 128, bf16 305 without, 289 and 286; 16,384, 16 over 2 1010, 998 and
    // 991; 4096, 16 over 4, capped 122, 108 and 112; 4096, 16 of 64, fp32 312, 288 and 288; but 16 sequences of 512 39, 40 and 41, and heads of 64, fp16 175, 194 and 181).
    constexpr bool kSoftFirst = MOD || sizeof(T) == 4 || DP == 128, kProductToo = !MOD && sizeof(T) == 2;
    typedef typename Elem<T>::Vec8 Vec8;
    auto &lds = *(char (*)[2][2][Keys::kBytes])memory;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
    const int row_wave = wave % RW, half = wave / RW;

    // Workgroups that read the same keys lie n_kv_heads (and n_seq) apart: with a multiple of 8 they are on one die, whose L2 then
    // holds them.  Tiles of rows in descending order, since under a causal mask the last rows see most keys.
    int s = 0, tile, head, split = 0;
    const int kv = b % a.n_kv_heads;
    b /= a.n_kv_heads;
    if (ROWS != kRowsShared && !a.q_ptr) { s = b % a.n_seq; b /= a.n_seq; }
    if constexpr (ROWS != kRowsOfHead) {
        head = kv * a.group;
    } else {
        head = kv * a.group + b % a.group;
        b /= a.group;
    }
    if constexpr (ROWS == kRowsShared) {
        split = b % a.n_split;
        b /= a.n_split;
    }
    if (ROWS != kRowsShared && a.q_ptr) {
        s = slot_sequence<false>(a.q_ptr, a.n_seq, 1, kRows, a.max_tiles, a.n_slots, b, tile);
        if (s < 0) return;
    } else {
        tile = a.n_slots - 1 - b;
    }

    // this lane's row: its token and head, and the keys [lo, hi) that it sees; and what any / all rows of the workgroup and of the wave see
    const int row = tile * kRows + row_wave * 32 + n;
    Seq e;
    int n_keys, token, my_head = head, pos, lo, hi, any_lo, any_hi, wave_lo, wave_hi, full_lo, full_hi;
    bool there;
    if constexpr (ROWS == kRowsShared) {
        __shared__ int ends[kWaves][2];
        n_keys = a.shared_len;
        there = row < a.n_seq * a.max_q * a.group;
        const int t = row / a.group;
        my_head = head + row % a.group;
        s = there ? t / a.max_q : 0;
        token = t - s * a.max_q;
        e = sequence(a, s);
        there = there && token < e.nq;
        pos = n_keys + e.nk - e.nq + token;
        lo = first_key(a, pos);
        hi = there ? min(n_keys, end_key(a, pos, a.prefix ? a.prefix[s] : 0, n_keys + e.nk)) : 0;
        wave_lo = there ? lo : INT32_MAX, wave_hi = hi, full_lo = there ? lo : 0, full_hi = there ? hi : INT32_MAX;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            wave_lo = min(wave_lo, __shfl_xor(wave_lo, d));
            wave_hi = max(wave_hi, __shfl_xor(wave_hi, d));
            full_lo = max(full_lo, __shfl_xor(full_lo, d));
            full_hi = min(full_hi, __shfl_xor(full_hi, d));
        }
        wave_lo = __builtin_amdgcn_readfirstlane(wave_lo), wave_hi = __builtin_amdgcn_readfirstlane(wave_hi);
        full_lo = __builtin_amdgcn_readfirstlane(full_lo), full_hi = __builtin_amdgcn_readfirstlane(full_hi);
        if (lane == 0) ends[wave][0] = wave_lo, ends[wave][1] = wave_hi;
        __syncthreads();
        any_lo = min(min(ends[0][0], ends[1][0]), min(ends[2][0], ends[3][0]));
        any_hi = max(max(ends[0][1], ends[1][1]), max(ends[2][1], ends[3][1]));
        any_lo = __builtin_amdgcn_readfirstlane(any_lo), any_hi = __builtin_amdgcn_readfirstlane(any_hi);
    } else {
        constexpr bool PACK = ROWS == kRowsPacked;
        e = sequence(a, s);
        n_keys = e.nk;
        const int n_rows = PACK ? e.nq * a.group : e.nq;
        if (tile * kRows >= n_rows) return;
        there = row < n_rows;
        token = PACK ? row / a.group : row;
        if constexpr (PACK) my_head = head + row % a.group;
        const int shift = e.nk - e.nq, prefix = a.prefix ? max(a.prefix[s], a.shared_len) - a.shared_len : 0;
        pos = token + shift;
        lo = first_key(a, pos), hi = end_key(a, pos, prefix, n_keys);
        const int last = min(n_rows, tile * kRows + kRows) - 1, w0 = tile * kRows + row_wave * 32, w1 = min(n_rows, w0 + 32) - 1;
        auto of = [&](int r) { return (PACK ? r / a.group : r) + shift; };
        any_lo = first_key(a, of(tile * kRows)), any_hi = end_key(a, of(last), prefix, n_keys);
        wave_lo = first_key(a, of(w0)), wave_hi = w1 < w0 ? 0 : end_key(a, of(w1), prefix, n_keys);
        full_lo = first_key(a, of(max(w1, 0))), full_hi = end_key(a, of(w0), prefix, n_keys);
    }

    const T *q = q_base<T>(a, a.q, e, s, my_head) + (int64_t)token * a.q_row;
    const T *k = ROWS == kRowsShared ? (const T *)a.shared_k + kv * a.k_head : k_base<T>(a, a.k, e, s, kv);
    const T *v = ROWS == kRowsShared ? (const T *)a.shared_v + kv * a.v_head : v_base<T>(a, a.v, e, s, kv);
    Vec8 qf[DP / 16];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) qf[c] = global_operand<T>(q, there, 16 * c + 8 * h, a.head_dim);

    floatx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = zero16();
    const float scale = a.scale;
    Bend<T> bend;
    if constexpr (MOD) bend.init(scale, a.cap);
    const float unit = MOD ? 1.f : scale * kLog2e;  // scores in registers to powers of two
    const float raise = 8.f / unit;
    const float slope = MOD && a.slopes && there ? a.slopes[my_head] * kLog2e : 0.f;
    float m = -INFINITY, sum = 0.f;

    const int n_tiles = any_hi > any_lo ? (any_hi - any_lo + KT - 1) / KT : 0;
    const int each = ROWS == kRowsShared ? (n_tiles + a.n_split - 1) / a.n_split : n_tiles;
    const int first = split * each, last = min(n_tiles, first + each);
    const int row_bytes = a.head_dim * (int)sizeof(T);
    const uint32_t k_stride = (uint32_t)(a.k_row * sizeof(T)), v_stride = (uint32_t)(a.v_row * sizeof(T));
    auto request = [&](int t) {
        const int key = any_lo + t * KT;
        char *to = lds[t & 1][0];
        Keys::template request<kWaves>(to, (const char *)(k + key * a.k_row), k_stride, n_keys - key, row_bytes, wave, lane);
        Keys::template request<kWaves>(to + Keys::kBytes, (const char *)(v + key * a.v_row), v_stride, n_keys - key, row_bytes, wave, lane);
    };
    if (first < last) request(first);
    for (int t = first; t < last; ++t) {
        tiles_arrived();
        if (t + 1 < last) request(t + 1);
        const int key = any_lo + t * KT + half * 32 * KB;
        if (key + 32 * KB <= wave_lo || key >= wave_hi) continue;
        const char *kt = lds[t & 1][0], *vt = lds[t & 1][1];

        int l = lane;
        if constexpr (MOD) asm volatile("" : "+v"(l));  // (places in LDS made anew in every tile: kept, they would not fit the registers)
        floatx16 x[KB];
#pragma unroll
        for (int i = 0; i < KB; ++i) x[i] = zero16();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
            for (int i = 0; i < KB; ++i) x[i] = Elem<T>::mma(Keys::row_operand(kt, 32 * (half * KB + i), c, l), qf[c], x[i]);

        if constexpr (kSoftFirst) __builtin_amdgcn_s_setprio(1);
        if constexpr (MOD) {
            if (bend.cap > 0.f) {
                bend.template apply<KB, false>(x, x);
            } else {
#pragma unroll
                for (int i = 0; i < KB; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[i][r] *= scale * kLog2e;
            }
            if (a.slopes) {
                const float at = (float)(pos - key - 4 * h);
#pragma unroll
                for (int i = 0; i < KB; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[i][r] = fmaf(-slope, fabsf(at - (float)(32 * i + 8 * (r >> 2) + (r & 3))), x[i][r]);
            }
        }
        if (key < full_lo || key + 32 * KB > full_hi) {
            const int at = key + 4 * h - lo;
            const uint32_t span = there && hi > lo ? hi - lo : 0;
#pragma unroll
            for (int i = 0; i < KB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    x[i][r] = (uint32_t)(at + 32 * i + 8 * (r >> 2) + (r & 3)) < span ? x[i][r] : -INFINITY;
        }
        float top = x[0][0];
#pragma unroll
        for (int i = 0; i < KB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, x[i][r]);
        top = halves_max(top);
        if (__any(top > m + raise || (m == -INFINITY && top > m))) {
            const float raised = fmaxf(m, top), by = raised == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - raised) * unit);
            m = raised;
            sum *= by;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= by;
        }
        const float base = m == -INFINITY ? 0.f : m * unit;
#pragma unroll
        for (int i = 0; i < KB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                x[i][r] = __builtin_amdgcn_exp2f(fmaf(x[i][r], unit, -base));
                sum += x[i][r];
            }
        if constexpr (kSoftFirst && !kProductToo) __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int i = 0; i < KB; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Vec8 p = operand<T>(x[i], c);
#pragma unroll
                for (int d = 0; d < DB; ++d) o[d] = Elem<T>::mma(Keys::column_operand(vt, d, 2 * (half * KB + i) + c, l), p, o[d]);
            }
        if constexpr (kSoftFirst && kProductToo) __builtin_amdgcn_s_setprio(0);
    }

    sum = halves_sum(sum);
    m = m == -INFINITY ? m : m * unit;
    if constexpr (RW < kWaves) {
        // the halves of the keys: [element of the lane / 4][lane] of 16 bytes, maximum and sum
        static_assert(RW * 128 * DP + RW * 256 <= (int)sizeof lds);
        __syncthreads();
        floatx4 *other = (floatx4 *)((char *)lds + row_wave * 128 * DP);
        float2 *other_ml = (float2 *)((char *)lds + RW * 128 * DP) + row_wave * 32;
        if (half) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) other[(4 * d + i) * 64 + lane] = floatx4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            if (h == 0) other_ml[n] = make_float2(m, sum);
        }
        __syncthreads();
        if (half) return;
        const float2 ml = other_ml[n];
        const float top = fmaxf(m, ml.x), w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top), u = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
        m = top, sum = sum * w + ml.y * u;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const floatx4 y = other[(4 * d + i) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) o[d][4 * i + j] = o[d][4 * i + j] * w + y[j] * u;
            }
    }
    const int64_t at = (e.lse0 + token) * a.n_heads + my_head;
    if constexpr (ROWS == kRowsShared) {
        if (!there) return;
        const int64_t all = a.rows * a.n_heads, part = a.part0 + split;
        float *to = a.part_o + (part * all + at) * a.head_dim;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = 32 * d + 8 * i + 4 * h;
                if (col < a.head_dim) *(floatx4 *)(to + col) = floatx4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            }
        if (h == 0) a.part_ml[part * all + at] = make_float2(m, sum);
    } else {
        if (there && a.lse && h == 0) a.lse[at] = (m + __builtin_amdgcn_logf(sum)) * kLn2;
        const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        if constexpr (sizeof(T) == 2) {
            static_assert(RW * 128 * DP + RW * 256 + RW * 64 * DP <= kLds || RW == kWaves);
            if constexpr (RW == kWaves) __syncthreads();  // (the tiles have been read by all)
        }
        const int row0 = tile * kRows + row_wave * 32;
        store_turned<T, DP>(memory + (RW == kWaves ? 0 : RW * 128 * DP + RW * 256) + row_wave * 64 * DP, o, by, a.head_dim, lane, [&](int r) -> T * {
            const int at_row = row0 + r;
            if constexpr (ROWS == kRowsOfHead) {
                return at_row < e.nq ? (T *)o_base<T>(a, a.out, e, s, my_head) + (int64_t)at_row * a.o_row : nullptr;
            } else {  // (few: a quotient each)
                const int t = at_row / a.group;
                return at_row < e.nq * a.group ? (T *)o_base<T>(a, a.out, e, s, head + at_row % a.group) + (int64_t)t * a.o_row : nullptr;
            }
        });
    }
}

}  // namespace sddmm
