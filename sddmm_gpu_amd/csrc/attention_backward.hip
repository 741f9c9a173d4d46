// Dense attention, backward (gfx950).
//
//   p_ij = exp(s_ij - lse_i);  dv_j = sum_i p_ij do_i;  ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = do_i . o_i
//   dt_ij = ds_ij (1 - tanh^2);  dq_i = scale sum_j dt_ij k_j;  dk_j = scale sum_i dt_ij q_i
//
// Scores are computed again from q and k: nothing but lse comes from the forward pass.  Two kernels, one that keeps rows of keys and
// walks the rows that see them (dk, dv), and one that keeps rows of queries and walks their keys (dq), compute them twice: seven
// products where five would do with atomic additions, but each result is summed by one wave in a fixed order.
#include "attention.hpp"
#include "attention_launch.hpp"
#include "launch.hpp"

namespace sddmm {

namespace {

constexpr int kRows = 128, kWaves = 4;  // rows (or keys) of a workgroup, 32 to a wave

// stats[head][row] = (lse in powers of two, dout . out).  A row that saw nothing gets +infinity, so that 2^(s - lse) is 0.
template <class T, int DP>
__global__ __launch_bounds__(256)
void sddmm_attention_stats_kernel(const AttnArgs a)
{
    constexpr int kLanes = DP / 8, kPer = 256 / kLanes;
    const int lane = threadIdx.x % kLanes;
    const int64_t at = (int64_t)blockIdx.x * kPer + threadIdx.x / kLanes;
    if (at >= a.rows * a.n_heads) return;
    const int head = (int)(at % a.n_heads);
    const int64_t row = at / a.n_heads;
    int64_t off;
    if (a.q_ptr) {
        if (row < a.q_ptr[0] || row >= a.q_ptr[a.n_seq]) return;
        off = row * a.o_row;
    } else {
        const int s = (int)(row / a.max_q), i = (int)(row % a.max_q);
        if (a.q_len && i >= min(a.q_len[s], a.max_q)) return;
        off = s * a.o_seq + i * a.o_row;
    }
    off += head * a.o_head;
    const auto x = __builtin_convertvector(global_operand<T>((const T *)a.out + off, true, 8 * lane, a.head_dim), floatx8);
    const auto y = __builtin_convertvector(global_operand<T>((const T *)a.dout + off, true, 8 * lane, a.head_dim), floatx8);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(x[j], y[j], sum);
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) sum += __shfl_xor(sum, d);
    const float lse = a.lse[at];
    if (lane == 0) {
        a.stat_lse[head * a.rows + row] = lse == -INFINITY ? INFINITY : lse * kLog2e;
        a.stat_delta[head * a.rows + row] = sum;
    }
}

// scores in powers of two from products, and what they have to be multiplied by on the way back
template <bool MOD>
__device__ __forceinline__ void bend(floatx16 &x, floatx16 &back, float scale, float cap, float cap_inv, bool bias, float slope, float at, float step)
{
    if constexpr (MOD) {
        if (cap > 0.f) {
            const float to = cap * kLog2e;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float y = tanh_any(x[r] * cap_inv);
                back[r] = fmaf(-y, y, 1.f);
                x[r] = to * y;
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) back[r] = 1.f, x[r] *= scale * kLog2e;
        }
        if (bias) {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = fmaf(-slope, fabsf(at + step * (float)(8 * (r >> 2) + (r & 3))), x[r]);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] *= scale * kLog2e;
    }
}

// The rows that see key j: [first, end).
__device__ __forceinline__ int first_row(const AttnArgs &a, int j, int prefix, int shift)
{
    return a.right < 0 || j < prefix ? 0 : max(0, j - min(a.right, j) - shift);
}
__device__ __forceinline__ int end_row(const AttnArgs &a, int j, int shift, int n_rows)
{
    return a.left < 0 ? n_rows : min(n_rows, max(0, min(j, INT32_MAX / 2) + min(a.left, INT32_MAX / 2) + 1 - shift));
}

// dk and dv.  A wave holds 32 keys: k and v as operands, the sums of dk and dv turned (element of the head by key).  Per tile of rows, q and
// do of which the four waves share in LDS with their statistics: S = Q K^T and dP = dO V^T, a lane holding one key's; P and dS are
// operands of dV^T += dO^T P and dK^T += Q^T dS as they lie, q and do being read a second time, in the transposing way.  The query heads that share a key
// head follow each other in the same sums.
template <class T, int DP, bool MOD>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 && DP == 128 ? 1 : 2)
void sddmm_attention_dkv_kernel(const AttnArgs a)
{
    constexpr int QT = 32, DB = DP / 32;
    typedef Tile<T, DP, QT> Rows;
    typedef Tile<T, DP, kRows> Values;
    typedef typename Elem<T>::Vec8 Vec8;
    // (registers: 128 for the sums, 32 for k, 32 for a tile's scores; v would be 32 more than two waves to a SIMD leave)
    constexpr bool kKeepV = sizeof(T) == 4 || DP == 64;
    __shared__ __align__(1024) char lds[2][2][Rows::kBytes];
    __shared__ __align__(1024) char values[kKeepV ? 16 : Values::kBytes];
    __shared__ __align__(16) float stat[2][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;

    int b = blockIdx.x, s, tile, split = 0;
    const int kv = b % a.n_kv_heads;
    b /= a.n_kv_heads;
    if (!a.k_ptr) { s = b % a.n_seq; b /= a.n_seq; }
    if (a.n_split > 1) { split = b % a.n_split; b /= a.n_split; }
    if (a.k_ptr) s = slot_sequence(a.k_ptr, a.n_seq, kRows, b, tile); else tile = b;
    const Seq e = sequence(a, s);
    if (tile * kRows >= e.nk) return;
    const int shift = e.nk - e.nq, prefix = a.prefix ? a.prefix[s] : 0;
    const int key = tile * kRows + wave * 32 + n;
    const bool there = key < e.nk;
    const int lo = first_row(a, key, prefix, shift), hi = there ? end_row(a, key, shift, e.nq) : 0;
    const int k0 = tile * kRows, k1 = min(e.nk, k0 + kRows) - 1, w0 = k0 + wave * 32, w1 = min(e.nk, w0 + 32) - 1;
    const int any_lo = first_row(a, k0, prefix, shift), any_hi = end_row(a, k1, shift, e.nq);
    const int wave_lo = first_row(a, w0, prefix, shift), wave_hi = w1 < w0 ? 0 : end_row(a, w1, shift, e.nq);
    const int full_lo = first_row(a, max(w1, 0), prefix, shift), full_hi = w1 < w0 + 31 ? 0 : end_row(a, w0, shift, e.nq);

    const int row_bytes = a.head_dim * (int)sizeof(T);
    Vec8 kf[DP / 16], vf[kKeepV ? DP / 16 : 1];
    {
        const T *k = k_base<T>(a, a.k, e, s, kv) + key * a.k_row, *v = v_base<T>(a, a.v, e, s, kv);
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) kf[c] = global_operand<T>(k, there, 16 * c + 8 * h, a.head_dim);
        if constexpr (kKeepV) {
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) vf[c] = global_operand<T>(v + key * a.v_row, there, 16 * c + 8 * h, a.head_dim);
        } else {
            Values::template request<kWaves>(values, (const char *)(v + k0 * a.v_row), (uint32_t)(a.v_row * sizeof(T)), e.nk - k0, row_bytes, wave, lane);
        }
    }
    floatx16 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();

    const float scale = a.scale, cap = a.cap, cap_inv = MOD && cap > 0.f ? scale / cap : 0.f;
    const int tiles = any_hi > any_lo ? (any_hi - any_lo + QT - 1) / QT : 0, all = tiles * a.group;
    const int each = (all + a.n_split - 1) / a.n_split, first = split * each, last = min(all, first + each);
    const uint32_t q_stride = (uint32_t)(a.q_row * sizeof(T)), o_stride = (uint32_t)(a.o_row * sizeof(T));
    auto request = [&](int t) {
        const int head = kv * a.group + t / tiles, row = any_lo + t % tiles * QT;
        char *to = lds[t & 1][0];
        Rows::template request<kWaves>(to, (const char *)(q_base<T>(a, a.q, e, s, head) + row * a.q_row), q_stride, e.nq - row, row_bytes, wave, lane);
        Rows::template request<kWaves>(to + Rows::kBytes, (const char *)(o_base<T>(a, a.dout, e, s, head) + row * a.o_row), o_stride, e.nq - row, row_bytes, wave, lane);
        if (wave < 2) request_floats<QT>(stat[t & 1][wave], (wave ? a.stat_delta : a.stat_lse) + head * a.rows + e.lse0 + row, e.nq - row, lane);
    };
    if (first < last) request(first);
    for (int t = first; t < last; ++t) {
        tiles_arrived();
        if (t + 1 < last) request(t + 1);
        const char *qt = lds[t & 1][0], *dot = lds[t & 1][1];
        const float slope = MOD && a.slopes ? a.slopes[kv * a.group + t / tiles] * kLog2e : 0.f;
#pragma unroll 1
        for (int u = 0; u < QT / 32; ++u) {
            const int row = any_lo + t % tiles * QT + 32 * u;
            if (row + 32 <= wave_lo || row >= wave_hi) continue;
            int l = lane;  // (places in LDS made anew in every tile: kept, they would not fit the registers)
            asm volatile("" : "+v"(l));
            floatx16 x = zero16(), y = zero16(), back;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) x = Elem<T>::mma(Rows::row_operand(qt, 32 * u, c, l), kf[c], x);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) y = Elem<T>::mma(Rows::row_operand(dot, 32 * u, c, l), kKeepV ? vf[kKeepV ? c : 0] : Values::row_operand(values, 32 * wave, c, l), y);
            bend<MOD>(x, back, scale, cap, cap_inv, a.slopes != nullptr, slope, (float)(row + 4 * h + shift - key), 1.f);
            const bool masked = row < full_lo || row + 32 > full_hi;
            const int at = row + 4 * h - lo;
            const uint32_t span = hi > lo ? hi - lo : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const floatx4 lse = *(const floatx4 *)&stat[t & 1][0][32 * u + 8 * i + 4 * h], delta = *(const floatx4 *)&stat[t & 1][1][32 * u + 8 * i + 4 * h];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = 4 * i + j;
                    x[r] = __builtin_amdgcn_exp2f(x[r] - lse[j]);
                    y[r] -= delta[j];
                }
            }
            if (masked) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool seen = (uint32_t)(at + 8 * (r >> 2) + (r & 3)) < span;
                    x[r] = seen ? x[r] : 0.f;
                    y[r] = seen ? y[r] : 0.f;
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                y[r] *= x[r];
                if constexpr (MOD) y[r] *= back[r];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Vec8 p = operand<T>(x, c), ds = operand<T>(y, c);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    dv[d] = Elem<T>::mma(Rows::column_operand(dot, d, 2 * u + c, l), p, dv[d]);
                    dk[d] = Elem<T>::mma(Rows::column_operand(qt, d, 2 * u + c, l), ds, dk[d]);
                }
            }
        }
    }
    if (!there) return;
#pragma unroll
    for (int d = 0; d < DB; ++d) dk[d] *= scale;
    if (a.n_split > 1) {
        // parts of dk, then of dv: [part][key][key head][head_dim]
        const int64_t place = ((e.k0 + (a.k_ptr ? 0 : (int64_t)s * a.max_k) + key) * a.n_kv_heads + kv) * a.head_dim, part = a.key_rows * a.n_kv_heads * a.head_dim;
        float *to = a.part_o + split * part + place, *to_v = to + a.n_split * part;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = 32 * d + 8 * i + 4 * h;
                if (col >= a.head_dim) continue;
                *(floatx4 *)(to + col) = floatx4{dk[d][4 * i], dk[d][4 * i + 1], dk[d][4 * i + 2], dk[d][4 * i + 3]};
                *(floatx4 *)(to_v + col) = floatx4{dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]};
            }
        return;
    }
    typedef typename Elem<T>::Vec4 Vec4;
    T *to = (T *)k_base<T>(a, a.dk, e, s, kv) + key * a.k_row, *to_v = (T *)v_base<T>(a, a.dv, e, s, kv) + key * a.v_row;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 32 * d + 8 * i + 4 * h;
            if (col >= a.head_dim) continue;
            *(Vec4 *)(to + col) = __builtin_convertvector((floatx4{dk[d][4 * i], dk[d][4 * i + 1], dk[d][4 * i + 2], dk[d][4 * i + 3]}), Vec4);
            *(Vec4 *)(to_v + col) = __builtin_convertvector((floatx4{dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]}), Vec4);
        }
}

// The sum of the parts of dk and dv, four elements a thread.
template <class T>
__global__ __launch_bounds__(256)
void sddmm_attention_dkv_sum_kernel(const AttnArgs a)
{
    const int64_t per = a.n_kv_heads * (a.head_dim / 4), at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= a.key_rows * per) return;
    const int64_t row = at / per;
    const int rest = (int)(at % per), kv = rest / (a.head_dim / 4), col = rest % (a.head_dim / 4) * 4;
    int64_t k_off, v_off;
    if (a.k_ptr) {
        if (row < a.k_ptr[0] || row >= a.k_ptr[a.n_seq]) return;
        k_off = row * a.k_row, v_off = row * a.v_row;
    } else {
        const int s = (int)(row / a.max_k), i = (int)(row % a.max_k);
        if (a.k_len && i >= min(a.k_len[s], a.max_k)) return;
        k_off = s * a.k_seq + i * a.k_row, v_off = s * a.v_seq + i * a.v_row;
    }
    const int64_t part = a.key_rows * a.n_kv_heads * a.head_dim;
    const float *from = a.part_o + at * 4, *from_v = from + a.n_split * part;
    floatx4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
    for (int p = 0; p < a.n_split; ++p) {
        x += *(const floatx4 *)(from + p * part);
        y += *(const floatx4 *)(from_v + p * part);
    }
    typedef typename Elem<T>::Vec4 Vec4;
    *(Vec4 *)((T *)a.dk + k_off + kv * a.k_head + col) = __builtin_convertvector(x, Vec4);
    *(Vec4 *)((T *)a.dv + v_off + kv * a.v_head + col) = __builtin_convertvector(y, Vec4);
}

// dq.  A wave holds 32 rows: q and do as operands, the sums of dq turned.  Per tile of keys in LDS: S^T = K Q^T, dP^T = V dO^T, then
// dQ^T += K^T dS^T.
//
// The gradient of a head's slope, - sum ds |p_i - j|, is asked to fp32 whatever the operands' type, and delta, which comes from the rounded
// output, would put an error of every row times its mean distance into it.  So it is made of sums that need no delta:
// with far = |p_i - j|, - sum_i (sum_j p dp far - (sum_j p dp) (sum_j p far) / sum_j p).
template <class T, int DP, bool MOD>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 && DP == 128 ? 1 : 2)
void sddmm_attention_dq_kernel(const AttnArgs a)
{
    constexpr int KT = sizeof(T) == 2 ? 64 : 32, DB = DP / 32;
    typedef Tile<T, DP, KT> Keys;
    typedef typename Elem<T>::Vec8 Vec8;
    __shared__ __align__(1024) char lds[2][2][Keys::kBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;

    int b = blockIdx.x, s = 0, tile;  // (as in the forward kernel)
    const int kv = b % a.n_kv_heads;
    b /= a.n_kv_heads;
    if (!a.q_ptr) { s = b % a.n_seq; b /= a.n_seq; }
    const int head = kv * a.group + b % a.group;
    b /= a.group;
    const int slot = a.n_slots - 1 - b;
    double *slope_part = MOD && a.slope_part ? a.slope_part + (int64_t)head * a.slope_parts + (a.q_ptr ? slot : slot * a.n_seq + s) : nullptr;
    if (slope_part && threadIdx.x == 0) *slope_part = 0.;
    if (a.q_ptr) s = slot_sequence(a.q_ptr, a.n_seq, kRows, slot, tile); else tile = slot;
    const Seq e = sequence(a, s);
    if (tile * kRows >= e.nq) return;
    const int row = tile * kRows + wave * 32 + n, shift = e.nk - e.nq, prefix = a.prefix ? a.prefix[s] : 0, pos = row + shift;
    const bool there = row < e.nq;
    const int lo = first_key(a, pos), hi = there ? end_key(a, pos, prefix, e.nk) : 0;
    const int r1 = min(e.nq, tile * kRows + kRows) - 1, w0 = tile * kRows + wave * 32, w1 = min(e.nq, w0 + 32) - 1;
    const int any_lo = first_key(a, tile * kRows + shift), any_hi = end_key(a, r1 + shift, prefix, e.nk);
    const int wave_lo = first_key(a, w0 + shift), wave_hi = w1 < w0 ? 0 : end_key(a, w1 + shift, prefix, e.nk);
    const int full_lo = first_key(a, w1 + shift), full_hi = w1 < w0 + 31 ? 0 : end_key(a, w0 + shift, prefix, e.nk);

    Vec8 qf[DP / 16], of[DP / 16];
    {
        const T *q = q_base<T>(a, a.q, e, s, head) + row * a.q_row, *dout = o_base<T>(a, a.dout, e, s, head) + row * a.o_row;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) qf[c] = global_operand<T>(q, there, 16 * c + 8 * h, a.head_dim);
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) of[c] = global_operand<T>(dout, there, 16 * c + 8 * h, a.head_dim);
    }
    const int64_t at_stat = (int64_t)head * a.rows + e.lse0 + row;
    const float lse = there ? a.stat_lse[at_stat] : INFINITY, delta = there ? a.stat_delta[at_stat] : 0.f;
    const T *k = k_base<T>(a, a.k, e, s, kv), *v = v_base<T>(a, a.v, e, s, kv);
    floatx16 dq[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) dq[d] = zero16();
    const float scale = a.scale, cap = a.cap, cap_inv = MOD && cap > 0.f ? scale / cap : 0.f;
    const float slope = MOD && a.slopes ? a.slopes[head] * kLog2e : 0.f;
    double far_ds = 0., far_p = 0., sum_ds = 0., sum_p = 0.;

    const int last = any_hi > any_lo ? (any_hi - any_lo + KT - 1) / KT : 0;
    const int row_bytes = a.head_dim * (int)sizeof(T);
    const uint32_t k_stride = (uint32_t)(a.k_row * sizeof(T)), v_stride = (uint32_t)(a.v_row * sizeof(T));
    auto request = [&](int t) {
        const int key = any_lo + t * KT;
        char *to = lds[t & 1][0];
        Keys::template request<kWaves>(to, (const char *)(k + key * a.k_row), k_stride, e.nk - key, row_bytes, wave, lane);
        Keys::template request<kWaves>(to + Keys::kBytes, (const char *)(v + key * a.v_row), v_stride, e.nk - key, row_bytes, wave, lane);
    };
    if (last > 0) request(0);
    for (int t = 0; t < last; ++t) {
        tiles_arrived();
        if (t + 1 < last) request(t + 1);
        const char *kt = lds[t & 1][0], *vt = lds[t & 1][1];
#pragma unroll 1
        for (int u = 0; u < KT / 32; ++u) {
            const int key = any_lo + t * KT + 32 * u;
            if (key + 32 <= wave_lo || key >= wave_hi) continue;
            int l = lane;  // (places in LDS made anew in every tile: kept, they would not fit the registers)
            asm volatile("" : "+v"(l));
            floatx16 x = zero16(), y = zero16(), back;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) x = Elem<T>::mma(Keys::row_operand(kt, 32 * u, c, l), qf[c], x);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) y = Elem<T>::mma(Keys::row_operand(vt, 32 * u, c, l), of[c], y);
            const float away = (float)(pos - key - 4 * h);
            bend<MOD>(x, back, scale, cap, cap_inv, a.slopes != nullptr, slope, away, -1.f);
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(x[r] - lse);
            if (key < full_lo || key + 32 > full_hi) {
                const int at = key + 4 * h - lo;
                const uint32_t span = hi > lo ? hi - lo : 0;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool seen = (uint32_t)(at + 8 * (r >> 2) + (r & 3)) < span;
                    x[r] = seen ? x[r] : 0.f;
                    y[r] = seen ? y[r] : 0.f;
                }
            }
            if constexpr (MOD) {
                if (slope_part) {
                    float w0 = 0.f, w1 = 0.f, w2 = 0.f, w3 = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float far = fabsf(away - (float)(8 * (r >> 2) + (r & 3))), z = x[r] * y[r];
                        w0 = fmaf(z, far, w0), w1 = fmaf(x[r], far, w1), w2 += z, w3 += x[r];
                    }
                    far_ds += w0, far_p += w1, sum_ds += w2, sum_p += w3;
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                y[r] = x[r] * (y[r] - delta);
                if constexpr (MOD) y[r] *= back[r];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Vec8 ds = operand<T>(y, c);
#pragma unroll
                for (int d = 0; d < DB; ++d) dq[d] = Elem<T>::mma(Keys::column_operand(kt, d, 2 * u + c, l), ds, dq[d]);
            }
        }
    }
    if (MOD && slope_part) {
        __shared__ double parts[kWaves];
        far_ds += __shfl_xor(far_ds, 32), far_p += __shfl_xor(far_p, 32), sum_ds += __shfl_xor(sum_ds, 32), sum_p += __shfl_xor(sum_p, 32);
        double g = sum_p > 0. || sum_p != sum_p ? sum_ds * far_p / sum_p - far_ds : 0.;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) g += __shfl_xor(g, d);
        if (lane == 0) parts[wave] = g;
        __syncthreads();
        if (threadIdx.x == 0) *slope_part = parts[0] + parts[1] + parts[2] + parts[3];
    }
    if (!there) return;
    typedef typename Elem<T>::Vec4 Vec4;
    T *to = (T *)q_base<T>(a, a.dq, e, s, head) + row * a.q_row;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 32 * d + 8 * i + 4 * h;
            if (col < a.head_dim)
                *(Vec4 *)(to + col) = __builtin_convertvector((floatx4{dq[d][4 * i], dq[d][4 * i + 1], dq[d][4 * i + 2], dq[d][4 * i + 3]} * scale), Vec4);
        }
}

// The slopes' gradients: a head's parts in a fixed order.
__global__ __launch_bounds__(256)
void sddmm_attention_dslopes_kernel(const AttnArgs a)
{
    __shared__ double sums[256];
    double x = 0.;
    for (int p = threadIdx.x; p < a.slope_parts; p += 256) x += a.slope_part[(int64_t)blockIdx.x * a.slope_parts + p];
    sums[threadIdx.x] = x;
    __syncthreads();
    for (int d = 128; d > 0; d /= 2) {
        if ((int)threadIdx.x < d) sums[threadIdx.x] += sums[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.dslopes[blockIdx.x] = (float)sums[0];
}

template <class T, int DP>
hipError_t launch_typed(const AttnArgs &a, unsigned kv_grid, unsigned q_grid, int q_slots, hipStream_t st)
{
    const bool mod = a.cap > 0.f || a.slopes;
    constexpr int kPer = 256 / (DP / 8);
    hipError_t e = hipSuccess;
    if (q_grid) e = launch(sddmm_attention_stats_kernel<T, DP>, dim3((unsigned)((a.rows * a.n_heads + kPer - 1) / kPer)), dim3(256), 0, st, a);
    if (e == hipSuccess && kv_grid) e = launch(mod ? sddmm_attention_dkv_kernel<T, DP, true> : sddmm_attention_dkv_kernel<T, DP, false>, dim3(kv_grid), dim3(64 * kWaves), 0, st, a);
    if (e == hipSuccess && kv_grid && a.n_split > 1)
        e = launch(sddmm_attention_dkv_sum_kernel<T>, dim3((unsigned)((a.key_rows * a.n_kv_heads * (a.head_dim / 4) + 255) / 256)), dim3(256), 0, st, a);
    AttnArgs b = a;
    b.n_slots = q_slots;
    if (e == hipSuccess && q_grid) e = launch(mod ? sddmm_attention_dq_kernel<T, DP, true> : sddmm_attention_dq_kernel<T, DP, false>, dim3(q_grid), dim3(64 * kWaves), 0, st, b);
    if (e == hipSuccess && a.dslopes) e = launch(sddmm_attention_dslopes_kernel, dim3((unsigned)a.n_heads), dim3(256), 0, st, a);
    return e;
}

template <class T>
hipError_t launch_dims(const AttnArgs &a, unsigned kv_grid, unsigned q_grid, int q_slots, hipStream_t st)
{
    return a.head_dim <= 64 ? launch_typed<T, 64>(a, kv_grid, q_grid, q_slots, st) : launch_typed<T, 128>(a, kv_grid, q_grid, q_slots, st);
}

}  // namespace

int attention_backward_rows() { return kRows; }

hipError_t launch_attention_backward(const AttnArgs &a, int type, unsigned kv_grid, unsigned q_grid, int q_slots, hipStream_t st)
{
    return type == SDDMM_TYPE_F32 ? launch_dims<float>(a, kv_grid, q_grid, q_slots, st)
         : type == SDDMM_TYPE_F16 ? launch_dims<_Float16>(a, kv_grid, q_grid, q_slots, st) : launch_dims<__bf16>(a, kv_grid, q_grid, q_slots, st);
}

}  // namespace sddmm
