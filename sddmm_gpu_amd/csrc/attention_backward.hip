// Dense attention, backward (gfx950).
//
//   p_ij = exp(s_ij - lse_i);  dv_j = sum_i p_ij do_i;  ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = do_i . o_i
//   dt_ij = ds_ij (1 - tanh^2);  dq_i = scale sum_j dt_ij k_j;  dk_j = scale sum_i dt_ij q_i
//
// Scores are computed again from q and k: nothing but lse comes from the forward pass.  Two kernels, one that keeps rows of queries and
// walks their keys (dq), and one that keeps rows of keys and walks the rows that see them (dk, dv), compute them twice: seven
// products where five would do with atomic additions, but each result is summed in a fixed order.  The first leaves every row's
// statistics (lse in powers of two, delta; [n_heads][rows]) for the second.
//
// Roundings with 16-bit operands: P and dt to the element type, as operands; delta comes from the rounded output.  With bf16 dq and dk are off by 0.0025
// of their size where rounding the results alone makes 0.0017 (fp32 operands: 3e-7).  A second operand for what dt loses would be two products beside seven.
//
// 8192 tokens, causal, 16 heads of 128, bf16: dq 0.40 ms and dk, dv 0.56 ms, 1.03 and 0.97 PFLOP/s of their products (a large library product 1.17);
// fp32, 4096 tokens, 16 heads of 64 1.2 ms, 98 TFLOP/s (154): matrix and vector instructions of a SIMD, which alternate, bound both.
#include "attention.hpp"
#include "attention_launch.hpp"
#include "launch.hpp"

namespace sddmm {

namespace {

constexpr int kWaves = 4, kFewKeys = 32;  // keys of a workgroup of the dk, dv kernel for few

// 16-bit operands, heads of more than 64 or scores that are bent or biased: a wave that is past its first products goes before another one of its SIMD that is at them, so
// that one's vector instructions run beside the other's products; of plain scores the second products too (us without and with, causal: 8192 tokens, 16 heads of
// 128, bf16 1020 and 959; 4096, 16 over 4, capped 405 and 386; 8192, 16 of 64, capped 900 and 819, 2048 in 3 sequences, 12 of 64, capped 187 and 189; but
// plain scores of heads of 64, fp16 596 and 628, fp32 1212 and 1245).
template <class T, int DP, bool MOD> __device__ __forceinline__ void raise_priority() { if constexpr (sizeof(T) == 2 && (DP == 128 || MOD)) __builtin_amdgcn_s_setprio(1); }
template <class T, int DP, bool MOD> __device__ __forceinline__ void lower_priority() { if constexpr (sizeof(T) == 2 && (DP == 128 || MOD)) __builtin_amdgcn_s_setprio(0); }

// scores in powers of two from products, and what their gradients have to be multiplied by on the way back
template <bool MOD, class T>
__device__ __forceinline__ void scores(floatx16 &x, floatx16 &back, const Bend<T> &bend, float unit, bool bias, float slope, float at, float step)
{
    if constexpr (MOD) {
        if (bend.cap > 0.f) {
            floatx16 y[1] = {x}, z[1];
            bend.template apply<1, true>(y, z);
            x = y[0], back = z[0];
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) back[r] = 1.f, x[r] *= unit;
        }
        if (bias) {
#pragma unroll
            for (int r = 0; r < 16; ++r) x[r] = fmaf(-slope, fabsf(at + step * (float)(8 * (r >> 2) + (r & 3))), x[r]);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] *= unit;
    }
}

// The keys of a workgroup (KEYS of them), and how the rows that see them are cut into pieces (a.n_split at most, of about a.chunk rows of all
// heads): a key tile early in a long sequence has many times the rows of others.
struct KeyTile {
    Seq e;
    int s, kv, tile, shift, prefix, any_lo, any_hi, pieces;
};
template <int KEYS>
__device__ __forceinline__ bool key_tile(const AttnArgs &a, int b, KeyTile &k)
{
    k.kv = b % a.n_kv_heads;
    b /= a.n_kv_heads;
    if (a.k_ptr) {
        k.s = slot_sequence<true>(a.k_ptr, a.n_seq, 1, KEYS, a.max_tiles, a.n_slots, b, k.tile);
        if (k.s < 0) return false;
    } else {
        k.s = b % a.n_seq, k.tile = b / a.n_seq;
    }
    k.e = sequence(a, k.s);
    if (k.tile * KEYS >= k.e.nk) return false;
    k.shift = k.e.nk - k.e.nq, k.prefix = a.prefix ? a.prefix[k.s] : 0;
    k.any_lo = first_row(a, k.tile * KEYS, k.prefix, k.shift);
    k.any_hi = end_row(a, min(k.e.nk, k.tile * KEYS + KEYS) - 1, k.shift, k.e.nq);
    const int64_t rows = (int64_t)max(0, k.any_hi - k.any_lo) * a.group;
    k.pieces = (int)max((int64_t)1, min((int64_t)a.n_split, (rows + a.chunk - 1) / a.chunk));
    return true;
}

// 32 keys of a wave: k as an operand, the sums of dk and dv turned (element of the head by key).  Per tile of 32 rows, q and do of which are in LDS
// with their statistics: S = Q K^T and dP = dO V^T, a lane holding one key's; P and dS are operands of dV^T += dO^T P and dK^T += Q^T dS as
// they lie, q and do being read a second time, in the transposing way.
template <class T, int DP, bool MOD>
struct DkvKeys {
    static constexpr int DB = DP / 32;
    typedef typename Elem<T>::Vec8 Vec8;
    typedef Tile<T, DP, 32> Rows;
    Vec8 kf[DP / 16];
    floatx16 dk[DB], dv[DB];
    float unit;
    Bend<T> bend;
    bool bias, there;
    int key, lo, hi, wave_lo, wave_hi, full_lo, full_hi, shift, h;

    __device__ __forceinline__ void init(const AttnArgs &a, const KeyTile &t, int first, int lane)
    {
        h = lane >> 5, key = first + (lane & 31), shift = t.shift;
        there = key < t.e.nk;
        lo = first_row(a, key, t.prefix, shift), hi = there ? end_row(a, key, shift, t.e.nq) : 0;
        const int last = min(t.e.nk, first + 32) - 1;
        wave_lo = first_row(a, first, t.prefix, shift), wave_hi = last < first ? 0 : end_row(a, last, shift, t.e.nq);
        full_lo = first_row(a, max(last, 0), t.prefix, shift), full_hi = last < first + 31 ? 0 : end_row(a, first, shift, t.e.nq);
        const T *k = k_base<T>(a, a.k, t.e, t.s, t.kv) + key * a.k_row;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) kf[c] = global_operand<T>(k, there, 16 * c + 8 * h, a.head_dim);
#pragma unroll
        for (int d = 0; d < DB; ++d) dk[d] = dv[d] = zero16();
        unit = a.scale * kLog2e, bias = a.slopes != nullptr;
        if constexpr (MOD) bend.init(a.scale, a.cap);
    }
    __device__ __forceinline__ bool sees(int row) const { return row + 32 > wave_lo && row < wave_hi; }
    // EARLY: dP begins at - delta, a subtraction less for each score, where registers are left (300 tokens, 16 heads over 4 of 128, bf16 40 and 38 us; in the kernel of
    // whole tiles they are not: 960 and 1060 us).
    // rows `row` on: their tiles, log-sum-exps and - deltas; v(c): 16 elements of v as an operand
    template <bool EARLY, class V> __device__ __forceinline__ void add(const char *qt, const char *dot, const float *lse, const float *minus_delta, int row, float slope, int l, V v)
    {
        floatx16 x = zero16(), y = zero16(), back;
        if constexpr (EARLY) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const floatx4 d = *(const floatx4 *)(minus_delta + 8 * i + 4 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j) y[4 * i + j] = d[j];
            }
        }
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) x = Elem<T>::mma(Rows::row_operand(qt, 0, c, l), kf[c], x);
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) y = Elem<T>::mma(Rows::row_operand(dot, 0, c, l), v(c), y);
        raise_priority<T, DP, MOD>();
        scores<MOD, T>(x, back, bend, unit, bias, slope, (float)(row + 4 * h + shift - key), 1.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const floatx4 m = *(const floatx4 *)(lse + 8 * i + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = __builtin_amdgcn_exp2f(x[4 * i + j] - m[j]);
            if constexpr (!EARLY) {
                const floatx4 d = *(const floatx4 *)(minus_delta + 8 * i + 4 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j) y[4 * i + j] += d[j];
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            y[r] *= x[r];
            if constexpr (MOD) y[r] *= back[r];
        }
        if (row < full_lo || row + 32 > full_hi) {  // (last: a factor of what is not seen may be NaN)
            const int at = row + 4 * h - lo;
            const uint32_t span = hi > lo ? hi - lo : 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool seen = (uint32_t)(at + 8 * (r >> 2) + (r & 3)) < span;
                x[r] = seen ? x[r] : 0.f;
                y[r] = seen ? y[r] : 0.f;
            }
        }
        if constexpr (MOD) lower_priority<T, DP, MOD>();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const Vec8 p = operand<T>(x, c), ds = operand<T>(y, c);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                dv[d] = Elem<T>::mma(Rows::column_operand(dot, d, c, l), p, dv[d]);
                dk[d] = Elem<T>::mma(Rows::column_operand(qt, d, c, l), ds, dk[d]);
            }
        }
        if constexpr (!MOD) lower_priority<T, DP, MOD>();
    }
    // calls f(i, four elements) for the pieces i = 0 .. 8 DB - 1 of a lane's sums: dk, then dv
    template <class F> __device__ __forceinline__ void pieces(F f) const
    {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f(4 * d + i, floatx4{dk[d][4 * i], dk[d][4 * i + 1], dk[d][4 * i + 2], dk[d][4 * i + 3]});
                f(4 * (DB + d) + i, floatx4{dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]});
            }
    }
    template <class F> __device__ __forceinline__ void join(F f)
    {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const floatx4 y = f(4 * d + i), z = f(4 * (DB + d) + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) dk[d][4 * i + j] += y[j], dv[d][4 * i + j] += z[j];
            }
    }
    static __device__ __forceinline__ void store(const AttnArgs &a, const KeyTile &t, int key, int i, int h, floatx4 y)
    {
        typedef typename Elem<T>::Vec4 Vec4;
        const int col = 8 * (i % (4 * DB)) + 4 * h;
        if (col >= a.head_dim) return;
        if (i < 4 * DB) y *= a.scale;
        T *to = i < 4 * DB ? (T *)k_base<T>(a, a.dk, t.e, t.s, t.kv) + key * a.k_row : (T *)v_base<T>(a, a.dv, t.e, t.s, t.kv) + key * a.v_row;
        *(Vec4 *)(to + col) = __builtin_convertvector(y, Vec4);
    }
};

// dk and dv of 32 keys to each of KW waves, which share the tiles of rows.  The query heads that share a key head follow each other in the same sums.
// 13 documents of 22 to 2281 tokens, 8192 in all, 16 heads over 4 of 128, bf16: 151 us, and 21 to sum the parts: a compute unit has work for 70 % of it.
// With two such waves the other two take every second tile of rows, and the sums are joined at the end: twice the workgroups, of half the length.
template <class T, int DP, bool MOD, int KW>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 && DP == 128 ? 1 : 2)
void sddmm_attention_dkv_kernel(const AttnArgs a)
{
    typedef DkvKeys<T, DP, MOD> Keys;
    typedef typename Keys::Rows Rows;
    constexpr int kKeys = 32 * KW, kTiles = kWaves / KW;  // tiles of rows in LDS together
    typedef Tile<T, DP, kKeys> Values;
    typedef typename Elem<T>::Vec8 Vec8;
    // (registers: 128 for the sums, 32 for k, 32 for a tile's scores; v would be 32 more than two waves to a SIMD leave)
    constexpr bool kKeepV = sizeof(T) == 4 || DP <= 64;
    __shared__ __align__(1024) char lds[2][kTiles][2][Rows::kBytes];
    __shared__ __align__(1024) char values[kKeepV ? 16 : Values::kBytes];
    __shared__ __align__(16) float stat[2][kTiles][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int key_wave = wave % KW, part = wave / KW;

    KeyTile at;
    // (pieces outermost: next to each other they would go to different dies, the later ones, of which there are fewer, always to the same)
    const int groups = gridDim.x / a.n_split, split = blockIdx.x / groups;
    if (!key_tile<kKeys>(a, blockIdx.x - split * groups, at) || split >= at.pieces) return;
    const int row_bytes = a.head_dim * (int)sizeof(T), k0 = at.tile * kKeys;
    Keys keys;
    keys.init(a, at, k0 + 32 * key_wave, lane);
    Vec8 vf[kKeepV ? DP / 16 : 1];
    {
        const T *v = v_base<T>(a, a.v, at.e, at.s, at.kv);
        if constexpr (kKeepV) {
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) vf[c] = global_operand<T>(v + keys.key * a.v_row, keys.there, 16 * c + 8 * h, a.head_dim);
        } else {
            Values::template request<kWaves>(values, (const char *)(v + k0 * a.v_row), (uint32_t)(a.v_row * sizeof(T)), at.e.nk - k0, row_bytes, wave, lane);
        }
    }
    const int tiles = at.any_hi > at.any_lo ? (at.any_hi - at.any_lo + 31) / 32 : 0, all = tiles * a.group;
    const int each = (all + at.pieces - 1) / at.pieces, first = split * each, last = min(all, first + each);
    const uint32_t q_stride = (uint32_t)(a.q_row * sizeof(T)), o_stride = (uint32_t)(a.o_row * sizeof(T));
    auto request = [&](int t, int turn) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            if (t + i >= last) break;
            const int head = at.kv * a.group + (t + i) / tiles, row = at.any_lo + (t + i) % tiles * 32;
            char *to = lds[turn][i][0];
            Rows::template request<kWaves>(to, (const char *)(q_base<T>(a, a.q, at.e, at.s, head) + row * a.q_row), q_stride, at.e.nq - row, row_bytes, wave, lane);
            Rows::template request<kWaves>(to + Rows::kBytes, (const char *)(o_base<T>(a, a.dout, at.e, at.s, head) + row * a.o_row), o_stride, at.e.nq - row, row_bytes, wave, lane);
            if (wave / 2 == i % 2) request_floats<32>(stat[turn][i][wave & 1], (wave & 1 ? a.stat_delta : a.stat_lse) + head * a.rows + at.e.lse0 + row, at.e.nq - row, lane);
        }
    };
    request(first, 0);
    for (int t = first, turn = 0; t < last; t += kTiles, turn ^= 1) {
        tiles_arrived();
        request(t + kTiles, turn ^ 1);
        const int mine = t + part;
        if (kTiles > 1 && mine >= last) continue;
        const float slope = MOD && a.slopes ? a.slopes[at.kv * a.group + mine / tiles] * kLog2e : 0.f;
        const int row = at.any_lo + mine % tiles * 32;
        if (!keys.sees(row)) continue;
        int l = lane;  // (places in LDS made anew in every tile: kept, they would not fit the registers)
        asm volatile("" : "+v"(l));
        keys.template add<false>(lds[turn][part][0], lds[turn][part][1], stat[turn][part][0], stat[turn][part][1], row, slope, l,
                 [&](int c) { if constexpr (kKeepV) return vf[c]; else return Values::row_operand(values, 32 * key_wave, c, l); });
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // (where there were no rows v may still be under way to LDS)
    constexpr int kPart = 8 * Keys::DB * 64;  // pieces of 16 bytes of a wave's sums
    if constexpr (KW < kWaves) {
        static_assert(kTiles == 2 && KW * kPart * 16 <= (int)sizeof lds);
        __syncthreads();
        floatx4 *other = (floatx4 *)lds + key_wave * kPart + lane;
        if (part) keys.pieces([&](int i, floatx4 y) { other[i * 64] = y; });
        __syncthreads();
        if (part) return;
        keys.join([&](int i) { return other[i * 64]; });
    }
    if (at.pieces > 1) {
        // parts of dk and dv as they lie in the registers: [part][workgroup][wave][piece][lane] of 16 bytes
        floatx4 *to = (floatx4 *)a.part_o + ((int64_t)blockIdx.x * KW + key_wave) * kPart + lane;
        keys.pieces([&](int i, floatx4 y) { to[i * 64] = y; });
        return;
    }
    if constexpr (sizeof(T) == 2 && KW == kWaves) __syncthreads();  // (the tiles have been read by all)
    char *mine = (char *)lds + key_wave * (KW == kWaves ? 64 * DP : kPart * 16);
    static_assert(sizeof(T) == 4 || kWaves * 64 * DP <= (int)sizeof lds);
    const int key0 = k0 + 32 * key_wave;
    store_turned<T, DP>(mine, keys.dk, a.scale, a.head_dim, lane,
                        [&](int r) { return key0 + r < at.e.nk ? (T *)k_base<T>(a, a.dk, at.e, at.s, at.kv) + (key0 + r) * a.k_row : nullptr; });
    store_turned<T, DP>(mine, keys.dv, 1.f, a.head_dim, lane,
                        [&](int r) { return key0 + r < at.e.nk ? (T *)v_base<T>(a, a.dv, at.e, at.s, at.kv) + (key0 + r) * a.v_row : nullptr; });
}

// The same where workgroups of 128 keys would leave most compute units without work: 32 keys to a workgroup, each wave on every NW-th tile of rows, in LDS of
// its own and without a barrier; sums are joined at the end.  fp32 heads of more than 64: one tile at a time, since a tile's products take eight
// times as long as its way to LDS, and v in LDS.  300 tokens, 16 heads over 4 of 128, bf16 24 us, fp32 31: latency of loads and of chains of products.
template <class T, int DP, bool MOD, int NW>
__global__ __launch_bounds__(64 * NW, 1)
void sddmm_attention_dkv_few_kernel(const AttnArgs a)
{
    typedef DkvKeys<T, DP, MOD> Keys;
    typedef typename Keys::Rows Rows;
    typedef typename Elem<T>::Vec8 Vec8;
    constexpr int kLoads = 2 * Rows::kBytes / 1024 + 2;
    constexpr bool kLarge = sizeof(T) == 4 && DP == 128;
    constexpr int kTurns = kLarge ? 1 : 2;
    __shared__ __align__(1024) char lds[NW][kTurns][2][Rows::kBytes];
    __shared__ __align__(1024) char values[kLarge ? Rows::kBytes : 16];
    __shared__ __align__(16) float stat[NW][kTurns][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
    KeyTile at;
    const int groups = gridDim.x / a.n_split, split = blockIdx.x / groups;
    if (!key_tile<kFewKeys>(a, blockIdx.x - split * groups, at) || split >= at.pieces) return;
    const int row_bytes = a.head_dim * (int)sizeof(T), k0 = at.tile * kFewKeys;
    const int tiles = at.any_hi > at.any_lo ? (at.any_hi - at.any_lo + 31) / 32 : 0, all = tiles * a.group;
    const int each = (all + at.pieces - 1) / at.pieces, first = split * each, last = min(all, first + each);
    const uint32_t q_stride = (uint32_t)(a.q_row * sizeof(T)), o_stride = (uint32_t)(a.o_row * sizeof(T));
    // (behind the last tile nothing is read, but the requests are made, so that the waits count the same)
    auto request = [&](int t, int turn) {
        const bool more = t < last;
        const int head = more ? at.kv * a.group + t / tiles : 0, row = more ? at.any_lo + t % tiles * 32 : 0, valid = more ? at.e.nq - row : 0;
        const int64_t stats = head * a.rows + at.e.lse0 + row;
        Rows::template request<1>(lds[wave][turn][0], (const char *)(q_base<T>(a, a.q, at.e, at.s, head) + row * a.q_row), q_stride, valid, row_bytes, 0, lane);
        Rows::template request<1>(lds[wave][turn][1], (const char *)(o_base<T>(a, a.dout, at.e, at.s, head) + row * a.o_row), o_stride, valid, row_bytes, 0, lane);
        request_floats<32>(stat[wave][turn][0], a.stat_lse + stats, valid, lane);
        request_floats<32>(stat[wave][turn][1], a.stat_delta + stats, valid, lane);
    };
    request(first + wave, 0);
    Keys keys;
    keys.init(a, at, k0, lane);
    Vec8 vf[kLarge ? 1 : DP / 16];
    const T *v = v_base<T>(a, a.v, at.e, at.s, at.kv);
    if constexpr (kLarge) {
        Rows::template request<NW>(values, (const char *)(v + k0 * a.v_row), (uint32_t)(a.v_row * sizeof(T)), at.e.nk - k0, row_bytes, wave, lane);
        tiles_arrived();
    } else {
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) vf[c] = global_operand<T>(v + keys.key * a.v_row, keys.there, 16 * c + 8 * h, a.head_dim);
        __builtin_amdgcn_s_waitcnt(0x0f70);  // the first tile and the keys: from here on only tiles are under way
    }
    for (int t = first + wave, turn = 0; t < last; t += NW, turn = (turn + 1) % kTurns) {
        if constexpr (!kLarge) request(t + NW, turn ^ 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLarge ? 0 : kLoads) : "memory");
        const float slope = MOD && a.slopes ? a.slopes[at.kv * a.group + t / tiles] * kLog2e : 0.f;
        const int row = at.any_lo + t % tiles * 32;
        if (keys.sees(row)) {
            keys.template add<true>(lds[wave][turn][0], lds[wave][turn][1], stat[wave][turn][0], stat[wave][turn][1], row, slope, lane,
                     [&](int c) { if constexpr (kLarge) return Rows::row_operand(values, 0, c, lane); else return vf[c]; });
#pragma unroll
            for (int d = 0; d < Keys::DB; ++d) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(keys.dk[d]), "+v"(keys.dv[d]) :: "memory");
        }
        if constexpr (kLarge) request(t + NW, 0);
    }
    // join the waves: [piece][lane] of 16 bytes for each
    static_assert(2 * kTurns * Rows::kBytes >= 256 * DP);
    __builtin_amdgcn_s_waitcnt(0x0070);
    floatx4 *mine = (floatx4 *)lds[wave][0][0];
    keys.pieces([&](int i, floatx4 y) { mine[i * 64 + lane] = y; });
    __syncthreads();
    floatx4 *part = (floatx4 *)a.part_o + (int64_t)blockIdx.x * (8 * Keys::DB * 64) + lane;
#pragma unroll
    for (int j = 0; j < 8 * Keys::DB / NW; ++j) {
        const int i = wave * (8 * Keys::DB / NW) + j;
        floatx4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) y += ((const floatx4 *)lds[w][0][0])[i * 64 + lane];
        if (at.pieces > 1) part[i * 64] = y;
        else if (keys.there) Keys::store(a, at, k0 + n, i, h, y);
    }
}

// The slopes' gradients: a head's parts in a fixed order.  A kernel of their own, or further workgroups of the one below, whose launch they then share.
__device__ __forceinline__ void sum_slopes(const AttnArgs &a, int head)
{
    __shared__ double sums[256];
    double x = 0.;
    for (int p = threadIdx.x; p < a.slope_parts; p += 256) x += a.slope_part[(int64_t)head * a.slope_parts + p];
    sums[threadIdx.x] = x;
    __syncthreads();
    for (int d = 128; d > 0; d /= 2) {
        if ((int)threadIdx.x < d) sums[threadIdx.x] += sums[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.dslopes[head] = (float)sums[0];
}
__global__ __launch_bounds__(256)
void sddmm_attention_dslopes_kernel(const AttnArgs a) { sum_slopes(a, blockIdx.x); }

// The sum of the parts of dk and dv of the keys whose rows were cut: pieces of four elements, one to a thread where there are few keys (us, 148 tokens, 16
// heads over 2 of 96, fp32 9 with eight and 5 with one), two where there are many, whose workgroups would spend their time on finding their sequence.
template <int KEYS> constexpr int kSumPieces = KEYS == kFewKeys ? 1 : 2;
template <class T, int DP, int KEYS>
__global__ __launch_bounds__(256)
void sddmm_attention_dkv_sum_kernel(const AttnArgs a, const int n_sum)
{
    typedef DkvKeys<T, DP, false> Keys;
    if ((int)blockIdx.x >= n_sum) {
        sum_slopes(a, blockIdx.x - n_sum);
        return;
    }
    constexpr int kEach = 2 * Keys::DB / kSumPieces<KEYS>;  // workgroups to 32 keys
    KeyTile at;
    const int unit = blockIdx.x / kEach;
    if (!key_tile<KEYS>(a, unit / (KEYS / 32), at) || at.pieces == 1) return;
    const int lane = threadIdx.x & 63, key = at.tile * KEYS + unit % (KEYS / 32) * 32 + (lane & 31), i0 = blockIdx.x % kEach * 4 + (threadIdx.x >> 6);
    if (key >= at.e.nk) return;
    const int64_t part = (int64_t)(n_sum / kEach) * (8 * Keys::DB * 64);
    const floatx4 *from = (const floatx4 *)a.part_o + (int64_t)unit * (8 * Keys::DB * 64) + lane;
    floatx4 x[kSumPieces<KEYS>] = {};
#pragma unroll 8 / kSumPieces<KEYS>
    for (int p = 0; p < at.pieces; ++p)
#pragma unroll
        for (int j = 0; j < kSumPieces<KEYS>; ++j) x[j] += from[p * part + (i0 + 4 * kEach * j) * 64];
#pragma unroll
    for (int j = 0; j < kSumPieces<KEYS>; ++j) Keys::store(a, at, key, i0 + 4 * kEach * j, lane >> 5, x[j]);
}

// dq.  A wave holds 32 rows: q and do as operands, the sums of dq turned.  Per tile of 32 keys in LDS: S^T = K Q^T, dP^T = V dO^T, then
// dQ^T += K^T dS^T.
//
// The gradient of a head's slope, - sum ds |p_i - j|, is asked to fp32 whatever the operands' type, and delta, which comes from the rounded
// output, would put an error of every row times its mean distance into it.  So it is made of sums that need no delta:
// with far = |p_i - j|, - sum_i (sum_j p dp far - (sum_j p dp) (sum_j p far) / sum_j p).
template <class T, int DP, bool MOD>
struct DqRows {
    static constexpr int DB = DP / 32;
    typedef typename Elem<T>::Vec8 Vec8;
    Vec8 qf[DP / 16], of[DP / 16];
    floatx16 dq[DB];
    float lse, delta, unit, slope;
    Bend<T> bend;
    bool bias, slopes_too, there;
    int pos, lo, hi, h;
    double far_ds, far_p, sum_ds, sum_p;

    __device__ __forceinline__ void init(const AttnArgs &a, const Seq &e, int s, int head, int row, int prefix, bool want_slopes, bool write_stats, int lane)
    {
        h = lane >> 5;
        there = row < e.nq;
        pos = row + e.nk - e.nq, lo = first_key(a, pos), hi = there ? end_key(a, pos, prefix, e.nk) : 0;
        const T *q = q_base<T>(a, a.q, e, s, head) + row * a.q_row, *dout = o_base<T>(a, a.dout, e, s, head) + row * a.o_row;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) qf[c] = global_operand<T>(q, there, 16 * c + 8 * h, a.head_dim);
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) of[c] = global_operand<T>(dout, there, 16 * c + 8 * h, a.head_dim);
        const T *out = o_base<T>(a, a.out, e, s, head) + row * a.o_row;
        delta = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
            const floatx8 x = __builtin_convertvector(of[c], floatx8), y = __builtin_convertvector(global_operand<T>(out, there, 16 * c + 8 * h, a.head_dim), floatx8);
#pragma unroll
            for (int j = 0; j < 8; ++j) delta = fmaf(x[j], y[j], delta);
        }
        delta = halves_sum(delta);
        // (a row that saw nothing gets +infinity, so that 2^(s - lse) is 0)
        const float m = there ? a.lse[(e.lse0 + row) * a.n_heads + head] : -INFINITY;
        lse = m == -INFINITY ? INFINITY : m * kLog2e;
        if (there && h == 0 && write_stats) {
            const int64_t at = (int64_t)head * a.rows + e.lse0 + row;
            a.stat_lse[at] = lse, a.stat_delta[at] = -delta;
        }
#pragma unroll
        for (int d = 0; d < DB; ++d) dq[d] = zero16();
        unit = a.scale * kLog2e;
        if constexpr (MOD) bend.init(a.scale, a.cap);
        bias = MOD && a.slopes, slope = bias ? a.slopes[head] * kLog2e : 0.f;
        slopes_too = MOD && want_slopes;
        far_ds = far_p = sum_ds = sum_p = 0.;
    }
    template <class Keys> __device__ __forceinline__ floatx16 product(const char *tile, int block, const Vec8 (&f)[DP / 16], int lane) const
    {
        floatx16 x = zero16();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) x = Elem<T>::mma(Keys::row_operand(tile, block, c, lane), f[c], x);
        return x;
    }
    // from the products with k and v of the 32 keys from `key` on to the gradients of their scores, in y
    __device__ __forceinline__ void gradients(floatx16 &x, floatx16 &y, int key, bool masked)
    {
        floatx16 back;
        const float away = (float)(pos - key - 4 * h);
        scores<MOD, T>(x, back, bend, unit, bias, slope, away, -1.f);
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = __builtin_amdgcn_exp2f(x[r] - lse);
        if (masked) {
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
            if (slopes_too) {
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
    }
    template <class Keys> __device__ __forceinline__ void add(const char *kt, int block, const floatx16 &y, int lane)
    {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const Vec8 ds = operand<T>(y, c);
#pragma unroll
            for (int d = 0; d < DB; ++d) dq[d] = Elem<T>::mma(Keys::column_operand(kt, d, block / 16 + c, lane), ds, dq[d]);
        }
    }
    // both halves of the wave hold parts of the rows' sums
    __device__ __forceinline__ void join_halves()
    {
        if constexpr (!MOD) return;
        far_ds += __shfl_xor(far_ds, 32), far_p += __shfl_xor(far_p, 32), sum_ds += __shfl_xor(sum_ds, 32), sum_p += __shfl_xor(sum_p, 32);
    }
    static __device__ __forceinline__ double of_slope(double far_ds, double far_p, double sum_ds, double sum_p)
    {
        double g = sum_p > 0. || sum_p != sum_p ? sum_ds * far_p / sum_p - far_ds : 0.;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) g += __shfl_xor(g, d);
        return g;
    }
};

template <class T>
__device__ __forceinline__ void store_dq(const AttnArgs &a, T *to, int col, floatx4 y)
{
    typedef typename Elem<T>::Vec4 Vec4;
    if (col < a.head_dim) *(Vec4 *)(to + col) = __builtin_convertvector(y * a.scale, Vec4);
}

// RW: as in the forward kernel.
template <class T, int DP, bool MOD, int RW>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 && DP == 128 ? 1 : 2)
void sddmm_attention_dq_kernel(const AttnArgs a)
{
    constexpr int KT = sizeof(T) == 2 || RW == 2 ? 64 : 32, KB = KT / 32 / (kWaves / RW), DB = DP / 32, kRows = 32 * RW;
    typedef Tile<T, DP, KT> Keys;
    __shared__ __align__(1024) char lds[2][2][Keys::kBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
    const int row_wave = wave % RW, half = wave / RW;

    int b = blockIdx.x, s = 0, tile;  // (as in the forward kernel)
    const int kv = b % a.n_kv_heads;
    b /= a.n_kv_heads;
    if (!a.q_ptr) { s = b % a.n_seq; b /= a.n_seq; }
    const int head = kv * a.group + b % a.group;
    b /= a.group;
    double *slope_part = MOD && a.slope_part ? a.slope_part + (int64_t)head * a.slope_parts + (a.q_ptr ? b : (int64_t)b * a.n_seq + s) : nullptr;
    if (slope_part && threadIdx.x == 0) *slope_part = 0.;
    if (a.q_ptr) {
        s = slot_sequence<false>(a.q_ptr, a.n_seq, 1, kRows, a.max_tiles, a.n_slots, b, tile);
        if (s < 0) return;
    } else {
        tile = a.n_slots - 1 - b;
    }
    const Seq e = sequence(a, s);
    if (tile * kRows >= e.nq) return;
    const int row = tile * kRows + row_wave * 32 + n, shift = e.nk - e.nq, prefix = a.prefix ? a.prefix[s] : 0;
    const int r1 = min(e.nq, tile * kRows + kRows) - 1, w0 = tile * kRows + row_wave * 32, w1 = min(e.nq, w0 + 32) - 1;
    const int any_lo = first_key(a, tile * kRows + shift), any_hi = end_key(a, r1 + shift, prefix, e.nk);
    const int wave_lo = first_key(a, w0 + shift), wave_hi = w1 < w0 ? 0 : end_key(a, w1 + shift, prefix, e.nk);
    const int full_lo = first_key(a, w1 + shift), full_hi = w1 < w0 + 31 ? 0 : end_key(a, w0 + shift, prefix, e.nk);
    DqRows<T, DP, MOD> rows;
    rows.init(a, e, s, head, row, prefix, slope_part != nullptr, half == 0, lane);
    const T *k = k_base<T>(a, a.k, e, s, kv), *v = v_base<T>(a, a.v, e, s, kv);

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
        for (int u = half * KB; u < half * KB + KB; ++u) {
            const int key = any_lo + t * KT + 32 * u;
            if (key + 32 <= wave_lo || key >= wave_hi) continue;
            int l = lane;  // (places in LDS made anew in every tile: kept, they would not fit the registers)
            asm volatile("" : "+v"(l));
            floatx16 x = rows.template product<Keys>(kt, 32 * u, rows.qf, l), y = rows.template product<Keys>(vt, 32 * u, rows.of, l);
            raise_priority<T, DP, MOD>();
            rows.gradients(x, y, key, key < full_lo || key + 32 > full_hi);
            if constexpr (MOD) lower_priority<T, DP, MOD>();
            rows.template add<Keys>(kt, 32 * u, y, l);
            if constexpr (!MOD) lower_priority<T, DP, MOD>();
        }
    }
    if constexpr (RW < kWaves) {  // the halves of the keys
        static_assert(RW * 128 * DP + RW * 1024 <= (int)sizeof lds);
        __syncthreads();
        floatx4 *other = (floatx4 *)((char *)lds + row_wave * 128 * DP);
        double *other_sums = (double *)((char *)lds + RW * 128 * DP) + row_wave * 128 + n * 4;
        rows.join_halves();
        if (half) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) other[(4 * d + i) * 64 + lane] = floatx4{rows.dq[d][4 * i], rows.dq[d][4 * i + 1], rows.dq[d][4 * i + 2], rows.dq[d][4 * i + 3]};
            if (MOD && h == 0) other_sums[0] = rows.far_ds, other_sums[1] = rows.far_p, other_sums[2] = rows.sum_ds, other_sums[3] = rows.sum_p;
        }
        __syncthreads();
        if (!half) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const floatx4 y = other[(4 * d + i) * 64 + lane];
#pragma unroll
                    for (int j = 0; j < 4; ++j) rows.dq[d][4 * i + j] += y[j];
                }
            if constexpr (MOD) rows.far_ds += other_sums[0], rows.far_p += other_sums[1], rows.sum_ds += other_sums[2], rows.sum_p += other_sums[3];
        }
    } else {
        rows.join_halves();
    }
    if (MOD && slope_part) {
        __shared__ double parts[kWaves];
        const double g = half ? 0. : rows.of_slope(rows.far_ds, rows.far_p, rows.sum_ds, rows.sum_p);
        if (lane == 0) parts[wave] = g;
        __syncthreads();
        if (threadIdx.x == 0) *slope_part = parts[0] + parts[1] + parts[2] + parts[3];
    }
    if (half) return;
    if constexpr (sizeof(T) == 2) {
        static_assert(RW * 128 * DP + RW * 1024 + RW * 64 * DP <= (int)sizeof lds || RW == kWaves);
        if constexpr (RW == kWaves) __syncthreads();  // (the tiles have been read by all)
    }
    const int row0 = tile * kRows + row_wave * 32;
    store_turned<T, DP>((char *)lds + (RW == kWaves ? 0 : RW * 128 * DP + RW * 1024) + row_wave * 64 * DP, rows.dq, a.scale, a.head_dim, lane,
                        [&](int r) { return row0 + r < e.nq ? (T *)q_base<T>(a, a.dq, e, s, head) + (row0 + r) * a.q_row : nullptr; });
}

// dq where workgroups of 128 rows would leave compute units without work: 32 rows to a workgroup, each wave on every NW-th tile of keys, in LDS of its
// own (keys twice, since they are needed to the end of a tile's work; not fp32 heads of more than 64, see above) and without a barrier; sums
// are joined at the end.  300 tokens, 16 heads over 4 of 128, bf16 11 us, fp32 30.
constexpr int kFewRows = 32;
template <class T, int DP, bool MOD, int NW>
__global__ __launch_bounds__(64 * NW, 1)
void sddmm_attention_dq_few_kernel(const AttnArgs a)
{
    constexpr int KT = 32, DB = DP / 32;
    typedef Tile<T, DP, KT> Keys;
    constexpr int kLoads = Keys::kBytes / 1024;
    constexpr bool kLarge = sizeof(T) == 4 && DP == 128;
    constexpr int kTurns = kLarge ? 1 : 2;
    __shared__ __align__(1024) char lds[NW][kTurns + 1][Keys::kBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
    int b = blockIdx.x, s = 0, tile;
    const int head = b % a.n_heads, kv = head / a.group;
    b /= a.n_heads;
    if (!a.q_ptr) { s = b % a.n_seq; b /= a.n_seq; }
    double *slope_part = MOD && a.slope_part ? a.slope_part + (int64_t)head * a.slope_parts + (a.q_ptr ? b : (int64_t)b * a.n_seq + s) : nullptr;
    if (slope_part && threadIdx.x == 0) *slope_part = 0.;
    if (a.q_ptr) {
        s = slot_sequence<false>(a.q_ptr, a.n_seq, 1, kFewRows, a.max_tiles, a.n_slots, b, tile);
        if (s < 0) return;
    } else {
        tile = a.n_slots - 1 - b;
    }
    const Seq e = sequence(a, s);
    if (tile * kFewRows >= e.nq) return;
    const int row = tile * kFewRows + n, shift = e.nk - e.nq, prefix = a.prefix ? a.prefix[s] : 0;
    const int w0 = tile * kFewRows, w1 = min(e.nq, w0 + kFewRows) - 1;
    const int any_lo = first_key(a, w0 + shift), any_hi = end_key(a, w1 + shift, prefix, e.nk);
    const int full_lo = first_key(a, w1 + shift), full_hi = w1 < w0 + 31 ? 0 : end_key(a, w0 + shift, prefix, e.nk);
    DqRows<T, DP, MOD> rows;
    rows.init(a, e, s, head, row, prefix, slope_part != nullptr, wave == 0, lane);
    const T *k = k_base<T>(a, a.k, e, s, kv), *v = v_base<T>(a, a.v, e, s, kv);

    const int last = any_hi > any_lo ? (any_hi - any_lo + KT - 1) / KT : 0;
    const int row_bytes = a.head_dim * (int)sizeof(T);
    const uint32_t k_stride = (uint32_t)(a.k_row * sizeof(T)), v_stride = (uint32_t)(a.v_row * sizeof(T));
    // (behind the last tile nothing is read, but the requests are made, so that the waits count the same)
    auto request = [&](char *to, const T *base, int64_t step, uint32_t stride, int t) {
        const int key = any_lo + t * KT;
        const bool more = t < last;
        Keys::template request<1>(to, (const char *)(base + (more ? key : 0) * step), stride, more ? e.nk - key : 0, row_bytes, 0, lane);
    };
    char *vt = lds[wave][kTurns];
    __builtin_amdgcn_s_waitcnt(0x0f70);  // the rows: from here on only tiles are under way
    request(lds[wave][0], k, a.k_row, k_stride, wave);
    request(vt, v, a.v_row, v_stride, wave);
    for (int t = wave, turn = 0; t < last; t += NW, turn = (turn + 1) % kTurns) {
        const int key = any_lo + t * KT;
        const char *kt = lds[wave][turn];
        if constexpr (!kLarge) request(lds[wave][turn ^ 1], k, a.k_row, k_stride, t + NW);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLarge ? 0 : 2 * kLoads) : "memory");
        floatx16 x = rows.template product<Keys>(kt, 0, rows.qf, lane);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLarge ? 0 : kLoads) : "memory");
        floatx16 y = rows.template product<Keys>(vt, 0, rows.of, lane);
        asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(x), "+v"(y) :: "memory");  // (all of the values have been read)
        request(vt, v, a.v_row, v_stride, t + NW);
        rows.gradients(x, y, key, key < full_lo || key + 32 > full_hi);
        rows.template add<Keys>(kt, 0, y, lane);
#pragma unroll
        for (int d = 0; d < DB; ++d) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(rows.dq[d]) :: "memory");
        if constexpr (kLarge) request(lds[wave][0], k, a.k_row, k_stride, t + NW);
    }
    // join the waves: [element of the lane / 4][lane] of 16 bytes for each wave
    static_assert((kTurns + 1) * Keys::kBytes >= 128 * DP);
    __builtin_amdgcn_s_waitcnt(0x0070);
    floatx4 *mine = (floatx4 *)lds[wave][0];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[(4 * d + i) * 64 + lane] = floatx4{rows.dq[d][4 * i], rows.dq[d][4 * i + 1], rows.dq[d][4 * i + 2], rows.dq[d][4 * i + 3]};
    if (MOD && slope_part) {
        __shared__ double sums[NW][32][4];
        rows.join_halves();
        if (h == 0) sums[wave][n][0] = rows.far_ds, sums[wave][n][1] = rows.far_p, sums[wave][n][2] = rows.sum_ds, sums[wave][n][3] = rows.sum_p;
        __syncthreads();
        if (wave == 0) {
            double y[4] = {0., 0., 0., 0.};
            for (int w = 0; w < NW; ++w)
                for (int i = 0; i < 4; ++i) y[i] += sums[w][n][i];
            const double g = rows.of_slope(y[0], y[1], y[2], y[3]);
            if (lane == 0) *slope_part = g;
        }
    }
    __syncthreads();
    if (!rows.there) return;
    T *to = (T *)q_base<T>(a, a.dq, e, s, head) + row * a.q_row;
#pragma unroll
    for (int piece = wave; piece < 4 * DB; piece += NW) {
        floatx4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) y += ((const floatx4 *)lds[i][0])[piece * 64 + lane];
        store_dq(a, to, 8 * piece + 4 * h, y);
    }
}

template <class T, int DP>
hipError_t launch_typed(const AttnArgs &a, const AttnArgs &b, unsigned kv_grid, int keys, unsigned q_grid, int q_rows, hipStream_t st)
{
    const bool mod = a.cap > 0.f || a.slopes;
    // Waves of the kernels for few: 4, which share a compute unit with another workgroup's, or 8 where that is not to be had anyway and their tiles fit: 16-bit
    // heads up to 64 (us of forward and backward, causal, bf16, heads of 64, with 4 and 8: 1000 tokens, 8 heads over 2 55 and 48; 1013 in 2, 4 over 2, capped and
    // biased 46 and 39; but 8 sequences of 512, 8 heads, which fill the card, 50 and 61), and dq of fp32 heads up to 32 (the second of these 72 and 66; with
    // dk and dv as well 73, and 1000 tokens, 8 over 2 86 and 96).
    constexpr int kMore = sizeof(T) == 2 && DP == 64 ? 8 : 4, kMoreQ = sizeof(T) * DP <= 128 ? 8 : 4;
    constexpr unsigned kUnits = 512;  // (workgroups that can be there together)
    const int kv_waves = kv_grid <= kUnits ? kMore : 4, q_waves = q_grid <= kUnits ? kMoreQ : 4;
    const auto dkv_few = kv_waves == 4 ? (mod ? sddmm_attention_dkv_few_kernel<T, DP, true, 4> : sddmm_attention_dkv_few_kernel<T, DP, false, 4>)
                                       : (mod ? sddmm_attention_dkv_few_kernel<T, DP, true, kMore> : sddmm_attention_dkv_few_kernel<T, DP, false, kMore>);
    const auto dq_few = q_waves == 4 ? (mod ? sddmm_attention_dq_few_kernel<T, DP, true, 4> : sddmm_attention_dq_few_kernel<T, DP, false, 4>)
                                     : (mod ? sddmm_attention_dq_few_kernel<T, DP, true, kMoreQ> : sddmm_attention_dq_few_kernel<T, DP, false, kMoreQ>);
    auto dkv = mod ? sddmm_attention_dkv_kernel<T, DP, true, 4> : sddmm_attention_dkv_kernel<T, DP, false, 4>;
    auto sum = keys == kFewKeys ? sddmm_attention_dkv_sum_kernel<T, DP, kFewKeys> : sddmm_attention_dkv_sum_kernel<T, DP, 128>;
    if constexpr (DP <= 64) {
        if (keys == 64) dkv = mod ? sddmm_attention_dkv_kernel<T, DP, true, 2> : sddmm_attention_dkv_kernel<T, DP, false, 2>, sum = sddmm_attention_dkv_sum_kernel<T, DP, 64>;
    }
    const auto dq = q_rows == 64 ? (mod ? sddmm_attention_dq_kernel<T, DP, true, 2> : sddmm_attention_dq_kernel<T, DP, false, 2>)
                                 : (mod ? sddmm_attention_dq_kernel<T, DP, true, 4> : sddmm_attention_dq_kernel<T, DP, false, 4>);
    hipError_t e = hipSuccess;
    if (q_grid) e = q_rows == kFewRows ? launch(dq_few, dim3(q_grid), dim3(64 * q_waves), 0, st, b) : launch(dq, dim3(q_grid), dim3(64 * kWaves), 0, st, b);
    if (e == hipSuccess && kv_grid) e = keys == kFewKeys ? launch(dkv_few, dim3(kv_grid), dim3(64 * kv_waves), 0, st, a) : launch(dkv, dim3(kv_grid), dim3(64 * kWaves), 0, st, a);
    const unsigned n_slopes = a.dslopes ? a.n_heads : 0, n_sum = (unsigned)attention_sum_grid(kv_grid, a.n_split, keys, DP, 0);
    if (e == hipSuccess && n_sum) e = launch(sum, dim3(n_sum + n_slopes), dim3(256), 0, st, a, (int)n_sum);
    else if (e == hipSuccess && n_slopes) e = launch(sddmm_attention_dslopes_kernel, dim3(n_slopes), dim3(256), 0, st, a);
    return e;
}

template <class T>
hipError_t launch_dims(const AttnArgs &a, const AttnArgs &b, unsigned kv_grid, int keys, unsigned q_grid, int q_rows, hipStream_t st)
{
    if constexpr (sizeof(T) == 4) {
        if (a.head_dim <= 32) return launch_typed<T, 32>(a, b, kv_grid, keys, q_grid, q_rows, st);
    }
    return a.head_dim <= 64 ? launch_typed<T, 64>(a, b, kv_grid, keys, q_grid, q_rows, st) : launch_typed<T, 128>(a, b, kv_grid, keys, q_grid, q_rows, st);
}

}  // namespace

int64_t attention_sum_grid(int64_t kv_grid, int splits, int keys, int padded_dim, int slope_heads)
{
    return (splits > 1 ? kv_grid / splits * (keys / 32) * (padded_dim / 16) / (keys == kFewKeys ? 1 : kSumPieces<128>) : 0) + slope_heads;
}

hipError_t launch_attention_backward(const AttnArgs &a, const AttnArgs &b, int type, unsigned kv_grid, int keys, unsigned q_grid, int q_rows, hipStream_t st)
{
    return type == SDDMM_TYPE_F32 ? launch_dims<float>(a, b, kv_grid, keys, q_grid, q_rows, st)
         : type == SDDMM_TYPE_F16 ? launch_dims<_Float16>(a, b, kv_grid, keys, q_grid, q_rows, st) : launch_dims<__bf16>(a, b, kv_grid, keys, q_grid, q_rows, st);
}

}  // namespace sddmm
