// Dense attention (gfx950): arguments of the kernels, and the pieces that they share -- fragments of the matrix
// instructions, tiles of rows in LDS, masks and scores.
//
// Every product is made of 32 x 32 x 16 matrix instructions (fp32: eight of 32 x 32 x 2).  A lane l of a wave holds, with
// n = l % 32 and h = l / 32:
//   operands   row (or column) n, elements 8 h + j of the 16 that are summed over, j = 0 .. 7
//   results    column n, rows 8 (i / 4) + 4 h + i % 4, i = 0 .. 15
// The order of summation is free as long as both operands agree, so the eight results i = 8 c .. 8 c + 7 of a lane, rounded to
// the element type, are an operand of the next product as they are: its sum then runs over 16 c + 8 (j / 4) + 4 h + j % 4,
// which is how `column_operand` reads the other operand.  Probabilities and their gradients never leave the registers.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>
#include "../../include/sddmm.h"
#include "attention_intervals.hpp"
#include "bf16_parts.hpp"

namespace sddmm {

// One call, as the kernels see it (strides in elements).
struct AttnArgs {
    const void *q, *k, *v;
    void *out;                  // forward: written; backward: read
    float *lse;                 // [rows][n_heads] or null; backward: read
    const void *shared_k, *shared_v;
    const void *dout;
    void *dq, *dk, *dv;
    float *part_o;              // partial results of split keys: [part][row of all heads][head_dim]
    float2 *part_ml;            // [part][row of all heads]: maximum (in powers of two) and sum
    float *stat_lse, *stat_delta;  // backward: [n_heads][all rows] log-sum-exp in powers of two, - sum of dout * out
    double *slope_part;         // backward: [n_heads][slope_parts] parts of the slopes' gradients, or null
    float *dslopes;
    int64_t q_seq, q_row, q_head, k_seq, k_row, k_head, v_seq, v_row, v_head, o_seq, o_row, o_head;
    const int32_t *q_ptr, *k_ptr, *q_len, *k_len, *prefix;
    const float *slopes;
    int64_t rows, key_rows;     // rows and keys of all sequences (of q_ptr, k_ptr: at most)
    int32_t head_dim, n_heads, n_kv_heads, group, n_seq, max_q, max_k, left, right, shared_len;
    int32_t n_slots;            // tiles of rows (or keys) that the grid holds
    int32_t max_tiles;          // tiles of a sequence at most
    int32_t n_split;            // pieces that the keys of a tile of rows are cut into
    int32_t part0, n_part;      // first piece of this launch, pieces in all
    int32_t slope_parts;
    int32_t chunk;              // backward: rows (of all query heads) that a workgroup of keys walks, more being cut into pieces
    float scale, cap;
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

template <class T> struct Elem;
template <> struct Elem<__bf16> {
    typedef bf16x8 Vec8;
    typedef bf16x4 Vec4;
    static __device__ __forceinline__ floatx16 mma(Vec8 a, Vec8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<_Float16> {
    typedef half8 Vec8;
    typedef half4 Vec4;
    static __device__ __forceinline__ floatx16 mma(Vec8 a, Vec8 b, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<float> {
    typedef floatx8 Vec8;
    typedef floatx4 Vec4;
    static __device__ __forceinline__ floatx16 mma(Vec8 a, Vec8 b, floatx16 c)
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

__device__ __forceinline__ floatx16 zero16()
{
    return floatx16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}

// results 8 c .. 8 c + 7 as an operand, rounded to the element type
template <class T>
__device__ __forceinline__ typename Elem<T>::Vec8 operand(const floatx16 &r, int c)
{
    floatx8 x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = r[8 * c + j];
    return __builtin_convertvector(x, typename Elem<T>::Vec8);
}

// the two halves of a wave hold parts of the same column: both get the maximum / the sum
__device__ __forceinline__ float halves_max(float x)
{
    const uint2v r = __builtin_bit_cast(uint2v, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float halves_sum(float x)
{
    const uint2v r = __builtin_bit_cast(uint2v, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}

// A tile of R rows of DP elements in LDS.  A row's 16-byte pieces are exchanged among themselves by its number so that both
// ways of reading are free of bank conflicts: 16 rows at one piece (`row_operand`), and 4 rows at 64 consecutive bytes (`column_operand`).
template <class T, int DP, int R>
struct Tile {
    static constexpr int kRowBytes = DP * (int)sizeof(T);
    static constexpr int kBytes = R * kRowBytes;
    static constexpr int kPieces = kRowBytes / 16;
    static_assert(kRowBytes == 128 || kRowBytes == 256 || kRowBytes == 512);

    static __device__ __forceinline__ int turn(int row)
    {
        return kRowBytes == 128 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
    }

    // Requests the tile: rows 0 .. R - 1 at `base`, `stride` bytes apart, of which `valid` exist and have `bytes` bytes; all
    // else becomes 0.  NW waves share the work; what arrives goes straight to LDS.
    template <int NW>
    static __device__ __forceinline__ void request(char *lds, const char *base, uint32_t stride, int valid, int bytes, int wave, int lane)
    {
        const uint32_t range = valid > 0 ? (uint32_t)(min(valid, R) - 1) * stride + (uint32_t)bytes : 0u;
        uint4v src = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)base),
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)((uintptr_t)base >> 32) & 0xffffu)),
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)range), 0x00020000u};
        uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds);
        asm volatile("s_nop 4" : "+s"(src), "+s"(to));  // (scalars that a vector instruction wrote, before a load reads them)
        constexpr int kSteps = kBytes / 1024 / NW;
        static_assert(kSteps * NW * 1024 == kBytes);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int at = (i * NW + wave) * 1024;
            const int pos = at + lane * 16, row = pos / kRowBytes, piece = (pos % kRowBytes / 16) ^ turn(row);
            const uint32_t off = piece * 16 < bytes ? (uint32_t)row * stride + (uint32_t)piece * 16 : 0x7ffffff0u;
            // (not the builtin: behind it the compiler waits for all loads before it reads LDS in the transposing way.  It keeps
            // nothing in m0 by itself, and nothing else in these kernels needs that register.)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to + at), "v"(off), "s"(src) : "memory");
        }
    }

    // elements 16 c + 8 h + j of row block + n
    static __device__ __forceinline__ typename Elem<T>::Vec8 row_operand(const char *lds, int block, int c, int lane)
    {
        const int row = block + (lane & 31), h = lane >> 5;
        const char *p = lds + row * kRowBytes;
        if constexpr (sizeof(T) == 2) {
            return *(const typename Elem<T>::Vec8 *)(p + (((2 * c + h) ^ turn(row)) << 4));
        } else {
            const floatx4 a = *(const floatx4 *)(p + (((4 * c + 2 * h) ^ turn(row)) << 4));
            const floatx4 b = *(const floatx4 *)(p + (((4 * c + 2 * h + 1) ^ turn(row)) << 4));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }

    // element 32 d + n of the rows 16 c + 8 (j / 4) + 4 h + j % 4 (a transposing read: 16 lanes take 4 rows of 16 elements)
    static __device__ __forceinline__ typename Elem<T>::Vec8 column_operand(const char *lds, int d, int c, int lane)
    {
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            const int i = lane & 15, piece = 4 * d + ((lane >> 3) & 2) + ((i >> 1) & 1);
            short4v r[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int row = 16 * c + 8 * k + 4 * h + (i >> 2);
                r[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) short4v *)(lds + row * kRowBytes + ((piece ^ turn(row)) << 4) + (i & 1) * 8));
            }
            typedef short short8 __attribute__((ext_vector_type(8)));
            const short8 s = __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(typename Elem<T>::Vec8, s);
        } else {
            floatx8 x;
            const int col = 32 * d + (lane & 31);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = 16 * c + 8 * (j >> 2) + 4 * h + (j & 3);
                x[j] = *(const float *)(lds + row * kRowBytes + (((col >> 2) ^ turn(row)) << 4) + (col & 3) * 4);
            }
            return x;
        }
    }
};

// Stores 32 rows of results that a wave holds turned (o[d] of lane (n, h): row n, columns 32 d + 8 (i / 4) + 4 h + i % 4), times `by` of the row:
// to(r) gives row r's place, or null.  16-bit results go through LDS (`mine`: 32 rows of the wave's own), so that whole lines are
// written instead of 16 bytes of each of 32 rows at a time (16 heads of 128, one key a row, 8192 rows 30.8 and 27.8 us, 65,536 rows 202 and 162).
template <class T, int DP, class F>
__device__ __forceinline__ void store_turned(char *mine, const floatx16 (&o)[DP / 32], float by, int dim, int lane, F to)
{
    typedef typename Elem<T>::Vec4 Vec4;
    const int n = lane & 31, h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        typedef Tile<T, DP, 32> Rows;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(Vec4 *)(mine + n * Rows::kRowBytes + (((4 * d + i) ^ Rows::turn(n)) << 4) + 8 * h) =
                    __builtin_convertvector((floatx4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * by), Vec4);
        asm volatile("" ::: "memory");
        constexpr int kPer = 64 / Rows::kPieces;
#pragma unroll
        for (int j = 0; j < 32 / kPer; ++j) {
            const int r = j * kPer + lane / Rows::kPieces, piece = lane % Rows::kPieces;
            T *row = to(r);
            if (row && 8 * piece < dim) *(uint4v *)(row + 8 * piece) = *(const uint4v *)(mine + r * Rows::kRowBytes + ((piece ^ Rows::turn(r)) << 4));
        }
    } else {
        T *row = to(n);
        if (!row) return;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = 32 * d + 8 * i + 4 * h;
                if (col < dim) *(floatx4 *)(row + col) = floatx4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * by;
            }
    }
}

// Requests R floats at `base`, of which `valid` exist (all else becomes 0), by one wave.
template <int R>
__device__ __forceinline__ void request_floats(float *lds, const float *base, int valid, int lane)
{
    static_assert(R <= 64);
    uint4v src = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)base),
                  (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)((uintptr_t)base >> 32) & 0xffffu)),
                  (uint32_t)__builtin_amdgcn_readfirstlane(max(0, min(valid, R)) * 4), 0x00020000u};
    uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)(char *)lds);
    const uint32_t off = lane * 4;
    asm volatile("s_nop 4" : "+s"(src), "+s"(to));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(off), "s"(src) : "memory");
}

// All requested tiles have arrived, for every wave, and no wave reads the other buffer any more.
__device__ __forceinline__ void tiles_arrived()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0), in a form that the compiler counts
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Eight elements of a row in global memory, 0 behind its end.
template <class T>
__device__ __forceinline__ typename Elem<T>::Vec8 global_operand(const T *row, bool there, int at, int dim)
{
    typename Elem<T>::Vec8 x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (T)0.f;
    if (there && at < dim) x = *(const typename Elem<T>::Vec8 *)(row + at);
    return x;
}

// A sequence: where its rows and keys begin and how many there are.  Lengths and places from the device are held to their bounds.
struct Seq {
    int64_t q0, k0;  // first row and key, in rows of q_row and k_row (0 where sequences have strides of their own)
    int64_t lse0;    // first row in lse
    int32_t nq, nk;
};
__device__ __forceinline__ Seq sequence(const AttnArgs &a, int s)
{
    Seq r;
    if (a.q_ptr) {
        const int first = min(max(0, a.q_ptr[s]), (int)a.rows);
        r.q0 = r.lse0 = first;
        r.nq = min(max(0, min(a.q_ptr[s + 1], (int)a.rows) - first), a.max_q);
    } else {
        r.q0 = 0;
        r.lse0 = (int64_t)s * a.max_q;
        r.nq = a.q_len ? min(max(0, a.q_len[s]), a.max_q) : a.max_q;
    }
    if (a.k_ptr) {
        const int first = min(max(0, a.k_ptr[s]), (int)a.key_rows);
        r.k0 = first;
        r.nk = min(max(0, min(a.k_ptr[s + 1], (int)a.key_rows) - first), a.max_k);
    } else {
        r.k0 = 0;
        r.nk = a.k_len ? min(max(0, a.k_len[s]), a.max_k) : a.max_k;
    }
    return r;
}
template <class T> __device__ __forceinline__ const T *q_base(const AttnArgs &a, const void *q, const Seq &e, int s, int head)
{
    return (const T *)q + (a.q_ptr ? e.q0 * a.q_row : s * a.q_seq) + head * a.q_head;
}
template <class T> __device__ __forceinline__ const T *o_base(const AttnArgs &a, const void *o, const Seq &e, int s, int head)
{
    return (const T *)o + (a.q_ptr ? e.q0 * a.o_row : s * a.o_seq) + head * a.o_head;
}
template <class T> __device__ __forceinline__ const T *k_base(const AttnArgs &a, const void *k, const Seq &e, int s, int kv)
{
    return (const T *)k + (a.k_ptr ? e.k0 * a.k_row : s * a.k_seq) + kv * a.k_head;
}
template <class T> __device__ __forceinline__ const T *v_base(const AttnArgs &a, const void *v, const Seq &e, int s, int kv)
{
    return (const T *)v + (a.k_ptr ? e.k0 * a.v_row : s * a.v_seq) + kv * a.v_head;
}

// Tiles of `size` rows of packed sequences (of `per` pairs for each row): sequence s takes the slots from ptr[s] * per / size + s on, which
// is at least as many as it needs, so that no count of all tiles has to be known beforehand.
//
// Up to 64 sequences of up to 64 tiles: the slots go to the tiles of all sequences in the order of their distance from their sequence's
// first one, the farthest first (LAST: from the last one).  Under a causal mask that is the order of their work, so that no long tile starts when
// the others are done (13 documents, 8192 tokens, 16 heads of 128: forward 82 and 73, dq 132 and 112 us).  Returns -1 for a slot that is none.
template <bool LAST>
__device__ __forceinline__ int slot_sequence(const int32_t *ptr, int n_seq, int per, int size, int max_tiles, int n_slots, int slot, int &tile)
{
    if (n_seq <= 64 && max_tiles <= 64) {
        const int lane = threadIdx.x & 63;
        int tiles = 0;
        if (lane < n_seq) tiles = (int)min((max((int64_t)0, (int64_t)ptr[lane + 1] - ptr[lane]) * per + size - 1) / size, (int64_t)max_tiles);
        for (int r = max_tiles - 1; r >= 0; --r) {
            uint64_t some = __ballot(tiles > r);
            const int n = __builtin_popcountll(some);
            if (slot < n) {
                for (; slot > 0; --slot) some &= some - 1;
                const int s = __builtin_ctzll(some);
                tile = LAST ? __builtin_amdgcn_readlane(tiles, s) - 1 - r : r;
                return s;
            }
            slot -= n;
        }
        return -1;
    }
    if (!LAST) slot = n_slots - 1 - slot;
    int lo = 0, hi = n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)max(0, ptr[mid]) * per / size + mid <= slot) lo = mid; else hi = mid;
    }
    tile = slot - (int)min((int64_t)max(0, ptr[lo]) * per / size + lo, (int64_t)INT32_MAX);
    return tile < 0 ? -1 : lo;
}

// (attention_intervals.hpp, of a call)
__device__ __forceinline__ int first_key(const AttnArgs &a, int pos) { return first_key(a.left, pos); }
__device__ __forceinline__ int end_key(const AttnArgs &a, int pos, int prefix, int n_keys) { return end_key(a.right, pos, prefix, n_keys); }
__device__ __forceinline__ int first_row(const AttnArgs &a, int j, int prefix, int shift) { return first_row(a.right, j, prefix, shift); }
__device__ __forceinline__ int end_row(const AttnArgs &a, int j, int shift, int n_rows) { return end_row(a.left, j, shift, n_rows); }

// The bound of scores: cap tanh(t / cap), t = scale * product, of N results in registers, in powers of two (BACK: and 1 - tanh^2 of each).
// Where all of the wave's |y|, y = t / cap, are 0.25 at most, which they mostly are, by powers of y^2 with everything else in their factors: six
// instructions, where 1 - 2 / (1 + e^2y) takes two of the slow kind and as many others, and to the last place, since that difference loses 24 bits
// below 1.  What the powers leave out is 8.5e-9 of the result; with 16-bit operands, whose probabilities are rounded to 2^-9 or 2^-12, the
// last of them is left out too (3.4e-7).
template <class T>
struct Bend {
    float limit, by2, twice, to, cap, c0, c1, c2, c3, c4;
    __device__ __forceinline__ void init(float scale, float cap_)
    {
        cap = cap_;
        const float by = cap > 0.f ? scale / cap : 0.f;
        to = cap * kLog2e, twice = by * (2.f * kLog2e), limit = cap > 0.f ? 0.25f / by : 0.f, by2 = by * by;
        c0 = scale * kLog2e, c1 = c0 * -0.33333334f, c2 = c0 * 0.13333334f, c3 = c0 * -0.053968254f, c4 = c0 * 0.021869489f;
    }
    __device__ __forceinline__ float near(float x) const
    {
        const float s = x * x * by2, last = sizeof(T) == 4 ? fmaf(s, c4, c3) : c3;
        return x * fmaf(s, fmaf(s, fmaf(s, last, c2), c1), c0);
    }
    template <int N, bool BACK>
    __device__ __forceinline__ void apply(floatx16 (&x)[N], floatx16 (&back)[N]) const
    {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(x[i][r]));
        if (__any(!(most <= limit))) {
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float away = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x[i][r] * twice)), 1.f) * to;
                    x[i][r] = fabsf(x[i][r]) <= limit ? near(x[i][r]) : away;
                }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[i][r] = near(x[i][r]);
        }
        if constexpr (BACK) {
            const float from = 1.f / to;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float y = x[i][r] * from;
                    back[i][r] = fmaf(-y, y, 1.f);
                }
        }
    }
};

}  // namespace sddmm
