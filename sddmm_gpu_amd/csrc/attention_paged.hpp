// Attention over a cache in pages (gfx950): pieces that the kernels share -- codes as operands of the matrix instructions, scores, places in the cache.
//
// The products of few rows are made of 16 x 16 x 32 matrix instructions (fp32: eight of 16 x 16 x 4).  A lane l of a wave holds, with n = l % 16 and g = l / 16:
//   operands   row (or column) n, elements 8 g + j of the 32 that are summed over, j = 0 .. 7
//   results    column n, rows 4 g + i, i = 0 .. 3
#pragma once
#include "attention.hpp"
#include "cache.hpp"

namespace sddmm {

template <class T> __device__ __forceinline__ floatx4 mma16(typename Elem<T>::Vec8 a, typename Elem<T>::Vec8 b, floatx4 c);
template <> __device__ __forceinline__ floatx4 mma16<__bf16>(bf16x8 a, bf16x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
template <> __device__ __forceinline__ floatx4 mma16<_Float16>(half8 a, half8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
template <> __device__ __forceinline__ floatx4 mma16<float>(floatx8 a, floatx8 b, floatx4 c)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// the sum, in the place of a row's first part, of a row that is not the kernel's for many rows
constexpr float kNone = -1.f;

// Eight codes, four to a register, as an operand: both kinds are exact in 16 bits.
template <class T, int HELD> __device__ __forceinline__ typename Elem<T>::Vec8 expand(uint32_t lo, uint32_t hi)
{
    typename Elem<T>::Vec8 r;
    if constexpr (HELD == kHeldE4m3) {
        if constexpr (sizeof(T) == 4) {
            const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(lo, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(lo, true);
            const auto c = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
            r[0] = a[0], r[1] = a[1], r[2] = b[0], r[3] = b[1], r[4] = c[0], r[5] = c[1], r[6] = d[0], r[7] = d[1];
        } else {
            typedef T Vec2 __attribute__((ext_vector_type(2)));
            Vec2 p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t w = i < 2 ? lo : hi;
                if constexpr (__is_same(T, __bf16)) p[i] = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false);
                else p[i] = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
                r[2 * i] = p[i][0], r[2 * i + 1] = p[i][1];
            }
        }
    } else if constexpr (__is_same(T, _Float16)) {
        // 1024 + (code + 128) is a half whose last bits are the code's, with the sign turned over
        typedef _Float16 half2v __attribute__((ext_vector_type(2)));
        const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
        const uint32_t w[4] = {__builtin_amdgcn_perm(a, 0x64646464u, 0x00050004u), __builtin_amdgcn_perm(a, 0x64646464u, 0x00070006u),
                               __builtin_amdgcn_perm(b, 0x64646464u, 0x00050004u), __builtin_amdgcn_perm(b, 0x64646464u, 0x00070006u)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const half2v h = __builtin_bit_cast(half2v, w[i]) - half2v{(_Float16)1152.f, (_Float16)1152.f};
            r[2 * i] = h[0], r[2 * i + 1] = h[1];
        }
    } else if constexpr (__is_same(T, __bf16)) {
        // (an integer below 2^8 fits the upper half of its float)
        uint4v w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t c = i < 2 ? lo : hi;
            const float x = (float)(int8_t)(c >> (16 * (i & 1))), y = (float)(int8_t)(c >> (16 * (i & 1) + 8));
            w[i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
        }
        r = __builtin_bit_cast(bf16x8, w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = (float)(int8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
    return r;
}

// bytes 0 .. 3 of four registers, turned: byte d of each in register d
__device__ __forceinline__ void turn4(uint32_t (&x)[4])
{
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
    x[0] = __builtin_amdgcn_perm(c, a, 0x05040100u), x[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    x[2] = __builtin_amdgcn_perm(d, b, 0x05040100u), x[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// The bound of scores (Bend in attention.hpp) of N scores of a lane.
template <class T, int N> __device__ __forceinline__ void bend_scores(const Bend<T> &bend, float (&x)[N])
{
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(x[i]));
    if (__any(!(most <= bend.limit))) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float away = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x[i] * bend.twice)), 1.f) * bend.to;
            x[i] = fabsf(x[i]) <= bend.limit ? bend.near(x[i]) : away;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = bend.near(x[i]);
    }
}

// the four lane groups of 16 hold parts of the same column: all get the maximum / the sum
__device__ __forceinline__ float groups_max(float x)
{
    x = fmaxf(x, __shfl_xor(x, 16));
    return halves_max(x);
}
__device__ __forceinline__ float groups_sum(float x)
{
    x += __shfl_xor(x, 16);
    return halves_sum(x);
}

}  // namespace sddmm
