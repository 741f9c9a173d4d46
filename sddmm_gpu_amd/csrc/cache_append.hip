// New tokens into a paged cache (gfx950): keys turned by their positions and values, in the operands' type or in 8 bits with a scale for each
// block of tokens and head; and their queries turned on the way.
#include <hip/hip_runtime.h>
#include <cstdlib>
#include <cstring>
#include <type_traits>
#include "cache.hpp"
#include "internal.hpp"
#include "launch.hpp"

using namespace sddmm;

namespace {

constexpr int kBlock = 256;
constexpr int kUnit = 16;  // tokens of a wave's unit of work

struct AppendArgs {
    AttnArgs a;      // q, k, v: the new rows; out: the turned queries
    CacheArgs c;
    const double *freq;
    int32_t rot_dim, half, chunk_shift, max_chunks, heads_per, head_groups, fast, table;  // table: entries of a chunk's angles
    float amplitude;
};

// cos and sin of 64-bit angles: the angle less its nearest multiple of pi / 2, which is subtracted in two parts (Cody and Waite), then the
// series up to the terms below 2^-57.
__device__ __forceinline__ double2 cos_sin(double angle)
{
    const double k = rint(angle * 0.63661977236758134308);
    const double x = fma(-k, 6.123233995736766036e-17, fma(-k, 1.570796326794896558, angle)), z = x * x;
    double s = fma(z, 1. / 355687428096000., -1. / 1307674368000.);
    s = fma(z, s, 1. / 6227020800.), s = fma(z, s, -1. / 39916800.), s = fma(z, s, 1. / 362880.), s = fma(z, s, -1. / 5040.);
    s = fma(z, s, 1. / 120.), s = fma(z, s, -1. / 6.), s = fma(x * z, s, x);
    double c = fma(z, 1. / 20922789888000., -1. / 87178291200.);
    c = fma(z, c, 1. / 479001600.), c = fma(z, c, -1. / 3628800.), c = fma(z, c, 1. / 40320.), c = fma(z, c, -1. / 720.);
    c = fma(z, c, 1. / 24.), c = fma(z, c, -0.5), c = fma(z, c, 1.);
    const int quarter = (int)(k - 4. * floor(k * 0.25));
    return quarter == 0 ? double2{c, s} : quarter == 1 ? double2{-s, c} : quarter == 2 ? double2{-c, -s} : double2{s, -c};
}

// The chunk of `slot` among packed sequences: sequence s takes the slots from ptr[s] / chunk + 2 s on, as many as its rows need wherever they begin in their chunks.
// 64 sequences are looked at in a step.
__device__ __forceinline__ int find_sequence(const AppendArgs &p, int slot, int &chunk)
{
    const int lane = threadIdx.x & 63;
    auto begin = [&](int s) { return (int)min((int64_t)(max(0, p.a.q_ptr[s]) >> p.chunk_shift) + 2 * (int64_t)s, (int64_t)INT32_MAX); };
    int lo = 0, n = p.a.n_seq;  // the last of n sequences from lo on that begins at `slot` or before
    while (n > 1) {
        const int step = (n + 63) / 64, s = lane * step;
        const uint64_t some = __ballot(s < n && begin(lo + s) <= slot);
        const int at = some ? (63 - __builtin_clzll(some)) * step : 0;
        lo += at, n = min(step, n - at);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    chunk = slot - begin(lo);
    return chunk < 0 ? -1 : lo;
}

template <class T> struct Piece { typedef T Vec __attribute__((ext_vector_type(8))); };
template <class T> __device__ __forceinline__ void store8(T *p, const float (&x)[8])
{
    typedef T Vec __attribute__((ext_vector_type(8)));
    Vec v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (T)x[j];
    *(Vec *)p = v;
}

// Eight codes of values in steps of a scale, rounded to nearest even; beyond the largest code, the largest.
template <int HELD> __device__ __forceinline__ uint2 codes_of(const float (&x)[8])
{
    uint32_t r[2];
    if constexpr (HELD == kHeldI8) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            r[w] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y = x[4 * w + j];
                const int code = y == y ? (int)fminf(fmaxf(rintf(y), -127.f), 127.f) : 0;
                r[w] |= ((uint32_t)code & 255u) << (8 * j);
            }
        }
    } else {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = x[4 * w + j];
                y[j] = v > 448.f ? 448.f : v < -448.f ? -448.f : v;
            }
            const int low = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            r[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], low, true);
        }
    }
    return make_uint2(r[0], r[1]);
}
// The same for finite values within the range and a scale whose reciprocal is exact: the integer is the last byte of 1.5 * 2^23 and it.
template <int HELD> __device__ __forceinline__ uint2 codes_of_scaled(const float (&x)[8], float by)
{
    uint32_t r[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        if constexpr (HELD == kHeldI8) {
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __float_as_uint(fmaf(x[4 * w + j], by, 12582912.f));
            r[w] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], 0x0c0c0400u), __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400u), 0x05040100u);
        } else {
            const int low = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w] * by, x[4 * w + 1] * by, 0, false);
            r[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w + 2] * by, x[4 * w + 3] * by, low, true);
        }
    }
    return make_uint2(r[0], r[1]);
}

// The maximum over 2^`levels` lanes in a row: 0 to 6.
__device__ __forceinline__ float lanes_max(float x, int levels)
{
    auto dpp = [](float y, auto ctrl) { return fmaxf(y, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(y), (int)__float_as_uint(y), decltype(ctrl)::value, 0xf, 0xf, false))); };
    if (levels > 0) x = dpp(x, std::integral_constant<int, 0xB1>());   // lanes 1 apart,
    if (levels > 1) x = dpp(x, std::integral_constant<int, 0x4E>());   // 2 apart,
    if (levels > 2) x = dpp(x, std::integral_constant<int, 0x141>());  // eight turned round (fours are alike by now),
    if (levels > 3) x = dpp(x, std::integral_constant<int, 0x140>());  // sixteen turned round
    if (levels > 4) x = fmaxf(x, __shfl_xor(x, 16));
    if (levels > 5) x = halves_max(x);
    return x;
}

template <int HELD> __device__ __forceinline__ void values_of(uint2 codes, float (&x)[8])
{
    const uint32_t r[2] = {codes.x, codes.y};
#pragma unroll
    for (int w = 0; w < 2; ++w)
        if constexpr (HELD == kHeldI8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * w + j] = (float)(int8_t)(r[w] >> (8 * j));
        } else {
            const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(r[w], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(r[w], true);
            x[4 * w] = a[0], x[4 * w + 1] = a[1], x[4 * w + 2] = b[0], x[4 * w + 3] = b[1];
        }
}

// The least power of two, from 2^-126 on, that `top` is at most `most` times of.
__device__ __forceinline__ float least_scale(float top, float most)
{
    int e = -125;
    if (top > 0.f) frexpf(top / most, &e);
    const float scale = ldexpf(1.f, max(e - 1, -126));
    return top > scale * most ? 2.f * scale : scale;
}

// A workgroup takes a chunk of 16 positions (of a whole block of tokens, where blocks are longer) of a sequence, with the angles' cosines and sines in LDS
// once for all heads, and some of its key heads.  LPR lanes hold a row, two pieces of eight elements each -- the two halves of pairs where
// those lie in halves; a wave a unit of 16 tokens of a key head's keys or values in registers: read once, turned, the largest element of each block found by
// exchanges between lanes (between waves for blocks of 32 and 64), and written as codes.  Bound by bytes: 16,384 tokens of 32 + 8 heads of 128 in 86 us, 4.3 TB/s (vector instructions 41 %
// of the time); a few tokens by the launch (7 us).
//
// Turned in 64 bits: a code is a rounding to few bits, whose borders products in 32 bits would cross for one element in 10^5, so that codes depended on the way
// of computing.
template <class T, int HELD, int LPR>
__global__ __launch_bounds__(kBlock, sizeof(T) == 4 ? 2 : 3)
void sddmm_cache_append_kernel(const AppendArgs p)
{
    constexpr int kRows = 64 / LPR, kPasses = kUnit / kRows;  // of a wave at a time, of a unit
    constexpr float kMost = HELD == kHeldI8 ? 127.f : 448.f;
    // Cosines and sines in 64 bits for what becomes codes or fp32, in 32 bits for what becomes 16.
    constexpr bool kCoarse = sizeof(T) == 2, kKeysCoarse = kCoarse && HELD == kHeldOwn;
    extern __shared__ double2 angles[];
    float2 *const coarse = (float2 *)(angles + (kKeysCoarse ? 0 : p.table));
    __shared__ float tops[4];
    const AttnArgs &a = p.a;
    const CacheArgs &c = p.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = lane / LPR, item = lane % LPR;
    const int slot = blockIdx.x / p.head_groups, head0 = blockIdx.x % p.head_groups * p.heads_per, n_heads = min(p.heads_per, a.n_kv_heads - head0);
    int s, chunk;
    if (a.q_ptr) {
        s = find_sequence(p, slot, chunk);
        if (s < 0) return;
    } else {
        s = slot / p.max_chunks, chunk = slot % p.max_chunks;
    }
    const Seq e = sequence(a, s);
    const int start = e.nk - e.nq;  // (below 0 where more rows come than the length counts)
    const int64_t first_of = ((int64_t)(start >> p.chunk_shift) + chunk) << p.chunk_shift;
    if (first_of >= e.nk) return;
    const int p0 = (int)first_of, lo = max(p0, start), hi = min(p0 + (1 << p.chunk_shift), e.nk), n = hi - lo;
    if (n <= 0) return;  // (no new rows)
    // the places of this lane's two pieces in a row (or none): pairs that lie in halves, then the rest two by two
    const int hp = p.half && p.fast ? p.rot_dim / 16 : 0, n_pieces = a.head_dim / 8;
    int at[2];
    at[0] = item < hp ? 8 * item : 8 * (2 * hp + 2 * (item - hp));
    at[1] = item < hp ? 8 * (item + hp) : at[0] + 8;
    const bool there[2] = {at[0] < 8 * n_pieces, at[1] < 8 * n_pieces};
    typedef typename Piece<T>::Vec Vec;
    auto fetch = [&](const T *row, Vec (&x)[2]) {  // (a lane without a piece takes the row's first)
#pragma unroll
        for (int i = 0; i < 2; ++i) x[i] = *(const Vec *)(row + (there[i] ? at[i] : 0));
    };

    // keys and values: units of 16 tokens, those of a block next to each other, a wave's first requested before the angles are made
    const int units_per = 1 << (p.chunk_shift - 4), n_units = n_heads * 2 * units_per;
    const T *rows = nullptr;
    int64_t row = 0;
    Vec raw[kPasses][2];
    auto request = [&](int u) {
        const int part = u % units_per, is_v = (u / units_per) & 1, kv = head0 + u / (2 * units_per), first = p0 + kUnit * part;
        rows = is_v ? (const T *)a.v + (a.q_ptr ? e.q0 * a.v_row : s * a.v_seq) + kv * a.v_head : (const T *)a.k + (a.q_ptr ? e.q0 * a.k_row : s * a.k_seq) + kv * a.k_head;
        row = is_v ? a.v_row : a.k_row;
#pragma unroll
        for (int t = 0; t < kPasses; ++t) fetch(rows + (min(max(first + t * kRows + mine, lo), hi - 1) - start) * row, raw[t]);
    };
    if (wave < n_units) request(wave);

    // (element e of a token's pairs at place (e % 8) * eighths + e / 8: the lanes of a row, which take eight pairs each, read next to each other)
    const int pairs = p.rot_dim / 2, eighths = (pairs + 7) / 8;
    for (int i = threadIdx.x; i < n * pairs; i += kBlock) {
        const int r = i / pairs, pair = i - r * pairs, to = (r * 9 + (pair & 7)) * eighths + (pair >> 3);
        double2 cs = cos_sin((double)(lo + r) * p.freq[pair]);
        cs.x *= p.amplitude, cs.y *= p.amplitude;
        if (!kKeysCoarse) angles[to] = cs;
        if (kCoarse) coarse[to] = make_float2((float)cs.x, (float)cs.y);
    }
    if (pairs) __syncthreads();

    // a row's two pieces, turned
    auto turned = [&]<bool COARSE>(std::bool_constant<COARSE>, const Vec (&r)[2], const T *row, int token, bool turn, float (&x)[2][8]) {
        typedef std::conditional_t<COARSE, float, double> F;
        typedef std::conditional_t<COARSE, float2, double2> F2;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] = there[i] ? (float)r[i][j] : 0.f;
        if (!turn || at[0] >= p.rot_dim) return;
        const F2 *cs;
        if constexpr (COARSE) cs = coarse; else cs = angles;
        cs += (token - lo) * 9 * eighths;
        if (hp) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const F2 w = cs[j * eighths + item];
                const F u = x[0][j], v = x[1][j];
                x[0][j] = (float)(u * w.x - v * w.y), x[1][j] = (float)(u * w.y + v * w.x);
            }
        } else if (!p.half) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 8; j += 2)
                    if (at[i] + j < p.rot_dim) {
                        const F2 w = cs[(4 * i + j / 2) * eighths + item];
                        const F u = x[i][j], v = x[i][j + 1];
                        x[i][j] = (float)(u * w.x - v * w.y), x[i][j + 1] = (float)(u * w.y + v * w.x);
                    }
        } else {
            // halves that are no whole pieces: an element's partner by itself
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int k = at[i] + j;
                    if (k >= p.rot_dim) continue;
                    const bool first = k < pairs;
                    const int pair = first ? k : k - pairs;
                    const F2 w = cs[(pair & 7) * eighths + (pair >> 3)];
                    const F u = x[i][j], v = (float)row[first ? k + pairs : k - pairs];
                    x[i][j] = (float)(first ? u * w.x - v * w.y : v * w.y + u * w.x);
                }
        }
    };

    for (int u0 = 0; u0 < n_units; u0 += 4) {
        const int u = u0 + wave, part = u % units_per, is_v = (u / units_per) & 1, kv = head0 + u / (2 * units_per), first = p0 + kUnit * part;
        // (units of a block's earlier tokens too, where blocks are longer than units)
        const bool some = u < n_units && first >= 0 && first < hi && (first + kUnit > lo || 1 << c.block_shift > kUnit) && c.n_pages > 0;
        const int page = some ? c.page(s, first >> c.page_shift) : 0, in_page = first & ((1 << c.page_shift) - 1);
        char *cache = is_v ? c.v_at(page, kv, in_page) : c.k_at(page, kv, in_page);
        const uint32_t cache_row = is_v ? c.v_row : c.k_row;
        float x[kPasses][2][8], top[kPasses];
        bool fresh[kPasses], odd = false;
#pragma unroll
        for (int t = 0; t < kPasses; ++t) {
            const int pos = first + t * kRows + mine;
            fresh[t] = some && pos >= max(lo, 0) && pos < hi;
            top[t] = 0.f;
            if (!fresh[t]) continue;
            turned(std::bool_constant<kKeysCoarse>(), raw[t], rows + (pos - start) * row, pos, !is_v, x[t]);
            if constexpr (HELD == kHeldOwn) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (there[i]) store8((T *)(cache + (uint32_t)(t * kRows + mine) * cache_row) + at[i], x[t][i]);
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        top[t] = fmaxf(top[t], fabsf(x[t][i][j]));
                        if (sizeof(T) == 4) odd = odd || x[t][i][j] != x[t][i][j];  // (a NaN of 16 bits ends in a byte of 0, as its code does)
                    }
                odd = odd || top[t] == INFINITY;
            }
        }
        if (u + 4 < n_units) request(u + 4);
        if constexpr (HELD != kHeldOwn) {
            const bool plain = !__any(odd);
            if (!plain) {  // the largest finite element
#pragma unroll
                for (int t = 0; t < kPasses; ++t) {
                    top[t] = 0.f;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (fresh[t] && fabsf(x[t][i][j]) < INFINITY) top[t] = fmaxf(top[t], fabsf(x[t][i][j]));
                }
            }
            const int block = 1 << c.block_shift;
            if (kPasses == 2 && block > kRows) top[0] = top[kPasses - 1] = fmaxf(top[0], top[kPasses - 1]);
#pragma unroll
            for (int t = 0; t < kPasses; ++t) top[t] = lanes_max(top[t], (LPR == 8 ? 3 : 2) + min(c.block_shift, LPR == 8 ? 3 : 4));
            if (block > kUnit) {
                __syncthreads();
                if (lane == 0) tops[wave] = top[0];
                __syncthreads();
                // (waves of a block: part 0 .. units_per - 1, of which there are 2 or 4)
                float most = 0.f;
                for (int i = 0; i < units_per; ++i) most = fmaxf(most, tops[wave - part + i]);
#pragma unroll
                for (int t = 0; t < kPasses; ++t) top[t] = most;
            }
            float *scales = is_v ? c.v_scale : c.k_scale;
            float scale[kPasses];
            bool begins[kPasses];
#pragma unroll
            for (int t = 0; t < kPasses; ++t) {
                const int place = t * kRows + mine, pos = first + place, begin = pos & ~(block - 1);  // of its block
                begins[t] = false;
                if (!some || begin + block <= lo || begin >= hi) continue;
                begins[t] = pos == begin && item == 0;
                const float old = begin < start ? scales[c.scale_at(page, kv, in_page + place)] : 0.f;
                scale[t] = old;
                if (!(old > 0.f && top[t] <= old * kMost)) scale[t] = least_scale(top[t], kMost);
                char *to = cache + (uint32_t)place * cache_row;
                const uint32_t bits = __float_as_uint(scale[t]);
                if (fresh[t] && plain && (bits & 0x7fffffu) == 0 && bits - 0x00800000u < 0x7e000000u) {
                    const float by = __uint_as_float(0x7f000000u - bits);  // (a power of two's reciprocal)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (there[i]) *(uint2 *)(to + at[i]) = codes_of_scaled<HELD>(x[t][i], by);
                } else if (fresh[t]) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (!there[i]) continue;
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[t][i][j] /= scale[t];
                        *(uint2 *)(to + at[i]) = codes_of<HELD>(x[t][i]);
                    }
                } else if (pos < start && scale[t] != old) {
                    // an earlier token of a block whose steps grow
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (!there[i]) continue;
                        float y[8];
                        values_of<HELD>(*(const uint2 *)(to + at[i]), y);
#pragma unroll
                        for (int j = 0; j < 8; ++j) y[j] = y[j] * old / scale[t];
                        *(uint2 *)(to + at[i]) = codes_of<HELD>(y);
                    }
                }
            }
            // (every lane of a block has its scale before one of them writes it)
            if (block > kUnit) __syncthreads();
#pragma unroll
            for (int t = 0; t < kPasses; ++t)
                if (begins[t]) scales[c.scale_at(page, kv, in_page + t * kRows + mine)] = scale[t];
        }
    }

    // queries: rows of (token, head)
    if (!a.q) return;
    const int heads = n_heads * a.group, all = n * heads;
    const T *from = (const T *)a.q + (a.q_ptr ? e.q0 * a.q_row : s * a.q_seq);
    T *to = (T *)a.out + (a.q_ptr ? e.q0 * a.q_row : s * a.q_seq);
    // (token and head of a lane's row, going on by so many of each; kSets rows of a lane under way)
    constexpr int kSets = sizeof(T) == 2 ? 4 : 2;
    const int step_tokens = 4 * kRows / heads, step_heads = 4 * kRows % heads;
    int i = (3 - wave) * kRows + mine, t = i / heads, head = i - t * heads;
    while (i - mine < all) {
        Vec set[kSets][2];
        int64_t place[kSets];
        int token[kSets];
#pragma unroll
        for (int k = 0; k < kSets; ++k) {
            token[k] = lo + t;
            place[k] = (lo + min(t, n - 1) - start) * a.q_row + (head0 * a.group + head) * a.q_head;
            if (i - mine + k * 4 * kRows < all) fetch(from + place[k], set[k]);
            t += step_tokens, head += step_heads;
            if (head >= heads) head -= heads, ++t;
        }
#pragma unroll
        for (int k = 0; k < kSets; ++k) {
            if (i + k * 4 * kRows < all) {
                float x[2][8];
                turned(std::bool_constant<kCoarse>(), set[k], from + place[k], token[k], true, x);
                __builtin_amdgcn_wave_barrier();  // (in place: partners are read before anything of the row is written)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (there[j]) store8(to + place[k] + at[j], x[j]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        i += kSets * 4 * kRows;
    }
}

template <class T, int HELD>
hipError_t launch_held(const AppendArgs &p, unsigned grid, size_t lds, hipStream_t st)
{
    auto *fn = p.a.head_dim <= 64 ? sddmm_cache_append_kernel<T, HELD, 4> : sddmm_cache_append_kernel<T, HELD, 8>;
    if (lds > 32768) {  // (blocks of 64 tokens: more than a launch takes without asking)
        const hipError_t e = hipFuncSetAttribute((const void *)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    return launch(fn, dim3(grid), dim3(kBlock), lds, st, p);
}
template <class T>
hipError_t launch_typed(const AppendArgs &p, int held, unsigned grid, size_t lds, hipStream_t st)
{
    return held == kHeldI8 ? launch_held<T, kHeldI8>(p, grid, lds, st) : held == kHeldE4m3 ? launch_held<T, kHeldE4m3>(p, grid, lds, st) : launch_held<T, kHeldOwn>(p, grid, lds, st);
}

}  // namespace

extern "C" {

void sddmm_cache_desc_init(sddmm_cache_desc *cache)
{
    if (!cache) return;
    memset(cache, 0, sizeof *cache);
    cache->block_len = 1;
    cache->rot_amplitude = 1.f;
}

int sddmm_cache_append(const sddmm_attention_desc *desc, const sddmm_cache_desc *cache, const void *d_q, void *d_q_out, const void *d_k,
                       const void *d_v, void *stream)
{
    const char *who = "sddmm_cache_append";
    if (!desc) return fail(SDDMM_ERR_ARG, "%s: NULL description", who);
    // (new keys and values are numbered as the queries are; o_ strides are not looked at)
    sddmm_attention_desc rows = *desc;
    rows.k_ptr = desc->q_ptr ? desc->q_ptr : desc->k_ptr, rows.k_rows = desc->q_ptr ? desc->q_rows : desc->k_rows;
    if (desc->q_ptr) rows.k_len = nullptr;
    rows.o_seq = rows.q_seq, rows.o_row = rows.q_row, rows.o_head = rows.q_head;
    if (int rc = check_desc(who, &rows)) return rc;
    if ((uintptr_t)desc->k_len & 3u) return fail(SDDMM_ERR_ARG, "%s: arrays of the description must be aligned to their elements", who);
    if (int rc = check_cache(who, *desc, cache)) return rc;
    const sddmm_attention_desc d = held(*desc);
    const sddmm_cache_desc &c = *cache;
    if (c.rot_layout != SDDMM_ROTARY_HALF && c.rot_layout != SDDMM_ROTARY_INTERLEAVED) return fail(SDDMM_ERR_ARG, "%s: unknown layout %d", who, c.rot_layout);
    if (c.rot_dim < 0 || c.rot_dim % 2 || c.rot_dim > d.head_dim) return fail(SDDMM_ERR_ARG, "%s: rot_dim = %d has to be even and 0 .. head_dim = %d", who, c.rot_dim, d.head_dim);
    if (!std::isfinite(c.rot_amplitude)) return fail(SDDMM_ERR_ARG, "%s: rot_amplitude must be finite", who);
    const int64_t new_rows = rows_of(d);
    if (new_rows == 0) return SDDMM_OK;
    if (!d_k || !d_v || (d_q && !d_q_out) || (c.rot_dim > 0 && !c.rot_freq)) return fail(SDDMM_ERR_ARG, "%s: NULL device pointer", who);
    if ((uintptr_t)c.rot_freq & 7u) return fail(SDDMM_ERR_ARG, "%s: arrays of the description must be aligned to their elements", who);
    if (!aligned({d_q, d_q_out, d_k, d_v})) return fail(SDDMM_ERR_ARG, "%s: pointers must be 16-byte aligned", who);
    const int64_t seqs = d.q_ptr ? 1 : d.n_seq, per_seq = d.q_ptr ? d.q_rows : d.max_q;
    if (d_q && !apart(d, d.q_seq, d.q_row, d.q_head, seqs, per_seq, d.n_heads)) return fail(SDDMM_ERR_ARG, "%s: rows of the turned queries overlap", who);
    // rows of the cache, as [page][token][head] or in any other order
    sddmm_attention_desc pages = d;
    if (!apart(pages, c.k_page, c.k_row, c.k_head, c.n_pages, c.page_len, d.n_kv_heads) || !apart(pages, c.v_page, c.v_row, c.v_head, c.n_pages, c.page_len, d.n_kv_heads))
        return fail(SDDMM_ERR_ARG, "%s: rows of the cache overlap", who);
    if (c.type != d.type) {
        // (keys' scales and values' are read and written by different waves)
        const int64_t scales = c.n_pages * d.n_kv_heads * (c.page_len / c.block_len) * (int64_t)sizeof(float), between = std::llabs((int64_t)((intptr_t)c.k_scale - (intptr_t)c.v_scale));
        if (c.k_scale && c.v_scale && (between < scales || in_place_of({c.k_scale, c.v_scale}, {d_q, d_q ? d_q_out : nullptr, d_k, d_v, c.k, c.v})))
            return fail(SDDMM_ERR_ARG, "%s: scales are in another array's place", who);
    }
    if (in_place_of({c.k, c.v}, {d_q, d_q_out, d_k, d_v}) || (c.k && c.k == c.v) || (d_q && in_place_of({d_q_out}, {d_k, d_v})))
        return fail(SDDMM_ERR_ARG, "%s: a result is in an operand's or another result's place", who);

    AppendArgs p{};
    p.a = arguments(d), p.c = cache_arguments(d, c);
    p.a.q = d_q, p.a.k = d_k, p.a.v = d_v, p.a.out = d_q_out;
    p.freq = c.rot_freq, p.rot_dim = c.rot_dim, p.half = c.rot_layout == SDDMM_ROTARY_HALF, p.fast = c.rot_dim % 16 == 0, p.amplitude = c.rot_amplitude;
    const int held = held_as(d, c);
    p.chunk_shift = std::max(4, (int)p.c.block_shift);
    const int64_t chunk = (int64_t)1 << p.chunk_shift;
    p.max_chunks = (int32_t)((d.max_q + chunk - 2) / chunk + 1);
    const int64_t slots = d.q_ptr ? new_rows / chunk + 2 * (int64_t)d.n_seq : (int64_t)d.n_seq * p.max_chunks;
    // Key heads of a workgroup: so few that there are 2048 workgroups, but, where there are 512 all the same, as many as make a row for each of 16 groups of lanes (us with 512, 1024, 2048, 4096
    // workgroups: 16,384 tokens, 32 heads over 8 of 128 96 / 96 / 84 / 88; 5999 tokens, 12 heads of 64 18 / 22 / 26 / 26).
    const int64_t lane_rows = d.head_dim <= 64 ? 2 + p.a.group : 4 + 2 * (int64_t)p.a.group;  // groups of rows that a wave takes at a time, of a key head
    const int64_t many = div_up(d.n_kv_heads, std::min<int64_t>(d.n_kv_heads, div_up(512, slots)));
    p.heads_per = (int32_t)std::max(div_up(d.n_kv_heads, std::min<int64_t>(d.n_kv_heads, div_up(2048, slots))), std::min(many, div_up(16, lane_rows)));
    p.head_groups = (int32_t)div_up(d.n_kv_heads, p.heads_per);
    if (slots > INT32_MAX || !launchable(slots * p.head_groups, kBlock)) return fail(SDDMM_ERR_RANGE, "%s: too many rows and heads for one launch", who);
    p.table = (int32_t)(chunk * div_up(c.rot_dim / 2, 8) * 9);
    const size_t lds = p.table * (d.type == SDDMM_TYPE_F32 ? sizeof(double2) : held == kHeldOwn ? sizeof(float2) : sizeof(double2) + sizeof(float2));
    const unsigned grid = (unsigned)(slots * p.head_groups);
    const hipStream_t st = (hipStream_t)stream;
    const hipError_t e = d.type == SDDMM_TYPE_F32 ? launch_typed<float>(p, held, grid, lds, st) : d.type == SDDMM_TYPE_F16 ? launch_typed<_Float16>(p, held, grid, lds, st)
                                                                                                                        : launch_typed<__bf16>(p, held, grid, lds, st);
    if (e != hipSuccess) return fail(SDDMM_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
    return SDDMM_OK;
}

}  // extern "C"
