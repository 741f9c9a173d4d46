// Attention over a cache in pages (gfx950): a tile of rows against tiles of keys.
#pragma once
#include <cfloat>
#include "attention_paged.hpp"

namespace sddmm {

// What products of codes are made of: fp16 for 16-bit operands (an 8-bit code times a power of two is exact in it, and it comes from eight bits in
// fewer instructions than bf16), else the operands' type.
template <class T, int HELD> struct Product { typedef T Type; };
template <> struct Product<__bf16, kHeldI8> { typedef _Float16 Type; };
template <> struct Product<__bf16, kHeldE4m3> { typedef _Float16 Type; };

// Eight codes times `by`, as an operand: fp16 by a power of two within the range of `fold` (exact), fp32 by any scale.
template <class U, int HELD> __device__ __forceinline__ typename Elem<U>::Vec8 expand_by(uint32_t lo, uint32_t hi, float by)
{
    typename Elem<U>::Vec8 r;
    if constexpr (sizeof(U) == 4) {
        r = expand<U, HELD>(lo, hi) * by;
    } else if constexpr (HELD == kHeldE4m3) {
        typedef _Float16 half2v __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const half2v h = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(i < 2 ? lo : hi, by, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(i < 2 ? lo : hi, by, false);
            r[2 * i] = h[0], r[2 * i + 1] = h[1];
        }
    } else {
        // (1152 + code) * by - 1152 * by, the sum being a half whose last bits are the code's with the sign turned over
        typedef _Float16 half2v __attribute__((ext_vector_type(2)));
        const _Float16 b = (_Float16)by, o = (_Float16)(by * -1152.f);
        const uint32_t x = lo ^ 0x80808080u, y = hi ^ 0x80808080u;
        const uint32_t w[4] = {__builtin_amdgcn_perm(x, 0x64646464u, 0x00050004u), __builtin_amdgcn_perm(x, 0x64646464u, 0x00070006u),
                               __builtin_amdgcn_perm(y, 0x64646464u, 0x00050004u), __builtin_amdgcn_perm(y, 0x64646464u, 0x00070006u)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const half2v h = __builtin_elementwise_fma(__builtin_bit_cast(half2v, w[i]), half2v{b, b}, half2v{o, o});
            r[2 * i] = h[0], r[2 * i + 1] = h[1];
        }
    }
    return r;
}

// A scale's power of two, as far as codes times it are exact in fp16, and what is left of the scale.
template <class U, int HELD> __device__ __forceinline__ float fold(float scale, float &left)
{
    if constexpr (sizeof(U) == 4) {
        left = 1.f;
        return scale;
    } else {
        constexpr int kLeast = HELD == kHeldI8 ? -24 : -15, kMost = HELD == kHeldI8 ? 5 : 7;
        const int e = min(max(__builtin_amdgcn_frexp_expf(scale) - 1, kLeast), kMost);
        const float by = __uint_as_float((uint32_t)((e << 23) + 0x3f800000));
        left = __builtin_amdgcn_ldexpf(scale, -e);
        return by;
    }
}

// The rows of a workgroup are (token, head) pairs that share a key head, 32 to each of NW waves; they go over the keys as the dense kernel's do (attention_tile.hpp):
// a running maximum that is raised when a row's exceeds it by more than 2^8, S^T = K Q^T and O^T += V^T P^T, tiles of keys in LDS, two in turn.  What differs is how tiles
// come: rows of the operands' type go from their pages to LDS by themselves, sixteen being in one page; codes are taken into registers while the tile before is multiplied, and
// written to LDS as operands times their scales' powers of two, once for all rows of a workgroup.  Scales that are no powers of two (sddmm_cache_append makes none) leave a factor to each
// token, which goes to scores and probabilities in tiles that have any; weights are in units of each row's own then, so that no scale of another's keys costs a row its bits.
//
// 2048 tokens behind 14,336, 16 heads over 2 of 128, 8 bits: 314 us, 0.82 PFLOP/s (a prompt of 4096, 32 heads over 8, bf16 cache: 0.90).  Vector instructions take 49 % of the time, matrix ones
// 33, compute units are busy for 88.  Halves of a workgroup half a tile apart, one at products while the other is at the rest, were slower (345 to 367): the vector
// instructions of one wave and the matrix instructions of the other on its SIMD slow each other.
template <class T, int HELD, int DP, bool MOD, int NW>
struct PagedTile {
    typedef typename Product<T, HELD>::Type U;
    static constexpr int KT = sizeof(U) == 2 ? 64 : 32;
    static constexpr int kRows = 32 * NW;
    typedef Tile<U, DP, KT> Keys;
    static constexpr int kTiles = 4 * Keys::kBytes;
    static constexpr int kLds = kTiles + (HELD != kHeldOwn ? 4 * (KT * 4 + 8) : 0);
    static __device__ __forceinline__ void run(const AttnArgs &a, const CacheArgs &c, int b, char (&memory)[kLds]);
};

template <class T, int HELD, int DP, bool MOD, int NW>
__device__ __forceinline__ void PagedTile<T, HELD, DP, MOD, NW>::run(const AttnArgs &a, const CacheArgs &c, int b, char (&memory)[kLds])
{
    constexpr int KB = KT / 32, DB = DP / 32;
    constexpr bool kCodes = HELD != kHeldOwn, kHalves = kCodes && sizeof(U) == 2;
    constexpr float kShift = kHalves ? 7.f : 0.f;  // probabilities are up to 2^(8 + this): fp16's small ones lose nothing that counts
    typedef typename Elem<U>::Vec8 Vec8;
    // tiles of keys and of values, two in turn; for each of them what is left of scales, and whether a wave's rows have any that is not 1
    auto place_of = [&](int which, int t) { return (t & 1) * 2 + which; };
    auto tile_at = [&](int which, int t) { return memory + place_of(which, t) * Keys::kBytes; };
    static_assert(8 % NW == 0);
    float *left = (float *)(memory + kTiles);
    uint8_t *any_left = (uint8_t *)(left + 4 * KT);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, h = lane >> 5;

    int s = 0, tile;
    const int kv = b % a.n_kv_heads;
    b /= a.n_kv_heads;
    const int split = b % a.n_split;
    b /= a.n_split;
    if (a.q_ptr) {
        s = slot_sequence<false>(a.q_ptr, a.n_seq, a.group, kRows, a.max_tiles, a.n_slots, b, tile);
        if (s < 0) return;
    } else {
        s = b % a.n_seq, tile = a.max_tiles - 1 - b / a.n_seq;
    }
    const Seq e = sequence(a, s);
    const int n_rows = e.nq * a.group, n_keys = c.n_pages > 0 ? e.nk : 0;
    if (tile * kRows >= n_rows || n_rows <= a.few_rows) return;
    const int row = tile * kRows + wave * 32 + n;
    const bool there = row < n_rows;
    const int token = row / a.group, head = kv * a.group + row % a.group;
    const int shift = e.nk - e.nq, prefix = a.prefix ? a.prefix[s] : 0, pos = token + shift;
    const int lo = first_key(a, pos), hi = end_key(a, pos, prefix, n_keys);
    const int w0 = tile * kRows + wave * 32, w1 = min(n_rows, w0 + 32) - 1;
    auto of = [&](int r) { return r / a.group + shift; };
    const int any_lo = first_key(a, of(tile * kRows)), any_hi = end_key(a, of(min(n_rows, tile * kRows + kRows) - 1), prefix, n_keys);
    const int wave_lo = first_key(a, of(w0)), wave_hi = w1 < w0 ? 0 : end_key(a, of(w1), prefix, n_keys);
    const int full_lo = first_key(a, of(max(w1, 0))), full_hi = end_key(a, of(w0), prefix, n_keys);

    // the row's elements; bf16 rows that meet codes in fp16 by a power of two, so that the largest is below 2^13 (what is 2^-27 of it keeps all of its bits)
    const T *q = q_base<T>(a, a.q, e, s, head) + (int64_t)token * a.q_row;
    float by_row = 1.f;
    Vec8 qf[DP / 16];
    if constexpr (!__is_same(T, U)) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const auto x = global_operand<T>(q, there, 16 * i + 8 * h, a.head_dim);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf((float)x[j]));
        }
        most = halves_max(most);
        const int ex = (int)(__float_as_uint(most) >> 23) - 126;
        // (no further than the scores' unit stays a normal number, which matters to rows of nothing but tiny elements)
        const int most_up = min((int)(__float_as_uint(a.scale * kLog2e) >> 23) - 2, 126);
        const int up = most < INFINITY ? min(13 - ex, most_up) : 0;
        const float to = __uint_as_float((uint32_t)(127 + up) << 23);
        by_row = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const auto x = global_operand<T>(q, there, 16 * i + 8 * h, a.head_dim);
#pragma unroll
            for (int j = 0; j < 8; ++j) qf[i][j] = (U)((float)x[j] * to);
        }
    } else {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) qf[i] = global_operand<T>(q, there, 16 * i + 8 * h, a.head_dim);
    }

    floatx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = zero16();
    const float scale = a.scale;
    Bend<T> bend;
    if constexpr (MOD) bend.init(scale, a.cap);
    const float unit = MOD ? 1.f : scale * kLog2e * by_row;  // scores in registers to powers of two
    const float raise = fminf(8.f / unit, FLT_MAX);  // (finite: added to a maximum of -infinity)
    const float slope = MOD && a.slopes && there ? a.slopes[head] * kLog2e : 0.f;
    float m = -INFINITY, sum = 0.f;
    float norm = 1.f, best = 0.f;  // codes in 16 bits: the unit of the row's weights, and the largest of them in units of 2^15 (see `weights`)

    // tiles begin at multiples of 16, so that sixteen rows lie in one page
    const int key0 = any_lo & ~15, n_tiles = any_hi > any_lo ? (any_hi - key0 + KT - 1) / KT : 0;
    const int each = (n_tiles + a.n_split - 1) / a.n_split, first = split * each, last = min(n_tiles, first + each);
    uint32_t pages = 0;
    int pages0 = INT32_MIN / 2;
    const int in_page = (1 << c.page_shift) - 1;
    // (whole waves ask, for keys that do not fall)
    auto hold_pages = [&](int key) {
        const int i = min(key, n_keys - 1) >> c.page_shift, top = min(key + KT - 1, n_keys - 1) >> c.page_shift;
        if (i < pages0 || top - pages0 >= 64) {
            pages0 = i;
            pages = c.page(s, min(i + lane, (n_keys - 1) >> c.page_shift));
        }
    };
    auto page_of = [&](int key) { return __builtin_amdgcn_readlane((int)pages, (min(key, n_keys - 1) >> c.page_shift) - pages0); };

    // codes: RPW rows to a wave at a time, kPiece bytes to a lane
    constexpr int kPiece = DP == 32 ? 8 : 16, kLanes = DP / kPiece, RPW = 64 / kLanes, kSteps = (KT + RPW * NW - 1) / (RPW * NW), kWords = kPiece / 4;
    uint32_t raw[kCodes ? kSteps : 1][2][kWords];
    float scales[kCodes ? kSteps : 1][2];
    // (of the lanes that write to LDS together, eight, half are four rows behind the others, whose pieces lie in the other banks)
    const int my_row = kPiece == 8 ? lane / kLanes : kLanes == 8 ? (lane >> 4) | (lane & 4) : ((lane >> 3) & 3) | (lane & 4) | ((lane >> 2) & 8);
    const int my_piece = (kPiece == 8 ? lane % kLanes : kLanes == 8 ? (lane & 3) | ((lane >> 1) & 4) : lane & 3) * kPiece;
    static_assert(kLanes == 8 || kLanes == 4);
    // (16 rows at most, of which `rows` exist: what lies behind them and behind the head's end becomes 0 and is not read)
    auto rows_at = [&](const char *base, uint32_t row, int rows) {
        const uint64_t begin = (uint64_t)base;
        const uint32_t lo32 = __builtin_amdgcn_readfirstlane((int)(uint32_t)begin), hi32 = __builtin_amdgcn_readfirstlane((int)(uint32_t)(begin >> 32));
        return __builtin_amdgcn_make_buffer_rsrc((void *)((uint64_t)hi32 << 32 | lo32), 0, __builtin_amdgcn_readfirstlane(rows > 0 ? (min(rows, 16) - 1) * (int)row + a.head_dim : 0), 0x00020000);
    };
    auto request = [&](int t) {
        const int key = key0 + t * KT;
        hold_pages(key);
        if constexpr (kCodes) {
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const int row0 = (j * NW + wave) * RPW;
                if (row0 >= KT) break;
                const int at = key + row0, page = page_of(at), place = at & in_page, r = at + my_row;
                const uint32_t off = r >= any_lo && my_piece < a.head_dim ? my_piece : 0x7ffffff0u;
                const auto src_k = rows_at(c.k_at(page, kv, place), c.k_row, any_hi - at), src_v = rows_at(c.v_at(page, kv, place), c.v_row, any_hi - at);
                const uint32_t off_k = off + (uint32_t)(my_row * (int)c.k_row), off_v = off + (uint32_t)(my_row * (int)c.v_row);
                if constexpr (kPiece == 16) {
                    const uint4v x = __builtin_amdgcn_raw_buffer_load_b128(src_k, off_k, 0, 0), y = __builtin_amdgcn_raw_buffer_load_b128(src_v, off_v, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) raw[j][0][i] = x[i], raw[j][1][i] = y[i];
                } else {
                    const uint2v x = __builtin_amdgcn_raw_buffer_load_b64(src_k, off_k, 0, 0), y = __builtin_amdgcn_raw_buffer_load_b64(src_v, off_v, 0, 0);
#pragma unroll
                    for (int i = 0; i < 2; ++i) raw[j][0][i] = x[i], raw[j][1][i] = y[i];
                }
                const int64_t first_scale = c.scale_at(page, kv, 0);
                const uint32_t mine = (uint32_t)((place + my_row) >> c.block_shift);
                scales[j][0] = (c.k_scale + first_scale)[mine], scales[j][1] = (c.v_scale + first_scale)[mine];
            }
        } else {
            constexpr int kStep = 1024 / Keys::kRowBytes;  // rows of a request
            static_assert(kStep <= 16);
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                char *to = tile_at(which, t);
#pragma unroll
                for (int i = 0; i < Keys::kBytes / 1024 / NW; ++i) {
                    const int block = (i * NW + wave) * 1024, row0 = block / Keys::kRowBytes, group = row0 & ~15;
                    // rows from any_lo on, up to any_hi, of the sixteen: others are taken as 0
                    const int at = key + group, place = at & in_page, valid = min(any_hi - at, 16);
                    const int page = page_of(at);
                    Keys::request_rows(to, which ? c.v_at(page, kv, place) : c.k_at(page, kv, place), which ? c.v_row : c.k_row, valid, max(any_lo - at, 0), a.head_dim * (int)sizeof(T), block, group, lane);
                }
            }
        }
    };
    auto place_codes = [&](int t) {
        if constexpr (kCodes) {
            const int key = key0 + t * KT;
            bool some[2] = {false, false};
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                const int row0 = (j * NW + wave) * RPW;
                if (row0 >= KT) break;
                const int r = row0 + my_row, at = key + r;
                const bool in = at >= any_lo && at < any_hi;
                if (kPiece == 16 && (a.head_dim & 8)) {  // (a head of 8 elements more than whole pieces: what follows them may be anything)
#pragma unroll
                    for (int i = 0; i < 4; ++i) raw[j][i & 1][2 + i / 2] = my_piece + 8 < a.head_dim ? raw[j][i & 1][2 + i / 2] : 0u;
                }
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    float rest;
                    const float by = fold<U, HELD>(in ? scales[j][which] : 1.f, rest);
                    some[which] = some[which] || rest != 1.f;
                    if (!in) rest = 0.f;  // (no key: no factor of its own, where the tile's factors are compared)
                    if (kHalves && my_piece == 0) left[place_of(which, t) * KT + r] = rest;
                    char *to = tile_at(which, t) + r * Keys::kRowBytes;
#pragma unroll
                    for (int i = 0; i < kPiece / 8; ++i) {
                        const Vec8 x = expand_by<U, HELD>(raw[j][which][2 * i], raw[j][which][2 * i + 1], by);
                        const int p = (my_piece + 8 * i) * (int)sizeof(U) / 16;
                        if constexpr (sizeof(U) == 2) {
                            *(Vec8 *)(to + ((p ^ Keys::turn(r)) << 4)) = x;
                        } else {
                            *(floatx4 *)(to + ((p ^ Keys::turn(r)) << 4)) = __builtin_shufflevector(x, x, 0, 1, 2, 3);
                            *(floatx4 *)(to + (((p + 1) ^ Keys::turn(r)) << 4)) = __builtin_shufflevector(x, x, 4, 5, 6, 7);
                        }
                    }
                }
            }
            if constexpr (kHalves) {
                const bool k_some = __any(some[0]), v_some = __any(some[1]);
                if (lane < 8 / NW) any_left[place_of(0, t) * 8 + wave * (8 / NW) + lane] = k_some, any_left[place_of(1, t) * 8 + wave * (8 / NW) + lane] = v_some;
            }
        }
    };
    uint2v some_left[2] = {{0u, 0u}, {0u, 0u}};  // of the tile in hand, read while its keys are multiplied
    auto any_of = [&](int which) { return __builtin_amdgcn_readfirstlane((int)(some_left[which].x | some_left[which].y)) != 0; };
    floatx16 x[KB];
    Vec8 p[2 * KB];
    // S^T = K Q^T, with operands two steps ahead: LDS answers after as long as four products take
    auto key_products = [&](int t) {
        const char *kt = tile_at(0, t);
        if constexpr (kHalves) {
#pragma unroll
            for (int which = 0; which < 2; ++which) some_left[which] = *(const uint2v *)(any_left + place_of(which, t) * 8);
        }
#pragma unroll
        for (int i = 0; i < KB; ++i) x[i] = zero16();
        constexpr int kAhead = sizeof(U) == 2 ? 2 : 0;
        Vec8 kx[kAhead + 1][KB];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int k = 0; k < KB; ++k) kx[i][k] = Keys::row_operand(kt, 32 * k, i, lane);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
            for (int k = 0; k < KB; ++k)
                if (i + kAhead < DP / 16) kx[(i + kAhead) % (kAhead + 1)][k] = Keys::row_operand(kt, 32 * k, i + kAhead, lane);
#pragma unroll
            for (int k = 0; k < KB; ++k) x[k] = Elem<U>::mma(kx[i % (kAhead + 1)][k], qf[i], x[k]);
            if constexpr (kAhead > 0) __builtin_amdgcn_sched_barrier(0);
        }
    };
    // scores to probabilities, with the maximum raised where it has to be
    auto weights = [&](int t) {
        const int key = key0 + t * KT;
        if constexpr (kHalves) {
            if (any_of(0)) {
                const float *by = left + place_of(0, t) * KT;
#pragma unroll
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const floatx4 f = *(const floatx4 *)(by + 32 * k + 8 * i + 4 * h);
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[k][4 * i + j] *= f[j];
                    }
            }
        }
        if constexpr (MOD) {
            if constexpr (!__is_same(T, U)) {
#pragma unroll
                for (int k = 0; k < KB; ++k) x[k] *= by_row;
            }
            if (bend.cap > 0.f) {
                bend.template apply<KB, false>(x, x);
            } else {
#pragma unroll
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[k][r] *= scale * kLog2e;
            }
            if (a.slopes) {
                const float at = (float)(pos - key - 4 * h);
#pragma unroll
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[k][r] = fmaf(-slope, fabsf(at - (float)(32 * k + 8 * (r >> 2) + (r & 3))), x[k][r]);
            }
        }
        if (key < full_lo || key + KT > full_hi) {
            const int at = key + 4 * h - lo;
            const uint32_t span = there && hi > lo ? hi - lo : 0;
#pragma unroll
            for (int k = 0; k < KB; ++k)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[k][r] = (uint32_t)(at + 32 * k + 8 * (r >> 2) + (r & 3)) < span ? x[k][r] : -INFINITY;
        }
        float top = x[0][0];
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, x[k][r]);
        top = halves_max(top);
        if (__any(top > m + raise)) {
            const float raised = fmaxf(m, top), by = raised == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - raised) * unit);
            m = raised;
            sum *= by, best *= by;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= by;
        }
        const float base = (m == -INFINITY ? 0.f : m * unit) - kShift;
        float sum_odd = 0.f;
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                x[k][r] = __builtin_amdgcn_exp2f(fmaf(x[k][r], unit, -base));
                (r & 1 ? sum_odd : sum) += x[k][r];
            }
        sum += sum_odd;
        if constexpr (kHalves) {
            // Weights: probabilities times what is left of values' scales, in units of a power of two of the row's own, so that its largest so far is from 2^7 to 2^15 of them
            // whatever the scales, those of other rows' keys among them (where all are 0 the unit stays).  1, and nothing to do, while no scale leaves anything.
            // (`largest` without an else: one would cost a hundred spilled registers)
            float largest = fmaxf(best, __builtin_amdgcn_exp2f(fmaf(top, unit, -base)) * 0x1p-15f);
            if (any_of(1) || __any(norm != 1.f)) {
                const float *by = left + place_of(1, t) * KT;
                float most = 0.f;
#pragma unroll
                for (int k = 0; k < KB; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const floatx4 f = *(const floatx4 *)(by + 32 * k + 8 * i + 4 * h) * 0x1p-15f;
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[k][4 * i + j] *= f[j], most = fmaxf(most, x[k][4 * i + j]);
                    }
                best = fmaxf(best, halves_max(most));
                largest = best;
                const bool change = best > norm || (best < norm * 0x1p-8f && best > 0.f);
                if (__any(change)) {
                    // (2^-111 and more, so that 2^15 of its reciprocals are a number)
                    const int e = best <= 1.f && best >= 0x1p-8f ? 0 : max(__builtin_amdgcn_frexp_expf(best), -111);
                    const float to = change ? __uint_as_float((uint32_t)(127 + e) << 23) : norm;
                    const int up = (int)(__float_as_uint(norm) >> 23) - (int)(__float_as_uint(to) >> 23);
                    norm = to;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[d][i] = __builtin_amdgcn_ldexpf(o[d][i], up);
                }
                const float in = __uint_as_float(0x7f000000u - __float_as_uint(norm)) * 0x1p15f;  // (a power of two's reciprocal)
#pragma unroll
                for (int k = 0; k < KB; ++k) x[k] *= in;
            }
            best = largest;
        }
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i) p[i] = operand<U>(x[i / 2], i & 1);
    };
    // O^T += V^T P^T, the next step's operands being under way
    auto value_products = [&](int t) {
        const char *vt = tile_at(1, t);
        constexpr int kSet = sizeof(U) == 2 ? 2 : 1;
        Vec8 vx[kSet][DB];
        if constexpr (kSet == 2) {
#pragma unroll
            for (int d = 0; d < DB; ++d) vx[0][d] = Keys::column_operand(vt, d, 0, lane);
        }
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i) {
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                if (kSet == 1) vx[0][d] = Keys::column_operand(vt, d, i, lane);
                else if (i + 1 < 2 * KB) vx[(i + 1) & 1][d] = Keys::column_operand(vt, d, i + 1, lane);
            }
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] = Elem<U>::mma(vx[kSet == 2 ? i & 1 : 0][d], p[i], o[d]);
        }
    };
    auto seen = [&](int t) { return key0 + t * KT + KT > wave_lo && key0 + t * KT < wave_hi; };
    if (first < last) {
        request(first);
        place_codes(first);
    }
    for (int t = first; t < last; ++t) {
        tiles_arrived();
        if (t + 1 < last) request(t + 1);
        if (seen(t)) {
            key_products(t);
            __builtin_amdgcn_s_setprio(1);
            weights(t);
            value_products(t);
            __builtin_amdgcn_s_setprio(0);
        }
        if (t + 1 < last) place_codes(t + 1);
    }

    sum = halves_sum(sum);
    m = m == -INFINITY ? m : m * unit - kShift;
    if constexpr (kHalves) {
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= norm;
    }
    const int64_t at = (e.lse0 + token) * a.n_heads + head, all = a.rows * a.n_heads;
    if (a.n_split > 1) {
        if (!there) return;
        float *to = a.part_o + (split * all + at) * a.head_dim;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = 32 * d + 8 * i + 4 * h;
                if (col < a.head_dim) *(floatx4 *)(to + col) = floatx4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            }
        if (h == 0) a.part_ml[split * all + at] = make_float2(m, sum);
        return;
    }
    if (there && a.lse && h == 0) a.lse[at] = (m + __builtin_amdgcn_logf(sum)) * kLn2;
    const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    __syncthreads();  // (the tiles have been read by all)
    store_turned<T, DP>(memory + wave * 64 * DP, o, by, a.head_dim, lane, [&](int r) -> T * {
        const int at_row = tile * kRows + wave * 32 + r, t = at_row / a.group;
        return at_row < n_rows ? (T *)o_base<T>(a, a.out, e, s, kv * a.group + at_row % a.group) + (int64_t)t * a.o_row : nullptr;
    });
}

}  // namespace sddmm
