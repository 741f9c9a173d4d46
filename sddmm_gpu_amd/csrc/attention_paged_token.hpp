// Attention over a cache in pages for few rows (gfx950): the newest tokens of every sequence.
#pragma once
#include <type_traits>
#include "attention_paged.hpp"
#include "attention_paged_launch.hpp"
#include "launch.hpp"

namespace sddmm {

// The (token, head) pairs that share a key head are the rows, R tiles of 16: they read every key once.  Every wave of a workgroup takes keys of its own,
// each NW-th tile of 32, from memory to registers without LDS or a barrier: S^T = K Q^T with the keys' rows as they lie -- a lane takes pieces of its token's row, in
// the order that memory has, and q's elements are in that order too -- and O^T += V^T P^T, the probabilities as they lie, a lane taking DP / 16
// elements in a row of each of the eight tokens that its probabilities are of, so that element d of all lanes, over these tokens, is an operand after an exchange of bytes
// within the lane.  Codes are made 16-bit operands in registers (two instructions for two to four of them); scales go to scores and probabilities.
// The next keys are requested when the scores are done, the next values when the products are; waves have statistics and sums of their own, which
// are joined at the end.
//
// Bound by reading the caches where there are many (64 users of 284 to 8192 keys, 8 key heads of 128, 8 bits: 119 us, 4.6 TB/s; a large copy makes 4.7; vector instructions for 41 % of
// the time, matrix ones for 9), by chains of loads -- lengths, pages, keys, the next keys -- where there are few (4 users of up to 32,768 keys, 2 key heads: 13.2 us in 512 workgroups of
// four tiles a wave, compute units busy for 42 %).  Sixteen waves to a workgroup, which need no pieces and no join for one user, are slower: 16.2 us for 1501 keys where both launches
// take 10.2 (one compute unit's rate).
template <class T, int HELD, int DP, bool MOD, int R>
struct PagedToken {
    static constexpr int NW = 4;  // waves
    static constexpr int kLds = NW * 16 * (DP + 4) * 4 + NW * 16 * 8;
    static __device__ __forceinline__ void run(const AttnArgs &a, const CacheArgs &c, int kv, int split, int b, char (&memory)[kLds]);
};

template <class T, int HELD, int DP, bool MOD, int R>
__device__ __forceinline__ void PagedToken<T, HELD, DP, MOD, R>::run(const AttnArgs &a, const CacheArgs &c, int kv, int split, int b, char (&memory)[kLds])
{
    typedef typename Elem<T>::Vec8 Vec8;
    // What probabilities times scales and values' codes are multiplied in: fp16 rows over codes take bf16, whose range is that of the scales (in fp16 a value of 2^14 times the others,
    // whatever its probability, would cost the others' weights their bits).
    typedef std::conditional_t<__is_same(T, _Float16) && HELD != kHeldOwn, __bf16, T> W;
    typedef typename Elem<W>::Vec8 Weights;
    constexpr int KT = 32, S = DP / 32, E = DP / 16;           // keys of a tile, steps of a product over a head's elements, values' elements of a lane
    constexpr int kSize = HELD == kHeldOwn ? (int)sizeof(T) : 1;
    constexpr int kPiece = HELD != kHeldOwn && S > 1 ? 16 : 8 * kSize;  // bytes of a key's row that a lane takes at a time: of two steps, or of one
    constexpr int kKeyWords = S * 8 * kSize / 4;               // a lane's registers of a key's row
    constexpr int kValueBytes = E * kSize, kValueWords = (kValueBytes + 3) / 4;
    constexpr int kRows = 16 * R;
    auto &joined = *(float (*)[NW][16][DP + 4])memory;
    auto &ml = *(float2 (*)[NW][16])(memory + sizeof joined);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;

    int s, tile;
    if (a.q_ptr && a.max_tiles > 1) {
        s = slot_sequence<false>(a.q_ptr, a.n_seq, a.group, kRows, a.max_tiles, a.n_slots, b, tile);
        if (s < 0) return;
    } else if (a.max_tiles == 1) {
        s = b, tile = 0;
    } else {
        s = b % a.n_seq, tile = a.max_tiles - 1 - b / a.n_seq;
    }
    int pages0 = -64;  // the table's entries from here on are in lanes, 64 at a time
    uint32_t pages = 0;
    float scale_raw = 0.f;  // of the key of token `lane`, of the value of token `lane` - 32
    const float *scale_base = lane < 32 ? c.k_scale : c.v_scale;
    const Seq e = sequence(a, s);
    const int n_rows = e.nq * a.group, n_keys = c.n_pages > 0 ? e.nk : 0;
    if (tile * kRows >= n_rows || (a.few_rows && n_rows > a.few_rows)) return;
    const int shift = e.nk - e.nq, prefix = a.prefix ? a.prefix[s] : 0;
    const int t0 = tile * kRows / a.group, t1 = (min(n_rows, tile * kRows + kRows) - 1) / a.group;
    const int any_lo = first_key(a, t0 + shift), any_hi = end_key(a, t1 + shift, prefix, n_keys);
    const int full_lo = first_key(a, t1 + shift), full_hi = end_key(a, t0 + shift, prefix, n_keys);

    // tiles begin at multiples of 32, so that each half of one lies in a page
    const int key0 = any_lo & ~(KT - 1), n_tiles = any_hi > any_lo ? (any_hi - key0 + KT - 1) / KT : 0;
    const int first = split * a.chunk, last = min(n_tiles, first + a.chunk);

    int pos[R], lo[R], hi[R];
    float slope[R];
    Vec8 qf[R][S];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = tile * kRows + 16 * r + n;
        const bool there = row < n_rows;
        const int token = row / a.group, head = kv * a.group + row % a.group;
        pos[r] = token + shift;
        lo[r] = first_key(a, pos[r]), hi[r] = there ? end_key(a, pos[r], prefix, n_keys) : 0;
        slope[r] = MOD && a.slopes && there ? a.slopes[head] * kLog2e : 0.f;
        const T *q = q_base<T>(a, a.q, e, s, head) + (int64_t)token * a.q_row;
#pragma unroll
        for (int i = 0; i < S; ++i) qf[r][i] = global_operand<T>(q, there, kPiece == 16 && kSize == 1 ? 64 * (i / 2) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g, a.head_dim);
    }

    floatx4 o[R][E];
    float m[R], sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY, sum[r] = 0.f;
#pragma unroll
        for (int d = 0; d < E; ++d) o[r][d] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    const float scale = a.scale, unit = MOD ? 1.f : scale * kLog2e;
    Bend<T> bend;
    if constexpr (MOD) bend.init(scale, a.cap);

    // Places: the page of a half tile is the same for all lanes, a lane's place in it fits 32 bits.  What a half tile lacks -- rows behind the last key, all of a tile behind the
    // wave's last one, elements behind the head's end -- lies outside the range that its loads are given: it becomes 0 and is not read, and the requests are the same in every
    // tile, so that the waits for them are.
    constexpr int kLoads = S * 8 * kSize / kPiece;
    const int in_page = (1 << c.page_shift) - 1, row_bytes = a.head_dim * kSize;
    uint32_t k_off[kLoads], v_off[4];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int at = (kPiece == 16 && kSize == 1 ? 64 : 32 * kSize) * i + kPiece * g;
        k_off[i] = at < row_bytes ? (uint32_t)(n * (int)c.k_row) + at : 0x7ffffff0u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v_off[i] = kValueBytes * n < row_bytes ? (uint32_t)((4 * g + i) * (int)c.v_row) + kValueBytes * n : 0x7ffffff0u;
    int page0 = 0, page1 = 0;  // of the halves of the tile whose keys, and then values, are requested (no array: indexed by a lane's number it would be one in memory)
    uint32_t k_raw[2][kKeyWords], v_raw[8][kValueWords];
    auto range = [&](const char *base, uint32_t row, int key, int t) {
        const uint64_t begin = (uint64_t)base;
        const int rows = t < last ? min(any_hi - key, 16) : 0;
        const uint32_t lo32 = __builtin_amdgcn_readfirstlane((int)(uint32_t)begin), hi32 = __builtin_amdgcn_readfirstlane((int)(uint32_t)(begin >> 32));
        return __builtin_amdgcn_make_buffer_rsrc((void *)((uint64_t)hi32 << 32 | lo32), 0, __builtin_amdgcn_readfirstlane(rows > 0 ? (rows - 1) * (int)row + row_bytes : 0), 0x00020000);
    };
    auto request_keys = [&](int t) {
        const int last_page = (n_keys - 1) >> c.page_shift, i0 = min((key0 + t * KT) >> c.page_shift, last_page), i1 = min((key0 + t * KT + 16) >> c.page_shift, last_page);
        if (i0 < pages0 || i1 - pages0 >= 64) {
            pages0 = i0;
            pages = c.page(s, min(i0 + lane, last_page));
        }
        page0 = __builtin_amdgcn_readlane((int)pages, i0 - pages0), page1 = __builtin_amdgcn_readlane((int)pages, i1 - pages0);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int key = key0 + t * KT + 16 * u;
            const auto src = range(c.k_at(u ? page1 : page0, kv, key & in_page), c.k_row, key, t);
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                constexpr int W = kPiece / 4;
                if constexpr (W == 2) {
                    const uint2v x = __builtin_amdgcn_raw_buffer_load_b64(src, k_off[j], 0, 0);
                    k_raw[u][2 * j] = x.x, k_raw[u][2 * j + 1] = x.y;
                } else {
#pragma unroll
                    for (int w = 0; w < W / 4; ++w) {
                        const uint4v x = __builtin_amdgcn_raw_buffer_load_b128(src, k_off[j] + 16 * w, 0, 0);
#pragma unroll
                        for (int k = 0; k < 4; ++k) k_raw[u][W * j + 4 * w + k] = x[k];
                    }
                }
            }
        }
        if constexpr (HELD != kHeldOwn) {
            const int at = (key0 + t * KT + (lane & 31)) & in_page;
            scale_raw = scale_base[c.scale_at(lane & 16 ? page1 : page0, kv, at)];
        }
        __builtin_amdgcn_sched_barrier(0);  // (keys' requests before values' everywhere, or the waits for keys would be for both)
    };
    auto request_values = [&](int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int key = key0 + t * KT + 16 * u;
            const auto src = range(c.v_at(u ? page1 : page0, kv, key & in_page), c.v_row, key, t);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t (&to)[kValueWords] = v_raw[4 * u + i];
                if constexpr (kValueBytes == 2) to[0] = __builtin_amdgcn_raw_buffer_load_b16(src, v_off[i], 0, 0);
                else if constexpr (kValueBytes == 4) to[0] = __builtin_amdgcn_raw_buffer_load_b32(src, v_off[i], 0, 0);
                else if constexpr (kValueBytes == 8) {
                    const uint2v x = __builtin_amdgcn_raw_buffer_load_b64(src, v_off[i], 0, 0);
                    to[0] = x.x, to[1] = x.y;
                } else {
#pragma unroll
                    for (int w = 0; w < kValueWords / 4; ++w) {
                        const uint4v x = __builtin_amdgcn_raw_buffer_load_b128(src, v_off[i] + 16 * w, 0, 0);
#pragma unroll
                        for (int j = 0; j < 4; ++j) to[4 * w + j] = x[j];
                    }
                }
            }
        }
    };

    int t = first + wave;
    if (t < last) {
        request_keys(t);
        request_values(t);
    }
    for (; t < last; t += NW) {
        const int key = key0 + t * KT;
        floatx4 x[R][2];
        // (a head of 8 elements more than whole pieces: a piece's second half may be anything)
        if constexpr (kSize == 1 && kPiece == 16) {
            if (a.head_dim & 8) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < kKeyWords; ++i)
                        if (i % 4 >= 2) k_raw[u][i] = 64 * (i / 4) + 16 * g + 8 < a.head_dim ? k_raw[u][i] : 0u;
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int r = 0; r < R; ++r) x[r][u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < S; ++i) {
                Vec8 k;
                if constexpr (HELD != kHeldOwn) k = expand<T, HELD>(k_raw[u][2 * i], k_raw[u][2 * i + 1]);
                else {
                    typedef uint32_t Words __attribute__((ext_vector_type(2 * sizeof(T))));
                    Words w;
#pragma unroll
                    for (int j = 0; j < 2 * (int)sizeof(T); ++j) w[j] = k_raw[u][2 * sizeof(T) * i + j];
                    k = __builtin_bit_cast(Vec8, w);
                }
#pragma unroll
                for (int r = 0; r < R; ++r) x[r][u] = mma16<T>(k, qf[r][i], x[r][u]);
            }
        }
        float y[R][8], kk[8], vv[8];
        if constexpr (HELD != kHeldOwn) {
            // the scales of the lane's eight tokens, from the lanes that have them; one for four tokens where blocks are as long
            if (c.block_shift >= 2) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    kk[4 * u] = __shfl(scale_raw, 16 * u + 4 * g), vv[4 * u] = __shfl(scale_raw, 32 + 16 * u + 4 * g);
#pragma unroll
                    for (int i = 1; i < 4; ++i) kk[4 * u + i] = kk[4 * u], vv[4 * u + i] = vv[4 * u];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int from = 16 * (j >> 2) + 4 * g + (j & 3);
                    kk[j] = __shfl(scale_raw, from), vv[j] = __shfl(scale_raw, 32 + from);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < 8; ++j) y[r][j] = HELD != kHeldOwn ? x[r][j >> 2][j & 3] * kk[j] : x[r][j >> 2][j & 3];
        request_keys(t + NW);

        const bool edge = key < full_lo || key + KT > full_hi;
        float top[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (MOD) {
                if (bend.cap > 0.f) {
                    bend_scores(bend, y[r]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[r][j] *= scale * kLog2e;
                }
                if (a.slopes) {
                    const float at = (float)(pos[r] - key - 4 * g);
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[r][j] = fmaf(-slope[r], fabsf(at - (float)(16 * (j >> 2) + (j & 3))), y[r][j]);
                }
            }
            if (edge) {
                const int at = key + 4 * g - lo[r];
                const uint32_t span = hi[r] > lo[r] ? hi[r] - lo[r] : 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) y[r][j] = (uint32_t)(at + 16 * (j >> 2) + (j & 3)) < span ? y[r][j] : -INFINITY;
            }
            top[r] = y[r][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) top[r] = fmaxf(top[r], y[r][j]);
            top[r] = groups_max(top[r]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float raised = fmaxf(m[r], top[r]);
            if (__any(raised > m[r])) {
                const float by = raised == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[r] - raised) * unit);
                m[r] = raised;
                sum[r] *= by;
#pragma unroll
                for (int d = 0; d < E; ++d) o[r][d] *= by;
            }
            const float base = m[r] == -INFINITY ? 0.f : m[r] * unit;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[r][j] = __builtin_amdgcn_exp2f(fmaf(y[r][j], unit, -base));
                sum[r] += y[r][j];
            }
        }

        // values before the rows' keys may hold anything, and so may scales of what is no key of theirs
        if (key < any_lo || key + KT > any_hi) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int token = key + 4 * g + 16 * (j >> 2) + (j & 3);
                const bool in = token >= any_lo && token < any_hi;
#pragma unroll
                for (int w = 0; w < kValueWords; ++w) v_raw[j][w] = in ? v_raw[j][w] : 0u;
                vv[j] = in ? vv[j] : 0.f;
            }
        }
        // Probabilities as operands; 16 bits: with a second one for what the first, of 8 or 11 bits, leaves: an output is then off by its own rounding only (bf16: 0.0017 of its size, 0.0026
        // with one operand and few keys), for 1 % of the time, since products are far from what bounds this kernel (64 users of up to 8192 keys, 122 and 123 us).
        constexpr bool kRest = sizeof(T) == 2;
        Weights p[R], rest[kRest ? R : 1];
        auto round = [&](int r, const floatx8 &f) {
            p[r] = __builtin_convertvector(f, Weights);
            if constexpr (kRest) rest[r] = __builtin_convertvector(f - __builtin_convertvector(p[r], floatx8), Weights);
        };
        if constexpr (HELD != kHeldOwn) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                floatx8 f;
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = y[r][j] * vv[j];
                round(r, f);
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                floatx8 f;
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = y[r][j];
                round(r, f);
            }
        }
        auto add = [&](const Weights &v, int r, int d) {
            o[r][d] = mma16<W>(v, p[r], o[r][d]);
            if constexpr (kRest) o[r][d] = mma16<W>(v, rest[r], o[r][d]);
        };
        // element d of the lane's elements, of its eight tokens
        if constexpr (HELD != kHeldOwn) {
#pragma unroll
            for (int q = 0; q < (E + 3) / 4; ++q) {
                uint32_t x0[4], x1[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x0[j] = v_raw[j][q], x1[j] = v_raw[4 + j][q];
                turn4(x0);
                turn4(x1);
#pragma unroll
                for (int d = 0; d < (E < 4 ? E : 4); ++d) {
                    const Weights v = expand<W, HELD>(x0[d], x1[d]);
#pragma unroll
                    for (int r = 0; r < R; ++r) add(v, r, 4 * q + d);
                }
            }
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int d = 0; d < E; ++d) {
                uint4v w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = __builtin_amdgcn_perm(v_raw[2 * j + 1][d / 2], v_raw[2 * j][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
                const Weights v = __builtin_bit_cast(Weights, w);
#pragma unroll
                for (int r = 0; r < R; ++r) add(v, r, d);
            }
        } else {
#pragma unroll
            for (int d = 0; d < E; ++d) {
                Weights v;
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(v_raw[j][d]);
#pragma unroll
                for (int r = 0; r < R; ++r) add(v, r, d);
            }
        }
        request_values(t + NW);
    }

    // join the waves, 16 rows at a time: a lane holds DP / 4 elements in a row of its row
    const bool parts = a.n_part > 1;
    const int64_t all = a.few_rows ? (int64_t)a.n_seq * a.n_kv_heads * a.few_rows : a.rows * a.n_heads;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float total_of_wave = groups_sum(sum[r]);
        if (r) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < E; ++d) joined[wave][n][E * (4 * g + i) + d] = o[r][d][i];
        if (g == 0) ml[wave][n] = make_float2(m[r] == -INFINITY ? m[r] : m[r] * unit, total_of_wave);
        __syncthreads();
        constexpr int kEach = 16 * DP / 4 / (64 * NW);  // pieces of four elements to a thread
        static_assert(kEach * 64 * NW * 4 == 16 * DP || 16 * DP / 4 < 64 * NW);
#pragma unroll
        for (int i = 0; i < (kEach > 0 ? kEach : 1); ++i) {
            const int piece = i * 64 * NW + threadIdx.x, row_at = piece / (DP / 4), col = piece % (DP / 4) * 4;
            const int row = tile * kRows + 16 * r + row_at;
            if (row_at >= 16 || row >= n_rows) continue;
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[w][row_at].x);
            floatx4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float2 one = ml[w][row_at];
                const float by = one.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(one.x - top);
                total = fmaf(by, one.y, total);
                const floatx4 y = *(const floatx4 *)&joined[w][row_at][col];
                if (one.x != -INFINITY) z += y * by;
            }
            const int token = row / a.group, head = kv * a.group + row % a.group;
            const int64_t at = (e.lse0 + token) * a.n_heads + head;
            if (a.not_ml && split == 0 && col == 0) a.not_ml[at] = make_float2(-INFINITY, kNone);
            if (parts) {
                const int64_t to = split * all + (a.few_rows ? ((int64_t)s * a.n_kv_heads + kv) * a.few_rows + row : at);
                if (top != -INFINITY && col < a.head_dim) *(floatx4 *)(a.part_o + to * a.head_dim + col) = z;
                if (col == 0) a.part_ml[to] = make_float2(top, total);
            } else {
                z *= total > 0.f || total != total ? 1.f / total : 0.f;
                T *to = (T *)o_base<T>(a, a.out, e, s, head) + (int64_t)token * a.o_row;
                if (col < a.head_dim) *(typename Elem<T>::Vec4 *)(to + col) = __builtin_convertvector(z, typename Elem<T>::Vec4);
                if (a.lse && col == 0) a.lse[at] = (top + __builtin_amdgcn_logf(total)) * kLn2;
            }
        }
    }
}

}  // namespace sddmm
