// Attention over a cache in pages for few rows (gfx950): workgroups of four waves, and the sum of partial results of keys that were cut into pieces.
#include <algorithm>
#include "attention_paged_token.hpp"

namespace sddmm {

namespace {

// Two waves to a SIMD, but one for two tiles of rows over fp32 rows of 128 elements, which do not fit 256 registers (us with two, which spill, and one: 4 tokens of 42 users, 64 heads over 8,
// up to 1231 keys 166 and 112; 5 of 32, 16 over 4, 3000 108 and 77; 8 of one, 4096 24 and 19).
template <class T, int HELD, int DP, bool MOD, int R>
__global__ __launch_bounds__(256, sizeof(T) == 4 && HELD == kHeldOwn && DP == 128 && R == 2 ? 1 : 2)
void sddmm_attention_paged_token_kernel(const AttnArgs a, const CacheArgs c)
{
    typedef PagedToken<T, HELD, DP, MOD, R> Body;
    __shared__ __align__(16) char lds[Body::kLds];
    const uint32_t b = blockIdx.x / a.n_kv_heads;
    Body::run(a, c, blockIdx.x - b * a.n_kv_heads, b % a.n_split, b / a.n_split, lds);
}

template <class T, int HELD, int DP, int R>
hipError_t launch_dim(const AttnArgs &a, const CacheArgs &c, dim3 grid, hipStream_t st)
{
    const bool mod = a.cap > 0.f || a.slopes;
    return launch(mod ? sddmm_attention_paged_token_kernel<T, HELD, DP, true, R> : sddmm_attention_paged_token_kernel<T, HELD, DP, false, R>, grid, dim3(256), 0, st, a, c);
}
template <class T, int HELD, int R>
hipError_t launch_held(const AttnArgs &a, const CacheArgs &c, dim3 grid, hipStream_t st)
{
    if constexpr (sizeof(T) == 4) {
        if (a.head_dim <= 32) return launch_dim<T, HELD, 32, R>(a, c, grid, st);
    }
    return a.head_dim <= 64 ? launch_dim<T, HELD, 64, R>(a, c, grid, st) : launch_dim<T, HELD, 128, R>(a, c, grid, st);
}
template <class T, int R>
hipError_t launch_typed(const AttnArgs &a, const CacheArgs &c, int held, dim3 grid, hipStream_t st)
{
    return held == kHeldI8 ? launch_held<T, kHeldI8, R>(a, c, grid, st) : held == kHeldE4m3 ? launch_held<T, kHeldE4m3, R>(a, c, grid, st) : launch_held<T, kHeldOwn, R>(a, c, grid, st);
}
template <int R>
hipError_t launch_rows(const AttnArgs &a, const CacheArgs &c, int type, int held, dim3 grid, hipStream_t st)
{
    return type == SDDMM_TYPE_F32 ? launch_typed<float, R>(a, c, held, grid, st) : type == SDDMM_TYPE_F16 ? launch_typed<_Float16, R>(a, c, held, grid, st)
                                                                                                             : launch_typed<__bf16, R>(a, c, held, grid, st);
}

// The parts of a row: sums and totals in units of 2^(largest maximum).  Groups of DP / 4 lanes take parts in turn, N at a time with maxima and sums under way together, each
// with a running maximum of its own, and meet in LDS.  FEW: the parts of sequences of few rows beside others.
constexpr int kJoinThreads = 512;
template <class T, int DP, int N, bool FEW>
__device__ __forceinline__ void join_parts(const AttnArgs &a, int per_row, int block, floatx4 (&sums)[kJoinThreads / (DP / 4)][DP / 4], float2 (&stats)[kJoinThreads / (DP / 4)])
{
    constexpr int kLanes = DP / 4, kGroups = kJoinThreads / kLanes;
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, mine = group % per_row, col = lane * 4;
    const int64_t all = FEW ? (int64_t)a.n_seq * a.n_kv_heads * a.few_rows : a.rows * a.n_heads, at = (int64_t)block * (kGroups / per_row) + group / per_row;
    int64_t to_row = 0, to_lse = at;
    int head;
    bool there = at < all;
    if constexpr (FEW) {
        const int row = (int)(at % a.few_rows), kv = (int)(at / a.few_rows % a.n_kv_heads), s = (int)min(at / a.few_rows / a.n_kv_heads, (int64_t)a.n_seq - 1), token = row / a.group;
        const Seq e = sequence(a, s);
        head = kv * a.group + row % a.group;
        there = there && row < e.nq * a.group && e.nq * a.group <= a.few_rows;
        to_row = (e.q0 + token) * a.o_row, to_lse = (e.lse0 + token) * a.n_heads + head;
    } else {
        head = (int)(at % a.n_heads);
        const int64_t row = at / a.n_heads;
        if (a.q_ptr) {
            there = there && row >= a.q_ptr[0] && row < a.q_ptr[a.n_seq];
            to_row = row * a.o_row;
        } else if (there) {
            const int s = (int)(row / a.max_q), i = (int)(row % a.max_q);
            there = !a.q_len || i < min(a.q_len[s], a.max_q);
            to_row = s * a.o_seq + i * a.o_row;
        }
        if (there && a.few_rows && a.part_ml[at].y == kNone) there = false;
    }
    float top = -INFINITY, total = 0.f;
    floatx4 y = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = mine; there && p0 < a.n_part; p0 += N * per_row) {
        float2 ml[N];
        floatx4 x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int p = min(p0 + i * per_row, a.n_part - 1);
            ml[i] = a.part_ml[p * all + at];
            x[i] = col < a.head_dim ? *(const floatx4 *)(a.part_o + (p * all + at) * a.head_dim + col) : floatx4{0.f, 0.f, 0.f, 0.f};
        }
        float most = top;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (p0 + i * per_row >= a.n_part) ml[i] = make_float2(-INFINITY, 0.f);
            most = fmaxf(most, ml[i].x);
        }
        const float by = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - most);
        y *= by, total *= by, top = most;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (ml[i].x == -INFINITY) continue;  // (no keys: its sums were not written)
            const float w = __builtin_amdgcn_exp2f(ml[i].x - top);
            y += x[i] * w;
            total = fmaf(w, ml[i].y, total);
        }
    }
    if (per_row > 1) {
        sums[group][lane] = y;
        if (lane == 0) stats[group] = make_float2(top, total);
        __syncthreads();
        if (mine) return;
        float most = top;
        for (int g = 1; g < per_row; ++g) most = fmaxf(most, stats[group + g].x);
        const float by = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - most);
        y *= by, total *= by, top = most;
        for (int g = 1; g < per_row; ++g) {
            const float2 one = stats[group + g];
            if (one.x == -INFINITY) continue;
            const float w = __builtin_amdgcn_exp2f(one.x - top);
            y += sums[group + g][lane] * w;
            total = fmaf(w, one.y, total);
        }
    }
    if (!there) return;
    const float by = total > 0.f || total != total ? 1.f / total : 0.f;
    T *to = (T *)a.out + to_row + head * a.o_head;
    if (col < a.head_dim) *(typename Elem<T>::Vec4 *)(to + col) = __builtin_convertvector(y * by, typename Elem<T>::Vec4);
    if (a.lse && lane == 0) a.lse[to_lse] = (top + __builtin_amdgcn_logf(total)) * kLn2;
}
template <class T, int DP, int N>
__global__ __launch_bounds__(kJoinThreads)
void sddmm_attention_paged_join_kernel(const AttnArgs a, const int per_row)
{
    __shared__ floatx4 sums[kJoinThreads / (DP / 4)][DP / 4];
    __shared__ float2 stats[kJoinThreads / (DP / 4)];
    join_parts<T, DP, N, false>(a, per_row, blockIdx.x, sums, stats);
}
// The first n_first workgroups: a's parts; the others: those of `few`.
template <class T, int DP, int N>
__global__ __launch_bounds__(kJoinThreads)
void sddmm_attention_paged_join_both_kernel(const AttnArgs a, const int per_row, const AttnArgs few, const int per_row_few, const int n_first)
{
    __shared__ floatx4 sums[kJoinThreads / (DP / 4)][DP / 4];
    __shared__ float2 stats[kJoinThreads / (DP / 4)];
    if ((int)blockIdx.x < n_first) join_parts<T, DP, N, false>(a, per_row, blockIdx.x, sums, stats);
    else join_parts<T, DP, N, true>(few, per_row_few, blockIdx.x - n_first, sums, stats);
}

// lane groups of a workgroup of the kernel above, and how many of them share a row
int join_groups(int head_dim) { return kJoinThreads / ((head_dim <= 64 ? 64 : 128) / 4); }
int join_per_row(int n_part, int head_dim)
{
    int per_row = 1;
    while (per_row < join_groups(head_dim) && per_row * 2 < n_part) per_row *= 2;
    return per_row;
}
template <class T, int DP>
hipError_t launch_join_dim(const AttnArgs &a, const AttnArgs *few, hipStream_t st)
{
    const int per_row = join_per_row(a.n_part, a.head_dim), per_row_few = few ? join_per_row(few->n_part, a.head_dim) : 1;
    const unsigned first = a.n_part > 1 ? (unsigned)attention_paged_join_grid(a.rows * a.n_heads, a.n_part, a.head_dim) : 0;
    // As many at a time as a group has, up to eight (us of the whole call with 2 / 4 / 8: two parts, 2048 rows of 16 heads 309 / - / 312, 1053 of 32 heads 107 / - / 111; 64 parts - / 16.8 / 17.3;
    // 128 and 256 of one row - / 15.1 and 17.1 / 14.8 and 16.7).
    const int most = std::max((a.n_part + per_row - 1) / per_row, few ? (few->n_part + per_row_few - 1) / per_row_few : 0);
    if constexpr (sizeof(T) == 2) {
        if (few) {
            const unsigned second = (unsigned)attention_paged_join_grid((int64_t)few->n_seq * few->n_kv_heads * few->few_rows, few->n_part, a.head_dim);
            auto *fn = most <= 2 ? sddmm_attention_paged_join_both_kernel<T, DP, 2> : most <= 4 ? sddmm_attention_paged_join_both_kernel<T, DP, 4> : sddmm_attention_paged_join_both_kernel<T, DP, 8>;
            return launch(fn, dim3(first + second), dim3(kJoinThreads), 0, st, a, per_row, *few, per_row_few, (int)first);
        }
    }
    auto *fn = most <= 2 ? sddmm_attention_paged_join_kernel<T, DP, 2> : most <= 4 ? sddmm_attention_paged_join_kernel<T, DP, 4> : sddmm_attention_paged_join_kernel<T, DP, 8>;
    return launch(fn, dim3(first), dim3(kJoinThreads), 0, st, a, per_row);
}
template <class T>
hipError_t launch_join(const AttnArgs &a, const AttnArgs *few, hipStream_t st)
{
    return a.head_dim <= 64 ? launch_join_dim<T, 64>(a, few, st) : launch_join_dim<T, 128>(a, few, st);
}

}  // namespace

int64_t attention_paged_join_grid(int64_t rows_of_heads, int n_part, int head_dim)
{
    const int rows = join_groups(head_dim) / join_per_row(n_part, head_dim);
    return (rows_of_heads + rows - 1) / rows;
}

hipError_t launch_attention_paged_join(const AttnArgs &a, const AttnArgs *few, int type, hipStream_t st)
{
    return type == SDDMM_TYPE_F32 ? launch_join<float>(a, few, st) : type == SDDMM_TYPE_F16 ? launch_join<_Float16>(a, few, st) : launch_join<__bf16>(a, few, st);
}

hipError_t launch_attention_paged_token(const AttnArgs &a, const CacheArgs &c, int type, int held, int tiles, unsigned grid, hipStream_t st)
{
    return tiles == 1 ? launch_rows<1>(a, c, type, held, dim3(grid), st) : launch_rows<2>(a, c, type, held, dim3(grid), st);
}

}  // namespace sddmm
