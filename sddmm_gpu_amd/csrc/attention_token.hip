// Dense attention for few rows (gfx950): the kernel, and the sum of partial results of keys that were cut into pieces.
#include "attention_token.hpp"
#include "launch.hpp"

namespace sddmm {

namespace {

template <class T, int DP, bool MOD, int NW>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 4 && DP == 128 ? 1 : 2)
void sddmm_attention_token_kernel(const AttnArgs a)
{
    typedef TokenTile<T, DP, MOD, NW> Body;
    __shared__ __align__(1024) char lds[Body::kLds];
    Body::run(a, blockIdx.x, lds);
}

// The partial results of a row: weights 2^(m - largest m), sums of both.  Groups of head_dim / 4 lanes take the parts of a row in turn,
// as many groups to a row as it has parts (up to the workgroup's), with all requests under way together, and meet in LDS.  4 to 6 us: latency of a launch
// and of two dependent loads.  (Its own launch: the last workgroup to finish would have to be known by a counter that every call finds at 0, which the workspace,
// anyone's between calls, does not hold.)
constexpr int kJoinBlock = 256;
template <class T, int DP>
__global__ __launch_bounds__(kJoinBlock)
void sddmm_attention_join_kernel(const AttnArgs a, const int per_row)
{
    constexpr int kLanes = DP / 4, kGroups = kJoinBlock / kLanes;
    __shared__ floatx4 sums[kGroups][kLanes];
    __shared__ float totals[kGroups];
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, mine = group % per_row, col = lane * 4;
    const int64_t all = a.rows * a.n_heads, at = (int64_t)blockIdx.x * (kGroups / per_row) + group / per_row;
    const int head = (int)(at % a.n_heads);
    const int64_t row = at / a.n_heads;
    int64_t to_row = 0;
    bool there = at < all;
    if (a.q_ptr) {
        there = there && row >= a.q_ptr[0] && row < a.q_ptr[a.n_seq];
        to_row = row * a.o_row;
    } else if (there) {
        const int s = (int)(row / a.max_q), i = (int)(row % a.max_q);
        there = !a.q_len || i < min(a.q_len[s], a.max_q);
        to_row = s * a.o_seq + i * a.o_row;
    }
    float top = -INFINITY, total = 0.f;
    floatx4 y = {0.f, 0.f, 0.f, 0.f};
    if (there) {
        for (int p = lane; p < a.n_part; p += kLanes) top = fmaxf(top, a.part_ml[p * all + at].x);
#pragma unroll
        for (int d = 1; d < kLanes; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
#pragma unroll 4
        for (int p = mine; p < a.n_part; p += per_row) {
            const float2 ml = a.part_ml[p * all + at];
            const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
            const floatx4 x = col < a.head_dim && ml.x != -INFINITY ? *(const floatx4 *)(a.part_o + (p * all + at) * a.head_dim + col) : floatx4{0.f, 0.f, 0.f, 0.f};
            y += x * w;
            total = fmaf(w, ml.y, total);
        }
    }
    if (per_row > 1) {
        sums[group][lane] = y;
        if (lane == 0) totals[group] = total;
        __syncthreads();
        if (mine) return;
        for (int g = 1; g < per_row; ++g) {
            y += sums[group + g][lane];
            total += totals[group + g];
        }
    }
    if (!there) return;
    const float by = total > 0.f || total != total ? 1.f / total : 0.f;
    T *to = (T *)a.out + to_row + head * a.o_head;
    if (col < a.head_dim) *(typename Elem<T>::Vec4 *)(to + col) = __builtin_convertvector(y * by, typename Elem<T>::Vec4);
    if (a.lse && lane == 0) a.lse[at] = (top + __builtin_amdgcn_logf(total)) * kLn2;
}

template <class T, int DP>
hipError_t launch_typed(const AttnArgs &a, bool mod, unsigned grid, hipStream_t st)
{
    constexpr int NW = 4;
    return launch(mod ? sddmm_attention_token_kernel<T, DP, true, NW> : sddmm_attention_token_kernel<T, DP, false, NW>, dim3(grid), dim3(64 * NW), 0, st, a);
}

// lane groups of a workgroup of the kernel above, and how many of them share a row
int join_groups(int head_dim) { return kJoinBlock / ((head_dim <= 64 ? 64 : 128) / 4); }
int join_per_row(int n_part, int head_dim)
{
    int per_row = 1;
    while (per_row < join_groups(head_dim) && per_row < n_part) per_row *= 2;
    return per_row;
}

template <class T, int DP>
hipError_t join_typed(const AttnArgs &a, hipStream_t st)
{
    return launch(sddmm_attention_join_kernel<T, DP>, dim3((unsigned)attention_join_grid(a.rows * a.n_heads, a.n_part, a.head_dim)), dim3(kJoinBlock), 0, st, a,
                  join_per_row(a.n_part, a.head_dim));
}
template <class T>
hipError_t join_dims(const AttnArgs &a, hipStream_t st)
{
    return a.head_dim <= 64 ? join_typed<T, 64>(a, st) : join_typed<T, 128>(a, st);
}

}  // namespace

int64_t attention_join_grid(int64_t rows_of_heads, int n_part, int head_dim)
{
    const int rows = join_groups(head_dim) / join_per_row(n_part, head_dim);
    return (rows_of_heads + rows - 1) / rows;
}

hipError_t launch_attention_token(const AttnArgs &a, int type, unsigned grid, hipStream_t st)
{
    const bool mod = a.cap > 0.f || a.slopes;
    if (a.head_dim <= 32 && type == SDDMM_TYPE_F32) return launch_typed<float, 32>(a, mod, grid, st);
    if (a.head_dim <= 64)
        return type == SDDMM_TYPE_F32 ? launch_typed<float, 64>(a, mod, grid, st)
             : type == SDDMM_TYPE_F16 ? launch_typed<_Float16, 64>(a, mod, grid, st) : launch_typed<__bf16, 64>(a, mod, grid, st);
    return type == SDDMM_TYPE_F32 ? launch_typed<float, 128>(a, mod, grid, st)
         : type == SDDMM_TYPE_F16 ? launch_typed<_Float16, 128>(a, mod, grid, st) : launch_typed<__bf16, 128>(a, mod, grid, st);
}

hipError_t launch_attention_join(const AttnArgs &a, int type, hipStream_t st)
{
    return type == SDDMM_TYPE_F32 ? join_dims<float>(a, st) : type == SDDMM_TYPE_F16 ? join_dims<_Float16>(a, st) : join_dims<__bf16>(a, st);
}

}  // namespace sddmm
