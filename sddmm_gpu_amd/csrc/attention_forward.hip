// Dense attention, forward (gfx950): the kernels of one tile of rows to a workgroup.
#include "attention_tile.hpp"
#include "launch.hpp"

namespace sddmm {

namespace {

template <class T, int DP, bool MOD, int ROWS, int RW>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 && DP == 128 ? 1 : sizeof(T) == 2 && DP == 64 && !MOD ? 4 : 2)
void sddmm_attention_forward_kernel(const AttnArgs a)
{
    typedef ForwardTile<T, DP, MOD, ROWS, RW> Body;
    __shared__ __align__(1024) char lds[Body::kLds];
    Body::run(a, blockIdx.x, lds);
}

template <class T, int DP, bool MOD>
hipError_t launch_rows(const AttnArgs &a, int rows, int tile, unsigned grid, hipStream_t st)
{
    void (*fn)(AttnArgs) = rows == kRowsPacked ? (tile == 64 ? sddmm_attention_forward_kernel<T, DP, MOD, kRowsPacked, 2> : sddmm_attention_forward_kernel<T, DP, MOD, kRowsPacked, 4>)
                              : (tile == 64 ? sddmm_attention_forward_kernel<T, DP, MOD, kRowsOfHead, 2> : sddmm_attention_forward_kernel<T, DP, MOD, kRowsOfHead, 4>);
    return launch(fn, dim3(grid), dim3(64 * kWaves), 0, st, a);
}

template <class T>
hipError_t launch_typed(const AttnArgs &a, int rows, int tile, unsigned grid, hipStream_t st)
{
    const bool mod = a.cap > 0.f || a.slopes;
    if constexpr (sizeof(T) == 4) {
        if (a.head_dim <= 32) return mod ? launch_rows<T, 32, true>(a, rows, tile, grid, st) : launch_rows<T, 32, false>(a, rows, tile, grid, st);
    }
    if (a.head_dim <= 64) return mod ? launch_rows<T, 64, true>(a, rows, tile, grid, st) : launch_rows<T, 64, false>(a, rows, tile, grid, st);
    return mod ? launch_rows<T, 128, true>(a, rows, tile, grid, st) : launch_rows<T, 128, false>(a, rows, tile, grid, st);
}

}  // namespace

hipError_t launch_attention_forward(const AttnArgs &a, int type, int rows, int tile, unsigned grid, hipStream_t st)
{
    return type == SDDMM_TYPE_F32 ? launch_typed<float>(a, rows, tile, grid, st)
         : type == SDDMM_TYPE_F16 ? launch_typed<_Float16>(a, rows, tile, grid, st) : launch_typed<__bf16>(a, rows, tile, grid, st);
}

}  // namespace sddmm
