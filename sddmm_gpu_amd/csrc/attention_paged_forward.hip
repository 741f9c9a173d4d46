// Attention over a cache in pages for many rows (gfx950).
#include "attention_paged_launch.hpp"
#include "attention_paged_tile.hpp"
#include "launch.hpp"

namespace sddmm {

namespace {

template <class T, int HELD, int DP, bool MOD, int NW>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 4 && DP == 128 ? 1 : 2)
void sddmm_attention_paged_kernel(const AttnArgs a, const CacheArgs c)
{
    typedef PagedTile<T, HELD, DP, MOD, NW> Body;
    __shared__ __align__(1024) char lds[Body::kLds];
    Body::run(a, c, blockIdx.x, lds);
}

template <class T, int HELD, int DP>
hipError_t launch_dim(const AttnArgs &a, const CacheArgs &c, int tile, unsigned grid, hipStream_t st)
{
    const bool mod = a.cap > 0.f || a.slopes;
    if constexpr (sizeof(T) == 2 && DP == 128) {
        if (tile == 256) return launch(mod ? sddmm_attention_paged_kernel<T, HELD, DP, true, 8> : sddmm_attention_paged_kernel<T, HELD, DP, false, 8>, dim3(grid), dim3(512), 0, st, a, c);
    }
    return launch(mod ? sddmm_attention_paged_kernel<T, HELD, DP, true, 4> : sddmm_attention_paged_kernel<T, HELD, DP, false, 4>, dim3(grid), dim3(256), 0, st, a, c);
}
template <class T, int HELD>
hipError_t launch_held(const AttnArgs &a, const CacheArgs &c, int tile, unsigned grid, hipStream_t st)
{
    if constexpr (sizeof(T) == 4) {
        if (a.head_dim <= 32) return launch_dim<T, HELD, 32>(a, c, tile, grid, st);
    }
    return a.head_dim <= 64 ? launch_dim<T, HELD, 64>(a, c, tile, grid, st) : launch_dim<T, HELD, 128>(a, c, tile, grid, st);
}
template <class T>
hipError_t launch_typed(const AttnArgs &a, const CacheArgs &c, int held, int tile, unsigned grid, hipStream_t st)
{
    return held == kHeldI8 ? launch_held<T, kHeldI8>(a, c, tile, grid, st) : held == kHeldE4m3 ? launch_held<T, kHeldE4m3>(a, c, tile, grid, st) : launch_held<T, kHeldOwn>(a, c, tile, grid, st);
}

}  // namespace

hipError_t launch_attention_paged_forward(const AttnArgs &a, const CacheArgs &c, int type, int held, int tile, unsigned grid, hipStream_t st)
{
    return type == SDDMM_TYPE_F32 ? launch_typed<float>(a, c, held, tile, grid, st) : type == SDDMM_TYPE_F16 ? launch_typed<_Float16>(a, c, held, tile, grid, st) : launch_typed<__bf16>(a, c, held, tile, grid, st);
}

}  // namespace sddmm
