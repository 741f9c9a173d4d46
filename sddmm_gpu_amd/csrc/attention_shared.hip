// Dense attention of sequences that begin with the same keys (gfx950): one launch for both parts of the keys.
#include "attention_tile.hpp"
#include "attention_token.hpp"
#include "launch.hpp"

namespace sddmm {

namespace {

// The first `n_shared` workgroups take the rows of all sequences against the shared keys, which are read once for RW * 32 of them; the
// others a sequence's own keys.  Both leave partial results.  In one launch the two fill the card together: 48 sequences of 32 heads over 8 behind
// 16,000 keys, 25 to 700 of their own: 61 us in two launches, 47 in one.
template <class T, int DP, bool MOD, int RW>
__global__ __launch_bounds__(64 * kWaves, sizeof(T) == 4 && DP == 128 ? 1 : 2)
void sddmm_attention_shared_kernel(const AttnArgs a, const AttnArgs own, const int n_shared)
{
    typedef ForwardTile<T, DP, MOD, kRowsShared, RW> First;
    typedef TokenTile<T, DP, MOD, kWaves> Second;
    __shared__ __align__(1024) char lds[First::kLds > Second::kLds ? First::kLds : Second::kLds];
    if ((int)blockIdx.x < n_shared) First::run(a, blockIdx.x, *(char (*)[First::kLds])lds);
    else Second::run(own, blockIdx.x - n_shared, *(char (*)[Second::kLds])lds);
}

template <class T, int DP, bool MOD>
hipError_t launch_typed(const AttnArgs &a, const AttnArgs &own, int tile, unsigned n_shared, unsigned n_own, hipStream_t st)
{
    return launch(tile == 64 ? sddmm_attention_shared_kernel<T, DP, MOD, 2> : sddmm_attention_shared_kernel<T, DP, MOD, 4>, dim3(n_shared + n_own),
                  dim3(64 * kWaves), 0, st, a, own, (int)n_shared);
}
template <class T>
hipError_t launch_dims(const AttnArgs &a, const AttnArgs &own, int tile, unsigned n_shared, unsigned n_own, hipStream_t st)
{
    const bool mod = a.cap > 0.f || a.slopes;
    if constexpr (sizeof(T) == 4) {
        if (a.head_dim <= 32) return mod ? launch_typed<T, 32, true>(a, own, tile, n_shared, n_own, st) : launch_typed<T, 32, false>(a, own, tile, n_shared, n_own, st);
    }
    if (a.head_dim <= 64) return mod ? launch_typed<T, 64, true>(a, own, tile, n_shared, n_own, st) : launch_typed<T, 64, false>(a, own, tile, n_shared, n_own, st);
    return mod ? launch_typed<T, 128, true>(a, own, tile, n_shared, n_own, st) : launch_typed<T, 128, false>(a, own, tile, n_shared, n_own, st);
}

}  // namespace

hipError_t launch_attention_shared(const AttnArgs &a, const AttnArgs &own, int type, int tile, unsigned n_shared, unsigned n_own, hipStream_t st)
{
    return type == SDDMM_TYPE_F32 ? launch_dims<float>(a, own, tile, n_shared, n_own, st)
         : type == SDDMM_TYPE_F16 ? launch_dims<_Float16>(a, own, tile, n_shared, n_own, st) : launch_dims<__bf16>(a, own, tile, n_shared, n_own, st);
}

}  // namespace sddmm
