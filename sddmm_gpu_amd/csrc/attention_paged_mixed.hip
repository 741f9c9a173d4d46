// Attention over a cache in pages for batches of sequences with many rows and with few (gfx950): one launch for both.
#include "attention_paged_launch.hpp"
#include "attention_paged_tile.hpp"
#include "attention_paged_token.hpp"
#include "launch.hpp"

namespace sddmm {

namespace {

// Pieces of prompts beside the newest tokens of other users: the first `n_many` workgroups take tiles of the sequences with more than few_rows rows, which are at their
// products, the others a piece of the cache of one with fewer, which wait for memory (three pieces of prompts beside 29 tokens, 1053 rows of 32 heads over 8 of 128, up to 4096 keys: 107 us
// with the join, 153 where tiles of 128 rows take the single tokens too).  Each leaves the other's sequences alone, since only the lengths on the device say which is which.
template <class T, int HELD, int DP, bool MOD, int R>
__global__ __launch_bounds__(256, 2)
void sddmm_attention_paged_mixed_kernel(const AttnArgs many, const AttnArgs few, const CacheArgs c, const int n_many)
{
    typedef PagedTile<T, HELD, DP, MOD, 4> First;
    typedef PagedToken<T, HELD, DP, MOD, R> Second;
    __shared__ __align__(1024) char lds[First::kLds > Second::kLds ? First::kLds : Second::kLds];
    if ((int)blockIdx.x < n_many) {
        First::run(many, c, blockIdx.x, *(char (*)[First::kLds])lds);
    } else {
        int b = blockIdx.x - n_many;
        const int kv = b % few.n_kv_heads;
        b /= few.n_kv_heads;
        Second::run(few, c, kv, b % few.n_split, b / few.n_split, *(char (*)[Second::kLds])lds);
    }
}

template <class T, int HELD, int DP, int R>
hipError_t launch_rows(const AttnArgs &many, const AttnArgs &few, const CacheArgs &c, unsigned n_many, unsigned n_few, hipStream_t st)
{
    const bool mod = many.cap > 0.f || many.slopes;
    return launch(mod ? sddmm_attention_paged_mixed_kernel<T, HELD, DP, true, R> : sddmm_attention_paged_mixed_kernel<T, HELD, DP, false, R>, dim3(n_many + n_few), dim3(256), 0, st, many, few, c,
                  (int)n_many);
}
template <class T, int HELD>
hipError_t launch_held(const AttnArgs &many, const AttnArgs &few, const CacheArgs &c, unsigned n_many, unsigned n_few, hipStream_t st)
{
    if (many.head_dim <= 64) return few.few_rows <= 16 ? launch_rows<T, HELD, 64, 1>(many, few, c, n_many, n_few, st) : launch_rows<T, HELD, 64, 2>(many, few, c, n_many, n_few, st);
    return few.few_rows <= 16 ? launch_rows<T, HELD, 128, 1>(many, few, c, n_many, n_few, st) : launch_rows<T, HELD, 128, 2>(many, few, c, n_many, n_few, st);
}
template <class T>
hipError_t launch_typed(const AttnArgs &many, const AttnArgs &few, const CacheArgs &c, int held, unsigned n_many, unsigned n_few, hipStream_t st)
{
    return held == kHeldI8 ? launch_held<T, kHeldI8>(many, few, c, n_many, n_few, st) : held == kHeldE4m3 ? launch_held<T, kHeldE4m3>(many, few, c, n_many, n_few, st)
                                                                                                       : launch_held<T, kHeldOwn>(many, few, c, n_many, n_few, st);
}

}  // namespace

hipError_t launch_attention_paged_mixed(const AttnArgs &many, const AttnArgs &few, const CacheArgs &c, int type, int held, unsigned n_many, unsigned n_few, hipStream_t st)
{
    return type == SDDMM_TYPE_F16 ? launch_typed<_Float16>(many, few, c, held, n_many, n_few, st) : launch_typed<__bf16>(many, few, c, held, n_many, n_few, st);
}

}  // namespace sddmm
