// Launches of the attention over a cache in pages, for its entry point.
#pragma once
#include <hip/hip_runtime.h>

namespace sddmm {

struct AttnArgs;
struct CacheArgs;

// tiles: of 16 rows to a workgroup, 1 or 2; a.chunk: tiles of 32 keys to a piece
hipError_t launch_attention_paged_token(const AttnArgs &a, const CacheArgs &c, int type, int held, int tiles, unsigned grid, hipStream_t st);

// 128 rows to a workgroup
hipError_t launch_attention_paged_forward(const AttnArgs &a, const CacheArgs &c, int type, int held, unsigned grid, hipStream_t st);

}  // namespace sddmm
