// Launches of the attention over a cache in pages, for its entry point.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace sddmm {

struct AttnArgs;
struct CacheArgs;

// tiles: of 16 rows to a workgroup, 1 or 2; a.chunk: tiles of 32 keys to a piece
hipError_t launch_attention_paged_token(const AttnArgs &a, const CacheArgs &c, int type, int held, int tiles, unsigned grid, hipStream_t st);

// tile: rows of a workgroup, 128 or, of 16-bit heads of more than 64, 256
hipError_t launch_attention_paged_forward(const AttnArgs &a, const CacheArgs &c, int type, int held, int tile, unsigned grid, hipStream_t st);

// sequences of many rows (128 to a workgroup) and of few_rows at most (of 16 or 32); 16-bit operands
hipError_t launch_attention_paged_mixed(const AttnArgs &many, const AttnArgs &few, const CacheArgs &c, int type, int held, unsigned n_many, unsigned n_few, hipStream_t st);
int64_t attention_paged_join_grid(int64_t rows_of_heads, int n_part, int head_dim);  // workgroups of the join, of 512 threads
// a's parts, if it has any, and, where not null, those of `few`
hipError_t launch_attention_paged_join(const AttnArgs &a, const AttnArgs *few, int type, hipStream_t st);

}  // namespace sddmm
