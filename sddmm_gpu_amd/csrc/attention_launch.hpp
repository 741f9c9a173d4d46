// Launches of the dense attention kernels, for the entry points.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace sddmm {

struct AttnArgs;

enum { kRowsOfHead = 0, kRowsPacked = 1, kRowsShared = 2 };  // what the rows of a forward workgroup are (attention_tile.hpp)

constexpr int kAttentionThreads = 256;  // of a workgroup, at least (the backward pass takes 512 where there are up to 512 workgroups)
constexpr int kTokenRows = 32;  // of a workgroup of the kernel for few rows
// tile: rows of a workgroup, 128 or 64
hipError_t launch_attention_forward(const AttnArgs &a, int type, int rows, int tile, unsigned grid, hipStream_t st);
hipError_t launch_attention_token(const AttnArgs &a, int type, unsigned grid, hipStream_t st);
int64_t attention_sum_grid(int64_t kv_grid, int splits, int keys, int padded_dim, int slope_heads);  // workgroups of the last launch, at most
// a: the dealing out of keys (dk, dv); b: of rows (dq)
// keys: of a dk, dv workgroup, 128, 64 or 32; q_rows: rows of a dq workgroup, 128, 64 or 32
hipError_t launch_attention_backward(const AttnArgs &a, const AttnArgs &b, int type, unsigned kv_grid, int keys, unsigned q_grid, int q_rows, hipStream_t st);
// a: the shared keys (kRowsShared, tile as above); own: each sequence's, by the kernel for few rows
hipError_t launch_attention_shared(const AttnArgs &a, const AttnArgs &own, int type, int tile, unsigned n_shared, unsigned n_own, hipStream_t st);
int64_t attention_join_grid(int64_t rows_of_heads, int n_part, int head_dim);  // its workgroups
hipError_t launch_attention_join(const AttnArgs &a, int type, hipStream_t st);

}  // namespace sddmm
