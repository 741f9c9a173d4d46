// Launches of the dense attention kernels, for the entry points.
#pragma once
#include <hip/hip_runtime.h>

namespace sddmm {

struct AttnArgs;

enum { kRowsOfHead = 0, kRowsPacked = 1, kRowsShared = 2 };  // what the rows of a forward workgroup are (attention_tile.hpp)

constexpr int kTokenRows = 32;  // of a workgroup of the kernel for few rows
// tile: rows of a workgroup, 128 or 64
hipError_t launch_attention_forward(const AttnArgs &a, int type, int rows, int tile, unsigned grid, hipStream_t st);
hipError_t launch_attention_token(const AttnArgs &a, int type, unsigned grid, hipStream_t st);
// a: the dealing out of keys (dk, dv); b: of rows (dq)
// keys: of a dk, dv workgroup, 128, 64 or 32; q_rows: rows of a dq workgroup, 128, 64 or 32
hipError_t launch_attention_backward(const AttnArgs &a, const AttnArgs &b, int type, unsigned kv_grid, int keys, unsigned q_grid, int q_rows, hipStream_t st);
// a: the shared keys (kRowsShared, tile as above); own: each sequence's, by the kernel for few rows
hipError_t launch_attention_shared(const AttnArgs &a, const AttnArgs &own, int type, int tile, unsigned n_shared, unsigned n_own, hipStream_t st);
hipError_t launch_attention_join(const AttnArgs &a, int type, hipStream_t st);

}  // namespace sddmm
