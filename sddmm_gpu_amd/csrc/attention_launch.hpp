// Launches of the dense attention kernels, for the entry points.
#pragma once
#include <hip/hip_runtime.h>

namespace sddmm {

struct AttnArgs;

enum { kRowsOfHead = 0, kRowsPacked = 1, kRowsShared = 2 };  // what the rows of a forward workgroup are (attention_forward.hip)

int attention_forward_rows();  // rows of a workgroup
int attention_token_rows();
hipError_t launch_attention_forward(const AttnArgs &a, int type, int rows, unsigned grid, hipStream_t st);
hipError_t launch_attention_token(const AttnArgs &a, int type, unsigned grid, hipStream_t st);
int attention_backward_rows();
int attention_backward_few_rows();  // of a workgroup of the dq kernel for few rows
// a: the dealing out of keys (dk, dv); b: of rows (dq)
hipError_t launch_attention_backward(const AttnArgs &a, const AttnArgs &b, int type, unsigned kv_grid, unsigned q_grid, bool few, hipStream_t st);
hipError_t launch_attention_join(const AttnArgs &a, int type, hipStream_t st);

}  // namespace sddmm
