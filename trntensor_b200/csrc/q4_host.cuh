// Host side shared by the 4-bit matrix's translation units.
#pragma once
#include "common.cuh"

namespace tt {
namespace q4 {

// tiles as (y, z) with y <= 65535, x = splits; false when there are too many.
inline bool grid_of(long long tiles, int splits, dim3* grid) {
  const long long y = tiles < 65535 ? tiles : 65535, z = (tiles + y - 1) / y;
  if (z > 65535) return false;
  *grid = dim3((unsigned)splits, (unsigned)y, (unsigned)z);
  return true;
}

size_t gemm_workspace_bytes(int type, int scale_type, bool transposed, int M, int N, int K);
int run_gemm(bool transposed, const void* x, int type, long long ldx, const void* packed, const void* scales,
             int scale_type, const float* row_scale, int M, int N, int K, int group, void* y, long long ldy,
             void* workspace, size_t workspace_bytes, int* err, int dev, cudaStream_t s);
int run_row_scale(const void* scales, int scale_type, int N, int K, int group, float* out, cudaStream_t s);

}  // namespace q4
}  // namespace tt
