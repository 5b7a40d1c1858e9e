// norm.cuh -- arguments that the streaming (norm.cu) and the held (norm_held*.cu) group norm share.
#pragma once
#include "cell_ops.cuh"

namespace nca {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const uint32_t a = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(a), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(a), "l"(from), "n"(BYTES) : "memory");
}

struct NormArgs {
  long long n, cells;
  int channels, groups, per_group;
  float eps;
  long long x_sn, x_sl, dy_sn, dy_sl, m_sn, m_sl;
  int tx, ty;                // threads over channel vectors, over cells
  int ctiles;                // tiles of tx vectors over the channels
  int chunks;                // pieces of a sample's cells, one per block at a time
  long long chunk_cells;
  int param_dtype;
  const void* x;
  const void* weight;
  const void* bias;
  const uint8_t* mask;
  const void* dy;
  void* y;                   // forward: y; backward: dx
  float* stats;              // [n][groups][2] mean, rstd
  float2* part;              // backward: [n][chunks][channels] (sum dz, sum dz h)
  float4* gpart;             // [n][chunks][groups + ctiles]: (count, mean, M2) or (count, A, B) of a block's
                             // channels of a group, at group + tile (no two pairs share a sum: along the
                             // channels neither falls)
  float2* ab;                // backward: [n][groups] (A / n, B / n)
};

// The kernels that hold samples in shared memory: the blocks that share a sample (8 at most), or 0 where
// they do not apply.  `v` is the vector width that channels, strides and addresses allow.  The
// backward writes (sum dz, sum dz h) of every sample and slice to a.part as [n][slices][channels].
int norm_held_slices(const NormArgs& a, int dtype, int v, bool backward);
int32_t norm_held_forward(const NormArgs& a, int dtype, int act, int v, cudaStream_t s);
int32_t norm_held_backward(const NormArgs& a, int dtype, int act, int v, cudaStream_t s);

}  // namespace nca
