// cell_ops.cuh -- what the cell-training operators (norm.cu, gated.cu, distill.cu) share: element
// types, 16-byte vectors of them, and the activations with their derivatives.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/nca_b200.h"

namespace nca {

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V adjacent elements moved by one load or store of V * sizeof(T) bytes (1 to 16).
template <class T, int V>
struct alignas(V * sizeof(T)) Vec {
  T v[V];
};

// A parameter or gradient element of a type known at run time (once per channel, not per value).
__device__ __forceinline__ float load_param(const void* p, int dtype, long long i) {
  if (dtype == NCA_F32) return static_cast<const float*>(p)[i];
  if (dtype == NCA_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int dtype, long long i, float v) {
  if (dtype == NCA_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == NCA_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// ---------------------------------------------------------------------------------- activations
// 1 / (1 + exp(-z)): exp overflows to inf for z < -88, whose quotient is the limit 0.
__device__ __forceinline__ float sigmoid_f(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

template <int ACT>
__device__ __forceinline__ float act_f(float z) {
  if constexpr (ACT == NCA_ACT_RELU) return z < 0.f ? 0.f : z;  // keeps NaN
  if constexpr (ACT == NCA_ACT_SILU) return z * sigmoid_f(z);
  if constexpr (ACT == NCA_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  if constexpr (ACT == NCA_ACT_SIGMOID) return sigmoid_f(z);
  return z;
}

// act(z) and act'(z); relu'(0) = 0.
template <int ACT>
__device__ __forceinline__ float act_slope_f(float z, float& a) {
  if constexpr (ACT == NCA_ACT_RELU) {
    a = z < 0.f ? 0.f : z;
    return z > 0.f ? 1.f : 0.f;
  }
  if constexpr (ACT == NCA_ACT_SILU) {
    const float s = sigmoid_f(z);
    a = z * s;
    return s * (1.f + z * (1.f - s));
  }
  if constexpr (ACT == NCA_ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    a = z * cdf;
    return cdf + z * 0.39894228040143268f * __expf(-0.5f * z * z);  // phi(z) = exp(-z^2/2)/sqrt(2 pi)
  }
  if constexpr (ACT == NCA_ACT_SIGMOID) {
    const float s = sigmoid_f(z);
    a = s;
    return s * (1.f - s);
  }
  a = z;
  return 1.f;
}

// ------------------------------------------------------------------------------------ host side
inline int32_t launch_status() {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return NCA_OK;
  return e == cudaErrorNoKernelImageForDevice || e == cudaErrorInvalidDeviceFunction ? NCA_ERR_DEVICE
                                                                                    : NCA_ERR_CUDA;
}
inline size_t dtype_size(int dtype) { return dtype == NCA_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype >= NCA_F32 && dtype <= NCA_F16; }

// Calls fn with a value of the element type / the activation as a compile-time constant.
template <class F>
int32_t with_dtype(int dtype, F fn) {
  switch (dtype) {
    case NCA_F32: return fn(float{});
    case NCA_BF16: return fn(__nv_bfloat16{});
    case NCA_F16: return fn(__half{});
    default: return NCA_ERR_INVALID;
  }
}
template <int A>
struct ActTag {
  static constexpr int value = A;
};
template <class F>
int32_t with_act(int act, F fn) {
  switch (act) {
    case NCA_ACT_NONE: return fn(ActTag<NCA_ACT_NONE>{});
    case NCA_ACT_RELU: return fn(ActTag<NCA_ACT_RELU>{});
    case NCA_ACT_SILU: return fn(ActTag<NCA_ACT_SILU>{});
    case NCA_ACT_GELU: return fn(ActTag<NCA_ACT_GELU>{});
    case NCA_ACT_SIGMOID: return fn(ActTag<NCA_ACT_SIGMOID>{});
    default: return NCA_ERR_INVALID;
  }
}

}  // namespace nca
