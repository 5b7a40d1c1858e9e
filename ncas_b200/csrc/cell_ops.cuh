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

// ------------------------------------------------------------------------- packed fp32 arithmetic
// Two fp32 operations in one instruction of sm_100.
#define NCA_F32X2(name, op)                                                                        \
  __device__ __forceinline__ float2 name(float2 a, float2 b) {                                     \
    float2 d;                                                                                      \
    asm(op " %0, %1, %2;"                                                                          \
        : "=l"(reinterpret_cast<uint64_t&>(d))                                                     \
        : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));   \
    return d;                                                                                      \
  }
NCA_F32X2(add2, "add.rn.f32x2")
NCA_F32X2(mul2, "mul.rn.f32x2")
#undef NCA_F32X2
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------------------------- activations
// Two values at a time.  1 / (1 + exp(-z)): exp overflows to inf for z < -88, whose reciprocal is the
// limit 0.
__device__ __forceinline__ float2 sigmoid2(float2 z) {
  const float2 t = mul2(z, both(-1.4426950408889634f));
  const float2 d = add2(make_float2(ex2(t.x), ex2(t.y)), both(1.f));
  return make_float2(rcp(d.x), rcp(d.y));
}
__device__ __forceinline__ float2 normal_cdf2(float2 z) {
  const float2 t = mul2(z, both(0.70710678118654752f));
  return fma2(make_float2(erff(t.x), erff(t.y)), both(0.5f), both(0.5f));
}

template <int ACT>
__device__ __forceinline__ float2 act2(float2 z) {
  if constexpr (ACT == NCA_ACT_RELU) return make_float2(z.x < 0.f ? 0.f : z.x, z.y < 0.f ? 0.f : z.y);  // keeps NaN
  if constexpr (ACT == NCA_ACT_SILU) return mul2(z, sigmoid2(z));
  if constexpr (ACT == NCA_ACT_GELU) return mul2(z, normal_cdf2(z));
  if constexpr (ACT == NCA_ACT_SIGMOID) return sigmoid2(z);
  return z;
}

// act'(z), and act(z) in `a`; relu'(0) = 0.
template <int ACT>
__device__ __forceinline__ float2 act_slope2(float2 z, float2& a) {
  if constexpr (ACT == NCA_ACT_RELU) {
    a = act2<ACT>(z);
    return make_float2(z.x > 0.f ? 1.f : 0.f, z.y > 0.f ? 1.f : 0.f);
  }
  if constexpr (ACT == NCA_ACT_SILU) {
    const float2 s = sigmoid2(z);
    a = mul2(z, s);
    return fma2(s, mul2(z, fma2(s, both(-1.f), both(1.f))), s);  // s + s z (1 - s)
  }
  if constexpr (ACT == NCA_ACT_GELU) {
    const float2 cdf = normal_cdf2(z);
    a = mul2(z, cdf);
    // the density exp(-z^2 / 2) / sqrt(2 pi)
    const float2 t = mul2(mul2(z, z), both(-0.72134752044448170f));
    return fma2(mul2(z, both(0.39894228040143268f)), make_float2(ex2(t.x), ex2(t.y)), cdf);
  }
  if constexpr (ACT == NCA_ACT_SIGMOID) {
    a = sigmoid2(z);
    return mul2(a, fma2(a, both(-1.f), both(1.f)));
  }
  a = z;
  return both(1.f);
}
template <int ACT>
__device__ __forceinline__ float act_f(float z) { return act2<ACT>(both(z)).x; }

// V values of a vector as pairs (the pair of a single value repeats it).
template <class T, int V>
__device__ __forceinline__ void to_pairs(const Vec<T, V>& v, float2 (&f)[(V + 1) / 2]) {
  if constexpr (V == 1) {
    f[0] = both(to_f32(v.v[0]));
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) f[i] = make_float2(v.v[2 * i], v.v[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (__is_same(T, __nv_bfloat16)) f[i] = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162&>(v.v[2 * i]));
      else f[i] = __half22float2(reinterpret_cast<const __half2&>(v.v[2 * i]));
    }
  }
}
template <class T, int V>
__device__ __forceinline__ Vec<T, V> from_pairs(const float2 (&f)[(V + 1) / 2]) {
  Vec<T, V> v;
  if constexpr (V == 1) {
    v.v[0] = from_f32<T>(f[0].x);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) v.v[2 * i] = f[i].x, v.v[2 * i + 1] = f[i].y;
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (__is_same(T, __nv_bfloat16)) reinterpret_cast<__nv_bfloat162&>(v.v[2 * i]) = __float22bfloat162_rn(f[i]);
      else reinterpret_cast<__half2&>(v.v[2 * i]) = __float22half2_rn(f[i]);
    }
  }
  return v;
}

// ------------------------------------------------------------------- programmatic dependent launch
// A kernel launched by launch_after() may start while the kernel before it in the stream ends: it sets
// itself up, and after after_previous() everything that ran before is complete and visible.  Every
// such kernel calls both: may_start_next() early, after_previous() before its first access to memory.
__device__ __forceinline__ void may_start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ------------------------------------------------------------------------------ blocks of a cluster
// A block may write the shared memory of another of its cluster only once that one has started, which a
// launch alone does not promise.  Every thread of a kernel that does so arrives at its start and waits
// just before its block's first such write; what the kernel reads in between hides the wait.
__device__ __forceinline__ void cluster_started_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_started_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// ------------------------------------------------------------------------------------ host side
inline int32_t launch_status() {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return NCA_OK;
  return e == cudaErrorNoKernelImageForDevice || e == cudaErrorInvalidDeviceFunction ? NCA_ERR_DEVICE
                                                                                    : NCA_ERR_CUDA;
}
template <class... P, class... A>
int32_t launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  const int32_t st = launch_status();
  return e == cudaSuccess || st != NCA_OK ? st : NCA_ERR_CUDA;
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
