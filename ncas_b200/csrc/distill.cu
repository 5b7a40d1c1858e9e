// distill.cu -- distillation from a teacher's top logits, forward and backward (nca_b200_distill*).
//
// Row r has logits s_j over the classes, entries (t_k, i_k) of the teacher, a weight w:
//   p = softmax(t / tau) over the entries, q = softmax(s / tau) over the classes
//   loss = w tau^2 sum_k p_k (log p_k - log q_{i_k}),  dloss/ds_j = w tau (q_j - sum_{k: i_k = j} p_k)
// G lanes share a row: one pass keeps a running maximum m and sum of exp((s - m) / tau), a second
// writes the gradient.  exp runs as exp2((s - m) log2(e) / tau): the difference first, so that the
// rounding is relative to the distance from the maximum.
#include <math_constants.h>

#include "cell_ops.cuh"

using namespace nca;

namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
  long long rows, top;
  int classes;
  int teacher_dtype, index_bits;
  float tau;
  long long s_stride, t_stride, i_stride;
  const void* logits;
  const void* teacher;
  const void* index;
  const float* weight;
  float* loss;
  float* stats;       // [rows][2] (maximum, sum), may be null
  const float* grad;  // backward: upstream gradient of each row's loss
  long long grad_stride;
  void* dlogits;
};

__device__ __forceinline__ int index_of(const DistillArgs& a, long long r, long long k) {
  const long long i = a.index_bits == 64 ? static_cast<const long long*>(a.index)[r * a.i_stride + k]
                                         : (long long)static_cast<const int*>(a.index)[r * a.i_stride + k];
  return i >= 0 && i < a.classes ? (int)i : -1;
}
__device__ __forceinline__ float teacher_of(const DistillArgs& a, long long r, long long k) {
  return load_param(a.teacher, a.teacher_dtype, r * a.t_stride + k);
}

// The G lanes of one row: G <= 32 lanes of a warp, or the whole block of kThreads.
template <int G>
struct Lanes {
  int lane;
  unsigned mask;
  float* red;  // shared, for the block form
  __device__ explicit Lanes(float* r) : red(r) {
    if constexpr (G <= 32) {
      lane = threadIdx.x % G;
      const int first = (threadIdx.x & 31) / G * G;
      mask = G == 32 ? 0xffffffffu : ((1u << G) - 1u) << first;
    } else {
      lane = threadIdx.x;
      mask = 0xffffffffu;
    }
  }
  __device__ __forceinline__ void sync() const {
    if constexpr (G <= 32) __syncwarp(mask);
    else __syncthreads();
  }
  __device__ __forceinline__ float max_warp(float v) const {
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o));
    return v;
  }
  __device__ __forceinline__ float sum_warp(float v) const {
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    return v;
  }
  __device__ __forceinline__ float max(float v) const {
    v = max_warp(v);
    if constexpr (G > 32) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      __syncthreads();
      v = red[0];
      for (int i = 1; i < G / 32; ++i) v = fmaxf(v, red[i]);
    }
    return v;
  }
  __device__ __forceinline__ float sum(float v) const {
    v = sum_warp(v);
    if constexpr (G > 32) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      __syncthreads();
      v = red[0];
      for (int i = 1; i < G / 32; ++i) v += red[i];
    }
    return v;
  }
};

template <class T, int G, bool FWD>
__global__ void __launch_bounds__(kThreads) distill_kernel(DistillArgs a) {
  __shared__ float red[32];
  const Lanes<G> l(red);
  constexpr int kRows = kThreads / G;
  const float c2 = kLog2e / a.tau, inv_tau = 1.f / a.tau;
  for (long long r = (long long)blockIdx.x * kRows + threadIdx.x / G; r < a.rows;
       r += (long long)gridDim.x * kRows) {
    const T* s = static_cast<const T*>(a.logits) + r * a.s_stride;
    T* ds = a.dlogits ? static_cast<T*>(a.dlogits) + r * (long long)a.classes : nullptr;
    const float w = a.weight ? a.weight[r] : 1.f;
    // the teacher's softmax over the row's entries
    float tmax = -CUDART_INF_F;
    if (w != 0.f)
      for (long long k = l.lane; k < a.top; k += G)
        if (index_of(a, r, k) >= 0) {
          const float t = teacher_of(a, r, k);
          tmax = t != t ? CUDART_INF_F : fmaxf(tmax, t);  // NaN and +inf end in NaN
        }
    tmax = l.max(tmax);
    if (tmax == -CUDART_INF_F) {  // no entry, or no weight
      if (FWD && l.lane == 0) {
        a.loss[r] = 0.f;
        if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
      }
      if (ds)
        for (int j = l.lane; j < a.classes; j += G) ds[j] = from_f32<T>(0.f);
      continue;
    }
    float tsum = 0.f;
    for (long long k = l.lane; k < a.top; k += G)
      if (index_of(a, r, k) >= 0) tsum += exp2f((teacher_of(a, r, k) - tmax) * c2);
    tsum = l.sum(tsum);
    float m, sum;
    if constexpr (FWD) {
      m = -CUDART_INF_F;
      sum = 0.f;
      for (int j = l.lane; j < a.classes; j += G) {
        const float v = to_f32(s[j]);
        if (v > m) {
          sum *= exp2f((m - v) * c2);  // 0 times it at first; a NaN stays
          m = v;
        }
        if (v != -CUDART_INF_F) sum += exp2f((v - m) * c2);  // NaN and +inf end in NaN
      }
      const float all = l.max(m);
      sum = l.sum(sum * exp2f((m - all) * c2));
      m = all;
      if (a.stats && l.lane == 0) {
        a.stats[2 * r] = m;
        a.stats[2 * r + 1] = sum;
      }
      const float lnt = logf(tsum), lns = logf(sum);
      float loss = 0.f;
      for (long long k = l.lane; k < a.top; k += G) {
        const int i = index_of(a, r, k);
        if (i < 0) continue;
        const float t = (teacher_of(a, r, k) - tmax);
        const float p = exp2f(t * c2) / tsum;
        if (p > 0.f) loss += p * ((t * inv_tau - lnt) - ((to_f32(s[i]) - m) * inv_tau - lns));
      }
      loss = l.sum(loss);
      if (l.lane == 0) a.loss[r] = loss * w * a.tau * a.tau;
    } else {
      m = a.stats[2 * r];
      sum = a.stats[2 * r + 1];
    }
    if (!ds) continue;
    const float coef = w * a.tau * (a.grad ? a.grad[r * a.grad_stride] : 1.f);
    const float qs = 1.f / sum;
    for (int j = l.lane; j < a.classes; j += G)
      ds[j] = from_f32<T>(coef * (exp2f((to_f32(s[j]) - m) * c2) * qs));
    l.sync();
    // the classes with an entry, each by the lane of its first entry
    for (long long k = l.lane; k < a.top; k += G) {
      const int i = index_of(a, r, k);
      if (i < 0) continue;
      bool first = true;
      for (long long k2 = 0; k2 < k && first; ++k2) first = index_of(a, r, k2) != i;
      if (!first) continue;
      float p = 0.f;
      for (long long k2 = k; k2 < a.top; ++k2)
        if (index_of(a, r, k2) == i) p += exp2f((teacher_of(a, r, k2) - tmax) * c2);
      ds[i] = from_f32<T>(coef * (exp2f((to_f32(s[i]) - m) * c2) * qs - p / tsum));
    }
    l.sync();
  }
}

template <class T, int G, bool FWD>
int32_t launch(const DistillArgs& a, cudaStream_t s) {
  const long long blocks = (a.rows + kThreads / G - 1) / (kThreads / G);
  distill_kernel<T, G, FWD><<<(unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), kThreads, 0, s>>>(a);
  return launch_status();
}

template <bool FWD>
int32_t dispatch(const NcaDistillDesc& d, const DistillArgs& a, cudaStream_t s) {
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    if (a.classes <= 4) return launch<T, 1, FWD>(a, s);
    if (a.classes <= 64) return launch<T, 8, FWD>(a, s);
    if (a.classes <= 1024) return launch<T, 32, FWD>(a, s);
    return launch<T, kThreads, FWD>(a, s);
  });
}

int32_t check_desc(const NcaDistillDesc* d) {
  if (!d || d->rows < 0 || d->classes <= 0 || d->top < 0) return NCA_ERR_INVALID;
  if (!dtype_ok(d->dtype) || !dtype_ok(d->teacher_dtype)) return NCA_ERR_INVALID;
  if (d->index_bits != 32 && d->index_bits != 64) return NCA_ERR_INVALID;
  if (!(d->temperature > 0.f) || d->temperature > 1e30f) return NCA_ERR_INVALID;
  if (d->classes >= (1ll << 31) - 4096) return NCA_ERR_UNSUPPORTED;
  return NCA_OK;
}

DistillArgs args_of(const NcaDistillDesc& d, const void* logits, const void* teacher, const void* index,
                    const float* weight) {
  DistillArgs a{};
  a.rows = d.rows;
  a.top = d.top;
  a.classes = (int)d.classes;
  a.teacher_dtype = d.teacher_dtype;
  a.index_bits = d.index_bits;
  a.tau = d.temperature;
  a.s_stride = d.logits_stride;
  a.t_stride = d.teacher_stride;
  a.i_stride = d.index_stride;
  a.logits = logits;
  a.teacher = teacher;
  a.index = index;
  a.weight = weight;
  return a;
}

}  // namespace

extern "C" {

int32_t nca_b200_distill_workspace(const NcaDistillDesc* d, size_t* bytes) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK || !bytes) return st != NCA_OK ? st : NCA_ERR_INVALID;
  *bytes = 256;
  return NCA_OK;
}

int32_t nca_b200_distill(const NcaDistillDesc* d, const void* logits, const void* teacher, const void* index,
                         const float* weight, float* loss, float* stats, void* dlogits, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK) return st;
  if (d->rows == 0) return NCA_OK;
  if (!logits || !loss || (d->top && (!teacher || !index))) return NCA_ERR_INVALID;
  (void)workspace;
  (void)workspace_bytes;
  DistillArgs a = args_of(*d, logits, teacher, index, weight);
  a.loss = loss;
  a.stats = stats;
  a.dlogits = dlogits;
  return dispatch<true>(*d, a, static_cast<cudaStream_t>(stream));
}

int32_t nca_b200_distill_backward(const NcaDistillDesc* d, const void* logits, const void* teacher,
                                  const void* index, const float* weight, const float* stats,
                                  const float* grad, int64_t grad_stride, void* dlogits, void* stream) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK) return st;
  if (d->rows == 0) return NCA_OK;
  if (!logits || !stats || !grad || !dlogits || (d->top && (!teacher || !index))) return NCA_ERR_INVALID;
  DistillArgs a = args_of(*d, logits, teacher, index, weight);
  a.stats = const_cast<float*>(stats);
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.dlogits = dlogits;
  return dispatch<false>(*d, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
