// distill.cu -- distillation from a teacher's top logits, forward and backward (nca_b200_distill*).
//
// Row r has logits s_j over the classes, entries (t_k, i_k) of the teacher, a weight w:
//   p = softmax(t / tau) over the entries, q = softmax(s / tau) over the classes
//   loss = w tau^2 sum_k p_k (log p_k - log q_{i_k}),  dloss/ds_j = w tau (q_j - sum_{k: i_k = j} p_k)
// exp runs as exp2((s - m) log2(e) / tau), m the row's maximum: the difference first, so that the
// rounding is relative to the distance from the maximum.
#include "cell_ops.cuh"

using namespace nca;

namespace {

constexpr int kThreads = 256;
constexpr float kInf = __builtin_huge_valf();
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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// -------------------------------------------------------------------------------- few classes
// G lanes a row, K classes a lane in registers (class j of a row: lane j % G, register j / G), the
// entries likewise: one read of everything, no second pass.  For top <= G K.
template <class T, int G, int K, bool FWD>
__global__ void __launch_bounds__(kThreads) distill_small_kernel(DistillArgs a) {
  const Lanes<G> l(nullptr);
  constexpr int kRows = kThreads / G;
  const float c2 = kLog2e / a.tau, inv_tau = 1.f / a.tau;
  const int top = (int)a.top;
  for (long long r = (long long)blockIdx.x * kRows + threadIdx.x / G; r < a.rows;
       r += (long long)gridDim.x * kRows) {
    const T* s = static_cast<const T*>(a.logits) + r * a.s_stride;
    T* ds = static_cast<T*>(a.dlogits) + r * (long long)a.classes;
    const float w = a.weight ? a.weight[r] : 1.f;
    float v[K], t[K];
    int i[K];
    float m = -kInf, tmax = -kInf;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = k * G + l.lane;
      v[k] = j < a.classes ? to_f32(s[j]) : -kInf;
      i[k] = j < top ? index_of(a, r, j) : -1;
      t[k] = i[k] >= 0 ? teacher_of(a, r, j) : -kInf;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      m = fmaxf(m, v[k]);
      tmax = fmaxf(tmax, t[k] != t[k] ? kInf : t[k]);  // NaN and +inf end in NaN
    }
    tmax = l.max(tmax);
    if (w == 0.f || tmax == -kInf) {  // no weight, or no entry
      if (FWD && l.lane == 0) {
        a.loss[r] = 0.f;
        if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
      }
      if (a.dlogits)
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (k * G + l.lane < a.classes) ds[k * G + l.lane] = from_f32<T>(0.f);
      continue;
    }
    float sum = 0.f, tsum = 0.f, q[K];
    if constexpr (FWD) m = l.max(m);
    else m = a.stats[2 * r];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      q[k] = k * G + l.lane < a.classes ? ex2((v[k] - m) * c2) : 0.f;
      sum += q[k];
      tsum += i[k] >= 0 ? ex2((t[k] - tmax) * c2) : 0.f;
    }
    sum = FWD ? l.sum(sum) : a.stats[2 * r + 1];
    tsum = l.sum(tsum);
    const float ts = 1.f / tsum;
    float p[K], hit[K];  // each entry's p; each class's sum of them
#pragma unroll
    for (int k = 0; k < K; ++k) {
      p[k] = i[k] >= 0 ? ex2((t[k] - tmax) * c2) * ts : 0.f;
      hit[k] = 0.f;
    }
    float vi[K];  // the logit of each entry's class
#pragma unroll
    for (int k = 0; k < K; ++k) vi[k] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int o = 0; o < G; ++o) {
        if (k * G + o >= top) break;
        const int ik = G == 1 ? i[k] : __shfl_sync(l.mask, i[k], o, G);
        const float pk = G == 1 ? p[k] : __shfl_sync(l.mask, p[k], o, G);
        float mine = 0.f;
#pragma unroll
        for (int c = 0; c < K; ++c)
          if (c * G + l.lane == ik) {
            hit[c] += pk;
            mine = v[c];
          }
        if constexpr (FWD) {
          if constexpr (G > 1) mine = __shfl_sync(l.mask, mine, (ik < 0 ? 0 : ik) % G, G);
          if (o == l.lane) vi[k] = mine;
        }
      }
    if constexpr (FWD) {
      const float lnt = logf(tsum), lns = logf(sum);
      float loss = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (p[k] > 0.f) loss += p[k] * (((t[k] - tmax) * inv_tau - lnt) - ((vi[k] - m) * inv_tau - lns));
        else if (p[k] != p[k]) loss = p[k];
      loss = l.sum(loss);
      if (l.lane == 0) {
        a.loss[r] = loss * w * a.tau * a.tau;
        if (a.stats) {
          a.stats[2 * r] = m;
          a.stats[2 * r + 1] = sum;
        }
      }
    }
    if (a.dlogits) {
      const float coef = w * a.tau * (a.grad ? a.grad[r * a.grad_stride] : 1.f), qs = 1.f / sum;
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (k * G + l.lane < a.classes) ds[k * G + l.lane] = from_f32<T>(coef * (q[k] * qs - hit[k]));
    }
  }
}

// ------------------------------------------------------------------------------ many classes
// A row as 16-byte vectors between a ragged head and tail: the elements before the first 16-byte
// boundary and after the last.
template <class T>
struct RowSpan {
  static constexpr int kV = 16 / sizeof(T);
  int head, vecs, tail0, n;
  __device__ __forceinline__ RowSpan(const T* s, int classes) : n(classes) {
    const int off = (int)((reinterpret_cast<uintptr_t>(s) & 15) / sizeof(T));
    head = min(off ? kV - off : 0, classes);
    vecs = (classes - head) / kV;
    tail0 = head + vecs * kV;
  }
  __device__ __forceinline__ int ragged() const { return head + n - tail0; }
  __device__ __forceinline__ int ragged_at(int i) const { return i < head ? i : tail0 + i - head; }
};

template <class T>
__device__ __forceinline__ void unpack(const uint4& q, float (&f)[16 / sizeof(T)]) {
  const Vec<T, 16 / sizeof(T)>& v = reinterpret_cast<const Vec<T, 16 / sizeof(T)>&>(q);
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) f[i] = to_f32(v.v[i]);
}
template <class T>
__device__ __forceinline__ uint4 pack(const float (&f)[16 / sizeof(T)]) {
  uint4 q;
  Vec<T, 16 / sizeof(T)>& v = reinterpret_cast<Vec<T, 16 / sizeof(T)>&>(q);
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) v.v[i] = from_f32<T>(f[i]);
  return q;
}

// The running maximum and sum of exp2((v - m) c2).
struct Running {
  float m = -kInf, sum = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float (&f)[N], float c2) {
    float top = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, f[i]);
    if (top > m) {
      sum *= ex2((m - top) * c2);  // 0 times it at first; a NaN stays
      m = top;
    }
    const float base = m == -kInf ? 0.f : m;  // only -inf so far: exp2(-inf) = 0
#pragma unroll
    for (int i = 0; i < N; ++i) sum += ex2((f[i] - base) * c2);
  }
};

struct Entry {
  int index;
  float teacher;
};

// G lanes a row.  One pass over the row keeps the running maximum and sum, a second, which finds the
// row in L1 or L2, writes q; then the classes that have an entry are written again with q - p.
// `entries` (index, probability) of the row are staged in shared memory.
template <class T, int G, int NT, bool FWD>
__global__ void __launch_bounds__(NT) distill_row_kernel(DistillArgs a) {
  constexpr int kV = 16 / sizeof(T), kRows = NT / G, kWarps = G / 32;
  __shared__ float red_m[2][NT / 32], red_s[2][NT / 32];
  __shared__ float red_t[NT / 32];
  extern __shared__ Entry entries_all[];
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  Entry* entries = entries_all + (size_t)group * a.top;
  const auto sync = [] {
    if constexpr (G == 32) __syncwarp();
    else __syncthreads();
  };
  const float c2 = kLog2e / a.tau, inv_tau = 1.f / a.tau;
  const int top = (int)a.top;
  int flip = 0;
  for (long long r = (long long)blockIdx.x * kRows + group; r < a.rows; r += (long long)gridDim.x * kRows) {
    const T* s = static_cast<const T*>(a.logits) + r * a.s_stride;
    T* ds = a.dlogits ? static_cast<T*>(a.dlogits) + r * (long long)a.classes : nullptr;
    const float w = a.weight ? a.weight[r] : 1.f;
    const RowSpan<T> span(s, a.classes);
    const uint4* sv = reinterpret_cast<const uint4*>(s + span.head);
    const bool vec_out = ds && ((reinterpret_cast<uintptr_t>(ds) ^ reinterpret_cast<uintptr_t>(s)) & 15) == 0;
    // the first warp of the row: the teacher's softmax over the entries
    float tmax = -kInf, tsum = 0.f;
    if (lane < 32 && w != 0.f) {
      for (int k = lane; k < top; k += 32) {
        const int i = index_of(a, r, k);
        float t = i >= 0 ? teacher_of(a, r, k) : -kInf;
        entries[k] = Entry{i, t};
        tmax = fmaxf(tmax, t != t ? kInf : t);  // NaN and +inf end in NaN
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
      for (int k = lane; k < top; k += 32)
        if (entries[k].index >= 0) tsum += ex2((entries[k].teacher - tmax) * c2);
#pragma unroll
      for (int o = 16; o; o >>= 1) tsum += __shfl_xor_sync(0xffffffffu, tsum, o);
    }
    float m = 0.f, sum = 0.f;
    bool live = w != 0.f;
    if constexpr (FWD) {
      Running run;
      if (live) {
        int j = lane;
        for (; j + 3 * G < span.vecs; j += 4 * G) {
          uint4 q[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) q[u] = __ldg(sv + j + u * G);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            float f[kV];
            unpack<T>(q[u], f);
            run.add(f, c2);
          }
        }
        for (; j < span.vecs; j += G) {
          float f[kV];
          unpack<T>(__ldg(sv + j), f);
          run.add(f, c2);
        }
        for (int i = lane; i < span.ragged(); i += G) {
          const float f[1] = {to_f32(s[span.ragged_at(i)])};
          run.add(f, c2);
        }
      }
      float wm = run.m;
#pragma unroll
      for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
      float ws = run.sum * ex2((run.m - wm) * c2);
      if (run.m == -kInf) ws = run.sum;  // nothing, or only -inf (0), or NaN
#pragma unroll
      for (int o = 16; o; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
      if constexpr (G == 32) {
        m = wm;
        sum = ws;
      } else {
        if ((threadIdx.x & 31) == 0) {
          red_m[flip][threadIdx.x >> 5] = wm;
          red_s[flip][threadIdx.x >> 5] = ws;
        }
        if (threadIdx.x == 0) red_t[flip] = tmax, red_t[2 + flip] = tsum;
        __syncthreads();
        m = red_m[flip][0];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) m = fmaxf(m, red_m[flip][i]);
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
          const float e = red_m[flip][i];
          sum += e == -kInf ? red_s[flip][i] : red_s[flip][i] * ex2((e - m) * c2);
        }
      }
      if (m == -kInf) sum = m - m;  // a row of -inf only: NaN
    } else {
      m = a.stats[2 * r];
      sum = a.stats[2 * r + 1];
      if constexpr (G > 32) {
        if (threadIdx.x == 0) red_t[flip] = tmax, red_t[2 + flip] = tsum;
        __syncthreads();
      }
    }
    if constexpr (G > 32) {
      tmax = red_t[flip];
      tsum = red_t[2 + flip];
      flip ^= 1;
    } else {
      __syncwarp();
    }
    live = live && tmax != -kInf;
    if (!live) {  // no weight, or no entry
      if (FWD && lane == 0) {
        a.loss[r] = 0.f;
        if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
      }
      if (ds) {
        if (vec_out)
          for (int j = lane; j < span.vecs; j += G)
            reinterpret_cast<uint4*>(ds + span.head)[j] = make_uint4(0, 0, 0, 0);
        else
          for (int j = lane; j < span.vecs * kV; j += G) ds[span.head + j] = from_f32<T>(0.f);
        for (int i = lane; i < span.ragged(); i += G) ds[span.ragged_at(i)] = from_f32<T>(0.f);
      }
      sync();  // the entries have been read
      continue;
    }
    if (FWD && lane < 32) {
      const float lnt = logf(tsum), lns = logf(sum);
      float loss = 0.f;
      for (int k = lane; k < top; k += 32) {
        const int i = entries[k].index;
        if (i < 0) continue;
        const float t = entries[k].teacher - tmax;
        const float p = ex2(t * c2) / tsum;
        if (!(p <= 0.f)) loss += p * ((t * inv_tau - lnt) - ((to_f32(s[i]) - m) * inv_tau - lns));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
      if (lane == 0) {
        a.loss[r] = loss * w * a.tau * a.tau;
        if (a.stats) {
          a.stats[2 * r] = m;
          a.stats[2 * r + 1] = sum;
        }
      }
    }
    if (ds) {
      const float coef = w * a.tau * (a.grad ? a.grad[r * a.grad_stride] : 1.f);
      const float cq = coef / sum;
      const auto out = [&](float f) { return ex2((f - m) * c2) * cq; };
      if (vec_out) {
        uint4* dv = reinterpret_cast<uint4*>(ds + span.head);
        int j = lane;
        for (; j + 3 * G < span.vecs; j += 4 * G) {
          uint4 q[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) q[u] = __ldg(sv + j + u * G);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            float f[kV];
            unpack<T>(q[u], f);
#pragma unroll
            for (int i = 0; i < kV; ++i) f[i] = out(f[i]);
            __stcs(dv + j + u * G, pack<T>(f));
          }
        }
        for (; j < span.vecs; j += G) {
          float f[kV];
          unpack<T>(__ldg(sv + j), f);
#pragma unroll
          for (int i = 0; i < kV; ++i) f[i] = out(f[i]);
          __stcs(dv + j, pack<T>(f));
        }
      } else {
        for (int j = lane; j < span.vecs * kV; j += G) ds[span.head + j] = from_f32<T>(out(to_f32(s[span.head + j])));
      }
      for (int i = lane; i < span.ragged(); i += G)
        ds[span.ragged_at(i)] = from_f32<T>(out(to_f32(s[span.ragged_at(i)])));
      sync();
      // the classes with an entry, each by the lane of its first entry
      for (int k = lane; k < top; k += G) {
        const int i = entries[k].index;
        if (i < 0) continue;
        float p = 0.f;
        bool first = true;
        for (int k2 = 0; k2 < top; ++k2) {
          const Entry e = entries[k2];
          if (e.index != i) continue;
          first = first && k2 >= k;
          p += ex2((e.teacher - tmax) * c2);
        }
        if (first) ds[i] = from_f32<T>(coef * (ex2((to_f32(s[i]) - m) * c2) / sum - p / tsum));
      }
    }
    sync();  // the entries have been read
  }
}

template <class T, int G, int K, bool FWD>
int32_t launch_small(const DistillArgs& a, cudaStream_t s) {
  const long long blocks = (a.rows + kThreads / G - 1) / (kThreads / G);
  distill_small_kernel<T, G, K, FWD><<<(unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), kThreads, 0, s>>>(a);
  return launch_status();
}

constexpr int kMostEntries = 4096;  // staged in shared memory: 8 bytes each

template <class T, int G, int NT, bool FWD>
int32_t launch_rows(const DistillArgs& a, cudaStream_t s) {
  const long long blocks = (a.rows + NT / G - 1) / (NT / G);
  const size_t smem = (size_t)(NT / G) * a.top * sizeof(Entry);
  distill_row_kernel<T, G, NT, FWD><<<(unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), NT, smem, s>>>(a);
  return launch_status();
}

template <bool FWD>
int32_t dispatch(const NcaDistillDesc& d, const DistillArgs& a, cudaStream_t s) {
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    if (a.classes <= 4 && a.top <= 4) return launch_small<T, 1, 4, FWD>(a, s);
    if (a.classes <= 16 && a.top <= 16) return launch_small<T, 4, 4, FWD>(a, s);
    if (a.classes <= 64 && a.top <= 64) return launch_small<T, 8, 8, FWD>(a, s);
    if (a.classes <= 2048 && a.top <= 512) return launch_rows<T, 32, 256, FWD>(a, s);
    return launch_rows<T, 512, 512, FWD>(a, s);
  });
}

int32_t check_desc(const NcaDistillDesc* d) {
  if (!d || d->rows < 0 || d->classes <= 0 || d->top < 0) return NCA_ERR_INVALID;
  if (!dtype_ok(d->dtype) || !dtype_ok(d->teacher_dtype)) return NCA_ERR_INVALID;
  if (d->index_bits != 32 && d->index_bits != 64) return NCA_ERR_INVALID;
  if (!(d->temperature > 0.f) || d->temperature > 1e30f) return NCA_ERR_INVALID;
  if (d->classes >= (1ll << 31) - 4096 || d->top > kMostEntries) return NCA_ERR_UNSUPPORTED;
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
