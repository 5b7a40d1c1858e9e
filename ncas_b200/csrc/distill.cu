// distill.cu -- distillation from a teacher's top logits, forward and backward (nca_b200_distill*).
//
// Row r has logits s_j over the classes, entries (t_k, i_k) of the teacher, a weight w:
//   p = softmax(t / tau) over the entries, q = softmax(s / tau) over the classes
//   loss = w tau^2 sum_k p_k (log p_k - log q_{i_k}),  dloss/ds_j = w tau (q_j - sum_{k: i_k = j} p_k)
// exp runs as exp2((s - m) log2(e) / tau), m the row's maximum: the difference first, so that the
// rounding is relative to the distance from the maximum, and a row of the type's lowest values, whose
// product with the scale would overflow, still gives differences of 0.
//
// Which lanes share a row goes by its size (dispatch, below).  On a B200: 900,000 x 2 bf16 12.9 us in all
// (2.0 TB/s; instructions bind, 74% of the issue slots), 150,022 x 662 fp16 with 90 entries 246 to 261 us,
// 2047 x 32003 fp16 55 us (4.7 TB/s), 8192 x 131072 bf16 with gradient 770 to 840 us (5.1 to 5.6 TB/s,
// near HBM; the exponentials take 58% of their unit).
#include "cell_ops.cuh"
#include <atomic>
#include <type_traits>

using namespace nca;

namespace {

constexpr int kThreads = 256;
constexpr float kInf = __builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
  long long rows, top;
  int classes;
  int teacher_dtype, index_bits;
  float tau, c2, inv_tau;  // temperature, log2(e) / tau, 1 / tau
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

// The G lanes of a warp that share a row.
template <int G>
struct Lanes {
  int lane;
  unsigned mask;
  __device__ Lanes() {
    lane = threadIdx.x % G;
    mask = G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) / G * G);
  }
  __device__ __forceinline__ float max(float v) const {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o));
    return v;
  }
  __device__ __forceinline__ float sum(float v) const {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    return v;
  }
};

// -------------------------------------------------------------------------------- few classes
// A row of n <= K values into registers (one access when the row is K values wide and lies on its own
// size).  n is the same for all threads.
template <class E, int K>
__device__ __forceinline__ void load_values(const E* from, int n, bool whole, E (&v)[K]) {
  if (whole) {
    const Vec<E, K> w = *reinterpret_cast<const Vec<E, K>*>(from);
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = w.v[k];
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k < n) v[k] = from[k];
  }
}
template <class E, int K>
__device__ __forceinline__ bool whole_rows(const void* p, long long stride, int n) {
  return sizeof(E) * K <= 16 && n == K && stride % K == 0 && reinterpret_cast<uintptr_t>(p) % (sizeof(E) * K) == 0;
}

// G lanes a row, K classes a lane in registers (class j of a row: lane j % G, register j / G), the
// entries likewise in KE registers: one read of everything, no second pass.  For top <= G KE.  I: the index
// type; the teacher has the logits' type (SAME) or one that is looked up at each load.
template <class T, class I, int G, int K, int KE, bool SAME, bool FWD>
__global__ void __launch_bounds__(kThreads) distill_small_kernel(DistillArgs a) {
  const Lanes<G> l;
  constexpr int kRows = kThreads / G;
  const float c2 = a.c2, inv_tau = a.inv_tau;
  const int top = (int)a.top;
  const bool whole_s = G == 1 && whole_rows<T, K>(a.logits, a.s_stride, a.classes);
  const bool whole_d = G == 1 && a.dlogits && whole_rows<T, K>(a.dlogits, a.classes, a.classes);
  const bool whole_i = G == 1 && whole_rows<I, KE>(a.index, a.i_stride, top);
  const bool whole_t = G == 1 && SAME && whole_rows<T, KE>(a.teacher, a.t_stride, top);
  for (long long r = (long long)blockIdx.x * kRows + threadIdx.x / G; r < a.rows;
       r += (long long)gridDim.x * kRows) {
    const T* s = static_cast<const T*>(a.logits) + r * a.s_stride;
    const I* is = static_cast<const I*>(a.index) + r * a.i_stride;
    T* ds = static_cast<T*>(a.dlogits) + r * (long long)a.classes;
    const float w = a.weight ? a.weight[r] : 1.f;
    float v[K], t[KE];
    int i[KE];
    float m = -kInf, tmax = -kInf;
    // everything is asked for before anything is used
    T sv[K], tv[KE];
    I iv[KE];
    float tf[KE];
    if constexpr (G == 1) {
      load_values<T, K>(s, a.classes, whole_s, sv);
      load_values<I, KE>(is, top, whole_i, iv);
      if constexpr (SAME) load_values<T, KE>(static_cast<const T*>(a.teacher) + r * a.t_stride, top, whole_t, tv);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int j = k * G + l.lane;
        if (j < a.classes) sv[k] = s[j];
      }
#pragma unroll
      for (int k = 0; k < KE; ++k) {
        const int j = k * G + l.lane;
        if (j < top) iv[k] = is[j];
        if (SAME && j < top) tv[k] = static_cast<const T*>(a.teacher)[r * a.t_stride + j];
      }
    }
    if constexpr (!SAME) {
#pragma unroll
      for (int k = 0; k < KE; ++k)
        if (k * G + l.lane < top) tf[k] = teacher_of(a, r, k * G + l.lane);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = k * G + l.lane;
      v[k] = j < a.classes ? to_f32(sv[k]) : -kInf;
      m = fmaxf(m, v[k]);
    }
#pragma unroll
    for (int k = 0; k < KE; ++k) {
      const int j = k * G + l.lane;
      i[k] = j < top && iv[k] >= 0 && iv[k] < a.classes ? (int)iv[k] : -1;
      if constexpr (SAME) t[k] = i[k] >= 0 ? to_f32(tv[k]) : -kInf;
      else t[k] = i[k] >= 0 ? tf[k] : -kInf;
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
    }
#pragma unroll
    for (int k = 0; k < KE; ++k) {
      tsum += i[k] >= 0 ? ex2((t[k] - tmax) * c2) : 0.f;
    }
    sum = FWD ? l.sum(sum) : a.stats[2 * r + 1];
    tsum = l.sum(tsum);
    const float ts = rcp(tsum);
    float p[KE], vi[KE];  // each entry's p and the logit of its class
    float hit[K];         // each class's sum of p
#pragma unroll
    for (int k = 0; k < KE; ++k) {
      p[k] = i[k] >= 0 ? ex2((t[k] - tmax) * c2) * ts : 0.f;
      vi[k] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) hit[k] = 0.f;
#pragma unroll
    for (int k = 0; k < KE; ++k)
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
      for (int k = 0; k < KE; ++k)
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
      const float coef = w * a.tau * (a.grad ? a.grad[r * a.grad_stride] : 1.f), qs = rcp(sum);
      Vec<T, K> out;
#pragma unroll
      for (int k = 0; k < K; ++k) out.v[k] = from_f32<T>(coef * (q[k] * qs - hit[k]));
      if (whole_d) {
        *reinterpret_cast<Vec<T, K>*>(ds) = out;
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (k * G + l.lane < a.classes) ds[k * G + l.lane] = out.v[k];
      }
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

// (a - m) c2 of two values.
__device__ __forceinline__ float2 scaled2(float a0, float a1, float m, float c2) {
  float2 d;
  const float2 a = make_float2(a0, a1), n = make_float2(-m, -m), c = make_float2(c2, c2);
  asm("{\n\t.reg .b64 t;\n\tadd.rn.f32x2 t, %1, %2;\n\tmul.rn.f32x2 %0, t, %3;\n\t}"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(n)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
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
      sum *= ex2((m - top) * c2);  // 0 times 0 at first; a NaN stays
      m = top;
    }
    const float from = m == -kInf ? 0.f : m;  // only -inf so far: exp2(-inf) = 0
    if constexpr (N % 2 == 0) {
      float2 part = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 d = scaled2(f[i], f[i + 1], from, c2);
        part.x += ex2(d.x);
        part.y += ex2(d.y);
      }
      sum += part.x + part.y;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) sum += ex2((f[i] - from) * c2);
    }
  }
};
// `sum` counted from maximum m, as counted from `to` >= m.
__device__ __forceinline__ float rebase(float sum, float m, float to, float c2) {
  return m == -kInf ? sum : sum * ex2((m - to) * c2);  // nothing, only -inf (0), or NaN
}

struct Entry {
  int index;
  float teacher;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Writes two values into the shared memory of CTA `rank` of the cluster, at the place that `p` is here.
__device__ __forceinline__ void put_remote(float2* p, uint32_t rank, float2 v) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(r), "f"(v.x), "f"(v.y) : "memory");
}
constexpr int kMostSlices = 8;

// A block a row, or a cluster of `slices` blocks: rows that no cluster holds, more than 128 entries, and
// the loss alone of many long rows.
// One pass keeps the running maximum and sum, a
// second, which finds the row in L1 or L2, writes q; then the classes that have an entry are written
// again with q - p.  The row's entries are staged in shared memory.
template <class T, int NT, bool FWD>
__global__ void __launch_bounds__(NT) distill_row_kernel(DistillArgs a, int slices) {
  constexpr int kV = 16 / sizeof(T), G = NT, kWarps = NT / 32;
  __shared__ float red_m[2][NT / 32], red_s[2][NT / 32];
  __shared__ float2 red_t[2];
  __shared__ float2 red_c[2][kMostSlices];  // (maximum, sum) of each slice
  extern __shared__ Entry entries[];
  const int lane = threadIdx.x;
  const int slice = slices > 1 ? (int)cluster_rank() : 0;
  if (FWD && slices > 1) cluster_started_arrive();
  const float c2 = a.c2, inv_tau = a.inv_tau;
  const int top = (int)a.top;
  int flip = 0;
  for (long long r = blockIdx.x / slices; r < a.rows; r += gridDim.x / slices) {
    const T* s = static_cast<const T*>(a.logits) + r * a.s_stride;
    T* ds = a.dlogits ? static_cast<T*>(a.dlogits) + r * (long long)a.classes : nullptr;
    const float w = a.weight ? a.weight[r] : 1.f;
    const RowSpan<T> span(s, a.classes);
    const uint4* sv = reinterpret_cast<const uint4*>(s + span.head);
    const bool vec_out = ds && ((reinterpret_cast<uintptr_t>(ds) ^ reinterpret_cast<uintptr_t>(s)) & 15) == 0;
    // this block's vectors; the ragged ends belong to the first slice
    const int v0 = (int)((long long)span.vecs * slice / slices), v1 = (int)((long long)span.vecs * (slice + 1) / slices);
    const int ragged = slice == 0 ? span.ragged() : 0;
    // the first warp of the row: the teacher's softmax over the entries
    float tmax = -kInf, tsum = 0.f;
    if (lane < 32 && w != 0.f) {
      for (int k = lane; k < top; k += 32) {
        const int i = index_of(a, r, k);
        const float t = i >= 0 ? teacher_of(a, r, k) : -kInf;
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
        int j = v0 + lane;
        for (; j + 3 * G < v1; j += 4 * G) {
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
        for (; j < v1; j += G) {
          float f[kV];
          unpack<T>(__ldg(sv + j), f);
          run.add(f, c2);
        }
        for (int i = lane; i < ragged; i += G) {
          const float f[1] = {to_f32(s[span.ragged_at(i)])};
          run.add(f, c2);
        }
      }
      float wm = run.m;
#pragma unroll
      for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
      float ws = rebase(run.sum, run.m, wm, c2);
#pragma unroll
      for (int o = 16; o; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
      {
        if ((threadIdx.x & 31) == 0) {
          red_m[flip][threadIdx.x >> 5] = wm;
          red_s[flip][threadIdx.x >> 5] = ws;
        }
        if (threadIdx.x == 0) red_t[flip] = make_float2(tmax, tsum);
        __syncthreads();
        m = red_m[flip][0];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) m = fmaxf(m, red_m[flip][i]);
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
          const float e = red_m[flip][i];
          sum += rebase(red_s[flip][i], e, m, c2);
        }
        if (slices > 1) {  // for a row of weight 0 too: the barrier frees the places of the row before
          if (r < gridDim.x / slices) cluster_started_wait();  // the first row
          if (threadIdx.x < slices) put_remote(&red_c[flip][slice], threadIdx.x, make_float2(m, sum));
          cluster_barrier();
          m = red_c[flip][0].x;
          for (int i = 1; i < slices; ++i) m = fmaxf(m, red_c[flip][i].x);
          sum = 0.f;
          for (int i = 0; i < slices; ++i) {
            const float2 e = red_c[flip][i];
            sum += rebase(e.y, e.x, m, c2);
          }
        }
      }
      if (m == -kInf) sum = m - m;  // a row of -inf only: NaN
    } else {
      m = a.stats[2 * r];
      sum = a.stats[2 * r + 1];
      if (threadIdx.x == 0) red_t[flip] = make_float2(tmax, tsum);
      __syncthreads();
    }
    tmax = red_t[flip].x;
    tsum = red_t[flip].y;
    flip ^= 1;
    live = live && tmax != -kInf;
    if (!live) {  // no weight, or no entry
      if (FWD && lane == 0 && slice == 0) {
        a.loss[r] = 0.f;
        if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
      }
      if (ds) {
        if (vec_out)
          for (int j = v0 + lane; j < v1; j += G)
            reinterpret_cast<uint4*>(ds + span.head)[j] = make_uint4(0, 0, 0, 0);
        else
          for (int j = v0 * kV + lane; j < v1 * kV; j += G) ds[span.head + j] = from_f32<T>(0.f);
        for (int i = lane; i < ragged; i += G) ds[span.ragged_at(i)] = from_f32<T>(0.f);
      }
      __syncthreads();  // the entries have been read
      continue;
    }
    if (FWD && lane < 32 && slice == 0) {
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
      const auto write = [&](int j, const uint4& q) {
        float f[kV];
        unpack<T>(q, f);
#pragma unroll
        for (int i = 0; i < kV; i += 2) {
          const float2 d = scaled2(f[i], f[i + 1], m, c2);
          f[i] = ex2(d.x) * cq;
          f[i + 1] = ex2(d.y) * cq;
        }
        __stcs(reinterpret_cast<uint4*>(ds + span.head) + j, pack<T>(f));
      };
      const auto write_one = [&](int j) { ds[j] = from_f32<T>(ex2((to_f32(s[j]) - m) * c2) * cq); };
      if (vec_out) {
        int j = v0 + lane;
        for (; j + 3 * G < v1; j += 4 * G) {
          uint4 q[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) q[u] = __ldg(sv + j + u * G);
#pragma unroll
          for (int u = 0; u < 4; ++u) write(j + u * G, q[u]);
        }
        for (; j < v1; j += G) write(j, __ldg(sv + j));
      } else {
        for (int j = v0 * kV + lane; j < v1 * kV; j += G) write_one(span.head + j);
      }
      for (int i = lane; i < ragged; i += G) write_one(span.ragged_at(i));
      __syncthreads();
      // the classes with an entry in this slice, each by the lane of its first entry
      const int c0 = span.head + v0 * kV, c1 = span.head + v1 * kV;
      for (int k = lane; k < top; k += G) {
        const int i = entries[k].index;
        if (i < 0 || (slices > 1 && (i < c0 || i >= c1) && !(slice == 0 && (i < span.head || i >= span.tail0))))
          continue;
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
    __syncthreads();  // the entries have been read
  }
}

__device__ __forceinline__ void named_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

constexpr int kHeld = 8;       // 16-byte vectors of a row that a lane holds
constexpr int kLaneTop = 4;    // entries of a row that a lane holds

// The larger of m and a vector's values, 16-bit types two at a time (NaN is passed over: the sum finds it).
template <class T>
struct Largest {
  using T2 = std::conditional_t<__is_same(T, __nv_bfloat16), __nv_bfloat162, __half2>;
  T2 m;
  __device__ __forceinline__ explicit Largest(uint32_t low) : m(reinterpret_cast<const T2&>(low)) {}
  __device__ __forceinline__ void add(const uint4& q) {
    m = __hmax2(__hmax2(m, reinterpret_cast<const T2&>(q.x)), reinterpret_cast<const T2&>(q.y));
    m = __hmax2(__hmax2(m, reinterpret_cast<const T2&>(q.z)), reinterpret_cast<const T2&>(q.w));
  }
  __device__ __forceinline__ float get() const { return fmaxf(to_f32(m.x), to_f32(m.y)); }
};
template <>
struct Largest<float> {
  float m;
  __device__ __forceinline__ explicit Largest(uint32_t low) : m(reinterpret_cast<const float&>(low)) {}
  __device__ __forceinline__ void add(const uint4& q) {
    m = fmaxf(fmaxf(m, fmaxf(reinterpret_cast<const float&>(q.x), reinterpret_cast<const float&>(q.y))),
              fmaxf(reinterpret_cast<const float&>(q.z), reinterpret_cast<const float&>(q.w)));
  }
  __device__ __forceinline__ float get() const { return m; }
};
// A 16-byte read of shared memory that is done again at each use: kept values would not fit the registers.
__device__ __forceinline__ uint4 ld_shared(const uint4* p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"((uint32_t)__cvta_generic_to_shared(p)));
  return v;
}
template <class T>
__device__ __forceinline__ float exp_sum(const uint4& q, float from, float c2) {
  float f[16 / sizeof(T)], part = 0.f;
  unpack<T>(q, f);
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); i += 2) {
    const float2 d = scaled2(f[i], f[i + 1], from, c2);
    part += ex2(d.x) + ex2(d.y);
  }
  return part;
}

// A block, or a cluster of `slices` blocks, goes through rows that it holds: NS lanes hold kHeld
// 16-byte vectors each in registers and NSM in shared memory, loaded while the row before is written
// (a place is reloaded as soon as it has been used), so a row is read once and reads stay in flight
// through the reductions.  One
// more warp does everything else a row ahead or behind: the entries, the loss, the ragged ends, the
// weights, and after the others have written q, the classes that have an entry.
// One block barrier a row (and one of the cluster when slices > 1).
template <class T, int NS, int NSM, int BLOCKS, bool FWD>
__global__ void __launch_bounds__(NS + 32, BLOCKS) distill_held_kernel(DistillArgs a, int slices) {
  // vectors of a slice: the host's arithmetic, a row's `vecs` is classes / kV or one less
  const int per = (a.classes / (16 / (int)sizeof(T)) + slices - 1) / slices;
  constexpr int kV = 16 / sizeof(T), kWarps = NS / 32, NT = NS + 32;
  constexpr int kWritten = 1;  // named barrier: the lanes have written a row's q
  __shared__ float2 red[2][kWarps + 1];     // (maximum, sum) of each warp
  __shared__ float2 red_c[2][kMostSlices];  // and of each slice
  __shared__ float4 said[2];                // coef, live, next row has a weight, sum (backward: with red the maximum)
  __shared__ Entry entries[32 * kLaneTop];
  extern __shared__ uint4 held[];           // [NSM][NS]
  const int slice = slices > 1 ? (int)cluster_rank() : 0;
  if (FWD && slices > 1) cluster_started_arrive();
  const int lane = threadIdx.x & 31;
  const bool entry_warp = threadIdx.x >= NS;
  const float c2 = a.c2;
  const long long step = gridDim.x / slices;
  long long r = blockIdx.x / slices;
  int flip = 0;
  // the row's (maximum, sum) from the partial ones of all warps and slices
  // (every lane of a warp gets them: one partial result a lane, then butterflies)
  const auto butterfly = [&](float2 e, int n, float& m, float& sum) {
    m = e.x;
#pragma unroll
    for (int o = 16; o; o >>= 1)
      if (o < n) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    sum = rebase(e.y, e.x, m, c2);
#pragma unroll
    for (int o = 16; o; o >>= 1)
      if (o < n) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  };
  const auto combine = [&](float& m, float& sum) {
    constexpr int n = kWarps < 8 ? 8 : kWarps < 16 ? 16 : 32;  // partial results, rounded up
    butterfly((lane & (n - 1)) <= kWarps ? red[flip][lane & (n - 1)] : make_float2(-kInf, 0.f), n, m, sum);
    if (slices > 1) {
      if (r < step) cluster_started_wait();  // the first row
      if (threadIdx.x < slices) put_remote(&red_c[flip][slice], threadIdx.x, make_float2(m, sum));
      cluster_barrier();
      butterfly((lane & 7) < slices ? red_c[flip][lane & 7] : make_float2(-kInf, 0.f), 8, m, sum);
    }
    if (m == -kInf) sum = m - m;  // a row of -inf only: NaN
  };

  if (!entry_warp) {
    uint4 q[kHeld];
    const uint32_t low = sizeof(T) == 4 ? 0xFF800000u : (__is_same(T, __nv_bfloat16) ? 0xFF80FF80u : 0xFC00FC00u);  // -inf
    // this lane's vectors of row `at`: the first, and how many lie in the slice
    const auto place = [&](long long at, const uint4*& p, int& first, int& count) {
      const T* s = static_cast<const T*>(a.logits) + at * a.s_stride;
      const RowSpan<T> span(s, a.classes);
      const int v0 = min(span.vecs, slice * per), v1 = min(span.vecs, v0 + per);
      first = v0 + (int)threadIdx.x;
      p = reinterpret_cast<const uint4*>(s + span.head) + first;
      count = v1 - first;  // vectors at first, first + NS, ... while u * NS < count
    };
    const uint4* p;
    int first, count;
    // vector u of the row at p: u < kHeld in a register, above in this lane's place of `held`
    const auto fetch = [&](int u) {
      const bool on = u * NS < count;
      if (u < kHeld) {
        q[u] = on ? __ldcs(p + u * NS) : make_uint4(low, low, low, low);
      } else {
        uint4* to = &held[(u - kHeld) * NS + threadIdx.x];
        if (on)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)),
                       "l"(p + u * NS)
                       : "memory");
        else
          *to = make_uint4(low, low, low, low);
      }
    };
    if (r < a.rows) {
      place(r, p, first, count);
#pragma unroll
      for (int u = 0; u < kHeld + NSM; ++u) fetch(u);
    }
    for (; r < a.rows; r += step, flip ^= 1) {
      float m = -kInf, sum = 0.f;
      if constexpr (FWD) {
        Largest<T> most(low);
#pragma unroll
        for (int u = 0; u < kHeld; ++u) most.add(q[u]);
        if constexpr (NSM > 0) {
          asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 3
          for (int u = 0; u < NSM; ++u) most.add(ld_shared(&held[u * NS + threadIdx.x]));
        }
        m = most.get();
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float from = m == -kInf ? 0.f : m;
#pragma unroll
        for (int u = 0; u < kHeld; ++u) asm volatile("" : "+r"(q[u].x), "+r"(q[u].y), "+r"(q[u].z), "+r"(q[u].w));
#pragma unroll
        for (int u = 0; u < kHeld; ++u) sum += exp_sum<T>(q[u], from, c2);
#pragma unroll 1
        for (int u = 0; u < NSM; ++u) sum += exp_sum<T>(ld_shared(&held[u * NS + threadIdx.x]), from, c2);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) red[flip][threadIdx.x >> 5] = make_float2(m, sum);
      }
#pragma unroll
      for (int u = 0; u < kHeld; ++u)  // unpacked again below: the 32-bit values would not fit the registers
        asm volatile("" : "+r"(q[u].x), "+r"(q[u].y), "+r"(q[u].z), "+r"(q[u].w));
      __syncthreads();
      if constexpr (FWD) combine(m, sum);
      const float4 word = said[flip];
      if constexpr (!FWD) {
        m = red[flip][0].x;
        sum = word.w;
        if constexpr (NSM > 0) asm volatile("cp.async.wait_all;" ::: "memory");
      }
      const bool live = word.y != 0.f;
      const float from = live ? m : 0.f, cq = live ? word.x / sum : 0.f;
      const bool more = r + step < a.rows;
      T* ds = static_cast<T*>(a.dlogits) + r * (long long)a.classes;
      const int head = (int)(reinterpret_cast<const T*>(p) - (static_cast<const T*>(a.logits) + r * a.s_stride)) - first * kV;
      T* out = a.dlogits ? ds + head + first * kV : nullptr;
      const bool vec_out = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(p)) & 15) == 0;
      const int now = a.dlogits ? count : 0;
      if (more) place(r + step, p, first, count);
      if (!more || word.z == 0.f) count = 0;
#pragma unroll
      for (int u = 0; u < kHeld + NSM; ++u) {
        if (u * NS < now) {
          float f[kV];
          unpack<T>(u < kHeld ? q[u < kHeld ? u : 0] : ld_shared(&held[(u - kHeld) * NS + threadIdx.x]), f);
#pragma unroll
          for (int i = 0; i < kV; i += 2) {
            const float2 d = scaled2(f[i], f[i + 1], from, c2);
            f[i] = live ? ex2(d.x) * cq : 0.f;
            f[i + 1] = live ? ex2(d.y) * cq : 0.f;
          }
          if (vec_out) {
            __stcs(reinterpret_cast<uint4*>(out) + u * NS, pack<T>(f));
          } else {
#pragma unroll
            for (int i = 0; i < kV; ++i) out[(size_t)u * NS * kV + i] = from_f32<T>(f[i]);
          }
        }
        fetch(u);
      }
      if (more && word.z == 0.f) {  // nothing was loaded, but the row's zeros are to be written
        place(r + step, p, first, count);
      }
      named_arrive(kWritten, NT);
    }
  } else {
    const int top = (int)a.top;
    const float inv_tau = a.inv_tau;
    // raw words of the row ahead
    long long index[kLaneTop];
    float teach[kLaneTop];
    float weight = 0.f, weight1 = 0.f, up = 1.f;
    const auto weight_of = [&](long long at) { return at < a.rows ? (a.weight ? a.weight[at] : 1.f) : 0.f; };
    const auto fetch = [&](long long at) {
#pragma unroll
      for (int k = 0; k < kLaneTop; ++k) {
        const int e = k * 32 + lane;
        index[k] = -1;
        teach[k] = 0.f;
        if (at < a.rows && e < top) {
          index[k] = a.index_bits == 64 ? static_cast<const long long*>(a.index)[at * a.i_stride + e]
                                        : (long long)static_cast<const int*>(a.index)[at * a.i_stride + e];
          teach[k] = teacher_of(a, at, e);
        }
      }
      if (at < a.rows && a.grad) up = a.grad[at * a.grad_stride];
    };
    weight = weight_of(r);
    weight1 = weight_of(r + step);
    fetch(r);
    for (; r < a.rows; r += step, flip ^= 1) {
      const T* s = static_cast<const T*>(a.logits) + r * a.s_stride;
      const RowSpan<T> span(s, a.classes);
      const int v0 = min(span.vecs, slice * per), v1 = min(span.vecs, v0 + per);
      const int c0 = span.head + v0 * kV, c1 = span.head + v1 * kV;
      const bool ragged = slice == 0 && lane < span.ragged();
      const int ragged_at = ragged ? span.ragged_at(lane) : 0;
      const float end = ragged ? to_f32(s[ragged_at]) : -kInf;
      int i[kLaneTop];
      T v[kLaneTop];
      float t[kLaneTop], tmax = -kInf, tsum = 0.f;
#pragma unroll
      for (int k = 0; k < kLaneTop; ++k) {
        i[k] = index[k] >= 0 && index[k] < a.classes ? (int)index[k] : -1;
        t[k] = i[k] >= 0 ? teach[k] : -kInf;
        v[k] = s[i[k] >= 0 ? i[k] : 0];
        tmax = fmaxf(tmax, t[k] != t[k] ? kInf : t[k]);  // NaN and +inf end in NaN
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
      const bool live = weight != 0.f && tmax != -kInf;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kLaneTop; ++k) {
        t[k] -= tmax;
        const float p = i[k] >= 0 ? ex2(t[k] * c2) : 0.f;
        tsum += p;
        if (k * 32 + lane < top) entries[k * 32 + lane] = Entry{i[k], p};  // p up to its sum
      }
      __syncwarp();
#pragma unroll
      for (int o = 16; o; o >>= 1) tsum += __shfl_xor_sync(0xffffffffu, tsum, o);
      const float coef = live ? weight * a.tau * up : 0.f;
      const float weight_now = weight;
      float m = -kInf, sum = 0.f;
      if constexpr (FWD) {
        m = end;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        sum = ragged ? ex2((end - (m == -kInf ? 0.f : m)) * c2) : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
          red[flip][kWarps] = make_float2(m, sum);
          said[flip] = make_float4(coef, live ? 1.f : 0.f, weight1, 0.f);
        }
      } else {
        m = a.stats[2 * r];
        sum = a.stats[2 * r + 1];
        if (lane == 0) {
          red[flip][0].x = m;
          said[flip] = make_float4(coef, live ? 1.f : 0.f, weight1, sum);
        }
      }
      __syncthreads();
      // the row ahead, while the others write
      weight = weight1;
      weight1 = weight_of(r + 2 * step);
      fetch(r + step);
      if constexpr (FWD) combine(m, sum);
      if (FWD && slice == 0) {
        float loss = 0.f;
        if (live) {
          const float lnt = logf(tsum), lns = logf(sum);
#pragma unroll
          for (int k = 0; k < kLaneTop; ++k) {
            const float p = i[k] >= 0 ? ex2(t[k] * c2) / tsum : 0.f;
            if (!(p <= 0.f)) loss += p * ((t[k] * inv_tau - lnt) - ((to_f32(v[k]) - m) * inv_tau - lns));
          }
#pragma unroll
          for (int o = 16; o; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
        }
        if (lane == 0) {
          a.loss[r] = live ? loss * weight_now * a.tau * a.tau : 0.f;
          if (a.stats) {
            a.stats[2 * r] = live ? m : 0.f;
            a.stats[2 * r + 1] = live ? sum : 0.f;
          }
        }
      }
      // each class once, with the sum of its entries, by the lane of its first entry
      float hit[kLaneTop];
      unsigned mine = 0;
#pragma unroll
      for (int k = 0; k < kLaneTop; ++k) {
        hit[k] = 0.f;
        const bool here = (i[k] >= c0 && i[k] < c1) || (slice == 0 && (i[k] < span.head || i[k] >= span.tail0));
        if (i[k] >= 0 && here) mine |= 1u << k;
      }
      if (a.dlogits && live) {
#pragma unroll 4
        for (int k2 = 0; k2 < top; ++k2) {
          const Entry e = entries[k2];
#pragma unroll
          for (int k = 0; k < kLaneTop; ++k) {
            if (k * 32 >= top) break;
            if (e.index == i[k]) {
              hit[k] += e.teacher;
              if (k2 < k * 32 + lane) mine &= ~(1u << k);
            }
          }
        }
      }
      __syncwarp();  // the entries have been read
      T* ds = static_cast<T*>(a.dlogits) + r * (long long)a.classes;
      if (a.dlogits && ragged) ds[ragged_at] = from_f32<T>(live ? ex2((end - m) * c2) * (coef / sum) : 0.f);
      named_sync(kWritten, NT);
      if (a.dlogits && live) {
#pragma unroll
        for (int k = 0; k < kLaneTop; ++k)
          if (mine >> k & 1) ds[i[k]] = from_f32<T>(coef * (ex2((to_f32(v[k]) - m) * c2) / sum - hit[k] / tsum));
      }
    }
  }
}

// ------------------------------------------------------------------------- rows of up to 8 KB
// A warp a row, which it holds in registers (NV vectors a lane); the gradient is put together in shared
// memory in fp32: q, then minus p at the entries' classes, 32 entries at a time (equal classes among
// them are found by a match over the lanes and added up by the first), then stored in lines.  Rows in
// flight on other warps hide the latency of one row's steps.
template <class T, int NV, int WARPS, int KT, int BLOCKS, bool FWD>
__global__ void __launch_bounds__(32 * WARPS, BLOCKS) distill_warp_kernel(DistillArgs a) {
  constexpr int kV = 16 / sizeof(T), kWarps = WARPS;
  extern __shared__ float4 warp_smem[];  // a warp: its gradient row, then its entries' probabilities
  __shared__ float probs_all[kWarps][32 * KT];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* grad = reinterpret_cast<float*>(warp_smem) + warp * ((a.classes + 2 * kV + 3) / 4 * 4);
  float* probs = probs_all[warp];
  const float c2 = a.c2, inv_tau = a.inv_tau;
  const int top = (int)a.top;
  const uint32_t low = sizeof(T) == 4 ? 0xFF800000u : (__is_same(T, __nv_bfloat16) ? 0xFF80FF80u : 0xFC00FC00u);  // -inf
  for (long long r = (long long)blockIdx.x * kWarps + warp; r < a.rows; r += (long long)gridDim.x * kWarps) {
    const T* s = static_cast<const T*>(a.logits) + r * a.s_stride;
    const RowSpan<T> span(s, a.classes);
    const uint4* sv = reinterpret_cast<const uint4*>(s + span.head);
    // everything is asked for before anything is used
    const float w = a.weight ? a.weight[r] : 1.f;
    int i[KT];
    float t[KT];
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      i[k] = -1;
      t[k] = -kInf;
      if (k * 32 + lane < top) {
        i[k] = index_of(a, r, k * 32 + lane);
        t[k] = teacher_of(a, r, k * 32 + lane);
      }
    }
    uint4 q[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) q[u] = u * 32 + lane < span.vecs ? __ldg(sv + u * 32 + lane) : make_uint4(low, low, low, low);
    const bool ragged = lane < span.ragged();
    const float end = ragged ? to_f32(s[span.ragged_at(lane)]) : -kInf;
    T v[KT];
    float tmax = -kInf, tsum = 0.f;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      if (k * 32 >= top) break;
      v[k] = s[i[k] >= 0 ? i[k] : 0];
      t[k] = i[k] >= 0 ? t[k] : -kInf;
      tmax = fmaxf(tmax, t[k] != t[k] ? kInf : t[k]);  // NaN and +inf end in NaN
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
    T* ds = static_cast<T*>(a.dlogits) + r * (long long)a.classes;
    const bool vec_out = ((reinterpret_cast<uintptr_t>(ds) ^ reinterpret_cast<uintptr_t>(s)) & 15) == 0;
    if (w == 0.f || tmax == -kInf) {  // no weight, or no entry
      if (FWD && lane == 0) {
        a.loss[r] = 0.f;
        if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
      }
      if (a.dlogits) {
        if (vec_out) {
          for (int j = lane; j < span.vecs; j += 32) reinterpret_cast<uint4*>(ds + span.head)[j] = make_uint4(0, 0, 0, 0);
          if (ragged) ds[span.ragged_at(lane)] = from_f32<T>(0.f);
        } else {
          for (int j = lane; j < a.classes; j += 32) ds[j] = from_f32<T>(0.f);
        }
      }
      continue;
    }
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      if (k * 32 >= top) break;
      t[k] -= tmax;
      const float p = i[k] >= 0 ? ex2(t[k] * c2) : 0.f;
      probs[k * 32 + lane] = p;
      tsum += p;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) tsum += __shfl_xor_sync(0xffffffffu, tsum, o);
    float m, sum;
    if constexpr (FWD) {
      Largest<T> most(low);
#pragma unroll
      for (int u = 0; u < NV; ++u)
        if (u * 32 < span.vecs) most.add(q[u]);
      m = fmaxf(most.get(), end);
#pragma unroll
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float from = m == -kInf ? 0.f : m;
      sum = ragged ? ex2((end - from) * c2) : 0.f;
#pragma unroll
      for (int u = 0; u < NV; ++u)
        if (u * 32 < span.vecs) sum += exp_sum<T>(q[u], from, c2);
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (m == -kInf) sum = m - m;  // a row of -inf only: NaN
      const float lnt = logf(tsum), lns = logf(sum);
      float loss = 0.f;
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        if (k * 32 >= top) break;
        const float p = probs[k * 32 + lane] * rcp(tsum);
        if (i[k] >= 0 && !(p <= 0.f)) loss += p * ((t[k] * inv_tau - lnt) - ((to_f32(v[k]) - m) * inv_tau - lns));
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
    } else {
      m = a.stats[2 * r];
      sum = a.stats[2 * r + 1];
    }
    if (!a.dlogits) continue;
    const float coef = w * a.tau * (a.grad ? a.grad[r * a.grad_stride] : 1.f);
    const float cq = coef / sum, cp = coef / tsum;
    const int off = (kV - span.head) % kV;  // class j lies at grad[j + off]: vectors on their boundaries
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if (u * 32 >= span.vecs) break;
      const int j = u * 32 + lane;
      if (j < span.vecs) {
        float f[kV];
        unpack<T>(q[u], f);
        float4* to = reinterpret_cast<float4*>(grad + span.head + off + j * kV);
#pragma unroll
        for (int e = 0; e < kV; e += 4) {
          const float2 d0 = scaled2(f[e], f[e + 1], m, c2), d1 = scaled2(f[e + 2], f[e + 3], m, c2);
          to[e / 4] = make_float4(ex2(d0.x) * cq, ex2(d0.y) * cq, ex2(d1.x) * cq, ex2(d1.y) * cq);
        }
      }
    }
    if (ragged) grad[span.ragged_at(lane) + off] = ex2((end - m) * c2) * cq;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      if (k * 32 >= top) break;
      const unsigned peers = __match_any_sync(0xffffffffu, i[k]);
      if (i[k] >= 0 && __ffs(peers) - 1 == lane) {
        float p = 0.f;
        for (unsigned b = peers; b; b &= b - 1) p += probs[k * 32 + __ffs(b) - 1];
        grad[i[k] + off] -= cp * p;
      }
      __syncwarp();
    }
    if (vec_out) {
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        if (u * 32 >= span.vecs) break;
        const int j = u * 32 + lane;
        if (j < span.vecs) {
          const float4* from = reinterpret_cast<const float4*>(grad + span.head + off + j * kV);
          float f[kV];
#pragma unroll
          for (int e = 0; e < kV; e += 4) {
            const float4 x = from[e / 4];
            f[e] = x.x, f[e + 1] = x.y, f[e + 2] = x.z, f[e + 3] = x.w;
          }
          __stcs(reinterpret_cast<uint4*>(ds + span.head) + j, pack<T>(f));
        }
      }
      if (ragged) ds[span.ragged_at(lane)] = from_f32<T>(grad[span.ragged_at(lane) + off]);
    } else {
      for (int j = lane; j < a.classes; j += 32) ds[j] = from_f32<T>(grad[j + off]);
    }
    __syncwarp();  // the row has been read
  }
}

template <class T, int G, int K, int KE, bool FWD>
int32_t launch_small(const DistillArgs& a, bool same, cudaStream_t s) {
  const long long blocks = (a.rows + kThreads / G - 1) / (kThreads / G);
  const unsigned grid = (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16);  // several rows a thread pay its set-up
  const auto run = [&](auto index) {
    using I = decltype(index);
    if (same) distill_small_kernel<T, I, G, K, KE, true, FWD><<<grid, kThreads, 0, s>>>(a);
    else distill_small_kernel<T, I, G, K, KE, false, FWD><<<grid, kThreads, 0, s>>>(a);
  };
  if (a.index_bits == 32) run(int{});
  else run((long long){});
  return launch_status();
}

constexpr int kMostEntries = 4096;  // staged in shared memory: 8 bytes each

// A launch in clusters of `slices` blocks that go through rows: `most` clusters, but no more than run
// at once (a cluster that started after the others had ended would double the time).  `room` keeps
// that number by device and cluster size.
constexpr int kMaxDevices = 64;
using Room = std::atomic<int>[kMaxDevices][kMostSlices + 1];

int32_t launch_clusters(void (*kernel)(DistillArgs, int), Room& room, const DistillArgs& a, long long most, int slices,
                        int threads, size_t smem, cudaStream_t s) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return NCA_ERR_DEVICE;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = slices;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(slices);
  int n = room[dev][slices].load(std::memory_order_relaxed);
  if (n == 0) {
    if (smem > 32 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) {
      const int32_t st = launch_status();
      return st == NCA_OK ? NCA_ERR_CUDA : st;
    }
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      const int32_t st = launch_status();
      return st == NCA_OK ? NCA_ERR_CUDA : st;
    }
    room[dev][slices].store(n, std::memory_order_relaxed);
  }
  cfg.gridDim = dim3((unsigned)((most < n ? most : n) * slices));
  if (cudaLaunchKernelEx(&cfg, kernel, a, slices) != cudaSuccess) {
    const int32_t st = launch_status();
    return st == NCA_OK ? NCA_ERR_CUDA : st;
  }
  return launch_status();
}

template <class T, int NT, bool FWD>
int32_t launch_rows(const DistillArgs& a, int slices, cudaStream_t s) {
  static Room room;
  return launch_clusters(distill_row_kernel<T, NT, FWD>, room, a, a.rows, slices, NT, a.top * sizeof(Entry), s);
}

template <class T, int NV, int WARPS, int KT, int BLOCKS, bool FWD>
int32_t launch_warps(const DistillArgs& a, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  auto* kernel = distill_warp_kernel<T, NV, WARPS, KT, BLOCKS, FWD>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return NCA_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 72 * 1024) != cudaSuccess) {
      const int32_t st = launch_status();
      return st == NCA_OK ? NCA_ERR_CUDA : st;
    }
    ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  constexpr int kV = 16 / sizeof(T);
  const size_t smem = a.dlogits ? (size_t)WARPS * ((a.classes + 2 * kV + 3) / 4 * 4) * sizeof(float) : 0;
  const long long blocks = (a.rows + WARPS - 1) / WARPS;
  kernel<<<(unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 32 * WARPS, smem, s>>>(a);
  return launch_status();
}

template <class T, int NS, int NSM, int BLOCKS, bool FWD>
int32_t launch_held(const DistillArgs& a, int slices, cudaStream_t s) {
  static Room room;
  return launch_clusters(distill_held_kernel<T, NS, NSM, BLOCKS, FWD>, room, a, a.rows, slices, NS + 32,
                         (size_t)NSM * NS * 16, s);
}

// Blocks that share a row: as many as keep the rows in flight (two blocks a multiprocessor) small
// enough for L2 to hold them until the second pass, more when there are few rows.
int slices_of(const DistillArgs& a, size_t size) {
  int n = 1;
  while (n < kMostSlices && (a.classes * size / n > 131072 || a.rows * n < 148) && a.classes * size / n > 8192) n *= 2;
  return n;
}

template <bool FWD>
int32_t dispatch(const NcaDistillDesc& d, const DistillArgs& a, cudaStream_t s) {
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    const bool same = d.dtype == d.teacher_dtype;
    if (a.classes <= 2 && a.top <= 2) return launch_small<T, 1, 2, 2, FWD>(a, same, s);
    if (a.classes <= 4 && a.top <= 4) return launch_small<T, 1, 4, 4, FWD>(a, same, s);
    if (a.classes <= 16 && a.top <= 4) return launch_small<T, 4, 4, 1, FWD>(a, same, s);
    if (a.classes <= 16 && a.top <= 16) return launch_small<T, 4, 4, 4, FWD>(a, same, s);
    if (a.classes <= 64 && a.top <= 8) return launch_small<T, 8, 8, 1, FWD>(a, same, s);
    if (a.classes <= 128 && a.top <= 16) return launch_small<T, 16, 8, 1, FWD>(a, same, s);
    if (a.classes <= 256 && a.top <= 32) return launch_small<T, 32, 8, 1, FWD>(a, same, s);
    const size_t bytes = a.classes * sizeof(T);
    // many rows of up to 8 KB by warps; few ones go to blocks, whose lanes share a row's work.  With no
    // registers for more entries and vectors than there are, more warps fit (950,000 x 514 bf16, 2
    // entries: 823 us, as 8 vectors and 128 entries 1080).
    const bool many = a.rows >= 148 * 8 || bytes <= 2048;
    if (many && bytes <= 32 * 16 * 16 && a.top <= 32 * kLaneTop) {
      if (bytes <= 32 * 4 * 16 && a.top <= 32) return launch_warps<T, 4, 8, 1, 6, FWD>(a, s);
      if (bytes <= 32 * 4 * 16) return launch_warps<T, 4, 8, kLaneTop, 5, FWD>(a, s);
      if (bytes <= 32 * 8 * 16 && a.top <= 32) return launch_warps<T, 8, 8, 1, 4, FWD>(a, s);
      if (bytes <= 32 * 8 * 16) return launch_warps<T, 8, 8, kLaneTop, 4, FWD>(a, s);
      return launch_warps<T, 16, 4, kLaneTop, 4, FWD>(a, s);
    }
    constexpr auto held = [](int lanes, int in_smem) { return (size_t)lanes * (kHeld + in_smem) * 16; };
    constexpr size_t kMiddle = held(256, 8), kLarge = held(992, 9);
    if (a.top <= 32 * kLaneTop && bytes <= kMostSlices * kLarge) {
      if (bytes <= held(96, 0)) return launch_held<T, 96, 0, 8, FWD>(a, 1, s);
      // Many rows: the smallest block that holds one, so that a multiprocessor has several, each at
      // another row, and few places stay empty.  Measured, loss and gradient, against 256 x 16 vectors
      // (to 64 KB) or 992 x 17: 25000 x 12000 bf16 263 (437) us, 14873 x 16384 200 (281), 14873 x 17000
      // 252 (288), 7000 x 34528 217 (432), 4000 x 65536 211 (292).
      if (a.rows >= 148 * 4) {
        if (bytes <= held(192, 0)) return launch_held<T, 192, 0, 4, FWD>(a, 1, s);
        if (bytes <= held(256, 0)) return launch_held<T, 256, 0, 3, FWD>(a, 1, s);
        if (bytes <= held(384, 0)) return launch_held<T, 384, 0, 2, FWD>(a, 1, s);
        // the loss alone needs no second look at a row: 4000 x 65536 bf16 123 us, held 210
        if constexpr (FWD) {
          if (!a.dlogits && bytes > kMiddle) return launch_rows<T, 256, FWD>(a, 1, s);
        }
        if (bytes > kMiddle && bytes <= held(256, 13)) return launch_held<T, 256, 13, 3, FWD>(a, 1, s);
        if (bytes > kMiddle && bytes <= held(480, 10)) return launch_held<T, 480, 10, 2, FWD>(a, 1, s);
      }
      int slices = 1;  // a row over several blocks where one cannot hold it, or where there are few rows
      const bool middle = bytes <= kMiddle || (a.rows < 74 && bytes <= kMostSlices * kMiddle);
      while (bytes > slices * (middle ? kMiddle : kLarge) ||
             (slices * 2 <= kMostSlices && a.rows * slices < 148 && bytes > (size_t)slices * 8192))
        slices *= 2;
      return middle ? launch_held<T, 256, 8, 3, FWD>(a, slices, s) : launch_held<T, 992, 9, 1, FWD>(a, slices, s);
    }
    return launch_rows<T, 512, FWD>(a, slices_of(a, sizeof(T)), s);
  });
}

int32_t check_desc(const NcaDistillDesc* d) {
  if (!d || d->rows < 0 || d->classes <= 0 || d->top < 0) return NCA_ERR_INVALID;
  if (!dtype_ok(d->dtype) || !dtype_ok(d->teacher_dtype)) return NCA_ERR_INVALID;
  if (d->index_bits != 32 && d->index_bits != 64) return NCA_ERR_INVALID;
  // below, log2(e) / tau would overflow, and equal logits give 0 times infinity
  if (!(d->temperature >= 1e-30f) || d->temperature > 1e30f) return NCA_ERR_INVALID;
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
  a.c2 = kLog2e / d.temperature;
  a.inv_tau = 1.f / d.temperature;
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
  *bytes = 0;  // the kernels need none; the argument keeps room for one that does
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
