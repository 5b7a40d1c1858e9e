// norm_held_forward.cu -- the forward kernel of norm_held.cuh.
#include "norm_held.cuh"

namespace nca {
namespace {

template <class T, int V, int ACT, bool MASK, bool ONE>
__global__ void __launch_bounds__(kMaxThreads, 2) norm_held_forward_kernel(const __grid_constant__ HeldArgs h) {
  constexpr int P = (V + 1) / 2, U = ONE ? 1 : P;  // U: units of a thread, each in one group
  constexpr int kUnit = ONE ? V : 2;               // channels of a unit
  const NormArgs& a = h.a;
  extern __shared__ uint4 smem_raw[];
  using VecT = Vec<T, V>;
  if (h.slices > 1) cluster_started_arrive();
  may_start_next();
  after_previous();
  const Work w = work_of<V>(h);
  const uint32_t kept = kept_of<MASK>(a, w);
  const int threads = blockDim.x, groups = h.cb / a.per_group;
  float4* all = reinterpret_cast<float4*>(smem_raw);            // [slices][groups] (n, mean, M2)
  VecT* xs = reinterpret_cast<VecT*>(all + h.slices * groups);  // [iters][threads]
  float2* part = reinterpret_cast<float2*>(xs + h.iters * threads);  // [threads][U] (mean, M2)
  int* count = reinterpret_cast<int*>(part + threads * U);      // [ty] cells of a row of threads
  {
    const T* x = static_cast<const T*>(a.x) + w.sample * a.x_sn + w.ch + w.c0 * a.x_sl;
    each_cell<MASK>(a, w, kept, [&](int at, int c) { copy_async<sizeof(VecT)>(xs + at, x + c * a.x_sl); }, [](int, int) {});
  }
  float2 wt[P], b[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = min(w.ch + 2 * i, a.channels - 1), c1 = min(c + (V > 1), a.channels - 1);
    wt[i] = a.weight ? make_float2(load_param(a.weight, a.param_dtype, c), load_param(a.weight, a.param_dtype, c1)) : both(1.f);
    b[i] = a.bias ? make_float2(load_param(a.bias, a.param_dtype, c), load_param(a.bias, a.param_dtype, c1)) : both(0.f);
  }
  copy_wait();
  {
    float k[U];
    float2 s1[U], s2[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = 0.f, s1[u] = s2[u] = both(0.f);
    int cnt = 0;
    each_cell<MASK>(
        a, w, kept,
        [&](int at, int) {
          float2 f[P];
          to_pairs<T, V>(xs[at], f);
          if (cnt == 0) {
#pragma unroll
            for (int u = 0; u < U; ++u) k[u] = f[u].x;
          }
          ++cnt;
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const int u = ONE ? 0 : i;
            const float2 d = add2(f[i], both(-k[u]));
            s1[u] = add2(s1[u], d);
            s2[u] = fma2(d, d, s2[u]);
          }
        },
        [](int, int) {});
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float t1 = V > 1 ? s1[u].x + s1[u].y : s1[u].x, t2 = V > 1 ? s2[u].x + s2[u].y : s2[u].x;
      const float m = cnt ? t1 / (float)(cnt * kUnit) : 0.f;
      const float rest = t2 - t1 * m;
      part[threadIdx.x * U + u] = make_float2(k[u] + m, rest < 0.f ? 0.f : rest);  // keeps NaN
    }
    if (w.on && w.col == 0) count[w.row] = cnt;
  }
  __syncthreads();
  if (h.slices > 1) cluster_started_wait();
  // a warp a group: its ty x cols partial results, lanes over rows of threads
  const int cols = a.per_group / kUnit, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wide = cols < 32 ? cols : 32, high = 32 / wide, lrow = lane / wide, lcol = lane % wide;
  for (int g = warp; g < groups; g += threads >> 5) {
    float n = 0.f, mean = 0.f, m2 = 0.f;
    for (int row = lrow; row < a.ty && lrow < high; row += high) {
      const float f = (float)(count[row] * kUnit);
      for (int c = lcol; c < cols; c += wide) {
        n += f;
        if (f > 0.f) mean = fmaf(f, part[row * a.tx * U + g * cols + c].x, mean);
      }
    }
    n = warp_sum(n);
    mean = warp_sum(mean);
    mean = n > 0.f ? mean / n : 0.f;
    for (int row = lrow; row < a.ty && lrow < high; row += high) {
      const float f = (float)(count[row] * kUnit);
      for (int c = lcol; c < cols; c += wide) {
        const float2 e = part[row * a.tx * U + g * cols + c];
        const float d = e.x - mean;
        if (f > 0.f) m2 += fmaf(f * d, d, e.y);
      }
    }
    m2 = warp_sum(m2);
    const float4 mine = make_float4(n, mean, m2, 0.f);
    if (h.slices > 1) {
      if (lane < h.slices) put_remote(&all[w.rank * groups + g], lane, mine);
    } else if (lane == 0) {
      all[g] = mine;
    }
  }
  if (h.slices > 1) cluster_barrier();
  else __syncthreads();
  if (!w.on) return;
  float mean[U], rstd[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int group = (w.col * V + u * kUnit) / a.per_group;  // within the block
    float n = 0.f, mu = 0.f, m2 = 0.f;
    if (h.slices == 1) {
      const float4 e = all[group];
      n = e.x, mu = e.y, m2 = e.z;
    } else {
      for (int i = 0; i < h.slices; ++i) {
        const float4 e = all[i * groups + group];
        n += e.x;
        if (e.x > 0.f) mu = fmaf(e.x, e.y, mu);
      }
      mu = n > 0.f ? mu / n : 0.f;
      for (int i = 0; i < h.slices; ++i) {
        const float4 e = all[i * groups + group];
        const float d = e.y - mu;
        if (e.x > 0.f) m2 += fmaf(e.x * d, d, e.z);
      }
    }
    mean[u] = mu;
    rstd[u] = n > 0.f ? 1.f / sqrtf(m2 / n + a.eps) : 0.f;
    const int ch = w.ch + u * kUnit;
    if (a.stats && w.rank == 0 && w.row == 0 && ch % a.per_group == 0) {
      float* st = a.stats + 2 * (w.sample * a.groups + ch / a.per_group);
      st[0] = mean[u];
      st[1] = rstd[u];
    }
  }
#pragma unroll
  for (int i = 0; i < P; ++i) wt[i] = mul2(wt[i], both(rstd[ONE ? 0 : i]));
  T* y = static_cast<T*>(a.y) + (w.sample * a.cells + w.c0) * a.channels + w.ch;
  each_cell<MASK>(
      a, w, kept,
      [&](int at, int c) {
        float2 f[P];
        to_pairs<T, V>(xs[at], f);
#pragma unroll
        for (int i = 0; i < P; ++i) f[i] = act2<ACT>(fma2(add2(f[i], both(-mean[ONE ? 0 : i])), wt[i], b[i]));
        *reinterpret_cast<VecT*>(y + (long long)c * a.channels) = from_pairs<T, V>(f);
      },
      [&](int, int c) {
        VecT v;
#pragma unroll
        for (int i = 0; i < V; ++i) v.v[i] = from_f32<T>(0.f);
        *reinterpret_cast<VecT*>(y + (long long)c * a.channels) = v;
      });
}

struct Call {
  const NormArgs& a;
  const HeldPlan& p;
  cudaStream_t s;
  template <class T, int V, int ACT, bool MASK, bool ONE>
  int32_t operator()() const {
    static std::atomic<uint64_t> ready{0};
    return launch(norm_held_forward_kernel<T, V, ACT, MASK, ONE>, ready, a, p, s);
  }
};

}  // namespace

int32_t norm_held_forward(const NormArgs& a, int dtype, int act, int v, cudaStream_t s) {
  const HeldPlan p = plan_of(a, dtype, v, false);
  return dispatch_held(a, dtype, act, p, Call{a, p, s});
}

}  // namespace nca
