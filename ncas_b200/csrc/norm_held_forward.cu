// norm_held_forward.cu -- the forward kernel of norm_held.cuh.
#include "norm_held.cuh"

namespace nca {
namespace {

template <class T, int V, int ACT, bool MASK>
__global__ void __launch_bounds__(kMaxThreads, 2) norm_held_forward_kernel(const __grid_constant__ HeldArgs h) {
  constexpr int P = (V + 1) / 2;
  const NormArgs& a = h.a;
  extern __shared__ uint4 smem_raw[];
  using VecT = Vec<T, V>;
  may_start_next();
  after_previous();
  const Work w = work_of<V>(h);
  const uint32_t kept = kept_of<MASK>(a, w);
  const int threads = blockDim.x, groups = h.cb / a.per_group;
  float4* all = reinterpret_cast<float4*>(smem_raw);            // [slices][groups] (n, mean, M2)
  VecT* xs = reinterpret_cast<VecT*>(all + h.slices * groups);  // [iters][threads]
  float2* part = reinterpret_cast<float2*>(xs + h.iters * threads);  // [threads] (mean, M2)
  int* count = reinterpret_cast<int*>(part + threads);          // [ty] cells of a row of threads
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
    float k = 0.f;
    float2 s1 = both(0.f), s2 = both(0.f);
    int cnt = 0;
    each_cell<MASK>(
        a, w, kept,
        [&](int at, int) {
          float2 f[P];
          to_pairs<T, V>(xs[at], f);
          if (cnt == 0) k = f[0].x;
          ++cnt;
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 d = add2(f[i], both(-k));
            s1 = add2(s1, d);
            s2 = fma2(d, d, s2);
          }
        },
        [](int, int) {});
    const float t1 = V > 1 ? s1.x + s1.y : s1.x, t2 = V > 1 ? s2.x + s2.y : s2.x;
    const float m = cnt ? t1 / (float)(cnt * V) : 0.f;
    const float rest = t2 - t1 * m;
    part[threadIdx.x] = make_float2(k + m, rest < 0.f ? 0.f : rest);  // keeps NaN
    if (w.on && w.col == 0) count[w.row] = cnt;
  }
  __syncthreads();
  // a warp a group: its ty x cols partial results, lanes over rows of threads
  const int cols = a.per_group / V, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wide = cols < 32 ? cols : 32, high = 32 / wide, lrow = lane / wide, lcol = lane % wide;
  for (int g = warp; g < groups; g += threads >> 5) {
    float n = 0.f, mean = 0.f, m2 = 0.f;
    for (int row = lrow; row < a.ty && lrow < high; row += high) {
      const float f = (float)(count[row] * V);
      for (int c = lcol; c < cols; c += wide) {
        n += f;
        if (f > 0.f) mean = fmaf(f, part[row * a.tx + g * cols + c].x, mean);
      }
    }
    n = warp_sum(n);
    mean = warp_sum(mean);
    mean = n > 0.f ? mean / n : 0.f;
    for (int row = lrow; row < a.ty && lrow < high; row += high) {
      const float f = (float)(count[row] * V);
      for (int c = lcol; c < cols; c += wide) {
        const float2 e = part[row * a.tx + g * cols + c];
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
  float n = 0.f, mean = 0.f, m2 = 0.f;
  if (h.slices == 1) {
    const float4 e = all[w.group];
    n = e.x, mean = e.y, m2 = e.z;
  } else {
    for (int i = 0; i < h.slices; ++i) {
      const float4 e = all[i * groups + w.group];
      n += e.x;
      if (e.x > 0.f) mean = fmaf(e.x, e.y, mean);
    }
    mean = n > 0.f ? mean / n : 0.f;
    for (int i = 0; i < h.slices; ++i) {
      const float4 e = all[i * groups + w.group];
      const float d = e.y - mean;
      if (e.x > 0.f) m2 += fmaf(e.x * d, d, e.z);
    }
  }
  const float rstd = n > 0.f ? 1.f / sqrtf(m2 / n + a.eps) : 0.f;
  if (a.stats && w.rank == 0 && w.row == 0 && w.ch % a.per_group == 0) {
    float* st = a.stats + 2 * (w.sample * a.groups + w.ch / a.per_group);
    st[0] = mean;
    st[1] = rstd;
  }
#pragma unroll
  for (int i = 0; i < P; ++i) wt[i] = mul2(wt[i], both(rstd));
  T* y = static_cast<T*>(a.y) + (w.sample * a.cells + w.c0) * a.channels + w.ch;
  each_cell<MASK>(
      a, w, kept,
      [&](int at, int c) {
        float2 f[P];
        to_pairs<T, V>(xs[at], f);
#pragma unroll
        for (int i = 0; i < P; ++i) f[i] = act2<ACT>(fma2(add2(f[i], both(-mean)), wt[i], b[i]));
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
  template <class T, int V, int ACT, bool MASK>
  int32_t operator()() const {
    static std::atomic<uint64_t> ready{0};
    return launch(norm_held_forward_kernel<T, V, ACT, MASK>, ready, a, p, s);
  }
};

}  // namespace

int32_t norm_held_forward(const NormArgs& a, int dtype, int act, int v, cudaStream_t s) {
  const HeldPlan p = plan_of(a, dtype, v, false);
  return dispatch_held(a, dtype, act, p.v, Call{a, p, s});
}

}  // namespace nca
