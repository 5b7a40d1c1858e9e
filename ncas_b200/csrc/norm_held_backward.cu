// norm_held_backward.cu -- the backward kernel of norm_held.cuh.
//
// The first pass over the held values sums dz and dz h by channel, the second writes dx.  fp32 keeps
// dz in the place of dy between the two; 16-bit types work it out again (its rounding to their type
// would show in dx).
#include "norm_held.cuh"

namespace nca {
namespace {

template <class T, int V, int ACT, bool MASK, bool ONE>
__global__ void __launch_bounds__(kMaxThreads, 2) norm_held_backward_kernel(const __grid_constant__ HeldArgs h) {
  constexpr int P = (V + 1) / 2, U = ONE ? 1 : P;  // U: units of a thread, each in one group
  constexpr int kUnit = ONE ? V : 2;               // channels of a unit
  constexpr bool kKeep = sizeof(T) == 4;
  const NormArgs& a = h.a;
  extern __shared__ uint4 smem_raw[];
  using VecT = Vec<T, V>;
  const int threads = blockDim.x;
  const int groups = h.cb / a.per_group;
  float4* all = reinterpret_cast<float4*>(smem_raw);            // [slices][groups] (A, B, n)
  VecT* xs = reinterpret_cast<VecT*>(all + h.slices * groups);  // [iters][threads], then dy the same
  VecT* gs = xs + h.iters * threads;
  float2* red = reinterpret_cast<float2*>(gs + h.iters * threads);  // [ty][tx * V] (sum dz, sum dz h)
  float2* chan = red + a.ty * a.tx * V;                             // [cb] totals of the block
  int* count = reinterpret_cast<int*>(chan + h.cb);                 // [ty] cells of a row of threads
  if (h.slices > 1) cluster_started_arrive();
  may_start_next();
  after_previous();
  const Work w = work_of<V>(h);
  const uint32_t kept = kept_of<MASK>(a, w);
  {
    const T* x = static_cast<const T*>(a.x) + w.sample * a.x_sn + w.ch + w.c0 * a.x_sl;
    const T* dy = static_cast<const T*>(a.dy) + w.sample * a.dy_sn + w.ch + w.c0 * a.dy_sl;
    each_cell<MASK>(
        a, w, kept,
        [&](int at, int c) {
          copy_async<sizeof(VecT)>(xs + at, x + c * a.x_sl);
          copy_async<sizeof(VecT)>(gs + at, dy + c * a.dy_sl);
        },
        [](int, int) {});
  }
  float mean[U], rstd[U];
  float2 wt[P], b[P], s1[P], s2[P];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float* st = a.stats + 2 * (w.sample * a.groups + (w.ch + u * kUnit) / a.per_group);
    mean[u] = w.on ? st[0] : 0.f;
    rstd[u] = w.on ? st[1] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = min(w.ch + 2 * i, a.channels - 1), c1 = min(c + (V > 1), a.channels - 1);
    wt[i] = a.weight ? make_float2(load_param(a.weight, a.param_dtype, c), load_param(a.weight, a.param_dtype, c1)) : both(1.f);
    b[i] = a.bias ? make_float2(load_param(a.bias, a.param_dtype, c), load_param(a.bias, a.param_dtype, c1)) : both(0.f);
    s1[i] = s2[i] = both(0.f);
  }
  copy_wait();
  int cnt = 0;
  each_cell<MASK>(
      a, w, kept,
      [&](int at, int) {
        ++cnt;
        float2 f[P], g[P];
        to_pairs<T, V>(xs[at], f);
        to_pairs<T, V>(gs[at], g);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 hh = mul2(add2(f[i], both(-mean[ONE ? 0 : i])), both(rstd[ONE ? 0 : i]));
          float2 unused;
          g[i] = mul2(g[i], act_slope2<ACT>(fma2(hh, wt[i], b[i]), unused));
          s1[i] = add2(s1[i], g[i]);
          s2[i] = fma2(g[i], hh, s2[i]);
        }
        if constexpr (kKeep) gs[at] = from_pairs<T, V>(g);
      },
      [](int, int) {});
  if (w.on) {
    if (w.col == 0) count[w.row] = cnt;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float2* to = red + (w.row * a.tx + w.col) * V + 2 * i;
      to[0] = make_float2(s1[i].x, s2[i].x);
      if (V > 1) to[1] = make_float2(s1[i].y, s2[i].y);
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < h.cb; c += threads) {
    float2 s = both(0.f);
    for (int r = 0; r < a.ty; ++r) s = add2(s, red[r * a.tx * V + c]);
    chan[c] = s;
    if (a.part) a.part[(w.sample * h.slices + w.rank) * a.channels + w.ch0 + c] = s;  // of the parameters' gradients
  }
  __syncthreads();
  if (h.slices > 1) cluster_started_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < groups; g += threads >> 5) {
    float sa = 0.f, sb = 0.f, n = 0.f;
    for (int i = lane; i < a.per_group; i += 32) {
      const int c = g * a.per_group + i;
      const float wc = a.weight ? load_param(a.weight, a.param_dtype, w.ch0 + c) : 1.f;
      sa = fmaf(wc, chan[c].x, sa);
      sb = fmaf(wc, chan[c].y, sb);
    }
    for (int r = lane; r < a.ty; r += 32) n += (float)count[r];
    sa = warp_sum(sa);
    sb = warp_sum(sb);
    n = warp_sum(n) * (float)a.per_group;
    const float4 mine = make_float4(sa, sb, n, 0.f);
    if (h.slices > 1) {
      if (lane < h.slices) put_remote(&all[w.rank * groups + g], lane, mine);
    } else if (lane == 0) {
      all[g] = mine;
    }
  }
  if (h.slices > 1) cluster_barrier();
  else __syncthreads();
  if (!w.on || !a.y) return;
  float ga[U], gb[U];  // -A / n, -B / n
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int group = (w.col * V + u * kUnit) / a.per_group;  // within the block
    float sa = 0.f, sb = 0.f, n = 0.f;
    for (int i = 0; i < h.slices; ++i) {
      const float4 e = all[i * groups + group];
      sa += e.x;
      sb += e.y;
      n += e.z;
    }
    ga[u] = n > 0.f ? -sa / n : 0.f;
    gb[u] = n > 0.f ? -sb / n : 0.f;
  }
  T* dx = static_cast<T*>(a.y) + (w.sample * a.cells + w.c0) * a.channels + w.ch;
  each_cell<MASK>(
      a, w, kept,
      [&](int at, int c) {
        float2 f[P], g[P];
        to_pairs<T, V>(xs[at], f);
        to_pairs<T, V>(gs[at], g);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 hh = mul2(add2(f[i], both(-mean[ONE ? 0 : i])), both(rstd[ONE ? 0 : i]));
          float2 unused;
          if constexpr (!kKeep) g[i] = mul2(g[i], act_slope2<ACT>(fma2(hh, wt[i], b[i]), unused));
          // rstd (w dz - (A + h B) / n), each product rounded: one value a group gives exactly 0
          const int u = ONE ? 0 : i;
          f[i] = mul2(add2(mul2(wt[i], g[i]), fma2(hh, both(gb[u]), both(ga[u]))), both(rstd[u]));
        }
        *reinterpret_cast<VecT*>(dx + (long long)c * a.channels) = from_pairs<T, V>(f);
      },
      [&](int, int c) {
        VecT v;
#pragma unroll
        for (int i = 0; i < V; ++i) v.v[i] = from_f32<T>(0.f);
        *reinterpret_cast<VecT*>(dx + (long long)c * a.channels) = v;
      });
}

struct Call {
  const NormArgs& a;
  const HeldPlan& p;
  cudaStream_t s;
  template <class T, int V, int ACT, bool MASK, bool ONE>
  int32_t operator()() const {
    static std::atomic<uint64_t> ready{0};
    return launch(norm_held_backward_kernel<T, V, ACT, MASK, ONE>, ready, a, p, s);
  }
};

}  // namespace

int norm_held_slices(const NormArgs& a, int dtype, int v, bool backward) {
  const HeldPlan p = plan_of(a, dtype, v, backward);
  return p.ok ? p.slices : 0;
}
int32_t norm_held_backward(const NormArgs& a, int dtype, int act, int v, cudaStream_t s) {
  const HeldPlan p = plan_of(a, dtype, v, true);
  return dispatch_held(a, dtype, act, p, Call{a, p, s});
}

}  // namespace nca
