// norm.cu -- group norm with an activation over channels-last samples, forward and backward
// (nca_b200_group_norm*).
//
// A sample is cells x channels; a group is channels / groups adjacent channels of all its cells,
// and its statistics run over the cells that the mask keeps.
//   forward   h = (x - mean) rstd,  y = act(weight h + bias)
//   backward  z = weight h + bias, dz = dy act'(z);  dbias = sum dz, dweight = sum dz h (all samples);
//             A = sum weight dz, B = sum weight dz h (a group), dx = rstd (weight dz - (A + h B) / n)
//
// Sums.  A thread owns V adjacent channels of every TY-th cell.  For the variance it sums x - K and
// (x - K)^2 with K the first value it meets in the channel: since K is one of the values summed, the
// cancellation in sum (x-K)^2 - (sum (x-K))^2 / n loses at most about n ulps for the n values of one
// thread, however far the data lie from zero or K from the rest.  Partial results are (count, mean,
// M2 = sum (x - mean)^2) and merge as mean = sum n_i mean_i / n,
// M2 = sum M2_i + sum n_i (mean_i - mean)^2 (Chan, Golub, LeVeque 1979), in fp32 and in a fixed order.
//
// These are the streaming kernels, for samples that the held form (norm_held.cuh) does not take: two
// passes over the data with a merge between them.  On a B200, 16 x 16384 x 512 bf16, silu: statistics 56 us
// (4.8 TB/s, 73% of the issue slots), application 88 us (6.1 TB/s; the exponentials' unit 75%), gradient
// sums 107 us (5.0 TB/s, 60% of the issue slots), gradient 119 us (6.8 TB/s, part of it from L2).
#include <algorithm>
#include <atomic>

#include "norm.cuh"

using namespace nca;

namespace {

constexpr int kThreads = 256;

struct Place {  // what a block works on
  long long sample, c0, c1;  // cells [c0, c1)
  int chunk, ch;             // first channel of the thread
  bool active;
};

template <int V>
__device__ __forceinline__ Place place_of(const NormArgs& a, long long item) {
  Place p;
  const int ct = (int)(item % a.ctiles);
  const long long rest = item / a.ctiles;
  p.chunk = (int)(rest % a.chunks);
  p.sample = rest / a.chunks;
  p.c0 = p.chunk * a.chunk_cells;
  p.c1 = min(a.cells, p.c0 + a.chunk_cells);
  p.ch = (ct * a.tx + threadIdx.x % a.tx) * V;
  p.active = p.ch < a.channels;
  return p;
}

// The cells of a thread that the mask keeps, a bit each (a block's piece has at most 32 a thread).
template <bool MASK>
__device__ __forceinline__ uint32_t kept_of(const NormArgs& a, const Place& p, int n) {
  if constexpr (!MASK) return ~0u;
  uint32_t bits = 0;
  const long long step = a.ty * a.m_sl;
  const uint8_t* m = a.mask + p.sample * a.m_sn + (p.c0 + threadIdx.x / a.tx) * a.m_sl;
  for (int i = 0; i < n; i += 8, m += 8 * step) {
    uint8_t v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i + u < n ? m[u * step] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) bits |= (uint32_t)(v[u] != 0) << (i + u);
  }
  return bits;
}

// Goes through the thread's cells: use(cell of the piece, x vector, second vector) where the mask keeps the
// cell, left_out(cell) elsewhere.  The vectors (one or two tensors) come through a ring of kRing
// asynchronous copies in places of the thread's own, so that kRing cells are in flight all the time and
// no thread waits for another; single 16-bit values, which such copies cannot move, are loaded to registers,
// kRing cells at a time (417 x 2009 x 69 fp16 backward: 332 us, one at a time 399).
constexpr int kRing = 8;
template <class T, int V>
__host__ __device__ constexpr size_t ring_bytes(int tensors) {
  return V * sizeof(T) >= 4 ? (size_t)kRing * tensors * kThreads * V * sizeof(T) : 0;
}
template <class T, int V, int TENSORS, bool MASK, class U, class O>
__device__ __forceinline__ void each_cell(const NormArgs& a, const Place& p, void* ring, const T* x, long long x_step,
                                          const T* g, long long g_step, U use, O left_out) {
  using VecT = Vec<T, V>;
  const int row = threadIdx.x / a.tx;
  const int n = p.active ? (int)((p.c1 - p.c0 - row + a.ty - 1) / a.ty) : 0;  // cells of this thread
  if (n <= 0) return;
  uint32_t bits = kept_of<MASK>(a, p, n);
  x += (p.c0 + row) * x_step;
  x_step *= a.ty;
  if (TENSORS > 1) {
    g += (p.c0 + row) * g_step;
    g_step *= a.ty;
  }
  if constexpr (V * sizeof(T) >= 4) {
    VecT* place = static_cast<VecT*>(ring) + threadIdx.x;
    uint32_t to_fetch = bits;
    const auto fetch = [&](int slot, bool in) {
      if (in && (to_fetch & 1)) {
        copy_async<sizeof(VecT)>(place + slot * TENSORS * kThreads, x);
        if (TENSORS > 1) copy_async<sizeof(VecT)>(place + (slot * TENSORS + 1) * kThreads, g);
      }
      to_fetch = MASK ? to_fetch >> 1 : to_fetch;
      x += x_step;
      if (TENSORS > 1) g += g_step;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kRing; ++i) fetch(i, i < n);
    int slot = 0;
    for (int i = 0; i < n; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
      if (bits & 1) {
        const VecT xv = place[slot * TENSORS * kThreads];
        use(row + i * a.ty, xv, TENSORS > 1 ? place[(slot * TENSORS + 1) * kThreads] : xv);
      } else {
        left_out(row + i * a.ty);
      }
      bits = MASK ? bits >> 1 : bits;
      fetch(slot, i + kRing < n);
      slot = slot + 1 == kRing ? 0 : slot + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    for (int i = 0; i < n; i += kRing) {
      VecT xv[kRing], gv[TENSORS > 1 ? kRing : 1];
      const uint32_t in = n - i < kRing ? bits & ((1u << (n - i)) - 1) : bits;
#pragma unroll
      for (int u = 0; u < kRing; ++u, x += x_step, g += TENSORS > 1 ? g_step : 0)
        if (in >> u & 1) {
          xv[u] = *reinterpret_cast<const VecT*>(x);
          if (TENSORS > 1) gv[u] = *reinterpret_cast<const VecT*>(g);
        }
#pragma unroll
      for (int u = 0; u < kRing; ++u) {
        if (in >> u & 1)
          use(row + (i + u) * a.ty, xv[u], gv[TENSORS > 1 ? u : 0]);
        else if (MASK && i + u < n)
          left_out(row + (i + u) * a.ty);
      }
      bits = MASK ? bits >> kRing : bits;
    }
  }
}

// The channels of a block's tile, group by group: f(lanes, group, first channel of the tile, width) by as
// many lanes for each group as let all groups be done at once, a warp at most.
struct Lanes {
  int count, lane;  // count a power of two
  __device__ __forceinline__ float sum(float v) const {
    for (int o = count >> 1; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
  }
  // Through rows x width entries: f(row, column).
  template <class F>
  __device__ __forceinline__ void each(int rows, int width, F f) const {
    const int wide = min(width, count), high = wide ? count / wide : 0;
    const int r0 = wide ? lane / wide : 0, c0 = wide ? lane % wide : 0;
    if (r0 >= high) return;
    for (int r = r0; r < rows; r += high)
      for (int c = c0; c < width; c += wide) f(r, c);
  }
};
template <int V, class F>
__device__ __forceinline__ void each_group(const NormArgs& a, long long item, F f) {
  const int c_lo = (int)(item % a.ctiles) * a.tx * V, c_hi = min(a.channels, c_lo + a.tx * V);
  const int first = c_lo / a.per_group, groups = (c_hi - 1) / a.per_group - first + 1;
  const int threads = blockDim.x & ~31;
  if ((int)threadIdx.x >= threads) return;  // an incomplete warp
  Lanes l{32, 0};
  while (l.count > 1 && groups * l.count > threads) l.count >>= 1;
  l.lane = threadIdx.x & (l.count - 1);
  for (int base = 0; base < groups; base += threads / l.count) {
    const bool in = base + (int)(threadIdx.x / l.count) < groups;  // past the last group a width of 0
    const int g = first + (in ? base + (int)(threadIdx.x / l.count) : 0);  // (there g times per_group may pass 32 bits)
    const int lo = max(g * a.per_group, c_lo) - c_lo;
    f(l, g, lo, in ? min((g + 1) * a.per_group, c_hi) - c_lo - lo : 0);
  }
}

// ------------------------------------------------------------------------- forward: statistics
template <class T, int V, bool MASK>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(NormArgs a, long long items) {
  may_start_next();
  after_previous();
  constexpr int P = (V + 1) / 2;
  extern __shared__ float2 red[];  // the ring; after it [ty][tx * V] (mean, M2), then [ty] counts
  int* rc = reinterpret_cast<int*>(red + a.ty * a.tx * V);
  const int row = threadIdx.x / a.tx, col = (threadIdx.x % a.tx) * V;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const Place p = place_of<V>(a, item);
    float2 k[P], s1[P], s2[P];
#pragma unroll
    for (int i = 0; i < P; ++i) k[i] = s1[i] = s2[i] = both(0.f);
    int cnt = 0;
    const T* x = static_cast<const T*>(a.x) + p.sample * a.x_sn + p.ch;
    each_cell<T, V, 1, MASK>(
        a, p, red, x, a.x_sl, nullptr, 0,
        [&](int, const Vec<T, V>& xv, const Vec<T, V>&) {
          float2 f[P];
          to_pairs<T, V>(xv, f);
          if (cnt == 0) {
#pragma unroll
            for (int i = 0; i < P; ++i) k[i] = f[i];
          }
          ++cnt;
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 d = fma2(k[i], both(-1.f), f[i]);
            s1[i] = add2(s1[i], d);
            s2[i] = fma2(d, d, s2[i]);
          }
        },
        [](int) {});
    __syncthreads();  // the ring has been read
    const float inv = cnt ? 1.f / (float)cnt : 0.f;
    const auto put = [&](int v, float k, float s1, float s2) {
      const float m = s1 * inv, rest = s2 - s1 * m;
      red[row * a.tx * V + col + v] = make_float2(k + m, rest < 0.f ? 0.f : rest);  // keeps NaN
    };
#pragma unroll
    for (int i = 0; i < P; ++i) {
      put(2 * i, k[i].x, s1[i].x, s2[i].x);
      if (V > 1) put(2 * i + 1, k[i].y, s1[i].y, s2[i].y);
    }
    if (col == 0) rc[row] = cnt;
    __syncthreads();
    float4* to = a.gpart + (p.sample * a.chunks + p.chunk) * (a.groups + a.ctiles) + item % a.ctiles;
    each_group<V>(a, item, [&](const Lanes& l, int g, int lo, int width) {
      float n = 0.f, mean = 0.f, m2 = 0.f;
      l.each(a.ty, width, [&](int r, int c) {
        const float f = (float)rc[r];
        n += f;
        if (f > 0.f) mean = fmaf(f, red[r * a.tx * V + lo + c].x, mean);
      });
      n = l.sum(n);
      mean = l.sum(mean);
      mean = n > 0.f ? mean / n : 0.f;
      l.each(a.ty, width, [&](int r, int c) {
        const float2 e = red[r * a.tx * V + lo + c];
        const float f = (float)rc[r], d = e.x - mean;
        if (f > 0.f) m2 += fmaf(f * d, d, e.y);
      });
      m2 = l.sum(m2);
      if (l.lane == 0 && width) to[g] = make_float4(n, mean, m2, 0.f);
    });
    __syncthreads();  // the partial results have been read
  }
}

// L lanes (a warp, or a block of kMergeThreads) per (sample, group) go through its partial results, one for
// every chunk and tile of channels that it reaches into.
constexpr int kMergeThreads = 256;
template <int L, class F>
__device__ __forceinline__ void each_partial(const NormArgs& a, long long w, int tile, F f) {
  const int g = (int)(w % a.groups), t0 = g * a.per_group / tile, t1 = ((g + 1) * a.per_group - 1) / tile;
  const long long step = a.groups + a.ctiles;
  const float4* part = a.gpart + (w / a.groups) * a.chunks * step + g;
  for (int t = t0; t <= t1; ++t)
#pragma unroll 8
    for (int k = threadIdx.x % L; k < a.chunks; k += L) f(part[k * step + t]);
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v, float* red) {  // in every lane, in a fixed order
  v = warp_sum(v);
  if constexpr (L > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < L / 32; ++i) v += red[i];
  }
  return v;
}

template <int L>
__global__ void __launch_bounds__(kMergeThreads) norm_stats_merge_kernel(NormArgs a, int tile) {
  may_start_next();
  after_previous();
  __shared__ float red[kMergeThreads / 32];
  constexpr int kGroups = kMergeThreads / L;
  for (long long w = (long long)blockIdx.x * kGroups + threadIdx.x / L; w < a.n * a.groups; w += (long long)gridDim.x * kGroups) {
    float n = 0.f, mean = 0.f, m2 = 0.f;
    each_partial<L>(a, w, tile, [&](const float4& e) {
      n += e.x;
      if (e.x > 0.f) mean = fmaf(e.x, e.y, mean);
    });
    n = lanes_sum<L>(n, red);
    mean = lanes_sum<L>(mean, red);
    mean = n > 0.f ? mean / n : 0.f;
    each_partial<L>(a, w, tile, [&](const float4& e) {
      const float d = e.y - mean;
      if (e.x > 0.f) m2 += fmaf(e.x * d, d, e.z);
    });
    m2 = lanes_sum<L>(m2, red);
    if (threadIdx.x % L == 0) {
      a.stats[2 * w] = mean;
      a.stats[2 * w + 1] = n > 0.f ? 1.f / sqrtf(m2 / n + a.eps) : 0.f;
    }
  }
}

// The per-channel values of a thread.  h uses x - mean: x a + b with b = -mean a would cancel for a
// large mean.
// ONE: the V channels lie in one group.
template <int V, bool ONE>
struct ChannelValues {
  static constexpr int P = (V + 1) / 2, Q = ONE ? 1 : P;
  float2 away[Q], rstd[Q];  // -mean, 1 / sqrt(var + eps)
  float2 w[P], b[P];        // weight, bias
  __device__ __forceinline__ void load(const NormArgs& a, const Place& p) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const int c0 = p.ch + 2 * i, c1 = ONE ? c0 : c0 + (V > 1);
      const float* s0 = a.stats + 2 * (p.sample * a.groups + c0 / a.per_group);
      const float* s1 = a.stats + 2 * (p.sample * a.groups + c1 / a.per_group);
      away[i] = make_float2(-s0[0], -s1[0]);
      rstd[i] = make_float2(s0[1], s1[1]);
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c0 = p.ch + 2 * i, c1 = c0 + (V > 1);
      w[i] = a.weight ? make_float2(load_param(a.weight, a.param_dtype, c0), load_param(a.weight, a.param_dtype, c1)) : both(1.f);
      b[i] = a.bias ? make_float2(load_param(a.bias, a.param_dtype, c0), load_param(a.bias, a.param_dtype, c1)) : both(0.f);
    }
  }
  __device__ __forceinline__ float2 away_of(int i) const { return away[ONE ? 0 : i]; }
  __device__ __forceinline__ float2 rstd_of(int i) const { return rstd[ONE ? 0 : i]; }
};

template <class T, int V>
__device__ __forceinline__ void write_zeros(T* to) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.v[i] = from_f32<T>(0.f);
  *reinterpret_cast<Vec<T, V>*>(to) = v;
}

template <class T, int V, int ACT, bool MASK, bool ONE>
__global__ void __launch_bounds__(kThreads, 4) norm_apply_kernel(NormArgs a, long long items) {
  may_start_next();
  after_previous();
  constexpr int P = (V + 1) / 2;
  extern __shared__ uint4 ring[];
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    // from the end: L2 still holds what the pass before read last
    const Place p = place_of<V>(a, items - 1 - item);
    if (!p.active) continue;
    ChannelValues<V, ONE> cv;
    cv.load(a, p);
#pragma unroll
    for (int i = 0; i < P; ++i) cv.w[i] = mul2(cv.w[i], cv.rstd_of(i));
    const T* x = static_cast<const T*>(a.x) + p.sample * a.x_sn + p.ch;
    T* y = static_cast<T*>(a.y) + (p.sample * a.cells + p.c0) * a.channels + p.ch;
    each_cell<T, V, 1, MASK>(
        a, p, ring, x, a.x_sl, nullptr, 0,
        [&](int c, const Vec<T, V>& xv, const Vec<T, V>&) {
          float2 f[P];
          to_pairs<T, V>(xv, f);
#pragma unroll
          for (int i = 0; i < P; ++i) f[i] = act2<ACT>(fma2(add2(f[i], cv.away_of(i)), cv.w[i], cv.b[i]));
          *reinterpret_cast<Vec<T, V>*>(y + (long long)c * a.channels) = from_pairs<T, V>(f);
        },
        [&](int c) { write_zeros<T, V>(y + (long long)c * a.channels); });
  }
}

// ---------------------------------------------------------------------------------- backward
template <class T, int V, int ACT, bool MASK, bool ONE>
__global__ void __launch_bounds__(kThreads, 3) norm_grad_sums_kernel(NormArgs a, long long items) {
  may_start_next();
  after_previous();
  constexpr int P = (V + 1) / 2;
  // the ring; after it [ty][tx * V] (sum dz, sum dz h), then [ty] counts and [tx * V] weights
  extern __shared__ float2 red[];
  int* rc = reinterpret_cast<int*>(red + a.ty * a.tx * V);
  float* weights = reinterpret_cast<float*>(rc + a.ty);
  const int row = threadIdx.x / a.tx, col = (threadIdx.x % a.tx) * V;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const Place p = place_of<V>(a, item);
    ChannelValues<V, ONE> cv;
    if (p.active) cv.load(a, p);
    float2 s1[P], s2[P];
#pragma unroll
    for (int i = 0; i < P; ++i) s1[i] = s2[i] = both(0.f);
    int cnt = 0;
    const T* x = static_cast<const T*>(a.x) + p.sample * a.x_sn + p.ch;
    const T* dy = static_cast<const T*>(a.dy) + p.sample * a.dy_sn + p.ch;
    each_cell<T, V, 2, MASK>(
        a, p, red, x, a.x_sl, dy, a.dy_sl,
        [&](int, const Vec<T, V>& xv, const Vec<T, V>& gv) {
          ++cnt;
          float2 f[P], g[P];
          to_pairs<T, V>(xv, f);
          to_pairs<T, V>(gv, g);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 h = mul2(add2(f[i], cv.away_of(i)), cv.rstd_of(i));
            float2 unused;
            const float2 dz = mul2(g[i], act_slope2<ACT>(fma2(h, cv.w[i], cv.b[i]), unused));
            s1[i] = add2(s1[i], dz);
            s2[i] = fma2(dz, h, s2[i]);
          }
        },
        [](int) {});
    __syncthreads();  // the ring has been read
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float2* to = red + row * a.tx * V + col + 2 * i;
      to[0] = make_float2(s1[i].x, s2[i].x);
      if (V > 1) to[1] = make_float2(s1[i].y, s2[i].y);
      if (row == 0) {
        weights[col + 2 * i] = cv.w[i].x;
        if (V > 1) weights[col + 2 * i + 1] = cv.w[i].y;
      }
    }
    if (col == 0) rc[row] = cnt;
    __syncthreads();
    float2* part = a.part + (p.sample * a.chunks + p.chunk) * a.channels + (int)(item % a.ctiles) * a.tx * V;
    const int width = min(a.tx * V, a.channels - (int)(item % a.ctiles) * a.tx * V);
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (a.ty > 16) {
      if ((int)threadIdx.x >> 5 < warps)
        for (int i = threadIdx.x >> 5; i < width; i += warps) {
          float2 s = both(0.f);
          for (int r = lane; r < a.ty; r += 32) s = add2(s, red[r * a.tx * V + i]);
          s = make_float2(warp_sum(s.x), warp_sum(s.y));
          if (lane == 0) part[i] = red[i] = s;
        }
    } else {
      for (int i = threadIdx.x; i < width; i += blockDim.x) {
        float2 s = red[i];
        for (int r = 1; r < a.ty; ++r) s = add2(s, red[r * a.tx * V + i]);
        part[i] = red[i] = s;
      }
    }
    __syncthreads();
    float4* to = a.gpart + (p.sample * a.chunks + p.chunk) * (a.groups + a.ctiles) + item % a.ctiles;
    each_group<V>(a, item, [&](const Lanes& l, int g, int lo, int width) {
      float n = 0.f, sa = 0.f, sb = 0.f;
      for (int r = l.lane; r < a.ty; r += l.count) n += (float)rc[r];
      for (int c = l.lane; c < width; c += l.count) {
        sa = fmaf(weights[lo + c], red[lo + c].x, sa);
        sb = fmaf(weights[lo + c], red[lo + c].y, sb);
      }
      n = l.sum(n) * (float)width;
      sa = l.sum(sa);
      sb = l.sum(sb);
      if (l.lane == 0 && width) to[g] = make_float4(n, sa, sb, 0.f);
    });
    __syncthreads();  // the partial results have been read
  }
}

// A / n and B / n of every (sample, group).
template <int L>
__global__ void __launch_bounds__(kMergeThreads) norm_grad_merge_kernel(NormArgs a, int tile) {
  may_start_next();
  after_previous();
  __shared__ float red[kMergeThreads / 32];
  constexpr int kGroups = kMergeThreads / L;
  for (long long w = (long long)blockIdx.x * kGroups + threadIdx.x / L; w < a.n * a.groups; w += (long long)gridDim.x * kGroups) {
    float n = 0.f, sa = 0.f, sb = 0.f;
    each_partial<L>(a, w, tile, [&](const float4& e) {
      n += e.x;
      sa += e.y;
      sb += e.z;
    });
    n = lanes_sum<L>(n, red);
    sa = lanes_sum<L>(sa, red);
    sb = lanes_sum<L>(sb, red);
    if (threadIdx.x % L == 0) a.ab[w] = n > 0.f ? make_float2(sa / n, sb / n) : make_float2(0.f, 0.f);
  }
}

template <class T, int V, int ACT, bool MASK, bool ONE>
__global__ void __launch_bounds__(kThreads, 3) norm_grad_apply_kernel(NormArgs a, long long items) {
  may_start_next();
  after_previous();
  constexpr int P = (V + 1) / 2;
  extern __shared__ uint4 ring[];
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    // from the end: L2 still holds what the pass before read last
    const Place p = place_of<V>(a, items - 1 - item);
    if (!p.active) continue;
    ChannelValues<V, ONE> cv;
    cv.load(a, p);
    constexpr int Q = ONE ? 1 : P;
    float2 ga[Q], gb[Q];  // -A / n, -B / n
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const float2 e0 = a.ab[p.sample * a.groups + (p.ch + 2 * i) / a.per_group];
      const float2 e1 = a.ab[p.sample * a.groups + (p.ch + (ONE ? 0 : 2 * i + (V > 1))) / a.per_group];
      ga[i] = make_float2(-e0.x, -e1.x);
      gb[i] = make_float2(-e0.y, -e1.y);
    }
    const T* x = static_cast<const T*>(a.x) + p.sample * a.x_sn + p.ch;
    const T* dy = static_cast<const T*>(a.dy) + p.sample * a.dy_sn + p.ch;
    T* dx = static_cast<T*>(a.y) + (p.sample * a.cells + p.c0) * a.channels + p.ch;
    each_cell<T, V, 2, MASK>(
        a, p, ring, x, a.x_sl, dy, a.dy_sl,
        [&](int c, const Vec<T, V>& xv, const Vec<T, V>& gv) {
          float2 f[P], g[P];
          to_pairs<T, V>(xv, f);
          to_pairs<T, V>(gv, g);
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float2 h = mul2(add2(f[i], cv.away_of(i)), cv.rstd_of(i));
            float2 unused;
            const float2 dz = mul2(g[i], act_slope2<ACT>(fma2(h, cv.w[i], cv.b[i]), unused));
            // rstd (w dz - (A + h B) / n), each product rounded: one value a group gives exactly 0
            f[i] = mul2(add2(mul2(cv.w[i], dz), fma2(h, gb[ONE ? 0 : i], ga[ONE ? 0 : i])), cv.rstd_of(i));
          }
          *reinterpret_cast<Vec<T, V>*>(dx + (long long)c * a.channels) = from_pairs<T, V>(f);
        },
        [&](int c) { write_zeros<T, V>(dx + (long long)c * a.channels); });
  }
}

// Column sums of `rows` x channels float2 entries in two steps of a fixed order: block (32 channels
// x 8 rows) s sums the rows of its split, then one block a channel tile sums the splits.
__global__ void norm_param_sums_kernel(const float2* part, long long rows, int channels, int splits,
                                       float2* out) {
  may_start_next();
  after_previous();
  __shared__ float2 red[8][32];
  const int ch = blockIdx.x * 32 + threadIdx.x;
  const int split = blockIdx.y;
  const long long per = (rows + splits - 1) / splits;
  const long long r0 = split * per, r1 = min(rows, r0 + per);
  float2 s = make_float2(0.f, 0.f);
  if (ch < channels)
#pragma unroll 4
    for (long long r = r0 + threadIdx.y; r < r1; r += 8) s = add2(s, part[r * channels + ch]);
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && ch < channels) {
    for (int r = 1; r < 8; ++r) {
      s.x += red[r][threadIdx.x].x;
      s.y += red[r][threadIdx.x].y;
    }
    out[(long long)split * channels + ch] = s;
  }
}
__global__ void norm_param_store_kernel(const float2* part, int splits, int channels, void* dweight,
                                        void* dbias, int param_dtype) {
  may_start_next();
  after_previous();
  __shared__ float2 red[16][32];
  const int ch = blockIdx.x * 32 + threadIdx.x;
  float2 s = make_float2(0.f, 0.f);
  if (ch < channels)
    for (int k = threadIdx.y; k < splits; k += 16) s = add2(s, part[(long long)k * channels + ch]);
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y || ch >= channels) return;
  for (int k = 1; k < 16; ++k) s = add2(s, red[k][threadIdx.x]);
  if (dweight) store_param(dweight, param_dtype, ch, s.y);
  if (dbias) store_param(dbias, param_dtype, ch, s.x);
}

// ------------------------------------------------------------------------------------ host side
inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

constexpr int kParamSplits = 64;

int32_t check_desc(const NcaNormDesc* d) {
  if (!d || d->n < 0 || d->cells < 0 || d->channels <= 0 || d->groups <= 0) return NCA_ERR_INVALID;
  if (d->channels % d->groups) return NCA_ERR_INVALID;
  if (!dtype_ok(d->dtype) || (d->param_dtype != NCA_F32 && d->param_dtype != d->dtype)) return NCA_ERR_INVALID;
  if (d->act < NCA_ACT_NONE || d->act > NCA_ACT_SIGMOID || !(d->eps >= 0.f)) return NCA_ERR_INVALID;
  if (d->channels > (1 << 30) || d->cells > (1ll << 30) || d->n > (1ll << 40)) return NCA_ERR_UNSUPPORTED;
  return NCA_OK;
}

// Pieces of a sample: about 32 cells a thread when there are enough samples, fewer cells (8 at
// least) when the pieces would not fill the GPU.
void split_cells(const NcaNormDesc& d, int ty, int ctiles, int* chunks, long long* chunk_cells) {
  long long per = 32ll * ty;
  while (per > 8ll * ty && ((d.cells + per - 1) / per) * d.n * ctiles < 1184) per /= 2;
  *chunk_cells = per;
  *chunks = (int)((d.cells + per - 1) / per);
  if (*chunks < 1) *chunks = 1;
}

// The most chunks, and partial results of a sample's groups, over the vector widths.
void worst_chunks(const NcaNormDesc& d, size_t* chunks, size_t* partials) {
  *chunks = *partials = 1;
  for (int v = 1; v <= 8; v *= 2) {
    const int nv = (d.channels + v - 1) / v;
    const int tx = nv < kThreads ? nv : kThreads, ty = kThreads / tx, ct = (nv + tx - 1) / tx;
    int n;
    long long cc;
    split_cells(d, ty, ct, &n, &cc);
    *chunks = std::max(*chunks, (size_t)n);
    *partials = std::max(*partials, (size_t)n * (d.groups + ct));
  }
}

struct Layout {
  size_t stats, part, gpart, ab, params, total;
};
// held: the slices of the kernel that holds samples, 0 when the streaming kernels run.
Layout layout_of(const NcaNormDesc& d, bool backward, int held) {
  size_t chunks, partials;
  worst_chunks(d, &chunks, &partials);
  if (held) chunks = held;
  Layout l{};
  size_t at = 0;
  const auto take = [&](bool needed, size_t bytes) {
    const size_t here = at;
    if (needed) at += align256(bytes);
    return here;
  };
  l.stats = take(!backward && !held, (size_t)d.n * d.groups * sizeof(float2));
  l.part = take(backward, (size_t)d.n * chunks * d.channels * sizeof(float2));
  l.gpart = take(!held, (size_t)d.n * partials * sizeof(float4));
  l.ab = take(backward && !held, (size_t)d.n * d.groups * sizeof(float2));
  l.params = take(backward, (size_t)kParamSplits * d.channels * sizeof(float2));
  l.total = at;
  return l;
}

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

NormArgs args_of(const NcaNormDesc& d, const void* x, const void* weight, const void* bias,
                 const uint8_t* mask, const void* dy, void* y, float* stats) {
  NormArgs a{};
  a.n = d.n;
  a.cells = d.cells;
  a.channels = d.channels;
  a.groups = d.groups;
  a.per_group = d.channels / d.groups;
  a.eps = d.eps;
  a.x_sn = d.x_stride_n;
  a.x_sl = d.x_stride_cell;
  a.dy_sn = d.dy_stride_n;
  a.dy_sl = d.dy_stride_cell;
  a.m_sn = d.mask_stride_n;
  a.m_sl = d.mask_stride_cell;
  a.param_dtype = d.param_dtype;
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.mask = mask;
  a.dy = dy;
  a.y = y;
  a.stats = stats;
  return a;
}
void place(NormArgs& a, const Layout& l, void* ws) {
  uint8_t* w = static_cast<uint8_t*>(ws);
  if (!a.stats) a.stats = reinterpret_cast<float*>(w + l.stats);
  a.part = reinterpret_cast<float2*>(w + l.part);
  a.gpart = reinterpret_cast<float4*>(w + l.gpart);
  a.ab = reinterpret_cast<float2*>(w + l.ab);
}

// Widest vector (16 bytes at most) that the channel count, the strides and the addresses allow; single
// values where an address is on no 16-byte boundary.
int vector_width(const NcaNormDesc& d, bool backward) {
  if (d.unaligned) return 1;
  const size_t size = dtype_size(d.dtype);
  for (int v = (int)(16 / size); v > 1; v /= 2) {
    bool ok = d.channels % v == 0 && d.x_stride_n % v == 0 && d.x_stride_cell % v == 0;
    if (backward) ok = ok && d.dy_stride_n % v == 0 && d.dy_stride_cell % v == 0;
    if (ok) return v;
  }
  return 1;
}

// The streaming kernels exist for 16-byte vectors, pairs of 16-bit values and single values.
int streaming_width(int dtype, int v) {
  const int w = (int)(16 / dtype_size(dtype));
  return v == w ? v : (dtype != NCA_F32 && v >= 2 ? 2 : 1);
}

long long plan(const NcaNormDesc& d, NormArgs& a, int v) {
  const int nv = d.channels / v;
  a.tx = nv < kThreads ? nv : kThreads;
  a.ty = kThreads / a.tx;
  a.ctiles = (nv + a.tx - 1) / a.tx;
  split_cells(d, a.ty, a.ctiles, &a.chunks, &a.chunk_cells);
  return a.n * a.chunks * a.ctiles;
}

inline unsigned grid_of(long long items) { return (unsigned)(items < (1 << 20) ? items : (1 << 20)); }

int32_t param_grads(const float2* part, long long rows, int channels, void* dweight, void* dbias, int param_dtype,
                    float2* params, cudaStream_t s) {
  if (rows <= 256)  // few: the second step alone
    return launch_after(norm_param_store_kernel, dim3((channels + 31) / 32), dim3(32, 16), 0, s, 1, part, (int)rows, channels,
                        dweight, dbias, param_dtype);
  const int splits = (int)(rows < 8 * kParamSplits ? (rows + 7) / 8 : kParamSplits);
  const int32_t st = launch_after(norm_param_sums_kernel, dim3((channels + 31) / 32, splits), dim3(32, 8), 0, s, 1, part,
                                  rows, channels, splits, params);
  if (st != NCA_OK) return st;
  return launch_after(norm_param_store_kernel, dim3((channels + 31) / 32), dim3(32, 16), 0, s, 1, params, splits, channels,
                      dweight, dbias, param_dtype);
}

// Raises a kernel's shared-memory limit once a device, and launches it.
constexpr int kMaxDevices = 64;
int32_t launch(void (*kernel)(NormArgs, long long), std::atomic<uint64_t>& ready, const NormArgs& a, long long items,
               size_t smem, cudaStream_t s) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return NCA_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024) != cudaSuccess) {
      const int32_t st = launch_status();
      return st == NCA_OK ? NCA_ERR_CUDA : st;
    }
    ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  return launch_after(kernel, dim3(grid_of(items)), dim3(a.tx * a.ty), smem, s, 1, a, items);
}
// Shared memory of a kernel that leaves partial results: the ring, or those where they are more.
template <class T, int V>
size_t sums_smem(const NormArgs& a, int tensors) {
  return std::max(ring_bytes<T, V>(tensors), (size_t)a.ty * a.tx * V * sizeof(float2) + a.ty * sizeof(int) + a.tx * V * sizeof(float));
}
#define NCA_TRY(call)              \
  do {                             \
    const int32_t st_ = (call);    \
    if (st_ != NCA_OK) return st_; \
  } while (0)

// A warp a group for few partial results, a block for many.  tile: channels of a block.
int32_t merge(void (*warp)(NormArgs, int), void (*block)(NormArgs, int), const NormArgs& a, int tile, cudaStream_t s) {
  const long long groups = a.n * a.groups;
  if ((long long)a.chunks * (a.ctiles / a.groups + 1) <= 64 || groups >= 8192)
    return launch_after(warp, dim3(grid_of((groups + kMergeThreads / 32 - 1) / (kMergeThreads / 32))), dim3(kMergeThreads), 0,
                        s, 1, a, tile);
  return launch_after(block, dim3(grid_of(groups)), dim3(kMergeThreads), 0, s, 1, a, tile);
}

template <class T, int V, int ACT, bool MASK, bool ONE>
int32_t forward(const NcaNormDesc& d, NormArgs a, cudaStream_t s) {
  static std::atomic<uint64_t> ready[2];
  const long long items = plan(d, a, V);
  NCA_TRY(launch(norm_stats_kernel<T, V, MASK>, ready[0], a, items, sums_smem<T, V>(a, 1), s));
  NCA_TRY(merge(norm_stats_merge_kernel<32>, norm_stats_merge_kernel<kMergeThreads>, a, a.tx * V, s));
  return launch(norm_apply_kernel<T, V, ACT, MASK, ONE>, ready[1], a, items, ring_bytes<T, V>(1), s);
}

template <class T, int V, int ACT, bool MASK, bool ONE>
int32_t backward(const NcaNormDesc& d, NormArgs a, void* dweight, void* dbias, float2* params,
                 cudaStream_t s) {
  static std::atomic<uint64_t> ready[2];
  const long long items = plan(d, a, V);
  NCA_TRY(launch(norm_grad_sums_kernel<T, V, ACT, MASK, ONE>, ready[0], a, items, sums_smem<T, V>(a, 2), s));
  if (a.y) {
    NCA_TRY(merge(norm_grad_merge_kernel<32>, norm_grad_merge_kernel<kMergeThreads>, a, a.tx * V, s));
    NCA_TRY(launch(norm_grad_apply_kernel<T, V, ACT, MASK, ONE>, ready[1], a, items, ring_bytes<T, V>(2), s));
  }
  if (!dweight && !dbias) return NCA_OK;
  return param_grads(a.part, a.n * a.chunks, a.channels, dweight, dbias, a.param_dtype, params, s);
}

// Instantiates fn(T, V, ACT) for the run-time choice.
template <class F>
int32_t dispatch(const NcaNormDesc& d, int v, F fn) {
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    return with_act(d.act, [&](auto act) {
      constexpr int A = decltype(act)::value;
      constexpr int W = 16 / sizeof(T);
      if (v == W) return fn.template operator()<T, W, A>();
      if constexpr (sizeof(T) == 2)
        if (v == 2) return fn.template operator()<T, 2, A>();
      return fn.template operator()<T, 1, A>();
    });
  });
}

struct ForwardCall {
  const NcaNormDesc& d;
  const NormArgs& a;
  cudaStream_t s;
  template <class T, int V, int A>
  int32_t operator()() const { 
    if constexpr (V * sizeof(T) == 16) {
      if (a.per_group % V == 0)
        return a.mask ? forward<T, V, A, true, true>(d, a, s) : forward<T, V, A, false, true>(d, a, s);
    }
    return a.mask ? forward<T, V, A, true, V == 1>(d, a, s) : forward<T, V, A, false, V == 1>(d, a, s);
   }
};
struct BackwardCall {
  const NcaNormDesc& d;
  const NormArgs& a;
  void *dweight, *dbias;
  float2* params;
  cudaStream_t s;
  template <class T, int V, int A>
  int32_t operator()() const { 
    if constexpr (V * sizeof(T) == 16) {
      if (a.per_group % V == 0)
        return a.mask ? backward<T, V, A, true, true>(d, a, dweight, dbias, params, s)
                      : backward<T, V, A, false, true>(d, a, dweight, dbias, params, s);
    }
    return a.mask ? backward<T, V, A, true, V == 1>(d, a, dweight, dbias, params, s)
                  : backward<T, V, A, false, V == 1>(d, a, dweight, dbias, params, s);
   }
};

}  // namespace

// What a call does and needs, from its descriptor alone.
struct Choice {
  int v, held;
  Layout l;
};
Choice choose(const NcaNormDesc& d, bool backward) {
  static const uint8_t some = 1;
  Choice c;
  c.v = vector_width(d, backward);
  const NormArgs a = args_of(d, nullptr, nullptr, nullptr, d.masked ? &some : nullptr, nullptr, nullptr, nullptr);
  c.held = norm_held_slices(a, d.dtype, c.v, backward);
  c.l = layout_of(d, backward, c.held);
  return c;
}
bool addresses_ok(const NcaNormDesc& d, const uint8_t* mask, std::initializer_list<const void*> ps) {
  if ((mask != nullptr) != (d.masked != 0)) return false;
  if (!d.unaligned)
    for (const void* p : ps)
      if (!aligned(p, 16)) return false;
  return true;
}

extern "C" {

int32_t nca_b200_group_norm_workspace(const NcaNormDesc* d, int32_t backward, size_t* bytes) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK || !bytes) return st != NCA_OK ? st : NCA_ERR_INVALID;
  *bytes = d->n == 0 || d->cells == 0 ? 0 : choose(*d, backward != 0).l.total;
  return NCA_OK;
}

int32_t nca_b200_group_norm(const NcaNormDesc* d, const void* x, const void* weight, const void* bias,
                            const uint8_t* mask, void* y, float* stats, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK) return st;
  if (d->n == 0 || d->cells == 0) return NCA_OK;
  const Choice c = choose(*d, false);
  if (!x || !y || workspace_bytes < c.l.total || (c.l.total && !workspace) || !addresses_ok(*d, mask, {x, y}))
    return NCA_ERR_INVALID;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  NormArgs a = args_of(*d, x, weight, bias, mask, nullptr, y, stats);
  if (c.held) return norm_held_forward(a, d->dtype, d->act, c.v, s);
  place(a, c.l, workspace);
  return dispatch(*d, streaming_width(d->dtype, c.v), ForwardCall{*d, a, s});
}

int32_t nca_b200_group_norm_backward(const NcaNormDesc* d, const void* x, const void* weight,
                                     const void* bias, const uint8_t* mask, const float* stats,
                                     const void* dy, void* dx, void* dweight, void* dbias,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->n == 0 || d->cells == 0) {
    const size_t bytes = d->channels * dtype_size(d->param_dtype);
    if (dweight && cudaMemsetAsync(dweight, 0, bytes, s) != cudaSuccess) return NCA_ERR_CUDA;
    if (dbias && cudaMemsetAsync(dbias, 0, bytes, s) != cudaSuccess) return NCA_ERR_CUDA;
    return NCA_OK;
  }
  const Choice c = choose(*d, true);
  if (!x || !dy || !stats || !workspace || workspace_bytes < c.l.total || !addresses_ok(*d, mask, {x, dy, dx}))
    return NCA_ERR_INVALID;
  NormArgs a = args_of(*d, x, weight, bias, mask, dy, dx, const_cast<float*>(stats));
  place(a, c.l, workspace);
  float2* params = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + c.l.params);
  if (c.held) {
    if (!dweight && !dbias) a.part = nullptr;
    const int32_t r = norm_held_backward(a, d->dtype, d->act, c.v, s);
    if (r != NCA_OK || !a.part) return r;
    return param_grads(a.part, a.n * c.held, a.channels, dweight, dbias, a.param_dtype, params, s);
  }
  return dispatch(*d, streaming_width(d->dtype, c.v), BackwardCall{*d, a, dweight, dbias, params, s});
}

}  // extern "C"
