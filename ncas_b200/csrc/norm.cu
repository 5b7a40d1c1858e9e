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
#include <algorithm>

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

__device__ __forceinline__ bool kept(const NormArgs& a, const Place& p, long long cell) {
  return !a.mask || a.mask[p.sample * a.m_sn + cell * a.m_sl] != 0;
}

// ------------------------------------------------------------------------- forward: statistics
template <class T, int V>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(NormArgs a, long long items) {
  extern __shared__ float2 red[];  // [ty][tx * V] (mean, M2), then [ty] counts
  int* rc = reinterpret_cast<int*>(red + a.ty * a.tx * V);
  const int row = threadIdx.x / a.tx, col = (threadIdx.x % a.tx) * V;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const Place p = place_of<V>(a, item);
    float k[V], s1[V], s2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) k[v] = s1[v] = s2[v] = 0.f;
    int cnt = 0;
    const T* x = static_cast<const T*>(a.x) + p.sample * a.x_sn + p.ch;
    for (long long c = p.c0 + row; c < p.c1; c += a.ty) {
      if (!kept(a, p, c)) continue;
      if (p.active) {
        const Vec<T, V> xv = *reinterpret_cast<const Vec<T, V>*>(x + c * a.x_sl);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float f = to_f32(xv.v[v]);
          if (cnt == 0) k[v] = f;
          const float d = f - k[v];
          s1[v] += d;
          s2[v] = fmaf(d, d, s2[v]);
        }
      }
      ++cnt;
    }
    __syncthreads();  // the previous item's partials have been read
    const float inv = cnt ? 1.f / (float)cnt : 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float m = s1[v] * inv;
      red[row * a.tx * V + col + v] = make_float2(k[v] + m, fmaxf(s2[v] - s1[v] * m, 0.f));
    }
    if (col == 0) rc[row] = cnt;
    __syncthreads();
    int total = 0;
    for (int r = 0; r < a.ty; ++r) total += rc[r];
    for (int i = threadIdx.x; i < a.tx * V; i += blockDim.x) {
      const int ch = (int)(item % a.ctiles) * a.tx * V + i;
      if (ch >= a.channels) break;
      float mean = 0.f, m2 = 0.f;
      for (int r = 0; r < a.ty; ++r) mean += (float)rc[r] * red[r * a.tx * V + i].x;
      mean = total ? mean / (float)total : 0.f;
      for (int r = 0; r < a.ty; ++r) {
        const float2 e = red[r * a.tx * V + i];
        const float d = e.x - mean;
        m2 += rc[r] ? fmaf((float)rc[r] * d, d, e.y) : 0.f;
      }
      a.part[(p.sample * a.chunks + p.chunk) * a.channels + ch] = make_float2(mean, m2);
    }
    if (threadIdx.x == 0 && item % a.ctiles == 0) a.counts[p.sample * a.chunks + p.chunk] = total;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp per (sample, group): merges its chunks x per_group partials.
__global__ void norm_stats_merge_kernel(NormArgs a) {
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= a.n * a.groups) return;
  const long long sample = w / a.groups;
  const int g = (int)(w % a.groups);
  const int* cnt = a.counts + sample * a.chunks;
  const float2* part = a.part + sample * a.chunks * a.channels + g * a.per_group;
  const long long entries = (long long)a.chunks * a.per_group;
  float n = 0.f, mean = 0.f, m2 = 0.f;
  for (long long i = lane; i < entries; i += 32) {
    const int k = (int)(i / a.per_group), c = (int)(i % a.per_group);
    const float f = (float)cnt[k];
    n += f;
    mean = fmaf(f, part[(long long)k * a.channels + c].x, mean);
  }
  n = warp_sum(n);
  mean = warp_sum(mean);
  mean = n > 0.f ? mean / n : 0.f;
  for (long long i = lane; i < entries; i += 32) {
    const int k = (int)(i / a.per_group), c = (int)(i % a.per_group);
    const float f = (float)cnt[k];
    const float2 e = part[(long long)k * a.channels + c];
    const float d = e.x - mean;
    if (f > 0.f) m2 += fmaf(f * d, d, e.y);
  }
  m2 = warp_sum(m2);
  if (lane == 0) {
    a.stats[2 * w] = mean;
    a.stats[2 * w + 1] = n > 0.f ? 1.f / sqrtf(m2 / n + a.eps) : 0.f;
  }
}

// The per-channel values of a thread: mean, rstd * weight and bias (rstd and weight apart in the
// backward).  h uses x - mean: x a + b with b = -mean a would cancel for a large mean.
template <int V>
struct ChannelValues {
  float mean[V], rstd[V], w[V], b[V];
  __device__ __forceinline__ void load(const NormArgs& a, const Place& p) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const long long sg = p.sample * a.groups + (p.ch + v) / a.per_group;
      mean[v] = a.stats[2 * sg];
      rstd[v] = a.stats[2 * sg + 1];
      w[v] = a.weight ? load_param(a.weight, a.param_dtype, p.ch + v) : 1.f;
      b[v] = a.bias ? load_param(a.bias, a.param_dtype, p.ch + v) : 0.f;
    }
  }
};

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) norm_apply_kernel(NormArgs a, long long items) {
  const int row = threadIdx.x / a.tx;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const Place p = place_of<V>(a, item);
    if (!p.active) continue;
    ChannelValues<V> cv;
    cv.load(a, p);
    const T* x = static_cast<const T*>(a.x) + p.sample * a.x_sn + p.ch;
    T* y = static_cast<T*>(a.y) + p.sample * a.cells * a.channels + p.ch;
    for (long long c = p.c0 + row; c < p.c1; c += a.ty) {
      Vec<T, V> yv;
      if (kept(a, p, c)) {
        const Vec<T, V> xv = *reinterpret_cast<const Vec<T, V>*>(x + c * a.x_sl);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float h = (to_f32(xv.v[v]) - cv.mean[v]) * cv.rstd[v];
          yv.v[v] = from_f32<T>(act_f<ACT>(fmaf(h, cv.w[v], cv.b[v])));
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) yv.v[v] = from_f32<T>(0.f);
      }
      *reinterpret_cast<Vec<T, V>*>(y + c * a.channels) = yv;
    }
  }
}

// ---------------------------------------------------------------------------------- backward
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) norm_grad_sums_kernel(NormArgs a, long long items) {
  extern __shared__ float2 red[];  // [ty][tx * V] (sum dz, sum dz h), then [ty] counts
  int* rc = reinterpret_cast<int*>(red + a.ty * a.tx * V);
  const int row = threadIdx.x / a.tx, col = (threadIdx.x % a.tx) * V;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const Place p = place_of<V>(a, item);
    ChannelValues<V> cv;
    if (p.active) cv.load(a, p);
    float s1[V], s2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) s1[v] = s2[v] = 0.f;
    int cnt = 0;
    const T* x = static_cast<const T*>(a.x) + p.sample * a.x_sn + p.ch;
    const T* dy = static_cast<const T*>(a.dy) + p.sample * a.dy_sn + p.ch;
    for (long long c = p.c0 + row; c < p.c1; c += a.ty) {
      if (!kept(a, p, c)) continue;
      ++cnt;
      if (!p.active) continue;
      const Vec<T, V> xv = *reinterpret_cast<const Vec<T, V>*>(x + c * a.x_sl);
      const Vec<T, V> gv = *reinterpret_cast<const Vec<T, V>*>(dy + c * a.dy_sl);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float h = (to_f32(xv.v[v]) - cv.mean[v]) * cv.rstd[v];
        float unused;
        const float dz = to_f32(gv.v[v]) * act_slope_f<ACT>(fmaf(h, cv.w[v], cv.b[v]), unused);
        s1[v] += dz;
        s2[v] = fmaf(dz, h, s2[v]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) red[row * a.tx * V + col + v] = make_float2(s1[v], s2[v]);
    if (col == 0) rc[row] = cnt;
    __syncthreads();
    for (int i = threadIdx.x; i < a.tx * V; i += blockDim.x) {
      const int ch = (int)(item % a.ctiles) * a.tx * V + i;
      if (ch >= a.channels) break;
      float2 s = make_float2(0.f, 0.f);
      for (int r = 0; r < a.ty; ++r) {
        s.x += red[r * a.tx * V + i].x;
        s.y += red[r * a.tx * V + i].y;
      }
      a.part[(p.sample * a.chunks + p.chunk) * a.channels + ch] = s;
    }
    if (threadIdx.x == 0 && item % a.ctiles == 0) {
      int total = 0;
      for (int r = 0; r < a.ty; ++r) total += rc[r];
      a.counts[p.sample * a.chunks + p.chunk] = total;
    }
  }
}

// One warp per (sample, group): A / n and B / n.
__global__ void norm_grad_merge_kernel(NormArgs a) {
  const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= a.n * a.groups) return;
  const long long sample = w / a.groups;
  const int g = (int)(w % a.groups);
  const float2* part = a.part + sample * a.chunks * a.channels + g * a.per_group;
  const long long entries = (long long)a.chunks * a.per_group;
  float n = 0.f, sa = 0.f, sb = 0.f;
  for (long long i = lane; i < entries; i += 32) {
    const int k = (int)(i / a.per_group), c = (int)(i % a.per_group);
    const float wt = a.weight ? load_param(a.weight, a.param_dtype, g * a.per_group + c) : 1.f;
    const float2 e = part[(long long)k * a.channels + c];
    n += (float)a.counts[sample * a.chunks + k];
    sa = fmaf(wt, e.x, sa);
    sb = fmaf(wt, e.y, sb);
  }
  n = warp_sum(n);
  sa = warp_sum(sa);
  sb = warp_sum(sb);
  if (lane == 0) a.ab[w] = n > 0.f ? make_float2(sa / n, sb / n) : make_float2(0.f, 0.f);
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kThreads) norm_grad_apply_kernel(NormArgs a, long long items) {
  const int row = threadIdx.x / a.tx;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const Place p = place_of<V>(a, item);
    if (!p.active) continue;
    ChannelValues<V> cv;
    cv.load(a, p);
    float ga[V], gb[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 e = a.ab[p.sample * a.groups + (p.ch + v) / a.per_group];
      ga[v] = e.x;
      gb[v] = e.y;
    }
    const T* x = static_cast<const T*>(a.x) + p.sample * a.x_sn + p.ch;
    const T* dy = static_cast<const T*>(a.dy) + p.sample * a.dy_sn + p.ch;
    T* dx = static_cast<T*>(a.y) + p.sample * a.cells * a.channels + p.ch;
    for (long long c = p.c0 + row; c < p.c1; c += a.ty) {
      Vec<T, V> out;
      if (kept(a, p, c)) {
        const Vec<T, V> xv = *reinterpret_cast<const Vec<T, V>*>(x + c * a.x_sl);
        const Vec<T, V> gv = *reinterpret_cast<const Vec<T, V>*>(dy + c * a.dy_sl);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float h = (to_f32(xv.v[v]) - cv.mean[v]) * cv.rstd[v];
          float unused;
          const float dz = to_f32(gv.v[v]) * act_slope_f<ACT>(fmaf(h, cv.w[v], cv.b[v]), unused);
          out.v[v] = from_f32<T>(cv.rstd[v] * (__fmul_rn(cv.w[v], dz) - fmaf(h, gb[v], ga[v])));
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) out.v[v] = from_f32<T>(0.f);
      }
      *reinterpret_cast<Vec<T, V>*>(dx + c * a.channels) = out;
    }
  }
}

// Column sums of `rows` x channels float2 entries in two steps of a fixed order: block (32 channels
// x 8 rows) s sums the rows of its split, then one block a channel tile sums the splits.
__global__ void norm_param_sums_kernel(const float2* part, long long rows, int channels, int splits,
                                       float2* out) {
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
  if (d->cells > (1ll << 30) || d->n > (1ll << 40)) return NCA_ERR_UNSUPPORTED;
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

int worst_chunks(const NcaNormDesc& d) {  // over every vector width: one vector a thread, 8 cells
  int worst = 1;
  for (int v = 1; v <= 8; v *= 2) {
    const int nv = (d.channels + v - 1) / v;
    const int tx = nv < kThreads ? nv : kThreads, ty = kThreads / tx;
    int chunks;
    long long cc;
    split_cells(d, ty, (nv + tx - 1) / tx, &chunks, &cc);
    if (chunks > worst) worst = chunks;
  }
  return worst;
}

struct Layout {
  size_t part, counts, ab, params, total;
};
Layout layout_of(const NcaNormDesc& d) {
  const size_t chunks = std::max(worst_chunks(d), 16);  // the held backward has up to 16 slices
  Layout l;
  l.part = 0;
  l.counts = l.part + align256((size_t)d.n * chunks * d.channels * sizeof(float2));
  l.ab = l.counts + align256((size_t)d.n * chunks * sizeof(int));
  l.params = l.ab + align256((size_t)d.n * d.groups * sizeof(float2));
  l.total = l.params + align256((size_t)kParamSplits * d.channels * sizeof(float2));
  return l;
}

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

NormArgs args_of(const NcaNormDesc& d, const void* x, const void* weight, const void* bias,
                 const uint8_t* mask, const void* dy, void* y, float* stats, void* ws) {
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
  const Layout l = layout_of(d);
  uint8_t* w = static_cast<uint8_t*>(ws);
  a.part = reinterpret_cast<float2*>(w + l.part);
  a.counts = reinterpret_cast<int*>(w + l.counts);
  a.ab = reinterpret_cast<float2*>(w + l.ab);
  return a;
}

// Widest vector (16 bytes at most) that the channel count, the strides and the addresses allow.
int vector_width(const NcaNormDesc& d, const NormArgs& a, bool backward) {
  const size_t size = dtype_size(d.dtype);
  for (int v = (int)(16 / size); v > 1; v /= 2) {
    bool ok = d.channels % v == 0 && d.x_stride_n % v == 0 && d.x_stride_cell % v == 0 &&
              aligned(a.x, v * size) && aligned(a.y, v * size);
    if (backward) ok = ok && d.dy_stride_n % v == 0 && d.dy_stride_cell % v == 0 && aligned(a.dy, v * size);
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

void param_grads(const float2* part, long long rows, int channels, void* dweight, void* dbias, int param_dtype,
                 float2* params, cudaStream_t s) {
  const int splits = (int)(rows < 8 * kParamSplits ? (rows + 7) / 8 : kParamSplits);
  norm_param_sums_kernel<<<dim3((channels + 31) / 32, splits), dim3(32, 8), 0, s>>>(part, rows, channels, splits,
                                                                                 params);
  norm_param_store_kernel<<<(channels + 31) / 32, dim3(32, 16), 0, s>>>(params, splits, channels, dweight, dbias, param_dtype);
}

template <class T, int V, int ACT>
int32_t forward(const NcaNormDesc& d, NormArgs a, cudaStream_t s) {
  const long long items = plan(d, a, V);
  const int threads = a.tx * a.ty;
  const size_t smem = (size_t)a.ty * a.tx * V * sizeof(float2) + a.ty * sizeof(int);
  norm_stats_kernel<T, V><<<grid_of(items), threads, smem, s>>>(a, items);
  norm_stats_merge_kernel<<<(unsigned)((a.n * a.groups + 7) / 8), 256, 0, s>>>(a);
  norm_apply_kernel<T, V, ACT><<<grid_of(items), threads, 0, s>>>(a, items);
  return launch_status();
}

template <class T, int V, int ACT>
int32_t backward(const NcaNormDesc& d, NormArgs a, void* dweight, void* dbias, float2* params,
                 cudaStream_t s) {
  const long long items = plan(d, a, V);
  const int threads = a.tx * a.ty;
  const size_t smem = (size_t)a.ty * a.tx * V * sizeof(float2) + a.ty * sizeof(int);
  norm_grad_sums_kernel<T, V, ACT><<<grid_of(items), threads, smem, s>>>(a, items);
  if (a.y) {
    norm_grad_merge_kernel<<<(unsigned)((a.n * a.groups + 7) / 8), 256, 0, s>>>(a);
    norm_grad_apply_kernel<T, V, ACT><<<grid_of(items), threads, 0, s>>>(a, items);
  }
  if (dweight || dbias) param_grads(a.part, a.n * a.chunks, a.channels, dweight, dbias, a.param_dtype, params, s);
  return launch_status();
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
  int32_t operator()() const { return forward<T, V, A>(d, a, s); }
};
struct BackwardCall {
  const NcaNormDesc& d;
  const NormArgs& a;
  void *dweight, *dbias;
  float2* params;
  cudaStream_t s;
  template <class T, int V, int A>
  int32_t operator()() const { return backward<T, V, A>(d, a, dweight, dbias, params, s); }
};

}  // namespace

extern "C" {

int32_t nca_b200_group_norm_workspace(const NcaNormDesc* d, int32_t, size_t* bytes) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK || !bytes) return st != NCA_OK ? st : NCA_ERR_INVALID;
  *bytes = layout_of(*d).total;
  return NCA_OK;
}

int32_t nca_b200_group_norm(const NcaNormDesc* d, const void* x, const void* weight, const void* bias,
                            const uint8_t* mask, void* y, float* stats, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK) return st;
  if (d->n == 0 || d->cells == 0) return NCA_OK;
  if (!x || !y || !stats || !workspace || workspace_bytes < layout_of(*d).total) return NCA_ERR_INVALID;
  const NormArgs a = args_of(*d, x, weight, bias, mask, nullptr, y, stats, workspace);
  const int v = vector_width(*d, a, false);
  if (norm_held_applies(a, d->dtype, v, false))
    return norm_held_forward(a, d->dtype, d->act, v, static_cast<cudaStream_t>(stream));
  return dispatch(*d, streaming_width(d->dtype, v), ForwardCall{*d, a, static_cast<cudaStream_t>(stream)});
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
  if (!x || !dy || !stats || !workspace || workspace_bytes < layout_of(*d).total) return NCA_ERR_INVALID;
  const NormArgs a = args_of(*d, x, weight, bias, mask, dy, dx, const_cast<float*>(stats), workspace);
  float2* params = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + layout_of(*d).params);
  const int v = vector_width(*d, a, true);
  if (norm_held_applies(a, d->dtype, v, true)) {
    NormArgs b = a;
    if (!dweight && !dbias) b.part = nullptr;
    const int32_t r = norm_held_backward(b, d->dtype, d->act, v, s);
    if (r != NCA_OK || !b.part) return r;
    param_grads(a.part, a.n * norm_held_slices(a, d->dtype, v), a.channels, dweight, dbias, a.param_dtype, params, s);
    return launch_status();
  }
  return dispatch(*d, streaming_width(d->dtype, v), BackwardCall{*d, a, dweight, dbias, params, s});
}

}  // extern "C"
