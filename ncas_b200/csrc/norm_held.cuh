// norm_held.cuh -- group norm with an activation, samples held in shared memory: every value is read
// from memory once (forward: x in, y out; backward: x and dy in, dx out).
//
// A block, or a cluster of `slices` blocks that split the cells, takes one sample, or a block of its
// channels that ends on group borders.  A thread owns the same V adjacent channels (of one group, or pairs
// of one group each) of every TY-th cell and copies its values asynchronously into places of its own in shared memory, so that no
// thread waits for another's data (norm_held_forward.cu, norm_held_backward.cu); statistics are merged through shared memory, and over a cluster
// through distributed shared memory.
//
// The mathematics and the treatment of sums are those of norm.cu.  Bound by HBM and, close behind, by
// instructions; the copies of the blocks that share a multiprocessor overlap with each other's arithmetic
// and writes.  On a B200, 8000 samples of 81 x 64 fp32, silu: forward 58 to 61 us (5.4 to 5.7 TB/s, 66% of
// the issue slots), backward 109 to 115 us (4.3 to 4.6 TB/s; its arithmetic, 62% of the issue slots, and 4
// blocks a multiprocessor bind).
#pragma once
#include <algorithm>
#include <atomic>

#include "norm.cuh"

namespace nca {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxSlices = 8;
constexpr int kMaxGroups = 64;  // of one block

struct HeldArgs {
  NormArgs a;
  int cb;             // channels of a block
  int cblocks;        // blocks of channels
  int slices;
  long long slice_cells;
  int iters;          // places of a thread
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void put_remote(const float4* p, uint32_t rank, float4 v) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(r), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// What a thread works on.
struct Work {
  long long sample;
  int ch0, ch;         // first channel of the block, of the thread
  int col, row, rank;
  long long c0;        // first cell of the slice
  int cells;           // and how many
  bool on;
};
template <int V>
__device__ __forceinline__ Work work_of(const HeldArgs& h) {
  Work w;
  const long long id = blockIdx.x / h.slices;
  w.rank = h.slices > 1 ? (int)cluster_rank() : 0;
  w.sample = id / h.cblocks;
  w.ch0 = (int)(id % h.cblocks) * h.cb;
  w.col = threadIdx.x % h.a.tx;
  w.row = threadIdx.x / h.a.tx;
  w.ch = w.ch0 + w.col * V;
  w.c0 = w.rank * h.slice_cells;
  w.cells = (int)min(h.a.cells - w.c0, h.slice_cells);
  w.on = w.row < h.a.ty && w.ch < h.a.channels;
  return w;
}
// The cells of a thread that the mask keeps, a bit for each of its places (32 at most).
template <bool MASK>
__device__ __forceinline__ uint32_t kept_of(const NormArgs& a, const Work& w) {
  if (!w.on) return 0;
  if constexpr (!MASK) return ~0u;
  uint32_t bits = 0;
  const uint8_t* m = a.mask + w.sample * a.m_sn + (w.c0 + w.row) * a.m_sl;
  const long long step = a.ty * a.m_sl;
  int i = 0;
  for (int c = w.row; c < w.cells; c += 8 * a.ty, i += 8, m += 8 * step) {
    uint8_t v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = c + u * a.ty < w.cells ? m[u * step] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) bits |= (uint32_t)(v[u] != 0) << (i + u);
  }
  return bits;
}
// Goes through the thread's cells: f(place in shared memory, cell of the slice) where the cell counts, g
// where the mask leaves it out.
template <bool MASK, class F, class G>
__device__ __forceinline__ void each_cell(const NormArgs& a, const Work& w, uint32_t bits, F f, G g) {
  int at = threadIdx.x;
  for (int c = w.on ? w.row : w.cells; c < w.cells; c += a.ty, at += blockDim.x) {
    if (!MASK || (bits & 1)) f(at, c);
    else g(at, c);
    if (MASK) bits >>= 1;
  }
}

// --------------------------------------------------------------------------------- host side
struct HeldPlan {
  bool ok, one;       // one: a thread's channels lie in one group
  int v, cb, cblocks, slices, tx, ty, iters, threads;
  long long slice_cells;
  size_t smem;
};

HeldPlan plan_of(const NormArgs& a, int dtype, int width, bool backward) {
  HeldPlan p{};
  const size_t size = dtype_size(dtype);
  // 16-byte vectors where groups hold whole ones, or pairs of channels; else what divides a group
  int v = width;
  p.one = !(v * size == 16 && a.per_group % v != 0 && a.per_group % 2 == 0);
  while (p.one && v > 1 && a.per_group % v) v /= 2;
  if (v * size < 4) return p;  // an asynchronous copy moves 4 bytes at least
  p.v = v;
  const size_t tensors = backward ? 2 : 1;
  // channels of a block: all of them, or fewer whole groups when a sample would need more than 8 blocks of
  // 100 KB, 256 adjacent bytes of them at least.  With shorter pieces the streaming kernels are faster on
  // much data (64 x 4096 x 320 bf16 in 32 groups: forward 109 against 140 us, backward 189 against 480), but
  // not on little, where their three launches cost more (4 x 4096 x 1024: 45 against 28 us).
  const size_t all = (size_t)a.n * a.cells * a.channels * size;
  const size_t narrowest = all < (48u << 20) ? 64 : 256;
  const size_t kFew = (backward ? 56 : 32) * 1024, kTwo = 100 * 1024;
  const auto bytes_of = [&](int g) { return (size_t)a.cells * g * a.per_group * size * tensors; };
  int groups = a.groups;
  const auto whole = [&](int g) { return a.groups % g == 0 && g * a.per_group % v == 0; };
  while (bytes_of(groups) > kMaxSlices * kTwo || groups > kMaxGroups || groups * a.per_group / v > kMaxThreads) {
    int next = groups - 1;
    while (next > 0 && !whole(next)) --next;
    if (next <= 0 || next * a.per_group * size < narrowest) return p;
    groups = next;
  }
  p.cb = groups * a.per_group;
  p.cblocks = a.groups / groups;
  const size_t bytes = bytes_of(groups);
  long long slices = (long long)((bytes + kFew - 1) / kFew);
  if (slices > kMaxSlices) slices = (long long)((bytes + kTwo - 1) / kTwo);
  // few samples: over more blocks, 8 KB each at least
  while (slices < kMaxSlices && a.n * p.cblocks * slices < 148 && (long long)bytes / slices > 16384) slices *= 2;
  slices = std::min({slices, (long long)kMaxSlices, (long long)a.cells});
  p.slice_cells = (a.cells + slices - 1) / slices;
  p.slices = (int)((a.cells + p.slice_cells - 1) / p.slice_cells);
  p.tx = p.cb / v;
  const long long ty_max = kMaxThreads / p.tx;
  long long iters = (p.slice_cells + ty_max - 1) / ty_max;
  // 8000 9 x 9 boards of 64 fp32 channels and padded 59 x 59 mazes: 16 places a thread forward, 8 backward
  // (more threads hide the latency of a block's few steps, fewer share the cost of its sums)
  const long long least = backward ? 8 : 16;
  if (iters < least) iters = std::min<long long>(p.slice_cells, least);
  p.ty = (int)((p.slice_cells + iters - 1) / iters);
  p.iters = (int)((p.slice_cells + p.ty - 1) / p.ty);
  p.threads = (p.tx * p.ty + 31) / 32 * 32;
  p.smem = (size_t)p.iters * p.threads * v * size * tensors;
  p.smem += (size_t)p.slices * groups * sizeof(float4) + (size_t)p.ty * sizeof(int);
  if (backward) p.smem += ((size_t)p.ty * p.tx * v + p.cb) * sizeof(float2);
  else p.smem += (size_t)p.threads * (p.one ? 1 : v / 2) * sizeof(float2);
  p.ok = p.smem <= 208 * 1024 && p.iters <= 32 && a.n * p.cblocks * p.slices < (1ll << 31);
  return p;
}

constexpr int kMaxDevices = 64;

int32_t launch(void (*kernel)(HeldArgs), std::atomic<uint64_t>& ready, const NormArgs& a, const HeldPlan& p,
               cudaStream_t s) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return NCA_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 208 * 1024) != cudaSuccess) {
      const int32_t st = launch_status();
      return st == NCA_OK ? NCA_ERR_CUDA : st;
    }
    ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  HeldArgs h{a, p.cb, p.cblocks, p.slices, p.slice_cells, p.iters};
  h.a.tx = p.tx;
  h.a.ty = p.ty;
  return launch_after(kernel, dim3((unsigned)(a.n * p.cblocks * p.slices)), dim3(p.threads), p.smem, s, p.slices, h);
}


// Instantiates fn(T, V, ACT, MASK, ONE) for the run-time choice.
template <class F>
int32_t dispatch_held(const NormArgs& a, int dtype, int act, const HeldPlan& p, F fn) {
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int W = 16 / sizeof(T);
    return with_act(act, [&](auto tag) {
      constexpr int A = decltype(tag)::value;
      if (!p.one) return a.mask ? fn.template operator()<T, W, A, true, false>() : fn.template operator()<T, W, A, false, false>();
      if (p.v == W) return a.mask ? fn.template operator()<T, W, A, true, true>() : fn.template operator()<T, W, A, false, true>();
      if (p.v == W / 2)
        return a.mask ? fn.template operator()<T, W / 2, A, true, true>() : fn.template operator()<T, W / 2, A, false, true>();
      return a.mask ? fn.template operator()<T, W / 4, A, true, true>() : fn.template operator()<T, W / 4, A, false, true>();
    });
  });
}

}  // namespace
}  // namespace nca
