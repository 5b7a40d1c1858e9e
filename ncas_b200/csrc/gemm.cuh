// gemm.cuh -- the tcgen05 matrix-product kernel behind the gated feed-forward block (gated.cu).
//
// D[M, N] = sum_k A[m, k] B[n, k] with 16-bit operands and fp32 sums in tensor memory.  Either
// operand may be stored with k adjacent ("K-major") or with its rows adjacent ("MN-major": the
// transposed operand of a backward product is read as it lies, nothing is transposed in memory).
//
// One persistent CTA (CG = 1) or CTA pair (CG = 2, cta_group::2: one 256-row tile over two
// multiprocessors, each loading half of B) per multiprocessor.  Warp 0 loads tiles by TMA into a
// ring of shared-memory stages, warp 1 issues the MMAs, warp 2 owns the tensor memory, warps 4-11
// take finished accumulators out and apply the epilogue (two warps a quarter of the lanes, in turn
// over pieces of 32 columns).  They own rows of the accumulator, memory wants lines of columns: what
// is stored and loaded passes through 2.5 KB of shared memory of the warp.  Two accumulators in tensor memory let
// the epilogue of one tile run under the MMAs of the next.
#pragma once
#include <cuda.h>

#include "cell_ops.cuh"
#include "ptx.cuh"

namespace nca {

enum GemmEpilogue {
  EPI_STORE = 0,    // c = D (+ bias), rounded to the matrix type
  EPI_PARTIAL = 1,  // fp32 partial sums of one piece of a long k axis
  EPI_GATE = 2,     // columns are gate | up halves: h = act(gate) up (and gate, up when saved)
  EPI_DGATE = 3     // D = dh: dgate = dh up act'(gate), dup = dh act(gate)
};

struct GemmParams {
  CUtensorMap a[2], b[2];
  int m, n;            // logical rows and columns of D (columns of one half for EPI_GATE)
  int m_tiles, n_tiles;
  int batch;           // independent products: a[z], c[z] (1 or 2)
  int splits;          // pieces of the k axis (EPI_PARTIAL)
  int kb;              // k blocks of 64
  int kb_second;       // first k block that reads a[1], b[1] (kb when there is one source)
  void* c[2];          // EPI_STORE: outputs; EPI_GATE: h, -; EPI_DGATE: dgate, dup
  long long ldc;
  int vec_c;           // 16-byte stores allowed
  const void* bias[2];
  int bias_dtype;
  uint16_t* saved;     // pre-activations (SavedPlanes): EPI_GATE writes (may be null), EPI_DGATE reads
  long long plane;     // distance of the three planes
  float* part;         // [batch * splits][m][ldp]
  long long ldp;
  int* ctrl;
  unsigned long long timeout_ns;
};

constexpr int kGemmThreads = 384;
constexpr int kEpilogueWarps = 8;
constexpr int kBM = 128, kBK = 64;

// ------------------------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ uint32_t cta_rank_in_cluster() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void tc_alloc(uint32_t* dst, uint32_t cols) {
  if constexpr (CG == 1) {
    tmem_alloc(dst, cols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tc_dealloc(uint32_t addr, uint32_t cols) {
  if constexpr (CG == 1) tmem_dealloc(addr, cols);
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
// D[tmem] (+)= A[smem] B[smem]^T, 16-bit inputs of one type, fp32 accumulators.
template <int CG>
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives on `bar` (of both CTAs of a pair) when the MMAs issued so far have finished.
template <int CG>
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  if constexpr (CG == 1) {
    umma_commit(bar);
  } else {
    const uint16_t both = 3;
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(both)
        : "memory");
  }
}

// The same on a barrier of this CTA alone.
template <int CG>
__device__ __forceinline__ void umma_commit_local(uint64_t* bar) {
  if constexpr (CG == 1)
    umma_commit(bar);
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// Shared-memory descriptor of a 128-byte-swizzled operand tile.  K-major: rows of 64 values (128
// bytes), 8 rows a swizzle atom, `sbo` the distance of atoms along the rows (lbo unused).
// MN-major: k lines of 64 adjacent rows (128 bytes), 8 lines an atom; `sbo` the distance of atoms
// along k, `lbo` the distance of blocks of 64 rows.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(lbo >> 4) << 16;
  d |= (uint64_t)(sbo >> 4) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version of sm_100
  d |= (uint64_t)2 << 61;  // 128-byte swizzle
  return d;
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// 32 rows of 64 bytes between a lane's row (registers) and lines of memory: the warp's staging place
// has rows of 80 bytes, so that neither side meets a bank twice.
constexpr int kStageRow = 80;
struct Staging {
  uint8_t* smem;  // [32][kStageRow]
  int lane;
  // Writes `bytes` of each of the first `rows` rows to to + row * ld (bytes).  vec: 16 bytes at a time
  // (whole ones: the caller's rows are padded to that), else 2 at a time.
  __device__ __forceinline__ void put(uint8_t* to, long long ld, int rows, int bytes, bool vec, const uint4 (&v)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(smem + lane * kStageRow + 16 * i) = v[i];
    __syncwarp();
    if (vec) {
      const int piece = 16 * (lane & 3);
      const uint8_t* from = smem + (lane >> 2) * kStageRow + piece;
      to += (lane >> 2) * ld + piece;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (8 * i + (lane >> 2) < rows && piece < bytes)
          *reinterpret_cast<uint4*>(to + 8 * i * ld) = *reinterpret_cast<const uint4*>(from + 8 * i * kStageRow);
    } else {
      for (int r = 0; r < rows; ++r)
        if (2 * lane < bytes)
          *reinterpret_cast<uint16_t*>(to + r * ld + 2 * lane) = *reinterpret_cast<const uint16_t*>(smem + r * kStageRow + 2 * lane);
    }
    __syncwarp();
  }
  // The loads of a `take` that comes later: this lane's pieces of the 32 rows.
  static __device__ __forceinline__ void ask(const uint8_t* from, long long ld, int rows, int bytes, int lane, uint4 (&v)[4]) {
    const int piece = 16 * (lane & 3);
    from += (lane >> 2) * ld + piece;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = 8 * i + (lane >> 2) < rows && piece < bytes ? *reinterpret_cast<const uint4*>(from + 8 * i * ld)
                                                         : make_uint4(0, 0, 0, 0);
  }
  // Turns them into the lane's row.
  __device__ __forceinline__ void take(uint4 (&v)[4]) const {
    uint8_t* at = smem + (lane >> 2) * kStageRow + 16 * (lane & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(at + 8 * i * kStageRow) = v[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4*>(smem + lane * kStageRow + 16 * i);
    __syncwarp();
  }
};
template <class T>
__device__ __forceinline__ void pack_row(const float (&v)[32], uint4 (&q)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q[i] = make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                      pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7]));
}

// The pre-activations kept for the backward pass: the upper 24 bits of their fp32 values (relative
// error below 2^-15, the full fp32 range).  In the matrix type, bf16 would put 2^-8 more noise into
// every gradient, and fp16 would overflow where the fp32 sum does not; the third plane costs 2 of
// 8 bytes.  Three planes of 16-bit values: gate bits 31-16, up bits 31-16, and bits 15-8 of both
// (gate low byte, up high byte).
__device__ __forceinline__ void split_planes(const float (&g)[32], const float (&u)[32], uint4 (&a)[4], uint4 (&b)[4],
                                             uint4 (&c)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t hg[4], hu[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = 8 * i + 2 * j;
      const uint32_t g0 = __float_as_uint(g[k]), g1 = __float_as_uint(g[k + 1]);
      const uint32_t u0 = __float_as_uint(u[k]), u1 = __float_as_uint(u[k + 1]);
      hg[j] = __byte_perm(g0, g1, 0x7632);
      hu[j] = __byte_perm(u0, u1, 0x7632);
      lo[j] = __byte_perm(__byte_perm(g0, u0, 0x0051), __byte_perm(g1, u1, 0x0051), 0x5410);
    }
    a[i] = make_uint4(hg[0], hg[1], hg[2], hg[3]);
    b[i] = make_uint4(hu[0], hu[1], hu[2], hu[3]);
    c[i] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}
__device__ __forceinline__ void join_planes(const uint4 (&a)[4], const uint4 (&b)[4], const uint4 (&c)[4], float (&g)[32],
                                            float (&u)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t hg[4] = {a[i].x, a[i].y, a[i].z, a[i].w}, hu[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
    const uint32_t lo[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = 8 * i + 2 * j;
      g[k] = __uint_as_float((hg[j] << 16) | (lo[j] << 8 & 0xFF00u));
      g[k + 1] = __uint_as_float((hg[j] & 0xFFFF0000u) | (lo[j] >> 8 & 0xFF00u));
      u[k] = __uint_as_float((hu[j] << 16) | (lo[j] & 0xFF00u));
      u[k + 1] = __uint_as_float((hu[j] & 0xFFFF0000u) | (lo[j] >> 16 & 0xFF00u));
    }
  }
}

template <int CG, int BN>
struct GemmShape {
  static constexpr int kBNc = BN / CG;  // rows of B in one CTA
  static constexpr int kABytes = kBM * kBK * 2;
  static constexpr int kBBytes = kBNc * kBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = (196 * 1024) / kStageBytes;
  static constexpr int kBars = kStages * kStageBytes;  // barriers, then biases, then the staging places
  static constexpr int kBias = kBars + 256;
  static constexpr int kStaging = kBias + 2 * 256 * (int)sizeof(float);
  static constexpr int kSmem = kStaging + kEpilogueWarps * 32 * kStageRow + 1024;  // alignment
  static constexpr int kTmemCols = 2 * BN;
};

struct GemmTile {
  int m0, n0, batch, split, kb0, kb1;
};

// Tiles in groups of 8 tile rows, columns within, so that tiles that run together share operands
// in L2.  TN: columns of D that one tile covers.
template <int TM, int TN>
__device__ __forceinline__ GemmTile tile_of(const GemmParams& p, int t) {
  GemmTile r;
  const int per = p.m_tiles * p.n_tiles;
  const int z = t / per;
  int i = t - z * per;
  r.batch = z % p.batch;
  r.split = z / p.batch;
  const int group = 8 * p.n_tiles;
  const int g = i / group;
  const int rows = min(8, p.m_tiles - g * 8);
  i -= g * group;
  r.m0 = (g * 8 + i % rows) * TM;
  r.n0 = (i / rows) * TN;
  r.kb0 = (int)((long long)p.kb * r.split / p.splits);
  r.kb1 = (int)((long long)p.kb * (r.split + 1) / p.splits);
  return r;
}

template <class T, int CG, int BN, bool A_MN, bool B_MN, int EPI, int ACT>
__global__ void __launch_bounds__(kGemmThreads, 1) gemm_kernel(const __grid_constant__ GemmParams p) {
  using S = GemmShape<CG, BN>;
  constexpr int kTN = EPI == EPI_GATE ? BN / 2 : BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drained = acc_empty + 2;
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_base_s + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 1 ? 0 : cta_rank_in_cluster();
  const FailState fs{p.ctrl, abort_s, 0, p.timeout_ns};

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpilogueWarps * CG);
    }
    mbar_init(drained, 1);
    *abort_s = 0;
    fence_mbar_init();
  }
  if (warp == 2) tc_alloc<CG>(tmem_base_s, S::kTmemCols);
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_base_s;

  const int tiles = p.m_tiles * p.n_tiles * p.batch * p.splits;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      long long issued = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        const GemmTile tl = tile_of<kBM * CG, kTN>(p, t);
        const int am = tl.m0 + (int)rank * kBM;
        for (int kb = tl.kb0; kb < tl.kb1; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1, fs, 101)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[s], S::kStageBytes * CG);
          const uint32_t bar = CG == 1 ? smem_u32(&full[s]) : map_to_rank(smem_u32(&full[s]), 0);
          const uint32_t sa = smem_u32(smem + s * S::kStageBytes), sb = sa + S::kABytes;
          const int second = kb >= p.kb_second;
          const int k0 = (second ? kb - p.kb_second : kb) * kBK;
          const CUtensorMap* ma = &p.a[p.batch == 2 ? tl.batch : second];
          if constexpr (A_MN) {
#pragma unroll
            for (int i = 0; i < kBM / 64; ++i) tma_load_2d<CG>(sa + i * 8192, ma, bar, am + 64 * i, k0);
          } else {
            tma_load_2d<CG>(sa, ma, bar, k0, am);
          }
          if constexpr (EPI == EPI_GATE) {
            if constexpr (CG == 2) {
              tma_load_2d<CG>(sb, &p.b[rank], bar, k0, tl.n0);
            } else {
              tma_load_2d<CG>(sb, &p.b[0], bar, k0, tl.n0);
              tma_load_2d<CG>(sb + S::kBBytes / 2, &p.b[1], bar, k0, tl.n0);
            }
          } else {
            const CUtensorMap* mb = &p.b[second];
            const int bn = tl.n0 + (int)rank * S::kBNc;
            if constexpr (B_MN) {
#pragma unroll
              for (int i = 0; i < S::kBNc / 64; ++i) tma_load_2d<CG>(sb + i * 8192, mb, bar, bn + 64 * i, k0);
            } else {
              tma_load_2d<CG>(sb, mb, bar, k0, bn);
            }
          }
          ++issued;
          if (++s == S::kStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok && rank == 0) {  // loads in flight land before this CTA leaves (bounded)
        for (long long i = issued > S::kStages ? issued - S::kStages : 0; i < issued; ++i)
          for (int tries = 0; tries < 64 && !mbar_try_wait(&full[i % S::kStages], (i / S::kStages) & 1); ++tries) {
          }
      }
    }
  } else if (warp == 1 && rank == 0) {
    if (lane == 0) {
      constexpr bool is_bf16 = __is_same(T, __nv_bfloat16);
      constexpr uint32_t idesc = (1u << 4) | ((is_bf16 ? 1u : 0u) << 7) | ((is_bf16 ? 1u : 0u) << 10) |
                                 ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) |
                                 ((uint32_t)(kBM * CG >> 4) << 24);
      // one MMA takes 16 k: 32 bytes along a K-major row, 16 lines of 128 bytes MN-major
      constexpr uint32_t a_step = (A_MN ? 2048 : 32) >> 4, b_step = (B_MN ? 2048 : 32) >> 4;
      int s = 0, buf = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        const GemmTile tl = tile_of<kBM * CG, kTN>(p, t);
        if (!mbar_wait(&acc_empty[buf], acc_ph ^ 1, fs, 102)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + buf * BN;
        for (int kb = tl.kb0; kb < tl.kb1; ++kb) {
          if (!mbar_wait(&full[s], ph, fs, 103)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * S::kStageBytes), sb = sa + S::kABytes;
          const uint64_t da = smem_desc(sa, A_MN ? 8192 : 16, 1024);
          const uint64_t db = smem_desc(sb, B_MN ? 8192 : 16, 1024);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            umma_ss<CG>(d, da + k * a_step, db + k * b_step, idesc, kb > tl.kb0 || k > 0);
          tc_commit<CG>(&empty[s]);
          if (++s == S::kStages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        tc_commit<CG>(&acc_full[buf]);
        buf ^= 1;
        if (buf == 0) acc_ph ^= 1;
      }
      if (!ok) {  // the MMAs in flight end before the tensor memory is freed (bounded)
        umma_commit_local<CG>(drained);
        for (int tries = 0; tries < 64 && !mbar_try_wait(drained, 0); ++tries) {
        }
      }
    }
  } else if (warp >= 4) {
    const int q = (warp - 4) & 3, turn = (warp - 4) >> 2;  // tensor memory lanes 32 q .. 32 q + 31
    const Staging st{smem + S::kStaging + (warp - 4) * 32 * kStageRow, lane};
    float* bias_s = reinterpret_cast<float*>(smem + S::kBias);  // [2][256]
    const bool biased = (EPI == EPI_GATE || EPI == EPI_STORE) && (p.bias[0] || p.bias[1]);
    int buf = 0;
    uint32_t ph = 0;
    for (int t = first; t < tiles; t += step) {
      const GemmTile tl = tile_of<kBM * CG, kTN>(p, t);
      const int row0 = tl.m0 + (int)rank * kBM + 32 * q, rows = min(32, p.m - row0);
      const int cols = min(kTN, p.n - tl.n0);
      if (biased) {  // the tile's biases, as floats
        const int i = threadIdx.x - 128;
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the tile before has read its own
        if (i < cols) {
          bias_s[i] = p.bias[0] ? load_param(p.bias[0], p.bias_dtype, tl.n0 + i) : 0.f;
          if (EPI == EPI_GATE) bias_s[256 + i] = p.bias[1] ? load_param(p.bias[1], p.bias_dtype, tl.n0 + i) : 0.f;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      uint4 k0[4], k1[4], k2[4];  // EPI_DGATE: the saved planes, asked for ahead of the accumulator
      const auto ask = [&](int c) {
        const uint8_t* from = reinterpret_cast<const uint8_t*>(p.saved + (long long)row0 * p.ldc + tl.n0 + c);
        const int bytes = 2 * min(32, cols - c);
        Staging::ask(from, 2 * p.ldc, rows, bytes, lane, k0);
        Staging::ask(from + 2 * p.plane, 2 * p.ldc, rows, bytes, lane, k1);
        Staging::ask(from + 4 * p.plane, 2 * p.ldc, rows, bytes, lane, k2);
      };
      if (EPI == EPI_DGATE && 32 * turn < cols) ask(32 * turn);
      if (!mbar_wait(&acc_full[buf], ph, fs, 104)) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(32 * q) << 16);
      for (int c = 32 * turn; c < cols; c += 64) {
        const int col = tl.n0 + c, n = min(32, cols - c);
        uint32_t r0[32];
        tmem_ld32(acc + c, r0);
        if constexpr (EPI == EPI_GATE) {
          uint32_t r1[32];
          tmem_ld32(acc + kTN + c, r1);
          tc_wait_ld_regs(r0);
#pragma unroll
          for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r1[i]));
          float g[32], u[32], h[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            g[i] = __uint_as_float(r0[i]);
            u[i] = __uint_as_float(r1[i]);
          }
          if (biased) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              g[i] += bias_s[c + i];
              u[i] += bias_s[256 + c + i];
            }
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 a = mul2(act2<ACT>(make_float2(g[i], g[i + 1])), make_float2(u[i], u[i + 1]));
            h[i] = a.x;
            h[i + 1] = a.y;
          }
          const long long at = (long long)row0 * p.ldc + col;
          uint4 v[4];
          pack_row<T>(h, v);
          st.put(reinterpret_cast<uint8_t*>(static_cast<T*>(p.c[0]) + at), 2 * p.ldc, rows, 2 * n, true, v);
          if (p.saved) {
            uint4 v1[4], v2[4];
            split_planes(g, u, v, v1, v2);
            uint8_t* to = reinterpret_cast<uint8_t*>(p.saved + at);
            st.put(to, 2 * p.ldc, rows, 2 * n, true, v);
            st.put(to + 2 * p.plane, 2 * p.ldc, rows, 2 * n, true, v1);
            st.put(to + 4 * p.plane, 2 * p.ldc, rows, 2 * n, true, v2);
          }
        } else if constexpr (EPI == EPI_DGATE) {
          st.take(k0);
          st.take(k1);
          st.take(k2);
          float g[32], u[32];
          join_planes(k0, k1, k2, g, u);
          if (c + 64 < cols) ask(c + 64);
          tc_wait_ld_regs(r0);
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 dh = make_float2(__uint_as_float(r0[i]), __uint_as_float(r0[i + 1]));
            float2 a;
            const float2 slope = act_slope2<ACT>(make_float2(g[i], g[i + 1]), a);
            const float2 dg = mul2(mul2(dh, make_float2(u[i], u[i + 1])), slope), du = mul2(dh, a);
            g[i] = dg.x, g[i + 1] = dg.y;
            u[i] = du.x, u[i + 1] = du.y;
          }
          const long long at = (long long)row0 * p.ldc + col;
          uint4 v[4];
          pack_row<T>(g, v);
          st.put(reinterpret_cast<uint8_t*>(static_cast<T*>(p.c[0]) + at), 2 * p.ldc, rows, 2 * n, true, v);
          pack_row<T>(u, v);
          st.put(reinterpret_cast<uint8_t*>(static_cast<T*>(p.c[1]) + at), 2 * p.ldc, rows, 2 * n, true, v);
        } else if constexpr (EPI == EPI_PARTIAL) {
          tc_wait_ld_regs(r0);
          uint8_t* to = reinterpret_cast<uint8_t*>(
              p.part + ((long long)(tl.split * p.batch + tl.batch) * p.m + row0) * p.ldp + col);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i] = make_uint4(r0[16 * half + 4 * i], r0[16 * half + 4 * i + 1], r0[16 * half + 4 * i + 2],
                                r0[16 * half + 4 * i + 3]);
            st.put(to + 64 * half, 4 * p.ldp, rows, 4 * (n - 16 * half), true, v);
          }
        } else {
          tc_wait_ld_regs(r0);
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r0[i]) + (biased ? bias_s[c + i] : 0.f);
          uint4 v[4];
          pack_row<T>(f, v);
          st.put(reinterpret_cast<uint8_t*>(static_cast<T*>(p.c[tl.batch]) + (long long)row0 * p.ldc + col), 2 * p.ldc,
                 rows, 2 * n, p.vec_c, v);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(map_to_rank(smem_u32(&acc_empty[buf]), 0));
        else mbar_arrive(&acc_empty[buf]);
      }
      buf ^= 1;
      if (buf == 0) ph ^= 1;
    }
  }
  __syncwarp();
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  if (warp == 2) tc_dealloc<CG>(tmem, S::kTmemCols);
}

}  // namespace nca
