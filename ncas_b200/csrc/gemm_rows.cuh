// gemm_rows.cuh -- the gated block's products for few rows (64 at most), where reading the weights is all
// that counts.
//
// The weights take the 128-row side of the MMA and the rows of x its narrow side (N = 16, 32 or 64), so
// a weight is loaded once and no tensor-core work is spent on absent rows.  A CTA streams 128 outputs
// (128 of gate and 128 of up together) over a piece of the k axis; a cluster of `slices` CTAs covers the
// axis, and each of them gathers the pieces' fp32 sums of its share of the outputs through distributed
// shared memory, in the order of the pieces.  About 2 CTAs a multiprocessor, 100 KB of weights in flight
// each: one output tile a CTA over the whole axis would leave most multiprocessors without work.
// The second product is launched while the first runs (programmatic dependent launch) and loads its
// weights before it waits for h.  (Prefetching them into L2 from the first took 2 us
// longer in all: its own loads have the bandwidth.)
// On a B200, bf16, one row through 2048 -> 8192 -> 2048: 23.9 us in a CUDA graph for 100.7 MB (4.2 TB/s);
// 8 rows through 4096 -> 16384 -> 4096: 72 us (5.6 TB/s).  Bound by HBM and the two launches' ramps.
#pragma once
#include "gemm.cuh"

namespace nca {

struct RowsParams {
  CUtensorMap w[2];  // 128 x 64 boxes of the weights (gate, up; or down)
  CUtensorMap x;     // N x 64 boxes of the rows
  int rows, n;       // rows of x, outputs
  int kb;            // k blocks of 64
  int slices;
  int weights_first; // the launch before writes x alone: the weights need not wait for it
  void* out;         // [rows][ld]
  long long ld;
  const void* bias[2];
  int bias_dtype;
  int* ctrl;
  unsigned long long timeout_ns;
};

constexpr int kRowsThreads = 192;

template <int N, bool GATE>
struct RowsShape {
  static constexpr int kAcc = GATE ? 2 : 1;
  static constexpr int kWBytes = kAcc * kBM * kBK * 2;
  static constexpr int kXBytes = N * kBK * 2;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kRow = N + 4;  // floats: lanes that read a column meet few banks twice
  static constexpr int kSums = kAcc * kBM * kRow * (int)sizeof(float);  // [slice][acc][rows of the share][kRow]
  static constexpr int kBlocks = GATE && N == 64 ? 1 : 2;  // CTAs a multiprocessor
  static constexpr int kStages = (220 * 1024 / kBlocks - 2048 - kSums) / kStageBytes;
  static constexpr int kSumsAt = kStages * kStageBytes;
  static constexpr int kBars = kSumsAt + kSums;
  static constexpr int kSmem = kBars + 256 + 1024;
  static constexpr int kTmemCols = kAcc * N < 32 ? 32 : kAcc * N;
  static_assert(kStages >= 2, "ring too short");
};

template <class T, int N, bool GATE, int ACT>
__global__ void __launch_bounds__(kRowsThreads) gemm_rows_kernel(const __grid_constant__ RowsParams p) {
  using S = RowsShape<N, GATE>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* sums = reinterpret_cast<float*>(smem + S::kSumsAt);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + S::kStages;
  uint64_t* done = empty + S::kStages;
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_base_s + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.slices > 1 ? (int)cta_rank_in_cluster() : 0;
  const int tile = blockIdx.x / p.slices;
  const FailState fs{p.ctrl, abort_s, 0, p.timeout_ns, true};

  if (p.slices > 1) cluster_started_arrive();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    *abort_s = 0;
    fence_mbar_init();
  }
  if (warp == 1) tc_alloc<1>(tmem_base_s, S::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_base_s;
  const int kb0 = p.kb * rank / p.slices, kb1 = p.kb * (rank + 1) / p.slices;

  if (warp == 0) {
    if (lane == 0) {
      const auto load_w = [&](int s, int kb) {
        const uint32_t at = smem_u32(smem + s * S::kStageBytes), bar = smem_u32(&full[s]);
        mbar_arrive_expect_tx(&full[s], S::kStageBytes);
        tma_load_2d<1>(at, &p.w[0], bar, kb * kBK, tile * kBM);
        if (GATE) tma_load_2d<1>(at + kBM * kBK * 2, &p.w[1], bar, kb * kBK, tile * kBM);
      };
      const auto load_x = [&](int s, int kb) {
        tma_load_2d<1>(smem_u32(smem + s * S::kStageBytes) + S::kWBytes, &p.x, smem_u32(&full[s]), kb * kBK, 0);
      };
      const int n = kb1 - kb0, ahead = n < S::kStages ? n : S::kStages;
      // The next launch may load its weights before this one ends, so it must not start before all that
      // ran ahead of this one (which may have written them) has ended: only after after_previous().
      if (!p.weights_first) {
        after_previous();
        may_start_next();
      }
      for (int i = 0; i < ahead; ++i) load_w(i, kb0 + i);
      if (p.weights_first) {
        after_previous();
        may_start_next();
      }
      for (int i = 0; i < ahead; ++i) load_x(i, kb0 + i);
      int i = ahead;
      for (; i < n; ++i) {
        const int s = i % S::kStages;
        if (!mbar_wait(&empty[s], (i / S::kStages + 1) & 1, fs, 111)) break;
        load_w(s, kb0 + i);
        load_x(s, kb0 + i);
      }
      // loads in flight land before this CTA leaves, also when only another warp gave up (bounded)
      for (int j = i > S::kStages ? i - S::kStages : 0; j < i; ++j)
        for (int tries = 0; tries < 64 && !mbar_try_wait(&full[j % S::kStages], (j / S::kStages) & 1); ++tries) {
        }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr bool is_bf16 = __is_same(T, __nv_bfloat16);
      constexpr uint32_t idesc = (1u << 4) | ((is_bf16 ? 1u : 0u) << 7) | ((is_bf16 ? 1u : 0u) << 10) |
                                 ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
      for (int i = 0; i < kb1 - kb0; ++i) {
        const int s = i % S::kStages;
        if (!mbar_wait(&full[s], (i / S::kStages) & 1, fs, 112)) break;
        tc_fence_after();
        const uint32_t at = smem_u32(smem + s * S::kStageBytes);
        const uint64_t dx = smem_desc(at + S::kWBytes, 16, 1024);
#pragma unroll
        for (int a = 0; a < S::kAcc; ++a) {
          const uint64_t dw = smem_desc(at + a * kBM * kBK * 2, 16, 1024);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) umma_ss<1>(tmem + a * N, dw + 2 * k, dx + 2 * k, idesc, i > 0 || k > 0);
        }
        umma_commit(&empty[s]);
      }
      umma_commit(done);
      // they end before the tensor memory is freed, also when only the epilogue gave up (bounded)
      for (int tries = 0; tries < 64 && !mbar_try_wait(done, 0); ++tries) {
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3;  // tensor memory lanes 32 q .. 32 q + 31: an output each
    const bool ok = mbar_wait_warp(done, 0, fs, 113);
    tc_fence_after();
    if (p.slices > 1) cluster_started_wait();
    if (ok) {
      const int share = kBM / p.slices, row = 32 * q + lane;
      const int to = row / share, at = row % share;
#pragma unroll
      for (int a = 0; a < S::kAcc; ++a)
#pragma unroll
        for (int c = 0; c < N; c += 16) {
          uint32_t r[16];
          tmem_take16(tmem + a * N + c + ((uint32_t)(32 * q) << 16), r);
          float* mine = sums + ((rank * S::kAcc + a) * share + at) * S::kRow + c;
          if (p.slices > 1) {
            const uint32_t far = map_to_rank(smem_u32(mine), to);
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(far + 4 * i), "r"(r[i]),
                           "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
                           : "memory");
          } else {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<uint4*>(mine + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
          }
        }
    }
    tc_fence_before();
  }
  __syncwarp();
  if (p.slices > 1 && warp < 2) cluster_started_wait();  // the others have waited
  if (p.slices > 1) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) tc_dealloc<1>(tmem, S::kTmemCols);
  after_previous();  // every thread that writes
  // this CTA's share of the outputs, every row
  const int share = kBM / p.slices, first = tile * kBM + rank * share;
  for (int i = threadIdx.x; i < share * p.rows; i += kRowsThreads) {
    const int at = i % share, t = i / share, f = first + at;
    if (f >= p.n) continue;
    float v[S::kAcc];
#pragma unroll
    for (int a = 0; a < S::kAcc; ++a) {
      v[a] = 0.f;
      for (int s = 0; s < p.slices; ++s) v[a] += sums[((s * S::kAcc + a) * share + at) * S::kRow + t];
      if (p.bias[a]) v[a] += load_param(p.bias[a], p.bias_dtype, f);
    }
    float r = v[0];
    if constexpr (GATE) r = act_f<ACT>(v[0]) * v[1];
    static_cast<T*>(p.out)[t * p.ld + f] = from_f32<T>(r);
  }
}

}  // namespace nca
