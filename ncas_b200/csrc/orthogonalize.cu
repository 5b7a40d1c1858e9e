// orthogonalize.cu -- the orthogonalised update of a matrix by Newton-Schulz products
// (nca_b200_orthogonalize): X = M / (|M|_F + eps), then `steps` times
//
//   A = X X^T,  B = b A + c A^2,  X = a X + B X        (of a tall matrix A = X^T X, X = a X + X B)
//
// which brings the singular values of M towards 1.  The products run on the tensor cores with fp16 operands
// and fp32 sums, for bf16 input too: powers of two keep every operand in fp16's range (|X| <= 2 is checked
// for the coefficients), and its 11 bits leave an eighth of the error that bf16 operands would.  X is kept
// as hi + lo, two fp16 values of 22 bits together: a X amplifies what is left in the small singular
// directions by a at every step, and with X in 11 bits that would be rounding noise (6 % of the result
// for a matrix of rank 1).  The products read hi alone: their errors appear only beside large singular values,
// which nothing amplifies.  What a step leaves once the singular values have arrived stays, though: 1.0e-3 to 1.5e-3 of
// the result's norm a step, beside the 1.7e-3 of its own rounding to bf16 (2e-4 to fp16).  They have arrived
// about log(sqrt(rows)) / log(a) steps from the start, so of a bf16 matrix the steps beyond the first three from there on (5
// steps: matrices of fewer than 140 rows) read B and X in 22 bits in the largest product, hi hi + hi lo + lo hi, and of a
// fp16 matrix all of them in all three products.  Of matrices of fewer than 64 rows all steps
// do so in all products, whichever the type: nothing averages the few roundings of a small matrix, and beside a norm of sqrt(rows) an
// error of a strong direction weighs more (16 x 24 fp16, 6 steps: up to 4.6 times the rounding's without, 8 x 12
// bf16 3.5; 48 x 240 takes 36 us without and 48 with them in bf16, 45 and 48 in fp16).  One or two
// steps of a fp16 matrix do too, for a strong direction has arrived before the first (with nearly all of the norm in it, 1 step: up
// to 4.6 times the rounding's without; 1001 x 2730, 2 steps, 90 us without and 135 with them).  Errors of 1 to 8
// steps are then 1.0 to 1.4 times the rounding's on average, 1.9 at most (bf16, 8 steps).
//
// A and A^2 are symmetric: tiles above the diagonal are computed, and stored twice.  Where a product has few tiles, a
// cluster of 2 or 4 CTAs shares the k axis of each: every CTA adds up a share of the tile's columns through distributed
// shared memory and stores it.  Over a long axis A comes from pieces of it, stored in 22 bits, which a second kernel adds up.
//
// Matrices of up to 128 x 256 (and 256 x 256 where no step takes operands of 22 bits) run in one launch: a CTA (or a pair,
// cta_group::2) holds X as MMA operands in shared memory and in fp32 in tensor memory, beside the accumulator, for all
// steps.  256 x 256, 5 steps: 57 us, as 17 launches 98 (fp16 125 and 6 steps of bf16 128, which have no such form); a phase is
// about 2400 cycles of MMAs, 1400 to 3100 of epilogue and 1300 of cluster barrier (with twice the epilogue warps the same time), and
// 7 us pass before the first.
//
// Else one product kernel, built as gemm.cuh's: a persistent CTA or CTA pair (cta_group::2) a multiprocessor, warp 0
// loads tiles by TMA, warp 1 issues the MMAs, warps 4-11 take the accumulators out, add the terms that they load by
// TMA and store by TMA; two accumulators in tensor memory.  Matrices of a batch are the third dimension of
// the tensor maps, so that a tile reaches over its own matrix's edge into zeros and writes nothing there.
// 4096 x 16384 bf16: A, A^2 and the update take 194, 58 and 375 us a step, 1.1 to 1.5 PFLOP/s under the power cap; 12 x
// 1024 x 1024 22, 23 and 33 us, in few waves of tiles, half of their time ramps and epilogues.
#include "gemm.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>

using namespace nca;

namespace {

#define NCA_TRY(call)                    \
  do {                                   \
    const int32_t st_ = (call);          \
    if (st_ != NCA_OK) return st_;       \
  } while (0)

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
inline long long pad64(long long v) { return (v + 63) / 64 * 64; }
constexpr int kMaxDevices = 64;

// X is stored times 2^12: |X| <= 2 stays below 2^13, and the entries of a normalised matrix of 2^24 and more values
// are still normal fp16 numbers.  A, |A| <= 4, is stored times 2^10.
constexpr float kScaleX = 4096.f, kScaleA = 1024.f;

enum OrthoStep {
  STEP_POWER = 0,  // A, and B
  STEP_UPDATE = 1  // X, or the result
};

// alpha D + beta (src[0] + src[1]), stored as a value or as hi + lo.
struct OrthoParams {
  CUtensorMap a[2], b[2];  // hi and, where there are three passes, lo
  CUtensorMap src[2];  // boxes of 32 rows of 64 bytes: what the epilogue reads
  CUtensorMap out[2];
  int m, n;  // of D
  int m_tiles, n_tiles, batch, kb;
  int pieces;  // of the k axis, kb blocks each: matrix z / pieces, and results for every z
  int slices;  // SPLIT: CTAs that share a tile's k axis, 2 or 4
  int passes;  // over the k axis: 1, or 3 (hi lo, lo hi, hi hi: additions to a small sum lose less)
  int pair;    // the output as hi + lo
  int symmetric;
  int terms;  // matrices in src
  int last;   // STEP_UPDATE: out[0] is the result
  int out_bf16, plain_c;
  float alpha, beta, scale;
  uint16_t* c;  // the result, where its rows lie on no 16-byte boundaries
  long long ldc;
  int* ctrl;
  unsigned long long timeout_ns;
};

template <int CG>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if constexpr (CG == 1)
    tma_load_3d(dst, map, bar, x, y, z);
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
        "%5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// A lane's 32 values as a column of a place: row c of the place holds column c of the warp's 32 rows.
__device__ __forceinline__ void put_column(uint32_t place, int lane, const float (&f)[32]) {
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    const uint32_t at = place + 64 * c + ((16 * (lane >> 3)) ^ (16 * ((c >> 1) & 3))) + 2 * (lane & 7);
    asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(__half_as_ushort(__float2half_rn(f[c]))) : "memory");
  }
}
__device__ __forceinline__ void unpack_half(const uint4 (&q)[4], float (&f)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = __half22float2(reinterpret_cast<const __half2&>(w[j]));
      f[8 * i + 2 * j] = t.x;
      f[8 * i + 2 * j + 1] = t.y;
    }
  }
}

struct OrthoTile {
  int m0, n0, z;
};
// Symmetric: of tile row i the tiles from the diagonal on.
__host__ __device__ __forceinline__ int tiles_of(const OrthoParams& p, int tm, int tn) {
  if (!p.symmetric) return p.m_tiles * p.n_tiles;
  return p.m_tiles * p.n_tiles - (tm / tn) * (p.m_tiles * (p.m_tiles - 1) / 2);
}
template <int TM, int TN>
__device__ __forceinline__ OrthoTile tile_at(const OrthoParams& p, int per, int t) {
  OrthoTile r;
  r.z = t / per;
  int i = t - r.z * per;
  if (p.symmetric) {
    int row = 0;
    for (int left = p.n_tiles; i >= left; left -= TM / TN) {
      i -= left;
      ++row;
    }
    r.m0 = row * TM;
    r.n0 = (row * (TM / TN) + i) * TN;
  } else {  // groups of 8 tile rows, columns within: tiles that run together share operands in L2
    const int group = 8 * p.n_tiles, g = i / group, rows = min(8, p.m_tiles - g * 8);
    i -= g * group;
    r.m0 = (g * 8 + i % rows) * TM;
    r.n0 = (i / rows) * TN;
  }
  return r;
}

// A lane's row of a place (put_row's layout) in another block's shared memory.
__device__ __forceinline__ void put_remote(uint32_t place, int lane, const uint4 (&v)[4]) {
  const uint32_t row = place + 64 * lane, x = 16 * ((lane >> 1) & 3);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((16 * j) ^ x)), "r"(v[j].x), "r"(v[j].y),
                 "r"(v[j].z), "r"(v[j].w)
                 : "memory");
}

template <int CG, int BN>
using OrthoShape = GemmShape<CG, BN, EPI_DGATE>;  // four places an epilogue warp

// SPLIT (CG = 1): a cluster of p.slices CTAs works on one tile.
template <int CG, int BN, bool A_MN, bool B_MN, int STEP, bool SPLIT>
__global__ void __launch_bounds__(kGemmThreads, 1) ortho_kernel(const __grid_constant__ OrthoParams p) {
  using S = OrthoShape<CG, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drained = acc_empty + 2;
  uint64_t* loaded = drained + 1;  // the terms of each epilogue warp
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(loaded + kEpilogueWarps);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_base_s + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 1 ? 0 : cta_rank_in_cluster(), slice = SPLIT ? cta_rank_in_cluster() : 0;
  const FailState fs{p.ctrl, abort_s, 0, p.timeout_ns, true};

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
    for (int i = 0; i < kEpilogueWarps; ++i) mbar_init(&loaded[i], 1);
    *abort_s = 0;
    fence_mbar_init();
  }
  if (warp == 2) tc_alloc<CG>(tmem_base_s, S::kTmemCols);
  if (warp == 3 && lane < 8) {  // the maps come while the kernel before ends
    const CUtensorMap* map = lane < 2 ? &p.a[lane] : lane < 4 ? &p.b[lane - 2] : lane < 6 ? &p.src[lane - 4] : &p.out[lane - 6];
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
  }
  may_start_next();
  after_previous();
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_base_s;

  const int per = tiles_of(p, kBM * CG, BN), tiles = per * p.batch;
  const int width = SPLIT ? p.slices : CG, first = blockIdx.x / width, step = gridDim.x / width;
  // this CTA's part of the k axis
  const int blocks = p.kb * p.passes, from = SPLIT ? blocks * (int)slice / p.slices : 0;
  const int to = SPLIT ? blocks * ((int)slice + 1) / p.slices : blocks;

  // SPLIT: two meetings of the cluster.  After the first all MMAs have ended and the rings are free, after the second the
  // shares have arrived.  Every warp comes to both, whatever failed.
  const int share = SPLIT ? BN / p.slices : BN;
  const uint32_t ring = smem_u32(smem);
  bool first_met = false, met = false;
  const auto meet = [&] {
    __syncwarp();
    cluster_started_arrive();
    cluster_started_wait();
    first_met = true;
  };
  const auto part_of = [&](int from_slice, int q, int c) { return (from_slice * 4 + q) * (share / 16) + c / 16; };

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      long long issued = 0;
      bool ok = true;
      const bool low = p.passes == 3;
      for (int t = first; t < tiles && ok; t += step) {
        const OrthoTile tl = tile_at<kBM * CG, BN>(p, per, t);
        const int am = tl.m0 + (int)rank * kBM, bn = tl.n0 + (int)rank * S::kBNc;
        const int z = tl.z / p.pieces, k_from = (tl.z - z * p.pieces) * p.kb;
        for (int i = from, pass = from / p.kb, kb = from - pass * p.kb; i < to; ++i, kb + 1 < p.kb ? ++kb : (kb = 0, ++pass)) {
          const CUtensorMap *ma = &p.a[low && pass == 1], *mb = &p.b[low && pass == 0];
          if (!mbar_wait(&empty[s], ph ^ 1, fs, 111)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[s], S::kStageBytes * CG);
          const uint32_t bar = CG == 1 ? smem_u32(&full[s]) : map_to_rank(smem_u32(&full[s]), 0);
          const uint32_t sa = smem_u32(smem + s * S::kStageBytes), sb = sa + S::kABytes;
          const int k0 = (k_from + kb) * kBK;  // beyond the axis: zeros
          if constexpr (A_MN) {
#pragma unroll
            for (int j = 0; j < kBM / 64; ++j) load_tile<CG>(sa + j * 8192, ma, bar, am + 64 * j, k0, z);
          } else {
            load_tile<CG>(sa, ma, bar, k0, am, z);
          }
          if constexpr (B_MN) {
#pragma unroll
            for (int j = 0; j < S::kBNc / 64; ++j) load_tile<CG>(sb + j * 8192, mb, bar, bn + 64 * j, k0, z);
          } else {
            load_tile<CG>(sb, mb, bar, k0, bn, z);
          }
          ++issued;
          if (++s == S::kStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (rank == 0) {  // loads in flight land before this CTA leaves, whichever warp gave up (bounded)
        for (long long i = issued > S::kStages ? issued - S::kStages : 0; i < issued; ++i)
          for (int tries = 0; tries < 64 && !mbar_try_wait(&full[i % S::kStages], (i / S::kStages) & 1); ++tries) {
          }
      }
    }
  } else if (warp == 1 && rank == 0) {
    if (lane == 0) {
      constexpr uint32_t idesc = (1u << 4) | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                                 ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(kBM * CG >> 4) << 24);  // fp16, fp32 sums
      constexpr uint32_t a_step = (A_MN ? 2048 : 32) >> 4, b_step = (B_MN ? 2048 : 32) >> 4;
      int s = 0, buf = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        if (!mbar_wait(&acc_empty[buf], acc_ph ^ 1, fs, 112)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + buf * BN;
        for (int kb = from; kb < to; ++kb) {
          if (!mbar_wait(&full[s], ph, fs, 113)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * S::kStageBytes), sb = sa + S::kABytes;
          const uint64_t da = smem_desc(sa, A_MN ? 8192 : 16, 1024);
          const uint64_t db = smem_desc(sb, B_MN ? 8192 : 16, 1024);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) umma_ss<CG>(d, da + k * a_step, db + k * b_step, idesc, kb > from || k > 0);
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
      // the MMAs in flight end before the tensor memory is freed, also when only the epilogue gave up (bounded)
      umma_commit_local<CG>(drained);
      for (int tries = 0; tries < 64 && !mbar_try_wait(drained, 0); ++tries) {
      }
    }
  } else if (warp >= 4) {
    const int q = (warp - 4) & 3, turn = (warp - 4) >> 2;  // tensor memory lanes 32 q .. 32 q + 31
    // places: 0 and 3 stored from, 1 and 2 loaded to
    const uint32_t place = smem_u32(smem + S::kPlacesAt) + (warp - 4) * S::kPlaces * kPlace;
    uint64_t* mine = &loaded[warp - 4];
    uint32_t load_ph = 0, ph = 0;
    int buf = 0;
    bool ok = true, pending = false;  // pending: terms asked for and not yet waited for
    for (int t = first; t < tiles && ok; t += step) {
      const OrthoTile tl = tile_at<kBM * CG, BN>(p, per, t);
      const int row0 = tl.m0 + (int)rank * kBM + 32 * q, cols = min(BN, p.n - tl.n0);
      const bool rows = row0 < p.m;
      const bool mirror = STEP == STEP_POWER && p.symmetric && tl.n0 >= tl.m0 + kBM * CG;
      const auto ask = [&](int c) {
        pending = true;
        if (lane == 0) {
          mbar_arrive_expect_tx(mine, p.terms * kPlace);
          for (int i = 0; i < p.terms; ++i) tma_load_3d(place + (1 + i) * kPlace, &p.src[i], smem_u32(mine), tl.n0 + c, row0, tl.z);
        }
      };
      const bool asks = p.terms > 0 && rows;
      const int asked = (SPLIT ? slice * share : 0) + 32 * turn, end = SPLIT ? min(cols, (int)slice * share + share) : cols;
      if (asks && asked < end) ask(asked);
      ok = mbar_wait_warp(&acc_full[buf], ph, fs, 114);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(32 * q) << 16);
      if constexpr (SPLIT) {  // the others' shares of the columns to them, 16 columns a place, into their rings
        meet();
        for (int c = 16 * turn; c < BN; c += 32) {
          const uint32_t owner = c / share;
          if (owner == slice) continue;
          uint32_t r[16];
          tmem_take16(acc + c, r);
          uint4 v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
          put_remote(map_to_rank(ring + part_of(slice, q, c - owner * share) * kPlace, owner), lane, v);
        }
        cluster_sync_all();
        met = true;
      }
      for (int c = asked; c < end && rows; c += 64) {
        const int col = tl.n0 + c;
        float f[32];
        if (asks) {
          ok = mbar_wait_warp(mine, load_ph, fs, 115);
          if (!ok) break;
          load_ph ^= 1;
          pending = false;
          uint4 k0[4], k1[4];
          take_row(place + kPlace, lane, k0);
          if (p.terms == 2) take_row(place + 2 * kPlace, lane, k1);
          // every lane's reads come before the copy that overwrites them
          fence_async_proxy();
          __syncwarp();
          if (c + 64 < end) ask(c + 64);
          unpack_half(k0, f);
          if (p.terms == 2) {
            float lo[32];
            unpack_half(k1, lo);
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] += lo[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = 0.f;
        }
        uint32_t r[32];
        tmem_take32(acc + c, r);
        if constexpr (SPLIT) {
          for (int from_slice = 0; from_slice < p.slices; ++from_slice) {  // in the order of the slices
            if (from_slice == (int)slice) continue;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint4 v[4];
              take_row(ring + part_of(from_slice, q, c + 16 * half - (int)slice * share) * kPlace, lane, v);
              const uint32_t w[16] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w,
                                      v[2].x, v[2].y, v[2].z, v[2].w, v[3].x, v[3].y, v[3].z, v[3].w};
#pragma unroll
              for (int i = 0; i < 16; ++i)
                r[16 * half + i] = __float_as_uint(__uint_as_float(r[16 * half + i]) + __uint_as_float(w[i]));
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = fmaf(p.alpha, __uint_as_float(r[i]), p.beta * f[i]);
        uint4 v[4];
        if (STEP == STEP_UPDATE && p.last) {
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] *= p.scale;
          if (p.out_bf16) pack_row<__nv_bfloat16>(f, v);
          else pack_row<__half>(f, v);
        } else {
          pack_row<__half>(f, v);
        }
        if (lane == 0) bulk_wait_read<0>();  // the places have been read
        __syncwarp();
        put_row(place, lane, v);
        if (STEP == STEP_UPDATE && p.last && p.plain_c) {
          __syncwarp();
          store_plain(place, lane, p.c + ((long long)tl.z * p.m + row0) * p.ldc + col, p.ldc, min(32, p.m - row0),
                      min(32, cols - c));
          __syncwarp();
          continue;
        }
        if (mirror) put_column(place + 3 * kPlace, lane, f);
        const auto store = [&](const CUtensorMap* out, uint32_t from) {
          fence_async_proxy();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(out, from, col, row0, tl.z);
            if (mirror) tma_store_3d(out, place + 3 * kPlace, row0, col, tl.z);
            bulk_commit();
          }
        };
        store(&p.out[0], place);
        if (p.pair) {  // what hi leaves
          float hi[32];
          unpack_half(v, hi);
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] -= hi[i];
          pack_row<__half>(f, v);
          const uint32_t second = mirror ? place : place + 3 * kPlace;
          if (mirror) {  // both places are in use
            if (lane == 0) bulk_wait_read<0>();
            __syncwarp();
            put_column(place + 3 * kPlace, lane, f);
          }
          put_row(second, lane, v);
          store(&p.out[1], second);
        }
      }
      if (!ok) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster_relaxed(map_to_rank(smem_u32(&acc_empty[buf]), 0));
        else mbar_arrive_relaxed(&acc_empty[buf]);
      }
      buf ^= 1;
      if (buf == 0) ph ^= 1;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // the stores are done
    if (pending)  // after a wait that ran out: the load in flight lands before this CTA leaves (bounded)
      for (int tries = 0; tries < 64 && !mbar_try_wait(mine, load_ph); ++tries) {
      }
  }
  if constexpr (SPLIT) {
    if (!first_met) meet();
    if (!met) {
      __syncwarp();
      cluster_sync_all();
    }
  }
  __syncwarp();
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  if (warp == 2) tc_dealloc<CG>(tmem, S::kTmemCols);
}

// ------------------------------------------------------------------------- the norm and the first X
struct StartParams {
  const void* m;
  long long rows, cols, batch_stride, row_stride, pitch;
  double* part;  // [batch][parts]
  int parts;
  double eps;
  __half *hi, *lo;  // [batch][rows][pitch]
};
// Eight values of a row at once: WIDE, where all rows start on 16 bytes and end with a whole eight, in one load.
struct Eights {
  long long per, count;  // of a row, of the matrix
  bool narrow;           // 64-bit divisions cost more than the values
  __device__ __forceinline__ Eights(const StartParams& p) : per((p.cols + 7) / 8), count(p.rows * per), narrow(count < 1ll << 31) {}
  __device__ __forceinline__ void at(long long i, long long& row, long long& col) const {
    row = narrow ? (long long)((unsigned)i / (unsigned)per) : i / per;
    col = (i - row * per) * 8;
  }
};
template <class T, bool WIDE>
__device__ __forceinline__ Vec<T, 8> eight(const T* row, long long col, long long cols) {
  if constexpr (WIDE) return *reinterpret_cast<const Vec<T, 8>*>(row + col);
  Vec<T, 8> v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v.v[j] = col + j < cols ? row[col + j] : from_f32<T>(0.f);
  return v;
}
constexpr int kInFlight = 4;  // eights of a thread
// One block a part.  Sums of squares in 64 bits: squares of bf16 values leave the range of fp32, in which eight of them add
// up where none is large and some is not small.
template <class T, bool WIDE>
__global__ void __launch_bounds__(256) ortho_norm_kernel(const __grid_constant__ StartParams p) {
  may_start_next();
  after_previous();
  const long long z = blockIdx.y, step = (long long)gridDim.x * 256;
  const Eights all(p);
  const T* m = static_cast<const T*>(p.m) + z * p.batch_stride;
  double s = 0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all.count; i += kInFlight * step) {
    Vec<T, 8> v[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      if (i + k * step >= all.count) break;
      long long row, col;
      all.at(i + k * step, row, col);
      v[k] = eight<T, WIDE>(m + row * p.row_stride, col, p.cols);
    }
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      if (i + k * step >= all.count) break;
      float most = 0.f, near = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = to_f32<T>(v[k].v[j]);
        most = fmaxf(most, fabsf(d));
        near = fmaf(d, d, near);
      }
      if ((most >= 0x1p-50f && most <= 0x1p60f) || most == 0.f) {
        s += near;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const double d = to_f32<T>(v[k].v[j]);
          s = fma(d, d, s);
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __shared__ double red[8];
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 8; ++i) s += red[i];
  p.part[z * p.parts + blockIdx.x] = s;
}
// X_0 = M / (|M|_F + eps).  Rows of X have room for whole eights.
template <class T, bool WIDE>
__global__ void __launch_bounds__(256) ortho_start_kernel(const __grid_constant__ StartParams p) {
  may_start_next();
  after_previous();
  __shared__ double scale_s;
  const long long z = blockIdx.y, step = (long long)gridDim.x * 256;
  if (threadIdx.x < 32) {  // every block adds the parts up in the same order
    double s = 0;
    for (int i = threadIdx.x; i < p.parts; i += 32) s += p.part[z * p.parts + i];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) scale_s = kScaleX / (sqrt(s) + p.eps);
  }
  __syncthreads();
  const double scale = scale_s;
  const float small = (float)scale;
  const Eights all(p);
  const T* m = static_cast<const T*>(p.m) + z * p.batch_stride;
  const auto scaled = [&](auto times) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all.count; i += step) {
      long long row, col;
      all.at(i, row, col);
      const Vec<T, 8> v = eight<T, WIDE>(m + row * p.row_stride, col, p.cols);
      const long long at = (z * p.rows + row) * p.pitch + col;
      Vec<__half, 8> hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = times(to_f32<T>(v.v[j]));
        hi.v[j] = __float2half_rn(f);
        lo.v[j] = __float2half_rn(f - __half2float(hi.v[j]));
      }
      *reinterpret_cast<Vec<__half, 8>*>(p.hi + at) = hi;
      *reinterpret_cast<Vec<__half, 8>*>(p.lo + at) = lo;
    }
  };
  // norms at the ends of bf16: the product in 64 bits
  if (small >= 0x1p-120f && small <= 0x1p120f) scaled([&](float x) { return x * small; });
  else scaled([&](float x) { return (float)(x * scale); });
}

// A from its pieces (values in 22 bits), in their order.
struct JoinParams {
  const __half *hi, *lo;  // [batch][pieces][rows][pitch]
  __half *to_hi, *to_lo;  // [batch][rows][pitch]; to_lo: null where one value is enough
  long long eights;       // of a matrix
  int pieces;
};
__global__ void __launch_bounds__(256) ortho_join_kernel(const __grid_constant__ JoinParams p) {
  may_start_next();
  after_previous();
  using Eight = Vec<__half, 8>;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.eights) return;
  const long long z = blockIdx.y;
  const Eight* hi = reinterpret_cast<const Eight*>(p.hi) + z * p.pieces * p.eights + i;
  const Eight* lo = reinterpret_cast<const Eight*>(p.lo) + z * p.pieces * p.eights + i;
  float sum[8] = {};
#pragma unroll 4
  for (int k = 0; k < p.pieces; ++k) {
    const Eight a = hi[k * p.eights], b = lo[k * p.eights];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] += __half2float(a.v[j]) + __half2float(b.v[j]);
  }
  Eight a, b;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    a.v[j] = __float2half_rn(sum[j]);
    b.v[j] = __float2half_rn(sum[j] - __half2float(a.v[j]));
  }
  reinterpret_cast<Eight*>(p.to_hi)[z * p.eights + i] = a;
  if (p.to_lo) reinterpret_cast<Eight*>(p.to_lo)[z * p.eights + i] = b;
}

// ------------------------------------------------------------------------ small matrices in one launch
struct HeldParams {
  const uint16_t* m;
  uint16_t* out;
  long long batch_stride, si, sj;  // X[i][j] = m[i si + j sj]: X is the wide one of the matrix and its transpose
  long long out_batch, oi, oj;
  int small, large, steps;
  int bf16;         // type of the matrix and the result
  int wide_loads, wide_stores;  // 16 bytes at a time along j
  int precise, all; // steps with operands of 22 bits in the largest product; in all products
  float a, a_scale, b_acc, b_src, inverse_b;
  double eps;
  int* ctrl;
  unsigned long long timeout_ns;
};

// Operands in shared memory: blocks of 64 columns, rows of 128 bytes, 16-byte pieces at j ^ (row & 7).
//   CG = 1: X hi, X lo (256 columns each), A or B hi, lo (128 columns)
//   CG = 2: this CTA's 128 rows of X, its 128 columns of X (of all rows), its rows of A or B (256 columns)
template <int CG>
struct HeldShape {
  static constexpr int kX = 65536;
  static constexpr int kSecond = kX;       // X lo, or the columns
  static constexpr int kSquare = 2 * kX;   // A, then B
  static constexpr int kSquareLo = kSquare + 32768;
  static constexpr int kRest = 3 * kX;
  static constexpr int kSmem = kRest + 512 + 1024;
  static constexpr int kSquareCols = 128 * CG;
};
constexpr int kHeldThreads = 288;

__device__ __forceinline__ uint32_t piece_at(uint32_t base, int rows, int row, int col) {  // of 8 columns from col on
  return base + (col >> 6) * rows * 128 + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4);
}
__device__ __forceinline__ void put_piece(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 take_piece(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

template <int CG>
__global__ void __launch_bounds__(kHeldThreads, 1) ortho_held_kernel(const __grid_constant__ HeldParams p) {
  using S = HeldShape<CG>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* done = reinterpret_cast<uint64_t*>(smem + S::kRest);
  double* sums = reinterpret_cast<double*>(done + 1);  // of the warps, then of the CTAs
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(sums + 10);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_base_s + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 1 ? 0 : cta_rank_in_cluster();
  const FailState fs{p.ctrl, abort_s, 0, p.timeout_ns, true};
  if (threadIdx.x == 0) {
    mbar_init(done, 1);
    *abort_s = 0;
    fence_mbar_init();
  }
  if (warp == 8) tc_alloc<CG>(tmem_base_s, 512);
  cluster_started_arrive();
  may_start_next();
  after_previous();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_started_wait();
  const uint32_t tmem = *tmem_base_s, base = smem_u32(smem);
  // a phase's results to the next phase's MMAs, in both CTAs
  const auto meet = [&] {
    tc_fence_before();
    asm volatile("fence.proxy.async;" ::: "memory");
    __syncwarp();
    cluster_sync_all();
    asm volatile("fence.proxy.async;" ::: "memory");
    tc_fence_after();
  };

  const int q = warp & 3, half = warp >> 2, row = 32 * q + lane, i = (int)rank * 128 + row;  // warps 0 to 7: a lane a row of X
  const uint32_t acc = tmem + ((uint32_t)(32 * q) << 16), held = acc + 256;  // the accumulator, X in fp32
  const uint16_t* m = p.m + (blockIdx.x / CG) * p.batch_stride;
  const auto value = [&](uint32_t bits) {
    return p.bf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits));
  };
  const auto keep = [&](int c, const float (&f)[32]) {  // 32 columns of X in fp32
    uint32_t r[16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(f[16 * h + j]);
      tmem_st16(held + c + 16 * h, r);
    }
    tc_wait_st();
  };
  // the same as operands of the next products
  const auto spread = [&](int c, float (&f)[32], bool low) {
    uint4 v[4];
    pack_row<__half>(f, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) put_piece(piece_at(base, 128, row, c + 8 * j), v[j]);
    if constexpr (CG == 2) {
      const uint32_t to = map_to_rank(base + S::kSecond, c >> 7);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at(to, 256, i, (c & 127) + 8 * j)), "r"(v[j].x),
                     "r"(v[j].y), "r"(v[j].z), "r"(v[j].w)
                     : "memory");
    } else if (low) {
      float hi[32];
      unpack_half(v, hi);
#pragma unroll
      for (int j = 0; j < 32; ++j) f[j] -= hi[j];
      pack_row<__half>(f, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) put_piece(piece_at(base + S::kSecond, 128, row, c + 8 * j), v[j]);
    }
  };
  const auto precise_at = [&](int k) { return k + p.precise >= p.steps; };

  double sum = 0;
  if (warp < 8) {
    const int end = min(p.large, 128 * half + 128);
    uint4 v[4][4];  // all loads come first
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int c = 128 * half + 32 * t;
      if (p.wide_loads && i < p.small && c + 32 <= p.large) {
        const uint4* from = reinterpret_cast<const uint4*>(m + i * p.si + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[t][j] = from[j];
      } else if (c < end) {
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int at = c + 2 * j;
          const uint32_t low = i < p.small && at < p.large ? m[i * p.si + at * p.sj] : 0;
          w[j] = low | (uint32_t)(i < p.small && at + 1 < p.large ? m[i * p.si + (at + 1) * p.sj] : 0) << 16;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[t][j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int c = 128 * half + 32 * t;
      if (c >= end) break;
      float f[32];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w[4] = {v[t][j].x, v[t][j].y, v[t][j].z, v[t][j].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) f[8 * j + 2 * k] = value(w[k] & 0xffffu), f[8 * j + 2 * k + 1] = value(w[k] >> 16);
      }
      // squares of bf16 values leave the range of fp32: 32 of them add up in it where none is large and some is not small
      float most = 0.f, near = 0.f;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        most = fmaxf(most, fabsf(f[j]));
        near = fmaf(f[j], f[j], near);
      }
      if ((most >= 0x1p-50f && most <= 0x1p60f) || most == 0.f) {
        sum += near;
      } else {
#pragma unroll 1
        for (int j = 0; j < 32; ++j) {
          if (i >= p.small || c + j >= p.large) break;
          const double d = value(m[i * p.si + (c + j) * p.sj]);
          sum = fma(d, d, sum);
        }
      }
      keep(c, f);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[warp] = sum;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
    for (int w = 0; w < 8; ++w) sum += sums[w];
    for (uint32_t r = 0; r < CG; ++r)
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(map_to_rank(smem_u32(sums + 8 + rank), r)), "d"(sum) : "memory");
  }
  meet();
  if (warp < 8) {
    const double scale = kScaleX / (sqrt(CG == 2 ? sums[8] + sums[9] : sums[8]) + p.eps);
    const float one = (float)scale;
    const auto scaled = [&](auto times) {
#pragma unroll 1
      for (int c = 128 * half; c < min(p.large, 128 * half + 128); c += 32) {
        uint32_t r[32];
        float f[32];
        tmem_take32(held + c, r);
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] = times(__uint_as_float(r[j]));
        keep(c, f);
        spread(c, f, precise_at(0));
      }
    };
    if (one >= 0x1p-120f && one <= 0x1p120f) scaled([&](float x) { return x * one; });
    else scaled([&](float x) { return (float)(x * scale); });
  }
  meet();

  bool ok = true;
  uint32_t ph = 0, issued = 0;  // issued: the parity of the last phase whose MMAs were issued
  // D = a b^T over `blocks` of 16 k; b MN-major for the last product
  const auto multiply = [&](uint32_t a, uint32_t b, int blocks, bool mn, int n, bool more) {
    const uint32_t idesc = (1u << 4) | ((mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 * CG >> 4) << 24);
    // the one thread that issues them: few operations for each
    uint64_t da = smem_desc(a, 16, 1024), db = mn ? smem_desc(b, CG == 2 ? 32768 : 16384, 1024) : smem_desc(b, 16, 1024);
    const uint32_t step = mn ? 128 : 2;
    for (int k = 0; k < blocks; k += 4, da += 1024, db += mn ? 512 : 1024) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k + j < blocks) umma_ss<CG>(tmem, da + 2 * j, db + step * j, idesc, more || k + j > 0);
    }
  };
  const bool issues = warp == 8 && lane == 0 && rank == 0;
  const uint32_t x = base, x_lo = base + S::kSecond, columns = CG == 2 ? base + S::kSecond : base;
  const uint32_t square = base + S::kSquare, square_lo = base + S::kSquareLo;
  const int small_blocks = (p.small + 15) / 16, large_blocks = (p.large + 15) / 16;
  for (int k = 0; k < p.steps; ++k) {
    const bool last = k + 1 == p.steps, precise = CG == 1 && precise_at(k), all = precise && p.all;
    for (int phase = 0; phase < 3; ++phase) {
      const bool three = phase < 2 ? all : precise;
      if (issues && ok) {  // after a wait that ran out no more: one phase at most is in flight at the end
        const uint32_t a = phase == 0 ? x : square, b = phase == 0 ? x : phase == 1 ? square : columns;
        const int blocks = phase == 0 ? large_blocks : small_blocks, n = phase < 2 ? S::kSquareCols : 256;
        multiply(a, b, blocks, phase == 2, n, false);
        if (three) {
          const uint32_t al = phase == 0 ? x_lo : square_lo, bl = phase == 1 ? square_lo : x_lo;
          multiply(a, bl, blocks, phase == 2, n, true);
          multiply(al, b, blocks, phase == 2, n, true);
        }
        tc_commit<CG>(done);
        issued = ph;
      }
      __syncwarp();
      if (ok) ok = mbar_wait_warp(done, ph, fs, 121 + phase);
      ph ^= 1;
      tc_fence_after();
      if (warp < 8 && ok) {
        const int width = phase < 2 ? S::kSquareCols / 2 : 128, from = half * width;
        const int to = min(from + width, phase < 2 ? p.small : p.large);
        for (int c = from; c < to; c += 32) {
          uint32_t r[32];
          float f[32];
          tmem_take32(acc + c, r);
          if (phase < 2) {
            if (phase == 0) {
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j] = p.a_scale * __uint_as_float(r[j]);
            } else {
              uint4 v[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) v[j] = take_piece(piece_at(square, 128, row, c + 8 * j));
              unpack_half(v, f);
              if (all) {
                float lo[32];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = take_piece(piece_at(square_lo, 128, row, c + 8 * j));
                unpack_half(v, lo);
#pragma unroll
                for (int j = 0; j < 32; ++j) f[j] += lo[j];
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j] = fmaf(p.b_acc, __uint_as_float(r[j]), p.b_src * f[j]);
            }
            uint4 v[4];
            pack_row<__half>(f, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) put_piece(piece_at(square, 128, row, c + 8 * j), v[j]);
            if (phase == 0 ? all : precise) {
              float hi[32];
              unpack_half(v, hi);
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j] -= hi[j];
              pack_row<__half>(f, v);
#pragma unroll
              for (int j = 0; j < 4; ++j) put_piece(piece_at(square_lo, 128, row, c + 8 * j), v[j]);
            }
          } else {
            uint32_t h[32];
            tmem_take32(held + c, h);
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = fmaf(p.inverse_b, __uint_as_float(r[j]), p.a * __uint_as_float(h[j]));
            if (!last) {
              keep(c, f);
              spread(c, f, precise_at(k + 1));
            } else if (i < p.small) {
              uint16_t* to_row = p.out + (blockIdx.x / CG) * p.out_batch + i * p.oi;
              uint4 v[4];
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j] *= 1.f / kScaleX;
              if (p.bf16) pack_row<__nv_bfloat16>(f, v);
              else pack_row<__half>(f, v);
              const uint32_t w[16] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w,
                                      v[2].x, v[2].y, v[2].z, v[2].w, v[3].x, v[3].y, v[3].z, v[3].w};
              if (p.wide_stores && c + 32 <= p.large) {
#pragma unroll
                for (int j = 0; j < 4; ++j) reinterpret_cast<uint4*>(to_row + c)[j] = v[j];
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (c + j < p.large) to_row[(c + j) * p.oj] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
              }
            }
          }
        }
      }
      meet();
    }
  }
  // after a wait that ran out: the MMAs in flight end before the tensor memory is freed (bounded)
  if (issues && !ok)
    for (int tries = 0; tries < 64 && !mbar_try_wait(done, issued); ++tries) {
    }
  __syncwarp();
  cluster_sync_all();
  if (warp == 8) tc_dealloc<CG>(tmem, 512);
}

// --------------------------------------------------------------------------------------- host side
int sm_count() {
  static std::atomic<int> kept[kMaxDevices];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 148;
  n = kept[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    kept[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static std::atomic<EncodeFn> kept{nullptr};
  EncodeFn f = kept.load(std::memory_order_acquire);
  if (!f) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    f = reinterpret_cast<EncodeFn>(p);
    kept.store(f, std::memory_order_release);
  }
  return f;
}

// A stack of 16-bit matrices, rows `ld` values apart.
struct Stack {
  const void* p;
  long long rows, cols, ld, batch;
  long long apart;  // values between matrices
};
// Boxes of `box_cols` x `box_rows` of one matrix; outside reads as zero and is not written.
bool encode(CUtensorMap* map, const Stack& m, CUtensorMapDataType type, int box_cols, int box_rows) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, (cuuint64_t)m.batch};
  const cuuint64_t strides[2] = {(cuuint64_t)m.ld * 2, (cuuint64_t)m.apart * 2};
  const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  const cuuint32_t one[3] = {1, 1, 1};
  return fn(map, type, 3, const_cast<void*>(m.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool encode_operand(CUtensorMap* map, const Stack& m, bool mn, int rows) {
  return encode(map, m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 64, mn ? 64 : rows);
}
bool encode_places(CUtensorMap* map, const Stack& m, bool bf16 = false) {
  return encode(map, m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 32, 32);
}

template <int CG, int BN, bool A_MN, bool B_MN, int STEP, bool SPLIT = false>
int32_t launch(OrthoParams& p, const Stack (&a)[2], const Stack (&b)[2], cudaStream_t s) {
  using S = OrthoShape<CG, BN>;
  auto* kernel = ortho_kernel<CG, BN, A_MN, B_MN, STEP, SPLIT>;
  static_assert(!SPLIT || (CG == 1 && BN == 128 && S::kStages * S::kStageBytes >= 32 * kPlace), "the ring holds a tile in fp32");
  static std::atomic<uint64_t> ready{0};  // a bit for each device whose shared-memory limit is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return NCA_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess)
      return launch_status() == NCA_OK ? NCA_ERR_CUDA : NCA_ERR_DEVICE;
    ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  for (int i = 0; i < (p.passes == 1 ? 1 : 2); ++i)
    if (!encode_operand(&p.a[i], a[i], A_MN, kBM) || !encode_operand(&p.b[i], b[i], B_MN, S::kBNc)) return NCA_ERR_CUDA;
  p.m_tiles = (int)ceil_div(p.m, kBM * CG);
  // symmetric: whole blocks on the diagonal, the last of whose tiles may be empty
  p.n_tiles = p.symmetric ? p.m_tiles * (kBM * CG / BN) : (int)ceil_div(p.n, BN);
  if ((long long)p.m_tiles * p.n_tiles > (1ll << 31) - 1024) return NCA_ERR_UNSUPPORTED;
  const long long tiles = (long long)tiles_of(p, kBM * CG, BN) * p.batch;
  if (tiles > (1ll << 31) - 1024) return NCA_ERR_UNSUPPORTED;
  if (SPLIT) return launch_after(kernel, dim3((unsigned)(tiles * p.slices)), dim3(kGemmThreads), S::kSmem, s, p.slices, p);
  const long long room = sm_count() / CG;
  return launch_after(kernel, dim3((unsigned)((tiles < room ? tiles : room) * CG)), dim3(kGemmThreads), S::kSmem, s, CG, p);
}

// Clusters of 2 and 4 leave some multiprocessors of a processing cluster out: the share in percent that runs at once.
constexpr int kClusters2 = 88, kClusters4 = 80;

// The tile of a product by the cost of its waves, as the gated block's: a k block costs a 256 x 256 tile of a pair of
// multiprocessors 0.28 us, a 256 x 128 tile 0.24 and a 128 x 128 tile of one 0.25, a wave 6, 5 or 4 us besides (epilogue, ramps); CTAs
// that share the k axis 2 us more.
template <bool A_MN, bool B_MN, int STEP>
int32_t product(OrthoParams& p, const Stack (&a)[2], const Stack (&b)[2], cudaStream_t s) {
  static const struct {
    int cg, bn;
    double us, wave;
  } kinds[] = {{2, 256, 0.28, 6.0}, {2, 128, 0.24, 5.0}, {1, 128, 0.25, 4.0}};
  const long long blocks = (long long)p.kb * p.passes;
  int best = 0, slices = 1;
  double least = 1e30;
  for (int i = 0; i < 3; ++i) {
    const long long tm = 128 * kinds[i].cg, mt = ceil_div(p.m, tm);
    long long tiles = mt * ceil_div(p.n, kinds[i].bn);
    if (p.symmetric) tiles = (tm / kinds[i].bn) * (mt * (mt + 1) / 2);
    tiles *= p.batch;
    for (int z = 1; z <= (kinds[i].cg == 1 ? 4 : 1); z *= 2) {
      if (z > 1 && (tiles * z > sm_count() * (z == 2 ? kClusters2 : kClusters4) / 100 || blocks < 4 * z)) break;
      const double us = (double)ceil_div(tiles * z, sm_count() / kinds[i].cg) * (ceil_div(blocks, z) * kinds[i].us + kinds[i].wave) +
                        (z > 1 ? 2.0 : 0.0);
      if (us < least) {
        least = us;
        best = i;
        slices = z;
      }
    }
  }
  p.slices = slices;
  if (slices > 1) return launch<1, 128, A_MN, B_MN, STEP, true>(p, a, b, s);
  if (best == 0) return launch<2, 256, A_MN, B_MN, STEP>(p, a, b, s);
  return best == 1 ? launch<2, 128, A_MN, B_MN, STEP>(p, a, b, s) : launch<1, 128, A_MN, B_MN, STEP>(p, a, b, s);
}

int32_t check_desc(const NcaOrthoDesc* d) {
  if (!d || d->batch < 0 || d->rows < 0 || d->cols < 0 || d->steps < 1) return NCA_ERR_INVALID;
  if (!(d->eps >= 0) || !std::isfinite(d->eps)) return NCA_ERR_INVALID;
  for (int i = 0; i < 3; ++i)
    if (!std::isfinite(d->coefficients[i])) return NCA_ERR_INVALID;
  if (d->dtype != NCA_BF16 && d->dtype != NCA_F16) return dtype_ok(d->dtype) ? NCA_ERR_UNSUPPORTED : NCA_ERR_INVALID;
  const long long most = 1ll << 30;
  if (d->rows > most || d->cols > most || d->batch > most) return NCA_ERR_UNSUPPORTED;
  if (d->steps > 1000 || d->batch > 65535) return NCA_ERR_UNSUPPORTED;
  // the largest singular value after every step, from [0, 1]: x (a + b x^2 + c x^4) is largest at the end of the range
  // or where a + 3 b x^2 + 5 c x^4 = 0
  const double a = d->coefficients[0], b = d->coefficients[1], c = d->coefficients[2];
  const auto image = [&](double x) { return std::fabs(x * (a + x * x * (b + x * x * c))); };
  const double root = std::sqrt(std::max(0.0, 9 * b * b - 20 * a * c));
  const double inner[3] = {(-3 * b + root) / (10 * c), (-3 * b - root) / (10 * c), -a / (3 * b)};  // x^2; the last for c = 0
  double range = 1.0;
  for (int k = 0; k < d->steps; ++k) {
    double most = image(range);
    for (double x2 : inner)
      if (x2 > 0 && x2 < range * range) most = std::max(most, image(std::sqrt(x2)));
    if (!(most <= 2.0)) return NCA_ERR_UNSUPPORTED;
    range = most;
  }
  return NCA_OK;
}

// Whether a step with operands of 22 bits has them in all three products.
constexpr int64_t kFewRows = 64;
constexpr int kFewSteps = 2;
bool few_rows(const NcaOrthoDesc& d) { return std::min(d.rows, d.cols) < kFewRows; }
bool all_products(const NcaOrthoDesc& d) { return d.dtype == NCA_F16 || few_rows(d); }
// How many of the last steps take operands of 22 bits.
int precise_steps(const NcaOrthoDesc& d) {
  if (few_rows(d) || (d.dtype == NCA_F16 && d.steps <= kFewSteps)) return d.steps;
  const double small = (double)std::min(d.rows, d.cols), a = std::fabs(d.coefficients[0]);
  const double arrived = a > 1.05 ? std::max(0.0, d.steps - 0.5 * std::log(small) / std::log(a)) : d.steps;
  if (d.dtype == NCA_F16) return (int)std::min<double>(d.steps, std::ceil(arrived));
  return arrived <= 3.0 ? 0 : (int)std::ceil(arrived - 1.2);
}

// CTAs that hold a matrix in one launch; 0: it goes through the products.
int held_by(const NcaOrthoDesc& d) {
  const int64_t small = std::min(d.rows, d.cols), large = std::max(d.rows, d.cols);
  if (large > 256) return 0;
  return small <= 128 ? 1 : precise_steps(d) == 0 ? 2 : 0;
}

// Blocks of the k axis that one product adds up.  The accumulators lose 7.6e-8 of a sum of equal signs with every 16 terms, 16 %
// of 2^25; A over a longer axis is brought together from pieces of it (8e-5 at most), in fp32 from 22 bits.
constexpr long long kLongest = 16384 / kBK;
// Pieces of the long axis: also where A has so few tiles that its clusters leave much of the GPU idle, for as many CTAs as there
// are, where what they save (a block of the axis takes 0.25 us) is more than the second kernel's 4 us (64 x 16384, 5 steps:
// bf16 178 to 127 us, fp16 305 to 195; 2730 x 1001 fp16 291 to 274).
long long pieces_of(const NcaOrthoDesc& d, int passes) {
  const long long small = std::min(d.rows, d.cols), blocks = ceil_div(std::max(d.rows, d.cols), kBK);
  const long long side = ceil_div(small, 128), tiles = side * (side + 1) / 2 * d.batch;
  const long long want = std::min(sm_count() / std::max(tiles, 1ll), blocks * passes / 8);
  const int slices = tiles * 4 <= kClusters4 * sm_count() / 100 ? 4 : tiles * 2 <= kClusters2 * sm_count() / 100 ? 2 : 1;
  const bool worth = want > slices && 0.25 * blocks * passes * (1.0 / slices - 1.0 / want) > 4.0;
  const long long pieces = std::max(worth ? want : 1, ceil_div(blocks, kLongest));
  return ceil_div(blocks, ceil_div(blocks, pieces));  // no empty ones
}

struct Plan {
  long long small, large, pitch, small_pitch;
  bool tall;
  size_t x[2][2], a[2], b[2], pieces[2], part, total;  // x[buffer][hi, lo]; a, b, pieces: hi, lo
  int parts;
};
Plan plan_of(const NcaOrthoDesc& d) {
  Plan p{};
  p.tall = d.rows > d.cols;
  p.small = std::min(d.rows, d.cols);
  p.large = std::max(d.rows, d.cols);
  p.pitch = pad64(d.cols);
  p.small_pitch = pad64(p.small);
  size_t at = 0;
  const size_t x = align256((size_t)d.batch * d.rows * p.pitch * 2), a = align256((size_t)d.batch * p.small * p.small_pitch * 2);
  for (auto& buffer : p.x)
    for (size_t& part : buffer) {
      part = at;
      at += x;
    }
  for (int i = 0; i < 2; ++i) {
    p.a[i] = at;
    p.b[i] = at + a;
    if (i == 0 || precise_steps(d) > 0) at += 2 * a;
  }
  const long long pieces = std::max(pieces_of(d, 1), pieces_of(d, 3));
  for (size_t& part : p.pieces) {
    part = at;
    if (pieces > 1) at += align256((size_t)d.batch * pieces * p.small * p.small_pitch * 2);
  }
  p.part = at;
  p.parts = (int)std::max<long long>(1, std::min<long long>(ceil_div(d.rows * d.cols, 4096), ceil_div(592, d.batch ? d.batch : 1)));
  at += align256((size_t)d.batch * p.parts * sizeof(double));
  p.total = at + 256;
  return p;
}

template <class T, bool WIDE>
int32_t start(const StartParams& p, long long batch, cudaStream_t s) {
  if (batch > 65535) return NCA_ERR_UNSUPPORTED;
  NCA_TRY(launch_after(ortho_norm_kernel<T, WIDE>, dim3(p.parts, (unsigned)batch), dim3(256), 0, s, 1, p));
  const long long blocks = std::min<long long>(ceil_div(p.rows * ceil_div(p.cols, 8), 512), 148 * 8);
  return launch_after(ortho_start_kernel<T, WIDE>, dim3((unsigned)blocks, (unsigned)batch), dim3(256), 0, s, 1, p);
}

// |B| <= 4 |b| + 16 |c|: times the largest power of two, 2^10 at most, that leaves it below 2^15
double scale_of_b(const NcaOrthoDesc& d) {
  double scale = kScaleA;
  while (scale * (4 * std::fabs(d.coefficients[1]) + 16 * std::fabs(d.coefficients[2])) > 32768.0) scale /= 2;
  return scale;
}

template <int CG>
int32_t held_launch(const HeldParams& p, long long batch, cudaStream_t s) {
  auto* kernel = ortho_held_kernel<CG>;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return NCA_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, HeldShape<CG>::kSmem) != cudaSuccess)
      return launch_status() == NCA_OK ? NCA_ERR_CUDA : NCA_ERR_DEVICE;
    ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  return launch_after(kernel, dim3((unsigned)(batch * CG)), dim3(kHeldThreads), HeldShape<CG>::kSmem, s, CG, p);
}
int32_t held(const NcaOrthoDesc& d, const void* matrix, void* out, int32_t* ctrl, int32_t timeout_ms, cudaStream_t s) {
  HeldParams p{};
  const bool tall = d.rows > d.cols;
  p.m = static_cast<const uint16_t*>(matrix);
  p.out = static_cast<uint16_t*>(out);
  p.batch_stride = d.stride[0];
  p.si = tall ? 1 : d.stride[1];
  p.sj = tall ? d.stride[1] : 1;
  p.out_batch = d.rows * d.cols;
  p.oi = tall ? 1 : d.cols;
  p.oj = tall ? d.cols : 1;
  p.small = (int)std::min(d.rows, d.cols);
  p.large = (int)std::max(d.rows, d.cols);
  p.steps = d.steps;
  p.bf16 = d.dtype == NCA_BF16;
  p.wide_loads = !tall && (d.rows == 1 || d.stride[1] % 8 == 0) && (d.batch == 1 || d.stride[0] % 8 == 0) &&
                 reinterpret_cast<uintptr_t>(matrix) % 16 == 0;
  p.wide_stores = !tall && d.cols % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  p.precise = precise_steps(d);
  p.all = all_products(d);
  const double scale_b = scale_of_b(d);
  p.a = (float)d.coefficients[0];
  p.a_scale = kScaleA / (kScaleX * kScaleX);
  p.b_acc = (float)(d.coefficients[2] * scale_b / ((double)kScaleA * kScaleA));
  p.b_src = (float)(d.coefficients[1] * scale_b / kScaleA);
  p.inverse_b = (float)(1.0 / scale_b);
  p.eps = d.eps;
  p.ctrl = ctrl;
  p.timeout_ns = (unsigned long long)(timeout_ms > 0 ? timeout_ms : 10000) * 1000000ull;
  return held_by(d) == 1 ? held_launch<1>(p, d.batch, s) : held_launch<2>(p, d.batch, s);
}

}  // namespace

extern "C" {

int32_t nca_b200_orthogonalize_workspace(const NcaOrthoDesc* d, size_t* bytes) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK || !bytes) return st != NCA_OK ? st : NCA_ERR_INVALID;
  *bytes = d->batch && d->rows && d->cols && !held_by(*d) ? plan_of(*d).total : 0;
  return NCA_OK;
}

int32_t nca_b200_orthogonalize(const NcaOrthoDesc* d, const void* matrix, void* out, void* workspace,
                               size_t workspace_bytes, int32_t* ctrl, int32_t timeout_ms, void* stream) {
  NCA_TRY(check_desc(d));
  if (d->batch == 0 || d->rows == 0 || d->cols == 0) return NCA_OK;
  if (!matrix || !out || !ctrl) return NCA_ERR_INVALID;
  if (held_by(*d)) return held(*d, matrix, out, ctrl, timeout_ms, static_cast<cudaStream_t>(stream));
  const Plan pl = plan_of(*d);
  if (!workspace || workspace_bytes < pl.total) return NCA_ERR_SCRATCH;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~(uintptr_t)255);
  const auto x_of = [&](int buffer, int part) { return Stack{ws + pl.x[buffer][part], d->rows, d->cols, pl.pitch, d->batch, d->rows * pl.pitch}; };
  const auto square = [&](size_t at) { return Stack{ws + at, pl.small, pl.small, pl.small_pitch, d->batch, pl.small * pl.small_pitch}; };
  const Stack a_of[2] = {square(pl.a[0]), square(pl.a[1])}, b_of[2] = {square(pl.b[0]), square(pl.b[1])};

  StartParams sp{};
  sp.m = matrix;
  sp.rows = d->rows;
  sp.cols = d->cols;
  sp.batch_stride = d->stride[0];
  sp.row_stride = d->stride[1];
  sp.pitch = pl.pitch;
  sp.part = reinterpret_cast<double*>(ws + pl.part);
  sp.parts = pl.parts;
  sp.eps = d->eps;
  sp.hi = reinterpret_cast<__half*>(ws + pl.x[0][0]);
  sp.lo = reinterpret_cast<__half*>(ws + pl.x[0][1]);
  const bool wide = d->cols % 8 == 0 && (d->rows == 1 || d->stride[1] % 8 == 0) && (d->batch == 1 || d->stride[0] % 8 == 0) &&
                    reinterpret_cast<uintptr_t>(matrix) % 16 == 0;
  if (d->dtype == NCA_BF16)
    NCA_TRY((wide ? start<__nv_bfloat16, true>(sp, d->batch, s) : start<__nv_bfloat16, false>(sp, d->batch, s)));
  else
    NCA_TRY((wide ? start<__half, true>(sp, d->batch, s) : start<__half, false>(sp, d->batch, s)));

  const double c0 = d->coefficients[0], c1 = d->coefficients[1], c2 = d->coefficients[2];
  const double scale_b = scale_of_b(*d);
  OrthoParams p{};
  p.batch = (int)d->batch;
  p.ctrl = ctrl;
  p.timeout_ns = (unsigned long long)(timeout_ms > 0 ? timeout_ms : 10000) * 1000000ull;
  p.out_bf16 = d->dtype == NCA_BF16;
  for (int k = 0; k < d->steps; ++k) {
    const Stack x[2] = {x_of(k & 1, 0), x_of(k & 1, 1)};
    const bool last = k + 1 == d->steps, precise = k + precise_steps(*d) >= d->steps, all = precise && all_products(*d);
    p.passes = all ? 3 : 1;
    p.m = p.n = (int)pl.small;
    p.symmetric = 1;
    p.last = 0;
    p.terms = 0;
    p.alpha = kScaleA / (kScaleX * kScaleX);
    p.beta = 0.f;
    const long long blocks = ceil_div(pl.large, kBK);
    p.pieces = (int)pieces_of(*d, p.passes);
    p.kb = (int)ceil_div(blocks, p.pieces);
    p.batch = (int)d->batch * p.pieces;
    p.pair = all || p.pieces > 1;
    for (int i = 0; i <= p.pair; ++i) {
      Stack to = p.pieces > 1 ? square(pl.pieces[i]) : a_of[i];
      to.batch = p.batch;
      if (!encode_places(&p.out[i], to)) return NCA_ERR_CUDA;
    }
    NCA_TRY((pl.tall ? product<true, true, STEP_POWER>(p, x, x, s) : product<false, false, STEP_POWER>(p, x, x, s)));
    if (p.pieces > 1) {
      JoinParams j{};
      j.hi = reinterpret_cast<const __half*>(ws + pl.pieces[0]);
      j.lo = reinterpret_cast<const __half*>(ws + pl.pieces[1]);
      j.to_hi = reinterpret_cast<__half*>(ws + pl.a[0]);
      j.to_lo = all ? reinterpret_cast<__half*>(ws + pl.a[1]) : nullptr;
      j.eights = pl.small * pl.small_pitch / 8;
      j.pieces = p.pieces;
      NCA_TRY(launch_after(ortho_join_kernel, dim3((unsigned)ceil_div(j.eights, 256), (unsigned)d->batch), dim3(256), 0, s, 1, j));
    }
    p.pieces = 1;
    p.batch = (int)d->batch;

    p.kb = (int)ceil_div(pl.small, kBK);
    p.terms = 1 + all;
    p.pair = precise;
    p.alpha = (float)(c2 * scale_b / ((double)kScaleA * kScaleA));
    p.beta = (float)(c1 * scale_b / kScaleA);
    for (int i = 0; i < 2; ++i)
      if ((i < p.terms && !encode_places(&p.src[i], a_of[i])) || (i <= p.pair && !encode_places(&p.out[i], b_of[i])))
        return NCA_ERR_CUDA;
    NCA_TRY((product<false, false, STEP_POWER>(p, a_of, a_of, s)));

    p.m = (int)d->rows;
    p.n = (int)d->cols;
    p.symmetric = 0;
    p.passes = precise ? 3 : 1;
    p.terms = 2;
    p.pair = !last;
    p.last = last;
    p.alpha = (float)(1.0 / scale_b);
    p.beta = (float)c0;
    p.scale = 1.f / kScaleX;
    p.c = static_cast<uint16_t*>(out);
    p.ldc = d->cols;
    p.plain_c = d->cols % 8 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0;
    if (!encode_places(&p.src[0], x[0]) || !encode_places(&p.src[1], x[1])) return NCA_ERR_CUDA;
    if (!last) {
      if (!encode_places(&p.out[0], x_of(~k & 1, 0)) || !encode_places(&p.out[1], x_of(~k & 1, 1))) return NCA_ERR_CUDA;
    } else if (!p.plain_c && !encode_places(&p.out[0], Stack{out, d->rows, d->cols, d->cols, d->batch, d->rows * d->cols}, p.out_bf16)) {
      return NCA_ERR_CUDA;
    }
    NCA_TRY((pl.tall ? product<false, false, STEP_UPDATE>(p, x, b_of, s) : product<false, true, STEP_UPDATE>(p, b_of, x, s)));
  }
  return NCA_OK;
}

}  // extern "C"
