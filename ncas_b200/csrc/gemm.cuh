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
// over pieces of 32 columns).  What they store and load moves by TMA through 2 KB places of the warp's
// own (32 rows of 64 bytes, swizzled so that lanes that write rows meet no bank twice): with stores of
// 32 rows by lanes the forward product of a cell model took 71 us in place of 47.  Two accumulators in
// tensor memory let the epilogue of one tile run under the MMAs of the next.
// On a B200, bf16: 8192 x 4096 by 16384 x 4096 twice (gate and up, saved) 1.42 ms, 1.55 PFLOP/s; the six
// products of that block's training step 6.36 ms, 1.56 PFLOP/s, bound by the tensor cores (and, run
// for seconds, by the power cap).  81000 x 256 by 256 x 256 twice: 41 us for 207 MB (5.0 TB/s), bound by
// HBM and the epilogue's latency.
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
  CUtensorMap out[2];  // c[0], c[1] (or, EPI_PARTIAL, the pieces) in boxes of 32 rows of 64 bytes
  CUtensorMap planes;  // the saved pre-activations likewise
  int m, n;            // logical rows and columns of D (columns of one half for EPI_GATE)
  int m_tiles, n_tiles;
  int batch;           // independent products: a[z], c[z] (1 or 2)
  int splits;          // pieces of the k axis (EPI_PARTIAL)
  int kb;              // k blocks of 64
  int kb_second;       // first k block that reads a[1], b[1] (kb when there is one source)
  void* c[2];          // EPI_STORE: outputs; EPI_GATE: h, -; EPI_DGATE: dgate, dup
  long long ldc;
  int plain_c;         // EPI_STORE: rows of c on no 16-byte boundaries, stored by lanes
  const void* bias[2];
  int bias_dtype;
  int save;            // EPI_GATE: write the planes
  float* col_sums;     // EPI_DGATE: column sums of dgate, then dup, of every 32 rows [m / 32][2][col_ld] (may be null)
  long long col_ld;
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
// Relaxed: hands over tensor memory, which the tcgen05 fences order.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
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
// Stores of a 2 KB place of this CTA's shared memory; outside of the tensor nothing is written.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src),
               "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
               "r"(src), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

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

// A wait of a whole warp: it goes on only where no lane gave up, since loads from tensor memory take all lanes.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, const FailState& fs, int where) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, fs, where));
}

// Accumulators out of tensor memory, n columns of the warp's lanes.  One statement loads them and waits: the
// registers of a load in flight may not be touched, and between two statements the compiler may move them
// (with the wait behind the planes' barrier, dgate and dup of the first tiles were wrong now and then).
__device__ __forceinline__ void tmem_take16(uint32_t a, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15])
      : "r"(a)
      : "memory");
}
__device__ __forceinline__ void tmem_take32(uint32_t a, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a)
      : "memory");
}
// (&: written before a1 is read)
__device__ __forceinline__ void tmem_take32(uint32_t a0, uint32_t a1, uint32_t (&r0)[32], uint32_t (&r1)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=&r"(r0[0]), "=&r"(r0[1]), "=&r"(r0[2]), "=&r"(r0[3]), "=&r"(r0[4]), "=&r"(r0[5]), "=&r"(r0[6]),
        "=&r"(r0[7]), "=&r"(r0[8]), "=&r"(r0[9]), "=&r"(r0[10]), "=&r"(r0[11]), "=&r"(r0[12]), "=&r"(r0[13]),
        "=&r"(r0[14]), "=&r"(r0[15]), "=&r"(r0[16]), "=&r"(r0[17]), "=&r"(r0[18]), "=&r"(r0[19]), "=&r"(r0[20]),
        "=&r"(r0[21]), "=&r"(r0[22]), "=&r"(r0[23]), "=&r"(r0[24]), "=&r"(r0[25]), "=&r"(r0[26]), "=&r"(r0[27]),
        "=&r"(r0[28]), "=&r"(r0[29]), "=&r"(r0[30]), "=&r"(r0[31]), "=r"(r1[0]), "=r"(r1[1]), "=r"(r1[2]),
        "=r"(r1[3]), "=r"(r1[4]), "=r"(r1[5]), "=r"(r1[6]), "=r"(r1[7]), "=r"(r1[8]), "=r"(r1[9]),
        "=r"(r1[10]), "=r"(r1[11]), "=r"(r1[12]), "=r"(r1[13]), "=r"(r1[14]), "=r"(r1[15]), "=r"(r1[16]),
        "=r"(r1[17]), "=r"(r1[18]), "=r"(r1[19]), "=r"(r1[20]), "=r"(r1[21]), "=r"(r1[22]), "=r"(r1[23]),
        "=r"(r1[24]), "=r"(r1[25]), "=r"(r1[26]), "=r"(r1[27]), "=r"(r1[28]), "=r"(r1[29]), "=r"(r1[30]),
        "=r"(r1[31])
      : "r"(a0), "r"(a1)
      : "memory");
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
// A place of 32 rows of 64 bytes, 16-byte pieces swizzled as TMA's 64-byte mode does it (piece j of row
// r at j ^ (r / 2 % 4)): a lane's row, written or read.
__device__ __forceinline__ void put_row(uint32_t place, int lane, const uint4 (&v)[4]) {
  const uint32_t row = place + 64 * lane, x = 16 * ((lane >> 1) & 3);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((16 * j) ^ x)), "r"(v[j].x), "r"(v[j].y),
                 "r"(v[j].z), "r"(v[j].w)
                 : "memory");
}
__device__ __forceinline__ void take_row(uint32_t place, int lane, uint4 (&v)[4]) {
  const uint32_t row = place + 64 * lane, x = 16 * ((lane >> 1) & 3);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[j].x), "=r"(v[j].y), "=r"(v[j].z), "=r"(v[j].w)
                 : "r"(row + ((16 * j) ^ x))
                 : "memory");
}
// The first `rows` rows of a place to 16-bit rows that lie on no 16-byte boundaries, `cols` values each.
__device__ __forceinline__ void store_plain(uint32_t place, int lane, uint16_t* to, long long ld, int rows, int cols) {
#pragma unroll 8
  for (int r = 0; r < rows; ++r) {
    const uint32_t at = place + 64 * r + ((16 * (lane >> 3)) ^ (16 * ((r >> 1) & 3))) + 2 * (lane & 7);
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
    if (lane < cols) to[r * ld + lane] = v;
  }
}
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

// Adds up 32 columns over the lanes of a warp: lane l returns the sum of v[l].
__device__ __forceinline__ float column_sum(const float (&x)[32], int lane) {
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = x[i];
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const bool high = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = high ? v[i] : v[i + o], keep = high ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

constexpr int kPlace = 2048;

// Shared memory: the ring, the epilogue's places, biases, barriers.
template <int CG, int BN, int EPI>
struct GemmShape {
  static constexpr int kBNc = BN / CG;  // rows of B in one CTA
  static constexpr int kABytes = kBM * kBK * 2;
  static constexpr int kBBytes = kBNc * kBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // places of an epilogue warp: h (or dgate, then dup) and the three planes; else two in turn
  static constexpr int kPlaces = EPI == EPI_GATE || EPI == EPI_DGATE ? 4 : 2;
  static constexpr int kPlaceBytes = kEpilogueWarps * kPlaces * kPlace;
  static constexpr int kRest = BN * (int)sizeof(float) + 512;
  static constexpr int kMost = (227 * 1024 - 1024 - kPlaceBytes - kRest) / kStageBytes;
  static constexpr int kStages = kMost > 10 ? 10 : kMost;
  static constexpr int kPlacesAt = kStages * kStageBytes;
  static constexpr int kBias = kPlacesAt + kPlaceBytes;
  static constexpr int kBars = kBias + BN * (int)sizeof(float);
  static constexpr int kSmem = kBars + 512 + 1024;  // 1024: alignment
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
  using S = GemmShape<CG, BN, EPI>;
  constexpr int kTN = EPI == EPI_GATE ? BN / 2 : BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drained = acc_empty + 2;
  uint64_t* loaded = drained + 1;  // EPI_DGATE: the planes of each epilogue warp
  uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(loaded + kEpilogueWarps);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_base_s + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 1 ? 0 : cta_rank_in_cluster();
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
  may_start_next();
  after_previous();
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
      if (rank == 0) {  // loads in flight land before this CTA leaves, whichever warp gave up (bounded)
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
      // the MMAs in flight end before the tensor memory is freed, also when only the epilogue gave up (bounded)
      umma_commit_local<CG>(drained);
      for (int tries = 0; tries < 64 && !mbar_try_wait(drained, 0); ++tries) {
      }
    }
  } else if (warp >= 4) {
    const int q = (warp - 4) & 3, turn = (warp - 4) >> 2;  // tensor memory lanes 32 q .. 32 q + 31
    const uint32_t place = smem_u32(smem + S::kPlacesAt) + (warp - 4) * S::kPlaces * kPlace;
    uint32_t load_ph = 0;
    int flip = 0;
    bool ok = true, pending = false;  // pending: planes asked for and not yet waited for
    float* bias_s = reinterpret_cast<float*>(smem + S::kBias);  // [BN]: EPI_GATE those of gate, then of up
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
          if (EPI == EPI_GATE) bias_s[kTN + i] = p.bias[1] ? load_param(p.bias[1], p.bias_dtype, tl.n0 + i) : 0.f;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      if (!ok) continue;  // after a wait that ran out: nothing but the barriers that the other warps wait at
      // EPI_DGATE: the saved planes of the piece at column c, asked for ahead of their use
      const auto ask = [&](int c) {
        pending = true;
        if (lane == 0) {
          mbar_arrive_expect_tx(&loaded[warp - 4], 3 * kPlace);
#pragma unroll
          for (int i = 0; i < 3; ++i)
            tma_load_3d(place + (1 + i) * kPlace, &p.planes, smem_u32(&loaded[warp - 4]), tl.n0 + c, row0, i);
        }
      };
      if (EPI == EPI_DGATE && rows > 0 && 32 * turn < cols) ask(32 * turn);
      ok = mbar_wait_warp(&acc_full[buf], ph, fs, 104);
      if (!ok) continue;
      tc_fence_after();
      const uint32_t acc = tmem + buf * BN + ((uint32_t)(32 * q) << 16);
      for (int c = 32 * turn; c < cols; c += 64) {
        const int col = tl.n0 + c, n = min(32, cols - c);
        uint32_t r0[32];
        if constexpr (EPI == EPI_GATE) {
          uint32_t r1[32];
          tmem_take32(acc + c, acc + kTN + c, r0, r1);
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
              u[i] += bias_s[kTN + c + i];
            }
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 a = mul2(act2<ACT>(make_float2(g[i], g[i + 1])), make_float2(u[i], u[i + 1]));
            h[i] = a.x;
            h[i + 1] = a.y;
          }
          uint4 v[4], v1[4], v2[4];
          if (lane == 0) bulk_wait_read<0>();  // the places have been read
          __syncwarp();
          pack_row<T>(h, v);
          put_row(place, lane, v);
          if (p.save) {
            split_planes(g, u, v, v1, v2);
            put_row(place + kPlace, lane, v);
            put_row(place + 2 * kPlace, lane, v1);
            put_row(place + 3 * kPlace, lane, v2);
          }
          fence_async_proxy();
          __syncwarp();
          if (lane == 0 && rows > 0) {
            tma_store_2d(&p.out[0], place, col, row0);
            if (p.save) {
#pragma unroll
              for (int i = 0; i < 3; ++i) tma_store_3d(&p.planes, place + (1 + i) * kPlace, col, row0, i);
            }
            bulk_commit();
          }
        } else if constexpr (EPI == EPI_DGATE) {
          float g[32], u[32];
          if (rows > 0) {
            ok = mbar_wait_warp(&loaded[warp - 4], load_ph, fs, 105);
            if (!ok) break;
            load_ph ^= 1;
            pending = false;
            uint4 k0[4], k1[4], k2[4];
            take_row(place + kPlace, lane, k0);
            take_row(place + 2 * kPlace, lane, k1);
            take_row(place + 3 * kPlace, lane, k2);
            // every lane's reads come before the copy that overwrites them: without the fence some may be moved
            // behind it, and a warp that was then held up read the next piece's planes
            fence_async_proxy();
            __syncwarp();
            if (c + 64 < cols) ask(c + 64);
            join_planes(k0, k1, k2, g, u);
          }
          if (lane == 0) bulk_wait_read<0>();  // the places have been read
          __syncwarp();
          tmem_take32(acc + c, r0);
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 dh = make_float2(__uint_as_float(r0[i]), __uint_as_float(r0[i + 1]));
            float2 a;
            const float2 slope = act_slope2<ACT>(make_float2(g[i], g[i + 1]), a);
            const float2 dg = mul2(mul2(dh, make_float2(u[i], u[i + 1])), slope), du = mul2(dh, a);
            g[i] = dg.x, g[i + 1] = dg.y;
            u[i] = du.x, u[i + 1] = du.y;
          }
          if (p.col_sums && rows > 0) {  // of the biases' gradients, before the rounding; rows beyond m add 0
            float* to = p.col_sums + (long long)(row0 >> 5) * 2 * p.col_ld + col + lane;
            const float sg = column_sum(g, lane), su = column_sum(u, lane);
            if (lane < n) {
              to[0] = sg;
              to[p.col_ld] = su;
            }
          }
          uint4 v[4];
          __syncwarp();
          pack_row<T>(g, v);
          put_row(place, lane, v);
          fence_async_proxy();
          __syncwarp();
          pack_row<T>(u, v);
          if (lane == 0) {
            if (rows > 0) {
              tma_store_2d(&p.out[0], place, col, row0);
              bulk_commit();
            }
            bulk_wait_read<0>();
          }
          __syncwarp();
          put_row(place, lane, v);
          fence_async_proxy();
          __syncwarp();
          if (lane == 0 && rows > 0) {
            tma_store_2d(&p.out[1], place, col, row0);
            bulk_commit();
          }
        } else if constexpr (EPI == EPI_PARTIAL) {
          tmem_take32(acc + c, r0);
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i] = make_uint4(r0[16 * half + 4 * i], r0[16 * half + 4 * i + 1], r0[16 * half + 4 * i + 2],
                                r0[16 * half + 4 * i + 3]);
            put_row(place + half * kPlace, lane, v);
          }
          fence_async_proxy();
          __syncwarp();
          if (lane == 0 && rows > 0) {
            const int z = tl.split * p.batch + tl.batch;
            tma_store_3d(&p.out[0], place, col, row0, z);
            if (n > 16) tma_store_3d(&p.out[0], place + kPlace, col + 16, row0, z);
            bulk_commit();
          }
        } else {
          tmem_take32(acc + c, r0);
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(r0[i]);
          if (biased) {
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] += bias_s[c + i];
          }
          uint4 v[4];
          pack_row<T>(f, v);
          const uint32_t here = place + flip * kPlace;
          flip ^= 1;
          if (lane == 0) bulk_wait_read<1>();  // the store before the last has read this place
          __syncwarp();
          put_row(here, lane, v);
          if (p.plain_c) {
            __syncwarp();
            store_plain(here, lane, static_cast<uint16_t*>(p.c[tl.batch]) + (long long)row0 * p.ldc + col, p.ldc, rows, n);
          } else {
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) {  // a group for every piece, also one without rows: the wait above counts groups
              if (rows > 0) tma_store_2d(&p.out[tl.batch], here, col, row0);
              bulk_commit();
            }
          }
        }
      }
      if (!ok) continue;
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
      for (int tries = 0; tries < 64 && !mbar_try_wait(&loaded[warp - 4], load_ph); ++tries) {
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
