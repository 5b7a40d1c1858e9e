// gated.cu -- the gated feed-forward block, forward and backward (nca_b200_gated_*), on the tcgen05
// product kernel of gemm.cuh.  With T rows, D inputs, F hidden, O outputs:
//
//   forward   gate = x Wg^T + bg, up = x Wu^T + bu, h = act(gate) up       one product, fused epilogue
//             y = h Wd^T + bd                                              one product
//   backward  dh = dy Wd;  dgate = dh up act'(gate), dup = dh act(gate)    one product, fused epilogue
//             dx = dgate Wg + dup Wu                                       one product, k axis 2 F
//             dWd = dy^T h;  dWg = dgate^T x, dWu = dup^T x                products over the T rows
//             db = column sums of dgate, dup, dy
//
// Roundings: h, dgate and dup are rounded once to the matrix type, since they are operands of the
// next 16-bit product; gate and up are kept for the backward with 24 bits; sums stay in fp32.
//
// The products over T rows have small outputs and a long k axis in a cell model: the axis is then
// cut into pieces whose fp32 sums are added in a fixed order by a second kernel.
#include "gemm_rows.cuh"

#include <algorithm>
#include <atomic>

using namespace nca;

namespace {

#define NCA_TRY(call)                    \
  do {                                   \
    const int32_t st_ = (call);          \
    if (st_ != NCA_OK) return st_;       \
  } while (0)

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
inline long long pad8(long long v) { return (v + 7) / 8 * 8; }

constexpr int kMaxDevices = 64;

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

// A 16-bit matrix that TMA can read: `cols` adjacent values a row, rows `ld` values apart.
struct Matrix {
  const void* p;
  long long rows, cols, ld;
};

// Boxes of 64 columns (128 bytes, swizzled) x box_rows rows; outside reads as zero.
bool encode(CUtensorMap* map, const Matrix& m, int dtype, int box_rows) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows};
  const cuuint64_t strides[1] = {(cuuint64_t)m.ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  const cuuint32_t one[2] = {1, 1};
  return fn(map, dtype == NCA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
            const_cast<void*>(m.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Boxes of 64 bytes x 32 rows, 64-byte swizzle, of `planes` matrices `plane` bytes apart: what the
// epilogues store and load.
bool encode_boxes(CUtensorMap* map, const void* p, CUtensorMapDataType type, int size, long long cols, long long rows,
                  long long ld, int dims, long long planes, long long plane) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t d[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  const cuuint64_t strides[2] = {(cuuint64_t)(ld * size), (cuuint64_t)plane};
  const cuuint32_t box[3] = {(cuuint32_t)(64 / size), 32, 1};
  const cuuint32_t one[3] = {1, 1, 1};
  return fn(map, type, dims, const_cast<void*>(p), d, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
CUtensorMapDataType map_type(int dtype) {
  return dtype == NCA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}
// An output matrix of the matrix type with rows on 16-byte boundaries.
bool encode_out(CUtensorMap* map, const void* p, int dtype, long long rows, long long cols, long long ld) {
  return encode_boxes(map, p, map_type(dtype), 2, cols, rows, ld, 2, 1, 0);
}
// The three planes of the saved pre-activations.
bool encode_planes(CUtensorMap* map, const void* p, long long rows, long long cols, long long ld, long long plane) {
  return encode_boxes(map, p, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, cols, rows, ld, 3, 3, plane);
}
// The outputs of an EPI_STORE product (c[1] may repeat c[0]): by TMA where their rows allow it.
bool set_out(GemmParams& p, int dtype, void* c0, void* c1, long long rows, long long cols) {
  p.c[0] = c0;
  p.c[1] = c1;
  p.ldc = cols;
  p.plain_c = cols % 8 != 0 || reinterpret_cast<uintptr_t>(c0) % 16 != 0 || reinterpret_cast<uintptr_t>(c1) % 16 != 0;
  return p.plain_c || (encode_out(&p.out[0], c0, dtype, rows, cols, cols) &&
                        (c1 == c0 || encode_out(&p.out[1], c1, dtype, rows, cols, cols)));
}

// ------------------------------------------------------------------------------- small kernels
// dst[r][c] = src[r * sr + c * sc]: operands that TMA cannot read, copied to padded rows, all of a call in
// one launch (blockIdx.y).
struct Pack {
  const uint16_t* src;
  uint16_t* dst;
  long long rows, cols, sr, sc, ld;
};
struct Packs {
  Pack p[5];
};
// 16 bytes of a row that starts 2 m bytes after a 16-byte boundary, from the two aligned pieces that hold them.
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int m) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t v[5];
#pragma unroll
  for (int i = 0; i < 5; ++i)
    v[i] = m < 2 ? w[i] : m < 4 ? w[i + 1] : m < 6 ? w[i + 2] : w[min(i + 3, 7)];
  const int bits = 16 * (m & 1);
  return make_uint4(__funnelshift_r(v[0], v[1], bits), __funnelshift_r(v[1], v[2], bits),
                    __funnelshift_r(v[2], v[3], bits), __funnelshift_r(v[3], v[4], bits));
}
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Packs all) {
  may_start_next();
  after_previous();
  __shared__ uint16_t tile[32][34];
  const Pack& p = all.p[blockIdx.y];
  if (p.sc == 1) {  // rows of adjacent values: a warp a row, 8 a lane
    for (long long r = (long long)blockIdx.x * 8 + threadIdx.y; r < p.rows; r += (long long)gridDim.x * 8) {
      const uint16_t* row = p.src + r * p.sr;
      const int m = (int)(reinterpret_cast<uintptr_t>(row) & 15) / 2;
#pragma unroll 2
      for (long long c = 8 * threadIdx.x; c < p.ld; c += 256) {
        uint4 out;
        if (c >= 8 && c + 16 <= p.cols) {  // both aligned pieces lie inside the row
          const uint4* q = reinterpret_cast<const uint4*>(row + c - m);
          out = shifted(q[0], q[1], m);
        } else {
          uint32_t v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = c + 2 * j < p.cols ? row[c + 2 * j] : 0, hi = c + 2 * j + 1 < p.cols ? row[c + 2 * j + 1] : 0;
            v[j] = lo | hi << 16;
          }
          out = make_uint4(v[0], v[1], v[2], v[3]);
        }
        *reinterpret_cast<uint4*>(p.dst + r * p.ld + c) = out;
      }
    }
    return;
  }
  // any strides: 32 x 32 tiles through shared memory, read along whichever stride is 1
  const long long ct = (p.cols + 31) / 32, tiles = ct * ((p.rows + 31) / 32);
  for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
    const long long r0 = t / ct * 32, c0 = t % ct * 32;
    __syncthreads();
    for (int i = threadIdx.y; i < 32; i += 8) {
      const int r = p.sr == 1 ? threadIdx.x : i, c = p.sr == 1 ? i : threadIdx.x;
      if (r0 + r < p.rows && c0 + c < p.cols) tile[r][c] = p.src[(r0 + r) * p.sr + (c0 + c) * p.sc];
    }
    __syncthreads();
    for (int i = threadIdx.y; i < 32; i += 8)
      if (r0 + i < p.rows && c0 + threadIdx.x < p.cols) p.dst[(r0 + i) * p.ld + c0 + threadIdx.x] = tile[i][threadIdx.x];
  }
}

// c[z][m][n] = bias[n] + sum over the pieces of part[s * batch + z][m][n]: 32 lanes of 4 columns by 8 groups of
// pieces, which add up in the order of the groups.
template <class T>
__global__ void __launch_bounds__(256) join_kernel(const float* part, int splits, int batch, long long m, long long n,
                                                   long long ldp, T* c0, T* c1, const void* bias, int bias_dtype) {
  may_start_next();
  after_previous();
  __shared__ float4 red[8][32];
  const long long total = batch * m * ldp / 4, i = (long long)blockIdx.x * 32 + threadIdx.x;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < total) {
    const float4* from = reinterpret_cast<const float4*>(part) + i;
#pragma unroll 4
    for (int k = threadIdx.y; k < splits; k += 8) {
      const float4 v = from[k * total];
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y || i >= total) return;
  for (int k = 1; k < 8; ++k) {
    const float4 v = red[k][threadIdx.x];
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  const long long zr = 4 * i / ldp, c = 4 * i - zr * ldp, z = zr / m, r = zr - z * m;
  T* to = (z ? c1 : c0) + r * n + c;
  const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j < n) to[j] = from_f32<T>(f[j] + (bias ? load_param(bias, bias_dtype, c + j) : 0.f));
}

// Column sums of a [rows][cols] matrix, 8 columns a thread (rows lie on 16-byte boundaries): `wide` threads
// side by side, 256 / wide rows at a time, a block the rows of its piece, in a fixed order.
constexpr int kSumSplits = 256, kRowPieces = 32;
template <class T>
__global__ void __launch_bounds__(256) column_sums_kernel(const T* a, long long rows, long long cols, long long ld,
                                                          int splits, int wide, float* part, long long padded) {
  may_start_next();
  after_previous();
  __shared__ float2 red[256][4];
  const int high = 256 / wide, row = threadIdx.x / wide;
  const long long c = 8 * ((long long)blockIdx.x * wide + threadIdx.x % wide);
  const long long per = (rows + splits - 1) / splits, r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
  float2 s[4] = {both(0.f), both(0.f), both(0.f), both(0.f)};
  if (c < cols && row < high) {
    const T* from = a + c;
    const auto add = [&](const Vec<T, 8>& v) {
      float2 f[4];
      to_pairs<T, 8>(v, f);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = add2(s[i], f[i]);
    };
    if (c + 8 <= cols) {
#pragma unroll 8
      for (long long r = r0 + row; r < r1; r += high) add(*reinterpret_cast<const Vec<T, 8>*>(from + r * ld));
    } else {
      for (long long r = r0 + row; r < r1; r += high) {
        Vec<T, 8> v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v.v[i] = c + i < cols ? from[r * ld + i] : from_f32<T>(0.f);
        add(v);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) red[threadIdx.x][i] = s[i];
  __syncthreads();
  for (int i = threadIdx.x; i < 4 * wide; i += 256) {  // a pair of columns each
    const int v = i / 4;
    const long long at = 8 * ((long long)blockIdx.x * wide + v) + 2 * (i % 4);
    if (at >= padded) continue;
    float2 t = red[v][i % 4];
    for (int r = 1; r < high; ++r) t = add2(t, red[r * wide + v][i % 4]);
    *reinterpret_cast<float2*>(part + blockIdx.y * padded + at) = t;
  }
}
// Adds up the rows of up to three [rows][ld] fp32 matrices (blockIdx.z), a piece of them a block (blockIdx.y):
// into the next matrix, or where there is one piece into the gradient.
struct RowSums {
  const float* part[3];
  float* next[3];  // [pieces][ld], or null
  void* out[3];
  long long cols[3], ld[3];
  int rows[3];
};
__global__ void __launch_bounds__(512) row_sums_kernel(const __grid_constant__ RowSums p, int dtype) {
  may_start_next();
  after_previous();
  __shared__ float red[16][33];
  const int z = blockIdx.z;
  const long long c = (long long)blockIdx.x * 32 + threadIdx.x, ld = p.ld[z];
  const int per = (p.rows[z] + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = min(p.rows[z], r0 + per);
  float s = 0.f;
  if (c < p.cols[z]) {
    const float* from = p.part[z] + c;
#pragma unroll 8
    for (int r = r0 + threadIdx.y; r < r1; r += 16) s += from[r * ld];
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y || c >= p.cols[z]) return;
  for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x];
  if (gridDim.y > 1) p.next[z][blockIdx.y * ld + c] = s;
  else store_param(p.out[z], dtype, c, s);
}

// --------------------------------------------------------------------------------- the products
template <class T, int CG, int BN, bool A_MN, bool B_MN, int EPI, int ACT>
int32_t launch(GemmParams& p, cudaStream_t s) {
  using S = GemmShape<CG, BN, EPI>;
  constexpr int kTN = EPI == EPI_GATE ? BN / 2 : BN;
  auto* kernel = gemm_kernel<T, CG, BN, A_MN, B_MN, EPI, ACT>;
  static std::atomic<uint64_t> ready{0};  // a bit for each device whose shared-memory limit is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return NCA_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess)
      return launch_status() == NCA_OK ? NCA_ERR_CUDA : NCA_ERR_DEVICE;
    ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  p.m_tiles = (int)ceil_div(p.m, kBM * CG);
  p.n_tiles = (int)ceil_div(p.n, kTN);
  const long long tiles = (long long)p.m_tiles * p.n_tiles * p.batch * p.splits;
  if (tiles > (1ll << 31) - 1024) return NCA_ERR_UNSUPPORTED;
  const long long room = sm_count() / CG;
  return launch_after(kernel, dim3((unsigned)((tiles < room ? tiles : room) * CG)), dim3(kGemmThreads), S::kSmem, s, CG, p);
}

// Tiles and pieces of a product m x n over kb k blocks (`batch` of them).  A k block costs a 256 x 256 tile
// of a pair of multiprocessors 0.28 us (the MMAs), a 256 x 128 tile 0.24 and a 128 x 128 tile of one
// 0.25 (64 bytes a cycle from L2), a tile 5 us besides, and a product in pieces 3 us and 20 bytes of
// traffic an output and piece more.  The smallest sum wins; measured on 2000 x 1008 x 5472: 33, 30 and
// 32 us in one piece.
struct Shape {
  int cg, bn;
  int splits;
};
Shape shape_of(long long m, long long n, int batch, long long kb, bool may_split, bool gate) {
  static const struct {
    int cg, bn;
    double us;
  } kinds[] = {{2, 256, 0.28}, {2, 128, 0.24}, {1, 128, 0.25}};
  const long long sms = sm_count();
  Shape best{2, 256, 1};
  double least = 1e30;
  for (const auto& k : kinds) {
    const long long tiles = ceil_div(m, 128 * k.cg) * ceil_div(n, gate ? k.bn / 2 : k.bn) * batch;
    const long long room = sms / k.cg;
    if (tiles == 0) return best;  // no rows
    const long long most = may_split ? std::max(1ll, std::min(room / tiles, kb / 8)) : 1;
    for (long long s = 1; s <= most; s = s < most && 2 * s > most ? most : 2 * s) {
      const double waves = (double)ceil_div(tiles * s, room);
      double us = waves * ((double)ceil_div(kb, s) * k.us + 1.0) + 4.0;
      if (s > 1) us += 3.0 + 1e6 * 20.0 * s * batch * m * n / 6.4e12;
      if (us < least) {
        least = us;
        best = {k.cg, k.bn, (int)s};
      }
    }
  }
  return best;
}

struct Product {
  Matrix a[2], b[2];
  bool two_a, two_b;     // a[1] / b[1] present
  long long m, n, k;     // k: one source's length
  bool k_sources;        // a[1], b[1] continue the k axis
  int batch;
};

int32_t set_up(GemmParams& p, const Product& g, int dtype, bool a_mn, bool b_mn, int cg, int bn, bool gate) {
  const int bnc = gate ? bn / 2 : bn / cg;
  if (!encode(&p.a[0], g.a[0], dtype, a_mn ? 64 : kBM) || !encode(&p.b[0], g.b[0], dtype, b_mn ? 64 : bnc) ||
      (g.two_a && !encode(&p.a[1], g.a[1], dtype, a_mn ? 64 : kBM)) ||
      (g.two_b && !encode(&p.b[1], g.b[1], dtype, b_mn ? 64 : bnc)))
    return NCA_ERR_CUDA;
  if (!g.two_a) p.a[1] = p.a[0];
  if (!g.two_b) p.b[1] = p.b[0];
  p.m = (int)g.m;
  p.n = (int)g.n;
  p.batch = g.batch;
  p.splits = 1;
  const int kb = (int)ceil_div(g.k, kBK);
  p.kb = g.k_sources ? 2 * kb : kb;
  p.kb_second = kb;
  return NCA_OK;
}

template <class T, bool A_MN, bool B_MN, int EPI, int ACT>
int32_t product(GemmParams& p, const Product& g, int dtype, const Shape& sh, cudaStream_t s) {
  const int32_t st = set_up(p, g, dtype, A_MN, B_MN, sh.cg, sh.bn, EPI == EPI_GATE);
  if (st != NCA_OK) return st;
  p.splits = sh.splits;
  if (sh.cg == 1) return launch<T, 1, 128, A_MN, B_MN, EPI, ACT>(p, s);
  return sh.bn == 128 ? launch<T, 2, 128, A_MN, B_MN, EPI, ACT>(p, s) : launch<T, 2, 256, A_MN, B_MN, EPI, ACT>(p, s);
}

// A product whose outputs are stored as they are (plus a bias), through partial sums when its k axis is cut.
template <class T, bool A_MN, bool B_MN>
int32_t stored_product(GemmParams& p, const Product& g, int dtype, void* c0, void* c1, const void* bias, float* part,
                       cudaStream_t s) {
  const long long kb = ceil_div(g.k, kBK) * (g.k_sources ? 2 : 1);
  const Shape sh = shape_of(g.m, g.n, g.batch, kb, true, false);
  if (sh.splits == 1) {
    p.bias[0] = bias;
    if (!set_out(p, dtype, c0, c1, g.m, g.n)) return NCA_ERR_CUDA;
    return product<T, A_MN, B_MN, EPI_STORE, NCA_ACT_NONE>(p, g, dtype, sh, s);
  }
  const long long ldp = (g.n + 3) / 4 * 4;
  if (!encode_boxes(&p.out[0], part, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, g.n, g.m, ldp, 3, (long long)sh.splits * g.batch,
                    g.m * ldp * 4))
    return NCA_ERR_CUDA;
  const int32_t st = product<T, A_MN, B_MN, EPI_PARTIAL, NCA_ACT_NONE>(p, g, dtype, sh, s);
  if (st != NCA_OK) return st;
  const long long total = g.batch * g.m * ldp / 4;
  return launch_after(join_kernel<T>, dim3((unsigned)ceil_div(total, 32)), dim3(32, 8), 0, s, 1, part, sh.splits, g.batch,
                      g.m, g.n, ldp, static_cast<T*>(c0), static_cast<T*>(c1), bias, p.bias_dtype);
}
size_t part_bytes(long long m, long long n, int batch, long long k, int sources) {
  const Shape sh = shape_of(m, n, batch, ceil_div(k, kBK) * sources, true, false);
  return sh.splits == 1 ? 0 : (size_t)sh.splits * batch * m * ((n + 3) / 4 * 4) * sizeof(float);
}

// The products of few rows: out = act(x w0^T + b0) (x w1^T + b1), or x w0^T + b0.
constexpr long long kFewRows = 64;
template <class T, int N, bool GATE, int ACT>
int32_t rows_launch(RowsParams& p, cudaStream_t s) {
  using S = RowsShape<N, GATE>;
  auto* kernel = gemm_rows_kernel<T, N, GATE, ACT>;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return NCA_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess)
      return launch_status() == NCA_OK ? NCA_ERR_CUDA : NCA_ERR_DEVICE;
    ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  const long long tiles = ceil_div(p.n, kBM);
  if (tiles > (1ll << 27)) return NCA_ERR_UNSUPPORTED;
  // a power of two (it divides 128): as many CTAs as run at once, two k blocks a CTA at least; clusters of
  // 4 and 8 leave some multiprocessors of a processing cluster out
  p.slices = 1;
  const long long room = (long long)S::kBlocks * sm_count();
  while (p.slices < 8 && p.kb >= 4 * p.slices &&
         tiles * p.slices * 2 <= (p.slices == 1 ? room : p.slices == 2 ? room * 88 / 100 : room * 80 / 100))
    p.slices *= 2;
  return launch_after(kernel, dim3((unsigned)(tiles * p.slices)), dim3(kRowsThreads), S::kSmem, s, p.slices, p);
}
template <class T, bool GATE, int ACT>
int32_t rows_product(const GemmParams& base, const Matrix& x, const Matrix& w0, const Matrix& w1, const void* b0,
                     const void* b1, void* out, long long ld, bool weights_first, int dtype, cudaStream_t s) {
  RowsParams p{};
  const int n = x.rows <= 16 ? 16 : x.rows <= 32 ? 32 : 64;
  if (!encode(&p.x, x, dtype, n) || !encode(&p.w[0], w0, dtype, kBM) || (GATE && !encode(&p.w[1], w1, dtype, kBM)))
    return NCA_ERR_CUDA;
  p.rows = (int)x.rows;
  p.n = (int)w0.rows;
  p.kb = (int)ceil_div(x.cols, kBK);
  p.weights_first = weights_first;
  p.out = out;
  p.ld = ld;
  p.bias[0] = b0;
  p.bias[1] = b1;
  p.bias_dtype = base.bias_dtype;
  p.ctrl = base.ctrl;
  p.timeout_ns = base.timeout_ns;
  if (n == 16) return rows_launch<T, 16, GATE, ACT>(p, s);
  return n == 32 ? rows_launch<T, 32, GATE, ACT>(p, s) : rows_launch<T, 64, GATE, ACT>(p, s);
}

// --------------------------------------------------------------------------------- arguments
int32_t check_desc(const NcaGatedDesc* d) {
  if (!d || d->rows < 0 || d->d_in <= 0 || d->hidden <= 0 || d->d_out <= 0) return NCA_ERR_INVALID;
  if (d->dtype != NCA_BF16 && d->dtype != NCA_F16) return NCA_ERR_UNSUPPORTED;
  if (d->bias_dtype != NCA_F32 && d->bias_dtype != d->dtype) return NCA_ERR_INVALID;
  if (d->act < NCA_ACT_RELU || d->act > NCA_ACT_SIGMOID) return NCA_ERR_INVALID;
  const long long most = (1ll << 31) - 1024;
  if (d->rows > most || d->d_in > most || d->hidden > most || d->d_out > most) return NCA_ERR_UNSUPPORTED;
  return NCA_OK;
}

enum { OP_X, OP_WG, OP_WU, OP_WD, OP_DY, OPS };
struct Operand {
  long long rows, cols, sr, sc;
  bool packed;
  size_t at;  // offset of the copy in the workspace
};
struct Plan {
  Operand op[OPS];
  size_t h, dgate, dup, part, sums, cols, total;
  long long fp;  // padded hidden
};

// bias_sums: room for the column sums that the gradients of b_gate and b_up are made of.
Plan plan_of(const NcaGatedDesc& d, bool backward, bool bias_sums = true) {
  Plan p{};
  const long long rows[OPS] = {d.rows, d.hidden, d.hidden, d.d_out, d.rows};
  const long long cols[OPS] = {d.d_in, d.d_in, d.d_in, d.hidden, d.d_out};
  const int64_t* stride[OPS] = {d.x_stride, d.w_gate_stride, d.w_up_stride, d.w_down_stride, d.dy_stride};
  size_t at = 0;
  for (int i = 0; i < OPS; ++i) {
    Operand& o = p.op[i];
    o.rows = rows[i];
    o.cols = cols[i];
    o.sr = o.rows == 1 ? pad8(o.cols) : stride[i][0];  // the stride of a single row or column means nothing
    o.sc = o.cols == 1 ? 1 : stride[i][1];
    o.packed = o.sc != 1 || o.sr % 8 != 0 || o.sr < o.cols || o.sr >= (1ll << 38) || (d.unaligned >> i & 1);
    if (i == OP_DY && !backward) o.packed = false;
    if (o.packed) {
      if (o.rows == 1) o.sr = 0;
      o.at = at;
      at += align256((size_t)o.rows * pad8(o.cols) * 2);
    }
  }
  p.fp = pad8(d.hidden);
  const size_t tf = align256((size_t)d.rows * p.fp * 2);
  if (!backward) {
    p.h = at;
    at += tf;
    p.part = at;
    at += align256(part_bytes(d.rows, d.d_out, 1, d.hidden, 1));
  } else {
    p.dgate = at;
    at += tf;
    p.dup = at;
    at += tf;
    p.part = at;
    at += align256(std::max({part_bytes(d.rows, d.d_in, 1, d.hidden, 2), part_bytes(d.hidden, d.d_in, 2, d.rows, 1),
                             part_bytes(d.hidden, d.d_in, 1, d.rows, 1), part_bytes(d.d_out, d.hidden, 1, d.rows, 1)}));
    p.sums = at;
    at += align256(((size_t)kRowPieces * 2 * p.fp + (size_t)(kSumSplits + kRowPieces) * pad8(d.d_out)) * sizeof(float));
    p.cols = at;
    if (bias_sums) at += align256((size_t)ceil_div(d.rows, 128) * 4 * 2 * p.fp * sizeof(float));
  }
  p.total = at + 256;
  return p;
}

// The operands as TMA reads them: in place, or copied into the workspace by one launch.
struct Operands {
  Matrix m[OPS];
  Packs packs;
  int count = 0;
  long long most = 0;  // blocks for the largest copy: 8 rows each, or tiles
  int32_t add(int i, const Operand& o, const void* src, uint8_t* ws) {
    if (!src) return NCA_ERR_INVALID;
    if (!o.packed) {
      if (reinterpret_cast<uintptr_t>(src) % 16) return NCA_ERR_INVALID;  // `unaligned` did not say so
      m[i] = {src, o.rows, o.cols, o.sr};
      return NCA_OK;
    }
    uint16_t* dst = reinterpret_cast<uint16_t*>(ws + o.at);
    const long long ld = pad8(o.cols);
    packs.p[count++] = {static_cast<const uint16_t*>(src), dst, o.rows, o.cols, o.sr, o.sc, ld};
    most = std::max(most, o.sc == 1 ? ceil_div(o.rows, 8) : ceil_div(o.rows, 32) * ceil_div(o.cols, 32));
    m[i] = {dst, o.rows, o.cols, ld};
    return NCA_OK;
  }
  int32_t copy(cudaStream_t s) const {
    if (count == 0) return NCA_OK;
    return launch_after(pack_kernel, dim3((unsigned)std::min<long long>(most, 148 * 8), count), dim3(32, 8), 0, s, 1, packs);
  }
};


template <class T, int ACT>
int32_t forward(const NcaGatedDesc& d, const void* x, const void* w_gate, const void* w_up, const void* w_down,
                const void* b_gate, const void* b_up, const void* b_down, void* y, void* saved, uint8_t* ws,
                GemmParams& base, cudaStream_t s) {
  const Plan pl = plan_of(d, false);
  Operands in;
  NCA_TRY(in.add(OP_X, pl.op[OP_X], x, ws));
  NCA_TRY(in.add(OP_WG, pl.op[OP_WG], w_gate, ws));
  NCA_TRY(in.add(OP_WU, pl.op[OP_WU], w_up, ws));
  NCA_TRY(in.add(OP_WD, pl.op[OP_WD], w_down, ws));
  NCA_TRY(in.copy(s));
  const Matrix &mx = in.m[OP_X], &mg = in.m[OP_WG], &mu = in.m[OP_WU], &md = in.m[OP_WD];
  const size_t tf = align256((size_t)d.rows * pl.fp * 2);
  uint8_t* keep = static_cast<uint8_t*>(saved);
  void* h = keep ? keep + 3 * tf : ws + pl.h;
  if (!keep && d.rows <= kFewRows) {
    NCA_TRY((rows_product<T, true, ACT>(base, mx, mg, mu, b_gate, b_up, h, pl.fp, false, d.dtype, s)));
    return rows_product<T, false, NCA_ACT_NONE>(base, {h, d.rows, d.hidden, pl.fp}, md, md, b_down, nullptr, y, d.d_out,
                                                true, d.dtype, s);
  }
  {
    GemmParams p = base;
    Product g{{mx, mx}, {mg, mu}, false, true, d.rows, d.hidden, d.d_in, false, 1};
    if (!encode_out(&p.out[0], h, d.dtype, d.rows, d.hidden, pl.fp)) return NCA_ERR_CUDA;
    p.bias[0] = b_gate;
    p.bias[1] = b_up;
    p.save = keep != nullptr;
    if (keep && !encode_planes(&p.planes, keep, d.rows, d.hidden, pl.fp, (long long)tf)) return NCA_ERR_CUDA;
    NCA_TRY((product<T, false, false, EPI_GATE, ACT>(
        p, g, d.dtype, shape_of(g.m, g.n, 1, ceil_div(g.k, kBK), false, true), s)));
  }
  GemmParams p = base;
  const Matrix mh{h, d.rows, d.hidden, pl.fp};
  Product g{{mh, mh}, {md, md}, false, false, d.rows, d.d_out, d.hidden, false, 1};
  return stored_product<T, false, false>(p, g, d.dtype, y, y, b_down, reinterpret_cast<float*>(ws + pl.part), s);
}

template <class T, int ACT>
int32_t backward(const NcaGatedDesc& d, const void* x, const void* w_gate, const void* w_up, const void* w_down,
                 const void* saved, const void* dy, void* dx, void* dw_gate, void* dw_up, void* dw_down,
                 void* db_gate, void* db_up, void* db_down, uint8_t* ws, GemmParams& base, cudaStream_t s) {
  const Plan pl = plan_of(d, true);
  const size_t tf = align256((size_t)d.rows * pl.fp * 2);
  const uint8_t* keep = static_cast<const uint8_t*>(saved);
  const bool hidden_grads = dx || dw_gate || dw_up || db_gate || db_up;
  Operands in;
  NCA_TRY(in.add(OP_DY, pl.op[OP_DY], dy, ws));
  if (hidden_grads) NCA_TRY(in.add(OP_WD, pl.op[OP_WD], w_down, ws));
  if (dx) {
    NCA_TRY(in.add(OP_WG, pl.op[OP_WG], w_gate, ws));
    NCA_TRY(in.add(OP_WU, pl.op[OP_WU], w_up, ws));
  }
  if (dw_gate || dw_up) NCA_TRY(in.add(OP_X, pl.op[OP_X], x, ws));
  NCA_TRY(in.copy(s));
  const Matrix &mx = in.m[OP_X], &mg = in.m[OP_WG], &mu = in.m[OP_WU], &md = in.m[OP_WD], &mdy = in.m[OP_DY];
  const Matrix mh{keep + 3 * tf, d.rows, d.hidden, pl.fp};
  const Matrix mdg{ws + pl.dgate, d.rows, d.hidden, pl.fp}, mdu{ws + pl.dup, d.rows, d.hidden, pl.fp};
  float* part = reinterpret_cast<float*>(ws + pl.part);
  float* part_sums = reinterpret_cast<float*>(ws + pl.sums);
  float* col_sums = reinterpret_cast<float*>(ws + pl.cols);
  if (hidden_grads) {
    GemmParams p = base;
    Product g{{mdy, mdy}, {md, md}, false, false, d.rows, d.hidden, d.d_out, false, 1};
    if (!encode_out(&p.out[0], ws + pl.dgate, d.dtype, d.rows, d.hidden, pl.fp) ||
        !encode_out(&p.out[1], ws + pl.dup, d.dtype, d.rows, d.hidden, pl.fp) ||
        !encode_planes(&p.planes, keep, d.rows, d.hidden, pl.fp, (long long)tf))
      return NCA_ERR_CUDA;
    p.col_sums = db_gate || db_up ? col_sums : nullptr;
    p.col_ld = pl.fp;
    NCA_TRY((product<T, false, true, EPI_DGATE, ACT>(
        p, g, d.dtype, shape_of(g.m, g.n, 1, ceil_div(g.k, kBK), false, false), s)));
  }
  if (dx) {
    GemmParams p = base;
    Product g{{mdg, mdu}, {mg, mu}, true, true, d.rows, d.d_in, d.hidden, true, 1};
    NCA_TRY((stored_product<T, false, true>(p, g, d.dtype, dx, dx, nullptr, part, s)));
  }
  if (dw_gate || dw_up) {
    GemmParams p = base;
    if (dw_gate && dw_up) {
      Product g{{mdg, mdu}, {mx, mx}, true, false, d.hidden, d.d_in, d.rows, false, 2};
      NCA_TRY((stored_product<T, true, true>(p, g, d.dtype, dw_gate, dw_up, nullptr, part, s)));
    } else {
      const Matrix& m = dw_gate ? mdg : mdu;
      void* out = dw_gate ? dw_gate : dw_up;
      Product g{{m, m}, {mx, mx}, false, false, d.hidden, d.d_in, d.rows, false, 1};
      NCA_TRY((stored_product<T, true, true>(p, g, d.dtype, out, out, nullptr, part, s)));
    }
  }
  if (dw_down) {
    GemmParams p = base;
    Product g{{mdy, mdy}, {mh, mh}, false, false, d.d_out, d.hidden, d.rows, false, 1};
    NCA_TRY((stored_product<T, true, true>(p, g, d.dtype, dw_down, dw_down, nullptr, part, s)));
  }
  // the biases' gradients: sums of 32 rows each (or of pieces of dy), added up in one or two steps
  RowSums sums{};
  int count = 0, most = 0;
  long long widest = 0;
  const auto add = [&](const float* part, int rows, long long cols, long long ld, float* next, void* out) {
    if (!out) return;
    sums.part[count] = part;
    sums.next[count] = next;
    sums.out[count] = out;
    sums.cols[count] = cols;
    sums.ld[count] = ld;
    sums.rows[count++] = rows;
    most = std::max(most, rows);
    widest = std::max(widest, cols);
  };
  const int blocks = (int)ceil_div(d.rows, 32);
  add(col_sums, blocks, d.hidden, 2 * pl.fp, part_sums, db_gate);
  add(col_sums + pl.fp, blocks, d.hidden, 2 * pl.fp, part_sums + pl.fp, db_up);
  if (db_down) {
    const long long padded = pad8(d.d_out);
    const int splits = (int)std::max<long long>(1, std::min<long long>(kSumSplits, d.rows / 64));
    float* part = part_sums + kRowPieces * 2 * pl.fp;
    const int wide = (int)std::min<long long>(padded / 8, 32);
    NCA_TRY(launch_after(column_sums_kernel<T>, dim3((unsigned)ceil_div(padded, 8 * wide), splits), dim3(256), 0, s, 1,
                         static_cast<const T*>(mdy.p), d.rows, d.d_out, mdy.ld, splits, wide, part, padded));
    add(part, splits, d.d_out, padded, part + kSumSplits * padded, db_down);
  }
  if (count && most > 256) {
    NCA_TRY(launch_after(row_sums_kernel, dim3((unsigned)ceil_div(widest, 32), kRowPieces, count), dim3(32, 16), 0, s, 1, sums,
                         d.bias_dtype));
    for (int i = 0; i < count; ++i) {
      sums.part[i] = sums.next[i];
      sums.rows[i] = kRowPieces;
    }
  }
  if (count)
    return launch_after(row_sums_kernel, dim3((unsigned)ceil_div(widest, 32), 1, count), dim3(32, 16), 0, s, 1, sums,
                        d.bias_dtype);
  return NCA_OK;
}

template <class F>
int32_t dispatch(const NcaGatedDesc& d, F fn) {
  auto by_act = [&](auto t) {
    using T = decltype(t);
    switch (d.act) {
      case NCA_ACT_RELU: return fn.template operator()<T, NCA_ACT_RELU>();
      case NCA_ACT_SILU: return fn.template operator()<T, NCA_ACT_SILU>();
      case NCA_ACT_GELU: return fn.template operator()<T, NCA_ACT_GELU>();
      default: return fn.template operator()<T, NCA_ACT_SIGMOID>();
    }
  };
  return d.dtype == NCA_BF16 ? by_act(__nv_bfloat16{}) : by_act(__half{});
}

struct ForwardCall {
  const NcaGatedDesc& d;
  const void *x, *wg, *wu, *wd, *bg, *bu, *bd;
  void *y, *saved;
  uint8_t* ws;
  GemmParams& base;
  cudaStream_t s;
  template <class T, int A>
  int32_t operator()() const { return forward<T, A>(d, x, wg, wu, wd, bg, bu, bd, y, saved, ws, base, s); }
};
struct BackwardCall {
  const NcaGatedDesc& d;
  const void *x, *wg, *wu, *wd, *saved, *dy;
  void *dx, *dwg, *dwu, *dwd, *dbg, *dbu, *dbd;
  uint8_t* ws;
  GemmParams& base;
  cudaStream_t s;
  template <class T, int A>
  int32_t operator()() const {
    return backward<T, A>(d, x, wg, wu, wd, saved, dy, dx, dwg, dwu, dwd, dbg, dbu, dbd, ws, base, s);
  }
};

// Makes the current device's context current on this thread: the tensor-map encoder is a driver
// call, which a thread without one (autograd's, before its first runtime call) would fail.
int32_t bind_context() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess ? NCA_OK : NCA_ERR_DEVICE;
}

GemmParams base_params(const NcaGatedDesc& d, int32_t* ctrl, int32_t timeout_ms) {
  GemmParams p{};
  p.bias_dtype = d.bias_dtype;
  p.ctrl = ctrl;
  p.timeout_ns = (unsigned long long)(timeout_ms > 0 ? timeout_ms : 20000) * 1000000ull;
  return p;
}

}  // namespace

extern "C" {

int32_t nca_b200_gated_saved_bytes(const NcaGatedDesc* d, size_t* bytes) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK || !bytes) return st != NCA_OK ? st : NCA_ERR_INVALID;
  *bytes = 4 * align256((size_t)d->rows * pad8(d->hidden) * 2);
  return NCA_OK;
}

int32_t nca_b200_gated_workspace(const NcaGatedDesc* d, int32_t backward, size_t* bytes) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK || !bytes) return st != NCA_OK ? st : NCA_ERR_INVALID;
  *bytes = plan_of(*d, backward != 0, backward != 2).total;
  return NCA_OK;
}

int32_t nca_b200_gated_ffn(const NcaGatedDesc* d, const void* x, const void* w_gate, const void* w_up,
                           const void* w_down, const void* b_gate, const void* b_up, const void* b_down, void* y,
                           void* saved, void* workspace, size_t workspace_bytes, int32_t* ctrl, int32_t timeout_ms,
                           void* stream) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK) return st;
  if (d->rows == 0) return NCA_OK;
  if (!y || !workspace || !ctrl || workspace_bytes < plan_of(*d, false).total) return NCA_ERR_INVALID;
  NCA_TRY(bind_context());
  GemmParams base = base_params(*d, ctrl, timeout_ms);
  return dispatch(*d, ForwardCall{*d, x, w_gate, w_up, w_down, b_gate, b_up, b_down, y, saved,
                                  static_cast<uint8_t*>(workspace), base, static_cast<cudaStream_t>(stream)});
}

int32_t nca_b200_gated_ffn_backward(const NcaGatedDesc* d, const void* x, const void* w_gate, const void* w_up,
                                    const void* w_down, const void* saved, const void* dy, void* dx, void* dw_gate,
                                    void* dw_up, void* dw_down, void* db_gate, void* db_up, void* db_down,
                                    void* workspace, size_t workspace_bytes, int32_t* ctrl, int32_t timeout_ms,
                                    void* stream) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->rows == 0) {
    const size_t b = dtype_size(d->bias_dtype);
    const struct {
      void* p;
      size_t bytes;
    } outs[] = {{dw_gate, (size_t)d->hidden * d->d_in * 2}, {dw_up, (size_t)d->hidden * d->d_in * 2},
                {dw_down, (size_t)d->d_out * d->hidden * 2}, {db_gate, d->hidden * b}, {db_up, d->hidden * b},
                {db_down, d->d_out * b}};
    for (const auto& o : outs)
      if (o.p && cudaMemsetAsync(o.p, 0, o.bytes, s) != cudaSuccess) return NCA_ERR_CUDA;
    return NCA_OK;
  }
  if (!saved || !dy || !workspace || !ctrl || workspace_bytes < plan_of(*d, true, db_gate || db_up).total)
    return NCA_ERR_INVALID;
  NCA_TRY(bind_context());
  GemmParams base = base_params(*d, ctrl, timeout_ms);
  return dispatch(*d, BackwardCall{*d, x, w_gate, w_up, w_down, saved, dy, dx, dw_gate, dw_up, dw_down, db_gate, db_up,
                                   db_down, static_cast<uint8_t*>(workspace), base, s});
}

}  // extern "C"
