// sample.cu -- classes drawn from rows of logits with given uniform numbers (nca_b200_sample): temperature, top-k,
// top-p, min-p.
//
// With w_i = exp((z_i - max z) / T), classes in the order of z (largest first, ties by index): the first top_k; of
// those, the ones before which less than top_p of their mass lies; of those, the ones with w_i >= min_p.  A draw is
// the first class, by index, at which the sum of the kept w exceeds u times the whole.
//
// The answers are whole numbers, and a row of 131072 classes has a border every 1e-5 of its mass: weights are computed in
// 64 bits, to 1e-14 of themselves.  Sums are in fixed point: they do not depend on an order.  The largest weight is 2^bits of
// its units: 51 bits up to 2048 classes, one less for every doubling to 43 at 2^19, so that a row of nothing but large weights
// still adds up within 2^62.  A weight is off by half a unit at most and one below that has no mass, so a border is off by
// classes 2^-(bits + 1) of the largest weight at most: 5e-13 at 2048 classes, 2e-9 at 131072, 3e-8 at 2^19, half the spacing of
// uniform numbers beside 1.  Beyond, where that would be 12 % at 2^30, another pass bounds the row's sum first and the bits
// follow from it (62 less its own): classes 2^-52 of the sum at most, 2e-7 at 2^30.  The exponential is table-driven
// (Tang, ACM TOMS 15, 1989): 2^(j / 32) from a table, e^r of |r| < 0.0109 by five terms, 12 operations in 64 bits with
// the conversion to fixed point.  A table of 256 saves two of them and loses more by conflicts of banks (1024 x 131072 without
// cuts: 7 % slower than the 190 us of now).
//
// Up to 32 classes a row is a group of lanes, a class a lane, and ranks are counted.  Longer rows are a block's.  All three
// cuts keep a prefix of the order, so the kept set is always "from a place (z, index) on".
//   min_p: the least z of enough weight, by search.
//   a small top_k: the k-th largest of 2 k groups' maxima bounds the k-th largest entry from below; the few entries above it
//     are listed and sorted, and everything else happens in the list (as for all rows that fit it).
//   a larger top_k, of 1536 at most: its place in a histogram of counts over (top - z) / T, and the list likewise.
//   top_p alone: such a histogram bounds the mass before every bin within 0.5 %; one pass then
//     computes all weights, adds up those surely kept by segment and lists those about the border, which decide.
//   else: histograms over the ordered bits of z until the entries of the bin with the border can be listed.
// Segments of entries, a warp each, hold the sums of the kept weights; a draw looks through one segment.
#include "cell_ops.cuh"

#include <algorithm>
#include <atomic>

using namespace nca;

namespace {

struct SampleParams {
  const void* logits;
  const float* uniforms;
  long long* tokens;
  float* probs;
  long long rows, stride;  // of logits
  int classes, draws;
  int top_k;               // classes: all
  double inverse_t, top_p, min_p;
  double one;              // a weight of 1 in fixed point (up to kKnown classes)
};

// -inf for NaN (drawn as little as -inf), 0 for -0.
__device__ __forceinline__ float clean(float v) { return v != v ? __int_as_float(0xff800000) : v + 0.f; }
__device__ __forceinline__ bool possible(float v) { return v > __int_as_float(0xff800000); }

// w of [0, 1] in fixed point, to nearest; one: 2^51 at most.
__device__ __forceinline__ uint64_t fixed(double w, double one) {
  return (uint64_t)(__double_as_longlong(fma(w, one, 4503599627370496.0)) - 0x4330000000000000ll);
}
// What a draw's sum has to exceed.
__device__ __forceinline__ uint64_t threshold(float u, uint64_t total) {
  const double t = fmax((double)u, 0.0) * (double)total;  // u above 1: the last class, NaN: the first
  return t < (double)total ? min((uint64_t)t, total - 1) : total - 1;
}

// 2^(j / kTable)
constexpr int kTableBits = 5, kTable = 1 << kTableBits;  // parts of an octave: two addresses a bank
__constant__ double kPowers[kTable] = {
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924,
    1.1387886347566916, 1.1637248587775775, 1.189207115002721, 1.215247359980469, 1.241857812073484,
    1.2690509571917332, 1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228, 1.5422108254079407,
    1.5759808451078865, 1.6104903319492543, 1.645755478153965, 1.681792830507429, 1.718619298122478,
    1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474,
    1.9571441241754002};
// e^(c r) - 1 of c = ln(2) / kTable and |r| <= 1/2, to 3e-15
__device__ __forceinline__ double power_rest(double r) {
  constexpr double c = 0.69314718055994530942 / kTable;
  constexpr double c2 = c * c / 2, c3 = c2 * c / 3, c4 = c3 * c / 4, c5 = c4 * c / 5;
  return r * (c + r * (c2 + r * (c3 + r * (c4 + r * c5))));
}
constexpr double kNearest = 6755399441055744.0;  // 1.5 2^52: the low bits of a sum with it are the nearest whole number
// exp((v - top) / T) times table[0], from a table of kPowers times that; kTable log2(e) / T in `steep`.
__device__ __forceinline__ double weight_below(float v, float top, double steep, const double* table) {
  if (v == top) return table[0];  // also of infinities
  const double x = ((double)v - (double)top) * steep;
  if (!(x > -62.0 * kTable)) return 0.0;
  const double m = x + kNearest;
  const int k = __double2loint(m);
  const double t = table[k & (kTable - 1)], e = fma(t, power_rest(x - (m - kNearest)), t);
  return __hiloint2double(__double2hiint(e) + (k >> kTableBits << 20), __double2loint(e));
}

// ------------------------------------------------------------------------------- up to 32 classes
// Up to 4 classes and 4 draws: a row a thread, everything in registers (900000 rows of 2 bf16 classes: 11 us, with two
// lanes a row 17).
template <class T, int C>
__global__ void __launch_bounds__(256) sample_tiny_kernel(const __grid_constant__ SampleParams p) {
  may_start_next();
  after_previous();
  __shared__ double table[kTable];
  if (threadIdx.x < kTable) table[threadIdx.x] = kPowers[threadIdx.x] * p.one;
  __syncthreads();
  const long long row = (long long)blockIdx.x * 256 + threadIdx.x;
  if (row >= p.rows) return;
  const T* z = static_cast<const T*>(p.logits) + row * p.stride;
  float v[C];
  float top = __int_as_float(0xff800000);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    v[i] = i < p.classes ? clean(to_f32<T>(z[i])) : __int_as_float(0xff800000);
    top = fmaxf(top, v[i]);
  }
  const double steep = p.inverse_t * (kTable * 1.4426950408889634074), least = p.min_p * p.one;
  uint64_t w[C], mass = 0;
  bool heavy[C];
  int rank[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const double e = possible(v[i]) ? weight_below(v[i], top, steep, table) : 0.0;
    w[i] = fixed(e, 1.0);
    heavy[i] = e >= least;
    rank[i] = 0;
#pragma unroll
    for (int j = 0; j < C; ++j) rank[i] += v[j] > v[i] || (v[j] == v[i] && j < i);
    if (rank[i] < p.top_k) mass += w[i];
  }
  uint64_t c[C], total = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    bool keep = rank[i] < p.top_k && heavy[i];
    if (p.top_p < 1.0) {
      uint64_t before = 0;
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (rank[j] < rank[i]) before += w[j];
      keep = keep && (double)before < p.top_p * (double)mass;
    }
    total += keep ? w[i] : 0;
    c[i] = total;
  }
  for (int d = 0; d < p.draws; ++d) {
    const long long at = row * p.draws + d;
    int token = -1;
    float prob = 0.f;
    if (total) {
      const uint64_t t = threshold(p.uniforms[at], total);
      uint64_t below = 0, own = 0;
      token = 0;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const bool over = c[i] > t;
        if (!over) token = i + 1, below = c[i];
        if (over && !own) own = c[i] - below;
      }
      prob = (float)((double)own / (double)total);
    }
    p.tokens[at] = token;
    if (p.probs) p.probs[at] = prob;
  }
}

template <class T, int G>
__global__ void __launch_bounds__(256) sample_few_kernel(const __grid_constant__ SampleParams p) {
  may_start_next();
  after_previous();
  __shared__ uint64_t sums[256];
  __shared__ double table[kTable];
  if (threadIdx.x < kTable) table[threadIdx.x] = kPowers[threadIdx.x] * p.one;
  __syncthreads();
  const int lane = threadIdx.x % G, base = threadIdx.x - lane;
  const long long row = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool here = row < p.rows && lane < p.classes;
  const unsigned all = 0xffffffffu;
  const float v = here ? clean(to_f32<T>(static_cast<const T*>(p.logits)[row * p.stride + lane])) : clean(__int_as_float(0x7fc00000));
  float top = v;
#pragma unroll
  for (int o = G / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(all, top, o));
  const double weight = possible(v) ? weight_below(v, top, p.inverse_t * (kTable * 1.4426950408889634074), table) : 0.0;
  uint64_t w = fixed(weight, 1.0);
  // its place in the order, and the mass before it
  int rank = 0;
  uint64_t before = 0;
#pragma unroll 8
  for (int j = 0; j < G; ++j) {
    const float vj = __shfl_sync(all, v, j, G);
    const uint64_t wj = __shfl_sync(all, w, j, G);
    if (vj > v || (vj == v && j < lane)) {
      ++rank;
      before += wj;
    }
  }
  if (rank >= p.top_k) w = 0;
  if (p.top_p < 1.0) {
    uint64_t mass = w;
#pragma unroll
    for (int o = G / 2; o; o >>= 1) mass += __shfl_xor_sync(all, mass, o);
    if (!((double)before < p.top_p * (double)mass)) w = 0;
  }
  if (!(weight >= p.min_p * p.one)) w = 0;
  uint64_t c = w;  // sums in the order of the classes
#pragma unroll
  for (int o = 1; o < G; o <<= 1) {
    const uint64_t below = __shfl_up_sync(all, c, o, G);
    if (lane >= o) c += below;
  }
  const uint64_t total = __shfl_sync(all, c, G - 1, G);
  sums[threadIdx.x] = c;
  __syncwarp();
  if (row >= p.rows) return;
  for (int d = lane; d < p.draws; d += G) {
    const long long at = row * p.draws + d;
    if (total == 0) {
      p.tokens[at] = -1;
      if (p.probs) p.probs[at] = 0.f;
      continue;
    }
    const uint64_t t = threshold(p.uniforms[at], total);
    int token = 0;  // how many sums are at most t
#pragma unroll
    for (int step = G / 2; step; step >>= 1)
      if (sums[base + token + step - 1] <= t) token += step;
    p.tokens[at] = token;
    if (p.probs) p.probs[at] = (float)((double)(sums[base + token] - (token ? sums[base + token - 1] : 0)) / (double)total);
  }
}

// ------------------------------------------------------------------------------------ longer rows
constexpr int kBins = 2048;       // of the ordered bits
constexpr int kMassBins = 4096;   // of (top - z) / T
constexpr float kPerBin = 100.f;  // the last holds all beyond 40.9, whose weights are below 2^-58
constexpr int kSubBins = 256;
constexpr int kMostSegments = 1024;
constexpr int kMostTops = 2048;
constexpr int kKnown = 1 << 19;   // classes up to which their number alone gives the fixed point

// Floats in their order as whole numbers.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// Its place in the order: larger first, then the lower index.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int i) { return (uint64_t)key << 32 | (0xffffffffu - (uint32_t)i); }
__device__ __forceinline__ int index_of(uint64_t place) { return (int)(0xffffffffu - (uint32_t)place); }
__device__ __forceinline__ float value_of(uint64_t place) { return of_key((uint32_t)(place >> 32)); }
constexpr uint64_t kPossible = 0x00800000ull << 32;  // the places above -inf

// Blocks of 128 threads serve rows that the list holds whole.
template <int THREADS>
struct RowShared {
  static constexpr bool kLong = THREADS > 128;
  static constexpr int kList = kLong ? 2048 : 1024;      // entries with their masses
  static constexpr int kRegion = kLong ? 2048 : 1024;    // entries alone
  static constexpr int kSegments = kLong ? kMostSegments : 64;
  double table[kTable];
  uint64_t sums[kSegments];
  uint64_t warp_sums[32];
  union {
    uint64_t list[kRegion];
    struct {
      uint64_t list_[kList];
      uint64_t masses[kList];
    };
    struct {
      uint32_t counts[kLong ? kBins : 1];
      uint32_t low[kLong ? kBins : 1], high[kLong ? kBins : 1];  // masses of the bins
    };
    uint32_t mass_counts[kLong ? kMassBins : 1];
  };
  uint32_t sub_low[kLong ? kSubBins : 1], sub_high[kLong ? kSubBins : 1];
  float reds[64];
  float groups[THREADS];                      // their largest entries
  float chunk_tops[kLong ? kMostTops : 1];    // of the chunks, where there are not more
  uint32_t keys[64];
  int listed, found;
  uint64_t limit;
  long long amount;
};

__device__ __forceinline__ float warp_max(float v) {  // NaN aside
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
// Adds to a 64-bit sum of two words.
__device__ __forceinline__ void add_to(uint32_t* low, uint32_t* high, uint64_t m) {
  const uint32_t l = (uint32_t)m, old = atomicAdd(low, l);
  const uint32_t h = (uint32_t)(m >> 32) + (old + l < old ? 1u : 0u);
  if (h) atomicAdd(high, h);
}
__device__ __forceinline__ uint64_t warp_sum(uint64_t s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
template <class S>
__device__ __forceinline__ S warp_running(S s, int lane) {  // with this lane's own
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const S below = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += below;
  }
  return s;
}

// 16 bytes of a row: 8 entries, or 4 of fp32.
template <class T>
struct Entries {
  static constexpr int kV = 16 / sizeof(T);
  uint4 q;
  __device__ __forceinline__ float at(int j) const {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    if constexpr (__is_same(T, __nv_bfloat16)) return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    else return __half2float(__ushort_as_half((unsigned short)(j & 1 ? w[j / 2] >> 16 : w[j / 2])));
  }
  __device__ __forceinline__ void set(int j, T v) { reinterpret_cast<T*>(&q)[j] = v; }
  // the largest, NaN aside: of two, then of all
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) {
      return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    } else if constexpr (__is_same(T, __nv_bfloat16)) {
      const __nv_bfloat162 m = __hmax2(reinterpret_cast<__nv_bfloat162&>(a), reinterpret_cast<__nv_bfloat162&>(b));
      return reinterpret_cast<const uint32_t&>(m);
    } else {
      const __half2 m = __hmax2(reinterpret_cast<__half2&>(a), reinterpret_cast<__half2&>(b));
      return reinterpret_cast<const uint32_t&>(m);
    }
  }
  __device__ __forceinline__ uint32_t most() const { return max2(max2(q.x, q.y), max2(q.z, q.w)); }
  static __device__ __forceinline__ float value(uint32_t most) {
    if constexpr (sizeof(T) == 4) return clean(__uint_as_float(most));
    Entries e;
    e.q.x = most;
    return fmaxf(clean(e.at(0)), clean(e.at(1)));
  }
};

template <class T, int THREADS>
struct Row {
  using Sh = RowShared<THREADS>;
  using E = Entries<T>;
  static constexpr int kWarps = THREADS / 32, kV = E::kV, kChunk = 32 * kV;
  const SampleParams& p;
  Sh& sh;
  const T* z;
  const uint4* base;  // this lane's 16 bytes of chunk 0
  int n, shift, chunks, per_segment, segments;  // chunks of a warp's vectors; of a segment
  float top, lowest;      // of the entries; what lies below `lowest` has no mass
  double one;             // a weight of 1 in fixed point
  double steep, offset;   // v steep + offset = kTable log2(e) (v - top) / T
  bool far;               // ... but for a top whose offset 64 bits round
  uint64_t limit;         // places from here on are kept
  int warp, lane;

  __device__ __forceinline__ Row(const SampleParams& p_, Sh& sh_, long long row) : p(p_), sh(sh_) {
    z = static_cast<const T*>(p.logits) + row * p.stride;
    n = p.classes;
    shift = (int)(reinterpret_cast<uintptr_t>(z) % 16 / sizeof(T));  // chunks start on 16-byte boundaries
    chunks = (n + shift + kChunk - 1) / kChunk;
    per_segment = (chunks + Sh::kSegments - 1) / Sh::kSegments;
    segments = (chunks + per_segment - 1) / per_segment;
    limit = kPossible;
    warp = threadIdx.x / 32;
    lane = threadIdx.x % 32;
    base = reinterpret_cast<const uint4*>(z - shift) + lane;
    set_one(p.one);
  }
  __device__ __forceinline__ void set_one(double o) {
    one = o;
    if (threadIdx.x < kTable) sh.table[threadIdx.x] = kPowers[threadIdx.x] * one;
  }
  // The fixed point of a row of many classes, from a bound of its sum of weights: 8 exponentials at a time add up in fp32, all in 64
  // bits, each within 2e-5 (roundings of the exponent, 2^-23 of 60 octaves, and the exponential's).
  __device__ __forceinline__ void fit_one() {
    const float scale = (float)(p.inverse_t * 1.4426950408889634074);
    double sum = 0;
    each_chunk<2>([&](int, const E& e) {
      float some = 0.f;
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const float v = clean(e.at(j));
        some += v == top ? 1.f : ex2((v - top) * scale);
      }
      sum += some;
    });
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if (lane == 0) sh.warp_sums[warp] = (uint64_t)__double_as_longlong(sum);
    __syncthreads();
    sum = 0;
    for (int w = 0; w < kWarps; ++w) sum += __longlong_as_double((long long)sh.warp_sums[w]);
    int bits = 51;
    while (bits > 32 && 1.001 * sum > (double)(1ll << (62 - bits))) --bits;
    set_one((double)(1ll << bits));
    __syncthreads();
  }
  __device__ __forceinline__ void set_top(float t) {
    top = t;
    steep = p.inverse_t * (kTable * 1.4426950408889634074);
    offset = -(double)top * steep;
    far = !(fabs(offset) < 1024.0 * kTable);
    lowest = (float)((double)top - 42.0 / p.inverse_t);  // e^-42 < 2^-60
  }
  // This lane's entries of a chunk; entries outside of the row (in the first and last chunk) are -inf.
  __device__ __forceinline__ E fetch(int chunk) const {
    E e;
    if (chunk > 0 && chunk + 1 < chunks) {
      e.q = base[chunk * 32];
    } else {
      const int first = first_of(chunk);
      if (first >= 0 && first + kV <= n) {
        e.q = base[chunk * 32];
      } else {
#pragma unroll
        for (int j = 0; j < kV; ++j)
          e.set(j, first + j >= 0 && first + j < n ? z[first + j] : from_f32<T>(__int_as_float(0xff800000)));
      }
    }
    return e;
  }
  __device__ __forceinline__ int first_of(int chunk) const { return chunk * kChunk + lane * kV - shift; }
  // fn(chunk, entries): chunks in turn over the warps, AHEAD of them on their way.
  template <int AHEAD, class F>
  __device__ __forceinline__ void each_chunk(F fn) const {
    E next[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (warp + i * kWarps < chunks) next[i] = fetch(warp + i * kWarps);
    for (int c = warp; c < chunks;) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (c >= chunks) break;
        const E e = next[i];
        if (c + AHEAD * kWarps < chunks) next[i] = fetch(c + AHEAD * kWarps);
        fn(c, e);
        c += kWarps;
      }
    }
  }
  // Segments in turn over the warps: fn(chunk, entries), and after a segment's chunks done(segment).
  template <class F, class D>
  __device__ __forceinline__ void each_segment(F fn, D done) const {
    if (warp >= segments) return;
    int s = warp, c = s * per_segment;
    E next = fetch(c);
    while (s < segments) {
      const E e = next;
      const int here = c, segment = s;
      if (++c >= min((s + 1) * per_segment, chunks)) {
        s += kWarps;
        c = s * per_segment;
      }
      if (s < segments) next = fetch(c);
      fn(here, e);
      if (s != segment) done(segment);
    }
  }
  __device__ __forceinline__ bool kept(float v, int i) const { return place_of(key_of(v), i) >= limit; }  // of a clean v

  // exp((v - top) / T) times `one`
  template <bool FAR>
  __device__ __forceinline__ double weight_of(float v) const {
    if constexpr (FAR) {
      return weight_below(v, top, steep, sh.table);
    } else {
      const double x = fma((double)fmaxf(v, lowest), steep, offset), m = x + kNearest;
      const int k = __double2loint(m);
      const double t = sh.table[k & (kTable - 1)], e = fma(t, power_rest(x - (m - kNearest)), t);
      return __hiloint2double(__double2hiint(e) + (k >> kTableBits << 20), __double2loint(e));
    }
  }
  __device__ __forceinline__ double weight(float v) const { return far ? weight_of<true>(v) : weight_of<false>(v); }
  __device__ __forceinline__ uint64_t mass(float v) const { return fixed(weight(v), 1.0); }
  __device__ __forceinline__ uint64_t near_mass(float v) const { return fixed(weight_of<false>(v), 1.0); }

  // Running sums of a[0 .. count) in place; returns the whole.
  __device__ __forceinline__ uint64_t scan(uint64_t* a, int count) {
    uint64_t carry = 0;
    for (int b = 0; b < count; b += THREADS) {
      const int i = b + threadIdx.x;
      uint64_t s = warp_running(i < count ? a[i] : 0, lane);
      __syncthreads();
      if (lane == 31) sh.warp_sums[warp] = s;
      __syncthreads();
      s += carry;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) s += sh.warp_sums[w];
        carry += sh.warp_sums[w];
      }
      if (i < count) a[i] = s;
    }
    __syncthreads();
    return carry;
  }
  // The sum of a value of each warp.
  __device__ __forceinline__ uint64_t block_sum(uint64_t s) {
    __syncthreads();
    if (lane == 0) sh.warp_sums[warp] = s;
    __syncthreads();
    s = 0;
    for (int w = 0; w < kWarps; ++w) s += sh.warp_sums[w];
    return s;
  }
  // The first of count running sums above t.
  __device__ __forceinline__ int above(const uint64_t* a, int count, uint64_t t) const {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (a[mid] <= t) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  }
  // The list to descending order: a few entries by counting the larger ones, else filled up to a power of two.
  __device__ __forceinline__ void sort(int count) {
    if (count <= min(THREADS, 256)) {
      uint64_t mine = 0;
      int rank = 0;
      if (threadIdx.x < (count + 31) / 32 * 32) {
        mine = threadIdx.x < count ? sh.list[threadIdx.x] : 0;
        for (int i = 0; i < count; ++i) rank += sh.list[i] > mine;
      }
      __syncthreads();
      if (threadIdx.x < count) sh.list[rank] = mine;
      __syncthreads();
      return;
    }
    int size = 2;
    while (size < count) size <<= 1;
    for (int i = count + threadIdx.x; i < size; i += THREADS) sh.list[i] = 0;
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j; j >>= 1) {
        __syncthreads();
        for (int i = threadIdx.x; i < size / 2; i += THREADS) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const uint64_t x = sh.list[a], y = sh.list[b];
          if ((x < y) == ((a & k) == 0)) sh.list[a] = y, sh.list[b] = x;
        }
      }
    __syncthreads();
  }
  // All lanes of a warp call it.
  __device__ __forceinline__ int room_for(bool mine) {
    const unsigned who = __ballot_sync(0xffffffffu, mine);
    if (!who) return 0;
    int at = 0;
    if (lane == 0) at = atomicAdd(&sh.listed, __popc(who));
    return __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
  }
  __device__ __forceinline__ void append(bool mine, uint64_t place, int room) {
    const int at = room_for(mine);
    if (mine && at < room) sh.list[at] = place;
  }
  __device__ __forceinline__ void append(bool mine, float v, int i, int room) {
    const int at = room_for(mine);
    if (mine && at < room) sh.list[at] = place_of(key_of(clean(v)), i);
  }
  __device__ __forceinline__ void start_list() {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
  }

  // The largest entry, and those of the chunks.  k > 0: also a bound that k entries reach, the k-th largest of the largest
  // entries of `groups` groups (a power of two, at most THREADS, and at least k).
  __device__ __forceinline__ float largest(int k, int groups, float& bound) {
    const float least = __int_as_float(0xff800000);
    E none;
#pragma unroll
    for (int j = 0; j < kV; ++j) none.set(j, from_f32<T>(least));
    uint32_t most = none.q.x;
    each_chunk<4>([&](int chunk, const E& e) {
      const uint32_t m = e.most();
      most = E::max2(most, m);
      if (Sh::kLong) {
        const float t = warp_max(E::value(m));
        if (lane == 0 && chunk < kMostTops) sh.chunk_tops[chunk] = t;
      }
    });
    float m = E::value(most);
    const int wide = THREADS / groups;  // threads of a group
    for (int o = 1; o < min(wide, 32); o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    sh.groups[threadIdx.x] = m;
    m = warp_max(m);
    if (lane == 0) sh.reds[warp] = m;
    __syncthreads();
    m = sh.reds[0];
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sh.reds[w]);
    if (k > 0) {
      if (threadIdx.x < groups) {
        const auto of_group = [&](int g) {
          float f = sh.groups[g * wide];
          for (int i = 32; i < wide; i += 32) f = fmaxf(f, sh.groups[g * wide + i]);
          return f;
        };
        const float mine = of_group(threadIdx.x);
        int before = 0;  // in the order of the groups
        for (int g = 0; g < groups; ++g) {
          const float f = of_group(g);
          before += f > mine || (f == mine && g < threadIdx.x);
        }
        if (before == k - 1) sh.reds[32] = mine;
      }
      __syncthreads();
      bound = sh.reds[32];
    }
    return m;
  }
  // Whether a chunk can hold entries from `least` on.
  __device__ __forceinline__ bool reaches(int chunk, float least) const {
    return !Sh::kLong || chunk >= kMostTops || sh.chunk_tops[chunk] >= least;
  }
  // fn(chunk, entries) of those chunks, in turn over the warps; the next one is on its way.
  template <class F>
  __device__ __forceinline__ void each_reaching(float least, F fn) const {
    for (int c0 = warp; c0 < chunks; c0 += 32 * kWarps) {
      const int mine = c0 + lane * kWarps;
      unsigned which = __ballot_sync(0xffffffffu, mine < chunks && reaches(mine, least));
      if (!which) continue;
      E next = fetch(c0 + (__ffs(which) - 1) * kWarps);
      while (which) {
        const E e = next;
        const int c = c0 + (__ffs(which) - 1) * kWarps;
        which &= which - 1;
        if (which) next = fetch(c0 + (__ffs(which) - 1) * kWarps);
        fn(c, e);
      }
    }
  }

  // The least place of a weight of min_p, by a search of 32 keys at a time (every warp for itself).
  __device__ __forceinline__ uint64_t limit_of_weight(double min_p) const {
    const double least = min_p * one;
    uint32_t lo = (uint32_t)(kPossible >> 32), hi = key_of(top);  // hi is heavy enough
    while (lo < hi) {
      const uint32_t step = (hi - lo + 30) / 31, at = min(lo + lane * step, hi);
      const float v = of_key(at);
      const int first = __ffs(__ballot_sync(0xffffffffu, weight(v) >= least || at == hi)) - 1;  // of the 32
      const uint32_t found = __shfl_sync(0xffffffffu, at, first);
      lo = first == 0 ? lo : __shfl_sync(0xffffffffu, at, first - 1) + 1;
      hi = found;
    }
    return (uint64_t)lo << 32;
  }
  // The place at which the sorted list's masses, from `m` on, reach the target.
  __device__ __forceinline__ uint64_t limit_of_list(int count, uint64_t m, uint64_t target) {
    if (warp == 0) {
      int taken = 0;
      for (int b = 0; b < count; b += 32) {
        const uint64_t own = b + lane < count ? mass(value_of(sh.list[b + lane])) : 0, up = warp_running(own, lane);
        const unsigned in = __ballot_sync(0xffffffffu, b + lane < count && m + up - own < target);
        taken += __popc(in);
        m += __shfl_sync(0xffffffffu, up, 31);
        if (in != 0xffffffffu) break;
      }
      if (lane == 0) sh.limit = sh.list[max(taken, 1) - 1];
    }
    __syncthreads();
    const uint64_t l = sh.limit;
    __syncthreads();
    return l;
  }

  // How many entries lie at each (top - v) scale, to nearest; all beyond the bins, and NaN, in the last.
  __device__ __forceinline__ void count_bins(float scale) {
    for (int i = threadIdx.x; i < kMassBins; i += THREADS) sh.mass_counts[i] = 0;
    __syncthreads();
    each_chunk<2>([&](int, const E& e) {
#pragma unroll
      for (int j = 0; j < kV; ++j) {  // by the bits of a sum with 2^23
        const uint32_t b = __float_as_uint(fmaf(top - e.at(j), scale, 8388608.f)) - 0x4b000000u;
        atomicAdd(&sh.mass_counts[min(b, (uint32_t)kMassBins - 1)], 1u);
      }
    });
    __syncthreads();
  }
  // What k entries reach, but for roundings at the edge of a bin; -inf where it lies in the last.
  __device__ __forceinline__ float bound_by_count(int k) {
    if constexpr (Sh::kLong) {
      const float scale = kPerBin * (float)p.inverse_t;
      if (threadIdx.x == 0) sh.keys[0] = kMassBins - 1;
      count_bins(scale);
      constexpr int kPer = kMassBins / THREADS;
      int count = 0;
      for (int i = 0; i < kPer; ++i) count += sh.mass_counts[threadIdx.x * kPer + i];
      const int up = warp_running(count, lane);
      if (lane == 31) sh.keys[32 + warp] = up;
      __syncthreads();
      int before = up - count;
      for (int w = 0; w < warp; ++w) before += sh.keys[32 + w];
      for (int i = 0; i < kPer; ++i) {
        const int here = sh.mass_counts[threadIdx.x * kPer + i];
        if (before < k && before + here >= k) sh.keys[0] = threadIdx.x * kPer + i;  // one thread
        before += here;
      }
      __syncthreads();
      const uint32_t b = sh.keys[0];
      __syncthreads();
      if (b < kMassBins - 1) return top - (b + 0.51f) / scale;
    }
    return __int_as_float(0xff800000);
  }

  // top_p alone.  `least`: the limit by min_p.  Returns kCut where the limit is found, kSummed where sh.sums also holds the
  // segments' kept sums, kNot where the entries about the border do not fit the list.
  enum { kNot, kCut, kSummed };
  __device__ __forceinline__ int cut_mass(uint64_t least) {
    if constexpr (Sh::kLong) {
      const float scale = kPerBin * (float)p.inverse_t;
      for (int i = threadIdx.x; i < kSubBins; i += THREADS) sh.sub_low[i] = sh.sub_high[i] = 0;
      if (threadIdx.x < 8) sh.keys[threadIdx.x] = kMassBins - 1;
      count_bins(scale);
      // bin b lies at (b -+ 0.501) / 100 (roundings: 4096 2^-23 of a bin): bounds of the masses up to every bin
      constexpr int kPer = kMassBins / THREADS;
      constexpr float kLog = -1.4426950408889634f / kPerBin;
      float lower = 0.f, upper = 0.f;
      int count = 0;
      for (int i = 0; i < kPer; ++i) {
        const int b = threadIdx.x * kPer + i, c = b + 1 < kMassBins ? sh.mass_counts[b] : 0;
        count += c;
        lower += c * ex2((b + 0.501f) * kLog);
        upper += c * ex2((b - 0.501f) * kLog);
      }
      const float l_up = warp_running(lower, lane), u_up = warp_running(upper, lane);
      const int c_up = warp_running(count, lane);
      if (lane == 31) {
        sh.reds[warp] = l_up;
        sh.reds[32 + warp] = u_up;
        sh.keys[32 + warp] = c_up;
      }
      __syncthreads();
      float l = l_up - lower, u = u_up - upper, l_all = 0.f, u_all = 0.f;
      int c = c_up - count;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) l += sh.reds[w], u += sh.reds[32 + w], c += sh.keys[32 + w];
        l_all += sh.reds[w], u_all += sh.reds[32 + w];
      }
      // the first bins at which the border may have been reached, is likely to be, and must have been (fp32 sums of 4096
      // terms, in three levels: 2^-17 of themselves)
      const float may = (float)p.top_p * l_all * 0.9999f, must = (float)p.top_p * u_all * 1.0001f;
      const float likely = (float)p.top_p * 0.5f * (l_all + u_all);
      const int before = c;
      {
        uint32_t first[3] = {kMassBins - 1, kMassBins - 1, kMassBins - 1}, at_likely = 0;
        for (int i = 0; i < kPer; ++i) {
          const int b = threadIdx.x * kPer + i, here = b + 1 < kMassBins ? sh.mass_counts[b] : 0;
          l += here * ex2((b + 0.501f) * kLog);
          u += here * ex2((b - 0.501f) * kLog);
          if (u >= may) first[0] = min(first[0], b);
          if (0.5f * (l + u) >= likely && b < first[1]) first[1] = b, at_likely = c;
          if (l >= must) first[2] = min(first[2], b);
          c += here;
        }
        const uint32_t mid = __reduce_min_sync(0xffffffffu, first[1]);
        for (int i = 0; i < 3; ++i) {
          const uint32_t f = __reduce_min_sync(0xffffffffu, first[i]);
          if (lane == 0) atomicMin(&sh.keys[i], f);
        }
        __syncthreads();
        if (first[1] == sh.keys[1] && mid == first[1]) sh.amount = at_likely;
      }
      __syncthreads();
      uint32_t from = sh.keys[0], to = sh.keys[2];
      const float sure = top - (from - 0.501f) / scale;  // the border lies below
      if (value_of(least) > sure) {
        limit = least;
        __syncthreads();
        return kCut;
      }
      // so many entries about the likely one
      const int room = Sh::kRegion * 3 / 8, centre = (int)sh.amount;
      c = before;
      uint32_t low_bin = kMassBins - 1, high_bin = 0;
      for (int i = 0; i < kPer; ++i) {
        const uint32_t b = threadIdx.x * kPer + i;
        const int here = b + 1 < kMassBins ? sh.mass_counts[b] : 0;
        if (c >= centre - room) low_bin = min(low_bin, b);
        if (c + here <= centre + room) high_bin = max(high_bin, b);
        c += here;
      }
      low_bin = __reduce_min_sync(0xffffffffu, low_bin);
      high_bin = __reduce_max_sync(0xffffffffu, high_bin);
      if (threadIdx.x == 0) sh.keys[4] = 0;
      __syncthreads();
      if (lane == 0) {
        atomicMin(&sh.keys[3], low_bin);
        atomicMax(&sh.keys[4], high_bin);
      }
      start_list();
      from = max(from, sh.keys[3]);
      to = min(to, sh.keys[4]);
      if (from > to || to >= kMassBins - 1) return kNot;
      const float high = top - (from - 0.5f) / scale, low = top - (to + 0.5f) / scale;  // the list: low < v <= high
      __syncthreads();  // the list takes the counts' place
      uint64_t sure_sum = 0, all = 0, some = 0;
      each_segment(
          [&](int chunk, const E& e) {
            unsigned about = 0;
#pragma unroll
            for (int j = 0; j < kV; ++j) {
              const float v = e.at(j);
              const uint64_t m = near_mass(v);
              all += m;
              if (v > high) some += m;
              else if (v > low) about |= 1u << j;
            }
            while (__any_sync(0xffffffffu, about)) {  // few lanes, and of those the most have one
              const int i = first_of(chunk) + __ffs(about) - 1;
              append(about != 0, about ? to_f32<T>(z[i]) : 0.f, i, Sh::kRegion);
              about &= about - 1;
            }
          },
          [&](int s) {
            some = warp_sum(some);
            sure_sum += some;
            if (lane == 0) sh.sums[s] = some;
            some = 0;
          });
      sure_sum = block_sum(sure_sum);
      all = block_sum(warp_sum(all));
      const int listed = sh.listed;
      if (listed > Sh::kRegion) return kNot;
      const uint64_t target = (uint64_t)__double2ull_ru(p.top_p * (double)all);
      // the list by 256 bins of their own, then the border's
      const float fine = low < high ? kSubBins / (high - low) : 0.f;
      const auto sub_of = [&](float v) { return min(max((int)((high - v) * fine), 0), kSubBins - 1); };
      constexpr int kOwn = Sh::kRegion / THREADS;
      uint64_t own[kOwn], masses[kOwn];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int at = threadIdx.x + i * THREADS;
        own[i] = at < listed ? sh.list[at] : 0;
        masses[i] = 0;
        if (own[i]) {
          masses[i] = mass(value_of(own[i]));
          const int b = sub_of(value_of(own[i]));
          add_to(&sh.sub_low[b], &sh.sub_high[b], masses[i]);
        }
      }
      start_list();
      if (warp == 0) {
        uint64_t m = sure_sum;
        int border = -1;
        for (int b = 0; b < kSubBins && border < 0 && m < target; b += 32) {
          const uint64_t here = (uint64_t)sh.sub_high[b + lane] << 32 | sh.sub_low[b + lane], up = warp_running(here, lane);
          const unsigned reached = __ballot_sync(0xffffffffu, m + up >= target);
          const int at = reached ? __ffs(reached) - 1 : 31;
          if (reached) border = b + at;
          m += __shfl_sync(0xffffffffu, reached ? up - here : up, at);
        }
        if (lane == 0) {
          sh.found = border;
          sh.limit = m;
        }
      }
      __syncthreads();
      const int border = sh.found;
      const uint64_t reached = sh.limit;
      if (border < 0) return kNot;  // not about the likely place
      const auto join = [&](uint64_t place, uint64_t m) {
        const unsigned chunk = (unsigned)(index_of(place) + shift) / kChunk, s = per_segment == 1 ? chunk : chunk / per_segment;
        uint32_t* sum = reinterpret_cast<uint32_t*>(&sh.sums[s]);
        if (place >= least) add_to(sum, sum + 1, m);
      };
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int b = own[i] ? sub_of(value_of(own[i])) : kSubBins;
        if (b < border) join(own[i], masses[i]);
        append(b == border, own[i], Sh::kRegion);
      }
      __syncthreads();
      const int last = sh.listed;
      sort(last);
      const uint64_t at = limit_of_list(last, reached, target);
      for (int i = threadIdx.x; i < last; i += THREADS)
        if (sh.list[i] >= at) join(sh.list[i], mass(value_of(sh.list[i])));
      limit = max(at, least);
      __syncthreads();
      // the sums hold all above the list: where min_p cuts some of those too, they come again (in few rows: 1024 x 131072 bf16, top-p
      // 0.95 and min-p 0.02 take 196 us)
      return value_of(least) > high ? kCut : kSummed;
    } else {
      return kNot;
    }
  }

  // The first `need` of the entries from `limit` on (BY_MASS: those before which less than `share` of their mass lies) by
  // histograms over their keys: the new limit.
  template <bool BY_MASS>
  __device__ __forceinline__ void narrow(long long need, double share) {
    if constexpr (Sh::kLong) {
      uint32_t lo = (uint32_t)(limit >> 32), hi = key_of(top);
      uint64_t above_mass = 0, target = 0;
      long long above_count = 0;
      bool have_target = !BY_MASS;
      for (;;) {
        int bin_bits = 0;
        while ((hi - lo) >> bin_bits >= kBins) ++bin_bits;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += THREADS) sh.counts[i] = sh.low[i] = sh.high[i] = 0;
        __syncthreads();
        const float bottom = of_key(lo), ceiling = of_key(hi);
        each_reaching(bottom, [&](int chunk, const E& e) {
          const int first = first_of(chunk);
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const float v = clean(e.at(j));
            if (!(v >= bottom && v <= ceiling) || !kept(v, first + j)) continue;
            const uint32_t b = (key_of(v) - lo) >> bin_bits;
            atomicAdd(&sh.counts[b], 1u);
            if (BY_MASS) add_to(&sh.low[b], &sh.high[b], mass(v));
          }
        });
        __syncthreads();
        // from the largest bin down: the one with the border
        if (warp == 0) {
          const auto mass_of = [&](int b) { return (uint64_t)sh.high[b] << 32 | sh.low[b]; };
          constexpr int kPer = kBins / 32;
          uint64_t ms = 0;
          long long cs = 0;
          for (int i = 0; i < kPer; ++i) {  // lane 0: the largest bins
            const int b = kBins - 1 - (lane * kPer + i);
            cs += sh.counts[b];
            if (BY_MASS) ms += mass_of(b);
          }
          const uint64_t m_up = warp_running(ms, lane);
          if (!have_target) target = (uint64_t)__double2ull_ru(share * (double)__shfl_sync(0xffffffffu, m_up, 31));
          // the border lies in the bin at which the sum reaches what is asked for
          int at = -1;
          uint64_t m = above_mass + m_up - ms;
          long long c = above_count + warp_running(cs, lane) - cs;
          for (int i = 0; i < kPer && at < 0; ++i) {
            const int b = kBins - 1 - (lane * kPer + i);
            const uint32_t count = sh.counts[b];
            if (count && (BY_MASS ? m < target && m + mass_of(b) >= target : c < need && c + count >= need)) at = b;
            else m += BY_MASS ? mass_of(b) : 0, c += count;
          }
          const unsigned who = __ballot_sync(0xffffffffu, at >= 0);
          if (who ? lane == __ffs(who) - 1 : lane == 0) {
            sh.found = at;
            sh.limit = m;
            sh.amount = c;
          }
          if (lane == 0) sh.keys[0] = (uint32_t)target, sh.keys[1] = (uint32_t)(target >> 32);
        }
        __syncthreads();
        const int bin = sh.found;
        if (BY_MASS) target = (uint64_t)sh.keys[1] << 32 | sh.keys[0];
        have_target = true;
        if (bin < 0) return;  // everything
        above_mass = sh.limit;
        above_count = sh.amount;
        const uint32_t in_bin = sh.counts[bin];
        lo += (uint32_t)bin << bin_bits;
        hi = bin_bits ? min(hi, lo + ((1u << bin_bits) - 1)) : lo;
        if (in_bin <= Sh::kRegion) break;
        if (lo == hi) {  // so many ties: the first by index
          const uint64_t m = mass(of_key(lo));
          long long ties = need - above_count;
          if (BY_MASS) ties = m ? (long long)((target - above_mass + m - 1) / m) : in_bin;
          nth_tie(lo, ties);
          return;
        }
      }
      // the entries of the bin with the border, sorted
      start_list();
      const float bottom = of_key(lo), ceiling = of_key(hi);
      each_reaching(bottom, [&](int chunk, const E& e) {
        const int first = first_of(chunk);
#pragma unroll
        for (int j = 0; j < kV; ++j) {
          const float v = clean(e.at(j));
          append(v >= bottom && v <= ceiling && kept(v, first + j), v, first + j, Sh::kRegion);
        }
      });
      __syncthreads();
      const int count = sh.listed;
      sort(count);
      if (BY_MASS) limit = limit_of_list(count, above_mass, target);
      else limit = sh.list[max(1, (int)min((long long)count, need - above_count)) - 1];
      __syncthreads();
    }
  }
  // The limit that keeps the first `ties` entries of a key (and all larger ones).
  __device__ __forceinline__ void nth_tie(uint32_t key, long long ties) {
    const auto count_in = [&](int first, const E& e) {
      int count = 0;
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const float v = clean(e.at(j));
        count += key_of(v) == key && kept(v, first + j);
      }
      return count;
    };
    uint64_t some = 0;
    each_segment([&](int chunk, const E& e) { some += count_in(first_of(chunk), e); },
                 [&](int s) {
                   some = warp_sum(some);
                   if (lane == 0) sh.sums[s] = some;
                   some = 0;
                 });
    __syncthreads();
    if (warp == 0) {
      long long left = ties;
      int s = 0;
      while (s < segments - 1 && (long long)sh.sums[s] < left) left -= (long long)sh.sums[s++];
      int at = -1;
      for (int c = s * per_segment; c < min((s + 1) * per_segment, chunks) && at < 0; ++c) {
        const E e = fetch(c);
        const int first = first_of(c);
        const int mine = count_in(first, e), up = warp_running(mine, lane);
        if (up - mine < left && up >= left) {
          long long k = left - (up - mine);
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const float v = clean(e.at(j));
            if (key_of(v) == key && kept(v, first + j) && --k == 0) at = first + j;
          }
        }
        at = __reduce_max_sync(0xffffffffu, at);
        left -= __shfl_sync(0xffffffffu, up, 31);
      }
      if (lane == 0) sh.limit = place_of(key, at < 0 ? n : at);
    }
    __syncthreads();
    limit = sh.limit;
    __syncthreads();
  }

  __device__ __forceinline__ void none(long long row) {
    for (int d = threadIdx.x; d < p.draws; d += THREADS) {
      p.tokens[row * p.draws + d] = -1;
      if (p.probs) p.probs[row * p.draws + d] = 0.f;
    }
  }
  // The list holds the first top_k entries and maybe others: by rank, cut by top-p and min-p, then by index.
  __device__ __forceinline__ void draw_listed(long long row, uint64_t least) {
    const int listed = sh.listed, count = min(listed, p.top_k);
    sort(listed);
    int m = count;
    if (p.top_p < 1.0) {
      for (int i = threadIdx.x; i < count; i += THREADS) sh.masses[i] = mass(value_of(sh.list[i]));
      __syncthreads();
      const uint64_t all = scan(sh.masses, count), target = (uint64_t)__double2ull_ru(p.top_p * (double)all);
      m = above(sh.masses, count, target - 1) + 1;  // the first sum that reaches the target is the last one kept
    }
    for (int i = threadIdx.x; i < m; i += THREADS) {  // by index from the lowest: descending again
      const uint64_t place = sh.list[i];
      sh.list[i] = place << 32 | place >> 32;
    }
    __syncthreads();
    sort(m);
    for (int i = threadIdx.x; i < m; i += THREADS) {
      const uint64_t place = sh.list[i] << 32 | sh.list[i] >> 32;
      sh.masses[i] = place >= least ? mass(value_of(place)) : 0;
    }
    __syncthreads();
    const uint64_t total = scan(sh.masses, m);
    for (int d = threadIdx.x; d < p.draws; d += THREADS) {
      const long long at = row * p.draws + d;
      const int i = above(sh.masses, m, threshold(p.uniforms[at], total));
      p.tokens[at] = index_of(sh.list[i] >> 32);
      if (p.probs) p.probs[at] = (float)((double)(sh.masses[i] - (i ? sh.masses[i - 1] : 0)) / (double)total);
    }
  }
  // The kept entries are those from `limit` on: sums of segments (unless they are there), then a look through the
  // segment of each draw.
  __device__ __forceinline__ void draw_row(long long row, bool summed) {
    const float least = value_of(limit);
    const bool all = limit == kPossible;
    uint64_t some = 0;
    const auto done = [&](int s) {
      some = warp_sum(some);
      if (lane == 0) sh.sums[s] = some;
      some = 0;
    };
    if (!summed && all && !far)
      each_segment(
          [&](int, const E& e) {
#pragma unroll
            for (int j = 0; j < kV; ++j) some += near_mass(e.at(j));
          },
          done);
    else if (!summed)
      for (int s = warp; s < segments; s += kWarps) {
        for (int c = s * per_segment; c < min((s + 1) * per_segment, chunks); ++c) {
          if (!reaches(c, least)) continue;
          const E e = fetch(c);
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const float v = clean(e.at(j));
            if (v >= least && kept(v, first_of(c) + j)) some += mass(v);
          }
        }
        done(s);
      }
    __syncthreads();
    const uint64_t total = scan(sh.sums, segments);
    for (int d = warp; d < p.draws; d += kWarps) {
      const long long at = row * p.draws + d;
      const uint64_t t = threshold(p.uniforms[at], total);
      const int s = above(sh.sums, segments, t), end = min((s + 1) * per_segment, chunks);
      uint64_t sum = s ? sh.sums[s - 1] : 0;
      int last = -1;  // the last class of the walk that can be drawn
      uint64_t last_mass = 0;
      bool drawn = false;
      for (int c = s * per_segment; c < end && sum <= t; ++c) {
        const E e = fetch(c);
        const int first = first_of(c);
        uint64_t own[kV], mine = 0;
#pragma unroll
        for (int j = 0; j < kV; ++j) {
          const float v = clean(e.at(j));
          mine += own[j] = kept(v, first + j) ? mass(v) : 0;
          if (own[j]) last = first + j, last_mass = own[j];
        }
        const uint64_t up = warp_running(mine, lane);
        uint64_t run = sum + up - mine;
        sum += __shfl_sync(0xffffffffu, up, 31);
        if (run <= t && t < run + mine) {  // one lane
          drawn = true;
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            if (run <= t && t < run + own[j]) {
              p.tokens[at] = first + j;
              if (p.probs) p.probs[at] = (float)((double)own[j] / (double)total);
            }
            run += own[j];
          }
        }
      }
      // the walk ends with a class, as its sums are the segment's; no output stays unwritten if one were off
      if (!__any_sync(0xffffffffu, drawn)) {
        const int best = __reduce_max_sync(0xffffffffu, last);
        if (last == best && (best >= 0 || lane == 0)) {
          p.tokens[at] = best;
          if (p.probs) p.probs[at] = (float)((double)last_mass / (double)total);
        }
      }
    }
  }
};

// A k up to this is found through groups: the k-th largest of 2 k maxima or more leaves about 1.4 k entries.
constexpr int kSmallK = 256;

template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) sample_row_kernel(const __grid_constant__ SampleParams p) {
  may_start_next();
  after_previous();
  extern __shared__ __align__(16) uint8_t smem[];
  auto& sh = *reinterpret_cast<RowShared<THREADS>*>(smem);
  using R = Row<T, THREADS>;
  R r(p, sh, blockIdx.x);
  const bool cut_k = p.top_k < p.classes, cut_p = p.top_p < 1.0;
  const bool small_k = cut_k && p.top_k <= min(kSmallK, THREADS / 2);
  int groups = 1;
  while (small_k && groups < 2 * p.top_k) groups <<= 1;
  float bound = __int_as_float(0xff800000);
  const float top = r.largest(small_k ? p.top_k : 0, groups, bound);
  if (!possible(top)) {
    r.none(blockIdx.x);
    return;
  }
  r.set_top(top);
  if (R::Sh::kLong && p.classes > kKnown) r.fit_one();
  const uint64_t least = p.min_p > 0.0 ? r.limit_of_weight(p.min_p) : kPossible;
  const bool middle_k = cut_k && !small_k && p.classes > R::Sh::kList && p.top_k <= R::Sh::kList * 3 / 4 &&
                        top < __int_as_float(0x7f800000);
  if (middle_k) bound = r.bound_by_count(p.top_k);
  if (small_k || possible(bound) || ((cut_k || cut_p) && p.classes <= R::Sh::kList)) {
    r.start_list();
    r.each_reaching(bound, [&](int chunk, const typename R::E& e) {
      const int first = r.first_of(chunk);
#pragma unroll
      for (int j = 0; j < R::kV; ++j) {
        const float v = clean(e.at(j));
        r.append(v >= bound && possible(v), v, first + j, R::Sh::kList);
      }
    });
    __syncthreads();
    if (sh.listed <= R::Sh::kList && (!middle_k || sh.listed >= p.top_k)) {
      r.draw_listed(blockIdx.x, least);
      return;
    }
  }
  if (cut_k) r.template narrow<false>(p.top_k, 1.0);
  int cut = R::kNot;
  if (cut_p) {
    if (!cut_k && !r.far) cut = r.cut_mass(least);
    if (cut == R::kNot) r.template narrow<true>(0, p.top_p);
  }
  r.limit = max(r.limit, least);
  r.draw_row(blockIdx.x, cut == R::kSummed);
}

// --------------------------------------------------------------------------------------- host side
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

template <class T, int G>
int32_t few(const SampleParams& p, cudaStream_t s) {
  const long long blocks = ceil_div(p.rows, 256 / G);
  if (blocks > (1ll << 31) - 1) return NCA_ERR_UNSUPPORTED;
  return launch_after(sample_few_kernel<T, G>, dim3((unsigned)blocks), dim3(256), 0, s, 1, p);
}
template <class T, int C>
int32_t tiny(const SampleParams& p, cudaStream_t s) {
  const long long blocks = ceil_div(p.rows, 256);
  if (blocks > (1ll << 31) - 1) return NCA_ERR_UNSUPPORTED;
  return launch_after(sample_tiny_kernel<T, C>, dim3((unsigned)blocks), dim3(256), 0, s, 1, p);
}
template <class T, int THREADS>
int32_t row_blocks(const SampleParams& p, cudaStream_t s) {
  if (p.rows > (1ll << 31) - 1) return NCA_ERR_UNSUPPORTED;
  auto* kernel = sample_row_kernel<T, THREADS>;
  constexpr size_t bytes = sizeof(RowShared<THREADS>);
  static std::atomic<uint64_t> ready{0};  // a bit for each device whose shared-memory limit is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NCA_ERR_DEVICE;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
      return launch_status() == NCA_OK ? NCA_ERR_CUDA : NCA_ERR_DEVICE;
    ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  return launch_after(kernel, dim3((unsigned)p.rows), dim3(THREADS), bytes, s, 1, p);
}

}  // namespace

extern "C" int32_t nca_b200_sample(const NcaSampleDesc* d, const void* logits, const float* uniforms, int64_t* tokens,
                                   float* probs, void* stream) {
  if (!d || d->rows < 0 || d->classes <= 0 || d->draws < 0 || d->top_k < 0 || !dtype_ok(d->dtype)) return NCA_ERR_INVALID;
  if (!(d->temperature >= 0) || !(d->temperature <= 1e30) || (d->temperature > 0 && d->temperature < 1e-30) ||
      !(d->top_p > 0 && d->top_p <= 1) || !(d->min_p >= 0 && d->min_p <= 1))
    return NCA_ERR_INVALID;
  if (d->classes > (1ll << 30) || d->draws > (1ll << 30) || d->rows > (1ll << 40)) return NCA_ERR_UNSUPPORTED;
  if (d->rows == 0 || d->draws == 0) return NCA_OK;
  if (!logits || !uniforms || !tokens) return NCA_ERR_INVALID;
  SampleParams p{};
  p.logits = logits;
  p.uniforms = uniforms;
  p.tokens = reinterpret_cast<long long*>(tokens);
  p.probs = probs;
  p.rows = d->rows;
  p.stride = d->logits_stride;
  p.classes = (int)d->classes;
  p.draws = (int)d->draws;
  // temperature 0: the first of the largest
  p.top_k = d->temperature == 0 ? 1 : d->top_k == 0 ? p.classes : (int)std::min<int64_t>(d->top_k, d->classes);
  p.inverse_t = d->temperature == 0 ? 1.0 : 1.0 / d->temperature;
  p.top_p = d->top_p;
  p.min_p = d->min_p;
  int bits = 51;  // the sum of all weights stays below 2^62; beyond kKnown classes the rows' own sums decide
  while (std::min<int64_t>(d->classes, kKnown) > (1ll << (62 - bits))) --bits;
  p.one = (double)(1ll << bits);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return with_dtype(d->dtype, [&](auto t) -> int32_t {
    using T = decltype(t);
    if (p.classes <= 4 && p.draws <= 4) return p.classes <= 2 ? tiny<T, 2>(p, s) : tiny<T, 4>(p, s);
    if (p.classes <= 2) return few<T, 2>(p, s);
    if (p.classes <= 4) return few<T, 4>(p, s);
    if (p.classes <= 8) return few<T, 8>(p, s);
    if (p.classes <= 16) return few<T, 16>(p, s);
    if (p.classes <= 32) return few<T, 32>(p, s);
    // Smaller blocks, more rows at once, hide each other's short steps (2047 x 32003 fp16, top-k 50: 93 against 127 us, without cuts 104
    // against 122); top-p alone has few of them and works through its list faster in large ones (1024 x 20000 bf16, top-p 0.95: 110
    // against 121, 1024 x 131072 365 against 387), as longer rows do (131072 without cuts 190 against 199, min-p alone 126 against 134;
    // top-k 50 is the exception, 117 against 110).
    if (p.classes <= RowShared<128>::kList) return row_blocks<T, 128>(p, s);
    const bool by_mass = p.top_p < 1.0 && p.top_k == p.classes;
    return p.classes <= 65536 && !by_mass ? row_blocks<T, 256>(p, s) : row_blocks<T, 512>(p, s);
  });
}
