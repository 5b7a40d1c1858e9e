// sample.cu -- classes drawn from rows of logits with given uniform numbers (nca_b200_sample): temperature, top-k,
// top-p, min-p.
//
// With w_i = exp((z_i - max z) / T), classes in the order of z (largest first, ties by index): the first top_k; of
// those, the ones before which less than top_p of their mass lies; of those, the ones with w_i >= min_p.  A draw is
// the first class, by index, at which the sum of the kept w exceeds u times the whole.
//
// The answers are whole numbers, and a row of 131072 classes has a border every 1e-5 of its mass: weights are computed in
// 64 bits, so that an answer other than the exact one takes a u within about 1e-13 of a border.  Sums are in fixed
// point: they do not depend on an order, and a class of no mass is never drawn.  The exponential is table-driven
// (Tang, ACM TOMS 15, 1989): 2^(j / 64) from a table, e^r of |r| < 0.0055 by four terms, 9 operations in 64 bits.
//
// Up to 32 classes a row is a group of lanes, a class a lane, and ranks are counted.  Longer rows are a block's: the kept
// set is always "above a threshold (z, index)".  A small top_k: the least of k groups' maxima bounds the k-th largest
// from below, the few entries above it are listed and sorted.  Else histograms over the ordered bits of z (counts, masses)
// until the entries of the bin with the border can be listed.
// Segments of 256 entries, a warp each, then sum the kept weights, and a draw looks through one segment.
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
  double one;              // a weight of 1 in fixed point
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

// ------------------------------------------------------------------------------- up to 32 classes
template <class T, int G>
__global__ void __launch_bounds__(256) sample_few_kernel(const __grid_constant__ SampleParams p) {
  may_start_next();
  after_previous();
  __shared__ uint64_t sums[256];
  const int lane = threadIdx.x % G, base = threadIdx.x - lane;
  const long long row = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool here = row < p.rows && lane < p.classes;
  const unsigned all = 0xffffffffu;
  const float v = here ? clean(to_f32<T>(static_cast<const T*>(p.logits)[row * p.stride + lane])) : clean(__int_as_float(0x7fc00000));
  float top = v;
#pragma unroll
  for (int o = G / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(all, top, o));
  double weight = v == top ? 1.0 : exp(((double)v - (double)top) * p.inverse_t);
  if (!possible(v)) weight = 0.0;
  uint64_t w = fixed(weight, p.one);
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
  if (!(weight >= p.min_p)) w = 0;
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
constexpr int kBins = 2048;
constexpr int kMostSegments = 1024;

// Floats in their order as whole numbers.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// Its place in the order: larger first, then the lower index.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int i) { return (uint64_t)key << 32 | (0xffffffffu - (uint32_t)i); }
__device__ __forceinline__ int index_of(uint64_t place) { return (int)(0xffffffffu - (uint32_t)place); }

template <int THREADS>
struct RowShared {
  static constexpr int kList = THREADS >= 512 ? 2048 : 1024;
  double table[64];
  uint64_t sums[kMostSegments];
  uint64_t warp_sums[32];
  uint64_t list[kList];
  union {
    uint64_t masses[kList];
    uint32_t counts[kBins];
  };
  uint32_t low[kBins], high[kBins];  // masses of the bins, in fixed point
  float reds[64];
  uint32_t keys[64];
  int listed, found;
  uint64_t limit;
  long long amount;
};

template <class T, int THREADS>
struct Row {
  using Sh = RowShared<THREADS>;
  static constexpr int kWarps = THREADS / 32;
  const SampleParams& p;
  Sh& sh;
  const T* z;
  int n, shift, chunks, per_segment, segments;  // chunks of 256 entries; of a segment
  float top;
  uint64_t limit;  // places from here on up are kept
  int warp, lane;

  __device__ __forceinline__ Row(const SampleParams& p_, Sh& sh_, long long row) : p(p_), sh(sh_) {
    z = static_cast<const T*>(p.logits) + row * p.stride;
    n = p.classes;
    shift = (int)(reinterpret_cast<uintptr_t>(z) % 16 / sizeof(T));  // chunks start on 16-byte boundaries
    chunks = (n + shift + 255) / 256;
    per_segment = (chunks + kMostSegments - 1) / kMostSegments;
    segments = (chunks + per_segment - 1) / per_segment;
    limit = 0;
    warp = threadIdx.x / 32;
    lane = threadIdx.x % 32;
  }
  // This lane's 8 entries of a chunk, from entry `first` on; entries outside of the row are -inf.
  __device__ __forceinline__ int fetch(int chunk, float (&v)[8]) const {
    const int first = chunk * 256 + lane * 8 - shift;
    if (first >= 0 && first + 8 <= n) {
      constexpr int V = 16 / sizeof(T);
#pragma unroll
      for (int k = 0; k < 8 / V; ++k) {
        const Vec<T, V> q = *reinterpret_cast<const Vec<T, V>*>(z + first + k * V);
#pragma unroll
        for (int j = 0; j < V; ++j) v[k * V + j] = clean(to_f32<T>(q.v[j]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = first + j >= 0 && first + j < n ? clean(to_f32<T>(z[first + j])) : __int_as_float(0xff800000);
    }
    return first;
  }
  // exp((v - top) / T) of a possible v
  __device__ __forceinline__ double weight(float v) const {
    if (v == top) return 1.0;
    constexpr double kMagic = 6755399441055744.0;  // 1.5 2^52: the sum's low bits are the nearest whole number
    const double x = ((double)v - (double)top) * (p.inverse_t * 92.332482616893656770);  // 64 log2(e)
    if (!(x > -64.0 * 1000)) return 0.0;
    const double m = x + kMagic;
    const int k = __double2loint(m);
    const double r = x - (m - kMagic);
    constexpr double c = 0.010830424696249145;  // ln(2) / 64
    const double q = r * (c + r * (c * c / 2 + r * (c * c * c / 6 + r * (c * c * c * c / 24))));
    const double t = sh.table[k & 63];
    const double e = fma(t, q, t);
    return __hiloint2double(__double2hiint(e) + ((k >> 6) << 20), __double2loint(e));
  }
  __device__ __forceinline__ bool kept(float v, int i) const { return possible(v) && place_of(key_of(v), i) >= limit; }

  template <class F>
  __device__ __forceinline__ void each_chunk(F fn) const {
    for (int c = warp; c < chunks; c += kWarps) {
      float v[8];
      const int first = fetch(c, v);
      fn(first, v);
    }
  }
  __device__ __forceinline__ uint64_t mass(float v) const { return fixed(weight(v), p.one); }
  // Running sums of a[0 .. count) in place; returns the whole.
  __device__ __forceinline__ uint64_t scan(uint64_t* a, int count) {
    uint64_t carry = 0;
    for (int b = 0; b < count; b += THREADS) {
      const int i = b + threadIdx.x;
      uint64_t s = i < count ? a[i] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t below = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += below;
      }
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
  // list[0 .. size), size a power of two, to descending order
  __device__ __forceinline__ void sort(int size) {
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
  __device__ __forceinline__ int padded() {  // the list filled up with places below all others
    const int c = sh.listed;
    int size = 2;
    while (size < c) size <<= 1;
    for (int i = c + threadIdx.x; i < size; i += THREADS) sh.list[i] = 0;
    return size;
  }
  __device__ __forceinline__ void append(uint64_t place) {
    const int at = atomicAdd(&sh.listed, 1);
    if (at < Sh::kList) sh.list[at] = place;
  }

  // The largest entry; with `groups` (a power of two, at most THREADS) also a bound that so many entries reach.
  __device__ __forceinline__ float largest(int groups, float& bound) {
    float m = __int_as_float(0xff800000);
    each_chunk([&](int, const float (&v)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, v[j]);
    });
    const int wide = THREADS / groups;  // threads of a group
    for (int o = 1; o < min(wide, 32); o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float least = m;
    for (int o = min(wide, 32); o < 32; o <<= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
    }
    __syncthreads();
    if (lane == 0) {
      sh.reds[warp] = m;
      sh.reds[32 + warp] = least;
    }
    __syncthreads();
    const int warps = max(wide / 32, 1);  // of a group
    bound = __int_as_float(0x7f800000);
    for (int g = 0; g < kWarps; g += warps) {
      float most = __int_as_float(0xff800000);
      if (warps == 1) most = sh.reds[32 + g];
      else
        for (int w = 0; w < warps; ++w) most = fmaxf(most, sh.reds[g + w]);
      bound = fminf(bound, most);
    }
    m = sh.reds[0];
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sh.reds[w]);
    return m;
  }

  // The first `need` of the entries from `limit` on (BY_MASS: those before which less than `share` of their mass lies) by
  // histograms over their keys: the new limit.
  template <bool BY_MASS>
  __device__ __forceinline__ void narrow(long long need, double share) {
    uint32_t lo, hi;
    {  // the range of the keys
      uint32_t a = 0xffffffffu, b = 0;
      each_chunk([&](int first, const float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (kept(v[j], first + j)) a = min(a, key_of(v[j])), b = max(b, key_of(v[j]));
      });
      a = __reduce_min_sync(0xffffffffu, a);
      b = __reduce_max_sync(0xffffffffu, b);
      __syncthreads();
      if (lane == 0) sh.keys[warp] = a, sh.keys[32 + warp] = b;
      __syncthreads();
      lo = sh.keys[0], hi = sh.keys[32];
      for (int w = 1; w < kWarps; ++w) lo = min(lo, sh.keys[w]), hi = max(hi, sh.keys[32 + w]);
    }
    uint64_t above_mass = 0, target = 0;
    long long above_count = 0;
    bool have_target = !BY_MASS;
    for (;;) {
      int bin_bits = 0;
      while ((hi - lo) >> bin_bits >= kBins) ++bin_bits;
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += THREADS) sh.counts[i] = sh.low[i] = sh.high[i] = 0;
      __syncthreads();
      each_chunk([&](int first, const float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t key = key_of(v[j]);
          if (key < lo || key > hi || !kept(v[j], first + j)) continue;
          const uint32_t b = (key - lo) >> bin_bits;
          atomicAdd(&sh.counts[b], 1u);
          if (BY_MASS) {
            const uint64_t m = mass(v[j]);
            const uint32_t l = (uint32_t)m;
            uint32_t h = (uint32_t)(m >> 32);
            const uint32_t old = atomicAdd(&sh.low[b], l);
            if (old + l < old) ++h;  // the carry
            if (h) atomicAdd(&sh.high[b], h);
          }
        }
      });
      __syncthreads();
      // from the largest bin down: the one with the border (a thread; the loops over the row cost far more)
      if (warp == 0) {
        const auto mass_of = [&](int b) { return (uint64_t)sh.high[b] << 32 | sh.low[b]; };
        constexpr int kPer = kBins / 32;
        uint64_t ms = 0;
        uint32_t cs = 0;
        for (int i = 0; i < kPer; ++i) {  // lane 0: the largest bins
          const int b = kBins - 1 - (lane * kPer + i);
          cs += sh.counts[b];
          if (BY_MASS) ms += mass_of(b);
        }
        uint64_t m_before = 0, m_all = 0;
        uint32_t c_before = 0;
        for (int w = 0; w < 32; ++w) {
          const uint64_t mw = __shfl_sync(0xffffffffu, ms, w);
          const uint32_t cw = __shfl_sync(0xffffffffu, cs, w);
          m_all += mw;
          if (w < lane) m_before += mw, c_before += cw;
        }
        if (!have_target) target = (uint64_t)__double2ull_ru(share * (double)m_all);
        // the border lies in the bin at which the sum reaches what is asked for; in the last that holds anything otherwise
        int at = -1;
        uint64_t m = above_mass + m_before;
        long long c = above_count + c_before;
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
      __syncthreads();
      if (in_bin <= Sh::kList) break;
      if (lo == hi) {  // so many ties: the first by index
        const uint64_t m = mass(of_key(lo));
        long long ties = need - above_count;
        if (BY_MASS) ties = m ? (long long)((target - above_mass + m - 1) / m) : in_bin;
        nth_tie(lo, ties);
        return;
      }
    }
    // the entries of the bin with the border, sorted
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    each_chunk([&](int first, const float (&v)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t key = key_of(v[j]);
        if (key >= lo && key <= hi && kept(v[j], first + j)) append(place_of(key, first + j));
      }
    });
    __syncthreads();
    const int count = sh.listed;
    sort(padded());
    if (warp == 0) {
      int taken = BY_MASS ? 0 : (int)min((long long)count, need - above_count);
      uint64_t m = above_mass;
      for (int b = 0; BY_MASS && b < count; b += 32) {
        const uint64_t own = b + lane < count ? mass(of_key((uint32_t)(sh.list[b + lane] >> 32))) : 0;
        uint64_t up = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t below = __shfl_up_sync(0xffffffffu, up, o);
          if (lane >= o) up += below;
        }
        const unsigned in = __ballot_sync(0xffffffffu, b + lane < count && m + up - own < target);
        taken += __popc(in);
        m += __shfl_sync(0xffffffffu, up, 31);
        if (in != 0xffffffffu) break;
      }
      if (lane == 0) sh.limit = sh.list[max(taken, 1) - 1];
    }
    __syncthreads();
    limit = sh.limit;
    __syncthreads();
  }
  // The limit that keeps the first `ties` entries of a key (and all larger ones).
  __device__ __forceinline__ void nth_tie(uint32_t key, long long ties) {
    for (int s = warp; s < segments; s += kWarps) {
      int count = 0;
      for (int c = s * per_segment; c < min((s + 1) * per_segment, chunks); ++c) {
        float v[8];
        const int first = fetch(c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) count += key_of(v[j]) == key && kept(v[j], first + j);
      }
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 0) sh.sums[s] = count;
    }
    __syncthreads();
    if (warp == 0) {
      long long left = ties;
      int s = 0;
      while (s < segments - 1 && (long long)sh.sums[s] < left) left -= (long long)sh.sums[s++];
      int at = -1;
      for (int c = s * per_segment; c < min((s + 1) * per_segment, chunks) && at < 0; ++c) {
        float v[8];
        const int first = fetch(c, v);
        int mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) mine += key_of(v[j]) == key && kept(v[j], first + j);
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int below = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += below;
        }
        const int all = __shfl_sync(0xffffffffu, sum, 31);
        if (sum - mine < left && sum >= left) {
          long long k = left - (sum - mine);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (key_of(v[j]) == key && kept(v[j], first + j) && --k == 0) at = first + j;
        }
        at = __reduce_max_sync(0xffffffffu, at);
        left -= all;
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
  // The kept entries are in the list: by rank, cut by top-p and min-p, then by index.
  __device__ __forceinline__ void draw_listed(long long row) {
    const int count = min(sh.listed, p.top_k);
    sort(padded());
    int m = count;
    if (p.top_p < 1.0) {
      for (int i = threadIdx.x; i < count; i += THREADS) sh.masses[i] = mass(of_key((uint32_t)(sh.list[i] >> 32)));
      __syncthreads();
      const uint64_t all = scan(sh.masses, count), target = (uint64_t)__double2ull_ru(p.top_p * (double)all);
      m = above(sh.masses, count, target - 1) + 1;  // the first sum that reaches the target is the last one kept
    }
    for (int i = threadIdx.x; i < m; i += THREADS) {  // by index from the lowest: descending again
      const uint64_t place = sh.list[i];
      sh.list[i] = (uint64_t)(uint32_t)place << 32 | (uint32_t)(place >> 32);
    }
    if (threadIdx.x == 0) sh.listed = m;
    __syncthreads();
    sort(padded());
    for (int i = threadIdx.x; i < m; i += THREADS) {
      const double w = weight(of_key((uint32_t)sh.list[i]));
      sh.masses[i] = w >= p.min_p ? fixed(w, p.one) : 0;
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
  // The kept entries are those from `limit` on: sums of segments, then a look through the segment of each draw.
  __device__ __forceinline__ void draw_row(long long row) {
    const auto share = [&](float v, int i) -> uint64_t {
      if (!kept(v, i)) return 0;
      const double w = weight(v);
      return w >= p.min_p ? fixed(w, p.one) : 0;
    };
    for (int s = warp; s < segments; s += kWarps) {
      uint64_t sum = 0;
      for (int c = s * per_segment; c < min((s + 1) * per_segment, chunks); ++c) {
        float v[8];
        const int first = fetch(c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += share(v[j], first + j);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) sh.sums[s] = sum;
    }
    __syncthreads();
    const uint64_t total = scan(sh.sums, segments);
    for (int d = warp; d < p.draws; d += kWarps) {
      const long long at = row * p.draws + d;
      const uint64_t t = threshold(p.uniforms[at], total);
      const int s = above(sh.sums, segments, t);
      uint64_t sum = s ? sh.sums[s - 1] : 0;
      for (int c = s * per_segment; c < min((s + 1) * per_segment, chunks); ++c) {
        float v[8];
        const int first = fetch(c, v);
        uint64_t own[8], up = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) up += own[j] = share(v[j], first + j);
        const uint64_t mine = up;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t below = __shfl_up_sync(0xffffffffu, up, o);
          if (lane >= o) up += below;
        }
        uint64_t run = sum + up - mine;
        sum += __shfl_sync(0xffffffffu, up, 31);
        if (run <= t && t < run + mine) {  // one lane
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (run <= t && t < run + own[j]) {
              p.tokens[at] = first + j;
              if (p.probs) p.probs[at] = (float)((double)own[j] / (double)total);
            }
            run += own[j];
          }
        }
        if (sum > t) break;
      }
    }
  }
};

// A k up to this is found through the groups' maxima: k groups leave about k ln k entries.
constexpr int kSmallK = 256;

template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS) sample_row_kernel(const __grid_constant__ SampleParams p) {
  may_start_next();
  after_previous();
  extern __shared__ __align__(16) uint8_t smem[];
  auto& sh = *reinterpret_cast<RowShared<THREADS>*>(smem);
  using R = Row<T, THREADS>;
  if (threadIdx.x < 64) sh.table[threadIdx.x] = exp2(threadIdx.x / 64.0);
  if (threadIdx.x == 0) sh.listed = 0;
  R r(p, sh, blockIdx.x);
  const bool cut_k = p.top_k < p.classes, cut_p = p.top_p < 1.0;
  const bool short_list = cut_k && p.top_k <= min(kSmallK, THREADS);
  int groups = 1;
  while (short_list && groups < p.top_k) groups <<= 1;
  float bound;
  r.top = r.largest(groups, bound);
  if (!possible(r.top)) {
    r.none(blockIdx.x);
    return;
  }
  __syncthreads();
  const bool whole = (cut_k || cut_p) && p.classes <= R::Sh::kList;  // all of the row in the list
  if (short_list || whole) {
    const float least = short_list ? bound : __int_as_float(0xff800000);
    r.each_chunk([&](int first, const float (&v)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (v[j] >= least && possible(v[j])) r.append(place_of(key_of(v[j]), first + j));
    });
    __syncthreads();
    if (sh.listed <= R::Sh::kList) {
      r.draw_listed(blockIdx.x);
      return;
    }
  }
  if (cut_k) r.template narrow<false>(p.top_k, 1.0);
  if (cut_p) r.template narrow<true>(0, p.top_p);
  r.draw_row(blockIdx.x);
}

// --------------------------------------------------------------------------------------- host side
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

template <class T, int G>
int32_t few(const SampleParams& p, cudaStream_t s) {
  const long long blocks = ceil_div(p.rows, 256 / G);
  if (blocks > (1ll << 31) - 1) return NCA_ERR_UNSUPPORTED;
  return launch_after(sample_few_kernel<T, G>, dim3((unsigned)blocks), dim3(256), 0, s, 1, p);
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
  int bits = 51;  // the sum of all weights stays below 2^62
  while (d->classes > (1ll << (62 - bits))) --bits;
  p.one = (double)(1ll << bits);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return with_dtype(d->dtype, [&](auto t) -> int32_t {
    using T = decltype(t);
    if (p.classes <= 2) return few<T, 2>(p, s);
    if (p.classes <= 4) return few<T, 4>(p, s);
    if (p.classes <= 8) return few<T, 8>(p, s);
    if (p.classes <= 16) return few<T, 16>(p, s);
    if (p.classes <= 32) return few<T, 32>(p, s);
    return p.classes <= 4096 ? row_blocks<T, 128>(p, s) : row_blocks<T, 512>(p, s);
  });
}
