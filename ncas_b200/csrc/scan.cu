// scan.cu -- the gated scan h_t = a_t h_{t-1} + (1 - a_t) x_t, a = sigmoid(gate), along one axis, forward
// and backward (nca_b200_gated_scan*).
//
// With e = exp(gate), 1 - a is 1 / (1 + e), and a is e / (1 + e) up to 1/2 and 1 less the former from there on: both with full
// relative precision, and a the nearest fp32 where the former is small, so that open gates hold a state.  States, products
// and sums are fp32.
//
// Steps compose as maps h -> P h + H (P the product of the a), so a line can be cut anywhere.  A thread
// owns two adjacent 16-bit channels (or one channel) of kSub adjacent steps, all of which it holds in
// registers.  Where lines and channels fill the GPU, a thread walks along its line alone.  If they are that many and short, it
// takes 16 bytes of every row instead (8 backward): the work a row and a line costs besides is shared by more channels.  Else the
// threads of a block's warps split a stretch of the line: each builds its steps' maps from the identity on, the
// warps exchange the last through shared memory, and y_t = P_t h + H_t from the state h before the thread's
// steps.  Blocks walk along the line and load the next stretch while they work on this one.  Where that does not fill
// the GPU either, the line is cut into pieces for different blocks: a first kernel computes the
// pieces' maps, at the price of a second read.  Backward: G_t = dy_t + a_{t+1} G_{t+1} is the same scan
// from the end; the states come again from the inputs, from the state that the forward pass stored before
// each kSub steps (4 bytes for kSub elements).
//
// 72000 lines of 9 steps, 64 channels, bf16 take 44 us forward and 94 backward (87 and 67 % of the HBM rate; with two channels
// a thread 62 and 115 where these took 43 and 89, before `a` had its present form), 100000 single steps of 504 channels 93 and 217
// (two channels: 389 and 690).  One line of 100001 steps, 1024 channels takes 203 us forward (87 of them for the pieces' maps) and 289
// backward (88), at 55 to 62 % of the DRAM cycles and 57 to 67 % of the issue slots; with 16 steps a thread 217 and 331, for their
// registers.  Passes in a row take 580 to 595 in all, 80 to 100 more than the two alone: a kernel that starts while the one before
// ends settles on the multiprocessors that are free first, up to 8 blocks on one, and its grid holds no more than 5 for each (510 to
// 530 where every kernel waits for the one before).
#include "cell_ops.cuh"

#include <algorithm>

using namespace nca;

namespace {

constexpr int kSub = 8;             // steps of a thread
constexpr int kLanes = 32;           // columns of a block whose warps split a line
constexpr int kThreads = 128;
constexpr int kBlocksAlone = 8, kBlocks = 5, kBlocksBack = 4;  // of a multiprocessor, by their registers
constexpr int kMostPieces = 128;

struct ScanParams {
  const void *x, *gate, *dy;
  const float *state, *dlast;
  const uint8_t* mask;
  void *y, *dx, *dgate;
  float *last, *dstate;
  float* saved;        // states before steps kSub, 2 kSub, ... [lines][marks][channels]
  float *agg_p, *agg_h;  // maps of the pieces [pieces][lines][channels]
  long long m, steps, lines, columns, marks;
  long long stretches, per;  // stretches of subs * kSub steps; those of a piece
  int channels, per_line;    // columns of a line
  int subs, pieces, block_columns;
  long long xs[3], gs[3], ds[3], ys[3], ms[3];  // strides of (n, m, step); those of the step negative in a reversed scan
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The channels of a thread: one, or two whose operations go in pairs.
template <int V>
struct Ch;
template <>
struct Ch<1> {
  using F = float;
  static __device__ __forceinline__ F of(float v) { return v; }
  static __device__ __forceinline__ F add(F a, F b) { return a + b; }
  static __device__ __forceinline__ F mul(F a, F b) { return a * b; }
  static __device__ __forceinline__ F fma(F a, F b, F c) { return fmaf(a, b, c); }
  template <class O>
  static __device__ __forceinline__ F each(F a, O o) { return o(a); }
  // b where g is not negative (its sign bit), else c
  static __device__ __forceinline__ F pick(F g, F b, F c) { return __float_as_int(g) >= 0 ? b : c; }
};
template <>
struct Ch<2> {
  using F = float2;
  static __device__ __forceinline__ F of(float v) { return both(v); }
  static __device__ __forceinline__ F add(F a, F b) { return add2(a, b); }
  static __device__ __forceinline__ F mul(F a, F b) { return mul2(a, b); }
  static __device__ __forceinline__ F fma(F a, F b, F c) { return fma2(a, b, c); }
  template <class O>
  static __device__ __forceinline__ F each(F a, O o) { return make_float2(o(a.x), o(a.y)); }
  static __device__ __forceinline__ F pick(F g, F b, F c) { return make_float2(Ch<1>::pick(g.x, b.x, c.x), Ch<1>::pick(g.y, b.y, c.y)); }
};

template <class T, int V>
__device__ __forceinline__ typename Ch<V>::F take(uint32_t v) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(v);
  } else {
    float2 t;
    if constexpr (__is_same(T, __nv_bfloat16)) t = make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    else t = __half22float2(reinterpret_cast<const __half2&>(v));
    if constexpr (V == 2) return t;
    else return t.x;
  }
}
// keep = 1 - a, and a.  Beyond 87, 1 - a is below 2^-125.  NaN stays NaN.  For fp32 data the product
// gate log2(e) is taken with its rounding error, which would be worth 2^-24 |gate| of the exponential.
template <class T, int V>
__device__ __forceinline__ void coefficients(typename Ch<V>::F gate, typename Ch<V>::F& keep, typename Ch<V>::F& a) {
  using C = Ch<V>;
  typename C::F g = C::each(gate, [](float v) { return min_nan(v, 87.f); });
  if constexpr (sizeof(T) == 4) g = C::each(g, [](float v) { return max_nan(v, -87.f); });
  const typename C::F t = C::mul(g, C::of(1.4426950408889634f));
  typename C::F e = C::each(t, [](float v) { return ex2(v); });
  if constexpr (sizeof(T) == 4) {
    const typename C::F rest = C::fma(g, C::of(1.925963033500011e-8f), C::fma(g, C::of(1.4426950408889634f), C::mul(t, C::of(-1.f))));
    e = C::fma(e, C::mul(rest, C::of(0.6931471805599453f)), e);
  }
  keep = C::each(C::add(e, C::of(1.f)), [](float v) { return rcp(v); });
  // beside 1 the rounded 1 - keep: the product's own roundings would take 2^-24 off a held state at every step
  a = C::pick(g, C::fma(keep, C::of(-1.f), C::of(1.f)), C::mul(e, keep));
}
// Of a step that counts only where `live`: else a = 1, so that the state stays.
template <class T, int V, bool WHOLE>
__device__ __forceinline__ void coefficients(uint32_t gate, uint32_t live, typename Ch<V>::F& keep, typename Ch<V>::F& a) {
  coefficients<T, V>(take<T, V>(gate), keep, a);
  if (!WHOLE && !live) keep = Ch<V>::of(0.f), a = Ch<V>::of(1.f);
}

// The next row's place, from this one's: left to itself the compiler keeps 16 multiples of every stride in
// registers, three times what the data takes.
template <class P>
__device__ __forceinline__ void advance(P& at, long long step) {
  at += step;
  asm volatile("" : "+l"(at));
}

// The 4 bytes (one fp32 or two 16-bit channels; one 16-bit channel: 2 bytes) of a thread's steps.
struct Raw {
  uint32_t v[kSub];
};
template <class T, int V>
__device__ __forceinline__ uint32_t load_one(const T* at) {
  if constexpr (sizeof(T) * V == 4) {
    uint32_t v;
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(at));
    return v;
  } else {
    uint16_t v;
    asm volatile("ld.global.b16 %0, [%1];" : "=h"(v) : "l"(at));
    return v;
  }
}
// 0 where the step does not count
template <class T, int V>
__device__ __forceinline__ uint32_t load_one(const T* at, uint32_t live) {
  if constexpr (sizeof(T) * V == 4) {
    uint32_t v = 0;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}" : "+r"(v) : "l"(at), "r"(live));
    return v;
  } else {
    uint16_t v = 0;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p ld.global.b16 %0, [%1];\n\t}" : "+h"(v) : "l"(at), "r"(live));
    return v;
  }
}
// What a warp works on: all of its threads' steps, or (else) those of each thread's own bits, of which the last of the
// warp comes before `end`.
struct Steps {
  uint32_t in, on;  // that exist; that exist and the mask keeps
  int end;
  bool whole;
  __device__ __forceinline__ Steps(uint32_t in_, uint32_t on_) : in(in_), on(on_) {
    whole = __all_sync(0xffffffffu, on == (1u << kSub) - 1);
    end = whole ? kSub : __reduce_max_sync(0xffffffffu, 32 - __clz(in));
  }
};
// The tensors' rows of the steps, N of them side by side.
template <class T, int V, int N>
__device__ __forceinline__ void load(Raw (&r)[N], const T* const (&from)[N], const long long (&step)[N], const Steps& st) {
  const T* at[N];
#pragma unroll
  for (int n = 0; n < N; ++n) at[n] = from[n];
  if (st.whole) {
#pragma unroll
    for (int i = 0; i < kSub; ++i)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        r[n].v[i] = load_one<T, V>(at[n]);
        advance(at[n], step[n]);
      }
  } else {
#pragma unroll
    for (int i = 0; i < kSub; ++i) {
#pragma unroll
      for (int n = 0; n < N; ++n) r[n].v[i] = 0;
      if (i < st.end) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          r[n].v[i] = load_one<T, V>(at[n], st.on >> i & 1);
          advance(at[n], step[n]);
        }
      }
    }
  }
}
// Asks for the steps from t0 on in L2, a step a lane: the rows of a warp lie within a line of it.
template <class T>
__device__ __forceinline__ void ahead(const T* line, long long t0, long long step, long long steps, bool on) {
  const long long t = t0 + threadIdx.x % kSub;
  if (on && t < steps) asm volatile("prefetch.global.L2 [%0];" ::"l"(line + t * step));
}
template <class T, int V>
__device__ __forceinline__ void put(T* at, typename Ch<V>::F f) {
  if constexpr (V == 2) *reinterpret_cast<Vec<T, 2>*>(at) = from_pairs<T, 2>({f});
  else *at = from_f32<T>(f);
}
// Of a step in a stretch that is not whole: 0 where the mask is, nothing where there is no step.
template <class T, int V, bool WHOLE>
__device__ __forceinline__ void put(T* at, typename Ch<V>::F f, const Steps& st, int i) {
  if (WHOLE || (st.on >> i & 1)) put<T, V>(at, f);
  else if (st.in >> i & 1) put<T, V>(at, Ch<V>::of(0.f));
}
template <int V>
__device__ __forceinline__ typename Ch<V>::F load_f32(const float* p, long long at, bool on) {
  if constexpr (V == 2) return on && p ? *reinterpret_cast<const float2*>(p + at) : both(0.f);
  else return on && p ? p[at] : 0.f;
}
// (state, last and their gradients may start on any 4-byte boundary)
template <int V>
__device__ __forceinline__ typename Ch<V>::F load_edge(const float* p, long long at, bool on) {
  if constexpr (V == 2) return on && p ? make_float2(p[at], p[at + 1]) : both(0.f);
  else return on && p ? p[at] : 0.f;
}
template <int V>
__device__ __forceinline__ void store_edge(float* p, long long at, typename Ch<V>::F f) {
  if constexpr (V == 2) p[at] = f.x, p[at + 1] = f.y;
  else p[at] = f;
}
template <int V>
__device__ __forceinline__ void store_f32(float* p, long long at, typename Ch<V>::F f) {
  if constexpr (V == 2) *reinterpret_cast<float2*>(p + at) = f;
  else p[at] = f;
}

// One thread's place: its column (line and channels) and its place among the threads along the line.
template <int V>
struct Place {
  long long line, n, m;
  int c, sub, lane;
  bool on;
  __device__ __forceinline__ Place(const ScanParams& p) {
    lane = p.subs > 1 ? threadIdx.x % kLanes : threadIdx.x;
    sub = p.subs > 1 ? threadIdx.x / kLanes : 0;
    const long long col = (long long)blockIdx.x * p.block_columns + lane;
    on = col < p.columns;
    if (p.columns < 1ll << 31) {  // 64-bit divisions cost a short line more than its steps
      const unsigned i = on ? (unsigned)col : 0u, l = i / (unsigned)p.per_line, k = l / (unsigned)p.m;
      line = l;
      c = (int)(i - l * (unsigned)p.per_line) * V;
      n = k;
      m = l - k * (unsigned)p.m;
    } else {
      line = on ? col / p.per_line : 0;
      c = on ? (int)(col - line * p.per_line) * V : 0;
      n = line / p.m;
      m = line - n * p.m;
    }
  }
  __device__ __forceinline__ long long at(const long long (&s)[3]) const { return n * s[0] + m * s[1]; }
  // the steps of the kSub from t0 on that exist (bits), and those of them that the mask keeps
  __device__ __forceinline__ uint32_t inside(const ScanParams& p, long long t0) const {
    const long long left = p.steps - t0;
    return !on || left <= 0 ? 0u : left >= kSub ? (1u << kSub) - 1 : (1u << left) - 1;
  }
  __device__ __forceinline__ uint32_t kept(const ScanParams& p, long long t0, uint32_t in) const {
    if (!p.mask) return in;
    const uint8_t* at_mask = p.mask + at(p.ms) + t0 * p.ms[2];
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kSub; ++i) {
      if ((in >> i & 1) && *at_mask) bits |= 1u << i;
      advance(at_mask, p.ms[2]);
    }
    return bits;
  }
};

// Maps of the warps along a line, two buffers in turn: one barrier an exchange.
template <int V, int SUBS>
struct Exchange {
  using C = Ch<V>;
  using F = typename C::F;
  F p[2][SUBS][kLanes], h[2][SUBS][kLanes];
  // In: this warp's map (P, H) and the state before (or, BACK, behind) the stretch in `run`.  Out: that of this
  // warp's steps, and in `run` that of the next stretch.  Maps are applied in the order of the line.
  template <bool BACK>
  __device__ __forceinline__ F go(int buf, int sub, int lane, F P, F H, F& run) {
    p[buf][sub][lane] = P;
    h[buf][sub][lane] = H;
    __syncthreads();
    F start = run;
#pragma unroll
    for (int k = 0; k < SUBS; ++k) {
      const int s = BACK ? SUBS - 1 - k : k;
      if (s == sub) start = run;
      run = C::fma(p[buf][s][lane], run, h[buf][s][lane]);
    }
    return start;
  }
};
template <int V>
struct Exchange<V, 1> {};

// The state at the start (end) of this block's piece: through the maps of the pieces before (behind) it.
template <int V, bool BACK>
__device__ __forceinline__ typename Ch<V>::F enter(const ScanParams& p, const Place<V>& me) {
  const long long at = me.line * p.channels + me.c, piece = p.lines * p.channels;
  typename Ch<V>::F run = load_edge<V>(BACK ? p.dlast : p.state, at, me.on);
  const int count = BACK ? p.pieces - 1 - (int)blockIdx.y : (int)blockIdx.y;
#pragma unroll 8
  for (int k = 0; k < count; ++k) {
    const long long from = (BACK ? p.pieces - 1 - k : k) * piece + at;
    run = Ch<V>::fma(load_f32<V>(p.agg_p, from, me.on), run, load_f32<V>(p.agg_h, from, me.on));
  }
  return run;
}

// Whether all steps of a stretch exist and count, for all columns of the block.
template <int SUBS>
__device__ __forceinline__ bool whole_stretch(const ScanParams& p, long long k) {
  return !p.mask && (k + 1) * SUBS * kSub <= p.steps && ((long long)blockIdx.x + 1) * kLanes <= p.columns;
}

// SUBS: warps along a line (1: a thread walks along it alone, and there is one piece).
template <class T, int V, int SUBS>
__global__ void __launch_bounds__(kThreads, SUBS == 1 ? kBlocksAlone : kBlocks) scan_forward_kernel(const __grid_constant__ ScanParams p) {
  using C = Ch<V>;
  using F = typename C::F;
  may_start_next();
  after_previous();
  __shared__ Exchange<V, SUBS> exchange;
  const Place<V> me(p);
  const T* x = static_cast<const T*>(p.x) + me.at(p.xs) + me.c;
  const T* g = static_cast<const T*>(p.gate) + me.at(p.gs) + me.c;
  T* y = static_cast<T*>(p.y) + me.at(p.ys) + me.c;
  const long long k0 = blockIdx.y * p.per, k1 = min(k0 + p.per, p.stretches);
  F run = enter<V, false>(p, me);

  Raw r[2];
  const long long step[2] = {p.xs[2], p.gs[2]}, ystep = p.ys[2];
  for (long long k = k0; k < k1; ++k) {
    const long long t0 = (k * SUBS + me.sub) * kSub;
    const uint32_t in = me.inside(p, t0);
    const Steps st(in, me.kept(p, t0, in));
    load<T, V, 2>(r, {x + t0 * step[0], g + t0 * step[1]}, step, st);
    if (k + 1 < k1) {
      ahead(x, t0 + SUBS * kSub, step[0], p.steps, me.on);
      ahead(g, t0 + SUBS * kSub, step[1], p.steps, me.on);
    }
    const long long mark = t0 / kSub - 1;
    float* to_mark = p.saved && mark >= 0 && in ? p.saved + (me.line * p.marks + mark) * p.channels + me.c : nullptr;
    T* to = y + t0 * ystep;
    const auto work = [&](auto all) {
      constexpr bool W = decltype(all)::value != 0;
      if constexpr (SUBS == 1) {
        if (to_mark) store_f32<V>(to_mark, 0, run);
#pragma unroll
        for (int i = 0; i < kSub; ++i) {
          if (!W && i >= st.end) break;
          F keep, a;
          coefficients<T, V, W>(r[1].v[i], st.on >> i & 1, keep, a);
          run = C::fma(a, run, C::mul(keep, take<T, V>(r[0].v[i])));
          put<T, V, W>(to, run, st, i);
          advance(to, ystep);
        }
      } else {
        F P[kSub], H[kSub], prod = C::of(1.f), h = C::of(0.f);
#pragma unroll
        for (int i = 0; i < kSub; ++i) {
          F keep, a;
          coefficients<T, V, W>(r[1].v[i], st.on >> i & 1, keep, a);
          H[i] = h = C::fma(a, h, C::mul(keep, take<T, V>(r[0].v[i])));
          P[i] = prod = C::mul(prod, a);
        }
        const F start = exchange.template go<false>(k & 1, me.sub, me.lane, prod, h, run);
        if (to_mark) store_f32<V>(to_mark, 0, start);
#pragma unroll
        for (int i = 0; i < kSub; ++i) {
          put<T, V, W>(to, C::fma(P[i], start, H[i]), st, i);
          advance(to, ystep);
        }
      }
    };
    if (SUBS == 1 ? st.whole : whole_stretch<SUBS>(p, k)) work(ActTag<1>{});
    else work(ActTag<0>{});
  }
  if (me.on && me.sub == 0 && (int)blockIdx.y == p.pieces - 1) store_edge<V>(p.last, me.line * p.channels + me.c, run);
}

// The maps of the pieces.  Here a warp takes adjacent steps of the piece, so there is one exchange, at the end.
// Backward: r -> P r + H with r = a G, built in the order of the line: a later step's dy passes the a before it.
template <class T, int V, int SUBS, bool BACK>
__global__ void __launch_bounds__(kThreads, kBlocksAlone) scan_pieces_kernel(const __grid_constant__ ScanParams p) {
  using C = Ch<V>;
  using F = typename C::F;
  may_start_next();
  after_previous();
  __shared__ Exchange<V, SUBS> exchange;
  const Place<V> me(p);
  const long long z = BACK ? blockIdx.y + 1 : blockIdx.y;  // nothing enters the first piece, or behind the last
  const T* v = static_cast<const T*>(BACK ? p.dy : p.x) + me.at(BACK ? p.ds : p.xs) + me.c;
  const T* g = static_cast<const T*>(p.gate) + me.at(p.gs) + me.c;
  const long long vs = BACK ? p.ds[2] : p.xs[2];
  const long long count = min(p.per, p.stretches - z * p.per);
  long long t0 = (z * p.per * SUBS + me.sub * count) * kSub;
  F P = C::of(1.f), H = C::of(0.f);
  Raw r[2];
  const long long step[2] = {vs, p.gs[2]};
  for (long long k = 0; k < count; ++k, t0 += kSub) {
    const uint32_t in = me.inside(p, t0);
    const Steps st(in, me.kept(p, t0, in));
    load<T, V, 2>(r, {v + t0 * vs, g + t0 * step[1]}, step, st);
    if (k + 1 < count) {
      ahead(v, t0 + kSub, vs, p.steps, me.on);
      ahead(g, t0 + kSub, step[1], p.steps, me.on);
    }
    const auto work = [&](auto all) {
      constexpr bool W = decltype(all)::value != 0;
#pragma unroll
      for (int i = 0; i < kSub; ++i) {
        if (!W && i >= st.end) break;
        F keep, a;
        coefficients<T, V, W>(r[1].v[i], st.on >> i & 1, keep, a);
        P = C::mul(P, a);
        if constexpr (BACK) H = C::fma(P, take<T, V>(r[0].v[i]), H);
        else H = C::fma(a, H, C::mul(keep, take<T, V>(r[0].v[i])));
      }
    };
    if (st.whole) work(ActTag<1>{});
    else work(ActTag<0>{});
  }
  // the whole piece's map: its H from a state of 0, its P as the product over the warps
  F run = C::of(0.f), all = C::of(1.f);
  exchange.template go<BACK>(0, me.sub, me.lane, P, H, run);
  if (!me.on || me.sub != 0) return;
#pragma unroll
  for (int s = 0; s < SUBS; ++s) all = C::mul(all, exchange.p[0][s][me.lane]);
  const long long to = (z * p.lines + me.line) * p.channels + me.c;
  store_f32<V>(p.agg_p, to, all);
  store_f32<V>(p.agg_h, to, run);
}

template <class T, int V, int SUBS>
__global__ void __launch_bounds__(kThreads, kBlocksBack) scan_backward_kernel(const __grid_constant__ ScanParams p) {
  using C = Ch<V>;
  using F = typename C::F;
  may_start_next();
  after_previous();
  __shared__ Exchange<V, SUBS> exchange;
  const Place<V> me(p);
  const T* x = static_cast<const T*>(p.x) + me.at(p.xs) + me.c;
  const T* g = static_cast<const T*>(p.gate) + me.at(p.gs) + me.c;
  const T* dy = static_cast<const T*>(p.dy) + me.at(p.ds) + me.c;
  T* dx = static_cast<T*>(p.dx) + me.at(p.ys) + me.c;
  T* dg = static_cast<T*>(p.dgate) + me.at(p.ys) + me.c;
  const long long k0 = blockIdx.y * p.per, k1 = min(k0 + p.per, p.stretches);
  F run = enter<V, true>(p, me), r = run;

  Raw raw[3];
  const long long step[3] = {p.xs[2], p.gs[2], p.ds[2]}, ystep = p.ys[2];
  for (long long k = k1 - 1; k >= k0; --k) {
    const long long t0 = (k * SUBS + me.sub) * kSub;
    const uint32_t in = me.inside(p, t0);
    const Steps st(in, me.kept(p, t0, in));
    load<T, V, 3>(raw, {x + t0 * step[0], g + t0 * step[1], dy + t0 * step[2]}, step, st);
    const long long mark = t0 / kSub - 1;  // the state before these steps
    F h = mark < 0 ? load_edge<V>(p.state, me.line * p.channels + me.c, me.on)
                   : load_f32<V>(p.saved, (me.line * p.marks + mark) * p.channels + me.c, in != 0);
    if (k > k0) {
      ahead(x, t0 - SUBS * kSub, step[0], p.steps, me.on);
      ahead(g, t0 - SUBS * kSub, step[1], p.steps, me.on);
      ahead(dy, t0 - SUBS * kSub, step[2], p.steps, me.on);
    }
    const auto work = [&](auto all) {
      constexpr bool W = decltype(all)::value != 0;
      // Two channels of a thread alone along its line: one row for a and 1 - a, the smaller of them, as the gate's sign tells,
      // since the other is 1 less that.  Two rows do not fit the registers (800 lines of 200 steps, 512 channels bf16: 180 us; at 3
      // blocks a multiprocessor 175; folded 172).  1 - a alone (163) would lose a beside 1 - a of nearly 1.
      constexpr bool kFold = V == 2 && SUBS == 1;
      F keeps[kSub], w[kSub], as[kFold ? 1 : kSub];
      F P = C::of(1.f), H = C::of(0.f);
      // in the order of the line: the states again, w = a (h before - x), and the stretch's map of r = a G
#pragma unroll
      for (int i = 0; i < kSub; ++i) {
        if (SUBS == 1 && !W && i >= st.end) break;
        F keep, a;
        coefficients<T, V, W>(raw[1].v[i], st.on >> i & 1, keep, a);
        const F xi = take<T, V>(raw[0].v[i]);
        w[i] = C::mul(a, C::fma(xi, C::of(-1.f), h));
        h = C::fma(a, h, C::mul(keep, xi));
        if constexpr (SUBS > 1) {
          P = C::mul(P, a);
          H = C::fma(P, take<T, V>(raw[2].v[i]), H);
        }
        if constexpr (kFold) {
          keeps[i] = C::pick(take<T, V>(raw[1].v[i]), keep, a);
        } else {
          keeps[i] = keep;
          as[i] = a;
        }
      }
      if constexpr (SUBS > 1) r = exchange.template go<true>(k & 1, me.sub, me.lane, P, H, run);
      // from its end: dx = (1 - a) G, dgate = w dx, r = a G
      long long to = (t0 + kSub - 1) * ystep;
#pragma unroll
      for (int i = kSub - 1; i >= 0; --i) {
        if (W || i < st.end) {
          const F G = C::add(take<T, V>(raw[2].v[i]), r);
          F ox = C::mul(keeps[i], G);
          if constexpr (kFold) {
            const F rest = C::fma(ox, C::of(-1.f), G), gate = take<T, V>(raw[1].v[i]);
            r = C::pick(gate, rest, ox);
            ox = C::pick(gate, ox, rest);
          } else {
            r = C::mul(as[i], G);
          }
          if (p.dx) put<T, V, W>(dx + to, ox, st, i);
          if (p.dgate) put<T, V, W>(dg + to, C::mul(w[i], ox), st, i);
        }
        advance(to, -ystep);
      }
    };
    if (SUBS == 1 ? st.whole : whole_stretch<SUBS>(p, k)) work(ActTag<1>{});
    else work(ActTag<0>{});
    if constexpr (SUBS == 1) run = r;
  }
  if (p.dstate && me.on && me.sub == 0 && blockIdx.y == 0) store_edge<V>(p.dstate, me.line * p.channels + me.c, run);
}

// ------------------------------------------------------------------------------- many or short lines
// A thread takes WORDS words of a row, up to 16 bytes, of S steps at a time, alone along its line.  PLAIN: the compiler orders
// loads and places (4 steps: backward 55 against 68 us when it was chosen; of 8 steps it would keep 276 bytes outside of the registers).
template <class T, int WORDS, int S, bool PLAIN>
struct Wide {
  static constexpr int kV = sizeof(T) == 2 ? 2 : 1, kChannels = WORDS * kV;  // of a word; of a thread
  using C = Ch<kV>;
  using F = typename C::F;
  struct __align__(4 * WORDS) Row {
    uint32_t w[WORDS];
  };
  static __device__ __forceinline__ uint32_t pack(F f) {
    if constexpr (kV == 2) {
      const Vec<T, 2> v = from_pairs<T, 2>({f});
      return reinterpret_cast<const uint32_t&>(v);
    } else {
      return __float_as_uint(f);
    }
  }
  // The rows of the steps that count; others are 0.
  static __device__ __forceinline__ void load(Row (&q)[S], const T* from, long long step, uint32_t on) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
#pragma unroll
      for (uint32_t& w : q[i].w) w = 0;
      if constexpr (PLAIN) {
        if (on >> i & 1) q[i] = *reinterpret_cast<const Row*>(from + i * step);
        continue;
      }
      if (on >> i & 1) {
        if constexpr (WORDS == 4)
          asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(q[i].w[0]), "=r"(q[i].w[1]), "=r"(q[i].w[2]), "=r"(q[i].w[3])
                       : "l"(from));
        else
          asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(q[i].w[0]), "=r"(q[i].w[1]) : "l"(from));
      }
      advance(from, step);
    }
  }
  static __device__ __forceinline__ void store(T* to, long long step, const Row (&q)[S], uint32_t in, uint32_t on) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
      if (in >> i & 1) *reinterpret_cast<Row*>(PLAIN ? to + i * step : to) = on >> i & 1 ? q[i] : Row{};
      if constexpr (!PLAIN) advance(to, step);
    }
  }
  // Asks for S steps from t0 on in L2.
  static __device__ __forceinline__ void soon(const T* line, long long t0, long long step, long long steps) {
    const long long t = t0 + threadIdx.x % S;
    if (t >= 0 && t < steps) asm volatile("prefetch.global.L2 [%0];" ::"l"(line + t * step));
  }
  // fp32 states, on any 4-byte boundary
  static __device__ __forceinline__ void load_states(F (&f)[WORDS], const float* p, long long at) {
    float v[kChannels];
    if (!p) {
#pragma unroll
      for (float& t : v) t = 0.f;
    } else if (kChannels % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kChannels / 4; ++i) {
        const float4 t = reinterpret_cast<const float4*>(p + at)[i];
        v[4 * i] = t.x, v[4 * i + 1] = t.y, v[4 * i + 2] = t.z, v[4 * i + 3] = t.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kChannels; ++i) v[i] = p[at + i];
    }
#pragma unroll
    for (int u = 0; u < WORDS; ++u) {
      if constexpr (kV == 2) f[u] = make_float2(v[2 * u], v[2 * u + 1]);
      else f[u] = v[u];
    }
  }
  static __device__ __forceinline__ void store_states(float* p, long long at, const F (&f)[WORDS]) {
    float v[kChannels];
#pragma unroll
    for (int u = 0; u < WORDS; ++u) {
      if constexpr (kV == 2) v[2 * u] = f[u].x, v[2 * u + 1] = f[u].y;
      else v[u] = f[u];
    }
    if (kChannels % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kChannels / 4; ++i)
        reinterpret_cast<float4*>(p + at)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < kChannels; ++i) p[at + i] = v[i];
    }
  }
};

constexpr int kShort = 4;  // steps at a time
// ONCE: lines that end there.
template <class T, bool ONCE>
__global__ void __launch_bounds__(kThreads, ONCE ? 8 : 6) scan_wide_forward_kernel(const __grid_constant__ ScanParams p) {
  using W = Wide<T, 4, kShort, ONCE>;
  using C = typename W::C;
  may_start_next();
  after_previous();
  const Place<W::kChannels> me(p);
  if (!me.on) return;
  const T* x = static_cast<const T*>(p.x) + me.at(p.xs) + me.c;
  const T* g = static_cast<const T*>(p.gate) + me.at(p.gs) + me.c;
  T* y = static_cast<T*>(p.y) + me.at(p.ys) + me.c;
  const long long edge = me.line * p.channels + me.c;
  typename W::F run[4];
  W::load_states(run, p.state, edge);
  for (long long t0 = 0; t0 < p.steps; t0 += kShort) {
    const uint32_t in = me.inside(p, t0) & ((1u << kShort) - 1), on = me.kept(p, t0, in);
    typename W::Row xs[kShort], gs[kShort];
    W::load(xs, x + t0 * p.xs[2], p.xs[2], on);
    W::load(gs, g + t0 * p.gs[2], p.gs[2], on);
    if constexpr (!ONCE) {
      W::soon(x, t0 + kShort, p.xs[2], p.steps);
      W::soon(g, t0 + kShort, p.gs[2], p.steps);
    }
    if (!ONCE && p.saved && t0 && t0 % kSub == 0) W::store_states(p.saved, (me.line * p.marks + t0 / kSub - 1) * p.channels + me.c, run);
#pragma unroll
    for (int i = 0; i < kShort; ++i)
      if (on >> i & 1) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          typename W::F keep, a;
          coefficients<T, W::kV>(take<T, W::kV>(gs[i].w[u]), keep, a);
          run[u] = C::fma(a, run[u], C::mul(keep, take<T, W::kV>(xs[i].w[u])));
          xs[i].w[u] = W::pack(run[u]);
        }
      }
    W::store(y + t0 * p.ys[2], p.ys[2], xs, in, on);
    if (ONCE) break;
  }
  W::store_states(p.last, edge, run);
}

// As scan_backward_kernel, a word after the other.  S: kShort for lines that end there, else kSub, from the stored states.
template <class T, int WORDS, int S>
__global__ void __launch_bounds__(kThreads, 4) scan_wide_backward_kernel(const __grid_constant__ ScanParams p) {
  using W = Wide<T, WORDS, S, S == kShort>;
  using C = typename W::C;
  using F = typename W::F;
  may_start_next();
  after_previous();
  const Place<W::kChannels> me(p);
  if (!me.on) return;
  const T* x = static_cast<const T*>(p.x) + me.at(p.xs) + me.c;
  const T* g = static_cast<const T*>(p.gate) + me.at(p.gs) + me.c;
  const T* dy = static_cast<const T*>(p.dy) + me.at(p.ds) + me.c;
  T* dx = static_cast<T*>(p.dx) + me.at(p.ys) + me.c;
  T* dg = static_cast<T*>(p.dgate) + me.at(p.ys) + me.c;
  const long long edge = me.line * p.channels + me.c;
  F h[WORDS], r[WORDS];
  W::load_states(r, p.dlast, edge);
  for (long long t0 = S == kShort ? 0 : p.marks * S; t0 >= 0; t0 -= S) {
    const uint32_t in = me.inside(p, t0), on = me.kept(p, t0, in);
    typename W::Row xs[S], gs[S], ds[S];
    W::load(xs, x + t0 * p.xs[2], p.xs[2], on);
    W::load(gs, g + t0 * p.gs[2], p.gs[2], on);
    W::load(ds, dy + t0 * p.ds[2], p.ds[2], on);
    const long long mark = t0 / S - 1;
    if (S == kShort || mark < 0) W::load_states(h, p.state, edge);
    else W::load_states(h, p.saved, (me.line * p.marks + mark) * p.channels + me.c);
    if (S != kShort) {
      W::soon(x, t0 - S, p.xs[2], p.steps);
      W::soon(g, t0 - S, p.gs[2], p.steps);
      W::soon(dy, t0 - S, p.ds[2], p.steps);
    }
#pragma unroll
    for (int u = 0; u < WORDS; ++u) {
      F keeps[S], w[S], as[S];
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (on >> i & 1) {
          F a;
          coefficients<T, W::kV>(take<T, W::kV>(gs[i].w[u]), keeps[i], a);
          const F xi = take<T, W::kV>(xs[i].w[u]);
          w[i] = C::mul(a, C::fma(xi, C::of(-1.f), h[u]));
          h[u] = C::fma(a, h[u], C::mul(keeps[i], xi));
          as[i] = a;
        }
#pragma unroll
      for (int i = S - 1; i >= 0; --i)
        if (on >> i & 1) {
          const F G = C::add(take<T, W::kV>(ds[i].w[u]), r[u]), ox = C::mul(keeps[i], G);
          r[u] = C::mul(as[i], G);
          xs[i].w[u] = W::pack(ox);
          gs[i].w[u] = W::pack(C::mul(w[i], ox));
        }
    }
    if (p.dx) W::store(dx + t0 * p.ys[2], p.ys[2], xs, in, on);
    if (p.dgate) W::store(dg + t0 * p.ys[2], p.ys[2], gs, in, on);
  }
  if (p.dstate) W::store_states(p.dstate, edge, r);
}

// --------------------------------------------------------------------------------------- host side
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

int32_t check_desc(const NcaScanDesc* d) {
  if (!d || d->n < 0 || d->m < 0 || d->steps < 0 || d->channels < 0 || !dtype_ok(d->dtype)) return NCA_ERR_INVALID;
  const long long most = 1ll << 40;  // products of sizes stay far inside 64 bits
  if (d->n > most || d->m > most || d->steps > most || (d->n && d->m > most / d->n)) return NCA_ERR_UNSUPPORTED;
  const long long lines = d->n * d->m;
  if (lines && (d->channels > most / lines || (d->steps && d->steps > (1ll << 44) / (lines * std::max(d->channels, 1)))))
    return NCA_ERR_UNSUPPORTED;
  return NCA_OK;
}
bool strides_even(const int64_t (&s)[3]) { return ((s[0] | s[1] | s[2]) & 1) == 0; }

// Two 16-bit channels a thread where every row starts on a 4-byte boundary, else one.  A thread a line where that gives
// half the threads that run at once, or the line is short; else the warps of a block along a line, and pieces of
// it for as many blocks as run at once.
ScanParams plan_of(const NcaScanDesc& d, bool backward) {
  ScanParams p{};
  const bool pairs = d.dtype != NCA_F32 && d.channels % 2 == 0 && !d.unaligned && strides_even(d.x_stride) &&
                     strides_even(d.gate_stride) && strides_even(d.y_stride) && (!backward || strides_even(d.dy_stride));
  p.m = std::max<long long>(d.m, 1);
  p.lines = d.n * d.m;
  p.steps = d.steps;
  p.channels = d.channels;
  p.per_line = pairs ? d.channels / 2 : d.channels;
  p.columns = p.lines * p.per_line;
  p.marks = d.steps > kSub ? ceil_div(d.steps, kSub) - 1 : 0;
  const int threads = kThreads, resident = 148 * (backward ? kBlocksBack : kBlocks);
  p.subs = d.steps > 2 * kSub && p.columns < (long long)resident * threads / 2 ? threads / kLanes : 1;
  p.block_columns = threads / p.subs;
  p.stretches = ceil_div(d.steps, (long long)p.subs * kSub);
  const long long groups = ceil_div(p.columns, p.block_columns);
  long long pieces = 1;
  if (p.subs > 1 && groups > 0) pieces = std::min({(long long)kMostPieces, p.stretches / 4, resident / groups});
  p.per = ceil_div(p.stretches, std::max(pieces, 1ll));
  p.pieces = (int)std::max<long long>(1, ceil_div(p.stretches, std::max<long long>(p.per, 1)));
  return p;
}
bool two_wide(const ScanParams& p) { return p.per_line != p.channels; }
size_t workspace_of(const ScanParams& p) {
  return p.pieces == 1 ? 0 : 2 * (size_t)p.pieces * p.lines * p.channels * sizeof(float);
}

void strides(long long (&to)[3], const int64_t (&from)[3], const NcaScanDesc& d) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
  if (d.reverse) to[2] = -to[2];
}
// The first step's element: in a reversed scan the last of the line.
const void* first(const void* p, const int64_t (&s)[3], const NcaScanDesc& d, size_t size) {
  return p && d.reverse && d.steps ? static_cast<const uint8_t*>(p) + (d.steps - 1) * s[2] * (int64_t)size : p;
}
bool misaligned(const void* p, int bytes = 4) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }
// States in `saved` and maps in the workspace are read and written in pairs.
constexpr int kPairBytes = 8;

// Lines that a thread with 8 channels walks along are fewer threads than with 2, and each waits for its own loads: worth it
// for up to 64 steps (250 x 59 x 59, 32 channels, masked: 34 against 44 us forward; 800 lines of 200 steps, 512 channels, 98
// against 87), of as many lines as fill a quarter of the GPU.
constexpr long long kWideColumns = 148 * 256, kWideSteps = 64;
bool on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// Whether a thread can take `bytes` of every row (the tensors' bases aside); if so, the plan for it.
bool take_wide(ScanParams& p, const NcaScanDesc& d, int bytes, bool backward) {
  const long long channels = bytes / (long long)dtype_size(d.dtype);
  if (d.channels % channels != 0) return false;
  for (int i = 0; i < 3; ++i)
    if ((d.x_stride[i] | d.gate_stride[i] | d.y_stride[i] | (backward ? d.dy_stride[i] : 0)) % channels != 0) return false;
  const long long columns = p.lines * (d.channels / channels);
  if (d.steps > kShort && (columns < kWideColumns || d.steps > kWideSteps)) return false;
  p.per_line = (int)(d.channels / channels);
  p.columns = columns;
  p.subs = p.pieces = 1;
  p.block_columns = kThreads;
  return true;
}

template <class F>
int32_t with_kind(int dtype, bool pairs, F fn) {
  return with_dtype(dtype, [&](auto t) -> int32_t {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) {
      if (pairs) return fn(t, ActTag<2>{});
    }
    return fn(t, ActTag<1>{});
  });
}

template <class T, int V, int SUBS>
int32_t run_forward(const ScanParams& p, long long groups, cudaStream_t s) {
  if constexpr (SUBS > 1) {
    if (p.pieces > 1) {
      const int32_t e = launch_after(scan_pieces_kernel<T, V, SUBS, false>, dim3((unsigned)groups, p.pieces - 1),
                                     dim3(kThreads), 0, s, 1, p);
      if (e != NCA_OK) return e;
    }
  }
  return launch_after(scan_forward_kernel<T, V, SUBS>, dim3((unsigned)groups, p.pieces), dim3(kThreads), 0, s, 1, p);
}
template <class T, int V, int SUBS>
int32_t run_backward(const ScanParams& p, long long groups, cudaStream_t s) {
  if constexpr (SUBS > 1) {
    if (p.pieces > 1) {
      const int32_t e = launch_after(scan_pieces_kernel<T, V, SUBS, true>, dim3((unsigned)groups, p.pieces - 1),
                                     dim3(kThreads), 0, s, 1, p);
      if (e != NCA_OK) return e;
    }
  }
  return launch_after(scan_backward_kernel<T, V, SUBS>, dim3((unsigned)groups, p.pieces), dim3(kThreads), 0, s, 1, p);
}

}  // namespace

extern "C" {

int32_t nca_b200_gated_scan_saved_bytes(const NcaScanDesc* d, size_t* bytes) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK || !bytes) return st != NCA_OK ? st : NCA_ERR_INVALID;
  const ScanParams p = plan_of(*d, false);
  *bytes = (size_t)p.lines * p.marks * p.channels * sizeof(float);
  return NCA_OK;
}

int32_t nca_b200_gated_scan_workspace(const NcaScanDesc* d, int32_t backward, size_t* bytes) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK || !bytes) return st != NCA_OK ? st : NCA_ERR_INVALID;
  *bytes = workspace_of(plan_of(*d, backward != 0));
  return NCA_OK;
}

int32_t nca_b200_gated_scan(const NcaScanDesc* d, const void* x, const void* gate, const float* state,
                            const uint8_t* mask, void* y, float* last, float* saved, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK) return st;
  ScanParams p = plan_of(*d, false);
  if (p.columns == 0) return NCA_OK;
  if (!last || (d->steps && (!x || !gate || !y)) || (d->masked && d->steps && !mask)) return NCA_ERR_INVALID;
  if (two_wide(p) && (misaligned(x) || misaligned(gate) || misaligned(y))) return NCA_ERR_INVALID;
  if (p.marks && misaligned(saved, kPairBytes)) return NCA_ERR_INVALID;
  const size_t need = workspace_of(p);
  if (need && (!workspace || workspace_bytes < need)) return NCA_ERR_SCRATCH;
  if (need && misaligned(workspace, kPairBytes)) return NCA_ERR_INVALID;
  const size_t size = dtype_size(d->dtype);
  p.x = first(x, d->x_stride, *d, size);
  p.gate = first(gate, d->gate_stride, *d, size);
  p.y = const_cast<void*>(first(y, d->y_stride, *d, size));
  p.mask = d->masked ? static_cast<const uint8_t*>(first(mask, d->mask_stride, *d, 1)) : nullptr;
  strides(p.xs, d->x_stride, *d);
  strides(p.gs, d->gate_stride, *d);
  strides(p.ys, d->y_stride, *d);
  strides(p.ms, d->mask_stride, *d);
  p.state = state;
  p.last = last;
  p.saved = p.marks ? saved : nullptr;
  p.agg_p = static_cast<float*>(workspace);
  p.agg_h = p.agg_p + (size_t)p.pieces * p.lines * p.channels;
  const bool pairs = two_wide(p), wide = on(p.x, 16) && on(p.gate, 16) && on(p.y, 16) && take_wide(p, *d, 16, false);
  const long long groups = ceil_div(p.columns, p.block_columns);
  if (groups > (1ll << 31) - 1) return NCA_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (wide)
    return with_dtype(d->dtype, [&](auto t) -> int32_t {
      using T = decltype(t);
      const dim3 grid((unsigned)groups), block(kThreads);
      return p.steps <= kShort ? launch_after(scan_wide_forward_kernel<T, true>, grid, block, 0, s, 1, p)
                               : launch_after(scan_wide_forward_kernel<T, false>, grid, block, 0, s, 1, p);
    });
  return with_kind(d->dtype, pairs, [&](auto t, auto v) -> int32_t {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    return p.subs > 1 ? run_forward<T, V, kThreads / kLanes>(p, groups, s) : run_forward<T, V, 1>(p, groups, s);
  });
}

int32_t nca_b200_gated_scan_backward(const NcaScanDesc* d, const void* x, const void* gate, const float* state,
                                     const uint8_t* mask, const float* saved, const void* dy, const float* dlast,
                                     void* dx, void* dgate, float* dstate, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  const int32_t st = check_desc(d);
  if (st != NCA_OK) return st;
  ScanParams p = plan_of(*d, true);
  if (p.columns == 0) return NCA_OK;
  if ((d->steps && (!x || !gate || !dy)) || (p.marks && !saved) || (d->masked && d->steps && !mask)) return NCA_ERR_INVALID;
  if (two_wide(p) && (misaligned(x) || misaligned(gate) || misaligned(dy) || misaligned(dx) || misaligned(dgate)))
    return NCA_ERR_INVALID;
  if (p.marks && misaligned(saved, kPairBytes)) return NCA_ERR_INVALID;
  const size_t need = workspace_of(p);
  if (need && (!workspace || workspace_bytes < need)) return NCA_ERR_SCRATCH;
  if (need && misaligned(workspace, kPairBytes)) return NCA_ERR_INVALID;
  const size_t size = dtype_size(d->dtype);
  p.x = first(x, d->x_stride, *d, size);
  p.gate = first(gate, d->gate_stride, *d, size);
  p.dy = first(dy, d->dy_stride, *d, size);
  p.dx = const_cast<void*>(first(dx, d->y_stride, *d, size));
  p.dgate = const_cast<void*>(first(dgate, d->y_stride, *d, size));
  p.mask = d->masked ? static_cast<const uint8_t*>(first(mask, d->mask_stride, *d, 1)) : nullptr;
  strides(p.xs, d->x_stride, *d);
  strides(p.gs, d->gate_stride, *d);
  strides(p.ds, d->dy_stride, *d);
  strides(p.ys, d->y_stride, *d);
  strides(p.ms, d->mask_stride, *d);
  p.state = state;
  p.dlast = dlast;
  p.dstate = dstate;
  p.saved = const_cast<float*>(saved);
  p.agg_p = static_cast<float*>(workspace);
  p.agg_h = p.agg_p + (size_t)p.pieces * p.lines * p.channels;
  const bool pairs = two_wide(p);
  const int bytes = d->steps > kShort ? 8 : 16;
  const bool wide = on(p.x, bytes) && on(p.gate, bytes) && on(p.dy, bytes) && on(p.dx, bytes) && on(p.dgate, bytes) &&
                    take_wide(p, *d, bytes, true);
  const long long groups = ceil_div(p.columns, p.block_columns);
  if (groups > (1ll << 31) - 1) return NCA_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (wide)
    return with_dtype(d->dtype, [&](auto t) -> int32_t {
      using T = decltype(t);
      const dim3 grid((unsigned)groups), block(kThreads);
      return bytes == 16 ? launch_after(scan_wide_backward_kernel<T, 4, kShort>, grid, block, 0, s, 1, p)
                         : launch_after(scan_wide_backward_kernel<T, 2, kSub>, grid, block, 0, s, 1, p);
    });
  return with_kind(d->dtype, pairs, [&](auto t, auto v) -> int32_t {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    return p.subs > 1 ? run_backward<T, V, kThreads / kLanes>(p, groups, s) : run_backward<T, V, 1>(p, groups, s);
  });
}

}  // extern "C"
