// Gated linear recurrence over packed windows of rows (include/atl_b200.h, atlb_recurrence_*).
//
//   decay    h_t = a_t h_(t-1) + x_t                      a_t = gate_t
//   sigmoid  h_t = a_t h_(t-1) + (1 - a_t) x_t            a_t = 1 / (1 + exp(-gate_t))
// per column, with h before a window's first row equal to h0 (or zero).  Backward, from the last row of a window:
//   g_t = dh_t + u_(t+1)   (last row: dh_t + dhT)         u_t = a_t g_t          dh0 = u of the first row
//   decay    dgate = g_t h_(t-1)                          dx = g_t
//   sigmoid  dgate = g_t (h_(t-1) - x_t) a_t (1 - a_t)    dx = (1 - a_t) g_t
//
// Rows are cut into groups of kGroup; over a group the recurrence is an affine map h -> A h + C of the state that enters
// it (and u -> A u + C' backward, with the same A).  Three kernels: the maps of the groups, joined inside each CTA's
// chunk of groups (k_rec_map); the states between the chunks (k_rec_chain); the rows replayed from the true state of
// their group (k_rec_fwd, k_rec_bwd).  Inputs are read twice and nothing waits for another CTA: a single pass, with
// tiles in shared memory that post their maps to one another, reads them once but measured 647 us where this form took
// 376 (forward and backward, 1M rows of 64 bf16 columns; 378 now), the waits and the link costing more than the bytes.
// What bounds it is memory: 4M rows of 64 fp16 columns forward move 2.6 GB in 496 us (5.3 TB/s, 82 % of the copy rate),
// where one reading would be 1.5 GB.  Measured against 374 / 240 / 483 us (1M rows of 64 both ways; 16 windows of 2048
// rows of 1024; 4M rows forward): 16 bytes per thread 429 / 263 / 535, 8 rows in flight 404 / 264 / 515, rows through a
// ring in shared memory 399 / 241 / 549, CTAs of 128 threads 383 / 229 / 505, packed fp32 arithmetic 371 / 232 / 485,
// groups of 64 to 192 rows 384 to 426 / 225 to 357 / 467 to 479.
// The maps are joined in one fixed order.  States, maps and sums are fp32; an output is rounded once.  A row that
// begins a window drops what comes before it by selection, so nothing of one window, NaN included, reaches another.
#include "vec.cuh"

namespace atlb {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 32;          // rows of a group (16 measured 413, 8 510 us where 32 took 376: more maps to join)
constexpr int kPart = 8;            // rows between the states that the forward pass keeps for the backward pass
constexpr int kBytes = 8;           // of a row per thread, where the rows are whole multiples of it
constexpr int kSeg = 16;            // groups joined by one thread
constexpr int kChainCols = 8, kChainSegs = 128;

struct RecShape {
  long long N;             // rows, below 2^31
  unsigned T;              // rows per window where b is null
  int B, D;
  const long long* b;      // window of every row, or null
  int groups, chunks;      // groups of rows, chunks of groups
  int lanes;               // threads per row in k_rec_map and k_rec_fwd (a power of two)
  bool linked;             // false: every group begins a window, no state enters one
};

// a = 1 / (1 + exp(-z)) and 1 - a = exp(-z) a, so that neither cancels.  Below z = -87.3 a would be no normal number and
// counts as zero, so a large state leaves no trace behind a closed gate; 1 - a is one there (exp(-z) a would be 0 inf).
// (Holding a at exp(-87) let 0.02 through from a state of 2^120; it was 1.9 % faster, 1M bf16 rows of 64 both ways.)
// FINE, for fp32 gates: expf, whose error does not grow with |z|.  For 16-bit gates the bare exponential stays below 1e-6
// of the value for |z| < 10, far below the gates' own rounding, and is 4 % (1M rows, both ways) to 12 % (4M rows forward)
// faster.
template <bool FINE>
__device__ __forceinline__ void sigmoid2(float z, float* a, float* w) {
  float e;
  if (FINE)
    e = expf(-z);
  else
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(*a) : "f"(1.f + e));
  *w = z < -87.2f ? 1.f : e * *a;  // a NaN stays one
}

// The row's coefficient a and what it adds: (1 - a) x or x.
template <int KIND, typename T>
__device__ __forceinline__ void row_terms(T gate, T in, float* a, float* w, float* v) {
  const float x = to_f32(in);
  if (KIND == ATLB_REC_SIGMOID) {
    sigmoid2<sizeof(T) == 4>(to_f32(gate), a, w);
    *v = *w * x;
  } else {
    *a = to_f32(gate);
    *w = 1.f;
    *v = x;
  }
}

// ------------------------------------------------------------------------------------------------ maps
// The map h -> A h + C of some rows in one column; cut: they hold a window's border, so the state before them does not
// matter.  C is the state that a zero leaves behind, no larger than the magnitudes that the rows themselves go through.
// A has no such bound.  Sigmoid: a product of values in [0, 1], which may at worst vanish; plain fp32 (below 2^-149 over a
// group, a state before it counts as zero).
struct Map {
  float A, C;
  bool cut;
  __device__ __forceinline__ static Map identity() { return Map{1.f, 0.f, false}; }
};
__device__ __forceinline__ float apply(const Map& m, float s) { return m.cut ? m.C : fmaf(m.A, s, m.C); }
__device__ __forceinline__ Map then(const Map& a, const Map& b) { return Map{a.A * b.A, apply(b, a.C), a.cut || b.cut}; }

// Decay: gates of any size.  A product over a chunk may leave fp32's range where no state does (130 gates of 2 and 130 of
// 1/2 behind a state of 0.01), so A = m 2^e with |m| in [1, 2), or m = e = 0 for zero;
// where a gate is infinite or a NaN, so is C, and m says nothing.  Device time of 1M bf16 rows of
// 64 columns, both ways: 367 us, where plain fp32 products took 348 (with 1 % of zero gates 353 for 347 unpacked); 100k
// fp32 rows of 32: 48 and 44.
struct WideMap {
  float m, C;
  int e;
  bool cut;
  __device__ __forceinline__ static WideMap identity() { return WideMap{1.f, 0.f, 0, false}; }
};
constexpr int kMaxExp = 32000;  // more makes no difference: beyond 2^+-278 a state vanishes or overflows in any case
__device__ __forceinline__ int clamp_to(int e, int most) { return max(-most, min(most, e)); }
// 2^k for -127 < k < 128; 0 for -127.
__device__ __forceinline__ float power2(int k) { return __int_as_float((k + 127) << 23); }
// Half of 2^e goes to the state and half to m: neither leaves fp32's range where the product does not.
__device__ __forceinline__ float apply(const WideMap& w, float s) {
  const int e = clamp_to(w.e, 254), half = e >> 1;
  return w.cut ? w.C : fmaf(w.m * power2(e - half), s * power2(half), w.C);
}
__device__ __forceinline__ WideMap then(const WideMap& a, const WideMap& b) {
  const float m = a.m * b.m;
  const bool two = fabsf(m) >= 2.f;
  return WideMap{two ? 0.5f * m : m, apply(b, a.C), clamp_to(a.e + b.e + two, kMaxExp), a.cut || b.cut};
}
// v = m 2^e
__device__ __forceinline__ void split(float v, float* m, int* e) {
  const bool small = fabsf(v) < 0x1p-126f;  // zero or subnormal
  const unsigned b = __float_as_uint(small ? v * 0x1p64f : v);
  const int x = b >> 23 & 255;
  const bool plain = x != 255 && v != 0.f;
  *m = plain ? __uint_as_float((b & 0x807fffffu) | 0x3f800000u) : v;
  *e = plain ? x - (small ? 191 : 127) : 0;
}
// A 2^x times the gates of four rows, per column; |A| in [1, 2).  Their product is a normal number on the whole way where
// none is above 2^8 and the end is at least 2^-100.  A gate of zero takes the exponent far below any other's sum and leaves
// A as it was; where gates are too large or too small all the same, each one's exponent is taken apart.
constexpr int kZeroExp = -(1 << 20);
template <typename T, int E>
__device__ __forceinline__ void times(const Pack<T, E> (&gate)[4], float (&A)[E], int (&x)[E]) {
  float p[E];
  bool plain = true;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float a = to_f32(gate[0].v[e]), b = to_f32(gate[1].v[e]), c = to_f32(gate[2].v[e]), d = to_f32(gate[3].v[e]);
    p[e] = A[e] * a * b * c * d;
    plain = plain && fmaxf(fmaxf(fabsf(a), fabsf(b)), fmaxf(fabsf(c), fabsf(d))) <= 0x1p8f && fabsf(p[e]) >= 0x1p-100f;
  }
  if (!plain) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float top = 0.f;
      bool zero = false;
      p[e] = A[e];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = to_f32(gate[j].v[e]);
        zero = zero || a == 0.f;
        p[e] *= a == 0.f ? 1.f : a;
        top = fmaxf(top, fabsf(a));
      }
      if (zero) x[e] += kZeroExp;
      if (!(top <= 0x1p8f && fabsf(p[e]) >= 0x1p-100f)) {
        p[e] = A[e];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float m;
          int k;
          split(to_f32(gate[j].v[e]), &m, &k);
          if (m != 0.f) p[e] *= m;
          x[e] += k;
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const unsigned b = __float_as_uint(p[e]);
    x[e] += (int)(b >> 23 & 255) - 127;
    A[e] = __uint_as_float((b & 0x807fffffu) | 0x3f800000u);
  }
}

// Arrays of maps: A and C as 64 bits (a cut stands in the place of A, as a NaN that arithmetic does not make), or m and C
// with e beside them (kCutExp for a cut).
constexpr unsigned kCut = 0x7fc00c07u, kNan = 0x7fffffffu;
constexpr short kCutExp = SHRT_MIN;
struct Maps {
  uint2* ac;
  short* e;
  __device__ __forceinline__ void put(long long i, const Map& m) const {
    ac[i] = make_uint2(m.cut ? kCut : (m.A != m.A ? kNan : __float_as_uint(m.A)), __float_as_uint(m.C));
  }
  __device__ __forceinline__ void put(long long i, const WideMap& m) const {
    ac[i] = make_uint2(__float_as_uint(m.m), __float_as_uint(m.C));
    e[i] = m.cut ? kCutExp : (short)m.e;
  }
};
__device__ __forceinline__ void unpack(uint2 v, short, Map& m) {
  m = Map{__uint_as_float(v.x), __uint_as_float(v.y), v.x == kCut};
}
__device__ __forceinline__ void unpack(uint2 v, short e, WideMap& m) {
  m = WideMap{__uint_as_float(v.x), __uint_as_float(v.y), e, e == kCutExp};
}
template <typename M>
constexpr bool kHasExp = std::is_same<M, WideMap>::value;
template <typename M>  // from shared memory
__device__ __forceinline__ M map_at(const Maps& a, int i) {
  M m;
  unpack(a.ac[i], kHasExp<M> ? a.e[i] : 0, m);
  return m;
}
template <typename M>  // from an earlier kernel's array
__device__ __forceinline__ M map_of(const Maps& a, long long i) {
  M m;
  unpack(__ldg(a.ac + i), kHasExp<M> ? __ldg(a.e + i) : 0, m);
  return m;
}

template <int KIND>
using MapOf = std::conditional_t<KIND == ATLB_REC_DECAY, WideMap, Map>;

// ------------------------------------------------------------------------------------------------ windows
// Bit r of each word stands for row r of the group: `first` / `last` of its window, `none` when it belongs to no window
// or lies behind the last row.
struct Edges {
  unsigned first, last, none;
};

__device__ __forceinline__ void row_edges(const RecShape& S, long long n, bool* first, bool* last, bool* none) {
  if (n >= S.N) {
    *first = *last = false;
    *none = true;
  } else if (S.b) {
    const long long w = S.b[n];
    *none = w < 0 || w >= S.B;
    *first = n == 0 || S.b[n - 1] != w;
    *last = n + 1 == S.N || S.b[n + 1] != w;
  } else {
    const unsigned t = (unsigned)n % S.T;
    *none = false;
    *first = t == 0;
    *last = t + 1 == S.T;
  }
}

// The edges of this thread's group; a warp holds `per` neighbouring groups from g0 on, the thread's is number mine.
__device__ __forceinline__ Edges group_edges(const RecShape& S, long long g0, int per, int mine) {
  Edges e{0, 0, 0};
  for (int i = 0; i < per; ++i) {
    bool first, last, none;
    row_edges(S, (g0 + i) * kGroup + (threadIdx.x & 31), &first, &last, &none);
    const unsigned f = __ballot_sync(0xffffffffu, first), l = __ballot_sync(0xffffffffu, last),
                   v = __ballot_sync(0xffffffffu, none);
    if (i == mine) e = Edges{f, l, v};
  }
  return e;
}

__device__ __forceinline__ int window_of(const RecShape& S, long long n) {
  return S.b ? (int)S.b[n] : (int)((unsigned)n / S.T);
}

template <int E>
__device__ __forceinline__ void load_state(const float* p, long long row, int D, int c, bool in, float (&s)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = in && p ? p[row * D + c + e] : 0.f;
}

template <typename T, int E>
__device__ __forceinline__ Pack<T, E> load_or_zero(const T* p, bool in) {
  if (in) return load_pack<T, E>(p);
  Pack<T, E> r;
#pragma unroll
  for (int e = 0; e < E; ++e) r.v[e] = from_f32<T>(0.f);
  return r;
}

template <typename T>
struct Src {
  const T* p;
  long long ld;
};

// ------------------------------------------------------------------------------------------------ maps of the groups
// Threads `lanes` wide on a row, E neighbouring columns each; the CTA's groups are one chunk.  BWD walks from the last
// row to the first: in = dL/dh, and the state is u.  prefix: the map from the chunk's entry to the group's; chunk: the
// whole chunk's map.  1M rows of 64 bf16 columns: 65 us forward, 61 backward, 277 MB (4.3 and 4.5 TB/s); 4M rows 198 us
// (5.5 TB/s).
constexpr int kAhead = 4;  // rows in flight per thread

template <typename T, int E, int KIND, bool BWD>
__global__ void __launch_bounds__(kThreads, 4) k_rec_map(RecShape S, Src<T> gate, Src<T> in, const float* __restrict__ s0,
                                                      Maps prefix, Maps chunk) {
  using M = MapOf<KIND>;
  constexpr bool kWide = KIND == ATLB_REC_DECAY;
  constexpr int kSegs = 32 * E;  // segments x columns: 16 E, or 32 E where a warp takes a row
  __shared__ uint2 sm_ac[kThreads * E], seg_ac[kSegs];
  __shared__ short sm_e[kWide ? kThreads * E : 1], seg_e[kWide ? kSegs : 1];
  const Maps sm{sm_ac, sm_e}, seg{seg_ac, seg_e};
  const int sub = threadIdx.x & (S.lanes - 1), per = kThreads / S.lanes, mine = threadIdx.x / S.lanes;
  const int W = S.lanes * E, c = blockIdx.y * W + sub * E, warp_groups = S.lanes >= 32 ? 1 : 32 / S.lanes;
  const long long g = blockIdx.x * (long long)per + mine, r0 = g * kGroup;
  const bool col = c < S.D;
  const Edges ed = group_edges(S, g - mine % warp_groups, warp_groups, mine % warp_groups);
  const unsigned edge = (BWD ? ed.last : ed.first) | ed.none;
  float A[E], s[E];
  int x[kWide ? E : 1];  // A's exponents, where they are kept apart
#pragma unroll
  for (int e = 0; e < E; ++e) {
    A[e] = 1.f, s[e] = 0.f;
    if (kWide) x[e] = 0;
  }
  auto rows = [&](auto plain) {
    // rows are stepped through by pointer: a product with the stride per row costs as much as four additions.  Threads
    // behind the last column read the first and are not heard.
    const long long dg = BWD ? -gate.ld : gate.ld, di = BWD ? -in.ld : in.ld, from = r0 + (BWD ? kGroup - 1 : 0);
    const T *pg = gate.p + from * gate.ld + (col ? c : 0), *pi = in.p + from * in.ld + (col ? c : 0);
#pragma unroll 1
    for (int q = 0; q < kGroup; q += kAhead) {
      Pack<T, E> gp[kAhead], ip[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int r = BWD ? kGroup - 1 - q - j : q + j;
        const bool ok = decltype(plain)::value || !(ed.none >> r & 1);
        gp[j] = load_or_zero<T, E>(pg, ok);
        ip[j] = load_or_zero<T, E>(pi, ok);
        pg += dg;
        pi += di;
      }
      if constexpr (kWide) times(gp, A, x);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int r = BWD ? kGroup - 1 - q - j : q + j;
        if (!decltype(plain)::value && (edge >> r & 1)) {
          const bool ok = col && !(ed.none >> r & 1);
          load_state(s0, ok ? window_of(S, r0 + r) : 0, S.D, c, ok, s);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float a, w, v;
          row_terms<KIND>(gp[j].v[e], ip[j].v[e], &a, &w, &v);
          s[e] = BWD ? a * (to_f32(ip[j].v[e]) + s[e]) : fmaf(a, s[e], v);
          if (!kWide) A[e] *= a;
        }
      }
    }
  };
  if (__any_sync(0xffffffffu, edge != 0))
    rows(std::false_type());
  else
    rows(std::true_type());
  // joined along the walk, per column: kSeg groups by one thread, then the segments, then the groups again
  const int at = BWD ? per - 1 - mine : mine, segs = (per + kSeg - 1) / kSeg;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if constexpr (kWide) {
      const bool zero = x[e] < kZeroExp / 2;
      sm.put(at * W + sub * E + e, WideMap{zero ? 0.f : A[e], s[e], zero ? 0 : x[e], edge != 0});
    } else {
      sm.put(at * W + sub * E + e, Map{A[e], s[e], edge != 0});
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < segs * W; i += kThreads) {
    const int x = i % W, k0 = i / W * kSeg;
    M m = M::identity();
    for (int k = k0; k < k0 + kSeg && k < per; k += 4) {  // per is a multiple of eight; four loads on the way at once
      M next[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) next[j] = map_at<M>(sm, (k + j) * W + x);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sm.put((k + j) * W + x, m);
        m = then(m, next[j]);
      }
    }
    seg.put(i, m);
  }
  __syncthreads();
  for (int x = threadIdx.x; x < W; x += kThreads) {
    M m = M::identity();
    for (int k = 0; k < segs; ++k) {
      const M next = map_at<M>(seg, k * W + x);
      seg.put(k * W + x, m);
      m = then(m, next);
    }
    if (blockIdx.y * W + x < S.D) chunk.put(blockIdx.x * (long long)S.D + blockIdx.y * W + x, m);
  }
  __syncthreads();
  if (col && g < S.groups) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      prefix.put(g * S.D + c + e,
                 then(map_at<M>(seg, at / kSeg * W + sub * E + e), map_at<M>(sm, at * W + sub * E + e)));
  }
}

// ------------------------------------------------------------------------------------------------ between the chunks
// state[k]: what enters chunk k along the walk.  Per column kChainSegs threads each join a run of chunks; the runs are
// joined four to a warp, the warps' eight to a thread of the first warp, and every thread walks its run again from the
// true state.
__device__ __forceinline__ Map map_above(const Map& m, int by) {
  return Map{__shfl_up_sync(0xffffffffu, m.A, by), __shfl_up_sync(0xffffffffu, m.C, by),
             (bool)__shfl_up_sync(0xffffffffu, (int)m.cut, by)};
}
__device__ __forceinline__ WideMap map_above(const WideMap& m, int by) {
  return WideMap{__shfl_up_sync(0xffffffffu, m.m, by), __shfl_up_sync(0xffffffffu, m.C, by),
                 __shfl_up_sync(0xffffffffu, m.e, by)};
}
// The map of the runs before this thread's in its warp (lanes of one column are kChainCols apart); m becomes the map up
// to its own.
template <typename M>
__device__ __forceinline__ M warp_join(M& m, int lane) {
#pragma unroll
  for (int by = kChainCols; by < 32; by *= 2) {
    const M p = map_above(m, by);
    if (lane >= by) m = then(p, m);
  }
  const M before = map_above(m, kChainCols);
  return lane < kChainCols ? M::identity() : before;
}

template <typename M, bool BWD>
__global__ void __launch_bounds__(kChainCols * kChainSegs) k_rec_chain(Maps chunk, int chunks, int D,
                                                                       float* __restrict__ state) {
  constexpr int kWarps = kChainCols * kChainSegs / 32, kEach = kWarps * kChainCols / 32;
  __shared__ uint2 sm_ac[kWarps * kChainCols];
  __shared__ short sm_e[kWarps * kChainCols];
  __shared__ float in[kWarps][kChainCols];
  const Maps sm{sm_ac, sm_e};
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int x = threadIdx.x % kChainCols, sg = threadIdx.x / kChainCols, c = blockIdx.x * kChainCols + x;
  const int run = (chunks + kChainSegs - 1) / kChainSegs, k0 = sg * run, k1 = min(k0 + run, chunks);
  auto at = [&](int k) { return (long long)(BWD ? chunks - 1 - k : k) * D + c; };
  M m = M::identity();
  if (c < D) {
#pragma unroll 8
    for (int k = k0; k < k1; ++k) m = then(m, map_of<M>(chunk, at(k)));
  }
  const M before = warp_join(m, lane);
  if (lane >= 32 - kChainCols) sm.put(wid * kChainCols + x, m);
  __syncthreads();
  if (wid == 0) {
    const int w0 = lane / kChainCols * kEach;
    M t = M::identity();
#pragma unroll
    for (int w = 0; w < kEach; ++w) t = then(t, map_at<M>(sm, (w0 + w) * kChainCols + x));
    float s = apply(warp_join(t, lane), 0.f);
#pragma unroll
    for (int w = 0; w < kEach; ++w) {
      in[w0 + w][x] = s;
      s = apply(map_at<M>(sm, (w0 + w) * kChainCols + x), s);
    }
  }
  __syncthreads();
  if (c >= D) return;
  float s = apply(before, in[wid][x]);
#pragma unroll 8
  for (int k = k0; k < k1; ++k) {
    const M next = map_of<M>(chunk, at(k));
    state[at(k)] = s;
    s = apply(next, s);
  }
}

// The state that enters group g: the chunk's, through the map from there.  per: groups of a chunk.
template <typename M, int E>
__device__ __forceinline__ void group_state(const RecShape& S, const Maps& prefix, const float* state, long long g,
                                            int per, int c, bool in, float (&s)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    s[e] = 0.f;
    if (in && S.linked)
      s[e] = apply(map_of<M>(prefix, g * S.D + c + e), S.chunks > 1 ? state[g / per * S.D + c + e] : 0.f);
  }
}

// ------------------------------------------------------------------------------------------------ replay, forward
// 1M rows of 64 bf16 columns: 73 us, 400 MB of DRAM traffic with the kept states (5.5 TB/s); 4M fp16 rows without them
// 235 us (6.7 TB/s).  Under the cap of 5 CTAs (48 registers) four bf16 columns spill 68 bytes a thread.  A cap of 4 has no
// spills: 362 and 225 us on the device for 1M rows of 64 and 32k of 1024, both ways, where 5 take 365 and 230, but 466
// for 4M fp16 rows forward, where 5 take 459.
template <typename T, int E, int KIND>
__global__ void __launch_bounds__(kThreads, 5) k_rec_fwd(RecShape S, Src<T> gate, Src<T> x, const float* __restrict__ h0,
                                                      Maps prefix, const float* __restrict__ state, T* __restrict__ h,
                                                      float* __restrict__ hT, float* __restrict__ saved) {
  const int sub = threadIdx.x & (S.lanes - 1), per = kThreads / S.lanes, mine = threadIdx.x / S.lanes;
  const int c = (blockIdx.y * S.lanes + sub) * E, warp_groups = S.lanes >= 32 ? 1 : 32 / S.lanes;
  // from the last chunk to the first: what the maps' kernel read last may still be in L2
  const long long g = (gridDim.x - 1 - blockIdx.x) * (long long)per + mine, r0 = g * kGroup;
  const bool col = c < S.D;
  const Edges ed = group_edges(S, g - mine % warp_groups, warp_groups, mine % warp_groups);
  const unsigned edge = ed.first | ed.none;
  float s[E];
  group_state<MapOf<KIND>>(S, prefix, state, g, per, c, col && g < S.groups, s);
  auto rows = [&](auto plain) {
    const T *pg = gate.p + r0 * gate.ld + (col ? c : 0), *px = x.p + r0 * x.ld + (col ? c : 0);
    T* ph = h + r0 * S.D + c;
#pragma unroll 1
    for (int q = 0; q < kGroup; q += kAhead) {
      Pack<T, E> gp[kAhead], xp[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const bool ok = decltype(plain)::value || !(ed.none >> (q + j) & 1);
        gp[j] = load_or_zero<T, E>(pg, ok);
        xp[j] = load_or_zero<T, E>(px, ok);
        pg += gate.ld;
        px += x.ld;
      }
      if (saved && q % kPart == 0 && col && r0 + q < S.N) {
#pragma unroll
        for (int e = 0; e < E; ++e) saved[(r0 + q) / kPart * S.D + c + e] = s[e];
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int r = q + j;
        if (!decltype(plain)::value && (edge >> r & 1)) {
          const bool ok = col && !(ed.none >> r & 1);
          load_state(h0, ok ? window_of(S, r0 + r) : 0, S.D, c, ok, s);
        }
        Pack<T, E> o;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float a, w, v;
          row_terms<KIND>(gp[j].v[e], xp[j].v[e], &a, &w, &v);
          s[e] = fmaf(a, s[e], v);
          o.v[e] = from_f32<T>(s[e]);
        }
        if (col && (decltype(plain)::value || r0 + r < S.N)) store_pack(ph, o);
        ph += S.D;
        if (!decltype(plain)::value && hT && col && (ed.last & ~ed.none) >> r & 1) {
          const int win = window_of(S, r0 + r);
#pragma unroll
          for (int e = 0; e < E; ++e) hT[(long long)win * S.D + c + e] = s[e];
        }
      }
    }
  };
  if (__any_sync(0xffffffffu, (edge | (hT ? ed.last : 0)) != 0))
    rows(std::false_type());
  else
    rows(std::true_type());
}

// One row per window (a step of running windows): row by row in parallel, E columns per thread.
template <typename T, int E, int KIND>
__global__ void __launch_bounds__(kThreads) k_rec_step(RecShape S, Src<T> gate, Src<T> x, const float* __restrict__ h0,
                                                       T* __restrict__ h, float* __restrict__ hT,
                                                       float* __restrict__ saved) {
  const int per_row = S.D / E;
  const long long i = blockIdx.x * (long long)kThreads + threadIdx.x, n = i / per_row;
  const int c = (int)(i - n * per_row) * E;
  if (n >= S.N) return;
  const Pack<T, E> gp = load_pack<T, E>(gate.p + n * gate.ld + c), xp = load_pack<T, E>(x.p + n * x.ld + c);
  Pack<T, E> o;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float a, w, v;
    row_terms<KIND>(gp.v[e], xp.v[e], &a, &w, &v);
    const float s = fmaf(a, h0 ? h0[n * S.D + c + e] : 0.f, v);
    o.v[e] = from_f32<T>(s);
    if (hT) hT[n * S.D + c + e] = s;
    // every row begins a window, so the backward pass takes h0 in the place of what it finds here
    if (saved && n % kPart == 0) saved[n / kPart * S.D + c + e] = 0.f;
  }
  store_pack(h + n * S.D + c, o);
}

// ------------------------------------------------------------------------------------------------ replay, backward
// lanes_b threads on a row, E columns each (4 bytes), a group per `lanes_b` threads.  Each part of the group, the last
// one first: its rows in registers, the states forward from the one the forward pass kept, then u backward.  The states
// are found again in fp32 rather than read from h, which was rounded: h - x would lose what the gate's gradient needs.
// 1M rows of 64 bf16 columns: 145 us, 660 MB (4.6 TB/s).  (16-bit sigmoid rows spill 12 to 20 bytes a thread under the cap.)
template <typename T, int E, int KIND>
__global__ void __launch_bounds__(kThreads, 3) k_rec_bwd(RecShape S, int lanes_b, Src<T> gate, Src<T> x, Src<T> gh,
                                                         const float* __restrict__ h0, const float* __restrict__ ghT,
                                                         const float* __restrict__ saved, Maps prefix,
                                                         const float* __restrict__ state, T* __restrict__ ggate,
                                                         T* __restrict__ gx, float* __restrict__ gh0) {
  const int sub = threadIdx.x & (lanes_b - 1), per = kThreads / lanes_b, mine = threadIdx.x / lanes_b;
  const int c = (blockIdx.y * lanes_b + sub) * E, warp_groups = 32 / lanes_b;
  // from the first chunk to the last: the maps' kernel walked towards the first
  const long long g = blockIdx.x * (long long)per + mine, r0 = g * kGroup;
  const bool col = c < S.D;
  const Edges ed = group_edges(S, g - mine % warp_groups, warp_groups, mine % warp_groups);
  const unsigned edge = ed.first | ed.none, edge_u = ed.last | ed.none;
  float u[E];
  group_state<MapOf<KIND>>(S, prefix, state, g, kThreads / S.lanes, c, col && g < S.groups, u);
  auto part = [&](int lo, auto plain) {
    Pack<T, E> xp[kPart], dp[kPart];
    float a[kPart][E], w[kPart][E], hp[kPart][E], s[E];
    const int cc = col ? c : 0;
    const T *pg = gate.p + (r0 + lo) * gate.ld + cc, *px = x.p + (r0 + lo) * x.ld + cc,
            *pd = gh.p + (r0 + lo) * gh.ld + cc;
    Pack<T, E> gp[kPart];
#pragma unroll
    for (int r = 0; r < kPart; ++r) {
      const bool ok = decltype(plain)::value || !(ed.none >> (lo + r) & 1);
      gp[r] = load_or_zero<T, E>(pg, ok);
      xp[r] = load_or_zero<T, E>(px, ok);
      dp[r] = load_or_zero<T, E>(pd, ok);
      pg += gate.ld;
      px += x.ld;
      pd += gh.ld;
    }
    load_state(saved, (r0 + lo) / kPart, S.D, c, col && r0 + lo < S.N, s);
#pragma unroll
    for (int r = 0; r < kPart; ++r) {
      if (!decltype(plain)::value && (edge >> (lo + r) & 1)) {
        const bool ok = col && !(ed.none >> (lo + r) & 1);
        load_state(h0, ok ? window_of(S, r0 + lo + r) : 0, S.D, c, ok, s);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float v;
        const float xv = to_f32(xp[r].v[e]);
        row_terms<KIND>(gp[r].v[e], xp[r].v[e], &a[r][e], &w[r][e], &v);
        hp[r][e] = KIND == ATLB_REC_SIGMOID ? w[r][e] * (s[e] - xv) : s[e];  // what the gate's gradient takes
        s[e] = fmaf(a[r][e], s[e], v);
      }
    }
    long long at = (r0 + lo + kPart - 1) * S.D + c;
#pragma unroll
    for (int r = kPart - 1; r >= 0; --r) {
      if (!decltype(plain)::value && (edge_u >> (lo + r) & 1)) {
        const bool ok = col && !(ed.none >> (lo + r) & 1);
        load_state(ghT, ok ? window_of(S, r0 + lo + r) : 0, S.D, c, ok, u);
      }
      Pack<T, E> og, ox;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float gt = to_f32(dp[r].v[e]) + u[e];
        u[e] = a[r][e] * gt;
        og.v[e] = from_f32<T>(KIND == ATLB_REC_SIGMOID ? u[e] * hp[r][e] : gt * hp[r][e]);
        ox.v[e] = from_f32<T>(KIND == ATLB_REC_SIGMOID ? gt * w[r][e] : gt);
      }
      if (col && (decltype(plain)::value || r0 + lo + r < S.N)) {
        store_pack(ggate + at, og);
        store_pack(gx + at, ox);
      }
      at -= S.D;
      if (!decltype(plain)::value && gh0 && col && (ed.first & ~ed.none) >> (lo + r) & 1) {
        const int win = window_of(S, r0 + lo + r);
#pragma unroll
        for (int e = 0; e < E; ++e) gh0[(long long)win * S.D + c + e] = u[e];
      }
    }
  };
  const bool some = __any_sync(0xffffffffu, (edge | edge_u) != 0);
#pragma unroll 1
  for (int lo = kGroup - kPart; lo >= 0; lo -= kPart) {
    if (some)
      part(lo, std::false_type());
    else
      part(lo, std::true_type());
  }
}

long long groups_of(long long N) { return (N + kGroup - 1) / kGroup; }

struct RecWs {
  Maps prefix, chunk;
  float* state;
  size_t bytes;
};

// Room for chunks of the fewest groups (32 threads on a row).
RecWs carve(void* ws, long long N, long long D) {
  Carve c(ws);
  RecWs w;
  const long long g = groups_of(N), k = (g + kThreads / 32 - 1) / (kThreads / 32);
  w.prefix.ac = c.take<uint2>(g * D);
  w.chunk.ac = c.take<uint2>(k * D);
  w.prefix.e = c.take<short>(g * D);
  w.chunk.e = c.take<short>(k * D);
  w.state = c.take<float>(k * D);
  w.bytes = c.bytes_needed();
  return w;
}

// Packed windows may be empty: what theirs are to hold is copied ahead of the kernels, which overwrite the others'.
int fill_state(float* dst, const float* src, long long n, bool packed, cudaStream_t s) {
  if (!dst || n <= 0 || !packed) return ATLB_OK;
  const cudaError_t e = src ? cudaMemcpyAsync(dst, src, n * sizeof(float), cudaMemcpyDeviceToDevice, s)
                            : cudaMemsetAsync(dst, 0, n * sizeof(float), s);
  return e == cudaSuccess ? ATLB_OK : launch_status("recurrence");
}

template <typename Fn>
int with_kind(int kind, Fn&& fn) {
  if (kind == ATLB_REC_SIGMOID) return fn(std::integral_constant<int, ATLB_REC_SIGMOID>());
  return fn(std::integral_constant<int, ATLB_REC_DECAY>());
}

// The bytes that every row of the arrays and D are whole multiples of.
struct Unit {
  long long bits;
  template <typename T>
  void add(const void* p, long long ld) { bits |= (long long)(reinterpret_cast<uintptr_t>(p) | (ld * sizeof(T))); }
  bool fits(int bytes) const { return bits % bytes == 0; }
};

// Lanes on a row of D columns with E each: a power of two, at most `most`.
int lanes_for(long long D, int E, int most) {
  int l = 1;
  while (l < most && l * E < D) l *= 2;
  return l;
}

// Shape for k_rec_map and k_rec_fwd with E columns per thread: 16 threads read a whole 128-byte line of a row, single
// columns take a whole warp (odd widths, 1.9 times the time of even ones: D = 255 against 256 in bf16 535 against 277 us).
// 16 bytes per thread halve the warps that fit and measured 429 us where 8 took 372.
RecShape make_shape(long long N, long long B, long long D, const long long* b, int E) {
  RecShape S;
  S.N = N;
  S.T = b ? 0 : (unsigned)(N / B);
  S.B = (int)B;
  S.D = (int)D;
  S.b = b;
  S.lanes = lanes_for(D, E, E > 1 ? 128 / kBytes : 32);
  S.groups = (int)groups_of(N);
  S.chunks = (S.groups + kThreads / S.lanes - 1) / (kThreads / S.lanes);
  S.linked = S.groups > 1 && (b || kGroup % S.T != 0);
  return S;
}

template <typename T, int E, int KIND, bool BWD>
void find_states(const RecShape& S, Src<T> gate, Src<T> in, const float* s0, const RecWs& w, cudaStream_t s) {
  if (!S.linked) return;
  const int W = S.lanes * E;
  launch(k_rec_map<T, E, KIND, BWD>, dim3(S.chunks, (S.D + W - 1) / W), kThreads, 0, s, S, gate, in, s0, w.prefix,
         w.chunk);
  if (S.chunks > 1)
    launch(k_rec_chain<MapOf<KIND>, BWD>, (S.D + kChainCols - 1) / kChainCols, kChainCols * kChainSegs, 0, s, w.chunk, S.chunks, S.D,
           w.state);
}

}  // namespace

size_t recurrence_workspace_bytes(long long N, long long D) { return carve(nullptr, N, D).bytes; }
size_t recurrence_saved_bytes(long long N, long long D) {
  return (size_t)((N + kPart - 1) / kPart) * D * sizeof(float);
}

int recurrence_fwd(int dtype, int kind, const void* gate, long long ldg, const void* x, long long ldx,
                   const long long* b, long long N, long long B, long long D, const float* h0, void* h, float* hT,
                   float* saved, void* ws, cudaStream_t s) {
  if (D <= 0) return ATLB_OK;
  if (int st = fill_state(hT, h0, B * D, b || N <= 0, s)) return st;
  if (N <= 0) return ATLB_OK;
  const RecWs w = carve(ws, N, D);
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    Unit u{0};
    u.add<T>(gate, ldg);
    u.add<T>(x, ldx);
    u.add<T>(h, D);
    return with_kind(kind, [&](auto kd) {
      constexpr int KIND = decltype(kd)::value;
      const Src<T> sg{(const T*)gate, ldg}, sx{(const T*)x, ldx};
      auto go = [&](auto el) {
        constexpr int E = decltype(el)::value;
        const RecShape S = make_shape(N, B, D, b, E);
        const int W = S.lanes * E;
        if (!b && S.T == 1) {
          launch(k_rec_step<T, E, KIND>, (unsigned)((N * (D / E) + kThreads - 1) / kThreads), kThreads, 0, s, S, sg, sx, h0,
                 (T*)h, hT, saved);
          return launch_status("recurrence_fwd");
        }
        find_states<T, E, KIND, false>(S, sg, sx, h0, w, s);
        launch(k_rec_fwd<T, E, KIND>, dim3(S.chunks, (S.D + W - 1) / W), kThreads, 0, s, S, sg, sx, h0, w.prefix, w.state,
               (T*)h, hT, saved);
        return launch_status("recurrence_fwd");
      };
      if (u.fits(kBytes)) return go(std::integral_constant<int, kBytes / sizeof(T)>());
      return go(std::integral_constant<int, 1>());
    });
  });
}

int recurrence_bwd(int dtype, int kind, const void* gate, long long ldg, const void* x, long long ldx,
                   const long long* b, long long N, long long B, long long D, const float* h0, const float* saved,
                   const void* gh, long long ldgh, const float* ghT, void* ggate, void* gx, float* gh0, void* ws,
                   cudaStream_t s) {
  if (D <= 0) return ATLB_OK;
  if (int st = fill_state(gh0, ghT, B * D, b || N <= 0, s)) return st;
  if (N <= 0) return ATLB_OK;
  const RecWs w = carve(ws, N, D);
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    Unit u{0};
    u.add<T>(gate, ldg);
    u.add<T>(x, ldx);
    u.add<T>(gh, ldgh);
    u.add<T>(ggate, D);
    u.add<T>(gx, D);
    return with_kind(kind, [&](auto kd) {
      constexpr int KIND = decltype(kd)::value;
      const Src<T> sg{(const T*)gate, ldg}, sx{(const T*)x, ldx}, sd{(const T*)gh, ldgh};
      RecShape S;
      if (u.fits(kBytes)) {
        constexpr int E = kBytes / sizeof(T);
        S = make_shape(N, B, D, b, E);
        find_states<T, E, KIND, true>(S, sg, sd, ghT, w, s);
      } else {
        S = make_shape(N, B, D, b, 1);
        find_states<T, 1, KIND, true>(S, sg, sd, ghT, w, s);
      }
      auto go = [&](auto el) {
        constexpr int E = decltype(el)::value;
        const int lanes = lanes_for(D, E, 32), per = kThreads / lanes;
        launch(k_rec_bwd<T, E, KIND>, dim3((S.groups + per - 1) / per, (unsigned)((D + lanes * E - 1) / (lanes * E))),
               kThreads, 0, s, S, lanes, sg, sx, sd, h0, ghT, saved, w.prefix, w.state, (T*)ggate, (T*)gx, gh0);
        return launch_status("recurrence_bwd");
      };
      if constexpr (sizeof(T) == 2) {
        if (u.fits(4)) return go(std::integral_constant<int, 2>());
      }
      return go(std::integral_constant<int, 1>());
    });
  });
}

}  // namespace atlb
