// Gated linear recurrence over packed windows of rows (include/atl_b200.h, atlb_recurrence_*).
//
//   decay    h_t = a_t h_(t-1) + x_t                      a_t = gate_t
//   sigmoid  h_t = a_t h_(t-1) + (1 - a_t) x_t            a_t = 1 / (1 + exp(-gate_t))
// per column, with h before a window's first row equal to h0 (or zero).  Backward, from the last row of a window:
//   g_t = dh_t + u_(t+1)   (last row: dh_t + dhT)         u_t = a_t g_t          dh0 = u of the first row
//   decay    dgate = g_t h_(t-1)                          dx = g_t
//   sigmoid  dgate = g_t (h_(t-1) - x_t) a_t (1 - a_t)    dx = (1 - a_t) g_t
//
// Rows are cut into chunks of kRows; over a chunk the recurrence is an affine map h -> A h + C of the state that
// enters it (and u -> A u + C' backward, with the same A), so the chunks' maps are found side by side, chained, and
// the rows then replayed from their true state.  States, maps and sums are fp32; an output is rounded once.  A row
// that begins a window drops what comes before it by selection, so nothing of one window, NaN included, reaches
// another.
#include "vec.cuh"

namespace atlb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kWarpRows = 16;                 // rows of one warp
constexpr int kRows = kWarps * kWarpRows;     // rows of one chunk

struct RecShape {
  long long N, T;          // rows; rows per window where b is null
  int B, D;
  const long long* b;      // window of every row, or null
};

// Windows of a warp's rows: bit i of `first` / `last` marks row i as the first / last of its window, `valid` as one
// that belongs to a window at all; win is the window of row `lane`.
struct RowFlags {
  unsigned first, last, valid;
  int win;
};

__device__ __forceinline__ RowFlags row_flags(const RecShape& S, long long r0, int lane) {
  const long long n = r0 + lane;
  bool first = false, last = false, valid = false;
  int win = -1;
  if (lane < kWarpRows && n < S.N) {
    if (S.b) {
      const long long w = S.b[n];
      valid = w >= 0 && w < S.B;
      first = n == 0 || S.b[n - 1] != w;
      last = n + 1 == S.N || S.b[n + 1] != w;
      win = valid ? (int)w : -1;
    } else {
      win = (int)(n / S.T);
      const long long t = n - win * S.T;
      valid = true;
      first = t == 0;
      last = t + 1 == S.T;
    }
  }
  RowFlags f;
  f.first = __ballot_sync(0xffffffffu, first);
  f.last = __ballot_sync(0xffffffffu, last);
  f.valid = __ballot_sync(0xffffffffu, valid);
  f.win = win;
  return f;
}

// a = 1 / (1 + exp(-z)) and 1 - a, each from exp(-|z|), which does not overflow, so neither cancels.
__device__ __forceinline__ void sigmoid2(float z, float* a, float* na) {
  const float e = __expf(-fabsf(z));
  const float r = __fdividef(1.f, 1.f + e), s = e * r;
  *a = z >= 0.f ? r : s;
  *na = z >= 0.f ? s : r;
}

template <int KIND>
__device__ __forceinline__ void row_coeff(float gate, float* a, float* w) {
  if (KIND == ATLB_REC_SIGMOID) {
    sigmoid2(gate, a, w);
  } else {
    *a = gate;
    *w = 1.f;
  }
}

// State after rows whose map is (A, C).  A zero state leaves C: the product of many gates above one may overflow.
__device__ __forceinline__ float through(float A, float C, float s) { return s == 0.f ? C : fmaf(A, s, C); }

template <typename T, int E>
__device__ __forceinline__ Pack<T, E> load_row(const T* p, long long ld, long long n, int c, bool in) {
  Pack<T, E> r;
  if (in) {
    r = load_pack<T, E>(p + n * ld + c);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) r.v[e] = from_f32<T>(0.f);
  }
  return r;
}

// Maps of the chunks, forward (BWD false: C is the state after the chunk from zero) or backward (u before it).
// map holds A, then C, each (chunks, D); drop[chunk] is set when a window border inside the chunk cuts it off from
// the state that enters it.
template <typename T, int E, int KIND, bool BWD>
__global__ void __launch_bounds__(kThreads) k_rec_map(RecShape S, const T* __restrict__ gate, long long ldg,
                                                      const T* __restrict__ in, long long ldi,
                                                      const float* __restrict__ h0, const float* __restrict__ ghT,
                                                      long long chunks, float* __restrict__ map,
                                                      int* __restrict__ drop) {
  __shared__ float sA[kWarps][32 * E], sC[kWarps][32 * E];
  __shared__ int sDrop[kWarps];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c = (blockIdx.y * 32 + lane) * E;
  const bool col = c < S.D;
  const long long r0 = blockIdx.x * (long long)kRows + wid * kWarpRows;
  const RowFlags f = row_flags(S, r0, lane);
  float A[E], C[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { A[e] = 1.f; C[e] = 0.f; }
  bool cut = false;
#pragma unroll
  for (int k = 0; k < kWarpRows; ++k) {
    const int i = BWD ? kWarpRows - 1 - k : k;
    const long long n = r0 + i;
    const bool valid = f.valid >> i & 1, edge = (BWD ? f.last : f.first) >> i & 1;
    const int w = __shfl_sync(0xffffffffu, f.win, i);
    if (n >= S.N) continue;
    if (!valid) {
      cut = true;
#pragma unroll
      for (int e = 0; e < E; ++e) C[e] = 0.f;
      continue;
    }
    const Pack<T, E> gp = load_row<T, E>(gate, ldg, n, c, col), ip = load_row<T, E>(in, ldi, n, c, col);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float a, q;
      row_coeff<KIND>(to_f32(gp.v[e]), &a, &q);
      const float v = to_f32(ip.v[e]);
      if (BWD) {  // u = a (dh + u_next)
        const float nx = edge ? (ghT && col ? ghT[(long long)w * S.D + c + e] : 0.f) : C[e];
        C[e] = a * (v + nx);
      } else {
        const float pv = edge ? (h0 && col ? h0[(long long)w * S.D + c + e] : 0.f) : C[e];
        C[e] = fmaf(a, pv, KIND == ATLB_REC_SIGMOID ? q * v : v);
      }
      A[e] *= a;
    }
    cut = cut || edge;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) { sA[wid][lane * E + e] = A[e]; sC[wid][lane * E + e] = C[e]; }
  if (lane == 0) sDrop[wid] = cut;
  __syncthreads();
  if (wid == 0 && col) {
    bool d = false;
    float a[E], s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) { a[e] = 1.f; s[e] = 0.f; }
    for (int k = 0; k < kWarps; ++k) {
      const int w = BWD ? kWarps - 1 - k : k;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s[e] = sDrop[w] ? sC[w][lane * E + e] : through(sA[w][lane * E + e], sC[w][lane * E + e], s[e]);
        a[e] *= sA[w][lane * E + e];
      }
      d = d || sDrop[w];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      map[blockIdx.x * (long long)S.D + c + e] = a[e];
      map[(chunks + blockIdx.x) * (long long)S.D + c + e] = s[e];
    }
    if (lane == 0 && blockIdx.y == 0) drop[blockIdx.x] = d;
  }
}

// Chains the maps: state[chunk] is what enters the chunk (from the left, or BWD from the right).
template <bool BWD>
__global__ void __launch_bounds__(kThreads) k_rec_chain(const float* __restrict__ map, const int* __restrict__ drop,
                                                        long long chunks, int D, float* __restrict__ state) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= D) return;
  float s = 0.f;
  for (long long k = 0; k < chunks; ++k) {
    const long long q = BWD ? chunks - 1 - k : k;
    state[q * D + c] = s;
    const float A = map[q * D + c], C = map[(chunks + q) * D + c];
    s = drop[q] ? C : through(A, C, s);
  }
}

// The state that enters a warp's rows: the chunk's, passed through the warps before it (BWD: after it).
template <int E, bool BWD>
__device__ __forceinline__ void warp_state(const float (*sA)[32 * E], const float (*sC)[32 * E], const int* sDrop,
                                           int wid, int lane, float (&s)[E]) {
  for (int k = 0; k < (BWD ? kWarps - 1 - wid : wid); ++k) {
    const int w = BWD ? kWarps - 1 - k : k;
#pragma unroll
    for (int e = 0; e < E; ++e)
      s[e] = sDrop[w] ? sC[w][lane * E + e] : through(sA[w][lane * E + e], sC[w][lane * E + e], s[e]);
  }
}

template <typename T, int E, int KIND>
__global__ void __launch_bounds__(kThreads) k_rec_fwd(RecShape S, const T* __restrict__ gate, long long ldg,
                                                      const T* __restrict__ x, long long ldx,
                                                      const float* __restrict__ h0, const float* __restrict__ state,
                                                      T* __restrict__ h, float* __restrict__ hT) {
  __shared__ float sA[kWarps][32 * E], sC[kWarps][32 * E];
  __shared__ int sDrop[kWarps];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c = (blockIdx.y * 32 + lane) * E;
  const bool col = c < S.D;
  const long long r0 = blockIdx.x * (long long)kRows + wid * kWarpRows;
  const RowFlags f = row_flags(S, r0, lane);
  Pack<T, E> gp[kWarpRows], xp[kWarpRows];
#pragma unroll
  for (int i = 0; i < kWarpRows; ++i) {
    const bool in = col && (f.valid >> i & 1);
    gp[i] = load_row<T, E>(gate, ldg, r0 + i, c, in);
    xp[i] = load_row<T, E>(x, ldx, r0 + i, c, in);
  }
  float s[E];
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {  // the warp's map, then the rows from their true state
    float A[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      A[e] = 1.f;
      if (pass == 0) s[e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < kWarpRows; ++i) {
      const int w = __shfl_sync(0xffffffffu, f.win, i);
      const bool valid = f.valid >> i & 1, first = f.first >> i & 1, last = f.last >> i & 1;
      Pack<T, E> out;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float a, q;
        row_coeff<KIND>(to_f32(gp[i].v[e]), &a, &q);
        const float v = to_f32(xp[i].v[e]);
        const float pv = first ? (h0 && col && valid ? h0[(long long)w * S.D + c + e] : 0.f) : s[e];
        s[e] = valid ? fmaf(a, pv, KIND == ATLB_REC_SIGMOID ? q * v : v) : 0.f;
        A[e] *= a;
        out.v[e] = from_f32<T>(s[e]);
      }
      if (pass == 1 && col && r0 + i < S.N) {
        store_pack(h + (r0 + i) * S.D + c, out);
        if (hT && last && valid) {
#pragma unroll
          for (int e = 0; e < E; ++e) hT[(long long)w * S.D + c + e] = s[e];
        }
      }
    }
    if (pass == 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sA[wid][lane * E + e] = A[e];
        sC[wid][lane * E + e] = s[e];
      }
      if (lane == 0) sDrop[wid] = f.first != 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] = col ? state[blockIdx.x * (long long)S.D + c + e] : 0.f;
      warp_state<E, false>(sA, sC, sDrop, wid, lane, s);
    }
  }
}

template <typename T, int E, int KIND>
__global__ void __launch_bounds__(kThreads) k_rec_bwd(RecShape S, const T* __restrict__ gate, long long ldg,
                                                      const T* __restrict__ x, long long ldx,
                                                      const T* __restrict__ gh, long long ldgh,
                                                      const float* __restrict__ h0, const float* __restrict__ ghT,
                                                      const float* __restrict__ saved,
                                                      const float* __restrict__ state, T* __restrict__ ggate,
                                                      T* __restrict__ gx, float* __restrict__ gh0) {
  __shared__ float sA[kWarps][32 * E], sC[kWarps][32 * E], sU[kWarps][32 * E];
  __shared__ int sDrop[kWarps], sDropU[kWarps];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c = (blockIdx.y * 32 + lane) * E;
  const bool col = c < S.D;
  const long long r0 = blockIdx.x * (long long)kRows + wid * kWarpRows;
  const RowFlags f = row_flags(S, r0, lane);
  Pack<T, E> gp[kWarpRows], xp[kWarpRows], dp[kWarpRows];
#pragma unroll
  for (int i = 0; i < kWarpRows; ++i) {
    const bool in = col && (f.valid >> i & 1);
    gp[i] = load_row<T, E>(gate, ldg, r0 + i, c, in);
    xp[i] = load_row<T, E>(x, ldx, r0 + i, c, in);
    dp[i] = load_row<T, E>(gh, ldgh, r0 + i, c, in);
  }
  float s[E], u[E], A[E];
#pragma unroll
  for (int e = 0; e < E; ++e) { s[e] = 0.f; u[e] = 0.f; A[e] = 1.f; }
  // the warp's two maps
#pragma unroll
  for (int i = 0; i < kWarpRows; ++i) {
    const int w = __shfl_sync(0xffffffffu, f.win, i);
    const bool valid = f.valid >> i & 1, first = f.first >> i & 1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float a, q;
      row_coeff<KIND>(to_f32(gp[i].v[e]), &a, &q);
      const float v = to_f32(xp[i].v[e]);
      const float pv = first ? (h0 && col && valid ? h0[(long long)w * S.D + c + e] : 0.f) : s[e];
      s[e] = valid ? fmaf(a, pv, KIND == ATLB_REC_SIGMOID ? q * v : v) : 0.f;
      A[e] *= a;
    }
  }
#pragma unroll
  for (int i = kWarpRows - 1; i >= 0; --i) {
    const int w = __shfl_sync(0xffffffffu, f.win, i);
    const bool valid = f.valid >> i & 1, last = f.last >> i & 1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float a, q;
      row_coeff<KIND>(to_f32(gp[i].v[e]), &a, &q);
      const float nx = last ? (ghT && col && valid ? ghT[(long long)w * S.D + c + e] : 0.f) : u[e];
      u[e] = valid ? a * (to_f32(dp[i].v[e]) + nx) : 0.f;
      if (r0 + i >= S.N) u[e] = 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    sA[wid][lane * E + e] = A[e];
    sC[wid][lane * E + e] = s[e];
    sU[wid][lane * E + e] = u[e];
  }
  if (lane == 0) {
    sDrop[wid] = f.first != 0;
    sDropU[wid] = f.last != 0 || r0 + kWarpRows > S.N;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    s[e] = col ? saved[blockIdx.x * (long long)S.D + c + e] : 0.f;
    u[e] = col ? state[blockIdx.x * (long long)S.D + c + e] : 0.f;
  }
  warp_state<E, false>(sA, sC, sDrop, wid, lane, s);
  warp_state<E, true>(sA, sU, sDropU, wid, lane, u);
  float hp[kWarpRows][E];  // h before each row
#pragma unroll
  for (int i = 0; i < kWarpRows; ++i) {
    const int w = __shfl_sync(0xffffffffu, f.win, i);
    const bool valid = f.valid >> i & 1, first = f.first >> i & 1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float a, q;
      row_coeff<KIND>(to_f32(gp[i].v[e]), &a, &q);
      const float v = to_f32(xp[i].v[e]);
      hp[i][e] = first ? (h0 && col && valid ? h0[(long long)w * S.D + c + e] : 0.f) : s[e];
      s[e] = valid ? fmaf(a, hp[i][e], KIND == ATLB_REC_SIGMOID ? q * v : v) : 0.f;
    }
  }
#pragma unroll
  for (int i = kWarpRows - 1; i >= 0; --i) {
    const int w = __shfl_sync(0xffffffffu, f.win, i);
    const bool valid = f.valid >> i & 1, first = f.first >> i & 1, last = f.last >> i & 1;
    Pack<T, E> og, ox;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float a, q;
      row_coeff<KIND>(to_f32(gp[i].v[e]), &a, &q);
      const float nx = last ? (ghT && col && valid ? ghT[(long long)w * S.D + c + e] : 0.f) : u[e];
      const float g = to_f32(dp[i].v[e]) + nx;
      u[e] = valid && r0 + i < S.N ? a * g : 0.f;
      float dg, dx;
      if (KIND == ATLB_REC_SIGMOID) {
        dg = g * (hp[i][e] - to_f32(xp[i].v[e])) * a * q;
        dx = g * q;
      } else {
        dg = g * hp[i][e];
        dx = g;
      }
      og.v[e] = from_f32<T>(valid ? dg : 0.f);
      ox.v[e] = from_f32<T>(valid ? dx : 0.f);
    }
    if (col && r0 + i < S.N) {
      store_pack(ggate + (r0 + i) * S.D + c, og);
      store_pack(gx + (r0 + i) * S.D + c, ox);
      if (gh0 && first && valid) {
#pragma unroll
        for (int e = 0; e < E; ++e) gh0[(long long)w * S.D + c + e] = u[e];
      }
    }
  }
}

long long chunks_of(long long N) { return (N + kRows - 1) / kRows; }

struct RecWs {
  float *map, *state;
  int* drop;
  size_t bytes;
};

RecWs carve(void* ws, long long N, long long D) {
  Carve c(ws);
  RecWs w;
  const long long k = chunks_of(N);
  w.map = c.take<float>(2 * k * D);
  w.state = c.take<float>(k * D);
  w.drop = c.take<int>(k);
  w.bytes = c.bytes_needed();
  return w;
}

// The state before each window's rows, for windows that have none: copied ahead of the kernels, which overwrite it.
int fill_state(float* dst, const float* src, long long n, cudaStream_t s) {
  if (!dst || n <= 0) return ATLB_OK;
  const cudaError_t e = src ? cudaMemcpyAsync(dst, src, n * sizeof(float), cudaMemcpyDeviceToDevice, s)
                            : cudaMemsetAsync(dst, 0, n * sizeof(float), s);
  return e == cudaSuccess ? ATLB_OK : launch_status("recurrence");
}

template <typename Fn>
int with_kind(int kind, Fn&& fn) {
  if (kind == ATLB_REC_SIGMOID) return fn(std::integral_constant<int, ATLB_REC_SIGMOID>());
  return fn(std::integral_constant<int, ATLB_REC_DECAY>());
}

}  // namespace

size_t recurrence_workspace_bytes(long long N, long long D) { return carve(nullptr, N, D).bytes; }
size_t recurrence_saved_bytes(long long N, long long D) { return (size_t)chunks_of(N) * D * sizeof(float); }

int recurrence_fwd(int dtype, int kind, const void* gate, long long ldg, const void* x, long long ldx,
                   const long long* b, long long N, long long B, long long D, const float* h0, void* h, float* hT,
                   float* saved, void* ws, cudaStream_t s) {
  if (D <= 0) return ATLB_OK;
  if (int st = fill_state(hT, h0, B * D, s)) return st;
  if (N <= 0) return ATLB_OK;
  const RecShape S{N, b ? 0 : N / B, (int)B, (int)D, b};
  const RecWs w = carve(ws, N, D);
  const long long k = chunks_of(N);
  float* state = saved ? saved : w.state;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return with_kind(kind, [&](auto kd) {
      constexpr int KIND = decltype(kd)::value;
      auto go = [&](auto el) {
        constexpr int E = decltype(el)::value;
        const dim3 grid((unsigned)k, (unsigned)((D + 32 * E - 1) / (32 * E)));
        launch(k_rec_map<T, E, KIND, false>, grid, kThreads, 0, s, S, (const T*)gate, ldg, (const T*)x, ldx, h0,
               (const float*)nullptr, k, w.map, w.drop);
        launch(k_rec_chain<false>, (unsigned)((D + kThreads - 1) / kThreads), kThreads, 0, s, w.map, w.drop, k, (int)D,
               state);
        launch(k_rec_fwd<T, E, KIND>, grid, kThreads, 0, s, S, (const T*)gate, ldg, (const T*)x, ldx, h0, state,
               (T*)h, hT);
        return launch_status("recurrence_fwd");
      };
      if constexpr (sizeof(T) == 2) {
        if (D % 2 == 0 && ldg % 2 == 0 && ldx % 2 == 0 && aligned_to(gate, 4) && aligned_to(x, 4) && aligned_to(h, 4))
          return go(std::integral_constant<int, 2>());
      }
      return go(std::integral_constant<int, 1>());
    });
  });
}

int recurrence_bwd(int dtype, int kind, const void* gate, long long ldg, const void* x, long long ldx,
                   const long long* b, long long N, long long B, long long D, const float* h0, const float* saved,
                   const void* gh, long long ldgh, const float* ghT, void* ggate, void* gx, float* gh0, void* ws,
                   cudaStream_t s) {
  if (D <= 0) return ATLB_OK;
  if (int st = fill_state(gh0, ghT, B * D, s)) return st;
  if (N <= 0) return ATLB_OK;
  const RecShape S{N, b ? 0 : N / B, (int)B, (int)D, b};
  const RecWs w = carve(ws, N, D);
  const long long k = chunks_of(N);
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    return with_kind(kind, [&](auto kd) {
      constexpr int KIND = decltype(kd)::value;
      auto go = [&](auto el) {
        constexpr int E = decltype(el)::value;
        const dim3 grid((unsigned)k, (unsigned)((D + 32 * E - 1) / (32 * E)));
        launch(k_rec_map<T, E, KIND, true>, grid, kThreads, 0, s, S, (const T*)gate, ldg, (const T*)gh, ldgh,
               (const float*)nullptr, ghT, k, w.map, w.drop);
        launch(k_rec_chain<true>, (unsigned)((D + kThreads - 1) / kThreads), kThreads, 0, s, w.map, w.drop, k, (int)D,
               w.state);
        launch(k_rec_bwd<T, E, KIND>, grid, kThreads, 0, s, S, (const T*)gate, ldg, (const T*)x, ldx, (const T*)gh,
               ldgh, h0, ghT, saved, w.state, (T*)ggate, (T*)gx, gh0);
        return launch_status("recurrence_bwd");
      };
      if constexpr (sizeof(T) == 2) {
        if (D % 2 == 0 && ldg % 2 == 0 && ldx % 2 == 0 && ldgh % 2 == 0 && aligned_to(gate, 4) && aligned_to(x, 4) &&
            aligned_to(gh, 4) && aligned_to(ggate, 4) && aligned_to(gx, 4))
          return go(std::integral_constant<int, 2>());
      }
      return go(std::integral_constant<int, 1>());
    });
  });
}

}  // namespace atlb
