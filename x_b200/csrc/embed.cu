// Row lookup of a table and its gradient (include/atl_b200.h, atlb_embedding_*).
//
//   out[n, :] = scale * W[i_n, :]                      zero where i_n lies outside [0, V)
//   dW[v, :]  = scale * sum over n with i_n = v of g[n, :]
//
// The gradient sorts the row numbers first (stable, so equal rows keep the order of their events) and sums each run
// of equal rows in fp32 in that order: no atomics, the same result every time.  Runs that cross the border of a
// chunk leave partial sums, which a second kernel joins in order.
#include "vec.cuh"

namespace atlb {
namespace {

constexpr int kThreads = 256;

// ------------------------------------------------------------------------------------------------ forward
// A group of `lanes` threads (a power of two up to 32) per row, E neighbouring elements per thread.
template <typename T, int E>
__global__ void __launch_bounds__(kThreads) k_embed_fwd(const T* __restrict__ W, long long ldw, long long V, int D,
                                                        const long long* __restrict__ idx, long long N, float scale,
                                                        int lanes, T* __restrict__ out) {
  const int sub = threadIdx.x & (lanes - 1), per = kThreads / lanes;
  const long long stride = (long long)gridDim.x * per;
  for (long long n = blockIdx.x * (long long)per + threadIdx.x / lanes; n < N; n += stride) {
    const long long v = idx[n];
    const bool ok = v >= 0 && v < V;
    for (int c = sub * E; c < D; c += lanes * E) {
      Pack<T, E> r;
      if (ok) r = load_pack<T, E>(W + v * ldw + c);
#pragma unroll
      for (int e = 0; e < E; ++e) r.v[e] = from_f32<T>(ok ? to_f32(r.v[e]) * scale : 0.f);
      store_pack(out + n * D + c, r);
    }
  }
}

// ------------------------------------------------------------------------------------------------ sort
// Least-significant-digit radix sort of (row, event) pairs, up to kMaxBits per pass.  A tile is kTileItems
// neighbouring pairs; every pass counts the tile's digits, scans the counts (digit-major) and places the pairs.
constexpr int kItems = 8;
constexpr int kTileItems = kThreads * kItems;
constexpr int kMaxBits = 10;
constexpr int kMaxBins = 1 << kMaxBits;

// Row numbers outside the table sort behind the last row.
__device__ __forceinline__ unsigned row_key(long long v, unsigned V) {
  return v >= 0 && v < (long long)V ? (unsigned)v : V;
}

template <bool FIRST>
__device__ __forceinline__ unsigned sort_key(const void* src, long long i, unsigned V) {
  return FIRST ? row_key(static_cast<const long long*>(src)[i], V) : static_cast<const unsigned*>(src)[i];
}

template <bool FIRST>
__global__ void __launch_bounds__(kThreads) k_sort_count(const void* __restrict__ src, long long N, unsigned V,
                                                         int shift, int bins, int tiles, unsigned* __restrict__ counts) {
  __shared__ unsigned hist[kMaxBins];
  for (int d = threadIdx.x; d < bins; d += kThreads) hist[d] = 0;
  __syncthreads();
  const long long base = blockIdx.x * (long long)kTileItems;
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const long long i = base + r * kThreads + threadIdx.x;
    if (i < N) atomicAdd(&hist[(sort_key<FIRST>(src, i, V) >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kThreads) counts[(long long)d * tiles + blockIdx.x] = hist[d];
}

// Exclusive sum over 256 threads; returns this thread's, *total the whole.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* sm, unsigned* total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  unsigned inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) sm[wid] = inc;
  __syncthreads();
  unsigned before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < wid) before += sm[w];
    all += sm[w];
  }
  __syncthreads();
  *total = all;
  return before + inc - v;
}

// One CTA per digit: its counts over the tiles become offsets within the digit.
__global__ void __launch_bounds__(kThreads) k_sort_scan(unsigned* __restrict__ counts, int tiles,
                                                        unsigned* __restrict__ totals) {
  __shared__ unsigned sm[kThreads / 32];
  unsigned* row = counts + (long long)blockIdx.x * tiles;
  unsigned carry = 0;
  for (int t0 = 0; t0 < tiles; t0 += kThreads) {
    const int t = t0 + threadIdx.x;
    const unsigned v = t < tiles ? row[t] : 0;
    unsigned total;
    const unsigned ex = block_scan(v, sm, &total);
    if (t < tiles) row[t] = carry + ex;
    carry += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Stable placement: a warp ranks 32 neighbouring pairs at a time among equal digits (match), on top of the counts
// of the rounds and warps before it.
template <bool FIRST>
__global__ void __launch_bounds__(kThreads) k_sort_place(const void* __restrict__ src, const unsigned* __restrict__ pos,
                                                         long long N, unsigned V, int shift, int bins, int tiles,
                                                         const unsigned* __restrict__ counts,
                                                         const unsigned* __restrict__ totals,
                                                         unsigned* __restrict__ key_out, unsigned* __restrict__ pos_out) {
  constexpr int W = kThreads / 32;
  __shared__ unsigned short hist[W][kMaxBins];
  __shared__ unsigned start[kMaxBins];
  __shared__ unsigned sm[W];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  for (int d = threadIdx.x; d < bins; d += kThreads)
#pragma unroll
    for (int w = 0; w < W; ++w) hist[w][d] = 0;
  unsigned carry = 0;
  for (int d0 = 0; d0 < bins; d0 += kThreads) {
    const int d = d0 + threadIdx.x;
    unsigned total;
    const unsigned ex = block_scan(d < bins ? totals[d] : 0, sm, &total);
    if (d < bins) start[d] = carry + ex + counts[(long long)d * tiles + blockIdx.x];
    carry += total;
  }
  __syncthreads();
  const long long base = blockIdx.x * (long long)kTileItems + wid * (32 * kItems) + lane;
  unsigned key[kItems], rank[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const long long i = base + r * 32;
    const bool in = i < N;
    key[r] = in ? sort_key<FIRST>(src, i, V) : 0xffffffffu;
    const unsigned d = (key[r] >> shift) & (bins - 1);
    const unsigned peers = __match_any_sync(0xffffffffu, in ? d : 0xffffffffu);
    unsigned before = 0;
    if (in) before = hist[wid][d];
    __syncwarp();
    rank[r] = before + __popc(peers & ((1u << lane) - 1));
    if (in && lane == __ffs(peers) - 1) hist[wid][d] = (unsigned short)(before + __popc(peers));
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kThreads) {
    unsigned c = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const unsigned h = hist[w][d];
      hist[w][d] = (unsigned short)c;
      c += h;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const long long i = base + r * 32;
    if (i < N) {
      const unsigned d = (key[r] >> shift) & (bins - 1);
      const unsigned at = start[d] + hist[wid][d] + rank[r];
      key_out[at] = key[r];
      pos_out[at] = FIRST ? (unsigned)i : pos[i];
    }
  }
}

struct SortPlan {
  int passes, bits, tiles;
};

SortPlan sort_plan(long long N, long long V) {
  int need = 1;  // the keys 0 .. V
  while ((V >> need) != 0) ++need;
  SortPlan s;
  s.passes = (need + kMaxBits - 1) / kMaxBits;
  s.bits = (need + s.passes - 1) / s.passes;
  s.tiles = (int)((N + kTileItems - 1) / kTileItems);
  return s;
}

// ------------------------------------------------------------------------------------------------ sums
// A group of `lanes` threads walks the L sorted pairs of one chunk, keeping E columns per thread in fp32, and
// writes a gradient row when its run ends inside the chunk.  A run that came in from the chunk before leaves its
// sum in part[chunk][0], one that goes on into the next chunk in part[chunk][1] (in [0] if it does both).
constexpr int kAhead = 4;  // rows in flight per thread

template <typename T, int E>
__global__ void __launch_bounds__(kThreads) k_embed_sum(const T* __restrict__ g, long long ldg,
                                                        const unsigned* __restrict__ key,
                                                        const unsigned* __restrict__ pos, long long N, unsigned V,
                                                        int D, int L, int lanes, float scale, T* __restrict__ grad,
                                                        float* __restrict__ part) {
  const int sub = threadIdx.x & (lanes - 1), per = kThreads / lanes;
  const long long chunk = blockIdx.x * (long long)per + threadIdx.x / lanes;
  const int c = (blockIdx.y * lanes + sub) * E;
  const long long j0 = chunk * L, j1 = j0 + L < N ? j0 + L : N;
  if (j0 >= N || c >= D) return;
  const unsigned prev = j0 > 0 ? key[j0 - 1] : 0xffffffffu, next = j1 < N ? key[j1] : 0xffffffffu;
  unsigned cur = key[j0];
  bool head = cur == prev;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  auto to_part = [&](int slot) {
    float* p = part + (chunk * 2 + slot) * D + c;
#pragma unroll
    for (int e = 0; e < E; ++e) p[e] = acc[e];
  };
  auto to_grad = [&]() {
    Pack<T, E> r;
#pragma unroll
    for (int e = 0; e < E; ++e) r.v[e] = from_f32<T>(acc[e] * scale);
    store_pack(grad + (long long)cur * D + c, r);
  };
  for (long long j = j0; j < j1 && cur < V; j += kAhead) {
    unsigned k[kAhead];
    Pack<T, E> r[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      k[q] = j + q < j1 ? key[j + q] : V;
      if (k[q] < V) r[q] = load_pack<T, E>(g + (long long)pos[j + q] * ldg + c);
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (j + q >= j1) break;
      if (k[q] != cur) {
        if (cur < V) {
          if (head) to_part(0);
          else to_grad();
        }
        cur = k[q];
        head = false;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
      }
      if (k[q] < V) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += to_f32(r[q].v[e]);
      }
    }
  }
  if (cur >= V) return;
  if (head) to_part(0);
  else if (cur == next) to_part(1);
  else to_grad();
}

// The chunk in which a run over several chunks begins joins its partial sums, in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_embed_join(const unsigned* __restrict__ key, long long N, unsigned V,
                                                         int D, int L, float scale, const float* __restrict__ part,
                                                         T* __restrict__ grad) {
  const long long chunk = blockIdx.x;
  const long long j0 = chunk * L, j1 = j0 + L;
  if (j1 >= N) return;
  const unsigned cur = key[j1 - 1];
  if (cur >= V || key[j1] != cur) return;
  if (j0 > 0 && key[j0] == cur && key[j0 - 1] == cur) return;  // it began further left
  for (int c = threadIdx.x; c < D; c += kThreads) {
    float acc = part[(chunk * 2 + 1) * D + c];
    for (long long e = chunk + 1; e * L < N && key[e * L] == cur; ++e) acc += part[e * 2 * D + c];
    grad[(long long)cur * D + c] = from_f32<T>(acc * scale);
  }
}

int sum_chunk(long long N) {
  int L = 32;
  while (L < (1 << 20) && N / L > 8192) L *= 2;
  return L;
}

int group_lanes(int D, int E) {
  int l = 1;
  while (l < 32 && l * E < D) l *= 2;
  return l;
}

struct EmbedWs {
  unsigned *key[2], *pos[2], *counts, *totals;
  float* part;
  size_t bytes;
};

EmbedWs carve(void* ws, long long N, long long V, long long D) {
  const SortPlan s = sort_plan(N, V);
  const int L = sum_chunk(N);
  Carve c(ws);
  EmbedWs w;
  for (int i = 0; i < 2; ++i) {
    w.key[i] = c.take<unsigned>(N);
    w.pos[i] = c.take<unsigned>(N);
  }
  w.counts = c.take<unsigned>(((long long)s.tiles) << s.bits);
  w.totals = c.take<unsigned>(1LL << s.bits);
  w.part = c.take<float>((N + L - 1) / L * 2 * D);
  w.bytes = c.bytes_needed();
  return w;
}

}  // namespace

size_t embedding_workspace_bytes(long long N, long long V, long long D) { return carve(nullptr, N, V, D).bytes; }

int embedding_fwd(int dtype, const void* W, long long ldw, long long V, long long D, const long long* idx, long long N,
                  double scale, void* out, cudaStream_t s) {
  if (N <= 0 || D <= 0) return ATLB_OK;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    constexpr int E = 16 / sizeof(T);
    const bool wide = D % E == 0 && ldw % E == 0 && aligned_to(W, 16) && aligned_to(out, 16);
    const int lanes = group_lanes((int)D, wide ? E : 1);
    const int grid = clamp_grid((N + kThreads / lanes - 1) / (kThreads / lanes));
    if (wide)
      launch(k_embed_fwd<T, E>, grid, kThreads, 0, s, (const T*)W, ldw, V, (int)D, idx, N, (float)scale, lanes, (T*)out);
    else
      launch(k_embed_fwd<T, 1>, grid, kThreads, 0, s, (const T*)W, ldw, V, (int)D, idx, N, (float)scale, lanes, (T*)out);
    return launch_status("embedding_fwd");
  });
}

int embedding_bwd(int dtype, const void* g, long long ldg, const long long* idx, long long N, long long V, long long D,
                  double scale, void* grad, void* ws, cudaStream_t s) {
  if (V <= 0 || D <= 0) return ATLB_OK;
  const size_t esize = dtype == ATLB_F32 ? 4 : 2;
  if (cudaMemsetAsync(grad, 0, (size_t)V * D * esize, s) != cudaSuccess) return launch_status("embedding_bwd");
  if (N <= 0) return ATLB_OK;
  const SortPlan p = sort_plan(N, V);
  const EmbedWs w = carve(ws, N, V, D);
  const int bins = 1 << p.bits, L = sum_chunk(N);
  int at = 0;
  for (int i = 0; i < p.passes; ++i) {
    const int shift = i * p.bits;
    if (i == 0) {
      launch(k_sort_count<true>, p.tiles, kThreads, 0, s, (const void*)idx, N, (unsigned)V, shift, bins, p.tiles, w.counts);
      launch(k_sort_scan, bins, kThreads, 0, s, w.counts, p.tiles, w.totals);
      launch(k_sort_place<true>, p.tiles, kThreads, 0, s, (const void*)idx, (const unsigned*)nullptr, N, (unsigned)V, shift,
             bins, p.tiles, w.counts, w.totals, w.key[0], w.pos[0]);
    } else {
      launch(k_sort_count<false>, p.tiles, kThreads, 0, s, (const void*)w.key[at], N, (unsigned)V, shift, bins, p.tiles, w.counts);
      launch(k_sort_scan, bins, kThreads, 0, s, w.counts, p.tiles, w.totals);
      launch(k_sort_place<false>, p.tiles, kThreads, 0, s, (const void*)w.key[at], (const unsigned*)w.pos[at], N,
             (unsigned)V, shift, bins, p.tiles, w.counts, w.totals, w.key[at ^ 1], w.pos[at ^ 1]);
      at ^= 1;
    }
  }
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    constexpr int E = 16 / sizeof(T);
    const bool wide = D % E == 0 && ldg % E == 0 && aligned_to(g, 16) && aligned_to(grad, 16);
    const int lanes = group_lanes((int)D, wide ? E : 1), cols = lanes * (wide ? E : 1);
    const long long chunks = (N + L - 1) / L;
    const dim3 grid((unsigned)((chunks + kThreads / lanes - 1) / (kThreads / lanes)), (unsigned)((D + cols - 1) / cols));
    if (wide)
      launch(k_embed_sum<T, E>, grid, kThreads, 0, s, (const T*)g, ldg, w.key[at], w.pos[at], N, (unsigned)V, (int)D, L,
             lanes, (float)scale, (T*)grad, w.part);
    else
      launch(k_embed_sum<T, 1>, grid, kThreads, 0, s, (const T*)g, ldg, w.key[at], w.pos[at], N, (unsigned)V, (int)D, L,
             lanes, (float)scale, (T*)grad, w.part);
    launch(k_embed_join<T>, dim3((unsigned)chunks), kThreads, 0, s, w.key[at], N, (unsigned)V, (int)D, L, (float)scale,
           w.part, (T*)grad);
    return launch_status("embedding_bwd");
  });
}

}  // namespace atlb
