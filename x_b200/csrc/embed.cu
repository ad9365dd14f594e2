// Row lookup of a table and its gradient (include/atl_b200.h, atlb_embedding_*).
//
//   out[n, :] = scale * W[i_n, :]                      zero where i_n lies outside [0, V)
//   dW[v, :]  = scale * sum over n with i_n = v of g[n, :]
//
// The gradient sorts the row numbers first (stable, so equal rows keep the order of their events) and sums each run of
// equal rows in an order that N, V, D and the row numbers fix, without atomics: the same result every time.  fp32 inside
// a chunk of the sorted events; runs that cross a chunk's border leave partial sums, which a second kernel joins in 64
// bits.
#include "vec.cuh"

namespace atlb {
namespace {

constexpr int kThreads = 256;

// ------------------------------------------------------------------------------------------------ forward
// A group of `lanes` threads (up to 32) takes kRowsEach rows, E neighbouring columns per thread: the rows' numbers, then
// all their loads, then the stores.  Groups need not divide a warp: rows of 96 fp16 columns take 12 threads.  1M rows of
// 64 bf16 columns from 307200: 41 us (175 MB, 4.3 TB/s); 4M of 96 fp16 columns from 33 rows: 170 us (800 MB, 4.7 TB/s).
// 63 and 79 % of the issue slots, 34 and 53 % of DRAM's peak: instructions bound it rather than bytes.  (bf16 spills one
// pair of registers under the cap of 6 CTAs.)
constexpr int kRowsEach = 3;  // four (5 CTAs per SM) take 45 us where three take 42, eight (4 CTAs) 80

template <typename T, int E>
__global__ void __launch_bounds__(kThreads, 6) k_embed_fwd(const T* __restrict__ W, int ldw, int V, int D,
                                                           const long long* __restrict__ idx, int N, float scale,
                                                           int lanes, T* __restrict__ out) {
  const int per = kThreads / lanes, mine = threadIdx.x / lanes, c = (blockIdx.y * lanes + threadIdx.x % lanes) * E;
  if (mine >= per || c >= D) return;
  const unsigned n = blockIdx.x * (unsigned)(per * kRowsEach) + mine;
  int v[kRowsEach];  // -1: no row
#pragma unroll
  for (int k = 0; k < kRowsEach; ++k) {
    const long long i = n + k * per < N ? __ldg(idx + n + k * per) : -1;
    v[k] = i >= 0 && i < V ? (int)i : -1;
  }
  Pack<T, E> r[kRowsEach];
#pragma unroll
  for (int k = 0; k < kRowsEach; ++k) {
    if (v[k] >= 0) {
      r[k] = load_pack<T, E>(W + (long long)v[k] * ldw + c);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) r[k].v[e] = from_f32<T>(0.f);
    }
  }
#pragma unroll
  for (int k = 0; k < kRowsEach; ++k) {
    if (n + k * per >= N) break;
    if (v[k] >= 0) {  // a row outside the table stays zero whatever the scale
#pragma unroll
      for (int e = 0; e < E; ++e) r[k].v[e] = from_f32<T>(to_f32(r[k].v[e]) * scale);
    }
    store_pack(out + (long long)(n + k * per) * D + c, r[k]);
  }
}

// ------------------------------------------------------------------------------------------------ sort
// Least-significant-digit radix sort of (row, event) pairs, up to kMaxBits per pass.  A tile is 512 * ITEMS
// neighbouring pairs; every pass counts the tiles' digits, scans the counts and places the pairs.  Tiles of 4096 pairs
// spread the work per digit (a place per warp and digit to clear and to sum) over more pairs: lookup and gradient of 1M
// events 152 us on the device against 160 with 2048.  Below 64 tiles of that size the GPU would idle, and tiles of 2048 are taken.
// 1M pairs take 20 us a placement, bound by the latency of its steps (28 % of issue slots, 5 % of DRAM).
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxBits = 10;
constexpr int kMaxBins = 1 << kMaxBits;

struct Pair {
  unsigned row, event;
};

// Row numbers outside the table sort behind the last row.
__device__ __forceinline__ unsigned row_key(long long v, unsigned V) {
  return v >= 0 && v < (long long)V ? (unsigned)v : V;
}

template <bool FIRST>
__device__ __forceinline__ Pair sort_pair(const void* src, long long i, unsigned V) {
  if (FIRST) return Pair{row_key(__ldg(static_cast<const long long*>(src) + i), V), (unsigned)i};
  const uint2 q = __ldg(static_cast<const uint2*>(src) + i);
  return Pair{q.x, q.y};
}

// Zeros, by all threads of the CTAs that call it.
__device__ __forceinline__ void write_zeros(char* dst, long long bytes) {
  const long long vecs = bytes / 16, step = (long long)gridDim.x * kSortThreads;
  const long long i0 = blockIdx.x * (long long)kSortThreads + threadIdx.x;
  if (reinterpret_cast<uintptr_t>(dst) % 16 == 0) {
    for (long long i = i0; i < vecs; i += step) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0, 0, 0, 0);
    if (i0 < bytes % 16) dst[vecs * 16 + i0] = 0;
  } else {
    for (long long i = i0; i < bytes / 2; i += step) reinterpret_cast<unsigned short*>(dst)[i] = 0;
  }
}

template <bool FIRST, int ITEMS>
__global__ void __launch_bounds__(kSortThreads) k_sort_count(const void* __restrict__ src, long long N, unsigned V,
                                                             int shift, int bins, int tiles,
                                                             unsigned* __restrict__ counts, char* __restrict__ grad,
                                                             long long grad_bytes) {
  __shared__ unsigned hist[kMaxBins];
  // on the way, and in CTAs of their own behind the tiles: the gradient starts as zeros (rows that no pair names)
  if (FIRST) write_zeros(grad, grad_bytes);
  if (blockIdx.x >= tiles) return;
  for (int d = threadIdx.x; d < bins; d += kSortThreads) hist[d] = 0;
  __syncthreads();
  const long long base = blockIdx.x * (long long)(kSortThreads * ITEMS);
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const long long i = base + r * kSortThreads + threadIdx.x;
    if (i < N) atomicAdd(&hist[(sort_pair<FIRST>(src, i, V).row >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) counts[(long long)blockIdx.x * bins + d] = hist[d];
}

// Exclusive sum over the CTA's THREADS threads; returns this thread's, *total the whole.
template <int THREADS>
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
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < wid) before += sm[w];
    all += sm[w];
  }
  __syncthreads();
  *total = all;
  return before + inc - v;
}

// Up to this many tiles, each CTA of the placement sums the counts before its own itself: a launch less per pass (100k
// events, lookup and gradient: 114 us against 121).
constexpr int kFewTiles = 64;

// A CTA per 8 digits: their counts over the tiles become offsets within the digit.  A thread sums a run of tiles, the
// 128 runs of a digit are joined, and the thread walks its run again.
constexpr int kScanDigits = 8, kScanRuns = 128;
__global__ void __launch_bounds__(kScanDigits * kScanRuns) k_sort_scan(unsigned* __restrict__ counts, int bins, int tiles,
                                                                       unsigned* __restrict__ totals) {
  __shared__ unsigned sm[kScanDigits][kScanRuns + 1];
  const int x = threadIdx.x % kScanDigits, y = threadIdx.x / kScanDigits, d = blockIdx.x * kScanDigits + x;
  const int run = (tiles + kScanRuns - 1) / kScanRuns, t0 = y * run, t1 = min(t0 + run, tiles);
  unsigned sum = 0;
  if (d < bins) {
#pragma unroll 8
    for (int t = t0; t < t1; ++t) sum += counts[(long long)t * bins + d];
  }
  sm[x][y] = sum;
  __syncthreads();
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  if (wid < kScanDigits) {  // a warp per digit, four runs a lane
    unsigned v[4], inc = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) inc += v[k] = sm[wid][lane * 4 + k];
    const unsigned own = inc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    unsigned at = inc - own;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sm[wid][lane * 4 + k] = at;
      at += v[k];
    }
    if (lane == 31 && blockIdx.x * kScanDigits + wid < bins) totals[blockIdx.x * kScanDigits + wid] = inc;
  }
  __syncthreads();
  if (d >= bins) return;
  unsigned at = sm[x][y];
#pragma unroll 8
  for (int t = t0; t < t1; ++t) {
    const unsigned c = counts[(long long)t * bins + d];
    counts[(long long)t * bins + d] = at;
    at += c;
  }
}

// The order of one tile by a digit, stable.  A warp ranks 32 neighbouring pairs at a time among equal digits (match), on
// top of the counts of the rounds and warps before it; the pairs then stand in order in shared memory.
template <int ITEMS>
struct TileSort {
  static constexpr int kTile = kSortThreads * ITEMS;
  union {
    unsigned short hist[kSortWarps][kMaxBins];
    uint2 pair[kTile];  // in order, once the counts are not needed any more
  };
  unsigned local[kMaxBins];  // where each digit's pairs begin
  unsigned sm[kSortWarps];

  // Pair r of a thread is the tile's number wid * 32 * ITEMS + r * 32 + lane; the first n of the tile's exist.  Ends with
  // a barrier.
  __device__ __forceinline__ void order(const Pair (&p)[ITEMS], int n, int shift, int bins) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, first = wid * (32 * ITEMS) + lane;
    for (int d = lane; d < bins; d += 32) hist[wid][d] = 0;
    __syncwarp();
    unsigned at[ITEMS];  // rank among the warp's pairs of the digit, then the place in the tile
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const bool in = first + r * 32 < n;
      const unsigned d = in ? (p[r].row >> shift) & (bins - 1) : 0xffffffffu;
      const unsigned peers = __match_any_sync(0xffffffffu, d);
      const unsigned before = in ? hist[wid][d] : 0;
      __syncwarp();
      at[r] = before + __popc(peers & ((1u << lane) - 1));
      if (in && lane == __ffs(peers) - 1) hist[wid][d] = (unsigned short)(before + __popc(peers));
      __syncwarp();
    }
    __syncthreads();
    unsigned carry = 0;
    for (int d0 = 0; d0 < bins; d0 += kSortThreads) {
      const int d = d0 + threadIdx.x;
      unsigned c = 0, total;
      if (d < bins) {
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) {
          const unsigned h = hist[w][d];
          hist[w][d] = (unsigned short)c;
          c += h;
        }
      }
      const unsigned ex = block_scan<kSortThreads>(c, sm, &total);
      if (d < bins) local[d] = carry + ex;
      carry += total;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      if (first + r * 32 < n) {
        const unsigned d = (p[r].row >> shift) & (bins - 1);
        at[r] += local[d] + hist[wid][d];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
      if (first + r * 32 < n) pair[at[r]] = make_uint2(p[r].row, p[r].event);
    __syncthreads();
  }
};

// Placement of the tiles' pairs.  They leave in the tile's order, so that pairs of one digit leave side by side (4M pairs
// of 33 rows 34 us, scattered one by one 37).
template <bool FIRST, int ITEMS>
__global__ void __launch_bounds__(kSortThreads) k_sort_place(const void* __restrict__ src, long long N, unsigned V,
                                                             int shift, int bins, int tiles,
                                                             const unsigned* __restrict__ counts,
                                                             const unsigned* __restrict__ totals,
                                                             uint2* __restrict__ out) {
  using Tile = TileSort<ITEMS>;
  __shared__ Tile ts;
  __shared__ unsigned start[kMaxBins];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const long long tile0 = blockIdx.x * (long long)Tile::kTile;
  const int n = N - tile0 < Tile::kTile ? (int)(N - tile0) : Tile::kTile;
  Pair p[ITEMS];
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = wid * (32 * ITEMS) + r * 32 + lane;
    if (i < n) p[r] = sort_pair<FIRST>(src, tile0 + i, V);
  }
  unsigned carry = 0;
  for (int d0 = 0; d0 < bins; d0 += kSortThreads) {
    const int d = d0 + threadIdx.x;
    unsigned all = 0, before = 0, total;  // pairs of the digit, in all tiles and in those before this one
    if (d < bins) {
      if (tiles > kFewTiles) {
        all = totals[d];
        before = counts[(long long)blockIdx.x * bins + d];
      } else {
#pragma unroll 8
        for (int t = 0; t < tiles; ++t) {
          const unsigned c = counts[(long long)t * bins + d];
          all += c;
          before += t < blockIdx.x ? c : 0;
        }
      }
    }
    const unsigned ex = block_scan<kSortThreads>(all, ts.sm, &total);
    if (d < bins) start[d] = carry + ex + before;
    carry += total;
  }
  ts.order(p, n, shift, bins);
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = r * kSortThreads + threadIdx.x;
    if (i < n) {
      const uint2 q = ts.pair[i];
      const unsigned d = (q.x >> shift) & (bins - 1);
      out[start[d] - ts.local[d] + i] = q;
    }
  }
}

// One tile: all passes in one CTA, the pairs in shared memory between them; the CTAs behind it write zeros.
constexpr int kSmallItems = 8;
__global__ void __launch_bounds__(kSortThreads) k_sort_small(const long long* __restrict__ idx, int n, unsigned V, int passes,
                                                             int bits, uint2* __restrict__ out, char* __restrict__ grad,
                                                             long long grad_bytes) {
  __shared__ TileSort<kSmallItems> ts;
  write_zeros(grad, grad_bytes);
  if (blockIdx.x > 0) return;
  const int first = (threadIdx.x >> 5) * (32 * kSmallItems) + (threadIdx.x & 31);
  Pair p[kSmallItems];
#pragma unroll
  for (int r = 0; r < kSmallItems; ++r)
    if (first + r * 32 < n) p[r] = sort_pair<true>(idx, first + r * 32, V);
  for (int k = 0; k < passes; ++k) {
    if (k > 0) {
#pragma unroll
      for (int r = 0; r < kSmallItems; ++r)
        if (first + r * 32 < n) p[r] = Pair{ts.pair[first + r * 32].x, ts.pair[first + r * 32].y};
      __syncthreads();
    }
    ts.order(p, n, k * bits, 1 << bits);
  }
  for (int i = threadIdx.x; i < n; i += kSortThreads) out[i] = ts.pair[i];
}

struct SortPlan {
  int passes, bits, tiles;
  bool large;  // tiles of 4096 pairs, else 2048
};

SortPlan sort_plan(long long N, long long V) {
  int need = 1;  // the keys 0 .. V
  while ((V >> need) != 0) ++need;
  SortPlan s;
  s.passes = (need + kMaxBits - 1) / kMaxBits;
  s.bits = (need + s.passes - 1) / s.passes;
  s.large = N > 64 * 4096;
  const int tile = s.large ? 4096 : 2048;
  s.tiles = (int)((N + tile - 1) / tile);
  return s;
}

// ------------------------------------------------------------------------------------------------ sums
// A group of `lanes` threads walks the L sorted pairs of one chunk, keeping E columns per thread in fp32, and
// writes a gradient row when its run ends inside the chunk.  A run that came in from the chunk before leaves its
// sum in part[chunk][0], one that goes on into the next chunk in part[chunk][1] (in [0] if it does both).  Bound by its
// scattered row reads: 1M rows of 64 bf16 columns 42 us (149 MB of DRAM traffic, 3.5 TB/s), 4M of 96 fp16 columns 161 us
// (995 MB, 6.2 TB/s; rows of 192 bytes fetch parts of lines that others need later).  The order of a chunk's sum: fours of
// neighbouring events that share their row, (a + b) + (c + d), one event at a time where a four holds a border.
constexpr int kAhead = 4;  // rows in flight per thread, at 3 CTAs per SM: 4 CTAs with spilled registers took 47 us

template <typename T, int E>
__global__ void __launch_bounds__(kThreads, 3) k_embed_sum(const T* __restrict__ g, int ldg,
                                                           const uint2* __restrict__ pair, int N, unsigned V, int D,
                                                           int L, int lanes, float scale, T* __restrict__ grad,
                                                           float* __restrict__ part) {
  const int per = kThreads / lanes, mine = threadIdx.x / lanes, c = (blockIdx.y * lanes + threadIdx.x % lanes) * E;
  const unsigned chunk = blockIdx.x * (unsigned)per + mine;
  if (mine >= per || (long long)chunk * L >= N || c >= D) return;
  const int j0 = chunk * L, j1 = min(N - j0, L) + j0;
  const unsigned prev = j0 > 0 ? pair[j0 - 1].x : 0xffffffffu;
  unsigned cur = pair[j0].x;
  bool head = cur == prev;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  auto put = [&](bool to_part, int slot) {
    if (to_part) {
      float* p = part + ((long long)chunk * 2 + slot) * D + c;
#pragma unroll
      for (int e = 0; e < E; ++e) p[e] = acc[e];
    } else {
      Pack<T, E> r;
#pragma unroll
      for (int e = 0; e < E; ++e) r.v[e] = from_f32<T>(acc[e] * scale);
      store_pack(grad + (long long)cur * D + c, r);
    }
  };
  uint2 next[kAhead];  // the pairs of the next rows, on the way while these rows are summed
#pragma unroll
  for (int q = 0; q < kAhead; ++q) next[q] = j0 + q < j1 ? __ldg(pair + j0 + q) : make_uint2(V, 0);
#pragma unroll 1
  for (int j = j0; j < j1 && cur < V; j += kAhead) {
    unsigned row[kAhead];
    Pack<T, E> r[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      row[q] = next[q].x;
      if (row[q] < V) {
        r[q] = load_pack<T, E>(g + (long long)next[q].y * ldg + c);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) r[q].v[e] = from_f32<T>(0.f);
      }
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int m = j + kAhead + q;
      next[q] = m < j1 ? __ldg(pair + m) : make_uint2(V, 0);
    }
    // all of the run, as most are where runs are long: summed among themselves first (the pairs are sorted, so the last
    // row tells), a quarter of the roundings on the way
    static_assert(kAhead == 4, "four rows at a time");
    if (row[0] == cur && row[3] == cur) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        acc[e] += (to_f32(r[0].v[e]) + to_f32(r[1].v[e])) + (to_f32(r[2].v[e]) + to_f32(r[3].v[e]));
      continue;
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (j + q < j1 && row[q] != cur) {
        if (cur < V) put(head, 0);
        cur = row[q];
        head = false;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += to_f32(r[q].v[e]);
    }
  }
  if (cur >= V) return;
  const bool on = j1 < N && pair[j1].x == cur;  // goes on in the next chunk
  put(head || on, head ? 0 : 1);
}

// The chunk in which a run over several chunks begins joins its partial sums.  A CTA looks after 32 chunks: a warp each
// for the runs that go on over fewer than 32 more chunks, in order; then, for a longer one, all its threads, 64 rows of
// them over 16 columns: each takes every 64th partial sum, and these are added in order.  The few sums of sums are taken
// in 64 bits, which keeps long runs at the error of their chunks (1M events, lookup and gradient: 152 us on the device,
// 151 with fp32).
constexpr int kJoinThreads = 1024, kLongCols = 16, kLongRows = kJoinThreads / kLongCols;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) k_embed_join(const uint2* __restrict__ pair, int N, unsigned V, int D,
                                                             int L, unsigned chunks, float scale,
                                                             const float* __restrict__ part, T* __restrict__ grad) {
  __shared__ double sm[kLongRows][kLongCols + 1];
  __shared__ unsigned long_row[32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const unsigned chunk = blockIdx.x * 32 + wid;
  unsigned row = V;  // of a run that begins here and goes on
  if (chunk + 1 < chunks) {
    const int j0 = chunk * L, j1 = j0 + L;
    const unsigned cur = pair[j1 - 1].x, after = pair[j1].x, first = pair[j0].x, before = j0 > 0 ? pair[j0 - 1].x : V;
    if (cur < V && after == cur && !(first == cur && before == cur)) row = cur;
  }
  bool is_long = false;
  if (row < V) {
    // lane i: does the run end before chunk + 2 + i?
    const unsigned next = chunk + 2 + lane;
    const unsigned ends = __ballot_sync(0xffffffffu, next >= chunks || pair[(long long)next * L].x != row);
    is_long = ends == 0;
    if (!is_long && blockIdx.y == 0) {
      const unsigned last = chunk + __ffs(ends);
      for (int c = lane; c < D; c += 32) {
        double acc = part[((long long)chunk * 2 + 1) * D + c];
#pragma unroll 4
        for (unsigned e = chunk + 1; e <= last; ++e) acc += part[(long long)e * 2 * D + c];
        grad[(long long)row * D + c] = from_f32<T>((float)acc * scale);
      }
    }
  }
  if (lane == 0) long_row[wid] = is_long ? row : V;
  __syncthreads();
  const int x = threadIdx.x % kLongCols, y = threadIdx.x / kLongCols;
  for (int w = 0; w < 32; ++w) {  // at most one: a long run leaves the CTA's chunks
    if (long_row[w] >= V) continue;
    const unsigned from = blockIdx.x * 32 + w, r = long_row[w];
    unsigned last = from;
    for (;;) {
      const unsigned e = last + 1 + threadIdx.x;
      const int more = __syncthreads_count(e < chunks && pair[(long long)e * L].x == r);
      last += more;
      if (more < kJoinThreads) break;
    }
    for (int c0 = blockIdx.y * kLongCols; c0 < D; c0 += gridDim.y * kLongCols) {
      const int c = c0 + x;
      double acc = 0.0;
      if (c < D) {
        if (y == 0) acc = part[((long long)from * 2 + 1) * D + c];
#pragma unroll 8
        for (unsigned e = from + 1 + y; e <= last; e += kLongRows) acc += part[(long long)e * 2 * D + c];
      }
      sm[y][x] = acc;
      __syncthreads();
      if (y == 0 && c < D) {
#pragma unroll 8
        for (int k = 1; k < kLongRows; ++k) acc += sm[k][x];
        grad[(long long)r * D + c] = from_f32<T>((float)acc * scale);
      }
      __syncthreads();
    }
  }
}

// Threads on a row of D columns, E each.
int group_lanes(long long D, int E) { return D >= 32LL * E ? 32 : D < 1 ? 1 : (int)((D + E - 1) / E); }

// Pairs per chunk: one wave of groups on the GPU (148 SMs of 3 CTAs, groups of 16-byte threads on 16-bit rows), so that
// all end together.
int sum_chunk(long long N, long long D) {
  const long long wave = 148LL * 3 * (kThreads / group_lanes(D, 8)), L = (N + wave - 1) / wave;
  return (int)(L < 16 ? 16 : L);
}

struct EmbedWs {
  uint2* pair[2];
  unsigned *counts, *totals;
  float* part;
  size_t bytes;
};

EmbedWs carve(void* ws, long long N, long long V, long long D) {
  const SortPlan s = sort_plan(N, V);
  const int L = sum_chunk(N, D);
  Carve c(ws);
  EmbedWs w;
  for (int i = 0; i < 2; ++i) w.pair[i] = c.take<uint2>(s.passes > i ? N : 0);
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
    const int lanes = group_lanes(D, wide ? E : 1);
    const int E1 = wide ? E : 1;
    const long long per = kThreads / lanes * kRowsEach;
    const unsigned slabs = (unsigned)((D + lanes * E1 - 1) / (lanes * E1));
    const dim3 grid((unsigned)((N + per - 1) / per), slabs);
    auto go = [&](auto el) {
      launch(k_embed_fwd<T, decltype(el)::value>, grid, kThreads, 0, s, (const T*)W, (int)ldw, (int)V, (int)D, idx, (int)N,
             (float)scale, lanes, (T*)out);
    };
    if (wide)
      go(std::integral_constant<int, E>());
    else
      go(std::integral_constant<int, 1>());
    return launch_status("embedding_fwd");
  });
}

int embedding_bwd(int dtype, const void* g, long long ldg, const long long* idx, long long N, long long V, long long D,
                  double scale, void* grad, void* ws, cudaStream_t s) {
  if (V <= 0 || D <= 0) return ATLB_OK;
  const size_t grad_bytes = (size_t)V * D * (dtype == ATLB_F32 ? 4 : 2);
  if (N <= 0) return cudaMemsetAsync(grad, 0, grad_bytes, s) == cudaSuccess ? ATLB_OK : launch_status("embedding_bwd");
  const SortPlan p = sort_plan(N, V);
  const EmbedWs w = carve(ws, N, V, D);
  const int bins = 1 << p.bits, L = sum_chunk(N, D);
  const void* src = idx;
  // enough CTAs to write the zeros as well: 64 KB each, up to two per SM
  const int zero = (int)(grad_bytes / 65536 < 296 ? grad_bytes / 65536 : 296);
  const bool small = N <= TileSort<kSmallItems>::kTile;
  if (small) {
    launch(k_sort_small, zero > 1 ? zero : 1, kSortThreads, 0, s, idx, (int)N, (unsigned)V, p.passes, p.bits, w.pair[0],
           (char*)grad, (long long)grad_bytes);
    src = w.pair[0];
  }
  for (int i = 0; !small && i < p.passes; ++i) {
    uint2* dst = w.pair[i & 1];
    auto pass = [&](auto first, auto items) {
      constexpr bool F = decltype(first)::value;
      constexpr int I = decltype(items)::value;
      launch(k_sort_count<F, I>, F && zero > p.tiles ? zero : p.tiles, kSortThreads, 0, s, src, N, (unsigned)V, i * p.bits,
             bins, p.tiles, w.counts, (char*)grad, (long long)grad_bytes);
      if (p.tiles > kFewTiles)
        launch(k_sort_scan, (bins + kScanDigits - 1) / kScanDigits, kScanDigits * kScanRuns, 0, s, w.counts, bins,
               p.tiles, w.totals);
      launch(k_sort_place<F, I>, p.tiles, kSortThreads, 0, s, src, N, (unsigned)V, i * p.bits, bins, p.tiles,
             w.counts, w.totals, dst);
    };
    auto sized = [&](auto first) {
      if (p.large)
        pass(first, std::integral_constant<int, 8>());
      else
        pass(first, std::integral_constant<int, 4>());
    };
    if (i == 0)
      sized(std::true_type());
    else
      sized(std::false_type());
    src = dst;
  }
  const uint2* pair = static_cast<const uint2*>(src);
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    constexpr int E = 16 / sizeof(T);
    const bool wide = D % E == 0 && ldg % E == 0 && aligned_to(g, 16) && aligned_to(grad, 16);
    const int lanes = group_lanes(D, wide ? E : 1), cols = lanes * (wide ? E : 1);
    const long long chunks = (N + L - 1) / L;
    const dim3 grid((unsigned)((chunks + kThreads / lanes - 1) / (kThreads / lanes)), (unsigned)((D + cols - 1) / cols));
    auto go = [&](auto el) {
      launch(k_embed_sum<T, decltype(el)::value>, grid, kThreads, 0, s, (const T*)g, (int)ldg, pair, (int)N, (unsigned)V,
             (int)D, L, lanes, (float)scale, (T*)grad, w.part);
    };
    if (wide)
      go(std::integral_constant<int, E>());
    else
      go(std::integral_constant<int, 1>());
    // where runs are long on average, CTAs share the columns (4M events, 33 rows of 96: 40 us, 90 with one CTA to a run)
    const unsigned share = N / V >= 16LL * L ? (unsigned)(D < 128 ? (D + kLongCols - 1) / kLongCols : 8) : 1;
    if (chunks > 1)
      launch(k_embed_join<T>, dim3((unsigned)((chunks + 31) / 32), share), kJoinThreads, 0, s, pair, (int)N, (unsigned)V,
             (int)D, L, (unsigned)chunks, (float)scale, w.part, (T*)grad);
    return launch_status("embedding_bwd");
  });
}

}  // namespace atlb
