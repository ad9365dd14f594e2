// Dropout from a counter-based generator (include/atl_b200.h, atlb_dropout).
//
//   out_i = keep_i ? x_i / (1 - p) : 0, plus residual_i when there is one;
//   keep_i = word i % 4 of Philox4x32-10 at counter (i / 4, 2^31 | (i / 4) >> 32, call) >= floor(p 2^32 + 1/2)
//
// The mask is a function of (seed, call, i) alone, so it is never stored: the backward pass is this same kernel on
// the incoming gradient.  Bit 31 of the second counter word keeps the draws apart from the noise of rng.cuh.
// A dropped element is selected to zero, not multiplied, so an infinity or NaN there leaves no trace.
#include "rng.cuh"
#include "vec.cuh"

namespace atlb {
namespace {

constexpr int kThreads = 256;

struct Drop {
  unsigned key[20];             // the ten rounds' keys, so that a round takes them from constant memory
  unsigned long long call;
  const long long* call_dev;    // added to call when not null: a graph replay can draw anew
  unsigned threshold;           // keep when the word is at least this
  float scale;
};

// The four words of counter (q, hi): Philox4x32-10 (rng.cuh) with the keys laid out ahead.  The second word and the
// call are the same for all of a CTA, so two of the first two rounds' four products are taken once (start).
struct Start {
  unsigned y, w, hi1, lo1, x2hi, x2lo, c2x;
};
__device__ __forceinline__ Start drop_start(const Drop& D, unsigned long long call, unsigned hi) {
  Start s;
  s.y = hi | 0x80000000u;
  s.w = (unsigned)(call >> 32);
  mulhilo32(kPhiloxM1, (unsigned)call, &s.hi1, &s.lo1);
  s.c2x = s.hi1 ^ s.y ^ D.key[0];
  mulhilo32(kPhiloxM0, s.c2x, &s.x2hi, &s.x2lo);
  return s;
}
__device__ __forceinline__ void drop_words(const Drop& D, const Start& s, unsigned q, unsigned (&w)[4]) {
  unsigned hi0, lo0, hi1, lo1;
  mulhilo32(kPhiloxM0, q, &hi0, &lo0);
  mulhilo32(kPhiloxM1, hi0 ^ s.w ^ D.key[1], &hi1, &lo1);
  Philox4 c{hi1 ^ s.lo1 ^ D.key[2], lo1, s.x2hi ^ lo0 ^ D.key[3], s.x2lo};
#pragma unroll
  for (int r = 2; r < 10; ++r) c = philox_round(c, D.key[2 * r], D.key[2 * r + 1]);
  w[0] = c.x, w[1] = c.y, w[2] = c.z, w[3] = c.w;
}

__device__ __forceinline__ float drop_one(const Drop& D, unsigned word, float x) {
  return word >= D.threshold ? x * D.scale : 0.f;
}

// A vector of 16 bytes is one Philox call of fp32 or two of 16-bit elements.  VECS vectors per thread, their loads
// issued together; with four, the part of the words that a CTA shares is spread over the most calls.  fp32 runs at the
// copy rate (2M x 48 with a residual, forward and backward: 285 us, 1.92 GB).  64M bf16 elements take 57 us a pass, 256 MB,
// 70 % of the copy rate (two vectors 59, one 60; high and low halves as two products: the same): the words' 32 x 32-bit
// products hold the issue port for about four cycles each, 31 us, the bytes take 40, and at 57 % of the warps the two
// overlap in part only.  Element by element, where a pointer is not on a 16-byte boundary, a pass takes 95 us.
template <typename T, bool RES, int VECS>
__global__ void __launch_bounds__(kThreads) k_dropout_vec(Drop D, const T* __restrict__ x, const T* __restrict__ res,
                                                          long long n, T* __restrict__ out) {
  constexpr int E = 16 / sizeof(T);
  const unsigned long long call = D.call + (D.call_dev ? (unsigned long long)*D.call_dev : 0ull);
  const long long vecs = n / E, base = blockIdx.x * (long long)(kThreads * VECS), v0 = base + threadIdx.x;
  // a CTA's calls start on a multiple of a power of two: none crosses 2^32
  const Start st = drop_start(D, call, (unsigned)((unsigned long long)base * (E / 4) >> 32));
  Pack<T, E> xv[VECS], rv[VECS];
#pragma unroll
  for (int k = 0; k < VECS; ++k) {
    const long long v = v0 + k * kThreads;
    if (v < vecs) {
      xv[k] = load_pack<T, E>(x + v * E);
      if (RES) rv[k] = load_pack<T, E>(res + v * E);
    }
  }
#pragma unroll
  for (int k = 0; k < VECS; ++k) {
    const long long v = v0 + k * kThreads;
    if (v < vecs) {
#pragma unroll
      for (int g = 0; g < E / 4; ++g) {
        unsigned w[4];
        drop_words(D, st, (unsigned)v * (E / 4) + g, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float y = drop_one(D, w[j], to_f32(xv[k].v[g * 4 + j]));
          if (RES) y += to_f32(rv[k].v[g * 4 + j]);
          xv[k].v[g * 4 + j] = from_f32<T>(y);
        }
      }
      store_pack(out + v * E, xv[k]);
    }
  }
}

// Elements from `from` on, four (one Philox call) per thread.
template <typename T, bool RES>
__global__ void __launch_bounds__(kThreads) k_dropout(Drop D, const T* __restrict__ x, const T* __restrict__ res,
                                                      long long from, long long n, T* __restrict__ out) {
  const unsigned long long call = D.call + (D.call_dev ? (unsigned long long)*D.call_dev : 0ull);
  const long long groups = (n + 3) / 4, stride = (long long)gridDim.x * blockDim.x;
  for (long long q = from / 4 + blockIdx.x * (long long)blockDim.x + threadIdx.x; q < groups; q += stride) {
    unsigned w[4];
    drop_words(D, drop_start(D, call, (unsigned)(q >> 32)), (unsigned)q, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long i = q * 4 + j;
      if (i < n) {
        float y = drop_one(D, w[j], to_f32(x[i]));
        if (RES) y += to_f32(res[i]);
        out[i] = from_f32<T>(y);
      }
    }
  }
}

template <typename T, bool RES>
int run(const Drop& D, const T* x, const T* res, long long n, T* out, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T), VECS = 4;
  long long done = 0;
  if (aligned_to(x, 16) && aligned_to(out, 16) && (!RES || aligned_to(res, 16))) {
    const long long vecs = n / E, per = kThreads * VECS;
    if (vecs > 0)
      launch(k_dropout_vec<T, RES, VECS>, (unsigned)((vecs + per - 1) / per), kThreads, 0, s, D, x, res, n, out);
    done = vecs * E;
  }
  if (done < n) {  // the rest, fewer than E elements behind whole vectors
    const int grid = clamp_grid(((n - done + 3) / 4 + kThreads - 1) / kThreads);
    launch(k_dropout<T, RES>, grid, kThreads, 0, s, D, x, res, done, n, out);
  }
  return launch_status("dropout");
}

}  // namespace

int dropout(int dtype, const void* x, const void* residual, long long n, double p, unsigned long long seed,
            unsigned long long call, const long long* call_dev, void* out, cudaStream_t s) {
  if (n <= 0) return ATLB_OK;
  const unsigned long long t = (unsigned long long)(p * 4294967296.0 + 0.5);
  Drop D;
  philox_keys((unsigned)seed, (unsigned)(seed >> 32), D.key);
  D.call = call;
  D.call_dev = call_dev;
  D.threshold = (unsigned)t;
  D.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
  if (t > 0xffffffffull) {  // p rounds to 1: nothing is kept
    const size_t bytes = (size_t)n * (dtype == ATLB_F32 ? 4 : 2);
    const cudaError_t e = residual ? cudaMemcpyAsync(out, residual, bytes, cudaMemcpyDeviceToDevice, s)
                                   : cudaMemsetAsync(out, 0, bytes, s);
    return e == cudaSuccess ? ATLB_OK : launch_status("dropout");
  }
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (residual) return run<T, true>(D, (const T*)x, (const T*)residual, n, (T*)out, s);
    return run<T, false>(D, (const T*)x, nullptr, n, (T*)out, s);
  });
}

}  // namespace atlb
