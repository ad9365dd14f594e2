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
  unsigned k0, k1;              // seed words
  unsigned long long call;
  const long long* call_dev;    // added to call when not null: a graph replay can draw anew
  unsigned threshold;           // keep when the word is at least this
  bool none;                    // p rounds to 1: nothing is kept
  float scale;
};

__device__ __forceinline__ Philox4 drop_words(const Drop& D, unsigned long long call, unsigned long long q) {
  return philox4x32_10(Philox4{(unsigned)q, (unsigned)(q >> 32) | 0x80000000u, (unsigned)call, (unsigned)(call >> 32)},
                       D.k0, D.k1);
}

__device__ __forceinline__ float drop_one(const Drop& D, unsigned word, float x) {
  return (word >= D.threshold && !D.none) ? x * D.scale : 0.f;
}

// One thread per group of four elements (one Philox call).
template <typename T, bool RES>
__global__ void __launch_bounds__(kThreads) k_dropout(Drop D, const T* __restrict__ x, const T* __restrict__ res,
                                                      long long n, T* __restrict__ out) {
  const unsigned long long call = D.call + (D.call_dev ? (unsigned long long)*D.call_dev : 0ull);
  const long long groups = (n + 3) / 4, stride = (long long)gridDim.x * blockDim.x;
  for (long long q = blockIdx.x * (long long)blockDim.x + threadIdx.x; q < groups; q += stride) {
    const Philox4 w = drop_words(D, call, (unsigned long long)q);
    const unsigned word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long i = q * 4 + j;
      if (i < n) {
        float v = drop_one(D, word[j], to_f32(x[i]));
        if (RES) v += to_f32(res[i]);
        out[i] = from_f32<T>(v);
      }
    }
  }
}

}  // namespace

int dropout(int dtype, const void* x, const void* residual, long long n, double p, unsigned long long seed,
            unsigned long long call, const long long* call_dev, void* out, cudaStream_t s) {
  if (n <= 0) return ATLB_OK;
  const unsigned long long t = (unsigned long long)(p * 4294967296.0 + 0.5);
  Drop D{(unsigned)seed, (unsigned)(seed >> 32), call, call_dev, (unsigned)t, t > 0xffffffffull,
         p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f};
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    const int grid = clamp_grid((n / 4 + kThreads) / kThreads);
    if (residual)
      launch(k_dropout<T, true>, grid, kThreads, 0, s, D, (const T*)x, (const T*)residual, n, (T*)out);
    else
      launch(k_dropout<T, false>, grid, kThreads, 0, s, D, (const T*)x, (const T*)nullptr, n, (T*)out);
    return launch_status("dropout");
  });
}

}  // namespace atlb
