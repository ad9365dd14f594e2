// 16- and 32-bit element types of the event-sequence operators (embed.cu, dropout.cu, recurrence.cu): conversion
// to and from fp32, and loads and stores of several neighbouring elements as one access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace atlb {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// One rounding, to nearest even.
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// N neighbouring elements as they lie in memory; an access of the whole pack needs its alignment.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> r;
  if constexpr (sizeof(r) == 16) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    memcpy(&r, &q, 16);
  } else if constexpr (sizeof(r) == 8) {
    const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
    memcpy(&r, &q, 8);
  } else if constexpr (sizeof(r) == 4) {
    const unsigned q = __ldg(reinterpret_cast<const unsigned*>(p));
    memcpy(&r, &q, 4);
  } else {
    static_assert(sizeof(r) == 2, "packs of 2, 4, 8 or 16 bytes");
    const unsigned short q = __ldg(reinterpret_cast<const unsigned short*>(p));
    memcpy(&r, &q, 2);
  }
  return r;
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& r) {
  *reinterpret_cast<Pack<T, N>*>(p) = r;
}

inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Calls fn(T()) with the element type of an atlb_dtype (checked by the caller).
template <typename Fn>
inline int with_dtype(int dtype, Fn&& fn) {
  if (dtype == ATLB_BF16) return fn(__nv_bfloat16());
  if (dtype == ATLB_F16) return fn(__half());
  return fn(float());
}

// Consecutive arrays carved out of a caller's workspace, each on a 256-byte boundary; with a null base it only
// adds up the bytes.
struct Carve {
  char* base;
  size_t used = 0;
  explicit Carve(void* p) : base(static_cast<char*>(p)) {
    if (base) used = (256 - (reinterpret_cast<uintptr_t>(base) & 255)) & 255;
  }
  template <typename T>
  T* take(long long n) {
    T* r = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += ((size_t)n * sizeof(T) + 255) / 256 * 256;
    return r;
  }
  size_t bytes_needed() const { return used + 256; }  // slack for an unaligned base
};

}  // namespace atlb
