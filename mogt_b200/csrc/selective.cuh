// Shared pieces of the selective state space kernels: loads and stores of
// VEC consecutive elements as fp32, parameters of a run-time type, the
// activations, and sums over lanes that leave each lane a different item.
#pragma once

#include "../../include/mogt_selective.h"
#include "common.cuh"

namespace mogt {

template <int BYTES>
struct RawVec;
template <>
struct RawVec<2> { using type = uint16_t; };
template <>
struct RawVec<4> { using type = uint32_t; };
template <>
struct RawVec<8> { using type = uint2; };
template <>
struct RawVec<16> { using type = uint4; };

// VEC consecutive elements of T, read or written as one access of VEC * sizeof(T) bytes.
template <typename T, int VEC>
struct Pack {
  using Raw = typename RawVec<VEC * (int)sizeof(T)>::type;
  union {
    Raw raw;
    T e[VEC];
  };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(0.f);
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ float f(int i) const { return to_f32<T>(e[i]); }
  __device__ __forceinline__ void set(int i, float x) { e[i] = from_f32<T>(x); }
};

// A parameter array whose element type is known at run time.
__device__ __forceinline__ float ld_param(const void* p, int code, int64_t i) {
  if (code == MOGT_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (code == MOGT_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void st_param(void* p, int code, int64_t i, float x) {
  if (code == MOGT_DTYPE_F32) static_cast<float*>(p)[i] = x;
  else if (code == MOGT_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// Tokens of sequence b (clamped to [0, L]).
__device__ __forceinline__ int64_t seq_len(const int64_t* lengths, int64_t b, int64_t L) {
  if (!lengths) return L;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > L ? L : n);
}

}  // namespace mogt
