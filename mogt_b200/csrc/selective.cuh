// Shared pieces of the selective state space and loss kernels: loads and stores
// of VEC consecutive elements as fp32, parameters of a run-time type, the
// activations, packed fp32 pairs.
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

// Two elements in a 32-bit word (16-bit types) or a pair of floats, as fp32.
template <typename T>
__device__ __forceinline__ float2 unpack_two(const uint32_t* w);
template <>
__device__ __forceinline__ float2 unpack_two<float>(const uint32_t* w) {
  return make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
template <>
__device__ __forceinline__ float2 unpack_two<__nv_bfloat16>(const uint32_t* w) {
  return make_float2(__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack_two<__half>(const uint32_t* w) {
  return __half22float2(*reinterpret_cast<const __half2*>(w));
}
template <typename T>
__device__ __forceinline__ void pack_two(uint32_t* w, float a, float b);
template <>
__device__ __forceinline__ void pack_two<float>(uint32_t* w, float a, float b) {
  w[0] = __float_as_uint(a);
  w[1] = __float_as_uint(b);
}
template <>
__device__ __forceinline__ void pack_two<__nv_bfloat16>(uint32_t* w, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(w) = __floats2bfloat162_rn(a, b);
}
template <>
__device__ __forceinline__ void pack_two<__half>(uint32_t* w, float a, float b) {
  *reinterpret_cast<__half2*>(w) = __floats2half2_rn(a, b);
}

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

// Store to a parameter array whose element type is known at run time.
__device__ __forceinline__ void st_param(void* p, int code, int64_t i, float x) {
  if (code == MOGT_DTYPE_F32) static_cast<float*>(p)[i] = x;
  else if (code == MOGT_DTYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// Two fp32 in one 64-bit register: one instruction for both halves.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 un2(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// sum += x, with the rounding error of the addition collected in lost.
__device__ __forceinline__ void add_kept(F2& sum, F2& lost, F2 x) {
  const F2 minus = f2(-1.f, -1.f);
  const F2 s = add2(sum, x), part = fma2(sum, minus, s);     // what of x arrived
  const F2 e1 = fma2(fma2(part, minus, s), minus, sum);      // sum - (s - part)
  const F2 e2 = fma2(part, minus, x);                        // x - part
  lost = add2(lost, add2(e1, e2));
  sum = s;
}
__device__ __forceinline__ F2 exp2_2(F2 a) {
  const float2 v = un2(a);
  return f2(fast_exp2(v.x), fast_exp2(v.y));
}
__device__ __forceinline__ float hsum(F2 a) {
  const float2 v = un2(a);
  return v.x + v.y;
}

// Tokens of sequence b (clamped to [0, L]).
__device__ __forceinline__ int64_t seq_len(const int64_t* lengths, int64_t b, int64_t L) {
  if (!lengths) return L;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n > L ? L : n);
}

}  // namespace mogt
