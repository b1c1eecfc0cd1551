// Lane layout, tiles and dispatch shared by the selective scan's forward and backward.
#pragma once

#include <type_traits>

#include "selective.cuh"

namespace mogt {
namespace sel {

constexpr int NT = 128;      // threads per CTA of the forward
constexpr int NTB = 256;     // and of the backward
constexpr int NS = 4;        // states per thread
constexpr int kGroup = 8;    // tokens handled together
constexpr int kTile = 16;    // tokens per B/C tile and per saved state
constexpr int kMaxN = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// log(1 + e^x); above 20 it is x to the last bit of fp32.
__device__ __forceinline__ float softplus(float x) { return x > 20.f ? x : log1pf(expf(x)); }

// Lane = c + CPW * j: channel c of the warp's CPW, part j of its LPC.
template <int LPC>
struct Lane {
  static constexpr int CPW = 32 / LPC;                       // channels per warp
  static constexpr int NP = LPC * NS;                        // states, padded
  static constexpr int TPL = LPC >= kGroup ? 1 : kGroup / LPC;  // tokens of a group per lane
  static constexpr int DUP = LPC > kGroup ? LPC / kGroup : 1;   // lanes per token beyond that
};

struct Geo {
  int64_t Dg, nblk, nck;  // channels per group, channel blocks per group, saved states per sequence
};

// Channel, group and batch row of a thread.  grid = (nblk * G, segments, B).
template <int LPC>
struct Where {
  int warp, c, j;
  int64_t b, g, d;
  bool ok;
  __device__ __forceinline__ Where(const mogt_selective_args& p, const Geo& geo) {
    const int lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    c = lane % Lane<LPC>::CPW;
    j = lane / Lane<LPC>::CPW;
    b = blockIdx.z;
    g = blockIdx.x / geo.nblk;
    const int64_t i = (blockIdx.x % geo.nblk) * (int)(blockDim.x / LPC) + warp * Lane<LPC>::CPW + c;
    ok = i < geo.Dg;
    d = g * geo.Dg + (ok ? i : 0);
  }
  // first token of the group that this lane loads, and whether it stores it
  __device__ __forceinline__ int part_tok() const { return LPC >= kGroup ? j / Lane<LPC>::DUP : j * Lane<LPC>::TPL; }
  __device__ __forceinline__ bool owner() const { return Lane<LPC>::DUP == 1 || j % Lane<LPC>::DUP == 0; }
};

template <int LPC>
__device__ __forceinline__ void load_A(float (&A2)[NS], const mogt_selective_args& p, const Where<LPC>& w) {
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int n = w.j * NS + i;
    A2[i] = (w.ok && n < p.N) ? p.A[w.d * p.N + n] * kLog2e : 0.f;
  }
}

// Tile of B or C rows t0..t0+kTile-1 as fp32, padded states and dead tokens zero.
template <typename T, int NP, typename W>
__device__ __forceinline__ void load_bc(float (*dst)[NP], const mogt_selective_args& p, const W& w, const T* src,
                                        int64_t sb, int64_t sl, int64_t sg, int64_t t0, int64_t len) {
  const T* base = src + w.b * sb + w.g * sg;
  for (int i = threadIdx.x; i < kTile * NP; i += blockDim.x) {
    const int k = i / NP, n = i % NP;
    dst[k][n] = (n < p.N && t0 + k < len) ? to_f32(base[(t0 + k) * sl + n]) : 0.f;
  }
}

// Sums v[0..7][M] over the LPC parts of a channel.  Afterwards v[i] holds
// token part_tok() + i.  Each halving step exchanges half of what is left.
template <int LPC, int M>
__device__ __forceinline__ void sum_parts(float (&v)[kGroup][M], int j) {
  int n = kGroup;
#pragma unroll
  for (int bit = LPC / 2; bit > 0; bit >>= 1) {
    const bool hi = j & bit;
    const int off = bit * Lane<LPC>::CPW;
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < kGroup / 2; ++i)
        if (i < n)
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const float send = hi ? v[i][m] : v[i + n][m];
            const float keep = hi ? v[i + n][m] : v[i][m];
            v[i][m] = keep + __shfl_xor_sync(0xffffffffu, send, off);
          }
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m) v[0][m] += __shfl_xor_sync(0xffffffffu, v[0][m], off);
    }
  }
}

// Sums v[0..7][M] over the CPW channels of a warp.  Afterwards v[i] holds
// token chan_tok(c) + i (each token on chan_dup lanes).
template <int CPW>
struct ChanTok {
  static constexpr int TPL = CPW >= kGroup ? 1 : kGroup / CPW;
  static constexpr int DUP = CPW > kGroup ? CPW / kGroup : 1;
  __device__ static __forceinline__ int first(int c) { return CPW >= kGroup ? c / DUP : c * TPL; }
  __device__ static __forceinline__ bool owner(int c) { return DUP == 1 || c % DUP == 0; }
};
template <int CPW, int M>
__device__ __forceinline__ void sum_channels(float (&v)[kGroup][M], int c) {
  int n = kGroup;
#pragma unroll
  for (int bit = CPW / 2; bit > 0; bit >>= 1) {
    const bool hi = c & bit;
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < kGroup / 2; ++i)
        if (i < n)
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const float send = hi ? v[i][m] : v[i + n][m];
            const float keep = hi ? v[i + n][m] : v[i][m];
            v[i][m] = keep + __shfl_xor_sync(0xffffffffu, send, bit);
          }
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m) v[0][m] += __shfl_xor_sync(0xffffffffu, v[0][m], bit);
    }
  }
}

inline int lpc_of(int64_t N) {
  int l = 1;
  while (l * NS < N) l <<= 1;
  return l;
}

inline Geo geometry(const mogt_selective_args& p, int threads) {
  Geo g;
  g.Dg = p.D / p.G;
  const int64_t cpb = threads / lpc_of(p.N);
  g.nblk = (g.Dg + cpb - 1) / cpb;
  g.nck = (p.L + kTile - 1) / kTile;
  return g;
}

inline int check_args(const mogt_selective_args& p) {
  if (p.B < 0 || p.L < 0 || p.D < 0 || p.N <= 0 || p.G <= 0 || p.D % p.G) return MOGT_ERR_SHAPE;
  if (p.N > kMaxN || p.B > 65535) return MOGT_ERR_UNSUPPORTED;
  if (p.dtype < 0 || p.dtype > 2) return MOGT_ERR_DTYPE;
  return MOGT_OK;
}

template <typename T, typename F>
int dispatch_n(int64_t N, F&& f) {
  switch (lpc_of(N)) {
    case 1: return f(T{}, std::integral_constant<int, 1>{});
    case 2: return f(T{}, std::integral_constant<int, 2>{});
    case 4: return f(T{}, std::integral_constant<int, 4>{});
    case 8: return f(T{}, std::integral_constant<int, 8>{});
    case 16: return f(T{}, std::integral_constant<int, 16>{});
    case 32: return f(T{}, std::integral_constant<int, 32>{});
    default: return MOGT_ERR_UNSUPPORTED;
  }
}
template <typename F>
int dispatch(int dtype, int64_t N, F&& f) {
  switch (dtype) {
    case MOGT_DTYPE_F32: return dispatch_n<float>(N, f);
    case MOGT_DTYPE_BF16: return dispatch_n<__nv_bfloat16>(N, f);
    case MOGT_DTYPE_F16: return dispatch_n<__half>(N, f);
    default: return MOGT_ERR_DTYPE;
  }
}

}  // namespace sel
}  // namespace mogt
