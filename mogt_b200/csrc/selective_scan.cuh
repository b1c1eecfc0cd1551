// Lane layout, tiles and dispatch shared by the selective scan's forward and backward.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "selective.cuh"

namespace mogt {
namespace sel {

constexpr int NT = 128;      // threads per CTA of the forward
#ifndef MOGT_NTB
#define MOGT_NTB 256
#endif
constexpr int NTB = MOGT_NTB;  // and of the backward
constexpr int NS = 4;        // states per thread
constexpr int kGroup = 8;    // tokens handled together by the forward
constexpr int kGroupB = 4;   // and by the backward
constexpr int kTile = 16;    // tokens per B/C tile and per saved state
constexpr int kMaxN = 128;
constexpr int64_t kMaxStride = (int64_t)1 << 27;  // of a token, in elements
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// log(1 + e^x) = max(x, 0) + log1p(e), e = e^-|x| in (0, 1], with
// log1p(e) = 2 atanh(s) = 2 (s + s^3/3 + s^5/5 + ...), s = e / (2 + e) <= 1/3.
// Seven terms leave 1.5e-8; relative accuracy for small e, which the step
// sizes near softplus' lower end need, comes with the series.  The exponent's
// rounding error is put back (a product rounded at |x| = 10 is off by 5e-7).
__device__ __forceinline__ float exp_neg_abs(float x) {
  const float a = -fabsf(x), t = a * kLog2e;
  return fast_exp2(t) * fmaf(fmaf(a, kLog2e, -t), kLn2, 1.f);
}
__device__ __forceinline__ float softplus_e(float x, float e) {
  const float s = __fdividef(e, 2.f + e), q = s * s;
  float r = fmaf(q, 1.f / 13.f, 1.f / 11.f);
  r = fmaf(q, r, 1.f / 9.f);
  r = fmaf(q, r, 1.f / 7.f);
  r = fmaf(q, r, 1.f / 5.f);
  r = fmaf(q, r, 1.f / 3.f);
  r = fmaf(q * s, r, s);
  return x > -87.f ? fmaf(2.f, r, fmaxf(x, 0.f)) : (x == x ? 0.f : x);  // e^-87 is the last normal e
}
__device__ __forceinline__ float softplus(float x) { return softplus_e(x, exp_neg_abs(x)); }

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
__device__ __forceinline__ F2 exp2_2(F2 a) {
  const float2 v = un2(a);
  return f2(fast_exp2(v.x), fast_exp2(v.y));
}
__device__ __forceinline__ float hsum(F2 a) {
  const float2 v = un2(a);
  return v.x + v.y;
}

// Lane = c + CPW * j: channel c of the warp's CPW, part j of its LPC.
template <int LPC, int GROUP = kGroup>
struct Lane {
  static constexpr int CPW = 32 / LPC;                        // channels per warp
  static constexpr int NP = LPC * NS;                         // states, padded
  static constexpr int TPL = LPC >= GROUP ? 1 : GROUP / LPC;  // tokens of a group per lane
  static constexpr int DUP = LPC > GROUP ? LPC / GROUP : 1;   // lanes per token beyond that
};

struct Geo {
  int64_t Dg, nblk, nck;  // channels per group, channel blocks per group, tiles per sequence
  int64_t tps;            // tiles per segment
  int nseg;               // segments per sequence (gridDim.y)
};

// Channel, group and batch row of a thread.  grid = (nblk * G, segments, B).
template <int LPC, int GROUP = kGroup>
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
  __device__ __forceinline__ int part_tok() const {
    return LPC >= GROUP ? j / Lane<LPC, GROUP>::DUP : j * Lane<LPC, GROUP>::TPL;
  }
  __device__ __forceinline__ bool owner() const { return Lane<LPC, GROUP>::DUP == 1 || j % Lane<LPC, GROUP>::DUP == 0; }
};

// A lane's elements of one [B, L, D] operand for one tile: TPL tokens of each
// group of GROUP.  fetch() only issues the loads.  Tokens behind the end are
// read from the last live one and cleared where they are used: no load needs
// a predicate, and an address is one multiply-add.
template <typename T, int TPL, int GROUP>
struct TileRaw {
  T v[kTile / GROUP][TPL];
  // p: the tile's first token; tok: the lane's first; last: index of the last live token in the tile
  __device__ __forceinline__ void fetch(const T* p, int sl, int tok, int last) {
#pragma unroll
    for (int q = 0; q < kTile / GROUP; ++q)
#pragma unroll
      for (int i = 0; i < TPL; ++i) v[q][i] = p[(int64_t)min(q * GROUP + tok + i, last) * sl];
  }
};

// The same for one group of a tile (first token kk of the lane).
template <typename T, int TPL>
struct GroupRaw {
  T v[TPL];
  __device__ __forceinline__ void fetch(const T* p, int sl, int kk, int last) {
#pragma unroll
    for (int i = 0; i < TPL; ++i) v[i] = p[(int64_t)min(kk + i, last) * sl];
  }
};

// A thread's share of one B or C tile (kTile x NP values over THREADS threads).
template <typename T, int NP, int THREADS>
struct BcRaw {
  static constexpr int PER = (kTile * NP + THREADS - 1) / THREADS;
  T v[PER];
  __device__ __forceinline__ void fetch(const T* p, int sl, int N, int last) {
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      const int i = threadIdx.x + r * THREADS;
      v[r] = p[(int64_t)min(i / NP, last) * sl + min(i % NP, N - 1)];
    }
  }
  // value r, or 0 for padded states and dead tokens
  __device__ __forceinline__ float get(int r, int N, int last) const {
    const int i = threadIdx.x + r * THREADS;
    return i % NP < N && i / NP <= last ? to_f32(v[r]) : 0.f;
  }
  __device__ __forceinline__ void put(float (*dst)[NP], int N, int last) const {
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      const int i = threadIdx.x + r * THREADS;
      if (kTile * NP % THREADS == 0 || i < kTile * NP) dst[i / NP][i % NP] = get(r, N, last);
    }
  }
};

// Segment carries.  A segment maps the state h entering it to
// exp(A sum dt) h + loc (loc: its state from zero), a reverse segment the
// adjoint likewise, so what a segment starts from is a short chain over the
// segments before it.
struct SegScratch {
  float4* loc;  // [nseg - 1][B][D][LPC]
  float* sdt;   // [nseg - 1][B][D]
};

template <int LPC, typename W>
__device__ __forceinline__ void load_A(float (&A2)[NS], const mogt_selective_args& p, const W& w) {
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int n = w.j * NS + i;
    A2[i] = (w.ok && n < p.N) ? p.A[w.d * p.N + n] * kLog2e : 0.f;
  }
}

// Sums v[0..GROUP-1][M] over the LPC parts of a channel.  Afterwards v[i] holds
// token part_tok() + i.  Each halving step exchanges half of what is left.
template <int LPC, int GROUP, int M>
__device__ __forceinline__ void sum_parts(float (&v)[GROUP][M], int j) {
  int n = GROUP;
#pragma unroll
  for (int bit = LPC / 2; bit > 0; bit >>= 1) {
    const bool hi = j & bit;
    const int off = bit * Lane<LPC>::CPW;
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < GROUP / 2; ++i)
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

inline int lpc_of(int64_t N) {
  int l = 1;
  while (l * NS < N) l <<= 1;
  return l;
}

// Segments: the scan over one sequence is serial, so when channels and
// sequences alone do not fill the GPU the tiles are split into segments, at
// the price of a first pass over all but one of them (states from zero; about
// `cost` of the main pass).  Warps wanted: `warps_per_sm` on 148 SMs.
inline int64_t num_segments(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G, int threads, int warps_per_sm) {
  const int64_t cpb = threads / lpc_of(N);
  const int64_t warps = B * G * ((D / G + cpb - 1) / cpb) * (threads / 32);
  const int64_t nck = (L + kTile - 1) / kTile;
  int64_t s = (148 * (int64_t)warps_per_sm) / (warps > 0 ? warps : 1);
  if (s > nck / 4) s = nck / 4;  // a segment shorter than 4 tiles spends its time starting
  if (s > 64) s = 64;
  return s < 2 ? 1 : s;
}

inline Geo geometry(const mogt_selective_args& p, int threads, int warps_per_sm) {
  Geo g;
  g.Dg = p.D / p.G;
  const int64_t cpb = threads / lpc_of(p.N);
  g.nblk = (g.Dg + cpb - 1) / cpb;
  g.nck = (p.L + kTile - 1) / kTile;
  const int64_t s = num_segments(p.B, p.L, p.D, p.N, p.G, threads, warps_per_sm);
  g.tps = (g.nck + s - 1) / s;
  g.nseg = g.nck > 0 ? (int)((g.nck + g.tps - 1) / g.tps) : 1;
  return g;
}

inline size_t seg_scratch_bytes(int64_t B, int64_t D, int64_t N, int64_t nseg) {
  return nseg < 2 ? 0 : (size_t)((nseg - 1) * B * D) * (lpc_of(N) * NS + 1) * sizeof(float);
}
inline SegScratch seg_scratch(void* base, int64_t B, int64_t D, int64_t N, int64_t nseg) {
  SegScratch s;
  s.loc = static_cast<float4*>(base);
  s.sdt = static_cast<float*>(base) + (nseg - 1) * B * D * lpc_of(N) * NS;
  return s;
}

inline int check_args(const mogt_selective_args& p) {
  if (p.B < 0 || p.L < 0 || p.D < 0 || p.N <= 0 || p.G <= 0 || p.D % p.G) return MOGT_ERR_SHAPE;
  if (p.N > kMaxN || p.B > 65535 || p.L > kMaxStride || p.D > kMaxStride) return MOGT_ERR_UNSUPPORTED;
  // offsets inside a tile are 32-bit
  for (int64_t s : {p.u_sl, p.delta_sl, p.z ? p.z_sl : 0, p.B_sl, p.C_sl, p.dout ? p.dout_sl : 0})
    if (s > kMaxStride || s < 0) return MOGT_ERR_UNSUPPORTED;
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
