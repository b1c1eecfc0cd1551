// Lane layout, tiles and dispatch shared by the selective scan's forward and backward.
#pragma once

#include <cfloat>
#include <initializer_list>
#include <type_traits>

#include "selective.cuh"

namespace mogt {
namespace sel {

constexpr int NT = 128;      // threads per CTA of the forward
constexpr int NTB = 128;     // and of the backward
constexpr int NS = 4;        // states per thread, of each of its two channels
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
// |x| is cut off where e is 0 in any case: a delta of -inf or of the type's
// lowest value masks a step, and inf - inf must not be formed from it.
__device__ __forceinline__ float exp_neg_abs(float x) {
  const float a = -fminf(fabsf(x), 127.f), t = a * kLog2e;
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

// Four values, each for both halves of a register pair (both channels).
__device__ __forceinline__ void twice4(F2 (&r)[4], const float* p) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  r[0] = f2(v.x, v.x);
  r[1] = f2(v.y, v.y);
  r[2] = f2(v.z, v.z);
  r[3] = f2(v.w, v.w);
}
// exp(dt A) for the pair, A given times log2(e).  ex2.approx comes out low by
// 2e-8 on average where results lie in [0.7, 1) (measured over a million
// arguments: -1.7e-8 to -2.0e-8 for exponents in [-0.5, -1e-3]).  One step does
// not notice, but a state with a memory of a thousand steps would be off by a
// thousand times that, all in one direction; the exponent is shifted by as
// much, in the multiply-add that forms it.  dt = 0 still gives exactly 1.
constexpr float kExp2Shift = 2.8e-8f;
__device__ __forceinline__ F2 decay(F2 dt, F2 A2) {
  return exp2_2(fma2(dt, A2, f2(kExp2Shift, kExp2Shift)));
}

// Lane = c + CPW * j: channel pair c of the warp's CPW, part j of its LPC.
template <int LPC, int GROUP = kGroup>
struct Lane {
  static constexpr int CPW = 32 / LPC;                        // channel pairs per warp
  static constexpr int NP = LPC * NS;                         // states, padded
  static constexpr int TPL = LPC >= GROUP ? 1 : GROUP / LPC;  // tokens of a group per lane
  static constexpr int DUP = LPC > GROUP ? LPC / GROUP : 1;   // lanes per token beyond that
};

struct Geo {
  int64_t Dg, nblk, nck;  // channels per group, channel blocks per group, tiles per sequence
  int64_t tps;            // tiles per segment
  int nseg;               // segments per sequence (gridDim.y)
};

// CTAs of a forward (or first) pass on an SM: fewer lanes per pair hold more
// tokens each and need more registers.
constexpr int fwd_ctas(int lpc) { return lpc < 4 ? 2 : 4; }
inline int channels_per_cta(int threads, int lpc) { return 2 * threads / lpc; }

// Channels (a pair), group and batch row of a thread.  grid = (nblk * G, segments, B).
template <int LPC, int GROUP = kGroup>
struct Where {
  int warp, c, j;
  int64_t b, g, d;  // d: first channel of the pair (a channel of the group for idle lanes)
  bool ok, ok1;     // the first and the second channel exist
  __device__ __forceinline__ Where(const mogt_selective_args& p, const Geo& geo) {
    const int lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    c = lane % Lane<LPC>::CPW;
    j = lane / Lane<LPC>::CPW;
    b = blockIdx.z;
    g = blockIdx.x / geo.nblk;
    const int64_t i = (blockIdx.x % geo.nblk) * (int)(2 * blockDim.x / LPC) + 2 * (warp * Lane<LPC>::CPW + c);
    ok = i < geo.Dg;
    ok1 = i + 1 < geo.Dg;
    d = g * geo.Dg + (ok ? i : 0);
  }
  // first token of the group that this lane loads, and whether it stores it
  __device__ __forceinline__ int part_tok() const {
    return LPC >= GROUP ? j / Lane<LPC, GROUP>::DUP : j * Lane<LPC, GROUP>::TPL;
  }
  __device__ __forceinline__ bool owner() const { return Lane<LPC, GROUP>::DUP == 1 || j % Lane<LPC, GROUP>::DUP == 0; }
  // a per-channel parameter, 0 where it is not given
  __device__ __forceinline__ float2 param(const float* v) const {
    return v ? make_float2(v[d], v[d + ok1]) : make_float2(0.f, 0.f);
  }
  // [D, N] values of state n for both channels, 0 for padded states and missing channels
  __device__ __forceinline__ F2 state(const float* v, int64_t cell, int64_t N, int n) const {
    return f2(v && ok && n < N ? v[cell * N + n] : 0.f, v && ok1 && n < N ? v[(cell + 1) * N + n] : 0.f);
  }
  __device__ __forceinline__ void put_state(float* v, int64_t cell, int64_t N, int n, F2 x) const {
    if (n < N) {
      if (ok) v[cell * N + n] = un2(x).x;
      if (ok1) v[(cell + 1) * N + n] = un2(x).y;
    }
  }
  // The 4 states of a lane for both channels in [.., D, LPC] float4 arrays (i: first channel's index)
  __device__ __forceinline__ void put4(float4* v, int64_t i, const F2 (&x)[NS]) const {
    const float2 a = un2(x[0]), b = un2(x[1]), e = un2(x[2]), f = un2(x[3]);
    if (ok) v[i * LPC] = make_float4(a.x, b.x, e.x, f.x);
    if (ok1) v[(i + 1) * LPC] = make_float4(a.y, b.y, e.y, f.y);
  }
};

// Two neighbouring channels' elements.  VEC: one access (pairs aligned);
// otherwise two (one: distance to the second channel, 0 when there is none).
template <typename T>
struct Two {
  using Raw = typename RawVec<2 * (int)sizeof(T)>::type;
  union {
    Raw raw;
    T e[2];
  };
  __device__ __forceinline__ Two() {}
  template <bool VEC>
  __device__ __forceinline__ void load(const T* p, int one) {
    if (VEC) {
      raw = *reinterpret_cast<const Raw*>(p);
    } else {
      e[0] = p[0];
      e[1] = p[one];
    }
  }
  __device__ __forceinline__ float2 f() const { return make_float2(to_f32(e[0]), to_f32(e[1])); }
};
template <typename T, bool VEC>
__device__ __forceinline__ void store_two(T* p, float a, float b, bool second) {
  Two<T> v;
  v.e[0] = from_f32<T>(a);
  v.e[1] = from_f32<T>(b);
  if (VEC) {
    *reinterpret_cast<typename Two<T>::Raw*>(p) = v.raw;
  } else {
    p[0] = v.e[0];
    if (second) p[1] = v.e[1];
  }
}

// A lane's elements of one [B, L, D] operand for COUNT runs of TPL tokens,
// GROUP apart.  fetch() only issues the loads.  Tokens behind the end are read
// from the last live one and cleared where they are used: no load needs a
// predicate, and an address is one multiply-add.
template <typename T, int TPL, int GROUP, int COUNT, bool VEC>
struct Raws {
  Two<T> v[COUNT][TPL];
  // p: the tile's first token; tok: the lane's first; last: index of the last live token in the tile
  __device__ __forceinline__ void fetch(const T* p, int sl, int tok, int last, int one) {
#pragma unroll
    for (int q = 0; q < COUNT; ++q)
#pragma unroll
      for (int i = 0; i < TPL; ++i)
        v[q][i].template load<VEC>(p + (int64_t)min(q * GROUP + tok + i, last) * sl, one);
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

// dt and x = dt u of a pair from its raw operands, (0, 0) for dead tokens.
struct DtX {
  float2 dt, x;
};
__device__ __forceinline__ DtX make_dtx(float2 delta, float2 u, float2 bias, bool sp, bool dead) {
  DtX r;
  r.dt = make_float2(delta.x + bias.x, delta.y + bias.y);
  if (sp) r.dt = make_float2(softplus(r.dt.x), softplus(r.dt.y));
  r.x = make_float2(r.dt.x * u.x, r.dt.y * u.y);
  if (dead) r.dt = r.x = make_float2(0.f, 0.f);
  return r;
}

// States in XORed order (the backward): slot i of a lane of channel pair c
// holds state i ^ (c & mask).
template <int LPC>
struct Perm {
  static constexpr int COPIES = Lane<LPC>::CPW >= 4 ? 4 : Lane<LPC>::CPW;
  static constexpr int MASK = COPIES - 1;
  __device__ static __forceinline__ float4 apply(float4 v, int c) {
    if (COPIES > 1 && (c & 1)) v = make_float4(v.y, v.x, v.w, v.z);
    if (COPIES > 2 && (c & 2)) v = make_float4(v.z, v.w, v.x, v.y);
    return v;
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

// exp(dt A) x where exp(dt A) alone is beyond the largest float (growing
// states: A or dt of the other sign): nothing stays nothing, and by the square
// root twice a small x gets the value that it grows to.
__device__ __forceinline__ float grown(float dt, float A2, float x) {
  const float r = fast_exp2(0.5f * fmaf(dt, A2, kExp2Shift));
  return x == 0.f ? 0.f : x * r * r;
}
// a x + l for both halves, a = exp(sd A) over a whole segment.
__device__ __forceinline__ F2 carry(F2 sd, F2 A2, F2 x, F2 l) {
  const F2 a = decay(sd, A2);
  const float2 v = un2(a);
  if (!(fmaxf(v.x, v.y) > FLT_MAX)) return fma2(a, x, l);
  const float2 d = un2(sd), e = un2(A2), s = un2(x);
  return add2(f2(v.x > FLT_MAX ? grown(d.x, e.x, s.x) : v.x * s.x, v.y > FLT_MAX ? grown(d.y, e.y, s.y) : v.y * s.y), l);
}

// The state (or adjoint) entering a segment: the chain over segments
// first, first + step, ..., count of them.  x: what the chain starts from.
template <int LPC, typename W, bool PERM>
__device__ __forceinline__ void chain(F2 (&x)[NS], const F2 (&A2)[NS], const SegScratch& s, int first, int step,
                                      int count, int64_t BD, int64_t cell, const W& w) {
#pragma unroll 2
  for (int k = 0; k < count; ++k) {
    const int64_t i = (first + k * step) * BD + cell;
    float4 l0 = s.loc[i * LPC + w.j], l1 = s.loc[(i + w.ok1) * LPC + w.j];
    if (PERM) {
      l0 = Perm<LPC>::apply(l0, w.c);
      l1 = Perm<LPC>::apply(l1, w.c);
    }
    const F2 sd = f2(s.sdt[i], s.sdt[i + w.ok1]);
    x[0] = carry(sd, A2[0], x[0], f2(l0.x, l1.x));
    x[1] = carry(sd, A2[1], x[1], f2(l0.y, l1.y));
    x[2] = carry(sd, A2[2], x[2], f2(l0.z, l1.z));
    x[3] = carry(sd, A2[3], x[3], f2(l0.w, l1.w));
  }
}

// Sums v[0..GROUP-1][M] over the LPC parts of a channel (STEP lanes apart).  Afterwards v[i] holds
// token part_tok() + i.  Each halving step exchanges half of what is left.
template <int LPC, int STEP = 32 / LPC, int GROUP, int M>
__device__ __forceinline__ void sum_parts(float (&v)[GROUP][M], int j) {
  int n = GROUP;
#pragma unroll
  for (int bit = LPC / 2; bit > 0; bit >>= 1) {
    const bool hi = j & bit;
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < GROUP / 2; ++i)
        if (i < n)
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const float send = hi ? v[i][m] : v[i + n][m];
            const float keep = hi ? v[i + n][m] : v[i][m];
            v[i][m] = keep + __shfl_xor_sync(0xffffffffu, send, bit * STEP);
          }
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m) v[0][m] += __shfl_xor_sync(0xffffffffu, v[0][m], bit * STEP);
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
// the price of a first pass over all but one of them.  Of 1..64 segments (no
// shorter than 4 tiles) the count with the least estimated time is taken: a
// pass over a segment costs its length per wave of CTAs (`slots` resident at
// once), the first pass `agg` of that.
inline int64_t num_segments(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G, int threads, int slots, float agg) {
  const int64_t cpb = channels_per_cta(threads, lpc_of(N));
  const int64_t ctas = B * G * ((D / G + cpb - 1) / cpb), nck = (L + kTile - 1) / kTile;
  int64_t best = 1;
  double least = 1e30;
  for (int64_t s = 1; s <= 64 && s * 4 <= nck; ++s) {
    // a full wave runs at the full rate; a partly filled one gains little per missing CTA
    auto waves = [&](int64_t n) {
      const double full = (double)(n / slots), rest = (double)(n % slots) / slots;
      return full + (rest > 0 ? 0.5 + 0.5 * rest : 0.0);
    };
    // in tiles: starting a segment costs about one, each link of its chain a tenth
    const double len = (double)((nck + s - 1) / s) + 1.0;
    const double t = waves(ctas * s) * (len + 0.1 * (double)s) + agg * waves(ctas * (s - 1)) * len;
    if (t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

inline Geo geometry(const mogt_selective_args& p, int threads, int64_t segments) {
  Geo g;
  g.Dg = p.D / p.G;
  const int64_t cpb = channels_per_cta(threads, lpc_of(p.N));
  g.nblk = (g.Dg + cpb - 1) / cpb;
  g.nck = (p.L + kTile - 1) / kTile;
  g.tps = (g.nck + segments - 1) / segments;
  g.nseg = g.nck > 0 ? (int)((g.nck + g.tps - 1) / g.tps) : 1;
  return g;
}

// Pairs of channels can be accessed at once: even group width, row strides
// and sequence strides, and bases aligned to a pair.
inline bool pairs_aligned(const mogt_selective_args& p, bool backward) {
  const uintptr_t a = p.dtype == MOGT_DTYPE_F32 ? 8 : 4;
  bool ok = (p.D / p.G) % 2 == 0;
  auto strided = [&](const void* q, int64_t sb, int64_t sl) {
    if (q) ok = ok && reinterpret_cast<uintptr_t>(q) % a == 0 && sb % 2 == 0 && sl % 2 == 0;
  };
  auto dense = [&](const void* q) { ok = ok && reinterpret_cast<uintptr_t>(q) % a == 0; };
  strided(p.u, p.u_sb, p.u_sl);
  strided(p.delta, p.delta_sb, p.delta_sl);
  strided(p.z, p.z_sb, p.z_sl);
  if (backward) {
    strided(p.dout, p.dout_sb, p.dout_sl);
    dense(p.du);
    dense(p.ddelta);
    dense(p.dz);
  } else {
    dense(p.out);
  }
  return ok;
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
