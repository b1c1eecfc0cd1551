// Backward of the selective state space scan.  With dy_t = dout_t silu(z_t),
// a_t = exp(dt_t A), x_t = dt_t u_t and g_t the adjoint of h_t:
//   g_t = C_t dy_t + a_{t+1} g_{t+1}
//   dC_t = sum_d dy_t h_t          dB_t = sum_d g_t x_t
//   s_t = sum_n g_t B_t            q_t = g_t (a_t h_{t-1})
//   du_t = dt_t s_t + D dy_t       ddt_t = u_t s_t + sum_n A q_t
//   dA = sum_t dt_t q_t            dD = sum_t dy_t u_t
//   dz_t = dout_t y_t silu'(z_t)   ddelta_t = ddt_t softplus'(delta_t + bias)
// a_t h_{t-1} is kept as such (h_t - x_t B_t would cancel where a_t is small).
//
// The forward saved the state every 16 tokens.  A warp walks its channels'
// tiles backwards; a tile's first 12 tokens are stepped to get the states that
// enter its groups of 4, then each group is stepped again with a_t and
// a_t h_{t-1} kept in registers, and walked backwards.  Lanes are those of
// the forward (4 states each, LPC lanes per channel), and a long sequence is
// split into segments as there, the adjoint's carries from a first pass.
//
// dB and dC need sums over all channels.  Per token a lane holds 8 terms (4
// states of each), the warp's channels are added by halving exchanges that
// leave a lane one term: a lane keeps its states in an order XORed with its
// channel number (B and C come in as many permuted copies), so that what it
// sends is always the same registers and no selects are needed.  The CTA's
// warps add through shared memory and CTAs through a second kernel, in a
// fixed order.  Instruction issue bounds it (about 20 per token, channel and
// state), then the shuffles.
#include "selective_scan.cuh"

namespace mogt {
namespace sel {

#ifndef MOGT_BWD_WARPS
#define MOGT_BWD_WARPS 16
#endif
#ifndef MOGT_BWD_CTAS
#define MOGT_BWD_CTAS 2
#endif
constexpr int kBwdWarps = MOGT_BWD_WARPS;  // warps per SM that the backward asks for

struct BwdScratch {
  SegScratch seg;
  float* bc;   // [nblk][B][G][L][2][NP]
  float* dA;   // [nseg * B][D][NP]
  float* dv;   // [nseg * B][2][D]: dD, dbias
};

// States in XORed order: slot i of a lane of channel c holds state i ^ (c & mask).
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

// One token's B or C: for every 4 states their COPIES orders side by side, so
// that the lanes of a quarter warp (one part, 8 channels) read 64 consecutive
// bytes: [part][copy][4].
template <typename T, int LPC, int THREADS>
__device__ __forceinline__ void put_copies(float4 (*dst)[LPC][Perm<LPC>::COPIES],
                                           const BcRaw<T, Lane<LPC>::NP, THREADS>& r, int N, int last) {
  constexpr int NP = Lane<LPC>::NP;
#pragma unroll
  for (int x = 0; x < BcRaw<T, NP, THREADS>::PER; ++x) {
    const int i = threadIdx.x + x * THREADS;
    if (kTile * NP % THREADS == 0 || i < kTile * NP) {
      const int k = i / NP, n = i % NP;
      const float v = r.get(x, N, last);
#pragma unroll
      for (int q = 0; q < Perm<LPC>::COPIES; ++q) reinterpret_cast<float*>(&dst[k][n / NS][q])[(n % NS) ^ q] = v;
    }
  }
}

template <int LPC>
struct BwdSmem {
  // two tiles: the one being worked on and the one being fetched
  float4 B[2][kTile][LPC][Perm<LPC>::COPIES], C[2][kTile][LPC][Perm<LPC>::COPIES];
  float2 s1[2][NTB / 32][kTile][Lane<LPC>::CPW];   // (dt, x)
  float4 s2[2][NTB / 32][kTile][Lane<LPC>::CPW];   // (dy, u, softplus', dout silu'(z))
  float4 hs[kTile / kGroupB - 1][NTB];             // states entering the tile's groups
  float red[2][NTB / 32][kTile / 2][2][Lane<LPC>::NP];
};

// First pass over a split sequence: per segment (all but the first) the
// adjoint handed to the state before it, from nothing behind it, and sum dt.
template <typename T, int LPC>
__global__ void __launch_bounds__(NT, LPC < 4 ? 3 : 4) scan_bwd_agg_kernel(const mogt_selective_args p,
                                                                         const Geo geo, const SegScratch seg) {
  using Q = Lane<LPC>;
  constexpr int CPW = Q::CPW, TPL = Q::TPL, NP = Q::NP;
  __shared__ __align__(16) float sC[2][kTile][NP];
  __shared__ float2 stage[NT / 32][kTile][CPW];  // (dt, dy)
  const Where<LPC> w(p, geo);
  const int64_t len = seq_len(p.lengths, w.b, p.L);
  const int64_t k0 = (int64_t)(blockIdx.y + 1) * geo.tps, k1 = min(k0 + geo.tps, geo.nck);
  const int64_t kl = min(k1, (len + kTile - 1) / kTile);
  const int64_t cell = w.b * p.D + w.d;
  float A2[NS];
  load_A<LPC>(A2, p, w);
  const F2 A01 = f2(A2[0], A2[1]), A23 = f2(A2[2], A2[3]);
  F2 g01 = 0, g23 = 0;
  const float bias = p.bias ? p.bias[w.d] : 0.f;
  const int tok = w.part_tok(), N = (int)p.N;
  const int d_sl = (int)p.delta_sl, z_sl = (int)p.z_sl, o_sl = (int)p.dout_sl, C_sl = (int)p.C_sl;
  const bool gate = p.z, sp = p.softplus;
  const T* dp = static_cast<const T*>(p.delta) + w.b * p.delta_sb + w.d;
  const T* zp = static_cast<const T*>(p.z) + w.b * p.z_sb + w.d;
  const T* op = static_cast<const T*>(p.dout) + w.b * p.dout_sb + w.d;
  const T* Cp = static_cast<const T*>(p.Cm) + w.b * p.C_sb + w.g * p.C_sg;
  TileRaw<T, TPL, kGroup> rd, rz, ro;
  BcRaw<T, NP, NT> rC;
  int last = 0;
  auto fetch = [&](int64_t k) {
    const int64_t t0 = k * kTile;
    last = (int)min(len - 1 - t0, (int64_t)(kTile - 1));
    rC.fetch(Cp + t0 * C_sl, C_sl, N, last);
    rd.fetch(dp + t0 * d_sl, d_sl, tok, last);
    ro.fetch(op + t0 * o_sl, o_sl, tok, last);
    if (gate) rz.fetch(zp + t0 * z_sl, z_sl, tok, last);
  };
  float sdt = 0.f;
  if (k0 < kl) fetch(kl - 1);
  for (int64_t k = kl - 1; k >= k0; --k) {
    const int buf = (int)(k & 1), live = last;
    rC.put(sC[buf], N, live);
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int kk = q * kGroup + tok + i;
        float dt = to_f32(rd.v[q][i]) + bias, dy = to_f32(ro.v[q][i]);
        if (sp) dt = softplus(dt);
        if (gate) {
          const float z = to_f32(rz.v[q][i]);
          dy *= z * sigmoid(z);
        }
        if (kk > live) dt = dy = 0.f;
        if (Q::DUP == 1 || w.owner()) stage[w.warp][kk][w.c] = make_float2(dt, dy);
      }
    __syncthreads();
    if (k > k0) fetch(k - 1);
    float sd = 0.f;
#pragma unroll
    for (int kk = kTile - 1; kk >= 0; --kk) {
      const float2 s = stage[w.warp][kk][w.c];
      const F2 dt2 = f2(s.x, s.x), dy2 = f2(s.y, s.y);
      const ulonglong2 Cv = *reinterpret_cast<const ulonglong2*>(&sC[buf][kk][w.j * NS]);
      g01 = mul2(exp2_2(mul2(dt2, A01)), fma2(Cv.x, dy2, g01));
      g23 = mul2(exp2_2(mul2(dt2, A23)), fma2(Cv.y, dy2, g23));
      sd += s.x;
    }
    sdt += sd;
    __syncwarp();
  }
  if (w.ok) {
    const float2 a = un2(g01), b = un2(g23);
    const int64_t i = blockIdx.y * p.B * p.D + cell;
    seg.loc[i * LPC + w.j] = make_float4(a.x, a.y, b.x, b.y);
    if (w.j == 0) seg.sdt[i] = sdt;
  }
}

// Sums the 8 terms of one token (dB: v[0..3], dC: v[4..7], XORed order) over
// the warp's channels and leaves them in row r[2][NP] of shared memory.
template <int LPC>
__device__ __forceinline__ void channel_sums(F2 b01, F2 b23, F2 c01, F2 c23, float (*r)[Lane<LPC>::NP], int c,
                                             int j) {
  constexpr int CPW = Lane<LPC>::CPW;
  constexpr unsigned ALL = 0xffffffffu;
  const float2 b0 = un2(b01), b1 = un2(b23), c0 = un2(c01), c1 = un2(c23);
  float v[8] = {b0.x, b0.y, b1.x, b1.y, c0.x, c0.y, c1.x, c1.y};
  const int n0 = j * NS;
  if constexpr (CPW == 1) {
    *reinterpret_cast<float4*>(&r[0][n0]) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(&r[1][n0]) = make_float4(v[4], v[5], v[6], v[7]);
  } else if constexpr (CPW == 2) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) v[i] += __shfl_xor_sync(ALL, v[i + 1], 1);
    r[0][n0 + c] = v[0];
    r[0][n0 + 2 + c] = v[2];
    r[1][n0 + c] = v[4];
    r[1][n0 + 2 + c] = v[6];
  } else {
#pragma unroll
    for (int q = 0; q < 8; q += 4) {
      v[q] += __shfl_xor_sync(ALL, v[q + 2], 2);
      v[q + 1] += __shfl_xor_sync(ALL, v[q + 3], 2);
      v[q] += __shfl_xor_sync(ALL, v[q + 1], 1);
    }
    if constexpr (CPW == 4) {
      r[0][n0 + c] = v[0];
      r[1][n0 + c] = v[4];
    } else {
      const bool hi = c & 4;
      float t = (hi ? v[4] : v[0]) + __shfl_xor_sync(ALL, hi ? v[0] : v[4], 4);
      if constexpr (CPW >= 16) t += __shfl_xor_sync(ALL, t, 8);
      if constexpr (CPW >= 32) t += __shfl_xor_sync(ALL, t, 16);
      if (CPW == 8 || c < 8) r[hi ? 1 : 0][n0 + (c & 3)] = t;
    }
  }
}

template <typename T, int LPC>
__global__ void __launch_bounds__(NTB, LPC == 4 || LPC == 8 ? MOGT_BWD_CTAS : 1)
    scan_bwd_kernel(const mogt_selective_args p, const Geo geo, const BwdScratch sc) {
  using Q = Lane<LPC, kGroupB>;
  constexpr int CPW = Q::CPW, TPL = Q::TPL, NP = Q::NP, NG = kTile / kGroupB;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  BwdSmem<LPC>& sm = *reinterpret_cast<BwdSmem<LPC>*>(smem_raw);
  const Where<LPC, kGroupB> w(p, geo);
  const int64_t len = seq_len(p.lengths, w.b, p.L);
  const int64_t k0 = (int64_t)blockIdx.y * geo.tps, k1 = min(k0 + geo.tps, geo.nck);
  const int64_t kl = min(k1, (len + kTile - 1) / kTile);
  const int64_t cell = w.b * p.D + w.d;
  const int cq = w.c & Perm<LPC>::MASK;

  F2 A01, A23, cy01, cy23;
  {
    float A2[NS], cy[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int n = w.j * NS + (i ^ cq);
      A2[i] = (w.ok && n < p.N) ? p.A[w.d * p.N + n] * kLog2e : 0.f;
      cy[i] = (p.dfinal && w.ok && n < p.N) ? p.dfinal[cell * p.N + n] : 0.f;
    }
#pragma unroll 4
    for (int s = geo.nseg - 1; s > (int)blockIdx.y; --s) {
      const int64_t i = (s - 1) * p.B * p.D + cell;
      const float4 l = Perm<LPC>::apply(sc.seg.loc[i * LPC + w.j], w.c);
      const float sd = sc.seg.sdt[i];
      cy[0] = fmaf(fast_exp2(sd * A2[0]), cy[0], l.x);
      cy[1] = fmaf(fast_exp2(sd * A2[1]), cy[1], l.y);
      cy[2] = fmaf(fast_exp2(sd * A2[2]), cy[2], l.z);
      cy[3] = fmaf(fast_exp2(sd * A2[3]), cy[3], l.w);
    }
    A01 = f2(A2[0], A2[1]);
    A23 = f2(A2[2], A2[3]);
    cy01 = f2(cy[0], cy[1]);
    cy23 = f2(cy[2], cy[3]);
  }
  const F2 one = f2(1.f, 1.f);
  F2 sumA01 = 0, sumA23 = 0;
  float sumD = 0.f, sumb = 0.f;
  const float Dd = p.Dskip ? p.Dskip[w.d] : 0.f;
  const float bias = p.bias ? p.bias[w.d] : 0.f;
  const bool gate = p.z, sp = p.softplus, store = w.ok && w.owner();
  const int tok = w.part_tok(), N = (int)p.N, D = (int)p.D;
  const int u_sl = (int)p.u_sl, d_sl = (int)p.delta_sl, z_sl = (int)p.z_sl, o_sl = (int)p.dout_sl,
            B_sl = (int)p.B_sl, C_sl = (int)p.C_sl;
  const T* up = static_cast<const T*>(p.u) + w.b * p.u_sb + w.d;
  const T* dp = static_cast<const T*>(p.delta) + w.b * p.delta_sb + w.d;
  const T* zp = static_cast<const T*>(p.z) + w.b * p.z_sb + w.d;
  const T* op = static_cast<const T*>(p.dout) + w.b * p.dout_sb + w.d;
  const T* Bp = static_cast<const T*>(p.Bm) + w.b * p.B_sb + w.g * p.B_sg;
  const T* Cp = static_cast<const T*>(p.Cm) + w.b * p.C_sb + w.g * p.C_sg;
  const float4* saved = reinterpret_cast<const float4*>(p.saved) + (w.b * geo.nck * p.D + w.d) * LPC + w.j;
  const int64_t o0 = (w.b * p.L + tok) * p.D + w.d;
  T* du = static_cast<T*>(p.du) + o0;
  T* ddelta = static_cast<T*>(p.ddelta) + o0;
  T* dz = gate ? static_cast<T*>(p.dz) + o0 : nullptr;
  float* bcp = sc.bc + (((blockIdx.x % geo.nblk) * p.B + w.b) * p.G + w.g) * p.L * (2 * NP);

  // tiles behind the end
  for (int64_t t = max(kl, k0) * kTile; t < min(k1 * kTile, p.L); t += kGroupB)
#pragma unroll
    for (int i = 0; i < TPL; ++i)
      if (store && t + tok + i < p.L) {
        du[(t + i) * p.D] = from_f32<T>(0.f);
        ddelta[(t + i) * p.D] = from_f32<T>(0.f);
        if (gate) dz[(t + i) * p.D] = from_f32<T>(0.f);
      }

  // Fetching is spread over the groups of the tile before: a group's raw
  // values are loaded when a group begins and staged when it ends, so few
  // registers wait on memory.
  GroupRaw<T, TPL> ru, rd, rz, ro;
  BcRaw<T, NP, NTB> rB, rC;
  float4 rs;
  auto last_of = [&](int64_t k) { return (int)min(len - 1 - k * kTile, (int64_t)(kTile - 1)); };
  auto fetch_bc = [&](int64_t k) {
    rB.fetch(Bp + k * kTile * B_sl, B_sl, N, last_of(k));
    rC.fetch(Cp + k * kTile * C_sl, C_sl, N, last_of(k));
  };
  auto fetch = [&](int64_t k, int q) {
    const int64_t t0 = k * kTile;
    const int last = last_of(k), kk = q * kGroupB + tok;
    rd.fetch(dp + t0 * d_sl, d_sl, kk, last);
    ru.fetch(up + t0 * u_sl, u_sl, kk, last);
    ro.fetch(op + t0 * o_sl, o_sl, kk, last);
    if (gate) rz.fetch(zp + t0 * z_sl, z_sl, kk, last);
  };
  auto stage = [&](int64_t k, int q) {
    const int live = last_of(k);
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      const int kk = q * kGroupB + tok + i;
      const float u = to_f32(ru.v[i]);
      float dt = to_f32(rd.v[i]) + bias, dy = to_f32(ro.v[i]), ds = 1.f, zf = 0.f;
      if (sp) {
        const float e = exp_neg_abs(dt);
        ds = __fdividef(dt >= 0.f ? 1.f : e, 1.f + e);
        dt = softplus_e(dt, e);
      }
      if (gate) {
        const float z = to_f32(rz.v[i]), sg = sigmoid(z);
        zf = dy * sg * (1.f + z * (1.f - sg));
        dy *= z * sg;
      }
      float x = dt * u;
      // dead tokens, and lanes without a channel (they share the sums over channels)
      if (kk > live || !w.ok) dt = x = dy = 0.f;
      if (Q::DUP == 1 || w.owner()) {
        sm.s1[k & 1][w.warp][kk][w.c] = make_float2(dt, x);
        sm.s2[k & 1][w.warp][kk][w.c] = make_float4(dy, u, ds, zf);
      }
    }
  };
  if (k0 < kl) {
    fetch_bc(kl - 1);
    rs = saved[(kl - 1) * p.D * LPC];
    put_copies<T, LPC, NTB>(sm.B[(kl - 1) & 1], rB, N, last_of(kl - 1));
    put_copies<T, LPC, NTB>(sm.C[(kl - 1) & 1], rC, N, last_of(kl - 1));
#pragma unroll
    for (int q = 0; q < NG; ++q) {
      fetch(kl - 1, q);
      stage(kl - 1, q);
    }
    __syncthreads();
  }
  for (int64_t k = kl - 1; k >= k0; --k) {
    const int64_t t0 = k * kTile;
    const int buf = (int)(k & 1), live = last_of(k);
    const float2(*s1)[CPW] = sm.s1[buf][w.warp];
    const float4(*s2)[CPW] = sm.s2[buf][w.warp];
    float4 h0 = Perm<LPC>::apply(rs, w.c);
    if (!w.ok) h0 = make_float4(0.f, 0.f, 0.f, 0.f);
    // states entering the tile's groups: of the first and last in registers
    F2 h01 = f2(h0.x, h0.y), h23 = f2(h0.z, h0.w);
    const F2 hf01 = h01, hf23 = h23;
#pragma unroll
    for (int q = 0; q + 1 < NG; ++q) {
      if (q > 0) sm.hs[q - 1][threadIdx.x] = make_float4(un2(h01).x, un2(h01).y, un2(h23).x, un2(h23).y);
#pragma unroll
      for (int i = 0; i < kGroupB; ++i) {
        const int kk = q * kGroupB + i;
        const float2 s = s1[kk][w.c];
        const F2 dt2 = f2(s.x, s.x), x2 = f2(s.y, s.y);
        const ulonglong2 Bv = *reinterpret_cast<const ulonglong2*>(&sm.B[buf][kk][w.j][cq]);
        h01 = fma2(exp2_2(mul2(dt2, A01)), h01, mul2(x2, Bv.x));
        h23 = fma2(exp2_2(mul2(dt2, A23)), h23, mul2(x2, Bv.y));
      }
    }
    F2 tA01 = 0, tA23 = 0;
    float tD = 0.f, tb = 0.f;
    const int rows = (int)min(p.L - t0, (int64_t)kTile);
#pragma unroll
    for (int q = NG - 1; q >= 0; --q) {
      if (k > k0) {
        fetch(k - 1, q);
        if (q == NG - 1) fetch_bc(k - 1);
        if (q == 0) rs = saved[(k - 1) * p.D * LPC];
      }
      if (q == 0) {
        h01 = hf01;
        h23 = hf23;
      } else if (q < NG - 1) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.hs[q - 1][threadIdx.x]);
        h01 = v.x;
        h23 = v.y;
      }
      F2 a[kGroupB][2], ph[kGroupB][2];
#pragma unroll
      for (int i = 0; i < kGroupB; ++i) {
        const int kk = q * kGroupB + i;
        const float2 s = s1[kk][w.c];
        const F2 dt2 = f2(s.x, s.x), x2 = f2(s.y, s.y);
        const ulonglong2 Bv = *reinterpret_cast<const ulonglong2*>(&sm.B[buf][kk][w.j][cq]);
        a[i][0] = exp2_2(mul2(dt2, A01));
        a[i][1] = exp2_2(mul2(dt2, A23));
        ph[i][0] = mul2(a[i][0], h01);
        ph[i][1] = mul2(a[i][1], h23);
        h01 = fma2(x2, Bv.x, ph[i][0]);
        h23 = fma2(x2, Bv.y, ph[i][1]);
      }
      float ysw[kGroupB][3];
#pragma unroll
      for (int i = kGroupB - 1; i >= 0; --i) {
        const int kk = q * kGroupB + i;
        const float2 s = s1[kk][w.c];
        const float dyv = s2[kk][w.c].x;
        const F2 dt2 = f2(s.x, s.x), x2 = f2(s.y, s.y), dy2 = f2(dyv, dyv);
        const ulonglong2 Bv = *reinterpret_cast<const ulonglong2*>(&sm.B[buf][kk][w.j][cq]);
        const ulonglong2 Cv = *reinterpret_cast<const ulonglong2*>(&sm.C[buf][kk][w.j][cq]);
        h01 = fma2(x2, Bv.x, ph[i][0]);
        h23 = fma2(x2, Bv.y, ph[i][1]);
        const F2 g01 = fma2(Cv.x, dy2, cy01), g23 = fma2(Cv.y, dy2, cy23);
        const F2 q01 = mul2(g01, ph[i][0]), q23 = mul2(g23, ph[i][1]);
        ysw[i][0] = hsum(fma2(Cv.y, h23, mul2(Cv.x, h01)));
        ysw[i][1] = hsum(fma2(Bv.y, g23, mul2(Bv.x, g01)));
        ysw[i][2] = hsum(fma2(A23, q23, mul2(A01, q01)));
        tA01 = fma2(dt2, q01, tA01);
        tA23 = fma2(dt2, q23, tA23);
        cy01 = mul2(a[i][0], g01);
        cy23 = mul2(a[i][1], g23);
        channel_sums<LPC>(mul2(g01, x2), mul2(g23, x2), mul2(dy2, h01), mul2(dy2, h23),
                          sm.red[kk / (kTile / 2)][w.warp][kk % (kTile / 2)], w.c, w.j);
      }
      sum_parts<LPC>(ysw, w.j);
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int kk = q * kGroupB + i;  // + tok
        const float dt = s1[kk + tok][w.c].x;
        const float4 v = s2[kk + tok][w.c];  // (dy, u, softplus', dout silu'(z))
        float gu = fmaf(dt, ysw[i][1], Dd * v.x);
        float gd = fmaf(v.y, ysw[i][1], kLn2 * ysw[i][2]) * v.z;
        float gz = v.w * fmaf(Dd, v.y, ysw[i][0]);
        if (kk + tok > live) {
          gu = gd = gz = 0.f;
        } else {
          tD = fmaf(v.x, v.y, tD);
          tb += gd;
        }
        if (store && kk + tok < rows) {
          const int64_t o = (t0 + kk) * D;
          du[o] = from_f32<T>(gu);
          ddelta[o] = from_f32<T>(gd);
          if (gate) dz[o] = from_f32<T>(gz);
        }
      }
      if (k > k0) {
        stage(k - 1, q);
        if (q == NG - 1) {
          put_copies<T, LPC, NTB>(sm.B[buf ^ 1], rB, N, last_of(k - 1));
          put_copies<T, LPC, NTB>(sm.C[buf ^ 1], rC, N, last_of(k - 1));
        }
      }
      if (q % (NG / 2) == 0) {  // half a tile: add up the warps
        const int half = q / (NG / 2);
        __syncthreads();
#pragma unroll
        for (int i0 = 0; i0 < kTile * NP; i0 += NTB) {
          const int i = i0 + threadIdx.x;
          if (kTile * NP % NTB == 0 || i < kTile * NP) {
            float v = 0.f;
#pragma unroll
            for (int ww = 0; ww < NTB / 32; ++ww) v += (&sm.red[half][ww][0][0][0])[i];
            const int kk = half * (kTile / 2) + i / (2 * NP);
            if (kk <= live) bcp[(t0 + kk) * (2 * NP) + i % (2 * NP)] = v;
          }
        }
      }
    }
    sumA01 = fma2(one, tA01, sumA01);
    sumA23 = fma2(one, tA23, sumA23);
    sumD += tD;
    sumb += tb;
  }
  if (!w.owner()) sumD = sumb = 0.f;
  const int64_t row = blockIdx.y * p.B + w.b;
  if (w.ok) {
    const float2 a0 = un2(sumA01), a1 = un2(sumA23), c0 = un2(cy01), c1 = un2(cy23);
    const float sa[NS] = {a0.x, a0.y, a1.x, a1.y}, cc[NS] = {c0.x, c0.y, c1.x, c1.y};
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int n = w.j * NS + (i ^ cq);
      sc.dA[(row * p.D + w.d) * NP + n] = sa[i];
      if (p.dinit && blockIdx.y == 0 && n < p.N) p.dinit[cell * p.N + n] = cc[i];
    }
  }
#pragma unroll
  for (int o = CPW; o < 32; o <<= 1) {
    sumD += __shfl_xor_sync(0xffffffffu, sumD, o);
    sumb += __shfl_xor_sync(0xffffffffu, sumb, o);
  }
  if (w.ok && w.j == 0) {
    sc.dv[(row * 2 + 0) * p.D + w.d] = sumD;
    sc.dv[(row * 2 + 1) * p.D + w.d] = sumb;
  }
}

// dB, dC [B, L, G, N] from the CTAs' partial rows.
template <typename T>
__global__ void __launch_bounds__(256) reduce_bc_kernel(const mogt_selective_args p, int64_t nblk, int NP,
                                                        const float* bc) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t total = p.B * p.L * p.G * 2 * p.N;
  if (i >= total) return;
  const int64_t n = i % p.N, which = (i / p.N) % 2, g = (i / (2 * p.N)) % p.G, bt = i / (2 * p.N * p.G);
  const int64_t t = bt % p.L, b = bt / p.L;
  float v = 0.f;
  if (t < seq_len(p.lengths, b, p.L)) {
    const float* src = bc + ((b * p.G + g) * p.L + t) * (2 * NP) + which * NP + n;
    const int64_t stride = p.B * p.G * p.L * 2 * NP;
    for (int64_t k = 0; k < nblk; ++k) v += src[k * stride];
  }
  T* dst = static_cast<T*>(which ? p.dC : p.dB);
  dst[(bt * p.G + g) * p.N + n] = from_f32<T>(v);
}

// dA, dD, dbias from the partial sums of sequences and segments.
__global__ void __launch_bounds__(256) reduce_param_kernel(const mogt_selective_args p, int NP, int64_t rows,
                                                           const BwdScratch sc) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t na = p.D * p.N;
  if (i < na) {
    const int64_t d = i / p.N, n = i % p.N;
    double v = 0.0;
    for (int64_t r = 0; r < rows; ++r) v += sc.dA[(r * p.D + d) * NP + n];
    p.dA[i] = (float)v;
  } else if (i < na + 2 * p.D) {
    const int64_t k = i - na;
    double v = 0.0;
    for (int64_t r = 0; r < rows; ++r) v += sc.dv[r * 2 * p.D + k];
    float* dst = k < p.D ? p.dD : p.dbias;
    if (dst) dst[k % p.D] = (float)v;
  }
}

inline size_t bwd_floats(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G, int64_t nseg) {
  const int64_t np = lpc_of(N) * NS, cpb = NTB / lpc_of(N);
  const int64_t seg = (int64_t)(seg_scratch_bytes(B, D, N, nseg) / sizeof(float) + 3) / 4 * 4;
  return (size_t)(seg + (D / G + cpb - 1) / cpb * B * G * L * 2 * np + nseg * B * D * (np + 2));
}

}  // namespace sel
}  // namespace mogt

using namespace mogt;
using namespace mogt::sel;

extern "C" size_t mogt_selective_bwd_scratch_bytes(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G) {
  if (B <= 0 || L < 0 || D <= 0 || N <= 0 || N > kMaxN || G <= 0 || D % G) return 0;
  return bwd_floats(B, L, D, N, G, num_segments(B, L, D, N, G, NTB, kBwdWarps)) * sizeof(float);
}

extern "C" int mogt_selective_scan_bwd(const mogt_selective_args* args, void* stream) {
  if (!args) return MOGT_ERR_ARG;
  const mogt_selective_args& p = *args;
  if (int st = check_args(p)) return st;
  if (p.B == 0 || p.D == 0) return MOGT_OK;
  if (!p.A || !p.dA ||
      (p.L > 0 && (!p.u || !p.delta || !p.Bm || !p.Cm || !p.dout || !p.saved || !p.du || !p.ddelta || !p.dB ||
                   !p.dC || (p.z && !p.dz))))
    return MOGT_ERR_ARG;
  if (!p.scratch || p.scratch_bytes < mogt_selective_bwd_scratch_bytes(p.B, p.L, p.D, p.N, p.G))
    return MOGT_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(p.scratch) | reinterpret_cast<uintptr_t>(p.saved)) & 15u) return MOGT_ERR_ALIGN;
  const Geo geo = geometry(p, NTB, kBwdWarps);
  const int NP = lpc_of(p.N) * NS;
  BwdScratch sc;
  sc.seg = seg_scratch(p.scratch, p.B, p.D, p.N, geo.nseg);
  sc.dA = static_cast<float*>(p.scratch) + (seg_scratch_bytes(p.B, p.D, p.N, geo.nseg) / sizeof(float) + 3) / 4 * 4;
  sc.dv = sc.dA + geo.nseg * p.B * p.D * NP;
  sc.bc = sc.dv + geo.nseg * p.B * 2 * p.D;
  cudaStream_t s = (cudaStream_t)stream;
  return dispatch(p.dtype, p.N, [&](auto t, auto l) {
    using T = decltype(t);
    constexpr int LPC = decltype(l)::value;
    if (geo.nseg > 1) {
      Geo ga = geo;  // the first pass has smaller CTAs over the same segments
      ga.nblk = (geo.Dg + NT / LPC - 1) / (NT / LPC);
      scan_bwd_agg_kernel<T, LPC>
          <<<dim3((unsigned)(ga.nblk * p.G), geo.nseg - 1, (unsigned)p.B), NT, 0, s>>>(p, ga, sc.seg);
    }
    constexpr int bytes = (int)sizeof(BwdSmem<LPC>);
    auto kern = scan_bwd_kernel<T, LPC>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return (int)MOGT_ERR_LAUNCH;
    kern<<<dim3((unsigned)(geo.nblk * p.G), geo.nseg, (unsigned)p.B), NTB, bytes, s>>>(p, geo, sc);
    const int64_t nbc = p.B * p.L * p.G * 2 * p.N;
    if (nbc > 0) reduce_bc_kernel<T><<<(unsigned)((nbc + 255) / 256), 256, 0, s>>>(p, geo.nblk, NP, sc.bc);
    const int64_t np = p.D * p.N + 2 * p.D;
    reduce_param_kernel<<<(unsigned)((np + 255) / 256), 256, 0, s>>>(p, NP, geo.nseg * p.B, sc);
    return mogt_host::launch_status();
  });
}
