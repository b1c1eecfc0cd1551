// Backward of the selective state space scan.  With dy_t = dout_t silu(z_t),
// a_t = exp(dt_t A), x_t = dt_t u_t and g_t the adjoint of h_t:
//   g_t = C_t dy_t + a_{t+1} g_{t+1}
//   dC_t = sum_d dy_t h_t          dB_t = sum_d g_t x_t
//   s_t = sum_n g_t B_t            q_t = g_t (a_t h_{t-1})
//   du_t = dt_t s_t + D dy_t       ddt_t = u_t s_t + sum_n A q_t
//   dA = sum_t dt_t q_t            dD = sum_t dy_t u_t
//   dz_t = dout_t y_t silu'(z_t)   ddelta_t = ddt_t softplus'(delta_t + bias)
// q_t is formed as (a_t g_t) h_{t-1}: h_t - x_t B_t would cancel where a_t is
// small.
//
// The forward saved the state every 16 tokens.  A warp walks its channels'
// tiles backwards; a tile's first 12 tokens are stepped to get the states that
// enter its groups of 4, then each group is stepped again with a_t and h_t
// kept in registers, and walked backwards.  Lanes are those of the forward (4
// states of two channels each, LPC lanes per pair), and a long sequence is
// split into segments as there, the adjoint's carries from a first pass.
//
// dB and dC need sums over all channels.  Per token a lane holds 8 terms (4
// states of each, its two channels added), and the warp's pairs are added by
// halving exchanges that leave a lane one term: a lane keeps its states in an
// order XORed with its pair's number (B and C come in as many permuted
// copies), so that what it sends is always the same registers and no selects
// are needed.  The CTA's warps add through shared memory and CTAs through a
// second kernel, in a fixed order.
//
// 8192 x 1536 x 16 bf16: 320 us, with the first pass 402.  Nothing is at its
// limit: shared-memory wavefronts at 62 % of their peak, instruction issue at
// 54 % and HBM at 8 %, with 17 % of the warps resident, so that each waits on
// its own shuffles and shared memory.
#include "selective_scan.cuh"

namespace mogt {
namespace sel {

// CTAs on an SM by registers and shared memory.  For 4 lanes per pair (N = 16)
// three of 168 registers: 355 us at 8192 x 1536 (320 us since operands are
// copied asynchronously), against 427 us for two of 255 and 439 us for four of
// 128, which spill.  The others (two; one for N <= 4, whose lanes hold most
// tokens and registers) were not measured against their neighbours.
constexpr int bwd_ctas(int lpc) { return lpc == 4 ? 3 : lpc == 1 ? 1 : 2; }
// The first pass over a split sequence costs about a quarter of the main one.
inline int64_t bwd_segments(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G) {
  return num_segments(B, L, D, N, G, NTB, 148 * bwd_ctas(lpc_of(N)), 0.25f);
}

struct BwdScratch {
  SegScratch seg;
  float* bc;   // [nblk][B][G][L][2][NP]
  float* dA;   // [nseg * B][D][NP]
  float* dv;   // [nseg * B][2][D]: dD, dbias
};

// One token's B or C: for every 4 states their COPIES orders
// side by side, [part][copy][4], so that the lanes of one part read
// neighbouring copies.
template <typename T, int LPC>
__device__ __forceinline__ void put_copies(float (*dst)[LPC][Perm<LPC>::COPIES][NS],
                                           const BcRaw<T, Lane<LPC>::NP, NTB>& r, int N, int last) {
  constexpr int NP = Lane<LPC>::NP;
#pragma unroll
  for (int x = 0; x < BcRaw<T, NP, NTB>::PER; ++x) {
    const int i = threadIdx.x + x * NTB;
    if (kTile * NP % NTB == 0 || i < kTile * NP) {
      const int k = i / NP, n = i % NP;
      const float v = r.get(x, N, last);
#pragma unroll
      for (int q = 0; q < Perm<LPC>::COPIES; ++q) dst[k][n / NS][q][(n % NS) ^ q] = v;
    }
  }
}

// Tokens of a group of 4 that a lane takes: i-th of TPL.  The sums over parts
// halve over neighbouring tokens first (they can start after two tokens).
template <int LPC>
__device__ __forceinline__ int group_token(int j, int i) {
  if (LPC == 1) return i;
  if (LPC == 2) return 2 * i + j;
  const int t = j / (LPC >= 4 ? LPC / 4 : 1);
  return (t >> 1) + 2 * (t & 1);
}

// Halving step over lane bit `bit` of the part number: lanes without the bit
// keep (and receive the partner's share of) a, the others b.
template <int LPC>
__device__ __forceinline__ void halve(float (&a)[6], const float (&b)[6], int j, int bit) {
  const bool hi = j & bit;
#pragma unroll
  for (int m = 0; m < 6; ++m) {
    const float send = hi ? a[m] : b[m], keep = hi ? b[m] : a[m];
    a[m] = keep + __shfl_xor_sync(0xffffffffu, send, bit * Lane<LPC>::CPW);
  }
}

template <int LPC>
struct BwdSmem {
  float B[kTile][LPC][Perm<LPC>::COPIES][NS], C[kTile][LPC][Perm<LPC>::COPIES][NS];
  // per token and channel pair; a group's slots take the next tile's values once the group is done
  float4 s1[NTB / 32][kTile][Lane<LPC>::CPW];   // (dt, dt', x, x')
  float4 s2[NTB / 32][kTile][Lane<LPC>::CPW];   // (dy, dy', u, u')
  float4 s3[NTB / 32][kTile][Lane<LPC>::CPW];   // softplus' and dout silu'(z), both channels
  float4 hs[kTile / kGroupB - 1][2][NTB];       // states entering the tile's groups but the last
  float4 sumA[2][2][NTB];                       // a thread's sums for dA, and what their additions lost
  float red[2][NTB / 32][kTile / 2][2][Lane<LPC>::NP];
  // raw operands of the group and the states of the tile that are on their way, a thread's own
  uint2 raw[4][Lane<LPC, kGroupB>::TPL][NTB];
  float4 next[2][NTB];
};

// Asynchronous copy of BYTES (4, 8 or 16) to this thread's shared memory.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// First pass over a split sequence: per segment (all but the first) the
// adjoint handed to the state before it, from nothing behind it, and sum dt.
template <int LPC>
struct AggSmem {
  float C[2][kTile][Lane<LPC>::NP];
  float4 stage[NT / 32][kTile][Lane<LPC>::CPW];  // (dt, dt', dy, dy')
};

template <typename T, int LPC, bool VEC>
__global__ void __launch_bounds__(NT, fwd_ctas(LPC)) scan_bwd_agg_kernel(const mogt_selective_args p,
                                                                         const Geo geo, const SegScratch seg) {
  using Q = Lane<LPC>;
  constexpr int TPL = Q::TPL, NP = Q::NP;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  AggSmem<LPC>& sm = *reinterpret_cast<AggSmem<LPC>*>(smem_raw);
  const Where<LPC> w(p, geo);
  const int64_t len = seq_len(p.lengths, w.b, p.L);
  const int64_t k0 = (int64_t)(blockIdx.y + 1) * geo.tps, k1 = min(k0 + geo.tps, geo.nck);
  const int64_t kl = min(k1, (len + kTile - 1) / kTile);
  const int64_t cell = w.b * p.D + w.d;
  F2 A2[NS], g[NS];
  const F2 l2e = f2(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    A2[i] = mul2(w.state(p.A, w.d, p.N, w.j * NS + i), l2e);
    g[i] = 0;
  }
  const float2 bias = w.param(p.bias);
  const int tok = w.part_tok(), N = (int)p.N, one = w.ok1;
  const int d_sl = (int)p.delta_sl, z_sl = (int)p.z_sl, o_sl = (int)p.dout_sl, C_sl = (int)p.C_sl;
  const bool gate = p.z, sp = p.softplus;
  const T* dp = static_cast<const T*>(p.delta) + w.b * p.delta_sb + w.d;
  const T* zp = static_cast<const T*>(p.z) + w.b * p.z_sb + w.d;
  const T* op = static_cast<const T*>(p.dout) + w.b * p.dout_sb + w.d;
  const T* Cp = static_cast<const T*>(p.Cm) + w.b * p.C_sb + w.g * p.C_sg;
  Raws<T, TPL, kGroup, 2, VEC> rd, rz, ro;
  BcRaw<T, NP, NT> rC;
  int last = 0;
  auto fetch = [&](int64_t k) {
    const int64_t t0 = k * kTile;
    last = (int)min(len - 1 - t0, (int64_t)(kTile - 1));
    rC.fetch(Cp + t0 * C_sl, C_sl, N, last);
    rd.fetch(dp + t0 * d_sl, d_sl, tok, last, one);
    ro.fetch(op + t0 * o_sl, o_sl, tok, last, one);
    if (gate) rz.fetch(zp + t0 * z_sl, z_sl, tok, last, one);
  };
  float2 sdt = make_float2(0.f, 0.f);
  if (k0 < kl) fetch(kl - 1);
  for (int64_t k = kl - 1; k >= k0; --k) {
    const int buf = (int)(k & 1), live = last;
    rC.put(sm.C[buf], N, live);
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int kk = q * kGroup + tok + i;
        float2 dy = ro.v[q][i].f();
        if (gate) {
          const float2 z = rz.v[q][i].f();
          dy = make_float2(dy.x * z.x * sigmoid(z.x), dy.y * z.y * sigmoid(z.y));
        }
        // x of make_dtx is not used here: dy takes its place
        const DtX r = make_dtx(rd.v[q][i].f(), dy, bias, sp, kk > live);
        if (kk > live) dy = make_float2(0.f, 0.f);
        if (Q::DUP == 1 || w.owner()) sm.stage[w.warp][kk][w.c] = make_float4(r.dt.x, r.dt.y, dy.x, dy.y);
      }
    __syncthreads();
    if (k > k0) fetch(k - 1);
    F2 sd = 0;
#pragma unroll
    for (int kk = kTile - 1; kk >= 0; --kk) {
      const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(&sm.stage[w.warp][kk][w.c]);
      F2 Cn[NS];
      twice4(Cn, &sm.C[buf][kk][w.j * NS]);
#pragma unroll
      for (int m = 0; m < NS; ++m) g[m] = mul2(decay(s.x, A2[m]), fma2(Cn[m], s.y, g[m]));
      sd = add2(sd, s.x);
    }
    const float2 v = un2(sd);
    sdt = make_float2(sdt.x + v.x, sdt.y + v.y);
    __syncwarp();
  }
  const int64_t i = blockIdx.y * p.B * p.D + cell;
  w.put4(seg.loc + w.j, i, g);
  if (w.j == 0) {
    if (w.ok) seg.sdt[i] = sdt.x;
    if (w.ok1) seg.sdt[i + 1] = sdt.y;
  }
}

// Sums the 8 terms of one token (dB: b, dC: c, XORed order) over the warp's
// channels and leaves them in row r[2][NP] of shared memory.
template <int LPC>
__device__ __forceinline__ void channel_sums(const F2 (&b)[NS], const F2 (&d)[NS], float (*r)[Lane<LPC>::NP], int c,
                                             int j) {
  constexpr int CPW = Lane<LPC>::CPW;
  constexpr unsigned ALL = 0xffffffffu;
  float v[8];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    v[i] = hsum(b[i]);
    v[NS + i] = hsum(d[i]);
  }
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

template <typename T, int LPC, bool VEC>
__global__ void __launch_bounds__(NTB, bwd_ctas(LPC))
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

  F2 A2[NS], cy[NS];
  const F2 l2e = f2(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int n = w.j * NS + (i ^ cq);
    A2[i] = mul2(w.state(p.A, w.d, p.N, n), l2e);
    cy[i] = w.state(p.dfinal, cell, p.N, n);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sm.sumA[i / 2][i % 2][threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  chain<LPC, Where<LPC, kGroupB>, true>(cy, A2, sc.seg, geo.nseg - 2, -1, geo.nseg - 1 - (int)blockIdx.y, p.B * p.D,
                                        cell, w);
  F2 sumD = 0, lostD = 0, sumb = 0, lostb = 0;
  const float2 Dd = w.param(p.Dskip), bias = w.param(p.bias);
  const bool gate = p.z, sp = p.softplus, store = w.ok && w.owner();
  const int N = (int)p.N, D = (int)p.D, one = w.ok1;
  const int u_sl = (int)p.u_sl, d_sl = (int)p.delta_sl, z_sl = (int)p.z_sl, o_sl = (int)p.dout_sl,
            B_sl = (int)p.B_sl, C_sl = (int)p.C_sl;
  const T* up = static_cast<const T*>(p.u) + w.b * p.u_sb + w.d;
  const T* dp = static_cast<const T*>(p.delta) + w.b * p.delta_sb + w.d;
  const T* zp = static_cast<const T*>(p.z) + w.b * p.z_sb + w.d;
  const T* op = static_cast<const T*>(p.dout) + w.b * p.dout_sb + w.d;
  const T* Bp = static_cast<const T*>(p.Bm) + w.b * p.B_sb + w.g * p.B_sg;
  const T* Cp = static_cast<const T*>(p.Cm) + w.b * p.C_sb + w.g * p.C_sg;
  const float4* saved = reinterpret_cast<const float4*>(p.saved) + (w.b * geo.nck * p.D + w.d) * LPC + w.j;
  const int64_t o0 = w.b * p.L * p.D + w.d;
  T* du = static_cast<T*>(p.du) + o0;
  T* ddelta = static_cast<T*>(p.ddelta) + o0;
  T* dz = gate ? static_cast<T*>(p.dz) + o0 : nullptr;
  float* bcp = sc.bc + (((blockIdx.x % geo.nblk) * p.B + w.b) * p.G + w.g) * p.L * (2 * NP);

  // tiles behind the end
  for (int64_t t = max(kl, k0) * kTile; t < min(k1 * kTile, p.L); t += kGroupB)
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      const int64_t tt = t + group_token<LPC>(w.j, i);
      if (store && tt < p.L) {
        store_two<T, VEC>(du + tt * p.D, 0.f, 0.f, w.ok1);
        store_two<T, VEC>(ddelta + tt * p.D, 0.f, 0.f, w.ok1);
        if (gate) store_two<T, VEC>(dz + tt * p.D, 0.f, 0.f, w.ok1);
      }
    }

  // Fetching is spread over the groups of the tile before: a group's raw
  // values are fetched when a group begins and staged when it ends, so little
  // waits on memory: pairs as asynchronous copies into the thread's own slots
  // of shared memory, unaligned channels in registers.
  Two<T> ru[TPL], rd[TPL], rz[TPL], ro[TPL];
  BcRaw<T, NP, NTB> rB, rC;
  float4 rs0, rs1;
  auto last_of = [&](int64_t k) { return (int)min(len - 1 - k * kTile, (int64_t)(kTile - 1)); };
  auto fetch_bc = [&](int64_t k) {
    rB.fetch(Bp + k * kTile * B_sl, B_sl, N, last_of(k));
    rC.fetch(Cp + k * kTile * C_sl, C_sl, N, last_of(k));
  };
  auto fetch_saved = [&](int64_t k) {
    const float4* v = saved + k * p.D * LPC;
    if constexpr (VEC) {
      copy_async<16>(&sm.next[0][threadIdx.x], v);
      copy_async<16>(&sm.next[1][threadIdx.x], v + one * LPC);
    } else {
      rs0 = v[0];
      rs1 = v[one * LPC];
    }
  };
  auto fetch = [&](int64_t k, int q) {
    const int64_t t0 = k * kTile;
    const int last = last_of(k);
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      const int64_t t = t0 + min(q * kGroupB + group_token<LPC>(w.j, i), last);
      if constexpr (VEC) {
        constexpr int PAIR = 2 * (int)sizeof(T);
        copy_async<PAIR>(&sm.raw[0][i][threadIdx.x], dp + t * d_sl);
        copy_async<PAIR>(&sm.raw[1][i][threadIdx.x], up + t * u_sl);
        copy_async<PAIR>(&sm.raw[2][i][threadIdx.x], op + t * o_sl);
        if (gate) copy_async<PAIR>(&sm.raw[3][i][threadIdx.x], zp + t * z_sl);
      } else {
        rd[i].template load<false>(dp + t * d_sl, one);
        ru[i].template load<false>(up + t * u_sl, one);
        ro[i].template load<false>(op + t * o_sl, one);
        if (gate) rz[i].template load<false>(zp + t * z_sl, one);
      }
    }
    if constexpr (VEC) copies_issued();
  };
  auto stage = [&](int64_t k, int q) {
    const int live = last_of(k);
    if constexpr (VEC) copies_landed();
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      if constexpr (VEC) {
        using R = typename Two<T>::Raw;
        rd[i].raw = *reinterpret_cast<const R*>(&sm.raw[0][i][threadIdx.x]);
        ru[i].raw = *reinterpret_cast<const R*>(&sm.raw[1][i][threadIdx.x]);
        ro[i].raw = *reinterpret_cast<const R*>(&sm.raw[2][i][threadIdx.x]);
        if (gate) rz[i].raw = *reinterpret_cast<const R*>(&sm.raw[3][i][threadIdx.x]);
      }
      const int kk = q * kGroupB + group_token<LPC>(w.j, i);
      const float2 uu = ru[i].f(), dd = rd[i].f(), oo = ro[i].f();
      const float2 zz = gate ? rz[i].f() : make_float2(0.f, 0.f);
      const bool dead0 = kk > live || !w.ok, dead1 = kk > live || !w.ok1;
      float r[2][6];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float u = e ? uu.y : uu.x, z = e ? zz.y : zz.x;
        float dt = (e ? dd.y + bias.y : dd.x + bias.x), dy = e ? oo.y : oo.x, ds = 1.f, zf = 0.f;
        if (sp) {
          const float x = exp_neg_abs(dt);
          ds = __fdividef(dt >= 0.f ? 1.f : x, 1.f + x);
          dt = softplus_e(dt, x);
        }
        if (gate) {
          const float sg = sigmoid(z);
          zf = dy * sg * (1.f + z * (1.f - sg));
          dy *= z * sg;
        }
        // dead tokens, and channels that do not exist (they share the sums over channels)
        const bool dead = e ? dead1 : dead0;
        r[e][0] = dead ? 0.f : dt;
        r[e][1] = dead ? 0.f : dt * u;
        r[e][2] = dead ? 0.f : dy;
        r[e][3] = u;
        r[e][4] = ds;
        r[e][5] = zf;
      }
      if (Q::DUP == 1 || w.owner()) {
        sm.s1[w.warp][kk][w.c] = make_float4(r[0][0], r[1][0], r[0][1], r[1][1]);
        sm.s2[w.warp][kk][w.c] = make_float4(r[0][2], r[1][2], r[0][3], r[1][3]);
        sm.s3[w.warp][kk][w.c] = make_float4(r[0][4], r[1][4], r[0][5], r[1][5]);
      }
    }
  };
  if (k0 < kl) {
    fetch_bc(kl - 1);
    fetch_saved(kl - 1);
    put_copies<T, LPC>(sm.B, rB, N, last_of(kl - 1));
    put_copies<T, LPC>(sm.C, rC, N, last_of(kl - 1));
#pragma unroll 1
    for (int q = 0; q < NG; ++q) {
      fetch(kl - 1, q);
      stage(kl - 1, q);
    }
    __syncthreads();
  }
  const float4(*s1)[CPW] = sm.s1[w.warp];
  const float4(*s2)[CPW] = sm.s2[w.warp];
  for (int64_t k = kl - 1; k >= k0; --k) {
    const int64_t t0 = k * kTile;
    const int live = last_of(k);
    // states entering the tile's groups wait in shared memory
    F2 h[NS];
    {
      if constexpr (VEC) {
        rs0 = sm.next[0][threadIdx.x];
        rs1 = sm.next[1][threadIdx.x];
      }
      const float4 a = Perm<LPC>::apply(rs0, w.c), b = Perm<LPC>::apply(rs1, w.c);
      h[0] = f2(w.ok ? a.x : 0.f, w.ok1 ? b.x : 0.f);
      h[1] = f2(w.ok ? a.y : 0.f, w.ok1 ? b.y : 0.f);
      h[2] = f2(w.ok ? a.z : 0.f, w.ok1 ? b.z : 0.f);
      h[3] = f2(w.ok ? a.w : 0.f, w.ok1 ? b.w : 0.f);
    }
#pragma unroll 1
    for (int q = 0; q + 1 < NG; ++q) {
      *reinterpret_cast<ulonglong2*>(&sm.hs[q][0][threadIdx.x]) = make_ulonglong2(h[0], h[1]);
      *reinterpret_cast<ulonglong2*>(&sm.hs[q][1][threadIdx.x]) = make_ulonglong2(h[2], h[3]);
#pragma unroll
      for (int i = 0; i < kGroupB; ++i) {
        const int kk = q * kGroupB + i;
        const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(&s1[kk][w.c]);
        F2 Bn[NS];
        twice4(Bn, sm.B[kk][w.j][cq]);
#pragma unroll
        for (int m = 0; m < NS; ++m) h[m] = fma2(decay(s.x, A2[m]), h[m], mul2(s.y, Bn[m]));
      }
    }
    F2 tA[NS] = {0, 0, 0, 0};
    float2 tD = make_float2(0.f, 0.f), tb = make_float2(0.f, 0.f);
    const int rows = (int)min(p.L - t0, (int64_t)kTile);
#pragma unroll 1
    for (int q = NG - 1; q >= 0; --q) {
      if (k > k0) {
        if (q == 0) {
          fetch_bc(k - 1);
          fetch_saved(k - 1);  // goes with the group's copies
        }
        fetch(k - 1, q);
      }
      const int kq = q * kGroupB;
      if (q < NG - 1) {
        const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(&sm.hs[q][0][threadIdx.x]);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&sm.hs[q][1][threadIdx.x]);
        h[0] = a.x;
        h[1] = a.y;
        h[2] = b.x;
        h[3] = b.y;
      }
      // hh[i]: the state before token i, hh[i + 1] the one after it
      F2 a[kGroupB][NS], hh[kGroupB + 1][NS];
#pragma unroll
      for (int m = 0; m < NS; ++m) hh[0][m] = h[m];
#pragma unroll
      for (int i = 0; i < kGroupB; ++i) {
        const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(&s1[kq + i][w.c]);
        F2 Bn[NS];
        twice4(Bn, sm.B[kq + i][w.j][cq]);
#pragma unroll
        for (int m = 0; m < NS; ++m) {
          a[i][m] = decay(s.x, A2[m]);
          hh[i + 1][m] = fma2(a[i][m], hh[i][m], mul2(s.y, Bn[m]));
        }
      }
      float ysw[kGroupB][6];  // y, sum g B, sum A q of the pair, per token
#pragma unroll
      for (int i = kGroupB - 1; i >= 0; --i) {
        const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(&s1[kq + i][w.c]);
        const F2 dy = *reinterpret_cast<const F2*>(&s2[kq + i][w.c]);
        F2 Bn[NS], Cn[NS];
        twice4(Bn, sm.B[kq + i][w.j][cq]);
        twice4(Cn, sm.C[kq + i][w.j][cq]);
        F2 y = 0, ss = 0, ww = 0, db[NS], dc[NS];
#pragma unroll
        for (int m = 0; m < NS; ++m) {
          const F2 g = fma2(Cn[m], dy, cy[m]);
          cy[m] = mul2(a[i][m], g);
          const F2 qq = mul2(cy[m], hh[i][m]);  // g a h
          y = m ? fma2(Cn[m], hh[i + 1][m], y) : mul2(Cn[m], hh[i + 1][m]);
          ss = m ? fma2(Bn[m], g, ss) : mul2(Bn[m], g);
          ww = m ? fma2(A2[m], qq, ww) : mul2(A2[m], qq);
          tA[m] = fma2(s.x, qq, tA[m]);
          db[m] = mul2(g, s.y);
          dc[m] = mul2(dy, hh[i + 1][m]);
        }
        const float2 y2 = un2(y), s2v = un2(ss), w2 = un2(ww);
        ysw[i][0] = y2.x;
        ysw[i][1] = y2.y;
        ysw[i][2] = s2v.x;
        ysw[i][3] = s2v.y;
        ysw[i][4] = w2.x;
        ysw[i][5] = w2.y;
        channel_sums<LPC>(db, dc, sm.red[q / (NG / 2)][w.warp][(kq + i) % (kTile / 2)], w.c, w.j);
        if (LPC >= 2 && i % 2 == 0) halve<LPC>(ysw[i], ysw[i + 1], w.j, LPC / 2);
      }
      if (LPC >= 4) {
        halve<LPC>(ysw[0], ysw[2], w.j, LPC / 4);
#pragma unroll
        for (int bit = LPC / 8; bit > 0; bit >>= 1)
#pragma unroll
          for (int m = 0; m < 6; ++m) ysw[0][m] += __shfl_xor_sync(0xffffffffu, ysw[0][m], bit * CPW);
      }
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int kk = kq + group_token<LPC>(w.j, i);
        const float(&r)[6] = ysw[LPC == 2 ? 2 * i : i];
        const float4 v1 = s1[kk][w.c], v2 = s2[kk][w.c], v3 = sm.s3[w.warp][kk][w.c];
        float u0 = fmaf(v1.x, r[2], Dd.x * v2.x), u1 = fmaf(v1.y, r[3], Dd.y * v2.y);
        float d0 = fmaf(v2.z, r[2], kLn2 * r[4]) * v3.x, d1 = fmaf(v2.w, r[3], kLn2 * r[5]) * v3.y;
        float z0 = v3.z * fmaf(Dd.x, v2.z, r[0]), z1 = v3.w * fmaf(Dd.y, v2.w, r[1]);
        if (kk > live) {
          u0 = u1 = d0 = d1 = z0 = z1 = 0.f;
        } else {
          tD = make_float2(fmaf(v2.x, v2.z, tD.x), fmaf(v2.y, v2.w, tD.y));
          tb = make_float2(tb.x + d0, tb.y + d1);
        }
        if (store && kk < rows) {
          const int64_t o = (t0 + kk) * D;
          store_two<T, VEC>(du + o, u0, u1, w.ok1);
          store_two<T, VEC>(ddelta + o, d0, d1, w.ok1);
          if (gate) store_two<T, VEC>(dz + o, z0, z1, w.ok1);
        }
      }
      if (k > k0) {
        __syncwarp();  // the group's slots are free
        stage(k - 1, q);
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
    if (k > k0) {  // every warp is past its last use of this tile's B and C
      put_copies<T, LPC>(sm.B, rB, N, last_of(k - 1));
      put_copies<T, LPC>(sm.C, rC, N, last_of(k - 1));
      __syncthreads();
    }
    // The sums over a sequence cancel heavily (terms of both signs): a tile's
    // 16 terms are added as they are, the tiles' sums with what each addition
    // lost kept beside them.
#pragma unroll
    for (int m = 0; m < NS; m += 2) {
      ulonglong2* v = reinterpret_cast<ulonglong2*>(&sm.sumA[m / 2][0][threadIdx.x]);
      ulonglong2* lost = reinterpret_cast<ulonglong2*>(&sm.sumA[m / 2][1][threadIdx.x]);
      ulonglong2 sum = *v, l = *lost;
      add_kept(sum.x, l.x, tA[m]);
      add_kept(sum.y, l.y, tA[m + 1]);
      *v = sum;
      *lost = l;
    }
    add_kept(sumD, lostD, f2(tD.x, tD.y));
    add_kept(sumb, lostb, f2(tb.x, tb.y));
  }
  float2 endD = un2(add2(sumD, lostD)), endb = un2(add2(sumb, lostb));
  if (!w.owner()) endD = endb = make_float2(0.f, 0.f);
  const int64_t row = blockIdx.y * p.B + w.b;
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int n = w.j * NS + (i ^ cq);
    const F2* sum = reinterpret_cast<const F2*>(&sm.sumA[i / 2][0][threadIdx.x]);
    const F2* lost = reinterpret_cast<const F2*>(&sm.sumA[i / 2][1][threadIdx.x]);
    w.put_state(sc.dA, row * p.D + w.d, NP, n, add2(sum[i % 2], lost[i % 2]));
    if (p.dinit && blockIdx.y == 0) w.put_state(p.dinit, cell, p.N, n, cy[i]);
  }
#pragma unroll
  for (int o = CPW; o < 32; o <<= 1) {
    endD.x += __shfl_xor_sync(0xffffffffu, endD.x, o);
    endD.y += __shfl_xor_sync(0xffffffffu, endD.y, o);
    endb.x += __shfl_xor_sync(0xffffffffu, endb.x, o);
    endb.y += __shfl_xor_sync(0xffffffffu, endb.y, o);
  }
  if (w.j == 0) {
    float* v = sc.dv + row * 2 * p.D + w.d;
    if (w.ok) {
      v[0] = endD.x;
      v[p.D] = endb.x;
    }
    if (w.ok1) {
      v[1] = endD.y;
      v[p.D + 1] = endb.y;
    }
  }
}

// The partial rows added up, in one launch: CTAs below bc_ctas take dB and dC
// [B, L, G, N] (over channel blocks), the others dA, dD and dbias (over
// sequences and segments).
template <typename T>
__global__ void __launch_bounds__(256) reduce_kernel(const mogt_selective_args p, int64_t nblk, int NP, int64_t rows,
                                                     int64_t bc_ctas, const BwdScratch sc) {
  if ((int64_t)blockIdx.x < bc_ctas) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t total = p.B * p.L * p.G * 2 * p.N;
    if (i >= total) return;
    const int64_t n = i % p.N, which = (i / p.N) % 2, g = (i / (2 * p.N)) % p.G, bt = i / (2 * p.N * p.G);
    const int64_t t = bt % p.L, b = bt / p.L;
    float v = 0.f;
    if (t < seq_len(p.lengths, b, p.L)) {
      const float* src = sc.bc + ((b * p.G + g) * p.L + t) * (2 * NP) + which * NP + n;
      const int64_t stride = p.B * p.G * p.L * 2 * NP;
#pragma unroll 8
      for (int64_t k = 0; k < nblk; ++k) v += src[k * stride];
    }
    T* dst = static_cast<T*>(which ? p.dC : p.dB);
    dst[(bt * p.G + g) * p.N + n] = from_f32<T>(v);
    return;
  }
  const int64_t i = ((int64_t)blockIdx.x - bc_ctas) * 256 + threadIdx.x;
  const int64_t na = p.D * p.N;
  if (i < na) {
    const int64_t d = i / p.N, n = i % p.N;
    double v = 0.0;
#pragma unroll 8
    for (int64_t r = 0; r < rows; ++r) v += sc.dA[(r * p.D + d) * NP + n];
    p.dA[i] = (float)v;
  } else if (i < na + 2 * p.D) {
    const int64_t k = i - na;
    double v = 0.0;
#pragma unroll 8
    for (int64_t r = 0; r < rows; ++r) v += sc.dv[r * 2 * p.D + k];
    float* dst = k < p.D ? p.dD : p.dbias;
    if (dst) dst[k % p.D] = (float)v;
  }
}

inline size_t bwd_floats(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G, int64_t nseg) {
  const int64_t np = lpc_of(N) * NS, cpb = channels_per_cta(NTB, lpc_of(N));
  const int64_t seg = (int64_t)(seg_scratch_bytes(B, D, N, nseg) / sizeof(float) + 3) / 4 * 4;
  return (size_t)(seg + (D / G + cpb - 1) / cpb * B * G * L * 2 * np + nseg * B * D * (np + 2));
}

}  // namespace sel
}  // namespace mogt

using namespace mogt;
using namespace mogt::sel;

extern "C" size_t mogt_selective_bwd_scratch_bytes(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G) {
  if (B <= 0 || L < 0 || D <= 0 || N <= 0 || N > kMaxN || G <= 0 || D % G) return 0;
  return bwd_floats(B, L, D, N, G, bwd_segments(B, L, D, N, G)) * sizeof(float);
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
  const Geo geo = geometry(p, NTB, bwd_segments(p.B, p.L, p.D, p.N, p.G));
  const int NP = lpc_of(p.N) * NS;
  BwdScratch sc;
  sc.seg = seg_scratch(p.scratch, p.B, p.D, p.N, geo.nseg);
  sc.dA = static_cast<float*>(p.scratch) + (seg_scratch_bytes(p.B, p.D, p.N, geo.nseg) / sizeof(float) + 3) / 4 * 4;
  sc.dv = sc.dA + geo.nseg * p.B * p.D * NP;
  sc.bc = sc.dv + geo.nseg * p.B * 2 * p.D;
  cudaStream_t s = (cudaStream_t)stream;
  const bool vec = pairs_aligned(p, true);
  static_assert(NT == NTB, "the first pass takes the main pass's channel blocks");
  return dispatch(p.dtype, p.N, [&](auto t, auto l) {
    using T = decltype(t);
    constexpr int LPC = decltype(l)::value;
    auto go = [&](auto kern, int bytes, int nseg, const auto& scratch) {
      if (bytes > 48 * 1024 &&
          cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
        return false;
      kern<<<dim3((unsigned)(geo.nblk * p.G), nseg, (unsigned)p.B), NTB, bytes, s>>>(p, geo, scratch);
      return true;
    };
    bool ok = true;
    if (geo.nseg > 1)
      ok = vec ? go(scan_bwd_agg_kernel<T, LPC, true>, (int)sizeof(AggSmem<LPC>), geo.nseg - 1, sc.seg)
               : go(scan_bwd_agg_kernel<T, LPC, false>, (int)sizeof(AggSmem<LPC>), geo.nseg - 1, sc.seg);
    constexpr int bytes = (int)sizeof(BwdSmem<LPC>);
    ok = ok && (vec ? go(scan_bwd_kernel<T, LPC, true>, bytes, geo.nseg, sc)
                    : go(scan_bwd_kernel<T, LPC, false>, bytes, geo.nseg, sc));
    if (!ok) return (int)MOGT_ERR_LAUNCH;
    const int64_t bc = (p.B * p.L * p.G * 2 * p.N + 255) / 256, par = (p.D * p.N + 2 * p.D + 255) / 256;
    if (bc + par >= ((int64_t)1 << 31)) return (int)MOGT_ERR_UNSUPPORTED;
    reduce_kernel<T><<<(unsigned)(bc + par), 256, 0, s>>>(p, geo.nblk, NP, geo.nseg * p.B, bc, sc);
    return mogt_host::launch_status();
  });
}
