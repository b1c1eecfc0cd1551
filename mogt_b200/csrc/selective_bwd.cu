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
// tiles backwards; in a tile the first 8 tokens are stepped to get the state
// in the middle, then each half is stepped again with a_t and a_t h_{t-1} of
// its 8 tokens kept in registers, and walked backwards.  Lanes are those of
// the forward (4 states each, LPC lanes per channel).  dB and dC need sums
// over all channels: over the warp's by a halving butterfly that leaves each
// lane one token, over the CTA's warps through shared memory, over CTAs by a
// second kernel that adds the partial rows in a fixed order.  About 25
// instructions per (token, channel, state), so instruction issue bounds it.
#include "selective_scan.cuh"

namespace mogt {
namespace sel {

struct BwdScratch {
  float* bc;   // [nblk][B][G][L][2][NP]
  float* dA;   // [B][D][NP]
  float* dv;   // [B][2][D]: dD, dbias
};

template <int LPC>
struct BwdSmem {
  float B[kTile][Lane<LPC>::NP], C[kTile][Lane<LPC>::NP];
  float4 stage[NTB / 32][kTile][Lane<LPC>::CPW];
  float red[NTB / 32][kGroup][2][Lane<LPC>::NP];
};

template <typename T, int LPC>
__global__ void __launch_bounds__(NTB) scan_bwd_kernel(const mogt_selective_args p, const Geo geo,
                                                       const BwdScratch sc) {
  using Q = Lane<LPC>;
  constexpr int CPW = Q::CPW, TPL = Q::TPL, NP = Q::NP;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  BwdSmem<LPC>& sm = *reinterpret_cast<BwdSmem<LPC>*>(smem_raw);
  const Where<LPC> w(p, geo);
  const int64_t len = seq_len(p.lengths, w.b, p.L);

  float A2[NS], carry[NS], accA[NS];
  load_A<LPC>(A2, p, w);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int n = w.j * NS + i;
    carry[i] = (p.dfinal && w.ok && n < p.N) ? p.dfinal[(w.b * p.D + w.d) * p.N + n] : 0.f;
    accA[i] = 0.f;
  }
  const float Dd = p.Dskip && w.ok ? p.Dskip[w.d] : 0.f;
  const float bias = p.bias && w.ok ? p.bias[w.d] : 0.f;
  float accD = 0.f, accb = 0.f;
  const float4* saved = reinterpret_cast<const float4*>(p.saved);
  T* du = static_cast<T*>(p.du) + w.b * p.L * p.D + w.d;
  T* ddelta = static_cast<T*>(p.ddelta) + w.b * p.L * p.D + w.d;
  T* dz = p.z ? static_cast<T*>(p.dz) + w.b * p.L * p.D + w.d : nullptr;

  for (int64_t tile = geo.nck - 1; tile >= 0; --tile) {
    const int64_t t0 = tile * kTile;
    if (t0 >= len) {
      for (int k = w.part_tok(); k < kTile; k += kGroup)
#pragma unroll
        for (int i = 0; i < TPL; ++i) {
          const int64_t t = t0 + k + i;
          if (w.ok && w.owner() && t < p.L) {
            du[t * p.D] = from_f32<T>(0.f);
            ddelta[t * p.D] = from_f32<T>(0.f);
            if (dz) dz[t * p.D] = from_f32<T>(0.f);
          }
        }
      continue;
    }
    __syncthreads();
    load_bc<T, NP>(sm.B, p, w, static_cast<const T*>(p.Bm), p.B_sb, p.B_sl, p.B_sg, t0, len);
    load_bc<T, NP>(sm.C, p, w, static_cast<const T*>(p.Cm), p.C_sb, p.C_sl, p.C_sg, t0, len);
    float u[2][TPL], raw[2][TPL], z[2][TPL], go[2][TPL];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int64_t t = t0 + q * kGroup + w.part_tok() + i;
        float dt = 0.f;
        u[q][i] = raw[q][i] = z[q][i] = go[q][i] = 0.f;
        if (w.ok && t < len) {
          u[q][i] = to_f32(static_cast<const T*>(p.u)[w.b * p.u_sb + t * p.u_sl + w.d]);
          raw[q][i] = dt = to_f32(static_cast<const T*>(p.delta)[w.b * p.delta_sb + t * p.delta_sl + w.d]) + bias;
          if (p.softplus) dt = softplus(dt);
          go[q][i] = to_f32(static_cast<const T*>(p.dout)[w.b * p.dout_sb + t * p.dout_sl + w.d]);
          if (p.z) z[q][i] = to_f32(static_cast<const T*>(p.z)[w.b * p.z_sb + t * p.z_sl + w.d]);
        }
        const float dy = p.z ? go[q][i] * z[q][i] * sigmoid(z[q][i]) : go[q][i];
        if (w.owner())
          sm.stage[w.warp][q * kGroup + w.part_tok() + i][w.c] = make_float4(dt, dt * u[q][i], dy, 0.f);
      }
    __syncthreads();
    float h0[NS], hm[NS];
    {
      const float4 v = w.ok ? saved[((w.b * geo.nck + tile) * p.D + w.d) * LPC + w.j] : make_float4(0, 0, 0, 0);
      h0[0] = v.x; h0[1] = v.y; h0[2] = v.z; h0[3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) hm[i] = h0[i];
    if (t0 + kGroup < len) {
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        const float4 s = sm.stage[w.warp][k][w.c];
#pragma unroll
        for (int i = 0; i < NS; ++i)
          hm[i] = fmaf(fast_exp2(s.x * A2[i]), hm[i], s.y * sm.B[k][w.j * NS + i]);
      }
    }
#pragma unroll 1
    for (int q = 1; q >= 0; --q) {
      float a[kGroup][NS], ph[kGroup][NS], h[NS];
#pragma unroll
      for (int i = 0; i < NS; ++i) h[i] = q ? hm[i] : h0[i];
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        const float4 s = sm.stage[w.warp][q * kGroup + k][w.c];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          a[k][i] = fast_exp2(s.x * A2[i]);
          ph[k][i] = a[k][i] * h[i];
          h[i] = fmaf(s.y, sm.B[q * kGroup + k][w.j * NS + i], ph[k][i]);
        }
      }
      float ysw[kGroup][3], bc[kGroup][2 * NS];
#pragma unroll
      for (int k = kGroup - 1; k >= 0; --k) {
        const float4 s = sm.stage[w.warp][q * kGroup + k][w.c];
        float y = 0.f, ss = 0.f, ww = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          const float Bn = sm.B[q * kGroup + k][w.j * NS + i], Cn = sm.C[q * kGroup + k][w.j * NS + i];
          const float hk = fmaf(s.y, Bn, ph[k][i]);
          const float g = fmaf(Cn, s.z, carry[i]);
          y = fmaf(Cn, hk, y);
          bc[k][i] = g * s.y;
          bc[k][NS + i] = s.z * hk;
          ss = fmaf(g, Bn, ss);
          const float qq = g * ph[k][i];
          ww = fmaf(A2[i], qq, ww);
          accA[i] = fmaf(s.x, qq, accA[i]);
          carry[i] = a[k][i] * g;
        }
        ysw[k][0] = y;
        ysw[k][1] = ss;
        ysw[k][2] = ww;
      }
      sum_parts<LPC, 3>(ysw, w.j);
      sum_channels<CPW, 2 * NS>(bc, w.c);
      using CT = ChanTok<CPW>;
      if (CT::owner(w.c)) {
#pragma unroll
        for (int i = 0; i < CT::TPL; ++i) {
          float(*r)[NP] = sm.red[w.warp][CT::first(w.c) + i];
          *reinterpret_cast<float4*>(&r[0][w.j * NS]) = make_float4(bc[i][0], bc[i][1], bc[i][2], bc[i][3]);
          *reinterpret_cast<float4*>(&r[1][w.j * NS]) = make_float4(bc[i][4], bc[i][5], bc[i][6], bc[i][7]);
        }
      }
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int kk = w.part_tok() + i;
        const int64_t t = t0 + q * kGroup + kk;
        const float uu = q ? u[1][i] : u[0][i], rr = q ? raw[1][i] : raw[0][i];
        const float zz = q ? z[1][i] : z[0][i], gg = q ? go[1][i] : go[0][i];
        const float4 s = sm.stage[w.warp][q * kGroup + kk][w.c];
        const float gu = fmaf(s.x, ysw[i][1], Dd * s.z);
        float gd = fmaf(uu, ysw[i][1], kLn2 * ysw[i][2]);
        if (p.softplus) gd *= sigmoid(rr);
        if (w.ok && w.owner() && t < p.L) {
          const bool live = t < len;
          du[t * p.D] = from_f32<T>(live ? gu : 0.f);
          ddelta[t * p.D] = from_f32<T>(live ? gd : 0.f);
          if (dz) {
            const float sg = sigmoid(zz), yt = fmaf(Dd, uu, ysw[i][0]);
            dz[t * p.D] = from_f32<T>(live ? gg * yt * sg * (1.f + zz * (1.f - sg)) : 0.f);
          }
          if (live) {
            accD = fmaf(s.z, uu, accD);
            accb += gd;
          }
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < kGroup * 2 * NP; i += NTB) {
        float v = 0.f;
#pragma unroll
        for (int ww = 0; ww < NTB / 32; ++ww) v += (&sm.red[ww][0][0][0])[i];
        const int64_t t = t0 + q * kGroup + i / (2 * NP);
        if (t < len)
          sc.bc[((((blockIdx.x % geo.nblk) * p.B + w.b) * p.G + w.g) * p.L + t) * (2 * NP) + i % (2 * NP)] = v;
      }
      __syncthreads();
    }
  }
  if (w.ok) {
    *reinterpret_cast<float4*>(sc.dA + ((w.b * p.D + w.d) * LPC + w.j) * NS) =
        make_float4(accA[0], accA[1], accA[2], accA[3]);
    if (p.dinit) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int n = w.j * NS + i;
        if (n < p.N) p.dinit[(w.b * p.D + w.d) * p.N + n] = carry[i];
      }
    }
  }
#pragma unroll
  for (int o = CPW; o < 32; o <<= 1) {
    accD += __shfl_xor_sync(0xffffffffu, accD, o);
    accb += __shfl_xor_sync(0xffffffffu, accb, o);
  }
  if (w.ok && w.j == 0) {
    sc.dv[(w.b * 2 + 0) * p.D + w.d] = accD;
    sc.dv[(w.b * 2 + 1) * p.D + w.d] = accb;
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

// dA, dD, dbias from the per-sequence partial sums.
__global__ void __launch_bounds__(256) reduce_param_kernel(const mogt_selective_args p, int NP, int64_t rows,
                                                           const BwdScratch sc) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t na = p.D * p.N;
  if (i < na) {
    const int64_t d = i / p.N, n = i % p.N;
    float v = 0.f;
    for (int64_t r = 0; r < rows; ++r) v += sc.dA[(r * p.D + d) * NP + n];
    p.dA[i] = v;
  } else if (i < na + 2 * p.D) {
    const int64_t k = i - na;
    float v = 0.f;
    for (int64_t r = 0; r < rows; ++r) v += sc.dv[r * 2 * p.D + k];
    float* dst = k < p.D ? p.dD : p.dbias;
    if (dst) dst[k % p.D] = v;
  }
}

inline int64_t bc_floats(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G) {
  const int64_t cpb = NTB / lpc_of(N);
  return (D / G + cpb - 1) / cpb * B * G * L * 2 * lpc_of(N) * NS;
}

}  // namespace sel
}  // namespace mogt

using namespace mogt;
using namespace mogt::sel;

extern "C" size_t mogt_selective_bwd_scratch_bytes(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G) {
  if (B <= 0 || L < 0 || D <= 0 || N <= 0 || N > kMaxN || G <= 0 || D % G) return 0;
  return (size_t)(bc_floats(B, L, D, N, G) + B * D * (lpc_of(N) * NS + 2)) * sizeof(float);
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
  const Geo geo = geometry(p, NTB);
  const int NP = lpc_of(p.N) * NS;
  BwdScratch sc;
  sc.dA = static_cast<float*>(p.scratch);
  sc.dv = sc.dA + p.B * p.D * NP;
  sc.bc = sc.dv + 2 * p.B * p.D;
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid((unsigned)(geo.nblk * p.G), 1, (unsigned)p.B);
  return dispatch(p.dtype, p.N, [&](auto t, auto l) {
    using T = decltype(t);
    constexpr int LPC = decltype(l)::value;
    constexpr int bytes = (int)sizeof(BwdSmem<LPC>);
    auto kern = scan_bwd_kernel<T, LPC>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return (int)MOGT_ERR_LAUNCH;
    kern<<<grid, NTB, bytes, s>>>(p, geo, sc);
    const int64_t nbc = p.B * p.L * p.G * 2 * p.N;
    if (nbc > 0) reduce_bc_kernel<T><<<(unsigned)((nbc + 255) / 256), 256, 0, s>>>(p, geo.nblk, NP, sc.bc);
    const int64_t np = p.D * p.N + 2 * p.D;
    reduce_param_kernel<<<(unsigned)((np + 255) / 256), 256, 0, s>>>(p, NP, p.B, sc);
    return mogt_host::launch_status();
  });
}
