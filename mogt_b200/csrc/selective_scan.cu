// Selective state space scan, forward and single token.  Per channel d and
// state n (group g = d / (D / G)):
//   h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t,   y_t = sum_n C_t h_t + D u_t,
//   out_t = y_t silu(z_t).
// One exponential and four multiply-adds per (token, channel, state) against
// 8 bytes per (token, channel) in bf16: at N = 16 the exponentials (16 a clock
// and SM) bound it, not HBM.
//
// A thread keeps NS = 4 states of one channel in registers; LPC = N / 4
// (rounded up to a power of two) lanes share a channel, so a warp holds
// 32 / LPC channels.  Lane = channel + CPW * part.  Tokens come in groups of
// 8: the LPC lanes of a channel split the group's tokens for what is done once
// per (token, channel) (softplus, gate, loads, stores), hand (dt, dt u) to one
// another through shared memory, and sum y over the parts with a butterfly
// that leaves each lane the tokens it loaded.
#include "selective_scan.cuh"

namespace mogt {
namespace sel {

#ifndef MOGT_FWD_WARPS
#define MOGT_FWD_WARPS 16
#endif
#ifndef MOGT_FWD_CTAS
#define MOGT_FWD_CTAS 4
#endif
constexpr int kFwdWarps = MOGT_FWD_WARPS;  // warps per SM that the forward asks for

// grid = (channel blocks, segments, B).  AGG: the first pass over a split
// sequence, which leaves each segment's state from zero and its sum of dt.
template <typename T, int LPC, bool AGG>
__global__ void __launch_bounds__(NT, LPC < 4 ? 3 : MOGT_FWD_CTAS) scan_fwd_kernel(const mogt_selective_args p, const Geo geo,
                                                                     const SegScratch seg) {
  using Q = Lane<LPC>;
  constexpr int CPW = Q::CPW, TPL = Q::TPL, NP = Q::NP;
  __shared__ __align__(16) float sB[2][kTile][NP], sC[AGG ? 1 : 2][AGG ? 1 : kTile][NP];
  __shared__ float2 stage[NT / 32][kTile][CPW];  // (dt, x)
  const Where<LPC> w(p, geo);
  const int64_t len = seq_len(p.lengths, w.b, p.L);
  const int64_t k0 = (int64_t)blockIdx.y * geo.tps, k1 = min(k0 + geo.tps, geo.nck);
  const int64_t kl = min(k1, (len + kTile - 1) / kTile);  // first tile without a live token
  const int64_t cell = w.b * p.D + w.d;

  float A2[NS];
  load_A<LPC>(A2, p, w);
  const F2 A01 = f2(A2[0], A2[1]), A23 = f2(A2[2], A2[3]);
  F2 h01 = 0, h23 = 0;
  if (!AGG) {
    float h[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int n = w.j * NS + i;
      h[i] = (p.init && w.ok && n < p.N) ? p.init[cell * p.N + n] : 0.f;
    }
#pragma unroll 4
    for (int s = 0; s < (int)blockIdx.y; ++s) {
      const float4 l = seg.loc[(s * p.B * p.D + cell) * LPC + w.j];
      const float sd = seg.sdt[s * p.B * p.D + cell];
      h[0] = fmaf(fast_exp2(sd * A2[0]), h[0], l.x);
      h[1] = fmaf(fast_exp2(sd * A2[1]), h[1], l.y);
      h[2] = fmaf(fast_exp2(sd * A2[2]), h[2], l.z);
      h[3] = fmaf(fast_exp2(sd * A2[3]), h[3], l.w);
    }
    h01 = f2(h[0], h[1]);
    h23 = f2(h[2], h[3]);
  }
  const float Dd = !AGG && p.Dskip ? p.Dskip[w.d] : 0.f;
  const float bias = p.bias ? p.bias[w.d] : 0.f;
  const bool gate = !AGG && p.z, sp = p.softplus, store = w.ok && w.owner();
  const int tok = w.part_tok(), N = (int)p.N, D = (int)p.D;
  const int u_sl = (int)p.u_sl, d_sl = (int)p.delta_sl, z_sl = (int)p.z_sl, B_sl = (int)p.B_sl, C_sl = (int)p.C_sl;
  const T* up = static_cast<const T*>(p.u) + w.b * p.u_sb + k0 * kTile * p.u_sl + w.d;
  const T* dp = static_cast<const T*>(p.delta) + w.b * p.delta_sb + k0 * kTile * p.delta_sl + w.d;
  const T* zp = gate ? static_cast<const T*>(p.z) + w.b * p.z_sb + k0 * kTile * p.z_sl + w.d : nullptr;
  const T* Bp = static_cast<const T*>(p.Bm) + w.b * p.B_sb + w.g * p.B_sg + k0 * kTile * p.B_sl;
  const T* Cp = static_cast<const T*>(p.Cm) + w.b * p.C_sb + w.g * p.C_sg + k0 * kTile * p.C_sl;
  T* out = static_cast<T*>(p.out) + (w.b * p.L + k0 * kTile) * p.D + w.d;
  float4* saved = AGG || !p.saved || !w.ok
                      ? nullptr
                      : reinterpret_cast<float4*>(p.saved) + ((w.b * geo.nck + k0) * p.D + w.d) * LPC + w.j;

  TileRaw<T, TPL, kGroup> ru, rd, rz;
  BcRaw<T, NP, NT> rB, rC;
  float sdt = 0.f;
  int last = 0;  // last live token of the fetched tile
  auto fetch = [&](int64_t k) {
    last = (int)min(len - 1 - k * kTile, (int64_t)(kTile - 1));
    rB.fetch(Bp, B_sl, N, last);
    Bp += (int64_t)kTile * B_sl;
    rd.fetch(dp, d_sl, tok, last);
    dp += (int64_t)kTile * d_sl;
    ru.fetch(up, u_sl, tok, last);
    up += (int64_t)kTile * u_sl;
    if (!AGG) {
      rC.fetch(Cp, C_sl, N, last);
      Cp += (int64_t)kTile * C_sl;
      if (gate) {
        rz.fetch(zp, z_sl, tok, last);
        zp += (int64_t)kTile * z_sl;
      }
    }
  };
  if (k0 < kl) fetch(k0);
  for (int64_t k = k0; k < kl; ++k) {
    const int buf = (int)(k & 1), live = last;
    if (saved) {
      const float2 a = un2(h01), b = un2(h23);
      *saved = make_float4(a.x, a.y, b.x, b.y);
      saved += (int64_t)D * LPC;
    }
    rB.put(sB[buf], N, live);
    if (!AGG) rC.put(sC[buf], N, live);
    float u[2][TPL], gz[2][TPL];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int kk = q * kGroup + tok + i;
        u[q][i] = to_f32(ru.v[q][i]);
        float dt = to_f32(rd.v[q][i]) + bias;
        if (sp) dt = softplus(dt);
        float x = dt * u[q][i];
        if (kk > live) dt = x = 0.f;
        if (Q::DUP == 1 || w.owner()) stage[w.warp][kk][w.c] = make_float2(dt, x);
        if (gate) {
          const float z = to_f32(rz.v[q][i]);
          gz[q][i] = z * sigmoid(z);
        }
      }
    __syncthreads();
    if (k + 1 < kl) fetch(k + 1);
    float sd = 0.f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float y[kGroup][1];
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const int kk = q * kGroup + i;
        const float2 dx = stage[w.warp][kk][w.c];
        const F2 dt2 = f2(dx.x, dx.x), x2 = f2(dx.y, dx.y);
        const ulonglong2 Bv = *reinterpret_cast<const ulonglong2*>(&sB[buf][kk][w.j * NS]);
        h01 = fma2(exp2_2(mul2(dt2, A01)), h01, mul2(x2, Bv.x));
        h23 = fma2(exp2_2(mul2(dt2, A23)), h23, mul2(x2, Bv.y));
        if (AGG) {
          sd += dx.x;
        } else {
          const ulonglong2 Cv = *reinterpret_cast<const ulonglong2*>(&sC[AGG ? 0 : buf][AGG ? 0 : kk][w.j * NS]);
          y[i][0] = hsum(fma2(Cv.y, h23, mul2(Cv.x, h01)));
        }
      }
      if (!AGG) {
        sum_parts<LPC>(y, w.j);
        const int rows = (int)min(p.L - k * kTile, (int64_t)kTile);
#pragma unroll
        for (int i = 0; i < TPL; ++i) {
          const int kk = q * kGroup + tok + i;
          float o = fmaf(Dd, u[q][i], y[i][0]);
          if (gate) o *= gz[q][i];
          if (kk > live) o = 0.f;
          if (store && kk < rows) out[(int64_t)kk * D] = from_f32<T>(o);
        }
      }
    }
    out += (int64_t)kTile * D;
    sdt += sd;
    __syncwarp();  // the stage is rewritten for the next tile
  }
  if constexpr (AGG) {
    if (w.ok) {
      const float2 a = un2(h01), b = un2(h23);
      const int64_t i = blockIdx.y * p.B * p.D + cell;
      seg.loc[i * LPC + w.j] = make_float4(a.x, a.y, b.x, b.y);
      if (w.j == 0) seg.sdt[i] = sdt;
    }
  } else {
    // tiles behind the end
    for (int64_t t = max(kl, k0) * kTile + tok; t < min(k1 * kTile, p.L); t += kGroup)
#pragma unroll
      for (int i = 0; i < TPL; ++i)
        if (store && t + i < p.L) static_cast<T*>(p.out)[(w.b * p.L + t + i) * p.D + w.d] = from_f32<T>(0.f);
    if (p.final_state && w.ok && (int)blockIdx.y == geo.nseg - 1) {
      const float2 a = un2(h01), b = un2(h23);
      const float h[NS] = {a.x, a.y, b.x, b.y};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int n = w.j * NS + i;
        if (n < p.N) p.final_state[cell * p.N + n] = h[i];
      }
    }
  }
}

// One token: a thread per 4 states of a channel, the channel's lanes adjacent
// (a warp reads 512 consecutive bytes of the state when N is a multiple of 4).
template <typename T, int LPC, bool V4>
__global__ void __launch_bounds__(NT) step_kernel(const float* state, float* new_state, const T* u, int64_t u_sb,
                                                  const T* delta, int64_t delta_sb, const T* z, int64_t z_sb,
                                                  const T* Bm, int64_t B_sb, int64_t B_sg, const T* Cm, int64_t C_sb,
                                                  int64_t C_sg, const float* A, const float* Dskip, const float* bias,
                                                  T* y, int64_t B, int64_t D, int N, int64_t Dg, int sp) {
  const int64_t i0 = (int64_t)blockIdx.x * NT + threadIdx.x;
  const int j = (int)(i0 % LPC);
  const int64_t c = i0 / LPC;
  const bool ok = c < B * D;
  const int64_t b = ok ? c / D : 0, d = ok ? c % D : 0, g = d / Dg;
  const float uu = to_f32(u[b * u_sb + d]);
  float dt = to_f32(delta[b * delta_sb + d]) + (bias ? bias[d] : 0.f);
  if (sp) dt = softplus(dt);
  const float x = dt * uu;
  const int64_t so = (b * D + d) * N + j * NS;
  const float* Ap = A + d * N + j * NS;
  const T* Bp = Bm + b * B_sb + g * B_sg + j * NS;
  const T* Cp = Cm + b * C_sb + g * C_sg + j * NS;
  float h[NS], a[NS], s = 0.f;
  if constexpr (V4) {
    const bool in = j * NS < N;
    const float4 hv = in ? *reinterpret_cast<const float4*>(state + so) : make_float4(0, 0, 0, 0);
    const float4 av = in ? *reinterpret_cast<const float4*>(Ap) : make_float4(0, 0, 0, 0);
    h[0] = hv.x; h[1] = hv.y; h[2] = hv.z; h[3] = hv.w;
    a[0] = av.x; a[1] = av.y; a[2] = av.z; a[3] = av.w;
  } else {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const bool in = j * NS + i < N;
      h[i] = in ? state[so + i] : 0.f;
      a[i] = in ? Ap[i] : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const bool in = j * NS + i < N;
    const float Bn = in ? to_f32(Bp[i]) : 0.f, Cn = in ? to_f32(Cp[i]) : 0.f;
    h[i] = fmaf(fast_exp2(dt * (a[i] * kLog2e)), h[i], x * Bn);
    s = fmaf(Cn, h[i], s);
  }
#pragma unroll
  for (int o = 1; o < LPC; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (!ok) return;
  if constexpr (V4) {
    if (j * NS < N) *reinterpret_cast<float4*>(new_state + so) = make_float4(h[0], h[1], h[2], h[3]);
  } else {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (j * NS + i < N) new_state[so + i] = h[i];
  }
  if (j == 0) {
    float o = fmaf(Dskip ? Dskip[d] : 0.f, uu, s);
    if (z) {
      const float zz = to_f32(z[b * z_sb + d]);
      o *= zz * sigmoid(zz);
    }
    y[b * D + d] = from_f32<T>(o);
  }
}

}  // namespace sel
}  // namespace mogt

using namespace mogt;
using namespace mogt::sel;

extern "C" size_t mogt_selective_saved_bytes(int64_t B, int64_t L, int64_t D, int64_t N) {
  if (B <= 0 || L <= 0 || D <= 0 || N <= 0 || N > kMaxN) return 0;
  return (size_t)(B * ((L + kTile - 1) / kTile) * D * lpc_of(N) * NS) * sizeof(float);
}

extern "C" size_t mogt_selective_fwd_scratch_bytes(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G) {
  if (B <= 0 || L < 0 || D <= 0 || N <= 0 || N > kMaxN || G <= 0 || D % G) return 0;
  return seg_scratch_bytes(B, D, N, num_segments(B, L, D, N, G, NT, kFwdWarps));
}

extern "C" int mogt_selective_scan_fwd(const mogt_selective_args* args, void* stream) {
  if (!args) return MOGT_ERR_ARG;
  const mogt_selective_args& p = *args;
  if (int st = check_args(p)) return st;
  if (p.B == 0 || p.D == 0) return MOGT_OK;
  if (!p.A || (p.L > 0 && (!p.u || !p.delta || !p.Bm || !p.Cm || !p.out))) return MOGT_ERR_ARG;
  const Geo geo = geometry(p, NT, kFwdWarps);
  const size_t need = seg_scratch_bytes(p.B, p.D, p.N, geo.nseg);
  if (need && (!p.scratch || p.scratch_bytes < need)) return MOGT_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(p.saved) | (need ? reinterpret_cast<uintptr_t>(p.scratch) : 0)) & 15u)
    return MOGT_ERR_ALIGN;
  const SegScratch seg = seg_scratch(p.scratch, p.B, p.D, p.N, geo.nseg);
  cudaStream_t s = (cudaStream_t)stream;
  return dispatch(p.dtype, p.N, [&](auto t, auto l) {
    using T = decltype(t);
    constexpr int LPC = decltype(l)::value;
    const unsigned gx = (unsigned)(geo.nblk * p.G);
    if (geo.nseg > 1)
      scan_fwd_kernel<T, LPC, true><<<dim3(gx, geo.nseg - 1, (unsigned)p.B), NT, 0, s>>>(p, geo, seg);
    scan_fwd_kernel<T, LPC, false><<<dim3(gx, geo.nseg, (unsigned)p.B), NT, 0, s>>>(p, geo, seg);
    return mogt_host::launch_status();
  });
}

extern "C" int mogt_selective_step(const float* state, float* new_state, const void* u, int64_t u_sb,
                                   const void* delta, int64_t delta_sb, const void* z, int64_t z_sb, const void* Bm,
                                   int64_t B_sb, int64_t B_sg, const void* Cm, int64_t C_sb, int64_t C_sg,
                                   const float* A, const float* Dskip, const float* bias, void* y, int64_t B,
                                   int64_t D, int64_t N, int64_t G, int softplus, int dtype, void* stream) {
  if (B < 0 || D < 0 || N <= 0 || G <= 0 || D % G) return MOGT_ERR_SHAPE;
  if (N > kMaxN) return MOGT_ERR_UNSUPPORTED;
  if (B == 0 || D == 0) return MOGT_OK;
  if (!state || !new_state || !u || !delta || !Bm || !Cm || !A || !y) return MOGT_ERR_ARG;
  const bool v4 = N % 4 == 0 && ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(new_state) |
                                  reinterpret_cast<uintptr_t>(A)) & 15u) == 0;
  return dispatch(dtype, N, [&](auto t, auto l) {
    using T = decltype(t);
    constexpr int LPC = decltype(l)::value;
    const int64_t n = B * D * LPC;
    if ((n + NT - 1) / NT >= ((int64_t)1 << 31)) return (int)MOGT_ERR_UNSUPPORTED;
    const unsigned grid = (unsigned)((n + NT - 1) / NT);
    auto go = [&](auto kern) {
      kern<<<grid, NT, 0, (cudaStream_t)stream>>>(state, new_state, (const T*)u, u_sb, (const T*)delta, delta_sb,
                                                  (const T*)z, z_sb, (const T*)Bm, B_sb, B_sg, (const T*)Cm, C_sb, C_sg,
                                                  A, Dskip, bias, (T*)y, B, D, (int)N, D / G, softplus);
    };
    if (v4) go(step_kernel<T, LPC, true>);
    else go(step_kernel<T, LPC, false>);
    return mogt_host::launch_status();
  });
}
