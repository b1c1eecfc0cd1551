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

template <typename T, int LPC>
__global__ void __launch_bounds__(NT) scan_fwd_kernel(const mogt_selective_args p, const Geo geo) {
  using Q = Lane<LPC>;
  constexpr int CPW = Q::CPW, TPL = Q::TPL, NP = Q::NP;
  __shared__ float sB[kTile][NP], sC[kTile][NP];
  __shared__ float2 stage[NT / 32][kGroup][CPW];
  const Where<LPC> w(p, geo);
  const int64_t len = seq_len(p.lengths, w.b, p.L);

  float A2[NS], h[NS];
  load_A<LPC>(A2, p, w);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int n = w.j * NS + i;
    h[i] = (p.init && w.ok && n < p.N) ? p.init[(w.b * p.D + w.d) * p.N + n] : 0.f;
  }
  const float Dd = p.Dskip && w.ok ? p.Dskip[w.d] : 0.f;
  const float bias = p.bias && w.ok ? p.bias[w.d] : 0.f;
  T* out = static_cast<T*>(p.out) + (w.b * p.L) * p.D + w.d;
  float4* saved = reinterpret_cast<float4*>(p.saved);

  for (int64_t t0 = 0; t0 < p.L; t0 += kTile) {
    if (saved && w.ok)
      saved[((w.b * geo.nck + t0 / kTile) * p.D + w.d) * LPC + w.j] = make_float4(h[0], h[1], h[2], h[3]);
    if (t0 >= len) {
      for (int k = w.part_tok(); k < kTile; k += kGroup)
#pragma unroll
        for (int i = 0; i < TPL; ++i)
          if (w.ok && w.owner() && t0 + k + i < p.L) out[(t0 + k + i) * p.D] = from_f32<T>(0.f);
      continue;
    }
    __syncthreads();
    load_bc<T, NP>(sB, p, w, static_cast<const T*>(p.Bm), p.B_sb, p.B_sl, p.B_sg, t0, len);
    load_bc<T, NP>(sC, p, w, static_cast<const T*>(p.Cm), p.C_sb, p.C_sl, p.C_sg, t0, len);
    __syncthreads();
#pragma unroll
    for (int gq = 0; gq < kTile / kGroup; ++gq) {
      const int64_t tg = t0 + gq * kGroup;
      float u[TPL], z[TPL];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int64_t t = tg + w.part_tok() + i;
        float dt = 0.f;
        u[i] = z[i] = 0.f;
        if (w.ok && t < len) {
          u[i] = to_f32(static_cast<const T*>(p.u)[w.b * p.u_sb + t * p.u_sl + w.d]);
          dt = to_f32(static_cast<const T*>(p.delta)[w.b * p.delta_sb + t * p.delta_sl + w.d]) + bias;
          if (p.softplus) dt = softplus(dt);
          if (p.z) z[i] = to_f32(static_cast<const T*>(p.z)[w.b * p.z_sb + t * p.z_sl + w.d]);
        }
        if (w.owner()) stage[w.warp][w.part_tok() + i][w.c] = make_float2(dt, dt * u[i]);
      }
      __syncwarp();
      float y[kGroup][1];
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        const float2 dx = stage[w.warp][k][w.c];
        const float4 Bv = *reinterpret_cast<const float4*>(&sB[gq * kGroup + k][w.j * NS]);
        const float4 Cv = *reinterpret_cast<const float4*>(&sC[gq * kGroup + k][w.j * NS]);
        const float Bn[NS] = {Bv.x, Bv.y, Bv.z, Bv.w}, Cn[NS] = {Cv.x, Cv.y, Cv.z, Cv.w};
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          h[i] = fmaf(fast_exp2(dx.x * A2[i]), h[i], dx.y * Bn[i]);
          s = fmaf(Cn[i], h[i], s);
        }
        y[k][0] = s;
      }
      sum_parts<LPC, 1>(y, w.j);
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int64_t t = tg + w.part_tok() + i;
        float o = fmaf(Dd, u[i], y[i][0]);
        if (p.z) o *= z[i] * sigmoid(z[i]);
        if (w.ok && w.owner() && t < p.L) out[t * p.D] = from_f32<T>(t < len ? o : 0.f);
      }
    }
  }
  if (p.final_state && w.ok) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int n = w.j * NS + i;
      if (n < p.N) p.final_state[(w.b * p.D + w.d) * p.N + n] = h[i];
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

extern "C" size_t mogt_selective_fwd_scratch_bytes(int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

extern "C" int mogt_selective_scan_fwd(const mogt_selective_args* args, void* stream) {
  if (!args) return MOGT_ERR_ARG;
  const mogt_selective_args& p = *args;
  if (int st = check_args(p)) return st;
  if (p.B == 0 || p.D == 0) return MOGT_OK;
  if (!p.A || (p.L > 0 && (!p.u || !p.delta || !p.Bm || !p.Cm || !p.out))) return MOGT_ERR_ARG;
  const Geo geo = geometry(p, NT);
  const dim3 grid((unsigned)(geo.nblk * p.G), 1, (unsigned)p.B);
  return dispatch(p.dtype, p.N, [&](auto t, auto l) {
    scan_fwd_kernel<decltype(t), decltype(l)::value><<<grid, NT, 0, (cudaStream_t)stream>>>(p, geo);
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
