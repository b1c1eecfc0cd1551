// Selective state space scan, forward and single token.  Per channel d and
// state n (group g = d / (D / G)):
//   h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t,   y_t = sum_n C_t h_t + D u_t,
//   out_t = y_t silu(z_t).
// One exponential and four multiply-adds per (token, channel, state) against
// 8 bytes per (token, channel) in bf16: at N = 16 the exponentials (16 a clock
// and SM) bound it, not HBM.
//
// A thread keeps NS = 4 states of two neighbouring channels in registers, the
// pair in the halves of packed fp32 instructions; LPC = N / 4 (rounded up to a
// power of two) lanes share a pair.  Lane = pair + CPW * part.  Tokens come in
// tiles of 16 (the next tile's operands are loaded while one is worked on) and
// groups of 8: the LPC lanes of a pair split a group's tokens for what is done
// once per (token, channel) (softplus, gate, loads, stores), hand (dt, dt u)
// to one another through shared memory, and sum y over the parts with a
// butterfly that leaves each lane the tokens it loaded.
//
// When channels and sequences do not fill the GPU, a sequence is split into
// segments: a first pass leaves each segment's state from zero and its sum of
// dt, and a segment starts from the chain over those before it.
//
// 32768 x 1536 x 16 bf16, one sequence: 616 us (first pass 267 with the
// exponential pipe 75 % busy, main pass 349 at 62 %), against 173 us of
// exponentials in one pass.
#include "selective_scan.cuh"

namespace mogt {
namespace sel {

// The first pass costs about 0.75 of the main one (267 against 349 us at 32768 x
// 1536, N = 16; it takes one segment less).
inline int64_t fwd_segments(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G) {
  return num_segments(B, L, D, N, G, NT, 148 * fwd_ctas(lpc_of(N)), 0.7f);
}

template <int LPC, bool AGG>
struct FwdSmem {
  float B[2][kTile][Lane<LPC>::NP];
  float4 stage[NT / 32][kTile][Lane<LPC>::CPW];  // (dt, dt', x, x')
  float C[AGG ? 1 : 2][AGG ? 1 : kTile][Lane<LPC>::NP];
};

// grid = (channel blocks, segments, B).  AGG: the first pass over a split
// sequence, which leaves each segment's state from zero and its sum of dt.
template <typename T, int LPC, bool VEC, bool AGG>
__global__ void __launch_bounds__(NT, fwd_ctas(LPC)) scan_fwd_kernel(const mogt_selective_args p, const Geo geo,
                                                                       const SegScratch seg) {
  using Q = Lane<LPC>;
  constexpr int TPL = Q::TPL, NP = Q::NP;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  FwdSmem<LPC, AGG>& sm = *reinterpret_cast<FwdSmem<LPC, AGG>*>(smem_raw);
  const Where<LPC> w(p, geo);
  const int64_t len = seq_len(p.lengths, w.b, p.L);
  const int64_t k0 = (int64_t)blockIdx.y * geo.tps, k1 = min(k0 + geo.tps, geo.nck);
  const int64_t kl = min(k1, (len + kTile - 1) / kTile);  // first tile without a live token
  const int64_t cell = w.b * p.D + w.d;

  F2 A2[NS], h[NS];
  const F2 l2e = f2(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    A2[i] = mul2(w.state(p.A, w.d, p.N, w.j * NS + i), l2e);
    h[i] = AGG ? 0 : w.state(p.init, cell, p.N, w.j * NS + i);
  }
  if (!AGG) chain<LPC, Where<LPC>, false>(h, A2, seg, 0, 1, blockIdx.y, p.B * p.D, cell, w);
  const float2 Dd = AGG ? make_float2(0.f, 0.f) : w.param(p.Dskip), bias = w.param(p.bias);
  const bool gate = !AGG && p.z, sp = p.softplus, store = w.ok && w.owner();
  const int tok = w.part_tok(), N = (int)p.N, D = (int)p.D, one = w.ok1;
  const int u_sl = (int)p.u_sl, d_sl = (int)p.delta_sl, z_sl = (int)p.z_sl, B_sl = (int)p.B_sl, C_sl = (int)p.C_sl;
  const T* up = static_cast<const T*>(p.u) + w.b * p.u_sb + k0 * kTile * p.u_sl + w.d;
  const T* dp = static_cast<const T*>(p.delta) + w.b * p.delta_sb + k0 * kTile * p.delta_sl + w.d;
  const T* zp = gate ? static_cast<const T*>(p.z) + w.b * p.z_sb + k0 * kTile * p.z_sl + w.d : nullptr;
  const T* Bp = static_cast<const T*>(p.Bm) + w.b * p.B_sb + w.g * p.B_sg + k0 * kTile * p.B_sl;
  const T* Cp = static_cast<const T*>(p.Cm) + w.b * p.C_sb + w.g * p.C_sg + k0 * kTile * p.C_sl;
  T* out = static_cast<T*>(p.out) + (w.b * p.L + k0 * kTile) * p.D + w.d;
  float4* saved = AGG || !p.saved
                      ? nullptr
                      : reinterpret_cast<float4*>(p.saved) + ((w.b * geo.nck + k0) * p.D + w.d) * LPC + w.j;

  Raws<T, TPL, kGroup, 2, VEC> ru, rd, rz;
  BcRaw<T, NP, NT> rB, rC;
  float2 sdt = make_float2(0.f, 0.f);
  int last = 0;  // last live token of the fetched tile
  auto fetch = [&](int64_t k) {
    last = (int)min(len - 1 - k * kTile, (int64_t)(kTile - 1));
    rB.fetch(Bp, B_sl, N, last);
    Bp += (int64_t)kTile * B_sl;
    rd.fetch(dp, d_sl, tok, last, one);
    dp += (int64_t)kTile * d_sl;
    ru.fetch(up, u_sl, tok, last, one);
    up += (int64_t)kTile * u_sl;
    if (!AGG) {
      rC.fetch(Cp, C_sl, N, last);
      Cp += (int64_t)kTile * C_sl;
      if (gate) {
        rz.fetch(zp, z_sl, tok, last, one);
        zp += (int64_t)kTile * z_sl;
      }
    }
  };
  if (k0 < kl) fetch(k0);
  for (int64_t k = k0; k < kl; ++k) {
    const int buf = (int)(k & 1), live = last;
    if (saved) {
      w.put4(saved, 0, h);
      saved += (int64_t)D * LPC;
    }
    rB.put(sm.B[buf], N, live);
    if (!AGG) rC.put(sm.C[AGG ? 0 : buf], N, live);
    float2 u[2][TPL], gz[2][TPL];
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < TPL; ++i) {
        const int kk = q * kGroup + tok + i;
        u[q][i] = ru.v[q][i].f();
        const DtX r = make_dtx(rd.v[q][i].f(), u[q][i], bias, sp, kk > live);
        if (Q::DUP == 1 || w.owner()) sm.stage[w.warp][kk][w.c] = make_float4(r.dt.x, r.dt.y, r.x.x, r.x.y);
        if (gate) {
          const float2 z = rz.v[q][i].f();
          gz[q][i] = make_float2(z.x * sigmoid(z.x), z.y * sigmoid(z.y));
        }
      }
    __syncthreads();
    if (k + 1 < kl) fetch(k + 1);
    F2 sd = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float y[kGroup][2];
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const int kk = q * kGroup + i;
        const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(&sm.stage[w.warp][kk][w.c]);
        F2 Bn[NS];
        twice4(Bn, &sm.B[buf][kk][w.j * NS]);
#pragma unroll
        for (int m = 0; m < NS; ++m) h[m] = fma2(decay(s.x, A2[m]), h[m], mul2(s.y, Bn[m]));
        if (AGG) {
          sd = add2(sd, s.x);
        } else {
          F2 Cn[NS];
          twice4(Cn, &sm.C[AGG ? 0 : buf][AGG ? 0 : kk][w.j * NS]);
          const float2 v = un2(fma2(Cn[3], h[3], fma2(Cn[2], h[2], fma2(Cn[1], h[1], mul2(Cn[0], h[0])))));
          y[i][0] = v.x;
          y[i][1] = v.y;
        }
      }
      if (!AGG) {
        sum_parts<LPC>(y, w.j);
        const int rows = (int)min(p.L - k * kTile, (int64_t)kTile);
#pragma unroll
        for (int i = 0; i < TPL; ++i) {
          const int kk = q * kGroup + tok + i;
          float o0 = fmaf(Dd.x, u[q][i].x, y[i][0]), o1 = fmaf(Dd.y, u[q][i].y, y[i][1]);
          if (gate) {
            o0 *= gz[q][i].x;
            o1 *= gz[q][i].y;
          }
          if (kk > live) o0 = o1 = 0.f;
          if (store && kk < rows) store_two<T, VEC>(out + (int64_t)kk * D, o0, o1, w.ok1);
        }
      }
    }
    out += (int64_t)kTile * D;
    if (AGG) {
      const float2 v = un2(sd);
      sdt = make_float2(sdt.x + v.x, sdt.y + v.y);
    }
    __syncwarp();  // the stage is rewritten for the next tile
  }
  if constexpr (AGG) {
    const int64_t i = blockIdx.y * p.B * p.D + cell;
    w.put4(seg.loc + w.j, i, h);
    if (w.j == 0) {
      if (w.ok) seg.sdt[i] = sdt.x;
      if (w.ok1) seg.sdt[i + 1] = sdt.y;
    }
  } else {
    // tiles behind the end
    for (int64_t t = max(kl, k0) * kTile + tok; t < min(k1 * kTile, p.L); t += kGroup)
#pragma unroll
      for (int i = 0; i < TPL; ++i)
        if (store && t + i < p.L)
          store_two<T, VEC>(static_cast<T*>(p.out) + (w.b * p.L + t + i) * p.D + w.d, 0.f, 0.f, w.ok1);
    if (p.final_state && (int)blockIdx.y == geo.nseg - 1) {
#pragma unroll
      for (int i = 0; i < NS; ++i) w.put_state(p.final_state, cell, p.N, w.j * NS + i, h[i]);
    }
  }
}

// One token: a thread per 4 states of a channel, the channel's lanes adjacent
// (a warp reads 512 consecutive bytes of the state when N is a multiple of 4).
// Reading and writing the state is what it cannot do without; as it stands the
// scalar arithmetic on it counts as much (256 x 1536 x 16: 63 % of the issue
// slots, 23 % of HBM).  grid = (channels, B).
struct StepParams {
  const float* state;
  float* new_state;
  const void *u, *delta, *z, *Bm, *Cm;
  int64_t u_sb, delta_sb, z_sb, B_sb, B_sg, C_sb, C_sg;
  const float *A, *Dskip, *bias;
  void* y;
  int64_t B;
  int D, N, Dg, sp;
};

// 4 neighbouring values, one access when they are aligned to it.
template <typename T, bool V4>
__device__ __forceinline__ void four(Pack<T, 4>& v, const T* p, int left) {
  if (V4) {
    if (left > 0) v.load(p);
    else v.zero();
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v.e[i] = i < left ? p[i] : from_f32<T>(0.f);
  }
}

// NB sequences at a time, their loads issued together.  As in the prompt form
// the LPC lanes of a channel split what is done once per (sequence, channel)
// and hand (dt, dt u) around; y is summed over them so that a lane ends with
// the sequences it loaded.  V4: N, the strides and the bases are multiples of
// 4 elements.
template <typename T, int LPC, bool V4, int NB>
__global__ void __launch_bounds__(NT) step_kernel(const StepParams p) {
  using Q = Lane<LPC, NB>;
  constexpr int SPL = Q::TPL;  // sequences per lane
  const int i0 = (int)blockIdx.x * NT + threadIdx.x;
  const int j = i0 % LPC, dd = i0 / LPC, n0 = j * NS, left = p.N - n0;
  const bool ok = dd < p.D;
  const int d = ok ? dd : 0, g = p.Dg == p.D ? 0 : d / p.Dg;
  const int mine = LPC >= NB ? j / Q::DUP : j * SPL;  // first of this lane's sequences
  Pack<float, 4> a;
  four<float, V4>(a, p.A + (int64_t)d * p.N + n0, left);
  const float bias = p.bias ? p.bias[d] : 0.f, skip = p.Dskip ? p.Dskip[d] : 0.f;
  for (int64_t b0 = (int64_t)blockIdx.y * NB; b0 < p.B; b0 += (int64_t)gridDim.y * NB) {
    Pack<float, 4> h[NB];
    Pack<T, 4> Bn[NB], Cn[NB];
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      const int64_t b = min(b0 + r, p.B - 1);
      four<float, V4>(h[r], p.state + (b * p.D + d) * p.N + n0, left);
      four<T, V4>(Bn[r], static_cast<const T*>(p.Bm) + b * p.B_sb + g * p.B_sg + n0, left);
      four<T, V4>(Cn[r], static_cast<const T*>(p.Cm) + b * p.C_sb + g * p.C_sg + n0, left);
    }
    float u[SPL], dt[SPL], z[SPL];
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      const int64_t b = min(b0 + mine + i, p.B - 1);
      u[i] = to_f32(static_cast<const T*>(p.u)[b * p.u_sb + d]);
      dt[i] = to_f32(static_cast<const T*>(p.delta)[b * p.delta_sb + d]);
      z[i] = p.z ? to_f32(static_cast<const T*>(p.z)[b * p.z_sb + d]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      dt[i] += bias;
      if (p.sp) dt[i] = softplus(dt[i]);
      z[i] *= sigmoid(z[i]);
    }
    float y[NB][1];
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      // the lane of sequence r among this channel's
      const int from = LPC >= NB ? r * Q::DUP : r / SPL, slot = LPC >= NB ? 0 : r % SPL;
      const float t = LPC == 1 ? dt[slot] : __shfl_sync(0xffffffffu, dt[slot], from, LPC);
      const float x = LPC == 1 ? t * u[slot] : t * __shfl_sync(0xffffffffu, u[slot], from, LPC);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        h[r].e[i] = fmaf(fast_exp2(fmaf(t, a.e[i] * kLog2e, kExp2Shift)), h[r].e[i], x * Bn[r].f(i));
        s = fmaf(Cn[r].f(i), h[r].e[i], s);
      }
      y[r][0] = s;
      const int64_t b = b0 + r;
      if (ok && b < p.B) {
        float* to = p.new_state + (b * p.D + d) * p.N + n0;
        if (V4) {
          if (left > 0) h[r].store(to);
        } else {
#pragma unroll
          for (int i = 0; i < NS; ++i)
            if (i < left) to[i] = h[r].e[i];
        }
      }
    }
    sum_parts<LPC, 1>(y, j);
#pragma unroll
    for (int i = 0; i < SPL; ++i) {
      const int64_t b = b0 + mine + i;
      float o = fmaf(skip, u[i], y[i][0]);
      if (p.z) o *= z[i];
      if (ok && b < p.B && j % Q::DUP == 0) static_cast<T*>(p.y)[b * p.D + d] = from_f32<T>(o);
    }
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
  return seg_scratch_bytes(B, D, N, fwd_segments(B, L, D, N, G));
}

extern "C" int mogt_selective_scan_fwd(const mogt_selective_args* args, void* stream) {
  if (!args) return MOGT_ERR_ARG;
  const mogt_selective_args& p = *args;
  if (int st = check_args(p)) return st;
  if (p.B == 0 || p.D == 0) return MOGT_OK;
  if (!p.A || (p.L > 0 && (!p.u || !p.delta || !p.Bm || !p.Cm || !p.out))) return MOGT_ERR_ARG;
  const Geo geo = geometry(p, NT, fwd_segments(p.B, p.L, p.D, p.N, p.G));
  const size_t need = seg_scratch_bytes(p.B, p.D, p.N, geo.nseg);
  if (need && (!p.scratch || p.scratch_bytes < need)) return MOGT_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(p.saved) | (need ? reinterpret_cast<uintptr_t>(p.scratch) : 0)) & 15u)
    return MOGT_ERR_ALIGN;
  const SegScratch seg = seg_scratch(p.scratch, p.B, p.D, p.N, geo.nseg);
  cudaStream_t s = (cudaStream_t)stream;
  const bool vec = pairs_aligned(p, false);
  return dispatch(p.dtype, p.N, [&](auto t, auto l) {
    using T = decltype(t);
    constexpr int LPC = decltype(l)::value;
    auto go = [&](auto kern, int bytes, int nseg) {
      if (bytes > 48 * 1024 &&
          cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
        return false;
      kern<<<dim3((unsigned)(geo.nblk * p.G), nseg, (unsigned)p.B), NT, bytes, s>>>(p, geo, seg);
      return true;
    };
    bool ok = true;
    if (geo.nseg > 1) {
      constexpr int bytes = (int)sizeof(FwdSmem<LPC, true>);
      ok = vec ? go(scan_fwd_kernel<T, LPC, true, true>, bytes, geo.nseg - 1)
               : go(scan_fwd_kernel<T, LPC, false, true>, bytes, geo.nseg - 1);
    }
    constexpr int bytes = (int)sizeof(FwdSmem<LPC, false>);
    ok = ok && (vec ? go(scan_fwd_kernel<T, LPC, true, false>, bytes, geo.nseg)
                    : go(scan_fwd_kernel<T, LPC, false, false>, bytes, geo.nseg));
    return ok ? mogt_host::launch_status() : (int)MOGT_ERR_LAUNCH;
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
  const uintptr_t f32s = reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(new_state) |
                         reinterpret_cast<uintptr_t>(A);
  const uintptr_t bcs = reinterpret_cast<uintptr_t>(Bm) | reinterpret_cast<uintptr_t>(Cm);
  const bool v4 = N % 4 == 0 && f32s % 16 == 0 && bcs % (dtype == MOGT_DTYPE_F32 ? 16 : 8) == 0 &&
                  (B_sb | B_sg | C_sb | C_sg) % 4 == 0;
  // channels and their threads are counted in 32 bits
  if (D > kMaxStride || D * lpc_of(N) > INT32_MAX - NT) return MOGT_ERR_UNSUPPORTED;
  StepParams p{};
  p.state = state; p.new_state = new_state;
  p.u = u; p.delta = delta; p.z = z; p.Bm = Bm; p.Cm = Cm;
  p.u_sb = u_sb; p.delta_sb = delta_sb; p.z_sb = z_sb;
  p.B_sb = B_sb; p.B_sg = B_sg; p.C_sb = C_sb; p.C_sg = C_sg;
  p.A = A; p.Dskip = Dskip; p.bias = bias; p.y = y;
  p.B = B; p.D = (int)D; p.N = (int)N; p.Dg = (int)(D / G); p.sp = softplus;
  return dispatch(dtype, N, [&](auto t, auto l) {
    using T = decltype(t);
    constexpr int LPC = decltype(l)::value;
    // A CTA lives for little more than the latency of its loads: 4 sequences at
    // a time once one each would make more CTAs than are resident at once (256
    // sequences of 1536 x 16: 19.6 us one at a time, 11.7 us four at a time).
    const int64_t gx = (D * LPC + NT - 1) / NT;
    const bool many = gx * B > 148 * 16;
    const int64_t gy = many ? (B + 3) / 4 : B;
    auto go = [&](auto kern) {
      kern<<<dim3((unsigned)gx, (unsigned)(gy < 65535 ? gy : 65535)), NT, 0, (cudaStream_t)stream>>>(p);
    };
    if (v4) many ? go(step_kernel<T, LPC, true, 4>) : go(step_kernel<T, LPC, true, 1>);
    else many ? go(step_kernel<T, LPC, false, 4>) : go(step_kernel<T, LPC, false, 1>);
    return mogt_host::launch_status();
  });
}
