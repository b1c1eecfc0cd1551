// Short depthwise causal convolution over time, K taps (2, 3 or 4):
//   pre_t = b + sum_j w_j x_{t-K+1+j},   y_t = silu(pre_t)
// and its gradients, with g_t = dy_t act'(pre_t):
//   dx_t = sum_j w_j g_{t+K-1-j},  dw_j = sum_t g_t x_{t-K+1+j},  db = sum_t g_t.
// About ten (forward) and twenty (backward) instructions per pair of 2- or
// 4-byte elements and the same number of bytes, so HBM bounds it once the
// arithmetic is packed (fp32 pairs: one element at a time it took three times
// the instructions and twice the time): every element of x (and dy) should be
// read once and of y (dx) written once.  A thread keeps up to 8 bytes of
// neighbouring channels and walks a run of consecutive tokens with the last
// inputs in registers.  The run's tokens are taken UNR at a time, all their
// loads issued first: the kilobytes in flight per warp are what keeps HBM busy.
// Only the K-1 rows before a run are read twice (in the backward K-1 rows after
// it as well, for the g of the following tokens).
#include "selective.cuh"

namespace mogt {
namespace cconv {

constexpr int NT = 128;
// CTAs on an SM and tokens a thread loads ahead, by measurement at 4 x 8192 x
// 1536 bf16: forward 43 us with 6 and 4 (49 with 6 and 8, 48 with 5 and 8, 51
// with 8 and 4), backward 75 us with 3 and 4 (89 with 4 and 4, 95 with 3 and 2,
// 74 with 3 and 6).
constexpr int kFwdCtas = 6, kFwdUnr = 4, kBwdCtas = 3, kBwdUnr = 4;

struct Params {
  const void *x, *w, *bias, *init, *dy, *dfinal;
  const int64_t* lengths;
  void *y, *fin, *dx, *dinit;
  float* part;  // [runs * B][K + 1][D] partial sums of dw, db
  int64_t x_sb, x_sl, dy_sb, dy_sl;
  int64_t B, L, D, runs;  // runs per sequence
  int run;                // tokens per run
  int silu, pcode;
};

// Row t of the input history of sequence b: x for t >= 0, init below.
template <typename T, int VEC, int K>
__device__ __forceinline__ void hist(Pack<T, VEC>& v, const Params& p, int64_t b, int64_t t, int64_t d) {
  if (t >= 0) v.load(static_cast<const T*>(p.x) + b * p.x_sb + t * p.x_sl + d);
  else if (p.init) v.load(static_cast<const T*>(p.init) + (b * (K - 1) + (K - 1 + t)) * p.D + d);
  else v.zero();
}

// VEC channels as fp32 pairs (VEC = 1: the second half is unused and zero).
template <int VEC>
struct Ch {
  static constexpr int N = (VEC + 1) / 2;
};
template <typename T, int VEC>
__device__ __forceinline__ void widen(F2 (&r)[Ch<VEC>::N], const Pack<T, VEC>& v) {
  if constexpr (VEC == 1) {
    r[0] = f2(v.f(0), 0.f);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 f = unpack_two<T>(reinterpret_cast<const uint32_t*>(&v.raw) + i * (sizeof(T) == 4 ? 2 : 1));
      r[i] = f2(f.x, f.y);
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void narrow(Pack<T, VEC>& v, const F2 (&r)[Ch<VEC>::N]) {
  if constexpr (VEC == 1) {
    v.set(0, un2(r[0]).x);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 f = un2(r[i]);
      pack_two<T>(reinterpret_cast<uint32_t*>(&v.raw) + i * (sizeof(T) == 4 ? 2 : 1), f.x, f.y);
    }
  }
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 1 / (1 + e^-x) of both halves (1 / inf = 0).
__device__ __forceinline__ F2 sigmoid2(F2 x) {
  const float2 e = un2(add2(exp2_2(mul2(x, f2(-1.4426950408889634f, -1.4426950408889634f))), f2(1.f, 1.f)));
  return f2(rcp(e.x), rcp(e.y));
}

// The taps and bias of VEC channels.  The parameters' type is looked at once,
// so that all the loads can be in flight together.
template <typename P, int VEC, int K>
__device__ __forceinline__ void load_taps(F2 (&w)[K][Ch<VEC>::N], F2 (&bias)[Ch<VEC>::N], const void* wp,
                                          const void* bp, int64_t d) {
  const P* pw = static_cast<const P*>(wp) + d * K;
  const P* pb = static_cast<const P*>(bp) + d;
  P rw[K * VEC], rb[VEC];
#pragma unroll
  for (int i = 0; i < K * VEC; ++i) rw[i] = pw[i];
#pragma unroll
  for (int i = 0; i < VEC; ++i) rb[i] = bp ? pb[i] : from_f32<P>(0.f);
#pragma unroll
  for (int i = 0; i < Ch<VEC>::N; ++i) {
    constexpr int two = VEC > 1;
#pragma unroll
    for (int j = 0; j < K; ++j)
      w[j][i] = f2(to_f32(rw[2 * i * K + j]), two ? to_f32(rw[(2 * i + two) * K + j]) : 0.f);
    bias[i] = f2(to_f32(rb[2 * i]), two ? to_f32(rb[2 * i + two]) : 0.f);
  }
}
template <int VEC, int K>
__device__ __forceinline__ void taps(F2 (&w)[K][Ch<VEC>::N], F2 (&bias)[Ch<VEC>::N], const void* wp, const void* bp,
                                     int code, int64_t d) {
  if (code == MOGT_DTYPE_F32) load_taps<float, VEC, K>(w, bias, wp, bp, d);
  else if (code == MOGT_DTYPE_BF16) load_taps<__nv_bfloat16, VEC, K>(w, bias, wp, bp, d);
  else load_taps<__half, VEC, K>(w, bias, wp, bp, d);
}

// Thread -> (sequence, run, channels): channels fastest.
struct Spot {
  int64_t b, run, d;
  bool ok;
  __device__ __forceinline__ Spot(const Params& p, int vec) {
    const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x, cols = p.D / vec;
    ok = i < cols * p.runs * p.B;
    d = i % cols * vec;
    run = i / cols % p.runs;
    b = i / cols / p.runs;
  }
};

template <typename T, int VEC, int K>
__global__ void __launch_bounds__(NT, kFwdCtas) fwd_kernel(const Params p) {
  constexpr int UNR = kFwdUnr, NC = Ch<VEC>::N;
  const Spot at(p, VEC);
  if (!at.ok) return;
  const int64_t b = at.b, d = at.d;
  const int64_t len = seq_len(p.lengths, b, p.L);
  const int64_t t0 = at.run * p.run, t1 = min(t0 + p.run, p.L);
  if (p.fin && t0 == 0) {
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      Pack<T, VEC> v;
      hist<T, VEC, K>(v, p, b, len - (K - 1) + i, d);
      v.store(static_cast<T*>(p.fin) + (b * (K - 1) + i) * p.D + d);
    }
  }
  T* y = static_cast<T*>(p.y) + (b * p.L + t0) * p.D + d;
  const int64_t te = min(t1, len);
  if (t0 < te) {
    F2 w[K][NC], bias[NC], h[K][NC];  // h: the last K inputs, newest last
    taps<VEC, K>(w, bias, p.w, p.bias, p.pcode, d);
#pragma unroll
    for (int j = 1; j < K; ++j) {
      Pack<T, VEC> v;
      hist<T, VEC, K>(v, p, b, t0 - K + j, d);
      widen<T, VEC>(h[j], v);
    }
    const T* x = static_cast<const T*>(p.x) + b * p.x_sb + t0 * p.x_sl + d;
    // whole blocks step their pointers; only the last one clamps its loads and
    // guards its stores
    Pack<T, VEC> v[UNR], next[UNR];
    auto fetch = [&](int64_t t) {
      if (t + UNR <= te) {
#pragma unroll
        for (int r = 0; r < UNR; ++r) {
          next[r].load(x);
          x += p.x_sl;
        }
      } else {
#pragma unroll
        for (int r = 0; r < UNR; ++r) next[r].load(x + min((int)(te - t) - 1, r) * p.x_sl);
      }
    };
    fetch(t0);
    for (int64_t t = t0; t < te; t += UNR) {
      const int n = (int)min(te - t, (int64_t)UNR);
#pragma unroll
      for (int r = 0; r < UNR; ++r) v[r] = next[r];
      if (t + UNR < te) fetch(t + UNR);
#pragma unroll
      for (int r = 0; r < UNR; ++r) {
#pragma unroll
        for (int j = 0; j + 1 < K; ++j)
#pragma unroll
          for (int i = 0; i < NC; ++i) h[j][i] = h[j + 1][i];
        widen<T, VEC>(h[K - 1], v[r]);
        F2 o[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          F2 s = bias[i];
#pragma unroll
          for (int j = 0; j < K; ++j) s = fma2(w[j][i], h[j][i], s);
          o[i] = p.silu ? mul2(s, sigmoid2(s)) : s;
        }
        Pack<T, VEC> q;
        narrow<T, VEC>(q, o);
        if (r < n) q.store(y);
        y += p.D;
      }
    }
  }
  Pack<T, VEC> zero;
  zero.zero();
  for (int64_t t = max(te, t0); t < t1; ++t) zero.store(static_cast<T*>(p.y) + (b * p.L + t) * p.D + d);
}

// Walks t from t0 to t1 + K - 2: g_t of the run's own tokens and of the K-1
// after it; dx_{t-K+1} is complete once g_t is known.  The first run also
// emits the rows -(K-1)..-1, the gradients of the initial state.
template <typename T, int VEC, int K>
__global__ void __launch_bounds__(NT, kBwdCtas) bwd_kernel(const Params p) {
  constexpr int UNR = kBwdUnr, NC = Ch<VEC>::N;
  const Spot at(p, VEC);
  if (!at.ok) return;
  const int64_t b = at.b, d = at.d;
  const int64_t len = seq_len(p.lengths, b, p.L);
  const int64_t t0 = at.run * p.run, t1 = min(t0 + p.run, p.L);
  F2 w[K][NC], bias[NC], g[K][NC], h[K][NC], dw[K][NC], db[NC];
  taps<VEC, K>(w, bias, p.w, p.bias, p.pcode, d);
  const F2 one = f2(1.f, 1.f), minus = f2(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) g[j][i] = dw[j][i] = h[j][i] = 0;
    db[i] = 0;
  }
  const T* x = static_cast<const T*>(p.x) + b * p.x_sb + d;
  const T* dy = static_cast<const T*>(p.dy) + b * p.dy_sb + d;
  T* dx = static_cast<T*>(p.dx) + (b * p.L) * p.D + d;
  if (t0 < len) {
#pragma unroll
    for (int j = 1; j < K; ++j) {
      Pack<T, VEC> v;
      hist<T, VEC, K>(v, p, b, t0 - K + j, d);
      widen<T, VEC>(h[j], v);
    }
  }
  const int64_t first = t0 == 0 ? -(int64_t)(K - 1) : t0;  // first row emitted
  Pack<T, VEC> vx[UNR], vg[UNR], nx[UNR], ng[UNR];
  const T *xp = x + t0 * p.x_sl, *gp = dy + t0 * p.dy_sl;
  T* dp = dx + (t0 - (K - 1)) * p.D;  // row of the block's first tau
  auto fetch = [&](int64_t t) {
    if (t + UNR <= len) {
#pragma unroll
      for (int r = 0; r < UNR; ++r) {
        nx[r].load(xp);
        ng[r].load(gp);
        xp += p.x_sl;
        gp += p.dy_sl;
      }
    } else {  // tokens behind the end: the last one again
#pragma unroll
      for (int r = 0; r < UNR; ++r) {
        const int64_t tt = min(t + r, len - 1);
        nx[r].load(x + tt * p.x_sl);
        ng[r].load(dy + tt * p.dy_sl);
      }
    }
  };
  // EDGE: tokens of the run's ends and the sequence's; inside, every token is
  // live and counted, and every row is emitted as it is.
  auto block = [&](int64_t t, auto edge_c) {
    constexpr bool EDGE = decltype(edge_c)::value;
    // rows behind the end carry no gradient
    const int n = EDGE ? (int)max(min(len - t, (int64_t)UNR), (int64_t)0) : UNR;
#pragma unroll
    for (int r = 0; r < UNR; ++r) {
      const bool live = !EDGE || r < n, mine = !EDGE || t + r < t1;
      const int64_t tau = t + r - (K - 1);
#pragma unroll
      for (int j = 0; j + 1 < K; ++j)
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          g[j][i] = g[j + 1][i];
          h[j][i] = h[j + 1][i];
        }
      if (live) {
        F2 gy[NC];
        widen<T, VEC>(h[K - 1], vx[r]);
        widen<T, VEC>(gy, vg[r]);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          if (p.silu) {
            F2 s = bias[i];
#pragma unroll
            for (int j = 0; j < K; ++j) s = fma2(w[j][i], h[j][i], s);
            // silu'(s) = sg (1 + s (1 - sg))
            const F2 sg = sigmoid2(s);
            gy[i] = mul2(gy[i], mul2(sg, fma2(s, fma2(sg, minus, one), one)));
          }
          g[K - 1][i] = gy[i];
          if (mine) {
#pragma unroll
            for (int j = 0; j < K; ++j) dw[j][i] = fma2(gy[i], h[j][i], dw[j][i]);
            db[i] = add2(db[i], gy[i]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < NC; ++i) g[K - 1][i] = 0;
      }
      if (EDGE && (tau < first || tau >= t1)) continue;
      // g[m] = g_{tau + m}: dx_tau = sum_j w_j g_{tau + K - 1 - j}
      F2 v[NC];
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        v[i] = mul2(w[0][i], g[K - 1][i]);
#pragma unroll
        for (int j = 1; j < K; ++j) v[i] = fma2(w[j][i], g[K - 1 - j][i], v[i]);
      }
      Pack<T, VEC> o;
      if (EDGE) {
        const int64_t fi = tau - (len - (K - 1));
        if (p.dfinal && fi >= 0 && fi < K - 1) {
          F2 df[NC];
          o.load(static_cast<const T*>(p.dfinal) + (b * (K - 1) + fi) * p.D + d);
          widen<T, VEC>(df, o);
#pragma unroll
          for (int i = 0; i < NC; ++i) v[i] = add2(v[i], df[i]);
        }
        narrow<T, VEC>(o, v);
        if (tau >= 0) {
          if (tau >= len) o.zero();
          o.store(dx + tau * p.D);
        } else if (p.dinit) {
          o.store(static_cast<T*>(p.dinit) + (b * (K - 1) + (K - 1 + tau)) * p.D + d);
        }
      } else {
        narrow<T, VEC>(o, v);
        o.store(dp + r * p.D);
      }
    }
  };
  if (t0 < len) fetch(t0);
  for (int64_t t = t0; t < t1 + K - 1; t += UNR) {
#pragma unroll
    for (int r = 0; r < UNR; ++r) {
      vx[r] = nx[r];
      vg[r] = ng[r];
    }
    if (t0 < len && t + UNR < t1 + K - 1) fetch(t + UNR);
    // rows t - K + 1 .. t + UNR - K are emitted: none of them may be one of the last K - 1
    const bool inside = t - (K - 1) >= t0 && t + UNR <= t1 && t + UNR <= len;
    if (inside && t + UNR - K < len - (K - 1)) block(t, std::false_type{});
    else block(t, std::true_type{});
    dp += UNR * p.D;
  }
  float* part = p.part + (b * p.runs + at.run) * (K + 1) * p.D + d;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) part[j * p.D + i] = i % 2 ? un2(dw[j][i / 2]).y : un2(dw[j][i / 2]).x;
    part[K * p.D + i] = i % 2 ? un2(db[i / 2]).y : un2(db[i / 2]).x;
  }
}

// Sum of the partial rows in a fixed order: 32 columns x 8 row groups per CTA.
__global__ void __launch_bounds__(256) reduce_kernel(const float* part, int64_t rows, int64_t D, int K, void* dw,
                                                     void* db, int pcode) {
  __shared__ float sm[8][33];
  const int64_t col = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int grp = threadIdx.x >> 5;
  const int64_t cols = (K + 1) * D;
  float s = 0.f;
  if (col < cols)
#pragma unroll 8
    for (int64_t r = grp; r < rows; r += 8) s += part[r * cols + col];
  sm[grp][threadIdx.x & 31] = s;
  __syncthreads();
  if (grp == 0 && col < cols) {
    for (int i = 1; i < 8; ++i) s += sm[i][threadIdx.x];
    const int64_t j = col / D, d = col % D;
    if (j < K) st_param(dw, pcode, d * K + j, s);
    else if (db) st_param(db, pcode, d, s);
  }
}

// One token; the K-1 rows of the state are read before they are shifted, so
// new_state may be state.  grid = (channels, B).
template <typename T, int VEC, int K>
__global__ void __launch_bounds__(NT) step_kernel(const T* x, int64_t x_sb, const T* state, const void* w,
                                                  const void* bias, T* y, T* new_state, int64_t B, int64_t D,
                                                  int silu, int pcode) {
  constexpr int NC = Ch<VEC>::N;
  const int64_t d = ((int64_t)blockIdx.x * NT + threadIdx.x) * VEC;
  if (d >= D) return;
  F2 wv[K][NC], bv[NC];
  taps<VEC, K>(wv, bv, w, bias, pcode, d);
  for (int64_t b = blockIdx.y; b < B; b += gridDim.y) {
    Pack<T, VEC> h[K], q;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) h[j].load(state + (b * (K - 1) + j) * D + d);
    h[K - 1].load(x + b * x_sb + d);
    F2 o[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] = bv[i];
#pragma unroll
    for (int j = 0; j < K; ++j) {
      F2 v[NC];
      widen<T, VEC>(v, h[j]);
#pragma unroll
      for (int i = 0; i < NC; ++i) o[i] = fma2(wv[j][i], v[i], o[i]);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] = silu ? mul2(o[i], sigmoid2(o[i])) : o[i];
    narrow<T, VEC>(q, o);
    q.store(y + b * D + d);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) h[j + 1].store(new_state + (b * (K - 1) + j) * D + d);
  }
}

// Tokens per run for one wave of the CTAs that are resident at once, between
// 24 (the rows read twice stay few, and so do the backward's partial rows of dw
// and db, one per run) and 512.
inline int run_len(int64_t B, int64_t L, int64_t D, int vec, int ctas) {
  const int64_t per = (int64_t)148 * ctas * NT, all = B * L * (D / vec);
  const int64_t run = (all + per - 1) / per;
  return (int)(run < 24 ? 24 : (run > 512 ? 512 : run));
}
inline int64_t num_runs(int64_t L, int run) { return L > 0 ? (L + run - 1) / run : 1; }

inline bool al(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Widest access that every operand allows: at most 8 bytes, D and all row
// strides multiples of it, all bases aligned to it.
inline int pick_vec(int es, int64_t D, const int64_t* strides, int ns, const void* const* ptrs, int np) {
  for (int v = 8 / es; v > 1; v >>= 1) {
    bool ok = D % v == 0;
    for (int i = 0; i < ns; ++i) ok = ok && strides[i] % v == 0;
    for (int i = 0; i < np; ++i) ok = ok && al(ptrs[i], (size_t)v * es);
    if (ok) return v;
  }
  return 1;
}

template <typename F>
int dispatch_tk(int dtype, int vec, int64_t K, F&& f) {
#define MOGT_K(T, V)                                              \
  switch (K) {                                                    \
    case 2: return f(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 2>{}); \
    case 3: return f(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 3>{}); \
    case 4: return f(T{}, std::integral_constant<int, V>{}, std::integral_constant<int, 4>{}); \
    default: return MOGT_ERR_UNSUPPORTED;                         \
  }
#define MOGT_T(T)                \
  switch (vec) {                 \
    case 4: if constexpr (sizeof(T) == 2) { MOGT_K(T, 4) } else return MOGT_ERR_UNSUPPORTED; \
    case 2: MOGT_K(T, 2)         \
    default: MOGT_K(T, 1)        \
  }
  switch (dtype) {
    case MOGT_DTYPE_F32: MOGT_T(float)
    case MOGT_DTYPE_BF16: MOGT_T(__nv_bfloat16)
    case MOGT_DTYPE_F16: MOGT_T(__half)
    default: return MOGT_ERR_DTYPE;
  }
#undef MOGT_T
#undef MOGT_K
}

inline int check(int64_t B, int64_t L, int64_t D, int64_t K, int dtype, int pd) {
  if (B < 0 || L < 0 || D < 0) return MOGT_ERR_SHAPE;
  if (K < 2 || K > 4) return MOGT_ERR_UNSUPPORTED;
  if (dtype < 0 || dtype > 2 || pd < 0 || pd > 2) return MOGT_ERR_DTYPE;
  return MOGT_OK;
}

}  // namespace cconv
}  // namespace mogt

using namespace mogt;
using namespace mogt::cconv;

extern "C" int mogt_causal_conv_fwd(const void* x, int64_t x_sb, int64_t x_sl, const void* weight, const void* bias,
                                    const void* init, const int64_t* lengths, void* y, void* final_state, int64_t B,
                                    int64_t L, int64_t D, int64_t K, int silu, int dtype, int param_dtype,
                                    void* stream) {
  if (int st = check(B, L, D, K, dtype, param_dtype)) return st;
  if (B == 0 || D == 0 || (L == 0 && !final_state)) return MOGT_OK;
  if ((L > 0 && (!x || !y)) || !weight) return MOGT_ERR_ARG;
  Params p{};
  p.x = x; p.w = weight; p.bias = bias; p.init = init; p.lengths = lengths; p.y = y; p.fin = final_state;
  p.x_sb = x_sb; p.x_sl = x_sl; p.B = B; p.L = L; p.D = D; p.silu = silu; p.pcode = param_dtype;
  const int64_t st[2] = {x_sb, x_sl};
  const void* ptrs[4] = {x, init, y, final_state};
  const int vec = pick_vec(dtype == MOGT_DTYPE_F32 ? 4 : 2, D, st, 2, ptrs, 4);
  p.run = run_len(B, L, D, vec, kFwdCtas);
  p.runs = num_runs(L, p.run);
  const int64_t ctas = (B * p.runs * (D / vec) + NT - 1) / NT;
  if (ctas >= ((int64_t)1 << 31)) return MOGT_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)ctas;
  return dispatch_tk(dtype, vec, K, [&](auto t, auto v, auto k) {
    fwd_kernel<decltype(t), decltype(v)::value, decltype(k)::value><<<grid, NT, 0, (cudaStream_t)stream>>>(p);
    return mogt_host::launch_status();
  });
}

extern "C" size_t mogt_causal_conv_bwd_scratch_bytes(int64_t B, int64_t L, int64_t D, int64_t K) {
  if (B <= 0 || L < 0 || D <= 0) return 0;
  // a row per run: the widest access has the shortest runs, the most rows
  int64_t most = 0;
  for (int v = 1; v <= 4; v <<= 1) {
    const int64_t runs = num_runs(L, run_len(B, L, D, v, kBwdCtas));
    most = runs > most ? runs : most;
  }
  return (size_t)(B * most * (K + 1) * D) * sizeof(float);
}

extern "C" int mogt_causal_conv_bwd(const void* x, int64_t x_sb, int64_t x_sl, const void* weight, const void* bias,
                                    const void* init, const int64_t* lengths, const void* dy, int64_t dy_sb,
                                    int64_t dy_sl, const void* dfinal, void* dx, void* dweight, void* dbias,
                                    void* dinit, int64_t B, int64_t L, int64_t D, int64_t K, int silu, int dtype,
                                    int param_dtype, void* scratch, size_t scratch_bytes, void* stream) {
  if (int st = check(B, L, D, K, dtype, param_dtype)) return st;
  if (B == 0 || D == 0) return MOGT_OK;
  if ((L > 0 && (!x || !dy || !dx)) || !weight || !dweight) return MOGT_ERR_ARG;
  if (!scratch || scratch_bytes < mogt_causal_conv_bwd_scratch_bytes(B, L, D, K)) return MOGT_ERR_WORKSPACE;
  Params p{};
  p.x = x; p.w = weight; p.bias = bias; p.init = init; p.lengths = lengths; p.dy = dy; p.dfinal = dfinal;
  p.dx = dx; p.dinit = dinit; p.part = static_cast<float*>(scratch);
  p.x_sb = x_sb; p.x_sl = x_sl; p.dy_sb = dy_sb; p.dy_sl = dy_sl; p.B = B; p.L = L; p.D = D;
  p.silu = silu; p.pcode = param_dtype;
  const int64_t st[4] = {x_sb, x_sl, dy_sb, dy_sl};
  const void* ptrs[6] = {x, init, dy, dfinal, dx, dinit};
  const int vec = pick_vec(dtype == MOGT_DTYPE_F32 ? 4 : 2, D, st, 4, ptrs, 6);
  p.run = run_len(B, L, D, vec, kBwdCtas);
  p.runs = num_runs(L, p.run);
  const int64_t ctas = (B * p.runs * (D / vec) + NT - 1) / NT;
  if (ctas >= ((int64_t)1 << 31)) return MOGT_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)ctas;
  cudaStream_t s = (cudaStream_t)stream;
  const int r = dispatch_tk(dtype, vec, K, [&](auto t, auto v, auto k) {
    bwd_kernel<decltype(t), decltype(v)::value, decltype(k)::value><<<grid, NT, 0, s>>>(p);
    return mogt_host::launch_status();
  });
  if (r != MOGT_OK) return r;
  reduce_kernel<<<(unsigned)(((K + 1) * D + 31) / 32), 256, 0, s>>>(p.part, B * p.runs, D, (int)K, dweight, dbias,
                                                                    param_dtype);
  return mogt_host::launch_status();
}

extern "C" int mogt_causal_conv_step(const void* x, int64_t x_sb, const void* state, const void* weight,
                                     const void* bias, void* y, void* new_state, int64_t B, int64_t D, int64_t K,
                                     int silu, int dtype, int param_dtype, void* stream) {
  if (int st = check(B, 1, D, K, dtype, param_dtype)) return st;
  if (B == 0 || D == 0) return MOGT_OK;
  if (!x || !state || !weight || !y || !new_state) return MOGT_ERR_ARG;
  const void* ptrs[4] = {x, state, y, new_state};
  const int vec = pick_vec(dtype == MOGT_DTYPE_F32 ? 4 : 2, D, &x_sb, 1, ptrs, 4);
  const dim3 grid((unsigned)((D / vec + NT - 1) / NT), (unsigned)(B < 65535 ? B : 65535));
  return dispatch_tk(dtype, vec, K, [&](auto t, auto v, auto k) {
    using T = decltype(t);
    step_kernel<T, decltype(v)::value, decltype(k)::value><<<grid, NT, 0, (cudaStream_t)stream>>>(
        (const T*)x, x_sb, (const T*)state, weight, bias, (T*)y, (T*)new_state, B, D, silu, param_dtype);
    return mogt_host::launch_status();
  });
}
