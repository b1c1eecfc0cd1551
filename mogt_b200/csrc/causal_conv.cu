// Short depthwise causal convolution over time, K taps (2, 3 or 4):
//   pre_t = b + sum_j w_j x_{t-K+1+j},   y_t = silu(pre_t)
// and its gradients, with g_t = dy_t act'(pre_t):
//   dx_t = sum_j w_j g_{t+K-1-j},  dw_j = sum_t g_t x_{t-K+1+j},  db = sum_t g_t.
// About ten (forward) and thirty (backward) operations per 2- or 4-byte
// element, so HBM bounds it: every element of x (and dy) should be read once
// and of y (dx) written once.  A thread keeps VEC neighbouring channels (one
// access of up to 16 bytes, 8 in the backward, which holds three times the
// registers per channel) and walks a run of consecutive tokens with the last
// K-1 inputs in registers.  The run's tokens are taken UNR at a time, all
// their loads issued first: a few kilobytes in flight per warp is what keeps
// HBM busy.  Only the K-1 rows before a run are read twice (in the backward
// K-1 rows after it as well, for the g of the following tokens).
#include "selective.cuh"

namespace mogt {
namespace cconv {

constexpr int NT = 128;

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

// The taps and bias of VEC channels.  The parameters' type is looked at once,
// so that all the loads can be in flight together.
template <typename P, int VEC, int K>
__device__ __forceinline__ void load_taps(float (&w)[K][VEC], float (&bias)[VEC], const void* wp, const void* bp,
                                          int64_t d) {
  const P* pw = static_cast<const P*>(wp) + d * K;
  const P* pb = static_cast<const P*>(bp) + d;
  P rw[K * VEC], rb[VEC];
#pragma unroll
  for (int i = 0; i < K * VEC; ++i) rw[i] = pw[i];
#pragma unroll
  for (int i = 0; i < VEC; ++i) rb[i] = bp ? pb[i] : from_f32<P>(0.f);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) w[j][i] = to_f32(rw[i * K + j]);
    bias[i] = to_f32(rb[i]);
  }
}
template <int VEC, int K>
__device__ __forceinline__ void taps(float (&w)[K][VEC], float (&bias)[VEC], const void* wp, const void* bp, int code,
                                     int64_t d) {
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
__global__ void __launch_bounds__(NT, 4) fwd_kernel(const Params p) {
  constexpr int UNR = 8;
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
    float w[K][VEC], bias[VEC];
    taps<VEC, K>(w, bias, p.w, p.bias, p.pcode, d);
    // h[0..K-2]: the K-1 tokens before the block, then the block's
    Pack<T, VEC> h[K - 1 + UNR];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) hist<T, VEC, K>(h[j], p, b, t0 - (K - 1) + j, d);
    const T* x = static_cast<const T*>(p.x) + b * p.x_sb + t0 * p.x_sl + d;
    for (int64_t t = t0; t < te; t += UNR) {
      const int n = (int)min(te - t, (int64_t)UNR);
#pragma unroll
      for (int r = 0; r < UNR; ++r) h[K - 1 + r].load(x + min(r, n - 1) * p.x_sl);
#pragma unroll
      for (int r = 0; r < UNR; ++r) {
        Pack<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float s = bias[i];
#pragma unroll
          for (int j = 0; j < K; ++j) s = fmaf(w[j][i], h[r + j].f(i), s);
          o.set(i, p.silu ? s * sigmoid(s) : s);
        }
        if (r < n) o.store(y + r * p.D);
      }
#pragma unroll
      for (int j = 0; j < K - 1; ++j) h[j] = h[UNR + j];
      x += UNR * p.x_sl;
      y += UNR * p.D;
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
__global__ void __launch_bounds__(NT, 4) bwd_kernel(const Params p) {
  constexpr int UNR = 4;
  const Spot at(p, VEC);
  if (!at.ok) return;
  const int64_t b = at.b, d = at.d;
  const int64_t len = seq_len(p.lengths, b, p.L);
  const int64_t t0 = at.run * p.run, t1 = min(t0 + p.run, p.L);
  float w[K][VEC], bias[VEC], g[K][VEC], dw[K][VEC], db[VEC];
  taps<VEC, K>(w, bias, p.w, p.bias, p.pcode, d);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) g[j][i] = dw[j][i] = 0.f;
    db[i] = 0.f;
  }
  const T* x = static_cast<const T*>(p.x) + b * p.x_sb + d;
  const T* dy = static_cast<const T*>(p.dy) + b * p.dy_sb + d;
  T* dx = static_cast<T*>(p.dx) + (b * p.L) * p.D + d;
  Pack<T, VEC> h[K - 1 + UNR], gy[UNR];
  if (t0 < len) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) hist<T, VEC, K>(h[j], p, b, t0 - (K - 1) + j, d);
  }
  const int64_t first = t0 == 0 ? -(int64_t)(K - 1) : t0;  // first row emitted
  for (int64_t t = t0; t < t1 + K - 1; t += UNR) {
    // rows behind the end carry no gradient
    const int n = (int)max(min(len - t, (int64_t)UNR), (int64_t)0);
    if (n > 0) {
#pragma unroll
      for (int r = 0; r < UNR; ++r) {
        h[K - 1 + r].load(x + (t + min(r, n - 1)) * p.x_sl);
        gy[r].load(dy + (t + min(r, n - 1)) * p.dy_sl);
      }
    }
#pragma unroll
    for (int r = 0; r < UNR; ++r) {
      const bool live = r < n, mine = t + r < t1;
      const int64_t tau = t + r - (K - 1), fi = tau - (len - (K - 1));
      const bool emit = tau >= first && tau < t1;
      Pack<T, VEC> o, df;
      const bool has_f = p.dfinal && emit && fi >= 0 && fi < K - 1;
      if (has_f) df.load(static_cast<const T*>(p.dfinal) + (b * (K - 1) + fi) * p.D + d);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
#pragma unroll
        for (int j = 0; j + 1 < K; ++j) g[j][i] = g[j + 1][i];
        float hv[K], s = bias[i];
#pragma unroll
        for (int j = 0; j < K; ++j) {
          hv[j] = h[r + j].f(i);
          s = fmaf(w[j][i], hv[j], s);
        }
        float gt = gy[r].f(i);
        if (p.silu) {
          const float sg = sigmoid(s);
          gt *= sg * (1.f + s * (1.f - sg));
        }
        if (!live) gt = 0.f;
        if (live && mine) {
#pragma unroll
          for (int j = 0; j < K; ++j) dw[j][i] = fmaf(gt, hv[j], dw[j][i]);
          db[i] += gt;
        }
        g[K - 1][i] = gt;
        // g[m] = g_{tau + m}: dx_tau = sum_j w_j g_{tau + K - 1 - j}
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) v = fmaf(w[j][i], g[K - 1 - j][i], v);
        if (has_f) v += df.f(i);
        o.set(i, v);
      }
      if (emit) {
        if (tau >= 0) {
          if (tau >= len) o.zero();
          o.store(dx + tau * p.D);
        } else if (p.dinit) {
          o.store(static_cast<T*>(p.dinit) + (b * (K - 1) + (K - 1 + tau)) * p.D + d);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j) h[j] = h[UNR + j];
  }
  float* part = p.part + (b * p.runs + at.run) * (K + 1) * p.D + d;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int j = 0; j < K; ++j) part[j * p.D + i] = dw[j][i];
    part[K * p.D + i] = db[i];
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
// new_state may be state.
template <typename T, int VEC, int K>
__global__ void __launch_bounds__(NT) step_kernel(const T* x, int64_t x_sb, const T* state, const void* w,
                                                  const void* bias, T* y, T* new_state, int64_t B, int64_t D,
                                                  int silu, int pcode) {
  const int64_t i0 = (int64_t)blockIdx.x * NT + threadIdx.x;
  const int64_t per = D / VEC;
  if (i0 >= B * per) return;
  const int64_t b = i0 / per, d = (i0 % per) * VEC;
  Pack<T, VEC> h[K], o;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) h[j].load(state + (b * (K - 1) + j) * D + d);
  h[K - 1].load(x + b * x_sb + d);
  float wv[K][VEC], bv[VEC];
  taps<VEC, K>(wv, bv, w, bias, pcode, d);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float s = bv[i];
#pragma unroll
    for (int j = 0; j < K; ++j) s = fmaf(wv[j][i], h[j].f(i), s);
    o.set(i, silu ? s * sigmoid(s) : s);
  }
  o.store(y + b * D + d);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) h[j + 1].store(new_state + (b * (K - 1) + j) * D + d);
}

// Tokens per run for `waves` waves of the CTAs that are resident at once (4 on
// each SM), between 24 (the rows read twice stay few) and 512.  The backward
// takes one wave: a partial row of dw and db is written per run.
inline int run_len(int64_t B, int64_t L, int64_t D, int vec, int waves) {
  const int64_t per = (int64_t)148 * 4 * NT * waves, all = B * L * (D / vec);
  const int64_t run = (all + per - 1) / per;
  return (int)(run < 24 ? 24 : (run > 512 ? 512 : run));
}
inline int64_t num_runs(int64_t L, int run) { return L > 0 ? (L + run - 1) / run : 1; }

inline bool al(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Widest access that every operand allows: at most `most` bytes, D and all row
// strides multiples of it, all bases aligned to it.
inline int pick_vec(int most, int es, int64_t D, const int64_t* strides, int ns, const void* const* ptrs, int np) {
  for (int v = most / es; v > 1; v >>= 1) {
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
    case 8: if constexpr (sizeof(T) == 2) { MOGT_K(T, 8) } else return MOGT_ERR_UNSUPPORTED; \
    case 4: MOGT_K(T, 4)         \
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
  const int vec = pick_vec(16, dtype == MOGT_DTYPE_F32 ? 4 : 2, D, st, 2, ptrs, 4);
  p.run = run_len(B, L, D, vec, 2);
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
  // the narrowest access has the shortest runs
  int64_t most = 0;
  for (int v = 1; v <= 4; v <<= 1) {
    const int64_t runs = num_runs(L, run_len(B, L, D, v, 1));
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
  const int vec = pick_vec(8, dtype == MOGT_DTYPE_F32 ? 4 : 2, D, st, 4, ptrs, 6);
  p.run = run_len(B, L, D, vec, 1);
  p.runs = num_runs(L, p.run);
  const int64_t ctas = (B * p.runs * (D / vec) + NT - 1) / NT;
  if (ctas >= ((int64_t)1 << 31)) return MOGT_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)ctas;
  cudaStream_t s = (cudaStream_t)stream;
  const int r = dispatch_tk(dtype, vec, K, [&](auto t, auto v, auto k) {
    using T = decltype(t);
    if constexpr (decltype(v)::value * sizeof(T) <= 8) {
      bwd_kernel<T, decltype(v)::value, decltype(k)::value><<<grid, NT, 0, s>>>(p);
      return mogt_host::launch_status();
    } else {
      return (int)MOGT_ERR_UNSUPPORTED;  // pick_vec stops at 8 bytes
    }
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
  const int vec = pick_vec(16, dtype == MOGT_DTYPE_F32 ? 4 : 2, D, &x_sb, 1, ptrs, 4);
  const int64_t n = B * (D / vec);
  return dispatch_tk(dtype, vec, K, [&](auto t, auto v, auto k) {
    using T = decltype(t);
    step_kernel<T, decltype(v)::value, decltype(k)::value><<<(unsigned)((n + NT - 1) / NT), NT, 0, (cudaStream_t)stream>>>(
        (const T*)x, x_sb, (const T*)state, weight, bias, (T*)y, (T*)new_state, B, D, silu, param_dtype);
    return mogt_host::launch_status();
  });
}
