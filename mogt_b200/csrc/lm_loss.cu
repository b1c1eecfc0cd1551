// Post-training losses on logits rows: label log-probabilities, the clipped
// policy loss with a KL term, the paired preference loss, and their gradients.
//   lp = x_l - lse,  lse = m + log sum_v exp(x_v - m);
//   d lp / d x_v = [v = l] - exp(x_v - lse).
// About eight operations, one exponential among them, per logit of 2 or 4
// bytes and pass: HBM bounds all of it.  A CTA takes a row at a time; the
// maximum and the sum of exponentials are carried together over one pass
// (rescaled when the maximum grows, once per 4 vectors of 16 bytes, whose
// loads are issued together).  The policy loss knows a token's coefficient as
// soon as the row's sum is known, so its gradient row is written by the same
// CTA at once, while the row it has just read is still in L2: one read and one
// write of the logits in HBM for the loss and its gradient (8192 x 32000 bf16
// with 62 % of the rows counting: 163 us, 5.1 TB/s).
#include <type_traits>

#include "../../include/mogt_lm_loss.h"
#include "selective.cuh"

namespace mogt {
namespace lml {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSms = 148;
// Rows up to which every CTA counts the tokens itself (9 bytes each, from L2)
// instead of a launch of its own.
constexpr int64_t kInlineCount = 1024;

struct Rows {
  const void* logits;
  int64_t sb, sl;
  const int64_t* labels;
  const uint8_t* mask;
  int64_t L, V, rows;
  void* d;
  int64_t d_sb, d_sl;
  float* lp;
  float2* stats;
};

struct Policy {
  const float *old, *ref, *adv;
  int64_t adv_sb, adv_sl;
  float lo, hi, kl;
  float* inv_n;
  bool counted;  // *inv_n is there; otherwise the rows kernel counts
  float *tok, *coef;
};

__device__ __forceinline__ bool counts(const Rows& r, int64_t row) {
  return (!r.mask || r.mask[row]) && r.labels[row] >= 0;
}

// exp(x - m) with the subtraction first: exact for equal values of any size
// (rows of the type's lowest value included).
__device__ __forceinline__ float exp_diff(float x, float m) { return fast_exp2((x - m) * kLog2e); }

struct MS {
  float m, s;
};
__device__ __forceinline__ MS merge(MS a, MS b) {
  const float m = fmaxf(a.m, b.m);
  MS r{m, 0.f};
  // an empty side (s = 0, m = -inf) adds nothing; a NaN sum is kept
  if (a.s != 0.f) r.s += a.s * exp_diff(a.m, m);
  if (b.s != 0.f) r.s += b.s * exp_diff(b.m, m);
  return r;
}
__device__ __forceinline__ MS one(float x) { return MS{x, x == -INFINITY ? 0.f : 1.f}; }

// A row as a head of single elements up to a 16-byte boundary, whole 16-byte
// vectors, and a tail.
template <typename T>
struct Split {
  static constexpr int VEC = 16 / (int)sizeof(T);
  int64_t head, nvec, tail0;
  __device__ Split(const T* x, int64_t V) {
    const int64_t mis = (reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T);
    head = mis ? VEC - mis : 0;
    if (head > V) head = V;
    nvec = (V - head) / VEC;
    tail0 = head + nvec * VEC;
  }
};

// Threads, CTAs on an SM and 16-byte vectors a thread has in flight, chosen by
// measurement at 8192 x 32000 and 4096 x 32001 bf16: a kernel that reads and
// rereads its row (the policy loss with its gradient) runs best with 512, 4, 2
// (163 us; 182 with 256, 6, 4), one that goes over it once with 256, 6, 4
// (50 and 72 us; 55 and 73).  Few rows get one CTA of 1024 threads each.
template <int NT>
struct Tune {
  static constexpr int kUnroll = NT == 512 ? 2 : 4, kCtas = NT == 256 ? 6 : NT == 512 ? 4 : 1;
};

// Vectors i, i + NT, ... of a row; those behind the last hold -inf.
template <typename T, int NT, int UNR>
__device__ __forceinline__ void load_vectors(uint4 (&v)[UNR], const T* xv, int64_t i, int64_t nvec) {
  const uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
  for (int r = 0; r < UNR; ++r) {
    const int64_t k = i + (int64_t)r * NT;
    v[r] = k < nvec ? reinterpret_cast<const uint4*>(xv)[k] : make_uint4(none, none, none, none);
  }
}

// Maximum and sum of exponentials of a row, known to every thread.
template <typename T, int NT>
__device__ MS row_stats(const T* x, int64_t V, MS* red) {
  constexpr int VEC = Split<T>::VEC, W = VEC == 8 ? 1 : 2;  // words per pair
  constexpr int UNR = Tune<NT>::kUnroll;
  const Split<T> sp(x, V);
  const T* xv = x + sp.head;
  const F2 l2e = f2(kLog2e, kLog2e);
  float m = -INFINITY;
  F2 acc = 0;
  for (int64_t i = threadIdx.x; i < sp.nvec; i += (int64_t)NT * UNR) {
    uint4 v[UNR];
    load_vectors<T, NT, UNR>(v, xv, i, sp.nvec);
    float mx = m;
#pragma unroll
    for (int r = 0; r < UNR; ++r)
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        const float2 f = unpack_two<T>(reinterpret_cast<const uint32_t*>(&v[r]) + k * W);
        mx = fmaxf(mx, fmaxf(f.x, f.y));
      }
    const float ref = mx == -INFINITY ? 0.f : mx;
    const float sc = exp_diff(m, ref);
    const F2 neg = f2(-ref, -ref);
    acc = mul2(acc, f2(sc, sc));
    m = mx;
#pragma unroll
    for (int r = 0; r < UNR; ++r)
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        const float2 f = unpack_two<T>(reinterpret_cast<const uint32_t*>(&v[r]) + k * W);
        acc = add2(acc, exp2_2(mul2(add2(f2(f.x, f.y), neg), l2e)));
      }
  }
  MS a{m, hsum(acc)};
  const int64_t edge = threadIdx.x;
  if (edge < sp.head) a = merge(a, one(to_f32(x[edge])));
  if (sp.tail0 + edge < V) a = merge(a, one(to_f32(x[sp.tail0 + edge])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = merge(a, MS{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) red[w] = a;
  __syncthreads();
  a = red[lane % (NT / 32)];
#pragma unroll
  for (int o = NT / 64; o > 0; o >>= 1)
    a = merge(a, MS{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
  return a;
}

// d[v] = c * ([v = label] - p_v), p_v = exp(x_v - m) / s.
template <typename T, int NT>
__device__ void write_grad(const T* x, T* d, int64_t V, int64_t label, float c, float m, float inv_s) {
  constexpr int VEC = Split<T>::VEC, W = VEC == 8 ? 1 : 2, UNR = Tune<NT>::kUnroll;
  const Split<T> sp(x, V);
  const float f = -c * inv_s;
  const T* xv = x + sp.head;
  T* dv = d + sp.head;
  if (((reinterpret_cast<uintptr_t>(dv)) & 15u) == 0) {
    const F2 l2e = f2(kLog2e, kLog2e), neg = f2(-m, -m), ff = f2(f, f);
    for (int64_t i = threadIdx.x; i < sp.nvec; i += (int64_t)NT * UNR) {
      uint4 v[UNR];
      load_vectors<T, NT, UNR>(v, xv, i, sp.nvec);
#pragma unroll
      for (int r = 0; r < UNR; ++r) {
        uint4 o;
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          const float2 e = unpack_two<T>(reinterpret_cast<const uint32_t*>(&v[r]) + k * W);
          const float2 q = un2(mul2(ff, exp2_2(mul2(add2(f2(e.x, e.y), neg), l2e))));
          pack_two<T>(reinterpret_cast<uint32_t*>(&o) + k * W, q.x, q.y);
        }
        const int64_t k = i + (int64_t)r * NT;
        if (k < sp.nvec) reinterpret_cast<uint4*>(dv)[k] = o;
      }
    }
  } else {
    for (int64_t i = threadIdx.x; i < sp.nvec * VEC; i += NT) dv[i] = from_f32<T>(f * exp_diff(to_f32(xv[i]), m));
  }
  const int64_t edge = threadIdx.x;
  if (edge < sp.head) d[edge] = from_f32<T>(f * exp_diff(to_f32(x[edge]), m));
  if (sp.tail0 + edge < V) d[sp.tail0 + edge] = from_f32<T>(f * exp_diff(to_f32(x[sp.tail0 + edge]), m));
  __syncthreads();
  if (threadIdx.x == 0 && label < V) d[label] = from_f32<T>(fmaf(f, exp_diff(to_f32(x[label]), m), c));
}

template <typename T, int NT>
__device__ void write_zero(T* d, int64_t V) {
  constexpr int VEC = Split<T>::VEC;
  const Split<T> sp(d, V);
  Pack<T, VEC> z;
  z.zero();
  for (int64_t i = threadIdx.x; i < sp.nvec; i += NT) z.store(d + sp.head + i * VEC);
  const int64_t edge = threadIdx.x;
  if (edge < sp.head) d[edge] = from_f32<T>(0.f);
  if (sp.tail0 + edge < V) d[sp.tail0 + edge] = from_f32<T>(0.f);
}

__device__ __forceinline__ float nan_f32() { return __int_as_float(0x7fc00000); }

// 1 / max(number of counting tokens, 1), by a whole CTA.
template <int NT>
__device__ float inverse_count(const Rows& r) {
  __shared__ int sm[NT / 32];
  int n = 0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < r.rows; i += NT) n += counts(r, i);
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
  for (int i = 0; i < NT / 32; ++i) n += sm[i];
  return 1.f / (float)(n > 0 ? n : 1);
}

__global__ void __launch_bounds__(1024) count_kernel(const Rows r, float* inv_n) {
  const float v = inverse_count<1024>(r);
  if (threadIdx.x == 0) *inv_n = v;
}

// A CTA per row: log-probability; with POLICY the token's loss and
// coefficient, and with GRAD the row of the gradient.
template <typename T, int NT, bool POLICY, bool GRAD>
__global__ void __launch_bounds__(NT, Tune<NT>::kCtas) rows_kernel(const Rows r, const Policy q) {
  __shared__ MS red[NT / 32];
  float inv_n = 0.f;
  if (POLICY) {
    inv_n = q.counted ? *q.inv_n : inverse_count<NT>(r);
    if (!q.counted && blockIdx.x == 0 && threadIdx.x == 0) *q.inv_n = inv_n;
  }
  const int64_t row = blockIdx.x;
  const int64_t b = row / r.L, l = row % r.L;
  T* d = GRAD ? static_cast<T*>(r.d) + b * r.d_sb + l * r.d_sl : nullptr;
  if (!counts(r, row)) {
    if (GRAD) write_zero<T, NT>(d, r.V);
    if (threadIdx.x == 0) {
      r.lp[row] = 0.f;
      if (r.stats) r.stats[row] = make_float2(0.f, 1.f);
      if (POLICY) q.tok[row] = q.coef[row] = 0.f;
    }
    return;
  }
  const T* x = static_cast<const T*>(r.logits) + b * r.sb + l * r.sl;
  const int64_t label = r.labels[row];
  const MS a = row_stats<T, NT>(x, r.V, red);
  const float lp = label < r.V ? (to_f32(x[label]) - a.m) - logf(a.s) : nan_f32();
  float tok = 0.f, c = 0.f;
  if (POLICY) {
    const float adv = q.adv[b * q.adv_sb + l * q.adv_sl];
    const float rr = expf(lp - q.old[row]);
    const float s1 = rr * adv, s2 = fminf(fmaxf(rr, q.lo), q.hi) * adv;
    tok = -fminf(s1, s2);
    c = s1 <= s2 ? -s1 : 0.f;
    if (s1 != s1) tok = c = s1;  // NaN is not dropped by the minimum
    if (q.ref) {
      const float dd = q.ref[row] - lp, e = expm1f(dd);
      tok = fmaf(q.kl, e - dd, tok);
      c = fmaf(-q.kl, e, c);
    }
    c *= inv_n;
  }
  if (threadIdx.x == 0) {
    r.lp[row] = lp;
    if (r.stats) r.stats[row] = make_float2(a.m, a.s);
    if (POLICY) {
      q.tok[row] = tok;
      q.coef[row] = c;
    }
  }
  if (GRAD) write_grad<T, NT>(x, d, r.V, label, c, a.m, 1.f / a.s);
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT, Tune<NT>::kCtas) rows_bwd_kernel(const Rows r, const float* coef, int64_t coef_div,
                                                      const float* scale, bool unless_one) {
  if (unless_one && *scale == 1.f) return;
  const int64_t row = blockIdx.x;
  const int64_t b = row / r.L, l = row % r.L;
  T* d = static_cast<T*>(r.d) + b * r.d_sb + l * r.d_sl;
  if (!counts(r, row)) {
    write_zero<T, NT>(d, r.V);
    return;
  }
  float c = coef[row / coef_div];
  if (scale) c *= *scale;
  const int64_t label = r.labels[row];
  if (label >= r.V) c = nan_f32();
  const float2 st = r.stats[row];
  write_grad<T, NT>(static_cast<const T*>(r.logits) + b * r.sb + l * r.sl, d, r.V, label, c, st.x, 1.f / st.y);
}

__device__ double block_sum_1024(double v, double* sm) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < 32; ++i) v += sm[i];
  return v;
}

__global__ void __launch_bounds__(1024) token_mean_kernel(const float* tok, int64_t rows, const float* inv_n,
                                                          float* loss) {
  __shared__ double sm[32];
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) v += tok[i];
  v = block_sum_1024(v, sm);
  if (threadIdx.x == 0) *loss = (float)(v * (double)*inv_n);
}

__device__ __forceinline__ float log_sigmoid(float x) { return fminf(x, 0.f) - log1pf(expf(-fabsf(x))); }

// One CTA, a warp per pair: the sums of its two sequences and their difference
// stay in f64 up to the logit (two sums of thousands differ by a few units).
// R: float or double, the reference sums as they are given.
template <typename R>
__global__ void __launch_bounds__(1024) pairs_kernel(const float* lp, const R* ref, int64_t P, int64_t L, float beta,
                                                     float eps, float* loss, float* seq, float* coef) {
  __shared__ double sm[32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  double tot = 0.0;
  for (int64_t i = w; i < P; i += 32) {
    double s[2] = {0.0, 0.0};
#pragma unroll 4
    for (int64_t l = lane; l < L; l += 32) {
      s[0] += lp[i * L + l];
      s[1] += lp[(P + i) * L + l];
    }
    for (int o = 16; o > 0; o >>= 1) {
      s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
      s[1] += __shfl_xor_sync(0xffffffffu, s[1], o);
    }
    if (lane == 0) {
      const float x = (float)((double)beta * ((s[0] - (double)ref[i]) - (s[1] - (double)ref[P + i])));
      // a side without weight is no term: x is infinite for a response of probability 0
      tot -= (eps < 1.f ? (1.f - eps) * log_sigmoid(x) : 0.f) + (eps > 0.f ? eps * log_sigmoid(-x) : 0.f);
      const float c = beta / (float)P * (eps / (1.f + expf(-x)) - (1.f - eps) / (1.f + expf(x)));
      seq[i] = (float)s[0];
      seq[P + i] = (float)s[1];
      coef[i] = c;
      coef[P + i] = -c;
    }
  }
  tot = block_sum_1024(tot, sm);
  if (threadIdx.x == 0) *loss = (float)(tot / (double)(P > 0 ? P : 1));
}

template <typename F>
int by_type(int dtype, F&& f) {
  switch (dtype) {
    case MOGT_DTYPE_F32: return f(float{});
    case MOGT_DTYPE_BF16: return f(__nv_bfloat16{});
    case MOGT_DTYPE_F16: return f(__half{});
    default: return MOGT_ERR_DTYPE;
  }
}

template <int NT, typename F>
int by_rows(int64_t rows, F&& f) {
  return rows >= kSms * 2 ? f(std::integral_constant<int, NT>{}) : f(std::integral_constant<int, 1024>{});
}

inline int check(int64_t B, int64_t L, int64_t V, int dtype) {
  if (B < 0 || L < 0 || V <= 0) return MOGT_ERR_SHAPE;
  if (dtype < 0 || dtype > 2) return MOGT_ERR_DTYPE;
  if (B * L >= ((int64_t)1 << 31)) return MOGT_ERR_UNSUPPORTED;
  return MOGT_OK;
}

}  // namespace lml
}  // namespace mogt

using namespace mogt;
using namespace mogt::lml;

extern "C" int mogt_logprob_fwd(const void* logits, int64_t sb, int64_t sl, const int64_t* labels,
                                const uint8_t* mask, int64_t B, int64_t L, int64_t V, int dtype, float* logprobs,
                                float* stats, void* stream) {
  if (int st = check(B, L, V, dtype)) return st;
  if (B * L == 0) return MOGT_OK;
  if (!logits || !labels || !logprobs) return MOGT_ERR_ARG;
  Rows r{logits, sb, sl, labels, mask, L, V, B * L, nullptr, 0, 0, logprobs, reinterpret_cast<float2*>(stats)};
  return by_type(dtype, [&](auto t) {
    return by_rows<256>(r.rows, [&](auto n) {
      constexpr int NT = decltype(n)::value;
      rows_kernel<decltype(t), NT, false, false><<<(unsigned)r.rows, NT, 0, (cudaStream_t)stream>>>(r, Policy{});
      return mogt_host::launch_status();
    });
  });
}

extern "C" int mogt_logprob_bwd(const void* logits, int64_t sb, int64_t sl, const int64_t* labels,
                                const uint8_t* mask, const float* stats, const float* coef, int64_t coef_div,
                                const float* scale, int unless_one, void* dlogits, int64_t d_sb, int64_t d_sl,
                                int64_t B, int64_t L,
                                int64_t V, int dtype, void* stream) {
  if (int st = check(B, L, V, dtype)) return st;
  if (coef_div <= 0) return MOGT_ERR_SHAPE;
  if (B * L == 0) return MOGT_OK;
  if (!logits || !labels || !stats || !coef || !dlogits || (unless_one && !scale)) return MOGT_ERR_ARG;
  Rows r{logits, sb, sl, labels, mask, L, V, B * L, dlogits, d_sb, d_sl, nullptr,
         const_cast<float2*>(reinterpret_cast<const float2*>(stats))};
  return by_type(dtype, [&](auto t) {
    return by_rows<256>(r.rows, [&](auto n) {
      constexpr int NT = decltype(n)::value;
      rows_bwd_kernel<decltype(t), NT><<<(unsigned)r.rows, NT, 0, (cudaStream_t)stream>>>(
          r, coef, coef_div, scale, unless_one != 0);
      return mogt_host::launch_status();
    });
  });
}

extern "C" size_t mogt_policy_loss_scratch_bytes(int64_t B, int64_t L) {
  return B < 0 || L < 0 ? 0 : (size_t)(B * L + 1) * sizeof(float);
}

extern "C" int mogt_policy_loss(const void* logits, int64_t sb, int64_t sl, const int64_t* labels,
                                const uint8_t* mask, const float* old_logprobs, const float* ref_logprobs,
                                const float* adv, int64_t adv_sb, int64_t adv_sl, float clip_low, float clip_high,
                                float kl_coef, float* loss, float* logprobs, float* stats, float* coef, void* dlogits,
                                int64_t d_sb, int64_t d_sl, int64_t B, int64_t L, int64_t V, int dtype,
                                void* scratch, size_t scratch_bytes, void* stream) {
  if (int st = check(B, L, V, dtype)) return st;
  if (!loss) return MOGT_ERR_ARG;
  if (B * L > 0 && (!logits || !labels || !old_logprobs || !adv || !logprobs || !coef)) return MOGT_ERR_ARG;
  if (!scratch || scratch_bytes < mogt_policy_loss_scratch_bytes(B, L)) return MOGT_ERR_WORKSPACE;
  float* inv_n = static_cast<float*>(scratch);
  Rows r{logits, sb, sl, labels, mask, L, V, B * L, dlogits, d_sb, d_sl, logprobs, reinterpret_cast<float2*>(stats)};
  // a weight of 0 is no term: exp(ref - lp) may overflow, and 0 * inf is not 0
  Policy q{old_logprobs, kl_coef != 0.f ? ref_logprobs : nullptr, adv, adv_sb, adv_sl, 1.f - clip_low, 1.f + clip_high,
           kl_coef, inv_n, r.rows > kInlineCount || r.rows == 0, inv_n + 1, coef};
  cudaStream_t s = (cudaStream_t)stream;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (q.counted) count_kernel<<<1, 1024, 0, s>>>(r, inv_n);
    if (r.rows > 0)
      dlogits ? by_rows<512>(r.rows, [&](auto n) {
        constexpr int NT = decltype(n)::value;
        rows_kernel<T, NT, true, true><<<(unsigned)r.rows, NT, 0, s>>>(r, q);
        return 0;
      })
              : by_rows<256>(r.rows, [&](auto n) {
        constexpr int NT = decltype(n)::value;
        rows_kernel<T, NT, true, false><<<(unsigned)r.rows, NT, 0, s>>>(r, q);
        return 0;
      });
    token_mean_kernel<<<1, 1024, 0, s>>>(q.tok, r.rows, inv_n, loss);
    return mogt_host::launch_status();
  });
}

namespace {
template <typename R>
int preference_pairs(const float* logprobs, const R* ref, int64_t P, int64_t L, float beta, float eps, float* loss,
                     float* seq, float* coef, void* stream) {
  if (P < 0 || L < 0) return MOGT_ERR_SHAPE;
  if (!loss || (P > 0 && (!ref || !seq || !coef || (L > 0 && !logprobs)))) return MOGT_ERR_ARG;
  pairs_kernel<R><<<1, 1024, 0, (cudaStream_t)stream>>>(logprobs, ref, P, L, beta, eps, loss, seq, coef);
  return mogt_host::launch_status();
}
}  // namespace

extern "C" int mogt_preference_pairs(const float* logprobs, const float* ref, int64_t P, int64_t L, float beta,
                                     float eps, float* loss, float* seq, float* coef, void* stream) {
  return preference_pairs(logprobs, ref, P, L, beta, eps, loss, seq, coef, stream);
}

extern "C" int mogt_preference_pairs_f64(const float* logprobs, const double* ref, int64_t P, int64_t L, float beta,
                                         float eps, float* loss, float* seq, float* coef, void* stream) {
  return preference_pairs(logprobs, ref, P, L, beta, eps, loss, seq, coef, stream);
}
