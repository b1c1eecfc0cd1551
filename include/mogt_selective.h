/* mogt_selective.h — C ABI of the selective state space path of libmogt_scan.so:
 * the short depthwise causal convolution, the selective scan, their backward
 * passes and their single-token forms.
 *
 * Conventions are those of mogt_scan.h (device pointers, stream-ordered
 * asynchronous calls, int status, the caller owns every buffer), except that
 * activations may be strided: a [B, L, D] operand is given with its batch and
 * token strides in elements; its last dimension is dense.  Outputs are dense.
 * Element types: MOGT_DTYPE_F32, MOGT_DTYPE_BF16, MOGT_DTYPE_F16.  States,
 * A, D and the delta bias are f32; arithmetic is f32 throughout and every
 * output is rounded once.
 *
 * `lengths` (int64 [B], or NULL for L everywhere) gives each sequence's number
 * of tokens, clamped to [0, L].  Tokens behind it are never read into the
 * arithmetic (they may hold NaN): their outputs and gradients are zero and
 * the final state is the state after the last token.
 *
 * The reference compares against this layer family through a library model
 * (model_baseline_hf_mamba.py) and has no operator of its own for it.
 */
#ifndef MOGT_SELECTIVE_H_
#define MOGT_SELECTIVE_H_

#include "mogt_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------
 * Depthwise causal convolution over time with K taps, K in {2, 3, 4}:
 *   pre_t = bias + sum_j weight[:, j] x_{t-K+1+j},  y_t = silu(pre_t) or pre_t
 * x_{-1}, x_{-2}, ... are the rows of `init` ([B, K-1, D], oldest first) or 0;
 * `final` [B, K-1, D] receives the last K-1 inputs (init's rows included when
 * a sequence is shorter than that).  weight [D, K] and bias [D] are
 * param_dtype; init, final, y are dtype.
 * ------------------------------------------------------------------------- */
int mogt_causal_conv_fwd(const void* x, int64_t x_sb, int64_t x_sl, const void* weight,
                         const void* bias, const void* init, const int64_t* lengths, void* y,
                         void* final_state, int64_t B, int64_t L, int64_t D, int64_t K, int silu,
                         int dtype, int param_dtype, void* stream);
/* Gradients of sum <y, dy> + sum <final, dfinal>: dx [B, L, D] and dinit
 * [B, K-1, D] (or NULL) in dtype, dweight [D, K] and dbias [D] (or NULL) in
 * param_dtype.  dy strided like x; dfinal dense or NULL.  scratch: at least
 * mogt_causal_conv_bwd_scratch_bytes(B, L, D, K). */
size_t mogt_causal_conv_bwd_scratch_bytes(int64_t B, int64_t L, int64_t D, int64_t K);
int mogt_causal_conv_bwd(const void* x, int64_t x_sb, int64_t x_sl, const void* weight,
                         const void* bias, const void* init, const int64_t* lengths, const void* dy,
                         int64_t dy_sb, int64_t dy_sl, const void* dfinal, void* dx, void* dweight,
                         void* dbias, void* dinit, int64_t B, int64_t L, int64_t D, int64_t K,
                         int silu, int dtype, int param_dtype, void* scratch, size_t scratch_bytes,
                         void* stream);
/* One token: x [B, D] (row stride x_sb), state [B, K-1, D] -> y [B, D] and the
 * shifted state in new_state (may be state itself). */
int mogt_causal_conv_step(const void* x, int64_t x_sb, const void* state, const void* weight,
                          const void* bias, void* y, void* new_state, int64_t B, int64_t D,
                          int64_t K, int silu, int dtype, int param_dtype, void* stream);

/* ---------------------------------------------------------------------------
 * Selective state space scan.  Per channel d and state n, with
 *   dt_t = delta_t + bias, or softplus(delta_t + bias)
 *   h_t[d, n] = exp(dt_t[d] A[d, n]) h_{t-1}[d, n] + dt_t[d] u_t[d] B_t[g, n]
 *   y_t[d]    = sum_n C_t[g, n] h_t[d, n] + Dskip[d] u_t[d]
 *   out_t     = y_t silu(z_t)   (z given)   or   y_t
 * where g = d / (D / G) is the channel's group.
 * Limits: N <= 128, D a multiple of G, B <= 65535 for the scan; for the single
 * token D times N / 4, rounded up to a power of two, below 2^31.
 * ------------------------------------------------------------------------- */
typedef struct mogt_selective_args {
  const void *u, *delta, *z, *Bm, *Cm;            /* z may be NULL */
  int64_t u_sb, u_sl, delta_sb, delta_sl, z_sb, z_sl; /* [B, L, D] strides, in elements */
  int64_t B_sb, B_sl, B_sg, C_sb, C_sl, C_sg;     /* [B, L, G, N] strides, in elements */
  const float *A, *Dskip, *bias;                  /* [D, N]; [D] or NULL; [D] or NULL */
  const float *init;                              /* [B, D, N] or NULL */
  const int64_t *lengths;                         /* [B] or NULL */
  int64_t B, L, D, N, G;
  int32_t softplus, dtype;
  void *out;                                      /* [B, L, D] */
  float *final_state;                             /* [B, D, N] or NULL */
  void *saved;            /* forward: written when not NULL; backward: read */
  /* backward only */
  const void *dout;                               /* [B, L, D], strided */
  int64_t dout_sb, dout_sl;
  const float *dfinal;                            /* [B, D, N] or NULL */
  void *du, *ddelta, *dz;                         /* [B, L, D] dtype; dz NULL without z */
  void *dB, *dC;                                  /* [B, L, G, N] dtype */
  float *dA, *dD, *dbias, *dinit;                 /* f32; the last three may be NULL */
  void *scratch;
  size_t scratch_bytes;
} mogt_selective_args;

/* Bytes of `saved` (the states a backward starts from; f32, one per 16
 * tokens) and of each direction's scratch.  Most of the backward's holds
 * partial rows of dB and dC, one per token and block of 256 / (N / 4) channels:
 * it grows with D N^2 (D = 1536: 3 KB a token at N = 16, 49 KB at 64, 197 KB at
 * 128). */
size_t mogt_selective_saved_bytes(int64_t B, int64_t L, int64_t D, int64_t N);
size_t mogt_selective_fwd_scratch_bytes(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G);
size_t mogt_selective_bwd_scratch_bytes(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G);
int mogt_selective_scan_fwd(const mogt_selective_args* args, void* stream);
int mogt_selective_scan_bwd(const mogt_selective_args* args, void* stream);

/* One token: u, delta, z [B, D] (row strides), Bm, Cm [B, G, N] (strides),
 * state [B, D, N] f32 -> y [B, D] and new_state (may be state itself). */
int mogt_selective_step(const float* state, float* new_state, const void* u, int64_t u_sb,
                        const void* delta, int64_t delta_sb, const void* z, int64_t z_sb,
                        const void* Bm, int64_t B_sb, int64_t B_sg, const void* Cm, int64_t C_sb,
                        int64_t C_sg, const float* A, const float* Dskip, const float* bias, void* y,
                        int64_t B, int64_t D, int64_t N, int64_t G, int softplus, int dtype,
                        void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MOGT_SELECTIVE_H_ */
