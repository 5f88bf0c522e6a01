/*
 * axn_ext.h - further entry points of libaxn_gfx950.so: layer norm and AdamW, the
 * operators of a training step between and behind the Linear layers of axn.h.
 *
 * The conventions are those of axn.h: device pointers unless a name starts with
 * "h_", asynchronous on `stream`, AXN_OK or a negative axn_status with the text
 * in axn_last_error(), arguments checked before any HIP call, nothing allocated
 * on the device, no memory retained.  They have a version of their own, so that
 * a program that knows axn.h alone goes on as it is.
 */
#ifndef AXN_EXT_H_
#define AXN_EXT_H_

#include "axn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define AXN_EXT_ABI_VERSION 1
AXN_API int axn_ext_abi_version(void);

/* ------------------------------------------------------------------------
 * Layer norm over the last dimension, M rows of N elements:
 *   sum = round(x + residual)      (x itself where residual is NULL)
 *   mean = sum_j sum[j] / N,  rstd = 1 / sqrt(sum_j (sum[j] - mean)^2 / N + eps)
 *   y = (sum - mean) * rstd * weight + bias
 * Sums in fp32, y rounded once.
 *   dtype: of x, residual, y and sum (BF16, F16, F32); param_dtype: of weight
 *   and bias, dtype or F32.  weight and bias may each be NULL (1 and 0).
 *   x and residual have rows of ldx / ldr >= N elements, y and sum dense ones.
 *   sum is written if residual is given, and is then required.
 *   mean, rstd: fp32 [M] for the backward pass, or both NULL.
 * Pointers are aligned to their elements; 16-byte aligned rows are faster.  The
 * outputs overlap neither each other nor the inputs.
 * M >= 0 (0: nothing is done), 1 <= N < 2^31, eps >= 0. */
AXN_API int axn_layer_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias,
                       void* y, void* sum, float* mean, float* rstd, int dtype, int param_dtype,
                       int64_t M, int64_t N, int64_t ldx, int64_t ldr, float eps, void* stream);

/* The backward pass, xhat = (h - mean) * rstd, a = dy * weight, h the normalised
 * rows (x, or sum):
 *   dx = rstd * (a - sum_j a[j] / N - xhat * sum_j a[j] xhat[j] / N) + dsum
 *   dweight = sum over rows of dy * xhat,  dbias = sum over rows of dy
 *   dsum: the gradient that reaches h from elsewhere, or NULL; dx is then the
 *   gradient of x and of residual.  weight may be NULL.
 *   dx, dweight, dbias: each may be NULL, not all of them.  dweight and dbias
 *   have param_dtype, are summed in fp32 in a fixed order (equal calls give equal
 *   bits) and rounded once.
 *   workspace: axn_layer_norm_bwd_workspace_bytes(M, N) bytes, 16-byte aligned,
 *   used by this call alone until it has finished; needed for dweight and dbias
 *   unless it is of 0 bytes.
 * M = 0 writes zeros to dweight and dbias. */
AXN_API size_t axn_layer_norm_bwd_workspace_bytes(int64_t M, int64_t N);
AXN_API int axn_layer_norm_bwd(const void* dy, const void* h, const void* weight, const float* mean,
                       const float* rstd, const void* dsum, void* dx, void* dweight, void* dbias,
                       int dtype, int param_dtype, int64_t M, int64_t N, int64_t lddy, int64_t ldh,
                       int64_t lddsum, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------
 * AdamW over a list of tensors: axn_mt_adam with the weight decay taken from
 * the weights themselves,
 *   g = float(g_lowp) * inv_scale * clip_coef
 *   m += (g - m) * (1 - beta1);  v = v * beta2 + (1 - beta2) * g * g
 *   p = p * keep - lr_over_bc1 * m / (sqrt(v) * inv_sqrt_bc2 + eps)
 *   p_lowp = round_to_nearest_even(p)
 * List, gradient types, scan result, skipped steps and limit of a tensor as there.
 * Refused (AXN_EINVAL): written tensors that overlap, of one list or of two, and a
 * gradient that overlaps one, unless it lies where its own weight or copy does,
 * element for element.
 * ------------------------------------------------------------------------ */
typedef struct axn_adamw_hparams {
  float lr_over_bc1;      /* lr / (1 - beta1^t)          */
  float inv_sqrt_bc2;     /* 1 / sqrt(1 - beta2^t)       */
  float one_minus_beta1;
  float beta2;
  float one_minus_beta2;
  float eps;
  float keep;             /* 1 - lr * weight_decay       */
} axn_adamw_hparams;

AXN_API int axn_mt_adamw(const void* const* h_g, void* const* h_p, void* const* h_m, void* const* h_v,
                 void* const* h_plow, const int64_t* h_sizes, int64_t n, int g_dtype, int plow_dtype,
                 float inv_scale, const axn_scan_result* scan, const axn_adamw_hparams* hp, void* stream);

/* The same with the moments in 8 bits.  The elements of a tensor form blocks of
 * AXN_ADAMW8_BLOCK, the last one of them may be short; block i has
 *   2 * AXN_ADAMW8_BLOCK bytes from h_codes[t] + i * 2 * AXN_ADAMW8_BLOCK on: for every
 *   four elements four codes of m, then four of v (those behind the tensor's end
 *   are zero), and
 *   2 bytes from h_exponents[t] + i * 2 on: E of m, E of v.
 * A code of m is a sign (bit 7), four bits of exponent and three of mantissa, one of
 * v five and three:
 *   F(c) = c / 8 for c < 8, else (1 + (c & 7) / 8) * 2^((c >> 3) - 1)
 *   m = +-F(c & 127) * 2^(E - 141),  v = F(c) * 2^(E - 157)
 * E is the exponent field of the block's largest magnitude as a float, the next one
 * if its mantissa is 1.875 or more.  Zeroed codes and exponents are zero moments.
 * E = 255: the block is not finite (a gradient was not, or a moment came to 1.875 * 2^127);
 * all of it reads as NaN.
 * m and v of the step are rounded to codes stochastically: the upper one of the two
 * neighbours is taken from (u + 1/2) / 2^16 <= their distance to the lower one on, u
 * 16 bits of a word that seed (64 bits) and the element's place give; a v above zero
 * takes at least code 1.  Blocks are numbered through the list, empty tensors left
 * out; with the block's number b, the element's place j in it, q = 64 b + j / 4 and
 * 32-bit arithmetic the word is
 *   x = (lo(q) ^ lo(seed)) * 0x9E3779B9;  x = ((x ^ x >> 16) + hi(seed) + hi(q)) * 0x6A09E667
 *   x ^= x >> 15;  w = x * C[j % 4];  w ^= w >> 16
 *   C = {0xBB67AE85, 0x510E527F, 0x1F83D9AB, 0x5BE0CD19};  u: low half for m, high half for v.
 * Every step takes a seed of its own; equal calls give equal bits.  Each product and sum
 * of m and v is rounded by itself.
 *   h_codes[t]: 8-byte aligned, h_exponents[t]: 2-byte aligned; p, g and p_lowp
 *   aligned to 16, 4 elements and 4 elements are faster.  At most 2^26 - 1 blocks to a tensor. */
#define AXN_ADAMW8_BLOCK 256
AXN_API int axn_mt_adamw8(const void* const* h_g, void* const* h_p, void* const* h_codes,
                  void* const* h_exponents, void* const* h_plow, const int64_t* h_sizes, int64_t n,
                  int g_dtype, int plow_dtype, float inv_scale, uint64_t seed, const axn_scan_result* scan,
                  const axn_adamw_hparams* hp, void* stream);

/* The moments that the first n elements of a tensor's codes stand for, as dtype F32 or
 * BF16 (whose mantissa holds a code's; values below 2^-133 are rounded).  m or v may be
 * NULL.  Pointers aligned to 8 (codes), 2 (exponents) and their elements (m, v). */
AXN_API int axn_adamw8_moments(const void* codes, const void* exponents, void* m, void* v, int dtype,
                       int64_t n, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* AXN_EXT_H_ */
