/*
 * C ABI of the microscaled (MX) path: quantisation to block-scaled 4- and
 * 8-bit floating point, products of MX activations with MXFP4 weights on the
 * matrix cores, and the layer steps that hand MX activations on
 * (RMSNorm, SwiGLU).  In the same library and with the same conventions as
 * nvm_moe.h: device pointers, work on `stream`, no host synchronisation, no
 * device allocation, no workspace, NVM_OK or a negative NVM_ERR_* status
 * (message in nvm_last_error()).
 *
 * Formats (OCP Microscaling, blocks of 32 consecutive values of a row):
 *   scales  E8M0 bytes, row r's block j at scales[r * scale_ld + j]: byte b
 *           stands for 2^(b - 127), 255 for NaN
 *   codes   NVM_MX_FP4: E2M1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives),
 *           two a byte, the even value in the low half: rows of n / 2 bytes.
 *           (The words of an MLX "mxfp4" weight are these bytes.)
 *           NVM_MX_FP8: E4M3 (largest 448, no infinity): rows of n bytes
 * A value is element * 2^(b - 127).  Row lengths n are multiples of 32 up to
 * 2^20.  scale_ld is a multiple of 16, at least n / 32 rounded up to 16:
 * bytes past a row's n / 32 scales are neither written nor do they count, but
 * they are read, so the last row needs them too.  codes, scales and 16-bit or
 * float32 rows are 16-byte aligned.
 *
 * Quantisation of a block with the largest magnitude A:
 * b = clamp(floor(log2 A) - emax + 127, 0, 254) with emax = 2 (FP4) or 8
 * (FP8); elements are x * 2^(127 - b) rounded to the nearest element value
 * (ties to even), saturating.  A = 0 gives b = 0.  A block that holds a NaN or
 * an infinity gets b = 255 and codes of zero: it stands for NaNs, and every
 * product over it is NaN.
 */
#ifndef NVM_MX_H
#define NVM_MX_H

#include "nvm_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

enum nvm_mx_format { NVM_MX_FP4 = 0, NVM_MX_FP8 = 1 };

/* Or-ed into a product's a_format: E4M3 activations summed by the scaled matrix
 * instruction itself, at twice the rate of float32 sums.  It adds eight
 * neighbouring E4M3 by E2M1 products as integers in units of 2^-13 of (a power
 * of two not above) the largest of them and drops what lies below, less than
 * 7 * 2^-13 of the largest for each eight; of a layer's values that is 2^-17 to
 * 2^-15 of the sums in the root mean square, where float32 sums are 2^-25 off.
 * (E2M1 by E2M1 lies inside those units: with NVM_MX_FP4 the flag changes
 * nothing.) */
enum { NVM_MX_SHORT_SUMS = 16 };

/* Types of plain values (the codes of nvm_kv_dtype). */
enum nvm_mx_dtype { NVM_MX_F16 = 0, NVM_MX_BF16 = 1, NVM_MX_F32 = 2 };

/* x [rows, n] of `dtype` (rows x_ld values apart, a multiple of 16 bytes) to
 * MX codes and scales. */
int nvm_mx_quantize(const void *x, int64_t rows, int64_t n, int64_t x_ld, int dtype, int format,
                    void *codes, uint8_t *scales, int64_t scale_ld, nvm_stream_t stream);

/* The values of codes and scales, rounded once to `dtype`: out [rows, n]. */
int nvm_mx_dequantize(const void *codes, const uint8_t *scales, int64_t scale_ld, int64_t rows,
                      int64_t n, int format, int dtype, void *out, nvm_stream_t stream);

/* Rows ids[0], .. ids[T - 1] of a table [V, n] (an embedding), rounded once to
 * `dtype`: out [T, n].  Ids outside [0, V) give zero rows. */
int nvm_mx_embedding(const int32_t *ids, int64_t T, const void *codes, const uint8_t *scales,
                     int64_t scale_ld, int64_t V, int64_t n, int format, int dtype, void *out,
                     nvm_stream_t stream);

/* nvm_residual_rms_norm with an MX output: h_out = rnd(h + r) (r NULL: h
 * itself, h_out not written), and the MX codes of rms_norm(h_out) * w.  The
 * norm is computed in float64 and not rounded to the activation dtype before
 * the quantisation.  H a multiple of 32, at most 8192; dtype NVM_DTYPE_F16 or
 * NVM_DTYPE_BF16 (of h, r, w and h_out); h_out may be h. */
int nvm_residual_rms_norm_mx(const void *h, const void *r, const void *w, int64_t T, int64_t H,
                             float eps, int dtype, void *h_out, int format, void *codes,
                             uint8_t *scales, int64_t scale_ld, nvm_stream_t stream);

/* out[m, k] = rnd(sum_j a[m, j] * w[k, j]): a [M, N] in MX (a_format, perhaps
 * with NVM_MX_SHORT_SUMS), w [K, N] in MXFP4, out [M, K] of out_dtype.  Products
 * are exact and the sums float32.  (An E4M3 element of a block whose scale is
 * below 2^-124 counts in multiples of 2^-133.) */
int nvm_mx_matmul(const void *a_codes, const uint8_t *a_scales, int64_t a_scale_ld, int a_format,
                  const void *w_codes, const uint8_t *w_scales, int64_t w_scale_ld, int64_t M,
                  int64_t N, int64_t K, int out_dtype, void *out, nvm_stream_t stream);

/* Gate and up products with SwiGLU and an MX output: with g and u the two
 * products of `a` as nvm_mx_matmul sums them, the MX codes (out_format) of
 * g / (1 + exp(-g)) * u, [M, K].  K a multiple of 32. */
int nvm_mx_swiglu(const void *a_codes, const uint8_t *a_scales, int64_t a_scale_ld, int a_format,
                  const void *gate_codes, const uint8_t *gate_scales, int64_t gate_scale_ld,
                  const void *up_codes, const uint8_t *up_scales, int64_t up_scale_ld, int64_t M,
                  int64_t N, int64_t K, int out_format, void *out_codes, uint8_t *out_scales,
                  int64_t out_scale_ld, nvm_stream_t stream);

/* The kernel that nvm_mx_matmul (gate_up 0) or nvm_mx_swiglu (1) runs for these
 * sizes on the current device.  plan[0]: 0 for few rows, 1 for some hundred, 2 for
 * many, -1 if there is nothing to compute; plan[1], plan[2]: a block's outputs (of
 * both matrices for gate_up) and rows; plan[3]: the parts that the tiles past whole
 * rounds are computed in, 2 or 4, or 0. */
int nvm_mx_product_plan(int gate_up, int64_t M, int64_t N, int64_t K, int a_format, int plan[4]);

#ifdef __cplusplus
}
#endif

#endif /* NVM_MX_H */
