/*
 * C ABI of the 4-bit KV cache: the step that rotates and stores keys and
 * values, what stored rows stand for, and attention over them.  In the same
 * library and with the same conventions as nvm_moe.h: device pointers, work on
 * `stream`, no host synchronisation, no device allocation (callers pass
 * outputs and the workspace), NVM_OK or a negative NVM_ERR_* status (message
 * in nvm_last_error()).
 *
 * Pages hold MXFP4 as nvm_mx.h defines it, in blocks of 32 consecutive values
 * of a head's row:
 *   codes   [P, num_kv_heads, page_size, D / 2]   E2M1, two a byte, the even
 *           value in the low half
 *   scales  [P, num_kv_heads, page_size, D / 32]  E8M0 bytes, 255 for NaN
 * both contiguous and 16-byte aligned, for keys and for values: 4.25 bits a
 * value.  D is a multiple of 32, at most 256.  A pool may be larger than 4
 * GiB, with P * num_kv_heads * page_size below 2^31.
 */
#ifndef NVM_MX_CACHE_H
#define NVM_MX_CACHE_H

#include "nvm_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * nvm_qk_norm_rope_store into 4-bit pages: per head, RMSNorm of q and k with
 * q_norm_w/k_norm_w and rotation of both (halves i and i + D/2, by the float32
 * tables cos/sin[position][D/2]); k and v quantised into their slots, q handed
 * on.
 *   qkv          [T, (Hq + 2 Hkv) * D] of `dtype` (NVM_DTYPE_F16 or _BF16,
 *                16-byte aligned): q heads, then k heads, then v heads
 *   positions    [T] int32 (clamped into [0, max_pos)); cos, sin [max_pos, D/2]
 *   page_ids, slots [T] int32: where token t's k and v go.  Page ids outside
 *                [0, P) and slots outside [0, page_size) are not stored.  What
 *                a slot holds that two tokens name is not specified.
 *   q_out        [T, Hq, D], k_out and v_out [T, Hkv, D] or NULL, of out_dtype
 *                (NVM_KV_F32, or the code of `dtype`), 16-byte aligned: values
 *                rounded once to `dtype` (as stored pages are not)
 * q is computed in float32; k in float64 up to its quantisation, without a
 * rounding to `dtype` before it.
 */
int nvm_qk_norm_rope_store_mx(const void *qkv, int64_t T, int Hq, int Hkv, int64_t D,
                              const void *q_norm_w, const void *k_norm_w, float eps,
                              const int32_t *positions, const float *cos, const float *sin,
                              int64_t max_pos, const int32_t *page_ids, const int32_t *slots,
                              void *key_codes, uint8_t *key_scales, void *value_codes,
                              uint8_t *value_scales, int64_t P, int64_t page_size, int dtype,
                              int out_dtype, void *q_out, void *k_out, void *v_out,
                              nvm_stream_t stream);

/*
 * What stored rows stand for: k_out[t, h] and v_out[t, h] [T, Hkv, D] of slot
 * (page_ids[t], slots[t]), rounded once to out_dtype (NVM_KV_F16, NVM_KV_BF16
 * or NVM_KV_F32; 16-byte aligned).  Slots that are not there give zeros.
 */
int nvm_paged_kv_read_mx(const void *key_codes, const uint8_t *key_scales,
                         const void *value_codes, const uint8_t *value_scales, int64_t P, int Hkv,
                         int64_t page_size, int64_t D, const int32_t *page_ids,
                         const int32_t *slots, int64_t T, int out_dtype, void *k_out, void *v_out,
                         nvm_stream_t stream);

/*
 * nvm_paged_attention over 4-bit pages: out = softmax(q . key^T * scale) .
 * value, per query row; positions, absent pages, page ids >= P, causal bounds
 * and rows that see nothing as there.
 *   q    row i of request b's query head h: D consecutive values of q_dtype
 *        (NVM_KV_F16, NVM_KV_BF16 or NVM_KV_F32) from q + b * q_stride_b + h *
 *        q_stride_h + i * q_stride_l on (strides in values; rows 16-byte
 *        aligned)
 *   out  [B, L, num_heads, D] of out_dtype (the same three)
 * Codes times scales are exact, so are the products with q, and sums are
 * float32.  For D of 64 or 128 the softmax weights go into the product with the
 * values as two bf16 parts (2^-17 of each weight), whatever out_dtype is.
 * Workspace: nvm_paged_attention_mx_workspace_size, on the device that the call
 * runs on (zero bytes if no context is split; workspace may then be NULL).
 */
int nvm_paged_attention_mx_workspace_size(int64_t B, int64_t L, int64_t D, int64_t max_pages,
                                          int64_t page_size, int num_kv_heads, int num_heads,
                                          size_t *bytes);
int nvm_paged_attention_mx(const void *q, int q_dtype, int64_t q_stride_b, int64_t q_stride_h,
                           int64_t q_stride_l, int64_t B, int64_t L, int64_t D,
                           const void *key_codes, const uint8_t *key_scales,
                           const void *value_codes, const uint8_t *value_scales, int64_t P,
                           int64_t page_size, const int32_t *block_table, int64_t max_pages,
                           const int32_t *context_lens, float scale, int is_causal,
                           int num_kv_heads, int num_heads, int out_dtype, void *out,
                           void *workspace, size_t workspace_bytes, nvm_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* NVM_MX_CACHE_H */
