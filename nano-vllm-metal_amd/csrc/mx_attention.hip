// Paged attention over the 4-bit cache (declared in include/nvm_mx_cache.h).
//
// mx_rows_kernel: any head dim, one wavefront per query row.  A position's row
//   of codes goes to a group of GL lanes (eight values, one dword, a lane), so
//   64 / GL positions are in flight side by side, each group with a running
//   maximum and sum of its own; the groups meet at the end.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal.h"
#include "mx_common.h"
#include "nvm_mx_cache.h"

namespace nvm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowThreads = 256;

struct MxAttnArgs {
  const void *q;
  int64_t q_sb, q_sh, q_sl;
  const uint8_t *kc, *ks, *vc, *vs;
  const int32_t *bt, *lens;
  void *out;
  int out_dt;
  int B, L, D, P, page_size, max_pages, Hkv, Hq, R, causal;
  float scale2;  // scale * log2(e): scores are kept in base 2
};

__device__ __forceinline__ void store_out(void *out, int dt, int64_t i, float v) {
  if (dt == NVM_KV_F32)
    ((float *)out)[i] = v;
  else if (dt == NVM_KV_BF16)
    ((uint16_t *)out)[i] = Act<DT_BF16>::from_f32(v);
  else
    ((uint16_t *)out)[i] = Act<DT_F16>::from_f32(v);
}

template <int QT>
__device__ __forceinline__ float q_at(const void *q, int64_t i) {
  if constexpr (QT == NVM_KV_F32) return ((const float *)q)[i];
  if constexpr (QT == NVM_KV_BF16) return Act<DT_BF16>::to_f32(((const uint16_t *)q)[i]);
  return Act<DT_F16>::to_f32(((const uint16_t *)q)[i]);
}

// 2^(x - m) with m the running maximum: nothing seen so far (m = -inf) counts as
// zero, so that a masked score gives 0 and a NaN stays one.
__device__ __forceinline__ float exp2_below(float x, float m) {
  return __builtin_amdgcn_exp2f(x - (m == -INFINITY ? 0.f : m));
}

__device__ __forceinline__ void values8(uint32_t d, float s, float (&v)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 0);
  const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 1);
  const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 2);
  const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 3);
  v[0] = p0.x * s, v[1] = p0.y * s, v[2] = p1.x * s, v[3] = p1.y * s;
  v[4] = p2.x * s, v[5] = p2.y * s, v[6] = p3.x * s, v[7] = p3.y * s;
}

template <int QT, int GL>
__global__ __launch_bounds__(kRowThreads) void mx_rows_kernel(MxAttnArgs a, int64_t rows) {
  constexpr int NG = 64 / GL;
  const int64_t row = (int64_t)blockIdx.x * (kRowThreads / 64) + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & (GL - 1), grp = (threadIdx.x & 63) / GL;
  const int h = (int)(row % a.Hq);
  const int64_t bl = row / a.Hq;
  const int i = (int)(bl % a.L), b = (int)(bl / a.L);
  const int kvh = h / a.R, n8 = a.D / 8;
  const bool on = lane < n8;
  const int64_t len = a.lens[b];
  const int64_t cap = min(len, (int64_t)a.max_pages * a.page_size);
  const int last = (int)(a.causal ? min(cap, i + len - a.L + 1) : cap);
  const int32_t *bt = a.bt + (int64_t)b * a.max_pages;
  float qv[8], ov[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    qv[j] = on ? q_at<QT>(a.q, b * a.q_sb + h * a.q_sh + i * a.q_sl + 8 * lane + j) : 0.f;
  float m = -INFINITY, l = 0.f;
  for (int j = grp; j < last; j += NG) {
    const int pg = bt[j / a.page_size];
    if (pg < 0 || pg >= a.P) continue;  // (a whole group)
    const int64_t at = ((int64_t)pg * a.Hkv + kvh) * a.page_size + j % a.page_size;
    float k[8], v[8];
    values8(on ? ((const uint32_t *)a.kc)[at * n8 + lane] : 0u,
            on ? mx_scale(a.ks[at * (n8 / 4) + (lane >> 2)]) : 0.f, k);
    values8(on ? ((const uint32_t *)a.vc)[at * n8 + lane] : 0u,
            on ? mx_scale(a.vs[at * (n8 / 4) + (lane >> 2)]) : 0.f, v);
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) dot = fmaf(qv[e], k[e], dot);
#pragma unroll
    for (int x = 1; x < GL; x <<= 1) dot += __shfl_xor(dot, x);
    const float sc = dot * a.scale2, m_new = fmaxf(m, sc);
    const float alpha = exp2_below(m, m_new), p = exp2_below(sc, m_new);
    l = fmaf(l, alpha, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) ov[e] = fmaf(ov[e], alpha, p * v[e]);
    m = m_new;
  }
#pragma unroll
  for (int x = GL; x < 64; x <<= 1) {
    const float mo = __shfl_xor(m, x), lo = __shfl_xor(l, x), mm = fmaxf(m, mo);
    const float f = exp2_below(m, mm), g = exp2_below(mo, mm);
    l = l * f + lo * g;
#pragma unroll
    for (int e = 0; e < 8; ++e) ov[e] = ov[e] * f + __shfl_xor(ov[e], x) * g;
    m = mm;
  }
  if (grp == 0 && on) {
    // (a row that sees nothing: zeros; a NaN stays one)
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      store_out(a.out, a.out_dt, row * a.D + 8 * lane + e, l == 0.f ? 0.f : ov[e] * inv);
  }
}

template <int QT>
hipError_t launch_rows(const MxAttnArgs &a, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.L * a.Hq;
  const unsigned grid = (unsigned)((rows + kRowThreads / 64 - 1) / (kRowThreads / 64));
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(grid), dim3(kRowThreads), 0, st, a, rows);
  };
  if (a.D <= 32)
    go(mx_rows_kernel<QT, 4>);
  else if (a.D <= 64)
    go(mx_rows_kernel<QT, 8>);
  else if (a.D <= 128)
    go(mx_rows_kernel<QT, 16>);
  else
    go(mx_rows_kernel<QT, 32>);
  return hipGetLastError();
}

constexpr int64_t kMaxRows = 0x3FFFFFF;  // query rows of a call: wavefronts of a launch

int check_shape(const char *op, int64_t B, int64_t L, int64_t D, int64_t max_pages,
                int64_t page_size, int Hkv, int Hq) {
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv)
    return set_error(NVM_ERR_INVALID, "%s: num_heads must be divisible by num_kv_heads", op);
  if (B < 0 || L < 1 || D < 1 || page_size < 1 || max_pages < 0)
    return set_error(NVM_ERR_INVALID, "%s: bad shape B=%lld L=%lld D=%lld page_size=%lld "
                     "max_pages=%lld", op, (long long)B, (long long)L, (long long)D,
                     (long long)page_size, (long long)max_pages);
  if (D % 32 || D > 256)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: head dim %lld must be a multiple of 32, at most 256",
                     op, (long long)D);
  // (positions are 32-bit, with room for a tile past the last)
  if (max_pages > 0x7FFF0000ll / page_size)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: context capacity too large", op);
  if (B > kMaxRows || L > kMaxRows || B * L > kMaxRows / Hq)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: too many query rows", op);
  return NVM_OK;
}

}  // namespace

}  // namespace nvm

extern "C" {

int nvm_paged_attention_mx_workspace_size(int64_t B, int64_t L, int64_t D, int64_t max_pages,
                                          int64_t page_size, int num_kv_heads, int num_heads,
                                          size_t *bytes) {
  using namespace nvm;
  constexpr const char *op = "paged_attention_mx";
  if (int rc = check_shape(op, B, L, D, max_pages, page_size, num_kv_heads, num_heads)) return rc;
  if (!bytes) return set_error(NVM_ERR_INVALID, "%s: null bytes", op);
  *bytes = 0;
  return NVM_OK;
}

int nvm_paged_attention_mx(const void *q, int q_dtype, int64_t q_stride_b, int64_t q_stride_h,
                           int64_t q_stride_l, int64_t B, int64_t L, int64_t D,
                           const void *key_codes, const uint8_t *key_scales,
                           const void *value_codes, const uint8_t *value_scales, int64_t P,
                           int64_t page_size, const int32_t *block_table, int64_t max_pages,
                           const int32_t *context_lens, float scale, int is_causal,
                           int num_kv_heads, int num_heads, int out_dtype, void *out,
                           void *workspace, size_t workspace_bytes, nvm_stream_t stream) {
  using namespace nvm;
  constexpr const char *op = "paged_attention_mx";
  auto plain = [](int dt) { return dt == NVM_KV_F16 || dt == NVM_KV_BF16 || dt == NVM_KV_F32; };
  if (!plain(q_dtype) || !plain(out_dtype))
    return set_error(NVM_ERR_INVALID, "%s: query and out dtypes must be f16, bf16 or f32", op);
  if (int rc = check_shape(op, B, L, D, max_pages, page_size, num_kv_heads, num_heads)) return rc;
  if (int rc = mx_check_pages(op, num_kv_heads, D, P, page_size, key_codes, key_scales,
                              value_codes, value_scales))
    return rc;
  if (B == 0) return NVM_OK;
  if (!q || !out || !context_lens || (max_pages > 0 && !block_table))
    return set_error(NVM_ERR_INVALID, "%s: null pointer", op);
  const int64_t unit = q_dtype == NVM_KV_F32 ? 4 : 8;  // values of 16 bytes
  if (((uintptr_t)q & 15) || q_stride_b % unit || q_stride_h % unit || q_stride_l % unit)
    return set_error(NVM_ERR_INVALID, "%s: query rows must be 16-byte aligned", op);
  MxAttnArgs a{};
  a.q = q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.q_sl = q_stride_l;
  a.kc = (const uint8_t *)key_codes;
  a.ks = key_scales;
  a.vc = (const uint8_t *)value_codes;
  a.vs = value_scales;
  a.bt = block_table;
  a.lens = context_lens;
  a.out = out;
  a.out_dt = out_dtype;
  a.B = (int)B;
  a.L = (int)L;
  a.D = (int)D;
  a.P = (int)P;
  a.page_size = (int)page_size;
  a.max_pages = (int)max_pages;
  a.Hkv = num_kv_heads;
  a.Hq = num_heads;
  a.R = num_heads / num_kv_heads;
  a.causal = is_causal ? 1 : 0;
  a.scale2 = scale * kLog2e;
  hipStream_t st = (hipStream_t)stream;
  (void)workspace;
  (void)workspace_bytes;
  const hipError_t e = q_dtype == NVM_KV_F32    ? launch_rows<NVM_KV_F32>(a, st)
                       : q_dtype == NVM_KV_BF16 ? launch_rows<NVM_KV_BF16>(a, st)
                                                : launch_rows<NVM_KV_F16>(a, st);
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

}  // extern "C"
