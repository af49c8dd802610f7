// Shared by the kernels of paged attention over the 4-bit cache.
#pragma once

#include "common.h"
#include "mx_common.h"
#include "nvm_mx_cache.h"

namespace nvm {

struct MxAttnArgs {
  const void *q;
  int64_t q_sb, q_sh, q_sl;
  const uint8_t *kc, *ks, *vc, *vs;
  const int32_t *bt, *lens;
  void *out;
  int out_dt;
  int B, L, D, P, page_size, max_pages, Hkv, Hq, R, causal;
  float scale2;  // |scale| * log2(e): scores are kept in base 2
  uint32_t q_sign;  // the sign bits to flip in two 16-bit query parts, for a negative scale
  uint32_t ps_mul, ps_shift;  // position / page_size, see page_of
  int HG, S;                  // groups of query heads, most splits of a context
  float slots;                // blocks to be had for the splits, a kv head's group of query heads
  float *part_o, *part_ml;    // splits' outputs [row][S][D], maxima and sums [row][S][2]
};

// n / page_size of n below 2^31: with 2^(l-1) < page_size <= 2^l the factor is
// ceil(2^(31 + l) / page_size), off by less than 2^-31 of n, which no quotient
// notices (page_size 1: a factor of 0 stands for 2^32).
__device__ __forceinline__ int page_of(int n, uint32_t mul, uint32_t shift) {
  return mul ? (int)(__umulhi((uint32_t)n, mul) >> shift) : n;
}

__device__ __forceinline__ void store_out(void *out, int dt, int64_t i, float v) {
  if (dt == NVM_KV_F32)
    ((float *)out)[i] = v;
  else if (dt == NVM_KV_BF16)
    ((uint16_t *)out)[i] = Act<DT_BF16>::from_f32(v);
  else
    ((uint16_t *)out)[i] = Act<DT_F16>::from_f32(v);
}

// Four consecutive outputs, from element i on.
template <int DT>
__device__ __forceinline__ void store_out4(void *out, int64_t i, f32x4 v) {
  if constexpr (DT == NVM_KV_F32)
    *(f32x4 *)((float *)out + i) = v;
  else
    *(u32x2 *)((uint16_t *)out + i) =
        u32x2{Act<DT>::pack2(v[0], v[1]), Act<DT>::pack2(v[2], v[3])};
}

// 2^(x - m) with m the running maximum: nothing seen so far (m = -inf) counts as
// zero, so that a masked score gives 0 and a NaN stays one.
__device__ __forceinline__ float exp2_below(float x, float m) {
  return __builtin_amdgcn_exp2f(x - (m == -INFINITY ? 0.f : m));
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// A 4 x 16 block of 16-bit values in LDS, transposed: of a group of 16 lanes,
// lane i passes the address of values 4 (i % 4) .. + 3 of row i / 4 and gets
// column i.
__device__ __forceinline__ u32x2 lds_read_tr(const uint16_t *p) {
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p));
}

template <int QT>
constexpr int kParts = QT == NVM_KV_F32 ? 3 : QT == NVM_KV_F16 ? 2 : 1;

// Eight query values as bf16 parts whose sum they are.
template <int QT>
__device__ __forceinline__ void query8(const void *q, int64_t i, u32x4 (&p)[kParts<QT>]) {
  using A = Act<DT_BF16>;
  if constexpr (QT == NVM_KV_BF16) {
    p[0] = ldg16((const uint16_t *)q + i);
  } else {
    float x[8];
    if constexpr (QT == NVM_KV_F32) {
      const f32x4 a = *(const f32x4 *)((const float *)q + i);
      const f32x4 b = *(const f32x4 *)((const float *)q + i + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
    } else {
      const u32x4 a = ldg16((const uint16_t *)q + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[2 * j] = Act<DT_F16>::lo(a[j]), x[2 * j + 1] = Act<DT_F16>::hi(a[j]);
    }
#pragma unroll
    for (int k = 0; k < kParts<QT>; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[k][j] = A::pack2(x[2 * j], x[2 * j + 1]);
        x[2 * j] -= A::lo(p[k][j]);
        x[2 * j + 1] -= A::hi(p[k][j]);
      }
  }
}

// Eight codes times a scale (a float of that exponent), as an MFMA operand.
__device__ __forceinline__ u32x4 codes_bf16(uint32_t d, float s) {
  return u32x4{mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 0)),
               mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 1)),
               mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 2)),
               mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 3))};
}

// N dwords from p, 4 N-byte aligned.
template <int N>
__device__ __forceinline__ void load_dwords(const uint8_t *p, uint32_t (&d)[N]) {
  static_assert(N == 2 || N == 4, "a load");
  if constexpr (N == 4) {
    const u32x4 v = ldg16_once(p);
    d[0] = v.x, d[1] = v.y, d[2] = v.z, d[3] = v.w;
  } else {
    const u32x2 v = __builtin_nontemporal_load((const u32x2 *)p);
    d[0] = v.x, d[1] = v.y;
  }
}

__device__ __forceinline__ int context_of(const MxAttnArgs &a, int len) {
  return (int)max((int64_t)0, min((int64_t)len, (int64_t)a.max_pages * a.page_size));
}

// Several query rows a request (mx_prefill.hip): blocks of a kv head's columns, and
// the launch (D of 64 or 128; splits' outputs as those of single rows).
int64_t mx_prefill_blocks(int64_t L, int64_t R);
hipError_t launch_mx_prefill(int q_dtype, const MxAttnArgs &a, hipStream_t st);

}  // namespace nvm
