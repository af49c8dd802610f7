// Microscaled formats on the device (include/nvm_mx.h): rounding of a block,
// and the scaled matrix instruction's operands.
#pragma once

#include "common.h"
#include "nvm_mx.h"

namespace nvm {

// Activations of the products: an nvm_mx_format, or E4M3 summed by the scaled
// matrix instruction (NVM_MX_SHORT_SUMS).
constexpr int kMxShort = 2;

template <int FMT>
struct Mx {
  static constexpr int kEmax = FMT == NVM_MX_FP4 ? 2 : 8;  // exponent of the largest element
  static constexpr int kBits = FMT == NVM_MX_FP4 ? 4 : 8;
  static constexpr int kMfma = FMT == NVM_MX_FP4 ? 4 : 0;  // the instruction's format code
};

// Scale byte of a block from the float32 bits of its largest magnitude.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23);
  return e == 255 ? 255u : (uint32_t)max(0, e - Mx<FMT>::kEmax);
}
// 2^(127 - b), the factor that takes values to elements (b = 255, a block
// with a NaN or an infinity: zero; its codes do not come from the products).
__device__ __forceinline__ float mx_factor(uint32_t b) {
  return b == 255u ? 0.f : __uint_as_float((254u - b) << 23);
}
// 2^(b - 127); NaN for 255.
__device__ __forceinline__ float mx_scale(uint32_t b) {
  return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7FC00000u : b << 23);
}

// Eight values to element codes (FP4: one dword, FP8: two).  x * factor is
// exact (a power of two; results below float32's normal range round to zero
// either way); the conversions round to nearest even.  E2M1 saturates in the
// conversion, E4M3 is clamped before it (a conversion of larger values gives
// NaN).  `bad`: a block of NaNs or infinities, whose codes are zero.
template <int FMT>
__device__ __forceinline__ u32x2 mx_encode8(const float (&x)[8], float factor, bool bad) {
  u32x2 o = {0u, 0u};
  if constexpr (FMT == NVM_MX_FP4) {
    uint32_t d = 0;
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, x[0] * factor, x[1] * factor, 1.0f, 0);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, x[2] * factor, x[3] * factor, 1.0f, 1);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, x[4] * factor, x[5] * factor, 1.0f, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, x[6] * factor, x[7] * factor, 1.0f, 3);
    o.x = bad ? 0u : d;
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_amdgcn_fmed3f(x[i] * factor, -448.f, 448.f);
    int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], a, true);
    int b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], b, true);
    o.x = bad ? 0u : (uint32_t)a;
    o.y = bad ? 0u : (uint32_t)b;
  }
  return o;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Largest magnitude of eight values, as float32 bits (NaNs and infinities
// come out largest).
__device__ __forceinline__ uint32_t absmax8(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(x[i]));
  return m;
}

// Operands of a 16 x 16 x 128 product, row or column lane % 16.  Lane group G =
// lane / 16 passes the scale of k-values 32 G .. 32 G + 31, and holds these, 16
// bytes of E2M1 or 32 of E4M3.  Only where E4M3 goes into the scaled matrix
// instruction (kMxShort) that wants k-values 16 G .. + 15 and 64 + 16 G .. + 15
// in the lane, 16 bytes each.
typedef int mx_operand __attribute__((ext_vector_type(8)));

template <int FMT>
struct MxFrag {
  u32x4 v[FMT == NVM_MX_FP4 ? 1 : 2];
  __device__ __forceinline__ mx_operand operand() const {
    if constexpr (FMT == NVM_MX_FP4)
      return mx_operand{(int)v[0].x, (int)v[0].y, (int)v[0].z, (int)v[0].w, 0, 0, 0, 0};
    else
      return mx_operand{(int)v[0].x, (int)v[0].y, (int)v[0].z, (int)v[0].w,
                        (int)v[1].x, (int)v[1].y, (int)v[1].z, (int)v[1].w};
  }
};

// The first k-value of load c of a lane's activations, from the step's first on.
template <int FMT>
__device__ __forceinline__ int mx_act_at(int G, int c) {
  return FMT == NVM_MX_FP4 ? 32 * G : FMT == NVM_MX_FP8 ? 32 * G + 16 * c : 64 * c + 16 * G;
}

// c += w . x^T: rows (4 G + i of c) from the FP4 weights, columns (lane % 16)
// from the activations; the scales are byte BYTE of ws and xs.  In one scaled
// matrix instruction, v_mfma_scale_f32_16x16x128_f8f6f4.  It adds eight products
// as integers in units of 2^-13 of the largest: E2M1 by E2M1 fits into that
// (2^-2 to 36 in multiples of 2^-2), of E4M3 by E2M1 the small ones are lost,
// 2^-17 to 2^-15 of a layer's sums.  So E4M3 comes here only if the caller asked for it.
template <int FMT, int BYTE = 0>
__device__ __forceinline__ f32x4 mx_mfma(const MxFrag<NVM_MX_FP4> &w, uint32_t ws,
                                         const MxFrag<FMT> &x, uint32_t xs, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      w.operand(), x.operand(), c, Mx<NVM_MX_FP4>::kMfma, Mx<FMT>::kMfma, BYTE, (int)ws, BYTE,
      (int)xs);
}

// E4M3 by E2M1 with float32 sums: operands as bf16, in which an element times its
// scale is exact (4 bits, and bf16 has float32's exponents; below its subnormals,
// 2^-133, an element is rounded), and whose products are exact in float32.  Four
// v_mfma_f32_16x16x32_bf16, 64 cycles for the scaled instruction's 32, and a
// conversion for two values (4 cycles, beside the other wavefront's products).

// 2^(b - 127) of byte BYTE of a dword of scales, for the conversions: they take
// a float's exponent alone (of zero 2^-127, of 255 NaN).
template <int BYTE>
__device__ __forceinline__ float mx_scale_of(uint32_t s) {
  return __uint_as_float((s >> (8 * BYTE) & 255u) << 23);
}
template <class V>
__device__ __forceinline__ uint32_t mx_bits(V v) {
  static_assert(sizeof(V) == 4, "a dword");
  return __builtin_bit_cast(uint32_t, v);
}
// Values 8 i .. + 7 of the lane's 32 of a step.
__device__ __forceinline__ u32x4 mx_bf16(const MxFrag<NVM_MX_FP4> &q, int i, float s) {
  const uint32_t d = q.v[0][i];
  return u32x4{mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 0)),
               mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 1)),
               mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 2)),
               mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 3))};
}
__device__ __forceinline__ u32x4 mx_bf16(const MxFrag<NVM_MX_FP8> &q, int i, float s) {
  const uint32_t a = q.v[i >> 1][2 * (i & 1)], b = q.v[i >> 1][2 * (i & 1) + 1];
  return u32x4{mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false)),
               mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true)),
               mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, false)),
               mx_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, true))};
}

// acc[f][t] += w[f] . x[t]^T for all f and t, by either of the two; beside(i) is
// called before part i of the mx_parts that the products are cut into.  (The bf16
// operands are made a quarter of a step at a time: all of them need more
// registers than there are beside 8 x 4 sums.)
template <int FMT, int TF>
constexpr int mx_parts = FMT == NVM_MX_FP8 ? 4 * TF : TF;

template <int FMT, int BYTE, int TF, int TM, class F>
__device__ __forceinline__ void mx_products(const MxFrag<NVM_MX_FP4> (&w)[TF],
                                            const uint32_t (&ws)[TF], const MxFrag<FMT> (&x)[TM],
                                            const uint32_t (&xs)[TM], f32x4 (&acc)[TF][TM],
                                            F beside) {
  if constexpr (FMT == NVM_MX_FP8) {
    float wf[TF], xf[TM];
#pragma unroll
    for (int f = 0; f < TF; ++f) wf[f] = mx_scale_of<BYTE>(ws[f]);
#pragma unroll
    for (int t = 0; t < TM; ++t) xf[t] = mx_scale_of<BYTE>(xs[t]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 xb[TM];
#pragma unroll
      for (int t = 0; t < TM; ++t) xb[t] = mx_bf16(x[t], i, xf[t]);
#pragma unroll
      for (int f = 0; f < TF; ++f) {
        beside(i * TF + f);
        const u32x4 wb = mx_bf16(w[f], i, wf[f]);
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[f][t] = Act<DT_BF16>::mfma16(wb, xb[t], acc[f][t]);
      }
    }
  } else {
#pragma unroll
    for (int f = 0; f < TF; ++f) {
      beside(f);
#pragma unroll
      for (int t = 0; t < TM; ++t)
        acc[f][t] = mx_mfma<FMT, BYTE>(w[f], ws[f], x[t], xs[t], acc[f][t]);
    }
  }
}

// g / (1 + exp(-g)) * u.  exp(-g) = 2^t (1 + d ln 2) with t = -g log2(e) rounded
// and d what was left of it, the rest of log2(e) beyond a float32 included (without
// that the error grows with g, to 2^-19.7 at -87).  2^t is v_exp_f32 and the quotient
// v_rcp_f32, 1 ulp each, so 2^-20.8 in all, in 12 instructions for the 30 of the
// library's exp and division.  The quotient is taken of a quarter of the sum: of more
// than 2^126 v_rcp_f32 gives zero.  Where exp overflows (g below -88.7) so does the
// result.  Gates beyond 200 count as 200 in t, where 2^t is 0 or infinity already:
// g log2(e) itself may leave float32's range.  NaNs go through.
__device__ __forceinline__ float mx_swiglu(float g, float u) {
  constexpr float kL = -0x1.715476p+0f, kLow = -0x1.4ae0cp-26f, kLn2 = 0.69314718056f;
  const float c = __builtin_amdgcn_fmed3f(g, -200.f, 200.f);
  const float t = c * kL, d = __builtin_fmaf(c, kLow, __builtin_fmaf(c, kL, -t));
  const float e = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(d, kLn2, 1.f);
  return 0.25f * g * __builtin_amdgcn_rcpf(__builtin_fmaf(0.25f, e, 0.25f)) * u;
}

// Arguments of the products (gate/up: two weights, MX output).
struct MxMatmulArgs {
  const uint8_t *a, *as;  // activations [M][N], scales
  const uint8_t *w[2], *ws[2];
  int64_t as_ld, ws_ld[2];
  int64_t M;
  int N, K;
  int out_dtype;  // products: nvm_mx_dtype
  void *out;      // [M][K], or MX codes
  uint8_t *out_s;
  int64_t out_sld;
};
// The products for few rows (mx_gemv.hip, with the block's `tile` that
// mx_gemv_time names: of those that a launch takes the one of the least time, which
// it returns in us, infinity if there is none; columns and rows: its outputs, for
// gate/up of both matrices, and rows), for some (mx_gemm_pipe.hip, in tiles of bn
// outputs by bm rows) and for many (mx_gemm.hip: 256 by 256, those past whole
// rounds in `parts`: 0, 2 or 4, a part a block), of at most kMxMaxTiles output
// tiles.  hipErrorInvalidConfiguration: more than a launch takes.
constexpr int64_t kMxMaxTiles = 1 << 22;
struct MxBlock {
  int tile, columns, rows;
};
double mx_gemv_time(int format, bool dual, int64_t M, int N, int K, MxBlock *block);
hipError_t launch_mx_gemv(int format, int tile, bool dual, int out_format, const MxMatmulArgs &a,
                          hipStream_t st);
hipError_t launch_mx_gemm_pipe(int format, int bn, int bm, bool dual, int out_format,
                               const MxMatmulArgs &a, hipStream_t st);
hipError_t launch_mx_gemm(int format, int parts, bool dual, int out_format, const MxMatmulArgs &a,
                          hipStream_t st);

// f(integral constant) of an output type.
template <int V>
struct MxInt {
  static constexpr int value = V;
};
template <class F>
__host__ __device__ __forceinline__ void mx_by_dtype(int dtype, F f) {
  if (dtype == NVM_MX_F32)
    f(MxInt<NVM_MX_F32>{});
  else if (dtype == NVM_MX_BF16)
    f(MxInt<NVM_MX_BF16>{});
  else
    f(MxInt<NVM_MX_F16>{});
}

// Outputs k .. k + 3 of a row whose first is element `row` of out; those
// below `end` are stored.
template <int DT>
__device__ __forceinline__ void mx_store4(void *out, int64_t row, int k, int end, f32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (k + e >= end) break;
    if constexpr (DT == NVM_MX_F32)
      ((float *)out)[row + k + e] = v[e];
    else
      ((uint16_t *)out)[row + k + e] = Act<DT>::from_f32(v[e]);
  }
}

// Two neighbouring 16-row weight tiles' outputs of one activation row, from
// output k on: lane group G holds v0 = outputs 4 G .. + 3 and v1 = 16 + 4 G ..
// + 3.  Rows are a multiple of eight outputs, and so is `end`.  16-bit
// outputs trade places first (v_permlane16_swap: lane groups 1 and 3 of the
// first with 0 and 2 of the second), which leaves a lane with eight
// neighbours, 16 bytes: groups 0 and 2 of the first tile, 1 and 3 of the
// second.  Every lane of the wavefront is active.
template <int DT>
__device__ __forceinline__ void mx_store_pair(void *out, int G, int64_t row, int k, int end,
                                              f32x4 v0, f32x4 v1) {
  if constexpr (DT == NVM_MX_F32) {
    float *o = (float *)out + row + k + 4 * G;
    if (k + 4 * G < end) *(f32x4 *)o = v0;
    if (k + 16 + 4 * G < end) *(f32x4 *)(o + 16) = v1;
  } else {
    using A = Act<DT>;
    const auto a = __builtin_amdgcn_permlane16_swap(A::pack2(v0[0], v0[1]), A::pack2(v1[0], v1[1]),
                                                    false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(A::pack2(v0[2], v0[3]), A::pack2(v1[2], v1[3]),
                                                    false, false);
    k += 16 * (G & 1) + 8 * (G >> 1);
    if (k < end) *(u32x4 *)((uint16_t *)out + row + k) = u32x4{a[0], b[0], a[1], b[1]};
  }
}

// One block of 32 MX outputs of row m, from column k on: lane group G holds
// values 4 G .. + 3 and 16 + 4 G .. + 3 (h[0..3], h[4..7]).  The codes trade
// places as above, so a lane stores eight neighbours.  Every lane of the
// wavefront is active; `on`: the block is inside the output.
template <int OFMT>
__device__ __forceinline__ void mx_store_block(const float (&h)[8], int G, bool on, int64_t m,
                                               int k, const MxMatmulArgs &p) {
  uint32_t mx = absmax8(h);
  mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16));
  mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
  const uint32_t b = mx_scale_byte<OFMT>(mx);
  const u32x2 o = mx_encode8<OFMT>(h, mx_factor(b), b == 255u);
  const int64_t i = (m * p.K + k) / 8 + 2 * (G & 1) + (G >> 1);  // eight outputs
  if constexpr (OFMT == NVM_MX_FP4) {
    const auto a = __builtin_amdgcn_permlane16_swap(o.x & 0xFFFFu, o.x >> 16, false, false);
    if (on) ((uint32_t *)p.out)[i] = a[0] | (a[1] << 16);
  } else {
    const auto a = __builtin_amdgcn_permlane16_swap(o.x, o.y, false, false);
    if (on) ((u32x2 *)p.out)[i] = u32x2{a[0], a[1]};
  }
  if (on && G == 0) p.out_s[m * p.out_sld + k / 32] = (uint8_t)b;
}

}  // namespace nvm
