// Microscaled quantisation, its inverse, and the residual add + RMSNorm with
// an MX output (declared in include/nvm_mx.h).
//
// All three are one pass over the data.  A thread owns eight consecutive
// values, four neighbouring lanes one block: the block's largest magnitude is
// two quad swaps away.  Bound: HBM (4096 x 4096 bf16 to MXFP8 10.2 us, 5.0 TB/s,
// a copy's rate), at the smallest sizes the launch (2.05 us).
#include <math.h>

#include "common.h"
#include "internal.h"
#include "mx_common.h"

namespace nvm {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxChunks = 0xFFFFFFFFll - kThreads + 1;  // threads of a launch: below 2^32

__device__ __forceinline__ uint32_t max4_lanes(uint32_t v) {
  v = max(v, dpp_u32<0xB1>(v));
  return max(v, dpp_u32<0x4E>(v));
}

// Codes and the scale byte of a lane's eight values (chunk c of a row's
// n / 8); every lane of the block's four is active.
template <int FMT>
__device__ __forceinline__ void store_block(const float (&x)[8], int64_t row, int c, int n8,
                                            void *codes, uint8_t *scales, int64_t sld) {
  const uint32_t b = mx_scale_byte<FMT>(max4_lanes(absmax8(x)));
  const u32x2 o = mx_encode8<FMT>(x, mx_factor(b), b == 255u);
  if constexpr (FMT == NVM_MX_FP4)
    ((uint32_t *)codes)[row * n8 + c] = o.x;
  else
    ((u32x2 *)codes)[row * n8 + c] = o;
  if ((c & 3) == 0) scales[row * sld + (c >> 2)] = (uint8_t)b;
}

template <int DT>
__device__ __forceinline__ void load8(const void *x, int64_t i, float (&v)[8]) {
  if constexpr (DT == NVM_MX_F32) {
    const f32x4 a = *(const f32x4 *)((const float *)x + i);
    const f32x4 b = *(const f32x4 *)((const float *)x + i + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  } else {
    const u32x4 a = ldg16((const uint16_t *)x + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = Act<DT>::lo(a[j]);
      v[2 * j + 1] = Act<DT>::hi(a[j]);
    }
  }
}

// (row, chunk) of a flat chunk index.  (The host takes at most 2^32 chunks, a
// launch's limit of threads: a 64-bit division is a long software sequence.)
__device__ __forceinline__ void split_index(uint32_t i, int n8, int64_t &row, int &c) {
  const uint32_t q = i / (uint32_t)n8;
  row = q;
  c = (int)(i - q * (uint32_t)n8);
}

template <int DT, int FMT>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(const void *x, uint32_t total,
                                                               int n8, int64_t x_ld, void *codes,
                                                               uint8_t *scales, int64_t sld) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= total) return;  // (whole blocks: n8 is a multiple of 4)
  int64_t row;
  int c;
  split_index(i, n8, row, c);
  float v[8];
  load8<DT>(x, row * x_ld + 8 * c, v);
  store_block<FMT>(v, row, c, n8, codes, scales, sld);
}

// The values of rows 0, 1, ..., or (IDS) of rows ids[0], ids[1], ... of a table of `table_rows`:
// of ids outside it zeros.
template <int FMT, int DT, bool IDS>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(
    const int32_t *ids, int table_rows, const void *codes, const uint8_t *scales, int64_t sld,
    uint32_t total, int n8, void *out) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= total) return;
  int64_t row;
  int c;
  split_index(i, n8, row, c);
  bool inside = true;
  if constexpr (IDS) {
    row = ids[row];
    inside = row >= 0 && row < table_rows;
    row = inside ? row : 0;
  }
  const int64_t at = IDS ? row * n8 + c : (int64_t)i;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  f32x2 p[4];
  if constexpr (FMT == NVM_MX_FP4) {
    const uint32_t d = ((const uint32_t *)codes)[at];
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 3);
  } else {
    const u32x2 d = ((const u32x2 *)codes)[at];
    p[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)d.x, false);
    p[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)d.x, true);
    p[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)d.y, false);
    p[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)d.y, true);
  }
  // (the products are exact down to float32's subnormals: 2^-9 * 2^-127)
  const float s = inside ? mx_scale(scales[row * sld + (c >> 2)]) : 0.f;
  if (IDS && !inside) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = f32x2{0.f, 0.f};
  }
  if constexpr (DT == NVM_MX_F32) {
    float *o = (float *)out + 8 * (int64_t)i;
    *(f32x4 *)o = f32x4{p[0].x * s, p[0].y * s, p[1].x * s, p[1].y * s};
    *(f32x4 *)(o + 4) = f32x4{p[2].x * s, p[2].y * s, p[3].x * s, p[3].y * s};
  } else {
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = Act<DT>::pack2(p[j].x * s, p[j].y * s);
    *(u32x4 *)((uint16_t *)out + 8 * (int64_t)i) = o;
  }
}

// Residual add, RMSNorm and quantisation, a row per block of NT threads of NC
// 8-value chunks; every load of the row, of the residual and of the weights
// goes out before the first is used.  The sum of squares, its root and the
// scaled values are float64: squares of 16-bit values are exact there, and
// an E4M3 or E2M1 rounding border is then missed by 2^-52 instead of the
// sum's 2^-22 (one value in some 10^5 changed its code).  Bound: HBM and the
// ramp (4096 x 2048 14.9 us, 4.0 TB/s; 16384 x 2048 46 us, 5.1 TB/s), at few rows
// latency: 8 rows of 2048 in 2.65 us, with 128 threads of two chunks 3.4, with
// 64 of four 4.4.
template <int DT, int FMT, int NT, int NC>
__global__ __launch_bounds__(NT) void residual_rms_norm_mx_kernel(
    const uint16_t *h, const uint16_t *r, const uint16_t *w, int H8, float eps, uint16_t *h_out,
    void *codes, uint8_t *scales, int64_t sld) {
  using A = Act<DT>;
  __shared__ double s_part[NT / 64];
  hoist_args(h, r, w, H8, eps, h_out, codes, scales, sld);
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const rsrc_t hr = make_rsrc(h + row * H8 * 8, (uint32_t)H8 * 16);
  const rsrc_t rr = make_rsrc(r ? r + row * H8 * 8 : h, r ? (uint32_t)H8 * 16 : 0u);
  const rsrc_t wr = make_rsrc(w, (uint32_t)H8 * 16);
  u32x4 hv[NC], rv[NC], wv[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) hv[k] = bload16(hr, 16 * (tid + k * NT), 0);
#pragma unroll
  for (int k = 0; k < NC; ++k) rv[k] = bload16(rr, 16 * (tid + k * NT), 0);
#pragma unroll
  for (int k = 0; k < NC; ++k) wv[k] = bload16(wr, 16 * (tid + k * NT), 0);
  __builtin_amdgcn_sched_barrier(0);
  double ss = 0.0;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = tid + k * NT;
    if (r) {  // uniform
#pragma unroll
      for (int j = 0; j < 4; ++j)
        hv[k][j] = A::pack2(A::lo(hv[k][j]) + A::lo(rv[k][j]), A::hi(hv[k][j]) + A::hi(rv[k][j]));
      if (c < H8) *(u32x4 *)(h_out + (row * H8 + c) * 8) = hv[k];
    }
    // (chunks past the row's end were read as zeros)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double a = A::lo(hv[k][j]), b = A::hi(hv[k][j]);
      ss = fma(a, a, fma(b, b, ss));
    }
  }
  double tot = wave_reduce_f64(ss, [](double a, double b) { return a + b; });
  if constexpr (NT > 64) {
    if ((tid & 63) == 0) s_part[tid >> 6] = tot;
    __syncthreads();
    tot = s_part[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) tot += s_part[i];
  }
  // 1 / sqrt, from v_rsq_f64's 2^-14 or better to float64 in two steps (an
  // infinite sum keeps the instruction's zero: finite / inf)
  const double m = tot / (8.0 * H8) + (double)eps;
  double inv = __builtin_amdgcn_rsq(m);
  if (m < INFINITY) {
#pragma unroll
    for (int i = 0; i < 2; ++i) inv = inv * fma(-0.5 * m * inv, inv, 1.5);
  }
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = tid + k * NT;
    if (c >= H8) break;
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = round_to_odd((double)A::lo(hv[k][j]) * inv * (double)A::lo(wv[k][j]));
      v[2 * j + 1] = round_to_odd((double)A::hi(hv[k][j]) * inv * (double)A::hi(wv[k][j]));
    }
    store_block<FMT>(v, row, c, H8, codes, scales, sld);
  }
}

constexpr int kNormMaxH = 8192;
constexpr int64_t kNormMaxT = 0xFFFFFF;  // (blocks of 256 threads, below 2^32 in all)

template <int DT, int FMT>
void launch_norm_mx(const void *h, const void *r, const void *w, int64_t T, int64_t H, float eps,
                    void *h_out, void *codes, uint8_t *scales, int64_t sld, hipStream_t st) {
  auto go = [&](auto kern, int nt) {
    hipLaunchKernelGGL(kern, dim3((unsigned)T), dim3(nt), 0, st, (const uint16_t *)h,
                       (const uint16_t *)r, (const uint16_t *)w, (int)(H / 8), eps,
                       (uint16_t *)h_out, codes, scales, sld);
  };
  if (H <= 512)
    go(residual_rms_norm_mx_kernel<DT, FMT, 64, 1>, 64);
  else if (H <= 2048)
    go(residual_rms_norm_mx_kernel<DT, FMT, 256, 1>, 256);
  else if (H <= 4096)
    go(residual_rms_norm_mx_kernel<DT, FMT, 256, 2>, 256);
  else
    go(residual_rms_norm_mx_kernel<DT, FMT, 256, 4>, 256);
}

// f(integral constant) of a format.
template <class F>
void by_format(int format, F f) {
  if (format == NVM_MX_FP4)
    f(MxInt<NVM_MX_FP4>{});
  else
    f(MxInt<NVM_MX_FP8>{});
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int mx_check_rows(const char *op, int64_t rows, int64_t n, int format, const char *what) {
  if (format != NVM_MX_FP4 && format != NVM_MX_FP8)
    return set_error(NVM_ERR_INVALID, "%s: %s format must be mxfp4 or mxfp8", op, what);
  if (rows < 0 || n <= 0 || n % 32)
    return set_error(NVM_ERR_INVALID, "%s: bad shape of %s: %lld rows of %lld values (a multiple "
                     "of 32)", op, what, (long long)rows, (long long)n);
  if (n > kMxMaxRow || rows > INT32_MAX)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: %s of %lld rows of %lld values is too large", op,
                     what, (long long)rows, (long long)n);
  return NVM_OK;
}

int mx_check_tensor(const char *op, const void *codes, const uint8_t *scales, int64_t scale_ld,
                    int64_t n, const char *what) {
  if (!codes || !scales) return set_error(NVM_ERR_INVALID, "%s: null pointer (%s)", op, what);
  if (!aligned16(codes) || !aligned16(scales))
    return set_error(NVM_ERR_INVALID, "%s: codes and scales of %s must be 16-byte aligned", op,
                     what);
  const int64_t need = (n / 32 + 15) / 16 * 16;
  if (scale_ld % 16 || scale_ld < need || scale_ld > kMxMaxRow)
    return set_error(NVM_ERR_INVALID, "%s: scale rows of %s must be a multiple of 16 bytes apart, "
                     "at least %lld, got %lld", op, what, (long long)need, (long long)scale_ld);
  return NVM_OK;
}

// Values of `rows` rows (all of the tensor's, or those that ids names) to out.
static int mx_rows(const char *op, const int32_t *ids, int64_t rows, const void *codes,
                   const uint8_t *scales, int64_t scale_ld, int64_t table_rows, int64_t n,
                   int format, int dtype, void *out, hipStream_t st) {
  if (dtype != NVM_MX_F16 && dtype != NVM_MX_BF16 && dtype != NVM_MX_F32)
    return set_error(NVM_ERR_INVALID, "%s: dtype must be f16, bf16 or f32", op);
  if (int rc = mx_check_rows(op, table_rows, n, format, "input")) return rc;
  if (rows == 0) return NVM_OK;
  if (int rc = mx_check_tensor(op, codes, scales, scale_ld, n, "input")) return rc;
  if (!out || !aligned16(out))
    return set_error(NVM_ERR_INVALID, "%s: out must be a 16-byte aligned pointer", op);
  const int64_t total = rows * (n / 8);
  if (total > kMaxChunks)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: more than 2^35 values in one call", op);
  const dim3 grid((unsigned)((total + kThreads - 1) / kThreads));
  mx_by_dtype(dtype, [&](auto D) {
    by_format(format, [&](auto F) {
      auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, st, ids, (int)table_rows, codes, scales,
                           scale_ld, (uint32_t)total, (int)(n / 8), out);
      };
      if (ids)
        go(mx_dequantize_kernel<decltype(F)::value, decltype(D)::value, true>);
      else
        go(mx_dequantize_kernel<decltype(F)::value, decltype(D)::value, false>);
    });
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

}  // namespace nvm

extern "C" {

int nvm_mx_quantize(const void *x, int64_t rows, int64_t n, int64_t x_ld, int dtype, int format,
                    void *codes, uint8_t *scales, int64_t scale_ld, nvm_stream_t stream) {
  using namespace nvm;
  const char *op = "mx_quantize";
  if (dtype != NVM_MX_F16 && dtype != NVM_MX_BF16 && dtype != NVM_MX_F32)
    return set_error(NVM_ERR_INVALID, "%s: dtype must be f16, bf16 or f32", op);
  if (int rc = mx_check_rows(op, rows, n, format, "output")) return rc;
  if (rows == 0) return NVM_OK;
  if (!x) return set_error(NVM_ERR_INVALID, "%s: null pointer (x)", op);
  if (int rc = mx_check_tensor(op, codes, scales, scale_ld, n, "output")) return rc;
  const int64_t size = dtype == NVM_MX_F32 ? 4 : 2;
  if (!aligned16(x) || x_ld < n || x_ld > (int64_t)1 << 40 || x_ld * size % 16)
    return set_error(NVM_ERR_INVALID, "%s: rows of x must be 16-byte aligned and not overlap", op);
  const int64_t total = rows * (n / 8);
  if (total > kMaxChunks)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: more than 2^35 values in one call", op);
  const dim3 grid((unsigned)((total + kThreads - 1) / kThreads));
  mx_by_dtype(dtype, [&](auto D) {
    by_format(format, [&](auto F) {
      hipLaunchKernelGGL((mx_quantize_kernel<decltype(D)::value, decltype(F)::value>), grid,
                         dim3(kThreads), 0, (hipStream_t)stream, x, (uint32_t)total, (int)(n / 8),
                         x_ld, codes, scales, scale_ld);
    });
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

int nvm_mx_dequantize(const void *codes, const uint8_t *scales, int64_t scale_ld, int64_t rows,
                      int64_t n, int format, int dtype, void *out, nvm_stream_t stream) {
  return nvm::mx_rows("mx_dequantize", nullptr, rows, codes, scales, scale_ld, rows, n, format,
                      dtype, out, (hipStream_t)stream);
}

int nvm_mx_embedding(const int32_t *ids, int64_t T, const void *codes, const uint8_t *scales,
                     int64_t scale_ld, int64_t V, int64_t n, int format, int dtype, void *out,
                     nvm_stream_t stream) {
  using namespace nvm;
  if (T < 0 || T > INT32_MAX || V <= 0)
    return set_error(NVM_ERR_INVALID, "mx_embedding: bad shape T=%lld V=%lld", (long long)T,
                     (long long)V);
  if (T > 0 && !ids) return set_error(NVM_ERR_INVALID, "mx_embedding: null pointer (ids)");
  return mx_rows("mx_embedding", ids, T, codes, scales, scale_ld, V, n, format, dtype, out,
                 (hipStream_t)stream);
}

int nvm_residual_rms_norm_mx(const void *h, const void *r, const void *w, int64_t T, int64_t H,
                             float eps, int dtype, void *h_out, int format, void *codes,
                             uint8_t *scales, int64_t scale_ld, nvm_stream_t stream) {
  using namespace nvm;
  const char *op = "residual_rms_norm_mx";
  if (dtype != NVM_DTYPE_F16 && dtype != NVM_DTYPE_BF16)
    return set_error(NVM_ERR_INVALID, "%s: dtype must be f16 or bf16", op);
  if (int rc = mx_check_rows(op, T, H, format, "output")) return rc;
  if (H > kNormMaxH || T > kNormMaxT)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: H at most %d, T at most %lld", op, kNormMaxH,
                     (long long)kNormMaxT);
  if (T == 0) return NVM_OK;
  if (!h || !w || (r && !h_out)) return set_error(NVM_ERR_INVALID, "%s: null pointer", op);
  if (int rc = mx_check_tensor(op, codes, scales, scale_ld, H, "output")) return rc;
  if (!aligned16(h) || !aligned16(r) || !aligned16(w) || !aligned16(h_out))
    return set_error(NVM_ERR_INVALID, "%s: h, r, w and h_out must be 16-byte aligned", op);
  by_format(format, [&](auto F) {
    if (dtype == NVM_DTYPE_BF16)
      launch_norm_mx<DT_BF16, decltype(F)::value>(h, r, w, T, H, eps, h_out, codes, scales,
                                                  scale_ld, (hipStream_t)stream);
    else
      launch_norm_mx<DT_F16, decltype(F)::value>(h, r, w, T, H, eps, h_out, codes, scales,
                                                 scale_ld, (hipStream_t)stream);
  });
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

}  // extern "C"
