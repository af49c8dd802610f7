// Products of MX rows with MXFP4 weights: which kernel, and the entry points
// (include/nvm_mx.h).
#include <math.h>

#include "internal.h"
#include "mx_common.h"

namespace nvm {

// Tiles of the larger kernels (of outputs, for gate/up of both matrices', by
// rows), and the time of a launch: `fixed` + rounds over the CUs x (`start` +
// `row` x N / 2048) microseconds, for E2M1 activations, E4M3, and E4M3 in short
// sums (fitted; some 10 % off, more where the clock falls under the load, for all
// alike).  A step of the larger ones costs less for its outputs, but they leave
// more CUs idle.  In us on 256 x 256 in whole tiles, in parts (below), on 256 x
// 128, 128 x 128, 128 x 64 and 64 x 64:
//   E4M3
//   2048 -> 2048    512 rows   47.8   -    27.5  18.2  13.0  10.5
//                  1024 rows   48.5   -    28.0  19.2  13.9  15.3
//   2048 -> 5120    512 rows   48.2   -    29.0  19.5  24.2  20.1
//                  1536 rows   49.6   -    35.8  37.6  45.0
//                  4096 rows   97.0  73.7  87.5  95.1
//                  8192 rows  141.1 133.7 148.2 169.4
//   6144 -> 2048    512 rows  129.4   -    68.0  39.9  27.6  20.7
//                  1024 rows  127.4   -    68.2  41.2  30.2  32.5
//                  8192 rows  147.7   -   166.8 179.5
//   4096 -> 6144   3000 rows  176.1 127.5 142.5 142.4
//   8192 -> 8192   8192 rows  743     -   800   892
//   gate/up 2048 -> 6144
//                   128 rows    -     -    28.9  19.0  13.5
//                  1500 rows   97.5  75.5  82.2  84.5
//                  4096 rows  153     -   169   204
//   E4M3 in short sums
//   2048 -> 2048    512 rows    -     -     -    12.2   9.1   7.9
//                  1024 rows    -     -     -    12.7  10.0  11.2
//   2048 -> 5120    512 rows   24.0   -    17.2  13.2  16.6  15.4
//                  1536 rows   26.3   -    21.0  24.8
//                  4096 rows   48.9  44.4  47.0  59.0        (E2M1 42.0  35.8  35.7  46.3)
//                  8192 rows   77.3  73.1  78.7   -          (E2M1 67.1  61.7  61.8)
//   6144 -> 2048    512 rows    -     -     -    22.9  16.5  14.1
//                  4096 rows   57     -    45.5  54
//   4096 -> 6144   3000 rows   82.2  66.4  78.2   -
//   8192 -> 8192   8192 rows   367    -    424   553         (E2M1  293   -   350   420)
//   gate/up 2048 -> 6144
//                   128 rows   24.0   -    16.8  13.0   9.7
//                  1500 rows   50.5  40.4  46.0   -
//                  4096 rows   82     -    94.7  134
struct Tiles {
  int bn, bm;
  double fixed[3], start[3], row[3];  // by the activations: an nvm_mx_format or kMxShort
  double round(int format, int N) const { return start[format] + row[format] * (N / 2048.0); }
};
constexpr Tiles kBig = {256, 256, {3.0, 1.0, 3.0}, {4.5, 6.5, 7.5}, {14.0, 41.4, 15.5}};
constexpr Tiles kTiles[] = {{256, 128, {2.5, 1.0, 3.5}, {4.0, 5.6, 3.5}, {7.0, 20.7, 9.2}},
                            {128, 128, {1.0, 1.0, 1.5}, {4.0, 5.5, 4.0}, {4.1, 11.3, 6.3}},
                            {128, 64, {3.0, 1.0, 2.5}, {1.8, 4.3, 2.8}, {3.2, 7.1, 4.3}},
                            {64, 64, {3.5, 3.5, 3.5}, {1.0, 1.5, 0.9}, {2.1, 4.5, 3.1}}};

// The kernel of the least time, of those that take so many outputs.  Few rows: mx_gemv.hip (2048 -> 5120 of 128 rows
// 11.2 us, on 64 x 64 tiles 10.2, 64 rows 9.1 and 9.6), and 32 rows always: there
// reading the weights is more of the time than the fit knows (in short sums 2048 ->
// 151936 of 16 rows 42 us, on 256 x 128 49; gate/up 2912 -> 14240 of 27 rows 13.2
// and 17.4).
struct Choice {
  int kernel = -1;  // 0 mx_gemv.hip, 1 mx_gemm_pipe.hip, 2 mx_gemm.hip; -1: more outputs than any takes
  MxBlock block{};
  int parts = 0;
};
static Choice choose(int format, bool dual, int64_t M, int N, int K) {
  const int64_t columns = (int64_t)K * (dual ? 2 : 1), cus = cu_count() / 8 * 8;
  auto count = [&](const Tiles &t) {
    return (columns + t.bn - 1) / t.bn * ((M + t.bm - 1) / t.bm);
  };
  Choice c;
  const double few = mx_gemv_time(format, dual, M, N, K, &c.block);
  double least = few;
  if (few < INFINITY) {
    c.kernel = 0;
    if (M <= 32) return c;
  }
  auto take = [&](const Tiles &t, double time, int kernel, int parts) {
    if (time < least && count(t) <= kMxMaxTiles) {
      least = time;
      c = {kernel, {0, t.bn, t.bm}, parts};
    }
  };
  for (const Tiles &t : kTiles)
    if (!dual || t.bn != 64)
      take(t, t.fixed[format] + (count(t) + cus - 1) / cus * t.round(format, N), 1, 0);
  // A last round of 256 x 256 that no more than a quarter (half) of the CUs would
  // have is computed in parts, of 128 x 128 (256 x 128), by all of them.
  const int64_t n = count(kBig), rest = n % cus;
  const int parts = n < cus || rest == 0 || 2 * rest > cus ? 0 : 4 * rest > cus ? 2 : 4;
  take(kBig,
       kBig.fixed[format] + (parts ? n / cus : (n + cus - 1) / cus) * kBig.round(format, N) +
           (parts ? kTiles[parts == 4].round(format, N) : 0.0),
       2, parts);
  return c;
}

static hipError_t launch_mx_product(int format, bool dual, int out_format, const MxMatmulArgs &a,
                                    hipStream_t st) {
  const Choice c = choose(format, dual, a.M, a.N, a.K);
  if (c.kernel == 0) return launch_mx_gemv(format, c.block.tile, dual, out_format, a, st);
  if (c.kernel == 1)
    return launch_mx_gemm_pipe(format, c.block.columns, c.block.rows, dual, out_format, a, st);
  if (c.kernel == 2) return launch_mx_gemm(format, c.parts, dual, out_format, a, st);
  return hipErrorInvalidConfiguration;
}

// What the kernels take for an entry's a_format.
static int mx_activations(int a_format) {
  return a_format == (NVM_MX_FP8 | NVM_MX_SHORT_SUMS) ? kMxShort : a_format & ~NVM_MX_SHORT_SUMS;
}

}  // namespace nvm

extern "C" {

int nvm_mx_matmul(const void *a_codes, const uint8_t *a_scales, int64_t a_scale_ld, int a_format,
                  const void *w_codes, const uint8_t *w_scales, int64_t w_scale_ld, int64_t M,
                  int64_t N, int64_t K, int out_dtype, void *out, nvm_stream_t stream) {
  using namespace nvm;
  const char *op = "mx_matmul";
  if (out_dtype != NVM_MX_F16 && out_dtype != NVM_MX_BF16 && out_dtype != NVM_MX_F32)
    return set_error(NVM_ERR_INVALID, "%s: out_dtype must be f16, bf16 or f32", op);
  if (int rc = mx_check_rows(op, M, N, a_format & ~NVM_MX_SHORT_SUMS, "a")) return rc;
  if (int rc = mx_check_rows(op, K, N, NVM_MX_FP4, "w")) return rc;
  if (M == 0 || K == 0) return NVM_OK;
  if (int rc = mx_check_tensor(op, a_codes, a_scales, a_scale_ld, N, "a")) return rc;
  if (int rc = mx_check_tensor(op, w_codes, w_scales, w_scale_ld, N, "w")) return rc;
  if (!out || ((uintptr_t)out & 15))
    return set_error(NVM_ERR_INVALID, "%s: out must be a 16-byte aligned pointer", op);
  MxMatmulArgs a{};
  a.a = (const uint8_t *)a_codes;
  a.as = a_scales;
  a.as_ld = a_scale_ld;
  a.w[0] = (const uint8_t *)w_codes;
  a.ws[0] = w_scales;
  a.ws_ld[0] = w_scale_ld;
  a.M = M;
  a.N = (int)N;
  a.K = (int)K;
  a.out_dtype = out_dtype;
  a.out = out;
  const hipError_t e = launch_mx_product(mx_activations(a_format), false, NVM_MX_FP8, a, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: too many output tiles", op);
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

int nvm_mx_swiglu(const void *a_codes, const uint8_t *a_scales, int64_t a_scale_ld, int a_format,
                  const void *gate_codes, const uint8_t *gate_scales, int64_t gate_scale_ld,
                  const void *up_codes, const uint8_t *up_scales, int64_t up_scale_ld, int64_t M,
                  int64_t N, int64_t K, int out_format, void *out_codes, uint8_t *out_scales,
                  int64_t out_scale_ld, nvm_stream_t stream) {
  using namespace nvm;
  const char *op = "mx_swiglu";
  if (int rc = mx_check_rows(op, M, N, a_format & ~NVM_MX_SHORT_SUMS, "a")) return rc;
  if (int rc = mx_check_rows(op, K, N, NVM_MX_FP4, "gate and up")) return rc;
  if (int rc = mx_check_rows(op, M, K, out_format, "output")) return rc;
  if (M == 0) return NVM_OK;
  if (int rc = mx_check_tensor(op, a_codes, a_scales, a_scale_ld, N, "a")) return rc;
  if (int rc = mx_check_tensor(op, gate_codes, gate_scales, gate_scale_ld, N, "gate")) return rc;
  if (int rc = mx_check_tensor(op, up_codes, up_scales, up_scale_ld, N, "up")) return rc;
  if (int rc = mx_check_tensor(op, out_codes, out_scales, out_scale_ld, K, "output")) return rc;
  MxMatmulArgs a{};
  a.a = (const uint8_t *)a_codes;
  a.as = a_scales;
  a.as_ld = a_scale_ld;
  a.w[0] = (const uint8_t *)gate_codes;
  a.ws[0] = gate_scales;
  a.ws_ld[0] = gate_scale_ld;
  a.w[1] = (const uint8_t *)up_codes;
  a.ws[1] = up_scales;
  a.ws_ld[1] = up_scale_ld;
  a.M = M;
  a.N = (int)N;
  a.K = (int)K;
  a.out = out_codes;
  a.out_s = out_scales;
  a.out_sld = out_scale_ld;
  const hipError_t e = launch_mx_product(mx_activations(a_format), true, out_format, a, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: too many output tiles", op);
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

int nvm_mx_product_plan(int gate_up, int64_t M, int64_t N, int64_t K, int a_format, int *plan) {
  using namespace nvm;
  const char *op = "mx_product_plan";
  if (!plan) return set_error(NVM_ERR_INVALID, "%s: null pointer", op);
  if (int rc = mx_check_rows(op, M, N, a_format & ~NVM_MX_SHORT_SUMS, "a")) return rc;
  if (int rc = mx_check_rows(op, K, N, NVM_MX_FP4, "w")) return rc;
  if (gate_up)
    if (int rc = mx_check_rows(op, M, K, NVM_MX_FP4, "output")) return rc;
  Choice c;
  if (M > 0 && K > 0) {
    c = choose(mx_activations(a_format), gate_up != 0, M, (int)N, (int)K);
    if (c.kernel < 0) return set_error(NVM_ERR_UNSUPPORTED, "%s: too many output tiles", op);
  }
  plan[0] = c.kernel;
  plan[1] = c.block.columns;
  plan[2] = c.block.rows;
  plan[3] = c.parts;
  return NVM_OK;
}

}  // extern "C"
