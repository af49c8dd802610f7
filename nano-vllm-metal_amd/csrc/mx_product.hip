// Products of MX rows with MXFP4 weights: which kernel, and the entry points
// (include/nvm_mx.h).
#include <algorithm>

#include "internal.h"
#include "mx_common.h"

namespace nvm {

// Few rows: mx_gemv.hip, while its time as fitted (mx_gemv_time) is the least;
// that of tiles goes with the steps along a row alone until they fill the GPU.
// In us there and on tiles: 2048 -> 5120, 64 rows 7.6 and 10.8, 96 rows 8.0 and
// 11.3, 128 rows 9.8 and 12.0, 192 rows 12.7 and 12.5; 4096 -> 4096, 192 rows 15.5
// and 17; gate/up 2048 -> 6144, 64 rows 10.5 and 12.6, 80 rows 15.2 and 12.6.  16
// rows stay there whatever the columns, where reading the weights is all:
// 2048 -> 151936 of 1 row 31 and 50 us, of 16 rows 42 and 49.
//
// Many rows: the tiles whose rounds over the CUs cost least.  A step of the
// larger ones costs less for its outputs, but they leave more CUs idle.  Their
// costs, in steps of 256 x 256 at 20 (0.9 us each): E4M3 activations 13 and 9,
// E2M1 11 and 8 for 256 x 128 and 128 x 128.  A last round of 256 x 256 that no
// more than a quarter (half) of the CUs would have is computed in parts of those
// sizes.  In us on 256 x 256 in whole tiles, in parts, on 256 x 128 and 128 x 128,
// E4M3 unless said:
//   2048 -> 5120    512 rows   24.0   -    17.2  13.2
//                  1536 rows   26.3   -    21.0  24.8
//                  2048 rows   27.0   -    30.3  35.2
//                  4096 rows   48.9  44.4  47.0  59.0  (E2M1 42.0  35.8  35.7  46.3)
//                  8192 rows   77.3  73.1  78.7   -    (E2M1 67.1  61.7  61.8)
//   6144 -> 2048   1024 rows   54     -    34    24
//                  4096 rows   57     -    45.5  54
//   4096 -> 6144   3000 rows   82.2  66.4  78.2   -
//   8192 -> 8192   8192 rows   367    -    424   553   (E2M1  293   -   350   420)
//   gate/up 2048 -> 6144
//                   100 rows   24.0   -    16.8  12.6
//                  1000 rows   27.7   -    31.7  35.9
//                  1500 rows   50.5  40.4  46.0   -
//                  4096 rows   82     -    94.7  134
static hipError_t launch_mx_product(int format, bool dual, int out_format, const MxMatmulArgs &a,
                                    hipStream_t st) {
  const bool fp4 = format == NVM_MX_FP4;
  const int64_t columns = (int64_t)a.K * (dual ? 2 : 1), cus = cu_count() / 8 * 8;
  auto tiles = [&](int bn, int bm) { return (columns + bn - 1) / bn * ((a.M + bm - 1) / bm); };
  auto rounds = [&](int64_t n) { return (n + cus - 1) / cus; };
  const int64_t wide_round = fp4 ? 11 : 13, small_round = fp4 ? 8 : 9;
  const int64_t wide_rounds = rounds(tiles(256, 128)), small_rounds = rounds(tiles(128, 128));
  // (Fitted likewise, for rows of 2048 values.  Where a few rows' tiles read many
  // weights they take longer than that, and blocks of a second round less: a
  // tenth in favour of the former.)
  const double n2048 = a.N / 2048.0;
  const double wide_time = (fp4 ? 5.0 : 7.0) + (fp4 ? 6.4 : 9.0) * wide_rounds * n2048;
  const double small_time = (fp4 ? 5.0 : 5.5) + (fp4 ? 4.1 : 5.9) * small_rounds * n2048;
  int tile = 0;
  if (mx_gemv_time(format, dual, a, &tile) <= 1.1 * std::min(wide_time, small_time) || a.M <= 16)
    return launch_mx_gemv(format, tile, dual, out_format, a, st);
  const int64_t wide = wide_rounds * wide_round, small = small_rounds * small_round;
  const int64_t n = tiles(256, 256), rest = n % cus;
  const int parts = n < cus || rest == 0 || 2 * rest > cus ? 0 : 4 * rest > cus ? 2 : 4;
  const int64_t big = parts ? n / cus * 20 + (parts == 4 ? small_round : wide_round)
                            : rounds(n) * 20;
  if (big <= std::min(wide, small)) return launch_mx_gemm(format, parts, dual, out_format, a, st);
  return launch_mx_gemm_pipe(format, wide <= small, dual, out_format, a, st);
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
  if (int rc = mx_check_rows(op, M, N, a_format, "a")) return rc;
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
  const hipError_t e = launch_mx_product(a_format, false, NVM_MX_FP8, a, (hipStream_t)stream);
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
  if (int rc = mx_check_rows(op, M, N, a_format, "a")) return rc;
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
  const hipError_t e = launch_mx_product(a_format, true, out_format, a, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: too many output tiles", op);
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

}  // extern "C"
