// Products of many MX rows with MXFP4 weights (include/nvm_mx.h): prompts
// through the projections and through the dense MLP's gate/up pair.
//
// Bound: the scaled matrix instruction, 32 cycles a 16x16x128 product where an
// operand is E4M3 and 16 where both are E2M1, so feeding it.
//  * Nothing is unpacked: codes and scale bytes go from memory into LDS as
//    they are (buffer loads with an LDS target) and from there into the
//    instruction's operands.
//  * A stage is one 128-value step of the tile: BN weight rows of 64 bytes, BM
//    activation rows of 128 (E4M3) or 64, and four scale bytes a row.  ST
//    stages ring: step s + ST - 1 is requested while s is computed, with one
//    block barrier a step.
//  * 16-byte chunk k of row r lies at place k ^ f(r) of its row, f = (r >> 2)
//    & 3 for rows of 64 bytes and (r >> 1) & 7 for rows of 128: chunk k of 16
//    consecutive rows then falls into 16 different 16-byte groups of the
//    256-byte bank cycle.  The loads' lane-to-chunk assignment makes the
//    order (LDS is written in lane order).
//  * Rows past an operand repeat its last row, whose outputs are not stored;
//    a last step of less than 128 values is computed with the activations
//    behind the row replaced by zeros and scales by one in registers, so what
//    lies there does not matter (a weight code is finite whatever its bits).
#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "mx_common.h"

namespace nvm {

namespace {

__device__ __forceinline__ void lds_load16(rsrc_t r, void *lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16,
                                           voff, soff, 0, 0);
}
__device__ __forceinline__ void lds_load4(rsrc_t r, void *lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 4,
                                           voff, soff, 0, 0);
}

// BN weight rows (DUAL: half of them gate, half up) and BM activation rows a
// block, WF x WT wavefronts.
template <int FMT, int BN_, int BM_, int WF_, int WT_, int ST_>
struct Tile {
  static constexpr int BN = BN_, BM = BM_, WF = WF_, WT = WT_, ST = ST_, NW = WF * WT;
  static constexpr int XR = FMT == NVM_MX_FP4 ? 64 : 128;  // bytes of an activation row's step
  static constexpr int kW = BN * 64, kX = BM * XR, kS = (BN + BM) * 4;
  static constexpr int kStage = kW + kX + kS;
  static constexpr int kLds = ST * kStage;
  // a wavefront's loads of a stage
  static constexpr int LW = kW / 1024 / NW, LX = kX / 1024 / NW, LS = (BN + BM) / 64;
  static constexpr int kLoads = LW + LX + 1;
  static_assert(kW % (1024 * NW) == 0 && kX % (1024 * NW) == 0 && LS <= NW, "whole loads");
  static constexpr int TF = BN / WF / 16, TM = BM / WT / 16;
};

template <int FMT, int OFMT, bool DUAL, class T>
__global__ __launch_bounds__(64 * T::NW) void mx_gemm_kernel(const MxMatmulArgs p, int n_tiles,
                                                             int total) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int NX = FMT == NVM_MX_FP4 ? 1 : 2;
  constexpr int GR = T::BN / T::WF;          // LDS weight rows of a wavefront
  constexpr int BK = DUAL ? T::BN / 2 : T::BN;  // output columns of a block
  static_assert(!DUAL || GR % 128 == 0, "a scale load is of one matrix");
  // tiles in contiguous runs per XCD (blocks go to the XCDs in turn)
  const int per_xcd = (total + 7) >> 3;
  const int tile = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if (((int)blockIdx.x >> 3) >= per_xcd || tile >= total) return;
  const int mt = tile / n_tiles, nt = tile - mt * n_tiles;
  const int k0 = nt * BK;
  const int64_t m0 = (int64_t)mt * T::BM;
  const int nk = min(BK, p.K - k0), nm = (int)min((int64_t)T::BM, p.M - m0);
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, G = lane >> 4;
  const int wf = wv % T::WF, wt = wv / T::WF;
  const int WB = p.N / 2, XB = p.N * Mx<FMT>::kBits / 8, nb = p.N / 32;
  const int steps = (p.N + 127) / 128, whole = p.N / 128;

  // LDS weight row -> (matrix, row of the tile's columns)
  auto matrix = [&](int row) { return DUAL ? (row / (GR / 2)) & 1 : 0; };
  auto column = [&](int row) { return DUAL ? row / GR * (GR / 2) + row % (GR / 2) : row; };

  rsrc_t lw[T::LW];
  int vw[T::LW], vx[T::LX];
#pragma unroll
  for (int j = 0; j < T::LW; ++j) {
    const int row = 16 * (wv * T::LW + j) + (lane >> 2), d = matrix(16 * (wv * T::LW + j));
    lw[j] = make_rsrc(p.w[d] + (int64_t)k0 * WB, (uint32_t)(nk * WB));
    vw[j] = min(column(row), nk - 1) * WB + 16 * ((lane & 3) ^ (lane >> 4));
  }
  const rsrc_t lx = make_rsrc(p.a + m0 * XB, (uint32_t)(nm * XB));
#pragma unroll
  for (int j = 0; j < T::LX; ++j) {
    const int q = wv * T::LX + j;
    if constexpr (FMT == NVM_MX_FP4)
      vx[j] = min(16 * q + (lane >> 2), nm - 1) * XB + 16 * ((lane & 3) ^ (lane >> 4));
    else
      vx[j] = min(8 * q + (lane >> 3), nm - 1) * XB +
              16 * ((lane & 7) ^ ((4 * (q & 1) + (lane >> 4)) & 7));
  }
  // one load of scales a wavefront: 64 rows' four bytes of the step (those
  // wavefronts that are left over load what another loads)
  const int sq = wv % T::LS, srow = 64 * sq;
  const bool sw = srow < T::BN;
  const int sd = sw ? matrix(srow) : 0;
  const int sld = (int)(sw ? p.ws_ld[sd] : p.as_ld);
  const rsrc_t ls = sw ? make_rsrc(p.ws[sd] + (int64_t)k0 * sld, (uint32_t)(nk * sld))
                       : make_rsrc(p.as + m0 * sld, (uint32_t)(nm * sld));
  const int vs = (sw ? min(column(srow + lane), nk - 1) : min(srow - T::BN + lane, nm - 1)) * sld;

  auto request = [&](int s) {
    // (steps past the end load the first again, into a stage that nothing
    // reads any more: every step makes the same loads)
    const int so = s < steps ? s : 0;
    uint8_t *st = smem + s % T::ST * T::kStage;
#pragma unroll
    for (int j = 0; j < T::LW; ++j) lds_load16(lw[j], st + (wv * T::LW + j) * 1024, vw[j], 64 * so);
#pragma unroll
    for (int j = 0; j < T::LX; ++j)
      lds_load16(lx, st + T::kW + (wv * T::LX + j) * 1024, vx[j], T::XR * so);
    lds_load4(ls, st + T::kW + T::kX + sq * 256, vs, 4 * so);
  };

  f32x4 acc[T::TF][T::TM];
#pragma unroll
  for (int f = 0; f < T::TF; ++f)
#pragma unroll
    for (int t = 0; t < T::TM; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int rw = (wf * GR + col) * 64 + 16 * (G ^ ((col >> 2) & 3));
  const int xrow = wt * (T::BM / T::WT) + col;
  int rx[NX];
#pragma unroll
  for (int c = 0; c < NX; ++c)
    rx[c] = T::kW + xrow * T::XR +
            16 * (FMT == NVM_MX_FP4 ? G ^ ((col >> 2) & 3) : (4 * c + G) ^ ((col >> 1) & 7));
  const int rws = T::kW + T::kX + (wf * GR + col) * 4 + G;
  const int rxs = T::kW + T::kX + (T::BN + xrow) * 4 + G;
  auto compute = [&](int s, auto TAIL) {
    constexpr bool tail = decltype(TAIL)::value;
    const uint8_t *st = smem + s % T::ST * T::kStage;
    MxFrag<FMT> x[T::TM];
    uint32_t xs[T::TM];
#pragma unroll
    for (int t = 0; t < T::TM; ++t) {
#pragma unroll
      for (int c = 0; c < NX; ++c) {
        x[t].v[c] = *(const u32x4 *)(st + rx[c] + t * 16 * T::XR);
        if constexpr (tail)
          if (128 * s + (FMT == NVM_MX_FP4 ? 32 * G : 64 * c + 16 * G) >= p.N)
            x[t].v[c] = u32x4{0u, 0u, 0u, 0u};
      }
      xs[t] = st[rxs + t * 64];
      if constexpr (tail) xs[t] = 4 * s + G < nb ? xs[t] : 127u;
    }
#pragma unroll
    for (int f = 0; f < T::TF; ++f) {
      MxFrag<NVM_MX_FP4> w;
      w.v[0] = *(const u32x4 *)(st + rw + f * 1024);
      uint32_t ws = st[rws + f * 64];
      if constexpr (tail) ws = 4 * s + G < nb ? ws : 127u;
#pragma unroll
      for (int t = 0; t < T::TM; ++t) acc[f][t] = mx_mfma<FMT>(w, ws, x[t], xs[t], acc[f][t]);
    }
  };
  // Stage s has arrived when at most the loads of the ST - 2 later ones are
  // outstanding; the barrier extends that to every wavefront's share, and
  // says that every wavefront has read stage s - 1, which the next request
  // overwrites.
  auto arrive = [&] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((T::ST - 2) * T::kLoads) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int s = 0; s < T::ST - 1; ++s) request(s);
  for (int s = 0; s < whole; ++s) {
    arrive();
    request(s + T::ST - 1);
    compute(s, std::false_type{});
  }
  if (whole < steps) {
    arrive();
    compute(whole, std::true_type{});
  }
  // (no load may still be writing when the block's LDS is given back)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

#pragma unroll
  for (int t = 0; t < T::TM; ++t) {
    const int m = wt * (T::BM / T::WT) + 16 * t + col;
    if constexpr (!DUAL) {
      if (m >= nm) continue;
#pragma unroll
      for (int f = 0; f < T::TF; ++f) {
        const int k = wf * GR + 16 * f + 4 * G;
        mx_store4(p.out, p.out_dtype, (m0 + m) * p.K + k0 + k, acc[f][t], nk - k, p.K % 4 == 0);
      }
    } else {
#pragma unroll
      for (int f = 0; f < T::TF / 2; f += 2) {
        const int k = wf * (GR / 2) + 16 * f;
        float h[8];
        uint32_t mx = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          h[e] = mx_swiglu(acc[f + (e >> 2)][t][e & 3], acc[T::TF / 2 + f + (e >> 2)][t][e & 3]);
          mx = max(mx, abs_bits(h[e]));
        }
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16));
        mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
        if (m < nm && k < nk)
          mx_store_block<OFMT>(h, mx, m0 + m, k0 + k, G, p.K, p.out, p.out_s, p.out_sld);
      }
    }
  }
}

// more than 64 KB of dynamic LDS: allowed once per device and instance (a
// failure shows up as a failed launch)
template <class F>
void allow_lds(F kern, int bytes, bool (&done)[64]) {
  int dev = 0;
  if (hipGetDevice(&dev) == hipSuccess && dev >= 0 && dev < 64 && !done[dev]) {
    (void)hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                              bytes);
    done[dev] = true;
  }
}

template <int FMT, int OFMT, bool DUAL, class T>
hipError_t go(const MxMatmulArgs &a, hipStream_t st) {
  static bool done[64] = {false};
  constexpr int BK = DUAL ? T::BN / 2 : T::BN;
  auto kern = mx_gemm_kernel<FMT, OFMT, DUAL, T>;
  allow_lds(kern, T::kLds, done);
  const int n_tiles = (a.K + BK - 1) / BK;
  const int64_t total = (a.M + T::BM - 1) / T::BM * n_tiles;
  if (total > kMxMaxTiles) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kern, dim3((unsigned)(8 * ((total + 7) / 8))), dim3(64 * T::NW), T::kLds, st,
                     a, n_tiles, (int)total);
  return hipGetLastError();
}

template <int FMT>
hipError_t launch_fmt(bool dual, int out_format, const MxMatmulArgs &a, hipStream_t st) {
  using Large = Tile<FMT, 256, 256, 2, 4, FMT == NVM_MX_FP4 ? 4 : 3>;
  if (!dual) return go<FMT, NVM_MX_FP8, false, Large>(a, st);
  return out_format == NVM_MX_FP4 ? go<FMT, NVM_MX_FP4, true, Large>(a, st)
                                  : go<FMT, NVM_MX_FP8, true, Large>(a, st);
}

}  // namespace

hipError_t launch_mx_gemm(int format, bool dual, int out_format, const MxMatmulArgs &a,
                          hipStream_t st) {
  return format == NVM_MX_FP4 ? launch_fmt<NVM_MX_FP4>(dual, out_format, a, st)
                              : launch_fmt<NVM_MX_FP8>(dual, out_format, a, st);
}

// Few rows: the kernel without LDS staging.
static hipError_t launch_mx_product(int format, bool dual, int out_format, const MxMatmulArgs &a,
                                    hipStream_t st) {
  return a.M <= 64 ? launch_mx_gemv(format, dual, out_format, a, st)
                   : launch_mx_gemm(format, dual, out_format, a, st);
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
