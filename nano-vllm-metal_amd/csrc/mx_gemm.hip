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

constexpr int round_up(int v, int m) { return (v + m - 1) / m * m; }

// BN weight rows (DUAL: half of them gate, half up) and BM activation rows a
// block, WF x WT wavefronts, two of them on a SIMD.
template <int FMT, bool DUAL_, int BN_, int BM_, int WF_, int WT_, int ST_>
struct Tile {
  static constexpr bool DUAL = DUAL_;
  static constexpr int BN = BN_, BM = BM_, WF = WF_, WT = WT_, ST = ST_, NW = WF * WT;
  static constexpr int NM = DUAL ? 2 : 1;        // matrices
  static constexpr int BK = BN / NM;             // output columns
  static constexpr int XR = FMT == NVM_MX_FP4 ? 64 : 128;  // bytes of an activation row's step
  // pieces of a stage (1 KB of codes, 64 rows of scales: a load each)
  static constexpr int PW = BN * 64 / 1024, PX = BM * XR / 1024;
  static constexpr int PSM = (BK + 63) / 64, PSW = NM * PSM, PS = PSW + (BM + 63) / 64;
  static constexpr int kW = PW * 1024, kX = PX * 1024, kS = PS * 256;
  static constexpr int kStage = kW + kX + kS, kLds = ST * kStage;
  // a wavefront's loads of a stage
  static constexpr int LW = (PW + NW - 1) / NW, LX = (PX + NW - 1) / NW;
  static constexpr int kLoads = LW + LX + 1;
  static constexpr int TF = BN / WF / 16, TM = BM / WT / 16;
  static_assert(NW == 8 && PS <= NW && kLds <= 160 * 1024, "a block of eight wavefronts");
  static_assert(BK % (16 * WF) == 0 && BM % (16 * WT) == 0 && (!DUAL || BK % (32 * WF) == 0),
                "whole tiles of a wavefront");
};

template <int FMT, int OFMT, class T>
__global__ __launch_bounds__(64 * T::NW, 2) void mx_gemm_kernel(const MxMatmulArgs p, int n_tiles,
                                                                int total) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int NX = FMT == NVM_MX_FP4 ? 1 : 2;
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, G = lane >> 4;
  const int wf = wv % T::WF, wt = wv / T::WF;
  const int WB = p.N / 2, XB = p.N * Mx<FMT>::kBits / 8, nb = p.N / 32;
  const int steps = (p.N + 127) / 128;
  // tiles in contiguous runs per XCD (blocks go to the XCDs in turn), a run
  // dealt to the XCD's blocks
  const int per_xcd = (total + 7) >> 3, stride = (int)gridDim.x >> 3;
  const int run_end = min(((int)blockIdx.x & 7) * per_xcd + per_xcd, total);
  const int first = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if (first >= run_end) return;

  struct Place {
    int k0, nk, nm;
    int64_t m0;
  };
  auto place = [&](int tile) {
    Place q;
    const int mt = tile / n_tiles;
    q.k0 = (tile - mt * n_tiles) * T::BK;
    q.m0 = (int64_t)mt * T::BM;
    q.nk = min(T::BK, p.K - q.k0);
    q.nm = (int)min((int64_t)T::BM, p.M - q.m0);
    return q;
  };

  // What the requests read: step r_step of tile r_tile, into stage r_slot.
  // Weight row r of a stage is column r % BK of matrix r / BK.
  int r_tile = first, r_step = 0, r_slot = 0;
  rsrc_t rw[T::LW], rx, rs;
  int vw[T::LW], vx[T::LX], vs;
  const int sp = wv % T::PS;  // (left-over wavefronts load what others load)
  auto aim = [&](int tile) {
    const Place q = place(tile);
#pragma unroll
    for (int j = 0; j < T::LW; ++j) {
      const int row = 16 * min(wv + j * T::NW, T::PW - 1), d = T::DUAL && row >= T::BK;
      rw[j] = make_rsrc(p.w[d] + (int64_t)q.k0 * WB, (uint32_t)(q.nk * WB));
      vw[j] = min(row - d * T::BK + (lane >> 2), q.nk - 1) * WB + 16 * ((lane & 3) ^ (lane >> 4));
    }
    rx = make_rsrc(p.a + q.m0 * XB, (uint32_t)(q.nm * XB));
#pragma unroll
    for (int j = 0; j < T::LX; ++j) {
      const int i = min(wv + j * T::NW, T::PX - 1);
      if constexpr (FMT == NVM_MX_FP4)
        vx[j] = min(16 * i + (lane >> 2), q.nm - 1) * XB + 16 * ((lane & 3) ^ (lane >> 4));
      else
        vx[j] = min(8 * i + (lane >> 3), q.nm - 1) * XB +
                16 * ((lane & 7) ^ ((4 * i + (lane >> 4)) & 7));
    }
    if (sp < T::PSW) {
      const int d = T::DUAL && sp >= T::PSM, ld = (int)p.ws_ld[d];
      rs = make_rsrc(p.ws[d] + (int64_t)q.k0 * ld, (uint32_t)(q.nk * ld));
      vs = min(64 * (sp - d * T::PSM) + lane, q.nk - 1) * ld;
    } else {
      const int ld = (int)p.as_ld;
      rs = make_rsrc(p.as + q.m0 * ld, (uint32_t)(q.nm * ld));
      vs = min(64 * (sp - T::PSW) + lane, q.nm - 1) * ld;
    }
  };
  auto request = [&] {
    uint8_t *st = smem + r_slot * T::kStage;
#pragma unroll
    for (int j = 0; j < T::LW; ++j)
      lds_load16(rw[j], st + min(wv + j * T::NW, T::PW - 1) * 1024, vw[j], 64 * r_step);
#pragma unroll
    for (int j = 0; j < T::LX; ++j)
      lds_load16(rx, st + T::kW + min(wv + j * T::NW, T::PX - 1) * 1024, vx[j], T::XR * r_step);
    lds_load4(rs, st + T::kW + T::kX + sp * 256, vs, 4 * r_step);
    r_slot = r_slot + 1 == T::ST ? 0 : r_slot + 1;
    if (++r_step == steps) {
      r_step = 0;
      r_tile += stride;
      if (r_tile < run_end) aim(r_tile);
    }
  };

  // places in a stage that the wavefront's operands are read from
  const int wrow = wf * (T::BK / T::WF) + col, xrow = wt * (T::BM / T::WT) + col;
  const int aw = wrow * 64 + 16 * (G ^ ((col >> 2) & 3));
  int ax[NX];
#pragma unroll
  for (int c = 0; c < NX; ++c)
    ax[c] = T::kW + xrow * T::XR +
            16 * (FMT == NVM_MX_FP4 ? G ^ ((col >> 2) & 3) : (4 * c + G) ^ ((col >> 1) & 7));
  const int aws = T::kW + T::kX + wrow * 4 + G;
  const int axs = T::kW + T::kX + T::PSW * 256 + xrow * 4 + G;
  // weight tile f of the wavefront: rows further on in the stage
  auto ftile = [](int f) { return T::DUAL && f >= T::TF / 2 ? T::BK + 16 * (f - T::TF / 2) : 16 * f; };
  auto fscale = [](int f) {
    return T::DUAL && f >= T::TF / 2 ? T::PSM * 256 + 64 * (f - T::TF / 2) : 64 * f;
  };

  aim(first);
#pragma unroll
  for (int s = 0; s < T::ST - 1; ++s)
    if (r_tile < run_end) request();
  // the first stage, of every wavefront
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  // wavefronts 4 to 7 run half a step behind the others
  if (wv >= 4) __builtin_amdgcn_s_barrier();
  int slot = 0;
  for (int tile = first; tile < run_end; tile += stride) {
    f32x4 acc[T::TF][T::TM];
#pragma unroll
    for (int f = 0; f < T::TF; ++f)
#pragma unroll
      for (int t = 0; t < T::TM; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < steps; ++s) {
      const uint8_t *st = smem + slot * T::kStage;
      MxFrag<FMT> x[T::TM];
      MxFrag<NVM_MX_FP4> w[T::TF];
      uint32_t xs[T::TM], ws[T::TF];
#pragma unroll
      for (int t = 0; t < T::TM; ++t) {
#pragma unroll
        for (int c = 0; c < NX; ++c) x[t].v[c] = *(const u32x4 *)(st + ax[c] + t * 16 * T::XR);
        xs[t] = st[axs + t * 64];
      }
#pragma unroll
      for (int f = 0; f < T::TF; ++f) {
        w[f].v[0] = *(const u32x4 *)(st + aw + ftile(f) * 64);
        ws[f] = st[aws + fscale(f)];
      }
      const bool more = r_tile < run_end;
      if (more) request();
      if (128 * s + 128 > p.N) {  // a last step that the row ends in
#pragma unroll
        for (int t = 0; t < T::TM; ++t) {
#pragma unroll
          for (int c = 0; c < NX; ++c)
            if (128 * s + (FMT == NVM_MX_FP4 ? 32 * G : 64 * c + 16 * G) >= p.N)
              x[t].v[c] = u32x4{0u, 0u, 0u, 0u};
          if (4 * s + G >= nb) xs[t] = 127u;
        }
#pragma unroll
        for (int f = 0; f < T::TF; ++f)
          if (4 * s + G >= nb) ws[f] = 127u;
      }
      // The wavefront's share of the next step has arrived when at most the
      // ST - 2 later requests are outstanding.  This step's operands are in
      // registers, so its stage may be overwritten from the barrier on.
      if (more)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((T::ST - 2) * T::kLoads) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int f = 0; f < T::TF; ++f)
#pragma unroll
        for (int t = 0; t < T::TM; ++t)
          acc[f][t] = mx_mfma<FMT>(w[f], ws[f], x[t], xs[t], acc[f][t]);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      slot = slot + 1 == T::ST ? 0 : slot + 1;
    }

    const Place q = place(tile);
#pragma unroll
    for (int t = 0; t < T::TM; ++t) {
      const int m = wt * (T::BM / T::WT) + 16 * t + col;
      if constexpr (!T::DUAL) {
        if (m >= q.nm) continue;
#pragma unroll
        for (int f = 0; f < T::TF; ++f) {
          const int k = wf * (T::BK / T::WF) + 16 * f + 4 * G;
          mx_store4(p.out, p.out_dtype, (q.m0 + m) * p.K + q.k0 + k, acc[f][t], q.nk - k,
                    p.K % 4 == 0);
        }
      } else {
#pragma unroll
        for (int f = 0; f < T::TF / 2; f += 2) {
          const int k = wf * (T::BK / T::WF) + 16 * f;
          float h[8];
          uint32_t mx = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            h[e] = mx_swiglu(acc[f + (e >> 2)][t][e & 3], acc[T::TF / 2 + f + (e >> 2)][t][e & 3]);
            mx = max(mx, abs_bits(h[e]));
          }
          mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16));
          mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
          if (m < q.nm && k < q.nk)
            mx_store_block<OFMT>(h, mx, q.m0 + m, q.k0 + k, G, p.K, p.out, p.out_s, p.out_sld);
        }
      }
    }
  }
  if (wv < 4) __builtin_amdgcn_s_barrier();
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

template <int FMT, int OFMT, class T>
hipError_t go(const MxMatmulArgs &a, hipStream_t st) {
  static bool done[64] = {false};
  auto kern = mx_gemm_kernel<FMT, OFMT, T>;
  allow_lds(kern, T::kLds, done);
  const int n_tiles = (a.K + T::BK - 1) / T::BK;
  const int64_t total = (a.M + T::BM - 1) / T::BM * n_tiles;
  if (total > kMxMaxTiles) return hipErrorInvalidConfiguration;
  const int64_t grid = std::min<int64_t>(8 * ((total + 7) / 8), cu_count() / 8 * 8);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * T::NW), T::kLds, st, a, n_tiles,
                     (int)total);
  return hipGetLastError();
}

template <int FMT>
hipError_t launch_fmt(bool dual, int out_format, const MxMatmulArgs &a, hipStream_t st) {
  constexpr int ST = FMT == NVM_MX_FP4 ? 4 : 3;
  if (!dual) return go<FMT, NVM_MX_FP8, Tile<FMT, false, 256, 256, 2, 4, ST>>(a, st);
  using Dual = Tile<FMT, true, 256, 256, 2, 4, ST>;
  return out_format == NVM_MX_FP4 ? go<FMT, NVM_MX_FP4, Dual>(a, st)
                                  : go<FMT, NVM_MX_FP8, Dual>(a, st);
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
