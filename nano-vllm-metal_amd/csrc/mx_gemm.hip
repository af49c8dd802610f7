// Products of many MX rows with MXFP4 weights (include/nvm_mx.h) where tiles of
// 256 x 256 fill the GPU: long prompts through the projections and through the
// dense MLP's gate/up pair.  (Fewer rows: mx_gemm_pipe.hip.)
//
// Bound: the matrix instructions.  A 16x16x128 product is one scaled instruction
// where both operands are E2M1, 16 cycles, or for short sums of E4M3, 32; E4M3
// otherwise takes four bf16 ones, 64 cycles, and conversions beside them.
//  * Codes and scale bytes go from memory into LDS as they are (buffer loads with
//    an LDS target) and from there into registers.
//  * A stage is one 128-value step of the tile: weight rows of 64 bytes and
//    activation rows of 128 (E4M3) or 64.  Scales come 16 bytes a row, for
//    four steps at once, into a ring of their own.
//  * The wavefronts of a SIMD take turns: 0 to 3 read a step's operands from
//    LDS (and request a later step) while 4 to 7 run theirs through the matrix
//    cores, then the other way round, two block barriers a step.  That leaves
//    a wavefront's registers to its 8 x 4 sums and one step's operands, which
//    is what 256 x 256 needs; with reads and products in one wavefront side by
//    side (mx_gemm_pipe.hip) two steps' operands only fit beside 4 x 4 sums.
//  * Blocks are persistent and requests run on across tiles, so a tile's first
//    steps arrive during the epilogue of the one before.
//  * Tiles that would be a last round of at most a quarter (half) of the CUs are
//    computed in quarters (halves) by all of them, with the code of mx_pipe.h
//    (3000 rows of 4096 -> 6144, 288 tiles: 127 us with quarters, 176 without;
//    8192 rows of 2048 -> 5120, 640 tiles: 134 with halves, 141 without).
//  * A last step of less than 128 values is computed with the activations
//    behind the row replaced by zeros and scales by one in registers, so what
//    lies there does not matter (a weight code is finite whatever its bits).
//
// 8192 x 8192 x 8192: 729 us, 1.5 PFLOP/s, as a bf16 library product there (732);
// E2M1 293 us, 3.75; short sums 367 us, 3.0.  4096 rows of 2048
// through a gate/up pair of 6144: 153 us, 1.35 PFLOP/s; short sums 84 us, 2.5.
#include "mx_pipe.h"

namespace nvm {

namespace {

template <class X>
struct TypeOf {
  using type = X;
};

// The first `whole` tiles in turn; the others, if `parts` is not zero, in that
// many parts (2 or 4), a part a block.
template <int FMT, int OFMT, class T>
__global__ __launch_bounds__(64 * T::NW, 2) void mx_gemm_kernel(const MxMatmulArgs p, int n_tiles,
                                                                int m_tiles, int whole, int parts) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int NX = FMT == NVM_MX_FP4 ? 1 : 2;
  const int lane = threadIdx.x & 63, G = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wf = wv % T::WF, wt = wv / T::WF;
  const int nb = p.N / 32;
  // Steps of a tile.  The runs that ST consecutive stages touch are ST at most,
  // ST - 1 if no run has a single step: then a tile gets one of zeros more.
  int steps = (p.N + 127) / 128;
  if (T::SL < T::ST) steps += steps % 4 == 1;
  // tiles in contiguous runs per XCD (blocks go to the XCDs in turn), dealt to
  // the XCD's blocks
  const int per_xcd = (whole + 7) >> 3, stride = (int)gridDim.x >> 3;
  const int last = min(((int)blockIdx.x & 7) * per_xcd + per_xcd, whole);
  const int first = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if (first >= last) return;

  // What the requests read: step r_step of tile r_tile, into slot r_slot.
  int r_tile = first, r_step = 0, r_slot = 0, r_chunk = 0;
  typename T::Source src;
  typename T::ScaleSource scales;
  auto aim = [&] {
    if (r_tile >= last) {
      src.none(p);
      scales.s = make_rsrc(p.a, 0);
    } else {
      const typename T::Place q = T::place(p, r_tile, n_tiles, m_tiles);
      src.aim(p, q, wv, lane);
      scales.aim(p, q, wv, lane);
    }
  };
  uint8_t *const piece = smem + T::kScales + wv * 1024;  // the wavefront's of a scale slot
  // load i of the step's: scales (of its run's first step), weights, activations
  auto load = [&](int i) {
    if (i > 0)
      src.load(i - 1, r_step, smem + r_slot * T::kStage, wv);
    else if (r_step % 4 == 0 && wv < T::PS)
      lds_load16(scales.s, piece + r_chunk * T::kS, scales.v, 4 * r_step);
  };
  auto advance = [&] {
    if (r_step % 4 == 0) r_chunk = r_chunk + 1 == T::SL ? 0 : r_chunk + 1;
    r_slot = r_slot + 1 == T::ST ? 0 : r_slot + 1;
    if (++r_step == steps) {
      r_step = 0;
      r_tile += stride;
      aim();
    }
  };
  // All but the last ST - 2 requested steps have arrived.  (Where scales were
  // among the loads the wait is longer than it need be, never shorter.)
  auto arrived = [&] {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((T::ST - 2) * T::kLoads) : "memory");
  };
  auto turn = [&](int c) {  // (its reads before its writes)
    if (wv >= T::PS) return;
    const u32x4 raw = *(const u32x4 *)(piece + c * T::kS + 16 * lane);
    wave_lds_sync();
    T::turn(piece + c * T::kS, raw, lane);
  };
  const typename T::Reads at(wf, wt, 0, lane);
  auto phase_end = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  const bool late = wv >= 4;
  aim();
  for (int n = T::ST - 1; n > 0; --n) {
#pragma unroll
    for (int i = 0; i <= T::kLoads; ++i) load(i);
    advance();
  }
  // the first step, of every wavefront
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  turn(0);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  // wavefronts 4 to 7 run half a step behind the others
  if (late) __builtin_amdgcn_s_barrier();
  int slot = 0, chunk = T::SL - 1;
  for (int tile = first; tile < last; tile += stride) {
    f32x4 acc[T::TF][T::TM];
#pragma unroll
    for (int f = 0; f < T::TF; ++f)
#pragma unroll
      for (int t = 0; t < T::TM; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Scale bytes of the lane's block in the steps to come, the next lowest
    // (the matrix instruction takes a register's low byte).
    typename T::Scales sc;
    for (int s = 0;; ++s) {
      if (s % 4 == 0) chunk = chunk + 1 == T::SL ? 0 : chunk + 1;
      if (s % 4 == 0 || FMT == NVM_MX_FP8) {
        // (bf16 operands leave no registers to keep a run's scales in beside
        // them: a step reads them again)
        sc.read(smem, at, chunk, FMT == NVM_MX_FP8 ? s % 4 : 0);
      } else {
#pragma unroll
        for (int f = 0; f < T::TF; ++f) sc.w[f] >>= 8;
#pragma unroll
        for (int t = 0; t < T::TM; ++t) sc.x[t] >>= 8;
      }
      const uint8_t *st = smem + slot * T::kStage;
      MxFrag<FMT> x[T::TM];
      MxFrag<NVM_MX_FP4> w[T::TF];
      // (a load's issue waits for the address unit, which all wavefronts of a
      // phase share: the LDS reads go out in between)
      auto next = [&](int i) {
        constexpr int n = T::kLoads + 1, of = T::TM + T::TF;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = i * n / of; j < (i + 1) * n / of; ++j) load(j);
        __builtin_amdgcn_sched_barrier(0);
      };
#pragma unroll
      for (int t = 0; t < T::TM; ++t) {
        next(t);
        x[t] = at.act(st, t);
      }
#pragma unroll
      for (int f = 0; f < T::TF; ++f) {
        next(T::TM + f);
        w[f] = at.weight(st, f);
      }
      advance();
      if (128 * s + 128 > p.N) {  // a last step that the row ends in or before
#pragma unroll
        for (int t = 0; t < T::TM; ++t) {
#pragma unroll
          for (int c = 0; c < NX; ++c)
            if (128 * s + mx_act_at<FMT>(G, c) >= p.N)
              x[t].v[c] = u32x4{0u, 0u, 0u, 0u};
          if (4 * s + G >= nb) sc.x[t] = 127u;
        }
#pragma unroll
        for (int f = 0; f < T::TF; ++f)
          if (4 * s + G >= nb) sc.w[f] = 127u;
      }
      arrived();
      if (s + 1 == steps || (s + 1) % 4 == 0) turn(chunk + 1 == T::SL ? 0 : chunk + 1);
      // This step's operands are in registers, the next run's scales in place.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      mx_products<FMT, 0>(w, sc.w, x, sc.x, acc, [](int) {
        if constexpr (FMT == NVM_MX_FP8) __builtin_amdgcn_sched_barrier(0);
      });
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      slot = slot + 1 == T::ST ? 0 : slot + 1;
      if (s + 1 == steps) break;
      phase_end();
    }
    // Wavefronts 4 to 7 meet the tile's last barrier behind their epilogue, so
    // that it runs along with the others' (one after the other, they cost a
    // tile of 16 steps 6500 of 50000 cycles).
    if (!late) phase_end();
    T::template finish<OFMT, T::TM>(p, T::place(p, tile, n_tiles, m_tiles), acc, wf,
                                    wt * (T::BM / T::WT), lane);
    if (late) phase_end();
  }
  // (no load may write to LDS behind the block's end)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (!late) __builtin_amdgcn_s_barrier();
  // The tiles past whole rounds, in parts: one to a block.
  if (parts == 0) return;
  const int part = ((int)blockIdx.x & 7) * stride + ((int)blockIdx.x >> 3);
  const int tile = whole + part / parts, sub = part % parts;
  if (tile >= n_tiles * m_tiles) return;
  __syncthreads();  // (LDS changes hands)
  auto finish = [&](auto TILE) {
    using S = typename decltype(TILE)::type;
    constexpr int across = T::BK / S::BK;
    const typename T::Place from = T::place(p, tile, n_tiles, m_tiles);
    typename S::Place q;
    q.k0 = from.k0 + sub % across * S::BK;
    q.m0 = from.m0 + sub / across * S::BM;
    q.nk = min(S::BK, p.K - q.k0);
    q.nm = (int)min((int64_t)S::BM, p.M - q.m0);
    if (q.nk > 0 && q.nm > 0)
      mx_pipe_tiles<FMT, OFMT, S>(p, smem, 0, 1, 1, [&](int) { return q; });
  };
  if (parts == 4)
    finish(TypeOf<MxSmallTile<FMT, T::DUAL>>{});
  else
    finish(TypeOf<MxWideTile<FMT, T::DUAL>>{});
}

template <int FMT, int OFMT, bool DUAL>
hipError_t go(int parts, const MxMatmulArgs &a, hipStream_t st) {
  // (the rings fill the 160 KB of LDS)
  using T = std::conditional_t<FMT == NVM_MX_FP4, MxTile<FMT, DUAL, 256, 256, 2, 4, 1, 4, 4>,
                               MxTile<FMT, DUAL, 256, 256, 2, 4, 1, 3, 2>>;
  constexpr int kLds =
      std::max({T::kLds, MxSmallTile<FMT, DUAL>::kLds, MxWideTile<FMT, DUAL>::kLds});
  static bool allowed[64] = {false};
  int n_tiles, m_tiles;
  if (!mx_count_tiles<T>(a, n_tiles, m_tiles)) return hipErrorInvalidConfiguration;
  auto kern = mx_gemm_kernel<FMT, OFMT, T>;
  mx_allow_lds(kern, kLds, allowed);
  // blocks that walk tiles, one to a CU
  const int total = n_tiles * m_tiles;
  const int grid = std::min(8 * ((total + 7) / 8), cu_count() / 8 * 8);
  const int whole = parts ? total / grid * grid : total;
  if (parts && (whole == 0 || (total - whole) * parts > grid)) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * T::NW), kLds, st, a, n_tiles, m_tiles,
                     whole, parts);
  return hipGetLastError();
}

template <int FMT>
hipError_t launch_fmt(int parts, bool dual, int out_format, const MxMatmulArgs &a, hipStream_t st) {
  if (!dual) return go<FMT, NVM_MX_FP8, false>(parts, a, st);
  return out_format == NVM_MX_FP4 ? go<FMT, NVM_MX_FP4, true>(parts, a, st)
                                  : go<FMT, NVM_MX_FP8, true>(parts, a, st);
}

}  // namespace

hipError_t launch_mx_gemm(int format, int parts, bool dual, int out_format, const MxMatmulArgs &a,
                          hipStream_t st) {
  return format == NVM_MX_FP4   ? launch_fmt<NVM_MX_FP4>(parts, dual, out_format, a, st)
         : format == NVM_MX_FP8 ? launch_fmt<NVM_MX_FP8>(parts, dual, out_format, a, st)
                                : launch_fmt<kMxShort>(parts, dual, out_format, a, st);
}

}  // namespace nvm
