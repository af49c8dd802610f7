// Products of many MX rows with MXFP4 weights (include/nvm_mx.h): prompts
// through the projections and through the dense MLP's gate/up pair.
//
// Bound: the scaled matrix instruction, 32 cycles a 16x16x128 product where an
// operand is E4M3 and 16 where both are E2M1, so feeding it.
//  * Nothing is unpacked: codes and scale bytes go from memory into LDS as
//    they are (buffer loads with an LDS target) and from there into the
//    instruction's operands.
//  * A stage is one 128-value step of the tile: BN weight rows of 64 bytes and
//    BM activation rows of 128 (E4M3) or 64; ST stages ring.  Scales come 16
//    bytes a row, for four steps at once, into a ring of their own.
//  * The wavefronts of a SIMD take turns: 0 to 3 read a step's operands from
//    LDS (and request a later step) while 4 to 7 run theirs through the matrix
//    cores, then the other way round, two block barriers a step.
//  * Blocks are persistent and requests run on across tiles, so a tile's first
//    steps arrive during the epilogue of the one before.
//  * 16-byte chunk k of row r lies at place k ^ f(r) of its row, f = 3 ((r >>
//    3) & 1) for rows of 64 bytes and (r >> 1) & 7 for rows of 128.  A 16-byte
//    LDS read is served 16 lanes at a time: lanes 0-3, 12-15 and 20-27, then
//    4-11, 16-19 and 28-31 (and the same of the upper half), so rows 0-3 and
//    12-15 at one chunk with rows 4-11 at its neighbour k ^ 1; with these f
//    those fall into 16 different 16-byte groups of the 256-byte bank cycle.
//    (f = (r >> 2) & 3, right for 16 consecutive lanes, cost a second access
//    every weight read: 448 conflict cycles a block and step of 2800.)  The
//    loads' lane-to-chunk assignment makes the order (LDS is written in lane
//    order).
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

// BN weight rows (DUAL: half of them gate, half up) and BM activation rows a
// block of eight wavefronts, two on a SIMD.  KG = 1: WF x WT = 8 wavefronts
// share a 128-value step.  KG = 2: a stage is two steps, wavefronts 0 to 3 (WF
// x WT = 4 over the whole tile) take the first and 4 to 7 the second, and the
// two sums are joined at the end.
template <int FMT, bool DUAL_, int BN_, int BM_, int WF_, int WT_, int KG_, int ST_>
struct Tile {
  static constexpr bool DUAL = DUAL_;
  static constexpr int BN = BN_, BM = BM_, WF = WF_, WT = WT_, KG = KG_, ST = ST_, NW = 8;
  static constexpr int NM = DUAL ? 2 : 1;        // matrices
  static constexpr int BK = BN / NM;             // output columns
  static constexpr int XR = FMT == NVM_MX_FP4 ? 64 : 128;  // bytes of an activation row's step
  static constexpr int TF = BN / WF / 16, TM = BM / WT / 16;  // a wavefront's 16-row tiles
  // pieces of a step, 1 KB of codes, a load each
  static constexpr int PW = BN * 64 / 1024, PX = BM * XR / 1024;
  // pieces of a scale slot: four 16-row tiles of a wavefront's weights (of one
  // matrix) or activations
  static constexpr int QF = (TF / NM + 3) / 4, QT = (TM + 3) / 4;
  static constexpr int PSW = NM * WF * QF, PS = PSW + WT * QT;
  static constexpr int kW = PW * 1024, kX = PX * 1024, kS = PS * 1024;
  static constexpr int kStep = kW + kX, kStage = KG * kStep, kScales = ST * kStage;
  // Scale slots, of four steps (RUN stages).  The runs that ST consecutive
  // stages touch are ST at most, ST - 1 if no run has a single stage.
  static constexpr int RUN = 4 / KG;
  static constexpr int SL = kScales + ST * kS <= 160 * 1024 ? ST : ST - 1;
  static constexpr int kLds = kScales + SL * kS;
  // a wavefront's loads of a stage
  static constexpr int LW = (KG * PW + NW - 1) / NW, LX = (KG * PX + NW - 1) / NW;
  static constexpr int kLoads = LW + LX;
  static_assert(KG * WF * WT == NW && PS <= NW && kLds <= 160 * 1024, "a block's LDS and loads");
  static_assert(BK % (16 * WF) == 0 && BM % (16 * WT) == 0 && (!DUAL || BK % (32 * WF) == 0),
                "whole tiles of a wavefront");
  static_assert(KG == 1 || (TM % 2 == 0 && TF * TM * 4096 <= kScales), "the sums' exchange");
};

template <int FMT, int OFMT, class T>
__global__ __launch_bounds__(64 * T::NW, 2) void mx_gemm_kernel(const MxMatmulArgs p, int n_tiles,
                                                                int m_tiles) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int NX = FMT == NVM_MX_FP4 ? 1 : 2;
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, G = lane >> 4;
  const int kg = T::KG == 2 ? wv >> 2 : 0;  // whose step of a stage
  const int wf = wv % T::WF, wt = (T::KG == 2 ? wv & 3 : wv) / T::WF;
  const int WB = p.N / 2, XB = p.N * Mx<FMT>::kBits / 8, nb = p.N / 32;
  // stages of a tile (where the scale slots ask for it, one of zeros more)
  int stages = ((p.N + 127) / 128 + T::KG - 1) / T::KG;
  if (T::SL < T::ST) stages += stages % T::RUN == 1;
  // tiles in contiguous runs per XCD (blocks go to the XCDs in turn), a run
  // dealt to the XCD's blocks
  const int total = n_tiles * m_tiles, per_xcd = (total + 7) >> 3, stride = (int)gridDim.x >> 3;
  const int run_end = min(((int)blockIdx.x & 7) * per_xcd + per_xcd, total);
  const int first = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if (first >= run_end) return;

  struct Place {
    int k0, nk, nm;
    int64_t m0;
  };
  auto place = [&](int tile) {
    Place q;
    // groups of four tile rows, down the rows first: the XCD's 32 tiles of a
    // time are 4 x 8, which read less through its L2 than 1 x 32
    const int group = tile / (4 * n_tiles), r = tile - group * (4 * n_tiles);
    const int rows = min(4, m_tiles - 4 * group);
    const int nt = r / rows, mt = 4 * group + (r - nt * rows);
    q.k0 = nt * T::BK;
    q.m0 = (int64_t)mt * T::BM;
    q.nk = min(T::BK, p.K - q.k0);
    q.nm = (int)min((int64_t)T::BM, p.M - q.m0);
    return q;
  };

  // What the requests read: stage r_stage of tile r_tile, into slot r_slot.
  // Weight row r of a step is column r % BK of matrix r / BK.
  int r_tile = first, r_stage = 0, r_slot = 0, r_chunk = 0;
  rsrc_t rw[T::LW], rx, rs;
  int vw[T::LW], vx[T::LX], vs;
  const int sp = wv;  // its scale piece, if there is one
  auto w_piece = [&](int j) { return min(wv + j * T::NW, T::KG * T::PW - 1); };
  auto x_piece = [&](int j) { return min(wv + j * T::NW, T::KG * T::PX - 1); };
  auto aim = [&](int tile) {
    const Place q = place(tile);
#pragma unroll
    for (int j = 0; j < T::LW; ++j) {
      const int row = 16 * (w_piece(j) % T::PW), d = T::DUAL && row >= T::BK;
      rw[j] = make_rsrc(p.w[d] + (int64_t)q.k0 * WB, (uint32_t)(q.nk * WB));
      vw[j] = min(row - d * T::BK + (lane >> 2), q.nk - 1) * WB + 16 * ((lane & 3) ^ (3 * (lane >> 5)));
    }
    rx = make_rsrc(p.a + q.m0 * XB, (uint32_t)(q.nm * XB));
#pragma unroll
    for (int j = 0; j < T::LX; ++j) {
      const int i = x_piece(j) % T::PX;
      if constexpr (FMT == NVM_MX_FP4)
        vx[j] = min(16 * i + (lane >> 2), q.nm - 1) * XB + 16 * ((lane & 3) ^ (3 * (lane >> 5)));
      else
        vx[j] = min(8 * i + (lane >> 3), q.nm - 1) * XB +
                16 * ((lane & 7) ^ ((4 * i + (lane >> 4)) & 7));
    }
        if (sp < T::PSW) {
      const int d = sp / (T::WF * T::QF), w = sp % (T::WF * T::QF) / T::QF, ld = (int)p.ws_ld[d];
      rs = make_rsrc(p.ws[d] + (int64_t)q.k0 * ld, (uint32_t)(q.nk * ld));
      vs = min(w * (T::BK / T::WF) + 64 * (sp % T::QF) + lane, q.nk - 1) * ld;
    } else {
      const int ld = (int)p.as_ld, t = sp - T::PSW;
      rs = make_rsrc(p.as + q.m0 * ld, (uint32_t)(q.nm * ld));
      vs = min(t / T::QT * (T::BM / T::WT) + 64 * (t % T::QT) + lane, q.nm - 1) * ld;
    }
  };
  // load i of the stage's: scales (of its run's first stage), weights, activations
  auto load = [&](int i) {
    uint8_t *st = smem + r_slot * T::kStage;
    const int step = T::KG * r_stage;
    if (i == 0) {
      if (r_stage % T::RUN == 0 && sp < T::PS)
        lds_load16(rs, smem + T::kScales + r_chunk * T::kS + sp * 1024, vs, 4 * step);
    } else if (i <= T::LW) {
      const int j = i - 1, g = w_piece(j) / T::PW;
      lds_load16(rw[j], st + g * T::kStep + w_piece(j) % T::PW * 1024, vw[j], 64 * (step + g));
    } else {
      const int j = i - 1 - T::LW, g = x_piece(j) / T::PX;
      lds_load16(rx, st + g * T::kStep + T::kW + x_piece(j) % T::PX * 1024, vx[j],
                 T::XR * (step + g));
    }
  };
  auto advance = [&] {
    if (r_stage % T::RUN == 0) r_chunk = r_chunk + 1 == T::SL ? 0 : r_chunk + 1;
    r_slot = r_slot + 1 == T::ST ? 0 : r_slot + 1;
    if (++r_stage == stages) {
      r_stage = 0;
      r_tile += stride;
      if (r_tile < run_end) {
        aim(r_tile);
      } else {  // nothing more: the same loads, of nothing
#pragma unroll
        for (int j = 0; j < T::LW; ++j) rw[j] = make_rsrc(p.a, 0);
        rx = rs = make_rsrc(p.a, 0);
      }
    }
  };
  // All but the last ST - 2 requested stages have arrived.  (Where scales were
  // among the loads the wait is longer than it need be, never shorter.)
  auto arrived = [&] {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((T::ST - 2) * T::kLoads) : "memory");
  };

  // The wavefront's piece of scale slot c, row by row as it was loaded (lane l
  // has row l % 16 of tile l / 16: four steps of four blocks), to one dword of
  // four steps per (block, row, tile): a lane then reads four tiles' scales of
  // its block at once.  (Read a byte a tile and step, scales took as long as
  // 16 bytes each: 380 of 980 cycles of a stage's reading.)
  auto turn = [&](int c) {
    if (sp >= T::PS) return;
    uint8_t *at = smem + T::kScales + c * T::kS + sp * 1024;
    const u32x4 d = *(const u32x4 *)(at + 16 * lane);
    const uint32_t a = perm_b32(d[1], d[0], 0x05010400u), b = perm_b32(d[1], d[0], 0x07030602u);
    const uint32_t e = perm_b32(d[3], d[2], 0x05010400u), f = perm_b32(d[3], d[2], 0x07030602u);
    uint32_t *o = (uint32_t *)at + 4 * (lane & 15) + (lane >> 4);
    wave_lds_sync();
    o[0] = perm_b32(e, a, 0x05040100u);
    o[64] = perm_b32(e, a, 0x07060302u);
    o[128] = perm_b32(f, b, 0x05040100u);
    o[192] = perm_b32(f, b, 0x07060302u);
  };

  // places in a stage and a scale slot that the wavefront's operands are read from
  const int wrow = wf * (T::BK / T::WF) + col, xrow = wt * (T::BM / T::WT) + col;
  const int aw = kg * T::kStep + wrow * 64 + 16 * (G ^ (3 * (col >> 3)));
  int ax[NX];
#pragma unroll
  for (int c = 0; c < NX; ++c)
    ax[c] = kg * T::kStep + T::kW + xrow * T::XR +
            16 * (FMT == NVM_MX_FP4 ? G ^ (3 * (col >> 3)) : (4 * c + G) ^ ((col >> 1) & 7));
  const int aws = T::kScales + wf * (T::QF * 1024) + 256 * G + 16 * col;
  const int axs = T::kScales + (T::PSW + wt * T::QT) * 1024 + 256 * G + 16 * col;
  // weight tile f of the wavefront: rows further on in the stage
  auto ftile = [](int f) { return T::DUAL && f >= T::TF / 2 ? T::BK + 16 * (f - T::TF / 2) : 16 * f; };

  const bool late = wv >= 4;
  auto phase_end = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  aim(first);
  for (int n = T::ST - 1; n > 0; --n) {
#pragma unroll
    for (int i = 0; i <= T::kLoads; ++i) load(i);
    advance();
  }
  // the first stage, of every wavefront
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  turn(0);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  // wavefronts 4 to 7 run half a stage behind the others
  if (late) __builtin_amdgcn_s_barrier();
  int slot = 0, chunk = T::SL - 1;
  for (int tile = first; tile < run_end; tile += stride) {
    f32x4 acc[T::TF][T::TM];
#pragma unroll
    for (int f = 0; f < T::TF; ++f)
#pragma unroll
      for (int t = 0; t < T::TM; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Scale bytes of the lane's block in the steps to come, the next lowest
    // (the matrix instruction takes a register's low byte).
    uint32_t ws[T::TF], xs[T::TM];
    for (int s = 0;; ++s) {
      if (s % T::RUN == 0) {
        chunk = chunk + 1 == T::SL ? 0 : chunk + 1;
        const uint8_t *sc = smem + chunk * T::kS;
        constexpr int FM = T::TF / T::NM;  // tiles of a matrix
#pragma unroll
        for (int f = 0; f < T::TF; f += f % FM + 4 < FM ? 4 : FM - f % FM) {
          const u32x4 d = *(const u32x4 *)(sc + aws + (f / FM * T::WF * T::QF + f % FM / 4) * 1024);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (f % FM + i < FM) ws[f + i] = d[i] >> (8 * kg);
        }
#pragma unroll
        for (int t = 0; t < T::TM; t += 4) {
          const u32x4 d = *(const u32x4 *)(sc + axs + t / 4 * 1024);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t + i < T::TM) xs[t + i] = d[i] >> (8 * kg);
        }
      } else {
#pragma unroll
        for (int f = 0; f < T::TF; ++f) ws[f] >>= 8 * T::KG;
#pragma unroll
        for (int t = 0; t < T::TM; ++t) xs[t] >>= 8 * T::KG;
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
#pragma unroll
        for (int c = 0; c < NX; ++c) x[t].v[c] = *(const u32x4 *)(st + ax[c] + t * 16 * T::XR);
      }
#pragma unroll
      for (int f = 0; f < T::TF; ++f) {
        next(T::TM + f);
        w[f].v[0] = *(const u32x4 *)(st + aw + ftile(f) * 64);
      }
      advance();
      const int step = T::KG * s + kg;
      if (128 * step + 128 > p.N) {  // a last step that the row ends in or before
#pragma unroll
        for (int t = 0; t < T::TM; ++t) {
#pragma unroll
          for (int c = 0; c < NX; ++c)
            if (128 * step + (FMT == NVM_MX_FP4 ? 32 * G : 64 * c + 16 * G) >= p.N)
              x[t].v[c] = u32x4{0u, 0u, 0u, 0u};
          if (4 * step + G >= nb) xs[t] = 127u;
        }
#pragma unroll
        for (int f = 0; f < T::TF; ++f)
          if (4 * step + G >= nb) ws[f] = 127u;
      }
      arrived();
      if (s + 1 == stages || (s + 1) % T::RUN == 0) turn(chunk + 1 == T::SL ? 0 : chunk + 1);
      // This stage's operands are in registers, the next run's scales in place.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int f = 0; f < T::TF; ++f) {
#pragma unroll
        for (int t = 0; t < T::TM; ++t)
          acc[f][t] = mx_mfma<FMT>(w[f], ws[f], x[t], xs[t], acc[f][t]);
      }
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      slot = slot + 1 == T::ST ? 0 : slot + 1;
      if (s + 1 == stages) break;
      phase_end();
    }
    // Wavefronts 4 to 7 meet the tile's last barrier behind their epilogue, so
    // that it runs along with the others' (one after the other, they cost a
    // tile of 16 steps 6500 of 50000 cycles).
    if (T::KG == 2 || !late) phase_end();

    // KG = 2: each wavefront of a pair (w, w + 4) finishes one half of their
    // activation tiles and hands its sums of the other half over through the
    // stages, which nothing is loaded into any more.
    constexpr int TM = T::TM / T::KG;  // activation tiles that a wavefront finishes
    if constexpr (T::KG == 2) {
      f32x4 *mine = (f32x4 *)smem + wv * (T::TF * TM * 64) + lane;
      const f32x4 *other = (const f32x4 *)smem + (wv ^ 4) * (T::TF * TM * 64) + lane;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (!late) __builtin_amdgcn_s_barrier();  // the last step of 4 to 7 has been read
#pragma unroll
      for (int f = 0; f < T::TF; ++f)
#pragma unroll
        for (int t = 0; t < TM; ++t) mine[(f * TM + t) * 64] = kg ? acc[f][t] : acc[f][TM + t];
      __syncthreads();
#pragma unroll
      for (int f = 0; f < T::TF; ++f)
#pragma unroll
        for (int t = 0; t < TM; ++t)
          acc[f][t] = (kg ? acc[f][TM + t] : acc[f][t]) + other[(f * TM + t) * 64];
    }
    const Place q = place(tile);
    // (computed here: hoisted out of the tile loop, the epilogue's addresses
    // cost the k-loop its registers)
    int el = lane;
    asm volatile("" : "+v"(el));
    const int mrow = wt * (T::BM / T::WT) + 16 * TM * kg + (el & 15);
    if constexpr (!T::DUAL) {
      auto store = [&](auto DTYPE, auto WHOLE) {
#pragma unroll
        for (int t = 0; t < TM; ++t) {
          const int m = mrow + 16 * t;
          const int64_t row = (q.m0 + m) * p.K + q.k0;
          if constexpr (decltype(WHOLE)::value) {
            // (an odd last tile: with zeros that are not stored)
            const int k = wf * (T::BK / T::WF), end = min(q.nk, k + 16 * T::TF);
#pragma unroll
            for (int f = 0; f < T::TF; f += 2)
              mx_store_pair<decltype(DTYPE)::value>(
                  p.out, el >> 4, row, k + 16 * f, m < q.nm ? end : 0, acc[f][t],
                  f + 1 < T::TF ? acc[f + 1 < T::TF ? f + 1 : f][t] : f32x4{0.f, 0.f, 0.f, 0.f});
          } else {
            if (m < q.nm)
#pragma unroll
              for (int f = 0; f < T::TF; ++f)
                mx_store4<decltype(DTYPE)::value>(p.out, row, wf * (T::BK / T::WF) + 16 * f + 4 * (el >> 4),
                                                  q.nk, acc[f][t]);
          }
        }
      };
      mx_by_dtype(p.out_dtype, [&](auto DTYPE) {
        if (p.K % 8 == 0)
          store(DTYPE, std::true_type{});
        else
          store(DTYPE, std::false_type{});
      });
    } else {
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        const int m = mrow + 16 * t;
#pragma unroll
        for (int f = 0; f < T::TF / 2; f += 2) {
          const int k = wf * (T::BK / T::WF) + 16 * f;
          float h[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            h[e] = mx_swiglu(acc[f + (e >> 2)][t][e & 3], acc[T::TF / 2 + f + (e >> 2)][t][e & 3]);
          mx_store_block<OFMT>(h, el >> 4, m < q.nm && k < q.nk, q.m0 + m, q.k0 + k, p);
        }
      }
    }
    if (T::KG == 1 && late) phase_end();
  }
  // (no load may write to LDS behind the block's end)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (T::KG == 1 && !late) __builtin_amdgcn_s_barrier();
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
  const int64_t m_tiles = (a.M + T::BM - 1) / T::BM, total = m_tiles * n_tiles;
  if (total > kMxMaxTiles) return hipErrorInvalidConfiguration;
  // (KG = 2: the exchange of sums takes the stages, so a tile a block)
  const int64_t all = 8 * ((total + 7) / 8);
  const int64_t grid = T::KG == 2 ? all : std::min<int64_t>(all, cu_count() / 8 * 8);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * T::NW), T::kLds, st, a, n_tiles,
                     (int)m_tiles);
  return hipGetLastError();
}

#ifndef CFG
#define CFG 256, 256, 2, 4, 1
#endif
template <int FMT>
hipError_t launch_fmt(bool dual, int out_format, const MxMatmulArgs &a, hipStream_t st) {
  constexpr int ST = FMT == NVM_MX_FP4 ? 4 : 3;
#ifdef DUALONLY
  return go<FMT, NVM_MX_FP8, Tile<FMT, true, CFG, ST>>(a, st);
#else
  if (!dual) return go<FMT, NVM_MX_FP8, Tile<FMT, false, CFG, ST>>(a, st);
#ifndef NODUAL
  using Dual = Tile<FMT, true, CFG, ST>;
  return out_format == NVM_MX_FP4 ? go<FMT, NVM_MX_FP4, Dual>(a, st)
                                  : go<FMT, NVM_MX_FP8, Dual>(a, st);
#else
  return hipErrorInvalidValue;
#endif
#endif
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
