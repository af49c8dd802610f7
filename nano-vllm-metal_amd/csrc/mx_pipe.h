// Products of MX rows with MXFP4 weights (include/nvm_mx.h) between decode
// batches (mx_gemv.hip) and grids that tiles of 256 x 256 fill (mx_gemm.hip):
// prompts of some hundred rows.  Codes and scales go through LDS into the
// matrix instructions as they do there; the tiles are smaller, so that there are
// enough of them, and time goes by stages.
//
// Bound: of E4M3 the bf16 products (256 x 128, a round of 16 stages in 25 us: 1.4
// PFLOP/s, the library's rate).  Of E2M1, and in short sums, of which the figures
// to come are, the loads into LDS.  128 x 128 with KG = 2 (24 stages, 6144 -> 2048 of
// 512 rows, 23 us): 9 us without reading or multiplying, products alone 19, LDS
// reads alone 12, loads alone 22; a deeper ring changes nothing (2 stages 29
// us, 3 23, and of E2M1, which leaves room, 3 as fast as 4).  So where 128 x 128
// leaves CUs idle, smaller tiles are faster though they load more: those 512 rows
// 16.5 us on 128 x 64, 14.1 on 64 x 64, of which two blocks fit a CU.
//  * Every wavefront reads stage j + 1's operands from LDS into registers and
//    requests stage j + ST while it multiplies stage j's, instruction by
//    instruction side by side: one barrier a stage.
//  * A run of four steps is unrolled, because the scaled matrix instruction takes
//    the scale byte of a step as an immediate.  Its scales are requested two runs
//    ahead, turned (MxTile::turn) one ahead, read at the end of the run before.
//  * KG = 2: rows are loaded 128 bytes at a time, and few tiles still have
//    eight wavefronts, each with a 64 x 64 piece of the tile to multiply.
//  * KG = 1: blocks may have several tiles, and requests run on across them.
//  * A last run of less than 512 values is computed with the activations behind
//    the row replaced by zeros and scales by one in registers.
//
// 6144 -> 2048: 512 rows 20.7 us (0.62 PFLOP/s), 1024 rows 30.2 us on 128 x 64
// (0.85), 4096 rows 79.8 us on 256 x 128 (1.29); in short sums 14.1, 20.2 and 45.5.
#pragma once

#include "mx_tile.h"

namespace nvm {

// The block's tiles first, first + stride, ... below `last` (KG = 2: one), at
// place(tile).
template <int FMT, int OFMT, class T, class F>
__device__ __forceinline__ void mx_pipe_tiles(const MxMatmulArgs &p, uint8_t *smem, int first,
                                              int last, int stride, F place) {
  // (the wait for a stage covers the scales of its run: they are requested
  // RUN - 1 stages before they are turned)
  static_assert(T::SL == 2 && T::RUN - 1 >= T::ST - 2, "scales arrive with their stages");
  constexpr int NX = FMT == NVM_MX_FP4 ? 1 : 2;
  const int lane = threadIdx.x & 63, G = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int kg = T::KG == 2 ? wv >> 2 : 0;  // whose step of a stage
  const int wf = wv % T::WF, wt = (T::KG == 2 ? wv & 3 : wv) / T::WF;
  const int nb = p.N / 32, runs = (p.N + 511) / 512;
  // What the loads read: run d_run of tile d_tile, and run s_run of s_tile's
  // scales, which are requested earlier.
  int d_tile = first, d_run = 0, s_tile = first, s_run = 0;
  typename T::Source src;
  typename T::ScaleSource scales;
  auto aim = [&] {
    if (d_tile >= last)
      src.none(p);
    else
      src.aim(p, place(d_tile), wv, lane);
  };
  auto aim_scales = [&] {
    if (s_tile >= last)
      scales.s = make_rsrc(p.a, 0);
    else
      scales.aim(p, place(s_tile), wv, lane);
  };
  // load i of stage j of the run, into a slot
  auto load = [&](int i, int j, uint8_t *to) { src.load(i, 4 * d_run + T::KG * j, to, wv); };
  uint8_t *const piece = smem + T::kScales + wv * 1024;  // the wavefront's of a scale slot
  auto load_scales = [&](int c) {
    if (wv < T::PS) lds_load16(scales.s, piece + c * T::kS, scales.v, 16 * s_run);
    if (++s_run == runs) {
      s_run = 0;
      s_tile += stride;
      aim_scales();
    }
  };
  u32x4 raw;
  auto turn_read = [&](int c) {
    if (wv < T::PS) raw = *(const u32x4 *)(piece + c * T::kS + 16 * lane);
  };
  auto turn_write = [&](int c) {
    if (wv < T::PS) T::turn(piece + c * T::kS, raw, lane);
  };
  const typename T::Reads at(wf, wt, kg, lane);
  struct Frags {
    MxFrag<NVM_MX_FP4> w[T::TF];
    MxFrag<FMT> x[T::TM];
  };
  constexpr int NR = T::TF + T::TM;  // operand tiles
  auto read = [&](Frags &q, int i, const uint8_t *stage) {
    if (i < T::TM)
      q.x[i] = at.act(stage, i);
    else
      q.w[i - T::TM] = at.weight(stage, i - T::TM);
  };
  auto sync = [] {
    // (the builtin, not asm: the compiler counts on it for the operands that
    // were read before)
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  aim();
  aim_scales();
  load_scales(0);
  load_scales(1);
  // (stage j of a run: slot j where the ring is a run, else in turn)
  constexpr bool ring = T::ST == T::RUN;
  int r_slot = 0, slot = 0;  // loaded, read next
  auto next = [](int v) { return v + 1 == T::ST ? 0 : v + 1; };
  auto next_run = [&] {
    if (++d_run == runs) {
      d_run = 0;
      d_tile += stride;
      aim();
    }
  };
#pragma unroll
  for (int n = 0; n < T::ST; ++n) {
    if (n > 0 && n % T::RUN == 0) next_run();
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) load(i, n % T::RUN, smem + n * T::kStage);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  turn_read(0);
  turn_write(0);
  turn_read(1);
  sync();
  Frags fr[2];
  typename T::Scales sc[2];
#pragma unroll
  for (int i = 0; i < NR; ++i) read(fr[0], i, smem);
  sc[0].read(smem, at, 0, kg);
  int chunk = 0;  // scale slot of the run

  for (int tile = first; tile < last; tile += stride) {
    f32x4 acc[T::TF][T::TM];
#pragma unroll
    for (int f = 0; f < T::TF; ++f)
#pragma unroll
      for (int t = 0; t < T::TM; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Stage J of run r: its products, while stage J + 1's operands are read and
    // stage J + ST is requested into the slot that every wavefront has read.
    auto do_stage = [&](auto STAGE, auto TAIL, int r) {
      constexpr int J = decltype(STAGE)::value;
      Frags &q = fr[J & 1], &n = fr[(J + 1) & 1];
      // Everything that branches comes first: the products have to be in one
      // basic block with the reads and loads to be interleaved with them.
      // (Stage J + 1 has arrived when the ST - 2 later ones are outstanding;
      // a load of scales among them makes the wait longer, never shorter.)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((T::ST - 2) * T::kLoads) : "memory");
      sync();
      if constexpr ((J + T::ST) % T::RUN == 0) next_run();
      if constexpr (J == 0) {
        load_scales(chunk);  // of the run after the next (this run's are in registers)
        turn_write(chunk ^ 1);
      }
      if constexpr (J + 1 == T::RUN) turn_read(chunk);
      uint8_t *const to = smem + (ring ? J : r_slot) * T::kStage;
      const uint8_t *const from = smem + (ring ? (J + 1) % T::ST : next(slot)) * T::kStage;
      if constexpr (decltype(TAIL)::value) {
        const int step = 4 * r + T::KG * J + kg;
#pragma unroll
        for (int t = 0; t < T::TM; ++t)
#pragma unroll
          for (int c = 0; c < NX; ++c)
            if (128 * step + mx_act_at<FMT>(G, c) >= p.N)
              q.x[t].v[c] = u32x4{0u, 0u, 0u, 0u};
        if constexpr (J == 0) {
          const int in = min(max((nb - 16 * r - G + 3) >> 2, 0), 4);  // steps inside
          const uint32_t out = in == 4 ? 0u : (0xFFFFFFFFu << (8 * in)) >> (8 * kg);
#pragma unroll
          for (int f = 0; f < T::TF; ++f) sc[0].w[f] = (sc[0].w[f] & ~out) | (0x7F7F7F7Fu & out);
#pragma unroll
          for (int t = 0; t < T::TM; ++t) sc[0].x[t] = (sc[0].x[t] & ~out) | (0x7F7F7F7Fu & out);
        }
      }
      if constexpr (J + 1 == T::RUN) sc[1].read(smem, at, chunk ^ 1, kg);
      __builtin_amdgcn_sched_barrier(0);
      mx_products<FMT, T::KG * J>(q.w, sc[0].w, q.x, sc[0].x, acc, [&](int part) {
        constexpr int of = mx_parts<FMT, T::TF>;
        if (part > 0) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = part * NR / of; i < (part + 1) * NR / of; ++i) read(n, i, from);
#pragma unroll
        for (int i = part * T::kLoads / of; i < (part + 1) * T::kLoads / of; ++i)
          load(i, (J + T::ST) % T::RUN, to);
      });
      __builtin_amdgcn_sched_barrier(0);
      // (computed here: the compiler would move products whose sums it needs
      // later only past the next barrier)
#pragma unroll
      for (int f = 0; f < T::TF; ++f)
#pragma unroll
        for (int t = 0; t < T::TM; ++t) asm volatile("" : "+v"(acc[f][t]));
      if constexpr (!ring) {
        r_slot = next(r_slot);
        slot = next(slot);
      }
    };
    auto do_run = [&](auto TAIL, int r) {
      do_stage(MxInt<0>{}, TAIL, r);
      do_stage(MxInt<1>{}, TAIL, r);
      if constexpr (T::RUN == 4) {
        do_stage(MxInt<2>{}, TAIL, r);
        do_stage(MxInt<3>{}, TAIL, r);
      }
      sc[0] = sc[1];
      chunk ^= 1;
    };
    const int full = p.N / 512;
    for (int r = 0; r < full; ++r) do_run(std::false_type{}, r);
    if (full < runs) do_run(std::true_type{}, full);
    // KG = 2: each wavefront of a pair (w, w + 4) finishes one half of their
    // activation tiles and hands its sums of the other half over through the
    // stages, which nothing is loaded into any more (a tile a block).
    constexpr int TN = T::TM / T::KG;  // activation tiles that a wavefront finishes
    if constexpr (T::KG == 2) {
      f32x4 *mine = (f32x4 *)smem + wv * (T::TF * TN * 64) + lane;
      const f32x4 *other = (const f32x4 *)smem + (wv ^ 4) * (T::TF * TN * 64) + lane;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      sync();  // (the last stage's loads and reads)
#pragma unroll
      for (int f = 0; f < T::TF; ++f)
#pragma unroll
        for (int t = 0; t < TN; ++t) mine[(f * TN + t) * 64] = kg ? acc[f][t] : acc[f][TN + t];
      __syncthreads();
#pragma unroll
      for (int f = 0; f < T::TF; ++f)
#pragma unroll
        for (int t = 0; t < TN; ++t)
          acc[f][t] = (kg ? acc[f][TN + t] : acc[f][t]) + other[(f * TN + t) * 64];
    }
    T::template finish<OFMT, TN>(p, place(tile), acc, wf,
                                 wt * (T::BM / T::WT) + 16 * TN * kg, lane);
  }
  // (no load may write to LDS behind the block's end)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

}  // namespace nvm
