// What the products of many MX rows share (mx_gemm.hip, mx_pipe.h): a block's
// tile and its layout in LDS, the order of the tiles, the turn of the scales,
// the epilogue.
#pragma once

#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "mx_common.h"

namespace nvm {

__device__ __forceinline__ void lds_load16(rsrc_t r, void *lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16,
                                           voff, soff, 0, 0);
}

// BN weight rows (DUAL: half of them gate, half up) and BM activation rows a
// block of eight wavefronts, two on a SIMD.  KG = 1: WF x WT = 8 wavefronts
// share a 128-value step, which is a stage.  KG = 2: a stage is two steps,
// wavefronts 0 to 3 (WF x WT = 4 over the whole tile) take the first and 4 to
// 7 the second, and the two sums are joined at the end.  LDS holds a ring of ST
// stages and one of SL scale slots.
template <int FMT, bool DUAL_, int BN_, int BM_, int WF_, int WT_, int KG_, int ST_, int SL_>
struct MxTile {
  static constexpr bool DUAL = DUAL_;
  static constexpr int BN = BN_, BM = BM_, WF = WF_, WT = WT_, KG = KG_, ST = ST_, SL = SL_;
  static constexpr int NW = 8;
  static constexpr int NM = DUAL ? 2 : 1;                     // matrices
  static constexpr int BK = BN / NM;                          // output columns
  static constexpr int TF = BN / WF / 16, TM = BM / WT / 16;  // a wavefront's 16-row tiles
  static constexpr int FM = TF / NM;                          // its weight tiles of a matrix
  // Bytes of a row in LDS.  KG = 2: 128 of a weight row are the stage's two
  // steps, and so are 128 of E2M1 activations; E4M3: 128 are a step, and the
  // stage has XS = 2 of them one behind the other.
  static constexpr int WR = 64 * KG, XR = FMT == NVM_MX_FP4 ? WR : 128;
  static constexpr int XS = FMT == NVM_MX_FP4 ? 1 : KG;
  // pieces of 1 KB, a load each; of a scale slot: 64 rows of a matrix or of
  // the activations
  static constexpr int PW = BN * WR / 1024, PX = BM * XR / 1024;
  static constexpr int PSM = BK / 64, PSW = NM * PSM, PS = PSW + BM / 64;
  static constexpr int kW = PW * 1024, kX = PX * 1024, kS = PS * 1024;
  static constexpr int kStage = kW + XS * kX, kScales = ST * kStage, kLds = kScales + SL * kS;
  static constexpr int RUN = 4 / KG;  // stages of a scale slot, which holds four steps
  // a wavefront's loads of a stage: pieces wv, wv + NW, ...
  static constexpr int LW = PW / NW, LX = XS * PX / NW, kLoads = LW + LX;
  static_assert(PW % NW == 0 && PX % NW == 0, "whole loads");
  static_assert(BK % 64 == 0 && BM % 64 == 0, "whole scale pieces");
  static_assert(KG * WF * WT == NW && PS <= NW && kLds <= 160 * 1024, "a block's LDS and loads");
  static_assert(BK % (32 * WF) == 0 && BM % (16 * WT) == 0, "whole pairs of tiles of a wavefront");
  static_assert(KG == 1 || (TM % 2 == 0 && TF * TM * 4096 <= kScales), "the sums' exchange");
  static_assert((FM == 2 || FM % 4 == 0) && (TM == 2 || TM % 4 == 0), "whole reads of scales");

  // 16-byte chunk k of row r of W bytes lies at place k ^ turned.  A 16-byte
  // LDS read is served 16 lanes at a time: lanes 0-3, 12-15 and 20-27, then
  // 4-11, 16-19 and 28-31 (and the same of the upper half), so rows 0-3 and
  // 12-15 at one chunk with rows 4-11 at its neighbour k ^ 1; with these those
  // fall into 16 different 16-byte groups of the 256-byte bank cycle.  (With
  // (r >> 2) & 3, right for 16 consecutive lanes, every weight read took a
  // second access: 448 conflict cycles a block and step of 2800.)  The loads'
  // lane-to-chunk assignment makes the order: LDS is written in lane order.
  template <int W>
  static __device__ __forceinline__ int turned(int r) {
    return W == 64 ? 3 * ((r >> 3) & 1) : (r >> 1) & 7;
  }
  // row and source byte of the lane's 16 of a piece
  template <int W>
  static __device__ __forceinline__ int piece_row(int piece, int lane) {
    return piece * (1024 / W) + lane / (W / 16);
  }
  template <int W>
  static __device__ __forceinline__ int piece_at(int piece, int lane) {
    return 16 * (lane % (W / 16) ^ turned<W>(piece_row<W>(piece, lane)));
  }
  // The same of activation rows.  (E4M3 that is converted to bf16: a lane group's
  // chunks are 2 G and 2 G + 1, the neighbour's k ^ 2, so the places of rows 0-3
  // and 12-15, turned by even numbers, and those of rows 4-11, by odd ones, are
  // closed under that.)
  static __device__ __forceinline__ int turned_act(int r) {
    if constexpr (FMT != NVM_MX_FP8) return turned<XR>(r);
    const int i = r >> 1;
    return (i & 4) | ((i & 1) << 1) | ((i >> 1 ^ i >> 2) & 1);
  }
  static __device__ __forceinline__ int act_piece_at(int piece, int lane) {
    return 16 * (lane % (XR / 16) ^ turned_act(piece_row<XR>(piece, lane)));
  }

  // Where the loads of an output tile read.  Weight row r of a stage is column
  // r % BK of matrix r / BK; rows past an operand repeat its last row, whose
  // outputs are not stored.
  struct Place {
    int k0, nk, nm;
    int64_t m0;
  };
  static __device__ __forceinline__ Place place(const MxMatmulArgs &p, int tile, int n_tiles,
                                                int m_tiles) {
    Place q;
    // groups of four tile rows, down the rows first: the XCD's 32 tiles of a
    // time are 4 x 8, which read less through its L2 than 1 x 32
    const int group = tile / (4 * n_tiles), r = tile - group * (4 * n_tiles);
    const int rows = min(4, m_tiles - 4 * group);
    const int nt = r / rows, mt = 4 * group + (r - nt * rows);
    q.k0 = nt * BK;
    q.m0 = (int64_t)mt * BM;
    q.nk = min(BK, p.K - q.k0);
    q.nm = (int)min((int64_t)BM, p.M - q.m0);
    return q;
  }
  struct Source {
    rsrc_t w[LW], x;
    int vw[LW], vx[LX];
    __device__ __forceinline__ void none(const MxMatmulArgs &p) {  // the same loads, of nothing
#pragma unroll
      for (int j = 0; j < LW; ++j) w[j] = make_rsrc(p.a, 0);
      x = make_rsrc(p.a, 0);
    }
    __device__ __forceinline__ void aim(const MxMatmulArgs &p, const Place &q, int wv, int lane) {
      const int WB = p.N / 2, XB = p.N * Mx<FMT>::kBits / 8;
#pragma unroll
      for (int j = 0; j < LW; ++j) {
        const int i = wv + j * NW, d = DUAL && i * (1024 / WR) >= BK;
        w[j] = make_rsrc(p.w[d] + (int64_t)q.k0 * WB, (uint32_t)(q.nk * WB));
        vw[j] = min(piece_row<WR>(i, lane) - d * BK, q.nk - 1) * WB + piece_at<WR>(i, lane);
      }
      x = make_rsrc(p.a + q.m0 * XB, (uint32_t)(q.nm * XB));
#pragma unroll
      for (int j = 0; j < LX; ++j) {
        const int i = wv + j * NW % PX;
        vx[j] = min(piece_row<XR>(i, lane), q.nm - 1) * XB + act_piece_at(i, lane) +
                128 * (j * NW / PX);
      }
    }
    // load i of a stage that starts with 128-value step `step`
    __device__ __forceinline__ void load(int i, int step, uint8_t *stage, int wv) const {
      uint8_t *const mine = stage + wv * 1024;
      if (i < LW)
        lds_load16(w[i], mine + i * NW * 1024, vw[i], 64 * step);
      else
        lds_load16(x, mine + kW + (i - LW) * NW * 1024, vx[i - LW],
                   (FMT == NVM_MX_FP4 ? 64 : 128) * step);
    }
  };
  struct ScaleSource {  // of wavefronts 0 to PS - 1, a piece each
    rsrc_t s;
    int v;
    __device__ __forceinline__ void aim(const MxMatmulArgs &p, const Place &q, int wv, int lane) {
      if (wv < PSW) {
        const int d = wv / PSM, ld = (int)p.ws_ld[d];
        s = make_rsrc(p.ws[d] + (int64_t)q.k0 * ld, (uint32_t)(q.nk * ld));
        v = min(64 * (wv % PSM) + lane, q.nk - 1) * ld;
      } else {
        const int ld = (int)p.as_ld;
        s = make_rsrc(p.as + q.m0 * ld, (uint32_t)(q.nm * ld));
        v = min(64 * (wv - PSW) + lane, q.nm - 1) * ld;
      }
    }
  };

  // A piece of scales lies as it was loaded, lane l's 16 bytes (`raw`) the
  // four steps of four blocks of row l % 16 of tile l / 16.  It is turned into
  // one dword of four steps per (block, row, tile), so that a lane reads its
  // block's of four tiles at once.  (Read a byte a tile and step, scales took
  // as long as 16 bytes each: 380 of 980 cycles of a step's reading.)
  static __device__ __forceinline__ void turn(uint8_t *piece, u32x4 raw, int lane) {
    const uint32_t a = perm_b32(raw[1], raw[0], 0x05010400u);
    const uint32_t b = perm_b32(raw[1], raw[0], 0x07030602u);
    const uint32_t e = perm_b32(raw[3], raw[2], 0x05010400u);
    const uint32_t f = perm_b32(raw[3], raw[2], 0x07030602u);
    uint32_t *o = (uint32_t *)piece + 4 * (lane & 15) + (lane >> 4);
    o[0] = perm_b32(e, a, 0x05040100u);
    o[64] = perm_b32(e, a, 0x07060302u);
    o[128] = perm_b32(f, b, 0x05040100u);
    o[192] = perm_b32(f, b, 0x07060302u);
  }

  // Where a wavefront's operands are read from: bytes of a stage and of LDS.
  struct Reads {
    int w, x[FMT == NVM_MX_FP4 ? 1 : 2], ws, xs;
    __device__ __forceinline__ Reads(int wf, int wt, int kg, int lane) {
      const int col = lane & 15, G = lane >> 4;
      const int wrow = wf * (BK / WF) + col, xrow = wt * (BM / WT) + col;
      const int g = KG == 2 ? 4 * kg + G : G;  // chunk of the two steps in a row
      w = wrow * WR + 16 * (g ^ turned<WR>(wrow));
      if constexpr (FMT == NVM_MX_FP4) {
        x[0] = kW + xrow * XR + 16 * (g ^ turned_act(xrow));
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c)
          x[c] = kW + kg * kX + xrow * XR +
                 16 * ((mx_act_at<FMT>(G, c) / 16) ^ turned_act(xrow));
      }
      auto scale_at = [](int tile) { return tile / 4 * 1024 + 4 * (tile % 4); };
      ws = kScales + scale_at(wf * FM) + 256 * G + 16 * col;
      xs = kScales + PSW * 1024 + scale_at(wt * TM) + 256 * G + 16 * col;
    }
    __device__ __forceinline__ MxFrag<FMT> act(const uint8_t *stage, int t) const {
      MxFrag<FMT> q;
#pragma unroll
      for (int c = 0; c < (FMT == NVM_MX_FP4 ? 1 : 2); ++c)
        q.v[c] = *(const u32x4 *)(stage + x[c] + t * 16 * XR);
      return q;
    }
    __device__ __forceinline__ MxFrag<NVM_MX_FP4> weight(const uint8_t *stage, int f) const {
      MxFrag<NVM_MX_FP4> q;
      q.v[0] = *(const u32x4 *)(stage + w + (f / FM * BK + f % FM * 16) * WR);
      return q;
    }
  };
  // A run's scale bytes, step by step from the lowest byte on.
  struct Scales {
    uint32_t w[TF], x[TM];
    template <int n>
    static __device__ __forceinline__ void tiles(const uint8_t *at, uint32_t *o, int kg) {
      if constexpr (n == 2) {
        const u32x2 d = *(const u32x2 *)at;
        o[0] = d.x >> (8 * kg);
        o[1] = d.y >> (8 * kg);
      } else {
#pragma unroll
        for (int i = 0; i < n; i += 4) {
          const u32x4 d = *(const u32x4 *)(at + i / 4 * 1024);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i + e] = d[e] >> (8 * kg);
        }
      }
    }
    __device__ __forceinline__ void read(const uint8_t *smem, const Reads &at, int slot, int kg) {
      const uint8_t *sc = smem + slot * kS;
#pragma unroll
      for (int d = 0; d < NM; ++d) tiles<FM>(sc + at.ws + d * PSM * 1024, w + d * FM, kg);
      tiles<TM>(sc + at.xs, x, kg);
    }
  };

  // A wavefront's sums of activation tiles 0 .. TN - 1 (the first of them row
  // m_first of the tile) to the output.
  template <int OFMT, int TN>
  static __device__ __forceinline__ void finish(const MxMatmulArgs &p, const Place &q,
                                                const f32x4 (&acc)[TF][TM], int wf, int m_first,
                                                int lane) {
    // (computed here: hoisted out of the tile loop, the addresses cost the
    // k-loop its registers)
    int el = lane;
    asm volatile("" : "+v"(el));
    const int G = el >> 4, mrow = m_first + (el & 15), kw = wf * (BK / WF);
    if constexpr (!DUAL) {
      auto store = [&](auto DTYPE, auto WHOLE) {
        constexpr int DT = decltype(DTYPE)::value;
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          const int m = mrow + 16 * t;
          const int64_t row = (q.m0 + m) * p.K + q.k0;
          if constexpr (decltype(WHOLE)::value) {
#pragma unroll
            for (int f = 0; f < TF; f += 2)
              mx_store_pair<DT>(p.out, G, row, kw + 16 * f, m < q.nm ? q.nk : 0, acc[f][t],
                                acc[f + 1][t]);
          } else {
            if (m < q.nm)
#pragma unroll
              for (int f = 0; f < TF; ++f)
                mx_store4<DT>(p.out, row, kw + 16 * f + 4 * G, q.nk, acc[f][t]);
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
      for (int t = 0; t < TN; ++t) {
        const int m = mrow + 16 * t;
#pragma unroll
        for (int f = 0; f < FM; f += 2) {
          const int k = kw + 16 * f;
          float h[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            h[e] = mx_swiglu(acc[f + (e >> 2)][t][e & 3], acc[FM + f + (e >> 2)][t][e & 3]);
          mx_store_block<OFMT>(h, G, m < q.nm && k < q.nk, q.m0 + m, q.k0 + k, p);
        }
      }
    }
  }
};

// 128 outputs (gate/up: 64 of each) by 128 rows, and 256 by 128 (mx_pipe.h).
template <int FMT, bool DUAL>
using MxSmallTile = MxTile<FMT, DUAL, 128, 128, 2, 2, 2, 3, 2>;
template <int FMT, bool DUAL>
using MxWideTile = MxTile<FMT, DUAL, 256, 128, 4, 2, 1, 4, 2>;

// Output tiles of T; false: more than kMxMaxTiles.
template <class T>
bool mx_count_tiles(const MxMatmulArgs &a, int &n_tiles, int &m_tiles) {
  const int64_t n = ((int64_t)a.K + T::BK - 1) / T::BK, m = (a.M + T::BM - 1) / T::BM;
  if (n * m > kMxMaxTiles) return false;
  n_tiles = (int)n;
  m_tiles = (int)m;
  return true;
}

// More than 64 KB of dynamic LDS is allowed once per device and kernel (a
// failure shows up as a failed launch).
template <class F>
void mx_allow_lds(F kern, int bytes, bool (&allowed)[64]) {
  int dev = 0;
  if (hipGetDevice(&dev) == hipSuccess && dev >= 0 && dev < 64 && !allowed[dev]) {
    (void)hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                              bytes);
    allowed[dev] = true;
  }
}

}  // namespace nvm
