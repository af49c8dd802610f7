// Products of few MX rows with MXFP4 weights (include/nvm_mx.h): decode
// batches of the projections and of the dense MLP's gate/up pair.
//
// Bound: latency, then the weight stream (a projection's 5 to 7 MB are 1 to
// 1.4 us of HBM time).  Codes go from memory into registers and from there, E2M1
// as it is, E4M3 by way of bf16 (mx_common.h), into matrix instructions, so a
// wavefront is loads, products and one sum (E4M3, 2048 -> 5120: one row 4.1 us, 8
// rows 4.4; in short sums 3.6 and 3.9):
//  * a block owns RT 16-row tiles of the weights and MT 16-row tiles of the
//    activations; its four wavefronts take runs of four 128-value steps in
//    turn, and each requests a whole run (scales, weights, activations) before
//    it uses any of it.  Requests are what costs here, 16 lines each: a
//    wavefront makes none past its last run (such loads of nothing, and the
//    compiler's own order instead of row by row, cost 2048 -> 151936 of one row
//    12 of 44 us), and only the last run is compared with the row's end.  Eight
//    wavefronts, or runs of two steps, or a run requested ahead, were slower
//    nearly everywhere (short sums, 2048 -> 5120 of 8 rows: 4.0, 4.1 and 4.1 us for
//    3.9);
//  * operands go from memory straight into registers: a lane's 16 bytes of a
//    weight row are its 32 values of a step, a row's 16 scale bytes are the run's,
//    and the activations are few enough to come from L2;
//  * the wavefronts' sums meet in LDS once and are added in order.
// Weights are the row operand, so a lane ends up with four neighbouring
// outputs of one activation row, and a block of 32 outputs (SwiGLU's MX
// output) is two tiles of four lane groups.
#include <math.h>

#include <type_traits>

#include "internal.h"
#include "mx_common.h"

namespace nvm {

namespace {

constexpr int NW = 4;  // wavefronts of a block

// RT: weight tiles of a block (DUAL: RT / 2 of the gate and the same rows of
// the up projection).
template <int FMT, int OFMT, bool DUAL, int RT, int MT>
__global__ __launch_bounds__(64 * NW) void mx_gemv_kernel(const MxMatmulArgs p) {
  constexpr int NX = FMT == NVM_MX_FP4 ? 1 : 2;  // 16-byte loads of a lane's 32 activations
  constexpr int RF = DUAL ? RT / 2 : RT;         // tiles of output columns
  __shared__ f32x4 s_red[NW][RT * MT][64];
  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, G = lane >> 4;
  const int k0 = blockIdx.x * (RF * 16);
  const int64_t m0 = (int64_t)blockIdx.y * (MT * 16);
  const int nk = min(RF * 16, p.K - k0);
  const int nm = (int)min((int64_t)(MT * 16), p.M - m0);
  const int WB = p.N / 2, XB = p.N * Mx<FMT>::kBits / 8;  // bytes of a row
  const int nb = p.N / 32;

  rsrc_t wr[DUAL ? 2 : 1], wsr[DUAL ? 2 : 1];
#pragma unroll
  for (int d = 0; d < (DUAL ? 2 : 1); ++d) {
    wr[d] = make_rsrc(p.w[d] + (int64_t)k0 * WB, (uint32_t)(nk * WB));
    wsr[d] = make_rsrc(p.ws[d] + (int64_t)k0 * p.ws_ld[d], (uint32_t)(nk * (int)p.ws_ld[d]));
  }
  const rsrc_t xr = make_rsrc(p.a + m0 * XB, (uint32_t)(nm * XB));
  const rsrc_t xsr = make_rsrc(p.as + m0 * p.as_ld, (uint32_t)(nm * (int)p.as_ld));
  // byte offsets of the lane's rows (rows past the operand read as zeros)
  int wo[RT], wso[RT], xo[MT], xso[MT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = 16 * (DUAL ? t % RF : t) + col;
    wo[t] = r < nk ? r * WB + 16 * G : kMaskedOffset;
    wso[t] = r < nk ? r * (int)p.ws_ld[DUAL && t >= RF] : kMaskedOffset;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int r = 16 * t + col;
    xo[t] = r < nm ? r * XB + (FMT == NVM_MX_FP4 ? 16 * G : mx_act_at<FMT>(G, 0)) : kMaskedOffset;
    xso[t] = r < nm ? r * (int)p.as_ld : kMaskedOffset;
  }

  struct Run {
    MxFrag<NVM_MX_FP4> w[4][RT];
    MxFrag<FMT> x[4][MT];
    u32x4 ws[RT], xs[MT];  // dword j: step j, byte G of it the lane's block
  };
  // All of a run is requested before any of it is used, and a row's steps next
  // to each other: two share a 128-byte line.  (TAIL: values past the row read
  // as zeros.)
  auto load = [&](Run &q, int r, auto TAIL) {
    auto at = [&](int o, int value) {
      return decltype(TAIL)::value && 512 * r + value >= p.N ? kMaskedOffset : o;
    };
#pragma unroll
    for (int t = 0; t < RT; ++t) q.ws[t] = bload16(wsr[DUAL && t >= RF], wso[t], 16 * r);
#pragma unroll
    for (int t = 0; t < MT; ++t) q.xs[t] = bload16(xsr, xso[t], 16 * r);
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        q.w[j][t].v[0] =
            bload16(wr[DUAL && t >= RF], at(wo[t], 128 * j + 32 * G), 256 * r + 64 * j);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < NX; ++c)
          q.x[j][t].v[c] =
              bload16(xr, at(xo[t], 128 * j + mx_act_at<FMT>(G, c)),
                      FMT == NVM_MX_FP4 ? 256 * r + 64 * j
                                        : 512 * r + 128 * j + mx_act_at<FMT>(0, c));
    __builtin_amdgcn_sched_barrier(0);
  };
  f32x4 acc[RT][MT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto do_run = [&](int r, auto TAIL) {
    Run q;
    load(q, r, TAIL);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (behind a row: the scale of one, whatever lies there)
      const bool in = !decltype(TAIL)::value || 16 * r + 4 * j + G < nb;
      uint32_t xs[MT], ws[RT];
#pragma unroll
      for (int t = 0; t < MT; ++t) xs[t] = in ? q.xs[t][j] >> (8 * G) : 127u;
#pragma unroll
      for (int i = 0; i < RT; ++i) ws[i] = in ? q.ws[i][j] >> (8 * G) : 127u;
      mx_products<FMT, 0>(q.w[j], ws, q.x[j], xs, acc, [](int) {});
    }
  };
  const int full = p.N / 512;
  int r = wv;
  for (; r < full; r += NW) do_run(r, std::false_type{});
  if (r == full && 512 * full < p.N) do_run(r, std::true_type{});

#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) s_red[wv][r * MT + t][lane] = acc[r][t];
  __syncthreads();
  auto sum = [&](int tile) {
    f32x4 v = s_red[0][tile][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += s_red[w][tile][lane];
    return v;
  };
  if constexpr (!DUAL) {
    for (int i = wv; i < RT * MT; i += NW) {
      const int r = i / MT, m = 16 * (i % MT) + col;
      const f32x4 v = sum(i);
      if (m < nm)
        mx_by_dtype(p.out_dtype, [&](auto DTYPE) {
          mx_store4<decltype(DTYPE)::value>(p.out, (m0 + m) * p.K + k0, 16 * r + 4 * G, nk, v);
        });
    }
  } else {
    // a block of 32 outputs of a row: two tiles, four lane groups
    for (int i = wv; i < RF / 2 * MT; i += NW) {
      const int r = i / MT, t = i % MT, m = 16 * t + col;
      float h[8];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x4 g = sum((2 * r + j) * MT + t), u = sum((RF + 2 * r + j) * MT + t);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[4 * j + e] = mx_swiglu(g[e], u[e]);
      }
      mx_store_block<OFMT>(h, G, m < nm && 32 * r < nk, m0 + m, k0 + 32 * r, p);
    }
  }
}

// Blocks of a launch (DUAL: RT / 2 tiles of either matrix); false: more than it
// takes, 2^32 - 1 threads and 65535 rows of blocks.
bool grid_of(bool dual, int rt, int mt, int64_t M, int64_t K, int64_t &x, int64_t &y) {
  const int64_t columns = 16 * (dual ? rt / 2 : rt), rows = 16 * mt;
  x = (K + columns - 1) / columns;
  y = (M + rows - 1) / rows;
  return x * (64 * NW) <= (int64_t)UINT32_MAX && y <= 65535;
}

template <int FMT, int OFMT, bool DUAL, int RT, int MT>
hipError_t go(const MxMatmulArgs &a, hipStream_t st) {
  int64_t x, y;
  if (!grid_of(DUAL, RT, MT, a.M, a.K, x, y)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((mx_gemv_kernel<FMT, OFMT, DUAL, RT, MT>),
                     dim3((unsigned)x, (unsigned)y), dim3(64 * NW), 0, st, a);
  return hipGetLastError();
}

// Tiles of a block, and the time of a launch of such blocks: `fixed` + `round` x
// rounds over the CUs x N / 2048 microseconds, for E2M1 activations, E4M3, and E4M3
// in short sums (least squares over some hundred products of 16 to 512 rows each;
// the residual is 3 to 9 %, for 1 x 1 tiles of E4M3 14).  A round after the first
// takes kLeastRound, however short the rows (in short sums 32 -> 2048 of 2048 rows,
// 11 rounds of 3 x 2 tiles: 17.3 us).  Larger blocks read the activations, and a
// column of them the weights, less often, but a round of them is longer: 4096 ->
// 4096 of 128 rows 14.3 us on 256 blocks of 4 x 2 tiles, 16.5 on 512 of 2 x 2, 20.1
// on 1024 of 2 x 1; 2048 -> 2048 of 32 rows 4.2 on 256 of 1 x 1, 4.7 on 128 of 2 x
// 1, 6.5 on 64 of 2 x 2.
constexpr double kLeastRound = 1.8;
struct Blocks {
  int rt, mt;
  double fixed[3], round[3];  // by the activations: an nvm_mx_format or kMxShort
};
constexpr Blocks kLinear[] = {
    {1, 1, {2, 1.9, 2.2}, {1.15, 1.8, 1.5}}, {2, 1, {2.1, 2.6, 2.3}, {1.8, 2.2, 2.05}},
    {4, 1, {2.3, 3.5, 2.6}, {3, 3.2, 3.25}}, {2, 2, {2.4, 3.4, 2.6}, {2.4, 3.1, 3.3}},
    {2, 3, {2.7, 3.9, 2.7}, {2.9, 3.6, 4.5}}, {4, 2, {3, 4.6, 3.3}, {3.6, 4.3, 4.5}},
    {4, 3, {3.5, 0, 3.6}, {4.1, 0, 6}}};
// (4 x 3 of E4M3, 5.3 and 5, takes longer than 64 x 64 tiles whatever the sizes.)
constexpr int linear_blocks(int format) {
  return sizeof(kLinear) / sizeof(Blocks) - (format == NVM_MX_FP8);
}
// (SwiGLU: 32 outputs a block, which its scale needs: two tiles of each matrix.
// 2048 -> 6144 of 32 rows 9.3 us on 192 blocks of 2 tiles of rows, 10.4 on 384 of
// 1; 2048 -> 768 of 64 rows 6.5 on 96 of 1, 11.6 on 24 of 4)
constexpr Blocks kSwiglu[] = {{4, 1, {2.6, 2.9, 2.5}, {2.9, 3.6, 3.3}},
                              {4, 2, {2.8, 3.6, 3}, {3.5, 4.9, 4.3}},
                              {4, 3, {3.2, 2.7, 2.9}, {3.8, 7, 5.6}},
                              {4, 4, {3.2, 3, 3.4}, {4.7, 7.8, 6.8}}};

template <int FMT, int OFMT, bool DUAL, int I>
hipError_t launch_tile(int tile, const MxMatmulArgs &a, hipStream_t st) {
  constexpr const Blocks &b = DUAL ? kSwiglu[I] : kLinear[I];
  if constexpr (I > 0)
    if (tile != I) return launch_tile<FMT, OFMT, DUAL, I - 1>(tile, a, st);
  return go<FMT, OFMT, DUAL, b.rt, b.mt>(a, st);
}

template <int FMT>
hipError_t launch_fmt(int tile, bool dual, int out_format, const MxMatmulArgs &a,
                      hipStream_t st) {
  constexpr int nl = linear_blocks(FMT), ns = sizeof(kSwiglu) / sizeof(Blocks);
  if (!dual) return launch_tile<FMT, NVM_MX_FP8, false, nl - 1>(tile, a, st);
  return out_format == NVM_MX_FP4 ? launch_tile<FMT, NVM_MX_FP4, true, ns - 1>(tile, a, st)
                                  : launch_tile<FMT, NVM_MX_FP8, true, ns - 1>(tile, a, st);
}

double best_of(const Blocks *blocks, int count, int format, bool dual, int64_t M, int N, int K,
               MxBlock *block) {
  const int64_t cus = cu_count();
  double best = INFINITY;
  for (int i = 0; i < count; ++i) {
    const Blocks &b = blocks[i];
    int64_t x, y;
    if (!grid_of(dual, b.rt, b.mt, M, K, x, y)) continue;
    const double round = b.round[format] * (N / 2048.0);
    const double t = b.fixed[format] + round + ((x * y - 1) / cus) * fmax(round, kLeastRound);
    if (t < best) {
      best = t;
      *block = {i, 16 * b.rt, 16 * b.mt};
    }
  }
  return best;
}

}  // namespace

double mx_gemv_time(int format, bool dual, int64_t M, int N, int K, MxBlock *block) {
  constexpr int ns = sizeof(kSwiglu) / sizeof(Blocks);
  return dual ? best_of(kSwiglu, ns, format, dual, M, N, K, block)
              : best_of(kLinear, linear_blocks(format), format, dual, M, N, K, block);
}

hipError_t launch_mx_gemv(int format, int tile, bool dual, int out_format, const MxMatmulArgs &a,
                          hipStream_t st) {
  return format == NVM_MX_FP4   ? launch_fmt<NVM_MX_FP4>(tile, dual, out_format, a, st)
         : format == NVM_MX_FP8 ? launch_fmt<NVM_MX_FP8>(tile, dual, out_format, a, st)
                                : launch_fmt<kMxShort>(tile, dual, out_format, a, st);
}

}  // namespace nvm
