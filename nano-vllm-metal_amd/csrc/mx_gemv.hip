// Products of few MX rows with MXFP4 weights (include/nvm_mx.h): decode
// batches of the projections and of the dense MLP's gate/up pair.
//
// Bound: latency, then the weight stream (a projection's 5 to 7 MB are 1 to
// 1.4 us of HBM time).  The scaled matrix instruction takes the codes as they
// lie in memory, so a wavefront is loads, matrix instructions and one sum:
//  * a block owns RT 16-row tiles of the weights and MT 16-row tiles of the
//    activations; its four wavefronts take runs of four 128-value steps in
//    turn, and each requests a whole run (scales, weights, activations) before
//    it uses any of it.  Requests are what costs here, 16 lines each: a
//    wavefront makes none past its last run (such loads of nothing, and the
//    compiler's own order instead of row by row, cost 2048 -> 151936 of one row
//    12 of 44 us), and only the last run is compared with the row's end.  Eight
//    wavefronts, or runs of two steps, or a run requested ahead, were slower
//    nearly everywhere (2048 -> 5120 of 8 rows 4.0, 4.1 and 4.1 us for 3.9);
//  * operands go from memory straight into the instruction's registers: a
//    lane's 16 bytes of a weight row are its 32 values of a step, a row's 16
//    scale bytes are the run's, and the activations are few enough to come
//    from L2;
//  * the wavefronts' sums meet in LDS once and are added in order.
// Weights are the row operand, so a lane ends up with four neighbouring
// outputs of one activation row, and a block of 32 outputs (SwiGLU's MX
// output) is two tiles of four lane groups.
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
    xo[t] = r < nm ? r * XB + 16 * G : kMaskedOffset;
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
          // (FP4: the lane's 32 values; FP8: 16 at 16 G, 16 at 64 + 16 G)
          q.x[j][t].v[c] =
              FMT == NVM_MX_FP4
                  ? bload16(xr, at(xo[t], 128 * j + 32 * G), 256 * r + 64 * j)
                  : bload16(xr, at(xo[t], 128 * j + 64 * c + 16 * G), 512 * r + 128 * j + 64 * c);
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
      uint32_t xs[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) xs[t] = in ? q.xs[t][j] >> (8 * G) : 127u;
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const uint32_t ws = in ? q.ws[i][j] >> (8 * G) : 127u;
#pragma unroll
        for (int t = 0; t < MT; ++t)
          acc[i][t] = mx_mfma<FMT>(q.w[j][i], ws, q.x[j][t], xs[t], acc[i][t]);
      }
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

template <int FMT, int OFMT, bool DUAL, int RT, int MT>
hipError_t go(const MxMatmulArgs &a, hipStream_t st) {
  constexpr int RF = DUAL ? RT / 2 : RT;
  const int64_t x = ((int64_t)a.K + 16 * RF - 1) / (16 * RF), y = (a.M + 16 * MT - 1) / (16 * MT);
  // (threads of a launch's dimension: below 2^32)
  if (x * (64 * NW) > (int64_t)UINT32_MAX || y > 65535) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((mx_gemv_kernel<FMT, OFMT, DUAL, RT, MT>),
                     dim3((unsigned)x, (unsigned)y), dim3(64 * NW), 0, st, a);
  return hipGetLastError();
}

// The largest tile of a block that leaves kBlocks of them, without a half-used
// activation tile.  Larger blocks read the activations, and a column of them
// the weights, less often; too few leave CUs idle (2048 -> 5120 of 16 rows: 160
// blocks of 2 x 1 tiles 4.6 us, 320 of 1 x 1 5.2, 80 of 4 x 1 5.6; of 64 rows 214
// of 3 x 2 7.6, 320 of 4 x 1 9.2; 4096 -> 2048 of 32 rows: 256 of 1 x 1 5.4, 128
// of 2 x 1 6.7).
constexpr int64_t kBlocks = 160;

template <int FMT>
hipError_t launch_fmt(bool dual, int out_format, const MxMatmulArgs &a, hipStream_t st) {
  const int64_t mt = (a.M + 15) / 16;
  auto fits = [&](int rt, int m) {
    return mt % m == 0 && ((int64_t)a.K + 16 * rt - 1) / (16 * rt) * (mt / m) >= kBlocks;
  };
  if (!dual) {
    if (fits(3, 2)) return go<FMT, NVM_MX_FP8, false, 3, 2>(a, st);
    if (fits(4, 1)) return go<FMT, NVM_MX_FP8, false, 4, 1>(a, st);
    if (fits(2, 2)) return go<FMT, NVM_MX_FP8, false, 2, 2>(a, st);
    if (fits(2, 1)) return go<FMT, NVM_MX_FP8, false, 2, 1>(a, st);
    return go<FMT, NVM_MX_FP8, false, 1, 1>(a, st);
  }
  // SwiGLU: 32 outputs a block (its scale needs them), over all activation
  // rows of up to four tiles (2048 -> 6144 of 8 rows 6.2 us; of 17 rows 7.4 on 2
  // tiles, 10.2 on 1; of 64 rows 11.9 on 4, 13.4 on 2)
  auto swiglu = [&](auto OF) {
    constexpr int OFMT = decltype(OF)::value;
    if (mt == 1) return go<FMT, OFMT, true, 4, 1>(a, st);
    if (mt == 2) return go<FMT, OFMT, true, 4, 2>(a, st);
    return go<FMT, OFMT, true, 4, 4>(a, st);
  };
  return out_format == NVM_MX_FP4 ? swiglu(MxInt<NVM_MX_FP4>{}) : swiglu(MxInt<NVM_MX_FP8>{});
}

}  // namespace

hipError_t launch_mx_gemv(int format, bool dual, int out_format, const MxMatmulArgs &a,
                          hipStream_t st) {
  return format == NVM_MX_FP4 ? launch_fmt<NVM_MX_FP4>(dual, out_format, a, st)
                              : launch_fmt<NVM_MX_FP8>(dual, out_format, a, st);
}

}  // namespace nvm
