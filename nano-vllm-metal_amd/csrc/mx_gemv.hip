// Products of few MX rows with MXFP4 weights (include/nvm_mx.h): decode
// batches of the projections and of the dense MLP's gate/up pair.
//
// Bound: latency, then the weight stream (a projection's 5 to 7 MB are 1 to
// 1.4 us of HBM time).  The scaled matrix instruction takes the codes as they
// lie in memory, so a wavefront is loads, matrix instructions and one sum:
//  * a block owns RT 16-row tiles of the weights and MT 16-row tiles of the
//    activations; its NW wavefronts split the reduction in runs of whole
//    128-value steps, and each requests up to RING steps (weights, their
//    scales, activations) before it uses the first;
//  * operands go from memory straight into the instruction's registers: a
//    lane's 16 bytes of a weight row are its 32 values of a step, and the
//    activations are few enough to come from L2;
//  * the wavefronts' sums meet in LDS once and are added in order.
// Weights are the row operand, so a lane ends up with four neighbouring
// outputs of one activation row, and a block of 32 outputs (SwiGLU's MX
// output) is two tiles of four lane groups.
#include <algorithm>

#include "internal.h"
#include "mx_common.h"

namespace nvm {

namespace {

// RT: weight tiles of a block (DUAL: RT / 2 of the gate and the same rows of
// the up projection).
template <int FMT, int OFMT, bool DUAL, int RT, int MT, int NW, int RING>
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
  const int steps = (p.N + 127) / 128, per = (steps + NW - 1) / NW;
  const int s0 = wv * per, s1 = min(steps, s0 + per);

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

  struct Step {
    MxFrag<NVM_MX_FP4> w[RT];
    MxFrag<FMT> x[MT];
    uint32_t ws[RT], xs[MT];
  };
  // (steps past the wavefront's run, and values past the row: zeros with the
  // scale of one, whatever lies behind the row)
  auto load = [&](Step &q, int s) {
    const bool on = s < s1;
    const int so = on ? s : 0;
    const bool wk = on && 128 * so + 32 * G < p.N;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      q.w[t].v[0] = bload16(wr[DUAL && t >= RF], wk ? wo[t] : kMaskedOffset, 64 * so);
      q.ws[t] = bload4(wsr[DUAL && t >= RF], wk ? wso[t] : kMaskedOffset, 4 * so);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
      for (int c = 0; c < NX; ++c) {
        // (FP4: the lane's 32 values; FP8: 16 at 16 G, 16 at 64 + 16 G)
        const bool xk = FMT == NVM_MX_FP4 ? wk : on && 128 * so + 64 * c + 16 * G < p.N;
        q.x[t].v[c] = bload16(xr, xk ? xo[t] : kMaskedOffset,
                              FMT == NVM_MX_FP4 ? 64 * so : 128 * so + 64 * c);
      }
      q.xs[t] = bload4(xsr, wk ? xso[t] : kMaskedOffset, 4 * so);
    }
  };
  f32x4 acc[RT][MT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto use = [&](const Step &q, int s) {
    // the lane group's byte of the step's four
    const bool in = s < s1 && 4 * s + G < nb;
    auto pick = [&](uint32_t d) { return in ? d >> (8 * G) : 127u; };
    uint32_t ws[RT], xs[MT];
#pragma unroll
    for (int t = 0; t < RT; ++t) ws[t] = pick(q.ws[t]);
#pragma unroll
    for (int t = 0; t < MT; ++t) xs[t] = pick(q.xs[t]);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[r][t] = mx_mfma<FMT>(q.w[r], ws[r], q.x[t], xs[t], acc[r][t]);
  };
  Step ring[RING];
#pragma unroll
  for (int j = 0; j < RING; ++j) load(ring[j], s0 + j);
  for (int s = s0; s < s1; s += RING) {
#pragma unroll
    for (int j = 0; j < RING; ++j) {
      use(ring[j], s + j);
      load(ring[j], s + j + RING);
    }
  }

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
      const int r = i / MT, t = i % MT;
      const f32x4 v = sum(i);
      const int k = 16 * r + 4 * G, m = 16 * t + col;
      if (m >= nm) continue;
      mx_store4(p.out, p.out_dtype, (m0 + m) * p.K + k0 + k, v, nk - k, p.K % 4 == 0);
    }
  } else {
    // a block of 32 outputs of a row: two tiles, four lane groups
    for (int i = wv; i < RF / 2 * MT; i += NW) {
      const int r = i / MT, t = i % MT;
      float h[8];
      uint32_t mx = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x4 g = sum((2 * r + j) * MT + t), u = sum((RF + 2 * r + j) * MT + t);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h[4 * j + e] = mx_swiglu(g[e], u[e]);
          mx = max(mx, abs_bits(h[4 * j + e]));
        }
      }
      mx = max(mx, (uint32_t)__shfl_xor((int)mx, 16));
      mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
      const int m = 16 * t + col;
      if (m >= nm || 32 * r >= nk) continue;
      mx_store_block<OFMT>(h, mx, (m0 + m), k0 + 32 * r, G, p.K, p.out, p.out_s, p.out_sld);
    }
  }
}

template <int FMT, int OFMT, bool DUAL, int RT, int MT, int NW, int RING>
void go(const MxMatmulArgs &a, hipStream_t st) {
  constexpr int RF = DUAL ? RT / 2 : RT;
  const dim3 grid((unsigned)((a.K + 16 * RF - 1) / (16 * RF)),
                  (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((mx_gemv_kernel<FMT, OFMT, DUAL, RT, MT, NW, RING>), grid, dim3(64 * NW), 0,
                     st, a);
}

template <int FMT>
void launch_fmt(bool dual, int out_format, const MxMatmulArgs &a, hipStream_t st) {
  if (!dual)
    go<FMT, NVM_MX_FP8, false, 1, 1, 8, 2>(a, st);
  else if (out_format == NVM_MX_FP4)
    go<FMT, NVM_MX_FP4, true, 4, 1, 8, 2>(a, st);
  else
    go<FMT, NVM_MX_FP8, true, 4, 1, 8, 2>(a, st);
}

}  // namespace

hipError_t launch_mx_gemv(int format, bool dual, int out_format, const MxMatmulArgs &a,
                          hipStream_t st) {
  if (format == NVM_MX_FP4)
    launch_fmt<NVM_MX_FP4>(dual, out_format, a, st);
  else
    launch_fmt<NVM_MX_FP8>(dual, out_format, a, st);
  return hipGetLastError();
}

}  // namespace nvm
