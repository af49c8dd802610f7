// Products of some hundred MX rows (mx_pipe.h) as kernels of their own.
#include "mx_pipe.h"

namespace nvm {

namespace {

template <int FMT, int OFMT, class T>
__global__ __launch_bounds__(64 * T::NW, 2) void mx_gemm_pipe_kernel(const MxMatmulArgs p,
                                                                     int n_tiles, int m_tiles) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  // tiles in contiguous runs per XCD (blocks go to the XCDs in turn), dealt to
  // the XCD's blocks
  const int total = n_tiles * m_tiles, per_xcd = (total + 7) >> 3, stride = (int)gridDim.x >> 3;
  const int last = min(((int)blockIdx.x & 7) * per_xcd + per_xcd, total);
  const int first = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
  if (first >= last) return;
  mx_pipe_tiles<FMT, OFMT, T>(p, smem, first, last, stride, [&](int tile) {
    return T::place(p, tile, n_tiles, m_tiles);
  });
}

template <int FMT, int OFMT, class T>
hipError_t go(const MxMatmulArgs &a, hipStream_t st) {
  static bool allowed[64] = {false};
  int n_tiles, m_tiles;
  if (!mx_count_tiles<T>(a, n_tiles, m_tiles)) return hipErrorInvalidConfiguration;
  auto kern = mx_gemm_pipe_kernel<FMT, OFMT, T>;
  mx_allow_lds(kern, T::kLds, allowed);
  // (KG = 2: a tile a block; else blocks that walk tiles, one to a CU)
  const int all = 8 * ((n_tiles * m_tiles + 7) / 8);
  const int grid = T::KG == 2 ? all : std::min(all, cu_count() / 8 * 8);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * T::NW), T::kLds, st, a, n_tiles,
                     m_tiles);
  return hipGetLastError();
}

// (mx_product.hip chooses; 64 x 64 has no room for two matrices' scale pieces)
template <int FMT, int OFMT, bool DUAL>
hipError_t launch_tile(int bn, int bm, const MxMatmulArgs &a, hipStream_t st) {
  if (bn == 256) return go<FMT, OFMT, MxWideTile<FMT, DUAL>>(a, st);
  if (bm == 128) return go<FMT, OFMT, MxSmallTile<FMT, DUAL>>(a, st);
  if constexpr (!DUAL)
    if (bn == 64) return go<FMT, OFMT, MxTile<FMT, DUAL, 64, 64, 2, 2, 2, 3, 2>>(a, st);
  return go<FMT, OFMT, MxTile<FMT, DUAL, 128, 64, 2, 2, 2, 3, 2>>(a, st);
}

template <int FMT>
hipError_t launch_fmt(int bn, int bm, bool dual, int out_format, const MxMatmulArgs &a,
                      hipStream_t st) {
  if (!dual) return launch_tile<FMT, NVM_MX_FP8, false>(bn, bm, a, st);
  return out_format == NVM_MX_FP4 ? launch_tile<FMT, NVM_MX_FP4, true>(bn, bm, a, st)
                                  : launch_tile<FMT, NVM_MX_FP8, true>(bn, bm, a, st);
}

}  // namespace

hipError_t launch_mx_gemm_pipe(int format, int bn, int bm, bool dual, int out_format,
                               const MxMatmulArgs &a, hipStream_t st) {
  return format == NVM_MX_FP4   ? launch_fmt<NVM_MX_FP4>(bn, bm, dual, out_format, a, st)
         : format == NVM_MX_FP8 ? launch_fmt<NVM_MX_FP8>(bn, bm, dual, out_format, a, st)
                                : launch_fmt<kMxShort>(bn, bm, dual, out_format, a, st);
}

}  // namespace nvm
