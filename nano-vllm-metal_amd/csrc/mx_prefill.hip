// Several query rows a request over the 4-bit cache on the matrix cores: chunked
// prefill and prefill after a prefix (a launch of nvm_paged_attention_mx, declared
// in include/nvm_mx_cache.h; D of 64 or 128).
//
// A block owns (request, kv head, 128 columns, a split of the context), a column
// being one (query row, query head) of the heads that share the kv head, 32 of them
// a wavefront.  Per 64 positions the codes of keys and values are converted to bf16
// once for the block (exactly: E2M1 times a power of two) and put into LDS, two
// buffers, the next tile's codes being loaded meanwhile.
//   * S^T = K . Q^T on v_mfma_f32_32x32x16_bf16: lane (c, h) gets column c at
//     positions 8 j + 4 h + i; the query in as many bf16 parts as its type needs.
//   * Softmax in base 2, two lanes a column.  The maximum moves only where a score
//     exceeds it by more than 2^kSlack, so the sums are rarely rescaled.
//   * O^T += V^T . P^T: the scores lie as the operand P^T wants them; values come out
//     of LDS transposed (ds_read_b64_tr_b16).  P is two bf16 parts: a weight loses
//     2^-17 of itself, so a result at most 2^-16 of its column's largest value.  (One f16
//     part would lose 2^-11 of each weight, which shows beside a bf16 output's own 2^-8
//     where values cancel; it took 193 us where two take 247: 2048 rows over 6144
//     positions, 32/4 heads of 128.)
// Bound, at that size: the matrix cores are busy 52 % of the time and the vector
// instructions fill as much, with two wavefronts a SIMD to overlap them; LDS is active 54 %
// of it, half of that for bank conflicts of the keys' reads and of the stores.  With a
// float32 query of 128 dims, three parts, nine registers spill.
// Positions that are not there are row 0 with a finite scale, and masked.  So are the
// scales of value blocks of NaNs, since a zero weight would not hide them from rows
// that do not see their position; those that do are told at the end.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal.h"
#include "mx_attention.h"
#include "mx_common.h"
#include "nvm_mx_cache.h"

namespace nvm {

namespace {

constexpr int kCW = 4;             // wavefronts of a block (two blocks a CU)
constexpr int kCols = 32 * kCW;    // its columns
constexpr int kKeys = 64;          // positions of a tile
constexpr float kSlack = 6.f;

template <int QT, int DH>
__global__ __launch_bounds__(64 * kCW, 2) void mx_prefill_kernel(MxAttnArgs a, int blocks) {
  using A = Act<DT_BF16>;
  constexpr int QP = kParts<QT>;
  constexpr int NC = DH / 16;  // steps of a score MFMA
  constexpr int NT = DH / 32;  // tiles of the output
  // LDS pitch of a row: the four rows of a transposed read lie in banks of their own
  // (with 8 in place of 16 in pairs, and the keys' reads apart: 249 us for 247)
  constexpr int VP = DH + 16;
  constexpr int NB = DH / 32;  // scales of a row; dwords of codes of a quarter of it
  static_assert(4 * kKeys == 64 * kCW, "a quarter of a row a thread");
  __shared__ __attribute__((aligned(16))) uint16_t s_k[2][kKeys][VP], s_v[2][kKeys][VP];
  // of each wavefront's 16 positions: which are there; NaNs among their values?  of a
  // position: its value blocks of NaNs
  __shared__ __attribute__((aligned(8))) uint16_t s_ok[2][kCW];
  __shared__ int s_any[2][kCW];
  __shared__ uint8_t s_nan[2][kKeys];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c32 = lane & 31, h = lane >> 5;
  const int b = blockIdx.y, s = blockIdx.z;
  // (columns with the most positions first)
  const int blk = blocks - 1 - (int)blockIdx.x / a.Hkv, kvh = (int)blockIdx.x % a.Hkv;
  const int col = blk * kCols + 32 * wv + c32;
  const bool col_ok = col < a.L * a.R;
  const int qrow = col / a.R, head = kvh * a.R + col - qrow * a.R;
  const int len = max(a.lens[b], 0), ctx = context_of(a, len), off = len - a.L;
  const int32_t *bt = a.bt + (int64_t)b * a.max_pages;
  // positions that a column of the block may see, of these this split's tiles
  const int last_row = min((blk * kCols + kCols - 1) / a.R, a.L - 1);
  const int kend = a.causal ? min(ctx, last_row + off + 1) : ctx;
  const int tiles = (max(kend, 0) + kKeys - 1) / kKeys, per = (tiles + a.S - 1) / a.S;
  const int t0 = min(s * per, tiles), t1 = min(t0 + per, tiles);
  // of the wavefront's columns: up to which tile all see everything
  const int first_row = min((blk * kCols + 32 * wv) / a.R, a.L - 1);
  const int all_see = a.causal ? first_row + off + 1 : 0x7FFFFFFF;
  // the column's last position (any of the last row's for a column that is none)
  const int bound = a.causal ? min(qrow, a.L - 1) + off : 0x7FFFFFFF;

  u32x4 qop[NC][QP];
  {
    const int64_t at = b * a.q_sb + (col_ok ? head * a.q_sh + qrow * a.q_sl : 0);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      query8<QT>(a.q, at + 16 * k + 8 * h, qop[k]);
#pragma unroll
      for (int p = 0; p < QP; ++p) qop[k][p] = col_ok ? qop[k][p] ^ a.q_sign : u32x4{0u, 0u, 0u, 0u};
    }
  }

  // staging: this thread's position of a tile and quarter of its row
  const int key = tid >> 2, part = tid & 3;
  int pg;
  auto page_id = [&](int t) {
    const int pos = kKeys * t + key;
    pg = bt[max(min(page_of(pos, a.ps_mul, a.ps_shift), a.max_pages - 1), 0)];
  };
  uint32_t kd[NB], vd[NB], ksc, vsc;
  bool ok;
  auto stage_load = [&](int t) {
    const int pos = kKeys * t + key;
    const int slot = pos - page_of(pos, a.ps_mul, a.ps_shift) * a.page_size;
    ok = (pos < ctx) & ((uint32_t)pg < (uint32_t)a.P);
    const uint32_t row = (((uint32_t)pg * a.Hkv + kvh) * a.page_size + slot) & (ok ? ~0u : 0u);
    load_dwords<NB>(a.kc + (uint64_t)row * (DH / 2) + (DH / 8) * part, kd);
    load_dwords<NB>(a.vc + (uint64_t)row * (DH / 2) + (DH / 8) * part, vd);
    ksc = a.ks[(uint64_t)row * NB + (DH / 4) * part / 32];
    vsc = a.vs[(uint64_t)row * NB + (DH / 4) * part / 32];
  };
  auto stage_store = [&](int buf) {
    const bool nan = ok & (vsc == 255u);
    const float f = __uint_as_float(ok ? ksc << 23 : 0u);
    const float g = __uint_as_float(ok & !nan ? vsc << 23 : 0u);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      *(u32x4 *)&s_k[buf][key][(DH / 4) * part + 8 * j] = codes_bf16(kd[j], f);
      *(u32x4 *)&s_v[buf][key][(DH / 4) * part + 8 * j] = codes_bf16(vd[j], g);
    }
    // (lane i of the first sixteen: position i of the wavefront's)
    const uint64_t there = __builtin_amdgcn_ballot_w64(__shfl((int)ok, 4 * lane & 63) != 0);
    const uint64_t nans = __builtin_amdgcn_ballot_w64(nan);
    if (lane == 0) {
      s_ok[buf][wv] = (uint16_t)there;
      s_any[buf][wv] = nans != 0;
    }
    if (part == 0) {
      const uint32_t m = (uint32_t)(nans >> lane) & 15u;  // by quarters
      s_nan[buf][key] = (uint8_t)(NB == 4 ? m : (m & 1) | (m >> 1 & 2));
    }
  };

  float m_run = -INFINITY, l_run = 0.f;  // column c32's; l_run this lane's share
  uint32_t seen_nan = 0;                 // value blocks of NaNs that the column sees
  f32x16 oacc[NT];                       // O^T: column c32, dims 32 t + 8 j + 4 h + i
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) oacc[t][i] = 0.f;
  // (-1, 0) and (0, -1), which pick out of a pair (in registers: as a constant the
  // second is taken for the inline constant -1.0, in the other half)
  uint32_t pick0 = 0x0000BF80u, pick1 = 0xBF800000u;
  asm volatile("" : "+v"(pick0), "+v"(pick1));
  page_id(t0);
  stage_load(t0);
  page_id(t0 + 1);
  stage_store(0);
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    stage_load(t + 1);  // (past the last one: row 0, or another split's)
    page_id(t + 2);

    f32x16 acc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[u][i] = 0.f;
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const u32x4 kb = *(const u32x4 *)&s_k[buf][32 * u + c32][16 * k + 8 * h];
#pragma unroll
        for (int p = 0; p < QP; ++p) acc[u] = A::mfma32(kb, qop[k][p], acc[u]);
      }
    }
    const uint64_t there = *(const uint64_t *)s_ok[buf];
    if (there != ~0ull || kKeys * (t + 1) > all_see) {  // uniform
      // bits of what this column sees; those of this lane's element i of part u are
      // 8 (i / 4) + i % 4 of the word
      const int n = bound - kKeys * t;  // (the last of them; one more might not fit an int)
      const uint64_t seen = n >= 63 ? there : n < 0 ? 0 : there & ((2ull << n) - 1);
      const uint32_t w[2] = {(uint32_t)seen >> (4 * h), (uint32_t)(seen >> 32) >> (4 * h)};
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)w[u], 8 * (i >> 2) + (i & 3), 1);
          acc[u][i] = __uint_as_float((__float_as_uint(acc[u][i]) & m) | (~m & 0xFF800000u));
        }
    }
    if (s_any[buf][0] | s_any[buf][1] | s_any[buf][2] | s_any[buf][3]) {  // uniform
#pragma unroll 1
      for (int kl = 0; kl < kKeys; ++kl)
        if (kKeys * t + kl <= bound) seen_nan |= s_nan[buf][kl];
    }
    float tmax = acc[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, acc[u][i]);
    tmax *= a.scale2;
    if (__any(tmax > m_run + kSlack)) {
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(tmax), __float_as_uint(tmax),
                                                      false, false);
      const float m_new =
          fmaxf(m_run, fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
      const float alpha = exp2_below(m_run, m_new);
      l_run *= alpha;
#pragma unroll
      for (int k = 0; k < NT; ++k) oacc[k] *= alpha;
      m_run = m_new;
    }
    const float m_sub = m_run == -INFINITY ? 0.f : m_run;
    // P^T: slot 8 h + j of 16 positions' product is position 4 h + j, or 8 + 4 h + j
    // - 4 from j = 4 on
    u32x4 hi[4], lo[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 8 * (c & 1) + 2 * j;
        const float x = __builtin_amdgcn_exp2f(fmaf(acc[c >> 1][i], a.scale2, -m_sub));
        const float y = __builtin_amdgcn_exp2f(fmaf(acc[c >> 1][i + 1], a.scale2, -m_sub));
        l_run += x + y;
        hi[c][j] = A::pack2(x, y);
        lo[c][j] = A::pack2(A::dot2(hi[c][j], pick0, x), A::dot2(hi[c][j], pick1, y));
      }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint16_t *v0 = &s_v[buf][16 * c + 4 * h + ((lane & 15) >> 2)]
                               [16 * ((lane >> 4) & 1) + 4 * (lane & 3)];
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const u32x2 x = lds_read_tr(v0 + 32 * k), y = lds_read_tr(v0 + 8 * VP + 32 * k);
        const u32x4 va = {x.x, x.y, y.x, y.y};
        oacc[k] = A::mfma32(va, hi[c], oacc[k]);
        oacc[k] = A::mfma32(va, lo[c], oacc[k]);
      }
    }
    stage_store(buf ^ 1);
    __syncthreads();
  }

  l_run += __shfl_xor(l_run, 32);
  if (!col_ok) return;
  const int64_t n = ((int64_t)b * a.L + qrow) * a.Hq + head;
  const bool whole = a.S == 1;
  const float inv = whole ? (l_run == 0.f ? 0.f : 1.f / l_run) : 1.f;
  auto store = [&](void *out, int64_t row, auto dt) {
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o[i] = seen_nan >> k & 1 ? __builtin_nanf("")
                 : l_run == 0.f    ? 0.f
                                   : oacc[k][4 * j + i] * inv;
        store_out4<decltype(dt)::value>(out, row * DH + 32 * k + 8 * j + 4 * h, o);
      }
  };
  if (whole)
    mx_by_dtype(a.out_dt, [&](auto dt) { store(a.out, n, dt); });
  else
    store(a.part_o, n * a.S + s, MxInt<NVM_KV_F32>{});
  if (!whole && h == 0) {
    a.part_ml[(n * a.S + s) * 2] = m_run;
    a.part_ml[(n * a.S + s) * 2 + 1] = l_run;
  }
}

template <int QT>
hipError_t launch(const MxAttnArgs &a, hipStream_t st) {
  const int blocks = (int)mx_prefill_blocks(a.L, a.R);
  const dim3 grid(blocks * a.Hkv, a.B, a.S);
  if (a.D == 128)
    hipLaunchKernelGGL((mx_prefill_kernel<QT, 128>), grid, dim3(64 * kCW), 0, st, a, blocks);
  else
    hipLaunchKernelGGL((mx_prefill_kernel<QT, 64>), grid, dim3(64 * kCW), 0, st, a, blocks);
  return hipGetLastError();
}

}  // namespace

int64_t mx_prefill_blocks(int64_t L, int64_t R) { return (L * R + kCols - 1) / kCols; }

hipError_t launch_mx_prefill(int q_dtype, const MxAttnArgs &a, hipStream_t st) {
  return q_dtype == NVM_KV_F32    ? launch<NVM_KV_F32>(a, st)
         : q_dtype == NVM_KV_BF16 ? launch<NVM_KV_BF16>(a, st)
                                  : launch<NVM_KV_F16>(a, st);
}

}  // namespace nvm
