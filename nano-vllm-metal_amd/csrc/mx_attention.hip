// Paged attention over the 4-bit cache (declared in include/nvm_mx_cache.h).
//
// mx_decode_kernel: one query row a request, D of 64 or 128.  A block owns a
//   request, a kv head, a group of up to 16 of its query heads and a split of the
//   context, which it shares out from the context's own length; its wavefronts
//   take tiles of 32 positions in turn.
//   * S^T = K . Q^T on v_mfma_f32_16x16x32_bf16.  E2M1 times a power of two is
//     exact in bf16, two values an instruction, so codes go from memory into the
//     operand: lane (c, G) loads position c's D/4 values from D/4 G on, its own
//     part of a block, and takes them as its dims of the MFMA's D/32 steps; the
//     query's operand is laid out in that order.  It is split into as many bf16
//     parts as its type needs (bf16 one, f16 two, float32 three), so products
//     are exact, each part's sum float32.
//   * Softmax in base 2; the running maximum is looked at across lanes only where
//     a score exceeds it.
//   * O^T += V^T . P^T: the scores' layout is that of the operand P^T.  Value rows
//     go to LDS as bf16 and come back transposed (ds_read_b64_tr_b16).  P is two
//     bf16 parts (2^-17 of each weight, below a 16-bit output's rounding by 2^6 or
//     more, and for a float32 one what a third product would take away): with up to
//     eight query heads the MFMA's other eight columns hold the second part, so both
//     cost one product.
//   * A masked position has a finite scale and any codes: its weight is zero, and
//     zero times a finite value is zero.
//   The next tile's keys are requested when this one's are converted, the next
//   values when these are in LDS.  Bound: for long contexts HBM (16 requests of 40000
//   positions, 32/4 heads of 128: 62 us, 5.5 TB/s of codes and scales); for short ones
//   the chain of trips to memory, code among them: one request of 700 positions 7.0 us
//   with the merge, of 100 4.0 without (in a table for 4096 positions, as a captured
//   step has, 6.9: the merge's launch goes by the table).  With f16 queries, 128 dims and
//   blocks of eight wavefronts six registers spill.
// mx_rows_kernel: any head dim, one wavefront per query row.  A position's row
//   of codes goes to a group of GL lanes (eight values, one dword, a lane), so
//   64 / GL positions are in flight side by side, each group with a running
//   maximum and sum of its own; the groups meet at the end.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal.h"
#include "mx_attention.h"
#include "mx_common.h"
#include "nvm_mx_cache.h"

namespace nvm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowThreads = 256;

template <int QT>
__device__ __forceinline__ float q_at(const void *q, int64_t i) {
  if constexpr (QT == NVM_KV_F32) return ((const float *)q)[i];
  if constexpr (QT == NVM_KV_BF16) return Act<DT_BF16>::to_f32(((const uint16_t *)q)[i]);
  return Act<DT_F16>::to_f32(((const uint16_t *)q)[i]);
}

__device__ __forceinline__ void values8(uint32_t d, float s, float (&v)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 0);
  const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 1);
  const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 2);
  const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 3);
  v[0] = p0.x * s, v[1] = p0.y * s, v[2] = p1.x * s, v[3] = p1.y * s;
  v[4] = p2.x * s, v[5] = p2.y * s, v[6] = p3.x * s, v[7] = p3.y * s;
}

template <int QT, int GL>
__global__ __launch_bounds__(kRowThreads) void mx_rows_kernel(MxAttnArgs a, int64_t rows) {
  constexpr int NG = 64 / GL;
  const int64_t row = (int64_t)blockIdx.x * (kRowThreads / 64) + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & (GL - 1), grp = (threadIdx.x & 63) / GL;
  const int h = (int)(row % a.Hq);
  const int64_t bl = row / a.Hq;
  const int i = (int)(bl % a.L), b = (int)(bl / a.L);
  const int kvh = h / a.R, n8 = a.D / 8;
  const bool on = lane < n8;
  const int64_t len = a.lens[b];
  const int64_t cap = min(len, (int64_t)a.max_pages * a.page_size);
  // (from 0 on: below -2^31, of a length next to it, an int would come out positive)
  const int last = (int)max((int64_t)0, a.causal ? min(cap, i + len - a.L + 1) : cap);
  const int32_t *bt = a.bt + (int64_t)b * a.max_pages;
  float qv[8], ov[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    qv[j] = on ? q_at<QT>(a.q, b * a.q_sb + h * a.q_sh + i * a.q_sl + 8 * lane + j) : 0.f;
  float m = -INFINITY, l = 0.f;
  for (int j = grp; j < last; j += NG) {
    const int pg = bt[j / a.page_size];
    if (pg < 0 || pg >= a.P) continue;  // (a whole group)
    const int64_t at = ((int64_t)pg * a.Hkv + kvh) * a.page_size + j % a.page_size;
    float k[8], v[8];
    values8(on ? ((const uint32_t *)a.kc)[at * n8 + lane] : 0u,
            on ? mx_scale(a.ks[at * (n8 / 4) + (lane >> 2)]) : 0.f, k);
    values8(on ? ((const uint32_t *)a.vc)[at * n8 + lane] : 0u,
            on ? mx_scale(a.vs[at * (n8 / 4) + (lane >> 2)]) : 0.f, v);
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) dot = fmaf(qv[e], k[e], dot);
#pragma unroll
    for (int x = 1; x < GL; x <<= 1) dot += __shfl_xor(dot, x);
    const float sc = (a.q_sign ? -dot : dot) * a.scale2, m_new = fmaxf(m, sc);
    const float alpha = exp2_below(m, m_new), p = exp2_below(sc, m_new);
    l = fmaf(l, alpha, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) ov[e] = fmaf(ov[e], alpha, p * v[e]);
    m = m_new;
  }
#pragma unroll
  for (int x = GL; x < 64; x <<= 1) {
    const float mo = __shfl_xor(m, x), lo = __shfl_xor(l, x), mm = fmaxf(m, mo);
    const float f = exp2_below(m, mm), g = exp2_below(mo, mm);
    l = l * f + lo * g;
#pragma unroll
    for (int e = 0; e < 8; ++e) ov[e] = ov[e] * f + __shfl_xor(ov[e], x) * g;
    m = mm;
  }
  if (grp == 0 && on) {
    // (a row that sees nothing: zeros; a NaN stays one)
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      store_out(a.out, a.out_dt, row * a.D + 8 * lane + e, l == 0.f ? 0.f : ov[e] * inv);
  }
}

template <int QT>
hipError_t launch_rows(const MxAttnArgs &a, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.L * a.Hq;
  const unsigned grid = (unsigned)((rows + kRowThreads / 64 - 1) / (kRowThreads / 64));
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(grid), dim3(kRowThreads), 0, st, a, rows);
  };
  if (a.D <= 32)
    go(mx_rows_kernel<QT, 4>);
  else if (a.D <= 64)
    go(mx_rows_kernel<QT, 8>);
  else if (a.D <= 128)
    go(mx_rows_kernel<QT, 16>);
  else
    go(mx_rows_kernel<QT, 32>);
  return hipGetLastError();
}

// The largest over a column's four lanes (lane groups 0..3).
__device__ __forceinline__ float column_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

constexpr int kTile = 32;  // positions of a wavefront's step: two of the MFMA's 16 rows

// Sum over the wavefront, in an order of its own: the same in every lane and block.
__device__ __forceinline__ float wave_sum(float v) {
  auto step = [&](uint32_t o) { v += __uint_as_float(o); };
  step(dpp_u32<0xB1>(__float_as_uint(v)));
  step(dpp_u32<0x4E>(__float_as_uint(v)));
  step(dpp_u32<0x141>(__float_as_uint(v)));
  step(dpp_u32<0x140>(__float_as_uint(v)));
  float r = 0.f;
#pragma unroll
  for (int i = 0; i < 64; i += 16)
    r += __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), i));
  return r;
}

// Splits of a context of `tiles` tiles: its share of the slots by length (the host
// does not know the lengths), and no more than sqrt(2 tiles), past which the merge
// takes longer than the steps it saves (one request of 1024, 4096 and 16384
// positions: 8, 16 and 32 splits of four wavefronts 7.2, 9.1 and 12.4 us; half and
// twice as many 7.8 and 7.2, 10 and 9.8, 14.0 and 13.9).
__device__ __forceinline__ int splits_of(const MxAttnArgs &a, int tiles, int lane, int tile) {
  float total = 0.f;
  for (int i = lane; i < a.B; i += 64)
    total += (float)((context_of(a, a.lens[i]) + tile - 1) / tile);
  total = wave_sum(total);
  const float share = (float)tiles * a.slots / fmaxf(total, 1.f);
  return max(1, min(a.S, (int)ceilf(fminf(share, sqrtf(2.f * (float)tiles)))));
}

// DUP: at most eight query heads; columns 8..15 hold them again, for the second
// part of P.  Grid: requests, kv heads x groups of query heads, splits (last, so
// that those that a context does not use come behind all others).
//
// A tile is 32 positions and not 64: its code runs cold in each launch (from L2
// into the instruction cache some 50 cycles a line), and a short context is little
// else.
template <int QT, int DH, bool DUP, int NW>
__global__ __launch_bounds__(64 * NW, 4) void mx_decode_kernel(MxAttnArgs a) {
  using A = Act<DT_BF16>;
  constexpr int NC = DH / 32;       // steps of a score MFMA; dwords of a lane's codes
  constexpr int NT = DH / 16;       // tiles of the output
  constexpr int NB = DH / 32;       // scales of a row
  constexpr int NU = kTile / 16;    // 16-row parts of a tile
  constexpr int VP = DH + 8;        // LDS pitch of a value row
  constexpr int RP = DUP ? 8 : 16;  // query heads of a block
  constexpr int QP = kParts<QT>;
  constexpr int kVBytes = NW * kTile * VP * 2, kOBytes = NW * RP * DH * 4;
  __shared__ __attribute__((aligned(16))) char s_buf[kVBytes > kOBytes ? kVBytes : kOBytes];
  auto s_v = reinterpret_cast<uint16_t(*)[kTile][VP]>(s_buf);
  auto s_o = reinterpret_cast<float(*)[RP][DH]>(s_buf);
  __shared__ float s_m[NW][RP], s_l[NW][RP];
  __shared__ u32x4 s_q[NC][QP][64];  // the score MFMAs' query operand, by lane

  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, G = lane >> 4;
  const int b = blockIdx.x, s = blockIdx.z;
  int kvh = blockIdx.y, hg = 0;
  if (a.HG > 1) {
    kvh = blockIdx.y / a.HG;
    hg = blockIdx.y - kvh * a.HG;
  }
  const int nh = min(RP, a.R - hg * RP);
  const int h0 = kvh * a.R + hg * RP;
  const int32_t *bt = a.bt + (int64_t)b * a.max_pages;

  // The block's wavefronts take tiles first, first + step, ... of the context,
  // whose length they need not know for the first: its page ids are requested
  // beside it.  pidx, slot: of position kTile t + 16 u + c16 of the tile whose
  // page ids are requested next.
  const int first = s * NW + wv;
  int pidx[NU], slot[NU], pg[NU];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int pos = kTile * first + 16 * u + c16;
    pidx[u] = page_of(pos, a.ps_mul, a.ps_shift);
    slot[u] = pos - pidx[u] * a.page_size;
  }
  // (No load stands behind a branch: at a branch's end the compiler waits for all
  // loads, the values of this tile among them, and a step took twice as long.  So
  // ids past the table are its last, and a tile past the context is row 0.)
  auto page_ids = [&]() {
#pragma unroll
    for (int u = 0; u < NU; ++u) pg[u] = bt[max(min(pidx[u], a.max_pages - 1), 0)];
  };
  page_ids();
  const int ctx = context_of(a, a.lens[b]);
  const int t_end = (ctx + kTile - 1) / kTile;

  for (int k = wv; k < NC; k += NW) {
    const int h = DUP ? c16 & 7 : c16;
    const bool ok = h < nh;
    const int64_t at = b * a.q_sb + (h0 + (ok ? h : 0)) * a.q_sh;
    u32x4 q[QP];
    query8<QT>(a.q, at + (DH / 4) * G + 8 * k, q);
#pragma unroll
    for (int p = 0; p < QP; ++p) s_q[k][p][lane] = ok ? q[p] ^ a.q_sign : u32x4{0u, 0u, 0u, 0u};
  }

  // rows in the pool of tile t's positions, whose page ids are there, and which
  // lanes' positions exist (row 0 for others)
  auto rows = [&](int t, uint32_t (&row)[NU], uint64_t (&there)[NU]) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const bool ok = (c16 < ctx - kTile * t - 16 * u) & ((uint32_t)pg[u] < (uint32_t)a.P);
      row[u] = (((uint32_t)pg[u] * a.Hkv + kvh) * a.page_size + slot[u]) & (ok ? ~0u : 0u);
      there[u] = __builtin_amdgcn_ballot_w64(ok);
    }
  };
  // on to the next tile's ids
  int dpage, dslot;
  auto advance = [&]() {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      slot[u] += dslot;
      const bool over = slot[u] >= a.page_size;
      pidx[u] += dpage + (over ? 1 : 0);
      slot[u] -= over ? a.page_size : 0;
    }
    page_ids();
  };
  auto load = [&](const uint8_t *codes, const uint8_t *scales, const uint32_t (&row)[NU],
                  uint32_t (&d)[NU][NC], uint32_t (&sc)[NU]) {
#pragma unroll
    for (int u = 0; u < NU; ++u)
      load_dwords<NC>(codes + (uint64_t)row[u] * (DH / 2) + (DH / 8) * G, d[u]);
#pragma unroll
    for (int u = 0; u < NU; ++u) sc[u] = scales[(uint64_t)row[u] * NB + (DH / 4) * G / 32];
  };
  // a lane's scale of a part: a finite one for a position that is not there
  auto scale_of = [&](uint32_t sc, uint64_t there) {
    return __uint_as_float(__builtin_amdgcn_inverse_ballot_w64(there) ? sc << 23 : 0u);
  };

  float m_run = -INFINITY;  // column c16's
  f32x4 oacc[NT], lacc = {0.f, 0.f, 0.f, 0.f};  // O^T: column c16, dims 16 t + 4 G + i; sums of P
#pragma unroll
  for (int t = 0; t < NT; ++t) oacc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // with DUP columns 8..15 hold P less its first part: (-1, 0) and (0, -1) pick
  // that part out of a pair
  // (in registers: as a constant the second is taken for the inline constant -1.0,
  // whose value the instruction puts into the other half)
  uint32_t pick0 = DUP && c16 < 8 ? 0u : 0x0000BF80u, pick1 = pick0 << 16;
  asm volatile("" : "+v"(pick0), "+v"(pick1));
  const u32x4 ones = {A::kOne2, A::kOne2, A::kOne2, A::kOne2};

  uint32_t row[NU], kd[NU][NC], ksc[NU], vd[NU][NC], vsc[NU];
  uint64_t there[NU];
  int t = first;
  const int S = __builtin_amdgcn_readfirstlane(a.S > 1 ? splits_of(a, t_end, lane, kTile) : 1);
  const int step = S * NW;
  if (s >= S) {
    if (threadIdx.x < nh) {
      const int64_t n = (int64_t)b * a.Hq + h0 + threadIdx.x;
      a.part_ml[(n * a.S + s) * 2] = -INFINITY;
      a.part_ml[(n * a.S + s) * 2 + 1] = 0.f;
    }
    return;
  }
  dpage = page_of(kTile * step, a.ps_mul, a.ps_shift);
  dslot = kTile * step - dpage * a.page_size;
  rows(t, row, there);
  advance();  // (before the keys, in the loop's order)
  load(a.kc, a.ks, row, kd, ksc);
  load(a.vc, a.vs, row, vd, vsc);
  __syncthreads();  // the query is there
  for (; t < t_end; t += step) {
    // S^T: column c16 at positions 16 u + 4 G + i
    f32x4 acc[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      const float f = scale_of(ksc[u], there[u]);
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const u32x4 kb = codes_bf16(kd[u][k], f);
#pragma unroll
        for (int p = 0; p < QP; ++p) acc[u] = A::mfma16(kb, s_q[k][p][lane], acc[u]);
      }
    }
    uint64_t now[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) now[u] = there[u];
    rows(t + step, row, there);
    advance();
    load(a.kc, a.ks, row, kd, ksc);
    __builtin_amdgcn_sched_barrier(0);  // (requested before this tile's values are waited for)

    // (before the softmax, so that the next values are requested before it too)
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const float f = scale_of(vsc[u], now[u]);
#pragma unroll
      for (int k = 0; k < NC; ++k)
        *(u32x4 *)&s_v[wv][16 * u + c16][(DH / 4) * G + 8 * k] = codes_bf16(vd[u][k], f);
    }
    wave_lds_sync();
    load(a.vc, a.vs, row, vd, vsc);

    if ((now[0] & now[1]) != ~0ull) {  // uniform
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(((uint32_t)now[u] >> (4 * G + i)) & 1u)) acc[u][i] = -INFINITY;
    }
    float tmax = acc[0][0];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) tmax = fmaxf(tmax, acc[u][i]);
    tmax *= a.scale2;
    if (__any(tmax > m_run)) {
      const float m_new = fmaxf(m_run, column_max(tmax));
      const float alpha = exp2_below(m_run, m_new);
      lacc *= alpha;
#pragma unroll
      for (int k = 0; k < NT; ++k) oacc[k] *= alpha;
      m_run = m_new;
    }
    const float m_sub = m_run == -INFINITY ? 0.f : m_run;
    // P^T, which lies as the product's operand wants it: slot 8 G + j is position
    // 4 G + j, or 16 + 4 G + j - 4 from j = 4 on
    u32x4 hi, lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = __builtin_amdgcn_exp2f(fmaf(acc[j >> 1][2 * (j & 1)], a.scale2, -m_sub));
      const float y = __builtin_amdgcn_exp2f(fmaf(acc[j >> 1][2 * (j & 1) + 1], a.scale2, -m_sub));
      hi[j] = A::pack2(x, y);
      lo[j] = A::pack2(A::dot2(hi[j], pick0, x), A::dot2(hi[j], pick1, y));
    }
    const u32x4 pb = DUP ? lo : hi;

    // O^T += V^T . P^T
    const uint16_t *v0 = &s_v[wv][4 * G + (c16 >> 2)][4 * (c16 & 3)];
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      const u32x2 x = lds_read_tr(v0 + 16 * k), y = lds_read_tr(v0 + 16 * VP + 16 * k);
      const u32x4 va = {x.x, x.y, y.x, y.y};
      oacc[k] = A::mfma16(va, pb, oacc[k]);
      if constexpr (!DUP) oacc[k] = A::mfma16(va, lo, oacc[k]);
    }
    lacc = A::mfma16(ones, pb, lacc);
    if constexpr (!DUP) lacc = A::mfma16(ones, lo, lacc);
    wave_lds_sync();
  }

  // the wavefronts' outputs meet (with DUP columns h and h + 8 are one: lanes 8
  // apart in a row of 16)
  auto both = [&](float v) {
    if constexpr (DUP) v += __uint_as_float(dpp_u32<0x128>(__float_as_uint(v)));
    return v;
  };
  const float l_run = both(lacc[0]);  // (all of its rows are alike)
  __syncthreads();                    // every wavefront is past its last use of s_v
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    f32x4 o = oacc[k];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = both(o[i]);
    if (c16 < RP) *(f32x4 *)&s_o[wv][c16][16 * k + 4 * G] = o;
  }
  if (G == 0 && c16 < RP) {
    s_m[wv][c16] = m_run;
    s_l[wv][c16] = l_run;
  }
  __syncthreads();

  for (int e = threadIdx.x; e < RP * DH / 4; e += 64 * NW) {
    const int r = e / (DH / 4), d = 4 * (e % (DH / 4));
    if (r >= nh) break;
    float M = s_m[0][r];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, s_m[w][r]);
    float Ls = 0.f;
    f32x4 Os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = exp2_below(s_m[w][r], M);
      Ls += f * s_l[w][r];
      Os += f * *(const f32x4 *)&s_o[w][r][d];
    }
    const int64_t n = (int64_t)b * a.Hq + h0 + r;
    if (a.S == 1) {
      const float inv = 1.f / Ls;
      const f32x4 o = Ls == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : Os * inv;
      mx_by_dtype(a.out_dt, [&](auto dt) { store_out4<decltype(dt)::value>(a.out, n * DH + d, o); });
    } else {
      *(f32x4 *)(a.part_o + (n * a.S + s) * DH + d) = Os;
      if (d == 0) {
        a.part_ml[(n * a.S + s) * 2] = M;
        a.part_ml[(n * a.S + s) * 2 + 1] = Ls;
      }
    }
  }
}

// Splits of a row: sum_s 2^(M_s - M) O_s / sum_s 2^(M_s - M) L_s, a wavefront a
// row: lane s takes split s's maximum and sum, then each lane D / 64 dims of those
// that saw a position (others were perhaps not written).  A weight of zero does not
// leave a split out: its outputs may be NaN, and zero times NaN is NaN, as it is
// where a context is not split.
constexpr int kMaxSplits = 64;
// ONE: of single query rows, few and late: the first splits' outputs are asked for
// beside the maxima, whether they count or not (one request of 32768 positions 15.0 us
// for 16.4; of 3 x 100 rows, whose splits are a few MB, 17.8 for 16.7).
template <int DH, bool ONE>
__global__ __launch_bounds__(kRowThreads) void mx_combine_kernel(const float *__restrict__ part_o,
                                                                 const float *__restrict__ part_ml,
                                                                 int64_t rows, int S, void *out,
                                                                 int out_dt) {
  constexpr int PD = DH / 64;
  const int64_t n = (int64_t)blockIdx.x * (kRowThreads / 64) + (threadIdx.x >> 6);
  if (n >= rows) return;
  const int lane = threadIdx.x & 63;
  const float *po = part_o + n * S * DH + PD * lane;
  constexpr int kAhead = 8;
  float v[kAhead][PD];
  auto load = [&](int s0, int end) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int d = 0; d < PD; ++d) v[j][d] = po[(int64_t)min(s0 + j, end - 1) * DH + d];
  };
  if constexpr (ONE) load(0, S);
  float ms = -INFINITY, ls = 0.f;
  if (lane < S) {
    ms = part_ml[(n * S + lane) * 2];
    ls = part_ml[(n * S + lane) * 2 + 1];
  }
  float M = ms;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor(M, x));
  const float w = exp2_below(ms, M);
  const float L = wave_sum(w * ls);
  const uint64_t on = __builtin_amdgcn_ballot_w64(ms != -INFINITY || ls != 0.f);
  const int last = on ? 64 - __builtin_clzll(on) : 0;
  float acc[PD] = {};
  for (int s0 = 0; s0 < last; s0 += kAhead) {
    if (!ONE || s0 > 0) load(s0, last);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), (s0 + j) & 63));
#pragma unroll
      for (int d = 0; d < PD; ++d)
        acc[d] += s0 + j < last && (on >> ((s0 + j) & 63) & 1) ? f * v[j][d] : 0.f;
    }
  }
#pragma unroll
  for (int d = 0; d < PD; ++d)
    store_out(out, out_dt, n * DH + PD * lane + d, L == 0.f ? 0.f : acc[d] / L);
}

// query rows of a call: wavefronts of a launch, which has below 2^32 threads in whole blocks
constexpr int64_t kMaxRows = 0x3FFFFFC;

// Wavefronts a block and most splits of a context (which the kernel shares out by
// length).  us, 32/4 heads of 128: 64 requests of 4096 positions in blocks of 8 x 1
// wavefronts x splits 27, 4 x 1 36, 8 x 2 32; 16 of 4096 8 x 4 13.4, 4 x 4 and 4 x 8
// 14.4, 8 x 8 16; 16/16 heads of 64, 64 requests of 1024: 4 x 1 21.6, 8 x 1 23.6.
// (A long context among short ones has no more than an equal share: twice as many
// splits, half of them without work, 32 requests of 500 to 4096 positions 21.2 us
// for 19.6, and 16 of 38000 to 40960 81 for 62, since some CUs get two blocks.)
struct MxPlan {
  bool decode, prefill;
  int HG, S, NW;
  float slots;  // blocks for a kv head's group of query heads: one of 8 wavefronts or
                // two of 4 a CU
};
MxPlan mx_plan(int64_t B, int64_t L, int64_t D, int64_t max_pages, int64_t page_size, int Hkv,
               int Hq) {
  MxPlan p{false, false, 1, 1, 4, 1.f};
  if ((D != 64 && D != 128) || B == 0) return p;
  const int R = Hq / Hkv;
  if (L > 1) {
    // The splits of the least time, a tile of 64 positions taken as 1.55 us of a block,
    // half as much more beside another block of its CU, a merge as 3 us and its outputs'
    // way there and back at 5 TB/s.  A tile takes 1.75 us with a bf16 query of 128 dims,
    // 2.0 with f16, 1.6 with 64 dims; the smaller figure for all leaves a few splits
    // fewer, and the choice lies within 8 % of the best of these.  (us with 1, 2, 4, 8, 16, 32 splits.
    // bf16, 32/4 heads of 128: 512 rows over 4096 positions 117, 74, 68, 76, 102, 166; 4 x
    // 256 over 1280 44, 55, 65, 94, 158, 210; 16 over 8192 222, 118, 64, 38, 26, 23.  f16:
    // 512 over 4096 130, 81, 75, 83, 107, 172.  bf16, 16/8 heads of 64: 512 over 4096 102,
    // 59, 37, 35, 40, 52; f16, 14/2 of 64: 3 x 100 over 1501 42, 28, 19, 18, 19, 22.)
    const int64_t blocks = mx_prefill_blocks(L, R), cu = cu_count();
    if (B > 0xFFFF || blocks * Hkv > 0x7FFFFF) return p;
    p.prefill = true;
    const int64_t base = blocks * Hkv * B, tiles = (max_pages * page_size + 63) / 64;
    const int64_t most = std::min<int64_t>({2 * cu / base, tiles, (int64_t)kMaxSplits});
    double least = INFINITY;
    for (int64_t s = 1; s <= std::max<int64_t>(1, most); ++s) {
      const double t = (double)((tiles + s - 1) / s) * (base * s > cu ? 2.33 : 1.55) +
                       (s > 1 ? 3. + (double)(s * B * L * Hq * D) * 8 / 5e6 : 0.);
      if (t < least) least = t, p.S = (int)s;
    }
    return p;
  }
  p.HG = R <= 8 ? 1 : (R + 15) / 16;
  // (a launch has below 2^32 threads, and below 2^16 blocks but for the first dimension)
  const int64_t heads = (int64_t)Hkv * p.HG;
  if (B > kMaxRows / 8 || heads > 0xFFFF) return p;
  p.decode = true;
  const int64_t tiles = (max_pages * page_size + kTile - 1) / kTile, cu = cu_count();
  p.NW = B * heads >= 2 * cu || B * heads * 8 < cu ? 4 : 8;
  p.slots = (float)(8 / p.NW * cu) / (float)heads;
  if (B * heads < cu)
    p.S = (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)ceil(sqrt(2. * (double)tiles)),
                                                       (tiles + p.NW - 1) / p.NW,
                                                       8 / p.NW * cu / heads / B,
                                                       (int64_t)kMaxSplits}));
  return p;
}
size_t mx_workspace(const MxPlan &p, int64_t rows, int64_t D) {
  if (p.S == 1) return 0;
  const size_t o = ((size_t)rows * p.S * D * sizeof(float) + 255) & ~(size_t)255;
  return o + (size_t)rows * p.S * 2 * sizeof(float) + 256;
}

template <int QT, int DH, bool DUP>
void launch_decode_nw(const MxAttnArgs &a, int NW, hipStream_t st) {
  const dim3 grid(a.B, a.Hkv * a.HG, a.S);
  if (NW == 8)
    hipLaunchKernelGGL((mx_decode_kernel<QT, DH, DUP, 8>), grid, dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((mx_decode_kernel<QT, DH, DUP, 4>), grid, dim3(256), 0, st, a);
}

template <int QT>
hipError_t launch_decode(const MxAttnArgs &a, int NW, hipStream_t st) {
  if (a.D == 128)
    a.R <= 8 ? launch_decode_nw<QT, 128, true>(a, NW, st)
             : launch_decode_nw<QT, 128, false>(a, NW, st);
  else
    a.R <= 8 ? launch_decode_nw<QT, 64, true>(a, NW, st)
             : launch_decode_nw<QT, 64, false>(a, NW, st);
  return hipGetLastError();
}

// The splits' outputs together, if there are any.
hipError_t launch_combine(const MxAttnArgs &a, hipStream_t st) {
  if (a.S == 1) return hipSuccess;
  const int64_t rows = (int64_t)a.B * a.L * a.Hq;
  const unsigned blocks = (unsigned)((rows + kRowThreads / 64 - 1) / (kRowThreads / 64));
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(blocks), dim3(kRowThreads), 0, st, a.part_o, a.part_ml, rows, a.S,
                       a.out, a.out_dt);
  };
  if (a.L == 1)
    a.D == 128 ? go(mx_combine_kernel<128, true>) : go(mx_combine_kernel<64, true>);
  else
    a.D == 128 ? go(mx_combine_kernel<128, false>) : go(mx_combine_kernel<64, false>);
  return hipGetLastError();
}

int check_shape(const char *op, int64_t B, int64_t L, int64_t D, int64_t max_pages,
                int64_t page_size, int Hkv, int Hq) {
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv)
    return set_error(NVM_ERR_INVALID, "%s: num_heads must be divisible by num_kv_heads", op);
  if (B < 0 || L < 1 || D < 1 || page_size < 1 || max_pages < 0)
    return set_error(NVM_ERR_INVALID, "%s: bad shape B=%lld L=%lld D=%lld page_size=%lld "
                     "max_pages=%lld", op, (long long)B, (long long)L, (long long)D,
                     (long long)page_size, (long long)max_pages);
  if (D % 32 || D > 256)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: head dim %lld must be a multiple of 32, at most 256",
                     op, (long long)D);
  // (positions are 32-bit, with room for a tile past the last)
  if (max_pages > 0x7FFF0000ll / page_size)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: context capacity too large", op);
  if (B > kMaxRows || L > kMaxRows || B * L > kMaxRows / Hq)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: too many query rows", op);
  return NVM_OK;
}

}  // namespace

}  // namespace nvm

extern "C" {

int nvm_paged_attention_mx_workspace_size(int64_t B, int64_t L, int64_t D, int64_t max_pages,
                                          int64_t page_size, int num_kv_heads, int num_heads,
                                          size_t *bytes) {
  using namespace nvm;
  constexpr const char *op = "paged_attention_mx";
  if (int rc = check_shape(op, B, L, D, max_pages, page_size, num_kv_heads, num_heads)) return rc;
  if (!bytes) return set_error(NVM_ERR_INVALID, "%s: null bytes", op);
  *bytes = mx_workspace(mx_plan(B, L, D, max_pages, page_size, num_kv_heads, num_heads),
                        B * L * num_heads, D);
  return NVM_OK;
}

int nvm_paged_attention_mx(const void *q, int q_dtype, int64_t q_stride_b, int64_t q_stride_h,
                           int64_t q_stride_l, int64_t B, int64_t L, int64_t D,
                           const void *key_codes, const uint8_t *key_scales,
                           const void *value_codes, const uint8_t *value_scales, int64_t P,
                           int64_t page_size, const int32_t *block_table, int64_t max_pages,
                           const int32_t *context_lens, float scale, int is_causal,
                           int num_kv_heads, int num_heads, int out_dtype, void *out,
                           void *workspace, size_t workspace_bytes, nvm_stream_t stream) {
  using namespace nvm;
  constexpr const char *op = "paged_attention_mx";
  auto plain = [](int dt) { return dt == NVM_KV_F16 || dt == NVM_KV_BF16 || dt == NVM_KV_F32; };
  if (!plain(q_dtype) || !plain(out_dtype))
    return set_error(NVM_ERR_INVALID, "%s: query and out dtypes must be f16, bf16 or f32", op);
  if (int rc = check_shape(op, B, L, D, max_pages, page_size, num_kv_heads, num_heads)) return rc;
  if (int rc = mx_check_pages(op, num_kv_heads, D, P, page_size, key_codes, key_scales,
                              value_codes, value_scales))
    return rc;
  if (B == 0) return NVM_OK;
  if (!q || !out || !context_lens || (max_pages > 0 && !block_table))
    return set_error(NVM_ERR_INVALID, "%s: null pointer", op);
  const int64_t unit = q_dtype == NVM_KV_F32 ? 4 : 8;  // values of 16 bytes
  if (((uintptr_t)q & 15) || q_stride_b % unit || q_stride_h % unit || q_stride_l % unit)
    return set_error(NVM_ERR_INVALID, "%s: query rows must be 16-byte aligned", op);
  MxAttnArgs a{};
  a.q = q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.q_sl = q_stride_l;
  a.kc = (const uint8_t *)key_codes;
  a.ks = key_scales;
  a.vc = (const uint8_t *)value_codes;
  a.vs = value_scales;
  a.bt = max_pages ? block_table : context_lens;  // (ids are read before they are known to count)
  a.lens = context_lens;
  a.out = out;
  a.out_dt = out_dtype;
  a.B = (int)B;
  a.L = (int)L;
  a.D = (int)D;
  a.P = (int)P;
  a.page_size = (int)page_size;
  a.max_pages = (int)max_pages;
  a.Hkv = num_kv_heads;
  a.Hq = num_heads;
  a.R = num_heads / num_kv_heads;
  a.causal = is_causal ? 1 : 0;
  // (the largest score is the largest product then; a scale of zero as one that
  // takes any product to zero, but not -infinity to a NaN)
  a.scale2 = std::max(fabsf(scale) * kLog2e, 1.17549435e-38f);
  if (scale != scale) a.scale2 = scale;
  a.q_sign = scale < 0.f ? 0x80008000u : 0u;
  hipStream_t st = (hipStream_t)stream;
  uint32_t l = 0;
  while (((int64_t)1 << l) < page_size) ++l;
  a.ps_mul = l ? (uint32_t)((((uint64_t)1 << (31 + l)) + page_size - 1) / page_size) : 0;
  a.ps_shift = l ? l - 1 : 0;
  const MxPlan plan = mx_plan(B, L, D, max_pages, page_size, num_kv_heads, num_heads);
  const size_t need = mx_workspace(plan, B * L * num_heads, D);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(NVM_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", op, need);
  a.HG = plan.HG;
  a.S = plan.S;
  a.slots = plan.slots;
  if (plan.S > 1) {
    a.part_o = (float *)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
    a.part_ml = (float *)((char *)a.part_o +
                          (((size_t)(B * L * num_heads) * plan.S * D * sizeof(float) + 255) &
                           ~(size_t)255));
  }
  auto go = [&](auto qt) {
    constexpr int QT = decltype(qt)::value;
    return plan.decode ? launch_decode<QT>(a, plan.NW, st) : launch_rows<QT>(a, st);
  };
  hipError_t e = plan.prefill             ? launch_mx_prefill(q_dtype, a, st)
                 : q_dtype == NVM_KV_F32  ? go(MxInt<NVM_KV_F32>{})
                 : q_dtype == NVM_KV_BF16 ? go(MxInt<NVM_KV_BF16>{})
                                          : go(MxInt<NVM_KV_F16>{});
  if (e == hipSuccess) e = launch_combine(a, st);
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

}  // extern "C"
