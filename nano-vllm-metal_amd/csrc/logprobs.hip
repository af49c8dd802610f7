// Log probabilities of tokens, entropy and the most probable alternatives of
// rows of logits (declared in include/nvm_logprobs.h).
//
// One pass over a row, or over a part of it where there are few rows.  With L =
// log2 e as a float32 a lane keeps its largest value X and, of all its other ones, Z =
// sum 2^(x L - m) and S = sum 2^(x L - m) (x L - m), m being X L as a float32 (one that
// moves by steps of 16 only was no faster).  x L - m is one fma, whose product is exact.
// A vector's few terms are summed in float32, everything beyond in float64, where X
// joins them as a term of 1 at the reference X L, exact in float64.  So the row's
// largest term is exactly 1 and none of the others is lost beside it: a token that is
// all but certain has its log probability and entropy to float32's own precision (with
// X among the other terms both were off by 1e-7, more than they are).  At the end
// log p(t) = (x_t L - m - log2 Z) / L and the entropy H = (log2 Z - S / Z) / L.  L is
// log2 e less 1.3e-8 of itself, a temperature that far from 1: log p gets back the 1.3e-8 H
// that it takes away; the entropy is off by 1.3e-8 of the logits' variance.
//
// That fails for values beyond 2.3e38, whose x L is none, and S for -infinity: a
// tile whose S comes out NaN takes its terms again with the difference clamped, and
// a part with an X like that is read again with x - X in place of x L - m (a row of
// bf16's or float32's lowest values; a lane that sees nothing else suffices).  Both
// cost time (2048 x 151936 bf16, top 5, all but 1000 logits masked: -infinities 246 us, the
// lowest value 430, which all but 10000 masked do not reach).
//
// The largest logits, in the same pass, by a wavefront each: keys of 64 bits
// (the value's order, then the lower id), which are all different.  A threshold
// T that at least top_k keys reach is known from the first tile on: the top_k-th
// largest of the 64 lanes' maxima; later the block's.
// A vector whose maximum lies below T, nearly every one, costs a comparison; keys
// from T on go to a list in LDS, and a full list is cut to its top_k largest, which
// raises T; after the first tile and the fourth the block's lists are compared.  So
// the result does not depend on the order of anything, and rows in ascending order
// are slow, not wrong.
//
// Bound: HBM for many rows (2048 x 151936 bf16: 105 us, 5.9 TB/s; top 5 130 us, 20
// 172, 64 392, of the lists' first keys), a lane's 10 slots a value close behind (4 of
// them exp's, 1.5 to keep X out: 104 us for 103.5, top 5 129 for 125.5; with all of a
// tile's other values in registers, 110 for 94, 116 and 151); for one row (top 5: 13 us)
// latency, of two launches.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal.h"
#include "nvm_logprobs.h"

namespace nvm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLog2eOff = 1.0 - (double)kLog2e / 1.4426950408889634;
constexpr int kWaves = 4;
constexpr int kUnroll = 4;                    // vectors of a lane's tile
constexpr int kMaxTop = NVM_MAX_TOP_LOGPROBS;
constexpr int kList = kMaxTop + 128;          // keys of a wavefront's list
constexpr int kMaxSplits = 64;

struct LogprobArgs {
  const void *x;
  int64_t N, ld;
  int V, k, S;
  const int64_t *tokens;
  float *lp, *ent;
  int64_t *ids;
  float *top;
  // of splits: keys [N][S][k] (0: none) and sums [N][S][3]
  uint64_t *part_keys;
  double *part_sums;
};

template <int DT>
struct Logits {
  static constexpr int kSize = DT == NVM_LOGITS_F32 ? 4 : 2;
  static constexpr int kPer = 16 / kSize;  // values of a vector
  __device__ static __forceinline__ float at(u32x4 v, int i) {
    if constexpr (DT == NVM_LOGITS_F32) return __uint_as_float(v[i]);
    if constexpr (DT == NVM_LOGITS_BF16)
      return (i & 1) ? Act<DT_BF16>::hi(v[i >> 1]) : Act<DT_BF16>::lo(v[i >> 1]);
    return (i & 1) ? Act<DT_F16>::hi(v[i >> 1]) : Act<DT_F16>::lo(v[i >> 1]);
  }
  // The dword of value i, and the value in it, of i that differs by lane.
  __device__ static __forceinline__ uint32_t dword(u32x4 v, int i) {
    const int w = DT == NVM_LOGITS_F32 ? i : i >> 1;
    const uint32_t a = (w & 1) ? v[1] : v[0], b = (w & 1) ? v[3] : v[2];
    return (w & 2) ? b : a;
  }
  __device__ static __forceinline__ float of(uint32_t d, int i) {
    if constexpr (DT == NVM_LOGITS_F32) return __uint_as_float(d);
    const uint32_t h = (i & 1) ? d >> 16 : d & 0xFFFFu;
    return DT == NVM_LOGITS_BF16 ? Act<DT_BF16>::to_f32(h) : Act<DT_F16>::to_f32(h);
  }
  // Value i to -infinity.
  __device__ static __forceinline__ void lowest(u32x4 &v, int i) {
    if constexpr (DT == NVM_LOGITS_F32) {
      v[i] = 0xFF800000u;
    } else {
      constexpr uint32_t kLow = DT == NVM_LOGITS_BF16 ? 0xFF80u : 0xFC00u;
      v[i >> 1] = (i & 1) ? (v[i >> 1] & 0xFFFFu) | kLow << 16 : (v[i >> 1] & 0xFFFF0000u) | kLow;
    }
  }
  __device__ static __forceinline__ float one(const void *x, int64_t i) {
    if constexpr (DT == NVM_LOGITS_F32) return ((const float *)x)[i];
    if constexpr (DT == NVM_LOGITS_BF16) return Act<DT_BF16>::to_f32(((const uint16_t *)x)[i]);
    return Act<DT_F16>::to_f32(((const uint16_t *)x)[i]);
  }
};

// The larger, NaN if one of them is.
__device__ __forceinline__ float max_nan(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

// The smallest of values without NaNs.
__device__ __forceinline__ float min3(float a, float b, float c) {
  return __builtin_elementwise_minimum(__builtin_elementwise_minimum(a, b), c);
}

// Order of float32 values as that of unsigned integers: NaNs above +infinity,
// both zeros alike.
__device__ __forceinline__ uint32_t ordered(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu));
}
// (ids are below 2^31: no key is zero, which stands for none)
__device__ __forceinline__ uint64_t key_of(float v, int id) {
  return ((uint64_t)ordered(v) << 32) | (0xFFFFFFFFu - (uint32_t)id);
}
__device__ __forceinline__ int id_of(uint64_t key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }
__device__ __forceinline__ float value_of(uint64_t key) {
  return from_ordered((uint32_t)(key >> 32));
}

__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return ((uint64_t)hi << 32) | lo;
}

// The k-th largest of the lanes' keys (0: fewer than k of them).
__device__ __forceinline__ uint64_t kth_of_lanes(uint64_t key, int k) {
  int above = 0;
#pragma unroll 4
  for (int i = 0; i < 64; ++i) above += lane_of(key, i) > key;
  const uint64_t at = __builtin_amdgcn_ballot_w64(key != 0 && above == k - 1);
  return at ? lane_of(key, __builtin_ctzll(at)) : 0;
}

// What at least k keys reach (all of them, if there are fewer), from the lanes'
// largest values: the k-th of these, its lowest six bits cleared.  Those hold the
// lane for the ranks.  (By 64-bit keys of the values themselves, three times the
// instructions: 2048 rows of 151936, top 5, 135 us for 125.)
__device__ __forceinline__ uint64_t first_threshold(float top, int k, int lane) {
  const uint32_t o = (ordered(top) & ~63u) | (uint32_t)lane;
  int above = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) above += (uint32_t)__builtin_amdgcn_readlane((int)o, i) > o;
  const uint64_t at = __builtin_amdgcn_ballot_w64(above == k - 1);
  const uint32_t v = (uint32_t)__builtin_amdgcn_readlane((int)o, __builtin_ctzll(at));
  return (uint64_t)(v & ~63u) << 32;
}

// A wavefront's list of keys, in LDS.
struct TopList {
  uint64_t *keys;
  int n;       // uniform
  uint64_t T;  // uniform: at least k keys seen so far reach it (0: not known)

  // Appends the lanes' keys that reach T.
  __device__ __forceinline__ void push(uint64_t key, int k, int lane) {
    if (key < T) key = 0;
    uint64_t on = __builtin_amdgcn_ballot_w64(key != 0);
    if (n + __builtin_popcountll(on) > kList) {
      cut(k, lane);
      if (key < T) key = 0;
      on = __builtin_amdgcn_ballot_w64(key != 0);
    }
    const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(on >> 32),
                                                 __builtin_amdgcn_mbcnt_lo((uint32_t)on, 0));
    if (key != 0) keys[at] = key;
    n += __builtin_popcountll(on);
  }

  // The k largest (all, if there are fewer), in order; T the last of k.
  __device__ __forceinline__ void cut(int k, int lane) {
    constexpr int NK = (kList + 63) / 64;
    wave_lds_sync();
    if (n <= 64) {  // uniform, and the rule
      const uint64_t key = lane < n ? keys[lane] : 0;
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += lane_of(key, j) > key;
      wave_lds_sync();
      if (key != 0 && rank < k) keys[rank] = key;
      wave_lds_sync();
      n = min(n, k);
      if (n == k) T = max(T, keys[k - 1]);
      return;
    }
    uint64_t v[NK], most = 0;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      v[i] = lane + 64 * i < n ? keys[lane + 64 * i] : 0;
      most = max(most, v[i]);
    }
    // those below the k-th largest of the lanes' maxima go first
    const uint64_t floor_ = kth_of_lanes(most, k);
    wave_lds_sync();
    int m = 0;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const bool on = v[i] != 0 && v[i] >= floor_;
      const uint64_t b = __builtin_amdgcn_ballot_w64(on);
      const int at = m + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32),
                                                   __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
      if (on) keys[at] = v[i];
      m += __builtin_popcountll(b);
    }
    wave_lds_sync();
    int rank[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      v[i] = lane + 64 * i < m ? keys[lane + 64 * i] : 0;
      rank[i] = 0;
    }
#pragma unroll 1
    for (int j = 0; j < m; ++j) {
      const uint64_t o = keys[j];
#pragma unroll
      for (int i = 0; i < NK; ++i) rank[i] += o > v[i];
    }
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < NK; ++i)
      if (v[i] != 0 && rank[i] < k) keys[rank[i]] = v[i];
    wave_lds_sync();
    n = min(m, k);
    if (n == k) T = max(T, keys[k - 1]);
  }
};

// Sums of a part of a row.
struct Part {
  double m, z, s;
  // (the other part's at the larger reference; with nothing seen m is -1e39, below
  // every value's)
  __device__ __forceinline__ void add(const Part &o) {
    const double mm = max(m, o.m), da = m - mm, db = o.m - mm;
    const double fa = __builtin_amdgcn_exp2f((float)da), fb = __builtin_amdgcn_exp2f((float)db);
    s = fa * (s + z * da) + fb * (o.s + o.z * db);
    z = fa * z + fb * o.z;
    m = mm;
  }
};

struct BlockState {
  uint64_t keys[kWaves][kList];
  uint64_t T;  // the block's threshold
  int n[kWaves];
  double sums[kWaves][3];
};

// The block's sums from the wavefronts', in every thread.
__device__ __forceinline__ Part block_sums(BlockState &b, Part p, int lane, int wv) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    p.add(Part{__shfl_xor(p.m, o), __shfl_xor(p.z, o), __shfl_xor(p.s, o)});
  if (lane == 0) b.sums[wv][0] = p.m, b.sums[wv][1] = p.z, b.sums[wv][2] = p.s;
  __syncthreads();
  p = {b.sums[0][0], b.sums[0][1], b.sums[0][2]};
#pragma unroll
  for (int w = 1; w < kWaves; ++w) p.add(Part{b.sums[w][0], b.sums[w][1], b.sums[w][2]});
  return p;
}

// f(place, key) of the k largest of the wavefronts' lists, which are in order (a
// barrier lies behind them): a key's place is the number of larger ones, which a
// search by halves counts in each other list.
template <class F>
__device__ __forceinline__ void block_top(const BlockState &b, int k, int lane, int wv, F f) {
  for (int i = lane; i < b.n[wv]; i += 64) {
    const uint64_t v = b.keys[wv][i];
    int larger[kWaves] = {};
    for (int step = 1 << (31 - __builtin_clz(k)); step > 0; step >>= 1)
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int at = larger[w] + step;
        if (at <= b.n[w] && b.keys[w][at - 1] > v) larger[w] = at;
      }
    int place = 0;  // (in its own list, too)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) place += larger[w];
    if (place < k) f(place, v);
  }
}

// The block's threshold after so many tiles: the k-th largest of all lists, which
// lose what lies below it.  (With each wavefront's own, from its first 2048 logits,
// some k / 2048 of all others came after it: 2048 rows of 151936, top 5, 301 us.)
__device__ __forceinline__ void block_threshold(BlockState &b, TopList &list, int k, int lane,
                                                int wv) {
  list.cut(k, lane);
  if (lane == 0) b.n[wv] = list.n;
  __syncthreads();
  block_top(b, k, lane, wv, [&](int place, uint64_t v) {
    if (place == k - 1) b.T = v;
  });
  __syncthreads();
  list.T = max(list.T, b.T);
  const uint64_t mine = lane < list.n ? list.keys[lane] : 0;
  list.n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine != 0 && mine >= list.T));
}

template <int DT>
__device__ __forceinline__ void store_row(const LogprobArgs &a, BlockState &b, int64_t row,
                                          const Part &p, float xt, int lane, int wv) {
  // (x L - m first, exactly: of values of 1e38 their difference is all that counts)
  const double lz = log2(p.z), h = (lz - p.s / p.z) / (double)kLog2e;
  const double off = kLog2eOff * h;
  // (neither above zero nor, the entropy, below it by an error of exp2)
  auto logprob = [&](float v) {
    const double d = ((double)v * (double)kLog2e - p.m - lz) / (double)kLog2e + off;
    return d > 0.0 ? 0.f : (float)d;
  };
  if (threadIdx.x == 0) {
    const int64_t t = a.tokens[row];
    a.lp[row] = t >= 0 && t < a.V ? logprob(xt) : 0.f;
    a.ent[row] = h < 0.0 ? 0.f : (float)h;
  }
  if (a.k > 0)
    block_top(b, a.k, lane, wv, [&](int place, uint64_t v) {
      a.ids[row * a.k + place] = id_of(v);
      a.top[row * a.k + place] = logprob(value_of(v));
    });
}

// The logit of a row's token, or of token 0: asked for at the start, since it is two
// trips to memory away.
template <int DT>
__device__ __forceinline__ float token_logit(const LogprobArgs &a, int64_t row) {
  const int64_t t = a.tokens[row];
  return Logits<DT>::one(a.x, row * a.ld + (t >= 0 && t < a.V ? t : 0));
}

// Grid: rows, splits.
template <int DT>
__global__ __launch_bounds__(64 * kWaves) void token_logprobs_kernel(LogprobArgs a) {
  using X = Logits<DT>;
  constexpr int PER = X::kPer;
  constexpr int kTile = 64 * kUnroll;  // vectors of a wavefront's tile
  __shared__ BlockState s_b;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  const char *x = (const char *)a.x + row * a.ld * X::kSize;
  // vectors from the 16-byte border at or before the row: the first one's
  // leading values belong to another row
  const int lead = (int)(((uintptr_t)x & 15) / X::kSize);
  const char *base = x - lead * X::kSize;
  const int nv = (int)(((int64_t)lead + a.V + PER - 1) / PER);
  // of these this split's
  const int per = (nv + a.S - 1) / a.S, first = min((int)blockIdx.y * per, nv);
  const int end = min(first + per, nv);
  if (threadIdx.x == 0) s_b.T = 0;
  __syncthreads();
  const float xt = a.S == 1 ? token_logit<DT>(a, row) : 0.f;

  auto load = [&](int v0, u32x4 (&raw)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      raw[u] = ldg16_once(base + (int64_t)min(v0 + 64 * u + lane, nv - 1) * 16);
    // values outside the row (of its first and last vector), and vectors outside the split
    if (v0 + kTile > end || v0 + kTile >= nv || v0 == 0) {  // uniform
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int v = v0 + 64 * u + lane;
        const int64_t id = (int64_t)v * PER - lead;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (v >= end || id + i < 0 || id + i >= a.V) X::lowest(raw[u], i);
      }
    }
  };

  Part p = {-1e39, 0.0, 0.0};
  TopList list = {s_b.keys[wv], 0, 0};
  float m = -3.402823466e38f, top = -INFINITY;
  const int rounds = (end - first + kWaves * kTile - 1) / (kWaves * kTile);
  for (int it = 0; it < rounds; ++it) {
    const int v0 = first + (it * kWaves + wv) * kTile;
    if (v0 < end) {  // uniform
      u32x4 raw[kUnroll];
      load(v0, raw);
      float tmax[kUnroll], most = top;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float t = X::at(raw[u], 0);
#pragma unroll
        for (int i = 1; i < PER; ++i) t = max_nan(t, X::at(raw[u], i));
        tmax[u] = t;
        most = max_nan(most, t);
      }
      const bool above = most * kLog2e > m;
      if (__any(above)) {
        const float mn = fmaxf(m, most * kLog2e);
        const double d = (double)m - (double)mn, alpha = __builtin_amdgcn_exp2f((float)d);
        p.s = alpha * (p.s + p.z * d);
        p.z *= alpha;
        m = mn;
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        // the vector's values and X less the largest of them, which is X from here on
        float rest[PER], z = 0.f, s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; i += 2) {
          const float v = X::at(raw[u], i), w = X::at(raw[u], i + 1);
          rest[i] = min3(top, v, w);
          rest[i + 1] = __builtin_amdgcn_fmed3f(top, v, w);
          top = max_nan(max_nan(top, v), w);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const float d = fmaf(rest[i], kLog2e, -m);
          const float e = __builtin_amdgcn_exp2f(d);
          z += e;
          s = fmaf(e, d, s);
        }
        if (__any(s != s)) {  // (0 for -infinity)
          s = 0.f;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const float d = fmaf(rest[i], kLog2e, -m);
            s = fmaf(__builtin_amdgcn_exp2f(d), fmaxf(d, -1e30f), s);
          }
        }
        p.z += (double)z;
        p.s += (double)s;
      }
      if (a.k > 0) {  // uniform
        if (list.T == 0) list.T = first_threshold(top, a.k, lane);
        // (values below the lowest number's are -infinity's)
        const float limit = list.T >> 32 > 0x007FFFFFu ? value_of(list.T) : -INFINITY;
        uint64_t hit[kUnroll], any = 0;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          hit[u] = __builtin_amdgcn_ballot_w64(!(tmax[u] < limit) & (v0 + 64 * u + lane < end));
          any |= hit[u];
        }
        if (any) {
          // (of those that only reach T's value, from T's id on none counts)
          const int64_t idT = 0xFFFFFFFFu - (uint32_t)list.T;
#pragma unroll
          for (int u = 0; u < kUnroll; ++u)
            hit[u] &= __builtin_amdgcn_ballot_w64(
                tmax[u] != limit || (int64_t)(v0 + 64 * u + lane) * PER - lead <= idT);
#pragma unroll 1
          for (int u = 0; u < kUnroll; ++u) {
            uint64_t h = hit[0];
            u32x4 r = raw[0];
#pragma unroll
            for (int w = 1; w < kUnroll; ++w)
              if (u == w) h = hit[w], r = raw[w];
            // one lane's vector after the other, a value a lane: few have one that counts
            // (a second path, by value, for vectors of four lanes and more: top 64 of
            // 2048 rows of 151936 323 us for 380, but top 5 128 for 124, 20 178 for 162)
#pragma unroll 1
            while (h) {
              const int from = __builtin_ctzll(h), e = lane & (PER - 1);
              h &= h - 1;
              u32x4 one;
#pragma unroll
              for (int w = 0; w < 4; ++w)
                one[w] = (uint32_t)__builtin_amdgcn_readlane((int)r[w], from);
              const uint32_t d = X::dword(one, e);
              const int64_t id = (int64_t)(v0 + 64 * u + from) * PER + e - lead;
              const bool on = lane < PER && id >= 0 && id < a.V;
              list.push(on ? key_of(X::of(d, e), (int)id) : 0, a.k, lane);
            }
          }
        }
      }
    }
    // (uniform in the block)
    if (a.k > 0 && ((it == 0 && rounds > 2) || (it == 3 && rounds > 6)))
      block_threshold(s_b, list, a.k, lane, wv);
  }
  // (top: none of the values that are there, or one whose product with L is one)
  if (!__any(top != -INFINITY && !(fabsf(top * kLog2e) < INFINITY))) {
    if (top != -INFINITY) {
      const double r = (double)top * (double)kLog2e, d = (double)m - r;
      const double f = __builtin_amdgcn_exp2f((float)d);
      p = {r, 1.0 + f * p.z, f * (p.s + p.z * d)};
    }
  } else {
    p = {-1e39, 0.0, 0.0};
    top = -3.402823466e38f;
    for (int v0 = first + wv * kTile; v0 < end; v0 += kWaves * kTile) {
      u32x4 raw[kUnroll];
      load(v0, raw);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll 1
        for (int i = 0; i < PER; ++i) {
          const float f = X::at(raw[u], i);
          const float t = max_nan(top, f);
          const double d0 = ((double)top - (double)t) * (double)kLog2e;
          const double alpha = __builtin_amdgcn_exp2f((float)d0);
          const float d = (f - t) * kLog2e, e = __builtin_amdgcn_exp2f(d);
          p.s = alpha * (p.s + p.z * d0) + (double)(e * fmaxf(d, -1e30f));
          p.z = alpha * p.z + (double)e;
          top = t;
        }
    }
    p.m = (double)top * (double)kLog2e;
  }

  if (a.k > 0) list.cut(a.k, lane);
  if (lane == 0) s_b.n[wv] = list.n;
  p = block_sums(s_b, p, lane, wv);
  if (a.S == 1) {
    store_row<DT>(a, s_b, row, p, xt, lane, wv);
    return;
  }
  const int64_t at = row * a.S + blockIdx.y;
  if (threadIdx.x == 0) {
    double *o = a.part_sums + at * 3;
    o[0] = p.m, o[1] = p.z, o[2] = p.s;
  }
  if (a.k > 0) {
    uint64_t *o = a.part_keys + at * a.k;
    const int total = s_b.n[0] + s_b.n[1] + s_b.n[2] + s_b.n[3];
    if ((int)threadIdx.x >= total && (int)threadIdx.x < a.k) o[threadIdx.x] = 0;
    block_top(s_b, a.k, lane, wv, [&](int place, uint64_t v) { o[place] = v; });
  }
}

// A row's splits together.
template <int DT>
__global__ __launch_bounds__(64 * kWaves) void logprobs_merge_kernel(LogprobArgs a) {
  __shared__ BlockState s_b;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  const float xt = token_logit<DT>(a, row);
  Part p = {-1e39, 0.0, 0.0};
  if (threadIdx.x < a.S) {
    const double *o = a.part_sums + (row * a.S + threadIdx.x) * 3;
    p = {o[0], o[1], o[2]};
  }
  TopList list = {s_b.keys[wv], 0, 0};
  if (a.k > 0) {
    const uint64_t *keys = a.part_keys + row * a.S * a.k;
    const int n = a.S * a.k;
    uint64_t most = 0;
    for (int i = threadIdx.x; i < n; i += 64 * kWaves) most = max(most, keys[i]);
    list.T = kth_of_lanes(most, a.k);
    for (int i = 64 * wv; i < n; i += 64 * kWaves)  // uniform
      list.push(i + lane < n ? keys[i + lane] : 0, a.k, lane);
    list.cut(a.k, lane);
  }
  if (lane == 0) s_b.n[wv] = list.n;
  p = block_sums(s_b, p, lane, wv);
  store_row<DT>(a, s_b, row, p, xt, lane, wv);
}

template <int DT>
void launch_logprobs(const LogprobArgs &a, hipStream_t st) {
  hipLaunchKernelGGL(token_logprobs_kernel<DT>, dim3((unsigned)a.N, (unsigned)a.S),
                     dim3(64 * kWaves), 0, st, a);
  if (a.S > 1)
    hipLaunchKernelGGL(logprobs_merge_kernel<DT>, dim3((unsigned)a.N), dim3(64 * kWaves), 0, st, a);
}

// Splits of a row: four blocks a CU, none of less than a tile a wavefront (1 x 151936
// bf16 top 5 and 33 x 50257 float32 top 20: 13.2 and 22.6 us, with half a tile 13.0 and
// 24.4, with two 17.2 and 32.3).
int logprobs_splits(int64_t N, int64_t V, int dtype) {
  const int64_t vectors = V / (dtype == NVM_LOGITS_F32 ? 4 : 8) + 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>({4 * cu_count() / std::max<int64_t>(N, 1),
                                                      (vectors - 1) / (64 * kUnroll * kWaves) + 1,
                                                      (int64_t)kMaxSplits}));
}
size_t logprobs_workspace(int64_t N, int S, int k) {
  return S == 1 ? 0 : (size_t)N * S * (3 * sizeof(double) + (size_t)k * sizeof(uint64_t)) + 256;
}

int check_logprobs(const char *op, int64_t N, int64_t V, int dtype, int top_k) {
  if (dtype != NVM_LOGITS_F16 && dtype != NVM_LOGITS_BF16 && dtype != NVM_LOGITS_F32)
    return set_error(NVM_ERR_INVALID, "%s: logits must be f16, bf16 or f32", op);
  if (N < 0 || V <= 0)
    return set_error(NVM_ERR_INVALID, "%s: bad shape: %lld rows of %lld logits", op, (long long)N,
                     (long long)V);
  if (top_k < 0 || top_k > V)
    return set_error(NVM_ERR_INVALID, "%s: top_k must be in [0, V], got %d", op, top_k);
  if (top_k > kMaxTop)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: top_k at most %d, got %d", op, kMaxTop, top_k);
  if (V > INT32_MAX - 64 || N > 0xFFFFFF)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: %lld rows of %lld logits are too many", op,
                     (long long)N, (long long)V);
  return NVM_OK;
}

}  // namespace

}  // namespace nvm

extern "C" {

int nvm_token_logprobs_workspace_size(int64_t N, int64_t V, int dtype, int top_k, size_t *bytes) {
  using namespace nvm;
  constexpr const char *op = "token_logprobs";
  if (int rc = check_logprobs(op, N, V, dtype, top_k)) return rc;
  if (!bytes) return set_error(NVM_ERR_INVALID, "%s: null bytes", op);
  *bytes = logprobs_workspace(N, logprobs_splits(N, V, dtype), top_k);
  return NVM_OK;
}

int nvm_token_logprobs(const void *logits, int64_t N, int64_t V, int64_t ld, int dtype,
                       const int64_t *tokens, int top_k, float *logprobs, float *entropy,
                       int64_t *top_ids, float *top_logprobs, void *workspace,
                       size_t workspace_bytes, nvm_stream_t stream) {
  using namespace nvm;
  constexpr const char *op = "token_logprobs";
  if (int rc = check_logprobs(op, N, V, dtype, top_k)) return rc;
  if (N > 1 && ld < V)
    return set_error(NVM_ERR_INVALID, "%s: rows of %lld logits are %lld apart", op, (long long)V,
                     (long long)ld);
  if (N == 0) return NVM_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top_k > 0 && (!top_ids || !top_logprobs)))
    return set_error(NVM_ERR_INVALID, "%s: null pointer", op);
  if ((uintptr_t)logits & (dtype == NVM_LOGITS_F32 ? 3 : 1))
    return set_error(NVM_ERR_INVALID, "%s: logits must be aligned to their type", op);
  LogprobArgs a = {logits, N, ld, (int)V, top_k, logprobs_splits(N, V, dtype), tokens, logprobs,
                   entropy, top_ids, top_logprobs, nullptr, nullptr};
  const size_t need = logprobs_workspace(N, a.S, top_k);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(NVM_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", op, need);
  if (a.S > 1) {
    a.part_sums = (double *)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
    a.part_keys = (uint64_t *)(a.part_sums + (size_t)N * a.S * 3);
  }
  hipStream_t st = (hipStream_t)stream;
  if (dtype == NVM_LOGITS_F32)
    launch_logprobs<NVM_LOGITS_F32>(a, st);
  else if (dtype == NVM_LOGITS_BF16)
    launch_logprobs<NVM_LOGITS_BF16>(a, st);
  else
    launch_logprobs<NVM_LOGITS_F16>(a, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

}  // extern "C"
