// Log probabilities of tokens, entropy and the most probable alternatives of
// rows of logits (declared in include/nvm_logprobs.h).
//
// One pass over a row: a lane keeps a maximum m, Z = sum exp(x - m) and S = sum
// exp(x - m) (x - m) of what it read; then log p(t) = x_t - m - log Z and the
// entropy is log Z - S / Z, whose terms are all positive.  A vector's few terms
// are summed in float32, everything beyond in float64.
//
// The largest logits, in the same pass, by a wavefront each: keys of 64 bits
// (the value's order, then the lower id), which are all different.  A threshold
// T that at least top_k keys reach is known from the first tile on: the top_k-th
// largest of the 64 lanes' maxima.  A vector whose maximum lies below T, nearly
// every one, costs a comparison; keys from T on go to a list in LDS, and a full
// list is cut to its top_k largest, which raises T.  So the result does not
// depend on the order of anything, and rows in ascending order are slow, not
// wrong.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "internal.h"
#include "nvm_logprobs.h"

namespace nvm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4;
constexpr int kUnroll = 4;                    // vectors of a lane's tile
constexpr int kMaxTop = NVM_MAX_TOP_LOGPROBS;
constexpr int kList = kMaxTop + 128;          // keys of a wavefront's list

struct LogprobArgs {
  const void *x;
  int64_t N, ld;
  int V, k;
  const int64_t *tokens;
  float *lp, *ent;
  int64_t *ids;
  float *top;
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
__device__ __forceinline__ float value_of(uint64_t key) { return from_ordered((uint32_t)(key >> 32)); }

__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return ((uint64_t)hi << 32) | lo;
}

// The k-th largest of the lanes' keys (0: fewer than k of them).
__device__ __forceinline__ uint64_t kth_of_lanes(uint64_t key, int k) {
  int above = 0;
  for (int i = 0; i < 64; ++i) above += lane_of(key, i) > key;
  const uint64_t at = __builtin_amdgcn_ballot_w64(key != 0 && above == k - 1);
  return at ? lane_of(key, __builtin_ctzll(at)) : 0;
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
    if (n == k) T = keys[k - 1];
  }
};

// Sums of a part of a row: m, Z and S.
struct Part {
  float m;
  double z, s;
  // (the other part's sums at the larger maximum; a maximum of -FLT_MAX stands
  // for nothing seen)
  __device__ __forceinline__ void add(float mo, double zo, double so) {
    const float mm = max_nan(m, mo);
    const float da = m - mm, db = mo - mm;
    const double fa = __builtin_amdgcn_exp2f(da * kLog2e), fb = __builtin_amdgcn_exp2f(db * kLog2e);
    s = fa * (s + z * (double)fmaxf(da, -1e30f)) + fb * (so + zo * (double)fmaxf(db, -1e30f));
    z = fa * z + fb * zo;
    m = mm;
  }
};

template <int DT>
__global__ __launch_bounds__(64 * kWaves) void token_logprobs_kernel(LogprobArgs a) {
  using X = Logits<DT>;
  constexpr int PER = X::kPer;
  __shared__ uint64_t s_keys[kWaves][kList];
  __shared__ int s_n[kWaves];
  __shared__ float s_m[kWaves];
  __shared__ double s_z[kWaves], s_s[kWaves];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const char *x = (const char *)a.x + row * a.ld * X::kSize;
  // vectors from the 16-byte border at or before the row: the first one's
  // leading values belong to another row
  const int lead = (int)(((uintptr_t)x & 15) / X::kSize);
  const char *base = x - lead * X::kSize;
  const int nv = (int)(((int64_t)lead + a.V + PER - 1) / PER);
  Part p = {-3.402823466e38f, 0.0, 0.0};
  TopList list = {s_keys[wv], 0, 0};
  float limit = -INFINITY;  // value of T
  constexpr int kTile = 64 * kUnroll;
  for (int v0 = wv * kTile; v0 < nv; v0 += kWaves * kTile) {  // uniform
    u32x4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = v0 + 64 * u + lane;
      raw[u] = v < nv ? ldg16(base + (int64_t)v * 16) : u32x4{0u, 0u, 0u, 0u};
    }
    const bool edge = v0 == 0 || v0 + kTile >= nv;  // uniform: values outside the row
    auto value = [&](int u, int i) {
      const float f = X::at(raw[u], i);
      if (!edge) return f;
      const int64_t id = (int64_t)(v0 + 64 * u + lane) * PER + i - lead;
      return id >= 0 && id < a.V ? f : -INFINITY;
    };
    auto key = [&](int u, int i) -> uint64_t {
      const int64_t id = (int64_t)(v0 + 64 * u + lane) * PER + i - lead;
      return id >= 0 && id < a.V ? key_of(X::at(raw[u], i), (int)id) : 0;
    };
    float tmax[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float f[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) f[i] = value(u, i);
      float t = f[0];
#pragma unroll
      for (int i = 1; i < PER; ++i) t = max_nan(t, f[i]);
      tmax[u] = t;
      const float mn = max_nan(p.m, t);
      if (__any(mn != p.m)) {  // (NaN too)
        const float d = p.m - mn;
        const double alpha = __builtin_amdgcn_exp2f(d * kLog2e);
        p.s = alpha * (p.s + p.z * (double)fmaxf(d, -1e30f));
        p.z *= alpha;
        p.m = mn;
      }
      float z = 0.f, s = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const float d = f[i] - p.m;
        const float e = __builtin_amdgcn_exp2f(d * kLog2e);
        z += e;
        s = fmaf(e, fmaxf(d, -1e30f), s);  // (0 for -infinity)
      }
      p.z += (double)z;
      p.s += (double)s;
    }
    if (a.k > 0) {  // uniform
      if (list.T == 0) {
        uint64_t most = 0;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
          for (int i = 0; i < PER; ++i) most = max(most, key(u, i));
        list.T = kth_of_lanes(most, a.k);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (!__any(!(tmax[u] < limit))) continue;
#pragma unroll
        for (int i = 0; i < PER; ++i) list.push(key(u, i), a.k, lane);
      }
      if (list.T != 0) limit = value_of(list.T);
    }
  }

  // the wavefront's sums, then the block's
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    p.add(__shfl_xor(p.m, o), __shfl_xor(p.z, o), __shfl_xor(p.s, o));
  if (a.k > 0) list.cut(a.k, lane);
  if (lane == 0) {
    s_m[wv] = p.m;
    s_z[wv] = p.z;
    s_s[wv] = p.s;
    s_n[wv] = list.n;
  }
  __syncthreads();
  p = {s_m[0], s_z[0], s_s[0]};
#pragma unroll
  for (int w = 1; w < kWaves; ++w) p.add(s_m[w], s_z[w], s_s[w]);
  const double lz = log(p.z);
  if (threadIdx.x == 0) {
    const int64_t t = a.tokens[row];
    a.lp[row] = t >= 0 && t < a.V ? (float)((double)X::one(x, t) - (double)p.m - lz) : 0.f;
    a.ent[row] = (float)(lz - p.s / p.z);
  }
  if (a.k == 0) return;
  // the k largest of the wavefronts' lists: a key's place is the number of
  // larger ones
  for (int i = lane; i < s_n[wv]; i += 64) {
    const uint64_t v = s_keys[wv][i];
    int place = i;
    for (int w = 0; w < kWaves; ++w) {
      if (w == wv) continue;
      for (int j = 0; j < s_n[w]; ++j) place += s_keys[w][j] > v;
    }
    if (place < a.k) {
      a.ids[row * a.k + place] = id_of(v);
      a.top[row * a.k + place] = (float)((double)value_of(v) - (double)p.m - lz);
    }
  }
}

template <int DT>
void launch_logprobs(const LogprobArgs &a, hipStream_t st) {
  hipLaunchKernelGGL(token_logprobs_kernel<DT>, dim3((unsigned)a.N), dim3(64 * kWaves), 0, st, a);
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
  *bytes = 0;
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
  const LogprobArgs a = {logits, N, ld, (int)V, top_k, tokens, logprobs, entropy, top_ids,
                         top_logprobs};
  hipStream_t st = (hipStream_t)stream;
  (void)workspace;
  (void)workspace_bytes;
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
