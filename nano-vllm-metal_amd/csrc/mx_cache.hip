// The 4-bit KV cache: keys and values into their slots, and back (declared in
// include/nvm_mx_cache.h).
//
// qk_norm_rope_store_mx_kernel: a head's row per group of GL lanes (a power of
//   two, eight values a lane; groups of D / 8 < GL lanes leave the rest idle).
//   A lane takes its partner's values (elements i and i + D/2 sit D / 16 lanes
//   apart) as they were read, so one exchange of four dwords serves norm and
//   rotation; four neighbouring lanes hold a block, whose largest magnitude is
//   two quad swaps away.  Keys are float64 up to their codes: a value next to a
//   rounding border of E2M1 is a quarter of itself off if it falls on the wrong
//   side, and float32 sums in another order put one in some 10^5 there.  That
//   concerns Hkv of the Hq + 2 Hkv heads.
// paged_kv_read_mx_kernel: eight values a lane (4096 rows of 4 heads of 128: 4.3 us,
//   2.4 TB/s, of which the launch is 1.4; a dword of codes a lane keeps it from more).
#include <math.h>

#include "common.h"
#include "internal.h"
#include "mx_common.h"
#include "nvm_mx_cache.h"

namespace nvm {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxThreads = 0xFFFFFFFFll - kThreads + 1;  // of a launch: below 2^32
constexpr int kMaxD = 256;

struct StoreArgs {
  const uint16_t *qkv, *qw, *kw;
  const int32_t *pos, *pages, *slots;
  const float *cos, *sin;
  uint32_t *kc, *vc;
  uint8_t *ks, *vs;
  void *q_out, *k_out, *v_out;
  uint32_t items;  // T * (ceil(Hq / U) + 2 Hkv)
  int Hq, Hkv, D, max_pos, P, page_size;
  float eps;
};

template <int GL>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int x = 1; x < GL; x <<= 1) v += __shfl_xor(v, x);
  return v;
}
template <int GL>
__device__ __forceinline__ double group_sum(double v) {
#pragma unroll
  for (int x = 1; x < GL; x <<= 1) v += __shfl_xor(v, x);
  return v;
}

// Eight values as they leave: rounded to the activation dtype, stored in it or
// in float32.
template <int DT, bool F32>
__device__ __forceinline__ void store8(void *out, int64_t i, const float (&v)[8]) {
  using A = Act<DT>;
  u32x4 o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = A::pack2(v[2 * j], v[2 * j + 1]);
  if constexpr (F32) {
    float *f = (float *)out + i;
    *(f32x4 *)f = f32x4{A::lo(o[0]), A::hi(o[0]), A::lo(o[1]), A::hi(o[1])};
    *(f32x4 *)(f + 4) = f32x4{A::lo(o[2]), A::hi(o[2]), A::lo(o[3]), A::hi(o[3])};
  } else {
    *(u32x4 *)((uint16_t *)out + i) = o;
  }
}

// 1 / sqrt(m), from v_rsq_f64's 2^-14 or better to float64 in two steps (an
// infinite m keeps the instruction's zero).
__device__ __forceinline__ double rsqrt_f64(double m) {
  double r = __builtin_amdgcn_rsq(m);
  if (m < INFINITY) {
#pragma unroll
    for (int i = 0; i < 2; ++i) r = r * fma(-0.5 * m * r, r, 1.5);
  }
  return r;
}

// Norm and rotation of a lane's eight values x with their partners p, in F
// (float or double).
template <class F, int GL, int DT>
__device__ __forceinline__ void norm_rope(u32x4 x, u32x4 p, u32x4 wx, u32x4 wp, bool first, int D,
                                          float eps, const float (&c)[8], const float (&s)[8],
                                          F (&o)[8]) {
  using A = Act<DT>;
  auto el = [](u32x4 v, int j) { return (F)((j & 1) ? A::hi(v[j >> 1]) : A::lo(v[j >> 1])); };
  F ss = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss += el(x, j) * el(x, j);
  ss = group_sum<GL>(ss);
  F inv;
  if constexpr (sizeof(F) == 8)
    inv = rsqrt_f64(ss / (F)D + (F)eps);
  else
    inv = rsqrtf(ss / (F)D + eps);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const F y = el(x, j) * inv * el(wx, j), z = el(p, j) * inv * el(wp, j);
    // first half: y cos - z sin; second: y cos + z sin
    o[j] = y * (F)c[j] + (first ? -z : z) * (F)s[j];
  }
}

// Items of a token: U query heads each (the last may be fewer), then a key or a
// value head each.  Bound: for one token the launch and one load's latency, 2 us;
// for 4096 of 32/4 heads of 128 the 80 MB read and written, 20 us, 4.0 TB/s, and with
// keys and values handed on and all of it in float32 (a prompt's first pass) 130 MB,
// 29.4 us, 4.4 TB/s.  (Loads with the non-temporal hint: 25.4 -> 24.3 us with the read
// of the rows.)
template <int DT, bool F32, int GL, int U>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_store_mx_kernel(StoreArgs a) {
  using A = Act<DT>;
  const uint32_t item = (blockIdx.x * kThreads + threadIdx.x) / GL;
  if (item >= a.items) return;
  const int QI = (a.Hq + U - 1) / U, NI = QI + 2 * a.Hkv, D = a.D;
  const int lane = threadIdx.x & (GL - 1), n8 = D / 8, half = D / 2, Q = n8 / 2;
  const uint32_t t = item / (uint32_t)NI;
  const int r = (int)(item - t * (uint32_t)NI);
  const bool on = lane < n8;
  const bool is_q = r < QI, is_v = r >= QI + a.Hkv;
  const int head = is_q ? r * U : a.Hq + r - QI;
  const int kvh = is_v ? r - QI - a.Hkv : r - QI;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  const uint16_t *src = a.qkv + ((int64_t)t * (a.Hq + 2 * a.Hkv) + head) * D + 8 * lane;
  const bool first = lane < Q;
  const int mate = first ? lane + Q : lane - Q;
  // norm weights and angles of a lane's eight values
  u32x4 wx = zero, wp = zero;
  float c[8], s[8];
  auto operands = [&]() {
    const uint16_t *w = is_q ? a.qw : a.kw;
    wx = on ? ldg16(w + 8 * lane) : zero, wp = on ? ldg16(w + 8 * mate) : zero;
    const int p = min(max(a.pos[t], 0), a.max_pos - 1);
    const int64_t at = (int64_t)p * half + 8 * (first ? lane : mate);
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
      const f32x4 cv = on ? *(const f32x4 *)(a.cos + at + j) : z;
      const f32x4 sv = on ? *(const f32x4 *)(a.sin + at + j) : z;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[j + i] = cv[i];
        s[j + i] = sv[i];
      }
    }
  };
  auto partner = [&](u32x4 v) {
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (uint32_t)__shfl((int)v[j], on ? mate : lane, GL);
    return o;
  };
  if (is_q) {
    u32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = on && head + u < a.Hq ? ldg16_once(src + u * D) : zero;
    operands();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float out[8];
      norm_rope<float, GL, DT>(x[u], partner(x[u]), wx, wp, first, D, a.eps, c, s, out);
      if (on && head + u < a.Hq)
        store8<DT, F32>(a.q_out, ((int64_t)t * a.Hq + head + u) * D + 8 * lane, out);
    }
    return;
  }
  const u32x4 x = on ? ldg16(src) : zero;
  const int pg = a.pages[t], slot = a.slots[t];
  const bool there = pg >= 0 && pg < a.P && slot >= 0 && slot < a.page_size;
  const int64_t row = ((int64_t)pg * a.Hkv + kvh) * a.page_size + slot;
  float out[8];
  if (is_v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      out[2 * j] = A::lo(x[j]);
      out[2 * j + 1] = A::hi(x[j]);
    }
  } else {
    operands();
    double o[8];
    norm_rope<double, GL, DT>(x, partner(x), wx, wp, first, D, a.eps, c, s, o);
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = round_to_odd(o[j]);
  }
  // (the block's four lanes are on or off together)
  if (!on) return;
  uint32_t m = absmax8(out);
  m = max(m, dpp_u32<0xB1>(m));
  m = max(m, dpp_u32<0x4E>(m));
  const uint32_t b = mx_scale_byte<NVM_MX_FP4>(m);
  const uint32_t code = mx_encode8<NVM_MX_FP4>(out, mx_factor(b), b == 255u).x;
  if (there) {
    (is_v ? a.vc : a.kc)[row * n8 + lane] = code;
    if ((lane & 3) == 0) (is_v ? a.vs : a.ks)[row * (D / 32) + (lane >> 2)] = (uint8_t)b;
  }
  void *f = is_v ? a.v_out : a.k_out;
  if (f) store8<DT, F32>(f, ((int64_t)t * a.Hkv + kvh) * D + 8 * lane, out);
}

struct ReadArgs {
  const uint32_t *kc, *vc;
  const uint8_t *ks, *vs;
  const int32_t *pages, *slots;
  void *k_out, *v_out;
  uint32_t items;  // chunks of eight values of keys: T * Hkv * D / 8
  int Hkv, n8, P, page_size;
};

// Keys by the first half of the grid's y, values by the second.
template <int DT>
__global__ __launch_bounds__(kThreads) void paged_kv_read_mx_kernel(ReadArgs a) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.items) return;
  const uint32_t r = i / (uint32_t)a.n8;  // (token, head)
  const int c = (int)(i - r * (uint32_t)a.n8);
  const uint32_t t = r / (uint32_t)a.Hkv;
  const int h = (int)(r - t * (uint32_t)a.Hkv);
  const bool vals = blockIdx.y;
  const int pg = a.pages[t], slot = a.slots[t];
  uint32_t d = 0;
  float s = 0.f;
  if (pg >= 0 && pg < a.P && slot >= 0 && slot < a.page_size) {
    const int64_t row = ((int64_t)pg * a.Hkv + h) * a.page_size + slot;
    d = (vals ? a.vc : a.kc)[row * a.n8 + c];
    s = mx_scale((vals ? a.vs : a.ks)[row * (a.n8 / 4) + (c >> 2)]);
  }
  const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 0);
  const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 1);
  const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 2);
  const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, 1.0f, 3);
  const float v[8] = {p0.x * s, p0.y * s, p1.x * s, p1.y * s,
                      p2.x * s, p2.y * s, p3.x * s, p3.y * s};
  void *out = vals ? a.v_out : a.k_out;
  if constexpr (DT == NVM_KV_F32) {
    float *o = (float *)out + 8 * (int64_t)i;
    *(f32x4 *)o = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4 *)(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    store8<DT, false>(out, 8 * (int64_t)i, v);
  }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int mx_check_pages(const char *op, int Hkv, int64_t D, int64_t P, int64_t page_size,
                   const void *kc, const void *ks, const void *vc, const void *vs) {
  if (Hkv <= 0 || D <= 0 || P <= 0 || page_size <= 0)
    return set_error(NVM_ERR_INVALID, "%s: bad pages: P=%lld Hkv=%d page_size=%lld D=%lld", op,
                     (long long)P, Hkv, (long long)page_size, (long long)D);
  if (D % 32 || D > kMaxD)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: head dim %lld must be a multiple of 32, at most %d",
                     op, (long long)D, kMaxD);
  // (rows have 32-bit numbers, their bytes 64-bit addresses: at D = 128 2^31 rows
  // are 128 GiB of codes)
  if (page_size > INT32_MAX || P > INT32_MAX / Hkv / page_size)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: pool too large", op);
  if (!kc || !ks || !vc || !vs) return set_error(NVM_ERR_INVALID, "%s: null page pointer", op);
  if (!aligned16(kc) || !aligned16(ks) || !aligned16(vc) || !aligned16(vs))
    return set_error(NVM_ERR_INVALID, "%s: codes and scales must be 16-byte aligned", op);
  return NVM_OK;
}

}  // namespace nvm

extern "C" {

int nvm_qk_norm_rope_store_mx(const void *qkv, int64_t T, int Hq, int Hkv, int64_t D,
                              const void *q_norm_w, const void *k_norm_w, float eps,
                              const int32_t *positions, const float *cos, const float *sin,
                              int64_t max_pos, const int32_t *page_ids, const int32_t *slots,
                              void *key_codes, uint8_t *key_scales, void *value_codes,
                              uint8_t *value_scales, int64_t P, int64_t page_size, int dtype,
                              int out_dtype, void *q_out, void *k_out, void *v_out,
                              nvm_stream_t stream) {
  using namespace nvm;
  constexpr const char *op = "qk_norm_rope_store_mx";
  if (dtype != NVM_DTYPE_F16 && dtype != NVM_DTYPE_BF16)
    return set_error(NVM_ERR_INVALID, "%s: dtype must be f16 or bf16", op);
  if (out_dtype != NVM_KV_F32 && out_dtype != dtype)
    return set_error(NVM_ERR_INVALID, "%s: out dtype must be f32 or that of qkv", op);
  if (T < 0 || Hq <= 0 || max_pos <= 0)
    return set_error(NVM_ERR_INVALID, "%s: bad shape T=%lld Hq=%d max_pos=%lld", op, (long long)T,
                     Hq, (long long)max_pos);
  if (int rc = mx_check_pages(op, Hkv, D, P, page_size, key_codes, key_scales, value_codes,
                              value_scales))
    return rc;
  if (max_pos > INT32_MAX || Hq > (1 << 20) || Hkv > (1 << 20))
    return set_error(NVM_ERR_UNSUPPORTED, "%s: too many heads or positions", op);
  int gl = 4;
  while (8 * gl < D) gl *= 2;
  const int64_t NH = (int64_t)Hq + 2 * Hkv;
  if (T > kMaxThreads / gl / NH)
    return set_error(NVM_ERR_UNSUPPORTED, "%s: %lld tokens of %lld heads are too many for a launch",
                     op, (long long)T, (long long)NH);
  if (T == 0) return NVM_OK;
  if (!qkv || !q_norm_w || !k_norm_w || !positions || !cos || !sin || !page_ids || !slots || !q_out)
    return set_error(NVM_ERR_INVALID, "%s: null pointer", op);
  if (!aligned16(qkv) || !aligned16(q_norm_w) || !aligned16(k_norm_w) || !aligned16(cos) ||
      !aligned16(sin) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(v_out))
    return set_error(NVM_ERR_INVALID, "%s: operands must be 16-byte aligned", op);
  StoreArgs a{};
  a.qkv = (const uint16_t *)qkv;
  a.qw = (const uint16_t *)q_norm_w;
  a.kw = (const uint16_t *)k_norm_w;
  a.pos = positions;
  a.pages = page_ids;
  a.slots = slots;
  a.cos = cos;
  a.sin = sin;
  a.kc = (uint32_t *)key_codes;
  a.vc = (uint32_t *)value_codes;
  a.ks = key_scales;
  a.vs = value_scales;
  a.q_out = q_out;
  a.k_out = k_out;
  a.v_out = v_out;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.D = (int)D;
  a.max_pos = (int)max_pos;
  a.P = (int)P;
  a.page_size = (int)page_size;
  a.eps = eps;
  // four query heads a group from eight wavefronts a SIMD on (with the read of the
  // rows: 4096 tokens of 32/4 heads of 128 28.4 us by one, 25.4 by four; 1024 11.7
  // and 10.3; fewer leave CUs idle)
  const int U = T * NH * gl >= (int64_t)8 * 64 * 4 * cu_count() ? 4 : 1;
  a.items = (uint32_t)(T * ((Hq + U - 1) / U + 2 * Hkv));
  const unsigned grid = (unsigned)(((int64_t)a.items * gl + kThreads - 1) / kThreads);
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3(grid), dim3(kThreads), 0, st, a); };
  auto by_gl = [&](auto dt, auto f32) {
    constexpr int DT = decltype(dt)::value;
    constexpr bool F32 = decltype(f32)::value;
    auto by_u = [&](auto g) {
      constexpr int GL = decltype(g)::value;
      U == 4 ? go(qk_norm_rope_store_mx_kernel<DT, F32, GL, 4>)
             : go(qk_norm_rope_store_mx_kernel<DT, F32, GL, 1>);
    };
    switch (gl) {
      case 4: return by_u(MxInt<4>{});
      case 8: return by_u(MxInt<8>{});
      case 16: return by_u(MxInt<16>{});
      default: return by_u(MxInt<32>{});
    }
  };
  const bool f32 = out_dtype == NVM_KV_F32;
  if (dtype == NVM_DTYPE_BF16)
    f32 ? by_gl(MxInt<DT_BF16>{}, MxInt<1>{}) : by_gl(MxInt<DT_BF16>{}, MxInt<0>{});
  else
    f32 ? by_gl(MxInt<DT_F16>{}, MxInt<1>{}) : by_gl(MxInt<DT_F16>{}, MxInt<0>{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

int nvm_paged_kv_read_mx(const void *key_codes, const uint8_t *key_scales,
                         const void *value_codes, const uint8_t *value_scales, int64_t P, int Hkv,
                         int64_t page_size, int64_t D, const int32_t *page_ids,
                         const int32_t *slots, int64_t T, int out_dtype, void *k_out, void *v_out,
                         nvm_stream_t stream) {
  using namespace nvm;
  constexpr const char *op = "paged_kv_read_mx";
  if (out_dtype != NVM_KV_F16 && out_dtype != NVM_KV_BF16 && out_dtype != NVM_KV_F32)
    return set_error(NVM_ERR_INVALID, "%s: out dtype must be f16, bf16 or f32", op);
  if (int rc = mx_check_pages(op, Hkv, D, P, page_size, key_codes, key_scales, value_codes,
                              value_scales))
    return rc;
  if (T < 0) return set_error(NVM_ERR_INVALID, "%s: bad shape T=%lld", op, (long long)T);
  if (T > kMaxThreads / Hkv / (D / 8))
    return set_error(NVM_ERR_UNSUPPORTED, "%s: %lld rows are too many for a launch", op,
                     (long long)T);
  if (T == 0) return NVM_OK;
  if (!page_ids || !slots || !k_out || !v_out)
    return set_error(NVM_ERR_INVALID, "%s: null pointer", op);
  if (!aligned16(k_out) || !aligned16(v_out))
    return set_error(NVM_ERR_INVALID, "%s: outputs must be 16-byte aligned", op);
  ReadArgs a{};
  a.kc = (const uint32_t *)key_codes;
  a.vc = (const uint32_t *)value_codes;
  a.ks = key_scales;
  a.vs = value_scales;
  a.pages = page_ids;
  a.slots = slots;
  a.k_out = k_out;
  a.v_out = v_out;
  a.items = (uint32_t)(T * Hkv * (D / 8));
  a.Hkv = Hkv;
  a.n8 = (int)(D / 8);
  a.P = (int)P;
  a.page_size = (int)page_size;
  const dim3 grid((a.items + kThreads - 1) / kThreads, 2);
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(kThreads), 0, st, a); };
  if (out_dtype == NVM_KV_F32)
    go(paged_kv_read_mx_kernel<NVM_KV_F32>);
  else if (out_dtype == NVM_KV_BF16)
    go(paged_kv_read_mx_kernel<NVM_KV_BF16>);
  else
    go(paged_kv_read_mx_kernel<NVM_KV_F16>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(NVM_ERR_HIP, "%s: %s", op, hipGetErrorString(e));
  return NVM_OK;
}

}  // extern "C"
