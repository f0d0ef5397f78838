// Element-wise parts shared by the GEMM epilogue, its backward and the stand-alone dropout: the
// activations with their derivatives and counter-based dropout.  Everything is fp32; callers round
// once, where they store.
#pragma once

#include "common.cuh"
#include "../../include/radiance_nvfp4.h"

namespace rb {

// ---------------------------------------------------------------------------------------------
// Dropout
// ---------------------------------------------------------------------------------------------

// Element i of a tensor (its row-major index) takes the 16-bit half i % 2 of word (i % 8) / 2 of
// Philox4x32-10 (J. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with
// counter (i / 8, 0) and the 64-bit seed as key, and is dropped when that draw is below `threshold`.
// So the mask is a function of (seed, index) alone: the GEMM epilogue, the stand-alone kernel and
// both backward passes regenerate the same one, and nothing stores it.
// 16-bit draws: one generator call (20 wide multiplies) serves eight elements, one 16-byte vector
// of bf16.  They resolve p to 2^-16; kept elements are scaled by 65536 / (65536 - threshold), the
// reciprocal of the probability that is really used, so the expectation is exact.
struct DropoutArgs {
  const int64_t* seed;  // device; nullptr: no dropout
  uint32_t below;       // threshold * 2^16 - 1: a draw in the upper half of a word stays when the word is above it
  float scale;
};

// The ten rounds' keys, which depend on the seed alone.
struct PhiloxKeys {
  uint32_t k0[10], k1[10];
};

__device__ __forceinline__ PhiloxKeys philox_keys(const int64_t* seed) {
  PhiloxKeys k;
  const uint64_t s = seed != nullptr ? static_cast<uint64_t>(__ldg(reinterpret_cast<const long long*>(seed))) : 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    k.k0[r] = static_cast<uint32_t>(s) + r * 0x9E3779B9u;
    k.k1[r] = static_cast<uint32_t>(s >> 32) + r * 0xBB67AE85u;
  }
  return k;
}

__device__ __forceinline__ uint4 philox(uint64_t counter, const PhiloxKeys& key) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32), c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ key.k0[r];
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ key.k1[r];
    c3 = static_cast<uint32_t>(a);
  }
  return make_uint4(c0, c1, c2, c3);
}

// Drops from the eight elements 8 * group .. 8 * group + 7.  A dropped element is 0 whatever it
// held, infinities and NaN included.
__device__ __forceinline__ void dropout8(float2 (&v)[4], uint64_t group, const PhiloxKeys& key, uint32_t below,
                                         float scale) {
  const uint4 d = philox(group, key);
  const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j].x = (w[j] << 16) > below ? v[j].x * scale : 0.0f;
    v[j].y = w[j] > below ? v[j].y * scale : 0.0f;
  }
}

// One element, at any index.
__device__ __forceinline__ float dropout1(float v, uint64_t index, const PhiloxKeys& key, uint32_t below,
                                          float scale) {
  const uint4 d = philox(index >> 3, key);
  const uint32_t j = static_cast<uint32_t>(index) & 7u;
  const uint32_t lo = (j & 2) ? d.y : d.x, hi = (j & 2) ? d.w : d.z;
  const uint32_t w = (j & 4) ? hi : lo;
  return ((j & 1) ? w : w << 16) > below ? v * scale : 0.0f;
}

// ---------------------------------------------------------------------------------------------
// Activations (RB_ACT_*), two elements at a time on the packed fp32 pipe
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float rcp_approx(float x) {  // within 1 ulp; inf -> 0
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float ex2_approx(float x) {  // within 2 ulp; large x -> inf, large -x -> 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 relu2(float2 z) { return make_float2(max_nan(z.x, 0.0f), max_nan(z.y, 0.0f)); }
__device__ __forceinline__ float2 rcp2(float2 x) { return make_float2(rcp_approx(x.x), rcp_approx(x.y)); }
__device__ __forceinline__ float2 ex2_2(float2 x) { return make_float2(ex2_approx(x.x), ex2_approx(x.y)); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluA = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

// silu(z) = z / (1 + 2^x) for x = -log2(e) z, and the tanh form of GELU, 0.5 z (1 + tanh u) = z / (1 + exp(-2u)),
// is the same with another x: one exponential, and no cancellation where tanh nears -1.
__device__ __forceinline__ float2 silu_exponent(float2 z) { return __fmul2_rn(z, both(-kLog2e)); }
__device__ __forceinline__ float2 gelu_tanh_exponent(float2 z) {
  return __fmul2_rn(z, __ffma2_rn(__fmul2_rn(z, z), both(-kLog2e * kGeluA * kGeluB), both(-kLog2e * kGeluA)));
}
__device__ __forceinline__ float2 logistic2(float2 x) { return rcp2(__fadd2_rn(ex2_2(x), both(1.0f))); }

// The normal distribution's tail q = Phi(-|z|) = erfc(|z| / sqrt 2) / 2 and e = exp(-z^2 / 2), by
// Hastings' formula (C. Hastings, "Approximations for Digital Computers", 1955, sheet 45; 7.1.26 of
// Abramowitz and Stegun): erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2), t = 1 / (1 + p x), within
// 1.5e-7 for x >= 0.  Halved here.  One exponential and half a reciprocal, with e shared by the derivative, where
// erff takes a branch and some 25 instructions more.  `nz` is -|z| held above -128, where q is 0; for a NaN it is
// -128, and the NaN comes through e.
// kN pairs are taken through it step by step, which overlaps their latencies.
template <int kN>
struct NormalTail {
  float2 nz[kN], q[kN], e[kN];
};
template <int kN>
__device__ __forceinline__ NormalTail<kN> normal_tail(const float2* z) {
  NormalTail<kN> n;
  float2 t[kN], p[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    n.nz[i] = make_float2(fmaxf(-fabsf(z[i].x), -128.0f), fmaxf(-fabsf(z[i].y), -128.0f));
    t[i] = __ffma2_rn(n.nz[i], both(-0.3275911f * 0.70710678118654752f), both(1.0f));
  }
  // One reciprocal for the pair, that of the product (both factors lie in 1 .. 31): the special-function unit
  // takes 8 cycles a warp for each, and bounds this formula otherwise.
#pragma unroll
  for (int i = 0; i < kN; ++i) p[i].x = rcp_approx(t[i].x * t[i].y);
#pragma unroll
  for (int i = 0; i < kN; ++i) t[i] = __fmul2_rn(both(p[i].x), make_float2(t[i].y, t[i].x));
#pragma unroll
  for (int i = 0; i < kN; ++i) n.e[i] = __fmul2_rn(z[i], __fmul2_rn(z[i], both(-0.5f * kLog2e)));
#pragma unroll
  for (int i = 0; i < kN; ++i) n.e[i] = ex2_2(n.e[i]);
#pragma unroll
  for (int i = 0; i < kN; ++i) p[i] = __ffma2_rn(t[i], both(0.5f * 1.061405429f), both(0.5f * -1.453152027f));
#pragma unroll
  for (int i = 0; i < kN; ++i) p[i] = __ffma2_rn(t[i], p[i], both(0.5f * 1.421413741f));
#pragma unroll
  for (int i = 0; i < kN; ++i) p[i] = __ffma2_rn(t[i], p[i], both(0.5f * -0.284496736f));
#pragma unroll
  for (int i = 0; i < kN; ++i) p[i] = __ffma2_rn(t[i], p[i], both(0.5f * 0.254829592f));
#pragma unroll
  for (int i = 0; i < kN; ++i) n.q[i] = __fmul2_rn(__fmul2_rn(t[i], p[i]), n.e[i]);
  return n;
}

// kN pairs through the activation, in place.
template <int kAct, int kN>
__device__ __forceinline__ void act_batch(float2* v) {
  if constexpr (kAct == RB_ACT_RELU || kAct == RB_ACT_RELU2) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      v[i] = relu2(v[i]);
      if constexpr (kAct == RB_ACT_RELU2) v[i] = __fmul2_rn(v[i], v[i]);
    }
  } else if constexpr (kAct == RB_ACT_GELU) {  // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    const NormalTail<kN> n = normal_tail<kN>(v);
#pragma unroll
    for (int i = 0; i < kN; ++i)
      v[i] = __ffma2_rn(n.nz[i], n.q[i], make_float2(fmaxf(v[i].x, 0.0f), fmaxf(v[i].y, 0.0f)));
  } else if constexpr (kAct == RB_ACT_SILU || kAct == RB_ACT_GELU_TANH) {
    float2 s[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) s[i] = ex2_2(kAct == RB_ACT_SILU ? silu_exponent(v[i]) : gelu_tanh_exponent(v[i]));
#pragma unroll
    for (int i = 0; i < kN; ++i) s[i] = rcp2(__fadd2_rn(s[i], both(1.0f)));
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = __fmul2_rn(v[i], s[i]);
  }
}

template <int kAct>
__device__ __forceinline__ float2 act_derivative2(float2 z) {
  if constexpr (kAct == RB_ACT_RELU)
    return make_float2(z.x <= 0.0f ? 0.0f : (z.x != z.x ? z.x : 1.0f), z.y <= 0.0f ? 0.0f : (z.y != z.y ? z.y : 1.0f));
  else if constexpr (kAct == RB_ACT_RELU2)
    return make_float2(z.x <= 0.0f ? 0.0f : z.x + z.x, z.y <= 0.0f ? 0.0f : z.y + z.y);
  else if constexpr (kAct == RB_ACT_SILU) {
    const float2 s = logistic2(silu_exponent(z));
    return __fmul2_rn(s, __ffma2_rn(z, __ffma2_rn(s, both(-1.0f), both(1.0f)), both(1.0f)));
  } else if constexpr (kAct == RB_ACT_GELU) {
    const NormalTail<1> n = normal_tail<1>(&z);
    const float2 up = __ffma2_rn(n.q[0], both(-1.0f), both(1.0f));
    const float2 phi = make_float2(z.x < 0.0f ? n.q[0].x : up.x, z.y < 0.0f ? n.q[0].y : up.y);
    return __ffma2_rn(__fmul2_rn(z, both(kInvSqrt2Pi)), n.e[0], phi);
  } else if constexpr (kAct == RB_ACT_GELU_TANH) {
    const float2 s = logistic2(gelu_tanh_exponent(z));
    const float2 t = __fmul2_rn(s, __ffma2_rn(s, both(-1.0f), both(1.0f)));
    const float2 du = __ffma2_rn(__fmul2_rn(z, z), both(3.0f * kGeluA * kGeluB), both(kGeluA));
    const float2 d = __ffma2_rn(__fmul2_rn(z, t), du, s);
    return make_float2(t.x > 0.0f ? d.x : s.x, t.y > 0.0f ? d.y : s.y);  // t = 0 wherever du can overflow
  } else return both(1.0f);
}

// ---------------------------------------------------------------------------------------------
// Eight elements of a row to and from fp32
// ---------------------------------------------------------------------------------------------
template <typename T>
struct Io;

template <>
struct Io<__nv_bfloat16> {
  // Returns the largest magnitude stored, as fp32 bits (NaN above infinity).
  static __device__ __forceinline__ uint32_t store8(__nv_bfloat16* p, const float2 (&v)[4]) {
    uint32_t w[4], m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 b = __float22bfloat162_rn(v[j]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
      m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    return max(m << 16, m & 0xFFFF0000u);
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ uint32_t store(__nv_bfloat16* p, float v) {
    const __nv_bfloat16 b = __float2bfloat16_rn(v);
    *p = b;
    return __float_as_uint(__bfloat162float(b)) & 0x7FFFFFFFu;
  }
};

template <>
struct Io<float> {
  static __device__ __forceinline__ uint32_t store8(float* p, const float2 (&v)[4]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      m = max(m, max(__float_as_uint(v[j].x) & 0x7FFFFFFFu, __float_as_uint(v[j].y) & 0x7FFFFFFFu));
    return m;
  }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ uint32_t store(float* p, float v) {
    *p = v;
    return __float_as_uint(v) & 0x7FFFFFFFu;
  }
};

}  // namespace rb

namespace rb_host {

// Device arguments of dropout with probability p (0 <= p <= 1, checked by the caller) and a device seed.
inline rb::DropoutArgs dropout_args(double p, const int64_t* seed) {
  rb::DropoutArgs d;
  const uint32_t threshold = static_cast<uint32_t>(p * 65536.0 + 0.5);
  d.below = (threshold << 16) - 1u;  // 65536 (everything dropped): above every draw
  d.scale = threshold < 65536u ? static_cast<float>(65536.0 / (65536.0 - threshold)) : 0.0f;
  d.seed = threshold > 0 ? seed : nullptr;
  return d;
}

}  // namespace rb_host
