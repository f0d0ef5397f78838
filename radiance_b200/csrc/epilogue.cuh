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

constexpr float kLog2eLo = 1.9259630e-8f;  // log2(e) - kLog2e
constexpr float kLn2 = 0.69314718055994531f;

// kExact, here and below: for fp32 tensors, within a few 2^-23 of the function.  Without it, for results that are
// rounded to bf16, a step of 2^-8, the shorter forms.

// silu(z) = z / (1 + 2^x) for x = -log2(e) z, and the tanh form of GELU, 0.5 z (1 + tanh u) = z / (1 + exp(-2u)),
// is the same with x = z (kTanh3 z^2 + kTanh1): one exponential, and no cancellation where tanh nears -1.
// This is 2^x.  kExact: times 1 + ln(2) lo, lo what the roundings of x left out: they are 2^-24 of x, not of the
// result.  Past 2^126, where 1 / (1 + 2^x) is no normal number, and for infinities, the factor is left off.
constexpr float kTanh1 = -2.302208185195923f, kTanh1Lo = -1.2948402e-8f;   // their sum: -log2(e) 2 sqrt(2 / pi)
constexpr float kTanh3 = -0.10294324159622192f, kTanh3Lo = 2.0161985e-9f;  // and that times 0.044715
template <int kAct, bool kExact>
__device__ __forceinline__ float2 logistic_power(float2 z) {
  float2 x, lo = both(0.0f);
  if constexpr (kAct == RB_ACT_SILU) {
    x = __fmul2_rn(z, both(-kLog2e));
    if constexpr (kExact) lo = __ffma2_rn(z, both(-kLog2eLo), __ffma2_rn(z, both(-kLog2e), make_float2(-x.x, -x.y)));
  } else if constexpr (!kExact) {
    x = __fmul2_rn(z, __ffma2_rn(__fmul2_rn(z, z), both(kTanh3), both(kTanh1)));
  } else {
    const float2 u = __fmul2_rn(z, z), ul = __ffma2_rn(z, z, make_float2(-u.x, -u.y));
    const float2 m = __fmul2_rn(u, both(kTanh3));
    float2 l = __ffma2_rn(u, both(kTanh3), make_float2(-m.x, -m.y));
    l = __fadd2_rn(l, __ffma2_rn(ul, both(kTanh3), __ffma2_rn(u, both(kTanh3Lo), both(kTanh1Lo))));
    // p = m + kTanh1 and what its rounding left out (D. Knuth's two-sum)
    const float2 p = __fadd2_rn(m, both(kTanh1)), q = make_float2(p.x - m.x, p.y - m.y);
    l.x += (m.x - (p.x - q.x)) + (kTanh1 - q.x);
    l.y += (m.y - (p.y - q.y)) + (kTanh1 - q.y);
    x = __fmul2_rn(z, p);
    lo = __ffma2_rn(z, l, __ffma2_rn(z, p, make_float2(-x.x, -x.y)));
  }
  const float2 e = ex2_2(x);
  if constexpr (!kExact) return e;
  const float2 f = __ffma2_rn(e, __fmul2_rn(lo, both(kLn2)), e);
  return make_float2(fabsf(x.x) < 126.0f ? f.x : e.x, fabsf(x.y) < 126.0f ? f.y : e.y);
}
// 1 - s for s = 1 / (1 + e).  kExact: e s where s is past 2/3 and 1 - s would cancel.
template <bool kExact>
__device__ __forceinline__ float2 one_minus(float2 s, float2 e) {
  const float2 d = __ffma2_rn(s, both(-1.0f), both(1.0f));
  if constexpr (!kExact) return d;
  const float2 f = __fmul2_rn(e, s);
  return make_float2(e.x < 0.5f ? f.x : d.x, e.y < 0.5f ? f.y : d.y);
}

// The normal distribution's tail q = Phi(-|z|) = erfc(|z| / sqrt 2) / 2 and e = exp(-z^2 / 2), as q = e t P(t),
// t = 1 / (1 + p |z|): t P(t) stands for the tail without its exponential, which falls slowly and as 1 / |z|.  p and
// P's coefficients are this project's own: weighted least squares on a grid of |z| in 0 .. 13.5, reweighted until the
// largest error is smallest, with the coefficients as fp32 holds them.  One exponential and half a reciprocal, with e
// shared by the derivative, where erff takes a branch and some 25 instructions more.  `nz` is -|z| held above -128,
// where q is 0.
// P of degree 5: q within 7.5e-8, and within 3.8e-4 of itself far out, a tenth of bf16's half step.
// kExact: P of degree 6, within 1.3e-7 of q where |z| >= 1 (below that, see act_batch), a reciprocal with a
// Newton step, and e times 1 + ln(2) (what rounding the exponent left out).
// kN pairs are taken through it step by step, which overlaps their latencies.
template <int kN>
struct NormalTail {
  float2 nz[kN], q[kN], e[kN];
};
__device__ __forceinline__ float min_nan(float x, float y) {  // NaN if either is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
template <bool kExact, int kN>
__device__ __forceinline__ NormalTail<kN> normal_tail(const float2* z) {
  NormalTail<kN> n;
  float2 t[kN], p[kN];
  if constexpr (kExact) {
    constexpr float kP = 0.39f, kC = -0.5f * kLog2e;
    constexpr float kCoef[7] = {0.06286511570215225f, -0.1864839494228363f, 0.12463319301605225f, 0.04984919726848602f,
                                0.13879886269569397f, 0.15486139059066772f, 0.15561912953853607f};
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      n.nz[i] = make_float2(-min_nan(fabsf(z[i].x), 128.0f), -min_nan(fabsf(z[i].y), 128.0f));
      t[i] = __ffma2_rn(n.nz[i], both(-kP), both(1.0f));
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float2 r = rcp2(t[i]);
      t[i] = __ffma2_rn(r, __ffma2_rn(make_float2(-t[i].x, -t[i].y), r, both(1.0f)), r);
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float2 a = n.nz[i], s = __fmul2_rn(a, a), x = __fmul2_rn(s, both(kC));
      const float2 sl = __ffma2_rn(a, a, make_float2(-s.x, -s.y));
      float2 lo = __ffma2_rn(s, both(kC), make_float2(-x.x, -x.y));
      lo = __fadd2_rn(lo, __ffma2_rn(s, both(-0.5f * kLog2eLo), __fmul2_rn(sl, both(kC))));
      const float2 e = ex2_2(x);
      n.e[i] = __ffma2_rn(e, __fmul2_rn(lo, both(kLn2)), e);
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) p[i] = __ffma2_rn(t[i], both(kCoef[0]), both(kCoef[1]));
#pragma unroll
    for (int k = 2; k < 7; ++k) {
#pragma unroll
      for (int i = 0; i < kN; ++i) p[i] = __ffma2_rn(t[i], p[i], both(kCoef[k]));
    }
  } else {
    constexpr float kP = 0.4f;
    constexpr float kCoef[6] = {0.05205557495355606f, -0.2375888079404831f, 0.3129570186138153f,
                                0.03388453274965286f, 0.18078862130641937f, 0.15790298581123352f};
#pragma unroll
    for (int i = 0; i < kN; ++i) {  // for a NaN nz is -128, and the NaN comes through e
      n.nz[i] = make_float2(fmaxf(-fabsf(z[i].x), -128.0f), fmaxf(-fabsf(z[i].y), -128.0f));
      t[i] = __ffma2_rn(n.nz[i], both(-kP), both(1.0f));
    }
    // One reciprocal for the pair, that of the product (both factors lie in 1 .. 53): the special-function unit
    // takes 8 cycles a warp for each.
#pragma unroll
    for (int i = 0; i < kN; ++i) p[i].x = rcp_approx(t[i].x * t[i].y);
#pragma unroll
    for (int i = 0; i < kN; ++i) t[i] = __fmul2_rn(both(p[i].x), make_float2(t[i].y, t[i].x));
#pragma unroll
    for (int i = 0; i < kN; ++i) n.e[i] = __fmul2_rn(z[i], __fmul2_rn(z[i], both(-0.5f * kLog2e)));
#pragma unroll
    for (int i = 0; i < kN; ++i) n.e[i] = ex2_2(n.e[i]);
#pragma unroll
    for (int i = 0; i < kN; ++i) p[i] = __ffma2_rn(t[i], both(kCoef[0]), both(kCoef[1]));
#pragma unroll
    for (int k = 2; k < 6; ++k) {
#pragma unroll
      for (int i = 0; i < kN; ++i) p[i] = __ffma2_rn(t[i], p[i], both(kCoef[k]));
    }
  }
#pragma unroll
  for (int i = 0; i < kN; ++i) n.q[i] = __fmul2_rn(__fmul2_rn(t[i], p[i]), n.e[i]);
  return n;
}

// Phi(z) for |z| < 1, as 1/2 + z B(z^2), within 2^-24: there z Phi(z) from the tail would carry the tail's error,
// 2^-24 of 1/2 and more, into every small z.  B's coefficients: as P's above.
__device__ __forceinline__ float2 normal_body(float2 z) {
  constexpr float kCoef[6] = {-7.590575933136279e-06f, 0.00011333930888213217f, -0.0011862121755257249f,
                              0.009973285719752312f, -0.06649035215377808f, 0.3989422917366028f};
  const float2 u = __fmul2_rn(z, z);
  float2 b = __ffma2_rn(u, both(kCoef[0]), both(kCoef[1]));
#pragma unroll
  for (int k = 2; k < 6; ++k) b = __ffma2_rn(u, b, both(kCoef[k]));
  return __ffma2_rn(z, b, both(0.5f));
}
__device__ __forceinline__ float2 near_zero(float2 z, float2 inside, float2 outside) {
  return make_float2(fabsf(z.x) < 1.0f ? inside.x : outside.x, fabsf(z.y) < 1.0f ? inside.y : outside.y);
}

// kN pairs through the activation, in place.
template <int kAct, bool kExact, int kN>
__device__ __forceinline__ void act_batch(float2* v) {
  if constexpr (kAct == RB_ACT_RELU || kAct == RB_ACT_RELU2) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      v[i] = relu2(v[i]);
      if constexpr (kAct == RB_ACT_RELU2) v[i] = __fmul2_rn(v[i], v[i]);
    }
  } else if constexpr (kAct == RB_ACT_GELU) {  // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    const NormalTail<kN> n = normal_tail<kExact, kN>(v);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float2 g = __ffma2_rn(n.nz[i], n.q[i], make_float2(fmaxf(v[i].x, 0.0f), fmaxf(v[i].y, 0.0f)));
      if constexpr (kExact) v[i] = near_zero(v[i], __fmul2_rn(v[i], normal_body(v[i])), g);
      else v[i] = g;
    }
  } else if constexpr (kAct == RB_ACT_SILU || kAct == RB_ACT_GELU_TANH) {
    float2 s[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) s[i] = logistic_power<kAct, kExact>(v[i]);
#pragma unroll
    for (int i = 0; i < kN; ++i) s[i] = rcp2(__fadd2_rn(s[i], both(1.0f)));
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = __fmul2_rn(v[i], s[i]);
  }
}

template <int kAct, bool kExact>
__device__ __forceinline__ float2 act_derivative2(float2 z) {
  if constexpr (kAct == RB_ACT_RELU)
    return make_float2(z.x <= 0.0f ? 0.0f : (z.x != z.x ? z.x : 1.0f), z.y <= 0.0f ? 0.0f : (z.y != z.y ? z.y : 1.0f));
  else if constexpr (kAct == RB_ACT_RELU2)
    return make_float2(z.x <= 0.0f ? 0.0f : z.x + z.x, z.y <= 0.0f ? 0.0f : z.y + z.y);
  else if constexpr (kAct == RB_ACT_SILU) {
    const float2 e = logistic_power<kAct, kExact>(z), s = rcp2(__fadd2_rn(e, both(1.0f)));
    return __fmul2_rn(s, __ffma2_rn(z, one_minus<kExact>(s, e), both(1.0f)));
  } else if constexpr (kAct == RB_ACT_GELU) {
    const NormalTail<1> n = normal_tail<kExact, 1>(&z);
    const float2 up = __ffma2_rn(n.q[0], both(-1.0f), both(1.0f));
    float2 phi = make_float2(z.x < 0.0f ? n.q[0].x : up.x, z.y < 0.0f ? n.q[0].y : up.y);
    if constexpr (kExact) phi = near_zero(z, normal_body(z), phi);
    return __ffma2_rn(__fmul2_rn(z, both(kInvSqrt2Pi)), n.e[0], phi);
  } else if constexpr (kAct == RB_ACT_GELU_TANH) {
    const float2 e = logistic_power<kAct, kExact>(z), s = rcp2(__fadd2_rn(e, both(1.0f)));
    const float2 t = __fmul2_rn(s, one_minus<kExact>(s, e));
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
