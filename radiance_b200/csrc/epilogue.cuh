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
  uint32_t threshold;   // 0 .. 65536
  float scale;
};

struct PhiloxKey {
  uint32_t k0, k1;
};

__device__ __forceinline__ PhiloxKey philox_key(const int64_t* seed) {
  const uint64_t s = static_cast<uint64_t>(__ldg(reinterpret_cast<const long long*>(seed)));
  return {static_cast<uint32_t>(s), static_cast<uint32_t>(s >> 32)};
}

__device__ __forceinline__ uint4 philox(uint64_t counter, PhiloxKey key) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32), c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ key.k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ key.k1;
    c3 = static_cast<uint32_t>(a);
    key.k0 += 0x9E3779B9u;
    key.k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Drops from the eight elements 8 * group .. 8 * group + 7.  A dropped element is 0 whatever it
// held, infinities and NaN included.
__device__ __forceinline__ void dropout8(float (&v)[8], uint64_t group, PhiloxKey key, uint32_t threshold,
                                         float scale) {
  const uint4 d = philox(group, key);
  const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = (w[j] & 0xFFFFu) >= threshold ? v[2 * j] * scale : 0.0f;
    v[2 * j + 1] = (w[j] >> 16) >= threshold ? v[2 * j + 1] * scale : 0.0f;
  }
}

// One element, at any index.
__device__ __forceinline__ float dropout1(float v, uint64_t index, PhiloxKey key, uint32_t threshold, float scale) {
  const uint4 d = philox(index >> 3, key);
  const uint32_t j = static_cast<uint32_t>(index) & 7u;
  const uint32_t lo = (j & 2) ? d.y : d.x, hi = (j & 2) ? d.w : d.z;
  const uint32_t w = (j & 4) ? hi : lo;
  return ((j & 1) ? w >> 16 : w & 0xFFFFu) >= threshold ? v * scale : 0.0f;
}

// ---------------------------------------------------------------------------------------------
// Activations (RB_ACT_*)
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.0f, 1.0f + expf(-z)); }

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluA = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

// 0.5 z (1 + tanh(u)) = z sigmoid(2u): one exponential, and no cancellation where tanh nears -1.
template <int kAct>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (kAct == RB_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN passes through
  else if constexpr (kAct == RB_ACT_RELU2) return z < 0.0f ? 0.0f : z * z;
  else if constexpr (kAct == RB_ACT_SILU) return z * sigmoid(z);
  else if constexpr (kAct == RB_ACT_GELU) return 0.5f * z * (1.0f + erff(z * kSqrtHalf));
  else if constexpr (kAct == RB_ACT_GELU_TANH) return z * sigmoid(kGeluA * fmaf(kGeluB * z * z, z, z));
  else return z;
}

template <int kAct>
__device__ __forceinline__ float act_derivative(float z) {
  if constexpr (kAct == RB_ACT_RELU) return z <= 0.0f ? 0.0f : (z != z ? z : 1.0f);
  else if constexpr (kAct == RB_ACT_RELU2) return z <= 0.0f ? 0.0f : 2.0f * z;
  else if constexpr (kAct == RB_ACT_SILU) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  } else if constexpr (kAct == RB_ACT_GELU) {
    return fmaf(z, kInvSqrt2Pi * expf(-0.5f * z * z), 0.5f * (1.0f + erff(z * kSqrtHalf)));
  } else if constexpr (kAct == RB_ACT_GELU_TANH) {
    const float s = sigmoid(kGeluA * fmaf(kGeluB * z * z, z, z));
    const float t = s * (1.0f - s);  // 0 wherever the polynomial below could overflow
    return t > 0.0f ? fmaf(z * t, kGeluA * fmaf(3.0f * kGeluB * z, z, 1.0f), s) : s;
  } else return 1.0f;
}

// ---------------------------------------------------------------------------------------------
// Eight elements of a row to and from fp32
// ---------------------------------------------------------------------------------------------
template <typename T>
struct Io;

template <>
struct Io<__nv_bfloat16> {
  static __device__ __forceinline__ void load8(float (&v)[8], const __nv_bfloat16* p) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ void round8(float (&v)[8], uint4& q) {  // v becomes what q holds
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
    q = make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ void store8(__nv_bfloat16* p, float (&v)[8]) {
    uint4 q;
    round8(v, q);
    *reinterpret_cast<uint4*>(p) = q;
  }
  static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ float store(__nv_bfloat16* p, float v) {
    const __nv_bfloat16 b = __float2bfloat16_rn(v);
    *p = b;
    return __bfloat162float(b);
  }
};

template <>
struct Io<float> {
  static __device__ __forceinline__ void load8(float (&v)[8], const float* p) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  static __device__ __forceinline__ void store8(float* p, float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ float store(float* p, float v) { return *p = v; }
};

}  // namespace rb

namespace rb_host {

// Device arguments of dropout with probability p (0 <= p <= 1, checked by the caller) and a device seed.
inline rb::DropoutArgs dropout_args(double p, const int64_t* seed) {
  rb::DropoutArgs d;
  d.threshold = static_cast<uint32_t>(p * 65536.0 + 0.5);
  d.scale = d.threshold < 65536u ? static_cast<float>(65536.0 / (65536.0 - d.threshold)) : 0.0f;
  d.seed = p > 0.0 ? seed : nullptr;
  return d;
}

}  // namespace rb_host
