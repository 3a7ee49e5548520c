// What the feed-forward kernels share: 16-bit element conversion, the activations and their derivatives.
#pragma once
#include "ftb_host.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ftb {

inline int launch_status(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_last_cuda_error(static_cast<int>(e));
    return FTB_E_CUDA;
  }
  return FTB_OK;
}

inline int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A 16-bit element as fp32 and back (one rounding to nearest even).
__device__ __forceinline__ float from16(uint16_t v, bool f16) {
  if (f16) return __half2float(__ushort_as_half(v));
  return __uint_as_float(static_cast<uint32_t>(v) << 16);
}
__device__ __forceinline__ uint16_t to16(float v, bool f16) {
  if (f16) return __half_as_ushort(__float2half_rn(v));
  return __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// Two neighbouring elements of a 32-bit word.
__device__ __forceinline__ float2 unpack16(uint32_t v, bool f16) {
  if (f16) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack16(float a, float b, bool f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// 1 / (1 + exp(-x)); exp overflows to infinity for very negative x, which gives the limit 0.
__device__ __forceinline__ float sigmoid_f(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

// gelu_tanh(z) = z (1 + tanh(u)) / 2 = z sigmoid(2u).
// __fdividef returns 0 for a denominator in (2^126, 2^128) and x / inf = 0, which is the limit here; only the product
// with an infinite z needs care: relu keeps +inf, the others multiply z by a factor that has gone to 0 or 1, and
// -inf * 0 is NaN as it is in the formula.
__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case FTB_ACT_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays NaN
    case FTB_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.7071067811865476f));
    case FTB_ACT_GELU_TANH: return z * sigmoid_f(2.0f * kGeluC * (z + kGeluA * z * z * z));
    case FTB_ACT_SILU: return z * sigmoid_f(z);
    default: return z;
  }
}

// act'(z); relu has 0 at 0.
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case FTB_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case FTB_ACT_GELU:
      return 0.5f * (1.0f + erff(z * 0.7071067811865476f)) + z * 0.3989422804014327f * __expf(-0.5f * z * z);
    case FTB_ACT_GELU_TANH: {
      const float s = sigmoid_f(2.0f * kGeluC * (z + kGeluA * z * z * z));
      return s + 2.0f * z * s * (1.0f - s) * kGeluC * (1.0f + 3.0f * kGeluA * z * z);
    }
    case FTB_ACT_SILU: {
      const float s = sigmoid_f(z);
      return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.0f;
  }
}

}  // namespace ftb
