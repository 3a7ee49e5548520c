// What the feed-forward kernels share: 16-bit element conversion, the activations and their derivatives.
#pragma once
#include "ftb_host.h"
#include "ftb_ptx.cuh"

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

// Phi(z), the normal distribution function, and exp(-z^2/2) on the way.  Phi(-|z|) exp(z^2/2) is smooth in
// t = 1 / (1 + 0.36 |z|) and goes to 0 with it: t times a polynomial of degree 6, whose coefficients minimise the largest
// RELATIVE error for |z| up to 14.5 (a linear program over 1200 nodes; 9.5e-7), so the tail of a negative z is the product
// itself and keeps fp32's digits: in fp32 off by 1.4e-6 of itself to z = -3, 3.7e-6 to -8, 6.8e-6 to -13, where the exponent's
// rounding leads, far below half a step of a 16-bit result (2^-11).
__device__ __forceinline__ float normal_cdf(float z, float* bell) {
  const float t = __fdividef(1.0f, fmaf(0.36f, fabsf(z), 1.0f));
  const float e = __expf(-0.5f * z * z);
  float poly = fmaf(t, 0.046779383f, -0.178817928f);
  poly = fmaf(t, poly, 0.179667756f);
  poly = fmaf(t, poly, 0.0274331067f);
  poly = fmaf(t, poly, 0.139397204f);
  poly = fmaf(t, poly, 0.141831115f);
  poly = fmaf(t, poly, 0.1437089f);
  const float tail = t * poly * e;
  *bell = e;
  return z < 0.0f ? tail : 1.0f - tail;
}

// gelu_tanh(z) = z (1 + tanh(u)) / 2 = z sigmoid(2u).
// __fdividef returns 0 for a denominator in (2^126, 2^128) and x / inf = 0, which is the limit here; only the product
// with an infinite z needs care: relu keeps +inf, the others multiply z by a factor that has gone to 0 or 1, and
// -inf * 0 is NaN as it is in the formula.
__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case FTB_ACT_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays NaN
    case FTB_ACT_GELU: {
      float bell;
      return z * normal_cdf(z, &bell);
    }
    case FTB_ACT_GELU_TANH: return z * sigmoid_f(2.0f * kGeluC * (z + kGeluA * z * z * z));
    case FTB_ACT_SILU: return z * sigmoid_f(z);
    default: return z;
  }
}

// act(z) and act'(z) of N values (relu' is 0 at 0): one branch, then straight-line code that shares the exponential.
template <int N>
__device__ __forceinline__ void act_both(const float (&z)[N], float (&value)[N], float (&slope)[N], int act) {
  if (act == FTB_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = sigmoid_f(z[i]);
      value[i] = z[i] * s;
      slope[i] = s * (1.0f + z[i] * (1.0f - s));
    }
  } else if (act == FTB_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float bell;
      const float cdf = normal_cdf(z[i], &bell);
      value[i] = z[i] * cdf;
      slope[i] = fmaf(z[i] * 0.3989422804014327f, bell, cdf);
    }
  } else if (act == FTB_ACT_GELU_TANH) {
    // z^2 is held to 1e4 (s is 0 or 1 from |z| = 15 on), so that no power of a large finite z becomes 0 * inf
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float q = fminf(z[i] * z[i], 1e4f), s = sigmoid_f(2.0f * kGeluC * z[i] * fmaf(kGeluA, q, 1.0f));
      value[i] = z[i] * s;
      slope[i] = fmaf(z[i] * (s * (1.0f - s)), 2.0f * kGeluC * fmaf(3.0f * kGeluA, q, 1.0f), s);
    }
  } else if (act == FTB_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      value[i] = z[i] < 0.0f ? 0.0f : z[i];
      slope[i] = z[i] > 0.0f ? 1.0f : 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      value[i] = z[i];
      slope[i] = 1.0f;
    }
  }
}

// ------------------------------------------------------------------ launches that overlap
// Every kernel of the feed-forward operators is launched as a programmatic dependent: its set-up runs while the kernel
// before it in the stream drains.  Each waits (griddepcontrol.wait) before its first access to global memory, so what
// an earlier kernel of any kind wrote is seen, asks for tensor memory only after that wait, and lets its own successor
// start only once it holds it: no kernel can take columns that one it waits for still needs.
template <typename... Params, typename... Args>
inline int launch_overlapped(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream,
                             Args... args) {
  cudaLaunchConfig_t lc;
  memset(&lc, 0, sizeof(lc));
  lc.gridDim = grid;
  lc.blockDim = block;
  lc.dynamicSmemBytes = smem;
  lc.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    lc.numAttrs = 2;
  }
  const cudaError_t e = cudaLaunchKernelEx(&lc, kernel, static_cast<Params>(args)...);
  count_launch();
  return launch_status(e);
}

}  // namespace ftb
