// Activations of the fused linear layer and their slopes, in f32.
//   gelu       z * Phi(z), Phi(z) = erfc(-z / sqrt 2) / 2
//   gelu_tanh  z * (1 + tanh(u)) / 2 = z * sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3)
//   silu       z * sigmoid(z)
// erfc is approximation 7.1.26 of Abramowitz & Stegun, "Handbook of
// Mathematical Functions": erfc(a) = (a1 t + .. + a5 t^5) exp(-a^2) with
// t = 1 / (1 + p a), a >= 0, at most 1.5e-7 off: two special-function
// instructions and a short polynomial per value, which the GEMM's epilogue
// warps fit under the next tile's mainloop.  relu keeps a NaN.
#pragma once

#include "common.cuh"

namespace packr {
namespace act {

__device__ __forceinline__ float ex2(float a) {
  float d;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(a));
  return d;
}
__device__ __forceinline__ float rcp(float a) {
  float d;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(a));
  return d;
}

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kTanhC = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float kTanhK = 0.044715f;
constexpr float kInvSqrt2Pi = 0.3989422804014327f;

// Phi(z); e = exp(-z^2 / 2)
__device__ __forceinline__ float phi_cdf(float z, float& e) {
  const float a = fabsf(z) * 0.7071067811865476f;
  e = ex2(z * z * (-0.5f * kLog2E));
  const float t = rcp(fmaf(0.3275911f, a, 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float q = 0.5f * p * t * e;  // erfc(a) / 2
  return z < 0.0f ? q : 1.0f - q;
}

__device__ __forceinline__ float sigmoid(float v) { return rcp(1.0f + ex2(-kLog2E * v)); }

template <int ACT>
__device__ __forceinline__ float apply(float z) {
  if (ACT == PACKR_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if (ACT == PACKR_ACT_GELU) {
    float e;
    return z * phi_cdf(z, e);
  }
  if (ACT == PACKR_ACT_GELU_TANH) return z * sigmoid(2.0f * kTanhC * fmaf(kTanhK * z * z, z, z));
  if (ACT == PACKR_ACT_SILU) return z * sigmoid(z);
  return z;
}

template <int ACT>
__device__ __forceinline__ float slope(float z) {
  if (ACT == PACKR_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (ACT == PACKR_ACT_GELU) {
    float e;
    const float p = phi_cdf(z, e);
    return fmaf(z * e, kInvSqrt2Pi, p);
  }
  if (ACT == PACKR_ACT_GELU_TANH) {
    // s is 0 or 1 from |z| = 20 on, far below; z * z beyond the type's range would
    // make the product 0 * infinity
    const float zz = fminf(z * z, 400.0f);
    const float s = sigmoid(2.0f * kTanhC * fmaf(kTanhK * zz, z, z));
    return fmaf(z * s * (1.0f - s), 2.0f * kTanhC * fmaf(3.0f * kTanhK, zz, 1.0f), s);
  }
  if (ACT == PACKR_ACT_SILU) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  return 1.0f;
}

// v[0..n) = act(v), the choice made once for all of them.
template <int n>
__device__ __forceinline__ void apply_all(int a, float* v) {
  switch (a) {
    case PACKR_ACT_RELU:
#pragma unroll
      for (int j = 0; j < n; ++j) v[j] = apply<PACKR_ACT_RELU>(v[j]);
      break;
    case PACKR_ACT_GELU:
#pragma unroll
      for (int j = 0; j < n; ++j) v[j] = apply<PACKR_ACT_GELU>(v[j]);
      break;
    case PACKR_ACT_GELU_TANH:
#pragma unroll
      for (int j = 0; j < n; ++j) v[j] = apply<PACKR_ACT_GELU_TANH>(v[j]);
      break;
    case PACKR_ACT_SILU:
#pragma unroll
      for (int j = 0; j < n; ++j) v[j] = apply<PACKR_ACT_SILU>(v[j]);
      break;
    default: break;
  }
}

}  // namespace act

// Epilogue of the fused linear layer: z = acc + bias is stored when `z` is
// set, out = act(z) + residual.  residual, out and z are [M, N] row-major of
// one type (io_f32: f32, else bf16).
struct Epilogue {
  const void* residual;  // nullable
  void* out;
  void* z;               // nullable
  int io_f32;
  int act;
  int vec;               // all three 16-byte aligned, with rows a multiple of 16 bytes
};

__device__ __forceinline__ float load_io(const void* p, long long i, int f32) {
  return f32 ? __ldg(static_cast<const float*>(p) + i) : bf16_to_f32(__ldg(static_cast<const uint16_t*>(p) + i));
}
// The same for kernels that may start before their inputs are written
// (launch_overlapped).
__device__ __forceinline__ float load_io_late(const void* p, long long i, int f32) {
  return f32 ? __ldcg(static_cast<const float*>(p) + i) : bf16_to_f32(__ldcg(static_cast<const uint16_t*>(p) + i));
}
__device__ __forceinline__ void store_io(void* p, long long i, int f32, float v) {
  if (f32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<uint16_t*>(p)[i] = (uint16_t)(pack_bf16x2_rne(v, 0.0f) & 0xFFFFu);
}

}  // namespace packr
