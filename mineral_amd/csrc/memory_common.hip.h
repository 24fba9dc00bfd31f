// What the operators of include/mineral_memory.h share: element types, vector types, two-term bf16 splits.
#pragma once
#include "../../include/mineral_memory.h"
#include "../../include/mineral_ppo.h"

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>

namespace mrl {
void set_error(const char* msg);   // defined next to mrl_last_error()

namespace mem {
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// two fp32 values -> packed bf16, rounded to nearest even (v_cvt_pk_bf16_f32), and the fp32 values of the halves
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(unsigned, v);
}
// (v_perm for the low half: a shift makes the compiler convert that element a second time by itself)
__device__ __forceinline__ float half_lo(unsigned pk) { return __uint_as_float(__builtin_amdgcn_perm(pk, 0u, 0x05040c0cu)); }
__device__ __forceinline__ float half_hi(unsigned pk) { return __uint_as_float(pk & 0xffff0000u); }

// Activations and their derivatives at z, in fp32.  `act` is uniform over the launch.  The logistic function uses the hardware's
// exp2 and reciprocal (one spacing each); where a difference cancels near zero (ELU, erf) the library's functions do.
__device__ __forceinline__ float logistic(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }
// tanh from its series up to 1/4 (the first term left out is below 1e-8 of it) and from exp2 beyond, where the difference from one
// loses at most two bits
__device__ __forceinline__ float tanh_of(float z) {
  const float q = z * z, a = __builtin_fabsf(z);
  const float low = z * __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
  const float high = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a * 2.88539008f));
  return a < 0.25f ? low : __builtin_copysignf(high, z);
}
// Its derivative: 1 - t^2 up to 1/4; beyond, where t is nearly one and the difference would cancel, 4 r (1 - r) with the reciprocal r
// that t = 1 - 2 r is made of, which keeps its digits down to 2^-120 (relative error 4 |z| 2^-24 from the exponential's argument).
__device__ __forceinline__ float tanh_slope(float z) {
  const float a = __builtin_fabsf(z), t = tanh_of(z);
  const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(a * 2.88539008f));
  return a < 0.25f ? 1.0f - t * t : 4.0f * r * (1.0f - r);
}
template <int N> __device__ __forceinline__ void act_fwd(int act, float (&z)[N]) {
  switch (act) {
    case MRL_ACT_SILU:
#pragma unroll
      for (int e = 0; e < N; ++e) z[e] *= logistic(z[e]);
      break;
    case MRL_ACT_ELU:
#pragma unroll
      for (int e = 0; e < N; ++e) z[e] = z[e] > 0.0f ? z[e] : expm1f(z[e]);
      break;
    case MRL_ACT_RELU:
#pragma unroll
      for (int e = 0; e < N; ++e) z[e] = z[e] < 0.0f ? 0.0f : z[e];
      break;
    case MRL_ACT_TANH:
#pragma unroll
      for (int e = 0; e < N; ++e) z[e] = tanh_of(z[e]);
      break;
    case MRL_ACT_GELU:
#pragma unroll
      for (int e = 0; e < N; ++e) z[e] *= 0.5f * erfcf(z[e] * -0.70710678f);
      break;
    default: break;
  }
}
// act'(z) into d
template <int N> __device__ __forceinline__ void act_slope(int act, const float (&z)[N], float (&d)[N]) {
  switch (act) {
    case MRL_ACT_SILU:
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float s = logistic(z[e]);
        d[e] = s * (1.0f + z[e] * (1.0f - s));
      }
      break;
    case MRL_ACT_ELU:
#pragma unroll
      for (int e = 0; e < N; ++e) d[e] = z[e] > 0.0f ? 1.0f : expf(z[e]);
      break;
    case MRL_ACT_RELU:
#pragma unroll
      for (int e = 0; e < N; ++e) d[e] = z[e] <= 0.0f ? 0.0f : 1.0f;
      break;
    case MRL_ACT_TANH:
#pragma unroll
      for (int e = 0; e < N; ++e) d[e] = tanh_slope(z[e]);
      break;
    case MRL_ACT_GELU:
#pragma unroll
      for (int e = 0; e < N; ++e) d[e] = 0.5f * erfcf(z[e] * -0.70710678f) + z[e] * 0.39894228f * expf(-0.5f * z[e] * z[e]);
      break;
    default:
#pragma unroll
      for (int e = 0; e < N; ++e) d[e] = 1.0f;
      break;
  }
}
// d[e] *= act'(z[e])
template <int N> __device__ __forceinline__ void act_bwd(int act, const float (&z)[N], float (&d)[N]) {
  if (act == MRL_ACT_NONE) return;
  float s[N];
  act_slope<N>(act, z, s);
#pragma unroll
  for (int e = 0; e < N; ++e) d[e] = act == MRL_ACT_RELU && s[e] == 0.0f ? 0.0f : d[e] * s[e];
}

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
}  // namespace mem
}  // namespace mrl

#define MEM_FAIL(code, ...)                       \
  do {                                            \
    char b_[256];                                 \
    snprintf(b_, sizeof(b_), __VA_ARGS__);        \
    mrl::set_error(b_);                           \
    return (code);                                \
  } while (0)

#define MEM_CHECK_LAUNCH(what)                                                           \
  do {                                                                                   \
    hipError_t e_ = hipGetLastError();                                                   \
    if (e_ != hipSuccess) MEM_FAIL(MRL_EHIP, "%s: %s", what, hipGetErrorString(e_));     \
  } while (0)
