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
__device__ __forceinline__ float half_lo(unsigned pk) { return __uint_as_float(pk << 16); }
__device__ __forceinline__ float half_hi(unsigned pk) { return __uint_as_float(pk & 0xffff0000u); }

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
