// Row element types of the token-mixing operators (IC_DT_*): conversions to and from fp32.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "ic_common.h"

// 16-bit types as plain storage: arithmetic is fp32, each value rounded once (to nearest even) when it is stored
struct ic_bf16 { uint16_t u; };
struct ic_f16 { uint16_t u; };

__device__ __forceinline__ float ic_to_f(float v) { return v; }
__device__ __forceinline__ float ic_to_f(ic_bf16 v) { return __uint_as_float((uint32_t)v.u << 16); }
__device__ __forceinline__ float ic_to_f(ic_f16 v) { return __half2float(__ushort_as_half(v.u)); }

template <typename T>
__device__ __forceinline__ T ic_from_f(float v);
template <>
__device__ __forceinline__ float ic_from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ ic_bf16 ic_from_f<ic_bf16>(float v) {
  const __bf16 b = (__bf16)v;  // v_cvt_pk_bf16_f32: nearest even, NaN stays NaN
  return ic_bf16{__builtin_bit_cast(uint16_t, b)};
}
template <>
__device__ __forceinline__ ic_f16 ic_from_f<ic_f16>(float v) { return ic_f16{__half_as_ushort(__float2half_rn(v))}; }

// one value of a run-time type (IC_DT_*)
__device__ __forceinline__ float ic_load_dt(const void* p, int dt, int i) {
  return dt == IC_DT_F32 ? ((const float*)p)[i] : dt == IC_DT_BF16 ? ic_to_f(((const ic_bf16*)p)[i]) : ic_to_f(((const ic_f16*)p)[i]);
}
__device__ __forceinline__ void ic_store_dt(void* p, int dt, int i, float v) {
  if (dt == IC_DT_F32) ((float*)p)[i] = v;
  else if (dt == IC_DT_BF16) ((ic_bf16*)p)[i] = ic_from_f<ic_bf16>(v);
  else ((ic_f16*)p)[i] = ic_from_f<ic_f16>(v);
}

static inline int ic_dt_size(int dt) { return dt == IC_DT_F32 ? 4 : 2; }
static inline bool ic_dt_ok(int dt) { return dt == IC_DT_F32 || dt == IC_DT_BF16 || dt == IC_DT_F16; }
