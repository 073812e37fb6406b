// dig3d — element types of the 16-bit operators (rownorm.hip, head.hip): codes, conversions and row vectors.
#pragma once
#include "common.h"

#define DT_F32 0
#define DT_BF16 1
#define DT_F16 2

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// N elements of a row from any element address: rows of an odd width or stride start anywhere, and the global memory path
// takes a 16-byte access at every 2-byte address
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) RowVec {
  T v[N];
};

template <class T>
struct VecLen {
  static constexpr int n = 16 / (int)sizeof(T);
};

// float -> T, to nearest even (the only rounding of a result held in 16 bits)
template <class T>
__device__ __forceinline__ T to_t(float v) {
  return (T)v;
}

// parameter vectors and per-column outputs whose type is only known at run time
__device__ __forceinline__ float load_as(const void* p, int dt, int64_t i) {
  return dt == DT_F32 ? ((const float*)p)[i] : dt == DT_BF16 ? (float)((const bf16_t*)p)[i] : (float)((const f16_t*)p)[i];
}
__device__ __forceinline__ void store_as(void* p, int dt, int64_t i, float v) {
  if (dt == DT_F32) ((float*)p)[i] = v;
  else if (dt == DT_BF16) ((bf16_t*)p)[i] = (bf16_t)v;
  else ((f16_t*)p)[i] = (f16_t)v;
}
