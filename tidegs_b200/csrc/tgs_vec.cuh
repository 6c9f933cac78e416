// Typed loads and stores of the appearance operators: fp32, bf16 and fp16
// tensors, computed on in 32 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "tgs_common.cuh"

namespace tgs {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) {
    return v;
  } else if constexpr (std::is_same_v<T, __half>) {
    return __float2half_rn(v);
  } else {
    return __float2bfloat16_rn(v);
  }
}

// kVec values at p (aligned to their joint size), or zeros where !on.
template <class T, int kVec>
__device__ __forceinline__ void load_vec(const T* p, bool on, float (&v)[kVec]) {
  constexpr int kBytes = sizeof(T) * kVec;
  union {
    uint4 q;
    T t[kVec];
  } u;
  if constexpr (kBytes == 16) {
    u.q = on ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = to_f32(u.t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = on ? to_f32(p[i]) : 0.f;
  }
}

// kVec values as they lie in memory.
template <class T, int kVec>
struct Packed {
  static constexpr bool kWhole = sizeof(T) * kVec == 16;
  union {
    uint4 q;
    T t[kVec];
  };
  __device__ __forceinline__ Packed() {}
  __device__ __forceinline__ void load(const T* p, bool on) {
    if constexpr (kWhole) {
      q = on ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) t[i] = on ? p[i] : from_f32<T>(0.f);
    }
  }
  __device__ __forceinline__ float get(int i) const { return to_f32(t[i]); }
};

template <class T, int kVec>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[kVec]) {
  if constexpr (sizeof(T) * kVec == 16) {
    union {
      uint4 q;
      T t[kVec];
    } u;
#pragma unroll
    for (int i = 0; i < kVec; ++i) u.t[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = u.q;
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) p[i] = from_f32<T>(v[i]);
  }
}

// Two fp32 values in a register pair: one instruction for both.
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  }
  __device__ __forceinline__ explicit F2(uint64_t x) : v(x) {}
  __device__ __forceinline__ void get(float& a, float& b) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
  }
};
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.v), "l"(b.v));
  return F2(r);
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.v), "l"(b.v));
  return F2(r);
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a.v), "l"(b.v), "l"(c.v));
  return F2(r);
}

__device__ __forceinline__ float load_param(const void* p, int dtype, int64_t i) {
  switch (dtype) {
    case TGS_F32: return static_cast<const float*>(p)[i];
    case TGS_BF16: return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
    default: return to_f32(static_cast<const __half*>(p)[i]);
  }
}

__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
  switch (dtype) {
    case TGS_F32: static_cast<float*>(p)[i] = v; break;
    case TGS_BF16: static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v); break;
    default: static_cast<__half*>(p)[i] = from_f32<__half>(v); break;
  }
}

inline bool valid_dtype(int dtype) {
  return dtype == TGS_F32 || dtype == TGS_BF16 || dtype == TGS_F16;
}

}  // namespace tgs
