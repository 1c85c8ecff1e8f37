// 16-bit activations eight at a time (one 16-byte access), widened to fp32: the
// access pattern of the convolution and norm kernels.  Tag types choose bf16 or
// fp16 at compile time.
#pragma once

#include <cuda_fp16.h>

#include "gdn_common.cuh"

namespace gdn {

struct Bf16 {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(bf16_lo(w), bf16_hi(w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};

struct Fp16 {
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Read-only and streaming 16-byte loads, and a streaming store.
__device__ __forceinline__ uint4 ldg_u4(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
__device__ __forceinline__ uint4 ld_cs_u4(const void* p) {
  uint4 r;
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
__device__ __forceinline__ void st_u4(void* p, uint4 v) {
  asm volatile("st.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

template <class T>
__device__ __forceinline__ void unpack8(uint4 w, float* v) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = T::unpack(u[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <class T>
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(T::pack(v[0], v[1]), T::pack(v[2], v[3]), T::pack(v[4], v[5]),
                    T::pack(v[6], v[7]));
}

// x sigmoid(x) from the hardware 2^x and reciprocal (each within 2 ulp of fp32,
// far below the 16-bit output's step).  For x below -87 the reciprocal of 1 + e^-x is
// below fp32's normal range and the result -0 (less than 2^-119 in exact arithmetic);
// -inf gives -inf * 0 = NaN, like the formula evaluated in fp32.
__device__ __forceinline__ float silu(float x) { return x * sigmoid_fast(x); }

}  // namespace gdn
