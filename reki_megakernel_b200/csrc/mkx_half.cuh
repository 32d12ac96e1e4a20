// The two 16-bit types of the episode cache, as raw words: conversions and packing.
#pragma once
#include <stdint.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mkx {

template <int DT>
struct Half16;
template <>
struct Half16<0> {  // bf16
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&t);
  }
};
template <>
struct Half16<1> {  // fp16
  static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&t);
  }
};

}  // namespace mkx
