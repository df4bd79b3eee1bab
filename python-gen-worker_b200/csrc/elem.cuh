// Element types of the block operators (layer norm, rotary, gated linear):
// conversion of f32 / bf16 / f16 to f32 and back, and 16-byte vector access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace gwb {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

// f32 -> T, round to nearest even: the one rounding of every output
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

// VEC consecutive elements as one access: 16 bytes, or one element.
template <typename T, int VEC> struct Pack {
  static_assert(VEC == 1 || VEC * sizeof(T) == 16, "a vector is one element or 16 bytes");
  struct alignas(VEC == 1 ? sizeof(T) : 16) Raw { T v[VEC]; };
  Raw raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ float get(int j) const { return to_f32<T>(raw.v[j]); }
  __device__ __forceinline__ void set(int j, float f) { raw.v[j] = from_f32<T>(f); }
};

// Host-side status of a launch: clears the sticky-free error of this call only.
inline int launch_status() {
  return cudaGetLastError() == cudaSuccess ? GWB_SUCCESS : GWB_E_LAUNCH;
}

}  // namespace gwb
