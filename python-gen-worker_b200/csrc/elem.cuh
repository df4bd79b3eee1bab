// Element types of the block operators (layer norm, rotary, gated linear):
// conversion of f32 / bf16 / f16 to f32 and back, and 16-byte vector access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <atomic>
#include <cstdint>
#include <type_traits>

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
  __device__ __forceinline__ uint4 bits() const { return *reinterpret_cast<const uint4*>(&raw); }
  __device__ __forceinline__ void put(uint4 w) { *reinterpret_cast<uint4*>(&raw) = w; }
};

// Two f32 in one 64-bit register: sm_100 multiplies and adds both in one
// instruction, which halves the issue slots of f32 streaming arithmetic.
struct F2 { unsigned long long v; };

__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum2(F2 a) {
  const float2 s = split(a);
  return s.x + s.y;
}

// 16 bytes of T <-> pairs of f32
template <typename T> struct Pairs {
  static constexpr int N = 8 / (int)sizeof(T);       // pairs in 16 bytes
};
template <typename T>
__device__ __forceinline__ void unpack(const uint4& w, F2 (&o)[Pairs<T>::N]) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
  if constexpr (sizeof(T) == 4) {
    o[0] = f2(__uint_as_float(r[0]), __uint_as_float(r[1]));
    o[1] = f2(__uint_as_float(r[2]), __uint_as_float(r[3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        o[j] = f2(__uint_as_float(r[j] << 16), __uint_as_float(r[j] & 0xffff0000u));
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[j]));
        o[j] = f2(f.x, f.y);
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 repack(const F2 (&o)[Pairs<T>::N]) {
  uint32_t r[4];
  if constexpr (sizeof(T) == 4) {
    const float2 a = split(o[0]), b = split(o[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x),
                      __float_as_uint(b.y));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = split(o[j]);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
        r[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(f.x, f.y);
        r[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
}

// Lets a kernel use up to `most` bytes of dynamic shared memory, asked of the
// driver once per device (a call costs more than a launch). `ready` belongs to
// the kernel.
inline bool allow_smem(const void* kern, std::atomic<uint64_t>& ready, int most) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (ready.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
    return false;
  ready.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

// Host-side status of a launch: clears the sticky-free error of this call only.
inline int launch_status() {
  return cudaGetLastError() == cudaSuccess ? GWB_SUCCESS : GWB_E_LAUNCH;
}

}  // namespace gwb
