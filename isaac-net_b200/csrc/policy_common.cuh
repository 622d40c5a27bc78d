// Shared device helpers of the policy operators (policy_*.cu): element types, vector access, group reductions.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "isaac_net_b200.h"

namespace inb {
namespace pol {

using bf16 = __nv_bfloat16;
using f16 = __half;

constexpr uint32_t M32_ALL = 0xFFFFFFFFu;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(f16 v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ f16 from_f<f16>(float v) { return __float2half_rn(v); }

template <typename T> struct IsBf16 { static constexpr bool value = false; };
template <> struct IsBf16<bf16> { static constexpr bool value = true; };

// V consecutive elements moved by one access (V * sizeof(T) bytes, aligned to that)
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> ld(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void st(T* p, const Pack<T, V>& v) {
  *reinterpret_cast<Pack<T, V>*>(p) = v;
}

// Two fp32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// two elements to fp32 and back
__device__ __forceinline__ float2 up2(float a, float b) { return make_float2(a, b); }
__device__ __forceinline__ float2 up2(bf16 a, bf16 b) { return __bfloat1622float2(__halves2bfloat162(a, b)); }
__device__ __forceinline__ float2 up2(f16 a, f16 b) { return __half22float2(__halves2half2(a, b)); }
__device__ __forceinline__ void down2(float2 v, float& a, float& b) {
  a = v.x;
  b = v.y;
}
__device__ __forceinline__ void down2(float2 v, bf16& a, bf16& b) {
  const __nv_bfloat162 t = __float22bfloat162_rn(v);
  a = t.x;
  b = t.y;
}
__device__ __forceinline__ void down2(float2 v, f16& a, f16& b) {
  const __half2 t = __float22half2_rn(v);
  a = t.x;
  b = t.y;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// SMs of the current device (the library is built for one architecture; a process may see several devices)
inline int sm_count() {
  static int n[64] = {0};
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= 64) return 148;
  if (n[d] == 0) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, d) != cudaSuccess || v < 1) return 148;
    n[d] = v;
  }
  return n[d];
}

// Lets a kernel use `bytes` of dynamic shared memory on the current device: one call of the runtime for a kernel, device
// and thread (so that a thread's first call also makes the device's context current to it, see policy_ffn.cuh).  KEY: a type
// of the kernel's own.
template <typename KEY>
inline cudaError_t allow_smem(const void* kernel, int bytes) {
  static thread_local uint64_t done = 0;
  int d = 0;
  const cudaError_t e = cudaGetDevice(&d);
  if (e != cudaSuccess || (d < 64 && (done >> d & 1))) return e;
  const cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (r == cudaSuccess && d < 64) done |= 1ull << d;
  return r;
}
template <auto K>
struct KernelKey {};

inline int launch_status() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : -100 - (int)e;
}

}  // namespace pol
}  // namespace inb
