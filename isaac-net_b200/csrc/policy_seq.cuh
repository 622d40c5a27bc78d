// What the policy's memory kernels (policy_conv.cu, policy_scan*.cu, policy_distill.cu) share: sequences and resets, the
// scalar functions, and the column sums that join the blocks' partial gradients.
#pragma once
#include <cmath>

#include "policy_common.cuh"

namespace inb {
namespace pol {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float ex2(float v) {      // 2^v, 2 ulp
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {      // 1 / v, 1 ulp
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float sigmoid(float v) { return rcp(1.f + ex2(-v * LOG2E)); }

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 sigmoid2(float2 v) {
  const float2 t = mul2(v, both(-LOG2E)), d = add2(make_float2(ex2(t.x), ex2(t.y)), both(1.f));
  return make_float2(rcp(d.x), rcp(d.y));
}
// 2^v of two values without the special function unit, which makes 16 results a clock and SM and so bounds the scan: v = i + f,
// f in [-1/2, 1/2], 2^f = 1 + f P(f) with P the Chebyshev interpolation of (2^f - 1) / f of degree 5 (at most 1.2 * 2^-24
// off, no bias where 2^v is near 1), times 2^i through the exponent's bits.  v is held to [-127, 128]: 0 and infinity there.
__device__ __forceinline__ float2 ex2_poly(float2 v) {
  auto hold = [](float x) {
    float r;
    asm("max.NaN.f32 %0, %1, 0fC2FE0000;" : "=f"(r) : "f"(x));      // -127
    asm("min.NaN.f32 %0, %1, 0f43000000;" : "=f"(r) : "f"(r));      // 128
    return r;
  };
  v = make_float2(hold(v.x), hold(v.y));
  const float2 magic = both(12582912.f + 127.f);      // 1.5 * 2^23: the sum's low bits are i + 127
  const float2 r = add2(v, magic);
  const float2 f = fma2(add2(r, both(-12582912.f - 127.f)), both(-1.f), v);
  float2 p = fma2(both(0.00015453163359779865f), f, both(0.0013390863314270973f));
  p = fma2(p, f, both(0.009618083015084267f));
  p = fma2(p, f, both(0.055503569543361664f));
  p = fma2(p, f, both(0.24022650718688965f));
  p = fma2(p, f, both(0.6931471824645996f));
  p = fma2(p, f, both(1.f));
  return mul2(p, make_float2(__uint_as_float(__float_as_uint(r.x) << 23), __uint_as_float(__float_as_uint(r.y) << 23)));
}

// log(1 + e^v) = max(v, 0) + log(1 + u), u = e^-|v| in [0, 1].  log(1 + u) = u P(u), P the Chebyshev interpolation of
// log(1 + u) / u of degree 9 (at most 2.1 * 2^-24 off), so that small results keep their relative precision, which log of a
// rounded 1 + u would lose.
__device__ __forceinline__ float softplus_u(float v, float& u) {
  // a step that is to leave the state as it is has dt of -inf or of the type's lowest value: e^-128 is 0, and a NaN stays one
  float a;
  asm("max.NaN.f32 %0, %1, 0fC3000000;" : "=f"(a) : "f"(-fabsf(v)));      // -128
  const float t = a * LOG2E;
  const float low = fmaf(a, LOG2E, -t);              // what t's rounding lost, 2^-24 |v|, and would cost u relative
  const float e = ex2(t);
  u = fmaf(e, low * LN2, e);
  float p = fmaf(u, -0.0031760570127516985f, 0.019542526453733444f);
  p = fmaf(u, p, -0.056373611092567444f);
  p = fmaf(u, p, 0.10543623566627502f);
  p = fmaf(u, p, -0.1526966691017151f);
  p = fmaf(u, p, 0.1966327428817749f);
  p = fmaf(u, p, -0.24951615929603577f);
  p = fmaf(u, p, 0.33329710364341736f);
  p = fmaf(u, p, -0.49999892711639404f);
  p = fmaf(u, p, 1.f);
  return fmaf(u, p, fmaxf(v, 0.f));
}
__device__ __forceinline__ float softplus(float v) {
  float u;
  return softplus_u(v, u);
}
// s: the derivative, 1 / (1 + e^-v)
__device__ __forceinline__ float softplus(float v, float& s) {
  float u;
  const float r = softplus_u(v, u), i = rcp(1.f + u);
  s = v >= 0.f ? i : u * i;
  return r;
}

// An element as it lies in memory, in a register of its own: loads that stay on their way must not be packed with others
template <typename T>
__device__ __forceinline__ uint32_t ld_raw(const T* p) {
  if constexpr (sizeof(T) == 2)
    return *reinterpret_cast<const uint16_t*>(p);
  else
    return *reinterpret_cast<const uint32_t*>(p);
}
template <typename T>
__device__ __forceinline__ float raw_f(uint32_t v) {
  if constexpr (IsBf16<T>::value)
    return __uint_as_float(v << 16);
  else if constexpr (sizeof(T) == 2)
    return __half2float(__ushort_as_half((uint16_t)v));
  else
    return __uint_as_float(v);
}

// V (1, 2, 4 or 8; up to 16 bytes) neighbouring elements as they lie in memory; their values as pairs (V = 1: the first of one pair)
template <typename T, int V>
struct Words {
  static constexpr int P = V < 2 ? 1 : V / 2, N = V * sizeof(T) / 4 > 0 ? V * sizeof(T) / 4 : 1;
  uint32_t w[N];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) {
      w[0] = ld_raw(p);
    } else if constexpr (N == 1) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (N == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1 && sizeof(T) == 2)
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    else if constexpr (N == 1)
      *reinterpret_cast<uint32_t*>(p) = w[0];
    else if constexpr (N == 2)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void join(const uint32_t (&e)[V]) {      // of elements as ld_raw gives them
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = sizeof(T) == 4 || V == 1 ? e[i] : e[(2 * i) % V] | e[(2 * i + 1) % V] << 16;
  }
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (V == 1)
      return make_float2(raw_f<T>(w[0]), 0.f);
    else if constexpr (sizeof(T) == 4)
      return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else if constexpr (IsBf16<T>::value)
      return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    else
      return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  }
  __device__ __forceinline__ void set(int i, float2 v) {
    if constexpr (sizeof(T) == 4) {
      w[V == 1 ? 0 : 2 * i] = __float_as_uint(v.x);
      if constexpr (V > 1) w[2 * i + 1] = __float_as_uint(v.y);
    } else {
      if constexpr (IsBf16<T>::value) {
        const __nv_bfloat162 q = __float22bfloat162_rn(v);
        w[i] = *reinterpret_cast<const uint32_t*>(&q);
      } else {
        const __half2 q = __float22half2_rn(v);
        w[i] = *reinterpret_cast<const uint32_t*>(&q);
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ const T* row(const InbSeq& q, int64_t s, int64_t t) {
  return (const T*)q.p + s * q.seq + t * q.step;
}
template <typename T>
__device__ __forceinline__ T* row_out(const InbSeq& q, int64_t s, int64_t t) {
  return (T*)q.p + s * q.seq + t * q.step;
}
// The reset bytes of sequence s, or NULL.  s and rows are below 2^31 (the entry points hold rows to that): a 64-bit division
// takes five times as long as a step of the convolution.
__device__ __forceinline__ const uint8_t* resets(const InbReset& r, int64_t s) {
  return r.p == nullptr ? nullptr : r.p + (uint32_t)s / (uint32_t)r.rows * r.seq;
}

// In a branch that is seldom taken: keeps the compiler from running its moves on every step
__device__ __forceinline__ void keep_branch() { __syncwarp(__activemask()); }

inline bool is_aligned(const InbSeq& q, int64_t bytes, int64_t elem) {
  return q.p == nullptr || (((uint64_t)(uintptr_t)q.p | (uint64_t)(q.seq * elem) | (uint64_t)(q.step * elem)) & (bytes - 1)) == 0;
}
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ------------------------------------------------------------------------------------------------- column sums
// part [P, M] fp32 -> sums over P: columns [0, first) to out0, [first, second) to out1, the others to out2 (any may be NULL).
// A block takes 32 columns, its 32 warps rows p, p + 32, ...; the order of the sum does not depend on timing.  Bound by latency
// (4 loads of a thread on their way): 592 rows of 1280 columns 5.6 us.
constexpr int COLSUM_WARPS = 32;
template <typename T>
__global__ void __launch_bounds__(COLSUM_WARPS * 32) colsum_kernel(const float* part, int64_t P, int64_t M, int64_t first, int64_t second,
                                                                   T* out0, T* out1, T* out2) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < M) {
    int64_t p = w;
    for (; p + 3 * COLSUM_WARPS < P; p += 4 * COLSUM_WARPS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += part[(p + COLSUM_WARPS * i) * M + c];
    }
    for (; p < P; p += COLSUM_WARPS) v[0] += part[p * M + c];
  }
  __shared__ float sum[COLSUM_WARPS][33];
  sum[w][lane] = (v[0] + v[1]) + (v[2] + v[3]);
  __syncthreads();
  // a warp a column: the 32 warps' sums of it
  const float s = warp_sum(sum[lane][w]);
  const int64_t to = (int64_t)blockIdx.x * 32 + w;
  if (lane != 0 || to >= M) return;
  if (to < first) {
    if (out0 != nullptr) out0[to] = from_f<T>(s);
  } else if (to < second) {
    if (out1 != nullptr) out1[to - first] = from_f<T>(s);
  } else if (out2 != nullptr) {
    out2[to - second] = from_f<T>(s);
  }
}
template <typename T>
inline void colsum(const float* part, int64_t P, int64_t M, int64_t first, int64_t second, void* out0, void* out1, void* out2,
                   cudaStream_t s) {
  colsum_kernel<T><<<(unsigned)ceil_div(M, 32), COLSUM_WARPS * 32, 0, s>>>(part, P, M, first, second, (T*)out0, (T*)out1, (T*)out2);
}

}  // namespace pol
}  // namespace inb
