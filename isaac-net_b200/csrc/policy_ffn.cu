// gated_ffn: the gated feed-forward block and its gradients, six products on the tensor cores (policy_gemm.cuh).
//
//   forward   g = x Wg^T, u = x Wu^T, h = act(g) * u     one product over [Wg | Wu], activation and product in its epilogue
//             y = h Wd^T
//   backward  dh = dy Wd, dg = dh u act'(g), du = dh act(g)     one product, both gradients in its epilogue
//             dx = dg Wg + du Wu                                one product over k = 2 F
//             dWg = dg^T x, dWu = du^T x                        one product over m = 2 F
//             dWd = dy^T h
//
// A tile of the first product holds 128 columns of g and the same 128 of u, so act(g) * u needs no exchange.  g and u are
// kept for the backward pass in fp32: rounding them to the operand type would put two more roundings into dg and du (the
// weights' gradients then are 1.4 times as far from the exact ones), and reading them costs 16 bytes an element of h
// against the 18 D operations the step does for it.  h, dg and du are rounded to the operand type because the next
// product multiplies them.
#include "policy_gemm.cuh"

namespace inb {
namespace pol {

__device__ __forceinline__ float act_of(float g, int act) {
  if (act == INB_ACT_SILU) return g * __fdividef(1.f, 1.f + __expf(-g));
  return g * (0.5f * (1.f + erff(g * 0.70710678f)));
}
// act(g) and its derivative
__device__ __forceinline__ void act_both(float g, int act, float& a, float& da) {
  if (act == INB_ACT_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    a = g * s;
    da = s * (1.f + g * (1.f - s));
  } else {
    const float c = 0.5f * (1.f + erff(g * 0.70710678f));
    a = g * c;
    da = c + g * __expf(-0.5f * g * g) * 0.39894228f;
  }
}

// 32 values of one row to `p` (columns [0, n) of them), 16 bytes at a time where the row allows it
template <typename T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[32], int n, bool vec) {
  constexpr int W = 16 / (int)sizeof(T);
#pragma unroll
  for (int i = 0; i < 32; i += W) {
    if (vec && i + W <= n) {
      Pack<T, W> o;
#pragma unroll
      for (int e = 0; e < W; ++e) o.v[e] = from_f<T>(v[i + e]);
      st<T, W>(p + i, o);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (i + e < n) p[i + e] = from_f<T>(v[i + e]);
    }
  }
}

template <typename T>
struct EpiStore {
  T *c0, *c1;        // tiles below m_split, and from it on
  int64_t ld;
  int M, N, m_split;
  bool vec;
  __device__ void operator()(int tm, int tn, int row, uint32_t tmem) const {
    const bool second = tm >= m_split;
    const int r = (second ? tm - m_split : tm) * BM + row, n0 = tn * BN;
    T* c = (second ? c1 : c0) + (int64_t)r * ld + n0;
    for (int j = 0; j < BN && n0 + j < N; j += 32) {
      uint32_t v[32];
      tmem_ld32(tmem + j, v);
      tmem_ld_wait();
      float f[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
      if (r < M) store_row<T>(c + j, f, N - n0 - j, vec);
    }
  }
};

template <typename T>
struct EpiGate {
  T* h;
  float *g, *u;      // NULL: not kept
  int64_t ld;        // a multiple of 8
  int M, F, act;
  __device__ void operator()(int tm, int tn, int row, uint32_t tmem) const {
    const int r = tm * BM + row, n0 = tn * (BN / 2);
    const int64_t at = (int64_t)r * ld + n0;
    for (int j = 0; j < BN / 2 && n0 + j < F; j += 32) {
      uint32_t vg[32], vu[32];
      tmem_ld32(tmem + j, vg);
      tmem_ld32(tmem + BN / 2 + j, vu);
      tmem_ld_wait();
      float fg[32], fu[32], fh[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        fg[i] = __uint_as_float(vg[i]);
        fu[i] = __uint_as_float(vu[i]);
        fh[i] = act_of(fg[i], act) * fu[i];
      }
      if (r < M) {
        store_row<T>(h + at + j, fh, F - n0 - j, true);
        if (g != nullptr) {
          store_row<float>(g + at + j, fg, F - n0 - j, true);
          store_row<float>(u + at + j, fu, F - n0 - j, true);
        }
      }
    }
  }
};

template <typename T>
struct EpiDh {
  T *dg, *du;
  const float *g, *u;
  int64_t ld;        // a multiple of 8; g and u hold whole groups of 4 columns up to it
  int M, F, act;
  __device__ void operator()(int tm, int tn, int row, uint32_t tmem) const {
    const int r = tm * BM + row, n0 = tn * BN;
    const int64_t at = (int64_t)r * ld + n0;
    for (int j = 0; j < BN && n0 + j < F; j += 32) {
      uint32_t v[32];
      tmem_ld32(tmem + j, v);
      float fg[32], fu[32];
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        Pack<float, 4> pg = {}, pu = {};
        if (r < M && n0 + j + i < F) {
          pg = ld_pack(g + at + j + i);
          pu = ld_pack(u + at + j + i);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          fg[i + e] = pg.v[e];
          fu[i + e] = pu.v[e];
        }
      }
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float dh = __uint_as_float(v[i]);
        float a, da;
        act_both(fg[i], act, a, da);
        fg[i] = dh * fu[i] * da;
        fu[i] = dh * a;
      }
      if (r < M) {
        store_row<T>(dg + at + j, fg, F - n0 - j, true);
        store_row<T>(du + at + j, fu, F - n0 - j, true);
      }
    }
  }
  static __device__ __forceinline__ Pack<float, 4> ld_pack(const float* p) { return inb::pol::ld<float, 4>(p); }
};

// ------------------------------------------------------------------------------------------------- operands
// Rows that TMA cannot address (a base or a row stride off 16 bytes) are copied once to padded rows.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const T* src, T* dst, int64_t rows, int cols, int64_t ls, int64_t ldst) {
  const int64_t n = rows * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / cols;
    const int c = (int)(i - r * cols);
    dst[r * ldst + c] = src[r * ls + c];
  }
}

struct Operand {
  const void* p;
  int64_t rows, ld;
  int cols;
};
static int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
static bool addressable(Operand& o) {
  if (o.rows == 1) o.ld = pad8(o.cols);
  return ((uintptr_t)o.p & 15) == 0 && o.ld % 8 == 0;
}
static int64_t packed_bytes(Operand o) {
  return addressable(o) ? 0 : (o.rows * pad8(o.cols) * 2 + 255) / 256 * 256;
}
template <typename T>
static void pack(Operand& o, char*& work, cudaStream_t s) {
  const int64_t b = packed_bytes(o);
  addressable(o);
  if (b == 0) return;
  const int64_t blocks = (o.rows * o.cols + 1023) / 1024, most = (int64_t)sm_count() * 16;
  pack_kernel<T><<<(unsigned)(blocks < most ? blocks : most), 256, 0, s>>>((const T*)o.p, (T*)work, o.rows, o.cols, o.ld,
                                                                         pad8(o.cols));
  o.p = work;
  o.ld = pad8(o.cols);
  work += b;
}

template <typename T, int MAJOR>
static bool map_of(CUtensorMap* m, const Operand& o) {
  return make_map<T>(m, o.p, o.rows, o.cols, o.ld, MAJOR == MAJOR_K ? 128 : 64);
}

template <typename T, int AMAJ, int BMAJ, typename Epi>
static int gemm(const Operand& a0, const Operand& a1, const Operand& b0, const Operand& b1, GemmShape g, const Epi& epi,
                int* status, cudaStream_t s) {
  auto* k = gemm_kernel<T, AMAJ, BMAJ, Epi>;
  // before the maps: their driver call needs a current context, which a fresh thread (autograd's) only has after a
  // runtime call
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, GEMM_SMEM);
  if (e != cudaSuccess) return -100 - (int)e;
  CUtensorMap ma0, ma1, mb0, mb1;
  if (!map_of<T, AMAJ>(&ma0, a0) || !map_of<T, AMAJ>(&ma1, a1) || !map_of<T, BMAJ>(&mb0, b0) || !map_of<T, BMAJ>(&mb1, b1))
    return -6;
  const int64_t tiles = (int64_t)g.tiles_m * g.tiles_n;
  if (tiles > 0x7FFFFFFF) return -2;
  g.band = 16;
  const int grid = (int)(tiles < sm_count() ? tiles : sm_count());
  k<<<grid, GEMM_THREADS, GEMM_SMEM, s>>>(ma0, ma1, mb0, mb1, g, epi, status);
  return launch_status();
}

static int cdiv(int64_t a, int b) { return (int)((a + b - 1) / b); }

struct FfnOperands {
  Operand x, wg, wu, wd, dy, h, dg, du;
};
static FfnOperands operands(const InbFfnArgs& a) {
  FfnOperands o;
  o.x = {a.x, a.N, a.ldx, a.D};
  o.wg = {a.wg, a.F, a.ldwg, a.D};
  o.wu = {a.wu, a.F, a.ldwu, a.D};
  o.wd = {a.wd, a.D, a.ldwd, a.F};
  o.dy = {a.dy, a.N, a.lddy, a.D};
  o.h = {a.h, a.N, a.ldh, a.F};
  o.dg = {a.dg, a.N, a.ldh, a.F};
  o.du = {a.du, a.N, a.ldh, a.F};
  return o;
}
static int64_t ffn_work(const InbFfnArgs& a, bool bwd) {
  const FfnOperands o = operands(a);
  return packed_bytes(o.x) + packed_bytes(o.wg) + packed_bytes(o.wu) + packed_bytes(o.wd) + (bwd ? packed_bytes(o.dy) : 0);
}

template <typename T>
static EpiStore<T> store_to(void* c0, void* c1, int M, int N, int m_split) {
  const bool vec = (((uintptr_t)c0 | (uintptr_t)(c1 ? c1 : c0) | (uintptr_t)N * 2) & 15) == 0;
  return EpiStore<T>{(T*)c0, (T*)c1, N, M, N, m_split, vec};
}

template <typename T>
static int ffn_forward(const InbFfnArgs& a, cudaStream_t s) {
  FfnOperands o = operands(a);
  char* w = (char*)a.work;
  pack<T>(o.x, w, s);
  pack<T>(o.wg, w, s);
  pack<T>(o.wu, w, s);
  pack<T>(o.wd, w, s);
  const int tm = cdiv(a.N, BM);
  GemmShape g = {tm, cdiv(a.F, BN / 2), cdiv(a.D, BK), 0, tm, 1, 0};
  int rc = gemm<T, MAJOR_K, MAJOR_K>(o.x, o.x, o.wg, o.wu, g, EpiGate<T>{(T*)a.h, a.g, a.u, a.ldh, (int)a.N, a.F, a.act},
                                     a.status, s);
  if (rc != 0) return rc;
  g = {tm, cdiv(a.D, BN), cdiv(a.F, BK), 0, tm, 0, 0};
  return gemm<T, MAJOR_K, MAJOR_K>(o.h, o.h, o.wd, o.wd, g, store_to<T>(a.y, nullptr, (int)a.N, a.D, tm), a.status, s);
}

template <typename T>
static int ffn_backward(const InbFfnArgs& a, cudaStream_t s) {
  FfnOperands o = operands(a);
  char* w = (char*)a.work;
  pack<T>(o.x, w, s);
  pack<T>(o.wg, w, s);
  pack<T>(o.wu, w, s);
  pack<T>(o.wd, w, s);
  pack<T>(o.dy, w, s);
  const int tm = cdiv(a.N, BM), tf = cdiv(a.F, BM), td = cdiv(a.D, BM);
  int rc = 0;
  GemmShape g;
  if (a.dx != nullptr || a.dwg != nullptr) {
    g = {tm, cdiv(a.F, BN), cdiv(a.D, BK), 0, tm, 0, 0};
    rc = gemm<T, MAJOR_K, MAJOR_MN>(o.dy, o.dy, o.wd, o.wd, g,
                                    EpiDh<T>{(T*)a.dg, (T*)a.du, a.g, a.u, a.ldh, (int)a.N, a.F, a.act}, a.status, s);
    if (rc != 0) return rc;
  }
  if (a.dx != nullptr) {
    g = {tm, cdiv(a.D, BN), cdiv(a.F, BK), cdiv(a.F, BK), tm, 0, 0};
    rc = gemm<T, MAJOR_K, MAJOR_MN>(o.dg, o.du, o.wg, o.wu, g, store_to<T>(a.dx, nullptr, (int)a.N, a.D, tm), a.status, s);
    if (rc != 0) return rc;
  }
  if (a.dwg != nullptr) {
    g = {2 * tf, cdiv(a.D, BN), cdiv(a.N, BK), 0, tf, 0, 0};
    rc = gemm<T, MAJOR_MN, MAJOR_MN>(o.dg, o.du, o.x, o.x, g, store_to<T>(a.dwg, a.dwu, a.F, a.D, tf), a.status, s);
    if (rc != 0) return rc;
  }
  if (a.dwd != nullptr) {
    g = {td, cdiv(a.F, BN), cdiv(a.N, BK), 0, td, 0, 0};
    rc = gemm<T, MAJOR_MN, MAJOR_MN>(o.dy, o.dy, o.h, o.h, g, store_to<T>(a.dwd, nullptr, a.D, a.F, td), a.status, s);
  }
  return rc;
}

static int ffn_check(const InbFfnArgs* p, bool bwd, bool sizes_only) {
  if (p == nullptr) return -1;
  const InbFfnArgs& a = *p;
  if ((a.dtype != INB_BF16 && a.dtype != INB_F16) || (a.act != INB_ACT_SILU && a.act != INB_ACT_GELU) || a.N < 0 ||
      a.N > INB_MAX_FFN || a.D < 1 || a.D > INB_MAX_FFN || a.F < 1 || a.F > INB_MAX_FFN || a.ldh % 8 != 0 || a.ldh < a.F)
    return -2;
  if (a.N == 0) return 0;
  if (a.x == nullptr || a.wg == nullptr || a.wu == nullptr || a.wd == nullptr) return -3;
  if (sizes_only) return 0;
  if (a.h == nullptr || (((uintptr_t)a.h | (uintptr_t)a.g | (uintptr_t)a.u) & 15) != 0) return -3;
  if (!bwd && (a.y == nullptr || (a.g == nullptr) != (a.u == nullptr))) return -3;
  if (bwd && (a.dy == nullptr || a.g == nullptr || a.u == nullptr || (a.dwg == nullptr) != (a.dwu == nullptr) ||
              ((a.dx != nullptr || a.dwg != nullptr) &&
               (a.dg == nullptr || a.du == nullptr || (((uintptr_t)a.dg | (uintptr_t)a.du) & 15) != 0))))
    return -3;
  if (a.work_bytes < ffn_work(a, bwd) || (a.work_bytes > 0 && ((uintptr_t)a.work & 15) != 0)) return -5;
  return 0;
}

}  // namespace pol
}  // namespace inb

extern "C" int inb_gated_ffn_fwd(const InbFfnArgs* args, void* cuda_stream) {
  const int rc = inb::pol::ffn_check(args, false, false);
  if (rc != 0 || args->N == 0) return rc;
  if (args->dtype == INB_BF16) return inb::pol::ffn_forward<inb::pol::bf16>(*args, (cudaStream_t)cuda_stream);
  return inb::pol::ffn_forward<inb::pol::f16>(*args, (cudaStream_t)cuda_stream);
}

extern "C" int inb_gated_ffn_bwd(const InbFfnArgs* args, void* cuda_stream) {
  const int rc = inb::pol::ffn_check(args, true, false);
  if (rc != 0 || args->N == 0) return rc;
  if (args->dtype == INB_BF16) return inb::pol::ffn_backward<inb::pol::bf16>(*args, (cudaStream_t)cuda_stream);
  return inb::pol::ffn_backward<inb::pol::f16>(*args, (cudaStream_t)cuda_stream);
}

extern "C" int inb_gated_ffn_work(const InbFfnArgs* args, int32_t backward, int64_t* bytes) {
  if (bytes == nullptr) return -1;
  *bytes = 0;
  const int rc = inb::pol::ffn_check(args, backward != 0, true);
  if (rc != 0 || args->N == 0) return rc;
  *bytes = inb::pol::ffn_work(*args, backward != 0);
  return 0;
}
