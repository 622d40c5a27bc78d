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
// kept for the backward pass in the upper 24 bits of fp32: what is rounded off is below 2^-16 of a value, against the operand
// type's 2^-9 or 2^-12; rounding them to the operand type would put two more roundings into dg and du (the weights' gradients then
// are 1.4 times as far from the exact ones).  The whole step runs at the GPU's power limit, where bytes cost time whatever
// bounds a kernel: with all 32 bits it took 2180 us, not 1960 (N = 131072, D = 512, F = 1408, sustained).  h, dg and du are
// rounded to the operand type because the next product multiplies them.
#pragma once
#include <algorithm>
#include <initializer_list>

#include "policy_gemm.cuh"

namespace inb {
namespace pol {

template <int ACT>
__device__ __forceinline__ float act_of(float g) {
  if (ACT == INB_ACT_SILU) return g * __fdividef(1.f, 1.f + __expf(-g));
  return g * (0.5f * (1.f + erff(g * 0.70710678f)));
}
// act(g) and its derivative
template <int ACT>
__device__ __forceinline__ void act_both(float g, float& a, float& da) {
  if (ACT == INB_ACT_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    a = g * s;
    da = s * (1.f + g * (1.f - s));
  } else {
    const float c = 0.5f * (1.f + erff(g * 0.70710678f));
    a = g * c;
    da = c + g * __expf(-0.5f * g * g) * 0.39894228f;
  }
}
template <int N>
__device__ __forceinline__ void buffers_free(const EpiCtx& c) {      // all but this warp's last N sent tiles have left
  if (c.lane == 0) store_wait<N>();
  __syncwarp();
}

struct NoState {};

// C, or (tiles from m_split on) a second C, rounded.  A warp sends its 64 columns as two staged tiles, one a buffer.  The
// second may follow while the first is read out, but the first waits for both of the tile before: where the matrix ends
// within the 64 columns only the first buffer was sent, so the last group in flight need not be the other buffer's.
template <typename T, int CG>
struct EpiStore {
  using State = NoState;
  T *c0, *c1;
  int M, N, m_split;
  bool tma;
  __device__ void begin(const EpiCtx&, State&) const {}
  __device__ void operator()(const EpiCtx& c, State&, const CUtensorMap* o0, const CUtensorMap* o1) const {
    constexpr int COLS = BN / EPI_COLS;
    static_assert(COLS / 32 == EPI_BUFS, "a staged tile a buffer");
    const bool second = c.tm >= m_split;
    const int r0 = (second ? c.tm - m_split : c.tm) * Gemm<CG>::TM + (c.row & ~31), n0 = c.tn * BN + c.part * COLS;
    const uint32_t acc = c.tmem + c.part * COLS;
#pragma unroll
    for (int b = 0; b < COLS / 32; ++b) {
      if (n0 + b * 32 >= N) break;
      float v[2][16];
      tmem_ld16(acc + b * 32, v[0]);
      tmem_ld16(acc + b * 32 + 16, v[1]);
      if (tma && b == 0)
        buffers_free<0>(c);
      else if (tma)
        buffers_free<EPI_BUFS - 1>(c);
      tmem_ld_wait();
      stage16<T>(c.stage_ptr + b * EPI_BUF, c.lane, 0, v[0]);
      stage16<T>(c.stage_ptr + b * EPI_BUF, c.lane, 16, v[1]);
      send_stage<T>(tma ? (second ? o1 : o0) : nullptr, second ? c1 : c0, N, M, N, r0, n0 + b * 32, c, b);
    }
  }
};

// One part of k of a tile, fp32: [item][column group][row][4]
template <int CG>
struct EpiPartial {
  using State = NoState;
  float* part;
  __device__ void begin(const EpiCtx&, State&) const {}
  __device__ void operator()(const EpiCtx& c, State&, const CUtensorMap*, const CUtensorMap*) const {
    constexpr int COLS = BN / EPI_COLS;
    float* p = part + (((int64_t)c.item * (BN / 4) + c.part * (COLS / 4)) * Gemm<CG>::TM + c.row) * 4;
#pragma unroll
    for (int q = 0; q < COLS; q += 16) {
      float v[16];
      tmem_ld16(c.tmem + c.part * COLS + q, v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(p + (int64_t)(q / 4 + i) * Gemm<CG>::TM * 4) =
            make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
  }
};
// Adds the parts of every tile in order.  A block takes 32 rows x 64 columns of a tile: it reads with a row to a lane, as
// the parts lie, and writes with two columns to a lane, as the result does.
template <typename T, int CG>
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* part, const GemmShape g, T* c0, T* c1, int M, int N,
                                                        bool pairs) {
  __shared__ float sm[32][65];
  constexpr int TM = Gemm<CG>::TM;
  const int tiles = g.tiles_m * g.tiles_n, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int tm, tn;
  tile_at(g, blockIdx.x, tm, tn);
  const bool second = tm >= g.m_split;
  const int r0 = (second ? tm - g.m_split : tm) * TM + blockIdx.z * 32, n0 = tn * BN + blockIdx.y * 64;
  if (r0 >= M || n0 >= N) return;
  float4 s[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int k = 0; k < g.splits; ++k) {
    const float* p = part + ((((int64_t)k * tiles + blockIdx.x) * (BN / 4) + blockIdx.y * 16 + warp * 2) * TM +
                             blockIdx.z * 32 + lane) * 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(p + i * TM * 4);
      s[i].x += v.x, s[i].y += v.y, s[i].z += v.z, s[i].w += v.w;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float* d = &sm[lane][warp * 8 + i * 4];
    d[0] = s[i].x, d[1] = s[i].y, d[2] = s[i].z, d[3] = s[i].w;
  }
  __syncthreads();
  const int col = n0 + 2 * lane;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = warp * 4 + i;
    if (r0 + r >= M || col >= N) continue;
    T* d = (second ? c1 : c0) + (int64_t)(r0 + r) * N + col;
    Pack<T, 2> o;
    down2(make_float2(sm[r][2 * lane], sm[r][2 * lane + 1]), o.v[0], o.v[1]);
    if (pairs) {
      st<T, 2>(d, o);
    } else {
      d[0] = o.v[0];
      if (col + 1 < N) d[1] = o.v[1];
    }
  }
}

// h = act(g) u of 128 columns, 32 a warp; g and u kept as blocked() says (NULL: not kept)
template <typename T, int CG, int ACT>
struct EpiGate {
  using State = NoState;
  uint4 *g, *u;
  int M, F, groups;
  __device__ void begin(const EpiCtx&, State&) const {}
  __device__ void operator()(const EpiCtx& c, State&, const CUtensorMap* o0, const CUtensorMap*) const {
    constexpr int COLS = BN / 2 / EPI_COLS;
    static_assert(COLS == 32, "one staged tile a warp");
    const int r0 = c.tm * Gemm<CG>::TM + (c.row & ~31), r = r0 + c.lane, n0 = c.tn * (BN / 2) + c.part * COLS;
    if (n0 >= F) return;
    // Either buffer would do: both are free once buffers_free<0> returns.  Taking them in turn is worth 5 us of 2005 (a training
    // step, N = 131072, D = 512, F = 1408); waiting for one alone would need a count of the tiles that this warp has sent.
    const int buf = c.tn & 1;
    float vg[2][16], vu[2][16];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      tmem_ld16(c.tmem + c.part * COLS + 16 * q, vg[q]);
      tmem_ld16(c.tmem + BN / 2 + c.part * COLS + 16 * q, vu[q]);
    }
    buffers_free<0>(c);
    tmem_ld_wait();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float vh[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) vh[i] = act_of<ACT>(vg[q][i]) * vu[q][i];
      stage16<T>(c.stage_ptr + buf * EPI_BUF, c.lane, 16 * q, vh);
    }
    send_stage<T>(o0, (T*)nullptr, 0, M, F, r0, n0, c, buf);
    if (g == nullptr || r >= M) return;
    // after the staged tile has gone: its fence would wait for these stores.
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int cg = (n0 >> 4) + q;
      if (cg >= groups) break;
      const int64_t at = blocked(r, cg, groups);
      const Kept16 kg = keep16(vg[q]), ku = keep16(vu[q]);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        g[at + i * 128] = kg.w[i];
        u[at + i * 128] = ku.w[i];
      }
    }
  }
};

// dg = dh u act'(g), du = dh act(g) of 256 columns, 64 a warp
template <typename T, int CG, int ACT>
struct EpiDh {
  struct State {
    Kept16 g, u;                    // the next 16 columns, on their way while these are worked on
  };
  const uint4 *g, *u;
  int M, F, groups;
  __device__ __forceinline__ void fetch(State& s, int r, int col) const {
    const int64_t at = blocked(r, col >> 4, groups);
    const bool in = r < M && (col >> 4) < groups;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      s.g.w[i] = in ? g[at + i * 128] : make_uint4(0, 0, 0, 0);
      s.u.w[i] = in ? u[at + i * 128] : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ void begin(const EpiCtx& c, State& s) const {
    fetch(s, c.tm * Gemm<CG>::TM + c.row, c.tn * BN + c.part * (BN / EPI_COLS));
  }
  __device__ void operator()(const EpiCtx& c, State& s, const CUtensorMap* o0, const CUtensorMap* o1) const {
    constexpr int COLS = BN / EPI_COLS;
    const int r0 = c.tm * Gemm<CG>::TM + (c.row & ~31), r = r0 + c.lane, n0 = c.tn * BN + c.part * COLS;
    const uint32_t acc = c.tmem + c.part * COLS;
#pragma unroll
    for (int b = 0; b < COLS / 32; ++b) {
      if (n0 + b * 32 >= F) break;
#pragma unroll
      for (int q = 0; q < 32; q += 16) {
        float v[16], fg[16], fu[16];
        tmem_ld16(acc + b * 32 + q, v);
        kept16(s.g, fg);
        kept16(s.u, fu);
        if (b * 32 + q + 16 < COLS) fetch(s, r, n0 + b * 32 + q + 16);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float a, da;
          act_both<ACT>(fg[i], a, da);
          fg[i] = v[i] * fu[i] * da;
          fu[i] = v[i] * a;
        }
        if (q == 0) buffers_free<0>(c);
        stage16<T>(c.stage_ptr, c.lane, q, fg);
        stage16<T>(c.stage_ptr + EPI_BUF, c.lane, q, fu);
      }
      send_stage<T>(o0, (T*)nullptr, 0, M, F, r0, n0 + b * 32, c, 0);
      send_stage<T>(o1, (T*)nullptr, 0, M, F, r0, n0 + b * 32, c, 1);
    }
  }
};

// ------------------------------------------------------------------------------------------------- operands
// Rows that TMA cannot address (a base or a row stride off 16 bytes) are copied once to padded rows, all of a call's in one
// launch: blockIdx.z is the matrix.
struct PackJobs {
  const void* src[5];
  void* dst[5];
  int64_t rows[5], ls[5];
  int cols[5];
  int n;
};
inline int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
// A thread makes 8 elements of a row from the aligned words that hold them (rows start on any element: every other one of
// an odd stride half a word late).  Each word read holds at least one element of the row.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const PackJobs j) {
  const int m = blockIdx.z, cols = j.cols[m];
  const uint32_t per_row = (cols + 7) / 8;
  const int64_t all = j.rows[m] * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row;
    const int c = (int)(i - r * per_row) * 8, n = min(8, cols - c);
    const uintptr_t at = (uintptr_t)((const uint16_t*)j.src[m] + r * j.ls[m] + c);
    const uint32_t* w = (const uint32_t*)(at & ~(uintptr_t)3);
    const int shift = at & 2 ? 16 : 0, words = (n * 2 + (shift ? 2 : 0) + 3) / 4;
    uint32_t v[5], o[4];
#pragma unroll
    for (int k = 0; k < 5; ++k) v[k] = k < words ? w[k] : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = __funnelshift_r(v[k], v[k + 1], shift);
    reinterpret_cast<uint4*>((uint16_t*)j.dst[m] + r * per_row * 8)[c / 8] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

struct Operand {
  const void* p;
  int64_t rows, ld;
  int cols;
};
inline int cdiv(int64_t a, int b) { return (int)((a + b - 1) / b); }
inline bool addressable(Operand& o) {
  if (o.rows == 1) o.ld = pad8(o.cols);
  return ((uintptr_t)o.p & 15) == 0 && o.ld % 8 == 0;
}
inline int64_t packed_bytes(Operand o) {
  return addressable(o) ? 0 : (o.rows * pad8(o.cols) * 2 + 255) / 256 * 256;
}
template <typename T>
void pack(std::initializer_list<Operand*> os, char*& work, cudaStream_t s) {
  PackJobs j = {};
  int64_t most = 0;
  for (Operand* o : os) {
    const int64_t b = packed_bytes(*o);
    addressable(*o);
    if (b == 0) continue;
    j.src[j.n] = o->p, j.dst[j.n] = work, j.rows[j.n] = o->rows, j.cols[j.n] = o->cols, j.ls[j.n] = o->ld;
    ++j.n;
    most = std::max(most, o->rows * (pad8(o->cols) / 8));
    o->p = work;
    o->ld = pad8(o->cols);
    work += b;
  }
  if (j.n == 0) return;
  const unsigned blocks = (unsigned)std::min<int64_t>((most + 255) / 256, (int64_t)sm_count() * 8);
  pack_kernel<T><<<dim3(blocks, 1, j.n), 256, 0, s>>>(j);
}

// ------------------------------------------------------------------------------------------------- plans
// How a product of M (or twice M: `twin`) x N over kb slices is cut: blocks a tile and parts of k.
struct Plan {
  int cg, splits;
  int64_t part_floats;
};
// An estimate of a plan's time in us: waves of tiles, each its slices (512 cycles of the tensor cores) and a fill and
// drain; single blocks run their products slower than pairs; parts are written and read once.
inline double plan_time(int64_t M, int N, int kb, bool twin, int cg, int splits, int bn) {
  const int64_t tiles = (int64_t)cdiv(M, BM * cg) * (twin ? 2 : 1) * cdiv(N, bn);
  const int64_t waves = (tiles * splits * cg + sm_count() - 1) / sm_count();
  double t = waves * (cdiv(kb, splits) * 0.3 * (cg == 1 ? 1.2 : 1.0) + 2.0);
  if (splits > 1) t += 3.0 + (double)tiles * splits * BM * cg * BN * 8 / 5e6;
  return t;
}
inline Plan plan(int64_t M, int N, int kb, bool twin, bool may_split, int bn) {
  Plan best = {1, 1, 0};
  double least = 1e30;
  for (int cg = 1; cg <= 2; ++cg)
    for (int s = 1; s <= (may_split ? 16 : 1); ++s) {
      if (s > 1 && kb / s < 4) break;
      const int64_t parts = s == 1 ? 0 : (int64_t)cdiv(M, BM * cg) * (twin ? 2 : 1) * cdiv(N, bn) * s * BM * cg * BN;
      if (parts > (64 << 20)) break;
      const double t = plan_time(M, N, kb, twin, cg, s, bn);
      if (t < least) {
        least = t;
        best = {cg, s, parts};
      }
    }
  return best;
}

template <typename T, int MAJOR>
bool map_of(CUtensorMap* m, const Operand& o) {
  return make_map<T>(m, o.p, o.rows, o.cols, o.ld, 64, MAJOR == MAJOR_K ? 128 : 64);
}
template <typename T>
bool out_map(CUtensorMap* m, const Operand& o) {
  return make_map<T>(m, o.p, o.rows, o.cols, o.ld, 32, 32);
}

struct GemmMaps {
  CUtensorMap a0, a1, b0, b1, o0, o1;
};

template <typename T, int CG, int AMAJ, int BMAJ, typename Epi>
int gemm_launch(const GemmMaps& m, GemmShape g, const Epi& epi, int* status, cudaStream_t s) {
  auto* k = gemm_kernel<T, CG, AMAJ, BMAJ, Epi>;
  cudaError_t e = allow_smem<KernelKey<gemm_kernel<T, CG, AMAJ, BMAJ, Epi>>>((const void*)k, Gemm<CG>::SMEM);
  if (e != cudaSuccess) return -100 - (int)e;
  const int64_t items = (int64_t)g.tiles_m * g.tiles_n * g.splits, most = sm_count() / CG;
  if (items > 0x3FFFFFFF) return -2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items < most ? items : most) * CG);
  cfg.blockDim = dim3(GEMM_THREADS);
  cfg.dynamicSmemBytes = Gemm<CG>::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = CG;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = CG > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, k, m.a0, m.a1, m.b0, m.b1, m.o0, m.o1, g, epi, status);
  return e == cudaSuccess ? 0 : -100 - (int)e;
}

// Makes the current device's context current to this thread: the driver call that makes tensor maps needs it, and a fresh
// thread (autograd's) has none before a runtime call like this one, which a graph capture allows
template <typename T>
bool bind_context() {
  return allow_smem<KernelKey<pack_kernel<T>>>((const void*)pack_kernel<T>, 0) == cudaSuccess;
}

template <typename T, int AMAJ, int BMAJ>
bool operand_maps(GemmMaps& m, const Operand& a0, const Operand& a1, const Operand& b0, const Operand& b1) {
  if (!map_of<T, AMAJ>(&m.a0, a0) || !map_of<T, BMAJ>(&m.b0, b0)) return false;
  m.a1 = m.a0;
  m.b1 = m.b0;
  // the two weights may be views that start at one address with strides of their own
  auto equal = [](const Operand& p, const Operand& q) { return p.p == q.p && p.ld == q.ld; };
  return (equal(a1, a0) || map_of<T, AMAJ>(&m.a1, a1)) && (equal(b1, b0) || map_of<T, BMAJ>(&m.b1, b1));
}

// A product whose result is stored: C (and, twin, a second C under it, from a1)
template <typename T, int CG, int AMAJ, int BMAJ>
int product_cg(const GemmMaps& m, int64_t M, int N, int kb0, int kb1, bool twin, const Plan& pl, void* c0, void* c1, bool tma,
               float* part, int* status, cudaStream_t s) {
  const int tm = cdiv(M, BM * CG), kb = kb0 + kb1, kbs = cdiv(kb, pl.splits);
  GemmShape g = {twin ? 2 * tm : tm, cdiv(N, BN), kb0, kb1, tm, 0, 16 / CG, cdiv(kb, kbs), kbs};
  if (g.splits == 1)
    return gemm_launch<T, CG, AMAJ, BMAJ>(m, g, EpiStore<T, CG>{(T*)c0, (T*)c1, (int)M, N, tm, tma}, status, s);
  const int rc = gemm_launch<T, CG, AMAJ, BMAJ>(m, g, EpiPartial<CG>{part}, status, s);
  if (rc != 0) return rc;
  const bool pairs = (((uintptr_t)c0 | (uintptr_t)(c1 ? c1 : c0) | (uintptr_t)N * 2) & 3) == 0;
  sum_parts_kernel<T, CG><<<dim3(g.tiles_m * g.tiles_n, BN / 64, BM * CG / 32), 256, 0, s>>>(part, g, (T*)c0, (T*)c1, (int)M,
                                                                                           N, pairs);
  return launch_status();
}
template <typename T, int AMAJ, int BMAJ>
int product(const Operand& a0, const Operand& a1, const Operand& b0, const Operand& b1, int64_t M, int N, int64_t k, bool two_k,
            bool twin, void* c0, void* c1, float* part, int* status, cudaStream_t s) {
  GemmMaps m;
  if (!operand_maps<T, AMAJ, BMAJ>(m, a0, a1, b0, b1)) return -6;
  Operand o0 = {c0, M, N, N}, o1 = {c1 ? c1 : c0, M, N, N};
  const bool tma = addressable(o0) && addressable(o1) && out_map<T>(&m.o0, o0) && out_map<T>(&m.o1, o1);
  if (!tma) m.o0 = m.o1 = m.a0;
  const int kb = cdiv(k, BK);
  const Plan pl = plan(M, N, two_k ? 2 * kb : kb, twin, true, BN);
  if (pl.cg == 1)
    return product_cg<T, 1, AMAJ, BMAJ>(m, M, N, kb, two_k ? kb : 0, twin, pl, c0, c1, tma, part, status, s);
  return product_cg<T, 2, AMAJ, BMAJ>(m, M, N, kb, two_k ? kb : 0, twin, pl, c0, c1, tma, part, status, s);
}

struct FfnOperands {
  Operand x, wg, wu, wd, dy, h, dg, du;
};
inline FfnOperands operands(const InbFfnArgs& a) {
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
inline int64_t pack_bytes(const InbFfnArgs& a, bool bwd) {
  const FfnOperands o = operands(a);
  return packed_bytes(o.x) + packed_bytes(o.wg) + packed_bytes(o.wu) + packed_bytes(o.wd) + (bwd ? packed_bytes(o.dy) : 0);
}
// packed operands, then the largest product's parts
inline int64_t ffn_work(const InbFfnArgs& a, bool bwd) {
  int64_t parts = 0;
  auto need = [&](int64_t M, int N, int64_t k, bool two_k, bool twin) {
    const int64_t p = plan(M, N, (two_k ? 2 : 1) * cdiv(k, BK), twin, true, BN).part_floats;
    parts = p > parts ? p : parts;
  };
  if (!bwd) {
    need(a.N, a.D, a.F, false, false);
  } else {
    need(a.N, a.D, a.F, true, false);
    need(a.F, a.D, a.N, false, true);
    need(a.D, a.F, a.N, false, false);
  }
  return pack_bytes(a, bwd) + parts * 4;
}

// The two products with an activation in their epilogue
template <typename T, int CG, int ACT>
int gate_product(const GemmMaps& m, const InbFfnArgs& a, int kb, cudaStream_t s) {
  const int tm = cdiv(a.N, BM * CG);
  const GemmShape g = {tm, cdiv(a.F, BN / 2), kb, 0, tm, 1, 16 / CG, 1, kb};
  return gemm_launch<T, CG, MAJOR_K, MAJOR_K>(m, g, EpiGate<T, CG, ACT>{(uint4*)a.g, (uint4*)a.u, (int)a.N, a.F, cdiv(a.F, 16)}, a.status, s);
}
template <typename T, int CG, int ACT>
int dh_product(const GemmMaps& m, const InbFfnArgs& a, int kb, cudaStream_t s) {
  const int tm = cdiv(a.N, BM * CG);
  const GemmShape g = {tm, cdiv(a.F, BN), kb, 0, tm, 0, 16 / CG, 1, kb};
  return gemm_launch<T, CG, MAJOR_K, MAJOR_MN>(m, g, EpiDh<T, CG, ACT>{(const uint4*)a.g, (const uint4*)a.u, (int)a.N, a.F, cdiv(a.F, 16)}, a.status, s);
}

template <typename T>
int ffn_forward(const InbFfnArgs& a, cudaStream_t s) {
  if (!bind_context<T>()) return -6;
  FfnOperands o = operands(a);
  char* w = (char*)a.work;
  pack<T>({&o.x, &o.wg, &o.wu, &o.wd}, w, s);
  const int kb = cdiv(a.D, BK);
  GemmMaps m;
  if (!operand_maps<T, MAJOR_K, MAJOR_K>(m, o.x, o.x, o.wg, o.wu) || !out_map<T>(&m.o0, o.h)) return -6;
  m.o1 = m.o0;
  const int cg = plan(a.N, a.F, kb, false, false, BN / 2).cg;
  int rc;
  if (a.act == INB_ACT_SILU)
    rc = cg == 1 ? gate_product<T, 1, INB_ACT_SILU>(m, a, kb, s) : gate_product<T, 2, INB_ACT_SILU>(m, a, kb, s);
  else
    rc = cg == 1 ? gate_product<T, 1, INB_ACT_GELU>(m, a, kb, s) : gate_product<T, 2, INB_ACT_GELU>(m, a, kb, s);
  if (rc != 0) return rc;
  return product<T, MAJOR_K, MAJOR_K>(o.h, o.h, o.wd, o.wd, a.N, a.D, a.F, false, false, a.y, nullptr, (float*)w, a.status, s);
}

template <typename T>
int ffn_backward(const InbFfnArgs& a, cudaStream_t s) {
  if (!bind_context<T>()) return -6;
  FfnOperands o = operands(a);
  char* w = (char*)a.work;
  pack<T>({&o.x, &o.wg, &o.wu, &o.wd, &o.dy}, w, s);
  float* part = (float*)w;
  int rc = 0;
  if (a.dx != nullptr || a.dwg != nullptr) {
    const int kb = cdiv(a.D, BK);
    GemmMaps m;
    if (!operand_maps<T, MAJOR_K, MAJOR_MN>(m, o.dy, o.dy, o.wd, o.wd) || !out_map<T>(&m.o0, o.dg) ||
        !out_map<T>(&m.o1, o.du))
      return -6;
    const int cg = plan(a.N, a.F, kb, false, false, BN).cg;
    if (a.act == INB_ACT_SILU)
      rc = cg == 1 ? dh_product<T, 1, INB_ACT_SILU>(m, a, kb, s) : dh_product<T, 2, INB_ACT_SILU>(m, a, kb, s);
    else
      rc = cg == 1 ? dh_product<T, 1, INB_ACT_GELU>(m, a, kb, s) : dh_product<T, 2, INB_ACT_GELU>(m, a, kb, s);
    if (rc != 0) return rc;
  }
  if (a.dx != nullptr) {
    rc = product<T, MAJOR_K, MAJOR_MN>(o.dg, o.du, o.wg, o.wu, a.N, a.D, a.F, true, false, a.dx, nullptr, part, a.status, s);
    if (rc != 0) return rc;
  }
  if (a.dwg != nullptr) {
    rc = product<T, MAJOR_MN, MAJOR_MN>(o.dg, o.du, o.x, o.x, a.F, a.D, a.N, false, true, a.dwg, a.dwu, part, a.status, s);
    if (rc != 0) return rc;
  }
  if (a.dwd != nullptr)
    rc = product<T, MAJOR_MN, MAJOR_MN>(o.dy, o.dy, o.h, o.h, a.D, a.F, a.N, false, false, a.dwd, nullptr, part, a.status, s);
  return rc;
}

int ffn_bf16(const InbFfnArgs& a, bool bwd, cudaStream_t s);
int ffn_f16(const InbFfnArgs& a, bool bwd, cudaStream_t s);
int ffn_rows_any(const InbFfnArgs& a, cudaStream_t s);
// Whether a call is one of few rows that keeps nothing for a backward pass (policy_ffn_rows.cu)
inline bool few_rows(const InbFfnArgs& a, bool bwd) { return !bwd && a.g == nullptr && a.N <= INB_FFN_ROWS; }

}  // namespace pol
}  // namespace inb
