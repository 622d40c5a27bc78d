// gated_ffn on few rows (serving): both products stream the weights once, past a handful of rows that stay on chip.
//
// With N rows a weight takes part in N multiply-adds, so up to INB_FFN_ROWS rows the time is that of reading 3 D F weights
// from DRAM.  A block takes two groups of 16 weight rows (16 rows of Wg and the same of Wu; or 32 rows of Wd), its eight
// warps take turns along k, and where that leaves SMs idle a cluster of up to 8 blocks shares one k.  A thread copies 16
// bytes of a weight row at a time (cp.async, through its own places of a ring in shared memory: 96 KB on their way to an
// SM) and gives them to the m16n8k16 matrix instruction as they are: the sum over k may run in any order, so the 8
// consecutive elements a thread holds are simply declared to be the k slots that the instruction expects of it, for
// weights and activations alike, and nothing is exchanged.  (128-row tcgen05 tiles would
// spend 3/4 of their operand on padding here and gain nothing: the tensor cores idle either way.)  The warps' and the
// blocks' partial sums meet in shared memory, in a fixed order.
//
// For up to 8 rows h passes between the two products as hi + lo, two 16-bit values whose sum is h to 2^-16 or better: the
// second product runs both through the same weight registers, so h costs neither precision nor time (a single row's
// outputs would show its rounding).  From 9 rows on the second half of h's bytes does cost time (16 rows, D = 4096,
// F = 11264: 77 us against 65) and h is rounded as it is in the large products.  The second kernel is launched while
// the first runs, loads its first weights, and waits before it reads h.
#include <cooperative_groups.h>

#include "policy_ffn.cuh"

namespace cg = cooperative_groups;

namespace inb {
namespace pol {

constexpr int ROWS_WARPS = 8, ROWS_K = 32;      // k of one step of a warp: 4 threads x 8 elements

struct RowsArgs {
  const void *w0, *w1;        // first rows of the two groups' matrices
  int64_t ld0, ld1;
  const void *x, *x_lo;       // activations [N, K], and their low parts or NULL
  int64_t ldx;
  void *out, *out_lo;         // [N, M]
  int64_t ldo;
  int N, M, K;                // M: output columns
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, bf16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, f16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 elements from p, of which the first `n` exist
template <typename T>
__device__ __forceinline__ uint4 load8(const T* p, int n) {
  Pack<uint16_t, 8> e;
#pragma unroll
  for (int i = 0; i < 8; ++i) e.v[i] = i < n ? reinterpret_cast<const uint16_t*>(p)[i] : 0;
  return *reinterpret_cast<uint4*>(&e);
}
// 16 bytes into shared memory, the first `left` elements from p and zeros after them
__device__ __forceinline__ void copy16(uint32_t dst, const void* p, int left) {
  const int bytes = left >= 8 ? 16 : (left > 0 ? 2 * left : 0);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p), "r"(bytes) : "memory");
}

// A step of the sum: 4 weight pieces against NT pieces of x (and their low parts)
template <typename T, int NT, bool LO>
__device__ __forceinline__ void rows_step(float (&acc)[2][NT][4], const uint4 (&v)[4], const uint4 (&x)[LO ? 2 : 1][NT]) {
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int p = 0; p < (LO ? 2 : 1); ++p)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mma_16816(acc[i][j], v[2 * i].x, v[2 * i + 1].x, v[2 * i].y, v[2 * i + 1].y, x[p][j].x, x[p][j].y, T());
        mma_16816(acc[i][j], v[2 * i].z, v[2 * i + 1].z, v[2 * i].w, v[2 * i + 1].w, x[p][j].z, x[p][j].w, T());
      }
}

template <int NT, bool GATE>
struct RowsRing {
  static constexpr bool LO = !GATE && NT == 1;                     // x has low parts
  static constexpr int XS = LO ? 2 : 1;
  static constexpr int PIECES = 4 + NT * XS;                       // 16-byte pieces of one step in a thread
  static constexpr int S = NT == 4 ? 3 : 4;
  static constexpr int BYTES = S * PIECES * 16 * 32 * ROWS_WARPS;
  static constexpr int BLOCKS = NT == 4 ? 1 : 2;                   // on an SM: with the partial sums a block of NT = 4 has 132 KB
};

// NT: groups of 8 rows of x.  GATE: the two groups are g and u of the same columns, out = act(g) u (NT = 1: as hi + lo); else they
// are 32 columns of the output.  VEC: every row starts on 16 bytes.
template <typename T, int NT, bool VEC, bool GATE, int ACT>
__global__ void __launch_bounds__(32 * ROWS_WARPS, RowsRing<NT, GATE>::BLOCKS) ffn_rows_kernel(const RowsArgs a, int ranks) {
  __shared__ float part[ROWS_WARPS][2][16][8 * NT + 1];
  extern __shared__ __align__(16) unsigned char ring[];
  using Rg = RowsRing<NT, GATE>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
  const int rank = blockIdx.x % ranks, m0 = blockIdx.x / ranks * (GATE ? 16 : 32);
  const T* w[4];        // this thread's weight rows: r and r + 8 of both groups
  bool on[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + r + 8 * (i & 1) + (GATE ? 0 : 16 * (i >> 1));
    on[i] = m < a.M;
    w[i] = (const T*)(i < 2 ? a.w0 : a.w1) + (int64_t)(on[i] ? m : 0) * (i < 2 ? a.ld0 : a.ld1);
  }
  float acc[2][NT][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
  const int start = (rank * ROWS_WARPS + warp) * ROWS_K + q * 8, stride = ranks * ROWS_WARPS * ROWS_K;
  if constexpr (VEC) {
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring) + threadIdx.x * 16;
    constexpr int PIECE = 16 * 32 * ROWS_WARPS, SLOT = Rg::PIECES * PIECE;
    auto fetch_w = [&](int slot, int k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int left = on[i] ? a.K - k : 0;
        copy16(mine + slot * SLOT + i * PIECE, left > 0 ? w[i] + k : w[i], left);
      }
    };
    auto fetch_x = [&](int slot, int k) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int n = j * 8 + r, left = n < a.N ? a.K - k : 0;
        const int64_t at = left > 0 ? (int64_t)n * a.ldx + k : 0;
        copy16(mine + slot * SLOT + (4 + j) * PIECE, (const T*)a.x + at, left);
        if (Rg::LO) copy16(mine + slot * SLOT + (4 + NT + j) * PIECE, (const T*)a.x_lo + at, left);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int ahead = start;
#pragma unroll
    for (int i = 0; i < Rg::S - 1; ++i) fetch_w(i, start + i * stride);
    if (!GATE) asm volatile("griddepcontrol.wait;" ::: "memory");      // h of the first kernel
#pragma unroll
    for (int i = 0; i < Rg::S - 1; ++i, ahead += stride) fetch_x(i, ahead);
    int slot = 0;
    for (int k = start; k - q * 8 < a.K; k += stride, ahead += stride) {
      asm volatile("cp.async.wait_group %0;" ::"n"(Rg::S - 2) : "memory");
      const unsigned char* p = ring + threadIdx.x * 16 + slot * SLOT;
      uint4 v[4], x[Rg::XS][NT];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4*>(p + i * PIECE);
#pragma unroll
      for (int i = 0; i < Rg::XS; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) x[i][j] = *reinterpret_cast<const uint4*>(p + (4 + i * NT + j) * PIECE);
      const int next = slot == 0 ? Rg::S - 1 : slot - 1;               // the place read in the last turn
      fetch_w(next, ahead);
      fetch_x(next, ahead);
      slot = slot == Rg::S - 1 ? 0 : slot + 1;
      rows_step<T, NT, Rg::LO>(acc, v, x);
    }
  } else {
    if (!GATE) asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int k = start; k - q * 8 < a.K; k += stride) {
      uint4 v[4], x[Rg::XS][NT];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = load8(w[i] + k, on[i] ? a.K - k : 0);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int n = j * 8 + r, left = n < a.N ? a.K - k : 0;
        x[0][j] = load8((const T*)a.x + (int64_t)n * a.ldx + k, left);
        if constexpr (Rg::LO) x[1][j] = load8((const T*)a.x_lo + (int64_t)n * a.ldx + k, left);
      }
      rows_step<T, NT, Rg::LO>(acc, v, x);
    }
  }
  if (GATE) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[warp][i][r + 8 * (e >> 1)][j * 8 + 2 * q + (e & 1)] = acc[i][j][e];
  __syncthreads();
  // the block's sums, into its first warp's place
  for (int i = threadIdx.x; i < 2 * 16 * 8 * NT; i += 32 * ROWS_WARPS) {
    const int g = i / (16 * 8 * NT), m = i / (8 * NT) % 16, n = i % (8 * NT);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < ROWS_WARPS; ++k) s += part[k][g][m][n];
    part[0][g][m][n] = s;
  }
  if (ranks > 1) {
    cg::this_cluster().sync();
    if (rank != 0) {
      cg::this_cluster().sync();        // the first block has read this one's sums
      return;
    }
  } else {
    __syncthreads();
  }
  auto total = [&](int g, int m, int n) {
    float s = part[0][g][m][n];
    for (int k = 1; k < ranks; ++k) s += *cg::this_cluster().map_shared_rank(&part[0][g][m][n], k);
    return s;
  };
  if (GATE) {
    for (int i = threadIdx.x; i < 16 * 8 * NT; i += 32 * ROWS_WARPS) {
      const int m = i & 15, n = i >> 4;
      if (n < a.N && m0 + m < a.M) {
        const float h = act_of<ACT>(total(0, m, n)) * total(1, m, n);
        const T hi = from_f<T>(h);
        const int64_t at = (int64_t)n * a.ldo + m0 + m;
        ((T*)a.out)[at] = hi;
        // what hi left out (of an infinite hi nothing: inf - inf would be NaN)
        if (NT == 1) ((T*)a.out_lo)[at] = from_f<T>(isfinite(to_f(hi)) ? h - to_f(hi) : 0.f);
      }
    }
  } else {
    for (int i = threadIdx.x; i < 32 * 8 * NT; i += 32 * ROWS_WARPS) {
      const int m = i & 31, n = i >> 5;
      if (n < a.N && m0 + m < a.M) ((T*)a.out)[(int64_t)n * a.ldo + m0 + m] = from_f<T>(total(m >> 4, m & 15, n));
    }
  }
  if (ranks > 1) cg::this_cluster().sync();
}

template <typename T, int NT, bool VEC, bool GATE, int ACT>
static int rows_launch(const RowsArgs& a, cudaStream_t s) {
  using Rg = RowsRing<NT, GATE>;
  const int blocks = cdiv(a.M, GATE ? 16 : 32), smem = VEC ? Rg::BYTES : 0;
  auto* k = ffn_rows_kernel<T, NT, VEC, GATE, ACT>;
  // blocks of one k: enough for what an SM holds while a warp keeps the steps of a ring (planned for two blocks of NT = 4 an
  // SM, 32 rows at D = 4096, F = 11264 took 110 us, not 94: the second product came in four waves, not two)
  int ranks = 1;
  while (ranks < 8 && blocks * ranks < Rg::BLOCKS * sm_count() && a.K / (2 * ranks * ROWS_WARPS) >= ROWS_K * Rg::S) ranks *= 2;
  cudaError_t e = allow_smem<KernelKey<ffn_rows_kernel<T, NT, VEC, GATE, ACT>>>((const void*)k, smem);
  if (e != cudaSuccess) return -100 - (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(blocks * ranks));
  cfg.blockDim = dim3(32 * ROWS_WARPS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = GATE ? 1 : 2;
  e = cudaLaunchKernelEx(&cfg, k, a, ranks);
  return e == cudaSuccess ? 0 : -100 - (int)e;
}
template <typename T, int NT, bool GATE, int ACT>
static int rows_vec(const RowsArgs& a, cudaStream_t s) {
  const uint64_t m = (uintptr_t)a.w0 | (uintptr_t)a.w1 | (uintptr_t)a.x | (uint64_t)(a.ld0 | a.ld1 | a.ldx) * 2;
  return (m & 15) == 0 ? rows_launch<T, NT, true, GATE, ACT>(a, s) : rows_launch<T, NT, false, GATE, ACT>(a, s);
}
template <typename T, bool GATE, int ACT>
static int rows_go(const RowsArgs& a, cudaStream_t s) {
  if (a.N <= 8) return rows_vec<T, 1, GATE, ACT>(a, s);
  if (a.N <= 16) return rows_vec<T, 2, GATE, ACT>(a, s);
  return rows_vec<T, 4, GATE, ACT>(a, s);
}

template <typename T>
static int ffn_rows(const InbFfnArgs& a, cudaStream_t s) {
  RowsArgs g = {};
  g.w0 = a.wg, g.w1 = a.wu, g.ld0 = a.ldwg, g.ld1 = a.ldwu;
  g.x = a.x, g.ldx = a.ldx;
  g.out = a.h, g.out_lo = (T*)a.h + a.N * a.ldh, g.ldo = a.ldh;
  g.N = (int)a.N, g.M = a.F, g.K = a.D;
  const int rc = a.act == INB_ACT_SILU ? rows_go<T, true, INB_ACT_SILU>(g, s) : rows_go<T, true, INB_ACT_GELU>(g, s);
  if (rc != 0) return rc;
  RowsArgs d = {};
  d.w0 = d.w1 = a.wd, d.ld0 = d.ld1 = a.ldwd;
  d.x = a.h, d.x_lo = g.out_lo, d.ldx = a.ldh;
  d.out = a.y, d.ldo = a.D;
  d.N = (int)a.N, d.M = a.D, d.K = a.F;
  return rows_go<T, false, INB_ACT_SILU>(d, s);
}

int ffn_rows_any(const InbFfnArgs& a, cudaStream_t s) { return a.dtype == INB_BF16 ? ffn_rows<bf16>(a, s) : ffn_rows<f16>(a, s); }

}  // namespace pol
}  // namespace inb
