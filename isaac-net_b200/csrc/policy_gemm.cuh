// The tensor-core matrix product under the policy operators: sm_100a, tcgen05.mma from shared memory that TMA fills,
// accumulators in tensor memory.
//
//   C[m, n] = sum over k of A[m, k] B[n, k],  16-bit operands, fp32 accumulation
//
// One persistent block per SM walks the tiles of C (BM x BN = 128 x 256).  Warp 0 fills a ring of STAGES x (A, B) slices of
// 64 k with TMA, warp 1 issues the matrix instructions, four more warps read finished accumulators out and run the
// epilogue.  Tensor memory holds two accumulators of 256 columns, so the epilogue of one tile runs under the products of
// the next.  Each operand is read as it lies in memory, k or m / n contiguous: the 128-byte swizzle of the shared tiles
// and the descriptor's major bits cover both, so no operand is ever transposed by a pass of its own.
//
// Every wait has a time limit (WAIT_NS).  A wait that runs out sets the device status word and ends the block: its copies
// in flight are waited for, its tensor memory is freed, its results are not to be used.
#pragma once
#include <cuda.h>

#include "policy_common.cuh"

namespace inb {
namespace pol {

constexpr int BM = 128, BN = 256, BK = 64;
constexpr int STAGES = 4;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2;
constexpr int GEMM_THREADS = 192;                      // TMA, MMA, 4 x epilogue
constexpr int GEMM_SMEM = STAGES * (A_BYTES + B_BYTES) + 1024 + 256;
constexpr unsigned long long WAIT_NS = 2000000000ull;  // far above any tile's time
constexpr int MAJOR_K = 0, MAJOR_MN = 1;

// ------------------------------------------------------------------------------------------------- instructions
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Waits for a phase; false when the limit ran out or another role gave up (`stop`, in shared memory).
__device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* stop) {
  const unsigned long long t0 = now_ns();
  while (true) {
    for (int i = 0; i < 64; ++i)
      if (mbar_try(bar, parity)) return true;
    if (*stop) return false;
    if (now_ns() - t0 > WAIT_NS) {
      *stop = 1;
      return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* stop) {
  if (mbar_try(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, stop);
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// Shared-memory matrix descriptor of a 128-byte-swizzled tile.  K-major: rows of 128 bytes (64 k), groups of 8 rows 1024
// bytes apart.  MN-major: chunks of 64 m or n x 64 k, 8192 bytes apart; within a chunk groups of 8 k 1024 bytes apart.
template <int MAJOR>
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
  const uint64_t lead = MAJOR == MAJOR_K ? 1 : 8192 >> 4;
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (lead << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// 16 k further within the slice, in the descriptor's unit of 16 bytes
template <int MAJOR>
__host__ __device__ constexpr uint32_t desc_step() {
  return MAJOR == MAJOR_K ? 32 >> 4 : 2048 >> 4;
}
template <typename T, int AMAJ, int BMAJ>
__host__ __device__ constexpr uint32_t mma_desc(int m, int n) {
  return (1u << 4) | ((IsBf16<T>::value ? 1u : 0u) << 7) |
         ((IsBf16<T>::value ? 1u : 0u) << 10) | ((uint32_t)AMAJ << 15) | ((uint32_t)BMAJ << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
      "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// ------------------------------------------------------------------------------------------------- the product
// What the blocks multiply.  A and B may each come from two tensors: along k (`kb0` slices of the first pair, then `kb1`
// of the second), along m (tiles from `m_split` on read a1: two products that share B), or interleaved along n
// (`dual`: a tile of B is 128 rows of b0 and the same 128 rows of b1).
struct GemmShape {
  int tiles_m, tiles_n;
  int kb0, kb1;
  int m_split;        // first m tile that reads a1 (tiles_m: none)
  int dual;
  int band;           // m tiles that are walked together, see tile_at
};

// Tile order: bands of `band` m tiles, all n tiles within a band: the blocks that run at one time share their operands
// in L2.
__device__ __forceinline__ void tile_at(const GemmShape& g, int i, int& m, int& n) {
  const int per = g.band * g.tiles_n, b = i / per, r = i - b * per;
  const int h = min(g.band, g.tiles_m - b * g.band);
  n = r / h;
  m = b * g.band + r - n * h;
}

// The operand tile of 64 k at (row0, k0) into dst: one box of `rows` rows k-major, or boxes of 64 rows MN-major
template <int MAJOR>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int row0, int k0, int rows, uint32_t bar) {
  if (MAJOR == MAJOR_K) {
    for (int r = 0; r < rows; r += 128) tma_2d(dst + r * 128, map, k0, row0 + r, bar);
  } else {
    for (int r = 0; r < rows; r += 64) tma_2d(dst + r * 128, map, row0 + r, k0, bar);
  }
}

// Epi: struct with  __device__ void operator()(int tile_m, int tile_n, int row, uint32_t tmem) const, called by every
// thread of the four epilogue warps with its row (0..127) of the tile and the address of that row's warp's accumulator.
template <typename T, int AMAJ, int BMAJ, typename Epi>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
gemm_kernel(const __grid_constant__ CUtensorMap a0, const __grid_constant__ CUtensorMap a1,
            const __grid_constant__ CUtensorMap b0, const __grid_constant__ CUtensorMap b1, const GemmShape g,
            const Epi epi, int* status) {
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t bars = base + STAGES * (A_BYTES + B_BYTES);
  const uint32_t full = bars, empty = bars + 8 * STAGES, tfull = bars + 16 * STAGES, tempty = tfull + 16,
                 drain = tempty + 16;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int stop;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull + 8 * i, 1);
      mbar_init(tempty + 8 * i, 4);
    }
    mbar_init(drain, 1);
    stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    tc_before();
  }
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;
  const int tiles = g.tiles_m * g.tiles_n, kb = g.kb0 + g.kb1;
  const int bn = g.dual ? BN / 2 : BN;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
        int tm, tn;
        tile_at(g, t, tm, tn);
        const bool second = tm >= g.m_split;
        const int m0 = (second ? tm - g.m_split : tm) * BM, n0 = tn * bn;
        for (int k = 0; k < kb; ++k, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES && !mbar_wait(empty + 8 * s, (it / STAGES - 1) & 1, &stop)) {
            ok = false;
            break;
          }
          const bool seg = k >= g.kb0;
          const int k0 = (seg ? k - g.kb0 : k) * BK;
          const uint32_t sa = base + s * (A_BYTES + B_BYTES), sb = sa + A_BYTES, bar = full + 8 * s;
          mbar_expect(bar, A_BYTES + B_BYTES);
          load_tile<AMAJ>(sa, seg || second ? &a1 : &a0, m0, k0, BM, bar);
          if (g.dual) {
            load_tile<BMAJ>(sb, &b0, n0, k0, BN / 2, bar);
            load_tile<BMAJ>(sb + B_BYTES / 2, &b1, n0, k0, BN / 2, bar);
          } else {
            load_tile<BMAJ>(sb, seg ? &b1 : &b0, n0, k0, BN, bar);
          }
        }
      }
      if (stop) {       // the copies in flight still write this block's shared memory: wait for them, within a limit
        volatile int never = 0;
        for (uint32_t i = it > STAGES ? it - STAGES : 0; i < it; ++i)
          mbar_wait_slow(full + 8 * (i % STAGES), (i / STAGES) & 1, &never);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = mma_desc<T, AMAJ, BMAJ>(BM, BN);
      uint32_t it = 0, n = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x, ++n) {
        const uint32_t acc = n & 1, d = tmem + acc * BN;
        if (n >= 2 && !mbar_wait(tempty + 8 * acc, ((n >> 1) - 1) & 1, &stop)) break;
        tc_after();
        for (int k = 0; k < kb; ++k, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(full + 8 * s, (it / STAGES) & 1, &stop)) {
            ok = false;
            break;
          }
          tc_after();
          const uint32_t sa = base + s * (A_BYTES + B_BYTES);
          const uint64_t da = smem_desc<AMAJ>(sa), db = smem_desc<BMAJ>(sa + A_BYTES);
#pragma unroll
          for (int j = 0; j < BK / 16; ++j)
            mma_f16(d, da + j * desc_step<AMAJ>(), db + j * desc_step<BMAJ>(), idesc, (k | j) != 0);
          mma_commit(empty + 8 * s);
        }
        if (ok) mma_commit(tfull + 8 * acc);
      }
      if (stop) {
        volatile int never = 0;
        mma_commit(drain);
        mbar_wait_slow(drain, 0, &never);
      }
    }
  } else {
    const int quarter = warp & 3;            // the tensor-memory lanes that this warp can read
    uint32_t n = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
      int tm, tn;
      tile_at(g, t, tm, tn);
      const uint32_t acc = n & 1;
      const bool ok = mbar_wait(tfull + 8 * acc, (n >> 1) & 1, &stop);
      if (!__all_sync(M32_ALL, ok)) break;
      tc_after();
      epi(tm, tn, quarter * 32 + lane, tmem + acc * BN + ((uint32_t)(quarter * 32) << 16));
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty + 8 * acc);
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == 1) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
  if (threadIdx.x == 0 && stop && status != nullptr) atomicExch(status, 1);
}

// ------------------------------------------------------------------------------------------------- host side
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess) p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

// A row-major [rows, cols] matrix of 16-bit elements, rows `ld` elements apart, as an operand whose k runs along the columns
// (MAJOR_K, box 64 columns x `box_rows` rows) or along the rows (MAJOR_MN, box 64 x 64).  Needs ld % 8 == 0 and a 16-byte
// aligned base; what lies outside the matrix reads as zero.
template <typename T>
static bool make_map(CUtensorMap* m, const void* p, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, one[2] = {1, 1};
  EncodeTiled f = encode_tiled();
  return f != nullptr &&
         f(m, IsBf16<T>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(p),
           dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace pol
}  // namespace inb
