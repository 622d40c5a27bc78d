// The tensor-core matrix product under the policy operators: sm_100a, tcgen05.mma from shared memory that TMA fills,
// accumulators in tensor memory.
//
//   C[m, n] = sum over k of A[m, k] B[n, k],  16-bit operands, fp32 accumulation
//
// Persistent blocks walk the tiles of C, 128 CG x 256: one block a tile (CG = 1), or a cluster of two whose SMs work on it
// together (CG = 2: each holds half of A's rows and half of B's, so a slice of B crosses L2 once for both).  Warp 0 fills a
// ring of slices of 64 k with TMA, warp 1 of the first block issues the matrix instructions, sixteen more warps read
// finished accumulators out and run the epilogue (four to a scheduler: one alone waits on its own instructions most of the
// time, and a product over few slices is bound by its epilogue).  Tensor memory holds two accumulators of 256 columns, so
// the epilogue of one tile runs under the products of the next.  Each operand is read as it lies in memory, k or m / n
// contiguous: the 128-byte swizzle of the shared tiles and the descriptor's major bits cover both, so no operand is ever
// transposed by a pass of its own.  Where a product has fewer tiles than the GPU has SMs, its k is split and the parts are
// added by a second launch in a fixed order.
//
// Every wait has a time limit (WAIT_NS).  A wait that runs out sets the device status word and ends the block: its copies
// in flight are waited for, its tensor memory is freed, its results are not to be used.
#pragma once
#include <cuda.h>

#include "policy_common.cuh"

namespace inb {
namespace pol {

constexpr int BM = 128, BN = 256, BK = 64;             // of one block: rows of A; columns of C; k of a slice
constexpr int EPI_WARPS = 16, EPI_COLS = EPI_WARPS / 4; // four warps to each of four column ranges
constexpr int GEMM_THREADS = 64 + 32 * EPI_WARPS;      // TMA, MMA, epilogue
constexpr int EPI_BUF = 2048, EPI_BUFS = 2;            // an epilogue warp's staging: 32 rows x 64 bytes, and how many
constexpr unsigned long long WAIT_NS = 2000000000ull;  // far above any tile's time
constexpr int MAJOR_K = 0, MAJOR_MN = 1;
template <int CG>
struct Gemm {
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN / CG * BK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = CG == 1 ? 3 : 5;
  static constexpr int TM = BM * CG;
  static constexpr int EPI = STAGES * STAGE, BARS = EPI + EPI_WARPS * EPI_BUFS * EPI_BUF, SMEM = BARS + 256 + 1024;
};

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
static __device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* stop) {
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
// CG = 2: the barrier may be the other block's
template <int CG>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(src)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void store_wait() {       // all but the last N groups have been read out of shared memory
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
template <int CG>
__device__ __forceinline__ void group_sync() {       // the blocks of one tile
  if constexpr (CG == 1) {
    __syncthreads();
  } else {
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
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
template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// Arrives at the barrier once the matrix instructions issued so far are done; CG = 2: at both blocks' (same offset)
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t slot) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}
// 16 columns of a warp's 32 rows: thread = row
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
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
  int splits, kbs;    // parts of k, and slices of one
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
template <int MAJOR, int CG>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int row0, int k0, int rows, uint32_t bar) {
  if (MAJOR == MAJOR_K) {
    for (int r = 0; r < rows; r += 128) tma_2d<CG>(dst + r * 128, map, k0, row0 + r, bar);
  } else {
    for (int r = 0; r < rows; r += 64) tma_2d<CG>(dst + r * 128, map, row0 + r, k0, bar);
  }
}

// What an epilogue warp gets for one tile: its row (thread = row) and where it lies
struct EpiCtx {
  int tm, tn, split, item;   // tile, part of k, and the running number of both
  int row;                   // of the tile: 0 .. 128 CG - 1
  int part;                  // which of the EPI_COLS column ranges is this warp's
  int lane;
  uint32_t tmem;             // this warp's rows of the accumulator
  uint32_t stage;            // shared address of EPI_BUFS x EPI_BUF bytes of this warp's own
  unsigned char* stage_ptr;
};

// Epi: struct with  void begin(const EpiCtx&, State&) const  (before the accumulator is complete: what can be fetched early) and
// void operator()(const EpiCtx&, State&, const CUtensorMap* o0, const CUtensorMap* o1) const, called by the epilogue warps
// for every tile.
template <typename T, int CG, int AMAJ, int BMAJ, typename Epi>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
gemm_kernel(const __grid_constant__ CUtensorMap a0, const __grid_constant__ CUtensorMap a1,
            const __grid_constant__ CUtensorMap b0, const __grid_constant__ CUtensorMap b1,
            const __grid_constant__ CUtensorMap o0, const __grid_constant__ CUtensorMap o1, const GemmShape g, const Epi epi,
            int* status) {
  using G = Gemm<CG>;
  extern __shared__ unsigned char raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t full = base + G::BARS, empty = full + 8 * G::STAGES, tfull = empty + 8 * G::STAGES, tempty = tfull + 16,
                 drain = tempty + 16;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int stop;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 1 ? 0 : cluster_rank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < G::STAGES; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull + 8 * i, 1);
      mbar_init(tempty + 8 * i, EPI_WARPS * CG);
    }
    mbar_init(drain, 1);
    stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc<CG>(smem_u32(&tmem_slot));
    tc_before();
  }
  group_sync<CG>();
  tc_after();
  const uint32_t tmem = tmem_slot;
  const int tiles = g.tiles_m * g.tiles_n, items = tiles * g.splits, kb = g.kb0 + g.kb1;
  const int bn = g.dual ? BN / 2 : BN, first = blockIdx.x / CG, stride = gridDim.x / CG;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = first; ok && t < items; t += stride) {
        int tm, tn;
        const int split = t / tiles;
        tile_at(g, t - split * tiles, tm, tn);
        const bool second = tm >= g.m_split;
        const int m0 = (second ? tm - g.m_split : tm) * G::TM + (int)rank * BM, n0 = tn * bn;
        const int k1 = min(kb, (split + 1) * g.kbs);
        for (int k = split * g.kbs; k < k1; ++k, ++it) {
          const int s = it % G::STAGES;
          if (it >= G::STAGES && !mbar_wait(empty + 8 * s, (it / G::STAGES - 1) & 1, &stop)) {
            ok = false;
            break;
          }
          const bool seg = k >= g.kb0;
          const int k0 = (seg ? k - g.kb0 : k) * BK;
          const uint32_t sa = base + s * G::STAGE, sb = sa + G::A_BYTES;
          uint32_t bar = full + 8 * s;
          if (rank == 0) mbar_expect(bar, G::STAGE * CG);      // both blocks' bytes count on the first one's barrier
          if (CG == 2) bar = map_rank(bar, 0);
          load_tile<AMAJ, CG>(sa, seg || second ? &a1 : &a0, m0, k0, BM, bar);
          if (CG == 2) {
            if (g.dual)
              load_tile<BMAJ, CG>(sb, rank ? &b1 : &b0, n0, k0, BN / 2, bar);
            else
              load_tile<BMAJ, CG>(sb, seg ? &b1 : &b0, n0 + (int)rank * (BN / 2), k0, BN / 2, bar);
          } else if (g.dual) {
            load_tile<BMAJ, CG>(sb, &b0, n0, k0, BN / 2, bar);
            load_tile<BMAJ, CG>(sb + G::B_BYTES / 2, &b1, n0, k0, BN / 2, bar);
          } else {
            load_tile<BMAJ, CG>(sb, seg ? &b1 : &b0, n0, k0, BN, bar);
          }
        }
      }
      if (stop && rank == 0) {   // the copies in flight still write shared memory: wait for them, within a limit
        volatile int never = 0;
        for (uint32_t i = it > G::STAGES ? it - G::STAGES : 0; i < it; ++i)
          mbar_wait_slow(full + 8 * (i % G::STAGES), (i / G::STAGES) & 1, &never);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = mma_desc<T, AMAJ, BMAJ>(G::TM, BN);
      uint32_t it = 0, n = 0;
      bool ok = true;
      for (int t = first; ok && t < items; t += stride, ++n) {
        const uint32_t acc = n & 1, d = tmem + acc * BN;
        const int k1 = min(kb, (t / tiles + 1) * g.kbs);
        if (n >= 2 && !mbar_wait(tempty + 8 * acc, ((n >> 1) - 1) & 1, &stop)) break;
        tc_after();
        uint32_t more = 0;
        for (int k = t / tiles * g.kbs; k < k1; ++k, ++it) {
          const int s = it % G::STAGES;
          if (!mbar_wait(full + 8 * s, (it / G::STAGES) & 1, &stop)) {
            ok = false;
            break;
          }
          tc_after();
          const uint32_t sa = base + s * G::STAGE;
          const uint64_t da = smem_desc<AMAJ>(sa), db = smem_desc<BMAJ>(sa + G::A_BYTES);
#pragma unroll
          for (int j = 0; j < BK / 16; ++j) {
            mma_f16<CG>(d, da + j * desc_step<AMAJ>(), db + j * desc_step<BMAJ>(), idesc, more);
            more = 1;
          }
          mma_commit<CG>(empty + 8 * s);
        }
        if (ok) mma_commit<CG>(tfull + 8 * acc);
      }
      if (stop) {
        volatile int never = 0;
        mma_commit<CG>(drain);
        mbar_wait_slow(drain, 0, &never);
      }
    }
  } else {
    const int quarter = warp & 3;            // the tensor-memory lanes that this warp can read
    EpiCtx c;
    c.lane = lane;
    c.row = (int)rank * BM + quarter * 32 + lane;
    c.part = (warp - 2) >> 2;
    c.stage = base + G::EPI + (warp - 2) * EPI_BUFS * EPI_BUF;
    c.stage_ptr = raw + (c.stage - smem_u32(raw));
    uint32_t n = 0;
    for (int t = first; t < items; t += stride, ++n) {
      c.item = t;
      c.split = t / tiles;
      tile_at(g, t - c.split * tiles, c.tm, c.tn);
      const uint32_t acc = n & 1;
      typename Epi::State state;
      epi.begin(c, state);
      const bool ok = mbar_wait(tfull + 8 * acc, (n >> 1) & 1, &stop);
      if (!__all_sync(M32_ALL, ok)) break;
      tc_after();
      c.tmem = tmem + acc * BN + ((uint32_t)(quarter * 32) << 16);
      epi(c, state, &o0, &o1);
      tc_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 1)
          mbar_arrive(tempty + 8 * acc);
        else
          mbar_arrive_at(map_rank(tempty + 8 * acc, 0));
      }
    }
    if (lane == 0) store_wait<0>();
  }
  __syncwarp();
  group_sync<CG>();
  if (warp == 1) {
    tc_after();
    tmem_free<CG>(tmem);
  }
  if (threadIdx.x == 0 && stop && status != nullptr) atomicExch(status, 1);
}

// ------------------------------------------------------------------------------------------------- epilogue helpers
// 16 values of this thread's row into its warp's staging tile of 32 rows x 32 columns (the layout of a 64-byte-swizzled TMA
// box): columns q, q + 16
template <typename T>
__device__ __forceinline__ void stage16(unsigned char* buf, int lane, int q, const float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    Pack<T, 8> o;
#pragma unroll
    for (int e = 0; e < 8; e += 2) down2(make_float2(v[8 * i + e], v[8 * i + e + 1]), o.v[e], o.v[e + 1]);
    st<T, 8>(reinterpret_cast<T*>(buf + lane * 64 + (((q >> 3) + i) ^ ((lane >> 1) & 3)) * 16), o);
  }
}
// Sends a staged tile to rows [r0, r0 + 32) x columns [c0, c0 + 32) of a matrix of M rows x N columns: by TMA, which clips at
// its edges, or (rows that TMA cannot address: `p`, `ld`) by the warp itself, two rows at a time
template <typename T>
__device__ __forceinline__ void send_stage(const CUtensorMap* map, T* p, int64_t ld, int M, int N, int r0, int c0,
                                           const EpiCtx& c, int b) {
  if (map != nullptr) {
    proxy_fence();
    __syncwarp();
    if (c.lane == 0) {
      if (r0 < M) tma_store_2d(map, c0, r0, c.stage + b * EPI_BUF);
      store_commit();
    }
    return;
  }
  __syncwarp();
  const int rows = min(32, M - r0), col = 2 * (c.lane & 15);
  for (int r = c.lane >> 4; r < rows; r += 2) {
    const T* s = reinterpret_cast<const T*>(c.stage_ptr + b * EPI_BUF + r * 64 + (((col >> 3) ^ ((r >> 1) & 3)) * 16)) + (col & 7);
    T* d = p + (int64_t)(r0 + r) * ld + c0 + col;
    if (c0 + col < N) d[0] = s[0];
    if (c0 + col + 1 < N) d[1] = s[1];
  }
  __syncwarp();
}
// Matrices that only these kernels read keep the upper 24 bits of fp32: 16 columns of a row are three 16-byte pieces.  They lie
// in 128-row blocks, in them by groups of 16 columns, in them by pieces, in them by rows: a warp's 32 rows of a piece are 512
// consecutive bytes.  The place (in pieces) of group `cg` of row r, groups groups a row; its further pieces follow 128 on:
__device__ __forceinline__ int64_t blocked(int r, int cg, int groups) {
  return ((int64_t)(r >> 7) * groups + cg) * (3 * 128) + (r & 127);
}
struct Kept16 {
  uint4 w[3];
};
// The upper 24 bits of a value, rounded: cut, every value would lose on average 2^-16.5 of itself, and sums over rows would
// keep that.  A NaN is cut, because the carry would turn some of them into numbers; an infinity has no bits to carry.
__device__ __forceinline__ uint32_t rounded24(float v) {
  const uint32_t b = __float_as_uint(v);
  return v == v ? b + 0x80u : b;
}
__device__ __forceinline__ Kept16 keep16(const float (&v)[16]) {
  uint32_t o[12];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = rounded24(v[4 * i]), b = rounded24(v[4 * i + 1]), c = rounded24(v[4 * i + 2]),
                   d = rounded24(v[4 * i + 3]);
    o[3 * i] = __byte_perm(a, b, 0x5321);
    o[3 * i + 1] = __byte_perm(b, c, 0x6532);
    o[3 * i + 2] = __byte_perm(c, d, 0x7653);
  }
  Kept16 k;
#pragma unroll
  for (int i = 0; i < 3; ++i) k.w[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
  return k;
}
__device__ __forceinline__ void kept16(const Kept16& k, float (&v)[16]) {
  const uint32_t o[12] = {k.w[0].x, k.w[0].y, k.w[0].z, k.w[0].w, k.w[1].x, k.w[1].y,
                          k.w[1].z, k.w[1].w, k.w[2].x, k.w[2].y, k.w[2].z, k.w[2].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[4 * i] = __uint_as_float(o[3 * i] << 8);
    v[4 * i + 1] = __uint_as_float(__funnelshift_r(o[3 * i], o[3 * i + 1], 16) & 0xFFFFFF00u);
    v[4 * i + 2] = __uint_as_float(__funnelshift_r(o[3 * i + 1], o[3 * i + 2], 8) & 0xFFFFFF00u);
    v[4 * i + 3] = __uint_as_float(o[3 * i + 2] & 0xFFFFFF00u);
  }
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

// A row-major [rows, cols] matrix of 16-bit elements, rows `ld` elements apart, in boxes of `box_cols` x `box_rows`: as an
// operand whose k runs along the columns (MAJOR_K, 64 x 128) or along the rows (MAJOR_MN, 64 x 64), or as an epilogue's
// output (32 x 32).  The swizzle spans a box's row.  Needs ld % 8 == 0 and a 16-byte aligned base; what lies outside the
// matrix reads as zero and is not written.
template <typename T>
static bool make_map(CUtensorMap* m, const void* p, int64_t rows, int64_t cols, int64_t ld, int box_cols, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, one[2] = {1, 1};
  EncodeTiled f = encode_tiled();
  return f != nullptr &&
         f(m, IsBf16<T>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(p),
           dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace pol
}  // namespace inb
