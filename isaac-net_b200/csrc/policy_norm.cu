// block_norm: the norms before and after a residual block, with the block's gate and the residual scale.
//
//   y = x + s * gate * (post * h * rh),   rh = rsqrt(mean(h^2) + eps)     (post absent: gate * h)
//   n = w * y * ry,                       ry = rsqrt(mean(y^2) + eps)
//
// Backward, with gy, gn the gradients of y and n, hh = h rh, yh = y ry:
//   t  = gy + ry (q - yh mean(q yh)),  q = gn w                            = gx
//   gp = s gate t;  gh = rh (r - hh mean(r hh)),  r = gp post              (post absent: gh = gp)
//   gw = sum gn yh;  gpost = sum gp hh;  ggate = sum over the gate's rows of s t (post hh)
//
// One pass over the rows in each direction: a group of threads (a warp, or several) holds a row in registers, every
// statistic is fp32, and each output is rounded once.  The backward pass recomputes y from x and h in fp32 rather
// than reading the rounded y back: it moves the same bytes and loses nothing.  It keeps the column sums of its rows
// in registers, writes one fp32 partial row per block and a second launch adds those in a fixed order: no atomics, so
// equal inputs give equal bits.
//
// The forward pass is bound by DRAM, 4 row passes of N x D elements; the backward pass, with 6 of them, by the latency of
// its instructions: two dependent row sums a row and 8 warps an SM to hide them (N = 131072, D = 512, bf16, a gate for 32
// rows: 104 us at 5.2 TB/s, and 170 us at 4.7).
#include <algorithm>

#include "policy_common.cuh"

namespace inb {
namespace pol {

struct NormPlan {
  int V, IT;          // elements of one access, accesses of one thread
  bool mis;           // 16-bit elements that may start on half a word: accesses of 8 of them, by words (see Part)
  int tpr;            // threads of a row (multiple of 32)
  int block, groups;  // threads of a block, rows in flight in it
};

// Widest access that the pointers, strides and D allow.
static int norm_vec(const InbNormArgs& a, bool bwd) {
  const int esz = a.dtype == INB_F32 ? 4 : 2;
  uint64_t m = (uint64_t)a.D * esz;
  auto add = [&](const void* p, int64_t ld) {
    if (p != nullptr) m |= (uint64_t)(uintptr_t)p | (uint64_t)(ld * esz);
  };
  add(a.x, a.ldx);
  add(a.h, a.ldh);
  add(a.w, 0);
  add(a.post, 0);
  add(a.gate, 0);
  if (!bwd) {
    add(a.y, a.D);
    add(a.n, a.D);
  } else {
    add(a.gy, a.ldgy);
    add(a.gn, a.ldgn);
    add(a.gx, a.D);
    add(a.gh, a.D);
    add(a.ggate, a.D);
  }
  if ((m & 15) == 0) return 16 / esz;
  if (esz == 2 && (m & 3) == 0) return 2;
  return 1;
}

static NormPlan norm_plan(const InbNormArgs& a, bool bwd) {
  NormPlan p;
  p.V = norm_vec(a, bwd);
  p.mis = p.V == 1 && a.dtype != INB_F32;
  if (p.mis) p.V = 8;
  // elements of a row in a thread: 16, or 8 of a narrow row.  (The backward pass on N = 131072, D = 512 takes 175 us with 16,
  // of which one block of 256 threads fits an SM, and 210 with 8 and two blocks: a row's fixed work counts for more.)
  const int per = a.D > 256 ? 16 : 8;
  p.IT = per / p.V;
  const int lanes = (a.D + p.V * p.IT - 1) / (p.V * p.IT);
  p.tpr = (lanes + 31) / 32 * 32;
  p.groups = p.tpr >= 256 ? 1 : 256 / p.tpr;
  p.block = p.tpr * p.groups;
  return p;
}

// Sum over the threads of one row.  `buf`: 2 x 32 floats of the group; calls alternate its halves, so the one barrier
// inside also separates a call's reads from the next-but-one call's writes.
__device__ __forceinline__ float row_sum(float v, int tpr, int group, int t, float* buf, int& par) {
  v = warp_sum(v);
  if (tpr == 32) return v;
  float* b = buf + (par ^= 1) * 32;
  if ((t & 31) == 0) b[t >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(tpr) : "memory");
  float s = 0.f;
  for (int i = 0; i < (tpr >> 5); ++i) s += b[i];
  return s;
}

// Rows are cut into chunks that never cross a gate's rows: chunk c = rows [g R + k len, ...) of gate g = c / cpg.  All
// counts are below 2^31.
struct NormChunks {
  uint32_t n;       // chunks
  uint32_t rows;    // rows of one gate (N without a gate)
  uint32_t len;     // rows of a chunk
  uint32_t cpg;     // chunks of one gate
};
// Row strides in bytes, below 2^32: a row's address is one 32 x 32 -> 64-bit multiply-add
struct NormStrides {
  uint32_t x, h, gy, gn, d;      // d: of the contiguous tensors
};
__device__ __forceinline__ const char* row_at(const void* p, uint32_t row, uint32_t ld, int offset) {
  return (const char*)p + ((uint64_t)row * ld + offset);
}

// A worker's walk over the rows of its chunks
struct Cursor {
  uint32_t c, gate, row, end;
  bool first;      // row is the first of its chunk
  __device__ __forceinline__ void start(const NormChunks& ch, uint32_t chunk) {
    c = chunk;
    first = true;
    if (c >= ch.n) return;
    gate = c / ch.cpg;
    row = gate * ch.rows + (c - gate * ch.cpg) * ch.len;
    end = min(row + ch.len, (gate + 1) * ch.rows);
  }
  __device__ __forceinline__ void next(const NormChunks& ch, uint32_t stride) {
    first = false;
    if (++row == end) start(ch, c + stride);
  }
};

// Rows on their way: each thread copies its own part of the next rows of NT tensors (and 8 bytes of statistics) to its own
// places of a ring of S rows in shared memory (cp.async) and reads only those back, so the ring needs no barrier and keeps
// rows in flight that registers would have no room for.  S = 0: plain loads.
template <typename T, int V, int IT, int MAXT, int NT, int WANT, bool MIS>
struct Ring {
  static constexpr int WORDS = 5;                                      // MIS: the words that 8 elements may touch
  static constexpr int ROW = NT * IT * (MIS ? 4 * WORDS : V * (int)sizeof(T)) + 8;     // a thread's bytes of one row
  static constexpr int MOST = 176 * 1024;
  static constexpr int S = V * sizeof(T) < 4 ? 0 : (WANT * ROW * MAXT <= MOST ? WANT : (2 * ROW * MAXT <= MOST ? 2 : 0));
  static constexpr int BLOCKS = S > 0 && S * ROW * MAXT <= 88 * 1024 ? 2 : 1;       // of them on an SM
  static constexpr int ACCESS = MIS ? 4 : V * (int)sizeof(T), PER = MIS ? WORDS : 1;    // bytes and number of a copy's pieces
  // access i (and its word w) of tensor k in slot `slot`, and the statistics: byte offsets from `mine()`, constant but for
  // the slot
  static __device__ __forceinline__ int place(int slot, int k, int i, int w = 0) {
    return slot * (ROW * MAXT) + ((k * IT + i) * PER + w) * ACCESS * MAXT;
  }
  static __device__ __forceinline__ unsigned char* mine(unsigned char* ring) { return ring + threadIdx.x * ACCESS; }
  static __device__ __forceinline__ unsigned char* stat(unsigned char* ring, int slot) {
    return ring + slot * (ROW * MAXT) + (ROW - 8) * MAXT + threadIdx.x * 8;
  }
  // zero the places: what is never copied (columns beyond D, absent tensors) reads as zero
  static __device__ __forceinline__ void clear(unsigned char* ring) {
#pragma unroll 1
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
          for (int w = 0; w < PER; ++w)
#pragma unroll
            for (int b = 0; b < ACCESS; b += ACCESS < 4 ? 2 : 4)
              if constexpr (ACCESS < 4)
                *reinterpret_cast<uint16_t*>(mine(ring) + place(s, k, i, w) + b) = 0;
              else
                *reinterpret_cast<uint32_t*>(mine(ring) + place(s, k, i, w) + b) = 0;
  }
};
template <typename T, int V, int IT, int MAXT, bool MIS>
using FwdRing = Ring<T, V, IT, MAXT, 3, 3, MIS>;      // x, h, gate
template <typename T, int V, int IT, int MAXT, bool MIS>
using BwdRing = Ring<T, V, IT, MAXT, 5, 3, MIS>;      // x, h, gn, gy, gate
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else if constexpr (BYTES == 8)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
  else if constexpr (BYTES == 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A thread's part of a row: IT accesses of V elements, zero beyond D, as pairs of fp32 where it is worked on.
// MIS: rows of 16-bit elements that start anywhere.  An access of 8 elements is copied as the four or five aligned words that
// hold them (each holds at least one of the row's elements) and shifted into place when it is read; it is stored as words
// but for its ends.  (Element by element and without the ring, rows of odd length ran at a seventh of the aligned rate.)
template <typename T, int V, int IT, bool MIS>
struct Part {
  static constexpr int N2 = V * IT / 2;
  Pack<T, V> p[IT];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) p[i].v[e] = from_f<T>(0.f);
  }
  __device__ __forceinline__ void load(const T* row, int tpr, int t, int D) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * tpr + t) * V;
      if (MIS) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (c + e < D) p[i].v[e] = row[c + e];
      } else if (c < D) {
        p[i] = ld<T, V>(row + c);
      }
    }
  }
  // to and from a ring: `row` is the tensor's row at this thread's first column
  template <typename R>
  static __device__ __forceinline__ void fetch(unsigned char* ring, int slot, int k, const char* row, int tpr, int t, int D) {
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if ((i * tpr + t) * V < D) {
        const char* at = row + i * tpr * V * (int)sizeof(T);
        if constexpr (MIS) {
          const int half = (int)((uintptr_t)at & 2), words = (half + 2 * min(V, D - (i * tpr + t) * V) + 3) >> 2;
#pragma unroll
          for (int w = 0; w < R::WORDS; ++w)
            if (w < words)
              copy_async<4>((uint32_t)__cvta_generic_to_shared(R::mine(ring) + R::place(slot, k, i, w)), at - half + 4 * w);
        } else {
          copy_async<R::ACCESS>((uint32_t)__cvta_generic_to_shared(R::mine(ring) + R::place(slot, k, i)), at);
        }
      }
  }
  template <typename R>
  __device__ __forceinline__ void read(unsigned char* ring, int slot, int k, const char* row, int tpr, int t, int D) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if constexpr (MIS) {
        const int shift = (int)((uintptr_t)row & 2) * 8, left = D - (i * tpr + t) * V;
        uint32_t v[R::WORDS];
#pragma unroll
        for (int w = 0; w < R::WORDS; ++w) v[w] = *reinterpret_cast<const uint32_t*>(R::mine(ring) + R::place(slot, k, i, w));
        uint32_t* o = reinterpret_cast<uint32_t*>(&p[i]);
#pragma unroll
        for (int w = 0; w < V / 2; ++w) {
          o[w] = __funnelshift_r(v[w], v[w + 1], shift);
          // what lies beyond D in the last words, or was left there by a row that started on the other half
          if (2 * w + 1 >= left) o[w] = 2 * w < left ? o[w] & 0xFFFFu : 0u;
        }
      } else {
        p[i] = *reinterpret_cast<const Pack<T, V>*>(R::mine(ring) + R::place(slot, k, i));
      }
    }
  }
  __device__ __forceinline__ void store(T* row, int tpr, int t, int D) const {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * tpr + t) * V;
      if constexpr (MIS) {
        T* d = row + c;
        if (c + V <= D) {
          const bool half = ((uintptr_t)d & 2) != 0;
          if (half) d[0] = p[i].v[0];
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            if (!half)
              st<T, 2>(d + e, Pack<T, 2>{p[i].v[e], p[i].v[e + 1]});
            else if (e + 2 < V)
              st<T, 2>(d + e + 1, Pack<T, 2>{p[i].v[e + 1], p[i].v[e + 2]});
          }
          if (half) d[V - 1] = p[i].v[V - 1];
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (c + e < D) d[e] = p[i].v[e];
        }
      } else if (c < D) {
        st<T, V>(row + c, p[i]);
      }
    }
  }
  __device__ __forceinline__ float2 get(int j) const {
    return V == 1 ? up2(p[2 * j].v[0], p[2 * j + 1].v[0]) : up2(p[2 * j / V].v[2 * j % V], p[2 * j / V].v[2 * j % V + 1]);
  }
  __device__ __forceinline__ void set(int j, float2 v) {
    if constexpr (V == 1)
      down2(v, p[2 * j].v[0], p[2 * j + 1].v[0]);
    else
      down2(v, p[2 * j / V].v[2 * j % V], p[2 * j / V].v[2 * j % V + 1]);
  }
  // the column of element 2 j (x) and of element 2 j + 1 (y)
  static __device__ __forceinline__ int2 cols(int j, int tpr, int t) {
    if (V == 1) return make_int2(2 * j * tpr + t, (2 * j + 1) * tpr + t);
    const int c = (2 * j / V * tpr + t) * V + 2 * j % V;
    return make_int2(c, c + 1);
  }
};

// MAXT: the largest block it is launched with.
template <typename T, int V, int IT, int MAXT, bool MIS>
__global__ void __launch_bounds__(MAXT, FwdRing<T, V, IT, MAXT, MIS>::BLOCKS)
norm_fwd_kernel(const __grid_constant__ InbNormArgs a, int tpr, const NormChunks ch, const NormStrides ld) {
  __shared__ float red[8][64];
  extern __shared__ __align__(16) unsigned char ring[];
  using P = Part<T, V, IT, MIS>;
  using Rg = FwdRing<T, V, IT, MAXT, MIS>;
  constexpr int S = Rg::S;
  const int group = threadIdx.x / tpr, t = threadIdx.x % tpr, groups = blockDim.x / tpr;
  const int D = a.D, col = t * V * (int)sizeof(T);
  const float inv_d = 1.f / (float)D;
  const bool has_h = a.h != nullptr, has_post = a.post != nullptr;
  P w, post, x, h;
  w.zero();
  w.load((const T*)a.w, tpr, t, D);
  post.zero();
  if (has_post) post.load((const T*)a.post, tpr, t, D);
  x.zero();
  h.zero();
  float2 coef[P::N2];                // scale * gate * post of the chunk
  int par = 0;
  const uint32_t stride = gridDim.x * groups;
  Cursor at, ahead;
  at.start(ch, blockIdx.x * groups + group);
  ahead = at;
  auto fetch = [&](int slot) {
    if (ahead.c < ch.n) {
      P::template fetch<Rg>(ring, slot, 0, row_at(a.x, ahead.row, ld.x, col), tpr, t, D);
      if (has_h) P::template fetch<Rg>(ring, slot, 1, row_at(a.h, ahead.row, ld.h, col), tpr, t, D);
      if (a.gate && ahead.first) P::template fetch<Rg>(ring, slot, 2, row_at(a.gate, ahead.gate, ld.d, col), tpr, t, D);
      ahead.next(ch, stride);
    }
    copy_commit();
  };
  if constexpr (S > 0) {
    Rg::clear(ring);
    for (int i = 0; i < S - 1; ++i) fetch(i);
  }
  int slot = 0;
  for (; at.c < ch.n; at.next(ch, stride)) {
    P g;
    g.zero();
    if constexpr (S > 0) {
      copy_wait<S - 2>();
      x.template read<Rg>(ring, slot, 0, row_at(a.x, at.row, ld.x, col), tpr, t, D);
      if (has_h) h.template read<Rg>(ring, slot, 1, row_at(a.h, at.row, ld.h, col), tpr, t, D);
      if (a.gate && at.first) g.template read<Rg>(ring, slot, 2, row_at(a.gate, at.gate, ld.d, col), tpr, t, D);
      fetch(slot == 0 ? S - 1 : slot - 1);         // the place read in the last turn
      slot = slot == S - 1 ? 0 : slot + 1;
    } else {
      x.zero();             // beyond D it holds the last row's output, which a row that is not finite made NaN there too
      x.load((const T*)row_at(a.x, at.row, ld.x, 0), tpr, t, D);
      if (has_h) h.load((const T*)row_at(a.h, at.row, ld.h, 0), tpr, t, D);
      if (a.gate && at.first) g.load((const T*)row_at(a.gate, at.gate, ld.d, 0), tpr, t, D);
    }
    if (at.first && has_h) {
#pragma unroll
      for (int j = 0; j < P::N2; ++j) {
        coef[j] = both(a.scale);
        if (has_post) coef[j] = mul2(coef[j], post.get(j));
        if (a.gate) coef[j] = mul2(coef[j], g.get(j));
      }
    }
    float rh = 1.f;
    float2 s = both(0.f);
    if (has_post) {
#pragma unroll
      for (int j = 0; j < P::N2; ++j) s = fma2(h.get(j), h.get(j), s);
      rh = rsqrtf(row_sum(s.x + s.y, tpr, group, t, red[group], par) * inv_d + a.eps);
    }
    float2 y[P::N2];
    s = both(0.f);
#pragma unroll
    for (int j = 0; j < P::N2; ++j) {
      y[j] = x.get(j);
      if (has_h) y[j] = fma2(mul2(h.get(j), both(rh)), coef[j], y[j]);
      s = fma2(y[j], y[j], s);
    }
    if (has_h) {
#pragma unroll
      for (int j = 0; j < P::N2; ++j) x.set(j, y[j]);
      x.store((T*)row_at(a.y, at.row, ld.d, 0), tpr, t, D);
    }
    const float ry = rsqrtf(row_sum(s.x + s.y, tpr, group, t, red[group], par) * inv_d + a.eps);
    if (a.stats && t == 0) *reinterpret_cast<float2*>(a.stats + 2 * (int64_t)at.row) = make_float2(rh, ry);
#pragma unroll
    for (int j = 0; j < P::N2; ++j) x.set(j, mul2(mul2(y[j], both(ry)), w.get(j)));
    x.store((T*)row_at(a.n, at.row, ld.d, 0), tpr, t, D);
  }
}

// The row sums that gate's and post's gradients need differ only in factors that are fixed within a chunk:
// e = sum over the chunk of t hh;  ggate = s post e, gpost = sum over the chunks of s gate e.  So the rows add to one
// accumulator (and to gw's), and gpost's, touched once a chunk, lies in shared memory.
template <typename T, int V, int IT, int MAXT, bool MIS>
__global__ void __launch_bounds__(MAXT, BwdRing<T, V, IT, MAXT, MIS>::BLOCKS)
norm_bwd_kernel(const __grid_constant__ InbNormArgs a, int tpr, const NormChunks ch, const NormStrides ld) {
  __shared__ float red[8][64];
  extern __shared__ __align__(16) unsigned char ring[];
  using P = Part<T, V, IT, MIS>;
  using Rg = BwdRing<T, V, IT, MAXT, MIS>;
  constexpr int S = Rg::S;
  const int group = threadIdx.x / tpr, t = threadIdx.x % tpr, groups = blockDim.x / tpr;
  const int D = a.D, col = t * V * (int)sizeof(T);
  float* sums = reinterpret_cast<float*>(ring + S * Rg::ROW * MAXT);   // [groups][D]
  const float inv_d = 1.f / (float)D;
  const bool has_h = a.h != nullptr, has_post = a.post != nullptr;
  P w;
  w.zero();
  w.load((const T*)a.w, tpr, t, D);
  float2 aw[P::N2], coef[P::N2], ae[P::N2];
  float* mine = sums + group * D;
#pragma unroll
  for (int j = 0; j < P::N2; ++j) {
    aw[j] = both(0.f);
    const int2 c = P::cols(j, tpr, t);
    if (c.x < D) mine[c.x] = 0.f;
    if (c.y < D) mine[c.y] = 0.f;
  }
  int par = 0;
  float* part_gate = a.work + 2 * (int64_t)gridDim.x * D;
  const uint32_t stride = gridDim.x * groups;
  Cursor at, ahead;
  at.start(ch, blockIdx.x * groups + group);
  ahead = at;
  auto fetch = [&](int slot) {
    if (ahead.c < ch.n) {
      P::template fetch<Rg>(ring, slot, 0, row_at(a.x, ahead.row, ld.x, col), tpr, t, D);
      if (has_h) P::template fetch<Rg>(ring, slot, 1, row_at(a.h, ahead.row, ld.h, col), tpr, t, D);
      if (a.gn) P::template fetch<Rg>(ring, slot, 2, row_at(a.gn, ahead.row, ld.gn, col), tpr, t, D);
      if (a.gy) P::template fetch<Rg>(ring, slot, 3, row_at(a.gy, ahead.row, ld.gy, col), tpr, t, D);
      if (a.gate && ahead.first) P::template fetch<Rg>(ring, slot, 4, row_at(a.gate, ahead.gate, ld.d, col), tpr, t, D);
      copy_async<8>((uint32_t)__cvta_generic_to_shared(Rg::stat(ring, slot)), row_at(a.stats, ahead.row, 8, 0));
      ahead.next(ch, stride);
    }
    copy_commit();
  };
  if constexpr (S > 0) {
    Rg::clear(ring);
    for (int i = 0; i < S - 1; ++i) fetch(i);
  }
  int slot = 0;
  while (at.c < ch.n) {
    const int here = slot;
    // one tensor's part of this row; the passes below read it again rather than hold it, which would spill
    auto take = [&](P& v, int k, const void* p, uint32_t stride) {
      if constexpr (S > 0) {
        asm volatile("" ::: "memory");
        v.template read<Rg>(ring, here, k, row_at(p, at.row, stride, col), tpr, t, D);
      } else {
        v.zero();
        if (p != nullptr) v.load((const T*)row_at(p, at.row, stride, 0), tpr, t, D);
      }
    };
    float2 st;
    if constexpr (S > 0) {
      copy_wait<S - 2>();
      st = *reinterpret_cast<const float2*>(Rg::stat(ring, slot));
    } else {
      st = *reinterpret_cast<const float2*>(row_at(a.stats, at.row, 8, 0));
    }
    if (at.first) {
      P post, g;
      post.zero();
      if (has_post) post.load((const T*)a.post, tpr, t, D);
      g.zero();
      if (a.gate) {
        if constexpr (S > 0)
          g.template read<Rg>(ring, here, 4, row_at(a.gate, at.gate, ld.d, col), tpr, t, D);
        else
          g.load((const T*)row_at(a.gate, at.gate, ld.d, 0), tpr, t, D);
      }
#pragma unroll
      for (int j = 0; j < P::N2; ++j) {
        ae[j] = both(0.f);
        coef[j] = both(a.scale);
        if (has_post) coef[j] = mul2(coef[j], post.get(j));
        if (a.gate) coef[j] = mul2(coef[j], g.get(j));
      }
    }
    if constexpr (S > 0) {
      fetch(slot == 0 ? S - 1 : slot - 1);         // the place read in the last turn
      slot = slot == S - 1 ? 0 : slot + 1;
    }
    const float rh = st.x, ry = st.y;
    float2 v[P::N2], s = both(0.f);
    {
      P x, h, gn;                                  // v = yh
      take(x, 0, a.x, ld.x);
      take(h, 1, a.h, ld.h);
      take(gn, 2, a.gn, ld.gn);
#pragma unroll
      for (int j = 0; j < P::N2; ++j) {
        v[j] = x.get(j);
        if (has_h) v[j] = fma2(mul2(h.get(j), both(rh)), coef[j], v[j]);
        v[j] = mul2(v[j], both(ry));
        const float2 q = gn.get(j);
        aw[j] = fma2(q, v[j], aw[j]);
        s = fma2(mul2(q, w.get(j)), v[j], s);
      }
    }
    const float c1 = row_sum(s.x + s.y, tpr, group, t, red[group], par) * inv_d;
    s = both(0.f);
    {
      P gy, h, gn;                                 // v = t, then gp post
      take(gn, 2, a.gn, ld.gn);
      take(gy, 3, a.gy, ld.gy);
      take(h, 1, a.h, ld.h);
#pragma unroll
      for (int j = 0; j < P::N2; ++j) {
        const float2 q = fma2(v[j], both(-c1), mul2(gn.get(j), w.get(j)));
        v[j] = fma2(q, both(ry), gy.get(j));
        gy.set(j, v[j]);
        if (has_h) {
          const float2 hh = mul2(h.get(j), both(rh));
          ae[j] = fma2(v[j], hh, ae[j]);
          v[j] = mul2(v[j], coef[j]);
          s = fma2(v[j], hh, s);
        }
      }
      gy.store((T*)row_at(a.gx, at.row, ld.d, 0), tpr, t, D);
    }
    if (has_h) {
      const float c2 = has_post ? row_sum(s.x + s.y, tpr, group, t, red[group], par) * inv_d : 0.f;
      P h;
      take(h, 1, a.h, ld.h);
#pragma unroll
      for (int j = 0; j < P::N2; ++j) {
        if (has_post) v[j] = mul2(fma2(mul2(h.get(j), both(rh)), both(-c2), v[j]), both(rh));
        h.set(j, v[j]);
      }
      h.store((T*)row_at(a.gh, at.row, ld.d, 0), tpr, t, D);
    }
    const uint32_t gate = at.gate, chunk = at.c;
    const bool alone = at.first;
    at.next(ch, stride);
    if (at.first && (a.ggate || has_post)) {           // that was the chunk's last row
      P post, g, x;
      post.zero();
      g.zero();
      if (a.gate) {
        bool loaded = false;
        if constexpr (S > 0)
          if (alone) {
            g.template read<Rg>(ring, here, 4, row_at(a.gate, gate, ld.d, col), tpr, t, D);
            loaded = true;
          }
        if (!loaded) g.load((const T*)row_at(a.gate, gate, ld.d, 0), tpr, t, D);
      }
      if (has_post) post.load((const T*)a.post, tpr, t, D);
#pragma unroll
      for (int j = 0; j < P::N2; ++j) {
        const int2 c = P::cols(j, tpr, t);
        ae[j] = mul2(ae[j], both(a.scale));
        const float2 add = a.gate ? mul2(ae[j], g.get(j)) : ae[j];
        if (c.x < D) mine[c.x] += add.x;
        if (c.y < D) mine[c.y] += add.y;
        if (a.ggate) {
          if (has_post) ae[j] = mul2(ae[j], post.get(j));
          x.set(j, ae[j]);
          if (ch.cpg > 1) {
            if (c.x < D) part_gate[(int64_t)chunk * D + c.x] = ae[j].x;
            if (c.y < D) part_gate[(int64_t)chunk * D + c.y] = ae[j].y;
          }
        }
      }
      if (a.ggate && ch.cpg == 1) x.store((T*)a.ggate + (int64_t)gate * D, tpr, t, D);
    }
  }
  // the block's column sums, over its groups in order: gpost's lie in shared memory, then gw's take their place
  float* out = a.work + (int64_t)blockIdx.x * 2 * D;
  for (int kind = 1; kind >= 0; --kind) {
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      float s = 0.f;
      for (int g = 0; g < groups; ++g) s += sums[g * D + c];
      out[kind * D + c] = s;
    }
    if (kind == 0) break;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < P::N2; ++j) {
      const int2 c = P::cols(j, tpr, t);
      if (c.x < D) mine[c.x] = aw[j].x;
      if (c.y < D) mine[c.y] = aw[j].y;
    }
  }
}

// Adds the partial rows: blockIdx.y = 0: w, 1: post, 2 + g: gate g.  32 columns x 32 rows in flight per block.
template <typename T>
__global__ void __launch_bounds__(1024) norm_sum_kernel(InbNormArgs a, int blocks, NormChunks ch) {
  __shared__ float sm[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, D = a.D;
  const int c = blockIdx.x * 32 + cx;
  const int kind = (int)blockIdx.y;
  const float* src;
  int64_t n, ld;
  T* dst;
  if (kind < 2) {
    if (kind == 1 && a.post == nullptr) return;
    src = a.work + kind * D;
    n = blocks;
    ld = 2 * (int64_t)D;
    dst = (T*)(kind == 0 ? a.gw : a.gpost);
  } else {
    const int64_t g = kind - 2;
    src = a.work + 2 * (int64_t)blocks * D + g * ch.cpg * D;
    n = ch.cpg;
    ld = D;
    dst = (T*)a.ggate + g * D;
  }
  float s = 0.f;
  if (c < D)
    for (int64_t r = ry; r < n; r += 32) s += src[r * ld + c];
  sm[ry][cx] = s;
  __syncthreads();
  s = warp_sum(sm[cx][ry]);       // thread (ry, cx) holds row cx of column ry
  const int col = blockIdx.x * 32 + ry;
  if (cx == 0 && col < D) dst[col] = from_f<T>(s);
}

static int norm_check(const InbNormArgs* p, bool bwd, bool sizes_only = false) {
  if (p == nullptr) return -1;
  const InbNormArgs& a = *p;
  if (a.dtype < 0 || a.dtype > 2 || a.N < 0 || a.N > 0x7FFFFFFF || a.D < 1 || a.D > INB_MAX_NORM_D) return -2;
  if (a.N == 0) return 0;
  if (a.x == nullptr || a.w == nullptr) return -3;
  if (a.h == nullptr && (a.post != nullptr || a.gate != nullptr)) return -3;
  // the kernels hold a row's stride in bytes in 32 bits
  auto far = [](const void* q, int64_t ld) { return q != nullptr && (ld < 0 || ld > INB_MAX_NORM_LD); };
  if (far(a.x, a.ldx) || far(a.h, a.ldh) || (bwd && (far(a.gy, a.ldgy) || far(a.gn, a.ldgn)))) return -2;
  if (a.gate != nullptr && (a.gate_rows < 1 || a.N % a.gate_rows != 0)) return -4;
  if (sizes_only) return 0;
  if (!bwd && (a.n == nullptr || (a.h != nullptr && a.y == nullptr))) return -3;
  if (bwd && (a.stats == nullptr || a.gx == nullptr || a.gw == nullptr || a.work == nullptr ||
              (a.h != nullptr && a.gh == nullptr) || (a.post != nullptr && a.gpost == nullptr) ||
              (a.gate != nullptr && a.ggate == nullptr)))
    return -3;
  return 0;
}

static int norm_blocks(const NormPlan& p, int64_t units, int per_sm) {
  const int64_t need = (units + p.groups - 1) / p.groups, most = (int64_t)sm_count() * per_sm;
  return (int)(need < most ? need : most);
}

// per_sm: blocks that an SM holds (see Ring)
static NormChunks norm_chunks(const InbNormArgs& a, const NormPlan& p, bool bwd, int per_sm) {
  NormChunks c;
  // enough chunks for every worker; the forward pass, whose chunks leave no partial sums, takes four times as many so
  // that the workers end together (in the backward pass the partial rows cost what that gains)
  const int64_t workers = (int64_t)sm_count() * per_sm * p.groups * (bwd ? 1 : 4);
  const int64_t rows = a.gate != nullptr ? a.gate_rows : a.N, gates = a.N / rows;
  const int64_t cpg = std::min(rows, (workers + gates - 1) / gates);
  const int64_t len = (rows + cpg - 1) / cpg;
  c.rows = (uint32_t)rows;
  c.len = (uint32_t)len;
  c.cpg = (uint32_t)((rows + len - 1) / len);
  c.n = (uint32_t)(gates * c.cpg);
  return c;
}

// Runs the call, or (elems != NULL) says how many floats of work it needs
template <typename T, int V, int IT, int MAXT, bool MIS>
static int norm_launch(const InbNormArgs& a, const NormPlan& p, bool bwd, int64_t* elems, cudaStream_t s) {
  using F = FwdRing<T, V, IT, MAXT, MIS>;
  using B = BwdRing<T, V, IT, MAXT, MIS>;
  const int per_sm = bwd ? B::BLOCKS : F::BLOCKS;
  const NormChunks ch = norm_chunks(a, p, bwd, per_sm);
  const int blocks = norm_blocks(p, ch.n, per_sm);
  if (bwd) {
    const int64_t need = (2 * (int64_t)blocks + (a.gate != nullptr && ch.cpg > 1 ? ch.n : 0)) * a.D;
    if (elems != nullptr) {
      *elems = need;
      return 0;
    }
    if (a.work_elems < need) return -5;
  }
  const int smem = bwd ? B::S * B::ROW * MAXT + p.groups * a.D * 4 : F::S * F::ROW * MAXT;
  const uint32_t esz = sizeof(T);
  const NormStrides ld = {(uint32_t)a.ldx * esz, (uint32_t)a.ldh * esz, (uint32_t)a.ldgy * esz, (uint32_t)a.ldgn * esz,
                          (uint32_t)a.D * esz};
  if (smem > 48 * 1024) {
    // the most that any D asks of the kernel: a block has 16 elements of a row to a thread at most
    const cudaError_t e =
        bwd ? allow_smem<KernelKey<norm_bwd_kernel<T, V, IT, MAXT, MIS>>>((const void*)norm_bwd_kernel<T, V, IT, MAXT, MIS>,
                                                                     B::S * B::ROW * MAXT + MAXT * 16 * 4)
            : allow_smem<KernelKey<norm_fwd_kernel<T, V, IT, MAXT, MIS>>>((const void*)norm_fwd_kernel<T, V, IT, MAXT, MIS>,
                                                                     F::S * F::ROW * MAXT);
    if (e != cudaSuccess) return -100 - (int)e;
  }
  if (!bwd) {
    norm_fwd_kernel<T, V, IT, MAXT, MIS><<<blocks, p.block, smem, s>>>(a, p.tpr, ch, ld);
    return launch_status();
  }
  norm_bwd_kernel<T, V, IT, MAXT, MIS><<<blocks, p.block, smem, s>>>(a, p.tpr, ch, ld);
  const dim3 grid((a.D + 31) / 32, 2 + (a.gate != nullptr && ch.cpg > 1 ? ch.n / ch.cpg : 0));
  norm_sum_kernel<T><<<grid, 1024, 0, s>>>(a, blocks, ch);
  return launch_status();
}

template <typename T, int V, bool MIS>
static int norm_go(const InbNormArgs& a, const NormPlan& p, bool bwd, int64_t* elems, cudaStream_t s) {
  // rows of 8 elements a thread are narrow (D <= 256): they never need more than 256 threads
  if (p.IT * V == 8) return norm_launch<T, V, 8 / V, 256, MIS>(a, p, bwd, elems, s);
  return p.block > 256 ? norm_launch<T, V, 16 / V, 512, MIS>(a, p, bwd, elems, s)
                       : norm_launch<T, V, 16 / V, 256, MIS>(a, p, bwd, elems, s);
}

template <typename T>
static int norm_type(const InbNormArgs& a, bool bwd, int64_t* elems, cudaStream_t s) {
  const NormPlan p = norm_plan(a, bwd);
  if constexpr (sizeof(T) == 2) {
    if (p.mis) return norm_go<T, 8, true>(a, p, bwd, elems, s);
    return p.V == 8 ? norm_go<T, 8, false>(a, p, bwd, elems, s) : norm_go<T, 2, false>(a, p, bwd, elems, s);
  } else {
    return p.V == 4 ? norm_go<T, 4, false>(a, p, bwd, elems, s) : norm_go<T, 1, false>(a, p, bwd, elems, s);
  }
}

static int norm_run(const InbNormArgs& a, bool bwd, int64_t* elems, void* stream) {
  cudaStream_t s = (cudaStream_t)stream;
  if (a.dtype == INB_BF16) return norm_type<bf16>(a, bwd, elems, s);
  if (a.dtype == INB_F16) return norm_type<f16>(a, bwd, elems, s);
  return norm_type<float>(a, bwd, elems, s);
}

}  // namespace pol
}  // namespace inb

extern "C" int inb_block_norm_fwd(const InbNormArgs* args, void* cuda_stream) {
  const int rc = inb::pol::norm_check(args, false);
  if (rc != 0 || args->N == 0) return rc;
  return inb::pol::norm_run(*args, false, nullptr, cuda_stream);
}

extern "C" int inb_block_norm_work(const InbNormArgs* args, int64_t* elems) {
  if (elems == nullptr) return -1;
  *elems = 0;
  const int rc = inb::pol::norm_check(args, false, true);
  if (rc != 0 || args->N == 0) return rc;
  return inb::pol::norm_run(*args, true, elems, nullptr);
}

extern "C" int inb_block_norm_bwd(const InbNormArgs* args, void* cuda_stream) {
  const int rc = inb::pol::norm_check(args, true);
  if (rc != 0 || args->N == 0) return rc;
  return inb::pol::norm_run(*args, true, nullptr, cuda_stream);
}
