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
// Both directions are bound by DRAM: 4 (forward) and 6 (backward) row passes of N x D elements.
#include "policy_common.cuh"

namespace inb {
namespace pol {

struct NormPlan {
  int V, IT;          // elements of one access, accesses of one thread
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
  const int esz = a.dtype == INB_F32 ? 4 : 2;
  if (p.V * esz == 16)
    p.IT = esz == 2 ? (a.D > 256 ? 2 : 1) : (a.D > 2048 ? 4 : 2);
  else
    p.IT = p.V == 2 ? 8 : 16;
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

// MAXT: the largest block it is launched with, which sets the registers that a thread may hold a row in
template <typename T, int V, int IT, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_fwd_kernel(InbNormArgs a, int tpr) {
  __shared__ float red[8][64];
  const int group = threadIdx.x / tpr, t = threadIdx.x % tpr, groups = blockDim.x / tpr;
  const int D = a.D;
  const float inv_d = 1.f / (float)D;
  const T *w = (const T*)a.w, *post = (const T*)a.post;
  Pack<T, V> wr[IT], pr[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = (i * tpr + t) * V;
    if (c < D) {
      wr[i] = ld<T, V>(w + c);
      if (post) pr[i] = ld<T, V>(post + c);
    }
  }
  int par = 0;
  const int64_t stride = (int64_t)gridDim.x * groups;
  for (int64_t row = (int64_t)blockIdx.x * groups + group; row < a.N; row += stride) {
    const T* xp = (const T*)a.x + row * a.ldx;
    const T* hp = (const T*)a.h + row * a.ldh;
    const T* gp = a.gate ? (const T*)a.gate + row / a.gate_rows * D : nullptr;
    Pack<T, V> xr[IT], hr[IT], gr[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * tpr + t) * V;
      if (c < D) {
        xr[i] = ld<T, V>(xp + c);
        if (a.h) hr[i] = ld<T, V>(hp + c);
        if (gp) gr[i] = ld<T, V>(gp + c);
      }
    }
    float rh = 1.f;
    if (post) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if ((i * tpr + t) * V < D)
#pragma unroll
          for (int e = 0; e < V; ++e) s = fmaf(to_f(hr[i].v[e]), to_f(hr[i].v[e]), s);
      rh = rsqrtf(row_sum(s, tpr, group, t, red[group], par) * inv_d + a.eps);
    }
    float y[IT][V], s = 0.f;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * tpr + t) * V;
      if (c < D) {
        Pack<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float v = to_f(xr[i].v[e]);
          if (a.h) {
            float p = to_f(hr[i].v[e]);
            if (post) p = p * rh * to_f(pr[i].v[e]);
            v += (gp ? a.scale * to_f(gr[i].v[e]) : a.scale) * p;
          }
          y[i][e] = v;
          s = fmaf(v, v, s);
          o.v[e] = from_f<T>(v);
        }
        if (a.y) st<T, V>((T*)a.y + row * D + c, o);
      }
    }
    const float ry = rsqrtf(row_sum(s, tpr, group, t, red[group], par) * inv_d + a.eps);
    if (a.stats && t == 0) {
      a.stats[2 * row] = rh;
      a.stats[2 * row + 1] = ry;
    }
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * tpr + t) * V;
      if (c < D) {
        Pack<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.v[e] = from_f<T>(y[i][e] * ry * to_f(wr[i].v[e]));
        st<T, V>((T*)a.n + row * D + c, o);
      }
    }
  }
}

// Rows are cut into chunks that never cross a gate's rows: chunk c = rows [g R + k len, ...) of gate g = c / cpg.
struct NormChunks {
  int64_t n;       // chunks
  int64_t rows;    // rows of one gate (N without a gate)
  int64_t len;     // rows of a chunk
  int cpg;         // chunks of one gate
};

template <typename T, int V, int IT, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_bwd_kernel(InbNormArgs a, int tpr, NormChunks ch) {
  __shared__ float red[8][64];
  extern __shared__ float comb[];
  const int group = threadIdx.x / tpr, t = threadIdx.x % tpr, groups = blockDim.x / tpr;
  const int D = a.D;
  const float inv_d = 1.f / (float)D;
  const T *w = (const T*)a.w, *post = (const T*)a.post;
  const bool has_h = a.h != nullptr;
  Pack<T, V> wr[IT], pr[IT];
  float aw[IT][V], ap[IT][V];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = (i * tpr + t) * V;
    if (c < D) {
      wr[i] = ld<T, V>(w + c);
      if (post) pr[i] = ld<T, V>(post + c);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) aw[i][e] = ap[i][e] = 0.f;
  }
  int par = 0;
  float* part_gate = a.work + 2 * (int64_t)gridDim.x * D;
  for (int64_t c0 = (int64_t)blockIdx.x * groups + group; c0 < ch.n; c0 += (int64_t)gridDim.x * groups) {
    const int64_t gi = c0 / ch.cpg, k = c0 - gi * ch.cpg;
    const int64_t r0 = gi * ch.rows + k * ch.len;
    int64_t r1 = r0 + ch.len;
    if (r1 > (gi + 1) * ch.rows) r1 = (gi + 1) * ch.rows;
    Pack<T, V> gr[IT];
    float ag[IT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * tpr + t) * V;
      if (a.gate && c < D) gr[i] = ld<T, V>((const T*)a.gate + gi * D + c);
#pragma unroll
      for (int e = 0; e < V; ++e) ag[i][e] = 0.f;
    }
    for (int64_t row = r0; row < r1; ++row) {
      Pack<T, V> xr[IT], hr[IT], yr[IT], nr[IT];
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (i * tpr + t) * V;
        if (c < D) {
          xr[i] = ld<T, V>((const T*)a.x + row * a.ldx + c);
          if (has_h) hr[i] = ld<T, V>((const T*)a.h + row * a.ldh + c);
          if (a.gn) nr[i] = ld<T, V>((const T*)a.gn + row * a.ldgn + c);
          if (a.gy) yr[i] = ld<T, V>((const T*)a.gy + row * a.ldgy + c);
        }
      }
      const float rh = a.stats[2 * row], ry = a.stats[2 * row + 1];
      float tt[IT][V];
      // yh is recomputed from x and h, then replaced by t
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if ((i * tpr + t) * V < D)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float v = to_f(xr[i].v[e]);
            if (has_h) {
              float p = to_f(hr[i].v[e]);
              if (post) p = p * rh * to_f(pr[i].v[e]);
              v += (a.gate ? a.scale * to_f(gr[i].v[e]) : a.scale) * p;
            }
            v *= ry;
            tt[i][e] = v;
            if (a.gn) {
              const float gn = to_f(nr[i].v[e]);
              aw[i][e] = fmaf(gn, v, aw[i][e]);
              s = fmaf(gn * to_f(wr[i].v[e]), v, s);
            }
          }
      const float c1 = a.gn ? row_sum(s, tpr, group, t, red[group], par) * inv_d : 0.f;
      float s2 = 0.f;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (i * tpr + t) * V;
        if (c < D) {
          Pack<T, V> o;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float q = a.gn ? to_f(nr[i].v[e]) * to_f(wr[i].v[e]) : 0.f;
            float v = ry * (q - tt[i][e] * c1);
            if (a.gy) v += to_f(yr[i].v[e]);
            o.v[e] = from_f<T>(v);
            if (has_h) {
              const float hh = to_f(hr[i].v[e]) * rh;
              const float p = post ? hh * to_f(pr[i].v[e]) : hh;
              ag[i][e] = fmaf(v, p, ag[i][e]);
              v *= a.gate ? a.scale * to_f(gr[i].v[e]) : a.scale;   // gp
              if (post) {
                ap[i][e] = fmaf(v, hh, ap[i][e]);
                v *= to_f(pr[i].v[e]);
                s2 = fmaf(v, hh, s2);
              }
              tt[i][e] = v;
            }
          }
          st<T, V>((T*)a.gx + row * D + c, o);
        }
      }
      if (has_h) {
        const float c2 = post ? row_sum(s2, tpr, group, t, red[group], par) * inv_d : 0.f;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int c = (i * tpr + t) * V;
          if (c < D) {
            Pack<T, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e)
              o.v[e] = from_f<T>(post ? rh * (tt[i][e] - to_f(hr[i].v[e]) * rh * c2) : tt[i][e]);
            st<T, V>((T*)a.gh + row * D + c, o);
          }
        }
      }
    }
    if (a.ggate) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (i * tpr + t) * V;
        if (c < D) {
          if (ch.cpg == 1) {
            Pack<T, V> o;
#pragma unroll
            for (int e = 0; e < V; ++e) o.v[e] = from_f<T>(a.scale * ag[i][e]);
            st<T, V>((T*)a.ggate + gi * D + c, o);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) part_gate[c0 * D + c + e] = a.scale * ag[i][e];
          }
        }
      }
    }
  }
  // the block's column sums: group after group in order, then one partial row of each kind
  for (int kind = 0; kind < (post ? 2 : 1); ++kind) {
    for (int g = 0; g < groups; ++g) {
      if (g == group) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int c = (i * tpr + t) * V;
          if (c < D)
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float v = kind ? ap[i][e] : aw[i][e];
              const float sum = g == 0 ? v : comb[c + e] + v;
              if (g == groups - 1)
                a.work[((int64_t)blockIdx.x * 2 + kind) * D + c + e] = sum;
              else
                comb[c + e] = sum;
            }
        }
      }
      __syncthreads();
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

static NormChunks norm_chunks(const InbNormArgs& a, const NormPlan& p, int per_sm) {
  NormChunks c;
  const int64_t workers = (int64_t)sm_count() * per_sm * p.groups;
  c.rows = a.gate != nullptr ? a.gate_rows : a.N;
  const int64_t gates = a.N / c.rows;
  int64_t cpg = (workers + gates - 1) / gates;
  if (cpg > c.rows) cpg = c.rows;
  c.len = (c.rows + cpg - 1) / cpg;
  c.cpg = (int)((c.rows + c.len - 1) / c.len);
  c.n = gates * c.cpg;
  return c;
}

static int norm_bwd_per_sm(const NormPlan& p) { return p.block > 512 ? 1 : 2; }

static int64_t norm_work(const InbNormArgs& a) {
  const NormPlan p = norm_plan(a, true);
  const NormChunks ch = norm_chunks(a, p, norm_bwd_per_sm(p));
  const int64_t blocks = norm_blocks(p, ch.n, norm_bwd_per_sm(p));
  return (2 * blocks + (a.gate != nullptr && ch.cpg > 1 ? ch.n : 0)) * a.D;
}

template <typename T, int V, int IT, int MAXT>
static void norm_launch(const InbNormArgs& a, const NormPlan& p, bool bwd, cudaStream_t s) {
  if (!bwd) {
    norm_fwd_kernel<T, V, IT, MAXT><<<norm_blocks(p, a.N, p.block > 512 ? 2 : 8), p.block, 0, s>>>(a, p.tpr);
    return;
  }
  const NormChunks ch = norm_chunks(a, p, norm_bwd_per_sm(p));
  const int blocks = norm_blocks(p, ch.n, norm_bwd_per_sm(p));
  const int smem = p.groups > 1 ? a.D * 4 : 0;
  norm_bwd_kernel<T, V, IT, MAXT><<<blocks, p.block, smem, s>>>(a, p.tpr, ch);
  const dim3 grid((a.D + 31) / 32, 2 + (a.gate != nullptr && ch.cpg > 1 ? (unsigned)(ch.n / ch.cpg) : 0));
  norm_sum_kernel<T><<<grid, 1024, 0, s>>>(a, blocks, ch);
}

template <typename T, int V, int IT>
static void norm_go(const InbNormArgs& a, const NormPlan& p, bool bwd, cudaStream_t s) {
  if (p.block <= 256) norm_launch<T, V, IT, 256>(a, p, bwd, s);
  else if constexpr (V * IT == 16) {     // narrow rows, of fewer elements a thread, never need more threads
    norm_launch<T, V, IT, 512>(a, p, bwd, s);
  }
}

template <typename T>
static int norm_type(const InbNormArgs& a, bool bwd, cudaStream_t s) {
  const NormPlan p = norm_plan(a, bwd);
  constexpr int W = 16 / (int)sizeof(T);
  if (p.V == W) {
    if (p.IT == 1) norm_go<T, W, 1>(a, p, bwd, s);
    else if (p.IT == 2) norm_go<T, W, 2>(a, p, bwd, s);
    else if constexpr (sizeof(T) == 4) norm_go<T, W, 4>(a, p, bwd, s);
  } else if (p.V == 2) {
    if constexpr (sizeof(T) == 2) norm_go<T, 2, 8>(a, p, bwd, s);
  } else {
    norm_go<T, 1, 16>(a, p, bwd, s);
  }
  return launch_status();
}

static int norm_run(const InbNormArgs& a, bool bwd, void* stream) {
  cudaStream_t s = (cudaStream_t)stream;
  if (a.dtype == INB_BF16) return norm_type<bf16>(a, bwd, s);
  if (a.dtype == INB_F16) return norm_type<f16>(a, bwd, s);
  return norm_type<float>(a, bwd, s);
}

}  // namespace pol
}  // namespace inb

extern "C" int inb_block_norm_fwd(const InbNormArgs* args, void* cuda_stream) {
  const int rc = inb::pol::norm_check(args, false);
  if (rc != 0 || args->N == 0) return rc;
  return inb::pol::norm_run(*args, false, cuda_stream);
}

extern "C" int inb_block_norm_work(const InbNormArgs* args, int64_t* elems) {
  if (elems == nullptr) return -1;
  *elems = 0;
  const int rc = inb::pol::norm_check(args, false, true);
  if (rc != 0 || args->N == 0) return rc;
  *elems = inb::pol::norm_work(*args);
  return 0;
}

extern "C" int inb_block_norm_bwd(const InbNormArgs* args, void* cuda_stream) {
  const int rc = inb::pol::norm_check(args, true);
  if (rc != 0 || args->N == 0) return rc;
  if (args->work_elems < inb::pol::norm_work(*args)) return -5;
  return inb::pol::norm_run(*args, true, cuda_stream);
}
