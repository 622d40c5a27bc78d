// distill_loss: cross entropy from a teacher's top logits, less the teacher's own entropy, a row at a time.
//
//   z = logits / tau over the allowed elements, q = exp(z - m) / l, m = max z, l = sum exp(z - m)
//   p = softmax(teacher / tau) over the entries in use;  loss = tau^2 sum_k p_k (log p_k - log q_k)
//   glogits = gloss tau (q - p)
//
// Bound by DRAM where rows are long: the forward call reads the logits once (running maximum and sum, one exponential an
// element), the backward call reads them again and writes the gradient.  8192 rows of 32001 bf16: 121 us forward (4.3 TB/s),
// 178 us backward (5.9 TB/s).  Rows of up to 128 logits are 8 lanes', which hold them in registers, longer ones a warp's, very
// long ones and few a block's or a cluster of blocks' (forward: joined through distributed shared memory; 64 rows of 131072:
// 11 + 10 us).  Short rows are bound by latency and by their lists (131072 rows of 33, lists of 8: 21 + 23 us).  Rows may start
// anywhere: what lies before the first and behind the last 16-byte boundary goes element by element.
#include <cooperative_groups.h>

#include "policy_seq.cuh"

namespace inb {
namespace pol {
namespace cg = cooperative_groups;

// Which form a call takes, by the length of its rows and lists and by its rows.  Forward + backward, bf16:
//   GROUP, 8 lanes a row, against a warp a row: 262144 rows of 33 with lists of 8 86 us against 301, of 100 and 8 121 against
//     287, of 100 and 64 301 against 397; of 160 and 8 (131072 rows) 111 against 139, but of 256 and 32 212 against 152
//   WARP, one access of a lane on its way, 8 blocks an SM, against DEEP: 65536 rows of 700 121 us against 137, of 1024 166 against
//     184; but 4096 rows of 1024, fewer than the GPU holds warps, 27 against 21
//   DEEP, a warp a row, four accesses, 4 blocks an SM, against BLOCK: 32768 rows of 2048 113 us against 301, 16384 of 4000 104
//     against 182, 8192 of 8192 102 against 121, of 16384 176 against 178, of 32001 334 against 315; 2048 rows of 4000 31 against
//     35, 1024 rows 27 against 25, 64 rows 39 against 16: a warp's time goes by the row, the blocks' by the rows.
//     With lists of 512 32768 rows of 2048 867 us against 1411, 64 rows of 400 70 against 35
//   BLOCK: four accesses, 5 blocks an SM.  8192 rows of 32001: 315 us; 335 with 4 blocks, 346 with 6, 324 with 2 accesses and 8
//     blocks, 368 with 8 and 3; 320 with blocks of 128 threads, 342 of 512; 358 with resident blocks that send for the next row
//     by cp.async.  `parts` blocks, a cluster, share a row while all are resident: 64 rows of 131072 29 us with 8, 57 with 1
enum { DIST_GROUP, DIST_WARP, DIST_DEEP, DIST_BLOCK };
constexpr int DIST_THREADS = 256, DIST_GROUP_V = 128, DIST_GROUP_K = 64, DIST_WARP_V = 1024, DIST_DEEP_V = 16384, DIST_WARP_K = 512;
template <int FORM>
struct Form {
  static constexpr bool WARP = FORM != DIST_BLOCK;
  static constexpr int U = FORM == DIST_WARP ? 1 : 4;               // accesses of a thread on their way at once
  static constexpr int BLOCKS = FORM == DIST_WARP ? 8 : FORM == DIST_DEEP ? 4 : 5;      // an SM
};

template <typename T>
struct RowView {
  static constexpr int W = 16 / sizeof(T);      // elements of an access
  const T* x;
  const uint8_t* mask;
  int V, head, nvec;         // elements before the first access, accesses
  RowView() = default;
  __device__ RowView(const InbDistillArgs& a, int64_t r, const T* out) {
    x = (const T*)a.logits + r * a.ld;
    mask = a.mask != nullptr ? a.mask + r * a.ld_mask : nullptr;
    V = a.V;
    head = (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T);
    bool fits = head < V && (((uintptr_t)x) & (sizeof(T) - 1)) == 0;
    if (out != nullptr) fits = fits && (((uintptr_t)x ^ (uintptr_t)out) & 15) == 0;
    if (mask != nullptr) fits = fits && (((uintptr_t)mask + head) & (W - 1)) == 0;
    if (!fits) head = V;
    nvec = (V - head) / W;
  }
  // the elements of part r of n: accesses [v0, v1), and the elements [lo, hi) around them
  __device__ void part(int r, int n, int& v0, int& v1, int& lo, int& hi) const {
    v0 = (int)((int64_t)nvec * r / n), v1 = (int)((int64_t)nvec * (r + 1) / n);
    lo = r == 0 ? 0 : head + v0 * W;
    hi = r == n - 1 ? V : head + v1 * W;
  }
  // U accesses, `stride` apart from v, of those below end: all on their way before the first is used
  template <int U>
  struct Batch {
    Words<T, W> q[U];
    Words<uint8_t, W> m[U];
  };
  template <int U>
  __device__ __forceinline__ void load(Batch<U>& b, int v, int stride, int end) const {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * stride < end) {
        b.q[u].load(x + head + (v + u * stride) * W);
        if (mask != nullptr) b.m[u].load(mask + head + (v + u * stride) * W);
      }
  }
  // an access's elements, -inf where they are not allowed
  template <int U>
  __device__ __forceinline__ void get(const Batch<U>& b, int u, float (&o)[W]) const {
#pragma unroll
    for (int k = 0; k < W; k += 2) {
      const float2 p = b.q[u].pair(k / 2);
      o[k] = p.x, o[k + 1] = p.y;
    }
    if (mask != nullptr) {
#pragma unroll
      for (int k = 0; k < W; ++k)
        if ((b.m[u].w[k / 4] >> (k % 4 * 8) & 0xFF) == 0) o[k] = -INFINITY;
    }
  }
  __device__ float load1(int i) const { return mask == nullptr || mask[i] != 0 ? to_f(x[i]) : -INFINITY; }
};

// An entry of the teacher's list as it lies in memory, and after the student's logit there has been looked at: the teacher's
// logit, -inf where it is not in use (index then -1); z: the student's logit
struct Entry {
  int64_t i;
  float t, z;
  int index;
  __device__ __forceinline__ void fetch(const InbDistillArgs& a, int64_t at) {
    i = a.index[at];
    if (a.teacher_dtype == INB_BF16)
      t = to_f(((const bf16*)a.teacher)[at]);
    else if (a.teacher_dtype == INB_F16)
      t = to_f(((const f16*)a.teacher)[at]);
    else
      t = ((const float*)a.teacher)[at];
  }
  template <typename T>
  __device__ __forceinline__ void look(const InbDistillArgs& a, const RowView<T>& row) {
    const bool in = i >= 0 && i < a.V;
    index = in ? (int)i : -1;
    z = in ? row.load1(index) : -INFINITY;
    if (z == -INFINITY || t != t || t == -INFINITY) t = -INFINITY, index = -1;
  }
};

// running maximum and sum of exp((v - m) c / log2 e)
struct Soft {
  float m = -INFINITY, l = 0.f;
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N], float c) {
    float top = v[0];
#pragma unroll
    for (int k = 1; k < N; ++k) top = fmaxf(top, v[k]);
    if (top > m) {
      l *= ex2((m - top) * c);
      m = top;
    }
    const float at = m == -INFINITY ? 0.f : m;
    if constexpr (N % 2 == 0) {
      float2 s = make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        const float2 z = mul2(add2(make_float2(v[k], v[k + 1]), both(-at)), both(c));
        s = add2(s, make_float2(ex2(z.x), ex2(z.y)));
      }
      l += s.x + s.y;
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) l += ex2((v[k] - at) * c);
    }
  }
  __device__ __forceinline__ void join(float om, float ol, float c) {
    const float top = fmaxf(m, om), at = top == -INFINITY ? 0.f : top;
    l = l * ex2((m - at) * c) + ol * ex2((om - at) * c);
    m = top;
  }
  __device__ __forceinline__ void over_warp(float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xFFFFFFFFu, m, o), ol = __shfl_xor_sync(0xFFFFFFFFu, l, o);
      join(om, ol, c);
    }
  }
};
template <int L>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// What the backward call knows of a row: q = rl exp(z - m), p = rp exp(teacher / tau - top); 0 where no entry is in use, whatever
// the row's logits are
struct Grad {
  float4 stat;
  float g, gl, c;
  bool live;
  __device__ __forceinline__ Grad(const InbDistillArgs& a, int64_t r, float c) : c(c) {
    stat = *reinterpret_cast<const float4*>(a.stats + 4 * r);
    live = stat.w != 0.f;
    g = a.gloss[r] * a.tau, gl = g * stat.y;
  }
  __device__ __forceinline__ float value(float v) const { return live && v != -INFINITY ? gl * ex2((v - stat.x) * c) : 0.f; }
  // an entry of the row's list as (index or -1, p)
  template <typename T>
  __device__ __forceinline__ float2 listed(const InbDistillArgs& a, const RowView<T>& row, Entry e) const {
    e.look(a, row);
    return make_float2(__int_as_float(live ? e.index : -1), ex2((e.t - stat.z) * c) * stat.w);
  }
  // a listed element, from q and the sum of its entries: every entry of an index gives the same value
  __device__ __forceinline__ float at(float z, float p) const { return g * (stat.y * ex2((z - stat.x) * c) - p); }
};

__host__ __device__ inline int list_room(int K) { return (K + 1) / 2 * 2; }      // pairs of a list in shared memory
// A row's list by L lanes: some entries a lane in registers, on their way while the row is; those beyond them from memory later.
// Every lane of the warp takes part.
template <typename T, int L>
struct Entries {
  static constexpr int HELD = L == 8 ? 4 : L == 32 ? 2 : 1;
  Entry e[HELD];
  __device__ __forceinline__ void fetch(const InbDistillArgs& a, int64_t r, int lane) {
#pragma unroll
    for (int q = 0; q < HELD; ++q) {
      e[q].i = -1, e[q].t = 0.f;
      if (lane + q * L < a.K) e[q].fetch(a, r * a.K + lane + q * L);
    }
  }
  __device__ __forceinline__ void look(const InbDistillArgs& a, const RowView<T>& row) {
#pragma unroll
    for (int q = 0; q < HELD; ++q) e[q].look(a, row);
  }
  // backward: the list as pairs (index or -1, p), an even number of them
  __device__ __forceinline__ void write(const InbDistillArgs& a, const RowView<T>& row, int64_t r, const Grad& g, int lane, float2* list) const {
#pragma unroll
    for (int q = 0; q < HELD; ++q)
      if (lane + q * L < a.K) list[lane + q * L] = g.listed(a, row, e[q]);
    for (int k = lane + HELD * L; k < a.K; k += L) {
      Entry n;
      n.fetch(a, r * a.K + k);
      list[k] = g.listed(a, row, n);
    }
    if (lane == 0 && (a.K & 1) != 0) list[a.K] = make_float2(__int_as_float(-1), 0.f);
  }
  // and, once all of it is there, the listed elements within [lo, hi) of the gradient's row
  __device__ __forceinline__ void mark(const InbDistillArgs& a, const RowView<T>& row, const Grad& g, int lane, const float2* list, int lo,
                                       int hi, T* out) const {
    if (a.K <= L)
      mark_by<1>(a, row, g, lane, list, lo, hi, out);
    else
      mark_by<HELD>(a, row, g, lane, list, lo, hi, out);
  }
  // B elements a lane at a time, each the sum over the list
  template <int B>
  __device__ __forceinline__ void mark_by(const InbDistillArgs& a, const RowView<T>& row, const Grad& g, int lane, const float2* list, int lo,
                                          int hi, T* out) const {
    for (int k0 = lane; k0 < a.K; k0 += B * L) {
      int i[B];
      float z[B], p[B];
#pragma unroll
      for (int q = 0; q < B; ++q) {
        i[q] = k0 + q * L < a.K ? __float_as_int(list[k0 + q * L].x) : -1;
        if (i[q] < lo || i[q] >= hi) i[q] = -1;
        z[q] = i[q] >= 0 ? row.load1(i[q]) : 0.f;
        p[q] = 0.f;
      }
      for (int o = 0; o < a.K; o += 2) {
        const float4 two = *reinterpret_cast<const float4*>(list + o);
#pragma unroll
        for (int q = 0; q < B; ++q) {
          if (__float_as_int(two.x) == i[q]) p[q] += two.y;
          if (__float_as_int(two.z) == i[q]) p[q] += two.w;
        }
      }
#pragma unroll
      for (int q = 0; q < B; ++q)
        if (i[q] >= 0) out[i[q]] = from_f<T>(g.at(z[q], p[q]));
    }
  }
  // forward: the loss, and what the backward call needs
  __device__ __forceinline__ void finish(const InbDistillArgs& a, const RowView<T>& row, int64_t r, float m, float l, float c, int lane,
                                         bool on) const {
    float top = e[0].t;
#pragma unroll
    for (int q = 1; q < HELD; ++q) top = fmaxf(top, e[q].t);
    for (int k = lane + HELD * L; k < a.K; k += L) {
      Entry n;
      n.fetch(a, r * a.K + k);
      n.look(a, row);
      top = fmaxf(top, n.t);
    }
    top = lanes_max<L>(top);
    const bool live = top != -INFINITY;
    float mass = 0.f, sum = 0.f;
    const float inv = c * LN2;                      // 1 / tau
    auto add = [&](const Entry& n) {
      if (n.index < 0) return;
      const float w = ex2((n.t - top) * c);
      mass += w;
      sum = fmaf(w, ((n.t - top) - (n.z - m)) * inv, sum);
    };
#pragma unroll
    for (int q = 0; q < HELD; ++q) add(e[q]);
    for (int k = lane + HELD * L; k < a.K; k += L) {
      Entry n;
      n.fetch(a, r * a.K + k);
      n.look(a, row);
      add(n);
    }
    mass = lanes_sum<L>(mass);
    sum = lanes_sum<L>(sum);
    if (!on || lane != 0) return;
    a.loss[r] = live ? a.tau * a.tau * (sum / mass + (logf(l) - logf(mass))) : 0.f;
    if (a.stats != nullptr)
      *reinterpret_cast<float4*>(a.stats + 4 * r) = live ? make_float4(m, 1.f / l, top, 1.f / mass) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
};

// A row a warp, or (BLOCK) a row `parts` blocks
template <typename T, int FORM>
__global__ void __launch_bounds__(DIST_THREADS, Form<FORM>::BLOCKS) distill_fwd_kernel(InbDistillArgs a, int parts, float c) {
  constexpr bool WARP = Form<FORM>::WARP;
  constexpr int TPR = WARP ? 32 : DIST_THREADS, W = RowView<T>::W, U = Form<FORM>::U;
  const int tid = threadIdx.x % TPR, lane = threadIdx.x & 31;
  const int64_t r = WARP ? (int64_t)blockIdx.x * (DIST_THREADS / 32) + threadIdx.x / 32 : blockIdx.x / parts;
  const int part = WARP ? 0 : blockIdx.x % parts;
  if (WARP && r >= a.N) return;
  const RowView<T> row(a, r, nullptr);
  int v0, v1, lo, hi;
  row.part(part, parts, v0, v1, lo, hi);
  Soft s;
  Entries<T, 32> list;
  const bool lists = WARP || (part == 0 && threadIdx.x < 32);
  if (lists) list.fetch(a, r, lane);
  for (int v = v0 + tid; v < v1; v += TPR * U) {
    typename RowView<T>::template Batch<U> b;
    row.load(b, v, TPR, v1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v + u * TPR >= v1) break;
      float x[W];
      row.get(b, u, x);
      s.add(x, c);
    }
  }
  const int body = row.head + v0 * W, end = row.head + v1 * W;
  for (int i = lo + tid; i < body; i += TPR) {
    const float x[1] = {row.load1(i)};
    s.add(x, c);
  }
  for (int i = end + tid; i < hi; i += TPR) {
    const float x[1] = {row.load1(i)};
    s.add(x, c);
  }
  if (lists) list.look(a, row);
  s.over_warp(c);
  if (WARP) {
    list.finish(a, row, r, s.m, s.l, c, lane, true);
    return;
  }
  __shared__ float2 warps[DIST_THREADS / 32];
  __shared__ float2 block;
  if (lane == 0) warps[threadIdx.x / 32] = make_float2(s.m, s.l);
  __syncthreads();
  if (threadIdx.x < 32) {
    s = Soft();
    for (int w = 0; w < DIST_THREADS / 32; ++w) s.join(warps[w].x, warps[w].y, c);
    if (lane == 0) block = make_float2(s.m, s.l);
  }
  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (lists) {
      s = Soft();
      for (int p = 0; p < parts; ++p) {
        const float2 o = *cluster.map_shared_rank(&block, p);
        s.join(o.x, o.y, c);
      }
    }
    cluster.sync();         // a block's memory lives until it has been read
  }
  if (lists) list.finish(a, row, r, s.m, s.l, c, lane, true);
}

template <typename T, int FORM>
__global__ void __launch_bounds__(DIST_THREADS, Form<FORM>::BLOCKS) distill_bwd_kernel(InbDistillArgs a, int parts, float c) {
  constexpr bool WARP = Form<FORM>::WARP;
  constexpr int TPR = WARP ? 32 : DIST_THREADS, W = RowView<T>::W, U = Form<FORM>::U;
  extern __shared__ float4 lists[];
  const int tid = threadIdx.x % TPR;
  const int64_t r = WARP ? (int64_t)blockIdx.x * (DIST_THREADS / 32) + threadIdx.x / 32 : blockIdx.x / parts;
  const int part = WARP ? 0 : blockIdx.x % parts;
  if (WARP && r >= a.N) return;
  T* out = (T*)a.glogits + r * a.V;
  const RowView<T> row(a, r, out);
  int v0, v1, lo, hi;
  row.part(part, parts, v0, v1, lo, hi);
  const Grad g(a, r, c);
  float2* list = (float2*)lists + (WARP ? threadIdx.x / 32 * list_room(a.K) : 0);
  Entries<T, TPR> entries;
  entries.fetch(a, r, tid);
  for (int v = v0 + tid; v < v1; v += TPR * U) {
    typename RowView<T>::template Batch<U> b;
    row.load(b, v, TPR, v1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v + u * TPR >= v1) break;
      float x[W];
      row.get(b, u, x);
      Words<T, W> o;
#pragma unroll
      for (int k = 0; k < W; k += 2) o.set(k / 2, make_float2(g.value(x[k]), g.value(x[k + 1])));
      o.store(out + row.head + (v + u * TPR) * W);
    }
  }
  const int body = row.head + v0 * W, end = row.head + v1 * W;
  for (int i = lo + tid; i < body; i += TPR) out[i] = from_f<T>(g.value(row.load1(i)));
  for (int i = end + tid; i < hi; i += TPR) out[i] = from_f<T>(g.value(row.load1(i)));
  entries.write(a, row, r, g, tid, list);
  if (WARP)
    __syncwarp();
  else
    __syncthreads();
  entries.mark(a, row, g, tid, list, lo, hi, out);
}

// Short rows: 8 lanes hold one
template <typename T, int M, bool BACK>
__global__ void __launch_bounds__(DIST_THREADS) distill_short_kernel(InbDistillArgs a, float c) {
  constexpr int L = 8;
  extern __shared__ float4 lists[];
  const int lane = threadIdx.x % L;
  const int64_t r0 = (int64_t)blockIdx.x * (DIST_THREADS / L) + threadIdx.x / L;
  const bool on = r0 < a.N;
  const int64_t r = on ? r0 : a.N - 1;           // lanes without a row read the last one and write nothing
  RowView<T> row;
  row.x = (const T*)a.logits + r * a.ld;
  row.mask = a.mask != nullptr ? a.mask + r * a.ld_mask : nullptr;
  uint32_t raw[M], ok[M];
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int k = i * L + lane;
    raw[i] = ok[i] = 0;
    if (k < a.V) {
      raw[i] = ld_raw(row.x + k);
      ok[i] = row.mask != nullptr ? row.mask[k] : 1;
    }
  }
  Entries<T, L> entries;
  entries.fetch(a, r, lane);
  if constexpr (!BACK) {
    float x[M];
#pragma unroll
    for (int i = 0; i < M; ++i) x[i] = ok[i] ? raw_f<T>(raw[i]) : -INFINITY;
    float m = x[0];
#pragma unroll
    for (int i = 1; i < M; ++i) m = fmaxf(m, x[i]);
    m = lanes_max<L>(m);
    entries.look(a, row);
    const float at = m == -INFINITY ? 0.f : m;
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < M; ++i)
      if (i * L < a.V) l += ex2((x[i] - at) * c);
    l = lanes_sum<L>(l);
    entries.finish(a, row, r, m, l, c, lane, on);
  } else {
    T* out = (T*)a.glogits + r * a.V;
    const Grad g(a, r, c);
    float2* list = (float2*)lists + threadIdx.x / L * list_room(a.K);
    entries.write(a, row, r, g, lane, list);
#pragma unroll
    for (int i = 0; i < M; ++i)
      if (on && i * L + lane < a.V) out[i * L + lane] = from_f<T>(g.value(ok[i] ? raw_f<T>(raw[i]) : -INFINITY));
    __syncwarp();
    entries.mark(a, row, g, lane, list, 0, on ? a.V : 0, out);
  }
}

struct DistPlan {
  int form, parts, rows;         // blocks that share a row, rows of a block
  unsigned blocks;
};
static DistPlan dist_plan(const InbDistillArgs& a) {
  DistPlan p = {DIST_BLOCK, 1, 1, 0};
  const int64_t row = a.V > 8 * a.K ? a.V : 8 * a.K;      // what a warp's time goes by
  if (a.V <= DIST_GROUP_V && a.K <= DIST_GROUP_K)
    p.form = DIST_GROUP, p.rows = DIST_THREADS / 8;
  else if (a.V <= DIST_DEEP_V && a.K <= DIST_WARP_K && (row <= DIST_WARP_V / 2 || a.N * 2 >= row))
    p.form = a.V <= DIST_WARP_V && a.N >= sm_count() * 64 ? DIST_WARP : DIST_DEEP, p.rows = DIST_THREADS / 32;
  else
    while (p.parts < 8 && a.N * p.parts * 2 <= sm_count() * Form<DIST_BLOCK>::BLOCKS && a.V / (2 * p.parts) >= 4096) p.parts *= 2;
  p.blocks = (unsigned)(ceil_div(a.N, p.rows) * p.parts);
  return p;
}
template <typename T>
static int dist_fwd(const InbDistillArgs& a, cudaStream_t s) {
  const DistPlan p = dist_plan(a);
  const float c = LOG2E / a.tau;
  if (p.form == DIST_GROUP) {
    const auto kernel = a.V <= DIST_GROUP_V / 2 ? distill_short_kernel<T, 8, false> : distill_short_kernel<T, 16, false>;
    kernel<<<p.blocks, DIST_THREADS, 0, s>>>(a, c);
    return launch_status();
  }
  if (p.form != DIST_BLOCK) {
    const auto kernel = p.form == DIST_WARP ? distill_fwd_kernel<T, DIST_WARP> : distill_fwd_kernel<T, DIST_DEEP>;
    kernel<<<p.blocks, DIST_THREADS, 0, s>>>(a, 1, c);
    return launch_status();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.blocks);
  cfg.blockDim = dim3(DIST_THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)p.parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, distill_fwd_kernel<T, DIST_BLOCK>, a, p.parts, c);
  return e == cudaSuccess ? launch_status() : -100 - (int)e;
}
template <typename T>
static int dist_bwd(const InbDistillArgs& a, cudaStream_t s) {
  const DistPlan p = dist_plan(a);
  const float c = LOG2E / a.tau;
  const size_t smem = (size_t)p.rows * list_room(a.K) * 8;      // at most 32 KB
  if (p.form == DIST_GROUP) {
    const auto kernel = a.V <= DIST_GROUP_V / 2 ? distill_short_kernel<T, 8, true> : distill_short_kernel<T, 16, true>;
    kernel<<<p.blocks, DIST_THREADS, smem, s>>>(a, c);
  } else {
    const auto kernel = p.form == DIST_WARP   ? distill_bwd_kernel<T, DIST_WARP>
                        : p.form == DIST_DEEP ? distill_bwd_kernel<T, DIST_DEEP>
                                              : distill_bwd_kernel<T, DIST_BLOCK>;
    kernel<<<p.blocks, DIST_THREADS, smem, s>>>(a, p.parts, c);
  }
  return launch_status();
}
static int dist_check(const InbDistillArgs& a) {
  if (a.dtype < 0 || a.dtype > 2 || a.teacher_dtype < 0 || a.teacher_dtype > 2 || a.V < 1 || a.V > INB_MAX_SAMPLE_V || a.K < 1 ||
      a.K > INB_MAX_DISTILL_K || a.N < 0 || a.N > INB_MAX_SAMPLE_N || !(a.tau > 0.f) || a.tau > 3e38f)
    return -2;
  return 0;
}

}  // namespace pol
}  // namespace inb

extern "C" int inb_distill_fwd(const InbDistillArgs* args, void* cuda_stream) {
  if (args == nullptr) return -1;
  const InbDistillArgs& a = *args;
  const int rc = inb::pol::dist_check(a);
  if (rc != 0) return rc;
  if (a.N == 0) return 0;
  if (a.logits == nullptr || a.teacher == nullptr || a.index == nullptr || a.loss == nullptr || ((uintptr_t)a.stats & 15) != 0)
    return -3;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (a.dtype == INB_BF16) return inb::pol::dist_fwd<inb::pol::bf16>(a, s);
  if (a.dtype == INB_F16) return inb::pol::dist_fwd<inb::pol::f16>(a, s);
  return inb::pol::dist_fwd<float>(a, s);
}

extern "C" int inb_distill_bwd(const InbDistillArgs* args, void* cuda_stream) {
  if (args == nullptr) return -1;
  const InbDistillArgs& a = *args;
  const int rc = inb::pol::dist_check(a);
  if (rc != 0) return rc;
  if (a.N == 0) return 0;
  if (a.logits == nullptr || a.teacher == nullptr || a.index == nullptr || a.stats == nullptr || a.gloss == nullptr ||
      a.glogits == nullptr || ((uintptr_t)a.stats & 15) != 0)
    return -3;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (a.dtype == INB_BF16) return inb::pol::dist_bwd<inb::pol::bf16>(a, s);
  if (a.dtype == INB_F16) return inb::pol::dist_bwd<inb::pol::f16>(a, s);
  return inb::pol::dist_bwd<float>(a, s);
}
