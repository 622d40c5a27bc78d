// distill_loss: cross entropy from a teacher's top logits, less the teacher's own entropy, a row at a time.
//
//   z = logits / tau over the allowed elements, q = exp(z - m) / l, m = max z, l = sum exp(z - m)
//   p = softmax(teacher / tau) over the entries in use;  loss = tau^2 sum_k p_k (log p_k - log q_k)
//   glogits = gloss tau (q - p)
//
// Bound by DRAM: the forward call reads the logits once (running maximum and sum, one exponential an element), the
// backward call reads them again and writes the gradient.  Rows of up to 1024 logits are a warp's, longer ones a block's, and
// where rows are few a cluster of blocks shares one (forward: joined through distributed shared memory).  Rows may start
// anywhere: what lies before the first and behind the last 16-byte boundary goes element by element.
#include <cooperative_groups.h>

#include "policy_seq.cuh"

namespace inb {
namespace pol {
namespace cg = cooperative_groups;

constexpr int DIST_THREADS = 256, DIST_WARP_V = 1024, DIST_WARP_K = 128;

template <typename T>
struct RowView {
  static constexpr int W = 16 / sizeof(T);      // elements of an access
  const T* x;
  const uint8_t* mask;
  int V, head, nvec;         // elements before the first access, accesses
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
  __device__ bool allowed(int i) const { return mask == nullptr || mask[i] != 0; }
  // an access's elements, -inf where they are not allowed
  __device__ void load(int v, float (&o)[W]) const {
    const Pack<T, W> p = ld<T, W>(x + head + v * W);
#pragma unroll
    for (int k = 0; k < W; ++k) o[k] = to_f(p.v[k]);
    if (mask != nullptr) {
      const Pack<uint8_t, W> m = ld<uint8_t, W>(mask + head + v * W);
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (m.v[k] == 0) o[k] = -INFINITY;
    }
  }
  __device__ float load1(int i) const { return allowed(i) ? to_f(x[i]) : -INFINITY; }
};

// An entry of the teacher's list: its logit, -inf where it is not in use; z: the student's logit there
template <typename T>
__device__ __forceinline__ float entry(const InbDistillArgs& a, const RowView<T>& row, int64_t at, int& index, float& z) {
  const int64_t i = a.index[at];
  float t = -INFINITY;
  index = -1;
  z = 0.f;
  if (i < 0 || i >= a.V) return t;
  if (a.teacher_dtype == INB_BF16)
    t = to_f(((const bf16*)a.teacher)[at]);
  else if (a.teacher_dtype == INB_F16)
    t = to_f(((const f16*)a.teacher)[at]);
  else
    t = ((const float*)a.teacher)[at];
  z = row.load1((int)i);
  if (z == -INFINITY || t != t || t == -INFINITY) return -INFINITY;
  index = (int)i;
  return t;
}

// running maximum and sum of exp((v - m) c / log2 e)
struct Soft {
  float m = -INFINITY, l = 0.f;
  template <int W>
  __device__ void add(const float (&v)[W], float c) {
    float top = v[0];
#pragma unroll
    for (int k = 1; k < W; ++k) top = fmaxf(top, v[k]);
    if (top > m) {
      l *= ex2((m - top) * c);
      m = top;
    }
    const float at = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) s += ex2((v[k] - at) * c);
    l += s;
  }
  __device__ void join(float om, float ol, float c) {
    const float top = fmaxf(m, om), at = top == -INFINITY ? 0.f : top;
    l = l * ex2((m - at) * c) + ol * ex2((om - at) * c);
    m = top;
  }
  __device__ void over_warp(float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float om = __shfl_xor_sync(0xFFFFFFFFu, m, o), ol = __shfl_xor_sync(0xFFFFFFFFu, l, o);
      join(om, ol, c);
    }
  }
};
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

// The row's entries by one warp, after m and l are known
template <typename T>
__device__ __forceinline__ void finish(const InbDistillArgs& a, const RowView<T>& row, int64_t r, const Soft& s, float c, int lane) {
  float top = -INFINITY, z;
  int index;
  for (int k = lane; k < a.K; k += 32) top = fmaxf(top, entry(a, row, r * a.K + k, index, z));
  top = warp_max(top);
  const bool live = top != -INFINITY;
  float mass = 0.f, sum = 0.f;
  const float inv = c * LN2;                      // 1 / tau
  if (live)
    for (int k = lane; k < a.K; k += 32) {
      const float t = entry(a, row, r * a.K + k, index, z);
      if (index < 0) continue;
      const float e = ex2((t - top) * c);
      mass += e;
      sum = fmaf(e, ((t - top) - (z - s.m)) * inv, sum);
    }
  mass = warp_sum(mass);
  sum = warp_sum(sum);
  if (lane != 0) return;
  a.loss[r] = live ? a.tau * a.tau * (sum / mass + (logf(s.l) - logf(mass))) : 0.f;
  if (a.stats != nullptr)
    *reinterpret_cast<float4*>(a.stats + 4 * r) = live ? make_float4(s.m, 1.f / s.l, top, 1.f / mass) : make_float4(0.f, 0.f, 0.f, 0.f);
}

template <typename T, bool WARP>
__global__ void __launch_bounds__(DIST_THREADS) distill_fwd_kernel(InbDistillArgs a, int parts, float c) {
  constexpr int TPR = WARP ? 32 : DIST_THREADS;
  const int tid = threadIdx.x % TPR, lane = threadIdx.x & 31;
  const int64_t r = WARP ? (int64_t)blockIdx.x * (DIST_THREADS / 32) + threadIdx.x / 32 : blockIdx.x / parts;
  const int part = WARP ? 0 : blockIdx.x % parts;
  if (WARP && r >= a.N) return;
  const RowView<T> row(a, r, nullptr);
  int v0, v1, lo, hi;
  row.part(part, parts, v0, v1, lo, hi);
  Soft s;
  for (int v = v0 + tid; v < v1; v += TPR) {
    float x[RowView<T>::W];
    row.load(v, x);
    s.add(x, c);
  }
  const int body = row.head + v0 * row.W, end = row.head + v1 * row.W;
  for (int i = lo + tid; i < body; i += TPR) {
    const float x[1] = {row.load1(i)};
    s.add(x, c);
  }
  for (int i = end + tid; i < hi; i += TPR) {
    const float x[1] = {row.load1(i)};
    s.add(x, c);
  }
  s.over_warp(c);
  if (WARP) {
    finish(a, row, r, s, c, lane);
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
    if (part == 0 && threadIdx.x < 32) {
      s = Soft();
      for (int p = 0; p < parts; ++p) {
        const float2 o = *cluster.map_shared_rank(&block, p);
        s.join(o.x, o.y, c);
      }
    }
    cluster.sync();         // a block's memory lives until it has been read
  }
  if (part == 0 && threadIdx.x < 32) finish(a, row, r, s, c, lane);
}

template <typename T, bool WARP>
__global__ void __launch_bounds__(DIST_THREADS) distill_bwd_kernel(InbDistillArgs a, int parts, float c) {
  constexpr int TPR = WARP ? 32 : DIST_THREADS, W = RowView<T>::W;
  extern __shared__ float2 entries[];            // (index, p) of the row's list
  const int tid = threadIdx.x % TPR;
  const int64_t r = WARP ? (int64_t)blockIdx.x * (DIST_THREADS / 32) + threadIdx.x / 32 : blockIdx.x / parts;
  const int part = WARP ? 0 : blockIdx.x % parts;
  if (WARP && r >= a.N) return;
  T* out = (T*)a.glogits + r * a.V;
  const RowView<T> row(a, r, out);
  int v0, v1, lo, hi;
  row.part(part, parts, v0, v1, lo, hi);
  const float4 stat = *reinterpret_cast<const float4*>(a.stats + 4 * r);
  const bool live = stat.w != 0.f;                 // a row without an entry in use: 0, whatever its logits are
  const float g = a.gloss[r] * a.tau, gl = g * stat.y;
  float2* list = entries + (WARP ? threadIdx.x / 32 * a.K : 0);
  for (int k = tid; k < a.K; k += TPR) {
    float z;
    int index;
    const float t = entry(a, row, r * a.K + k, index, z);
    list[k] = make_float2(__int_as_float(live ? index : -1), ex2((t - stat.z) * c) * stat.w);
  }
  auto value = [&](float v) { return live && v != -INFINITY ? gl * ex2((v - stat.x) * c) : 0.f; };
  for (int v = v0 + tid; v < v1; v += TPR) {
    float x[W];
    Pack<T, W> o;
    row.load(v, x);
#pragma unroll
    for (int k = 0; k < W; ++k) o.v[k] = from_f<T>(value(x[k]));
    st<T, W>(out + row.head + v * W, o);
  }
  const int body = row.head + v0 * W, end = row.head + v1 * W;
  for (int i = lo + tid; i < body; i += TPR) out[i] = from_f<T>(value(row.load1(i)));
  for (int i = end + tid; i < hi; i += TPR) out[i] = from_f<T>(value(row.load1(i)));
  if (WARP)
    __syncwarp();
  else
    __syncthreads();
  // the listed elements again, from q and the sum of their entries: every entry of an index writes the same value
  for (int k = tid; k < a.K; k += TPR) {
    const int i = __float_as_int(list[k].x);
    if (i < lo || i >= hi) continue;
    float p = 0.f;
    for (int o = 0; o < a.K; ++o)
      if (__float_as_int(list[o].x) == i) p += list[o].y;
    out[i] = from_f<T>(g * (stat.y * ex2((row.load1(i) - stat.x) * c) - p));
  }
}

struct DistPlan {
  bool warp;
  int parts;
  unsigned blocks;
};
static DistPlan dist_plan(const InbDistillArgs& a) {
  DistPlan p = {a.V <= DIST_WARP_V && a.K <= DIST_WARP_K, 1, 0};
  if (p.warp) {
    p.blocks = (unsigned)ceil_div(a.N, DIST_THREADS / 32);
  } else {
    while (p.parts < 8 && a.N * p.parts < sm_count() * 4 && a.V / (2 * p.parts) >= 4096) p.parts *= 2;
    p.blocks = (unsigned)(a.N * p.parts);
  }
  return p;
}
template <typename T>
static int dist_fwd(const InbDistillArgs& a, cudaStream_t s) {
  const DistPlan p = dist_plan(a);
  const float c = LOG2E / a.tau;
  if (p.warp) {
    distill_fwd_kernel<T, true><<<p.blocks, DIST_THREADS, 0, s>>>(a, 1, c);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, distill_fwd_kernel<T, false>, a, p.parts, c);
  return e == cudaSuccess ? launch_status() : -100 - (int)e;
}
template <typename T>
static int dist_bwd(const InbDistillArgs& a, cudaStream_t s) {
  const DistPlan p = dist_plan(a);
  const float c = LOG2E / a.tau;
  const int rows = p.warp ? DIST_THREADS / 32 : 1;
  const size_t smem = (size_t)rows * a.K * 8;
  if (p.warp)
    distill_bwd_kernel<T, true><<<p.blocks, DIST_THREADS, smem, s>>>(a, 1, c);
  else
    distill_bwd_kernel<T, false><<<p.blocks, DIST_THREADS, smem, s>>>(a, p.parts, c);
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
  if (a.logits == nullptr || a.teacher == nullptr || a.index == nullptr || a.loss == nullptr) return -3;
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
      a.glogits == nullptr)
    return -3;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (a.dtype == INB_BF16) return inb::pol::dist_bwd<inb::pol::bf16>(a, s);
  if (a.dtype == INB_F16) return inb::pol::dist_bwd<inb::pol::f16>(a, s);
  return inb::pol::dist_bwd<float>(a, s);
}
