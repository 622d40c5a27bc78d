// causal_conv: depthwise causal convolution over time, 2 to 4 taps a channel, with resets inside the sequence.
//
//   pre[t] = bias + sum_j w[K - 1 - j] x[t - j],  y = act(pre);     taps before a reset, or before the sequence, are 0
//   g[t] = gy[t] act'(pre[t]);   gx[t] = sum_j w[K - 1 - j] g[t + j];   gw[K - 1 - j] = sum_t g[t] x[t - j];   gbias = sum_t g[t]
//
// Bound by DRAM: 2K operations an element against 2 (forward) or 4 (backward, which recomputes pre) moved elements.  A
// thread holds V neighbouring channels, walks along time and keeps the last K - 1 inputs in registers, so every element is
// read once; where sequences are few the time axis is split and a part re-reads K - 1 steps at its edge.
#include "policy_seq.cuh"

namespace inb {
namespace pol {

constexpr int CONV_U = 4;       // steps whose loads are sent at once, while the steps before are worked on
constexpr int CONV_FWD_BLOCKS = 4, CONV_STEP_BLOCKS = 4, CONV_BWD_BLOCKS = 3;      // of 128 threads, an SM
constexpr int CONV_STEP_B = 2;  // sequences whose loads are sent at once by a single step

struct ConvPlan {
  int64_t parts, len, tasks;    // parts of the time axis, their steps; sequences x parts
};

// V neighbouring channels as pairs (V = 1: the first of one pair)
template <typename T, int V, int K>
struct Taps {
  static constexpr int P = Words<T, V>::P;
  float2 w[K][P], bias[P];
  __device__ __forceinline__ void load(const InbConvArgs& a, int64_t ch, bool on) {
    auto get = [&](const void* p, int64_t i) { return on && p != nullptr ? to_f(((const T*)p)[i]) : 0.f; };
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int64_t c = ch + 2 * i;
      bias[i] = make_float2(get(a.bias, c), V > 1 ? get(a.bias, c + 1) : 0.f);
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][i] = make_float2(get(a.w, c * K + k), V > 1 ? get(a.w, (c + 1) * K + k) : 0.f);
    }
  }
};
// The last K - 1 inputs; x[j]: j + 1 steps back
template <typename T, int V, int K>
struct Window {
  static constexpr int P = Words<T, V>::P;
  float2 x[K - 1][P];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) x[j][i] = make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ void push(const float2 (&v)[P]) {
#pragma unroll
    for (int j = K - 2; j > 0; --j)
#pragma unroll
      for (int i = 0; i < P; ++i) x[j][i] = x[j - 1][i];
#pragma unroll
    for (int i = 0; i < P; ++i) x[0][i] = v[i];
  }
  __device__ __forceinline__ void push(const T* p) {
    Words<T, V> q;
    q.load(p);
    float2 v[P];
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = q.pair(i);
    push(v);
  }
  // what lies before step t0; returns how many steps back the episode reaches, up to K - 1
  __device__ __forceinline__ int before(const InbConvArgs& a, int64_t s, int64_t t0, const uint8_t* rs, int64_t ch) {
    zero();
    if (t0 == 0) {
      if (a.state != nullptr) {
        const T* p = (const T*)a.state + s * a.state_seq + ch;
        Words<T, V> q[K - 1];
#pragma unroll
        for (int j = 0; j < K - 1; ++j) q[j].load(p + j * a.C);
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
#pragma unroll
          for (int i = 0; i < P; ++i) x[K - 2 - j][i] = q[j].pair(i);
      }
      return K - 1;
    }
    int m = K - 1;                        // parts are longer than K - 1 steps
    for (int64_t t = t0 - (K - 1); t < t0; ++t) {
      if (rs != nullptr && rs[t * a.reset.step]) {
        m = 0;
        zero();
      }
      push(row<T>(a.x, s, t) + ch);
      m = m < K - 1 ? m + 1 : m;
    }
    return m;
  }
  __device__ __forceinline__ float2 pre(const Taps<T, V, K>& t, float2 now, int i) const {
    float2 p = fma2(now, t.w[K - 1][i], t.bias[i]);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) p = fma2(x[j][i], t.w[K - 2 - j][i], p);
    return p;
  }
};
// ---------------------------------------------------------------------------------------------- forward
// A block is blockDim.x channel vectors x blockDim.y tasks and strides over the tasks, so that weights are read once.
template <typename T, int V, int K>
__global__ void __launch_bounds__(128, CONV_FWD_BLOCKS) conv_fwd_kernel(InbConvArgs a, ConvPlan pl) {
  constexpr int P = Words<T, V>::P;
  const int64_t ch = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (ch >= a.C) return;
  Taps<T, V, K> taps;
  taps.load(a, ch, true);
  for (int64_t task = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; task < pl.tasks; task += (int64_t)gridDim.x * blockDim.y) {
    const int64_t part = pl.parts > 1 ? task / a.S : 0, s = task - part * a.S;      // the next task: the same steps of the next sequence
    const int64_t t0 = part * pl.len;
    const int n = (int)(t0 + pl.len < a.T ? pl.len : a.T - t0);
    const uint8_t* rs = resets(a.reset, s);
    const uint8_t* pr = rs != nullptr ? rs + t0 * a.reset.step : nullptr;
    const T* px = row<T>(a.x, s, t0) + ch;
    T* py = row_out<T>(a.y, s, t0) + ch;
    Words<T, V> x[CONV_U], nx[CONV_U];
    uint32_t reset[CONV_U] = {}, nr[CONV_U] = {};
    auto load = [&](Words<T, V>(&to)[CONV_U], uint32_t(&flag)[CONV_U], int left) {
#pragma unroll
      for (int u = 0; u < CONV_U; ++u) {
        if (u < left) to[u].load(px);
        px += a.x.step;
      }
      if (rs != nullptr) {
#pragma unroll
        for (int u = 0; u < CONV_U; ++u) {
          if (u < left) flag[u] = *pr;
          pr += a.reset.step;
        }
      }
    };
    load(x, reset, n);
    Window<T, V, K> win;
    win.before(a, s, t0, rs, ch);
    for (int left = n; left > 0; left -= CONV_U) {
      if (left > CONV_U) load(nx, nr, left - CONV_U);
#pragma unroll
      for (int u = 0; u < CONV_U; ++u) {
        if (u >= left) break;
        if (reset[u]) win.zero();
        Words<T, V> y;
        float2 now[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
          now[i] = x[u].pair(i);
          const float2 p = win.pre(taps, now[i], i);
          y.set(i, a.act == INB_ACT_SILU ? mul2(p, sigmoid2(p, V > 1)) : p);
        }
        win.push(now);
        y.store(py);
        py += a.y.step;
      }
#pragma unroll
      for (int u = 0; u < CONV_U; ++u) x[u] = nx[u], reset[u] = nr[u];
    }
    if (t0 + n == a.T && a.state_out != nullptr) {
      T* out = (T*)a.state_out + s * a.state_out_seq + ch;
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        Words<T, V> p;
#pragma unroll
        for (int i = 0; i < P; ++i) p.set(i, win.x[j][i]);      // what was read, or 0: exact
        p.store(out + (K - 2 - j) * a.C);
      }
    }
  }
}

// One step: bound by the states' bytes, of which a thread has CONV_STEP_B sequences' on their way at once; state_out may be state.
template <typename T, int V, int K>
__global__ void __launch_bounds__(128, CONV_STEP_BLOCKS) conv_step_kernel(InbConvArgs a) {
  constexpr int P = Words<T, V>::P;
  const int64_t ch = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (ch >= a.C) return;
  Taps<T, V, K> taps;
  taps.load(a, ch, true);
  const int64_t stride = (int64_t)gridDim.x * blockDim.y;
  for (int64_t s0 = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; s0 < a.S; s0 += stride * CONV_STEP_B) {
    Words<T, V> x[CONV_STEP_B], old[CONV_STEP_B][K - 1];
    uint32_t reset[CONV_STEP_B];
#pragma unroll
    for (int b = 0; b < CONV_STEP_B; ++b) {
      const int64_t s = s0 + b * stride;
      if (s >= a.S) break;
      x[b].load(row<T>(a.x, s, 0) + ch);
      reset[b] = a.reset.p != nullptr ? *resets(a.reset, s) : 0;
      if (a.state != nullptr) {
        const T* p = (const T*)a.state + s * a.state_seq + ch;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) old[b][j].load(p + j * a.C);
      }
    }
#pragma unroll
    for (int b = 0; b < CONV_STEP_B; ++b) {
      const int64_t s = s0 + b * stride;
      if (s >= a.S) break;
      if (reset[b] || a.state == nullptr) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
#pragma unroll
          for (int i = 0; i < Words<T, V>::N; ++i) old[b][j].w[i] = 0;
      }
      Words<T, V> y;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float2 p = fma2(x[b].pair(i), taps.w[K - 1][i], taps.bias[i]);
#pragma unroll
        for (int j = K - 2; j >= 0; --j) p = fma2(old[b][j].pair(i), taps.w[j][i], p);
        y.set(i, a.act == INB_ACT_SILU ? mul2(p, sigmoid2(p, V > 1)) : p);
      }
      y.store(row_out<T>(a.y, s, 0) + ch);
      if (a.state_out != nullptr) {
        T* out = (T*)a.state_out + s * a.state_out_seq + ch;
#pragma unroll
        for (int j = 0; j < K - 2; ++j) old[b][j + 1].store(out + j * a.C);
        x[b].store(out + (K - 2) * a.C);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- backward
// pend[j - 1] gathers gx[t - j] while later steps still add to it; step t completes gx[t - (K - 1)].  A part goes K - 1 steps
// beyond its end, for gx alone.  Blocks as in the forward pass, so that gw and gbias stay in registers; one partial row a
// block, [C K | C], added by a second launch.
template <typename T, int V, int K>
__global__ void __launch_bounds__(128, CONV_BWD_BLOCKS) conv_bwd_kernel(InbConvArgs a, ConvPlan pl) {
  constexpr int P = Words<T, V>::P;
  extern __shared__ float smem[];
  const int64_t ch = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  const bool on = ch < a.C;
  Taps<T, V, K> taps;
  taps.load(a, ch, on);
  const float2 zero = make_float2(0.f, 0.f);
  float2 gw[K][P], gb[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    gb[i] = zero;
#pragma unroll
    for (int k = 0; k < K; ++k) gw[k][i] = zero;
  }
  if (on)
    for (int64_t task = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; task < pl.tasks; task += (int64_t)gridDim.x * blockDim.y) {
      const int64_t part = pl.parts > 1 ? task / a.S : 0, s = task - part * a.S;
      const int64_t t0 = part * pl.len;
      const int n = (int)(t0 + pl.len < a.T ? pl.len : a.T - t0);                 // the part's steps,
      const int end = (int)(n + K - 1 < a.T - t0 ? n + K - 1 : a.T - t0);         // and with those that reach back into it
      const uint8_t* rs = resets(a.reset, s);
      const uint8_t* pr = rs != nullptr ? rs + t0 * a.reset.step : nullptr;
      const T *px = row<T>(a.x, s, t0) + ch, *pg = row<T>(a.gy, s, t0) + ch;
      Words<T, V> x[CONV_U], nx[CONV_U], gy[CONV_U], ng[CONV_U];
      uint32_t reset[CONV_U] = {}, nr[CONV_U] = {};
      auto load = [&](Words<T, V>(&to)[CONV_U], Words<T, V>(&tg)[CONV_U], uint32_t(&flag)[CONV_U], int left) {
#pragma unroll
        for (int u = 0; u < CONV_U; ++u) {
          if (u < left) to[u].load(px), tg[u].load(pg);
          px += a.x.step, pg += a.gy.step;
        }
        if (rs != nullptr) {
#pragma unroll
          for (int u = 0; u < CONV_U; ++u) {
            if (u < left) flag[u] = *pr;
            pr += a.reset.step;
          }
        }
      };
      load(x, gy, reset, end);
      Window<T, V, K> win;
      float2 pend[K - 1][P];
      int m = win.before(a, s, t0, rs, ch);      // how many steps before this one are seen
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) pend[j][i] = zero;
      T* pgx = row_out<T>(a.gx, s, t0) + ch;
      // step i of the part completes gx of step i - (K - 1); before the sequence it is the initial state's
      auto emit = [&](int i) {
        Words<T, V> p;
#pragma unroll
        for (int q = 0; q < P; ++q) p.set(q, pend[K - 2][q]);
        const int at = i - (K - 1);
        if (at >= 0) {
          p.store(pgx);
          pgx += a.gx.step;
        } else if (t0 == 0 && a.gstate != nullptr) {
          p.store((T*)a.gstate + (s * (K - 1) + at + K - 1) * a.C + ch);
        }
      };
      auto shift = [&](const float2 (&g)[P]) {
#pragma unroll
        for (int j = K - 2; j > 0; --j)
#pragma unroll
          for (int i = 0; i < P; ++i) pend[j][i] = pend[j - 1][i];
#pragma unroll
        for (int i = 0; i < P; ++i) pend[0][i] = mul2(taps.w[K - 1][i], g[i]);
      };
      for (int i0 = 0; i0 < end; i0 += CONV_U) {
        if (i0 + CONV_U < end) load(nx, ng, nr, end - i0 - CONV_U);
#pragma unroll
        for (int u = 0; u < CONV_U; ++u) {
          if (i0 + u >= end) break;
          if (reset[u]) {
            m = 0;
            win.zero();
          }
          float2 g[P], now[P];
#pragma unroll
          for (int i = 0; i < P; ++i) {
            now[i] = x[u].pair(i);
            g[i] = gy[u].pair(i);
            if (a.act == INB_ACT_SILU) {
              const float2 p = win.pre(taps, now[i], i);
              const float2 q = sigmoid2(p, V > 1);
              g[i] = mul2(g[i], mul2(q, fma2(p, fma2(q, both(-1.f), both(1.f)), both(1.f))));
            }
            if (i0 + u < n) {
              gb[i] = add2(gb[i], g[i]);
              gw[K - 1][i] = fma2(g[i], now[i], gw[K - 1][i]);
#pragma unroll
              for (int j = 0; j < K - 1; ++j) gw[K - 2 - j][i] = fma2(g[i], win.x[j][i], gw[K - 2 - j][i]);
            }
          }
#pragma unroll
          for (int j = 0; j < K - 1; ++j)
            if (j < m) {
#pragma unroll
              for (int i = 0; i < P; ++i) pend[j][i] = fma2(taps.w[K - 2 - j][i], g[i], pend[j][i]);
            }
          emit(i0 + u);
          shift(g);
          win.push(now);
          m = m < K - 1 ? m + 1 : m;
        }
#pragma unroll
        for (int u = 0; u < CONV_U; ++u) x[u] = nx[u], gy[u] = ng[u], reset[u] = nr[u];
      }
      // steps beyond the sequence: entry e of the final state is the input of step T - (K - 1) + e
      for (int i = end; i < n + K - 1; ++i) {
        const int e = (int)(t0 + i - a.T);
        if (a.gstate_out != nullptr && K - 1 - e <= m) {
          Words<T, V> p;
          p.load((const T*)a.gstate_out + (s * (K - 1) + e) * a.C + ch);
#pragma unroll
          for (int q = 0; q < P; ++q) pend[K - 2][q] = add2(pend[K - 2][q], p.pair(q));
        }
        emit(i);
        float2 none[P];
#pragma unroll
        for (int q = 0; q < P; ++q) none[q] = zero;
        shift(none);
      }
    }
  // the block's tasks, then one partial row
  const int n = blockDim.x * V * (K + 1);
  float* mine = smem + threadIdx.y * n;
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < K; ++k) mine[(threadIdx.x * V + v) * K + k] = v & 1 ? gw[k][v / 2].y : gw[k][v / 2].x;
    mine[blockDim.x * V * K + threadIdx.x * V + v] = v & 1 ? gb[v / 2].y : gb[v / 2].x;
  }
  __syncthreads();
  const int64_t c0 = (int64_t)blockIdx.y * blockDim.x * V;
  float* out = a.work + (int64_t)blockIdx.x * a.C * (K + 1);
  for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < n; i += blockDim.x * blockDim.y) {
    float v = 0.f;
    for (int y = 0; y < (int)blockDim.y; ++y) v += smem[y * n + i];
    const bool weight = i < (int)blockDim.x * V * K;
    const int64_t col = weight ? c0 * K + i : c0 + i - blockDim.x * V * K;
    if (weight) {
      if (col < (int64_t)a.C * K) out[col] = v;
    } else if (col < a.C) {
      out[(int64_t)a.C * K + col] = v;
    }
  }
}

// ---------------------------------------------------------------------------------------------- plans
// Blocks of 128 threads, channel vectors first; as many as the GPU holds at `resident` an SM, striding over the tasks.  The
// time axis is split where sequences are too few for that, into parts of 16 steps or more (a part re-reads K - 1).
struct ConvLaunch {
  ConvPlan plan;
  dim3 block, grid;
};
static ConvLaunch conv_plan(const InbConvArgs& a, int V, int resident) {
  ConvLaunch l;
  const int64_t cv = ceil_div(a.C, V), room = (int64_t)sm_count() * resident;
  unsigned tx = 1;
  while (tx < 128 && tx < cv) tx *= 2;
  l.block = dim3(tx, 128 / tx);
  const int64_t gy = ceil_div(cv, tx);
  int64_t parts = ceil_div(room * l.block.y, a.S * gy);
  if (parts > a.T / 16) parts = a.T / 16;
  if (parts < 1) parts = 1;
  l.plan.len = ceil_div(a.T, parts);
  l.plan.parts = ceil_div(a.T, l.plan.len);
  l.plan.tasks = a.S * l.plan.parts;
  const int64_t need = ceil_div(l.plan.tasks, l.block.y), gx = ceil_div(room, gy);
  l.grid = dim3((unsigned)(gx < need ? gx : need), (unsigned)gy);
  return l;
}
static int elem_size(int dtype) { return dtype == INB_F32 ? 4 : 2; }
static bool aligned_to(const void* p, int64_t seq, int64_t bytes, int64_t elem) {
  return p == nullptr || (((uint64_t)(uintptr_t)p | (uint64_t)(seq * elem)) & (bytes - 1)) == 0;
}
// Whether every row can be moved by accesses of `bytes`
static bool conv_aligned(const InbConvArgs& a, int64_t bytes) {
  const int64_t e = elem_size(a.dtype);
  return a.C * e % bytes == 0 && is_aligned(a.x, bytes, e) && is_aligned(a.y, bytes, e) && is_aligned(a.gy, bytes, e) &&
         is_aligned(a.gx, bytes, e) && aligned_to(a.state, a.state_seq, bytes, e) &&
         aligned_to(a.state_out, a.state_out_seq, bytes, e) && aligned_to(a.gstate_out, 0, bytes, e) &&
         aligned_to(a.gstate, 0, bytes, e);
}
static int conv_check(const InbConvArgs& a) {
  if (a.dtype < 0 || a.dtype > 2 || (a.act != -1 && a.act != INB_ACT_SILU) || a.C < 1 || a.C > INB_MAX_MEMORY_C || a.K < 2 ||
      a.K > 4 || a.S < 0 || a.S > INB_MAX_MEMORY_S || a.T < 0 || a.T > INB_MAX_MEMORY_S || (a.reset.p != nullptr && (a.reset.rows < 1 || a.reset.rows > INB_MAX_MEMORY_S)))
    return -2;
  return 0;
}

template <typename T, int V, int K>
static int conv_fwd_go(const InbConvArgs& a, cudaStream_t s) {
  if (a.T == 1) {
    const ConvLaunch l = conv_plan(a, V, CONV_STEP_BLOCKS);
    conv_step_kernel<T, V, K><<<l.grid, l.block, 0, s>>>(a);
  } else {
    const ConvLaunch l = conv_plan(a, V, CONV_FWD_BLOCKS);
    conv_fwd_kernel<T, V, K><<<l.grid, l.block, 0, s>>>(a, l.plan);
  }
  return launch_status();
}
template <typename T, int V, int K>
static int conv_bwd_go(const InbConvArgs& a, cudaStream_t s) {
  const ConvLaunch l = conv_plan(a, V, CONV_BWD_BLOCKS);
  conv_bwd_kernel<T, V, K><<<l.grid, l.block, 128 * V * (K + 1) * 4, s>>>(a, l.plan);
  colsum<T>(a.work, l.grid.x, (int64_t)a.C * (K + 1), (int64_t)a.C * K, (int64_t)a.C * (K + 1), a.gw, a.gbias, nullptr, s);
  return launch_status();
}
// Channels a thread: 16 bytes (forward) or 4 channels (backward, whose sums take the registers), moved by one access, where
// every row allows it, else one.
template <typename T>
static int conv_width(const InbConvArgs& a, bool backward) {
  const int v = backward ? 4 : 16 / (int)sizeof(T);
  return conv_aligned(a, v * sizeof(T)) ? v : 1;
}
template <typename T>
static int conv_go(const InbConvArgs& a, bool backward, cudaStream_t s) {
  constexpr int W = 16 / sizeof(T);
  if (backward) {
    if (conv_width<T>(a, true) == 4)
      return a.K == 2 ? conv_bwd_go<T, 4, 2>(a, s) : a.K == 3 ? conv_bwd_go<T, 4, 3>(a, s) : conv_bwd_go<T, 4, 4>(a, s);
    return a.K == 2 ? conv_bwd_go<T, 1, 2>(a, s) : a.K == 3 ? conv_bwd_go<T, 1, 3>(a, s) : conv_bwd_go<T, 1, 4>(a, s);
  }
  if (conv_width<T>(a, false) == W)
    return a.K == 2 ? conv_fwd_go<T, W, 2>(a, s) : a.K == 3 ? conv_fwd_go<T, W, 3>(a, s) : conv_fwd_go<T, W, 4>(a, s);
  return a.K == 2 ? conv_fwd_go<T, 1, 2>(a, s) : a.K == 3 ? conv_fwd_go<T, 1, 3>(a, s) : conv_fwd_go<T, 1, 4>(a, s);
}
static int conv_dispatch(const InbConvArgs& a, bool backward, cudaStream_t s) {
  if (a.dtype == INB_BF16) return conv_go<bf16>(a, backward, s);
  if (a.dtype == INB_F16) return conv_go<f16>(a, backward, s);
  return conv_go<float>(a, backward, s);
}

}  // namespace pol
}  // namespace inb

extern "C" int inb_causal_conv_fwd(const InbConvArgs* args, void* cuda_stream) {
  if (args == nullptr) return -1;
  const InbConvArgs& a = *args;
  const int rc = inb::pol::conv_check(a);
  if (rc != 0) return rc;
  if (a.S == 0 || a.T == 0) return 0;
  if (a.x.p == nullptr || a.y.p == nullptr || a.w == nullptr) return -3;
  return inb::pol::conv_dispatch(a, false, (cudaStream_t)cuda_stream);
}

extern "C" int inb_causal_conv_work(const InbConvArgs* args, int64_t* elems) {
  if (args == nullptr || elems == nullptr) return -1;
  const InbConvArgs& a = *args;
  const int rc = inb::pol::conv_check(a);
  if (rc != 0) return rc;
  *elems = 0;
  if (a.S == 0 || a.T == 0) return 0;
  const int v = a.dtype == INB_F32 ? inb::pol::conv_width<float>(a, true) : inb::pol::conv_width<inb::pol::bf16>(a, true);
  *elems = (int64_t)inb::pol::conv_plan(a, v, inb::pol::CONV_BWD_BLOCKS).grid.x * a.C * (a.K + 1);
  return 0;
}

extern "C" int inb_causal_conv_bwd(const InbConvArgs* args, void* cuda_stream) {
  int64_t need = 0;
  const int rc = inb_causal_conv_work(args, &need);
  if (rc != 0) return rc;
  const InbConvArgs& a = *args;
  if (a.S == 0 || a.T == 0) return 0;
  if (a.x.p == nullptr || a.w == nullptr || a.gy.p == nullptr || a.gx.p == nullptr || a.gw == nullptr) return -3;
  if (a.work == nullptr || a.work_elems < need) return -5;
  return inb::pol::conv_dispatch(a, true, (cudaStream_t)cuda_stream);
}
