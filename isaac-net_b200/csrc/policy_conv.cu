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
constexpr int CONV_STEP_B = 4;  // sequences whose loads are sent at once by a single step

struct ConvPlan {
  int64_t parts, len, tasks;    // parts of the time axis, their steps; sequences x parts
};

// V channels of the weights, [K] taps each
template <typename T, int V, int K>
struct Taps {
  float w[K][V], bias[V];
  __device__ void load(const InbConvArgs& a, int64_t ch, bool on) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      bias[v] = on && a.bias != nullptr ? to_f(((const T*)a.bias)[ch + v]) : 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][v] = on ? to_f(((const T*)a.w)[(ch + v) * K + k]) : 0.f;
    }
  }
};
// The last K - 1 inputs; x[j]: j + 1 steps back
template <typename T, int V, int K>
struct Window {
  float x[K - 1][V];
  __device__ void zero() {
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) x[j][v] = 0.f;
  }
  __device__ void push(const Pack<T, V>& p) {
#pragma unroll
    for (int j = K - 2; j > 0; --j)
#pragma unroll
      for (int v = 0; v < V; ++v) x[j][v] = x[j - 1][v];
#pragma unroll
    for (int v = 0; v < V; ++v) x[0][v] = to_f(p.v[v]);
  }
  __device__ float pre(const Taps<T, V, K>& t, float now, int v) const {
    float p = fmaf(now, t.w[K - 1][v], t.bias[v]);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) p = fmaf(x[j][v], t.w[K - 2 - j][v], p);
    return p;
  }
};

// ---------------------------------------------------------------------------------------------- forward
// A block is blockDim.x channel vectors x blockDim.y tasks and strides over the tasks, so that weights are read once.
template <typename T, int V, int K>
__global__ void __launch_bounds__(128, 6) conv_fwd_kernel(InbConvArgs a, ConvPlan pl) {
  const int64_t ch = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (ch >= a.C) return;
  Taps<T, V, K> taps;
  taps.load(a, ch, true);
  for (int64_t task = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; task < pl.tasks; task += (int64_t)gridDim.x * blockDim.y) {
    const int64_t part = pl.parts > 1 ? task / a.S : 0, s = task - part * a.S;      // the next task: the same steps of the next sequence
    const int64_t t0 = part * pl.len, t1 = t0 + pl.len < a.T ? t0 + pl.len : a.T;
    const uint8_t* rs = resets(a.reset, s);
    const T* px = row<T>(a.x, s, t0) + ch;
    T* py = row_out<T>(a.y, s, t0) + ch;
    Pack<T, V> x[CONV_U], nx[CONV_U];
    uint32_t reset[CONV_U], nr[CONV_U];
    // loads have no condition: the steps beyond the part's end read its last one again
    auto load = [&](Pack<T, V>(&to)[CONV_U], uint32_t(&flag)[CONV_U], int64_t t) {
#pragma unroll
      for (int u = 0; u < CONV_U; ++u) {
        to[u] = ld<T, V>(px);
        flag[u] = rs != nullptr ? rs[(t + u < t1 ? t + u : t1 - 1) * a.reset.step] : 0;
        if (t + u + 1 < t1) px += a.x.step;
      }
    };
    load(x, reset, t0);
    Window<T, V, K> win;
    win.zero();
    for (int64_t t = t0 - (K - 1); t < t0; ++t) {
      if (t >= 0) {
        if (rs != nullptr && rs[t * a.reset.step]) win.zero();
        win.push(ld<T, V>(row<T>(a.x, s, t) + ch));
      } else if (a.state != nullptr) {
        win.push(ld<T, V>((const T*)a.state + s * a.state_seq + (t + K - 1) * a.C + ch));
      }
    }
    for (int64_t t = t0; t < t1; t += CONV_U) {
      if (t + CONV_U < t1) load(nx, nr, t + CONV_U);
#pragma unroll
      for (int u = 0; u < CONV_U; ++u) {
        if (t + u >= t1) break;
        if (reset[u]) win.zero();
        Pack<T, V> y;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float p = win.pre(taps, to_f(x[u].v[v]), v);
          y.v[v] = from_f<T>(a.act == INB_ACT_SILU ? p * sigmoid(p) : p);
        }
        win.push(x[u]);
        st<T, V>(py, y);
        py += a.y.step;
      }
#pragma unroll
      for (int u = 0; u < CONV_U; ++u) x[u] = nx[u], reset[u] = nr[u];
    }
    if (t1 == a.T && a.state_out != nullptr) {
      T* out = (T*)a.state_out + s * a.state_out_seq + ch;
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        Pack<T, V> p;
#pragma unroll
        for (int v = 0; v < V; ++v) p.v[v] = from_f<T>(win.x[j][v]);      // what was read, or 0: exact
        st<T, V>(out + (K - 2 - j) * a.C, p);
      }
    }
  }
}

// One step: bound by the states' bytes, of which a thread has CONV_STEP_B sequences' on their way at once; state_out may be state.
template <typename T, int V, int K>
__global__ void __launch_bounds__(128, 6) conv_step_kernel(InbConvArgs a) {
  const int64_t ch = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (ch >= a.C) return;
  Taps<T, V, K> taps;
  taps.load(a, ch, true);
  const int64_t stride = (int64_t)gridDim.x * blockDim.y;
  for (int64_t s0 = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; s0 < a.S; s0 += stride * CONV_STEP_B) {
    Pack<T, V> x[CONV_STEP_B], old[CONV_STEP_B][K - 1];
    uint32_t reset[CONV_STEP_B];
#pragma unroll
    for (int b = 0; b < CONV_STEP_B; ++b) {
      const int64_t s = s0 + b * stride;
      if (s >= a.S) break;
      x[b] = ld<T, V>(row<T>(a.x, s, 0) + ch);
      reset[b] = a.reset.p != nullptr ? *resets(a.reset, s) : 0;
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
        if (a.state != nullptr) old[b][j] = ld<T, V>((const T*)a.state + s * a.state_seq + j * a.C + ch);
    }
#pragma unroll
    for (int b = 0; b < CONV_STEP_B; ++b) {
      const int64_t s = s0 + b * stride;
      if (s >= a.S) break;
      if (reset[b] || a.state == nullptr) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v) old[b][j].v[v] = from_f<T>(0.f);
      }
      Pack<T, V> y;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float p = fmaf(to_f(x[b].v[v]), taps.w[K - 1][v], taps.bias[v]);
#pragma unroll
        for (int j = K - 2; j >= 0; --j) p = fmaf(to_f(old[b][j].v[v]), taps.w[j][v], p);
        y.v[v] = from_f<T>(a.act == INB_ACT_SILU ? p * sigmoid(p) : p);
      }
      st<T, V>(row_out<T>(a.y, s, 0) + ch, y);
      if (a.state_out != nullptr) {
        T* out = (T*)a.state_out + s * a.state_out_seq + ch;
#pragma unroll
        for (int j = 0; j < K - 2; ++j) st<T, V>(out + j * a.C, old[b][j + 1]);
        st<T, V>(out + (K - 2) * a.C, x[b]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- backward
// pend[j - 1] gathers gx[t - j] while later steps still add to it; step t completes gx[t - (K - 1)].  A part goes K - 1 steps
// beyond its end, for gx alone.  Blocks as in the forward pass, so that gw and gbias stay in registers; one partial row a
// block, [C K | C], added by a second launch.
template <typename T, int V, int K>
__global__ void __launch_bounds__(128, 3) conv_bwd_kernel(InbConvArgs a, ConvPlan pl) {
  extern __shared__ float smem[];
  const int64_t ch = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  const bool on = ch < a.C;
  Taps<T, V, K> taps;
  taps.load(a, ch, on);
  float gw[K][V], gb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    gb[v] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) gw[k][v] = 0.f;
  }
  if (on)
    for (int64_t task = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; task < pl.tasks; task += (int64_t)gridDim.x * blockDim.y) {
      const int64_t part = pl.parts > 1 ? task / a.S : 0, s = task - part * a.S;
      const int64_t t0 = part * pl.len, t1 = t0 + pl.len < a.T ? t0 + pl.len : a.T;
      const int64_t last = t1 + K - 1, end = last < a.T ? last : a.T;
      const uint8_t* rs = resets(a.reset, s);
      const T *px = row<T>(a.x, s, t0) + ch, *pg = row<T>(a.gy, s, t0) + ch;
      Pack<T, V> x[CONV_U], nx[CONV_U], gy[CONV_U], ng[CONV_U];
      uint32_t reset[CONV_U], nr[CONV_U];
      auto load = [&](Pack<T, V>(&to)[CONV_U], Pack<T, V>(&tg)[CONV_U], uint32_t(&flag)[CONV_U], int64_t t) {
#pragma unroll
        for (int u = 0; u < CONV_U; ++u) {
          to[u] = ld<T, V>(px);
          tg[u] = ld<T, V>(pg);
          flag[u] = rs != nullptr ? rs[(t + u < end ? t + u : end - 1) * a.reset.step] : 0;
          if (t + u + 1 < end) px += a.x.step, pg += a.gy.step;
        }
      };
      load(x, gy, reset, t0);
      Window<T, V, K> win;
      float pend[K - 1][V];
      int m = K - 1;                        // how many steps before this one are seen
      win.zero();
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) pend[j][v] = 0.f;
      auto restart = [&] {
        m = 0;
        win.zero();
      };
      auto push = [&](const Pack<T, V>& p) {
        win.push(p);
        m = m < K - 1 ? m + 1 : m;
      };
      T* pgx = row_out<T>(a.gx, s, t0) + ch;
      // gx of step t - (K - 1) is complete; before the sequence it is the initial state's
      auto emit = [&](int64_t t) {
        const int64_t at = t - (K - 1);
        Pack<T, V> p;
#pragma unroll
        for (int v = 0; v < V; ++v) p.v[v] = from_f<T>(pend[K - 2][v]);
        if (at >= t0) {
          st<T, V>(pgx, p);
          pgx += a.gx.step;
        } else if (at < 0 && a.gstate != nullptr) {
          st<T, V>((T*)a.gstate + (s * (K - 1) + at + K - 1) * a.C + ch, p);
        }
      };
      auto shift = [&](const float (&g)[V]) {
#pragma unroll
        for (int j = K - 2; j > 0; --j)
#pragma unroll
          for (int v = 0; v < V; ++v) pend[j][v] = pend[j - 1][v];
#pragma unroll
        for (int v = 0; v < V; ++v) pend[0][v] = taps.w[K - 1][v] * g[v];
      };
      for (int64_t t = t0 - (K - 1); t < t0; ++t) {
        if (t >= 0) {
          if (rs != nullptr && rs[t * a.reset.step]) restart();
          push(ld<T, V>(row<T>(a.x, s, t) + ch));
        } else if (a.state != nullptr) {
          push(ld<T, V>((const T*)a.state + s * a.state_seq + (t + K - 1) * a.C + ch));
        }
      }
      for (int64_t t = t0; t < end; t += CONV_U) {
        if (t + CONV_U < end) load(nx, ng, nr, t + CONV_U);
#pragma unroll
        for (int u = 0; u < CONV_U; ++u) {
          if (t + u >= end) break;
          if (reset[u]) restart();
          const bool mine = t + u < t1;
          float g[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float xv = to_f(x[u].v[v]);
            g[v] = to_f(gy[u].v[v]);
            if (a.act == INB_ACT_SILU) {
              const float p = win.pre(taps, xv, v), q = sigmoid(p);
              g[v] *= q * fmaf(p, 1.f - q, 1.f);
            }
            if (mine) {
              gb[v] += g[v];
              gw[K - 1][v] = fmaf(g[v], xv, gw[K - 1][v]);
#pragma unroll
              for (int j = 0; j < K - 1; ++j) gw[K - 2 - j][v] = fmaf(g[v], win.x[j][v], gw[K - 2 - j][v]);
            }
          }
#pragma unroll
          for (int j = 0; j < K - 1; ++j)
            if (j < m) {
#pragma unroll
              for (int v = 0; v < V; ++v) pend[j][v] = fmaf(taps.w[K - 2 - j][v], g[v], pend[j][v]);
            }
          emit(t + u);
          shift(g);
          push(x[u]);
        }
#pragma unroll
        for (int u = 0; u < CONV_U; ++u) x[u] = nx[u], gy[u] = ng[u], reset[u] = nr[u];
      }
      // steps beyond the sequence: entry i of the final state is the input of step T - (K - 1) + i
      for (int64_t t = end; t < last; ++t) {
        const int i = (int)(t - a.T);
        if (a.gstate_out != nullptr && K - 1 - i <= m) {
          const Pack<T, V> p = ld<T, V>((const T*)a.gstate_out + (s * (K - 1) + i) * a.C + ch);
#pragma unroll
          for (int v = 0; v < V; ++v) pend[K - 2][v] += to_f(p.v[v]);
        }
        emit(t);
        const float none[V] = {};
        shift(none);
      }
    }
  // the block's tasks, then one partial row
  const int n = blockDim.x * V * (K + 1);
  float* mine = smem + threadIdx.y * n;
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < K; ++k) mine[(threadIdx.x * V + v) * K + k] = gw[k][v];
    mine[blockDim.x * V * K + threadIdx.x * V + v] = gb[v];
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
      a.K > 4 || a.S < 0 || a.S > INB_MAX_MEMORY_S || a.T < 0 || a.T > INB_MAX_MEMORY_S || (a.reset.p != nullptr && a.reset.rows < 1))
    return -2;
  return 0;
}

template <typename T, int V, int K>
static int conv_fwd_go(const InbConvArgs& a, cudaStream_t s) {
  if (a.T == 1) {
    const ConvLaunch l = conv_plan(a, V, 12);      // two rounds: a block's sequences are few
    conv_step_kernel<T, V, K><<<l.grid, l.block, 0, s>>>(a);
  } else {
    const ConvLaunch l = conv_plan(a, V, 6);
    conv_fwd_kernel<T, V, K><<<l.grid, l.block, 0, s>>>(a, l.plan);
  }
  return launch_status();
}
template <typename T, int V, int K>
static int conv_bwd_go(const InbConvArgs& a, cudaStream_t s) {
  const ConvLaunch l = conv_plan(a, V, 3);
  conv_bwd_kernel<T, V, K><<<l.grid, l.block, 128 * V * (K + 1) * 4, s>>>(a, l.plan);
  colsum<T>(a.work, l.grid.x, (int64_t)a.C * (K + 1), (int64_t)a.C * K, (int64_t)a.C * (K + 1), a.gw, a.gbias, nullptr, s);
  return launch_status();
}
template <typename T, int V>
static int conv_go(const InbConvArgs& a, bool backward, cudaStream_t s) {
  if (a.K == 2) return backward ? conv_bwd_go<T, V, 2>(a, s) : conv_fwd_go<T, V, 2>(a, s);
  if (a.K == 3) return backward ? conv_bwd_go<T, V, 3>(a, s) : conv_fwd_go<T, V, 3>(a, s);
  return backward ? conv_bwd_go<T, V, 4>(a, s) : conv_fwd_go<T, V, 4>(a, s);
}
// Four channels a thread, moved by one access, or one: 8 of 16 bits would hold twice the registers for no more bytes in flight.
static int conv_dispatch(const InbConvArgs& a, bool backward, cudaStream_t s) {
  const bool vec = conv_aligned(a, 4 * elem_size(a.dtype));
  if (a.dtype == INB_BF16) return vec ? conv_go<bf16, 4>(a, backward, s) : conv_go<bf16, 1>(a, backward, s);
  if (a.dtype == INB_F16) return vec ? conv_go<f16, 4>(a, backward, s) : conv_go<f16, 1>(a, backward, s);
  return vec ? conv_go<float, 4>(a, backward, s) : conv_go<float, 1>(a, backward, s);
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
  const bool vec = inb::pol::conv_aligned(a, 4 * inb::pol::elem_size(a.dtype));
  *elems = (int64_t)inb::pol::conv_plan(a, vec ? 4 : 1, 3).grid.x * a.C * (a.K + 1);
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
