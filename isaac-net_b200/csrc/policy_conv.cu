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

constexpr int CONV_U = 4;       // steps whose loads are on their way at once

struct ConvPlan {
  int64_t parts, len, tasks;    // parts of the time axis, their steps; sequences x parts
  uint32_t cv;                  // threads a task: vectors of V channels
};

// ---------------------------------------------------------------------------------------------- forward
template <typename T, int V, int K>
__global__ void __launch_bounds__(256) conv_fwd_kernel(InbConvArgs a, ConvPlan pl) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t task = i / pl.cv;
  if (task >= pl.tasks) return;
  const int64_t ch = (i - task * pl.cv) * V;
  const int64_t part = task / a.S, s = task - part * a.S;      // neighbouring threads: the same step of the next sequence
  const int64_t t0 = part * pl.len, t1 = t0 + pl.len < a.T ? t0 + pl.len : a.T;
  const uint8_t* rs = resets(a.reset, s);
  float w[K][V], bias[V], hist[K - 1][V];       // hist[j]: x[t - 1 - j]
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = a.bias != nullptr ? to_f(((const T*)a.bias)[ch + v]) : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][v] = to_f(((const T*)a.w)[(ch + v) * K + k]);
  }
  auto zero = [&] {
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) hist[j][v] = 0.f;
  };
  auto push = [&](const Pack<T, V>& x) {
#pragma unroll
    for (int j = K - 2; j > 0; --j)
#pragma unroll
      for (int v = 0; v < V; ++v) hist[j][v] = hist[j - 1][v];
#pragma unroll
    for (int v = 0; v < V; ++v) hist[0][v] = to_f(x.v[v]);
  };
  zero();
  for (int64_t t = t0 - (K - 1); t < t0; ++t) {
    if (t >= 0) {
      if (rs != nullptr && rs[t * a.reset.step]) zero();
      push(ld<T, V>(row<T>(a.x, s, t) + ch));
    } else if (a.state != nullptr) {
      push(ld<T, V>((const T*)a.state + s * a.state_seq + (t + K - 1) * a.C + ch));
    }
  }
  for (int64_t t = t0; t < t1; t += CONV_U) {
    Pack<T, V> x[CONV_U];
    bool reset[CONV_U];
#pragma unroll
    for (int u = 0; u < CONV_U; ++u)
      if (t + u < t1) {
        x[u] = ld<T, V>(row<T>(a.x, s, t + u) + ch);
        reset[u] = rs != nullptr && rs[(t + u) * a.reset.step];
      }
#pragma unroll
    for (int u = 0; u < CONV_U; ++u) {
      if (t + u >= t1) break;
      if (reset[u]) zero();
      Pack<T, V> y;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float p = fmaf(to_f(x[u].v[v]), w[K - 1][v], bias[v]);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) p = fmaf(hist[j][v], w[K - 2 - j][v], p);
        y.v[v] = from_f<T>(a.act == INB_ACT_SILU ? p * sigmoid(p) : p);
      }
      push(x[u]);
      st<T, V>(row_out<T>(a.y, s, t + u) + ch, y);
    }
  }
  if (t1 == a.T && a.state_out != nullptr) {
    T* out = (T*)a.state_out + s * a.state_out_seq + ch;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      Pack<T, V> p;
#pragma unroll
      for (int v = 0; v < V; ++v) p.v[v] = from_f<T>(hist[j][v]);      // what was read, or 0: exact
      st<T, V>(out + (K - 2 - j) * a.C, p);
    }
  }
}

// ---------------------------------------------------------------------------------------------- backward
// pend[j - 1] gathers gx[t - j] while later steps still add to it; step t completes gx[t - (K - 1)].  A part goes K - 1 steps
// beyond its end, for gx alone.  A block is tx channel vectors x ty tasks and strides over the tasks, so that gw and gbias
// stay in registers; one partial row a block, [C K | C], added by a second launch.
template <typename T, int V, int K>
__global__ void __launch_bounds__(128) conv_bwd_kernel(InbConvArgs a, ConvPlan pl) {
  extern __shared__ float smem[];
  const int64_t ch = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * V;
  const bool on = ch < a.C;
  float w[K][V], bias[V], gw[K][V], gb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = on && a.bias != nullptr ? to_f(((const T*)a.bias)[ch + v]) : 0.f;
    gb[v] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      w[k][v] = on ? to_f(((const T*)a.w)[(ch + v) * K + k]) : 0.f;
      gw[k][v] = 0.f;
    }
  }
  if (on)
    for (int64_t task = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; task < pl.tasks; task += (int64_t)gridDim.x * blockDim.y) {
      const int64_t part = task / a.S, s = task - part * a.S;
      const int64_t t0 = part * pl.len, t1 = t0 + pl.len < a.T ? t0 + pl.len : a.T;
      const int64_t last = t1 + K - 1, end = last < a.T ? last : a.T;
      const uint8_t* rs = resets(a.reset, s);
      float hist[K - 1][V], pend[K - 1][V];
      int m = K - 1;                        // how many steps before this one are seen
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) hist[j][v] = pend[j][v] = 0.f;
      auto restart = [&] {
        m = 0;
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
#pragma unroll
          for (int v = 0; v < V; ++v) hist[j][v] = 0.f;
      };
      auto push = [&](const Pack<T, V>& x) {
#pragma unroll
        for (int j = K - 2; j > 0; --j)
#pragma unroll
          for (int v = 0; v < V; ++v) hist[j][v] = hist[j - 1][v];
#pragma unroll
        for (int v = 0; v < V; ++v) hist[0][v] = to_f(x.v[v]);
        m = m < K - 1 ? m + 1 : m;
      };
      // gx of step t - (K - 1) is complete; before the sequence it is the initial state's
      auto emit = [&](int64_t t) {
        const int64_t at = t - (K - 1);
        Pack<T, V> p;
#pragma unroll
        for (int v = 0; v < V; ++v) p.v[v] = from_f<T>(pend[K - 2][v]);
        if (at >= t0)
          st<T, V>(row_out<T>(a.gx, s, at) + ch, p);
        else if (at < 0 && a.gstate != nullptr)
          st<T, V>((T*)a.gstate + (s * (K - 1) + at + K - 1) * a.C + ch, p);
      };
      auto shift = [&](const float (&g)[V]) {
#pragma unroll
        for (int j = K - 2; j > 0; --j)
#pragma unroll
          for (int v = 0; v < V; ++v) pend[j][v] = pend[j - 1][v];
#pragma unroll
        for (int v = 0; v < V; ++v) pend[0][v] = w[K - 1][v] * g[v];
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
        Pack<T, V> x[CONV_U], gy[CONV_U];
        bool reset[CONV_U];
#pragma unroll
        for (int u = 0; u < CONV_U; ++u)
          if (t + u < end) {
            x[u] = ld<T, V>(row<T>(a.x, s, t + u) + ch);
            gy[u] = ld<T, V>(row<T>(a.gy, s, t + u) + ch);
            reset[u] = rs != nullptr && rs[(t + u) * a.reset.step];
          }
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
              float p = fmaf(xv, w[K - 1][v], bias[v]);
#pragma unroll
              for (int j = 0; j < K - 1; ++j) p = fmaf(hist[j][v], w[K - 2 - j][v], p);
              const float q = sigmoid(p);
              g[v] *= q * fmaf(p, 1.f - q, 1.f);
            }
            if (mine) {
              gb[v] += g[v];
              gw[K - 1][v] = fmaf(g[v], xv, gw[K - 1][v]);
#pragma unroll
              for (int j = 0; j < K - 1; ++j) gw[K - 2 - j][v] = fmaf(g[v], hist[j][v], gw[K - 2 - j][v]);
            }
#pragma unroll
            for (int j = 0; j < K - 1; ++j)
              if (j < m) pend[j][v] = fmaf(w[K - 2 - j][v], g[v], pend[j][v]);
          }
          emit(t + u);
          shift(g);
          push(x[u]);
        }
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
// Parts of the time axis: as many as fill the GPU with threads, none shorter than 16 steps (a part re-reads K - 1).
static ConvPlan conv_plan(const InbConvArgs& a, int V, int64_t threads) {
  ConvPlan p;
  p.cv = (uint32_t)ceil_div(a.C, V);
  int64_t parts = ceil_div(threads, a.S * (int64_t)p.cv), most = a.T / 16;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  p.len = ceil_div(a.T, parts);
  p.parts = ceil_div(a.T, p.len);
  p.tasks = a.S * p.parts;
  return p;
}
struct ConvBwd {
  ConvPlan plan;
  dim3 block, grid;
  int smem;
};
static ConvBwd conv_bwd_plan(const InbConvArgs& a, int V) {
  ConvBwd b;
  const int64_t room = (int64_t)sm_count() * 4 * 128;
  b.plan = conv_plan(a, V, room);
  unsigned tx = 1;
  while (tx < 128 && tx < b.plan.cv) tx *= 2;
  b.block = dim3(tx, 128 / tx);
  const unsigned gy = (unsigned)ceil_div(b.plan.cv, tx);
  int64_t gx = ceil_div(sm_count() * 4, gy), need = ceil_div(b.plan.tasks, b.block.y);
  if (gx > need) gx = need;
  b.grid = dim3((unsigned)gx, gy);
  b.smem = 128 * V * (a.K + 1) * 4;
  return b;
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
  if (ceil_div(a.S * (int64_t)a.C, 256) > INT32_MAX / 2) return -2;      // blocks of one launch
  return 0;
}

template <typename T, int V, int K>
static int conv_fwd_go(const InbConvArgs& a, cudaStream_t s) {
  const ConvPlan p = conv_plan(a, V, (int64_t)sm_count() * 1024);
  conv_fwd_kernel<T, V, K><<<(unsigned)ceil_div(p.tasks * p.cv, 256), 256, 0, s>>>(a, p);
  return launch_status();
}
template <typename T, int V, int K>
static int conv_bwd_go(const InbConvArgs& a, cudaStream_t s) {
  const ConvBwd b = conv_bwd_plan(a, V);
  conv_bwd_kernel<T, V, K><<<b.grid, b.block, b.smem, s>>>(a, b.plan);
  colsum<T>(a.work, b.grid.x, (int64_t)a.C * (K + 1), (int64_t)a.C * K, (int64_t)a.C * (K + 1), a.gw, a.gbias, nullptr, s);
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
  *elems = (int64_t)inb::pol::conv_bwd_plan(a, vec ? 4 : 1).grid.x * a.C * (a.K + 1);
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
