// selective_scan: h[t, c, n] = exp(delta a[c, n]) h[t - 1, c, n] + delta x[t, c] b[t, n],  y = (<h, c> + d x) silu(z),
// delta = log(1 + exp(dt + dt_bias)), with resets (h before the step is 0) inside the sequence.  Forward pass and one step.
//
// The recurrence runs in registers: a thread holds the NS states of one channel (LN lanes share a channel above 16
// states), a warp neighbouring channels of one sequence, so b and c are the same for all its lanes and are read from
// shared memory by broadcast.  State and sums are fp32.
#include "policy_scan.cuh"

namespace inb {
namespace pol {

constexpr int SCAN_WARPS = 4;        // a block's warps work on their own; no barrier

// MODE 0: outputs; 1: outputs, and the state before every SCAN_STEPS steps is kept for the backward pass; 2: a part's
// end state from zero and its sum of delta (-1 where an episode began inside), 3: the same of the reverse recurrence
// r[t - 1] = exp(delta[t] a) (r[t] + c[t] g[t]), g = gy silu(z)
template <typename T, int NS, int LN, int MODE>
__global__ void __launch_bounds__(SCAN_WARPS * 32) scan_kernel(InbScanArgs a, ScanPlan pl, float* carry, int64_t tasks) {
  constexpr int NP = NS * LN, CW = 32 / LN, TC = SCAN_STEPS, BCL = (2 * TC * NP + 31) / 32;
  __shared__ alignas(16) float bc[SCAN_WARPS][TC][2][NP];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane % LN;
  const int64_t task = (int64_t)blockIdx.x * SCAN_WARPS + warp;
  if (task >= tasks) return;
  const int64_t tiles = (a.C + CW - 1) / CW, n4 = (a.N + 3) / 4 * 4;
  const int64_t tile = task % tiles, sp = task / tiles, s = sp % a.S, part = sp / a.S;
  const int64_t ch = tile * CW + lane / LN;
  const bool on = ch < a.C;
  const int64_t t0 = part * pl.len, t1 = t0 + pl.len < a.T ? t0 + pl.len : a.T;
  const uint8_t* rs = resets(a.reset, s);
  float A[NS], h[NS], dsum = 0.f;
  bool fresh = false;                              // an episode began in this part
  const float bias = on && a.dt_bias != nullptr ? a.dt_bias[ch] : 0.f;
  const float d = on && a.d != nullptr ? a.d[ch] : 0.f;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const int k = j * NS + n;
    A[n] = on && k < a.N ? a.a[ch * a.N + k] * LOG2E : 0.f;
    h[n] = 0.f;
    if (MODE < 2 && on && k < a.N) {
      if (part > 0)
        h[n] = carry[((s * pl.parts + part) * a.C + ch) * n4 + k];
      else if (a.state != nullptr)
        h[n] = a.state[s * a.state_seq + ch * a.N + k];
    }
  }
  // a chunk's inputs, on their way while the one before is worked on
  T x[TC], dt[TC], z[TC], g[TC], bcr[BCL];
  uint32_t rb = 0;
  const bool gate = a.z.p != nullptr;
  auto load = [&](int64_t t) {
#pragma unroll
    for (int i = 0; i < TC; ++i) {
      if (on && t + i < t1) {
        if (MODE != 3) x[i] = row<T>(a.x, s, t + i)[ch];
        dt[i] = row<T>(a.dt, s, t + i)[ch];
        if (gate && MODE != 2) z[i] = row<T>(a.z, s, t + i)[ch];
        if (MODE == 3) g[i] = row<T>(a.gy, s, t + i)[ch];
      }
    }
#pragma unroll
    for (int i = 0; i < BCL; ++i) {
      const int k = i * 32 + lane, which = k / (TC * NP), q = k % (TC * NP), tt = q / NP, n = q % NP;
      bcr[i] = from_f<T>(0.f);
      if (n < a.N && t + tt < t1 && which < 2 && !(MODE == 2 && which == 1) && !(MODE == 3 && which == 0))
        bcr[i] = row<T>(which ? a.c : a.b, s, t + tt)[n];
    }
    rb = reset_bits(rs, a.reset.step, t, t1, lane);
  };
  constexpr bool BACK = MODE == 3;
  const int64_t chunks = (t1 - t0 + TC - 1) / TC;
  load(BACK ? t0 + (chunks - 1) * TC : t0);
  for (int64_t q = 0; q < chunks; ++q) {
    const int64_t t = t0 + (BACK ? chunks - 1 - q : q) * TC;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < BCL; ++i) {
      const int k = i * 32 + lane, which = k / (TC * NP), r = k % (TC * NP);
      if (which < 2) bc[warp][r / NP][which][r % NP] = to_f(bcr[i]);
    }
    __syncwarp();
    if (MODE == 1 && t > 0 && on) {
      float* k = a.kept + ((s * ((a.T + TC - 1) / TC - 1) + t / TC - 1) * a.C + ch) * n4;
#pragma unroll
      for (int n = 0; n < NS; n += 4)
        if (j * NS + n < n4) *reinterpret_cast<float4*>(k + j * NS + n) = make_float4(h[n], h[n + 1], h[n + 2], h[n + 3]);
    }
    float xs[TC], ds[TC], zs[TC], gs[TC];
#pragma unroll
    for (int i = 0; i < TC; ++i) {
      xs[i] = MODE != 3 && on && t + i < t1 ? to_f(x[i]) : 0.f;
      ds[i] = on && t + i < t1 ? to_f(dt[i]) : 0.f;
      zs[i] = MODE != 2 && gate && on && t + i < t1 ? to_f(z[i]) : 0.f;
      gs[i] = MODE == 3 && on && t + i < t1 ? to_f(g[i]) : 0.f;
    }
    const uint32_t bits = rb;
    if (q + 1 < chunks) load(BACK ? t - TC : t + TC);
#pragma unroll
    for (int ii = 0; ii < TC; ++ii) {
      const int i = BACK ? TC - 1 - ii : ii;
      if (t + i >= t1) {
        if (BACK) continue;
        break;
      }
      float slope;
      const float delta = softplus(ds[i] + bias, slope);
      if (!BACK) {
        if (bits >> i & 1) {
          fresh = true;
#pragma unroll
          for (int n = 0; n < NS; ++n) h[n] = 0.f;
        }
        const float u = delta * xs[i];
        float y = 0.f;
#pragma unroll
        for (int n = 0; n < NS; n += 4) {
          const float4 b = *reinterpret_cast<const float4*>(&bc[warp][i][0][j * NS + n]);
          const float bb[4] = {b.x, b.y, b.z, b.w};
          float cc[4] = {};
          if (MODE < 2) {
            const float4 c = *reinterpret_cast<const float4*>(&bc[warp][i][1][j * NS + n]);
            cc[0] = c.x, cc[1] = c.y, cc[2] = c.z, cc[3] = c.w;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            h[n + k] = fmaf(ex2(delta * A[n + k]), h[n + k], u * bb[k]);
            if (MODE < 2) y = fmaf(h[n + k], cc[k], y);
          }
        }
        if (MODE < 2) {
#pragma unroll
          for (int o = 1; o < LN; o *= 2) y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
          y = fmaf(d, xs[i], y);
          if (gate) y *= zs[i] * sigmoid(zs[i]);
          if (on && j == 0) row_out<T>(a.y, s, t + i)[ch] = from_f<T>(y);
        } else {
          dsum += delta;
        }
      } else {
        const float gg = gate ? gs[i] * zs[i] * sigmoid(zs[i]) : gs[i];
        const bool cut = bits >> i & 1;
        fresh |= cut;
        dsum += delta;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          const float r = fmaf(bc[warp][i][1][j * NS + n], gg, h[n]);
          h[n] = cut ? 0.f : ex2(delta * A[n]) * r;
        }
      }
    }
  }
  if (!on) return;
  if (MODE < 2) {
    if (t1 == a.T && a.state_out != nullptr) {
#pragma unroll
      for (int n = 0; n < NS; ++n)
        if (j * NS + n < a.N) a.state_out[s * a.state_out_seq + ch * a.N + j * NS + n] = h[n];
    }
  } else {
    const int64_t at = (s * pl.parts + part) * a.C + ch;
#pragma unroll
    for (int n = 0; n < NS; ++n)
      if (j * NS + n < a.N) carry[at * n4 + j * NS + n] = h[n];
    if (j == 0) carry[a.S * pl.parts * a.C * n4 + at] = fresh ? -1.f : dsum;
  }
}

// The states that the parts begin (reverse: end) with, in place of what they end with from zero.  A thread a state.
__global__ void __launch_bounds__(256) scan_join_kernel(InbScanArgs a, ScanPlan pl, float* carry, bool reverse) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.S * a.C * a.N) return;
  const int n = (int)(i % a.N);
  const int64_t sc = i / a.N, ch = sc % a.C, s = sc / a.C, n4 = (a.N + 3) / 4 * 4;
  const float A = a.a[ch * a.N + n] * LOG2E;
  const float* sums = carry + a.S * pl.parts * a.C * n4;
  float h = 0.f;
  if (reverse) {
    if (a.gstate_out != nullptr) h = a.gstate_out[i];
  } else if (a.state != nullptr) {
    h = a.state[s * a.state_seq + ch * a.N + n];
  }
  for (int64_t q = 0; q < pl.parts; ++q) {
    const int64_t at = (s * pl.parts + (reverse ? pl.parts - 1 - q : q)) * a.C + ch;
    const float end = carry[at * n4 + n], sum = sums[at];
    carry[at * n4 + n] = h;
    h = sum < 0.f ? end : fmaf(ex2(sum * A), h, end);
  }
}

// One step: bound by the states' bytes.  V states a thread, moved by one access where they are aligned; `lanes` threads a
// channel (a power of two up to 16).
template <typename T, int V>
__global__ void __launch_bounds__(256) scan_step_kernel(InbScanArgs a, int lanes) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, sc = i / lanes;
  const int j = (int)(i % lanes);
  const bool on = sc < a.S * a.C;
  const int64_t ch = on ? sc % a.C : 0, s = on ? sc / a.C : 0;
  float y = 0.f;
  const bool cut = a.state == nullptr || (a.reset.p != nullptr && *resets(a.reset, s) != 0);
  const float x = to_f(row<T>(a.x, s, 0)[ch]), raw = to_f(row<T>(a.dt, s, 0)[ch]);
  const T *b = row<T>(a.b, s, 0), *c = row<T>(a.c, s, 0);
  float slope;
  const float delta = softplus(raw + (a.dt_bias != nullptr ? a.dt_bias[ch] : 0.f), slope), u = delta * x;
  if (on) {
    const float* A = a.a + ch * a.N;
    const float* old = a.state + s * a.state_seq + ch * a.N;
    float* out = a.state_out + s * a.state_out_seq + ch * a.N;
    for (int n = j * V; n < a.N; n += lanes * V) {
      Pack<float, V> h;
#pragma unroll
      for (int k = 0; k < V; ++k) h.v[k] = 0.f;
      if (!cut) h = ld<float, V>(old + n);
      const Pack<float, V> w = ld<float, V>(A + n);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        h.v[k] = fmaf(ex2(delta * w.v[k] * LOG2E), h.v[k], u * to_f(b[n + k]));
        y = fmaf(h.v[k], to_f(c[n + k]), y);
      }
      if (a.state_out != nullptr) st<float, V>(out + n, h);
    }
  }
  for (int o = 1; o < lanes; o *= 2) y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
  if (!on || j != 0) return;
  if (a.d != nullptr) y = fmaf(a.d[ch], x, y);
  if (a.z.p != nullptr) {
    const float z = to_f(row<T>(a.z, s, 0)[ch]);
    y *= z * sigmoid(z);
  }
  row_out<T>(a.y, s, 0)[ch] = from_f<T>(y);
}

int scan_check(const InbScanArgs& a) {
  if (a.dtype < 0 || a.dtype > 2 || a.C < 1 || a.C > INB_MAX_MEMORY_C || a.N < 1 || a.N > INB_MAX_SCAN_N || a.S < 0 ||
      a.S > INB_MAX_MEMORY_S || a.T < 0 || a.T > INB_MAX_MEMORY_S || (a.reset.p != nullptr && a.reset.rows < 1))
    return -2;
  if (a.S * (int64_t)a.C > (1ll << 34)) return -2;      // blocks of one launch
  return 0;
}
int scan_join(const InbScanArgs& a, const ScanPlan& p, float* carry, bool reverse, cudaStream_t s) {
  scan_join_kernel<<<(unsigned)ceil_div(a.S * a.C * a.N, 256), 256, 0, s>>>(a, p, carry, reverse);
  return launch_status();
}

template <typename T, int NS, int LN, int MODE>
static void scan_go(const InbScanArgs& a, const ScanPlan& p, float* carry, cudaStream_t s) {
  const int64_t tasks = a.S * p.parts * ceil_div(a.C, 32 / LN);
  scan_kernel<T, NS, LN, MODE><<<(unsigned)ceil_div(tasks, SCAN_WARPS), SCAN_WARPS * 32, 0, s>>>(a, p, carry, tasks);
}
template <typename T, int NS, int LN>
static int scan_mode(const InbScanArgs& a, const ScanPlan& p, float* carry, int mode, cudaStream_t s) {
  if (mode == 3) {
    scan_go<T, NS, LN, 3>(a, p, carry, s);
    return scan_join(a, p, carry, true, s);
  }
  if (p.split()) {
    scan_go<T, NS, LN, 2>(a, p, carry, s);
    const int rc = scan_join(a, p, carry, false, s);
    if (rc != 0) return rc;
  }
  if (a.kept != nullptr)
    scan_go<T, NS, LN, 1>(a, p, carry, s);
  else
    scan_go<T, NS, LN, 0>(a, p, carry, s);
  return launch_status();
}
template <typename T>
static int scan_type(const InbScanArgs& a, const ScanPlan& p, float* carry, int mode, cudaStream_t s) {
  if (a.N <= 4) return scan_mode<T, 4, 1>(a, p, carry, mode, s);
  if (a.N <= 8) return scan_mode<T, 8, 1>(a, p, carry, mode, s);
  if (a.N <= 16) return scan_mode<T, 16, 1>(a, p, carry, mode, s);
  if (a.N <= 32) return scan_mode<T, 16, 2>(a, p, carry, mode, s);
  return scan_mode<T, 16, 4>(a, p, carry, mode, s);
}
template <typename T>
static int scan_step(const InbScanArgs& a, cudaStream_t s) {
  const uint64_t m = (uint64_t)(uintptr_t)a.state | (uint64_t)(uintptr_t)a.state_out | (uint64_t)(uintptr_t)a.a |
                     (uint64_t)(a.state_seq * 4) | (uint64_t)(a.state_out_seq * 4) | (uint64_t)(a.N * 4);
  const bool vec = (m & 15) == 0;
  int lanes = 1;
  while (lanes < 16 && lanes * 4 < a.N) lanes *= 2;
  const unsigned blocks = (unsigned)ceil_div(a.S * a.C * lanes, 256);
  if (vec)
    scan_step_kernel<T, 4><<<blocks, 256, 0, s>>>(a, lanes);
  else
    scan_step_kernel<T, 1><<<blocks, 256, 0, s>>>(a, lanes);
  return launch_status();
}
// mode 0: the forward pass; 3: the backward pass's parts
int scan_launch(const InbScanArgs& a, const ScanPlan& p, float* carry, int mode, cudaStream_t s) {
  if (a.dtype == INB_BF16) return scan_type<bf16>(a, p, carry, mode, s);
  if (a.dtype == INB_F16) return scan_type<f16>(a, p, carry, mode, s);
  return scan_type<float>(a, p, carry, mode, s);
}

}  // namespace pol
}  // namespace inb

using namespace inb::pol;

extern "C" int inb_selective_scan_kept(const InbScanArgs* args, int64_t* elems) {
  if (args == nullptr || elems == nullptr) return -1;
  const int rc = scan_check(*args);
  if (rc != 0) return rc;
  *elems = args->S == 0 || args->T == 0 ? 0 : args->S * (scan_chunks(*args) - 1) * args->C * scan_n4(*args);
  return 0;
}

extern "C" int inb_selective_scan_fwd(const InbScanArgs* args, void* cuda_stream) {
  if (args == nullptr) return -1;
  const InbScanArgs& a = *args;
  const int rc = scan_check(a);
  if (rc != 0) return rc;
  if (a.S == 0 || a.T == 0) return 0;
  if (a.x.p == nullptr || a.dt.p == nullptr || a.b.p == nullptr || a.c.p == nullptr || a.y.p == nullptr || a.a == nullptr) return -3;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (a.T == 1) {
    if (a.dtype == INB_BF16) return scan_step<bf16>(a, s);
    if (a.dtype == INB_F16) return scan_step<f16>(a, s);
    return scan_step<float>(a, s);
  }
  const ScanPlan p = scan_plan(a, 32 / scan_lanes(a.N));
  if (p.split() && (a.work == nullptr || a.work_elems < scan_carry_elems(a, p))) return -5;
  return scan_launch(a, p, a.work, 0, s);
}
