// selective_scan: h[t, c, n] = exp(delta a[c, n]) h[t - 1, c, n] + delta x[t, c] b[t, n],  y = (<h, c> + d x) silu(z),
// delta = log(1 + exp(dt + dt_bias)), with resets (h before the step is 0) inside the sequence.  Forward pass and one step.
//
// The recurrence runs in registers: a thread holds the NS states of one channel (LN lanes share a channel above 16
// states), a warp neighbouring channels of one sequence, so b and c are the same for all its lanes and are read from
// shared memory by broadcast.  State and sums are fp32.
#include "policy_scan.cuh"

namespace inb {
namespace pol {

// A block's SCAN_WARPS warps work on their own; no barrier.
//
// MODE 0: outputs; 1: outputs, and the state before every SCAN_STEPS steps is kept for the backward pass; 2: a part's
// end state from zero and its sum of delta (-1 where an episode began inside), 3: the same of the reverse recurrence
// r[t - 1] = exp(delta[t] a) (r[t] + c[t] g[t]), g = gy silu(z), which runs from the part's last step to its first.
//
// Bound by the exponentials (one a state and step, 16 a clock and SM) and, next to that, by instruction issue: an eighth of
// them goes to the FMA pipe (ex2_poly), which evens the two out; all else is packed in pairs of states.  A chunk of
// SCAN_STEPS steps is prepared at once (delta, u, the gate), then the next one's loads are sent, then its steps run.
// 179 warp instructions a step (32 channels, 16 states), 137 cycles of the special function unit.  1024 x 32 sequences of 16
// steps, 128 channels, bf16, with the states kept: 540 us (2.5 TB/s); one of 4096 steps, 2048 channels, in 37 parts: 50 + 9 (join) + 68 us.
// WIDE: the rows of b and c are NS whole, aligned to 16 bytes and moved by that
template <typename T, int NS, int LN, int MODE, bool WIDE>
__global__ void __launch_bounds__(SCAN_WARPS * 32, 4) scan_kernel(InbScanArgs a, ScanPlan pl, float* carry) {
  constexpr int NP = NS * LN, CW = 32 / LN, TC = SCAN_STEPS, BCL = (2 * TC * NP + 31) / 32, NH = NS / 2, POLY = NS / 16;
  constexpr int BCW = 16 / sizeof(T);
  constexpr bool BACK = MODE == 3;
  __shared__ alignas(16) float bc[SCAN_WARPS][TC][2][NP];
  __shared__ float4 stage[SCAN_WARPS][TC][32];       // delta, u, silu(z) (1 without z), d x of this lane's channel
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = lane % LN;
  const int n4 = (a.N + 3) / 4 * 4;
  // a block is one sequence's: what depends on it is the same for all its threads
  const int64_t at = pl.parts > 1 ? blockIdx.x / (uint32_t)a.S : 0, s = blockIdx.x - at * a.S, part = at + BACK;
  const int c0 = (blockIdx.y * (blockDim.x >> 5) + warp) * CW + lane / LN;
  const bool on = c0 < a.C;
  const int ch = on ? c0 : a.C - 1;                // lanes beyond the last channel read it too and write nothing
  const int64_t t0 = part * pl.len, t1 = t0 + pl.len < a.T ? t0 + pl.len : a.T, first = BACK ? t1 - 1 : t0;
  constexpr int DIR = BACK ? -1 : 1;
  float2 A[NH], h[NH];
  float dsum = 0.f;
  bool fresh = false;                              // an episode began in this part
  const float bias = a.dt_bias != nullptr ? a.dt_bias[ch] : 0.f, d = MODE < 2 && a.d != nullptr ? a.d[ch] : 0.f;
  const float* h0 = nullptr;                       // the state before the first step
  if (MODE < 2) h0 = part > 0 ? carry + ((s * pl.parts + part) * a.C + ch) * n4 : a.state != nullptr ? a.state + s * a.state_seq + ch * a.N : nullptr;
  const float* pa = a.a + ch * a.N;
  if (a.N == NP && ((uintptr_t)a.a & 15) == 0 && (part > 0 || (((uintptr_t)a.state | (a.state_seq * 4)) & 15) == 0)) {
#pragma unroll
    for (int n = 0; n < NH; n += 2) {
      const float4 v = *reinterpret_cast<const float4*>(pa + j * NS + 2 * n);
      float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
      if (h0 != nullptr) w = *reinterpret_cast<const float4*>(h0 + j * NS + 2 * n);
      A[n] = mul2(make_float2(v.x, v.y), both(LOG2E)), A[n + 1] = mul2(make_float2(v.z, v.w), both(LOG2E));
      h[n] = make_float2(w.x, w.y), h[n + 1] = make_float2(w.z, w.w);
    }
  } else {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int k = j * NS + n;
      (n & 1 ? A[n / 2].y : A[n / 2].x) = k < a.N ? pa[k] * LOG2E : 0.f;
      (n & 1 ? h[n / 2].y : h[n / 2].x) = k < a.N && h0 != nullptr ? h0[k] : 0.f;
    }
  }
  const bool gate = a.z.p != nullptr && MODE != 2;
  const T *px = row<T>(BACK ? a.gy : a.x, s, first) + ch, *pd = row<T>(a.dt, s, first) + ch;
  const T* pz = gate ? row<T>(a.z, s, first) + ch : nullptr;
  T* py = MODE < 2 ? row_out<T>(a.y, s, first) + ch : nullptr;
  const T *pb = row<T>(a.b, s, first), *pc = row<T>(a.c, s, first);
  const uint8_t* rs = resets(a.reset, s);
  if (rs != nullptr) rs += first * a.reset.step;
  int64_t left = t1 - t0;
  uint32_t x[TC], dt[TC], z[TC], bcr[WIDE ? 1 : BCL], flag = 0;      // the next chunk's inputs; BACK: x is gy
  Words<T, BCW> wide[WIDE ? BCL / BCW : 1];
  auto load = [&](int steps) {
#pragma unroll
    for (int i = 0; i < TC; ++i) {
      if (i < steps) {
        x[i] = ld_raw(px);
        dt[i] = ld_raw(pd);
        if (gate) z[i] = ld_raw(pz);
      }
      px += DIR * (BACK ? a.gy.step : a.x.step);
      pd += DIR * a.dt.step;
      if (gate) pz += DIR * a.z.step;
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < BCL / BCW; ++i) {
        const int k = (i * 32 + lane) * BCW, which = k / (TC * NP), q = k % (TC * NP), tt = q / NP, n = q % NP;
        // the steps beyond the last one read it again
        const int tl = tt < steps ? tt : steps - 1;
        wide[i].load(which ? pc + (DIR * tl * a.c.step + n) : pb + (DIR * tl * a.b.step + n));
      }
    } else {
#pragma unroll
      for (int i = 0; i < BCL; ++i) {
        const int k = i * 32 + lane, which = k / (TC * NP), q = k % (TC * NP), tt = q / NP, n = q % NP;
        bcr[i] = 0;
        if (n < a.N && tt < steps && which < 2 && !(MODE == 2 && which == 1) && !(BACK && which == 0))
          bcr[i] = ld_raw(which ? pc + (DIR * tt * a.c.step + n) : pb + (DIR * tt * a.b.step + n));
      }
    }
    pb += DIR * TC * a.b.step;
    pc += DIR * TC * a.c.step;
    flag = reset_flag(rs, DIR * a.reset.step, steps, lane);
    if (rs != nullptr) rs += DIR * TC * a.reset.step;
  };
#pragma unroll
  for (int i = 0; i < TC; ++i) x[i] = dt[i] = z[i] = 0;
  load(left < TC ? (int)left : TC);
  float* kept = MODE == 1 ? a.kept + ((s * ((a.T + TC - 1) / TC - 1) + t0 / TC - 1) * a.C + ch) * n4 + j * NS : nullptr;
  for (; left > 0; left -= TC) {
    if (MODE == 1) {
      if (on && (part > 0 || left < t1 - t0)) {
#pragma unroll
        for (int n = 0; n < NS; n += 4)
          if (j * NS + n < n4)
            *reinterpret_cast<float4*>(kept + n) = make_float4(h[n / 2].x, h[n / 2].y, h[n / 2 + 1].x, h[n / 2 + 1].y);
      }
      kept += (int64_t)a.C * n4;
    }
    const int steps = left < TC ? (int)left : TC, ahead = left - TC < TC ? (int)(left - TC) : TC;      // now, and of the next chunk
    __syncwarp();
#pragma unroll
    for (int i = 0; i < TC; ++i) {
      const float xv = raw_f<T>(x[i]), delta = softplus(raw_f<T>(dt[i]) + bias);
      float o = 1.f;
      if (gate) {
        const float zv = raw_f<T>(z[i]);
        o = zv * sigmoid(zv);
      }
      // BACK: u is g, whose c (in place of b) it multiplies
      stage[warp][i][lane] = make_float4(delta, BACK ? xv * o : delta * xv, o, d * xv);
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < BCL / BCW; ++i) {
        const int k = (i * 32 + lane) * BCW, which = k / (TC * NP), r = k % (TC * NP);
        float4* to = reinterpret_cast<float4*>(&bc[warp][r / NP][which][r % NP]);
#pragma unroll
        for (int e = 0; e < BCW / 4; ++e) {
          const float2 p = wide[i].pair(2 * e), q = wide[i].pair(2 * e + 1);
          to[e] = make_float4(p.x, p.y, q.x, q.y);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < BCL; ++i) {
        const int k = i * 32 + lane, which = k / (TC * NP), r = k % (TC * NP);
        if (which < 2) bc[warp][r / NP][which][r % NP] = raw_f<T>(bcr[i]);
      }
    }
    const uint32_t bits = __ballot_sync(0xFFFFFFFFu, flag != 0);
    if (ahead > 0) load(ahead);
    __syncwarp();
    float delta = 0.f;                 // the chunk's sum
#pragma unroll 2
    for (int i = 0; i < steps; ++i) {
      const float4 in = stage[warp][i][lane];
      const float2 D = both(in.x), U = both(in.y);
      const bool cut = bits >> i & 1;
      if (MODE >= 2) fresh |= cut;
      if (!BACK && cut) {
#pragma unroll
        for (int n = 0; n < NH; ++n) h[n] = make_float2(0.f, 0.f);
        delta = 0.f;
        keep_branch();
      }
      delta += in.x;
      float2 y = make_float2(0.f, 0.f);
#pragma unroll
      for (int n = 0; n < NH; n += 2) {
        const float4 q = *reinterpret_cast<const float4*>(&bc[warp][i][BACK ? 1 : 0][j * NS + 2 * n]);
        float4 c = {};
        if (MODE < 2) c = *reinterpret_cast<const float4*>(&bc[warp][i][1][j * NS + 2 * n]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 v = mul2(D, A[n + k]), b = k ? make_float2(q.z, q.w) : make_float2(q.x, q.y);
          const float2 e = n + k < POLY ? ex2_poly(v) : make_float2(ex2(v.x), ex2(v.y));
          if (BACK)
            h[n + k] = mul2(e, fma2(b, U, h[n + k]));
          else
            h[n + k] = fma2(e, h[n + k], mul2(U, b));
          if (MODE < 2) y = fma2(h[n + k], k ? make_float2(c.z, c.w) : make_float2(c.x, c.y), y);
        }
      }
      if (BACK && cut) {
#pragma unroll
        for (int n = 0; n < NH; ++n) h[n] = make_float2(0.f, 0.f);
        keep_branch();
      }
      if (MODE < 2) {
        float o = y.x + y.y;
#pragma unroll
        for (int m = 1; m < LN; m *= 2) o += __shfl_xor_sync(0xFFFFFFFFu, o, m);
        o = (o + in.w) * in.z;
        if (on && j == 0) *py = from_f<T>(o);
        py += a.y.step;
      }
    }
    dsum += delta;
#pragma unroll
    for (int n = POLY; n < NH; ++n) h[n] = unbias(h[n], A[n], both(delta));
  }
  if (!on) return;
  if (MODE >= 2 && j == 0) carry[a.S * pl.parts * a.C * n4 + (s * pl.parts + part) * a.C + ch] = fresh ? -1.f : dsum;
  float* to = MODE >= 2 ? carry + ((s * pl.parts + part) * a.C + ch) * n4
                        : t1 == a.T && a.state_out != nullptr ? a.state_out + s * a.state_out_seq + ch * a.N : nullptr;
  if (to == nullptr) return;
  if (a.N == NP && (MODE >= 2 || (((uintptr_t)a.state_out | (a.state_out_seq * 4)) & 15) == 0)) {
#pragma unroll
    for (int n = 0; n < NH; n += 2) *reinterpret_cast<float4*>(to + j * NS + 2 * n) = make_float4(h[n].x, h[n].y, h[n + 1].x, h[n + 1].y);
  } else {
#pragma unroll
    for (int n = 0; n < NS; ++n)
      if (j * NS + n < a.N) to[j * NS + n] = n & 1 ? h[n / 2].y : h[n / 2].x;
  }
}

// The states that the parts begin (reverse: end) with, in place of what they end with from zero (the last one's, which no
// launch has written, is read and left unused).  A thread a state.
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
  constexpr int U = 16;               // parts whose loads are on their way at once
  for (int64_t q0 = 0; q0 < pl.parts; q0 += U) {
    float end[U], sum[U];
    int64_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t q = q0 + u < pl.parts ? q0 + u : pl.parts - 1;
      at[u] = (s * pl.parts + (reverse ? pl.parts - 1 - q : q)) * a.C + ch;
      end[u] = carry[at[u] * n4 + n], sum[u] = sums[at[u]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (q0 + u >= pl.parts) break;
      carry[at[u] * n4 + n] = h;
      h = sum[u] < 0.f ? end[u] : fmaf(ex2(sum[u] * A), h, end[u]);
    }
  }
}

// One step: bound by the states' bytes.  A thread holds V x G states of one channel (V moved by one access; `lanes` threads a
// channel, a power of two) and walks over sequences, STEP_B at a time, whose loads are on their way at once.  A block takes
// `chans` channels (a power of two, a warp's at least) of `runs` sequences at a time (MANY: more than one), next to one another, `per` times.
// 131072 sequences of 256 channels, N = 16: 800 us alone (5.7 TB/s).  23168 sequences of 18 channels, N = 4: 18 us with shared blocks, 57 with
// one sequence a block; as a variable, `runs` cost the large call 30 % in registers, hence MANY.
constexpr int STEP_THREADS = 256, STEP_B = 2;
template <typename T, int V, int G, bool MANY>
__global__ void __launch_bounds__(STEP_THREADS, 4) scan_step_kernel(InbScanArgs a, int lanes, int chans, int per) {
  if (!MANY) chans = STEP_THREADS / lanes;
  const int j = threadIdx.x % lanes, w = threadIdx.x / lanes;
  const int c0 = blockIdx.x * chans + (MANY ? w & (chans - 1) : w);
  const bool on = c0 < a.C;
  const int ch = on ? c0 : a.C - 1;
  const uint32_t runs = MANY ? STEP_THREADS / (lanes * chans) : 1;
  const int64_t b0 = (int64_t)blockIdx.y * per * runs, b1 = b0 + (int64_t)per * runs, s0 = MANY ? b0 + w / chans : b0;
  const int64_t s1 = b1 < a.S ? b1 : a.S;
  if (MANY && s0 >= a.S) return;
  const float bias = a.dt_bias != nullptr ? a.dt_bias[ch] : 0.f, d = a.d != nullptr ? a.d[ch] : 0.f;
  const bool gate = a.z.p != nullptr;
  float A[G][V];
  int at[G];                     // this thread's states; those beyond the last one are read as the last ones and not written
#pragma unroll
  for (int q = 0; q < G; ++q) {
    at[q] = (q * lanes + j) * V;
#pragma unroll
    for (int k = 0; k < V; ++k) A[q][k] = at[q] < a.N ? a.a[ch * a.N + at[q] + k] * LOG2E : 0.f;
  }
  // the reset flag's row, and how many sequences of it have passed
  const uint8_t* pr = resets(a.reset, s0);
  uint32_t of = pr != nullptr ? (uint32_t)s0 % (uint32_t)a.reset.rows : 0;
  for (int64_t s = s0; s < s1; s += STEP_B * runs) {
    const int n = s1 - s > (STEP_B - 1) * (int64_t)runs ? STEP_B : MANY ? (int)((s1 - s + runs - 1) / runs) : (int)(s1 - s);
    uint32_t x[STEP_B], dt[STEP_B], z[STEP_B], cut[STEP_B];
    Words<T, V> b[STEP_B][G], c[STEP_B][G];
    Pack<float, V> h[STEP_B][G];
    const T *px = row<T>(a.x, s, 0) + ch, *pd = row<T>(a.dt, s, 0) + ch, *pz = gate ? row<T>(a.z, s, 0) + ch : nullptr;
    const T *pb = row<T>(a.b, s, 0), *pc = row<T>(a.c, s, 0);
    const float* ph = a.state != nullptr ? a.state + s * a.state_seq + ch * a.N : nullptr;
    float* po = a.state_out != nullptr ? a.state_out + s * a.state_out_seq + ch * a.N : nullptr;
    T* py = row_out<T>(a.y, s, 0) + ch;
#pragma unroll
    for (int u = 0; u < STEP_B; ++u) {
      // the sequences beyond the last one read it again
      x[u] = ld_raw(px), dt[u] = ld_raw(pd);
      if (gate) z[u] = ld_raw(pz);
      cut[u] = 0;
      if (pr != nullptr && u < n) {
        cut[u] = *pr;
        of += runs;
        if (of >= (uint32_t)a.reset.rows) {
          const uint32_t past = MANY ? of / (uint32_t)a.reset.rows : 1;
          of = MANY ? of - past * (uint32_t)a.reset.rows : 0;
          if (s + (u + 1) * (int64_t)runs < a.S) pr += past * a.reset.seq;
        }
      }
#pragma unroll
      for (int q = 0; q < G; ++q) {
        const int k0 = at[q] < a.N ? at[q] : a.N - V;
        if (ph != nullptr) h[u][q] = ld<float, V>(ph + k0);
        b[u][q].load(pb + k0), c[u][q].load(pc + k0);
      }
      if (u + 1 < n) {
        px += runs * a.x.seq, pd += runs * a.dt.seq, pb += runs * a.b.seq, pc += runs * a.c.seq;
        if (gate) pz += runs * a.z.seq;
        if (ph != nullptr) ph += runs * a.state_seq;
      }
    }
#pragma unroll
    for (int u = 0; u < STEP_B; ++u) {
      if (u >= n) break;
      const float xv = raw_f<T>(x[u]);
      float y = 0.f;
      const float delta = softplus(raw_f<T>(dt[u]) + bias), in = delta * xv;
      const bool none = ph == nullptr || cut[u] != 0;
#pragma unroll
      for (int q = 0; q < G; ++q) {
        Pack<float, V> o;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float2 bp = b[u][q].pair(k / 2), cp = c[u][q].pair(k / 2);
          o.v[k] = fmaf(ex2(delta * A[q][k]), none ? 0.f : h[u][q].v[k], in * (k & 1 ? bp.y : bp.x));
          if (at[q] < a.N) y = fmaf(o.v[k], k & 1 ? cp.y : cp.x, y);
        }
        if (po != nullptr && on && at[q] < a.N) st<float, V>(po + at[q], o);
      }
      for (int o = 1; o < lanes; o *= 2) y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
      y = fmaf(d, xv, y);
      if (gate) {
        const float zv = raw_f<T>(z[u]);
        y *= zv * sigmoid(zv);
      }
      if (on && j == 0) *py = from_f<T>(y);
      py += runs * a.y.seq;
      if (po != nullptr) po += runs * a.state_out_seq;
    }
  }
}

int scan_check(const InbScanArgs& a) {
  if (a.dtype < 0 || a.dtype > 2 || a.C < 1 || a.C > INB_MAX_MEMORY_C || a.N < 1 || a.N > INB_MAX_SCAN_N || a.S < 0 ||
      a.S > INB_MAX_MEMORY_S || a.T < 0 || a.T > INB_MAX_MEMORY_S || (a.reset.p != nullptr && (a.reset.rows < 1 || a.reset.rows > INB_MAX_MEMORY_S)))
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
  const int64_t tiles = ceil_div(a.C, 32 / LN), warps = tiles < SCAN_WARPS ? tiles : SCAN_WARPS;      // as scan_plan has them
  // nothing begins with what the last part (reverse: the first) ends with
  const dim3 grid((unsigned)(a.S * (MODE < 2 ? p.parts : p.parts - 1)), (unsigned)ceil_div(tiles, warps));
  if constexpr (NS == 16 && LN == 1) {
    if (a.N == 16 && is_aligned(a.b, 16, sizeof(T)) && is_aligned(a.c, 16, sizeof(T))) {
      scan_kernel<T, NS, LN, MODE, true><<<grid, (unsigned)warps * 32, 0, s>>>(a, p, carry);
      return;
    }
  }
  scan_kernel<T, NS, LN, MODE, false><<<grid, (unsigned)warps * 32, 0, s>>>(a, p, carry);
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
template <typename T, int V, int G>
static int step_go(const InbScanArgs& a, int lanes, cudaStream_t s) {
  int chans = STEP_THREADS / lanes;
  while (chans / 2 >= a.C && chans * lanes > 32) chans /= 2;      // a warp is one sequence's
  const int64_t tiles = ceil_div(a.C, chans), runs = STEP_THREADS / (lanes * chans);
  // as many times as leave six blocks an SM, no more than 32, and a grid's second axis ends at 65535
  int64_t per = a.S * tiles / (sm_count() * 6 * runs);
  if (per > 32) per = 32;
  if (per > 1) per = ceil_div(per, STEP_B) * STEP_B;
  if (per < ceil_div(a.S, 65535 * runs)) per = ceil_div(a.S, 65535 * runs);
  if (per < 1) per = 1;
  const auto kernel = runs > 1 ? scan_step_kernel<T, V, G, true> : scan_step_kernel<T, V, G, false>;
  kernel<<<dim3((unsigned)tiles, (unsigned)ceil_div(a.S, per * runs)), STEP_THREADS, 0, s>>>(a, lanes, chans, (int)per);
  return launch_status();
}
template <typename T>
static int scan_step(const InbScanArgs& a, cudaStream_t s) {
  const uint64_t m = (uint64_t)(uintptr_t)a.state | (uint64_t)(uintptr_t)a.state_out | (uint64_t)(a.state_seq * 4) |
                     (uint64_t)(a.state_out_seq * 4) | (uint64_t)(a.N * 4);
  int lanes = 1;
  if ((m & 15) == 0 && is_aligned(a.b, 4 * sizeof(T), sizeof(T)) && is_aligned(a.c, 4 * sizeof(T), sizeof(T))) {
    // eight states a thread, so that what is a channel's (delta, the gate) is computed by N / 8 threads
    while (lanes < 8 && lanes * 8 < a.N) lanes *= 2;
    return a.N <= 4 ? step_go<T, 4, 1>(a, 1, s) : step_go<T, 4, 2>(a, lanes, s);
  }
  while (lanes < 16 && lanes * 4 < a.N) lanes *= 2;
  return step_go<T, 1, 4>(a, lanes, s);
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
  if (((uintptr_t)a.kept & 15) != 0 || ((uintptr_t)a.work & 15) != 0) return -3;
  if (a.T == 1) {
    if (a.dtype == INB_BF16) return scan_step<bf16>(a, s);
    if (a.dtype == INB_F16) return scan_step<f16>(a, s);
    return scan_step<float>(a, s);
  }
  const ScanPlan p = scan_plan(a);
  if (p.split() && (a.work == nullptr || a.work_elems < scan_carry_elems(a, p))) return -5;
  return scan_launch(a, p, a.work, 0, s);
}
