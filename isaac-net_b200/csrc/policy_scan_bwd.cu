// selective_scan's backward pass.  With g = gy silu(z), u = delta x, e = exp(delta a):
//
//   dh[t] = c[t] g[t] + e[t + 1] dh[t + 1]            (0 instead of the second term where t + 1 starts an episode)
//   gb[t, n] = sum_c dh u     gc[t, n] = sum_c h g     ga[c, n] = sum_t delta dh e h[t - 1]
//   s1 = sum_n dh b           w = sum_n a dh e h[t - 1]
//   gx = s1 delta + d g       gdt = (w + s1 x) / (1 + exp(-(dt + dt_bias)))     gz = gy silu'(z) (sum_n c h + d x)
//
// The forward pass kept the state before every SCAN_STEPS steps; a warp runs those steps forward again from there, with
// every state in shared memory, then backward.  A thread holds 4 states of 2 neighbouring channels.  gb and gc are added over
// the block's warps in shared memory and over blocks by a further launch, ga, gd, gdt_bias stay in registers over all the
// tasks of a block: no atomics.
#include "policy_scan.cuh"

namespace inb {
namespace pol {

template <int LN>
struct BwdShape {
  static constexpr int TC = SCAN_STEPS, NP = 4 * LN, CW = 64 / LN;  // channels a warp
  static constexpr int G = 32 / LN, G4 = CW / 4;                    // its groups of 2 channels (a lane's) and of 4 (staging, gradients)
  static constexpr int SLOTS = 2, LINE = 33;                        // float4 a lane and step: its states, then its parts of gb and gc
  static constexpr int H = TC * SLOTS * LINE * 4, CH = TC * CW;
  static constexpr int USED = H + 6 * CH, PAD = (40 - USED % 32) % 32;      // warps 8 floats apart in the banks
  static constexpr int WARP = USED + PAD;                           // floats of shared memory a warp
  static constexpr int BC = TC * NP * 2, BLOCK = 2 * BC;            // and a block: b and c, twice each
  static constexpr int LEAST = LN > 4 ? LN / 4 : 1;                 // warps a block, so that a thread loads no more than
  static constexpr int BCN = (2 * TC * NP + LEAST * 32 - 1) / (LEAST * 32);        // these of b and c
  static constexpr int STEP = 32 / G4, ITEMS = (TC + STEP - 1) / STEP;      // (step, group of 4) pairs: lane / G4 + k STEP, lane % G4
};

// A chunk of SCAN_STEPS steps of a task (a part of a sequence), the task's last one first
struct Chunk {
  int64_t task, s, part, t0, t1, t;
  int steps;
  __device__ void set() { steps = t1 - t < SCAN_STEPS ? (int)(t1 - t) : SCAN_STEPS; }
  __device__ void start(const InbScanArgs& a, const ScanPlan& pl) {
    part = pl.parts > 1 ? task / a.S : 0, s = task - part * a.S;
    t0 = part * pl.len, t1 = t0 + pl.len < a.T ? t0 + pl.len : a.T;
    t = t0 + (t1 - t0 - 1) / SCAN_STEPS * SCAN_STEPS;
    set();
  }
  __device__ bool on(const InbScanArgs& a, const ScanPlan& pl) const { return task < a.S * pl.parts; }
  __device__ void next(const InbScanArgs& a, const ScanPlan& pl) {
    if (t > t0) {
      t -= SCAN_STEPS;
      set();
    } else {
      task += gridDim.x;
      if (on(a, pl)) start(a, pl);
    }
  }
  __device__ bool newest() const { return t + SCAN_STEPS >= t1; }
  __device__ bool oldest() const { return t == t0; }
};

// Bound by instruction issue: some 270 warp instructions for 8 states a thread and step, of which 60 are packed multiplications and
// additions and 20 exponentials; next to that by the exponentials (160 of a step's 280 issue cycles).  1024 x 32 sequences of
// 16 steps, 128 channels, N = 16: 1750 us, of a pass of 2265 us (860 GB/s).  16 warps an SM (128 registers, 12 KB of shared
// memory a warp) cover their latency: with twice the states a thread, and so half the warps, the same work took 1750 to 2050
// us.  A chunk's inputs are loaded a
// chunk ahead.  What is summed over lanes: over a channel's LN by shuffles (s1, w, y), over channels (gb, gc) once a chunk
// through shared memory, where a lane leaves its parts in place of its states.
// VEC: rows of x, dt, z, gy and their gradients, d and dt_bias are moved four channels at a time (aligned, C a multiple of 4)
template <typename T, int LN, bool VEC>
__global__ void __launch_bounds__(256, 2) scan_bwd_kernel(InbScanArgs a, ScanPlan pl, const float* carry, float* part_bc,
                                                          float* part_par) {
  using S = BwdShape<LN>;
  constexpr int TC = S::TC, NP = S::NP, CW = S::CW, G = S::G, G4 = S::G4, ITEMS = S::ITEMS, SLOTS = S::SLOTS, LINE = S::LINE;
  extern __shared__ float4 smem4[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int j = lane % LN, gr = lane / LN;
  float *sB = (float*)smem4, *sC = sB + S::BC;
  float* base = sB + S::BLOCK + warp * S::WARP;
  float4* H = (float4*)base;
  float *sD = base + S::H, *sX = sD + S::CH, *sG = sX + S::CH, *sQ = sG + S::CH;      // sQ: s1, w, y of the chunk's steps
  const int c0 = (blockIdx.y * warps + warp) * CW, n4 = (a.N + 3) / 4 * 4;
  const int64_t chunks = (a.T + TC - 1) / TC;
  const bool gate = a.z.p != nullptr;
  // the channels whose inputs this lane stages and whose gradients it writes, and the step of its first item
  const int mine = c0 + lane % G4 * 4, step0 = lane / G4;
  const int many = a.C - mine < 4 ? (a.C - mine > 0 ? a.C - mine : 0) : 4;
  // this thread's two channels as a pair, state n of its four; 0 beyond the last channel and state
  const int ch0 = c0 + gr * 2;
  float2 A[4], dA[4], r[4], h[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const bool in = j * 4 + n < a.N;
    A[n].x = in && ch0 < a.C ? a.a[ch0 * a.N + j * 4 + n] * LOG2E : 0.f;
    A[n].y = in && ch0 + 1 < a.C ? a.a[(ch0 + 1) * a.N + j * 4 + n] * LOG2E : 0.f;
    dA[n] = r[n] = make_float2(0.f, 0.f);
  }
  float gd[4], gbias[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) gd[c] = gbias[c] = 0.f;
  auto per_channel = [&](const float* p, float (&v)[4]) {
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC && p != nullptr && many == 4) f = *reinterpret_cast<const float4*>(p + mine);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    if (!VEC && p != nullptr) {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = p[mine + c < a.C ? mine + c : a.C - 1];
    }
  };
  // a chunk's inputs as they lie in memory; beyond the channels and the states the last one is read again, and made 0 where
  // that matters
  using Four = Words<T, 4>;
  struct Raw {
    Four v;             // VEC
    uint32_t e[4];
    __device__ __forceinline__ float f(int c) const {
      if constexpr (!VEC) return raw_f<T>(e[c]);
      const float2 p = v.pair(c / 2);
      return c & 1 ? p.y : p.x;
    }
  };
  Raw rx[ITEMS], rd[ITEMS], rz[ITEMS], rg[ITEMS];
  constexpr int BCN = S::BCN;
  uint32_t rb[BCN], flag = 0, bits;
  float4 rh[2];
  const int chl = many == 4 ? mine : a.C - 4;
  auto four = [&](Raw& q, const T* p) {
    if constexpr (VEC) {
      q.v.load(p + chl);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) q.e[c] = ld_raw(p + (mine + c < a.C ? mine + c : a.C - 1));
    }
  };
  const bool flat = a.N % 4 == 0 && (((uintptr_t)a.state | (a.state_seq * 4)) & 15) == 0;      // the state's rows lie as the kept ones do
  const float* zero = nullptr;
  auto load = [&](const Chunk& q) {
    const T *px = row<T>(a.x, q.s, q.t), *pd = row<T>(a.dt, q.s, q.t), *pg = row<T>(a.gy, q.s, q.t);
    const T* pz = gate ? row<T>(a.z, q.s, q.t) : nullptr;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int t = step0 + i * S::STEP;
      if (t >= q.steps) continue;
      four(rx[i], px + t * a.x.step), four(rd[i], pd + t * a.dt.step), four(rg[i], pg + t * a.gy.step);
      if (gate) four(rz[i], pz + t * a.z.step);
    }
    const T *pb = row<T>(a.b, q.s, q.t), *pc = row<T>(a.c, q.s, q.t);
#pragma unroll
    for (int i = 0; i < BCN; ++i) {
      const int k = i * blockDim.x + threadIdx.x;
      if (k >= 2 * TC * NP) break;
      const int which = k / (TC * NP), tt = k % (TC * NP) / NP, n = k % NP;
      const int tl = tt < q.steps ? tt : q.steps - 1, nl = n < a.N ? n : a.N - 1;
      rb[i] = ld_raw(which ? pc + (tl * a.c.step + nl) : pb + (tl * a.b.step + nl));
    }
    const float* from = q.t > 0 ? a.kept + (q.s * (chunks - 1) + q.t / TC - 1) * a.C * n4
                                : flat && a.state != nullptr ? a.state + q.s * a.state_seq : zero;
    if (from != nullptr) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
        rh[c] = *reinterpret_cast<const float4*>(from + ((ch0 + c < a.C ? ch0 + c : a.C - 1) * n4 + (j * 4 < n4 ? j * 4 : 0)));
    } else {
      const float* p = a.state != nullptr ? a.state + q.s * a.state_seq : nullptr;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float v[4] = {};
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (p != nullptr && ch0 + c < a.C && j * 4 + n < a.N) v[n] = p[(ch0 + c) * a.N + j * 4 + n];
        rh[c] = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    const uint8_t* rs = resets(a.reset, q.s);
    flag = reset_flag(rs != nullptr ? rs + q.t * a.reset.step : nullptr, a.reset.step, q.steps, lane);
  };
  // 2^subs threads for four states of a step and of gb or gc
  int subs = 0;
  while (subs < 3 && TC * 2 * LN << (subs + 1) <= (int)blockDim.x) ++subs;
  Chunk q;
  q.task = blockIdx.x;
  q.start(a, pl);
  load(q);
  while (q.on(a, pl)) {
    __syncwarp();
    float gz[ITEMS][4], slope[ITEMS][4], bias[4];
    per_channel(a.dt_bias, bias);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int t = step0 + i * S::STEP;
      if (t >= TC) continue;
      float x[4], delta[4], g[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[c] = c < many ? rx[i].f(c) : 0.f, g[c] = c < many ? rg[i].f(c) : 0.f;
        delta[c] = softplus(rd[i].f(c) + bias[c], slope[i][c]);
        if (gate) {
          const float z = rz[i].f(c), w = sigmoid(z);
          gz[i][c] = g[c] * w * fmaf(z, 1.f - w, 1.f);
          g[c] *= z * w;
        }
      }
      const int o = t * CW + lane % G4 * 4;
      *(float4*)(sX + o) = make_float4(x[0], x[1], x[2], x[3]);
      *(float4*)(sD + o) = make_float4(delta[0], delta[1], delta[2], delta[3]);
      *(float4*)(sG + o) = make_float4(g[0], g[1], g[2], g[3]);
    }
#pragma unroll
    for (int i = 0; i < BCN; ++i) {
      const int k = i * blockDim.x + threadIdx.x;
      if (k >= 2 * TC * NP) break;
      *reinterpret_cast<float2*>(sB + 2 * k) = both(k % NP < a.N ? raw_f<T>(rb[i]) : 0.f);
    }
    {
      const bool in = j * 4 < n4, in0 = in && ch0 < a.C, in1 = in && ch0 + 1 < a.C;
      h[0] = make_float2(in0 ? rh[0].x : 0.f, in1 ? rh[1].x : 0.f), h[1] = make_float2(in0 ? rh[0].y : 0.f, in1 ? rh[1].y : 0.f);
      h[2] = make_float2(in0 ? rh[0].z : 0.f, in1 ? rh[1].z : 0.f), h[3] = make_float2(in0 ? rh[0].w : 0.f, in1 ? rh[1].w : 0.f);
    }
    bits = __ballot_sync(0xFFFFFFFFu, flag != 0);
    const Chunk now = q;
    const int steps = now.steps;
    q.next(a, pl);
    if (q.on(a, pl)) load(q);
    if (now.newest()) {              // the gradient that reaches the task's last state from later steps
#pragma unroll
      for (int n = 0; n < 4; ++n) r[n] = make_float2(0.f, 0.f);
      const float* from = pl.parts > 1 ? carry + (now.s * pl.parts + now.part) * a.C * n4
                                       : a.gstate_out != nullptr ? a.gstate_out + now.s * a.C * a.N : nullptr;
      if (from != nullptr) {
        const int ld = pl.parts > 1 ? n4 : a.N;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const bool in = j * 4 + n < a.N;
          r[n].x = in && ch0 < a.C ? from[ch0 * ld + j * 4 + n] : 0.f;
          r[n].y = in && ch0 + 1 < a.C ? from[(ch0 + 1) * ld + j * 4 + n] : 0.f;
        }
      }
    }
    __syncthreads();                 // this chunk is staged, and the block has read the parts of the one before
    // forward again: the state before each step
#pragma unroll 4
    for (int i = 0; i < steps; ++i) {
      if (bits >> i & 1) {
#pragma unroll
        for (int n = 0; n < 4; ++n) h[n] = make_float2(0.f, 0.f);
        keep_branch();
      }
      H[i * SLOTS * LINE + lane] = make_float4(h[0].x, h[0].y, h[1].x, h[1].y);
      H[(i * SLOTS + 1) * LINE + lane] = make_float4(h[2].x, h[2].y, h[3].x, h[3].y);
      if (i + 1 == steps) break;
      const float2 D = *(const float2*)(sD + i * CW + gr * 2), U = mul2(D, *(const float2*)(sX + i * CW + gr * 2));
      const float4 *B4 = (const float4*)(sB + (i * NP + j * 4) * 2), B0 = B4[0], B1 = B4[1];
      const float2 B[4] = {make_float2(B0.x, B0.y), make_float2(B0.z, B0.w), make_float2(B1.x, B1.y), make_float2(B1.z, B1.w)};
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float2 v = mul2(D, A[n]);
        h[n] = fma2(make_float2(ex2(v.x), ex2(v.y)), h[n], mul2(U, B[n]));
      }
    }
    float2 delta = make_float2(0.f, 0.f);      // the chunk's sum
#pragma unroll 4
    for (int i = steps - 1; i >= 0; --i) {
      const float2 D = *(const float2*)(sD + i * CW + gr * 2), U = mul2(D, *(const float2*)(sX + i * CW + gr * 2));
      const float2 GG = *(const float2*)(sG + i * CW + gr * 2);
      delta = add2(delta, D);
      const float4 *B4 = (const float4*)(sB + (i * NP + j * 4) * 2), B0 = B4[0], B1 = B4[1];
      const float4 *C4 = (const float4*)(sC + (i * NP + j * 4) * 2), C0 = C4[0], C1 = C4[1];
      const float2 B[4] = {make_float2(B0.x, B0.y), make_float2(B0.z, B0.w), make_float2(B1.x, B1.y), make_float2(B1.z, B1.w)};
      const float2 C[4] = {make_float2(C0.x, C0.y), make_float2(C0.z, C0.w), make_float2(C1.x, C1.y), make_float2(C1.z, C1.w)};
      float4* at = H + i * SLOTS * LINE + lane;
      const float4 P0 = at[0], P1 = at[LINE];
      const float2 P[4] = {make_float2(P0.x, P0.y), make_float2(P0.z, P0.w), make_float2(P1.x, P1.y), make_float2(P1.z, P1.w)};
      float gb[4], gc[4];
      float2 s1, w, yp;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float2 v = mul2(D, A[n]), e = make_float2(ex2(v.x), ex2(v.y));
        const float2 eh = mul2(e, P[n]), hh = fma2(U, B[n], eh), dh = fma2(C[n], GG, r[n]), f = mul2(dh, eh);
        const float2 pc = mul2(GG, hh), pb = mul2(U, dh);
        gc[n] = pc.x + pc.y, gb[n] = pb.x + pb.y;
        yp = n ? fma2(C[n], hh, yp) : mul2(C[n], hh);
        s1 = n ? fma2(B[n], dh, s1) : mul2(B[n], dh);
        w = n ? fma2(A[n], f, w) : mul2(A[n], f);
        dA[n] = fma2(D, f, dA[n]);
        r[n] = mul2(e, dh);
      }
      if (bits >> i & 1) {
#pragma unroll
        for (int n = 0; n < 4; ++n) r[n] = make_float2(0.f, 0.f);
        keep_branch();
      }
      // this lane's parts, in place of the states that it alone has read
      at[0] = make_float4(gb[0], gb[1], gb[2], gb[3]);
      at[LINE] = make_float4(gc[0], gc[1], gc[2], gc[3]);
      // over the channel's lanes: the upper half of them takes the second channel
      if constexpr (LN == 1) {
        *(float2*)(sQ + i * CW + gr * 2) = s1;
        *(float2*)(sQ + S::CH + i * CW + gr * 2) = w;
        *(float2*)(sQ + 2 * S::CH + i * CW + gr * 2) = yp;
      } else {
        const bool up = j >= LN / 2;
        auto sum = [&](float2 v) {
          float o = (up ? v.y : v.x) + __shfl_xor_sync(0xFFFFFFFFu, up ? v.x : v.y, LN / 2);
#pragma unroll
          for (int m = LN / 4; m > 0; m /= 2) o += __shfl_xor_sync(0xFFFFFFFFu, o, m);
          return o;
        };
        const float s1s = sum(s1), ws = sum(w), ys = gate ? sum(yp) : 0.f;
        if (j % (LN / 2) == 0) {
          float* to = sQ + i * CW + gr * 2 + up;
          to[0] = s1s, to[S::CH] = ws, to[2 * S::CH] = ys;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) r[n] = unbias(r[n], A[n], delta);
    if (now.oldest() && now.part == 0 && a.gstate != nullptr) {
      float* to = a.gstate + now.s * a.C * a.N + (ch0 * a.N + j * 4);
      if (a.N % 4 == 0 && ((uintptr_t)a.gstate & 15) == 0) {
        if (j * 4 < a.N && ch0 < a.C) *reinterpret_cast<float4*>(to) = make_float4(r[0].x, r[1].x, r[2].x, r[3].x);
        if (j * 4 < a.N && ch0 + 1 < a.C) *reinterpret_cast<float4*>(to + a.N) = make_float4(r[0].y, r[1].y, r[2].y, r[3].y);
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (j * 4 + n < a.N) {
            if (ch0 < a.C) to[n] = r[n].x;
            if (ch0 + 1 < a.C) to[a.N + n] = r[n].y;
          }
      }
    }
    __syncthreads();
    // gx, gdt, gz
    T *qx = row_out<T>(a.gx, now.s, now.t), *qd = row_out<T>(a.gdt, now.s, now.t);
    T* qz = gate ? row_out<T>(a.gz, now.s, now.t) : nullptr;
    float dd[4];
    per_channel(a.d, dd);
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int t = step0 + i * S::STEP;
      if (t >= steps || many == 0) continue;
      const int o = t * CW + lane % G4 * 4;
      const float4 s4 = *(const float4*)(sQ + o), w4 = *(const float4*)(sQ + S::CH + o), y4 = *(const float4*)(sQ + 2 * S::CH + o);
      const float4 x4 = *(const float4*)(sX + o), d4 = *(const float4*)(sD + o), g4 = *(const float4*)(sG + o);
      const float x[4] = {x4.x, x4.y, x4.z, x4.w}, delta[4] = {d4.x, d4.y, d4.z, d4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w};
      const float s1[4] = {s4.x, s4.y, s4.z, s4.w}, w[4] = {w4.x, w4.y, w4.z, w4.w}, yp[4] = {y4.x, y4.y, y4.z, y4.w};
      float ox[4], od[4], oz[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        od[c] = fmaf(LN2, w[c], s1[c] * x[c]) * slope[i][c];
        gd[c] = fmaf(g[c], x[c], gd[c]);
        gbias[c] += od[c];
        ox[c] = fmaf(s1[c], delta[c], dd[c] * g[c]);
        oz[c] = gate ? gz[i][c] * fmaf(dd[c], x[c], yp[c]) : 0.f;
      }
      auto put = [&](T* p, const float (&v)[4]) {
        if constexpr (VEC) {
          Four q;
          q.set(0, make_float2(v[0], v[1]));
          q.set(1, make_float2(v[2], v[3]));
          q.store(p);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < many) p[c] = from_f<T>(v[c]);
        }
      };
      put(qx + t * a.gx.step + mine, ox);
      put(qd + t * a.gdt.step + mine, od);
      if (gate) put(qz + t * a.gz.step + mine, oz);
    }
    // gb and gc: over the groups of every warp
    const int total = steps * 2 * LN << subs;
    for (int i0 = 0; i0 < total; i0 += blockDim.x) {
      const int i = i0 + threadIdx.x, o = i < total ? i >> subs : 0;
      const int t = o / (2 * LN), which = o / LN % 2, jj = o % LN;
      const float4* from = (const float4*)(sB + S::BLOCK) + (t * SLOTS + which) * LINE + jj;
      float2 v0 = make_float2(0.f, 0.f), v1 = v0;
      for (int k = i & (1 << subs) - 1; k < warps; k += 1 << subs) {
#pragma unroll
        for (int m = 0; m < G; ++m) {
          const float4 p = from[k * (S::WARP / 4) + m * LN];
          v0 = add2(v0, make_float2(p.x, p.y)), v1 = add2(v1, make_float2(p.z, p.w));
        }
      }
      float v[4] = {v0.x, v0.y, v1.x, v1.y};
      for (int m = 1; m < 1 << subs; m *= 2)
#pragma unroll
        for (int n = 0; n < 4; ++n) v[n] += __shfl_xor_sync(0xFFFFFFFFu, v[n], m);
      if (i >= total || (i & (1 << subs) - 1) != 0) continue;
      if (part_bc != nullptr) {
        float* to = part_bc + (((int64_t)blockIdx.y * a.S + now.s) * a.T + now.t + t) * 2 * a.N + which * a.N + jj * 4;
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (jj * 4 + n < a.N) to[n] = v[n];
      } else {
        T* to = row_out<T>(which ? a.gc : a.gb, now.s, now.t + t) + jj * 4;
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (jj * 4 + n < a.N) to[n] = from_f<T>(v[n]);
      }
    }
  }
  float* out = part_par + (int64_t)blockIdx.x * a.C * (a.N + 2);
#pragma unroll
  for (int n = 0; n < 4; ++n)
    if (j * 4 + n < a.N) {
      if (ch0 < a.C) out[(int64_t)ch0 * a.N + j * 4 + n] = dA[n].x;
      if (ch0 + 1 < a.C) out[(int64_t)(ch0 + 1) * a.N + j * 4 + n] = dA[n].y;
    }
  // the lanes that wrote other steps of the same channels
#pragma unroll
  for (int m = G4; m < 32; m *= 2)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      gd[c] += __shfl_xor_sync(0xFFFFFFFFu, gd[c], m);
      gbias[c] += __shfl_xor_sync(0xFFFFFFFFu, gbias[c], m);
    }
  if (lane < G4)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < many) {
        out[(int64_t)a.C * a.N + mine + c] = gd[c];
        out[(int64_t)a.C * (a.N + 1) + mine + c] = gbias[c];
      }
}

// gb and gc from the blocks' parts [P, S, T, 2 N]
template <typename T>
__global__ void __launch_bounds__(256) scan_bc_kernel(InbScanArgs a, const float* part, int P) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = a.S * a.T * 2 * a.N;
  if (i >= m) return;
  float v = 0.f;
  for (int p = 0; p < P; ++p) v += part[p * m + i];
  const int64_t st = i / (2 * a.N), s = st / a.T, t = st - s * a.T;
  const int n = (int)(i - st * 2 * a.N);
  if (n < a.N)
    row_out<T>(a.gb, s, t)[n] = from_f<T>(v);
  else
    row_out<T>(a.gc, s, t)[n - a.N] = from_f<T>(v);
}

struct BwdPlan {
  ScanPlan plan;
  int lanes, warps, tiles, blocks, smem;       // tiles: blocks over the channels
  int64_t carry, bc, par;                      // floats of scratch
};
template <int LN>
static void bwd_shape(BwdPlan& b, int64_t C) {
  using S = BwdShape<LN>;
  const int64_t all = ceil_div(C, S::CW);
  // 8 warps a block; of N = 5 to 8 that leaves shared memory for one block an SM, 7 warps for two (256 sequences of 300 steps of 512
  // channels, N = 8, forward + backward: 1035 us against 1091).  Of N <= 4 two blocks of 5 are no faster (1789 us against 1717).
  constexpr int most = LN == 2 ? 7 : 8;
  b.tiles = (int)ceil_div(all, most);
  b.warps = (int)ceil_div(all, b.tiles);
  if (b.warps < S::LEAST) b.warps = S::LEAST;
  b.smem = (S::BLOCK + b.warps * S::WARP) * 4;
}
static BwdPlan bwd_plan(const InbScanArgs& a) {
  BwdPlan b;
  b.lanes = a.N <= 4 ? 1 : a.N <= 8 ? 2 : a.N <= 16 ? 4 : a.N <= 32 ? 8 : 16;
  if (b.lanes == 1) bwd_shape<1>(b, a.C);
  if (b.lanes == 2) bwd_shape<2>(b, a.C);
  if (b.lanes == 4) bwd_shape<4>(b, a.C);
  if (b.lanes == 8) bwd_shape<8>(b, a.C);
  if (b.lanes == 16) bwd_shape<16>(b, a.C);
  int64_t fit = 227 * 1024 / (b.smem + 1024);
  if (fit > 16 / b.warps) fit = 16 / b.warps;                      // registers
  int64_t blocks = sm_count() * fit / b.tiles;
  if (blocks < 1) blocks = 1;
  b.plan = scan_split(a.T, a.S, blocks, 5);
  const int64_t tasks = a.S * b.plan.parts;
  b.blocks = (int)(blocks < tasks ? blocks : tasks);
  b.carry = (scan_carry_elems(a, b.plan) + 3) / 4 * 4;
  b.bc = b.tiles > 1 ? b.tiles * a.S * a.T * 2 * a.N : 0;
  b.par = (int64_t)b.blocks * a.C * (a.N + 2);
  return b;
}
template <typename T, int LN, bool VEC>
static int bwd_launch(const InbScanArgs& a, const BwdPlan& b, const float* carry, float* bc, float* par, cudaStream_t s) {
  constexpr auto kernel = scan_bwd_kernel<T, LN, VEC>;
  const cudaError_t e = allow_smem<KernelKey<scan_bwd_kernel<T, LN, VEC>>>((const void*)kernel, (BwdShape<LN>::BLOCK + 8 * BwdShape<LN>::WARP) * 4);
  if (e != cudaSuccess) return -100 - (int)e;
  kernel<<<dim3(b.blocks, b.tiles), b.warps * 32, b.smem, s>>>(a, b.plan, carry, b.bc > 0 ? bc : nullptr, par);
  return 0;
}
template <typename T, int LN>
static int bwd_go(const InbScanArgs& a, const BwdPlan& b, cudaStream_t s) {
  float *carry = a.work, *bc = carry + b.carry, *par = bc + b.bc;
  int rc = b.plan.split() ? scan_launch(a, b.plan, carry, 3, s) : 0;
  if (rc != 0) return rc;
  bool vec = a.C % 4 == 0;
  for (const InbSeq& q : {a.x, a.dt, a.z, a.gy, a.gx, a.gdt, a.gz}) vec = vec && is_aligned(q, 4 * sizeof(T), sizeof(T));
  vec = vec && (((uintptr_t)a.d | (uintptr_t)a.dt_bias) & 15) == 0;
  rc = vec ? bwd_launch<T, LN, true>(a, b, carry, bc, par, s) : bwd_launch<T, LN, false>(a, b, carry, bc, par, s);
  if (rc != 0) return rc;
  if (b.bc > 0) scan_bc_kernel<T><<<(unsigned)ceil_div(a.S * a.T * 2 * a.N, 256), 256, 0, s>>>(a, bc, b.tiles);
  colsum<float>(par, b.blocks, (int64_t)a.C * (a.N + 2), (int64_t)a.C * a.N, (int64_t)a.C * (a.N + 1), a.ga, a.gd, a.gdt_bias, s);
  return launch_status();
}
template <typename T>
static int bwd_type(const InbScanArgs& a, const BwdPlan& b, cudaStream_t s) {
  switch (b.lanes) {
    case 1: return bwd_go<T, 1>(a, b, s);
    case 2: return bwd_go<T, 2>(a, b, s);
    case 4: return bwd_go<T, 4>(a, b, s);
    case 8: return bwd_go<T, 8>(a, b, s);
    default: return bwd_go<T, 16>(a, b, s);
  }
}

}  // namespace pol
}  // namespace inb

using namespace inb::pol;

extern "C" int inb_selective_scan_work(const InbScanArgs* args, int32_t backward, int64_t* elems) {
  if (args == nullptr || elems == nullptr) return -1;
  const InbScanArgs& a = *args;
  const int rc = scan_check(a);
  if (rc != 0) return rc;
  *elems = 0;
  if (a.S == 0 || a.T == 0) return 0;
  if (backward) {
    const BwdPlan b = bwd_plan(a);
    *elems = b.carry + b.bc + b.par;
  } else if (a.T > 1) {
    *elems = scan_carry_elems(a, scan_plan(a));
  }
  return 0;
}

extern "C" int inb_selective_scan_bwd(const InbScanArgs* args, void* cuda_stream) {
  int64_t need = 0;
  const int rc = inb_selective_scan_work(args, 1, &need);
  if (rc != 0) return rc;
  const InbScanArgs& a = *args;
  if (a.S == 0 || a.T == 0) return 0;
  if (a.x.p == nullptr || a.dt.p == nullptr || a.b.p == nullptr || a.c.p == nullptr || a.a == nullptr || a.gy.p == nullptr ||
      a.gx.p == nullptr || a.gdt.p == nullptr || a.gb.p == nullptr || a.gc.p == nullptr || a.ga == nullptr ||
      (a.z.p != nullptr && a.gz.p == nullptr) || (a.T > SCAN_STEPS && a.kept == nullptr) || ((uintptr_t)a.kept & 15) != 0 ||
      ((uintptr_t)a.work & 15) != 0)
    return -3;
  if (a.work == nullptr || a.work_elems < need) return -5;
  const BwdPlan b = bwd_plan(a);
  if (a.dtype == INB_BF16) return bwd_type<bf16>(a, b, (cudaStream_t)cuda_stream);
  if (a.dtype == INB_F16) return bwd_type<f16>(a, b, (cudaStream_t)cuda_stream);
  return bwd_type<float>(a, b, (cudaStream_t)cuda_stream);
}
