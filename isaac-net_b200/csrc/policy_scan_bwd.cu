// selective_scan's backward pass.  With g = gy silu(z), u = delta x, e = exp(delta a):
//
//   dh[t] = c[t] g[t] + e[t + 1] dh[t + 1]            (0 instead of the second term where t + 1 starts an episode)
//   gb[t, n] = sum_c dh u     gc[t, n] = sum_c h g     ga[c, n] = sum_t delta dh e h[t - 1]
//   s1 = sum_n dh b           w = sum_n a dh e h[t - 1]
//   gx = s1 delta + d g       gdt = (w + s1 x) / (1 + exp(-(dt + dt_bias)))     gz = gy silu'(z) (sum_n c h + d x)
//
// The forward pass kept the state before every SCAN_STEPS steps; a warp runs those steps forward again from there, with
// every state in shared memory, then backward.  A thread holds 4 states of 4 neighbouring channels, so that sums over channels
// (gb, gc) and over states (s1, w, y) leave it as 20 parts a step where a channel a thread would leave 32.  gb and gc are added
// over the block's warps in shared memory and over blocks by a further launch, ga, gd, gdt_bias stay in registers over all
// the tasks of a block: no atomics.
#include "policy_scan.cuh"

namespace inb {
namespace pol {

template <int LN>
struct BwdShape {
  static constexpr int TC = SCAN_STEPS, NP = 4 * LN, CW = 128 / LN, G = 32 / LN;       // G: groups of 4 channels
  static constexpr int SLOTS = 5;                                   // float4 a lane and step: states, then partial sums
  static constexpr int LINE = 33;                                   // float4 from slot to slot: one more than lanes, for the banks
  static constexpr int H = TC * SLOTS * LINE * 4, CH = TC * CW, BC = TC * NP * 2;
  static constexpr int WARP = H + 3 * CH + 2 * BC;                  // floats of shared memory a warp
  static constexpr int STEP = 32 / G, ITEMS = (TC + STEP - 1) / STEP;       // (step, group) pairs: lane / G + k STEP, lane % G
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

// Bound by issue and by the exponentials together: of a step's 300 warp instructions for 16 states a thread 120 are packed
// multiplications and additions and 36 exponentials, which take 8 cycles each.  The sums over lanes go through shared memory
// once a chunk: a lane leaves its parts where its states were, and one lane adds four channels' of a step.  Shared memory
// (25 KB a warp, of it 20 for states and parts) leaves 8 warps an SM, so a chunk's inputs are loaded a chunk ahead.
// VEC: rows of x, dt, z, gy and their gradients are moved four channels at a time (aligned, C a multiple of 4)
// WIDE: b and c have NP states whose rows are aligned to 16 bytes and moved by that
template <typename T, int LN, bool VEC, bool WIDE>
__global__ void __launch_bounds__(256, 1) scan_bwd_kernel(InbScanArgs a, ScanPlan pl, const float* carry, float* part_bc,
                                                          float* part_par) {
  using S = BwdShape<LN>;
  constexpr int TC = S::TC, NP = S::NP, CW = S::CW, G = S::G, BCL = TC * NP / 32, ITEMS = S::ITEMS, SLOTS = S::SLOTS,
                LINE = S::LINE, UNROLL = 2, BCW = 16 / sizeof(T);
  // words of b and c a lane loads: in all, and by 16 bytes
  constexpr int BCN = 2 * TC * NP / (32 * BCW) > 0 ? 2 * TC * NP / (32 * BCW) : 1;
  extern __shared__ float4 smem4[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int j = lane % LN, gr = lane / LN;
  float* base = (float*)smem4 + warp * S::WARP;
  float4* H = (float4*)base;
  float *sD = base + S::H, *sX = sD + S::CH, *sG = sX + S::CH, *sB = sG + S::CH, *sC = sB + S::BC;       // b and c twice each
  const int c0 = (blockIdx.y * warps + warp) * CW, n4 = (a.N + 3) / 4 * 4;
  const int64_t chunks = (a.T + TC - 1) / TC;
  const bool gate = a.z.p != nullptr;
  // the channels whose inputs this lane stages and whose gradients it writes, and the step of its first item
  const int mine = c0 + lane % G * 4, step0 = lane / G;
  const int many = a.C - mine < 4 ? (a.C - mine > 0 ? a.C - mine : 0) : 4;
  // pairs of channels (2 p, 2 p + 1) of this thread's four, state n of its four; 0 beyond the last channel and state
  float2 A[2][4], dA[2][4], r[2][4], h[2][4];
  auto at = [](float2 (&v)[2][4], int c, int n) -> float& { return c & 1 ? v[c / 2][n].y : v[c / 2][n].x; };
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int ch = c0 + gr * 4 + c;
      at(A, c, n) = ch < a.C && j * 4 + n < a.N ? a.a[ch * a.N + j * 4 + n] * LOG2E : 0.f;
      at(dA, c, n) = at(r, c, n) = 0.f;
    }
  float bias[4], dd[4], gd[4], gbias[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    bias[c] = c < many && a.dt_bias != nullptr ? a.dt_bias[mine + c] : 0.f;
    dd[c] = c < many && a.d != nullptr ? a.d[mine + c] : 0.f;
    gd[c] = gbias[c] = 0.f;
  }
  // a chunk's inputs as they lie in memory.  Loads have no condition: beyond the chunk's steps, the channels and the states
  // the last one is read again, and made 0 where that matters.
  using Four = Pack<T, 4>;
  struct Raw {
    Four v;             // VEC
    uint32_t e[4];
    __device__ float f(int c) const { return VEC ? to_f(v.v[c]) : raw_f<T>(e[c]); }
  };
  Raw rx[ITEMS], rd[ITEMS], rz[ITEMS], rg[ITEMS];
  uint32_t rb[WIDE ? 1 : BCL], rc[WIDE ? 1 : BCL], flag = 0, bits;
  Words<T, BCW> wide[WIDE ? BCN : 1];
  float4 rh[4];
  const int chl = VEC ? (many == 4 ? mine : a.C - 4) : 0;
  auto four = [&](Raw& r, const T* p) {
    if constexpr (VEC) {
      r.v = ld<T, 4>(p + chl);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) r.e[c] = ld_raw(p + (mine + c < a.C ? mine + c : a.C - 1));
    }
  };
  const bool flat = a.N % 4 == 0 && (((uintptr_t)a.state | (a.state_seq * 4)) & 15) == 0;      // the state's rows lie as the kept ones do
  const float* zero = nullptr;
  auto load = [&](const Chunk& q) {
    const T *px = row<T>(a.x, q.s, q.t), *pd = row<T>(a.dt, q.s, q.t), *pg = row<T>(a.gy, q.s, q.t);
    const T* pz = gate ? row<T>(a.z, q.s, q.t) : nullptr;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int t = step0 + i * S::STEP, tl = t < q.steps ? t : q.steps - 1;
      four(rx[i], px + tl * a.x.step), four(rd[i], pd + tl * a.dt.step), four(rg[i], pg + tl * a.gy.step);
      if (gate) four(rz[i], pz + tl * a.z.step);
    }
    const T *pb = row<T>(a.b, q.s, q.t), *pc = row<T>(a.c, q.s, q.t);
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < BCN; ++i) {
        const int k = (i * 32 + lane) * BCW, which = k / (TC * NP), tt = k % (TC * NP) / NP, n = k % NP;
        const int tl = tt < q.steps ? tt : q.steps - 1;
        wide[i].load(which ? pc + (tl * a.c.step + n) : pb + (tl * a.b.step + n));
      }
    } else {
#pragma unroll
    for (int i = 0; i < BCL; ++i) {
      const int tt = (i * 32 + lane) / NP, n = (i * 32 + lane) % NP;
      const int tl = tt < q.steps ? tt : q.steps - 1, nl = n < a.N ? n : a.N - 1;
      rb[i] = ld_raw(pb + (tl * a.b.step + nl)), rc[i] = ld_raw(pc + (tl * a.c.step + nl));
    }
    }
    const float* from = q.t > 0 ? a.kept + (q.s * (chunks - 1) + q.t / TC - 1) * a.C * n4
                                : flat && a.state != nullptr ? a.state + q.s * a.state_seq : zero;
    if (from != nullptr) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int ch = c0 + gr * 4 + c;
        rh[c] = *reinterpret_cast<const float4*>(from + ((ch < a.C ? ch : a.C - 1) * n4 + (j * 4 < n4 ? j * 4 : 0)));
      }
    } else {
      const float* p = a.state != nullptr ? a.state + q.s * a.state_seq : nullptr;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int ch = c0 + gr * 4 + c;
        float v[4] = {};
#pragma unroll
        for (int n = 0; n < 4; ++n)
          if (p != nullptr && ch < a.C && j * 4 + n < a.N) v[n] = p[ch * a.N + j * 4 + n];
        rh[c] = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    const uint8_t* rs = resets(a.reset, q.s);
    flag = reset_flag(rs != nullptr ? rs + q.t * a.reset.step : nullptr, a.reset.step, q.steps, lane);
  };
  Chunk q;
  q.task = blockIdx.x;
  q.start(a, pl);
  load(q);
  while (q.on(a, pl)) {
    __syncwarp();
    float gz[ITEMS][4], slope[ITEMS][4];
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
      const int o = t * CW + lane % G * 4;
      *(float4*)(sX + o) = make_float4(x[0], x[1], x[2], x[3]);
      *(float4*)(sD + o) = make_float4(delta[0], delta[1], delta[2], delta[3]);
      *(float4*)(sG + o) = make_float4(g[0], g[1], g[2], g[3]);
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < BCN; ++i) {
        const int k = (i * 32 + lane) * BCW, which = k / (TC * NP);
        float4* to = (float4*)((which ? sC : sB) + 2 * (k % (TC * NP)));
#pragma unroll
        for (int e = 0; e < BCW / 2; ++e) {
          const float2 p = wide[i].pair(e);
          to[e] = make_float4(p.x, p.x, p.y, p.y);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < BCL; ++i) {
        const bool in = (i * 32 + lane) % NP < a.N;
        *reinterpret_cast<float2*>(sB + 2 * (i * 32 + lane)) = both(in ? raw_f<T>(rb[i]) : 0.f);
        *reinterpret_cast<float2*>(sC + 2 * (i * 32 + lane)) = both(in ? raw_f<T>(rc[i]) : 0.f);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bool in = c0 + gr * 4 + c < a.C && j * 4 < n4;
      at(h, c, 0) = in ? rh[c].x : 0.f, at(h, c, 1) = in ? rh[c].y : 0.f, at(h, c, 2) = in ? rh[c].z : 0.f, at(h, c, 3) = in ? rh[c].w : 0.f;
    }
    bits = __ballot_sync(0xFFFFFFFFu, flag != 0);
    const Chunk now = q;
    const int steps = now.steps;
    q.next(a, pl);
    if (q.on(a, pl)) load(q);
    if (now.newest()) {              // the gradient that reaches the task's last state from later steps
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int ch = c0 + gr * 4 + c, k = j * 4 + n;
          float v = 0.f;
          if (ch < a.C && k < a.N) {
            if (pl.parts > 1)
              v = carry[((now.s * pl.parts + now.part) * a.C + ch) * n4 + k];
            else if (a.gstate_out != nullptr)
              v = a.gstate_out[(now.s * a.C + ch) * a.N + k];
          }
          at(r, c, n) = v;
        }
    }
    __syncthreads();                 // this chunk is staged, and the block has read the parts of the one before
    // forward again: the state before each step
#pragma unroll UNROLL
    for (int i = 0; i < TC; ++i) {
      if (i >= steps) break;
      if (bits >> i & 1) {
#pragma unroll
        for (int n = 0; n < 4; ++n) h[0][n] = h[1][n] = make_float2(0.f, 0.f);
        keep_branch();
      }
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int n = 0; n < 4; n += 2)
          H[(i * SLOTS + p * 2 + n / 2) * LINE + lane] = make_float4(h[p][n].x, h[p][n].y, h[p][n + 1].x, h[p][n + 1].y);
      if (i + 1 == steps) break;
      const float4 D4 = *(const float4*)(sD + i * CW + gr * 4), X4 = *(const float4*)(sX + i * CW + gr * 4);
      const float4 *B4 = (const float4*)(sB + (i * NP + j * 4) * 2), B0 = B4[0], B1 = B4[1];
      const float2 D[2] = {make_float2(D4.x, D4.y), make_float2(D4.z, D4.w)};
      const float2 U[2] = {mul2(D[0], make_float2(X4.x, X4.y)), mul2(D[1], make_float2(X4.z, X4.w))};
      const float2 B[4] = {make_float2(B0.x, B0.y), make_float2(B0.z, B0.w), make_float2(B1.x, B1.y), make_float2(B1.z, B1.w)};
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float2 v = mul2(D[p], A[p][n]);
          h[p][n] = fma2(make_float2(ex2(v.x), ex2(v.y)), h[p][n], mul2(U[p], B[n]));
        }
    }
#pragma unroll UNROLL
    for (int i = TC - 1; i >= 0; --i) {
      if (i >= steps) continue;
      const float4 D4 = *(const float4*)(sD + i * CW + gr * 4), X4 = *(const float4*)(sX + i * CW + gr * 4),
                   G4 = *(const float4*)(sG + i * CW + gr * 4);
      const float4 *B4 = (const float4*)(sB + (i * NP + j * 4) * 2), B0 = B4[0], B1 = B4[1];
      const float4 *C4 = (const float4*)(sC + (i * NP + j * 4) * 2), C0 = C4[0], C1 = C4[1];
      const float2 D[2] = {make_float2(D4.x, D4.y), make_float2(D4.z, D4.w)};
      const float2 U[2] = {mul2(D[0], make_float2(X4.x, X4.y)), mul2(D[1], make_float2(X4.z, X4.w))};
      const float2 GG[2] = {make_float2(G4.x, G4.y), make_float2(G4.z, G4.w)};
      const float2 B[4] = {make_float2(B0.x, B0.y), make_float2(B0.z, B0.w), make_float2(B1.x, B1.y), make_float2(B1.z, B1.w)};
      const float2 C[4] = {make_float2(C0.x, C0.y), make_float2(C0.z, C0.w), make_float2(C1.x, C1.y), make_float2(C1.z, C1.w)};
      float2 gb[4], gc[4], s1[2], w[2], yp[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float4 P4 = H[(i * SLOTS + p * 2 + n / 2) * LINE + lane];
          const float2 P = n & 1 ? make_float2(P4.z, P4.w) : make_float2(P4.x, P4.y);
          const float2 v = mul2(D[p], A[p][n]), e = make_float2(ex2(v.x), ex2(v.y));
          const float2 eh = mul2(e, P), hh = fma2(U[p], B[n], eh), dh = fma2(C[n], GG[p], r[p][n]), f = mul2(dh, eh);
          yp[p] = n ? fma2(C[n], hh, yp[p]) : mul2(C[n], hh);
          gc[n] = p ? fma2(GG[p], hh, gc[n]) : mul2(GG[p], hh);
          gb[n] = p ? fma2(U[p], dh, gb[n]) : mul2(U[p], dh);
          s1[p] = n ? fma2(B[n], dh, s1[p]) : mul2(B[n], dh);
          dA[p][n] = fma2(D[p], f, dA[p][n]);
          w[p] = n ? fma2(A[p][n], f, w[p]) : mul2(A[p][n], f);
          r[p][n] = mul2(e, dh);
        }
      }
      if (bits >> i & 1) {
#pragma unroll
        for (int n = 0; n < 4; ++n) r[0][n] = r[1][n] = make_float2(0.f, 0.f);
        keep_branch();
      }
      // this lane's parts, in place of the states that it alone has read
      float4* to = H + i * SLOTS * LINE + lane;
      to[0] = make_float4(gb[0].x + gb[0].y, gb[1].x + gb[1].y, gb[2].x + gb[2].y, gb[3].x + gb[3].y);
      to[LINE] = make_float4(gc[0].x + gc[0].y, gc[1].x + gc[1].y, gc[2].x + gc[2].y, gc[3].x + gc[3].y);
      to[2 * LINE] = make_float4(s1[0].x, s1[0].y, s1[1].x, s1[1].y);
      to[3 * LINE] = make_float4(w[0].x, w[0].y, w[1].x, w[1].y);
      if (gate) to[4 * LINE] = make_float4(yp[0].x, yp[0].y, yp[1].x, yp[1].y);
    }
    if (now.oldest() && now.part == 0 && a.gstate != nullptr) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int ch = c0 + gr * 4 + c;
          if (ch < a.C && j * 4 + n < a.N) a.gstate[(now.s * a.C + ch) * a.N + j * 4 + n] = at(r, c, n);
        }
    }
    __syncthreads();
    // gx, gdt, gz: over the LN lanes that share a group of channels
    T *qx = row_out<T>(a.gx, now.s, now.t), *qd = row_out<T>(a.gdt, now.s, now.t);
    T* qz = gate ? row_out<T>(a.gz, now.s, now.t) : nullptr;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int t = step0 + i * S::STEP;
      if (t >= steps || many == 0) continue;
      const float4* from = H + t * SLOTS * LINE + lane % G * LN;
      float2 s1[2], w[2], yp[2];
#pragma unroll
      for (int k = 0; k < LN; ++k) {
        // each lane begins with another of its parts, so that eight lanes read from eight groups of banks
        const int kk = (k + (LN == 4 ? lane % G / 2 : lane % G)) % LN;
        const float4 p = from[2 * LINE + kk], v = from[3 * LINE + kk];
        s1[0] = k ? add2(s1[0], make_float2(p.x, p.y)) : make_float2(p.x, p.y);
        s1[1] = k ? add2(s1[1], make_float2(p.z, p.w)) : make_float2(p.z, p.w);
        w[0] = k ? add2(w[0], make_float2(v.x, v.y)) : make_float2(v.x, v.y);
        w[1] = k ? add2(w[1], make_float2(v.z, v.w)) : make_float2(v.z, v.w);
        if (gate) {
          const float4 y = from[4 * LINE + kk];
          yp[0] = k ? add2(yp[0], make_float2(y.x, y.y)) : make_float2(y.x, y.y);
          yp[1] = k ? add2(yp[1], make_float2(y.z, y.w)) : make_float2(y.z, y.w);
        }
      }
      const int o = t * CW + lane % G * 4;
      const float4 x4 = *(const float4*)(sX + o), d4 = *(const float4*)(sD + o), g4 = *(const float4*)(sG + o);
      const float x[4] = {x4.x, x4.y, x4.z, x4.w}, delta[4] = {d4.x, d4.y, d4.z, d4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w};
      Pack<T, 4> ox, od, oz;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float sv = c & 1 ? s1[c / 2].y : s1[c / 2].x, wv = c & 1 ? w[c / 2].y : w[c / 2].x;
        const float gdt = fmaf(LN2, wv, sv * x[c]) * slope[i][c];
        gd[c] = fmaf(g[c], x[c], gd[c]);
        gbias[c] += gdt;
        ox.v[c] = from_f<T>(fmaf(sv, delta[c], dd[c] * g[c]));
        od.v[c] = from_f<T>(gdt);
        if (gate) oz.v[c] = from_f<T>(gz[i][c] * fmaf(dd[c], x[c], c & 1 ? yp[c / 2].y : yp[c / 2].x));
      }
      auto put = [&](T* p, const Pack<T, 4>& v) {
        if constexpr (VEC) {
          st<T, 4>(p, v);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < many) p[c] = v.v[c];
        }
      };
      put(qx + t * a.gx.step + mine, ox);
      put(qd + t * a.gdt.step + mine, od);
      if (gate) put(qz + t * a.gz.step + mine, oz);
    }
    // gb and gc: over the groups of every warp.  Four states of a step and of b or c a thread.
    for (int i = threadIdx.x; i < steps * 2 * LN; i += blockDim.x) {
      const int t = i / (2 * LN), which = i / LN % 2, jj = i % LN;
      float2 v0 = make_float2(0.f, 0.f), v1 = v0;
      for (int k = 0; k < warps; ++k) {
        const float4* from = (const float4*)((const float*)smem4 + k * S::WARP) + (t * SLOTS + which) * LINE + jj;
#pragma unroll
        for (int m = 0; m < G; ++m) {
          const float4 p = from[m * LN];
          v0 = add2(v0, make_float2(p.x, p.y)), v1 = add2(v1, make_float2(p.z, p.w));
        }
      }
      const float v[4] = {v0.x, v0.y, v1.x, v1.y};
      float* to = part_bc + (((int64_t)blockIdx.y * a.S + now.s) * a.T + now.t + t) * 2 * a.N + which * a.N + jj * 4;
      T* out = row_out<T>(which ? a.gc : a.gb, now.s, now.t + t) + jj * 4;
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (jj * 4 + n < a.N) {
          if (part_bc != nullptr)
            to[n] = v[n];
          else
            out[n] = from_f<T>(v[n]);
        }
    }
  }
  float* out = part_par + (int64_t)blockIdx.x * a.C * (a.N + 2);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int ch = c0 + gr * 4 + c;
      if (ch < a.C && j * 4 + n < a.N) out[(int64_t)ch * a.N + j * 4 + n] = at(dA, c, n);
    }
  // the lanes that wrote other steps of the same channels
#pragma unroll
  for (int m = G; m < 32; m *= 2)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      gd[c] += __shfl_xor_sync(0xFFFFFFFFu, gd[c], m);
      gbias[c] += __shfl_xor_sync(0xFFFFFFFFu, gbias[c], m);
    }
  if (lane < G)
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
  int most = 8;
  while (most > 1 && (most * S::WARP * 4 + 1024) > 227 * 1024) --most;
  b.tiles = (int)ceil_div(all, most);
  b.warps = (int)ceil_div(all, b.tiles);
  b.smem = b.warps * S::WARP * 4;
}
static BwdPlan bwd_plan(const InbScanArgs& a) {
  BwdPlan b;
  b.lanes = a.N <= 4 ? 1 : a.N <= 8 ? 2 : a.N <= 16 ? 4 : a.N <= 32 ? 8 : 16;
  b.plan = scan_plan(a, 128 / b.lanes);
  if (b.lanes == 1) bwd_shape<1>(b, a.C);
  if (b.lanes == 2) bwd_shape<2>(b, a.C);
  if (b.lanes == 4) bwd_shape<4>(b, a.C);
  if (b.lanes == 8) bwd_shape<8>(b, a.C);
  if (b.lanes == 16) bwd_shape<16>(b, a.C);
  const int64_t fit = 227 * 1024 / (b.smem + 1024), tasks = a.S * b.plan.parts;
  int64_t blocks = sm_count() * fit / b.tiles;
  if (blocks < 1) blocks = 1;
  b.blocks = (int)(blocks < tasks ? blocks : tasks);
  b.carry = (scan_carry_elems(a, b.plan) + 3) / 4 * 4;
  b.bc = b.tiles > 1 ? b.tiles * a.S * a.T * 2 * a.N : 0;
  b.par = (int64_t)b.blocks * a.C * (a.N + 2);
  return b;
}
template <typename T, int LN, bool VEC, bool WIDE>
static int bwd_launch(const InbScanArgs& a, const BwdPlan& b, const float* carry, float* bc, float* par, cudaStream_t s) {
  constexpr auto kernel = scan_bwd_kernel<T, LN, VEC, WIDE>;
  const cudaError_t e = allow_smem<KernelKey<scan_bwd_kernel<T, LN, VEC, WIDE>>>((const void*)kernel, 227 * 1024);
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
  const bool wide = LN >= 4 && vec && a.N == 4 * LN && is_aligned(a.b, 16, sizeof(T)) && is_aligned(a.c, 16, sizeof(T));
  if (wide)
    rc = bwd_launch<T, LN, true, LN >= 4>(a, b, carry, bc, par, s);
  else
    rc = vec ? bwd_launch<T, LN, true, false>(a, b, carry, bc, par, s) : bwd_launch<T, LN, false, false>(a, b, carry, bc, par, s);
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
    *elems = scan_carry_elems(a, scan_plan(a, 32 / scan_lanes(a.N)));
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
      (a.z.p != nullptr && a.gz.p == nullptr) || (a.T > SCAN_STEPS && a.kept == nullptr))
    return -3;
  if (a.work == nullptr || a.work_elems < need) return -5;
  const BwdPlan b = bwd_plan(a);
  if (a.dtype == INB_BF16) return bwd_type<bf16>(a, b, (cudaStream_t)cuda_stream);
  if (a.dtype == INB_F16) return bwd_type<f16>(a, b, (cudaStream_t)cuda_stream);
  return bwd_type<float>(a, b, (cudaStream_t)cuda_stream);
}
