// selective_scan's backward pass.  With g = gy silu(z), u = delta x, e = exp(delta a):
//
//   dh[t] = c[t] g[t] + e[t + 1] dh[t + 1]            (0 instead of the second term where t + 1 starts an episode)
//   gb[t, n] = sum_c dh u     gc[t, n] = sum_c h g     ga[c, n] = sum_t delta dh e h[t - 1]
//   s1 = sum_n dh b           w = sum_n a dh e h[t - 1]
//   gx = s1 delta + d g       gdt = (w + s1 x) / (1 + exp(-(dt + dt_bias)))     gz = gy silu'(z) (sum_n c h + d x)
//
// The forward pass kept the state before every SCAN_STEPS steps; a warp runs those steps forward again from there, with
// every state in shared memory, then backward.  A thread holds 4 states of 4 neighbouring channels: sums over channels (gb,
// gc) and over states (s1, w, y) then take 7 + 9 shuffles a step where a channel a thread would take 31.  gb and gc are
// added over the block's warps in shared memory and over blocks by a further launch, ga, gd, gdt_bias stay in registers
// over all the tasks of a block: no atomics.
#include "policy_scan.cuh"

namespace inb {
namespace pol {

// One level of a sum over lanes: each value is added to that of the lane that differs in `mask`.  While there are several
// values, a lane keeps half of them: the upper half where its bit is set.
template <int M, int NV>
__device__ __forceinline__ void halve(float (&v)[NV], int lane, int mask) {
  if constexpr (M > 1) {
    const bool up = lane & mask;
#pragma unroll
    for (int i = 0; i < M / 2; ++i) {
      const float send = up ? v[i] : v[i + M / 2], keep = up ? v[i + M / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, mask);
    }
  } else {
    v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], mask);
  }
}
// Over LN lanes, the highest bit first: lane j is left with values [j * M / LN, ...)
template <int M, int LN, int NV>
__device__ __forceinline__ void over_states(float (&v)[NV], int lane) {
  if constexpr (LN > 1) {
    halve<M>(v, lane, LN / 2);
    over_states<(M > 1 ? M / 2 : 1), LN / 2>(v, lane);
  }
}
// Over the lanes of the bits MASK .. 16, likewise
template <int M, int BIT, int MASK, int NV>
__device__ __forceinline__ void over_channels(float (&v)[NV], int lane) {
  if constexpr (BIT >= MASK) {
    halve<M>(v, lane, BIT);
    over_channels<(M > 1 ? M / 2 : 1), BIT / 2, MASK>(v, lane);
  }
}

template <int LN>
struct BwdShape {
  static constexpr int TC = SCAN_STEPS, NP = 4 * LN, CW = 128 / LN, OWN = LN < 4 ? 4 / LN : 1;
  static constexpr int H = TC * 4 * 32 * 4, CH = TC * CW, BC = TC * NP * 2, OUT = TC * 2 * NP;
  static constexpr int WARP = H + 5 * CH + 2 * BC + 2 * OUT;        // floats of shared memory a warp
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

// Bound by issue and by the exponentials together: of a step's 330 warp instructions for 16 states a thread 120 are packed
// multiplications and additions and 36 exponentials, which take 8 cycles each.  Shared memory (25 KB a warp, of it 16 for
// the states) leaves 8 warps an SM, so a chunk's inputs are loaded a chunk ahead.
template <typename T, int LN>
__global__ void __launch_bounds__(256, 1) scan_bwd_kernel(InbScanArgs a, ScanPlan pl, const float* carry, float* part_bc,
                                                          float* part_par) {
  using S = BwdShape<LN>;
  constexpr int TC = S::TC, NP = S::NP, CW = S::CW, OWN = S::OWN, G = 32 / LN, BCL = TC * NP / 32;
  extern __shared__ float4 smem4[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int j = lane % LN, gr = lane / LN;
  float* base = (float*)smem4 + warp * S::WARP;
  float4* H = (float4*)base;
  float *sD = base + S::H, *sX = sD + S::CH, *sG = sX + S::CH, *sZ = sG + S::CH, *sS = sZ + S::CH;
  float *sB = sS + S::CH, *sC = sB + S::BC, *sO = sC + S::BC;       // b and c twice each: operands of packed products
  const int64_t c0 = ((int64_t)blockIdx.y * warps + warp) * CW, n4 = (a.N + 3) / 4 * 4, chunks = (a.T + TC - 1) / TC;
  const bool gate = a.z.p != nullptr;
  const int own = lane * 4 / LN;                 // this lane's channels [own, own + OWN) of the warp's
  const bool writer = LN <= 4 || (lane % (LN / 4 > 0 ? LN / 4 : 1)) == 0;
  // channels beyond the last one: dt and z are read as the last one's, a, x, gy and the state are 0, nothing is written
  auto clip = [&](int64_t ch) { return ch < a.C ? ch : (int64_t)a.C - 1; };
  // pairs of channels (2 p, 2 p + 1) of this thread's four, state n of its four
  float2 A[2][4], dA[2][4], r[2][4], h[2][4];
  float bias[OWN], dd[OWN], gd[OWN], gbias[OWN];
  auto at = [](float2 (&v)[2][4], int c, int n) -> float& { return c & 1 ? v[c / 2][n].y : v[c / 2][n].x; };
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int64_t ch = c0 + gr * 4 + c;
      at(A, c, n) = ch < a.C && j * 4 + n < a.N ? a.a[ch * a.N + j * 4 + n] * LOG2E : 0.f;
      at(dA, c, n) = 0.f;
    }
#pragma unroll
  for (int k = 0; k < OWN; ++k) {
    const int64_t ch = clip(c0 + own + k);
    bias[k] = a.dt_bias != nullptr ? a.dt_bias[ch] : 0.f;
    dd[k] = a.d != nullptr ? a.d[ch] : 0.f;
    gd[k] = gbias[k] = 0.f;
  }
  // a chunk's inputs as they lie in memory
  T rx[TC][OWN], rd[TC][OWN], rz[TC][OWN], rg[TC][OWN], rb[BCL], rc[BCL];
  float4 rh[4];
  uint32_t bits, later = 0;
  auto load = [&](const Chunk& q) {
    const T *px = row<T>(a.x, q.s, q.t), *pd = row<T>(a.dt, q.s, q.t), *pg = row<T>(a.gy, q.s, q.t);
    const T* pz = gate ? row<T>(a.z, q.s, q.t) : nullptr;
    const int64_t ch = clip(c0 + own);
    px += ch, pd += ch, pg += ch;
    if (gate) pz += ch;
    // the other channels of this lane lie next to it, but for those beyond the last one
    const int more = (int)(clip(c0 + own + OWN - 1) - ch);
#pragma unroll
    for (int i = 0; i < TC; ++i) {
      if (i < q.steps) {
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
          const int o = k < more ? k : more;
          rx[i][k] = px[o], rd[i][k] = pd[o], rg[i][k] = pg[o];
          if (gate) rz[i][k] = pz[o];
        }
      }
      px += a.x.step, pd += a.dt.step, pg += a.gy.step;
      if (gate) pz += a.z.step;
    }
    const T *pb = row<T>(a.b, q.s, q.t), *pc = row<T>(a.c, q.s, q.t);
#pragma unroll
    for (int i = 0; i < BCL; ++i) {
      const int tt = (i * 32 + lane) / NP, n = (i * 32 + lane) % NP;
      rb[i] = rc[i] = from_f<T>(0.f);
      if (tt < q.steps && n < a.N) rb[i] = pb[tt * a.b.step + n], rc[i] = pc[tt * a.c.step + n];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t hc = clip(c0 + gr * 4 + c);
      rh[c] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c0 + gr * 4 + c >= a.C) continue;
      if (q.t > 0) {
        if (j * 4 < n4)
          rh[c] = *reinterpret_cast<const float4*>(a.kept + ((q.s * (chunks - 1) + q.t / TC - 1) * a.C + hc) * n4 + j * 4);
      } else if (a.state != nullptr) {
        const float* p = a.state + q.s * a.state_seq + hc * a.N + j * 4;
        if (j * 4 < a.N) rh[c].x = p[0];
        if (j * 4 + 1 < a.N) rh[c].y = p[1];
        if (j * 4 + 2 < a.N) rh[c].z = p[2];
        if (j * 4 + 3 < a.N) rh[c].w = p[3];
      }
    }
    const uint8_t* rs = resets(a.reset, q.s);
    later = reset_bits(rs != nullptr ? rs + q.t * a.reset.step : nullptr, a.reset.step, q.steps, lane);
  };
  Chunk q;
  q.task = blockIdx.x;
  q.start(a, pl);
  load(q);
  for (int flip = 0; q.on(a, pl); flip ^= 1) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < TC; ++i)
#pragma unroll
      for (int k = 0; k < OWN; ++k) {
        if (i >= q.steps) break;
        float slope, g = to_f(rg[i][k]), gz = 0.f;
        const float delta = softplus(to_f(rd[i][k]) + bias[k], slope);
        if (gate) {
          const float z = to_f(rz[i][k]), w = sigmoid(z);
          gz = g * w * fmaf(z, 1.f - w, 1.f);
          g *= z * w;
        }
        const bool in = c0 + own + k < a.C;
        const int o = i * CW + own + k;
        sX[o] = in ? to_f(rx[i][k]) : 0.f, sD[o] = delta, sG[o] = in ? g : 0.f, sZ[o] = gz, sS[o] = slope;
      }
#pragma unroll
    for (int i = 0; i < BCL; ++i) {
      *reinterpret_cast<float2*>(sB + 2 * (i * 32 + lane)) = both(to_f(rb[i]));
      *reinterpret_cast<float2*>(sC + 2 * (i * 32 + lane)) = both(to_f(rc[i]));
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) at(h, c, 0) = rh[c].x, at(h, c, 1) = rh[c].y, at(h, c, 2) = rh[c].z, at(h, c, 3) = rh[c].w;
    bits = later;
    const Chunk now = q;
    const int steps = now.steps;
    q.next(a, pl);
    if (q.on(a, pl)) load(q);
    if (now.newest()) {              // the gradient that reaches the task's last state from later steps
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int64_t ch = c0 + gr * 4 + c;
          const int k = j * 4 + n;
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
    __syncwarp();
    // forward again: the state before each step
    for (int i = 0; i < steps; ++i) {
      if (bits >> i & 1) {
#pragma unroll
        for (int n = 0; n < 4; ++n) h[0][n] = h[1][n] = make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int n = 0; n < 4; n += 2)
          H[(i * 4 + p * 2 + n / 2) * 32 + lane] = make_float4(h[p][n].x, h[p][n].y, h[p][n + 1].x, h[p][n + 1].y);
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
    T *qx = row_out<T>(a.gx, now.s, now.t + steps - 1), *qd = row_out<T>(a.gdt, now.s, now.t + steps - 1);
    T* qz = gate ? row_out<T>(a.gz, now.s, now.t + steps - 1) : nullptr;
    for (int i = steps - 1; i >= 0; --i) {
      const float4 D4 = *(const float4*)(sD + i * CW + gr * 4), X4 = *(const float4*)(sX + i * CW + gr * 4),
                   G4 = *(const float4*)(sG + i * CW + gr * 4);
      const float4 *B4 = (const float4*)(sB + (i * NP + j * 4) * 2), B0 = B4[0], B1 = B4[1];
      const float4 *C4 = (const float4*)(sC + (i * NP + j * 4) * 2), C0 = C4[0], C1 = C4[1];
      const float2 D[2] = {make_float2(D4.x, D4.y), make_float2(D4.z, D4.w)};
      const float2 U[2] = {mul2(D[0], make_float2(X4.x, X4.y)), mul2(D[1], make_float2(X4.z, X4.w))};
      const float2 GG[2] = {make_float2(G4.x, G4.y), make_float2(G4.z, G4.w)};
      const float2 B[4] = {make_float2(B0.x, B0.y), make_float2(B0.z, B0.w), make_float2(B1.x, B1.y), make_float2(B1.z, B1.w)};
      const float2 C[4] = {make_float2(C0.x, C0.y), make_float2(C0.z, C0.w), make_float2(C1.x, C1.y), make_float2(C1.z, C1.w)};
      float2 gb[4], gc[4], s1p[2], wp[2], yp2[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float4 P4 = H[(i * 4 + p * 2 + n / 2) * 32 + lane];
          const float2 P = n & 1 ? make_float2(P4.z, P4.w) : make_float2(P4.x, P4.y);
          const float2 v = mul2(D[p], A[p][n]), e = make_float2(ex2(v.x), ex2(v.y));
          const float2 eh = mul2(e, P), hh = fma2(U[p], B[n], eh), dh = fma2(C[n], GG[p], r[p][n]), w = mul2(dh, eh);
          yp2[p] = n ? fma2(C[n], hh, yp2[p]) : mul2(C[n], hh);
          gc[n] = p ? fma2(GG[p], hh, gc[n]) : mul2(GG[p], hh);
          gb[n] = p ? fma2(U[p], dh, gb[n]) : mul2(U[p], dh);
          s1p[p] = n ? fma2(B[n], dh, s1p[p]) : mul2(B[n], dh);
          dA[p][n] = fma2(D[p], w, dA[p][n]);
          wp[p] = n ? fma2(A[p][n], w, wp[p]) : mul2(A[p][n], w);
          r[p][n] = mul2(e, dh);
        }
      }
      if (bits >> i & 1) {
#pragma unroll
        for (int n = 0; n < 4; ++n) r[0][n] = r[1][n] = make_float2(0.f, 0.f);
      }
      float bc[8], s1[4] = {s1p[0].x, s1p[0].y, s1p[1].x, s1p[1].y}, w[4] = {wp[0].x, wp[0].y, wp[1].x, wp[1].y},
                   yp[4] = {yp2[0].x, yp2[0].y, yp2[1].x, yp2[1].y};
#pragma unroll
      for (int n = 0; n < 4; ++n) bc[n] = gb[n].x + gb[n].y, bc[4 + n] = gc[n].x + gc[n].y;
      over_channels<8, 16, LN>(bc, lane);
      over_states<4, LN>(s1, lane);
      over_states<4, LN>(w, lane);
      if (gate) over_states<4, LN>(yp, lane);
      {
        // values [8 / G * gr, ...) of b's 4 and c's 4 are this lane's; with more lanes than values the first of each run's
        constexpr int LEFT = G < 8 ? 8 / G : 1, SAME = G > 8 ? G / 8 : 1;
        if (gr % SAME == 0)
#pragma unroll
          for (int k = 0; k < LEFT; ++k) {
            const int v = gr / SAME * LEFT + k;
            sO[flip * S::OUT + (i * 2 + v / 4) * NP + j * 4 + v % 4] = bc[k];
          }
      }
#pragma unroll
      for (int k = 0; k < OWN; ++k) {
        const int64_t ch = c0 + own + k;
        const int o = i * CW + own + k;
        const float x = sX[o], delta = sD[o], g = sG[o];
        const float gdt = fmaf(LN2, w[k], s1[k] * x) * sS[o];
        gd[k] = fmaf(g, x, gd[k]);
        gbias[k] += gdt;
        if (writer && ch < a.C) {
          qx[ch] = from_f<T>(fmaf(s1[k], delta, dd[k] * g));
          qd[ch] = from_f<T>(gdt);
          if (gate) qz[ch] = from_f<T>(sZ[o] * fmaf(dd[k], x, yp[k]));
        }
      }
      qx -= a.gx.step, qd -= a.gdt.step;
      if (gate) qz -= a.gz.step;
    }
    __syncthreads();
    const float* all = (const float*)smem4 + (sO - base) + flip * S::OUT;
    for (int i = threadIdx.x; i < steps * 2 * NP; i += blockDim.x) {
      const int tt = i / (2 * NP), which = i / NP % 2, n = i % NP;
      if (n >= a.N) continue;
      float v = 0.f;
      for (int k = 0; k < warps; ++k) v += all[k * S::WARP + i];
      if (part_bc != nullptr)
        part_bc[(((int64_t)blockIdx.y * a.S + now.s) * a.T + now.t + tt) * 2 * a.N + which * a.N + n] = v;
      else
        row_out<T>(which ? a.gc : a.gb, now.s, now.t + tt)[n] = from_f<T>(v);
    }
    if (now.oldest() && now.part == 0 && a.gstate != nullptr) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int64_t ch = c0 + gr * 4 + c;
          if (ch < a.C && j * 4 + n < a.N) a.gstate[(now.s * a.C + ch) * a.N + j * 4 + n] = at(r, c, n);
        }
    }
  }
  float* out = part_par + (int64_t)blockIdx.x * a.C * (a.N + 2);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int64_t ch = c0 + gr * 4 + c;
      if (ch < a.C && j * 4 + n < a.N) out[ch * a.N + j * 4 + n] = at(dA, c, n);
    }
#pragma unroll
  for (int k = 0; k < OWN; ++k) {
    const int64_t ch = c0 + own + k;
    if (writer && ch < a.C) {
      out[(int64_t)a.C * a.N + ch] = gd[k];
      out[(int64_t)a.C * (a.N + 1) + ch] = gbias[k];
    }
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
template <typename T, int LN>
static int bwd_go(const InbScanArgs& a, const BwdPlan& b, cudaStream_t s) {
  const cudaError_t e = allow_smem<KernelKey<scan_bwd_kernel<T, LN>>>((const void*)scan_bwd_kernel<T, LN>, 227 * 1024);
  if (e != cudaSuccess) return -100 - (int)e;
  float *carry = a.work, *bc = carry + b.carry, *par = bc + b.bc;
  if (b.plan.split()) {
    const int rc = scan_launch(a, b.plan, carry, 3, s);
    if (rc != 0) return rc;
  }
  scan_bwd_kernel<T, LN><<<dim3(b.blocks, b.tiles), b.warps * 32, b.smem, s>>>(a, b.plan, carry, b.bc > 0 ? bc : nullptr, par);
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
