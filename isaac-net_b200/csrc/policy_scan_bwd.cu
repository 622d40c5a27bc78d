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
  static constexpr int H = TC * 4 * 32 * 4, CH = TC * CW, BC = TC * NP, OUT = TC * 2 * NP;
  static constexpr int WARP = H + 5 * CH + 2 * BC + 2 * OUT;        // floats of shared memory a warp
};

template <typename T, int LN>
__global__ void __launch_bounds__(256) scan_bwd_kernel(InbScanArgs a, ScanPlan pl, const float* carry, float* part_bc,
                                                       float* part_par) {
  using S = BwdShape<LN>;
  constexpr int TC = S::TC, NP = S::NP, CW = S::CW, OWN = S::OWN, G = 32 / LN;
  extern __shared__ float4 smem4[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int j = lane % LN, gr = lane / LN;
  float* base = (float*)smem4 + warp * S::WARP;
  float4* H = (float4*)base;
  float *sD = base + S::H, *sX = sD + S::CH, *sG = sX + S::CH, *sZ = sG + S::CH, *sS = sZ + S::CH;
  float *sB = sS + S::CH, *sC = sB + S::BC, *sO = sC + S::BC;
  const int64_t c0 = ((int64_t)blockIdx.y * warps + warp) * CW, n4 = (a.N + 3) / 4 * 4, chunks = (a.T + TC - 1) / TC;
  const bool gate = a.z.p != nullptr;
  const int own = lane * 4 / LN;                 // this lane's channels [own, own + OWN) of the warp's
  const bool writer = LN <= 4 || (lane % (LN / 4 > 0 ? LN / 4 : 1)) == 0;
  float A[4][4], dA[4][4], bias[OWN], dd[OWN], gd[OWN], gbias[OWN];
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int64_t ch = c0 + gr * 4 + c;
      A[c][n] = ch < a.C && j * 4 + n < a.N ? a.a[ch * a.N + j * 4 + n] * LOG2E : 0.f;
      dA[c][n] = 0.f;
    }
#pragma unroll
  for (int k = 0; k < OWN; ++k) {
    const int64_t ch = c0 + own + k;
    bias[k] = ch < a.C && a.dt_bias != nullptr ? a.dt_bias[ch] : 0.f;
    dd[k] = ch < a.C && a.d != nullptr ? a.d[ch] : 0.f;
    gd[k] = gbias[k] = 0.f;
  }
  int flip = 0;
  for (int64_t task = blockIdx.x; task < a.S * pl.parts; task += gridDim.x) {
    const int64_t part = task / a.S, s = task - part * a.S;
    const int64_t t0 = part * pl.len, t1 = t0 + pl.len < a.T ? t0 + pl.len : a.T;
    const uint8_t* rs = resets(a.reset, s);
    float r[4][4];              // the gradient that reaches the state from later steps
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int64_t ch = c0 + gr * 4 + c;
        const int k = j * 4 + n;
        r[c][n] = 0.f;
        if (ch < a.C && k < a.N) {
          if (pl.parts > 1)
            r[c][n] = carry[((s * pl.parts + part) * a.C + ch) * n4 + k];
          else if (a.gstate_out != nullptr)
            r[c][n] = a.gstate_out[(s * a.C + ch) * a.N + k];
        }
      }
    for (int64_t t = t0 + (t1 - t0 - 1) / TC * TC; t >= t0; t -= TC, flip ^= 1) {
      const int steps = t1 - t < TC ? (int)(t1 - t) : TC;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < TC; ++i)
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
          const int64_t ch = c0 + own + k;
          float x = 0.f, delta = 0.f, g = 0.f, gz = 0.f, slope = 0.f;
          if (i < steps && ch < a.C) {
            x = to_f(row<T>(a.x, s, t + i)[ch]);
            g = to_f(row<T>(a.gy, s, t + i)[ch]);
            delta = softplus(to_f(row<T>(a.dt, s, t + i)[ch]) + bias[k], slope);
            if (gate) {
              const float z = to_f(row<T>(a.z, s, t + i)[ch]), q = sigmoid(z);
              gz = g * q * fmaf(z, 1.f - q, 1.f);
              g *= z * q;
            }
          }
          const int at = i * CW + own + k;
          sX[at] = x, sD[at] = delta, sG[at] = g, sZ[at] = gz, sS[at] = slope;
        }
#pragma unroll
      for (int i = lane; i < TC * NP; i += 32) {
        const int tt = i / NP, n = i % NP;
        const bool in = tt < steps && n < a.N;
        sB[i] = in ? to_f(row<T>(a.b, s, t + tt)[n]) : 0.f;
        sC[i] = in ? to_f(row<T>(a.c, s, t + tt)[n]) : 0.f;
      }
      const uint32_t bits = reset_bits(rs, a.reset.step, t, t1, lane);
      float h[4][4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int64_t ch = c0 + gr * 4 + c;
#pragma unroll
        for (int n = 0; n < 4; ++n) h[c][n] = 0.f;
        if (ch >= a.C) continue;
        if (t > 0) {
          if (j * 4 < n4) {
            const float4 v = *reinterpret_cast<const float4*>(a.kept + ((s * (chunks - 1) + t / TC - 1) * a.C + ch) * n4 + j * 4);
            h[c][0] = v.x, h[c][1] = v.y, h[c][2] = v.z, h[c][3] = v.w;
          }
        } else if (a.state != nullptr) {
#pragma unroll
          for (int n = 0; n < 4; ++n)
            if (j * 4 + n < a.N) h[c][n] = a.state[s * a.state_seq + ch * a.N + j * 4 + n];
        }
      }
      __syncwarp();
      // forward again: the state before each step
      for (int i = 0; i < steps; ++i) {
        if (bits >> i & 1) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int n = 0; n < 4; ++n) h[c][n] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) H[(i * 4 + c) * 32 + lane] = make_float4(h[c][0], h[c][1], h[c][2], h[c][3]);
        if (i + 1 == steps) break;
        const float4 D4 = *(const float4*)(sD + i * CW + gr * 4), X4 = *(const float4*)(sX + i * CW + gr * 4);
        const float4 B4 = *(const float4*)(sB + i * NP + j * 4);
        const float D[4] = {D4.x, D4.y, D4.z, D4.w}, U[4] = {D4.x * X4.x, D4.y * X4.y, D4.z * X4.z, D4.w * X4.w};
        const float B[4] = {B4.x, B4.y, B4.z, B4.w};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int n = 0; n < 4; ++n) h[c][n] = fmaf(ex2(D[c] * A[c][n]), h[c][n], U[c] * B[n]);
      }
      for (int i = steps - 1; i >= 0; --i) {
        const float4 D4 = *(const float4*)(sD + i * CW + gr * 4), X4 = *(const float4*)(sX + i * CW + gr * 4),
                     G4 = *(const float4*)(sG + i * CW + gr * 4);
        const float4 B4 = *(const float4*)(sB + i * NP + j * 4), C4 = *(const float4*)(sC + i * NP + j * 4);
        const float D[4] = {D4.x, D4.y, D4.z, D4.w}, U[4] = {D4.x * X4.x, D4.y * X4.y, D4.z * X4.z, D4.w * X4.w};
        const float GG[4] = {G4.x, G4.y, G4.z, G4.w}, B[4] = {B4.x, B4.y, B4.z, B4.w}, C[4] = {C4.x, C4.y, C4.z, C4.w};
        float bc[8], s1[4], w[4], yp[4];
#pragma unroll
        for (int n = 0; n < 8; ++n) bc[n] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float4 P4 = H[(i * 4 + c) * 32 + lane];
          const float P[4] = {P4.x, P4.y, P4.z, P4.w};
          s1[c] = w[c] = yp[c] = 0.f;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float e = ex2(D[c] * A[c][n]), eh = e * P[n], hh = fmaf(U[c], B[n], eh);
            const float dh = fmaf(C[n], GG[c], r[c][n]), q = dh * eh;
            yp[c] = fmaf(C[n], hh, yp[c]);
            bc[4 + n] = fmaf(GG[c], hh, bc[4 + n]);
            bc[n] = fmaf(U[c], dh, bc[n]);
            s1[c] = fmaf(B[n], dh, s1[c]);
            dA[c][n] = fmaf(D[c], q, dA[c][n]);
            w[c] = fmaf(A[c][n], q, w[c]);
            r[c][n] = e * dh;
          }
        }
        if (bits >> i & 1) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int n = 0; n < 4; ++n) r[c][n] = 0.f;
        }
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
          const int at = i * CW + own + k;
          const float x = sX[at], delta = sD[at], g = sG[at];
          const float gdt = fmaf(LN2, w[k], s1[k] * x) * sS[at];
          gd[k] = fmaf(g, x, gd[k]);
          gbias[k] += gdt;
          if (writer && ch < a.C) {
            row_out<T>(a.gx, s, t + i)[ch] = from_f<T>(fmaf(s1[k], delta, dd[k] * g));
            row_out<T>(a.gdt, s, t + i)[ch] = from_f<T>(gdt);
            if (gate) row_out<T>(a.gz, s, t + i)[ch] = from_f<T>(sZ[at] * fmaf(dd[k], x, yp[k]));
          }
        }
      }
      __syncthreads();
      const float* all = (const float*)smem4 + (sO - base) + flip * S::OUT;
      for (int i = threadIdx.x; i < steps * 2 * NP; i += blockDim.x) {
        const int tt = i / (2 * NP), which = i / NP % 2, n = i % NP;
        if (n >= a.N) continue;
        float v = 0.f;
        for (int k = 0; k < warps; ++k) v += all[k * S::WARP + i];
        if (part_bc != nullptr)
          part_bc[(((int64_t)blockIdx.y * a.S + s) * a.T + t + tt) * 2 * a.N + which * a.N + n] = v;
        else
          row_out<T>(which ? a.gc : a.gb, s, t + tt)[n] = from_f<T>(v);
      }
    }
    if (part == 0 && a.gstate != nullptr) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int64_t ch = c0 + gr * 4 + c;
          if (ch < a.C && j * 4 + n < a.N) a.gstate[(s * a.C + ch) * a.N + j * 4 + n] = r[c][n];
        }
    }
  }
  float* out = part_par + (int64_t)blockIdx.x * a.C * (a.N + 2);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int64_t ch = c0 + gr * 4 + c;
      if (ch < a.C && j * 4 + n < a.N) out[ch * a.N + j * 4 + n] = dA[c][n];
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
