// selective_scan: what its forward and backward launches share (formulas: policy_scan.cu).
#pragma once
#include "policy_seq.cuh"

namespace inb {
namespace pol {

constexpr int SCAN_STEPS = 8;        // steps a warp stages at once; the backward pass starts from states kept this far apart

constexpr int SCAN_WARPS = 4;        // a block of the forward pass

// The time axis in parts of `len` steps (a multiple of SCAN_STEPS), so that few sequences still fill the GPU: their states
// are joined between two passes (scan_kernel's modes 2 and 3, scan_join_kernel).
struct ScanPlan {
  int64_t parts, len;
  bool split() const { return parts > 1; }
};
// As many parts as end soonest.  One takes `units` blocks, of which the GPU holds `room`, and blocks that find no room wait for a
// whole round; a step takes as long beside 16 warps an SM as alone (0.4 us).  A split pass costs `split` / 4 of one that is
// not, and the join as much as 16 steps.
inline ScanPlan scan_split(int64_t T, int64_t units, int64_t room, int split) {
  ScanPlan best = {1, ceil_div(T, SCAN_STEPS) * SCAN_STEPS};
  int64_t cost = ceil_div(units, room) * T * 4;
  for (int64_t n = 2; n <= T / 16 && n <= 256 && units * n <= 4 * room; ++n) {
    const int64_t len = ceil_div(ceil_div(T, n), SCAN_STEPS) * SCAN_STEPS, parts = ceil_div(T, len);
    const int64_t c = ceil_div(units * parts, room) * len * split + 64;
    if (c < cost) cost = c, best = {parts, len};
  }
  return best;
}
inline int64_t scan_n4(const InbScanArgs& a) { return (a.N + 3) / 4 * 4; }       // states of a channel in scratch
inline int64_t scan_chunks(const InbScanArgs& a) { return ceil_div(a.T, SCAN_STEPS); }
// Forward pass: states a thread (NS) and lanes a channel (LN) for N states
inline int scan_lanes(int n) { return n <= 16 ? 1 : n <= 32 ? 2 : 4; }
inline ScanPlan scan_plan(const InbScanArgs& a) {
  const int64_t tiles = ceil_div(a.C, 32 / scan_lanes(a.N)), warps = tiles < SCAN_WARPS ? tiles : SCAN_WARPS;
  return scan_split(a.T, a.S * ceil_div(tiles, warps), (int64_t)sm_count() * (4 * SCAN_WARPS / warps), 8);
}
// floats of the parts' states [S, parts, C, N4] and of their sums of delta [S, parts, C]
inline int64_t scan_carry_elems(const InbScanArgs& a, const ScanPlan& p) {
  return p.split() ? a.S * p.parts * a.C * (scan_n4(a) + 1) : 0;
}

int scan_check(const InbScanArgs& a);
int scan_launch(const InbScanArgs& a, const ScanPlan& p, float* carry, int mode, cudaStream_t s);
int scan_join(const InbScanArgs& a, const ScanPlan& p, float* carry, bool reverse, cudaStream_t s);

// ex2.approx is low: measured on a B200, by 0.1 * 2^-24 on average for results 2^-v with v below 2^-9, by 0.3 to 0.45 for v from
// 2^-8 to 1/4, by 0.6 to 0.85 beyond.  A state that fades slowly multiplies hundreds of such decays, whose random errors average
// out and whose common one adds up (1.7e-6 of a state after 90 steps of 0.01).  So once a chunk a state is raised by what its
// decays have lost: `delta`, the chunk's sum, times -a, held to what a state keeps of a chunk.
__device__ __forceinline__ float2 unbias(float2 h, float2 a, float2 delta) {
  const float2 t = mul2(mul2(delta, both(-1.f)), a), low = mul2(t, both(78.f)), high = fma2(t, both(-0.4f), both(3.2f));
  const float2 k = make_float2(fmaxf(0.f, fminf(low.x, high.x)), fmaxf(0.f, fminf(low.y, high.y)));
  return fma2(h, mul2(k, both(1.f / 16777216)), h);
}

// The reset flag of this lane's step among the next `steps` (lanes beyond: 0); a ballot makes them the same bits in every lane
__device__ __forceinline__ uint32_t reset_flag(const uint8_t* at, int64_t step, int steps, int lane) {
  return at != nullptr && lane < steps ? at[lane * step] : 0u;
}

}  // namespace pol
}  // namespace inb
