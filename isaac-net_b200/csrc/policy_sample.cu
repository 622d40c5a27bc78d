// sample_logits: one token a row from temperature, top-k, top-p, min-p and a given uniform, with its log-probability.
//
//   m = max l;  z_i = (l_i - m) / T;  w_i = exp(z_i);  q_i = floor(2^40 w_i)
//   order: larger l first, ties by lower index
//   top-k keeps the first k; top-p keeps an element while the mass before it is < p times the mass top-k left;
//   min-p keeps w_i >= min_p;  token = first kept i by index with sum of q up to i > floor(u S), S = the kept mass
//   logp = z - log(2^-40 S)
//
// The masses are integers, so a sum has one value whatever its order: no result depends on how a row is split over
// lanes, warps or blocks, and the token is a function of the inputs alone.  2^-40 of the largest weight is the unit:
// 2^20 elements together cannot be off by more than 2^-20 of the largest one, and 2^22 of them (the longest
// row) do not overflow 64 bits.
//
// Rows of up to 384 logits take 8, 16 or 32 lanes of a warp each: the cut-offs are found by bisection, and then by taking
// the largest remaining logit away until the count or the mass is reached.  Longer rows take a block, or a cluster of 2 to 8
// blocks when there are fewer rows than SMs: the row stays in shared memory, a histogram over z finds the bin of the
// cut-off, and histograms over the float's ordered bits narrow that bin to one value.  Either way the logits are read from
// memory once, which is the floor; what bounds the kernel is the latency of its passes, not DRAM.
#include <cooperative_groups.h>

#include <type_traits>

#include "policy_common.cuh"

namespace cg = cooperative_groups;

namespace inb {
namespace pol {

constexpr uint32_t KEY_NEG_INF = 0x007FFFFFu;      // ordered bits of -inf
constexpr float Z_SPAN = 28.f;                     // exp(-28) < 2^-40: below it the mass is 0
constexpr float Z_SURE = 27.f;                     // exp(-27) > 2^-39: above it the mass is not 0
constexpr float Q_ONE = 1099511627776.f;           // 2^40

// order-preserving map of a float to unsigned
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// a logit as the operator sees it: masked and NaN entries are -inf, and -0 is +0
__device__ __forceinline__ float clean(float l, bool ok) { return ok && l == l ? l + 0.f : -INFINITY; }

struct RowParams {
  float inv_t, top_p, min_p, u;
  int k;               // 0: off
};
__device__ __forceinline__ RowParams row_params(const InbSampleArgs& a, int64_t row) {
  RowParams p;
  const float t = a.temperature_row ? a.temperature_row[row] : a.temperature;
  p.top_p = a.top_p_row ? a.top_p_row[row] : a.top_p;
  if (p.top_p != p.top_p) p.top_p = 0.f;      // NaN: the first element alone, never a filter that is off
  p.min_p = a.min_p_row ? a.min_p_row[row] : a.min_p;
  p.k = a.top_k_row ? a.top_k_row[row] : a.top_k;
  if (p.k < 0) p.k = 0;
  if (!(t > 0.f)) {      // 0 (or below, or NaN): greedy
    p.inv_t = 1.f;
    p.k = 1;
  } else {
    p.inv_t = __fdiv_rn(1.f, t);
  }
  p.u = a.u[row];
  return p;
}
__device__ __forceinline__ float z_of(float l, float m, float inv_t) {
  return l == m ? 0.f : (l == -INFINITY ? -INFINITY : __fmul_rn(__fsub_rn(l, m), inv_t));
}
__device__ __forceinline__ long long q_of(float w) { return __float2ll_rz(__fmul_rn(w, Q_ONE)); }

// how many of c equal masses q come before the mass thr is reached, `before` being what is above them (at least 1)
__device__ __forceinline__ uint32_t ties_kept(long long before, long long q, uint32_t c, double thr) {
  uint32_t lo = 1, hi = c;           // the first r in [1, c] with before + r q >= thr
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (__ll2double_rn(before + (long long)mid * q) >= thr)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}
__device__ __forceinline__ double p_threshold(float p, long long total) {
  const double t = __dmul_rn((double)p, __ll2double_rn(total));
  return t > 1.0 ? t : 1.0;          // p <= 0 keeps the first element
}
__device__ __forceinline__ long long draw_at(float u, long long total) {
  const double t = __dmul_rn((double)u, __ll2double_rn(total));
  if (!(t > 0.0)) return 0;
  const long long v = __double2ll_rz(t);
  return v < total ? v : total - 1;
}
__device__ __forceinline__ float logp_of(float z, long long total) {
  return (float)((double)z - log(__ll2double_rn(total) * (1.0 / 1099511627776.0)));
}

// ------------------------------------------------------------------------------------------------ a warp per row
// Groups of GW lanes (8, 16 or 32) work on a row each; every lane of a warp takes part in every step.
template <int GW>
struct Group {
  static __device__ __forceinline__ int lane() { return threadIdx.x & (GW - 1); }
  static __device__ __forceinline__ uint32_t below() { return (1u << lane()) - 1u; }
  static __device__ __forceinline__ uint32_t max_of(uint32_t v) {
    if constexpr (GW == 32) {
      return __reduce_max_sync(M32_ALL, v);
    } else {
#pragma unroll
      for (int o = GW / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(M32_ALL, v, o));
      return v;
    }
  }
  static __device__ __forceinline__ uint32_t sum_of(uint32_t v) {
    if constexpr (GW == 32) {
      return __reduce_add_sync(M32_ALL, v);
    } else {
#pragma unroll
      for (int o = GW / 2; o > 0; o >>= 1) v += __shfl_xor_sync(M32_ALL, v, o);
      return v;
    }
  }
  static __device__ __forceinline__ uint32_t ballot(bool p) {
    const uint32_t b = __ballot_sync(M32_ALL, p);
    return GW == 32 ? b : (b >> (threadIdx.x & 31 & ~(GW - 1))) & ((1u << (GW & 31)) - 1u);
  }
  template <typename V>
  static __device__ __forceinline__ V get(V v, int src) {
    return __shfl_sync(M32_ALL, v, src, GW);
  }
};

// Masses of up to 512 elements as two words, q = hi 2^20 + lo with lo < 2^20: either sum fits 32 bits
__device__ __forceinline__ long long mass_of(uint32_t hi, uint32_t lo) { return ((long long)hi << 20) + lo; }

// One row: keys, exponents z and masses of its elements, EPL a lane, element j * GW + lane.  cut() zeroes the masses that a
// filter takes away: by count (top-k) or by mass (top-p).  Bisection over the z that the row has, on the high words alone,
// narrows the range that holds the cut-off; then the largest remaining value is taken away until the target is reached.  (A
// policy before training has logits that hardly differ: from a fixed range the bisection left all of a row's 33 values to
// the second part, 80 us for 32768 rows against 25.)
template <int GW, int EPL>
struct WarpRow {
  using G = Group<GW>;
  // of the bisection: each costs a sum, and halves the values that are then taken away one by one.  32768 rows, top-p 0.95:
  // V = 64 31 us with 6, 33 with 5; V = 128 56 with 7, 69 with 5; V = 200 91 with 9, 101 with 12.
  static constexpr int STEPS = EPL > 4 ? 9 : (EPL == 4 ? 7 : 6);
  uint32_t key[EPL], hi[EPL], lo[EPL];
  float z[EPL];

  __device__ __forceinline__ bool has(int j) const { return (hi[j] | lo[j]) != 0; }
  __device__ __forceinline__ long long mass_from(float least) const {
    uint32_t h = 0, l = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (z[j] >= least) {
        h += hi[j];
        l += lo[j];
      }
    return mass_of(G::sum_of(h), G::sum_of(l));
  }
  __device__ __forceinline__ uint32_t count_from(float least) const {
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) c += __popc(G::ballot(z[j] >= least && has(j)));
    return c;
  }
  // live: whether this group's row is to be cut at all
  template <bool MASS>
  __device__ __forceinline__ void cut(bool live, long long target) {
    // z >= up lies above the target's value; z >= down, the least z of all, holds it, or every element stays
    uint32_t least = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j) least = max(least, has(j) ? __float_as_uint(z[j]) : 0u);     // z <= 0: the bits fall with z
    float up = 1.f, down = __uint_as_float(G::max_of(least)), mid = fmaxf(-4.f, 0.5f * down);
    const uint32_t want = (uint32_t)(MASS ? target >> 20 : target);
    bool open = true;
#pragma unroll 1
    for (int i = 0; i < STEPS; ++i) {
      bool reached;
      if (MASS) {
        uint32_t h = 0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) h += z[j] >= mid ? hi[j] : 0u;
        h = G::sum_of(h);                        // the low words add less than GW EPL to it
        reached = h > want;
        if (!reached && h + GW * EPL >= want) open = false;      // the high words cannot tell
      } else {
        reached = count_from(mid) >= want;
      }
      if (open) {
        if (reached)
          down = mid;
        else
          up = mid;
        mid = 0.5f * (fminf(up, 0.f) + down);
      }
    }
    long long before = MASS ? mass_from(up) : (long long)count_from(up);
    uint32_t tau = M32_ALL;
#pragma unroll 1
    while (true) {
      uint32_t b = 0;
#pragma unroll
      for (int j = 0; j < EPL; ++j) b = max(b, key[j] < tau && z[j] < up && has(j) ? key[j] : 0u);
      b = G::max_of(b);
      live = live && b != 0;                     // 0: the target is beyond what there is, all stay
      if (!__any_sync(M32_ALL, live)) return;
      uint32_t c = 0, qh = 0, ql = 1, tie[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        tie[j] = G::ballot(key[j] == b && has(j));
        if (MASS) {
          const int src = tie[j] ? __ffs(tie[j]) - 1 : 0;
          const uint32_t h = G::get(hi[j], src), l = G::get(lo[j], src);
          if (tie[j] != 0) qh = h, ql = l;
        }
        c += __popc(tie[j]);
      }
      tau = b;
      const long long qb = mass_of(qh, ql);
      if (live) {
        if (before + (long long)c * qb >= target) {
          const uint32_t r = c == 1 ? 1u : (uint32_t)((target - before + qb - 1) / qb);     // the first r of them
          uint32_t rank = 0;
#pragma unroll
          for (int j = 0; j < EPL; ++j) {
            if (key[j] < tau || (key[j] == tau && rank + __popc(tie[j] & G::below()) >= r)) hi[j] = lo[j] = 0;
            rank += __popc(tie[j]);
          }
          live = false;
        } else {
          before += (long long)c * qb;
        }
      }
    }
  }
  // z holds the logits: makes z and the masses (none where m is the -inf of a row that allows nothing)
  __device__ __forceinline__ void weigh(float m, float inv_t) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      z[j] = m == -INFINITY ? -INFINITY : z_of(z[j], m, inv_t);
      // floor(2^40 w) in two words: w 2^20 and what its whole part leaves are exact
      const float w = __fmul_rn(expf(z[j]), 1048576.f);              // exp(-inf) = 0
      hi[j] = __float2uint_rz(w);
      lo[j] = __float2uint_rz(__fmul_rn(__fsub_rn(w, __uint2float_rn(hi[j])), 1048576.f));
    }
  }
  // top-k (0: off), top-p (thr: the mass to reach, 0: that share of what top-k left) and min-p, in that order
  __device__ __forceinline__ void filter(int k, float top_p, double thr, float min_p, uint32_t top) {
    if (__any_sync(M32_ALL, k > 1)) cut<false>(k > 1, k);
    if (__any_sync(M32_ALL, k == 1)) {           // the first of the largest
      bool taken = false;
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const uint32_t tie = G::ballot(key[j] == top);
        if (k == 1 && (key[j] != top || taken || (tie & G::below()) != 0)) hi[j] = lo[j] = 0;
        taken = taken || tie != 0;
      }
    }
    if (__any_sync(M32_ALL, top_p < 1.f)) {
      // every sum is exact in a double, so x >= threshold is x >= its ceiling in integers
      const long long total = mass_from(-Z_SPAN);
      cut<true>(top_p < 1.f && total > 0, __double2ll_ru(thr == 0.0 ? p_threshold(top_p, total) : thr));
    }
    if (min_p > 0.f)
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (expf(z[j]) < min_p && key[j] != top) hi[j] = lo[j] = 0;     // the first element always stays
  }
  // the element drawn (-1: there is none), its z, and the kept mass
  __device__ __forceinline__ int draw(float u, float& z_out, long long& total) const {
    total = mass_from(-Z_SPAN);
    long long at = draw_at(u, total);
    int token = -1;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      uint32_t h = hi[j], l = lo[j];
#pragma unroll
      for (int o = 1; o < GW; o <<= 1) {
        const uint32_t vh = __shfl_up_sync(M32_ALL, h, o, GW), vl = __shfl_up_sync(M32_ALL, l, o, GW);
        if (G::lane() >= o) {
          h += vh;
          l += vl;
        }
      }
      const long long run = mass_of(h, l);
      const uint32_t over = G::ballot(run > at);
      const int src = over ? __ffs(over) - 1 : 0;
      const float zj = G::get(z[j], src);
      if (token < 0 && over != 0) {
        token = j * GW + src;
        z_out = zj;
      }
      at -= G::get(run, GW - 1);
      if (j + 1 < EPL && __all_sync(M32_ALL, token >= 0)) break;
    }
    return token;
  }
};

// A group takes `rows` rows, one after another: its lane i holds the settings of the i-th and finishes it (the logarithm)
// with the others
template <typename T, int GW, int EPL>
__global__ void __launch_bounds__(128) sample_warp_kernel(InbSampleArgs a, int rows) {
  using G = Group<GW>;
  constexpr int GROUPS = 32 / GW;
  const int lane = G::lane();
  const int64_t warp_first = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * rows * GROUPS;
  if (warp_first >= a.N) return;
  const int64_t first = warp_first + (threadIdx.x & 31) / GW * rows;      // of this group
  const int n = first >= a.N ? 0 : (a.N - first < rows ? (int)(a.N - first) : rows);
  RowParams mine = {1.f, 1.f, 0.f, 0.f, 0};
  if (lane < n) mine = row_params(a, first + lane);
  int my_token = -1;
  float my_z = 0.f;
  long long my_total = 0;
  const T* lp = (const T*)a.logits + first * a.ld + lane;
  const uint8_t* mp = a.mask ? a.mask + first * a.ld_mask + lane : nullptr;
  T next[EPL];
  bool ok[EPL];
  auto fetch = [&](bool on) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      ok[j] = on && j * GW + lane < a.V;
      if (ok[j]) {
        next[j] = lp[j * GW];
        if (mp) ok[j] = mp[j * GW] != 0;
      }
    }
    lp += a.ld;
    if (mp) mp += a.ld_mask;
  };
  fetch(n > 0);
#pragma unroll 1
  for (int r = 0; r < rows; ++r) {
    WarpRow<GW, EPL> R;
    uint32_t top = KEY_NEG_INF;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      R.z[j] = clean(ok[j] ? to_f(next[j]) : 0.f, ok[j]);
      R.key[j] = key_of(R.z[j]);
      top = max(top, R.key[j]);
    }
    if (r + 1 < rows) fetch(r + 1 < n);
    top = G::max_of(top);
    const int k = G::get(mine.k, r);
    R.weigh(of_key(top), G::get(mine.inv_t, r));
    R.filter(k < a.V ? k : 0, G::get(mine.top_p, r), 0.0, G::get(mine.min_p, r), top);
    float z = 0.f;
    long long total;
    const int token = R.draw(G::get(mine.u, r), z, total);
    if (lane == r) {
      my_token = token;
      my_z = z;
      my_total = total;
    }
  }
  if (lane < n) {
    a.token[first + lane] = my_token;
    a.logp[first + lane] = my_token < 0 ? -INFINITY : logp_of(my_z, my_total);
  }
}

template <typename T, int GW, int EPL>
static int warp_launch(const InbSampleArgs& a, cudaStream_t s) {
  // a group takes one row while the SMs' 64 warps are not all busy, and up to 8 then
  constexpr int GROUPS = 32 / GW;
  int64_t rows = a.N / ((int64_t)sm_count() * 64 * GROUPS);
  rows = rows < 1 ? 1 : (rows > 8 ? 8 : rows);
  const int64_t per = 4 * rows * GROUPS;
  sample_warp_kernel<T, GW, EPL><<<(unsigned)((a.N + per - 1) / per), 128, 0, s>>>(a, (int)rows);
  return launch_status();
}

// ------------------------------------------------------------------------------------- a block or cluster per row
// What the blocks of a cluster exchange (read through distributed shared memory)
struct Exchange {
  uint32_t umax, umin;
  long long mass;
};

template <int NT>
struct BlockState {
  static constexpr int BINS = 2 * NT, LIST = 4 * NT;
  uint32_t cnt[BINS];                      // histogram: elements, and their mass where it is asked for
  unsigned long long mass[BINS];
  float lv[LIST];                          // the elements that can be kept, by index, where they are few
  int li[LIST];
  Exchange ex[2];                          // alternated, see all_reduce
  uint32_t wu[32], wt[32];
  long long wm[32];
  uint32_t f_bin, f_cnt_above, f_count, f_key;
  long long f_mass_above;
};

// Which of a vector's elements are at least `least`, one bit each
template <int W>
__device__ __forceinline__ uint32_t ge_bits(const Pack<float, W>& v, float least) {
  uint32_t b = 0;
#pragma unroll
  for (int e = 0; e < W; ++e) b |= (uint32_t)(v.v[e] >= least) << e;
  return b;
}
template <int W>
__device__ __forceinline__ uint32_t ge_bits(const Pack<bf16, W>& v, float least) {
  const __nv_bfloat162 t = __bfloat162bfloat162(__float2bfloat16_ru(least));      // l >= least is l >= the next bf16 up
  uint32_t b = 0;
#pragma unroll
  for (int e = 0; e < W; e += 2) {
    const uint32_t m = __hge2_mask(__halves2bfloat162(v.v[e], v.v[e + 1]), t);
    b |= (m & (1u << e)) | ((m >> 16) & (2u << e));
  }
  return b;
}
template <int W>
__device__ __forceinline__ uint32_t ge_bits(const Pack<f16, W>& v, float least) {
  const __half2 t = __half2half2(__float2half_ru(least));
  uint32_t b = 0;
#pragma unroll
  for (int e = 0; e < W; e += 2) {
    const uint32_t m = __hge2_mask(__halves2half2(v.v[e], v.v[e + 1]), t);
    b |= (m & (1u << e)) | ((m >> 16) & (2u << e));
  }
  return b;
}
// The larger of each element, a number before a NaN
template <int W>
__device__ __forceinline__ void keep_max(Pack<float, W>& a, const Pack<float, W>& v) {
#pragma unroll
  for (int e = 0; e < W; ++e) a.v[e] = fmaxf(a.v[e], v.v[e]);
}
template <int W>
__device__ __forceinline__ void keep_max(Pack<bf16, W>& a, const Pack<bf16, W>& v) {
#pragma unroll
  for (int e = 0; e < W; e += 2) {
    const __nv_bfloat162 m = __hmax2(__halves2bfloat162(a.v[e], a.v[e + 1]), __halves2bfloat162(v.v[e], v.v[e + 1]));
    a.v[e] = m.x;
    a.v[e + 1] = m.y;
  }
}
template <int W>
__device__ __forceinline__ void keep_max(Pack<f16, W>& a, const Pack<f16, W>& v) {
#pragma unroll
  for (int e = 0; e < W; e += 2) {
    const __half2 m = __hmax2(__halves2half2(a.v[e], a.v[e + 1]), __halves2half2(v.v[e], v.v[e + 1]));
    a.v[e] = m.x;
    a.v[e + 1] = m.y;
  }
}

// The smaller of each element, +inf in place of -inf and a number before a NaN
template <int W>
__device__ __forceinline__ void keep_min(Pack<float, W>& a, const Pack<float, W>& v) {
#pragma unroll
  for (int e = 0; e < W; ++e) a.v[e] = fminf(a.v[e], v.v[e] == -INFINITY ? INFINITY : v.v[e]);
}
template <typename T, int W>
__device__ __forceinline__ void keep_min(Pack<T, W>& a, const Pack<T, W>& v) {
  constexpr uint32_t INF = std::is_same<T, bf16>::value ? 0x7F807F80u : 0x7C007C00u, SIGN = 0x80008000u;
  using Two = typename std::conditional<std::is_same<T, bf16>::value, __nv_bfloat162, __half2>::type;
  const uint32_t* vw = reinterpret_cast<const uint32_t*>(&v);
  uint32_t* aw = reinterpret_cast<uint32_t*>(&a);
#pragma unroll
  for (int e = 0; e < W / 2; ++e) {
    const uint32_t none = INF | SIGN, w = vw[e];
    const uint32_t at = __heq2_mask(*reinterpret_cast<const Two*>(&w), *reinterpret_cast<const Two*>(&none));
    const uint32_t up = w ^ (at & SIGN);
    const Two m = __hmin2(*reinterpret_cast<const Two*>(&aw[e]), *reinterpret_cast<const Two*>(&up));
    aw[e] = *reinterpret_cast<const uint32_t*>(&m);
  }
}

// Elements that a slice of `len` takes in shared memory: it is filled up with -inf to a whole 16-byte access
template <typename T>
__host__ __device__ constexpr int padded(int len) {
  constexpr int W = 16 / (int)sizeof(T);
  return (len + W - 1) / W * W;
}

// A 64-bit sum in shared memory by 32-bit atomics, which it has natively: low word, then high word with the carry
__device__ __forceinline__ void add_mass(unsigned long long& sum, long long q) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&sum);
  const uint32_t ql = (uint32_t)q, old = atomicAdd(w, ql), qh = (uint32_t)(q >> 32) + (old + ql < old ? 1u : 0u);
  if (qh != 0) atomicAdd(w + 1, qh);
}

// The row (or, once `list` is set, the list of its candidates in the first block) as the passes see it
template <typename T, int NT, bool RES>
struct Row {
  static constexpr int BINS = 2 * NT, LIST = 4 * NT, LOG_BINS = NT == 128 ? 8 : 10, W = 16 / (int)sizeof(T);
  static constexpr int RANKS = NT == 128 ? 1 : 8;      // the most blocks a row takes; loads from all come before their uses
  const InbSampleArgs& a;
  BlockState<NT>& s;
  T* buf;
  int64_t row;
  int first, len;      // this block's slice
  int ranks, rank;
  float m, inv_t;
  bool list;
  int par;
  // bins of the histogram over z to a unit of z.  They span what the row's own logits span: where those hardly differ a
  // fixed span puts all in one bin (64 x 131072, top-k 1000, top-p 0.9: 216 us, not 33).
  float bins;

  __device__ __forceinline__ float at(int i) const {
    if (list) return s.lv[i];
    if (RES) return to_f(buf[i]) + 0.f;      // -0 counts as +0; a NaN stays one and compares as out of every range
    return clean(to_f(((const T*)a.logits)[row * a.ld + first + i]),
                 a.mask == nullptr || a.mask[row * a.ld_mask + first + i] != 0);
  }
  __device__ __forceinline__ int index(int i) const { return list ? s.li[i] : first + i; }
  __device__ __forceinline__ float z(float l) const { return z_of(l, m, inv_t); }
  __device__ __forceinline__ int z_bin(float z) const { return min(BINS - 1, (int)(-z * bins)); }
  __device__ __forceinline__ void sync() {
    if (ranks > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }
  __device__ __forceinline__ BlockState<NT>* peer(int r) {
    return ranks > 1 ? cg::this_cluster().map_shared_rank(&s, r) : &s;
  }
  // max, min and mass over the row; every thread gets them.  `ex` alternates between two slots, so the one
  // barrier after the write also keeps a slot from being rewritten before every block has read it.
  __device__ Exchange all_reduce(uint32_t umax, uint32_t umin, long long mass, bool with_mass) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    umax = __reduce_max_sync(M32_ALL, umax);
    umin = __reduce_min_sync(M32_ALL, umin);
    if (with_mass)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(M32_ALL, mass, o);
    __syncthreads();
    if (lane == 0) {
      s.wu[wid] = umax;
      s.wt[wid] = umin;
      s.wm[wid] = mass;
    }
    __syncthreads();
    par ^= 1;
    if (threadIdx.x < 32) {
      umax = __reduce_max_sync(M32_ALL, lane < NT / 32 ? s.wu[lane] : 0u);
      umin = __reduce_min_sync(M32_ALL, lane < NT / 32 ? s.wt[lane] : M32_ALL);
      if (with_mass) {
        mass = lane < NT / 32 ? s.wm[lane] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(M32_ALL, mass, o);
      }
      if (lane == 0) {
        s.ex[par].umax = umax;
        s.ex[par].umin = umin;
        s.ex[par].mass = mass;
      }
    }
    sync();
    Exchange e = s.ex[par];
    if (ranks > 1) {                          // a lane reads a block's
      e = peer(lane < ranks ? lane : rank)->ex[par];
      e.umax = __reduce_max_sync(M32_ALL, e.umax);
      e.umin = __reduce_min_sync(M32_ALL, e.umin);
      if (with_mass) {
        if (lane >= ranks) e.mass = 0;
#pragma unroll
        for (int o = RANKS / 2; o > 0; o >>= 1) e.mass += __shfl_xor_sync(M32_ALL, e.mass, o);
        e.mass = __shfl_sync(M32_ALL, e.mass, 0);
      }
    }
    return e;
  }
  __device__ void clear() {
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += NT) {
      s.cnt[b] = 0;
      s.mass[b] = 0;
    }
    __syncthreads();
  }
  // Histogram over z of each thread's largest logit: the k-th of them is at most the k-th of the row
  __device__ void fill_best(float best) {
    clear();
    const float zi = z(best);
    if (zi > -Z_SPAN && q_of(expf(zi)) > 0) atomicAdd(&s.cnt[z_bin(zi)], 1u);
  }
  // Histogram over z of the elements that have a mass; with_mass: their masses too, whose sum (this thread's) it returns
  __device__ long long fill(bool with_mass) {
    clear();
    long long sum = 0;
    for (int i = threadIdx.x; i < len; i += NT) {
      const float zi = z(at(i));
      if (zi > -Z_SPAN) {
        if (with_mass) {
          const long long q = q_of(expf(zi));
          if (q > 0) {
            atomicAdd(&s.cnt[z_bin(zi)], 1u);
            add_mass(s.mass[z_bin(zi)], q);
            sum += q;
          }
        } else if (zi > -Z_SURE || q_of(expf(zi)) > 0) {
          atomicAdd(&s.cnt[z_bin(zi)], 1u);
        }
      }
    }
    return sum;
  }
  // Over the histogram of the row (bin 0 = largest logits): the first bin at which the count (by_mass false) or the mass
  // reaches the target, given what lies above the histogram.  False: no bin does.
  __device__ bool cross(bool by_mass, uint32_t k, double thr, uint32_t& cnt_above, long long& mass_above, uint32_t& bin,
                        uint32_t& count) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, b = 2 * threadIdx.x;
    __syncthreads();                          // the last call's result has been read
    if (threadIdx.x == 0) s.f_bin = M32_ALL;
    sync();                                   // every block's histogram is complete
    uint32_t c[2] = {s.cnt[b], s.cnt[b + 1]};
    long long q[2] = {(long long)s.mass[b], (long long)s.mass[b + 1]};
#pragma unroll 1
    for (int r0 = 1; r0 < ranks; r0 += 4) {       // the others, four at a time
      uint2 pc[4];
      ulonglong2 pq[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const BlockState<NT>* o = peer(r0 + i < ranks ? (rank + r0 + i) % ranks : rank);
        pc[i] = *reinterpret_cast<const uint2*>(&o->cnt[b]);
        pq[i] = *reinterpret_cast<const ulonglong2*>(&o->mass[b]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + i < ranks) {
          c[0] += pc[i].x, c[1] += pc[i].y;
          q[0] += (long long)pq[i].x, q[1] += (long long)pq[i].y;
        }
    }
    uint32_t ci = c[0] + c[1];
    long long qi = q[0] + q[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t vc = __shfl_up_sync(M32_ALL, ci, o);
      const long long vq = __shfl_up_sync(M32_ALL, qi, o);
      if (lane >= o) {
        ci += vc;
        qi += vq;
      }
    }
    if (lane == 31) {
      s.wu[wid] = ci;
      s.wm[wid] = qi;
    }
    __syncthreads();
    uint32_t ca = cnt_above + ci - c[0] - c[1];
    long long qa = mass_above + qi - q[0] - q[1];
    for (int i = 0; i < wid; ++i) {
      ca += s.wu[i];
      qa += s.wm[i];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool was = by_mass ? __ll2double_rn(qa) >= thr : ca >= k;
      const bool is = by_mass ? __ll2double_rn(qa + q[i]) >= thr : ca + c[i] >= k;
      if (is && !was) {
        s.f_bin = b + i;
        s.f_cnt_above = ca;
        s.f_mass_above = qa;
        s.f_count = c[i];
      }
      ca += c[i];
      qa += q[i];
    }
    sync();                                   // every block has read the histograms, and this one's result is there
    bin = s.f_bin;
    if (bin == M32_ALL) return false;
    cnt_above = s.f_cnt_above;
    mass_above = s.f_mass_above;
    count = s.f_count;
    return true;
  }
  // The smallest key whose element lies in z bins 0 .. bin: z_bin falls with the key, so a warp finds it in seven rounds
  // of 32 probes.
  __device__ uint32_t bin_floor(uint32_t bin) {
    if (threadIdx.x < 32) {
      uint32_t lo = KEY_NEG_INF, hi = key_of(m);          // lo does not lie there, hi does
      while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 31) / 32;
        const uint64_t probe = (uint64_t)lo + (uint64_t)step * (threadIdx.x + 1);
        bool in = true;
        if (probe < hi) {
          const float zi = z(of_key((uint32_t)probe));
          in = zi > -Z_SPAN && z_bin(zi) <= (int)bin;
        }
        const int f = __ffs(__ballot_sync(M32_ALL, in));     // the last probe is at or above hi: one is in
        const uint64_t up = (uint64_t)lo + (uint64_t)step * f;
        lo = lo + step * (f - 1);
        hi = up < hi ? (uint32_t)up : hi;
      }
      if (threadIdx.x == 0) s.f_key = hi;
    }
    __syncthreads();
    return s.f_key;
  }
  // The run of the slice that a warp owns: whole accesses of 32 lanes
  __device__ __forceinline__ void run(int& s0, int& s1) const {
    constexpr int nw = NT / 32, unit = RES ? 32 * W : 32;
    const int seg = (len + nw * unit - 1) / (nw * unit) * unit, wid = threadIdx.x >> 5;
    s0 = min(len, wid * seg);
    s1 = min(len, s0 + seg);
  }
  // Which of the W (RES) or 1 elements from i on are at least `least`, one bit each
  __device__ __forceinline__ uint32_t at_least(int i, int end, float least) const {
    if (!RES) return i < end && at(i) >= least;
    if (i >= end) return 0;
    const Pack<T, W> v = ld<T, W>(buf + i);           // what lies beyond the slice is -inf
    return ge_bits(v, least);
  }
  // Moves the elements from key `floor` up to the first block's list, by index.  0: they are more than the list holds and
  // nothing was moved; 1: moved, and this is the first block; 2: moved, and this block is done.
  __device__ int gather(uint32_t floor) {
    constexpr int STEP = RES ? W : 1;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const float least = of_key(floor);
    int s0, s1;
    run(s0, s1);
    uint32_t n = 0;
    for (int i = s0 + lane * STEP; i < s1; i += 32 * STEP) n += __popc(at_least(i, s1, least));
    n = __reduce_add_sync(M32_ALL, n);
    if (lane == 0) s.wt[wid] = n;
    sync();
    uint32_t before = 0, total = 0, v[RANKS];
#pragma unroll
    for (int r = 0; r < RANKS; ++r) v[r] = lane < NT / 32 ? peer(r < ranks ? r : rank)->wt[lane] : 0u;
#pragma unroll
    for (int r = 0; r < RANKS; ++r)
      if (r < ranks) {
        total += v[r];
        before += r < rank || (r == rank && lane < wid) ? v[r] : 0u;
      }
    total = __reduce_add_sync(M32_ALL, total);
    before = __reduce_add_sync(M32_ALL, before);
    if (total > (uint32_t)LIST) {
      sync();           // the counts have been read
      return 0;
    }
    BlockState<NT>* to = peer(0);
    if (n > 0)
      for (int i0 = s0; i0 < s1; i0 += 32 * STEP) {
        const int i = i0 + lane * STEP;
        uint32_t bits = at_least(i, s1, least);
        if (__ballot_sync(M32_ALL, bits != 0) == 0) continue;
        const uint32_t c = __popc(bits);
        uint32_t slot = c;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const uint32_t v = __shfl_up_sync(M32_ALL, slot, d);
          if (lane >= d) slot += v;
        }
        const uint32_t all = __shfl_sync(M32_ALL, slot, 31);
        slot += before - c;
        for (; bits != 0; bits &= bits - 1, ++slot) {
          const int e = i + __ffs(bits) - 1;
          to->lv[slot] = at(e);
          to->li[slot] = first + e;
        }
        before += all;
      }
    sync();
    if (rank != 0) return 2;
    list = true;
    len = (int)total;
    ranks = 1;
    return 1;
  }
  // With the histogram filled (and `crossed`: its bin found): the value tau at which the target is reached, how many hold
  // it, and what lies above it.
  __device__ bool find(bool by_mass, uint32_t k, double thr, bool crossed, uint32_t bin, uint32_t& tau, uint32_t& count,
                       uint32_t& cnt_above, long long& mass_above) {
    if (!crossed) {
      cnt_above = 0;
      mass_above = 0;
      if (!cross(by_mass, k, thr, cnt_above, mass_above, bin, count)) return false;
    }
    // the keys of that bin: what its elements span (a short pass over a list), or all that fall there
    uint32_t lo = M32_ALL, hi = 0;
    if (list) {
      for (int i = threadIdx.x; i < len; i += NT) {
        const float l = at(i), zi = z(l);
        if (zi > -Z_SPAN && z_bin(zi) == (int)bin && q_of(expf(zi)) > 0) {
          hi = max(hi, key_of(l));
          lo = min(lo, key_of(l));
        }
      }
      const Exchange e = all_reduce(hi, lo, 0, false);
      hi = e.umax;
      lo = e.umin;
    } else {
      lo = bin_floor(bin);
      __syncthreads();                        // f_key has been read
      hi = bin > 0 ? bin_floor(bin - 1) - 1 : key_of(m);
    }
    // the low bits of a 16-bit type's keys are all 0 or all 1 and decide nothing
    constexpr int LOW = sizeof(T) == 4 ? 0 : (std::is_same<T, bf16>::value ? 16 : 13);
    const uint32_t least = lo, most = hi;
    lo >>= LOW;
    hi >>= LOW;
    while (hi != lo) {
      const int bits = 32 - __clz(hi - lo), shift = max(0, bits - LOG_BINS);
      clear();
      for (int i = threadIdx.x; i < len; i += NT) {
        const float l = at(i);
        const uint32_t full = key_of(l), key = full >> LOW;
        if (full >= least && full <= most && key >= lo && key <= hi) {
          const long long q = q_of(expf(z(l)));
          if (q > 0) {
            const uint32_t b = (hi - key) >> shift;
            atomicAdd(&s.cnt[b], 1u);
            add_mass(s.mass[b], q);
          }
        }
      }
      cross(by_mass, k, thr, cnt_above, mass_above, bin, count);   // the target lies within: a bin is found
      hi = hi - (bin << shift);
      const uint32_t span = (1u << shift) - 1u;
      lo = hi - lo > span ? hi - span : lo;
    }
    tau = hi << LOW;
    if ((tau & 0x80000000u) == 0) tau |= (1u << LOW) - 1u;
    return true;
  }
};

// What costs here is the latency of the passes between barriers, so 64 registers: with 100, one block an SM less, 64 rows of
// 131072 (top-k 1000, top-p 0.9) take 48 us, not 34.
template <typename T, int NT, bool RES>
__global__ void __launch_bounds__(NT, 1024 / NT) sample_block_kernel(InbSampleArgs a, int ranks, int slice) {
  extern __shared__ __align__(16) unsigned char dyn[];
  BlockState<NT>& s = *reinterpret_cast<BlockState<NT>*>(dyn);
  constexpr int STATE = (sizeof(BlockState<NT>) + 15) / 16 * 16;
  T* buf = reinterpret_cast<T*>(dyn + STATE);
  const int64_t row = (int64_t)blockIdx.x / ranks;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int own = (int)(blockIdx.x % ranks);       // clusters are consecutive blocks: also the rank in the cluster
  const int first = own * slice;
  int len = a.V - first;
  len = len < 0 ? 0 : (len > slice ? slice : len);
  const RowParams p = row_params(a, row);
  Row<T, NT, RES> R{a, s, buf, row, first, len, ranks, own, 0.f, p.inv_t, false, 0, 0.f};
  const bool select_k = p.k > 0 && p.k < a.V, select_p = p.top_p < 1.f;

  // the slice, and the row's largest logit
  float best = -INFINITY, low = INFINITY;      // the largest of this thread's elements, and the smallest that is not -inf
  if (RES) {
    const T* lp = (const T*)a.logits + row * a.ld + first;
    const uint8_t* mp = a.mask ? a.mask + row * a.ld_mask + first : nullptr;
    constexpr int W = 16 / (int)sizeof(T);
    const T none = from_f<T>(-INFINITY);
    int i0 = 0;
    if (((uintptr_t)lp & 15) == 0 && ((uintptr_t)mp & (W - 1)) == 0) {
      i0 = len / W * W;
      Pack<T, W> most, least;
#pragma unroll
      for (int e = 0; e < W; ++e) most.v[e] = none, least.v[e] = from_f<T>(INFINITY);
#pragma unroll 4
      for (int i = threadIdx.x * W; i < i0; i += NT * W) {
        Pack<T, W> v = ld<T, W>(lp + i);
        if (mp) {
          const Pack<uint8_t, W> ok = ld<uint8_t, W>(mp + i);
#pragma unroll
          for (int e = 0; e < W; ++e)
            if (ok.v[e] == 0) v.v[e] = none;
        }
        keep_max(most, v);
        keep_min(least, v);
        st<T, W>(buf + i, v);
      }
#pragma unroll
      for (int e = 0; e < W; ++e) best = fmaxf(best, to_f(most.v[e])), low = fminf(low, to_f(least.v[e]));
    }
    // the rest, and -inf up to a whole access
    for (int i = i0 + threadIdx.x; i < padded<T>(len); i += NT) {
      const T l = i < len && (mp == nullptr || mp[i] != 0) ? lp[i] : none;
      best = fmaxf(best, to_f(l));
      if (to_f(l) > -INFINITY) low = fminf(low, to_f(l));
      buf[i] = l;
    }
    best += 0.f;
  } else {
    for (int i = threadIdx.x; i < len; i += NT) {
      const float l = R.at(i);
      best = fmaxf(best, l);
      if (l > -INFINITY) low = fminf(low, l);
    }
  }
  const Exchange ends = R.all_reduce(key_of(best), key_of(low), 0, false);
  const uint32_t top = ends.umax;
  if (top <= KEY_NEG_INF) {
    if (own == 0 && threadIdx.x == 0) {
      a.token[row] = -1;
      a.logp[row] = -INFINITY;
    }
    R.sync();           // no block leaves while another may still read its shared memory
    return;
  }
  const float m = of_key(top);
  R.m = m;
  const float span = fminf(Z_SPAN, -R.z(of_key(ends.umin)));
  R.bins = R.BINS / (span > 1e-30f ? span : Z_SPAN);
  if (p.k == 1) {       // the first of the largest
    uint32_t i1 = M32_ALL;
    for (int i = threadIdx.x; i < R.len; i += NT)
      if (R.at(i) == m) i1 = min(i1, (uint32_t)(first + i));
    i1 = R.all_reduce(0, i1, 0, false).umin;
    if (own == 0 && threadIdx.x == 0) {
      a.token[row] = i1;
      a.logp[row] = 0.f;
    }
    R.sync();
    return;
  }

  // the cut-off (tau, kept): elements above tau stay, and the first `kept` of those equal to it
  uint32_t tau = 0, kept = 0;
  if (select_k || select_p) {
    uint32_t count, above = 0, bin = 0;
    long long total = 0, mass_above = 0;
    double thr = 0.0;
    bool crossed = false;
    if (select_k) {
      // the k-th of the threads' largest bounds the k-th of the row from below: what lies above it is few enough, or else
      // the k-th bin of every element is looked for
      R.fill_best(best);
      int done = R.cross(false, (uint32_t)p.k, 0.0, above, mass_above, bin, count) ? R.gather(R.bin_floor(bin)) : 0;
      if (done == 0) {
        above = 0;
        R.fill(false);
        if (R.cross(false, (uint32_t)p.k, 0.0, above, mass_above, bin, count) && above + count <= (uint32_t)R.LIST)
          done = R.gather(R.bin_floor(bin));
      }
      if (done == 2) return;
    } else {
      total = R.all_reduce(0, M32_ALL, R.fill(true), true).mass;
      thr = p_threshold(p.top_p, total);
      crossed = R.cross(true, 0, thr, above, mass_above, bin, count);
      if (crossed && above + count <= (uint32_t)R.LIST && R.gather(R.bin_floor(bin)) == 2) return;
    }
    if (R.list && R.len <= 128) {        // few enough for one warp
      if (wid > 0) return;
      WarpRow<32, 4> w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = j * 32 + lane;
        w.z[j] = i < R.len ? s.lv[i] : -INFINITY;
        w.key[j] = key_of(w.z[j]);
      }
      w.weigh(m, p.inv_t);
      w.filter(select_k ? p.k : 0, p.top_p, thr, p.min_p, top);
      float z;
      long long kept_mass;
      const int i = w.draw(p.u, z, kept_mass);
      if (lane == 0) {
        a.token[row] = s.li[i];
        a.logp[row] = logp_of(z, kept_mass);
      }
      return;
    }
    if (select_k || R.list) {
      const long long sum = R.fill(true);
      if (select_k) total = R.all_reduce(0, M32_ALL, sum, true).mass;     // stays if fewer than k have a mass
    }
    if (select_k && R.find(false, (uint32_t)p.k, 0.0, false, 0, tau, count, above, mass_above)) {
      kept = (uint32_t)p.k - above;
      total = mass_above + (long long)kept * q_of(expf(R.z(of_key(tau))));
      if (select_p) R.fill(true);
    }
    if (select_p) {
      if (select_k) thr = p_threshold(p.top_p, total);
      uint32_t tp;
      if (R.find(true, 0, thr, crossed && !R.list, bin, tp, count, above, mass_above)) {
        tau = tp;
        kept = ties_kept(mass_above, q_of(expf(R.z(of_key(tau)))), count, thr);
      }
    }
  }

  // the kept mass of each warp's run, by index
  constexpr int nw = NT / 32;
  int s0, s1;
  R.run(s0, s1);
  const float w_tau = expf(R.z(of_key(tau)));
  const long long q_tau = tau == 0 || (w_tau < p.min_p && tau != top) ? 0 : q_of(w_tau);
  long long mass = 0;
  uint32_t ties = 0;
  for (int i = s0 + lane; i < s1; i += 32) {
    const float l = R.at(i);
    const uint32_t key = key_of(l);
    if (key == tau) {
      ++ties;
    } else if (key > tau) {
      const float z = R.z(l);
      if (z > -Z_SPAN) {
        const float w = expf(z);
        if (!(w < p.min_p) || key == top) mass += q_of(w);
      }
    }
  }
  ties = __reduce_add_sync(M32_ALL, ties);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(M32_ALL, mass, o);
  R.sync();
  if (lane == 0) {
    s.wt[wid] = ties;
    s.wm[wid] = mass;
  }
  R.sync();
  // every warp: the mass of the row, what comes before its own run, and the ties before it
  long long total = 0, before = 0;
  uint32_t seen = 0, my_seen = 0, pt[R.RANKS];
  long long pv[R.RANKS];
#pragma unroll
  for (int r = 0; r < R.RANKS; ++r) {
    const BlockState<NT>* o = R.peer(r < R.ranks ? r : R.rank);
    pt[r] = lane < nw ? o->wt[lane] : 0u;
    pv[r] = lane < nw ? o->wm[lane] : 0;
  }
#pragma unroll
  for (int r = 0; r < R.RANKS; ++r) {
    if (r >= R.ranks) break;
    uint32_t t = pt[r], ti = t;
    long long v = pv[r];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t x = __shfl_up_sync(M32_ALL, ti, d);
      if (lane >= d) ti += x;
    }
    const uint32_t tb = seen + ti - t;                                    // ties before warp `lane` of rank r
    const uint32_t here = tb >= kept ? 0u : min(t, kept - tb);
    v += (long long)here * q_tau;
    long long vi = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long x = __shfl_up_sync(M32_ALL, vi, d);
      if (lane >= d) vi += x;
    }
    if (r == R.rank) {
      before = total + __shfl_sync(M32_ALL, vi - v, wid);
      my_seen = __shfl_sync(M32_ALL, tb, wid);
      mass = __shfl_sync(M32_ALL, v, wid);
    }
    total += __shfl_sync(M32_ALL, vi, 31);
    seen += __shfl_sync(M32_ALL, ti, 31);
  }
  R.sync();             // no block leaves while another may still read its shared memory
  const long long at = draw_at(p.u, total);
  if (at < before || at >= before + mass) return;
  long long run = before;
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    uint32_t key = 0;
    float z = -INFINITY;
    long long q = 0;
    if (i < s1) {
      const float l = R.at(i);
      key = key_of(l);
      z = R.z(l);
      if (key > tau && z > -Z_SPAN) {
        const float w = expf(z);
        if (!(w < p.min_p) || key == top) q = q_of(w);
      }
    }
    const uint32_t tie = __ballot_sync(M32_ALL, i < s1 && key == tau);
    if (i < s1 && key == tau && my_seen + __popc(tie & ((1u << lane) - 1u)) < kept) q = q_tau;
    my_seen += __popc(tie);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long x = __shfl_up_sync(M32_ALL, q, d);
      if (lane >= d) q += x;
    }
    const uint32_t over = __ballot_sync(M32_ALL, run + q > at);
    if (over != 0) {
      if (lane == __ffs(over) - 1) {
        a.token[row] = R.index(i);
        a.logp[row] = logp_of(z, total);
      }
      return;
    }
    run += __shfl_sync(M32_ALL, q, 31);
  }
}

constexpr int SMEM_MOST = 227 * 1024;

template <typename T, int NT, bool RES>
static int block_launch(const InbSampleArgs& a, int ranks, int slice, cudaStream_t s) {
  const size_t smem = (sizeof(BlockState<NT>) + 15) / 16 * 16 + (RES ? (size_t)padded<T>(slice) * sizeof(T) : 0);
  auto* k = sample_block_kernel<T, NT, RES>;
  cudaError_t e;
  if (smem > 48 * 1024) {
    e = allow_smem<KernelKey<sample_block_kernel<T, NT, RES>>>((const void*)k, SMEM_MOST);
    if (e != cudaSuccess) return -100 - (int)e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.N * ranks));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = ranks;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, k, a, ranks, slice);
  return e == cudaSuccess ? 0 : -100 - (int)e;
}

template <typename T>
static int sample_type(const InbSampleArgs& a, cudaStream_t s) {
  // lanes of a row: fewer make a row's fixed work cheaper and its steps longer.  131072 rows, top-p 0.95: V = 16 31 us with
  // 8 lanes, 60 with 32; V = 33 74 with 16, 79 with 32; V = 64 110 with 16, 90 with 32.
  // A warp a row against a block: 32768 rows, top-k 50: V = 200 80 us and 255, V = 384 138 and 187; one row, top-p 0.95:
  // V = 256 8 and 15.  Beyond, a lane's elements outgrow its registers (V = 512, top-k 50: 249 and 189).
  if (a.V <= 8) return warp_launch<T, 8, 1>(a, s);
  if (a.V <= 16) return warp_launch<T, 8, 2>(a, s);
  if (a.V <= 32) return warp_launch<T, 16, 2>(a, s);
  if (a.V <= 48) return warp_launch<T, 16, 3>(a, s);
  if (a.V <= 64) return warp_launch<T, 32, 2>(a, s);
  if (a.V <= 128) return warp_launch<T, 32, 4>(a, s);
  if (a.V <= 256) return warp_launch<T, 32, 8>(a, s);
  if (a.V <= 384) return warp_launch<T, 32, 12>(a, s);
  // threads of a block: top-p 0.9 after top-k 1000, 6 rows: V = 1000 19 us with 128 and 17 with 512, V = 2026 35 and 23,
  // V = 4000 52 and 23; 250 rows: V = 1000 21 and 21, V = 2026 41 and 29.  With more rows than the SMs take of the large
  // blocks at a time the small ones keep more rows in flight.
  if (a.V <= 1536 || (a.V <= 4096 && a.N > 2 * sm_count())) return block_launch<T, 128, true>(a, 1, a.V, s);
  // blocks of a row: enough to give every SM one while a slice keeps 4096 logits, and enough for the row to be resident
  constexpr int CAP = (SMEM_MOST - (int)((sizeof(BlockState<512>) + 15) / 16 * 16)) / (int)sizeof(T) / 16 * 16;
  int ranks = 1;
  while (ranks < 8 && (a.N * ranks < sm_count() || (a.V + ranks - 1) / ranks > CAP) && a.V / (2 * ranks) >= 4096)
    ranks *= 2;
  const int slice = ((a.V + ranks - 1) / ranks + 15) / 16 * 16;
  if (slice <= CAP) return block_launch<T, 512, true>(a, ranks, slice, s);
  return block_launch<T, 512, false>(a, ranks, slice, s);
}

}  // namespace pol
}  // namespace inb

extern "C" int inb_sample(const InbSampleArgs* args, void* cuda_stream) {
  if (args == nullptr) return -1;
  const InbSampleArgs& a = *args;
  if (a.dtype < 0 || a.dtype > 2 || a.N < 0 || a.N > INB_MAX_SAMPLE_N || a.V < 1 || a.V > INB_MAX_SAMPLE_V) return -2;
  if (a.N == 0) return 0;
  if (a.logits == nullptr || a.u == nullptr || a.token == nullptr || a.logp == nullptr) return -3;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (a.dtype == INB_BF16) return inb::pol::sample_type<inb::pol::bf16>(a, s);
  if (a.dtype == INB_F16) return inb::pol::sample_type<inb::pol::f16>(a, s);
  return inb::pol::sample_type<float>(a, s);
}
