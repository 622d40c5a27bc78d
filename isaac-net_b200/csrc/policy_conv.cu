// causal_conv: depthwise causal convolution over time, 2 to 4 taps a channel, with resets inside the sequence.
//
//   pre[t] = bias + sum_j w[K - 1 - j] x[t - j],  y = act(pre);     taps before a reset, or before the sequence, are 0
//   g[t] = gy[t] act'(pre[t]);   gx[t] = sum_j w[K - 1 - j] g[t + j];   gw[K - 1 - j] = sum_t g[t] x[t - j];   gbias = sum_t g[t]
//
// Bound by DRAM: 2K operations an element against 2 (forward) or 3 (backward, which recomputes pre) moved elements.  A
// thread holds V neighbouring channels, walks along time and keeps the last K - 1 inputs in registers, so every element is
// read once; where sequences are few the time axis is split and a part re-reads K - 1 steps at its edge.
// 1024 x 32 sequences of 16 steps, 256 channels, K = 4, bf16, SiLU: forward 121 us (4.4 TB/s), backward 256 us (3.1 TB/s: the 15
// warps an SM that its 128 registers leave issue 55 % of the time, waiting on their own results).
#include "policy_seq.cuh"

namespace inb {
namespace pol {

// Blocks of 128 threads, an SM.  80 sequences of 3373 steps of 458 bf16 channels, 2 a thread: forward 199 us with 4, 279 with 6, 330
// with 8; backward 402 with 4, 421 with 6, 516 with 8.
constexpr int CONV_FWD_BLOCKS = 4, CONV_BWD_BLOCKS = 4;
// A single step's: 16880 sequences of 458 channels, 2 a thread by one access, bf16 59 us with 4, 49 with 6, 43 with 8, fp32 78, 53, 63;
// by two accesses (457 channels) 86, 92, 88 and 78, 91, 87
constexpr int conv_step_blocks(int V, bool wide) { return V == 2 && wide ? 6 : 4; }
// Sequences whose loads are sent at once by a single step: more leave the registers (3 and 4 at 2 channels a thread: 49 -> 46 and
// 51 us bf16, 53 -> 72 and 84 us fp32)
constexpr int CONV_STEP_B = 2;

struct ConvPlan {
  int64_t parts, len, tasks;    // parts of the time axis, their steps; sequences x parts
};

// A thread's V channels: neighbours, moved by one access of V sizeof(T) bytes where every row is aligned to that, or (WIDE
// false) blockDim.x apart, each moved by itself, so that a warp's accesses still lie side by side.
template <typename T, int V, bool WIDE>
struct Lanes {
  int64_t first;
  int gap, count, x;              // count: those below C
  __device__ __forceinline__ Lanes(const InbConvArgs& a) : gap(WIDE ? 1 : (int)blockDim.x), x(threadIdx.x) {
    const int64_t c0 = (int64_t)blockIdx.y * blockDim.x * V;
    first = WIDE ? c0 + x * V : c0 + x;
    const int64_t left = a.C - first;
    count = left <= 0 ? 0 : WIDE ? V : (int)((left + gap - 1) / gap < V ? (left + gap - 1) / gap : V);
  }
  __device__ __forceinline__ int64_t at(int v) const { return first + (int64_t)v * gap; }
  __device__ __forceinline__ int local(int v) const { return WIDE ? x * V + v : v * gap + x; }      // in the block's blockDim.x V channels
  __device__ __forceinline__ void load(Words<T, V>& w, const T* row) const {
    if constexpr (WIDE) {
      w.load(row + first);
    } else {
      uint32_t e[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        e[v] = 0;
        if (v < count) e[v] = ld_raw(row + at(v));
      }
      w.join(e);
    }
  }
  __device__ __forceinline__ void store(T* row, const Words<T, V>& w) const {
    if constexpr (WIDE) {
      w.store(row + first);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (v < count) {
          if constexpr (sizeof(T) == 4)
            reinterpret_cast<uint32_t*>(row)[at(v)] = w.w[v];
          else
            reinterpret_cast<uint16_t*>(row)[at(v)] = (uint16_t)(v & 1 ? w.w[v / 2] >> 16 : w.w[v / 2]);
        }
    }
  }
};
// The weights of a thread's channels, as pairs
template <typename T, int V, int K>
struct Taps {
  static constexpr int P = Words<T, V>::P;
  float2 w[K][P], bias[P];
  template <bool WIDE>
  __device__ __forceinline__ void load(const InbConvArgs& a, const Lanes<T, V, WIDE>& io) {
    if constexpr (WIDE) {
      // the V K weights of neighbouring channels lie together
      if ((((uintptr_t)a.w | (uintptr_t)a.bias) & (V * sizeof(T) - 1)) == 0) {
        Words<T, V> q[K], b;
        if (io.count > 0) {
#pragma unroll
          for (int k = 0; k < K; ++k) q[k].load((const T*)a.w + io.first * K + k * V);
          if (a.bias != nullptr) b.load((const T*)a.bias + io.first);
        }
        auto element = [&](int e) {
          const float2 p = q[e / V].pair(e % V / 2);
          return e & 1 ? p.y : p.x;
        };
#pragma unroll
        for (int i = 0; i < P; ++i) {
          bias[i] = io.count > 0 && a.bias != nullptr ? b.pair(i) : make_float2(0.f, 0.f);
#pragma unroll
          for (int k = 0; k < K; ++k)
            w[k][i] = io.count > 0 ? make_float2(element(2 * i * K + k), element((2 * i + 1) * K + k)) : make_float2(0.f, 0.f);
        }
        return;
      }
    }
    auto get = [&](const void* p, int v, int64_t of, int64_t k) { return v < io.count && p != nullptr ? to_f(((const T*)p)[io.at(v) * of + k]) : 0.f; };
#pragma unroll
    for (int i = 0; i < P; ++i) {
      bias[i] = make_float2(get(a.bias, 2 * i, 1, 0), get(a.bias, 2 * i + 1, 1, 0));
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][i] = make_float2(get(a.w, 2 * i, K, k), get(a.w, 2 * i + 1, K, k));
    }
  }
};
// The last K - 1 inputs; x[j]: j + 1 steps back
template <typename T, int V, int K>
struct Window {
  static constexpr int P = Words<T, V>::P;
  float2 x[K - 1][P];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) x[j][i] = make_float2(0.f, 0.f);
  }
  __device__ __forceinline__ void push(const float2 (&v)[P]) {
#pragma unroll
    for (int j = K - 2; j > 0; --j)
#pragma unroll
      for (int i = 0; i < P; ++i) x[j][i] = x[j - 1][i];
#pragma unroll
    for (int i = 0; i < P; ++i) x[0][i] = v[i];
  }
  __device__ __forceinline__ void push(const Words<T, V>& q) {
    float2 v[P];
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = q.pair(i);
    push(v);
  }
  __device__ __forceinline__ float2 pre(const Taps<T, V, K>& t, float2 now, int i) const {
    float2 p = fma2(now, t.w[K - 1][i], t.bias[i]);
#pragma unroll
    for (int j = 0; j < K - 1; ++j) p = fma2(x[j][i], t.w[K - 2 - j][i], p);
    return p;
  }
};
// ---------------------------------------------------------------------------------------------- rows on their way
// A task's rows go by chunks through memory that the thread alone writes and reads (no barrier): while one chunk is
// worked on, the next one's rows, the next task's among them, are on their way by cp.async; rows of 2 bytes, which cp.async
// cannot move, by registers.  A task's first chunk also brings the K - 1 rows before it, of the state or of the part before.
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// STREAMS 2: x and gy, whose rows end with those that reach back into the part
template <typename T, int V, bool WIDE, int K, int STREAMS>
struct Feed {
  static constexpr bool HELD = !WIDE && sizeof(T) == 2;        // by registers
  static constexpr int R = HELD ? 4 : 8;                       // rows of a chunk
  static constexpr int B = V * sizeof(T), ROWS = K - 1 + R * STREAMS, STAGE = ROWS * 128 * B;
  using Io = Lanes<T, V, WIDE>;
  // a chunk: sequence s, rows [lo, hi) of its part [t0, t0 + n)
  struct Chunk {
    int64_t task, s, t0;
    int n, to, lo, hi;
    bool on;
  };
  char* base;
  uint32_t held[HELD ? ROWS * V : 1];
  uint32_t flag[2];
  int64_t stride, rounds, round;
  int chunks, chunk, tx, lane, stage;
  Chunk next;
  __device__ __forceinline__ char* slot(int st, int row) const { return base + st * STAGE + row * 128 * B; }
  __device__ __forceinline__ void put(const Io& io, int row, const T* p) {
    if constexpr (WIDE && B == 16) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_at(slot(stage, row))), "l"(p + io.first) : "memory");
    } else if constexpr (WIDE) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_at(slot(stage, row))), "l"(p + io.first), "n"(B) : "memory");
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (v < io.count) {
          if constexpr (HELD)
            held[row * V + v] = ld_raw(p + io.at(v));
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_at(slot(stage, row)) + 4 * v), "l"(p + io.at(v)) : "memory");
        }
    }
  }
  __device__ __forceinline__ Words<T, V> get(int row) const {      // of the chunk that now() gave
    Words<T, V> w;
    w.load((const T*)slot(stage ^ 1, row));
    return w;
  }
  __device__ __forceinline__ void place(const InbConvArgs& a, const ConvPlan& pl) {
    next.lo = chunk * R;
    if (chunk == 0) {
      next.on = next.task < pl.tasks;
      const int64_t part = pl.parts > 1 ? next.task / a.S : 0;      // the next task: the same steps of the next sequence
      next.s = next.task - part * a.S;
      next.t0 = part * pl.len;
      const int64_t left = a.T - next.t0;
      next.n = (int)(pl.len < left ? pl.len : left);
      next.to = STREAMS == 1 ? next.n : next.n + K - 1 < left ? next.n + K - 1 : (int)left;
    }
    next.hi = next.lo + R < next.to ? next.lo + R : next.to;
  }
  __device__ __forceinline__ void send(const InbConvArgs& a, const Io& io) {
    flag[0] = flag[1] = 0;
    if (next.on && next.lo < next.hi) {
      const int count = next.hi - next.lo;
      if (io.count > 0) rows(a, io, count);
      const uint8_t* rs = resets(a.reset, next.s);
      if (rs != nullptr) {
        rs += (next.t0 + next.lo) * a.reset.step;
        const int l = threadIdx.x & 31;           // the lanes of a task read its flags together, those beyond the channels too
        if (l < R && l < count) flag[0] = rs[l * a.reset.step];
        if (tx == 4 && l + 4 < count) flag[1] = rs[(l + 4) * a.reset.step];
      }
    }
    if constexpr (!HELD) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void rows(const InbConvArgs& a, const Io& io, int count) {
    const T* p = row<T>(a.x, next.s, next.t0 + next.lo);
    const T* g = STREAMS > 1 ? row<T>(a.gy, next.s, next.t0 + next.lo) : nullptr;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < count) {
        put(io, K - 1 + i, p);
        p += a.x.step;
        if (STREAMS > 1) {
          put(io, K - 1 + R + i, g);
          g += a.gy.step;
        }
      }
    if (chunk == 0 && (next.t0 > 0 || a.state != nullptr)) {
      const bool state = next.t0 == 0;
      const T* h = state ? (const T*)a.state + next.s * a.state_seq : row<T>(a.x, next.s, next.t0 - (K - 1));
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        put(io, j, h);
        h += state ? a.C : a.x.step;
      }
    }
  }
  __device__ __forceinline__ void start(const InbConvArgs& a, const ConvPlan& pl, char* smem, const Io& io) {
    tx = blockDim.x;
    const int id = threadIdx.y * tx + threadIdx.x;
    base = smem + id * B;
    lane = id & 31;
    stride = (int64_t)gridDim.x * blockDim.y;
    rounds = (pl.tasks + stride - 1) / stride;
    const int64_t rows = pl.parts > 1 && STREAMS > 1 ? pl.len + K - 1 : pl.len;
    chunks = (int)((rows + R - 1) / R);
    round = chunk = stage = 0;
    next.task = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    place(a, pl);
    send(a, io);
  }
  __device__ __forceinline__ bool more() const { return round < rounds; }      // the same for every thread of the block
  // the next chunk, landed; bit i of `cuts`: its row i starts an episode.  The chunk after it is sent for.
  __device__ __forceinline__ Chunk now(const InbConvArgs& a, const ConvPlan& pl, const Io& io, uint32_t& cuts) {
    const Chunk c = next;
    if constexpr (HELD) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        Words<T, V> w;
        w.join(reinterpret_cast<const uint32_t(&)[V]>(held[i * V]));
        w.store((T*)slot(stage, i));
      }
    }
    const int first = lane & ~((tx < 32 ? tx : 32) - 1);
    cuts = __ballot_sync(0xFFFFFFFFu, flag[0] != 0) >> first & (tx == 4 ? 0xFu : 0xFFu);
    if (tx == 4) cuts |= (__ballot_sync(0xFFFFFFFFu, flag[1] != 0) >> first & 0xFu) << 4;
    stage ^= 1;
    if (++chunk == chunks) chunk = 0, ++round, next.task += stride;
    if (round < rounds) {
      place(a, pl);
      send(a, io);
    } else if constexpr (!HELD) {
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if constexpr (!HELD) asm volatile("cp.async.wait_group 1;" ::: "memory");
    return c;
  }
};

// ---------------------------------------------------------------------------------------------- forward
// A block is blockDim.x channel vectors x blockDim.y tasks and strides over the tasks, so that weights are read once.
template <typename T, int V, bool WIDE, int K>
__global__ void __launch_bounds__(128, CONV_FWD_BLOCKS) conv_fwd_kernel(InbConvArgs a, ConvPlan pl) {
  constexpr int P = Words<T, V>::P;
  extern __shared__ float4 smem4[];
  const Lanes<T, V, WIDE> io(a);
  Feed<T, V, WIDE, K, 1> feed;
  feed.start(a, pl, (char*)smem4, io);
  Taps<T, V, K> taps;
  taps.load(a, io);
  Window<T, V, K> win;
  T* py = nullptr;
  while (feed.more()) {
    uint32_t cuts;
    const auto q = feed.now(a, pl, io, cuts);
    if (!q.on || io.count == 0) continue;
    if (q.lo == 0) {
      win.zero();
      if (q.t0 > 0 || a.state != nullptr) {
        const uint8_t* rs = q.t0 > 0 ? resets(a.reset, q.s) : nullptr;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
          if (rs != nullptr && rs[(q.t0 - (K - 1) + j) * a.reset.step] != 0) win.zero();
          win.push(feed.get(j));
        }
      }
      py = row_out<T>(a.y, q.s, q.t0);
    }
    const int count = q.hi - q.lo;
    auto step = [&](int i, bool cut) {
      const Words<T, V> x = feed.get(K - 1 + i);
      if (cut) win.zero();
      float2 now[P];
      Words<T, V> y;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        now[k] = x.pair(k);
        const float2 p = win.pre(taps, now[k], k);
        y.set(k, a.act == INB_ACT_SILU ? mul2(p, sigmoid2(p)) : p);
      }
      io.store(py, y);
      py += a.y.step;
      win.push(now);
    };
    if (cuts == 0 && count == feed.R) {      // without a branch between them, rows overlap
#pragma unroll 4
      for (int i = 0; i < feed.R; ++i) step(i, false);
    } else {
#pragma unroll 4
      for (int i = 0; i < count; ++i) step(i, cuts >> i & 1);
    }
    if (q.hi == q.n && q.lo < q.hi && q.t0 + q.n == a.T && a.state_out != nullptr) {
      T* out = (T*)a.state_out + q.s * a.state_out_seq;
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        Words<T, V> p;
#pragma unroll
        for (int k = 0; k < P; ++k) p.set(k, win.x[j][k]);      // what was read, or 0: exact
        io.store(out + (K - 2 - j) * a.C, p);
      }
    }
  }
}

// One step: bound by the states' bytes, of which a thread has CONV_STEP_B sequences' on their way at once; state_out may be state.
// 131072 sequences of 512 channels, K = 4, bf16: 172 us (6.2 TB/s).
template <typename T, int V, bool WIDE, int K>
__global__ void __launch_bounds__(128, conv_step_blocks(V, WIDE)) conv_step_kernel(InbConvArgs a) {
  constexpr int P = Words<T, V>::P;
  const Lanes<T, V, WIDE> io(a);
  if (io.count == 0) return;
  Taps<T, V, K> taps;
  taps.load(a, io);
  const int64_t stride = (int64_t)gridDim.x * blockDim.y;
  for (int64_t s0 = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; s0 < a.S; s0 += stride * CONV_STEP_B) {
    Words<T, V> x[CONV_STEP_B], old[CONV_STEP_B][K - 1];
    uint32_t reset[CONV_STEP_B];
#pragma unroll
    for (int b = 0; b < CONV_STEP_B; ++b) {
      const int64_t s = s0 + b * stride;
      if (s >= a.S) break;
      io.load(x[b], row<T>(a.x, s, 0));
      reset[b] = a.reset.p != nullptr ? *resets(a.reset, s) : 0;
      if (a.state != nullptr) {
        const T* p = (const T*)a.state + s * a.state_seq;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) io.load(old[b][j], p + j * a.C);
      }
    }
#pragma unroll
    for (int b = 0; b < CONV_STEP_B; ++b) {
      const int64_t s = s0 + b * stride;
      if (s >= a.S) break;
      if (reset[b] || a.state == nullptr) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
#pragma unroll
          for (int i = 0; i < Words<T, V>::N; ++i) old[b][j].w[i] = 0;
      }
      Words<T, V> y;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float2 p = fma2(x[b].pair(i), taps.w[K - 1][i], taps.bias[i]);
#pragma unroll
        for (int j = K - 2; j >= 0; --j) p = fma2(old[b][j].pair(i), taps.w[j][i], p);
        y.set(i, a.act == INB_ACT_SILU ? mul2(p, sigmoid2(p)) : p);
      }
      io.store(row_out<T>(a.y, s, 0), y);
      if (a.state_out != nullptr) {
        T* out = (T*)a.state_out + s * a.state_out_seq;
#pragma unroll
        for (int j = 0; j < K - 2; ++j) io.store(out + j * a.C, old[b][j + 1]);
        io.store(out + (K - 2) * a.C, x[b]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------- backward
// pend[j - 1] gathers gx[t - j] while later steps still add to it; step t completes gx[t - (K - 1)].  Where an episode begins
// the K - 1 before it are complete already: they are stored there, and what is gathered for them afterwards is dropped.  A part
// goes K - 1 steps beyond its end, for gx alone.  Blocks as in the forward pass, so that gw and gbias stay in registers; one
// partial row a block, [C K | C], added by a second launch.
template <typename T, int V, bool WIDE, int K>
__global__ void __launch_bounds__(128, CONV_BWD_BLOCKS) conv_bwd_kernel(InbConvArgs a, ConvPlan pl) {
  constexpr int P = Words<T, V>::P;
  extern __shared__ float4 smem4[];
  float* smem = (float*)smem4;
  const Lanes<T, V, WIDE> io(a);
  Taps<T, V, K> taps;
  taps.load(a, io);
  const float2 zero = make_float2(0.f, 0.f);
  float2 gw[K][P], gb[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    gb[i] = zero;
#pragma unroll
    for (int k = 0; k < K; ++k) gw[k][i] = zero;
  }
  Window<T, V, K> win;
  float2 pend[K - 1][P];
  int seen = 0;                           // rows since the episode or the part began, up to K - 1
  T* pgx = nullptr;
  Feed<T, V, WIDE, K, 2> feed;
  feed.start(a, pl, (char*)smem, io);
  while (feed.more()) {
    uint32_t cuts;
    const auto q = feed.now(a, pl, io, cuts);
    if (!q.on || io.count == 0) continue;
    // gx of the row `at` (pgx's) is complete; before the sequence it is the initial state's
    auto store = [&](int at, const float2 (&v)[P]) {
      Words<T, V> p;
#pragma unroll
      for (int k = 0; k < P; ++k) p.set(k, v[k]);
      if (at >= 0)
        io.store(row_out<T>(a.gx, q.s, q.t0 + at), p);
      else if (q.t0 == 0 && a.gstate != nullptr)
        io.store((T*)a.gstate + (q.s * (K - 1) + at + K - 1) * a.C, p);
    };
    // an episode begins at row i: the rows before it are complete, but for those that were when the last one began
    auto flush = [&](int i) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
        if (j < seen && i - 1 - j < q.n) store(i - 1 - j, pend[j]);
    };
    auto clear = [&] {
      win.zero();
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
#pragma unroll
        for (int k = 0; k < P; ++k) pend[j][k] = zero;
    };
    auto shift = [&](const float2 (&g)[P]) {
#pragma unroll
      for (int j = K - 2; j > 0; --j)
#pragma unroll
        for (int k = 0; k < P; ++k) pend[j][k] = pend[j - 1][k];
#pragma unroll
      for (int k = 0; k < P; ++k) pend[0][k] = mul2(taps.w[K - 1][k], g[k]);
    };
    if (q.lo == 0) {
      clear();
      seen = q.t0 == 0 ? K - 1 : 0;       // what lies before a later part is that part's to store
      if (q.t0 > 0 || a.state != nullptr) {
        const uint8_t* rs = q.t0 > 0 ? resets(a.reset, q.s) : nullptr;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
          if (rs != nullptr && rs[(q.t0 - (K - 1) + j) * a.reset.step] != 0) win.zero();
          win.push(feed.get(j));
        }
      }
      pgx = row_out<T>(a.gx, q.s, q.t0);
    }
    const int count = q.hi - q.lo;
    // MIDDLE: rows of the part, whose gx is stored K - 1 rows later
    auto step = [&](int i, bool cut, bool middle) {
      const Words<T, V> x = feed.get(K - 1 + i), gy = feed.get(K - 1 + feed.R + i);
      const int row = q.lo + i;
      if (cut) {
        flush(row);
        clear();
        seen = 0;
      }
      float2 now[P], g[P];
#pragma unroll
      for (int k = 0; k < P; ++k) {
        now[k] = x.pair(k);
        g[k] = gy.pair(k);
        if (a.act == INB_ACT_SILU) {
          const float2 p = win.pre(taps, now[k], k), s = sigmoid2(p);
          g[k] = mul2(g[k], mul2(s, fma2(p, fma2(s, both(-1.f), both(1.f)), both(1.f))));
        }
      }
      if (middle || row < q.n) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
          gb[k] = add2(gb[k], g[k]);
          gw[K - 1][k] = fma2(g[k], now[k], gw[K - 1][k]);
#pragma unroll
          for (int j = 0; j < K - 1; ++j) gw[K - 2 - j][k] = fma2(g[k], win.x[j][k], gw[K - 2 - j][k]);
        }
      }
#pragma unroll
      for (int j = 0; j < K - 1; ++j)
#pragma unroll
        for (int k = 0; k < P; ++k) pend[j][k] = fma2(taps.w[K - 2 - j][k], g[k], pend[j][k]);
      if (middle || (row >= K - 1 && seen == K - 1)) {
        Words<T, V> p;
#pragma unroll
        for (int k = 0; k < P; ++k) p.set(k, pend[K - 2][k]);
        io.store(pgx, p);
      } else if (seen == K - 1) {
        store(row - (K - 1), pend[K - 2]);
      }
      if (middle || row >= K - 1) pgx += a.gx.step;
      shift(g);
      win.push(now);
      if (!middle) seen = seen < K - 1 ? seen + 1 : seen;
    };
    if (cuts == 0 && count == feed.R && q.hi <= q.n && seen == K - 1) {      // without a branch between them, rows overlap
      if (q.lo == 0) {
#pragma unroll
        for (int i = 0; i < K - 1; ++i) step(i, false, false);
#pragma unroll
        for (int i = K - 1; i < feed.R; ++i) step(i, false, true);
      } else {
#pragma unroll 4
        for (int i = 0; i < feed.R; ++i) step(i, false, true);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < count; ++i) step(i, cuts >> i & 1, false);
    }
    if (q.hi == q.to && q.lo < q.hi) {
      // the rows that nothing follows: those of the sequence's end, to which the final state's gradient adds
      // (its entry e is the input of step T - (K - 1) + e)
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        const int at = q.to - 1 - j;
        if (at >= q.n || j >= seen) continue;
        const int e = (int)(q.t0 + at - a.T) + K - 1;
        if (a.gstate_out != nullptr && e >= 0) {
          Words<T, V> p;
          io.load(p, (const T*)a.gstate_out + (q.s * (K - 1) + e) * a.C);
#pragma unroll
          for (int k = 0; k < P; ++k) pend[j][k] = add2(pend[j][k], p.pair(k));
        }
        store(at, pend[j]);
      }
    }
  }
  __syncthreads();                        // the rows' memory holds the block's sums from here on
  // the block's tasks, then one partial row
  const int n = blockDim.x * V * (K + 1);
  float* mine = smem + threadIdx.y * n;
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < K; ++k) mine[io.local(v) * K + k] = v & 1 ? gw[k][v / 2].y : gw[k][v / 2].x;
    mine[blockDim.x * V * K + io.local(v)] = v & 1 ? gb[v / 2].y : gb[v / 2].x;
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
  // lanes of a task: as few beyond the last channel as may be, the more the better; 4 at least, which share the reading of the
  // task's reset flags
  unsigned tx = 128;
  for (unsigned t = 64; t >= (cv >= 16 ? 16 : 4); t /= 2)
    if (ceil_div(cv, t) * t < ceil_div(cv, tx) * tx) tx = t;
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
      a.K > 4 || a.S < 0 || a.S > INB_MAX_MEMORY_S || a.T < 0 || a.T > INB_MAX_MEMORY_S || (a.reset.p != nullptr && (a.reset.rows < 1 || a.reset.rows > INB_MAX_MEMORY_S)))
    return -2;
  return 0;
}

template <typename T, int V, bool WIDE, int K>
static int conv_fwd_go(const InbConvArgs& a, cudaStream_t s) {
  if (a.T == 1) {
    const ConvLaunch l = conv_plan(a, V, conv_step_blocks(V, WIDE));
    conv_step_kernel<T, V, WIDE, K><<<l.grid, l.block, 0, s>>>(a);
    return launch_status();
  }
  constexpr auto kernel = conv_fwd_kernel<T, V, WIDE, K>;
  constexpr int smem = 2 * Feed<T, V, WIDE, K, 1>::STAGE;
  const cudaError_t e = allow_smem<KernelKey<conv_fwd_kernel<T, V, WIDE, K>>>((const void*)kernel, smem);
  if (e != cudaSuccess) return -100 - (int)e;
  const ConvLaunch l = conv_plan(a, V, CONV_FWD_BLOCKS);
  kernel<<<l.grid, l.block, smem, s>>>(a, l.plan);
  return launch_status();
}
template <typename T, int V, bool WIDE, int K>
static int conv_bwd_go(const InbConvArgs& a, cudaStream_t s) {
  constexpr auto kernel = conv_bwd_kernel<T, V, WIDE, K>;
  constexpr int rows = 2 * Feed<T, V, WIDE, K, 2>::STAGE, sums = 128 * V * (K + 1) * 4, smem = rows > sums ? rows : sums;
  const cudaError_t e = allow_smem<KernelKey<conv_bwd_kernel<T, V, WIDE, K>>>((const void*)kernel, smem);
  if (e != cudaSuccess) return -100 - (int)e;
  const ConvLaunch l = conv_plan(a, V, CONV_BWD_BLOCKS);
  kernel<<<l.grid, l.block, smem, s>>>(a, l.plan);
  colsum<T>(a.work, l.grid.x, (int64_t)a.C * (K + 1), (int64_t)a.C * K, (int64_t)a.C * (K + 1), a.gw, a.gbias, nullptr, s);
  return launch_status();
}
// Channels a thread, by what one access can move: 16 bytes forward; 4 channels backward, whose sums take the registers (8 bytes of
// bf16, 16 of fp32); where rows are not aligned to that 2; and where not even to 2 channels, 2 by an access each.  80 sequences
// of 3373 steps, fp16, forward + backward: 464 channels (4 backward) 332 us, 460 (4 both ways) 346, 458 (2) 582, 457 (2 by two) 684
// (2654 with 4 by four accesses, which leave the registers).
template <typename T, int V, bool WIDE>
static int conv_taps(const InbConvArgs& a, bool backward, cudaStream_t s) {
  if (backward) {
    if constexpr (V <= 4) return a.K == 2 ? conv_bwd_go<T, V, WIDE, 2>(a, s) : a.K == 3 ? conv_bwd_go<T, V, WIDE, 3>(a, s) : conv_bwd_go<T, V, WIDE, 4>(a, s);
    return -2;
  }
  return a.K == 2 ? conv_fwd_go<T, V, WIDE, 2>(a, s) : a.K == 3 ? conv_fwd_go<T, V, WIDE, 3>(a, s) : conv_fwd_go<T, V, WIDE, 4>(a, s);
}
template <typename T>
static int conv_type(const InbConvArgs& a, bool backward, cudaStream_t s) {
  constexpr int W = 16 / sizeof(T), E = sizeof(T);
  if (!backward && W > 4 && conv_aligned(a, 16)) return conv_taps<T, W, true>(a, false, s);
  if (conv_aligned(a, 4 * E)) return conv_taps<T, 4, true>(a, backward, s);
  if (conv_aligned(a, 2 * E)) return conv_taps<T, 2, true>(a, backward, s);
  return conv_taps<T, 2, false>(a, backward, s);
}
static int conv_dispatch(const InbConvArgs& a, bool backward, cudaStream_t s) {
  if (a.dtype == INB_BF16) return conv_type<bf16>(a, backward, s);
  if (a.dtype == INB_F16) return conv_type<f16>(a, backward, s);
  return conv_type<float>(a, backward, s);
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
  // the rows' alignment, which decides on the channels a thread, is the launch's to find out
  for (int v : {2, 4}) {
    const int64_t n = (int64_t)inb::pol::conv_plan(a, v, inb::pol::CONV_BWD_BLOCKS).grid.x * a.C * (a.K + 1);
    if (n > *elems) *elems = n;
  }
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
