// counter_dropout: dropout whose mask is a function of the engine's counter RNG and is never stored.
//
//   key(e) = the counter-RNG chain over (s0, env_id[e], episode[e], channel INB_CH_DROPOUT, ctr[e], stream)
//   word j of env e = elem(key(e), j); its low half decides element 2j of the env's row, its high half 2j + 1
//   out = x * 65536 / (65536 - t) where half >= t, else 0;   t = round(65536 p)
//
// The draw depends on the global env id, not on the shard, like every other draw of the engine.  Sixteen bits a draw
// make one hash serve two elements: the hash is what bounds the kernel next to DRAM (18 integer operations a word), p
// is held to 2^-17 and the scale uses the probability as held, so the expectation is exact.
//
// The forward call derives the keys and can store them ([E] words); the backward call reads those, so that an episode
// or a counter that moved on in between (the engine updates both in place) does not change the mask.
#include "nr_common.cuh"
#include "policy_common.cuh"

namespace inb {
namespace pol {

constexpr int DROP_THREADS = 256;
constexpr int DROP_SPAN = 16;     // elements of one thread
constexpr int DROP_TILE = DROP_THREADS * DROP_SPAN;

// One block per tile of one env's row.  Bound by instruction issue: a word takes 17 operations to hash and 10 to apply to
// its two elements.  184.5 M bf16 elements take 135 us alone, 141 each in a forward and backward pair, and their bytes 113
// at the measured copy rate.  Tried and slower: several tiles a block with the next one loaded ahead (7 us more), shifts as
// multiplies on the idle pipe (3 us more).
template <typename T, int V>
__global__ void __launch_bounds__(DROP_THREADS) dropout_kernel(InbDropoutArgs a, uint32_t tiles, float scale) {
  const uint32_t e = blockIdx.x / tiles, tile = blockIdx.x - e * tiles;
  const int64_t n = a.n;
  const T* x = (const T*)a.x + (int64_t)e * n;
  T* y = (T*)a.y + (int64_t)e * n;
  constexpr int W = V < 2 ? 2 : V;           // elements of one step: whole words
  const int64_t start = (int64_t)tile * DROP_TILE + threadIdx.x * W;
  // the elements are on their way before the key, which takes a few dependent loads of its own
  T in[DROP_SPAN];
#pragma unroll
  for (int i = 0; i < DROP_SPAN / W; ++i) {
    const int64_t c = start + i * DROP_THREADS * W;
    if (V >= 2) {
      if (c < n) {
        const Pack<T, W> p = ld<T, W>(x + c);
#pragma unroll
        for (int k = 0; k < W; ++k) in[i * W + k] = p.v[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k) in[i * W + k] = c + k < n ? x[c + k] : from_f<T>(0.f);
    }
  }
  __shared__ uint32_t key;
  if (threadIdx.x == 0) {
    uint32_t k;
    if (a.keys_in != nullptr) {
      k = a.keys_in[e];
    } else {
      k = key_stream(key_env(a.s0, a.env_id[e], a.episode != nullptr ? a.episode[e] : 0, INB_CH_DROPOUT,
                             a.ctr != nullptr ? a.ctr[e] : 0), a.stream);
      if (a.keys_out != nullptr && tile == 0) a.keys_out[e] = k;
    }
    key = k;
  }
  __syncthreads();
  // a half is compared with the threshold in the upper half of a word, without being taken out; 65536 does not fit there
  const uint32_t base = key, thr = a.threshold << 16;
  const bool none = a.threshold > 65535u;
#pragma unroll
  for (int i = 0; i < DROP_SPAN / W; ++i) {
    const int64_t c = start + i * DROP_THREADS * W;
    if (c >= n) break;
    Pack<T, W> o;
    const uint32_t word = base + (uint32_t)(c >> 1) * GOLD;      // c is even
#pragma unroll
    for (int k = 0; k < W; k += 2) {
      const uint32_t w = mix32(mix32(word + (uint32_t)(k / 2) * GOLD) ^ base);      // elem(base, c / 2 + k / 2)
      const float2 v = mul2(up2(in[i * W + k], in[i * W + k + 1]), both(scale));
      down2(make_float2(w << 16 >= thr && !none ? v.x : 0.f, w >= thr && !none ? v.y : 0.f), o.v[k], o.v[k + 1]);
    }
    if (V >= 2) {
      st<T, W>(y + c, o);
    } else {
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (c + k < n) y[c + k] = o.v[k];
    }
  }
}

template <typename T>
static int dropout_go(const InbDropoutArgs& a, cudaStream_t s) {
  const uint64_t tiles = ((uint64_t)a.n + DROP_TILE - 1) / DROP_TILE, grid = tiles * (uint64_t)a.E;
  if (grid > 0x7FFFFFFFull) return -2;
  const float scale = a.threshold < 65536u ? 65536.f / (float)(65536u - a.threshold) : 0.f;
  constexpr int W = 16 / (int)sizeof(T);
  const uint64_t m = (uint64_t)(uintptr_t)a.x | (uint64_t)(uintptr_t)a.y | (uint64_t)a.n * sizeof(T);
  if ((m & 15) == 0)
    dropout_kernel<T, W><<<(unsigned)grid, DROP_THREADS, 0, s>>>(a, (uint32_t)tiles, scale);
  else
    dropout_kernel<T, 1><<<(unsigned)grid, DROP_THREADS, 0, s>>>(a, (uint32_t)tiles, scale);
  return launch_status();
}

}  // namespace pol
}  // namespace inb

extern "C" int inb_dropout(const InbDropoutArgs* args, void* cuda_stream) {
  if (args == nullptr) return -1;
  const InbDropoutArgs& a = *args;
  if (a.dtype < 0 || a.dtype > 2 || a.E < 0 || a.n < 0 || a.n > 0x1FFFFFFFFll || a.threshold > 65536u) return -2;
  if (a.E == 0 || a.n == 0) return 0;
  if (a.x == nullptr || a.y == nullptr || (a.keys_in == nullptr && a.env_id == nullptr)) return -3;
  cudaStream_t s = (cudaStream_t)cuda_stream;
  if (a.dtype == INB_BF16) return inb::pol::dropout_go<inb::pol::bf16>(a, s);
  if (a.dtype == INB_F16) return inb::pol::dropout_go<inb::pol::f16>(a, s);
  return inb::pol::dropout_go<float>(a, s);
}
