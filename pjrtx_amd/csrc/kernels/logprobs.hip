// Log probabilities of given tokens, the distribution's entropy and its
// likeliest tokens, in one pass over the logits; and their gradient.
//
// A row is split over workgroups, which read it in chunks of 8192 elements
// held in registers. Each thread keeps an online softmax of its own: m, the
// largest x so far, l = sum e^d and a = sum e^d d with d = x - m, from which
// log p of x = (x - m) - log l, lse = m + log l and entropy = log l - a / l.
// Everything is taken about m, not about zero, so nothing large cancels, also
// in rows that hold nothing but the type's lowest value. Elements that may be among the
// row's top_k (bounded below by the threads' maxima, then by the top_k found so
// far) go to a list in LDS and are ranked there by value, then by lowest index.
// logprobs_join folds a row's splits.
//
// Many rows are bound by HBM (1000 x 32000 f32, 128 MB, in 26.9 us), or by the
// exponentials beside it (4000 x 32000 bf16, 256 MB, in 48). Few rows are bound
// by latency: 64 x 128256 bf16 with 20 likeliest 11.5 us in 8 splits a row, two
// dependent chunks each with its maximum, bound, list and ranking, and 4.1 for
// the join. (Ranking only when the list is long saves barriers, but the looser
// bound scans more: 4000 x 32000 bf16, 5 likeliest, 14% longer.)
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kernels/operators.h"
#include "kernels/vec.h"

namespace pjrtx {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;               // elements a workgroup holds in registers
constexpr int kCandidates = 1024;          // list of a chunk's candidates in LDS
constexpr int kJoinKeys = 2048;            // keys of all splits that the join holds in LDS
constexpr int kJoinSplits = 64;            // a lane each
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
// Largest |m| whose elements take their distances by one fma: 4000 x 32000 bf16
// in 48.9 us, by a subtraction and a product 49.9 (600 x 128256, 5 likeliest:
// 52.6 and 54.7). Past it the rounding of m log2(e), which the chunk's sums are
// corrected by, would be more than 2^-17, and near 2^31 more than exp2 takes.
constexpr float kNear = 128.f;

// The order of top_k on floats: the sign-magnitude order of their bits, so
// that -0 < +0 and NaN (positive) is above +inf. 0 is below every float's
// image but that of the negative NaN of all ones.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __builtin_bit_cast(float, o ^ (o & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
// Larger key: larger value, then lower index. Keys of a row are distinct; 0
// is no key (an index is below 2^31).
__device__ __forceinline__ uint64_t key_of(float x, int64_t i) {
  return ((uint64_t)order_of(x) << 32) | (uint32_t)~(uint32_t)i;
}


// One thread's or split's softmax state.
struct Soft {
  float m, l, a;
};
// The state about the larger maximum m >= s.m.
__device__ __forceinline__ void raise(Soft& s, float m) {
  // A side of no elements has l = a = 0 at -inf: its shift is made finite.
  const float d = fmaxf(s.m - m, -1e4f), f = __builtin_amdgcn_exp2f(d * kLog2e);
  s.a = f * (s.a + d * s.l);
  s.l *= f;
  s.m = m;
}
__device__ __forceinline__ Soft join(Soft x, Soft y) {
  const float m = fmaxf(x.m, y.m);
  if (m != -INFINITY) {  // else 0s, or NaNs
    raise(x, m);
    raise(y, m);
  }
  return {m, x.l + y.l, x.a + y.a};
}

// The split's results: {m, l, a}, then top_k keys, largest first, 0 past the last.
__host__ __device__ constexpr int64_t split_words(int top_k) { return 4 + 2 * (int64_t)top_k; }

// The largest of a wave's values, on every lane (register moves, no LDS).
__device__ __forceinline__ uint32_t wave_max_u(uint32_t x) {
  const auto take = [](uint32_t a, int b) { return std::max(a, (uint32_t)b); };
  x = take(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false));  // the lane 1 before in its 16
  x = take(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
  x = take(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
  x = take(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
  x = take(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));  // lane 15 of the 16 before
  x = take(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));  // lane 31
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
// The k-th largest of a wave's values (k >= 1).
__device__ __forceinline__ uint32_t wave_kth_u(uint32_t x, int k) {
  uint32_t top = 0;
  for (int i = 0; i < k; ++i) {
    top = wave_max_u(x);
    const uint64_t who = __ballot(x == top);
    if ((int)(threadIdx.x & 63) == __ffsll((unsigned long long)who) - 1) x = 0;
  }
  return top;
}

// Ranks the n distinct keys at `cand` together with the `held` at `best` and
// leaves the top_k largest in order at `to`; kLanes lanes take a key. Called by
// the whole workgroup.
template <int kLanes>
__device__ __forceinline__ void rank_keys_by(const uint64_t* cand, int n, const uint64_t* best, int held, uint64_t* to,
                                             int top_k) {
  const int lane = threadIdx.x % kLanes;
  for (int i0 = 0; i0 < n + held; i0 += kThreads / kLanes) {
    const int i = i0 + threadIdx.x / kLanes;
    const uint64_t mine = i < n ? cand[i] : i < n + held ? best[i - n] : ~0ull;
    int above = 0;
#pragma unroll 8
    for (int j = lane; j < n; j += kLanes) above += cand[j] > mine ? 1 : 0;
#pragma unroll 4
    for (int j = lane; j < held; j += kLanes) above += best[j] > mine ? 1 : 0;
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) above += __shfl_xor(above, d);
    if (i < n + held && lane == 0 && above < top_k) to[above] = mine;
  }
}
__device__ __forceinline__ void rank_keys(const uint64_t* cand, int n, const uint64_t* best, int held, uint64_t* to,
                                          int top_k) {
  if (n + held <= kThreads / 4) rank_keys_by<4>(cand, n, best, held, to, top_k);
  else if (n + held <= kThreads / 2) rank_keys_by<2>(cand, n, best, held, to, top_k);
  else rank_keys_by<1>(cand, n, best, held, to, top_k);
}

__device__ __forceinline__ int64_t read_token(const void* tokens, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(tokens)[i] : (int64_t)static_cast<const int32_t*>(tokens)[i];
}

struct Results {
  float *logprobs, *entropy, *lse, *top_logprobs;
  int32_t* top_tokens;
};
// By one thread: the row's numbers, `chosen` its token's logit.
__device__ __forceinline__ void write_row(const Results& r, int64_t row, const Soft& s, bool known, float chosen) {
  const float log_l = logf(s.l);
  r.logprobs[row] = known ? (chosen - s.m) - log_l : 0.f;
  r.entropy[row] = log_l - s.a / s.l;
  r.lse[row] = s.m + log_l;
}
// By the workgroup: the row's likeliest tokens, ranked.
__device__ __forceinline__ void write_top(const Results& r, int64_t row, float m, float log_l, const uint64_t* best, int top_k) {
  for (int i = threadIdx.x; i < top_k; i += kThreads) {
    r.top_logprobs[row * top_k + i] = (value_of((uint32_t)(best[i] >> 32)) - m) - log_l;
    r.top_tokens[row * top_k + i] = (int32_t)~(uint32_t)best[i];
  }
}

// A workgroup's share of a row: elements [lo, hi). A row of one share is
// finished here. (5 waves a SIMD: 4000 x 32000 bf16, 5 likeliest, 65 us, with
// the registers of 4 72.)
template <typename T, bool kTop, bool kStream>
__global__ void __launch_bounds__(kThreads, kTop ? 5 : 8)
    logprobs_split(LogprobsParams p, int nsplit, int64_t per, const T* __restrict__ logits,
                   const void* __restrict__ tokens, uint32_t* __restrict__ part, Results r) {
  constexpr int E = kVecElems<T>;
  constexpr int NV = kChunk / kThreads / E;
  constexpr int kWaves = kThreads / 64;
  __shared__ uint64_t cand[kTop ? kCandidates : 1];
  __shared__ uint64_t best[2][kTop ? kLogprobsMaxTopK : 1];
  __shared__ uint32_t kth[kWaves];
  __shared__ uint64_t pick[kWaves];
  __shared__ int count_s;
  __shared__ Soft soft_s[kWaves];
  const int64_t row = blockIdx.x / nsplit;
  const int split = (int)(blockIdx.x % nsplit);
  const T* x = logits + row * p.V;
  const int64_t lo = split * per, hi = std::min(p.V, lo + per);
  const int tid = threadIdx.x;
  Soft s = {-INFINITY, 0.f, 0.f};
  int held = 0, turn = 0;  // keys at best[turn]
  for (int64_t base = lo; base < hi; base += kChunk) {
    typename Vec<T>::type v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t at = base + (int64_t)(i * kThreads + tid) * E;
      v[i] = load_vec<T, kStream>(x + std::min(at, p.V - 1), hi - at, (T)-INFINITY);
    }
    float cm = -INFINITY;  // NaN where one is
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) cm = __builtin_elementwise_maximum(cm, (float)v[i][e]);
    if constexpr (kTop) {
      // Each of the 4 waves has ceil(top_k / 4) threads whose largest element
      // is at or above the least of these: top_k elements or more are.
      if (held < p.top_k) {
        const uint32_t k = wave_kth_u(order_of(cm), (p.top_k + kWaves - 1) / kWaves);
        if ((tid & 63) == 0) kth[tid >> 6] = k;
      }
      if (tid == 0) count_s = 0;
    }
    const float m = fmaxf(s.m, cm);
    if (m > s.m) raise(s, m);  // also the first finite chunk, from l = a = 0
    const float ref = m == -INFINITY ? 0.f : m;
    // -inf weighs nothing: its distance is made finite for a's product.
    if (fabsf(ref) <= kNear) {
      // y = d log2(e) + r by one fma, r what rounding m log2(e) left (a fma
      // gives it exactly). The chunk's sums give it back: over 2^r = 1 + c, |c|
      // below 2^-17, to c^2. The largest element's 1 + c becomes 1, so that no
      // sum is below 1 and no log probability above 0; a sum of e^d d above 0 is
      // rounding, and no entropy is below 0.
      const float ref2 = ref * kLog2e, r = fmaf(ref, kLog2e, -ref2);
      float l2 = 0.f, a2 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float y = __builtin_elementwise_maximum(fmaf((float)v[i][e], kLog2e, -ref2), -1e4f);
          const float w = __builtin_amdgcn_exp2f(y);
          l2 += w;
          a2 = fmaf(w, y, a2);
        }
      const float c = __builtin_amdgcn_exp2f(r) - 1.f;
      a2 = fmaf(-r, l2, a2);
      s.l += fmaf(-c, l2, l2);
      s.a = fmaf(__builtin_elementwise_minimum(fmaf(-c, a2, a2), 0.f), kLn2, s.a);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float d = __builtin_elementwise_maximum((float)v[i][e] - ref, -1e4f);
          const float w = __builtin_amdgcn_exp2f(d * kLog2e);
          s.l += w;
          s.a = fmaf(w, d, s.a);
        }
    }
    if constexpr (kTop) {
      const int64_t left = hi - base;
      __syncthreads();
      // Elements at the bound count in the first chunk; behind top_k keys that
      // were found before (at lower indices) the next float is the bound. NaNs
      // always count.
      const float bound = value_of(held == p.top_k ? (uint32_t)(best[turn][p.top_k - 1] >> 32) + 1
                                                   : std::min(std::min(kth[0], kth[1]), std::min(kth[2], kth[3])));
      auto may = [&](float y) { return !(y < bound); };
      if (may(cm)) {
        // Which of the thread's elements, in bits, and the last one's value:
        // most threads have one. Others are read again.
        uint32_t bits = 0;
        float value = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const bool yes = may((float)v[i][e]);
            bits |= yes ? 1u << (i * E + e) : 0u;
            value = yes ? (float)v[i][e] : value;
          }
        for (bool read = false; bits; read = true) {
          const int j = 31 - __clz(bits);
          bits ^= 1u << j;
          const int64_t index = (int64_t)(j / E * kThreads + tid) * E + j % E;
          const int at = index < left ? atomicAdd(&count_s, 1) : kCandidates;
          if (at < kCandidates) cand[at] = key_of(read ? (float)x[base + index] : value, base + index);
        }
      }
      __syncthreads();
      int n = count_s;
      if (n > kCandidates) {
        // Too many equal or ordered elements for the list: the top_k of the
        // chunk one after another, each the largest key below the last (read
        // again: held in registers for this they would halve the waves).
        uint64_t last = ~0ull;
        for (int k = 0; k < p.top_k; ++k) {
          uint64_t mine = 0;
          for (int64_t i = tid; i < std::min<int64_t>(left, kChunk); i += kThreads) {
            const uint64_t key = key_of((float)x[base + i], base + i);
            if (key < last && key > mine) mine = key;
          }
#pragma unroll
          for (int d = 32; d >= 1; d >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)mine, d);
            mine = std::max(mine, other);
          }
          if ((tid & 63) == 0) pick[tid >> 6] = mine;
          __syncthreads();
          last = std::max(std::max(pick[0], pick[1]), std::max(pick[2], pick[3]));
          if (tid == 0) cand[k] = last;
          __syncthreads();
        }
        n = p.top_k;
      }
      if (n > 0) {
        rank_keys(cand, n, best[turn], held, best[turn ^ 1], p.top_k);
        held = std::min(p.top_k, held + n);
        turn ^= 1;
        __syncthreads();
      }
    }
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s = join(s, Soft{__shfl_xor(s.m, d), __shfl_xor(s.l, d), __shfl_xor(s.a, d)});
  if ((tid & 63) == 0) soft_s[tid >> 6] = s;
  __syncthreads();
  const Soft t = join(join(soft_s[0], soft_s[1]), join(soft_s[2], soft_s[3]));
  if (nsplit == 1) {
    if (tid == 0) {
      const int64_t token = read_token(tokens, p.token_bytes, row);
      const bool known = token >= 0 && token < p.V;
      write_row(r, row, t, known, known ? (float)x[token] : 0.f);
    }
    if constexpr (kTop) write_top(r, row, t.m, logf(t.l), best[turn], p.top_k);
    return;
  }
  uint32_t* out = part + (row * nsplit + split) * split_words(p.top_k);
  if (tid == 0) {
    out[0] = __builtin_bit_cast(uint32_t, t.m);
    out[1] = __builtin_bit_cast(uint32_t, t.l);
    out[2] = __builtin_bit_cast(uint32_t, t.a);
  }
  if constexpr (kTop) {
    for (int i = tid; i < p.top_k; i += kThreads) {
      const uint64_t key = i < held ? best[turn][i] : 0;
      out[4 + 2 * i] = (uint32_t)key;
      out[5 + 2 * i] = (uint32_t)(key >> 32);
    }
  }
}

// The splits of a row: their softmax states folded by halves (a lane each), and
// their keys ranked. Of nsplit ordered lists the ceil(top_k / nsplit)-th keys
// bound the top_k from below: few keys are at or above the least of them.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    logprobs_join(LogprobsParams p, int nsplit, const T* __restrict__ logits, const void* __restrict__ tokens,
                  const uint32_t* __restrict__ part, Results r) {
  __shared__ uint64_t keys[kJoinKeys];
  __shared__ uint64_t best[kLogprobsMaxTopK];
  __shared__ int count_s;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const int64_t words = split_words(p.top_k);
  const uint32_t* in = part + row * nsplit * words;
  // Each wave folds the states, and takes the bound, alone.
  Soft s = {-INFINITY, 0.f, 0.f};
  uint32_t high = ~0u;
  if (lane < nsplit) {
    const uint32_t* w = in + lane * words;
    s = {__builtin_bit_cast(float, w[0]), __builtin_bit_cast(float, w[1]), __builtin_bit_cast(float, w[2])};
    if (p.top_k) high = w[4 + 2 * ((p.top_k + nsplit - 1) / nsplit - 1) + 1];
  }
  const int n = nsplit * p.top_k;
  constexpr int kMine = kJoinKeys / kThreads;
  uint64_t mine[kMine];
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    const int i = j * kThreads + threadIdx.x;
    mine[j] = 0;
    if (i < n) {
      const int split = i / p.top_k;
      const uint32_t* w = in + split * words + 4 + 2 * (i - split * p.top_k);
      mine[j] = (uint64_t)w[1] << 32 | w[0];
    }
  }
  const int64_t token = read_token(tokens, p.token_bytes, row);
  const bool known = token >= 0 && token < p.V;
  const float chosen = known ? (float)logits[row * p.V + token] : 0.f;
  if (threadIdx.x == 0) count_s = 0;
  for (int d = 1; d < nsplit; d <<= 1)
    s = join(s, Soft{__shfl_xor(s.m, d), __shfl_xor(s.l, d), __shfl_xor(s.a, d)});
  if (threadIdx.x == 0) write_row(r, row, s, known, chosen);
  if (p.top_k == 0) return;
  const uint32_t bound = ~wave_max_u(~high);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kMine; ++j)
    if (mine[j] != 0 && (uint32_t)(mine[j] >> 32) >= bound) keys[atomicAdd(&count_s, 1)] = mine[j];
  __syncthreads();
  rank_keys(keys, count_s, best, 0, best, p.top_k);
  __syncthreads();
  write_top(r, row, __shfl(s.m, 0), logf(__shfl(s.l, 0)), best, p.top_k);
}

// Elementwise over the logits, a row's numbers read once a workgroup. Bound by
// HBM: 2000 x 32000 bf16, 256 MB, in 45 us (5.7 TB/s).
template <typename T, bool kStream>
__global__ void __launch_bounds__(kThreads)
    logprobs_grad(LogprobsParams p, int nsplit, const T* __restrict__ logits, const void* __restrict__ tokens,
                  const float* __restrict__ lse, const float* __restrict__ entropy,
                  const float* __restrict__ d_logprobs, const float* __restrict__ d_entropy, T* __restrict__ dx) {
  constexpr int E = kVecElems<T>;
  constexpr int NV = kChunk / kThreads / E;
  const int64_t row = blockIdx.x / nsplit;
  const int64_t base = (int64_t)(blockIdx.x % nsplit) * kChunk;
  const T* x = logits + row * p.V;
  typename Vec<T>::type v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t at = base + (int64_t)(i * kThreads + threadIdx.x) * E;
    v[i] = load_vec<T, kStream>(x + std::min(at, p.V - 1), p.V - at, (T)0.f);
  }
  const int64_t token = read_token(tokens, p.token_bytes, row);
  const bool known = token >= 0 && token < p.V;
  const float g = known ? d_logprobs[row] : 0.f, h = d_entropy[row], z = lse[row], H = entropy[row];
  // h == 0 leaves the entropy out: where it is NaN or infinite, and g's part alone is not.
  const float c0 = h == 0.f ? -g : -fmaf(h, H, g);
  // A row that no gradient reaches has none, whatever it holds (a padded row).
  const bool none = g == 0.f && h == 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int64_t at = base + (int64_t)(i * kThreads + threadIdx.x) * E;
    const int64_t n = p.V - at;
    if (n <= 0) continue;
    typename Vec<T>::type o;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      // p log p is 0 at p = 0: -inf's distance is made finite.
      const float d = __builtin_elementwise_maximum((float)v[i][e] - z, -1e4f);
      const float w = __builtin_amdgcn_exp2f(d * kLog2e);
      float y = none ? 0.f : w * fmaf(-h, d, c0);
      if (at + e == token) y += g;
      o[e] = (T)y;
    }
    store_vec<T, kStream>(dx + row * p.V + at, n, o);
  }
}

// Splits of a row, whole chunks each: those of the least estimated time, in us.
// A workgroup alone takes `alone`; together they take `all`, of which the chip
// does 1024 chunks, 4 workgroups a CU, in `unit` (by HBM for f32, by the
// exponentials and the candidates for 16 bits), with 0.7 of a chunk to begin
// and end each and half a round more where there are rounds; where both count,
// they add as squares do. Measured (estimated), bf16, 20 likeliest, V = 128256:
// 8 rows in 16 / 8 / 4 splits 12.4 / 13.9 / 19.6 us (13.1 / 14.4 / 18.6), 64 rows
// in 16 / 8 17.6 / 16.2 (16.9 / 16.4), 128 rows in 8 / 4 / 2 20.7 / 22.8 / 28.7
// (21.1 / 22.7 / 30.3); 5 likeliest: 256 rows in 4 / 2 / 1 26.8 / 31.6 / 38.1
// (30.2 / 33.2 / 41.2), 256 rows of 32000 in 4 / 1 14.2 / 13.2 (14.3 / 13.5).
struct Split {
  int n;
  int64_t per;
};
Split split_of(const LogprobsParams& p, DType t) {
  const int64_t chunks = (p.V + kChunk - 1) / kChunk;
  const int64_t most = std::min<int64_t>(chunks, p.top_k ? std::min(kJoinSplits, kJoinKeys / p.top_k) : kJoinSplits);
  const double k = p.top_k, unit = t == DType::kF32 ? 6.5 : p.top_k ? 5.0 : 3.3;
  int64_t best = chunks;
  double least = INFINITY;
  for (int64_t n = 1; n <= most; ++n) {
    const int64_t per = (chunks + n - 1) / n;
    const double rounds = static_cast<double>(p.rows) * n / 1024;
    const double all = unit * (per + 0.7) * (rounds > 1 ? rounds + 0.5 : rounds);
    const double alone = p.top_k ? 4.3 + 0.025 * k + (1.8 + 0.03 * k) * per : 3.4 + 1.5 * per;
    const double time = std::sqrt(all * all + alone * alone) + (n == 1 ? 0 : p.top_k ? 3.6 + 0.007 * n * k : 3.2);
    if (time < least) {
      least = time;
      best = per;
    }
  }
  return {static_cast<int>((chunks + best - 1) / best), best * kChunk};
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(Code::kInternal, strformat("%s launch failed: %s", what, hipGetErrorString(e)));
}

}  // namespace

size_t token_logprobs_scratch_bytes(const LogprobsParams& p, DType t) {
  const int n = split_of(p, t).n;
  return n > 1 ? static_cast<size_t>(p.rows) * n * split_words(p.top_k) * sizeof(uint32_t) : 0;
}

void launch_token_logprobs(hipStream_t s, const LogprobsParams& p, DType t, const void* logits, const void* tokens,
                           float* logprobs, float* entropy, float* lse, float* top_logprobs, int32_t* top_tokens,
                           void* scratch) {
  if (p.rows == 0) return;
  const Split sp = split_of(p, t);
  const dim3 grid(static_cast<uint32_t>(p.rows * sp.n)), block(kThreads);
  uint32_t* part = static_cast<uint32_t*>(scratch);
  const Results r = {logprobs, entropy, lse, top_logprobs, top_tokens};
  auto go = [&](auto tag) {
    using T = decltype(tag);
    const T* x = static_cast<const T*>(logits);
    const bool stream = p.rows * p.V * static_cast<int64_t>(sizeof(T)) >= kStreamBytes;
#define PJRTX_LOGPROBS(TOP, STREAM) \
  hipLaunchKernelGGL((logprobs_split<T, TOP, STREAM>), grid, block, 0, s, p, sp.n, sp.per, x, tokens, part, r)
    if (p.top_k && stream) PJRTX_LOGPROBS(true, true);
    else if (p.top_k) PJRTX_LOGPROBS(true, false);
    else if (stream) PJRTX_LOGPROBS(false, true);
    else PJRTX_LOGPROBS(false, false);
#undef PJRTX_LOGPROBS
    if (sp.n > 1)
      hipLaunchKernelGGL((logprobs_join<T>), dim3(static_cast<uint32_t>(p.rows)), block, 0, s, p, sp.n, x, tokens, part,
                         r);
  };
  if (t == DType::kF32) go(float());
  else if (t == DType::kBF16) go(bf16_t());
  else go(f16_t());
  check_launch("token_logprobs");
}

void launch_token_logprobs_grad(hipStream_t s, const LogprobsParams& p, DType t, const void* logits,
                                const void* tokens, const float* lse, const float* entropy, const float* d_logprobs,
                                const float* d_entropy, void* d_logits) {
  if (p.rows == 0) return;
  const int n = static_cast<int>((p.V + kChunk - 1) / kChunk);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    const dim3 grid(static_cast<uint32_t>(p.rows * n)), block(kThreads);
    const T* x = static_cast<const T*>(logits);
    T* dx = static_cast<T*>(d_logits);
    if (p.rows * p.V * static_cast<int64_t>(sizeof(T)) >= kStreamBytes)
      hipLaunchKernelGGL((logprobs_grad<T, true>), grid, block, 0, s, p, n, x, tokens, lse, entropy, d_logprobs,
                         d_entropy, dx);
    else
      hipLaunchKernelGGL((logprobs_grad<T, false>), grid, block, 0, s, p, n, x, tokens, lse, entropy, d_logprobs,
                         d_entropy, dx);
  };
  if (t == DType::kF32) go(float());
  else if (t == DType::kBF16) go(bf16_t());
  else go(f16_t());
  check_launch("token_logprobs_grad");
}

}  // namespace pjrtx
