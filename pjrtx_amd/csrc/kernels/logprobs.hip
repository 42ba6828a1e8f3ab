// Log probabilities of given tokens, the distribution's entropy and its
// likeliest tokens, in one pass over the logits; and their gradient.
//
// A row is split over workgroups, which read it in chunks of 8192 elements
// held in registers. Each thread keeps an online softmax of its own (largest
// x so far m, l = sum e^(x-m), a = sum e^(x-m) (x-m)), from which lse = m +
// log l and entropy = log l - a / l: the entropy's terms are taken about m,
// not about zero, so nothing large cancels. Elements that may be among the
// row's top_k (bounded below by the top_k-th largest of the threads' maxima,
// then by the best found so far) go to a list in LDS and are ranked there by
// value, then by lowest index. logprobs_join folds a row's splits in order.
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
constexpr int kJoinKeys = 1024;            // top_k keys of all splits that the join ranks
constexpr float kLog2e = 1.44269504088896340736f;

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
__device__ __forceinline__ Soft join(const Soft& x, const Soft& y) {
  const float m = fmaxf(x.m, y.m);
  if (m == -INFINITY) return {m, x.l + y.l, x.a + y.a};  // 0s, or NaNs
  // A side of no elements has l = a = 0 at m = -inf: its shift is finite here.
  const float dx = fmaxf(x.m - m, -1e4f), dy = fmaxf(y.m - m, -1e4f);
  const float fx = exp2f(dx * kLog2e), fy = exp2f(dy * kLog2e);
  return {m, x.l * fx + y.l * fy, fx * (x.a + dx * x.l) + fy * (y.a + dy * y.l)};
}

// The split's results: {m, l, a}, then top_k keys, largest first.
__host__ __device__ constexpr int64_t split_words(int top_k) { return 4 + 2 * (int64_t)top_k; }

// Ranks the n distinct keys at `keys` and leaves the top_k largest (or n, then
// zeros) in order at `best`. Called by the whole workgroup.
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int n, uint64_t* best, int top_k) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = keys[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += keys[j] > mine ? 1 : 0;
    if (above < top_k) best[above] = mine;
  }
  for (int i = n + threadIdx.x; i < top_k; i += kThreads) best[i] = 0;
}

__device__ __forceinline__ int64_t read_token(const void* tokens, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(tokens)[i] : (int64_t)static_cast<const int32_t*>(tokens)[i];
}

// A workgroup's share of a row: elements [lo, hi).
template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads)
    logprobs_split(LogprobsParams p, int nsplit, int64_t per, const T* __restrict__ logits,
                   uint32_t* __restrict__ part) {
  constexpr int E = kVecElems<T>;
  constexpr int NV = kChunk / kThreads / E;
  __shared__ uint64_t cand[kTop ? kCandidates + kLogprobsMaxTopK : 1];
  __shared__ uint64_t best[kTop ? kLogprobsMaxTopK : 1];
  __shared__ uint32_t maxima[kTop ? kThreads : 1];
  __shared__ uint64_t pick[kTop ? kThreads / 64 : 1];
  __shared__ uint32_t bound_s;
  __shared__ int count_s;
  __shared__ Soft soft_s[kThreads / 64];
  const int64_t row = blockIdx.x / nsplit;
  const int split = (int)(blockIdx.x % nsplit);
  const T* x = logits + row * p.V;
  const int64_t lo = split * per, hi = std::min(p.V, lo + per);
  const int tid = threadIdx.x;
  Soft s = {-INFINITY, 0.f, 0.f};
  uint32_t bound = 0;  // elements of a lower order are not among the top_k
  bool have = false;   // best holds top_k keys of this split
  if constexpr (kTop) {
    for (int i = tid; i < p.top_k; i += kThreads) best[i] = 0;
  }
  for (int64_t base = lo; base < hi; base += kChunk) {
    typename Vec<T>::type v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t at = base + (int64_t)(i * kThreads + tid) * E;
      v[i] = load_vec<T>(x + std::min(at, p.V - 1), hi - at, (T)-INFINITY);
    }
    float cm = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) cm = fmaxf(cm, (float)v[i][e]);
    const float m = fmaxf(s.m, cm);
    if (m > s.m) {  // also the first finite chunk, from l = a = 0
      const float d = fmaxf(s.m - m, -1e4f), f = exp2f(d * kLog2e);
      s.a = f * (s.a + d * s.l);
      s.l *= f;
      s.m = m;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        // -inf weighs nothing: its distance is made finite for a's product.
        const float d = __builtin_elementwise_maximum((float)v[i][e] - ref, -1e4f);
        const float w = __builtin_amdgcn_exp2f(d * kLog2e);
        s.l += w;
        s.a = fmaf(w, d, s.a);
      }
    if constexpr (kTop) {
      const int64_t left = hi - base;
      auto index = [&](int i, int e) { return (int64_t)(i * kThreads + tid) * E + e; };
      if (!have) {
        // top_k <= 128 < 256 threads: the top_k-th largest of the threads'
        // maxima is at or below the top_k-th largest element.
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (index(i, e) < left) mine = std::max(mine, order_of((float)v[i][e]));
        maxima[tid] = mine;
        __syncthreads();
        int above = 0;
        for (int j = 0; j < kThreads; ++j) above += maxima[j] > mine || (maxima[j] == mine && j < tid) ? 1 : 0;
        if (above == p.top_k - 1) bound_s = mine;
        __syncthreads();
        bound = bound_s;
      }
      if (tid == 0) count_s = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t o = order_of((float)v[i][e]);
          // With top_k keys in hand their last one's order must be passed, or
          // met at a lower index: those all came before.
          if ((have ? o > bound : o >= bound) && index(i, e) < left) {
            const int at = atomicAdd(&count_s, 1);
            if (at < kCandidates) cand[at] = key_of((float)v[i][e], base + index(i, e));
          }
        }
      __syncthreads();
      const int n = count_s;
      if (n > kCandidates) {
        // Too many equal or ordered elements for the list: the top_k of the
        // chunk one after another, each the largest key below the last.
        uint64_t last = ~0ull;
        for (int k = 0; k < p.top_k; ++k) {
          uint64_t mine = 0;
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (index(i, e) < left) {
                const uint64_t key = key_of((float)v[i][e], base + index(i, e));
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
          if (last == 0) break;
        }
      }
      int m_keys = n > kCandidates ? p.top_k : n;
      if (m_keys > 0) {
        for (int i = tid; i < p.top_k; i += kThreads) cand[m_keys + i] = best[i];
        __syncthreads();
        // Empty places of `best` are equal keys of 0 behind all others.
        int held = p.top_k;
        if (best[p.top_k - 1] == 0) {
          held = 0;
          for (int i = 0; i < p.top_k; ++i) held += best[i] != 0 ? 1 : 0;
        }
        __syncthreads();
        rank_keys(cand, m_keys + held, best, p.top_k);
        __syncthreads();
      }
      const uint64_t least = best[p.top_k - 1];
      have = least != 0;
      bound = (uint32_t)(least >> 32);
      __syncthreads();
    }
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s = join(s, Soft{__shfl_xor(s.m, d), __shfl_xor(s.l, d), __shfl_xor(s.a, d)});
  if ((tid & 63) == 0) soft_s[tid >> 6] = s;
  __syncthreads();
  uint32_t* out = part + (row * nsplit + split) * split_words(p.top_k);
  if (tid == 0) {
    const Soft t = join(join(soft_s[0], soft_s[1]), join(soft_s[2], soft_s[3]));
    out[0] = __builtin_bit_cast(uint32_t, t.m);
    out[1] = __builtin_bit_cast(uint32_t, t.l);
    out[2] = __builtin_bit_cast(uint32_t, t.a);
  }
  if constexpr (kTop) {
    for (int i = tid; i < p.top_k; i += kThreads) {
      out[4 + 2 * i] = (uint32_t)best[i];
      out[5 + 2 * i] = (uint32_t)(best[i] >> 32);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    logprobs_join(LogprobsParams p, int nsplit, const T* __restrict__ logits, const void* __restrict__ tokens,
                  const uint32_t* __restrict__ part, float* __restrict__ logprobs, float* __restrict__ entropy,
                  float* __restrict__ lse_out, float* __restrict__ top_logprobs, int32_t* __restrict__ top_tokens) {
  __shared__ uint64_t keys[kJoinKeys];
  __shared__ uint64_t best[kLogprobsMaxTopK];
  __shared__ float lse_s;
  __shared__ int count_s;
  const int64_t row = blockIdx.x;
  const int64_t words = split_words(p.top_k);
  const uint32_t* in = part + row * nsplit * words;
  if (threadIdx.x == 0) {
    count_s = 0;
    Soft s = {-INFINITY, 0.f, 0.f};
    for (int k = 0; k < nsplit; ++k)
      s = join(s, Soft{__builtin_bit_cast(float, in[k * words]), __builtin_bit_cast(float, in[k * words + 1]),
                       __builtin_bit_cast(float, in[k * words + 2])});
    const float log_l = logf(s.l);
    const float lse = s.m + log_l;
    const int64_t token = read_token(tokens, p.token_bytes, row);
    logprobs[row] = token >= 0 && token < p.V ? (float)logits[row * p.V + token] - lse : 0.f;
    entropy[row] = log_l - s.a / s.l;
    lse_out[row] = lse;
    lse_s = lse;
  }
  if (p.top_k == 0) return;
  __syncthreads();
  for (int i = threadIdx.x; i < nsplit * p.top_k; i += kThreads) {
    const uint32_t* w = in + (i / p.top_k) * words + 4 + 2 * (i % p.top_k);
    const uint64_t key = (uint64_t)w[1] << 32 | w[0];
    if (key != 0) keys[atomicAdd(&count_s, 1)] = key;  // distinct: their order does not matter
  }
  __syncthreads();
  rank_keys(keys, count_s, best, p.top_k);
  __syncthreads();
  for (int i = threadIdx.x; i < p.top_k; i += kThreads) {
    top_logprobs[row * p.top_k + i] = value_of((uint32_t)(best[i] >> 32)) - lse_s;
    top_tokens[row * p.top_k + i] = (int32_t)~(uint32_t)best[i];
  }
}

// Elementwise over the logits, a row's numbers read once a workgroup.
template <typename T>
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
    v[i] = load_vec<T>(x + std::min(at, p.V - 1), p.V - at, (T)0.f);
  }
  const int64_t token = read_token(tokens, p.token_bytes, row);
  const bool known = token >= 0 && token < p.V;
  const float g = known ? d_logprobs[row] : 0.f, h = d_entropy[row], z = lse[row], H = entropy[row];
  // h == 0 leaves the entropy out: where it is NaN or infinite, and g's part alone is not.
  const float c0 = h == 0.f ? -g : -fmaf(h, H, g);
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
      float y = w * fmaf(-h, d, c0);
      if (at + e == token) y += g;
      o[e] = (T)y;
    }
    store_vec<T>(dx + row * p.V + at, n, o);
  }
}

// Splits of a row: enough workgroups for the chip, whole chunks each, and no
// more keys than the join ranks.
struct Split {
  int n;
  int64_t per;
};
Split split_of(const LogprobsParams& p) {
  const int64_t chunks = (p.V + kChunk - 1) / kChunk;
  int64_t want = std::max<int64_t>(1, (1024 + p.rows - 1) / std::max<int64_t>(1, p.rows));
  want = std::min<int64_t>(want, p.top_k ? kJoinKeys / p.top_k : 64);
  const int64_t n = std::max<int64_t>(1, std::min(chunks, want));
  const int64_t per = (chunks + n - 1) / n * kChunk;
  return {static_cast<int>((p.V + per - 1) / per), per};
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(Code::kInternal, strformat("%s launch failed: %s", what, hipGetErrorString(e)));
}

}  // namespace

size_t token_logprobs_scratch_bytes(const LogprobsParams& p, DType t) {
  return static_cast<size_t>(p.rows) * split_of(p).n * split_words(p.top_k) * sizeof(uint32_t);
}

void launch_token_logprobs(hipStream_t s, const LogprobsParams& p, DType t, const void* logits, const void* tokens,
                           float* logprobs, float* entropy, float* lse, float* top_logprobs, int32_t* top_tokens,
                           void* scratch) {
  if (p.rows == 0) return;
  const Split sp = split_of(p);
  const dim3 grid(static_cast<uint32_t>(p.rows * sp.n)), rows(static_cast<uint32_t>(p.rows)), block(kThreads);
  uint32_t* part = static_cast<uint32_t*>(scratch);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    const T* x = static_cast<const T*>(logits);
    if (p.top_k) hipLaunchKernelGGL((logprobs_split<T, true>), grid, block, 0, s, p, sp.n, sp.per, x, part);
    else hipLaunchKernelGGL((logprobs_split<T, false>), grid, block, 0, s, p, sp.n, sp.per, x, part);
    hipLaunchKernelGGL((logprobs_join<T>), rows, block, 0, s, p, sp.n, x, tokens, part, logprobs, entropy, lse,
                       top_logprobs, top_tokens);
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
    hipLaunchKernelGGL((logprobs_grad<T>), dim3(static_cast<uint32_t>(p.rows * n)), dim3(kThreads), 0, s, p, n,
                       static_cast<const T*>(logits), tokens, lse, entropy, d_logprobs, d_entropy,
                       static_cast<T*>(d_logits));
  };
  if (t == DType::kF32) go(float());
  else if (t == DType::kBF16) go(bf16_t());
  else go(f16_t());
  check_launch("token_logprobs_grad");
}

}  // namespace pjrtx
