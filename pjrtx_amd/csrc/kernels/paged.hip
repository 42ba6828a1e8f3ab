// Attention of one new token a sequence over a paged key-value cache, and the
// rows that are written into its pages.
//
// Work units. A row is one sequence with one key-value head and up to 16 of
// the query heads that share it, so that keys and values are read once for
// them. The host knows the table's capacity but no length, so the device cuts
// the work: every workgroup adds the sequences' 32-key tiles (`lengths` is one
// short read, most of it from L2) and takes unit blockIdx.x of rows x splits,
// where a split is `unit_tiles` tiles: about kUnits splits in all, of one size
// whatever the lengths are. A table far larger than its sequences costs
// nothing, and a long sequence among short ones is cut finer than they are.
//
// A split of a row that has several writes its softmax's (max, sum,
// unnormalised output) to scratch; paged_combine folds them in split order.
#include <algorithm>
#include <cmath>

#include "kernels/operators.h"
#include "kernels/vec.h"

namespace pjrtx {
namespace {

constexpr int kTileKeys = 32;
constexpr int kUnits = 512;      // splits aimed at: two workgroups a CU
constexpr int kHeads = 16;       // query heads of a row
constexpr int kWaves = 4;
constexpr float kLog2e = 1.44269504088896340736f;

// What the kernels are given beside the tensors.
struct Shape {
  PagedParams p;
  int group;       // query heads of a key-value head
  int head_tiles;  // rows of a (sequence, key-value head)
  int heads;       // query heads of a row at most
  int rows;        // rows of a sequence: Hkv * head_tiles
  int64_t cap;     // keys the table holds
};

struct Sequence {
  int64_t lo, hi;  // attended keys
  int tile0, tiles;
};
__device__ __forceinline__ Sequence sequence_of(const Shape& s, const int32_t* lengths, int64_t b) {
  Sequence q;
  q.hi = std::min<int64_t>(std::max(lengths[b], 0), s.cap);
  q.lo = s.p.window > 0 ? std::max<int64_t>(0, q.hi - s.p.window) : 0;
  q.tile0 = (int)(q.lo / kTileKeys);
  q.tiles = (int)((q.hi + kTileKeys - 1) / kTileKeys) - q.tile0;
  return q;
}

__device__ __forceinline__ uint32_t wave_sum_u(uint32_t x) {
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) x += __shfl_xor(x, k);
  return x;
}

// Tiles of a split: whole rounds of the workgroup's waves.
__device__ __forceinline__ uint32_t unit_tiles(const Shape& s, const int32_t* lengths) {
  uint32_t total = 0;
#pragma unroll 4
  for (int64_t b = threadIdx.x & 63; b < s.p.B; b += 64) total += (uint32_t)sequence_of(s, lengths, b).tiles;
  total = wave_sum_u(total);
  const uint64_t per = ((uint64_t)total * s.rows + kUnits - 1) / kUnits;
  return (uint32_t)std::max<uint64_t>(kWaves, (per + kWaves - 1) / kWaves * kWaves);
}
__device__ __forceinline__ uint32_t splits_of(int tiles, uint32_t per) {
  return tiles <= (int)per ? 1u : ((uint32_t)tiles + per - 1) / per;
}

// Where a sequence stands in the order of units and of scratch slots: those of
// the sequences before it, in splits. `slots` counts those with several only.
struct Place {
  int64_t b;
  uint32_t before, slots, n;
};
// The sequence that holds split index `at` of the sequences' splits laid end
// to end, or (kByB) sequence `at` itself. Each wave of the workgroup finds it
// alone; false past the last.
template <bool kByB>
__device__ __forceinline__ bool find_place(const Shape& s, const int32_t* lengths, uint32_t per, uint32_t at,
                                           Place* out) {
  const int lane = threadIdx.x & 63;
  uint32_t before = 0, slots = 0;
  for (int64_t b0 = 0; b0 < s.p.B; b0 += 64) {
    const int64_t b = b0 + lane;
    const uint32_t n = b < s.p.B ? splits_of(sequence_of(s, lengths, b).tiles, per) : 0u;
    const uint32_t k = n > 1 ? n : 0u;
    uint32_t sum = n, ksum = k;  // inclusive over the lanes
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t a = __shfl_up(sum, d), c = __shfl_up(ksum, d);
      if (lane >= d) {
        sum += a;
        ksum += c;
      }
    }
    const uint32_t first = before + sum - n;
    const bool mine = kByB ? b == (int64_t)at : at >= first && at < first + n;
    const uint64_t who = __ballot(mine);
    if (who) {
      const int src = __ffsll((unsigned long long)who) - 1;
      out->b = b0 + src;
      out->before = __shfl(first, src);
      out->slots = __shfl(slots + ksum - k, src);
      out->n = __shfl(n, src);
      return true;
    }
    before += __shfl(sum, 63);
    slots += __shfl(ksum, 63);
  }
  return false;
}

struct Unit {
  int64_t b;
  int kv_head, head0, heads;  // query heads head0 .. head0 + heads - 1
  uint32_t split, n;
  int64_t slot;               // scratch slot (n > 1)
  int64_t lo, hi;             // the sequence's attended keys
  int tile0, tile1;           // the split's tiles
};
__device__ __forceinline__ bool find_unit(const Shape& s, const int32_t* lengths, Unit* u) {
  const uint32_t per = unit_tiles(s, lengths);
  const uint32_t r = blockIdx.x % (uint32_t)s.rows;
  Place pl;
  if (!find_place<false>(s, lengths, per, blockIdx.x / (uint32_t)s.rows, &pl)) return false;
  const Sequence q = sequence_of(s, lengths, pl.b);
  u->b = pl.b;
  u->kv_head = (int)r / s.head_tiles;
  const int ht = (int)r % s.head_tiles;
  u->head0 = u->kv_head * s.group + ht * kHeads;
  u->heads = std::min(kHeads, s.group - ht * kHeads);
  u->split = blockIdx.x / (uint32_t)s.rows - pl.before;
  u->n = pl.n;
  u->slot = (int64_t)pl.slots * s.rows + (int64_t)r * pl.n + u->split;
  u->lo = q.lo;
  u->hi = q.hi;
  u->tile0 = q.tile0 + (int)(u->split * per);
  u->tile1 = std::min(q.tile0 + q.tiles, u->tile0 + (int)per);
  return true;
}

// Key j's row of the pages (in rows of D elements), -1 where the table's entry
// names no page. j is clamped to the table.
__device__ __forceinline__ int64_t row_of(const Shape& s, const int32_t* table, int64_t b, int kv_head, int64_t j) {
  const int64_t e = std::min(j / s.p.S, s.p.M - 1);
  const int64_t page = table[b * s.p.M + e];
  if (page < 0 || page >= s.p.P) return -1;
  return (page * s.p.Hkv + kv_head) * s.p.S + (j - e * s.p.S);
}

// Scratch of a slot: (max, sum) of each head, then each head's D outputs. A
// sum of -1 marks a split without any attended key.
__device__ __forceinline__ float* slot_state(const Shape& s, float* scratch, int64_t slot) {
  return scratch + slot * s.heads * (s.p.D + 2);
}

// The workgroup's waves meet over one head: state of wave w in ml[w], its
// outputs in o[w]. Writes the row's result, or the split's partial one.
template <typename T>
__device__ __forceinline__ void finish_head(const Shape& s, const Unit& u, int head, const float (*ml)[2],
                                            const float* o, int o_stride, T* out, float* scratch) {
  float m = -INFINITY;
  bool any = false;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (ml[w][1] < 0.f) continue;
    any = true;
    m = fmaxf(m, ml[w][0]);
  }
  const float ref = m == -INFINITY ? 0.f : m;
  float f[kWaves], l = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    f[w] = ml[w][1] < 0.f ? 0.f : exp2f(ml[w][0] - ref);
    l += ml[w][1] < 0.f ? 0.f : ml[w][1] * f[w];
  }
  float* state = u.n > 1 ? slot_state(s, scratch, u.slot) : nullptr;
  if (state && threadIdx.x == 0) {
    state[2 * head] = m;
    state[2 * head + 1] = any ? l : -1.f;
  }
  for (int d = threadIdx.x; d < s.p.D; d += kWaves * 64) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (ml[w][1] >= 0.f || ml[w][1] != ml[w][1]) v += f[w] * o[w * o_stride + d];
    if (state) state[2 * s.heads + (int64_t)head * s.p.D + d] = v;
    else out[(u.b * s.p.Hq + u.head0 + head) * s.p.D + d] = (T)(any ? v / l : 0.f);
  }
}

// Any head dim up to 512 and any page size: a wave takes a key at a time, its
// lanes across the head dim, one query head after another.
constexpr int kMaxHeadDim = 512;
template <typename T>
__global__ void __launch_bounds__(kWaves * 64)
    paged_any(Shape s, const T* __restrict__ q, const T* __restrict__ k_pages, const T* __restrict__ v_pages,
              const int32_t* __restrict__ table, const int32_t* __restrict__ lengths, T* __restrict__ out,
              float* __restrict__ scratch) {
  constexpr int J = kMaxHeadDim / 64;
  __shared__ float ml[kWaves][2];
  __shared__ float ow[kWaves][kMaxHeadDim];
  Unit u;
  if (!find_unit(s, lengths, &u)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int D = s.p.D;
  for (int h = 0; h < u.heads; ++h) {
    const T* qr = q + (u.b * s.p.Hq + u.head0 + h) * D;
    float qv[J], o[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      qv[j] = lane + 64 * j < D ? (float)qr[lane + 64 * j] : 0.f;
      o[j] = 0.f;
    }
    float m = -INFINITY, l = -1.f;
    for (int t = u.tile0 + wave; t < u.tile1; t += kWaves) {
      const int64_t first = std::max<int64_t>(u.lo, (int64_t)t * kTileKeys);
      const int64_t last = std::min<int64_t>(u.hi, ((int64_t)t + 1) * kTileKeys);
      for (int64_t key = first; key < last; ++key) {
        const int64_t row = row_of(s, table, u.b, u.kv_head, key);
        if (row < 0) continue;
        const T *kr = k_pages + row * D, *vr = v_pages + row * D;
        float dot = 0.f, vv[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int d = lane + 64 * j;
          if (d < D) dot = fmaf(qv[j], (float)kr[d], dot);
          vv[j] = d < D ? (float)vr[d] : 0.f;
        }
        const float x = wave_sum(dot) * s.p.scale * kLog2e;
        if (l < 0.f) l = 0.f;
        const float mn = fmaxf(m, x);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2f(m - ref), pe = exp2f(x - ref);
        l = l * alpha + pe;
#pragma unroll
        for (int j = 0; j < J; ++j) o[j] = fmaf(pe, vv[j], o[j] * alpha);
        m = mn;
      }
    }
    if (lane == 0) {
      ml[wave][0] = m;
      ml[wave][1] = l;
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (lane + 64 * j < D) ow[wave][lane + 64 * j] = o[j];
    __syncthreads();
    finish_head<T>(s, u, h, ml, ow[0], kMaxHeadDim, out, scratch);
    __syncthreads();
  }
}

// One workgroup a query head: folds the splits of its row in split order.
template <typename T>
__global__ void __launch_bounds__(256)
    paged_combine(Shape s, const int32_t* __restrict__ lengths, const float* __restrict__ scratch,
                  T* __restrict__ out) {
  __shared__ float m_s[kUnits + 1], l_s[kUnits + 1];
  const int64_t b = blockIdx.x / s.p.Hq;
  const int hq = (int)(blockIdx.x % s.p.Hq);
  const uint32_t per = unit_tiles(s, lengths);
  Place pl;
  if (!find_place<true>(s, lengths, per, (uint32_t)b, &pl) || pl.n <= 1) return;
  const int kv_head = hq / s.group, ht = (hq % s.group) / kHeads, head = (hq % s.group) % kHeads;
  const int64_t slot0 = (int64_t)pl.slots * s.rows + (int64_t)(kv_head * s.head_tiles + ht) * pl.n;
  const int64_t words = (int64_t)s.heads * (s.p.D + 2);
  const float* base = scratch + slot0 * words;
  for (uint32_t i = threadIdx.x; i < pl.n; i += 256) {
    m_s[i] = base[i * words + 2 * head];
    l_s[i] = base[i * words + 2 * head + 1];
  }
  __syncthreads();
  float m = -INFINITY;
  bool any = false;
  for (uint32_t i = 0; i < pl.n; ++i) {
    if (l_s[i] < 0.f) continue;
    any = true;
    m = fmaxf(m, m_s[i]);
  }
  const float ref = m == -INFINITY ? 0.f : m;
  for (int d = threadIdx.x; d < s.p.D; d += 256) {
    float l = 0.f, v = 0.f;
    for (uint32_t i = 0; i < pl.n; ++i) {
      if (l_s[i] < 0.f) continue;
      const float f = exp2f(m_s[i] - ref);
      l += l_s[i] * f;
      v += f * base[i * words + 2 * s.heads + (int64_t)head * s.p.D + d];
    }
    out[(b * s.p.Hq + hq) * s.p.D + d] = (T)(any ? v / l : 0.f);
  }
}

Shape shape_of(const PagedParams& p) {
  Shape s;
  s.p = p;
  s.group = p.Hq / p.Hkv;
  s.head_tiles = (s.group + kHeads - 1) / kHeads;
  s.heads = std::min(s.group, kHeads);
  s.rows = p.Hkv * s.head_tiles;
  s.cap = p.M * p.S;
  return s;
}
// Splits a sequence can have at most, were it alone as long as the table.
int64_t most_splits(const Shape& s) {
  const int64_t tiles = (s.cap + kTileKeys - 1) / kTileKeys;
  return std::min<int64_t>((tiles + kWaves - 1) / kWaves, kUnits);
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(Code::kInternal, strformat("%s launch failed: %s", what, hipGetErrorString(e)));
}

}  // namespace

size_t paged_attention_scratch_bytes(const PagedParams& p, DType t) {
  const Shape s = shape_of(p);
  if (p.B == 0 || most_splits(s) <= 1) return 0;
  // A sequence of n > 1 splits has more than n / 2 of unit_tiles each, so the
  // split sequences' rows have fewer than 2 kUnits of them in all.
  const int64_t slots = std::min<int64_t>(2 * kUnits, p.B * s.rows * most_splits(s));
  return static_cast<size_t>(slots) * s.heads * (p.D + 2) * sizeof(float);
}

void launch_paged_attention(hipStream_t stream, const PagedParams& p, DType t, const void* q, const void* k_pages,
                            const void* v_pages, const int32_t* page_table, const int32_t* lengths, void* out,
                            void* scratch) {
  if (p.B == 0) return;
  const Shape s = shape_of(p);
  const int64_t rows = p.B * s.rows;
  // Splits of unit_tiles tiles, and one that is short a row.
  const int64_t units = std::min<int64_t>(rows * most_splits(s), rows + kUnits);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL((paged_any<T>), dim3(static_cast<uint32_t>(units)), dim3(kWaves * 64), 0, stream, s,
                       static_cast<const T*>(q), static_cast<const T*>(k_pages), static_cast<const T*>(v_pages),
                       page_table, lengths, static_cast<T*>(out), static_cast<float*>(scratch));
    if (scratch)
      hipLaunchKernelGGL((paged_combine<T>), dim3(static_cast<uint32_t>(p.B * p.Hq)), dim3(256), 0, stream, s, lengths,
                         static_cast<const float*>(scratch), static_cast<T*>(out));
  };
  if (t == DType::kF32) go(float());
  else if (t == DType::kBF16) go(bf16_t());
  else go(f16_t());
  check_launch("paged_attention");
}

// ------------------------------------------------------------------ append
// A workgroup copies the keys and values of kRows new rows. Of rows that name
// one slot the last stays whatever order the workgroups run in: each reads
// the slots after its rows and leaves a row out whose slot comes again. The
// scan is 4 bytes a later row and workgroup (8 rows: 16 MB of L2 reads at 8192
// rows, whose copy moves 64 MB and more).
namespace {

template <typename U, int kRows>
__global__ void __launch_bounds__(256)
    append_rows(AppendParams p, int64_t units, U* __restrict__ k_pages, U* __restrict__ v_pages,
                const U* __restrict__ k_new, const U* __restrict__ v_new, const void* __restrict__ slots) {
  __shared__ int64_t slot_s[kRows];
  __shared__ int again_s[kRows];
  const int64_t n0 = (int64_t)blockIdx.x * kRows;
  auto slot_at = [&](int64_t i) {
    return p.slot_bytes == 8 ? static_cast<const int64_t*>(slots)[i] : (int64_t)static_cast<const int32_t*>(slots)[i];
  };
  if (threadIdx.x < kRows) {
    const int64_t n = n0 + threadIdx.x;
    const int64_t slot = n < p.N ? slot_at(n) : -1;
    slot_s[threadIdx.x] = slot >= 0 && slot < p.P * p.S ? slot : -1;
    again_s[threadIdx.x] = 0;
  }
  __syncthreads();
  for (int64_t j = n0 + 1 + threadIdx.x; j < p.N; j += 256) {
    const int64_t other = slot_at(j);
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (other == slot_s[r] && j > n0 + r) again_s[r] = 1;  // only ever set
  }
  __syncthreads();
  // `units` of U make a head's D elements.
  const int64_t per_row = p.Hkv * units;
  for (int r = 0; r < kRows; ++r) {
    const int64_t slot = slot_s[r];
    if (slot < 0 || again_s[r]) continue;
    const int64_t page = slot / p.S, at = slot - page * p.S;
    for (int64_t i = threadIdx.x; i < per_row; i += 256) {
      const int64_t h = i / units, c = i - h * units;
      const int64_t to = ((page * p.Hkv + h) * p.S + at) * units + c, from = (n0 + r) * per_row + i;
      k_pages[to] = k_new[from];
      v_pages[to] = v_new[from];
    }
  }
}

}  // namespace

void launch_paged_append(hipStream_t s, const AppendParams& p, int elem_bytes, void* k_pages, void* v_pages,
                         const void* k_new, const void* v_new, const void* slots) {
  if (p.N == 0 || p.Hkv == 0 || p.D == 0 || p.P == 0 || p.S == 0) return;
  const int64_t row_bytes = p.D * elem_bytes;
  uint64_t addresses = static_cast<uint64_t>(row_bytes);
  for (const void* x : {static_cast<const void*>(k_pages), static_cast<const void*>(v_pages), k_new, v_new})
    addresses |= reinterpret_cast<uint64_t>(x);
  auto go = [&](auto tag) {
    using U = decltype(tag);
    const int64_t units = row_bytes / static_cast<int64_t>(sizeof(U));
    U *kp = static_cast<U*>(k_pages), *vp = static_cast<U*>(v_pages);
    const U *kn = static_cast<const U*>(k_new), *vn = static_cast<const U*>(v_new);
    if (p.N <= 1024)
      hipLaunchKernelGGL((append_rows<U, 1>), dim3(static_cast<uint32_t>(p.N)), dim3(256), 0, s, p, units, kp, vp, kn,
                         vn, slots);
    else
      hipLaunchKernelGGL((append_rows<U, 8>), dim3(static_cast<uint32_t>((p.N + 7) / 8)), dim3(256), 0, s, p, units,
                         kp, vp, kn, vn, slots);
  };
  // The widest unit that every row starts on.
  if (addresses % 16 == 0) go(uint4());
  else if (addresses % 4 == 0) go(uint32_t());
  else if (addresses % 2 == 0) go(uint16_t());
  else go(uint8_t());
  check_launch("paged_append");
}

}  // namespace pjrtx
