// Attention of one new token a sequence over a paged key-value cache, and the
// rows that are written into its pages.
//
// Work. A row is one sequence with one key-value head and up to 64 of the
// query heads that share it, so that keys and values are read once for them.
// The host knows the table's capacity but no length, so the device cuts the
// work: every workgroup adds the sequences' 32-key tiles (`lengths` is one
// short read, most of it from L2), and takes its equal share of the rows' tiles
// laid end to end: the end of one row, whole ones, the start of another. All
// workgroups of a launch are resident at once and end together whatever the
// lengths are; a table far larger than its sequences costs nothing. (64 rows of
// 32 to 4064 keys by 8 heads, 538 MB: splits of rows, each a workgroup, left
// the last ones alone on the chip, 113 us at best; shares take 100.) Where the
// table itself is so small that shares are one tile a wave, rows start on a
// workgroup's first tile instead, so that no workgroup walks two.
//
// A share of a row that is not all of it writes its softmax's (max, sum,
// unnormalised output) to scratch; paged_combine folds them in order.
//
// Long caches are bound by HBM: 2 sequences of 131072 keys by 8 heads of 128,
// f16, 537 MB in 99 us (5.4 TB/s), the 64 ragged ones 538 MB in 101 us. The
// fold takes 4 us where few keys do (600 keys: 5.6 + 4.3 us, all of it the
// latency of dependent reads: length, table, keys) and 8 at those sizes, about
// half of it behind the tiles. In the last arriving workgroup instead of its
// own launch it was no faster (10.7 and 10.5 us at 600 keys; 17.4 and 13.9 at
// 7 x 1500 f32), and a device-scope fence for it cost the tiles their L2 (321
// us for 101).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kernels/operators.h"
#include "kernels/vec.h"

namespace pjrtx {
namespace {

constexpr int kTileKeys = 32;
constexpr int kHeads = 16;       // query heads of a wave
constexpr int kSets = 4;         // such sets of a row at most
constexpr int kRowCost = 4;      // tiles; 0 / 2 / 4 / 8: 115 / 106 / 101 / 102 us at those 64 sequences
constexpr int kCus = 256;
constexpr int kMaxParts = 2 * kCus;  // of a row: at most one a workgroup
constexpr int kWaves = 4, kWavesLog = 2;
constexpr float kLog2e = 1.44269504088896340736f;

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery, 1994).
struct Divisor {
  uint32_t d = 1, m = 0, s = 0;
};
Divisor divisor_of(uint32_t d) {
  Divisor v;
  v.d = d;
  while (v.s < 31 && (1u << v.s) < d) ++v.s;
  v.m = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << v.s) - d)) / d + 1);
  return v;
}
__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divisor& v) { return (__umulhi(n, v.m) + n) >> v.s; }

// What the kernels are given beside the tensors.
struct Shape {
  PagedParams p;
  int group;       // query heads of a key-value head
  int sets;        // sets of kHeads query heads in a row: 1, 2 or 4,
  int sets_log;    // 2 to this
  int head_rows;   // rows of a (sequence, key-value head)
  int heads;       // query heads of a row at most
  int rows;        // rows of a sequence: Hkv * head_rows
  uint32_t cap;    // keys the table holds, below 2^31
  Divisor page;    // keys of a page
  int groups;      // workgroups of the launch
  bool aligned;    // rows start on a workgroup's first tile,
  int each;        // and have so many workgroups
};

struct Sequence {
  uint32_t lo, hi;  // attended keys
  int tile0, tiles;
};
__device__ __forceinline__ Sequence sequence_of(const Shape& s, const int32_t* lengths, int64_t b) {
  Sequence q;
  q.hi = std::min((uint32_t)std::max(lengths[b], 0), s.cap);
  q.lo = 0;
  q.tile0 = 0;  // known before the length is, where there is no window
  if (s.p.window > 0 && s.p.window < q.hi) {
    q.lo = q.hi - (uint32_t)s.p.window;
    q.tile0 = (int)(q.lo / kTileKeys);
  }
  q.tiles = (int)((q.hi + kTileKeys - 1) / kTileKeys) - q.tile0;
  return q;
}

__device__ __forceinline__ uint32_t wave_sum_u(uint32_t x) {
#pragma unroll
  for (int k = 32; k >= 1; k >>= 1) x += __shfl_xor(x, k);
  return x;
}

// Tiles that a row counts for in the rows laid end to end: its own, at least
// one, so that some workgroup answers for it; then kRowCost for the time that a
// workgroup takes to begin it.
__device__ __forceinline__ uint32_t span_of(int tiles) { return (uint32_t)std::max(tiles, 1) + kRowCost; }
// Tiles of a workgroup's share.
__device__ __forceinline__ uint32_t share_of(const Shape& s, const int32_t* lengths) {
  uint32_t total = 0;
#pragma unroll 4
  for (int64_t b = threadIdx.x & 63; b < s.p.B; b += 64) total += span_of(sequence_of(s, lengths, b).tiles);
  total = wave_sum_u(total) * (uint32_t)s.rows;
  return std::max<uint32_t>(kWaves, (total + s.groups - 1) / s.groups);
}

// The sequence whose rows hold tile `at` of all rows', and the tiles before it.
// Each wave of the workgroup finds it alone; false past the last.
__device__ __forceinline__ bool find_sequence(const Shape& s, const int32_t* lengths, uint32_t at, int64_t* b_out,
                                              uint32_t* before_out) {
  const int lane = threadIdx.x & 63;
  uint32_t before = 0;
  for (int64_t b0 = 0; b0 < s.p.B; b0 += 64) {
    const int64_t b = b0 + lane;
    const uint32_t n = b < s.p.B ? span_of(sequence_of(s, lengths, b).tiles) * (uint32_t)s.rows : 0u;
    uint32_t sum = n;  // inclusive over the lanes
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t a = __shfl_up(sum, d);
      if (lane >= d) sum += a;
    }
    const uint32_t first = before + sum - n;
    const uint64_t who = __ballot(at >= first && at < first + n);
    if (who) {
      const int src = __ffsll((unsigned long long)who) - 1;
      *b_out = b0 + src;
      *before_out = (uint32_t)__builtin_amdgcn_readlane((int)first, src);
      return true;
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  }
  return false;
}

// Key j's row of the pages (in rows of D elements), -1 where the table's entry
// names no page or j is past the table, as the keys of a last tile may be: its
// entry is read all the same, clamped, so that the read waits for no length.
// The pages have fewer than 2^31 rows.
__device__ __forceinline__ int row_of(const Shape& s, const int32_t* table, int64_t b, int kv_head, uint32_t j) {
  const uint32_t e = std::min(quotient(j, s.page), (uint32_t)s.p.M - 1);
  const int page = table[b * s.p.M + e];
  if (page < 0 || page >= s.p.P || j >= s.cap) return -1;
  return (page * s.p.Hkv + kv_head) * (int)s.page.d + (int)(j - e * s.page.d);
}

// What the workgroup that starts a row leaves for paged_combine, before the
// slots (unless rows start on a workgroup's first tile): the row's parts are
// that workgroup's and the n - 1 after it.
struct Row {
  uint32_t group, n;
};
// A workgroup has a slot for the end of a row that others start, and one for
// the start of a row.
__host__ __device__ constexpr int64_t slot_of(int64_t group, bool start) { return 2 * group + (start ? 1 : 0); }
// Scratch of a slot: (max, sum) of each head, then each head's D outputs. A
// sum of -1 marks a split without any attended key.
__device__ __forceinline__ float* slot_state(const Shape& s, float* scratch, int64_t slot) {
  return scratch + 2 * s.p.B * s.rows + slot * s.heads * (s.p.D + 2);
}

// The part of a row that a workgroup is at.
struct Unit {
  int64_t b;
  int kv_head, head0, heads;  // query heads head0 .. head0 + heads - 1
  bool whole;                 // all of the row
  int64_t slot;               // scratch slot otherwise
  uint32_t lo, hi;            // the sequence's attended keys
  int tile0, tile1;           // the part's tiles
};

__device__ __forceinline__ void set_unit(const Shape& s, Unit* u, uint32_t r, const Sequence& q, uint32_t tile,
                                         uint32_t n) {
  u->kv_head = (int)r / s.head_rows;
  const int first = ((int)r - u->kv_head * s.head_rows) * kHeads * s.sets;
  u->head0 = u->kv_head * s.group + first;
  u->heads = std::min(kHeads * s.sets, s.group - first);
  u->whole = tile == 0 && (int)n >= q.tiles;
  u->slot = slot_of(blockIdx.x, tile == 0);
  u->lo = q.lo;
  u->hi = q.hi;
  u->tile0 = q.tile0 + (int)tile;
  u->tile1 = q.tile0 + std::min(q.tiles, (int)(tile + n));
}

// Calls part(unit) for each part of the workgroup's share, the same on every
// thread.
template <bool kAligned, typename F>
__device__ __forceinline__ void for_parts(const Shape& s, const int32_t* lengths, float* scratch, const F& part) {
  Unit u;
  if constexpr (kAligned) {
    // Row by row, as many workgroups each as the table's keys could take.
    const uint32_t row = blockIdx.x / (uint32_t)s.each, tile = (blockIdx.x - row * (uint32_t)s.each) * kWaves;
    u.b = row / (uint32_t)s.rows;
    const Sequence q = sequence_of(s, lengths, u.b);
    if (tile > 0 && (int)tile >= q.tiles) return;
    set_unit(s, &u, row - (uint32_t)u.b * s.rows, q, tile, kWaves);
    part(u);
  } else {
    Row* rows = reinterpret_cast<Row*>(scratch);
    const uint32_t per = share_of(s, lengths);
    uint32_t at = blockIdx.x * per, before;
    if (!find_sequence(s, lengths, at, &u.b, &before)) return;
    const uint32_t end = at + per;
    Sequence q = sequence_of(s, lengths, u.b);
    uint32_t span = span_of(q.tiles);
    uint32_t r = (at - before) / span, tile = (at - before) % span;
    for (;;) {
      const uint32_t own = (uint32_t)std::max(q.tiles, 1);
      const uint32_t n = std::min(end - at, span - tile);
      set_unit(s, &u, r, q, tile, n);
      if (tile == 0 && threadIdx.x == 0)
        rows[u.b * s.rows + r] = {blockIdx.x, (at + own - 1) / per - blockIdx.x + 1};
      if (tile < own) part(u);
      at += n;
      if (at >= end) return;
      tile = 0;
      if (++r == (uint32_t)s.rows) {
        r = 0;
        if (++u.b >= s.p.B) return;
        q = sequence_of(s, lengths, u.b);
        span = span_of(q.tiles);
      }
      __syncthreads();  // the part before has been read from LDS
    }
  }
}

// The workgroup's waves meet. Wave w holds set w % sets of the heads, for its
// share of the keys: ml[w][c] is the state of its head c, a sum of -1 where it
// attended no key, and o[(w slots + c) D] its outputs. Writes the row's results,
// or the part's, of the unit's heads first .. first + heads - 1.
template <int V, bool kManySets, typename T>
__device__ __forceinline__ void finish_heads(const Shape& s, const Unit& u, int first, int heads, int slots,
                                             const float (*ml)[kHeads][2], const float* o, T* out, float* scratch) {
  constexpr int kMost = kManySets ? kSets * kHeads : kHeads;
  __shared__ float f_s[kWaves][kMost], l_s[kMost];
  const int sets = kManySets ? s.sets : 1;
  const int D = s.p.D, lanes = D / V;
  float* state = u.whole ? nullptr : slot_state(s, scratch, u.slot);
  if ((int)threadIdx.x < heads) {
    // The head's weights of the waves, -1 where a wave's outputs were not
    // written, and its sum, -1 where none were.
    const int h = threadIdx.x, c = kManySets ? h % kHeads : h;
    auto none_of = [&](int w) { return (kManySets && (w & (sets - 1)) != h / kHeads) || ml[w][c][1] < 0.f; };
    float m = -INFINITY, l = 0.f;
    bool any = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const bool none = none_of(w);
      any = any || !none;
      m = none ? m : fmaxf(m, ml[w][c][0]);
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const bool none = none_of(w);
      const float f = none ? -1.f : exp2f(ml[w][c][0] - ref);
      f_s[w][h] = f;
      l += none ? 0.f : ml[w][c][1] * f;
    }
    l_s[h] = any ? l : -1.f;
    if (state) {
      state[2 * (first + h)] = m;
      state[2 * (first + h) + 1] = l_s[h];
    }
  }
  __syncthreads();
  typedef float vec __attribute__((ext_vector_type(V)));
  typedef T tvec __attribute__((ext_vector_type(V)));
  typedef vec vec_at __attribute__((aligned(4)));
  typedef tvec tvec_at __attribute__((aligned(sizeof(T))));
  for (int i = threadIdx.x; i < heads * lanes; i += kWaves * 64) {
    const int h = i / lanes, d = (i - h * lanes) * V;
    vec v = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = f_s[w][h];
      const vec x = *reinterpret_cast<const vec_at*>(o + (w * slots + (kManySets ? h % kHeads : h)) * D + d);
      if (!(f < 0.f)) v += x * f;
    }
    if (state) {
      *reinterpret_cast<vec_at*>(state + 2 * s.heads + (int64_t)(first + h) * D + d) = v;
      continue;
    }
    const float l = l_s[h];
    tvec y;
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = (T)(l < 0.f ? 0.f : v[e] / l);
    *reinterpret_cast<tvec_at*>(out + (u.b * s.p.Hq + u.head0 + first + h) * D + d) = y;
  }
}

// Any head dim up to 512 and any page size: a wave takes a key at a time, its
// lanes across the head dim, one query head after another.
constexpr int kMaxHeadDim = 512;
template <typename T>
__device__ __forceinline__ void any_part(const Shape& s, const Unit& u, const T* __restrict__ q,
                                         const T* __restrict__ k_pages, const T* __restrict__ v_pages,
                                         const int32_t* __restrict__ table, T* __restrict__ out, float* scratch,
                                         float (*ml)[kHeads][2], float* ow) {
  constexpr int J = kMaxHeadDim / 64;
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
      const uint32_t first = std::max(u.lo, (uint32_t)t * kTileKeys);
      const uint32_t last = std::min(u.hi, ((uint32_t)t + 1) * kTileKeys);
      for (uint32_t key = first; key < last; ++key) {
        const int row = row_of(s, table, u.b, u.kv_head, key);
        if (row < 0) continue;
        const T *kr = k_pages + (int64_t)row * D, *vr = v_pages + (int64_t)row * D;
        float dot = 0.f, vv[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int d = lane + 64 * j;
          if (d < D) dot = fmaf(qv[j], (float)kr[d], dot);
          vv[j] = d < D ? (float)vr[d] : 0.f;
        }
        float x = wave_sum(dot) * s.p.scale * kLog2e;
        // Rounded here, not in a fma below: the largest is 0 off itself,
        // however large.
        asm("" : "+v"(x));
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
      ml[wave][0][0] = m;
      ml[wave][0][1] = l;
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (lane + 64 * j < D) ow[wave * D + lane + 64 * j] = o[j];
    __syncthreads();
    finish_heads<1, false>(s, u, h, 1, 1, ml, ow, out, scratch);
    __syncthreads();
  }
}

template <typename T, bool kAligned>
__global__ void __launch_bounds__(kWaves * 64)
    paged_any(Shape s, const T* __restrict__ q, const T* __restrict__ k_pages, const T* __restrict__ v_pages,
              const int32_t* __restrict__ table, const int32_t* __restrict__ lengths, T* __restrict__ out,
              float* __restrict__ scratch) {
  __shared__ float ml[kWaves][kHeads][2];
  __shared__ float ow[kWaves * kMaxHeadDim];  // [waves][D]
  for_parts<kAligned>(s, lengths, scratch,
            [&](const Unit& u) { any_part<T>(s, u, q, k_pages, v_pages, table, out, scratch, ml, ow); });
}

// ------------------------------------------------------------------- tiles
// Head dims that are whole matrix steps. A wave takes 32 keys at a time (16 in
// f32) for its heads: S^T = K.Q^T with the keys as the matrix rows
// and the heads as its 16 columns, so a lane holds scores of one head (its
// column, lane & 15) for keys 4g + r of each 16 (g = lane / 16), and these are,
// as they lie, the right operand of O^T += V^T.P^T. K goes from memory to the
// registers of the left operand (16 bytes a lane of a key's row). V^T's
// operand needs 8 keys of one column a lane: a lane loads its 8 keys' pieces
// of neighbouring columns and v_perm pairs them up, column after column; the
// columns then lie in the order lane, element, which the output undoes. No
// LDS and no barrier until the waves' states meet.
//
// Bound by HBM: the matrix steps are 8% of a tile's time at 5 TB/s, whether a
// row has 1 head or 16. The next tile's rows are loaded before this one's are
// used; head dims above 128 have no registers for that.

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (std::is_same_v<T, f16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}
// Two weights in two pieces of the type, a first one below the weight and the rest
// of it: 2^-16 of a weight is lost in bf16, 2^-21 in f16. No rest of a weight is
// 0, so that an infinite value's product with it is no NaN: bf16 has room for a
// least one, f16 leaves a part in 2^11 to it (a weight below 2^-28 of the largest
// may have a rest of 0 all the same).
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& first, uint32_t& rest) {
  if constexpr (std::is_same_v<T, f16_t>) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a * (1.f - 0x1p-11f), b * (1.f - 0x1p-11f));
    first = __builtin_bit_cast(uint32_t, h);
    rest = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a - (float)h[0], b - (float)h[1]}, f16x2));
  } else {
    const uint32_t u = __builtin_bit_cast(uint32_t, a), v = __builtin_bit_cast(uint32_t, b);
    first = __builtin_amdgcn_perm(v, u, 0x07060302u);
    const f32x2 r = {__builtin_amdgcn_fmed3f(a - __builtin_bit_cast(float, u & 0xffff0000u), 0x1p-126f, a),
                     __builtin_amdgcn_fmed3f(b - __builtin_bit_cast(float, v & 0xffff0000u), 0x1p-126f, b)};
    rest = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
  }
}

// The larger of the four 16-lane groups' values, on every lane: swapped halves
// and rows instead of LDS shuffles.
__device__ __forceinline__ float groups_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const float y = fmaxf(__builtin_bit_cast(float, (uint32_t)h[0]), __builtin_bit_cast(float, (uint32_t)h[1]));
  const uint32_t v = __builtin_bit_cast(uint32_t, y);
  const auto w = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)w[0]), __builtin_bit_cast(float, (uint32_t)w[1]));
}

// What a weight of 1 goes to the matrix steps as, and counts as in its sum. f16
// holds 2^-24 at least and 65504 at most: as 2^14 a small weight loses at most
// 2^-39 there, and 2^20 of them 2^-19; as 1 they would lose 2^-5.
template <typename T>
constexpr float kLift = std::is_same_v<T, f16_t> ? 16384.f : 1.f;

template <typename T, int D>
struct TileShape {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kHalves = kHalf ? 2 : 1;             // 16-key halves of a step
  static constexpr int kKeys = 16 * kHalves;
  static constexpr int kKWords = D * (int)sizeof(T) / 16;   // dwords of a key's row a lane holds (a quarter)
  static constexpr int kRows = 4 * kHalves;                 // value rows of a lane
  static constexpr int kVWords = D * (int)sizeof(T) / 64;   // dwords of a value row a lane holds (a sixteenth)
  static constexpr int kPieces = kVWords / 4;               // of 4 dwords, then one of the rest
  static constexpr int kRest = kVWords % 4;
  static constexpr int kAcc = D / 16;                       // output columns a lane's row of the accumulators holds
  static constexpr bool kAhead = kHalves * kKWords + kRows * kVWords <= 64;
};

// One step's keys and values, and which of the lane's keys 16 t + 4g + r are
// attended (bit 4t + r).
template <typename T, int D>
struct Tile {
  using Sh = TileShape<T, D>;
  uint32_t k[Sh::kHalves][Sh::kKWords];
  uint32_t v[Sh::kRows][Sh::kVWords];
  uint32_t mask;
};

template <typename T, int D, bool kPage16>
__device__ __forceinline__ void load_tile(const Shape& s, const Unit& u, const T* __restrict__ k_pages,
                                          const T* __restrict__ v_pages, const int32_t* __restrict__ table,
                                          uint32_t key0, Tile<T, D>& t) {
  using Sh = TileShape<T, D>;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  t.mask = 0;
#pragma unroll
  for (int h = 0; h < Sh::kHalves; ++h) {
    const uint32_t key = key0 + 16 * h;
    int krow, vrow[4];
    bool ok[4];
    if constexpr (kPage16) {
      // 16 keys from a multiple of 16 lie in one page: the same for every lane.
      const int row = row_of(s, table, u.b, u.kv_head, key);
      krow = row < 0 ? c : row + c;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        vrow[r] = (row < 0 ? 0 : row) + 4 * g + r;
        ok[r] = row >= 0;
      }
    } else {
      const int row = row_of(s, table, u.b, u.kv_head, key + c);
      krow = std::max(row, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int x = __shfl(row, 4 * g + r);
        vrow[r] = std::max(x, 0);
        ok[r] = x >= 0;
      }
    }
    const T* kr = k_pages + (int64_t)krow * D;
#pragma unroll
    for (int i = 0; i < Sh::kKWords / 4; ++i) load_words<4>(kr + (4 * i + g) * (16 / (int)sizeof(T)), t.k[h] + 4 * i);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t j = key + 4 * g + r;
      if (ok[r] && j >= u.lo && j < u.hi) t.mask |= 1u << (4 * h + r);
      const T* vr = v_pages + (int64_t)vrow[r] * D;
      constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < Sh::kPieces; ++i) load_words<4>(vr + (16 * i + c) * E, t.v[4 * h + r] + 4 * i);
      if constexpr (Sh::kRest > 0)
        load_words<Sh::kRest>(vr + 16 * E * Sh::kPieces + c * (Sh::kRest * 4 / (int)sizeof(T)),
                              t.v[4 * h + r] + 4 * Sh::kPieces);
    }
  }
}

// Output column of accumulator a, matrix row i.
template <typename T, int D>
__device__ __forceinline__ int column_of(int a, int i) {
  using Sh = TileShape<T, D>;
  constexpr int E = 16 / (int)sizeof(T), R = Sh::kRest * 4 / (int)sizeof(T);
  return a < Sh::kPieces * E ? (a / E * 16 + i) * E + a % E : Sh::kPieces * 16 * E + i * R + (a - Sh::kPieces * E);
}

template <typename T, int D>
struct Heads {
  uint32_t q[TileShape<T, D>::kKWords];
  f32x4 o[TileShape<T, D>::kAcc];
  f32x4 l4;   // 16-bit: the weights' sum, from a matrix step with rows of ones
  float l;    // f32: this lane's keys' share of it
  float m;
  uint32_t seen;
};

template <typename T, int D>
__device__ __forceinline__ void use_tile(float scale2, Tile<T, D>& t, Heads<T, D>& st) {
  using Sh = TileShape<T, D>;
  f32x4 x[Sh::kHalves];
#pragma unroll
  for (int h = 0; h < Sh::kHalves; ++h) {
    x[h] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (Sh::kHalf) {
#pragma unroll
      for (int i = 0; i < Sh::kKWords; i += 4)
        x[h] = mfma16<T>(u32x4{t.k[h][i], t.k[h][i + 1], t.k[h][i + 2], t.k[h][i + 3]},
                         u32x4{st.q[i], st.q[i + 1], st.q[i + 2], st.q[i + 3]}, x[h]);
    } else {
#pragma unroll
      for (int i = 0; i < Sh::kKWords; ++i)
        x[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, t.k[h][i]),
                                                    __builtin_bit_cast(float, st.q[i]), x[h], 0, 0, 0);
    }
  }
  constexpr uint32_t kAll = (1u << Sh::kRows) - 1;
  if (__any(t.mask != kAll)) {
    // What is not attended weighs nothing whatever its rows hold.
#pragma unroll
    for (int r = 0; r < Sh::kRows; ++r)
      if (!(t.mask >> r & 1)) {
#pragma unroll
        for (int i = 0; i < Sh::kVWords; ++i) t.v[r][i] = 0;
      }
  }
  st.seen |= t.mask;
  float mx = -INFINITY;
#pragma unroll
  for (int h = 0; h < Sh::kHalves; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[h][r] = t.mask >> (4 * h + r) & 1 ? x[h][r] * scale2 : -INFINITY;
      mx = fmaxf(mx, x[h][r]);
    }
  mx = groups_max(mx);
  if (__any(mx > st.m)) {
    const float mn = fmaxf(st.m, mx);
    const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m - mn);
    st.m = mn;
    st.l *= alpha;
    st.l4 *= alpha;
#pragma unroll
    for (int a = 0; a < Sh::kAcc; ++a) st.o[a] *= alpha;
  }
  const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
  for (int h = 0; h < Sh::kHalves; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r) x[h][r] = __builtin_amdgcn_exp2f(x[h][r] - ref) * kLift<T>;
  if constexpr (Sh::kHalf) {
    // A weight goes to the matrix steps in two pieces. They are summed as they
    // are, so that a key of all the weight answers its value. (64 sequences of 32
    // to 4064 keys, bf16: 107.3 us, a relative error of 1.7e-3 that is the result's
    // rounding; in one piece 107.4 us and 2.1e-3.)
    u32x4 p, rest;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t first, second;
      split2<T>(x[i / 2][2 * (i % 2)], x[i / 2][2 * (i % 2) + 1], first, second);
      p[i] = first;
      rest[i] = second;
    }
    constexpr uint32_t one = std::is_same_v<T, f16_t> ? 0x3c003c00u : 0x3f803f80u;
    st.l4 = mfma16<T>(u32x4{one, one, one, one}, p, st.l4);
    st.l4 = mfma16<T>(u32x4{one, one, one, one}, rest, st.l4);
#pragma unroll
    for (int w = 0; w < Sh::kVWords; ++w)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t sel = e ? 0x07060302u : 0x05040100u;
        const u32x4 a = {__builtin_amdgcn_perm(t.v[1][w], t.v[0][w], sel), __builtin_amdgcn_perm(t.v[3][w], t.v[2][w], sel),
                         __builtin_amdgcn_perm(t.v[5][w], t.v[4][w], sel), __builtin_amdgcn_perm(t.v[7][w], t.v[6][w], sel)};
        st.o[2 * w + e] = mfma16<T>(a, p, st.o[2 * w + e]);
        st.o[2 * w + e] = mfma16<T>(a, rest, st.o[2 * w + e]);
      }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      st.l += x[0][r];
#pragma unroll
      for (int w = 0; w < Sh::kVWords; ++w)
        st.o[w] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, t.v[r][w]), x[0][r], st.o[w], 0, 0, 0);
    }
  }
}

template <typename T, int D, bool kPage16, bool kManySets>
__device__ __forceinline__ void tiles_part(const Shape& s, const Unit& u, const T* __restrict__ q,
                                           const T* __restrict__ k_pages, const T* __restrict__ v_pages,
                                           const int32_t* __restrict__ table, T* __restrict__ out, float* scratch,
                                           float (*ml)[kHeads][2], float* ow) {
  using Sh = TileShape<T, D>;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The wave's heads, and its share of the keys beside the other waves of the
  // set. (The sets' waves read a tile about at once: it comes from HBM once.)
  const int log = kManySets ? s.sets_log : 0, key_waves = kWaves >> log, key_wave = wave >> log;
  const int head0 = kManySets ? (wave & (s.sets - 1)) * kHeads : 0;
  const int heads = std::min(kHeads, u.heads - head0), slots = std::min(kHeads, u.heads);
  Heads<T, D> st;
  st.m = -INFINITY;
  st.l = 0.f;
  st.l4 = f32x4{0.f, 0.f, 0.f, 0.f};
  st.seen = 0;
#pragma unroll
  for (int a = 0; a < Sh::kAcc; ++a) st.o[a] = f32x4{0.f, 0.f, 0.f, 0.f};
  const T* qr = q + (u.b * s.p.Hq + u.head0 + std::min(head0 + c, u.heads - 1)) * D;
#pragma unroll
  for (int i = 0; i < Sh::kKWords / 4; ++i) {
    load_words<4>(qr + (4 * i + g) * (16 / (int)sizeof(T)), st.q + 4 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) st.q[4 * i + e] = c < heads ? st.q[4 * i + e] : 0u;
  }
  const float scale2 = s.p.scale * kLog2e;
  // Step i of the wave: its tiles are every key_waves-th from tile0 + key_wave.
  constexpr int kSteps = kTileKeys / Sh::kKeys;
  const int tiles = u.tile1 - u.tile0 - key_wave;
  const int steps = heads > 0 && tiles > 0 ? ((tiles + key_waves - 1) >> (kWavesLog - log)) * kSteps : 0;
  auto key_of = [&](int i) {
    return (uint32_t)(u.tile0 + key_wave + i / kSteps * key_waves) * kTileKeys + i % kSteps * Sh::kKeys;
  };
  if (steps > 0) {
    Tile<T, D> t;
    if constexpr (Sh::kAhead) {
      load_tile<T, D, kPage16>(s, u, k_pages, v_pages, table, key_of(0), t);
      for (int i = 1; i < steps; ++i) {
        Tile<T, D> next;
        load_tile<T, D, kPage16>(s, u, k_pages, v_pages, table, key_of(i), next);
        use_tile<T, D>(scale2, t, st);
        t = next;
      }
      use_tile<T, D>(scale2, t, st);
    } else {
      for (int i = 0; i < steps; ++i) {
        load_tile<T, D, kPage16>(s, u, k_pages, v_pages, table, key_of(i), t);
        use_tile<T, D>(scale2, t, st);
      }
    }
  }
  float l = st.l4[0];
  if constexpr (!Sh::kHalf) l = st.l + __shfl_xor(st.l, 16), l += __shfl_xor(l, 32);
  const bool any = __any(st.seen != 0);
  if (lane < heads) {
    ml[wave][lane][0] = st.m;
    ml[wave][lane][1] = any ? l : -1.f;
  }
  if (any && c < heads) {
#pragma unroll
    for (int a = 0; a < Sh::kAcc; ++a)
#pragma unroll
      for (int r = 0; r < 4; ++r) ow[(wave * slots + c) * D + column_of<T, D>(a, 4 * g + r)] = st.o[a][r];
  }
  __syncthreads();
  finish_heads<4, kManySets>(s, u, 0, u.heads, slots, ml, ow, out, scratch);
}

template <typename T, int D, bool kPage16, bool kAligned, bool kManySets>
__global__ void __launch_bounds__(kWaves * 64, D > 192 ? 1 : 2)
    paged_tiles(Shape s, const T* __restrict__ q, const T* __restrict__ k_pages, const T* __restrict__ v_pages,
                const int32_t* __restrict__ table, const int32_t* __restrict__ lengths, T* __restrict__ out,
                float* __restrict__ scratch) {
  __shared__ float ml[kWaves][kHeads][2];
  extern __shared__ float ow[];  // [waves][heads of a wave][D]
  for_parts<kAligned>(s, lengths, scratch, [&](const Unit& u) {
    tiles_part<T, D, kPage16, kManySets>(s, u, q, k_pages, v_pages, table, out, scratch, ml, ow);
  });
}

// One workgroup a query head: folds the parts of its row. Lanes take V outputs
// each, groups of them every G-th part, and the groups are added in order.
template <typename T, int V, bool kAligned>
__global__ void __launch_bounds__(256)
    paged_combine(Shape s, const int32_t* __restrict__ lengths, const float* __restrict__ scratch,
                  T* __restrict__ out) {
  __shared__ float f_s[kMaxParts], l_s[kMaxParts];
  __shared__ float red[2][4];
  __shared__ float sums[256 * V];
  const int64_t b = blockIdx.x / (uint32_t)s.p.Hq;
  const int hq = (int)(blockIdx.x - (uint32_t)b * (uint32_t)s.p.Hq);
  const int kv_head = hq / s.group, of_head = hq - kv_head * s.group, head = of_head % (kHeads * s.sets);
  const int64_t at = b * s.rows + kv_head * s.head_rows + of_head / (kHeads * s.sets);
  // The row's first workgroup, and its parts: as many as its keys take, or as
  // many as there may be, whose states and outputs are requested with the
  // length that tells.
  const Row row = kAligned ? Row{(uint32_t)at * (uint32_t)s.each, (uint32_t)s.each}
                           : reinterpret_cast<const Row*>(scratch)[at];
  const int D = s.p.D, most = (int)row.n;
  if (!kAligned && most <= 1) return;
  // Part i's slot: the first starts the row, the others continue it.
  auto part = [&](int i) {
    return slot_state(s, const_cast<float*>(scratch), slot_of((int64_t)row.group + i, i == 0));
  };
  const int lanes = std::min(256, (D + V - 1) / V), groups = 256 / lanes;
  const int g = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  float first[V];
  if (g < std::min(groups, most) && lane * V < D)
    __builtin_memcpy(first, part(g) + 2 * s.heads + (int64_t)head * D + lane * V, sizeof(first));
  float m0 = -INFINITY, l0 = -1.f;
  if ((int)threadIdx.x < most) {
    m0 = part(threadIdx.x)[2 * head];
    l0 = part(threadIdx.x)[2 * head + 1];
  }
  int n = most;
  if constexpr (kAligned) {
    n = (sequence_of(s, lengths, b).tiles + kWaves - 1) / kWaves;
    if (n <= 1) return;
  }
  float m = -INFINITY;
  for (int i = threadIdx.x; i < n; i += 256) {
    const bool here = i == (int)threadIdx.x;
    f_s[i] = here ? m0 : part(i)[2 * head];
    l_s[i] = here ? l0 : part(i)[2 * head + 1];
    if (!(l_s[i] < 0.f)) m = fmaxf(m, f_s[i]);
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float ref = m == -INFINITY ? 0.f : m;
  // Each part's weight, once; a part without any attended key (a sum of -1)
  // has no outputs, and weighs -1.
  float l = 0.f;
  bool any = false;
  for (int i = threadIdx.x; i < n; i += 256) {
    const bool none = l_s[i] < 0.f;
    f_s[i] = none ? -1.f : exp2f(f_s[i] - ref);
    l += none ? 0.f : l_s[i] * f_s[i];
    any = any || !none;
  }
  l = wave_sum(l);
  if ((threadIdx.x & 63) == 0) red[1][threadIdx.x >> 6] = l;
  any = __syncthreads_or(any);
  l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  for (int d0 = 0; d0 < D; d0 += lanes * V) {
    const int d = d0 + lane * V;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
    if (g < groups && d < D) {
#pragma unroll 4
      for (int i = g; i < n; i += groups) {
        float x[V];
        if (i == g && d0 == 0) __builtin_memcpy(x, first, sizeof(x));
        else __builtin_memcpy(x, part(i) + 2 * s.heads + (int64_t)head * D + d, sizeof(x));
        const float f = f_s[i];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += f < 0.f ? 0.f : x[e] * f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) sums[threadIdx.x * V + e] = acc[e];
    __syncthreads();
    for (int i = threadIdx.x; i < lanes * V && d0 + i < D; i += 256) {
      float v = 0.f;
      for (int k = 0; k < groups; ++k) v += sums[k * lanes * V + i];
      out[(b * s.p.Hq + hq) * D + d0 + i] = (T)(any ? v / l : 0.f);
    }
  }
}

// Workgroups a CU holds of the kernel that takes the shape: what its registers
// leave, so that a launch's workgroups run at once.
int groups_per_cu(const PagedParams& p) { return p.D > 192 ? 1 : 2; }

// Head dims that paged_tiles takes.
bool takes_tiles(int D) { return D == 32 || D == 64 || D == 96 || D == 128 || D == 192 || D == 256; }

Shape shape_of(const PagedParams& p) {
  Shape s;
  s.p = p;
  s.group = p.Hq / p.Hkv;
  // 8 sequences of 8192 keys, 8 heads of 128 with 32 query heads each, bf16:
  // 90 us in rows of 16, 73 in rows of 32, whose two sets load a tile each.
  s.sets = s.group <= kHeads || !takes_tiles(p.D) ? 1 : s.group <= 2 * kHeads ? 2 : kSets;
  s.sets_log = s.sets / 2;
  s.heads = std::min(s.group, kHeads * s.sets);
  s.head_rows = (s.group + kHeads * s.sets - 1) / (kHeads * s.sets);
  s.rows = p.Hkv * s.head_rows;
  s.cap = static_cast<uint32_t>(p.M * p.S);
  s.page = divisor_of(static_cast<uint32_t>(p.S));
  // The table's tiles as workgroups of one tile a wave, row by row: where they
  // are no more than run at once, that is the launch.
  const int64_t tiles = (static_cast<int64_t>(s.cap) + kTileKeys - 1) / kTileKeys;
  const int64_t each = (tiles + kWaves - 1) / kWaves, most = kCus * groups_per_cu(p);
  s.aligned = s.sets == 1 && p.B * s.rows * each <= most;
  s.each = static_cast<int>(each);
  s.groups = static_cast<int>(s.aligned ? p.B * s.rows * each : most);
  return s;
}
// Whether a row may be cut.
bool may_cut(const Shape& s) { return !s.aligned || s.cap > kWaves * kTileKeys; }

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(Code::kInternal, strformat("%s launch failed: %s", what, hipGetErrorString(e)));
}

}  // namespace

size_t paged_attention_scratch_bytes(const PagedParams& p, DType t) {
  const Shape s = shape_of(p);
  if (p.B == 0 || !may_cut(s)) return 0;
  return static_cast<size_t>(p.B) * s.rows * sizeof(Row) +
         static_cast<size_t>(slot_of(s.groups, false)) * s.heads * (p.D + 2) * sizeof(float);
}

void launch_paged_attention(hipStream_t stream, const PagedParams& p, DType t, const void* q, const void* k_pages,
                            const void* v_pages, const int32_t* page_table, const int32_t* lengths, void* out,
                            void* scratch) {
  if (p.B == 0) return;
  const Shape s = shape_of(p);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    const T *qp = static_cast<const T*>(q), *kp = static_cast<const T*>(k_pages), *vp = static_cast<const T*>(v_pages);
    const dim3 grid(static_cast<uint32_t>(s.groups)), block(kWaves * 64);
    T* op = static_cast<T*>(out);
    float* sp = static_cast<float*>(scratch);
#define PJRTX_PAGED_AS(...) \
  hipLaunchKernelGGL((__VA_ARGS__), grid, block, lds, stream, s, qp, kp, vp, page_table, lengths, op, sp)
#define PJRTX_PAGED_PAGES(DIM, ALIGNED, SETS)                                       \
  do {                                                                              \
    if (p.S % 16 == 0) PJRTX_PAGED_AS(paged_tiles<T, DIM, true, ALIGNED, SETS>);    \
    else PJRTX_PAGED_AS(paged_tiles<T, DIM, false, ALIGNED, SETS>);                 \
  } while (0)
#define PJRTX_PAGED(DIM)                                         \
  case DIM:                                                      \
    if (s.sets > 1) PJRTX_PAGED_PAGES(DIM, false, true);         \
    else if (s.aligned) PJRTX_PAGED_PAGES(DIM, true, false);     \
    else PJRTX_PAGED_PAGES(DIM, false, false);                   \
    break
    size_t lds = static_cast<size_t>(kWaves) * std::min(s.heads, kHeads) * p.D * sizeof(float);  // the waves' outputs
    switch (p.D) {
      PJRTX_PAGED(32);
      PJRTX_PAGED(64);
      PJRTX_PAGED(96);
      PJRTX_PAGED(128);
      PJRTX_PAGED(192);
      PJRTX_PAGED(256);
      default:
        lds = 0;
        if (s.aligned) PJRTX_PAGED_AS(paged_any<T, true>);
        else PJRTX_PAGED_AS(paged_any<T, false>);
    }
#undef PJRTX_PAGED_AS
#undef PJRTX_PAGED_PAGES
#undef PJRTX_PAGED
    if (!sp) return;
    const dim3 heads(static_cast<uint32_t>(p.B * p.Hq));
#define PJRTX_COMBINE(V, ALIGNED) \
  hipLaunchKernelGGL((paged_combine<T, V, ALIGNED>), heads, block, 0, stream, s, lengths, sp, op)
    if (p.D % 4 == 0 && s.aligned) PJRTX_COMBINE(4, true);
    else if (p.D % 4 == 0) PJRTX_COMBINE(4, false);
    else if (s.aligned) PJRTX_COMBINE(1, true);
    else PJRTX_COMBINE(1, false);
#undef PJRTX_COMBINE
  };
  if (t == DType::kF32) go(float());
  else if (t == DType::kBF16) go(bf16_t());
  else go(f16_t());
  check_launch("paged_attention");
}

// ------------------------------------------------------------------ append
// A workgroup copies the keys and values of kRows new rows, a thread the same
// unit of each, all in flight at once. Of rows that name one slot the last
// stays whatever order the workgroups run in: each reads the slots after its
// rows and leaves a row out whose slot comes again, while its first units are
// on their way. The scan is 4 bytes a later row and workgroup: at 8192 rows 16
// MB of L2 reads beside the 64 MB and more of the copy. It grows as the square of
// the rows, so a launch takes kAppendRows at most, and the next launch's rows
// come later by the stream's order. 131072 rows of 8 heads of 128, bf16, in one
// launch 866 us, in launches of 32768 / 16384 / 8192 378 / 316 / 260; of one head
// of 128 742, and 245 / 182 / 196.
namespace {

constexpr int64_t kAppendRows = 8192;

// Past the L2, which the scattered rows would fill line by line: 8000 rows of 8
// heads of 128, f16, 25.4 us without and 15.2 us with.
template <typename U>
__device__ __forceinline__ void store_streaming(U* p, const U& x) {
  if constexpr (sizeof(U) == 16)
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, x), reinterpret_cast<u32x4*>(p));
  else
    __builtin_nontemporal_store(x, p);
}

template <typename U, int kRows>
__global__ void __launch_bounds__(256)
    append_rows(AppendParams p, Divisor page, Divisor units, U* __restrict__ k_pages, U* __restrict__ v_pages,
                const U* __restrict__ k_new, const U* __restrict__ v_new, const void* __restrict__ slots) {
  static_assert(kRows <= 32, "a bit a row");
  __shared__ uint32_t again_s;
  const int64_t n0 = (int64_t)blockIdx.x * kRows;
  // A row's slot, or -1 where it names none.
  auto slot_at = [&](int64_t i) {
    const int64_t x = p.slot_bytes == 8 ? static_cast<const int64_t*>(slots)[i]
                                        : (int64_t)static_cast<const int32_t*>(slots)[i];
    return x >= 0 && x < p.P * p.S ? (int)x : -1;
  };
  // `units` of U make a head's D elements; a row's keys, then its values.
  const uint32_t half = (uint32_t)p.Hkv * units.d, total = 2 * half;
  U x[kRows];
  auto request = [&](uint32_t i) {
    const U* from = (i < half ? k_new + i : v_new + (i - half)) + n0 * half;
#pragma unroll
    for (int r = 0; r < kRows; ++r) x[r] = from[std::min<int64_t>(r, p.N - 1 - n0) * half];
  };
  uint32_t i = threadIdx.x;
  if (i < total) request(i);
  int slot[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) slot[r] = n0 + r < p.N ? slot_at(n0 + r) : -1;
  if (threadIdx.x == 0) {
    uint32_t again = 0;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int o = r + 1; o < kRows; ++o) again |= slot[r] == slot[o] ? 1u << r : 0u;
    again_s = again;
  }
  __syncthreads();
  uint32_t again = 0;
#pragma unroll 8
  for (int64_t j = n0 + kRows + threadIdx.x; j < p.N; j += 256) {
    const int other = slot_at(j);
#pragma unroll
    for (int r = 0; r < kRows; ++r) again |= other == slot[r] ? 1u << r : 0u;
  }
  if (again) atomicOr(&again_s, again);
  __syncthreads();
  again = again_s;
  for (; i < total; i += 256) {
    if (i >= 256) request(i);
    const uint32_t at = i < half ? i : i - half, h = quotient(at, units), c = at - h * units.d;
    U* to = (i < half ? k_pages : v_pages) + c;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (slot[r] < 0 || (again >> r & 1)) continue;
      const uint32_t pg = quotient((uint32_t)slot[r], page), pos = (uint32_t)slot[r] - pg * page.d;
      store_streaming(to + (((int64_t)pg * p.Hkv + h) * p.S + pos) * units.d, x[r]);
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
    const Divisor units = divisor_of(static_cast<uint32_t>(row_bytes / sizeof(U)));
    const Divisor page = divisor_of(static_cast<uint32_t>(p.S));
    U *kp = static_cast<U*>(k_pages), *vp = static_cast<U*>(v_pages);
    for (int64_t n0 = 0; n0 < p.N; n0 += kAppendRows) {
      AppendParams part = p;
      part.N = std::min(kAppendRows, p.N - n0);
      const int64_t at = n0 * p.Hkv * units.d;
      const U *kn = static_cast<const U*>(k_new) + at, *vn = static_cast<const U*>(v_new) + at;
      const void* sl = static_cast<const char*>(slots) + n0 * p.slot_bytes;
      if (part.N <= 1024)
        hipLaunchKernelGGL((append_rows<U, 1>), dim3(static_cast<uint32_t>(part.N)), dim3(256), 0, s, part, page, units,
                           kp, vp, kn, vn, sl);
      else
        hipLaunchKernelGGL((append_rows<U, 8>), dim3(static_cast<uint32_t>((part.N + 7) / 8)), dim3(256), 0, s, part,
                           page, units, kp, vp, kn, vn, sl);
    }
  };
  // The widest unit that every row starts on.
  if (addresses % 16 == 0) go(uint4());
  else if (addresses % 4 == 0) go(uint32_t());
  else go(uint16_t());
  check_launch("paged_append");
}

}  // namespace pjrtx
