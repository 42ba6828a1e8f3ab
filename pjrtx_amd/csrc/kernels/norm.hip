// Residual addition with the root-mean-square norm, and its gradient.
//
// Forward: t = x + residual, y = t * r * gain with r = 1 / sqrt(mean(t^2) +
// eps). A row is read once: its floats stay in registers between the sum of
// squares and the results (and, for 8 bits, between the row's largest |y| and
// the rounding). The sum is held unrounded for the norm; what is written as
// the sum is rounded once to the type. Bound by HBM: x and the residual in,
// the sum and y out (8192 x 4096 bf16 to 8 bits 235 MB in 41 us, 5.7 TB/s).
// One row of 2048 takes 2.7 us, which is a launch's.
#include <algorithm>
#include <cmath>

#include "kernels/operators.h"
#include "kernels/vec.h"

namespace pjrtx {
namespace {

// Sum and max over the TPR threads of a row: one wave, or every wave of the
// workgroup through `red` (one float a wave, its own words each call).
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
  x = wave_sum(x);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) x += red[w];
  }
  return x;
}
template <int TPR>
__device__ __forceinline__ float row_max_nan(float x, float* red) {
  x = wave_max_nan(x);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) x = __builtin_elementwise_maximum(x, red[w]);
  }
  return x;
}

// y over the row's scale, rounded to the nearest even; NaN counts as 0 (its
// scale is NaN, so what it stands for stays NaN). Under an infinite scale an
// infinite y is +-127, which stands for itself.
struct Quant {
  float scale, inv;
  bool divide;
};
__device__ __forceinline__ Quant quant_of(float amax) {
  Quant q;
  q.scale = amax / 127.f;
  // The reciprocal of a scale below 2^-120 could overflow: those rows divide.
  q.divide = !(q.scale >= 0x1p-120f && q.scale < HUGE_VALF);
  q.inv = q.divide ? 0.f : 1.f / q.scale;
  return q;
}
__device__ __forceinline__ int8_t quantize(float y, const Quant& q) {
  float v = q.divide ? (fabsf(y) == HUGE_VALF ? y : q.scale > 0.f ? y / q.scale : 0.f) : y * q.inv;
  v = fminf(fmaxf(rintf(v), -127.f), 127.f);  // fmaxf(NaN, -127) is -127
  return y == y ? (int8_t)v : (int8_t)0;
}

// TPR threads a row, NV vectors a thread: NV * TPR vectors cover the row.
// kStream: 8192 x 4096 bf16 to 8 bits 46.0 us without, 41.9 with.
template <typename T, int TPR, int NV, bool kQuant, bool kStream>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
    norm_rows(NormParams p, const T* __restrict__ x, const T* __restrict__ residual, const T* __restrict__ gain,
              T* __restrict__ y, int8_t* __restrict__ y8, float* __restrict__ scales, T* __restrict__ sum) {
  constexpr int E = kVecElems<T>;
  constexpr int RPW = TPR < 256 ? 256 / TPR : 1;  // rows a workgroup
  __shared__ float red[2][TPR / 64];
  const int64_t row = (int64_t)blockIdx.x * RPW + (TPR < 256 ? threadIdx.x / TPR : 0);
  if (row >= p.rows) return;  // whole waves, and no barrier when rows share a workgroup
  const int lane = threadIdx.x % TPR;
  const T* xr = x + row * p.D;
  const T* rr = residual ? residual + row * p.D : nullptr;
  typedef typename Vec<T>::type V;
  V a[NV], b[NV], g[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t at = (int64_t)(v * TPR + lane) * E, n = p.D - at, to = std::min(at, p.D - 1);
    a[v] = load_vec<T, kStream>(xr + to, n, (T)0.f);
    if (rr) b[v] = load_vec<T, kStream>(rr + to, n, (T)0.f);
    g[v] = load_vec<T>(gain + to, n, (T)0.f);
  }
  float t[NV][E];
  float ss = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      t[v][e] = rr ? (float)a[v][e] + (float)b[v][e] : (float)a[v][e];
      ss = fmaf(t[v][e], t[v][e], ss);
    }
  const float r = 1.f / sqrtf(row_sum<TPR>(ss, red[0]) / (float)p.D + p.eps);
  float amax = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t at = (int64_t)(v * TPR + lane) * E;
    const int64_t n = p.D - at;
    if (n <= 0) continue;
    if (sum) {
      typename Vec<T>::type o;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = (T)t[v][e];
      store_vec<T, kStream>(sum + row * p.D + at, n, o);
    }
    V o;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      t[v][e] = t[v][e] * r * (float)g[v][e];
      if constexpr (kQuant) amax = __builtin_elementwise_maximum(amax, fabsf(t[v][e]));
      else o[e] = (T)t[v][e];
    }
    if constexpr (!kQuant) store_vec<T, kStream>(y + row * p.D + at, n, o);
  }
  if constexpr (kQuant) {
    const Quant q = quant_of(row_max_nan<TPR>(amax, red[1]));
    if (lane == 0) scales[row] = q.scale;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int64_t at = (int64_t)(v * TPR + lane) * E;
      const int64_t n = p.D - at;
      if (n <= 0) continue;
      int8_t* o = y8 + row * p.D + at;
      if (n >= E) {
        uint32_t w[E / 4];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t b = (uint32_t)(uint8_t)quantize(t[v][e], q) << (8 * (e & 3));
          w[e / 4] = e & 3 ? w[e / 4] | b : b;
        }
        __builtin_memcpy(o, w, E);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e < n) o[e] = quantize(t[v][e], q);
      }
    }
  }
}

// Rows that no launch above holds in registers: read again for each pass.
template <typename T, bool kQuant>
__global__ void __launch_bounds__(1024)
    norm_long_rows(NormParams p, const T* __restrict__ x, const T* __restrict__ residual, const T* __restrict__ gain,
                   T* __restrict__ y, int8_t* __restrict__ y8, float* __restrict__ scales, T* __restrict__ sum) {
  __shared__ float red[2][16];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * p.D;
  const T* rr = residual ? residual + row * p.D : nullptr;
  auto total = [&](int64_t i) { return rr ? (float)xr[i] + (float)rr[i] : (float)xr[i]; };
  float ss = 0.f;
  for (int64_t i = threadIdx.x; i < p.D; i += 1024) {
    const float t = total(i);
    ss = fmaf(t, t, ss);
  }
  const float r = 1.f / sqrtf(row_sum<1024>(ss, red[0]) / (float)p.D + p.eps);
  float amax = 0.f;
  for (int64_t i = threadIdx.x; i < p.D; i += 1024) {
    const float t = total(i), v = t * r * (float)gain[i];
    if (sum) sum[row * p.D + i] = (T)t;
    if constexpr (kQuant) amax = __builtin_elementwise_maximum(amax, fabsf(v));
    else y[row * p.D + i] = (T)v;
  }
  if constexpr (kQuant) {
    const Quant q = quant_of(row_max_nan<1024>(amax, red[1]));
    if (threadIdx.x == 0) scales[row] = q.scale;
    for (int64_t i = threadIdx.x; i < p.D; i += 1024)
      y8[row * p.D + i] = quantize(total(i) * r * (float)gain[i], q);
  }
}

template <typename T, bool kQuant, bool kStream>
void launch_norm_as(hipStream_t s, const NormParams& p, const T* x, const T* res, const T* gain, T* y, int8_t* y8,
                 float* scales, T* sum) {
  const int64_t nvec = (p.D + kVecElems<T> - 1) / kVecElems<T>;
#define PJRTX_NORM(TPR, NV)                                                                                     \
  hipLaunchKernelGGL((norm_rows<T, TPR, NV, kQuant, kStream>),                                                  \
                     dim3((uint32_t)((p.rows + (TPR < 256 ? 256 / TPR : 1) - 1) / (TPR < 256 ? 256 / TPR : 1))), \
                     dim3(TPR < 256 ? 256 : TPR), 0, s, p, x, res, gain, y, y8, scales, sum)
  if (nvec <= 64) PJRTX_NORM(64, 1);
  else if (nvec <= 128) PJRTX_NORM(64, 2);
  else if (nvec <= 256) PJRTX_NORM(256, 1);
  else if (nvec <= 512) PJRTX_NORM(256, 2);
  else if (nvec <= 1024) PJRTX_NORM(256, 4);
  else if (nvec <= 2048) PJRTX_NORM(512, 4);
  else if (nvec <= 4096) PJRTX_NORM(1024, 4);
  else
    hipLaunchKernelGGL((norm_long_rows<T, kQuant>), dim3((uint32_t)p.rows), dim3(1024), 0, s, p, x, res, gain, y, y8,
                       scales, sum);
#undef PJRTX_NORM
}

template <typename T, bool kQuant>
void launch_norm(hipStream_t s, const NormParams& p, const T* x, const T* res, const T* gain, T* y, int8_t* y8,
                 float* scales, T* sum) {
  if (p.rows * p.D * static_cast<int64_t>(sizeof(T)) >= kStreamBytes)
    launch_norm_as<T, kQuant, true>(s, p, x, res, gain, y, y8, scales, sum);
  else
    launch_norm_as<T, kQuant, false>(s, p, x, res, gain, y, y8, scales, sum);
}

// ---------------------------------------------------------------- gradient
// Two sums a row: of t^2 and of dy gain t, since mean(dn n) = r mean(dy gain
// t). A workgroup takes every W-th row and keeps its columns' share of dgain
// in registers; the W shares are added by norm_gain_sum in a fixed order, so
// that a gradient is the same bits each time (atomics would not give that).
// Bound by HBM: 8000 x 2048 bf16, 131 MB, in 29 us and 4.7 for the sum.

// The next row is on its way while this one is reduced.
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR)
    norm_grad_rows(NormParams p, const T* __restrict__ dy, const T* __restrict__ dsum, const T* __restrict__ t,
                   const T* __restrict__ gain, T* __restrict__ dx, float* __restrict__ part) {
  constexpr int E = kVecElems<T>;
  typedef typename Vec<T>::type V;
  __shared__ float2 red[2][TPR / 64];
  float acc[NV][E];
  V g[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t at = (int64_t)(v * TPR + threadIdx.x) * E;
    g[v] = load_vec<T>(gain + std::min(at, p.D - 1), p.D - at, (T)0.f);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[v][e] = 0.f;
  }
  struct Raw {
    V t[NV], dy[NV], ds[NV];
  };
  auto request = [&](int64_t row, Raw& x) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int64_t at = (int64_t)(v * TPR + threadIdx.x) * E, n = p.D - at, to = row * p.D + std::min(at, p.D - 1);
      x.t[v] = load_vec<T>(t + to, n, (T)0.f);
      x.dy[v] = load_vec<T>(dy + to, n, (T)0.f);
      if (dsum) x.ds[v] = load_vec<T>(dsum + to, n, (T)0.f);
    }
  };
  Raw next;
  request(blockIdx.x, next);
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const Raw x = next;
    // Unconditional, so that what is waited for below is this row alone.
    request(std::min<int64_t>(row + gridDim.x, p.rows - 1), next);
    float ss = 0.f, sd = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float a = (float)x.t[v][e];
        ss = fmaf(a, a, ss);
        sd = fmaf((float)x.dy[v][e] * (float)g[v][e], a, sd);
      }
    ss = wave_sum(ss);
    sd = wave_sum(sd);
    if constexpr (TPR > 64) {
      if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = make_float2(ss, sd);
      __syncthreads();
      ss = sd = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) {
        ss += red[turn][w].x;
        sd += red[turn][w].y;
      }
    }
    const float r = 1.f / sqrtf(ss / (float)p.D + p.eps);
    const float along = r * r * (sd / (float)p.D);  // mean(dn n) / r, times r^2
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int64_t at = (int64_t)(v * TPR + threadIdx.x) * E;
      const int64_t n = p.D - at;
      if (n <= 0) continue;
      V o;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float a = (float)x.t[v][e], b = (float)x.dy[v][e];
        acc[v][e] = fmaf(b, a * r, acc[v][e]);
        const float back = r * (b * (float)g[v][e] - a * along);
        o[e] = (T)(dsum ? (float)x.ds[v][e] + back : back);
      }
      store_vec<T>(dx + row * p.D + at, n, o);
    }
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int64_t at = (int64_t)(v * TPR + threadIdx.x) * E;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (at + e < p.D) part[(int64_t)blockIdx.x * p.D + at + e] = acc[v][e];
  }
}

// Long rows: each row's two numbers first, then columns.
template <typename T>
__global__ void __launch_bounds__(1024)
    norm_grad_stats(NormParams p, const T* __restrict__ dy, const T* __restrict__ t, const T* __restrict__ gain,
                    float2* __restrict__ stats) {
  __shared__ float red[2][16];
  const int64_t row = blockIdx.x;
  float ss = 0.f, sd = 0.f;
  for (int64_t i = threadIdx.x; i < p.D; i += 1024) {
    const float a = (float)t[row * p.D + i];
    ss = fmaf(a, a, ss);
    sd = fmaf((float)dy[row * p.D + i] * (float)gain[i], a, sd);
  }
  ss = row_sum<1024>(ss, red[0]);
  sd = row_sum<1024>(sd, red[1]);
  if (threadIdx.x == 0) {
    const float r = 1.f / sqrtf(ss / (float)p.D + p.eps);
    stats[row] = make_float2(r, r * r * (sd / (float)p.D));
  }
}
template <typename T>
__global__ void __launch_bounds__(256)
    norm_grad_columns(NormParams p, const T* __restrict__ dy, const T* __restrict__ dsum, const T* __restrict__ t,
                      const T* __restrict__ gain, const float2* __restrict__ stats, T* __restrict__ dx,
                      float* __restrict__ part) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.D) return;
  const float g = (float)gain[i];
  float acc = 0.f;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float2 st = stats[row];
    const float a = (float)t[row * p.D + i], b = (float)dy[row * p.D + i];
    acc = fmaf(b, a * st.x, acc);
    const float back = st.x * (b * g - a * st.y);
    dx[row * p.D + i] = (T)(dsum ? (float)dsum[row * p.D + i] + back : back);
  }
  part[(int64_t)blockIdx.y * p.D + i] = acc;
}

// dgain[c] = sum of part[w][c] over w < W, in an order that W alone sets: 16
// lanes take every 16th share, and are added in lane order.
template <typename T>
__global__ void __launch_bounds__(256)
    norm_gain_sum(int64_t W, int64_t D, const float* __restrict__ part, T* __restrict__ dgain) {
  __shared__ float lanes[16][17];
  const int c = threadIdx.x & 15, l = threadIdx.x >> 4;
  const int64_t col = (int64_t)blockIdx.x * 16 + c;
  float acc = 0.f;
  if (col < D) {
#pragma unroll 8
    for (int64_t w = l; w < W; w += 16) acc += part[w * D + col];
  }
  lanes[l][c] = acc;
  __syncthreads();
  if (l == 0 && col < D) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += lanes[k][c];
    dgain[col] = (T)s;
  }
}

// Rows that the kernel above holds, this one and the next, without spilling: 2
// vectors a thread of 512 (16 bits) or 1024 (f32).
bool grad_in_registers(const NormParams& p) { return p.D <= 8192; }
// Shares of dgain: two workgroups of up to 256 threads, or one of more, a CU. Rows
// and the shares' sum, with two and with one of more: 4000 x 8192 bf16 56.7 + 6.8
// and 51.3 + 5.0 us, 1283 x 4928 and 1000 x 8192 f32 33.5 + 6.5 and 27.8 + 4.8.
// Rows of up to 64 vectors have one wave a workgroup, two a CU, and are bound by
// its latency: 16384 x 512 bf16 31.0 + 4.7 us, 67 MB. Rows of more than 8192
// elements are read twice: 1000 x 16384 bf16 23.3 + 59.5 + 11.8 us, 131 MB.
int64_t grad_shares(const NormParams& p, DType t) {
  const int64_t nvec = (p.D + 16 / static_cast<int64_t>(dtype_size(t)) - 1) / (16 / static_cast<int64_t>(dtype_size(t)));
  return std::min<int64_t>(p.rows, nvec <= 512 || !grad_in_registers(p) ? 512 : 256);
}

template <typename T>
void launch_grad(hipStream_t s, const NormParams& p, const T* dy, const T* dsum, const T* t, const T* gain, T* dx,
                 T* dgain, void* scratch, bool registers, int64_t W) {
  float2* stats = static_cast<float2*>(scratch);
  float* part = registers ? static_cast<float*>(scratch) : reinterpret_cast<float*>(stats + p.rows);
  if (registers) {
    const int64_t nvec = (p.D + kVecElems<T> - 1) / kVecElems<T>;
#define PJRTX_NORM_GRAD(TPR, NV) \
  hipLaunchKernelGGL((norm_grad_rows<T, TPR, NV>), dim3((uint32_t)W), dim3(TPR), 0, s, p, dy, dsum, t, gain, dx, part)
    if (nvec <= 64) PJRTX_NORM_GRAD(64, 1);
    else if (nvec <= 256) PJRTX_NORM_GRAD(256, 1);
    else if (nvec <= 512) PJRTX_NORM_GRAD(256, 2);
    else if (nvec <= 1024) PJRTX_NORM_GRAD(512, 2);
    else if constexpr (kVecElems<T> == 4) PJRTX_NORM_GRAD(1024, 2);
#undef PJRTX_NORM_GRAD
  } else {
    hipLaunchKernelGGL((norm_grad_stats<T>), dim3((uint32_t)p.rows), dim3(1024), 0, s, p, dy, t, gain, stats);
    hipLaunchKernelGGL((norm_grad_columns<T>), dim3((uint32_t)((p.D + 255) / 256), (uint32_t)W), dim3(256), 0, s, p,
                       dy, dsum, t, gain, stats, dx, part);
  }
  hipLaunchKernelGGL((norm_gain_sum<T>), dim3((uint32_t)((p.D + 15) / 16)), dim3(256), 0, s, W, p.D, part, dgain);
}

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(Code::kInternal, strformat("%s launch failed: %s", what, hipGetErrorString(e)));
}

}  // namespace

void launch_add_rms_norm(hipStream_t s, const NormParams& p, DType t, const void* x, const void* residual,
                         const void* gain, void* y, int8_t* y8, float* scales, void* sum) {
  if (p.rows == 0) return;
  auto go = [&](auto tag) {
    using T = decltype(tag);
    const T *xp = static_cast<const T*>(x), *rp = static_cast<const T*>(residual), *gp = static_cast<const T*>(gain);
    if (y8) launch_norm<T, true>(s, p, xp, rp, gp, nullptr, y8, scales, static_cast<T*>(sum));
    else launch_norm<T, false>(s, p, xp, rp, gp, static_cast<T*>(y), nullptr, nullptr, static_cast<T*>(sum));
  };
  if (t == DType::kF32) go(float());
  else if (t == DType::kBF16) go(bf16_t());
  else go(f16_t());
  check_launch("add_rms_norm");
}

size_t add_rms_norm_grad_scratch_bytes(const NormParams& p, DType t) {
  const size_t part = static_cast<size_t>(std::max<int64_t>(1, grad_shares(p, t))) * p.D * sizeof(float);
  return part + (grad_in_registers(p) ? 0 : static_cast<size_t>(p.rows) * sizeof(float2));
}

void launch_add_rms_norm_grad(hipStream_t s, const NormParams& p, DType t, const void* dy, const void* dsum,
                              const void* sum, const void* gain, void* dx, void* dgain, void* scratch) {
  auto go = [&](auto tag) {
    using T = decltype(tag);
    if (p.rows == 0)  // the sum of no rows
      hipLaunchKernelGGL((norm_gain_sum<T>), dim3((uint32_t)((p.D + 15) / 16)), dim3(256), 0, s, 0, p.D,
                         static_cast<const float*>(scratch), static_cast<T*>(dgain));
    else
      launch_grad<T>(s, p, static_cast<const T*>(dy), static_cast<const T*>(dsum), static_cast<const T*>(sum),
                     static_cast<const T*>(gain), static_cast<T*>(dx), static_cast<T*>(dgain), scratch,
                     grad_in_registers(p), grad_shares(p, t));
  };
  if (t == DType::kF32) go(float());
  else if (t == DType::kBF16) go(bf16_t());
  else go(f16_t());
  check_launch("add_rms_norm_grad");
}

}  // namespace pjrtx
