// Layer norm of rows and its gradients, on sm_100a.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r, y = h w + b
//   t = dy w:  dx = r (t - mean(t) - h mean(t h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// Both are bound by HBM: a row is read once, into registers, and everything that is computed of it comes from there. A row is shared by
// as many threads as leave each some sixteen to thirty-two values; sums and the weights' gradients are fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "sm100_ptx.cuh"

namespace b200 {

struct LayerNormParams {
  const void* x;
  int64_t x_stride;
  void* y;
  int64_t y_stride;
  const void* w;
  const void* b;
  float2* stats;
  const void* dy;
  int64_t dy_stride;
  void* dx;
  int64_t dx_stride;
  float* partial;   // [CTAs][2][dim]: this CTA's part of dw and of db
  int want_dw;      // any of the two
  int wide;         // weights are fp32
  int64_t rows;
  int dim;
  float eps, inverse_dim;
};

template <typename T>
__device__ __forceinline__ float ln_float(T v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T ln_round(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// VEC values side by side: 16 bytes of T where rows allow it, else one value.
template <typename T, int VEC>
struct LnVec {
  alignas(VEC > 1 ? 16 : alignof(T)) T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ LnVec<T, VEC> ln_load(const T* p) {
  LnVec<T, VEC> r;
  if constexpr (sizeof(r) == 16) *reinterpret_cast<uint4*>(&r) = __ldcs(reinterpret_cast<const uint4*>(p));  // read once
  else r.v[0] = *p;
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void ln_store(T* p, const LnVec<T, VEC>& r) {
  if constexpr (sizeof(r) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  else *p = r.v[0];
}
// VEC weights of the rows' type or, `wide`, fp32 (beside a 16-bit row two 16-byte loads).
template <typename T, int VEC>
__device__ __forceinline__ void ln_weights(const void* base, int c, bool wide, float (&out)[VEC]) {
  if (wide && !std::is_same<T, float>::value) {
    const float* const p = static_cast<const float*>(base) + c;
    if constexpr (VEC == 1) {
      out[0] = __ldg(p);
    } else {
#pragma unroll
      for (int i = 0; i < VEC / 4; ++i) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(p) + i);
        out[4 * i] = f.x;
        out[4 * i + 1] = f.y;
        out[4 * i + 2] = f.z;
        out[4 * i + 3] = f.w;
      }
    }
  } else {
    const T* const p = static_cast<const T*>(base) + c;
    if constexpr (VEC == 1) {
      out[0] = ln_float(*p);
    } else {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
#pragma unroll
      for (int j = 0; j < VEC; ++j) out[j] = ln_float(reinterpret_cast<const T*>(&raw)[j]);
    }
  }
}

__device__ __forceinline__ float2 ln_warp_sum2(float2 v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, d);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, d);
  }
  return v;
}

// Sums over the THREADS threads of a row (a warp, or the whole CTA; `turn` alternates between two places, so that one barrier a sum is enough).
template <int THREADS>
__device__ __forceinline__ float2 ln_row_sum2(float2 v, float2 (*place)[32], int& turn) {
  v = ln_warp_sum2(v);
  if constexpr (THREADS > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) place[turn][warp] = v;
    __syncthreads();
    v = lane < THREADS / 32 ? place[turn][lane] : make_float2(0.f, 0.f);
    v = ln_warp_sum2(v);
    turn ^= 1;
  }
  return v;
}

constexpr int kLnForwardRows = 4;  // rows of a CTA whose rows are a warp's each

// Forward. THREADS of a row: 32 (four rows a CTA) or the CTA. A thread has N vectors, THREADS * VEC values apart.
template <typename T, int VEC, int N, int THREADS>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kLnForwardRows : THREADS) norm_rows_kernel(const LayerNormParams p) {
  __shared__ float2 place[2][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t row = THREADS == 32 ? static_cast<int64_t>(blockIdx.x) * kLnForwardRows + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= p.rows) return;  // (a whole warp, where rows are warps'; never where they are CTAs')
  const int at = (threadIdx.x & (THREADS - 1)) * VEC;
  const T* const x = static_cast<const T*>(p.x) + row * p.x_stride;
  LnVec<T, VEC> raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (at + i * THREADS * VEC < p.dim) raw[i] = ln_load<T, VEC>(x + at + i * THREADS * VEC);
  int turn = 0;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (at + i * THREADS * VEC < p.dim) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += ln_float(raw[i].v[j]);
    }
  // Divided: times the rounded 1 / dim, a row of one value would come out as that value's last bit over sqrt(eps).
  const float mean = ln_row_sum2<THREADS>(make_float2(s, 0.f), place, turn).x / static_cast<float>(p.dim);
  float q = 0.f;  // of the differences: no cancellation where the mean is large
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (at + i * THREADS * VEC < p.dim) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = ln_float(raw[i].v[j]) - mean;
        q = fmaf(d, d, q);
      }
    }
  const float var = ln_row_sum2<THREADS>(make_float2(q, 0.f), place, turn).x * p.inverse_dim;
  const float r = 1.f / sqrtf(var + p.eps);
  if (p.stats != nullptr && at == 0) p.stats[row] = make_float2(mean, r);
  T* const y = static_cast<T*>(p.y) + row * p.y_stride;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = at + i * THREADS * VEC;
    if (c < p.dim) {
      float w[VEC], b[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        w[j] = 1.f;
        b[j] = 0.f;
      }
      if (p.w != nullptr) ln_weights<T, VEC>(p.w, c, p.wide != 0, w);
      if (p.b != nullptr) ln_weights<T, VEC>(p.b, c, p.wide != 0, b);
      LnVec<T, VEC> out;
#pragma unroll
      for (int j = 0; j < VEC; ++j) out.v[j] = ln_round<T>(fmaf((ln_float(raw[i].v[j]) - mean) * r, w[j], b[j]));
      ln_store<T, VEC>(y + c, out);
    }
  }
}

constexpr int kLnGradWarps = 8;  // rows of a CTA at a time, where rows are a warp's each

// Gradients. CTAs stay and take every so-manieth row (or rows, a warp each); a thread keeps its columns' part of dw and db in
// registers, and the next row is on its way while this one is worked on. The CTA's parts go to p.partial, which norm_join_kernel adds up.
template <typename T, int VEC, int N, int THREADS>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kLnGradWarps : THREADS) norm_rows_grad_kernel(const LayerNormParams p) {
  constexpr int kRows = THREADS == 32 ? kLnGradWarps : 1;
  __shared__ float2 place[2][32];
  extern __shared__ float joined[];  // [2][dim], where rows are warps'
  grid_dependency_wait();
  grid_launch_dependents();
  const int at = (threadIdx.x & (THREADS - 1)) * VEC, warp = threadIdx.x >> 5;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  float dw[N][VEC], db[N][VEC];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[i][j] = db[i][j] = 0.f;
  LnVec<T, VEC> x[N], g[N];
  float2 stats = make_float2(0.f, 0.f);
  const auto fetch = [&](int64_t row) {
    const T* const xr = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* const gr = static_cast<const T*>(p.dy) + row * p.dy_stride;
    stats = __ldg(p.stats + row);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at + i * THREADS * VEC < p.dim) {
        x[i] = ln_load<T, VEC>(xr + at + i * THREADS * VEC);
        g[i] = ln_load<T, VEC>(gr + at + i * THREADS * VEC);
      }
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + (THREADS == 32 ? warp : 0);
  if (row < p.rows) fetch(row);
  int turn = 0;
  for (; row < p.rows; row += step) {
    const float mean = stats.x, r = stats.y;
    float t[N][VEC], h[N][VEC];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = at + i * THREADS * VEC;
      if (c < p.dim) {
        float w[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) w[j] = 1.f;
        if (p.w != nullptr) ln_weights<T, VEC>(p.w, c, p.wide != 0, w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = ln_float(g[i].v[j]);
          h[i][j] = (ln_float(x[i].v[j]) - mean) * r;
          db[i][j] += d;
          dw[i][j] = fmaf(d, h[i][j], dw[i][j]);
          t[i][j] = d * w[j];
          s.x += t[i][j];
          s.y = fmaf(t[i][j], h[i][j], s.y);
        }
      }
    }
    if (row + step < p.rows) fetch(row + step);
    if (p.dx == nullptr) continue;
    s = ln_row_sum2<THREADS>(s, place, turn);
    const float mean_t = s.x * p.inverse_dim, mean_th = s.y * p.inverse_dim;
    T* const dx = static_cast<T*>(p.dx) + row * p.dx_stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = at + i * THREADS * VEC;
      if (c < p.dim) {
        LnVec<T, VEC> out;
#pragma unroll
        for (int j = 0; j < VEC; ++j) out.v[j] = ln_round<T>(r * (t[i][j] - mean_t - h[i][j] * mean_th));
        ln_store<T, VEC>(dx + c, out);
      }
    }
  }
  if (!p.want_dw) return;
  float* const out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.dim;
  if constexpr (THREADS == 32) {  // the warps' parts, one after the other
    for (int turn_of = 0; turn_of < kRows; ++turn_of) {
      if (warp == turn_of) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int c = at + i * THREADS * VEC + j;
            if (c < p.dim) {
              joined[c] = (turn_of == 0 ? 0.f : joined[c]) + dw[i][j];
              joined[p.dim + c] = (turn_of == 0 ? 0.f : joined[p.dim + c]) + db[i][j];
            }
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * p.dim; c += 32 * kRows) out[c] = joined[c];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = at + i * THREADS * VEC + j;
        if (c < p.dim) {
          out[c] = dw[i][j];
          out[p.dim + c] = db[i][j];
        }
      }
  }
}

// The CTAs' parts of dw and db added up: 32 columns a CTA, a warp every 32nd part, then the warps' sums in their order.
struct NormJoinParams {
  const float* partial;  // [parts][2][dim]
  int parts, dim;
  void* dw;
  void* db;
};
constexpr int kLnJoinWarps = 32;

template <typename W>
__global__ void __launch_bounds__(32 * kLnJoinWarps) norm_join_kernel(const NormJoinParams p) {
  __shared__ float sums[kLnJoinWarps][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  grid_launch_dependents();
  const int c = blockIdx.x * 32 + lane, which = blockIdx.y;
  W* const out = static_cast<W*>(which == 0 ? p.dw : p.db);
  if (out == nullptr) return;
  float s = 0.f;
  if (c < p.dim) {
#pragma unroll 4
    for (int i = warp; i < p.parts; i += kLnJoinWarps) s += __ldg(p.partial + (static_cast<int64_t>(i) * 2 + which) * p.dim + c);
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= p.dim) return;
#pragma unroll
  for (int i = 1; i < kLnJoinWarps; ++i) s += sums[i][lane];
  out[c] = ln_round<W>(s);
}

}  // namespace b200
