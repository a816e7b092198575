// Layer norm of rows and its gradients, on sm_100a.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r, y = h w + b
//   t = dy w:  dx = r (t - mean(t) - h mean(t h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// Both have their floor in HBM's bytes: a row is read once, into registers, and everything that is computed of it comes from there. What binds them above it
// is the chain of a row (load, two sums over its threads, store): in 16 bits neither memory nor issue slots are at their end. A row is shared by
// as many threads as leave each some sixteen to thirty-two values; sums and the weights' gradients are fp32. norm_rows_kernel is the forward pass;
// norm_ring_grad_kernel the gradients of rows on 16-byte boundaries of up to 8192 16-bit or 4096 fp32 values, norm_rows_grad_kernel of all others.
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
  int slots;        // rows of a group's ring
  uint32_t* status;
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
// Two neighbouring values of sixteen bytes.
template <typename T>
__device__ __forceinline__ float2 ln_pair(const uint4& raw, int j) {
  if constexpr (std::is_same<T, float>::value) {
    return reinterpret_cast<const float2*>(&raw)[j];
  } else {
    const uint32_t v = reinterpret_cast<const uint32_t*>(&raw)[j];
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
}

// Eight (fp32: four) values rounded and packed: pairs convert in one instruction.
template <typename T, int PAIRS>
__device__ __forceinline__ uint4 ln_packed(const float2 (&v)[PAIRS]) {
  if constexpr (std::is_same<T, float>::value) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  } else {
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[j].x, v[j].y);
        out[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[j].x, v[j].y);
        out[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
  }
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

// The same in pairs, or `missing` without weights.
template <typename T, int VEC, int PAIRS>
__device__ __forceinline__ void ln_weight_pairs(const void* base, int c, bool wide, float missing, float2 (&out)[PAIRS]) {
  if (base == nullptr) {
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) out[j] = make_float2(missing, missing);
  } else if constexpr (VEC == 1) {
    float v[1];
    ln_weights<T, 1>(base, c, wide, v);
    out[0] = make_float2(v[0], 0.f);
  } else if (wide && !std::is_same<T, float>::value) {
    const float4* const from = reinterpret_cast<const float4*>(static_cast<const float*>(base) + c);
#pragma unroll
    for (int j = 0; j < PAIRS; j += 2) {
      const float4 f = __ldg(from + j / 2);
      out[j] = make_float2(f.x, f.y);
      out[j + 1] = make_float2(f.z, f.w);
    }
  } else {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(base) + c));
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) out[j] = ln_pair<T>(raw, j);
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

__device__ __forceinline__ float ln_warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// s / n as s times the rounded 1 / n and one correction: times that alone, a row of one value would come out as the product's error over sqrt(eps).
__device__ __forceinline__ float ln_mean(float s, float n, float inverse_n) {
  const float m = s * inverse_n;
  return fmaf(fmaf(-m, n, s), inverse_n, m);
}

// Sums over the THREADS threads of a row (a warp, or the whole CTA; `turn` alternates between two places, so that one barrier a sum is enough).
template <int THREADS>
__device__ __forceinline__ float ln_row_sum(float v, float2 (*place)[32], int& turn) {
  v = ln_warp_sum(v);
  if constexpr (THREADS > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) place[turn][warp].x = v;
    __syncthreads();
    v = ln_warp_sum(lane < THREADS / 32 ? place[turn][lane].x : 0.f);
    turn ^= 1;
  }
  return v;
}
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

// Forward. THREADS of a row: 32 (four rows a CTA) or the CTA; ROWS rows at a time, which share weights and barriers (forward_forms in b200_training.cu).
// A thread has N vectors, THREADS * VEC values apart; they go in pairs, which the packed instructions take at once. us, value by value -> in pairs, one row at a
// time and one input again and again (part of it in L2): 8192 x 4096 in bf16 28.9 -> 24.3, 21920 x 1024 17.9 -> 15.3. Now, several inputs in turn, and the time of
// the bytes: 8192 x 4096 27.3 (20.5), 21920 x 1024 18.2 (13.7), 16384 x 2048 25.7 (20.5), 21920 x 768 in fp16 16.0 (10.3), 8192 x 4096 in fp32 43.0 (41.0).
// 197 x 768: 2.7, the launch and a chain of latencies.
template <typename T, int VEC, int N, int THREADS, int ROWS>
__global__ void __launch_bounds__(THREADS == 32 ? 32 * kLnForwardRows : THREADS) norm_rows_kernel(const LayerNormParams p) {
  __shared__ float2 place[2][32];
  grid_dependency_wait();
  grid_launch_dependents();
  constexpr int kStep = THREADS * VEC, kPairs = VEC > 1 ? VEC / 2 : 1, kWarpRows = THREADS == 32 ? kLnForwardRows : 1;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kWarpRows * ROWS + (THREADS == 32 ? threadIdx.x >> 5 : 0);  // and kWarpRows further on
  if (row0 >= p.rows) return;  // (a whole warp, where rows are warps'; never where they are CTAs')
  const int at = (threadIdx.x & (THREADS - 1)) * VEC;
  const auto there = [&](int k) { return k == 0 || row0 + kWarpRows < p.rows; };
  LnVec<T, VEC> raw[ROWS][N];
#pragma unroll
  for (int k = 0; k < ROWS; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at + i * kStep < p.dim && there(k)) raw[k][i] = ln_load<T, VEC>(static_cast<const T*>(p.x) + (row0 + k * kWarpRows) * p.x_stride + at + i * kStep);
  // Kept as it came, and converted at each of three uses: held as fp32, it cost warps (8192 x 4096 in bf16, one row at a time, 34.7 us; so 24.3).
  // A single value is a pair whose second half does not count.
  const auto pair = [&](int k, int i, int j) {
    if constexpr (VEC > 1) return ln_pair<T>(*reinterpret_cast<const uint4*>(&raw[k][i]), j);
    else return make_float2(ln_float(raw[k][i].v[0]), 0.f);
  };
  int turn = 0;
  const auto row_sums = [&](const float2 (&s)[ROWS]) {
    if constexpr (ROWS == 1) return make_float2(ln_row_sum<THREADS>(s[0].x + s[0].y, place, turn), 0.f);
    else return ln_row_sum2<THREADS>(make_float2(s[0].x + s[0].y, s[1].x + s[1].y), place, turn);
  };
  float2 s[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    s[k] = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at + i * kStep < p.dim) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) s[k] = fadd2(s[k], pair(k, i, j));
      }
  }
  const float2 sums = row_sums(s);
  float2 minus[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const float mean = ln_mean(k == 0 ? sums.x : sums.y, static_cast<float>(p.dim), p.inverse_dim);
    minus[k] = make_float2(-mean, VEC > 1 ? -mean : 0.f);
    s[k] = make_float2(0.f, 0.f);  // of the differences: no cancellation where the mean is large
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at + i * kStep < p.dim) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const float2 d = fadd2(pair(k, i, j), minus[k]);
          s[k] = ffma2(d, d, s[k]);
        }
      }
  }
  const float2 squares = row_sums(s);
  float2 r2[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const float r = rsqrtf((k == 0 ? squares.x : squares.y) * p.inverse_dim + p.eps);
    r2[k] = make_float2(r, r);
    if (p.stats != nullptr && at == 0 && there(k)) p.stats[row0 + k * kWarpRows] = make_float2(-minus[k].x, r);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = at + i * kStep;
    if (c < p.dim) {
      float2 w[kPairs], b[kPairs];
      ln_weight_pairs<T, VEC>(p.w, c, p.wide != 0, 1.f, w);
      ln_weight_pairs<T, VEC>(p.b, c, p.wide != 0, 0.f, b);
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        if (!there(k)) continue;
        T* const y = static_cast<T*>(p.y) + (row0 + k * kWarpRows) * p.y_stride + c;
        float2 v[kPairs];
#pragma unroll
        for (int j = 0; j < kPairs; ++j) v[j] = ffma2(fmul2(fadd2(pair(k, i, j), minus[k]), r2[k]), w[j], b[j]);
        if constexpr (VEC > 1) *reinterpret_cast<uint4*>(y) = ln_packed<T>(v);
        else *y = ln_round<T>(v[0].x);
      }
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

// ---- gradients, rows through shared memory -----------------------------------------------------------------------------------------------
// Sums behind dw and db want the CTAs to stay, and then what HBM needs in flight does not fit beside a row in registers. G warps share a row, and every
// such group has a ring of rows that one of its lanes fills with bulk copies (cp.async.bulk, 16-byte addresses and sizes), some 200 KB an
// SM. A slot is filled again as soon as the group has it in registers. Slots are as wide as G warps of N vectors, with zeros behind the row, so that
// no value is tested for being one; weights stay in registers as fp32 pairs (with a test and a conversion at each use a value took 29
// instructions, and 8192 rows of 4096 54 us). us with the join, of bf16: a row a CTA with the next one in registers (norm_rows_grad_kernel) -> here, and
// the time of the bytes: 8192 x 4096 75.0 -> 40.9 (30.8), 21920 x 1024 48.4 -> 30.8 (20.6), 30000 x 512 64.4 -> 20.5 (14.1), 300 x 4096 18.3 -> 7.8; fp32
// 8192 x 4096 74.3 -> 67.7 (61.6), 5480 x 384 14.5 -> 8.9 (3.9). Bound in fp32 by HBM and in 16 bits, at sixteen warps an SM, by the chain of copy, sums and
// barrier of each row (8192 x 4096: DRAM 53 %, issue slots 41 %). The same for the forward pass was slower than rows in registers but for the largest calls (several
// inputs in turn: 1200 x 4096 10.1 against 7.6, 5000 x 4096 19.7 and 19.6, 10000 x 4096 30.7 and 32.8): two barriers a row, and nothing that has to stay. (Groups added one after the other into one place took 5 us more at 16 groups.)
constexpr int kLnMostWarps = 16, kLnMostSlots = 16, kLnRingBytes = 208 * 1024;
constexpr uint32_t kStatusNormWait = 1u << 24;
// Warps of a CTA, one on each SM, as the registers of so many values a thread allow. (Two CTAs of eight warps leave twice as many parts to join.)
constexpr int ln_ring_warps(int values) { return values <= 16 ? 16 : 8; }

struct LnRingSmem {
  uint64_t full[kLnMostWarps][kLnMostSlots];
  alignas(16) float2 place[kLnMostWarps][2][8];  // of each group, alternately: its warps' sums
  uint32_t abort;
};

__device__ __forceinline__ void ln_bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               :
               : "r"(smem_dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int G>
__device__ __forceinline__ void ln_group_sync(int group) {
  if constexpr (G == 1) __syncwarp();
  else asm volatile("barrier.cta.sync %0, %1;" ::"r"(group + 1), "n"(G * 32) : "memory");
}
// Both sums over a group, in the order of its warps: the halves of a warp take one each after the first exchange. Behind it every thread of the
// group has passed the point where it was called.
template <int G>
__device__ __forceinline__ float2 ln_group_sum2(float2 v, LnRingSmem& sm, int group, int& turn) {
  const int lane = threadIdx.x & 31;
  float one = lane < 16 ? v.x : v.y;
  one += __shfl_xor_sync(0xffffffffu, lane < 16 ? v.y : v.x, 16);
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) one += __shfl_xor_sync(0xffffffffu, one, d);
  if constexpr (G == 1) {
    const float other = __shfl_xor_sync(0xffffffffu, one, 16);
    return lane < 16 ? make_float2(one, other) : make_float2(other, one);
  } else {
    if ((lane & 15) == 0) reinterpret_cast<float*>(&sm.place[group][turn][(threadIdx.x >> 5) % G])[lane >> 4] = one;
    ln_group_sync<G>(group);
    const float4* const from = reinterpret_cast<const float4*>(sm.place[group][turn]);
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < G / 2; ++i) {
      const float4 o = from[i];
      sum = fadd2(fadd2(sum, make_float2(o.x, o.y)), make_float2(o.z, o.w));
    }
    turn ^= 1;
    return sum;
  }
}
// A group's ring: rows first, first + step, ... of x and dy, a slot for both.
struct LnRing {
  uint32_t slots;  // of this group, in shared memory
  uint64_t* full;
  const uint8_t *a, *b;  // the next row to be asked for
  int64_t a_step, b_step;  // bytes
  int64_t next, step, rows;
  uint32_t bytes, row_bytes;  // of a row, and of its place
  int count, slot;
  uint32_t phase;
  bool leader;

  __device__ __forceinline__ void fill(int at, const uint32_t* abort) {
    if (next < rows) {
      if (leader && *static_cast<const volatile uint32_t*>(abort) == 0) {
        mbar_arrive_expect_tx(&full[at], 2 * bytes);
        ln_bulk_load(slots + 2 * at * row_bytes, a, bytes, &full[at]);
        ln_bulk_load(slots + (2 * at + 1) * row_bytes, b, bytes, &full[at]);
      }
      next += step;
      a += a_step;
      b += b_step;
    }
  }
  __device__ __forceinline__ uint32_t wait(uint32_t* abort, uint32_t* status) {
    if (!mbar_wait(&full[slot], phase, abort) && atomicExch(abort, 1u) == 0) atomicOr(status, kStatusNormWait);  // the rest runs through, with what is there
    return slots + 2 * slot * row_bytes;
  }
  __device__ __forceinline__ void advance() {
    if (++slot == count) {
      slot = 0;
      phase ^= 1;
    }
  }
  // Copies still on their way when a wait has run out must land before the CTA goes. (Each slot's last use; where one was never used, its
  // barrier stands at phase 0, and the wait for phase 1 ends at once.)
  __device__ __forceinline__ void drain(const uint32_t* abort) const {
    if (*static_cast<const volatile uint32_t*>(abort) == 0 || !leader) return;
    uint32_t no_abort = 0;
    for (int i = 0; i < count; ++i) mbar_wait(&full[i], i < slot ? phase : phase ^ 1, &no_abort);
  }
};

template <typename T, int VEC, int N, int G>
__device__ __forceinline__ LnRing ln_ring(LnRingSmem& sm, uint8_t* memory, const LayerNormParams& p) {
  constexpr int kWarps = ln_ring_warps(N * VEC), kGroups = kWarps / G;
  const int group = (threadIdx.x >> 5) / G;
  LnRing r;
  r.bytes = static_cast<uint32_t>(p.dim * sizeof(T));
  r.row_bytes = G * 32 * VEC * N * sizeof(T);
  r.count = p.slots;
  r.slots = smem_u32(memory) + 2 * group * p.slots * r.row_bytes;
  r.full = sm.full[group];
  r.rows = p.rows;
  r.step = static_cast<int64_t>(gridDim.x) * kGroups;
  r.next = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  r.a = reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.x) + r.next * p.x_stride);
  r.b = reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.dy) + r.next * p.dy_stride);
  r.a_step = r.step * p.x_stride * static_cast<int64_t>(sizeof(T));
  r.b_step = r.step * p.dy_stride * static_cast<int64_t>(sizeof(T));
  r.slot = 0;
  r.phase = 0;
  r.leader = threadIdx.x % (G * 32) == 0;
  if (threadIdx.x == 0) {
    for (int g = 0; g < kGroups; ++g)
      for (int i = 0; i < p.slots; ++i) mbar_init(&sm.full[g][i], 1);
    sm.abort = 0;
    mbar_init_fence();
  }
  const uint32_t tail = r.row_bytes - r.bytes;  // a multiple of 16, as both are
  if (tail > 0) {
    const int words = static_cast<int>(tail >> 4), places = 2 * kGroups * p.slots;
    for (int i = threadIdx.x; i < places * words; i += 32 * kWarps) {
      const int at = i / words;
      st_shared_v4(smem_u32(memory) + at * r.row_bytes + r.bytes + (i - at * words) * 16, make_uint4(0, 0, 0, 0));
    }
  }
  __syncthreads();
  return r;
}

// Gradients: one pass for the sums, dw and db, one barrier, dx from registers.
template <typename T, int VEC, int N, int G>
__global__ void __launch_bounds__(32 * ln_ring_warps(N * VEC), 1) norm_ring_grad_kernel(const LayerNormParams p) {
  extern __shared__ __align__(128) uint8_t ln_memory[];
  __shared__ LnRingSmem sm;
  constexpr int kStep = G * 32 * VEC, kWarps = ln_ring_warps(N * VEC), kGroups = kWarps / G, kPairs = VEC / 2;
  const int group = (threadIdx.x >> 5) / G, at = (threadIdx.x % (G * 32)) * VEC;
  LnRing ring = ln_ring<T, VEC, N, G>(sm, ln_memory, p);
  grid_dependency_wait();
  grid_launch_dependents();
  int64_t row = ring.next;
  for (int i = 0; i < ring.count; ++i) ring.fill(i, &sm.abort);
  float2 w[N][kPairs], dw[N][kPairs], db[N][kPairs];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    ln_weight_pairs<T, VEC>(at + i * kStep < p.dim ? p.w : nullptr, at + i * kStep, p.wide != 0, 1.f, w[i]);
#pragma unroll
    for (int j = 0; j < kPairs; ++j) dw[i][j] = db[i][j] = make_float2(0.f, 0.f);
  }
  float2 stats = row < p.rows ? __ldg(p.stats + row) : make_float2(0.f, 0.f);
  T* dx = static_cast<T*>(p.dx) + row * p.dx_stride + at;
  const int64_t dx_step = ring.step * p.dx_stride;
  int turn = 0;
  for (; row < p.rows; row += ring.step, dx += dx_step) {
    const float2 minus = make_float2(-stats.x, -stats.x), r2 = make_float2(stats.y, stats.y);
    const uint32_t slot = ring.wait(&sm.abort, p.status) + at * static_cast<int>(sizeof(T));
    if (row + ring.step < p.rows) stats = __ldg(p.stats + row + ring.step);
    float2 t[N][kPairs], h[N][kPairs], s = make_float2(0.f, 0.f), q = s;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint4 x = ld_shared_v4(slot + i * kStep * static_cast<int>(sizeof(T))), g = ld_shared_v4(slot + ring.row_bytes + i * kStep * static_cast<int>(sizeof(T)));
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const float2 d = ln_pair<T>(g, j);
        h[i][j] = fmul2(fadd2(ln_pair<T>(x, j), minus), r2);
        db[i][j] = fadd2(db[i][j], d);
        dw[i][j] = ffma2(d, h[i][j], dw[i][j]);
        t[i][j] = fmul2(d, w[i][j]);
        s = fadd2(s, t[i][j]);
        q = ffma2(t[i][j], h[i][j], q);
      }
    }
    s = ln_group_sum2<G>(make_float2(s.x + s.y, q.x + q.y), sm, group, turn);
    if constexpr (G == 1) __syncwarp();
    ring.fill(ring.slot, &sm.abort);
    ring.advance();
    if (p.dx == nullptr) continue;
    const float mean_t = s.x * p.inverse_dim, mean_th = s.y * p.inverse_dim;
    const float2 mt2 = make_float2(-mean_t, -mean_t), mh2 = make_float2(-mean_th, -mean_th);
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) t[i][j] = fmul2(ffma2(h[i][j], mh2, fadd2(t[i][j], mt2)), r2);
      if (at + i * kStep < p.dim) *reinterpret_cast<uint4*>(dx + i * kStep) = ln_packed<T>(t[i]);
    }
  }
  ring.drain(&sm.abort);
  if (!p.want_dw) return;
  // The groups' parts side by side in what was the ring (every copy has landed; every slot has been read), then added in the order of the groups.
  float* const out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.dim;
  if constexpr (kGroups > 1) {
    float* const joined = reinterpret_cast<float*>(ln_memory);
    __syncthreads();
    float* const mine = joined + static_cast<size_t>(group) * 2 * p.dim + at;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (at + i * kStep >= p.dim) continue;
#pragma unroll
      for (int j = 0; j < kPairs; j += 2) {
        *reinterpret_cast<float4*>(mine + i * kStep + 2 * j) = make_float4(dw[i][j].x, dw[i][j].y, dw[i][j + 1].x, dw[i][j + 1].y);
        *reinterpret_cast<float4*>(mine + p.dim + i * kStep + 2 * j) = make_float4(db[i][j].x, db[i][j].y, db[i][j + 1].x, db[i][j + 1].y);
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.dim / 2; c += 32 * kWarps) {
      float4 sum = reinterpret_cast<const float4*>(joined)[c];
      for (int g = 1; g < kGroups; ++g) {
        const float4 more = reinterpret_cast<const float4*>(joined + static_cast<size_t>(g) * 2 * p.dim)[c];
        sum.x += more.x;
        sum.y += more.y;
        sum.z += more.z;
        sum.w += more.w;
      }
      reinterpret_cast<float4*>(out)[c] = sum;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at + i * kStep < p.dim) {
#pragma unroll
        for (int j = 0; j < kPairs; j += 2) {
          *reinterpret_cast<float4*>(out + at + i * kStep + 2 * j) = make_float4(dw[i][j].x, dw[i][j].y, dw[i][j + 1].x, dw[i][j + 1].y);
          *reinterpret_cast<float4*>(out + p.dim + at + i * kStep + 2 * j) = make_float4(db[i][j].x, db[i][j].y, db[i][j + 1].x, db[i][j + 1].y);
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
#pragma unroll 10
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
