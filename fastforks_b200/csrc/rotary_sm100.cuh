// Rotary positions of heads, with or without the root-mean-square norm of each head in front, and their gradients:
//   h = x r w,  r = rsqrt(mean(x^2) + eps)                  (norm; else h = x)
//   y_a = h_a c - h_b s,  y_b = h_b c + h_a s               for each pair (a, b) of the first `rot` dimensions, y = h for the rest
// and backwards, with t = the same rotation by -s of the incoming gradient g:
//   dx = t                                                   without a norm
//   dx = r (t w - x r mean(t w x r)),  dw = sum over all heads and tokens of t x r.
// Everything is fp32 and rounded once. The products of a rotation are rounded before they are added, so that the 4-bit cache's
// codes, which round these sums again, come out as elementwise arithmetic gives them.
//
// Bound by HBM: each value is read once and written once (backward with a norm: two reads). A head is a row; 16 consecutive or
// paired values of it are one lane's, so that a row is a group of 2, 4, 8, 16 or 32 lanes, its sums are shuffles within the group and
// its accesses whole 16-byte words. Rows are numbered with the heads of one token next to one another: the token's row of the
// table comes from L1.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "sm100_ptx.cuh"

namespace b200 {

struct RotaryTensor {
  const void* x;
  void* y;
  const void* g;
  const void* w;
  void* dw;
  int64_t xs[3], ys[3], gs[3];  // element strides: batch, token, head
  int heads;
};
struct RotaryParams {
  RotaryTensor t[2];
  const float* cs;
  const int32_t* positions;
  int64_t ps[2];
  uint64_t heads_magic, tokens_magic, t_magic[2];
  uint32_t rows;  // of both tensors
  uint32_t t_rows[2];
  int table_rows, tokens, dim, rot, lanes, heads;
  bool interleaved, w_f32, vec;  // vec: every row of every tensor is 16-byte aligned
  float eps, sign;               // sign: -1 turns back
  float* partial;                // norm, backward: [2][CTAs][dim]
  uint32_t* counter;
  uint32_t* status;
};

constexpr int kRotaryThreads = 256;
constexpr uint32_t kStatusPosition = 1u << 20, kStatusPage = 1u << 21;

__device__ __forceinline__ uint32_t magic_div(uint32_t n, uint64_t magic) { return magic == 0 ? n : static_cast<uint32_t>(__umul64hi(n, magic)); }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight values as they lie in memory, 16-byte aligned.
template <typename T>
struct Raw8 {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void unpack(float* f) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = d.x;
        f[2 * i + 1] = d.y;
      } else {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void unpack(float* f) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
};
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* f) {
  if constexpr (std::is_same<T, float>::value) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
  }
}

// How a row lies in its lanes. kRowHalves: lane j < rot / 16 holds dimensions 8 j .. and rot / 2 + 8 j .. (the partners), the lanes behind
// them 16 consecutive dimensions each. kRowPairs: 16 consecutive dimensions. Both want rot and dim in multiples of 16. kRowAny: 16
// consecutive dimensions, partners through shared memory, any rot and dim.
enum RowForm { kRowHalves = 0, kRowPairs = 1, kRowAny = 2 };

template <int FORM>
__device__ __forceinline__ void lane_places(int j, int rot, int* a, int* b) {
  *a = 16 * j;
  *b = 16 * j + 8;
  if (FORM == kRowHalves && 16 * j < rot) {
    *a = 8 * j;
    *b = (rot >> 1) + 8 * j;
  }
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)), y = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
  b = y;
}

// Rotates a lane's 16 values f (8 at its first place, 8 at its second). `cs`: the token's row of the table (nullptr: not rotated), the
// cosines at 0 and the sines at rot / 2. `row`: the group's floats in shared memory (kRowAny).
template <int FORM>
__device__ __forceinline__ void rotate16(float* f, const float* cs, int j, int rot, int dim, float sign, bool interleaved, float* row) {
  if constexpr (FORM != kRowAny) {
    if (cs == nullptr || 16 * j >= rot) return;
    const float4* c4 = reinterpret_cast<const float4*>(cs + 8 * j);
    const float4* s4 = reinterpret_cast<const float4*>(cs + (rot >> 1) + 8 * j);
    const float4 c0 = __ldg(c4), c1 = __ldg(c4 + 1), s0 = __ldg(s4), s1 = __ldg(s4 + 1);
    const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (FORM == kRowHalves) turn(f[i], f[8 + i], c[i], sign * s[i]);
      else turn(f[2 * i], f[2 * i + 1], c[i], sign * s[i]);
    }
  } else {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (16 * j + i < dim) row[16 * j + i] = f[i];
    __syncwarp();
    if (cs == nullptr) return;
    const int half = rot >> 1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = 16 * j + i;
      if (e >= rot) continue;
      const bool first = interleaved ? (e & 1) == 0 : e < half;
      const int at = interleaved ? e >> 1 : first ? e : e - half;
      const float other = row[interleaved ? e ^ 1 : first ? e + half : e - half];
      const float c = __ldg(cs + at), s = sign * __ldg(cs + half + at);
      f[i] = first ? __fsub_rn(__fmul_rn(f[i], c), __fmul_rn(other, s)) : __fadd_rn(__fmul_rn(f[i], c), __fmul_rn(other, s));
    }
  }
}

// A lane's 16 values of the row at `p`, zeros past `dim`.
template <typename T, int FORM>
__device__ __forceinline__ void load16(float* f, const T* p, int a, int b, int dim, bool vec) {
  if (FORM != kRowAny || (vec && a + 16 <= dim)) {
    Raw8<T> u, v;
    u.load(p + a);
    v.load(p + b);
    u.unpack(f);
    v.unpack(f + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = a + i < dim ? to_f32(p[a + i]) : 0.f;
  }
}
template <typename T, int FORM>
__device__ __forceinline__ void store16(T* p, const float* f, int a, int b, int dim, bool vec) {
  if (FORM != kRowAny || (vec && a + 16 <= dim)) {
    store8<T>(p + a, f);
    store8<T>(p + b, f + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (a + i < dim) p[a + i] = from_f32<T>(f[i]);
  }
}

// The table's row of a token, nullptr where it is not rotated.
__device__ __forceinline__ const float* table_row(const float* cs, int rot, int rows, int at, uint32_t* status) {
  if (at < 0 || rot == 0) return nullptr;
  if (at >= rows) {
    atomicOr(status, kStatusPosition);
    return nullptr;
  }
  return cs + static_cast<int64_t>(at) * rot;
}
__device__ __forceinline__ const float* token_row(const RotaryParams& p, uint32_t b, uint32_t n) {
  return p.rot == 0 ? nullptr : table_row(p.cs, p.rot, p.table_rows, p.positions == nullptr ? static_cast<int>(n) : p.positions[b * p.ps[0] + n * p.ps[1]], p.status);
}

__device__ __forceinline__ float group_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A lane's 16 weights, ones where there are none.
template <typename T, int FORM>
__device__ __forceinline__ void load_weight(float* f, const RotaryParams& p, const void* w, int a, int b) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int e = (i < 8 ? a : b - 8) + i;
    f[i] = w == nullptr || e >= p.dim ? 1.f : p.w_f32 ? __ldg(static_cast<const float*>(w) + e) : to_f32(static_cast<const T*>(w)[e]);
  }
}

// Forward, and backward without a norm (x = g, sign = -1).
template <typename T, int FORM, bool NORM>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p) {
  extern __shared__ float rotary_smem[];
  grid_dependency_wait();
  grid_launch_dependents();
  const int j = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes, groups = kRotaryThreads / p.lanes;
  float* row_smem = rotary_smem + group * p.dim;
  int a, b;
  lane_places<FORM>(j, p.rot, &a, &b);
  const bool mine = 16 * j < p.dim;
  const uint32_t row = blockIdx.x * groups + group;
  const bool there = row < p.rows;
  const uint32_t token = magic_div(there ? row : 0, p.heads_magic);
  uint32_t h = (there ? row : 0) - token * p.heads;
  const bool second = h >= static_cast<uint32_t>(p.t[0].heads);
  const RotaryTensor& t = p.t[second ? 1 : 0];
  if (second) h -= p.t[0].heads;
  const uint32_t img = magic_div(token, p.tokens_magic), n = token - img * p.tokens;
  const T* x = static_cast<const T*>(t.x) + img * t.xs[0] + n * t.xs[1] + h * t.xs[2];
  float f[16];
  if (there && mine) {
    load16<T, FORM>(f, x, a, b, p.dim, p.vec);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = 0.f;
  }
  const float* cs = token_row(p, img, n);
  if constexpr (NORM) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = fmaf(f[i], f[i], sum);
    const float r = rsqrtf(group_sum(sum, p.lanes) / p.dim + p.eps);
    float w[16];
    if (mine) load_weight<T, FORM>(w, p, t.w, a, b);
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = f[i] * r * w[i];
  }
  rotate16<FORM>(f, cs, j, p.rot, p.dim, p.sign, p.interleaved, row_smem);
  if (there && mine) store16<T, FORM>(static_cast<T*>(t.y) + img * t.ys[0] + n * t.ys[1] + h * t.ys[2], f, a, b, p.dim, p.vec);
}

// Gradients through norm and rotation. A CTA walks rows of the first tensor, then of the second, and keeps its lanes' sums for dw in
// registers; they go through shared memory to a line of `partial`, and the CTA that counts last adds the lines in their order.
template <typename T, int FORM>
__global__ void __launch_bounds__(kRotaryThreads) norm_rotary_backward_kernel(const RotaryParams p) {
  extern __shared__ float rotary_smem[];
  grid_dependency_wait();
  grid_launch_dependents();
  const int j = threadIdx.x & (p.lanes - 1), group = threadIdx.x / p.lanes, groups = kRotaryThreads / p.lanes;
  float* row_smem = rotary_smem + group * p.dim;
  int a, b;
  lane_places<FORM>(j, p.rot, &a, &b);
  const bool mine = 16 * j < p.dim;
  for (int k = 0; k < 2; ++k) {
    if (p.t_rows[k] == 0) continue;
    const RotaryTensor& t = p.t[k];
    float w[16], dw[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 1.f, dw[i] = 0.f;
    if (mine) load_weight<T, FORM>(w, p, t.w, a, b);
    for (uint32_t first = blockIdx.x * groups; first < p.t_rows[k]; first += gridDim.x * groups) {
      const bool there = first + group < p.t_rows[k];
      const uint32_t row = there ? first + group : 0;
      const uint32_t token = magic_div(row, p.t_magic[k]), h = row - token * t.heads;
      const uint32_t img = magic_div(token, p.tokens_magic), n = token - img * p.tokens;
      float f[16], g[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = g[i] = 0.f;
      if (there && mine) {
        load16<T, FORM>(f, static_cast<const T*>(t.x) + img * t.xs[0] + n * t.xs[1] + h * t.xs[2], a, b, p.dim, p.vec);
        load16<T, FORM>(g, static_cast<const T*>(t.g) + img * t.gs[0] + n * t.gs[1] + h * t.gs[2], a, b, p.dim, p.vec);
      }
      rotate16<FORM>(g, token_row(p, img, n), j, p.rot, p.dim, -1.f, p.interleaved, row_smem);
      float sum = 0.f, along = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sum = fmaf(f[i], f[i], sum);
        along = fmaf(g[i] * w[i], f[i], along);
      }
      sum = group_sum(sum, p.lanes);
      along = group_sum(along, p.lanes);
      const float r = rsqrtf(sum / p.dim + p.eps);
      const float back = along * r / p.dim;  // mean(t w x r)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float hat = f[i] * r;
        dw[i] = fmaf(g[i], hat, dw[i]);
        f[i] = r * (g[i] * w[i] - hat * back);
      }
      if (there && mine) store16<T, FORM>(static_cast<T*>(t.y) + img * t.ys[0] + n * t.ys[1] + h * t.ys[2], f, a, b, p.dim, p.vec);
    }
    if (t.dw == nullptr) continue;
    // Lanes with the same place: within a warp by shuffles, then over the warps through shared memory.
    for (int o = p.lanes; o < 32; o <<= 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
    }
    __syncthreads();  // rows of kRowAny, and the other tensor's sums
    if ((threadIdx.x & 31) < p.lanes && mine) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int e = (i < 8 ? a : b - 8) + i;
        if (e < p.dim) rotary_smem[(threadIdx.x >> 5) * p.dim + e] = dw[i];
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.dim; e += kRotaryThreads) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < kRotaryThreads / 32; ++i) v += rotary_smem[i * p.dim + e];
      p.partial[(static_cast<int64_t>(k) * gridDim.x + blockIdx.x) * p.dim + e] = v;
    }
    __syncthreads();
  }
  if (p.t[0].dw == nullptr && p.t[1].dw == nullptr) return;
  __shared__ uint32_t last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(p.counter, 1u) == gridDim.x - 1 ? 1u : 0u;
  __syncthreads();
  if (last == 0) return;
  __threadfence();
  // Eight warps take every eighth line each; a warp's sums of a column are added to the others' in their order.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int k = 0; k < 2; ++k) {
    const RotaryTensor& t = p.t[k];
    if (p.t_rows[k] == 0 || t.dw == nullptr) continue;
    const float* lines = p.partial + static_cast<int64_t>(k) * gridDim.x * p.dim;
    for (int e = lane; e < p.dim; e += 32) {
      float v = 0.f;
#pragma unroll 8
      for (uint32_t c = warp; c < gridDim.x; c += 8) v += __ldcg(lines + static_cast<int64_t>(c) * p.dim + e);
      rotary_smem[warp * p.dim + e] = v;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.dim; e += kRotaryThreads) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += rotary_smem[i * p.dim + e];
      if (p.w_f32) static_cast<float*>(t.dw)[e] = v;
      else static_cast<T*>(t.dw)[e] = from_f32<T>(v);
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.counter = 0;
}

}  // namespace b200
