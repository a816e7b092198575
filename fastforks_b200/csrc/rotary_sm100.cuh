// Rotary positions of heads, with or without the root-mean-square norm of each head in front, and their gradients:
//   h = x r w,  r = rsqrt(mean(x^2) + eps)                  (norm; else h = x)
//   y_a = h_a c - h_b s,  y_b = h_b c + h_a s               for each pair (a, b) of the first `rot` dimensions, y = h for the rest
// and backwards, with t = the same rotation by -s of the incoming gradient g:
//   dx = t                                                   without a norm
//   dx = r (t w - x r mean(t w x r)),  dw = sum over all heads and tokens of t x r.
// Everything is fp32 and rounded once. The products of a rotation are rounded before they are added, so that the 4-bit cache's
// codes, which round these sums again, come out as elementwise arithmetic gives them.
//
// Bound by HBM: each value is read once and written once (backward with a norm: two reads). Measured, as parts of the measured copy
// bandwidth of 6.5 TB/s: q of [32, 1029, 3, 16, 64] fp16 25.6 us (81 %), [4, 4096, 32, 128] bf16 forward and back 100 us (82 %), norms of 24 + 24
// heads of 64 of 8 x 1370 tokens 28.2 us (73 %), of 32 + 8 heads of 128 of 2 x 4096 with all gradients 98.0 us (66 %); with a norm the
// instructions weigh too (66 % of issue slots). A head is a row; 16 consecutive or
// paired values of it are one lane's, so that a row is a group of 2, 4, 8, 16 or 32 lanes, its sums are shuffles within the group and
// its accesses whole 16-byte words. The rows of a token are dealt to a few groups of lanes, which load the token's cosines and sines once.
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
  uint64_t tokens_magic;
  uint32_t all_tokens;  // batch * tokens
  int table_rows, tokens, dim, rot, tensors;
  int lanes_log2, steps_log2[2];      // lanes of a row; rows of a token that are worked on at once, for each tensor
  bool interleaved, w_f32, vec;       // vec: every row of every tensor is 16-byte aligned
  float eps, inv_dim, sign;           // sign: -1 turns back
  float* partial;                // norm, backward: [2][CTAs][dim]
  uint32_t* counter;
  uint32_t* status;
};

constexpr int kRotaryThreads = 256;
constexpr uint32_t kStatusPosition = 1u << 20, kStatusPage = 1u << 21;

__device__ __forceinline__ uint32_t magic_div(uint32_t n, uint64_t magic) { return magic == 0 ? n : static_cast<uint32_t>(__umul64hi(n, magic)); }

__device__ __forceinline__ bool aligned_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
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

// How a row lies in its lanes, eight dimensions at a first and eight at a second place, so that neighbouring lanes' words are neighbours.
// kRowHalves: lane j < rot / 16 holds dimensions 8 j .. and rot / 2 + 8 j .. (the partners), the lanes behind them the rest in the same way; dim and
// rot in multiples of 16. kRowPairs (neighbours are partners, dim in multiples of 16 and rot of 8), kRowLoose (the same, any rot) and kRowSplit (halves, any
// rot; partners through shared memory): the first half of the row's words of eight dimensions and the second, the last lane's second one
// may be none; dim in multiples of 8.
// kRowAny: 16 consecutive dimensions, partners through shared memory, any rot and dim.
enum RowForm { kRowHalves = 0, kRowPairs = 1, kRowSplit = 2, kRowLoose = 3, kRowAny = 4 };
constexpr int kRowForms = 5;

template <int FORM>
__device__ __forceinline__ void lane_places(int j, int rot, int dim, int* a, int* b) {
  if (FORM == kRowAny) {
    *a = 16 * j;
    *b = 16 * j + 8;
  } else if (FORM != kRowHalves) {
    *a = 8 * j;
    *b = 8 * ((dim + 8) >> 4) + 8 * j;
  } else if (16 * j < rot) {
    *a = 8 * j;
    *b = (rot >> 1) + 8 * j;
  } else {
    *a = (rot >> 1) + 8 * j;
    *b = (dim >> 1) + 8 * j;
  }
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)), y = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = x;
  b = y;
}

// The rotation with fused multiply-adds, behind a norm.
__device__ __forceinline__ void turn_fused(float& a, float& b, float c, float s) {
  const float x = fmaf(a, c, -(b * s)), y = fmaf(b, c, a * s);
  a = x;
  b = y;
}

// A lane's cosines and sines of a token's row of the table, the cosines at 0 and the sines at rot / 2 (nullptr: not rotated).
template <int FORM>
struct Turns {
  float c[8], s[8];
  int first, second;  // pairs of the lane's places that are rotated; but for kRowLoose all of a place's or none
  __device__ __forceinline__ void load(const float* cs, int a, int b, int rot, float sign) {
    if (FORM == kRowLoose) {
      first = cs == nullptr ? 0 : min(max((rot - a) >> 1, 0), 4);
      second = cs == nullptr ? 0 : min(max((rot - b) >> 1, 0), 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if ((i & 3) >= (i < 4 ? first : second)) continue;
        const int at = (i < 4 ? a : b - 8) / 2 + i;
        c[i] = __ldg(cs + at);
        s[i] = __ldg(cs + (rot >> 1) + at);
      }
    } else {
      first = cs != nullptr && (FORM == kRowPairs ? a : b) < rot ? 4 : 0;
      second = cs != nullptr && b < rot ? 4 : 0;
      if (first != 0) get(cs, FORM == kRowPairs ? a >> 1 : a, rot, 0);
      if (second != 0) get(cs, FORM == kRowPairs ? b >> 1 : a + 4, rot, 4);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] *= sign;
  }
  __device__ __forceinline__ void get(const float* cs, int at, int rot, int i) {
    const float4 x = __ldg(reinterpret_cast<const float4*>(cs + at)), y = __ldg(reinterpret_cast<const float4*>(cs + (rot >> 1) + at));
    c[i] = x.x, c[i + 1] = x.y, c[i + 2] = x.z, c[i + 3] = x.w;
    s[i] = y.x, s[i + 1] = y.y, s[i + 2] = y.z, s[i + 3] = y.w;
  }
  template <bool FUSED>
  __device__ __forceinline__ void apply(float* f, float*, int, bool) const {  // a lane's 16 values, 8 at its first place and 8 at its second
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (FORM == kRowLoose ? (i & 3) >= (i < 4 ? first : second) : (FORM == kRowHalves || i < 4 ? first : second) == 0) continue;
      float &x = FORM == kRowHalves ? f[i] : f[2 * i], &y = FORM == kRowHalves ? f[8 + i] : f[2 * i + 1];
      if (FUSED) turn_fused(x, y, c[i], s[i]);
      else turn(x, y, c[i], s[i]);
    }
  }
};

// Halves of any rot: a value's partner is looked up in `row`, the group's floats in shared memory; one that is not turned has cosine 1 and
// sine 0, and a zero for a partner (no branches: sixteen of them do not fit the predicate registers).
template <>
struct Turns<kRowSplit> {
  float c[16], s[16];
  uint32_t partner[8];  // two of 16 bits; all ones: none
  int a, b;
  __device__ __forceinline__ void load(const float* cs, int first_place, int second_place, int rot, float sign) {
    a = first_place, b = second_place;
    const int half = rot >> 1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = i < 8 ? a + i : b + i - 8;
      const bool turned = cs != nullptr && e < rot, late = e >= half;
      const int at = late ? e - half : e;
      c[i] = turned ? __ldg(cs + at) : 1.f;
      s[i] = turned ? (late ? sign : -sign) * __ldg(cs + half + at) : 0.f;
      const uint32_t other = turned ? late ? e - half : e + half : 0xffffu;
      partner[i >> 1] = i & 1 ? partner[i >> 1] | other << 16 : other;
    }
  }
  template <bool FUSED>
  __device__ __forceinline__ void apply(float* f, float* row, int dim, bool) const {
    __syncwarp();
    if (a < dim) store8<float>(row + a, f);
    if (b < dim) store8<float>(row + b, f + 8);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t at = i & 1 ? partner[i >> 1] >> 16 : partner[i >> 1] & 0xffffu;
      const float held = row[at == 0xffffu ? 0 : at], other = at == 0xffffu ? 0.f : held;
      f[i] = FUSED ? fmaf(f[i], c[i], other * s[i]) : __fadd_rn(__fmul_rn(f[i], c[i]), __fmul_rn(other, s[i]));
    }
  }
};

// The same for rows of any form: partners are looked up in `row`, the group's floats in shared memory.
template <>
struct Turns<kRowAny> {
  const float* cs;
  int a, rot;
  float sign;
  __device__ __forceinline__ void load(const float* table, int place, int, int n, float by) { cs = table, a = place, rot = n, sign = by; }
  template <bool FUSED>
  __device__ __forceinline__ void apply(float* f, float* row, int dim, bool interleaved) const {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (a + i < dim) row[a + i] = f[i];
    __syncwarp();
    if (cs == nullptr) return;
    const int half = rot >> 1;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = a + i;
      if (e >= rot) continue;
      const bool first = interleaved ? (e & 1) == 0 : e < half;
      const int at = interleaved ? e >> 1 : first ? e : e - half;
      const float other = row[interleaved ? e ^ 1 : first ? e + half : e - half];
      const float c = __ldg(cs + at), s = sign * __ldg(cs + half + at);
      f[i] = first ? __fsub_rn(__fmul_rn(f[i], c), __fmul_rn(other, s)) : __fadd_rn(__fmul_rn(f[i], c), __fmul_rn(other, s));
    }
  }
};

// 16 values from `at` on of a row, zeros past `dim`. vec: the row starts on 16 bytes.
template <typename T>
__device__ __forceinline__ void load16(float* f, const T* p, int at, int dim, bool vec) {
  if (vec && at + 16 <= dim) {
    Raw8<T> u, v;
    u.load(p + at);
    v.load(p + at + 8);
    u.unpack(f);
    v.unpack(f + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = at + i < dim ? to_f32(p[at + i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const float* f, int at, int dim, bool vec) {
  if (vec && at + 16 <= dim) {
    store8<T>(p + at, f);
    store8<T>(p + at + 8, f + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (at + i < dim) p[at + i] = from_f32<T>(f[i]);
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

__device__ __forceinline__ float group_sum(float v, int lanes_log2) {
  for (int o = 1 << lanes_log2 >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A lane's 16 weights, ones where there are none.
template <typename T, int FORM>
__device__ __forceinline__ void load_weight(float* f, const RotaryParams& p, const void* w, int a, int b) {
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = 1.f;
  if (w == nullptr) return;
  if (FORM != kRowAny && b < p.dim && aligned_16(w)) {
    if (p.w_f32) {
      Raw8<float> u, v;
      u.load(static_cast<const float*>(w) + a);
      v.load(static_cast<const float*>(w) + b);
      u.unpack(f);
      v.unpack(f + 8);
    } else {
      Raw8<T> u, v;
      u.load(static_cast<const T*>(w) + a);
      v.load(static_cast<const T*>(w) + b);
      u.unpack(f);
      v.unpack(f + 8);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int e = (i < 8 ? a : b - 8) + i;
    if (e < p.dim) f[i] = p.w_f32 ? __ldg(static_cast<const float*>(w) + e) : to_f32(static_cast<const T*>(w)[e]);
  }
}

enum RotaryMode { kTurn = 0, kNormTurn = 1, kNormBack = 2 };

// Rows that a lane has in flight, in its own places in shared memory: 128 KB an SM in 16 bits.
template <typename T, int MODE, int FORM>
struct RotaryStream {
  static constexpr int kCtasPerSm = MODE == kNormBack || (MODE == kNormTurn && FORM == kRowSplit) ? 2 : MODE == kNormTurn || FORM == kRowSplit ? 3 : 4;
  static constexpr int kParts = sizeof(T) / 2 * 2;                        // 16-byte words of a row in a lane
  static constexpr int kTensors = MODE == kNormBack ? 2 : 1;             // x, and g
  static constexpr int kDepth = sizeof(T) == 4 ? 2 : 4;
  static constexpr int kSlot = kTensors * kParts * kRotaryThreads * 16;  // bytes of one row of all lanes
  static constexpr int kBytes = kDepth * kSlot;
};

__host__ __device__ constexpr int line_floats(int dim) { return (dim + 3) & ~3; }

// Sums for dw: the lanes' own of tensor k go to this CTA's line of `partial`. A lane's places are a .. a + 7 and b .. b + 7.
__device__ __forceinline__ void put_sums(const RotaryParams& p, float* dw, float* smem, int k, int a, int b, bool place) {
  // Lanes with the same place: within a warp by shuffles, then over the warps through shared memory.
  for (int o = 1 << p.lanes_log2; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < 16; ++i) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
  }
  __syncthreads();  // what lay there before
  if ((threadIdx.x & 31) >> p.lanes_log2 == 0 && place) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = (i < 8 ? a : b - 8) + i;
      if (e < p.dim) smem[(threadIdx.x >> 5) * p.dim + e] = dw[i];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.dim; e += kRotaryThreads) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kRotaryThreads / 32; ++i) v += smem[i * p.dim + e];
    p.partial[(static_cast<int64_t>(k) * gridDim.x + blockIdx.x) * line_floats(p.dim) + e] = v;
  }
  __syncthreads();
}

// The CTA that counts last adds all lines: a thread takes four columns of every so-manieth line, and these sums are added in their order.
template <typename T>
__device__ __forceinline__ void join_sums(const RotaryParams& p, float* smem) {
  __shared__ uint32_t last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(p.counter, 1u) == gridDim.x - 1 ? 1u : 0u;
  __syncthreads();
  if (last == 0) return;
  __threadfence();
  const int quads = line_floats(p.dim) / 4, columns = 2 * quads, shares = kRotaryThreads / columns;  // both tensors' columns
  const int share = threadIdx.x / columns, column = threadIdx.x - share * columns;
  const int k = column >= quads ? 1 : 0;
  float4* sums = reinterpret_cast<float4*>(smem);
  if (share < shares && p.t[k].dw != nullptr) {
    const float4* line = reinterpret_cast<const float4*>(p.partial) + static_cast<int64_t>(k) * gridDim.x * quads + (column - k * quads);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kAtOnce = 16;  // loads in flight, the last ones too
    for (uint32_t c = share; c < gridDim.x; c += kAtOnce * shares) {
      float4 x[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) x[i] = c + i * shares < gridDim.x ? __ldcg(line + static_cast<int64_t>(c + i * shares) * quads) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) v.x += x[i].x, v.y += x[i].y, v.z += x[i].z, v.w += x[i].w;
    }
    sums[threadIdx.x] = v;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * p.dim; e += kRotaryThreads) {
    const int i = e >= p.dim ? 1 : 0, d = e - i * p.dim;
    if (p.t[i].dw == nullptr) continue;
    float v = 0.f;
    for (int n = 0; n < shares; ++n) v += smem[(n * columns + i * quads) * 4 + d];
    if (p.w_f32) static_cast<float*>(p.t[i].dw)[d] = v;
    else static_cast<T*>(p.t[i].dw)[d] = from_f32<T>(v);
  }
  if (threadIdx.x == 0) *p.counter = 0;
}

// Rows of whole lanes on 16 bytes. A lane streams its rows through places of its own in shared memory, kDepth rows ahead, so that what is
// in flight costs no registers; nobody else reads them, so nothing but its own copies has to be waited for. A CTA has an equal run of the
// tokens, and walks it with the first tensor, then with the second (the weights, and backward the sums for dw, are one tensor's at a time);
// its groups of lanes take a few heads each of a few tokens at once, and keep a token's cosines and sines for its heads.
template <typename T, int FORM, int MODE>
__global__ void __launch_bounds__(kRotaryThreads, RotaryStream<T, MODE, FORM>::kCtasPerSm) rotary_stream_kernel(const RotaryParams p) {
  using S = RotaryStream<T, MODE, FORM>;
  extern __shared__ __align__(16) float rotary_smem[];
  grid_dependency_wait();
  grid_launch_dependents();
  const int j = threadIdx.x & ((1 << p.lanes_log2) - 1), group = threadIdx.x >> p.lanes_log2;
  int a, b;
  lane_places<FORM>(j, p.rot, p.dim, &a, &b);
  const int words = (p.dim + 8) >> 4;  // a row's words of eight dimensions, less those at second places
  const bool place = j < words, place_b = place && b < p.dim;
  if (FORM == kRowSplit && !place) a = b = p.dim;  // a lane that holds nothing of a row stores nothing of it (kRowSplit)
  constexpr bool kWhole = FORM == kRowHalves || FORM == kRowPairs;  // every lane has both places
  float* row_smem = rotary_smem + S::kBytes / 4 + group * p.dim;  // kRowSplit
  const uint32_t run_begin = static_cast<uint32_t>(static_cast<uint64_t>(p.all_tokens) * blockIdx.x / gridDim.x);
  const uint32_t run_end = static_cast<uint32_t>(static_cast<uint64_t>(p.all_tokens) * (blockIdx.x + 1) / gridDim.x);
  uint4* mine = reinterpret_cast<uint4*>(rotary_smem) + threadIdx.x;
  const uint32_t mine_at = smem_u32(mine);
  for (int k = 0; k < p.tensors; ++k) {
    const RotaryTensor& t = p.t[k];
    const int step = 1 << p.steps_log2[k], first = group & (step - 1), heads = t.heads;
    const uint32_t at_once = kRotaryThreads >> (p.lanes_log2 + p.steps_log2[k]);  // tokens
    const uint32_t token0 = run_begin + (group >> p.steps_log2[k]);
    const uint32_t warp0 = run_begin + ((threadIdx.x & ~31) >> (p.lanes_log2 + p.steps_log2[k]));  // the warp's first
    const int chunks = warp0 < run_end ? static_cast<int>((run_end - warp0 + at_once - 1) / at_once) : 0;
    float w[16], dw[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 1.f, dw[i] = 0.f;
    if (MODE != kTurn && place) load_weight<T, FORM>(w, p, t.w, a, b);
    // The place of the copies: a chunk of tokens, and the first of `step` heads in it.
    int ahead = 0, ahead_h = 0, slot = 0;
    bool ahead_there = false;
    const T *from_x = nullptr, *from_g = nullptr;
    const auto enter = [&]() {
      const uint32_t token = token0 + ahead * at_once;
      ahead_there = ahead < chunks && place && token < run_end;
      if (!ahead_there) return;
      const uint32_t img = magic_div(token, p.tokens_magic), n = token - img * p.tokens;
      from_x = static_cast<const T*>(t.x) + img * t.xs[0] + n * t.xs[1] + first * t.xs[2];
      if (MODE == kNormBack) from_g = static_cast<const T*>(t.g) + img * t.gs[0] + n * t.gs[1] + first * t.gs[2];
    };
    const auto copy = [&]() {
      if (ahead < chunks) {
        const bool valid = ahead_there && ahead_h + first < heads;
        const uint32_t to = mine_at + slot * S::kSlot;
        constexpr int kHalf = S::kParts / 2;
#pragma unroll
        for (int i = 0; i < S::kParts; ++i) {
          const int at = i < kHalf ? a + i * (16 / static_cast<int>(sizeof(T))) : b + (i - kHalf) * (16 / static_cast<int>(sizeof(T)));
          if (valid && (kWhole || i < kHalf || place_b)) {
            cp_async_16(to + i * kRotaryThreads * 16, from_x + at, true);
            if (MODE == kNormBack) cp_async_16(to + (S::kParts + i) * kRotaryThreads * 16, from_g + at, true);
          }
        }
        from_x += step * t.xs[2];
        if (MODE == kNormBack) from_g += step * t.gs[2];
        ahead_h += step;
        if (ahead_h >= heads) {
          ahead_h = 0;
          ++ahead;
          enter();
        }
      }
      cp_async_commit();
      slot = slot + 1 == S::kDepth ? 0 : slot + 1;
    };
    enter();
#pragma unroll
    for (int i = 0; i < S::kDepth - 1; ++i) copy();
    int use = 0;
    for (int chunk = 0; chunk < chunks; ++chunk) {  // the same for all lanes of a warp
      const uint32_t token = token0 + chunk * at_once;
      const bool there = place && token < run_end;
      const uint32_t img = there ? magic_div(token, p.tokens_magic) : 0, n = there ? token - img * p.tokens : 0;
      T* y = static_cast<T*>(t.y) + img * t.ys[0] + n * t.ys[1] + first * t.ys[2];
      Turns<FORM> turns;
      turns.load(there ? token_row(p, img, n) : nullptr, a, b, p.rot, MODE == kNormBack ? -1.f : p.sign);
      for (int h0 = 0; h0 < heads; h0 += step) {
        copy();
        cp_async_wait<S::kDepth - 1>();
        const uint4* at = mine + use * (S::kSlot / 16);
        use = use + 1 == S::kDepth ? 0 : use + 1;
        const bool valid = there && h0 + first < heads;
        float f[16];
        const auto read = [&](float* to, int part) {
          Raw8<T> u;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (!kWhole && i == 1 && !place_b) {
#pragma unroll
              for (int n = 8; n < 16; ++n) to[n] = 0.f;
              continue;
            }
            if constexpr (sizeof(T) == 4) {
              u.a = *reinterpret_cast<const float4*>(at + (part + 2 * i) * kRotaryThreads);
              u.b = *reinterpret_cast<const float4*>(at + (part + 2 * i + 1) * kRotaryThreads);
            } else {
              u.v = at[(part + i) * kRotaryThreads];
            }
            u.unpack(to + 8 * i);
          }
        };
        if (valid) {
          read(f, 0);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = 0.f;
        }
        if constexpr (MODE == kTurn) {
          turns.template apply<false>(f, row_smem, p.dim, false);
        } else {
          float e[16], sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum = fmaf(f[i], f[i], sum);
          if constexpr (MODE == kNormTurn) {
            const float r = rsqrtf(fmaf(group_sum(sum, p.lanes_log2), p.inv_dim, p.eps));
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = f[i] * r * w[i];
            turns.template apply<true>(f, row_smem, p.dim, false);
          } else {
            if (valid) {
              read(e, S::kParts);
            } else {
#pragma unroll
              for (int i = 0; i < 16; ++i) e[i] = 0.f;
            }
            turns.template apply<true>(e, row_smem, p.dim, false);
            float along = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) along = fmaf(e[i] * w[i], f[i], along);
            for (int o = 1 << p.lanes_log2 >> 1; o > 0; o >>= 1) {
              sum += __shfl_xor_sync(0xffffffffu, sum, o);
              along += __shfl_xor_sync(0xffffffffu, along, o);
            }
            const float r = valid ? rsqrtf(fmaf(sum, p.inv_dim, p.eps)) : 0.f;  // no row: nothing for dw, whatever eps is
            const float back = along * r * r * p.inv_dim;  // r mean(t w x r)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float hat = f[i] * r;
              dw[i] = fmaf(e[i], hat, dw[i]);
              f[i] = fmaf(r, e[i] * w[i], -(hat * back));
            }
          }
        }
        if (valid) {
          store8<T>(y + a, f);
          if (kWhole || place_b) store8<T>(y + b, f + 8);
        }
        y += step * t.ys[2];
      }
    }
    cp_async_wait<0>();
    if (MODE == kNormBack && t.dw != nullptr) put_sums(p, dw, rotary_smem, k, a, b, place);
    __syncthreads();  // the places are laid anew, and were smem of the sums
  }
  if (MODE == kNormBack && (p.t[0].dw != nullptr || p.t[1].dw != nullptr)) join_sums<T>(p, rotary_smem);
}

// Rows of any kind, one at a time.
template <typename T, int MODE>
__global__ void __launch_bounds__(kRotaryThreads, 2) rotary_any_kernel(const RotaryParams p) {
  extern __shared__ __align__(16) float rotary_smem[];
  grid_dependency_wait();
  grid_launch_dependents();
  const int j = threadIdx.x & ((1 << p.lanes_log2) - 1), group = threadIdx.x >> p.lanes_log2;
  float* row_smem = rotary_smem + group * p.dim;
  int a, b;
  lane_places<kRowAny>(j, p.rot, p.dim, &a, &b);
  const bool place = a < p.dim;
  for (int k = 0; k < p.tensors; ++k) {
    const RotaryTensor& t = p.t[k];
    const int step = 1 << p.steps_log2[k], first = group & (step - 1);
    const uint32_t in_chunk = group >> p.steps_log2[k], chunk_tokens = kRotaryThreads >> (p.lanes_log2 + p.steps_log2[k]);
    float w[16], dw[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 1.f, dw[i] = 0.f;
    if (MODE != kTurn && place) load_weight<T, kRowAny>(w, p, t.w, a, b);
    for (uint32_t token0 = blockIdx.x * chunk_tokens; token0 < p.all_tokens; token0 += gridDim.x * chunk_tokens) {
      const uint32_t token = token0 + in_chunk;
      const bool there = place && token < p.all_tokens;
      const uint32_t img = there ? magic_div(token, p.tokens_magic) : 0, n = there ? token - img * p.tokens : 0;
      Turns<kRowAny> turns;
      turns.load(there ? token_row(p, img, n) : nullptr, a, b, p.rot, MODE == kNormBack ? -1.f : p.sign);
      for (int h0 = 0; h0 < t.heads; h0 += step) {
        const int h = h0 + first;
        const bool valid = there && h < t.heads;
        float f[16];
        load16<T>(f, static_cast<const T*>(t.x) + img * t.xs[0] + n * t.xs[1] + h * t.xs[2], a, valid ? p.dim : 0, p.vec);
        if constexpr (MODE == kTurn) {
          turns.template apply<false>(f, row_smem, p.dim, p.interleaved);
        } else {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum = fmaf(f[i], f[i], sum);
          const float mean = fmaf(group_sum(sum, p.lanes_log2), p.inv_dim, p.eps), r = valid ? rsqrtf(mean) : 0.f;  // no row: nothing for dw, whatever eps is
          if constexpr (MODE == kNormTurn) {
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = f[i] * r * w[i];
            turns.template apply<false>(f, row_smem, p.dim, p.interleaved);
          } else {
            float e[16], along = 0.f;
            load16<T>(e, static_cast<const T*>(t.g) + img * t.gs[0] + n * t.gs[1] + h * t.gs[2], a, valid ? p.dim : 0, p.vec);
            turns.template apply<false>(e, row_smem, p.dim, p.interleaved);
#pragma unroll
            for (int i = 0; i < 16; ++i) along = fmaf(e[i] * w[i], f[i], along);
            const float back = group_sum(along, p.lanes_log2) * r * r * p.inv_dim;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float hat = f[i] * r;
              dw[i] = fmaf(e[i], hat, dw[i]);
              f[i] = fmaf(r, e[i] * w[i], -(hat * back));
            }
          }
        }
        if (valid) store16<T>(static_cast<T*>(t.y) + img * t.ys[0] + n * t.ys[1] + h * t.ys[2], f, a, p.dim, p.vec);
      }
    }
    if (MODE == kNormBack && t.dw != nullptr) put_sums(p, dw, rotary_smem, k, a, b, place);
  }
  if (MODE == kNormBack && (p.t[0].dw != nullptr || p.t[1].dw != nullptr)) join_sums<T>(p, rotary_smem);
}

}  // namespace b200
