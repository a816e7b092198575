// A paged cache of keys and values held in 4 bits: writing new tokens (keys and queries rotated on the way) and reading them back.
// The layout is stated in include/b200_decoder.h; it is the attention kernel's: a block of sixteen tokens of one head is contiguous, a
// lane's codes of K are consecutive, and a 32-bit word of V holds the same four dimensions of two neighbouring tokens, which is what a
// 16 x 8 tile of the second product takes from one lane.
//
// A head's vector of one token is a group: step = bf16((max - min) / 15), least = bf16(min), code = clamp(round((x - least) / step)). The
// codes are taken against the rounded pair, so they get back what its rounding costs but for the ends of the range: the largest value may
// lie 15 * 2^-9 of a step, and either end 2^-9 of |min|, outside of what codes reach. That is below a step as long as |min| is below 34 ranges; a vector
// whose values all lie near one large value comes back coarser (around 100 with deviation 0.25: up to 3.2 steps off). Division is by multiplication with the rounded reciprocal of 15 and of the step.
//
// Bound by launch latency for single tokens (64 of them: append 4.2 us, read 5.0) and by instructions and HBM for prompts (4 x 2047 tokens,
// 32 + 2 x 8 heads of 128: append 36 us, read 10; a kernel that kept a token's place for several of its heads, and one that streamed q apart,
// were no faster: 45 and 40 us where this one took 41 then). Rows (a head of q, k or v of one token) are four or eight lanes of
// sixteen values, as in the rotary kernels.
#pragma once

#include "rotary_sm100.cuh"

namespace b200 {

constexpr int kKv4Block = 16;  // tokens
template <int D>
struct Kv4Layout {
  static constexpr int kRowK = D / 2, kV = 8 * D, kRowV = D + 16, kBytes = 16 * (D + 8);
};

struct Kv4Params {
  uint8_t* cache;
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* lengths;
  const float* cs;
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;
  int64_t qs[3], ks[3], vs[3], qos[3], kos[3], vos[3];
  uint64_t heads_magic, tokens_magic, page_magic;
  uint32_t rows;
  int tokens, q_heads, kv_heads, rot, page, pages, table_pages, table_rows, heads;
  bool interleaved;
  uint32_t* status;
};

constexpr int kKv4Threads = 256;

// Address of the block that holds position `at` of sequence `b` for `head`, and the token's place in it; nullptr if there is none.
template <int D>
__device__ __forceinline__ uint8_t* kv4_block(const Kv4Params& p, uint32_t b, int at, int head, int* token) {
  const uint32_t col = magic_div(at, p.page_magic);
  if (col >= static_cast<uint32_t>(p.table_pages)) {
    atomicOr(p.status, kStatusPage);
    return nullptr;
  }
  const int page = p.page_table[b * p.table_stride + col];
  if (page < 0 || page >= p.pages) {
    atomicOr(p.status, kStatusPage);
    return nullptr;
  }
  const int in_page = at - static_cast<int>(col) * p.page;
  *token = in_page & (kKv4Block - 1);
  const int blocks = p.page / kKv4Block;
  return p.cache + ((static_cast<int64_t>(page) * p.kv_heads + head) * blocks + in_page / kKv4Block) * Kv4Layout<D>::kBytes;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Codes of a group's values, 16 in this lane and the others in the LANES - 1 lanes beside it: eight codes in either word, the first in the
// lowest bits. Returns the pair (step in the low, least value in the high half).
template <int LANES>
__device__ __forceinline__ uint32_t quantise16(const float* f, uint32_t* words) {
  float low = f[0], high = f[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) {
    low = min_nan(low, f[i]);
    high = max_nan(high, f[i]);
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  const float span = __fsub_rn(high, low);
  words[0] = words[1] = 0;
  if (!(fabsf(span) < INFINITY)) return 0x7fc07fc0u;
  float step = __bfloat162float(__float2bfloat16_rn(__fmul_rn(span, 1.f / 15.f)));
  const float least = __bfloat162float(__float2bfloat16_rn(low));
  if (!(fabsf(least) < INFINITY) || !(step < INFINITY)) return 0x7fc07fc0u;  // rounded past the largest bfloat16
  if (step < 1.17549435e-38f) {
    step = 0.f;
  } else {
    // A code between 0 and 15 is rounded to even by adding 1.5 * 2^23; four of them make a word of 16 bits, exact as a float.
    constexpr float kWhole = 12582912.f, kWord = 8388608.f;
    const float inverse = __frcp_rn(step);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      float word = kWord;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float t = fminf(fmaxf(__fmul_rn(__fsub_rn(f[4 * h + i], least), inverse), 0.f), 15.f);
        word = fmaf(__fsub_rn(__fadd_rn(t, kWhole), kWhole), static_cast<float>(1 << (4 * i)), word);
      }
      words[h >> 1] |= (__float_as_uint(word) & 0xffffu) << (16 * (h & 1));
    }
  }
  return (__float_as_uint(step) >> 16) | (__float_as_uint(least) & 0xffff0000u);
}

template <typename T, int D, int FORM>
__global__ void __launch_bounds__(kKv4Threads) kv4_append_kernel(const Kv4Params p) {
  constexpr int kLanes = D / 16, kGroups = kKv4Threads / kLanes;
  using L = Kv4Layout<D>;
  __shared__ __align__(16) float rows_smem[FORM == kRowSplit ? kGroups * D : 4];
  grid_dependency_wait();
  grid_launch_dependents();
  const int j = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const uint32_t row = blockIdx.x * kGroups + group;
  const bool there = row < p.rows;
  const uint32_t token = magic_div(there ? row : 0, p.heads_magic);
  int h = static_cast<int>((there ? row : 0) - token * p.heads);
  const uint32_t b = magic_div(token, p.tokens_magic), n = token - b * p.tokens;
  const int what = h < p.q_heads ? 0 : h < p.q_heads + p.kv_heads ? 1 : 2;
  h -= what == 0 ? 0 : what == 1 ? p.q_heads : p.q_heads + p.kv_heads;
  const int64_t* s = what == 0 ? p.qs : what == 1 ? p.ks : p.vs;
  const T* x = static_cast<const T*>(what == 0 ? p.q : what == 1 ? p.k : p.v) + b * s[0] + n * s[1] + h * s[2];
  int at0, at1;
  lane_places<FORM>(j, p.rot, D, &at0, &at1);
  if (what == 2) lane_places<kRowAny>(j, 0, D, &at0, &at1);
  float f[16];
  {
    Raw8<T> u, v;
    u.load(x + at0);
    v.load(x + at1);
    u.unpack(f);
    v.unpack(f + 8);
  }
  const int at = p.lengths[b] - p.tokens + static_cast<int>(n);
  const float* cs = what == 2 ? nullptr : table_row(p.cs, p.rot, p.table_rows, at, p.status);
  Turns<FORM> turns;
  turns.load(cs, at0, at1, p.rot, 1.f);
  turns.template apply<false>(f, rows_smem + (FORM == kRowSplit ? group * D : 0), D, p.interleaved);
  uint32_t words[2], pair = 0;
  if (__any_sync(0xffffffffu, what != 0)) pair = quantise16<kLanes>(f, words);
  if (!there) return;
  if (what == 0) {
    T* y = static_cast<T*>(p.q_out) + b * p.qos[0] + n * p.qos[1] + h * p.qos[2];
    store8<T>(y + at0, f);
    store8<T>(y + at1, f + 8);
    return;
  }
  if (at < 0) return;
  int t;
  uint8_t* block = kv4_block<D>(p, b, at, h, &t);
  if (block == nullptr) return;
  uint8_t* tail = block + L::kV + (t >> 1) * L::kRowV;
  if (what == 1) {
    uint32_t* codes = reinterpret_cast<uint32_t*>(block + t * L::kRowK);
    codes[at0 >> 3] = words[0];
    codes[at1 >> 3] = words[1];
  } else {
    uint16_t* codes = reinterpret_cast<uint16_t*>(tail) + (t & 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) codes[2 * (4 * j + i)] = static_cast<uint16_t>(words[i >> 1] >> (16 * (i & 1)));
  }
  if (j == 0) *reinterpret_cast<uint32_t*>(tail + D + (t & 1) * 8 + (what == 2 ? 4 : 0)) = pair;
}

// The values of the last tokens, in 16 bits: K and V of a head of one token by one group of lanes, whose places they share.
template <typename T, int D>
__global__ void __launch_bounds__(kKv4Threads) kv4_read_kernel(const Kv4Params p) {
  constexpr int kLanes = D / 16, kGroups = kKv4Threads / kLanes;
  using L = Kv4Layout<D>;
  grid_dependency_wait();
  grid_launch_dependents();
  const int j = threadIdx.x % kLanes;
  const uint32_t row = blockIdx.x * kGroups + threadIdx.x / kLanes;
  if (row >= p.rows) return;
  const uint32_t token = magic_div(row, p.heads_magic);
  const int h = static_cast<int>(row - token * p.heads);
  const uint32_t b = magic_div(token, p.tokens_magic), n = token - b * p.tokens;
  const int at = p.lengths[b] - p.tokens + static_cast<int>(n);
  int t = 0;
  const uint8_t* block = at < 0 ? nullptr : kv4_block<D>(p, b, at, h, &t);
  uint32_t words[4] = {0, 0, 0, 0};
  uint2 pairs = make_uint2(0, 0);
  if (block != nullptr) {
    const uint8_t* tail = block + L::kV + (t >> 1) * L::kRowV;
    const uint2 k = *reinterpret_cast<const uint2*>(block + t * L::kRowK + 8 * j);
    const uint4 v = *reinterpret_cast<const uint4*>(tail + 16 * j);
    pairs = *reinterpret_cast<const uint2*>(tail + D + (t & 1) * 8);
    const int half = t & 1 ? 0x7632 : 0x5410;  // this token's half of either word
    words[0] = k.x;
    words[1] = k.y;
    words[2] = __byte_perm(v.x, v.y, half);
    words[3] = __byte_perm(v.z, v.w, half);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t pair = i == 0 ? pairs.x : pairs.y;
    const float step = __uint_as_float(pair << 16), least = __uint_as_float(pair & 0xffff0000u);
    T* y = static_cast<T*>(i == 0 ? p.k_out : p.v_out) + (i == 0 ? b * p.kos[0] + n * p.kos[1] + h * p.kos[2] : b * p.vos[0] + n * p.vos[1] + h * p.vos[2]) + 16 * j;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = fmaf(step, static_cast<float>((words[2 * i + w] >> (4 * k)) & 15u), least);  // the product is exact
      store8<T>(y + 8 * w, f);
    }
  }
}

}  // namespace b200
