// Causal attention of the last queries of each sequence over the paged 4-bit cache (kv4_sm100.cuh).
//
// With K_t = ks_t u_t + kl_t and V_t = vs_t w_t + vl_t (u, w: codes 0 .. 15 of each dimension; ks, kl, vs, vl: one pair per token and head)
//   logit_t = scale (ks_t (q . u_t) + kl_t sum(q)),   o = sum_t p_t vs_t w_t + sum_t p_t vl_t,   p = softmax(logit)
// so the tensor cores multiply codes, never values: no value is ever unpacked. A code as it lies in its word is an fp16 subnormal,
// code * 2^-24 (or * 2^-20 for the nibble above it), which the tensor cores take exactly: eight codes become four operand words with
// one shift and four ANDs. 2^24 and the 16 between nibbles are folded into exact factors of q and of the output. q goes in as fp16
// after a power of two for each row that puts its largest value near 2^10; p vs goes in as fp16 after a power of two (shared by a warp,
// raised like a running maximum when a larger step comes along) that keeps p vs below 2^15. Logits, maxima, sums and both accumulators are fp32.
//
// A warp has 16 rows (queries x the q heads that share a kv head) and walks blocks of 16 tokens. CTAs of four warps: up to 16 rows all
// four warps share the rows and take every fourth block, each with its own softmax state, joined at the end; up to 32 two and two; above
// that four warps have 64 rows and share each block. Blocks are contiguous in the cache: one bulk copy brings codes and parameters of 16
// tokens into a ring in shared memory.
//
// Work is laid on one line: sequences, row tiles, kv heads, blocks. Each CTA takes an equal run of it, whatever the lengths are. An
// item (sequence, row tile, head) cut by the end of a run is finished by the CTA that counts last: partial outputs, maxima and sums go to
// the workspace and are joined in their order, so the result does not depend on which CTA that is.
#pragma once

#include "kv4_sm100.cuh"

namespace b200 {

struct Kv4AttnParams {
  const uint8_t* cache;
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* lengths;
  const void* q;
  void* o;
  int64_t qs[3], os[3];
  uint64_t group_magic, bpp_magic;
  float scale_log2;
  int batch, queries, q_heads, kv_heads, group, rows, row_tiles;
  int pages, table_pages, page_blocks;
  int min_run;         // blocks a CTA takes at least
  float* partial;      // [CTA][2][row][dim], unnormalised
  float2* partial_ml;  // [CTA][2][row]: maximum (log2) and sum
  uint32_t* counters;  // [CTA]
  uint32_t* status;
};

constexpr int kKv4AttnThreads = 128, kKv4Stages = 4;
constexpr uint32_t kStatusKv4Wait = 1u << 22;

template <int D, int RW>
struct Kv4AttnSmem {
  static constexpr int kTW = 4 / RW;  // warps that share rows
  static constexpr int kBlock = Kv4Layout<D>::kBytes;
  static constexpr int kRing = kTW * kKv4Stages * kBlock;
  static constexpr int kMerge = kTW > 1 ? 4 * 32 * (D / 2) * 4 : 0;  // each warp's accumulators
  static constexpr int kMl = kRing + kMerge;                         // [4][16] float2
  static constexpr int kBars = kMl + 4 * 16 * 8;                     // full, empty
  static constexpr int kFlags = kBars + 2 * kTW * kKv4Stages * 8;
  static constexpr int kBytes = kFlags + 16;
};

__device__ __forceinline__ void bulk_load(void* smem, const void* gmem, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem)), "l"(gmem), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}

// Four operand words of a word of eight codes: pairs (nibble i, nibble i + 4) for i = 0 .. 3; odd i come out 16 times too large.
__device__ __forceinline__ void split_codes(uint32_t w, uint32_t* pairs) {
  const uint32_t h = w >> 8;
  pairs[0] = w & 0x000f000fu;
  pairs[1] = w & 0x00f000f0u;
  pairs[2] = h & 0x000f000fu;
  pairs[3] = h & 0x00f000f0u;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// A CTA's place on the line: an item and the blocks of it that are this CTA's.
struct Kv4Segment {
  int b, tile, head;  // head runs fastest
  int len, blocks;    // of sequence b
  int s0, s1;
  int left;           // blocks of the run behind this segment
};

__device__ __forceinline__ int kv4_length(const Kv4AttnParams& p, int b) {
  const int n = p.lengths[b], most = p.table_pages * p.page_blocks * kKv4Block;
  return n < 0 ? 0 : n > most ? most : n;
}

__device__ __forceinline__ bool kv4_next(const Kv4AttnParams& p, Kv4Segment& s) {
  if (s.left <= 0) return false;
  if (++s.head == p.kv_heads) {
    s.head = 0;
    if (++s.tile == p.row_tiles) {
      s.tile = 0;
      do {  // blocks are left on the line, so a sequence with some follows
        if (++s.b >= p.batch) return false;
        s.len = kv4_length(p, s.b);
      } while (s.len == 0);
      s.blocks = (s.len + kKv4Block - 1) / kKv4Block;
    }
  }
  s.s0 = 0;
  s.s1 = min(s.blocks, s.left);
  s.left -= s.s1;
  return true;
}

// Blocks of the segment that some row of its tile sees: [s0, result).
template <int ROWS>
__device__ __forceinline__ int kv4_seen(const Kv4AttnParams& p, const Kv4Segment& s) {
  const int last = min(p.rows, (s.tile + 1) * ROWS) - 1;
  const int limit = s.len - p.queries + static_cast<int>(magic_div(last, p.group_magic)) + 1;
  return max(s.s0, min(s.s1, (limit + kKv4Block - 1) / kKv4Block));
}

template <typename T, int D, int RW>
__global__ void __launch_bounds__(kKv4AttnThreads, 3) kv4_attn_kernel(const Kv4AttnParams p) {
  using S = Kv4AttnSmem<D, RW>;
  using L = Kv4Layout<D>;
  constexpr int kTW = S::kTW, kRows = 16 * RW;
  constexpr int kWordsK = D / 32;            // words of codes of K in a lane, for each token
  constexpr int kTiles = D / 8;              // column tiles of the output
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int rw = warp % RW, tw = warp / RW;
  uint8_t* ring = smem + tw * kKv4Stages * S::kBlock;
  float* merge = reinterpret_cast<float*>(smem + S::kRing);
  float2* ml_smem = reinterpret_cast<float2*>(smem + S::kMl);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::kBars) + tw * kKv4Stages;
  uint64_t* empty = reinterpret_cast<uint64_t*>(smem + S::kBars) + (kTW + tw) * kKv4Stages;
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + S::kFlags);
  volatile uint32_t* last_flag = abort_flag + 1;
  if (threadIdx.x < kTW * kKv4Stages) {
    mbar_init(reinterpret_cast<uint64_t*>(smem + S::kBars) + threadIdx.x, 1);
    mbar_init(reinterpret_cast<uint64_t*>(smem + S::kBars) + kTW * kKv4Stages + threadIdx.x, RW);
  }
  if (threadIdx.x == 0) abort_flag[0] = abort_flag[2] = 0;
  mbar_init_fence();
  __syncthreads();
  grid_dependency_wait();
  grid_launch_dependents();

  // The line: blocks of all items, and this CTA's run of it.
  const int per = p.kv_heads * p.row_tiles;
  long long total = 0;
  {
    long long mine = 0;
    for (int b = lane; b < p.batch; b += 32) {
      const int n = p.lengths[b], len = kv4_length(p, b);
      if (n != len && n > 0 && threadIdx.x < 32 && blockIdx.x == 0) atomicOr(p.status, kStatusPage);
      mine += (len + kKv4Block - 1) / kKv4Block;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    total = mine * per;
  }
  const long long run = max(static_cast<long long>(p.min_run), (total + gridDim.x - 1) / gridDim.x);
  const long long begin = run * blockIdx.x, end = min(total, begin + run);

  // Rows that see nothing at all get zeros: whole sequences without tokens are on no CTA's run, and rows in front of a sequence's start
  // are written by whoever has their item.
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (kv4_length(p, b) != 0) continue;
    for (int i = threadIdx.x; i < p.queries * p.q_heads * (D / 8); i += kKv4AttnThreads) {
      const int d = i % (D / 8), h = i / (D / 8) % p.q_heads, n = i / (D / 8) / p.q_heads;
      *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + b * p.os[0] + n * p.os[1] + h * p.os[2] + 8 * d) = make_uint4(0, 0, 0, 0);
    }
  }
  if (begin >= end) return;

  Kv4Segment seg{};
  long long item_begin = 0;  // of the segment's item, on the line
  {
    // The sequence the run begins in: 32 lengths at a time.
    long long before = 0;
    int b0 = 0;
    for (;; b0 += 32) {
      const int b = b0 + lane;
      const int blocks = b < p.batch ? (kv4_length(p, b) + kKv4Block - 1) / kKv4Block : 0;
      long long sum = static_cast<long long>(blocks) * per;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, before + sum > begin);
      if (hit != 0) {  // always, at the latest with the last sequence: begin < total
        const int l = __ffs(hit) - 1;
        seg.b = b0 + l;
        seg.blocks = __shfl_sync(0xffffffffu, blocks, l);
        before += __shfl_sync(0xffffffffu, sum, l) - static_cast<long long>(seg.blocks) * per;
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
      if (b0 + 32 >= p.batch) return;
    }
    seg.len = kv4_length(p, seg.b);
    const long long in = begin - before;
    const int item = static_cast<int>(in / seg.blocks);
    seg.s0 = static_cast<int>(in - static_cast<long long>(item) * seg.blocks);
    seg.tile = item / p.kv_heads;
    seg.head = item - seg.tile * p.kv_heads;
    item_begin = begin - seg.s0;
    const long long count = end - begin;
    seg.s1 = static_cast<int>(min(static_cast<long long>(seg.blocks), seg.s0 + count));
    seg.left = static_cast<int>(count - (seg.s1 - seg.s0));
  }

  // The producer's own place: it runs kKv4Stages blocks ahead, over the ends of items. One lane of the first row warp of each token warp.
  const bool producer = rw == 0;
  Kv4Segment ahead = seg;
  int ahead_s = ahead.s0 + tw, ahead_end = kv4_seen<kRows>(p, ahead);
  bool more = true;
  uint32_t issued = 0, used = 0;  // blocks of this token warp, in order
  bool ok = true;
  auto issue = [&]() {
    while (more && ahead_s >= ahead_end) {
      more = kv4_next(p, ahead);
      if (more) {
        ahead_s = ahead.s0 + tw;
        ahead_end = kv4_seen<kRows>(p, ahead);
      }
    }
    if (!more) return;
    const uint32_t stage = issued % kKv4Stages, round = issued / kKv4Stages;
    if (RW > 1 && round > 0 && !mbar_wait(empty + stage, (round - 1) & 1, abort_flag)) {
      ok = false;
      more = false;
      return;
    }
    if (lane == 0) {
      const uint32_t col = magic_div(ahead_s, p.bpp_magic);
      int page = p.page_table[ahead.b * p.table_stride + col];
      if (page < 0 || page >= p.pages) {
        atomicOr(p.status, kStatusPage);
        page = 0;
      }
      const uint8_t* from = p.cache + ((static_cast<int64_t>(page) * p.kv_heads + ahead.head) * p.page_blocks + (ahead_s - static_cast<int>(col) * p.page_blocks)) * S::kBlock;
      mbar_arrive_expect_tx(full + stage, S::kBlock);
      bulk_load(ring + stage * S::kBlock, from, S::kBlock, full + stage);
    }
    __syncwarp();
    ++issued;
    ahead_s += kTW;
  };
  if (producer) {
    for (int i = 0; i < kKv4Stages; ++i) issue();
  }

  for (;;) {
    // Rows r and r + 8 of this warp's 16: their queries as operand words, in the order of a lane's codes.
    const int row0 = seg.tile * kRows + 16 * rw;
    uint32_t qa[2][4 * kWordsK];
    float rscale[2], qsum[2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, ms[2] = {0.f, 0.f};
    int pos[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = min(row0 + r + 8 * i, p.rows - 1);
      const int n = static_cast<int>(magic_div(row, p.group_magic)), g = row - n * p.group;
      pos[i] = seg.len - p.queries + n;
      const T* x = static_cast<const T*>(p.q) + seg.b * p.qs[0] + n * p.qs[1] + (seg.head * p.group + g) * p.qs[2] + c * (D / 4);
      float most = 0.f;
      Raw8<T> raw[kWordsK];
#pragma unroll
      for (int w = 0; w < kWordsK; ++w) raw[w].load(x + 8 * w);
#pragma unroll
      for (int w = 0; w < kWordsK; ++w) {
        float f[8];
        raw[w].unpack(f);
#pragma unroll
        for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(f[k]));
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // 2^e <= most < 2^(e + 1); a row of zeros, subnormals or infinities is taken at the end of the range
      const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100), 126);
      const float up = pow2(10 - e);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWordsK; ++w) {
        float f[8];
        raw[w].unpack(f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          f[k] *= up;
          sum += f[k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float by = k & 1 ? 0.0625f : 1.f;
          qa[i][4 * w + k] = pack2<__half>(f[k] * by, f[k + 4] * by);
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qsum[i] = sum * 5.9604644775390625e-08f;                   // the logits of this row are in units of 2^(e - 10) 2^24
      rscale[i] = p.scale_log2 * pow2(min(e + 14, 127));
    }
    const int seen_by_all = min(pos[0], pos[1]);  // (the lowest of the warp's rows is lane 0's, and all lanes ask it)
    const int lowest = __shfl_sync(0xffffffffu, seen_by_all, 0);
    float o[kTiles][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    int vexp = -120;      // steps of V are taken times 2^(6 - vexp)
    float vscale = 0.f;   // 2^(6 - vexp); 0: no step seen yet
    float vlimit = 0.f;   // steps from here on need a larger vexp
    float limit[2] = {-INFINITY, -INFINITY};  // logits above need a larger maximum

    const int seen = kv4_seen<kRows>(p, seg);
#pragma unroll 1
    for (int s = seg.s0 + tw; s < seen; s += kTW) {
      const uint32_t stage = used % kKv4Stages, round = used / kKv4Stages;
      ok = ok && mbar_wait(full + stage, round & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const uint8_t* block = ring + stage * S::kBlock;
      // q . u of two tiles of eight tokens
      float x[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint32_t w[kWordsK];
        const uint8_t* at = block + (8 * t + r) * L::kRowK + c * (D / 8);
        if constexpr (D == 128) {
          const uint4 v = *reinterpret_cast<const uint4*>(at);
          w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(at);
          w[0] = v.x, w[1] = v.y;
        }
        x[t][0] = x[t][1] = x[t][2] = x[t][3] = 0.f;
#pragma unroll
        for (int i = 0; i < kWordsK; ++i) {
          uint32_t u[4];
          split_codes(w[i], u);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t a[4] = {qa[0][4 * i + 2 * k], qa[1][4 * i + 2 * k], qa[0][4 * i + 2 * k + 1], qa[1][4 * i + 2 * k + 1]};
            mma_16816<__half>(x[t], a, u[2 * k], u[2 * k + 1]);
          }
        }
      }
      // steps and least values of tokens 2 c, 2 c + 1 and 8 behind them
      float ks[4], kl[4], vs[4], vl[4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint4 v = *reinterpret_cast<const uint4*>(block + L::kV + (c + 4 * t) * L::kRowV + D);
        ks[2 * t] = __uint_as_float(v.x << 16), kl[2 * t] = __uint_as_float(v.x & 0xffff0000u);
        vs[2 * t] = __uint_as_float(v.y << 16), vl[2 * t] = __uint_as_float(v.y & 0xffff0000u);
        ks[2 * t + 1] = __uint_as_float(v.z << 16), kl[2 * t + 1] = __uint_as_float(v.z & 0xffff0000u);
        vs[2 * t + 1] = __uint_as_float(v.w << 16), vl[2 * t + 1] = __uint_as_float(v.w & 0xffff0000u);
      }
      const int base = s * kKv4Block;
      const bool masked = base + kKv4Block - 1 > lowest;
      if (masked) {  // parameters behind the sequence's end are whatever the page held
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (base + 2 * c + (k & 1) + 8 * (k >> 1) >= seg.len) ks[k] = kl[k] = vs[k] = vl[k] = 0.f;
      }
      bool raise = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float& y = x[k >> 1][2 * i + (k & 1)];
          y = fmaf(ks[k], y, kl[k] * qsum[i]);
          if (masked && base + 2 * c + (k & 1) + 8 * (k >> 1) > pos[i]) y = -INFINITY;
        }
        const float most = fmaxf(fmaxf(x[0][2 * i], x[0][2 * i + 1]), fmaxf(x[1][2 * i], x[1][2 * i + 1]));
        raise = raise || most > limit[i];
      }
      const float step = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
      raise = raise || step >= vlimit;
      if (__any_sync(0xffffffffu, raise)) {
        // New maxima for the rows and for the steps of V. Infinite and NaN steps are left out: they show in the rows that see them.
        float big = step < INFINITY ? step : 0.f;
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int e = max(vexp, min(static_cast<int>(__float_as_uint(big) >> 23) - 127, 126));
        const float shrink = e == vexp || vscale == 0.f ? 1.f : pow2(max(vexp - e, -126));
        vexp = e;
        vscale = pow2(6 - e);
        vlimit = e >= 126 ? INFINITY : pow2(e + 1);
        float alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float most = fmaxf(fmaxf(x[0][2 * i], x[0][2 * i + 1]), fmaxf(x[1][2 * i], x[1][2 * i + 1]));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
          most = fmaxf(most, m[i]);
          alpha[i] = m[i] == -INFINITY ? 0.f : exp2_approx((m[i] - most) * rscale[i]);
          m[i] = most;
          limit[i] = most == -INFINITY ? most : most + 8.f / rscale[i];
          l[i] *= alpha[i];
          ms[i] *= alpha[i];
          alpha[i] *= shrink;
        }
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          o[i][0] *= alpha[0];
          o[i][1] *= alpha[0];
          o[i][2] *= alpha[1];
          o[i][3] *= alpha[1];
        }
      }
      uint32_t a[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float off = m[i] == -INFINITY ? 0.f : m[i] * rscale[i];
        float e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float y = x[k >> 1][2 * i + (k & 1)];
          const float pk = exp2_approx(fmaf(y, rscale[i], -off));
          l[i] += pk;
          const bool none = masked && y == -INFINITY;  // a masked token's parameters may be anything
          ms[i] = none ? ms[i] : fmaf(pk, vl[k], ms[i]);
          e[k] = none ? 0.f : pk * (vs[k] * vscale);
        }
        a[i] = pack2<__half>(e[0], e[1]);
        a[2 + i] = pack2<__half>(e[2], e[3]);
      }
      {
        uint32_t w0[kWordsK], w1[kWordsK];
        const uint8_t* at = block + L::kV + c * L::kRowV + r * (D / 8);
        if constexpr (D == 128) {
          const uint4 v0 = *reinterpret_cast<const uint4*>(at), v1 = *reinterpret_cast<const uint4*>(at + 4 * L::kRowV);
          w0[0] = v0.x, w0[1] = v0.y, w0[2] = v0.z, w0[3] = v0.w;
          w1[0] = v1.x, w1[1] = v1.y, w1[2] = v1.z, w1[3] = v1.w;
        } else {
          const uint2 v0 = *reinterpret_cast<const uint2*>(at), v1 = *reinterpret_cast<const uint2*>(at + 4 * L::kRowV);
          w0[0] = v0.x, w0[1] = v0.y;
          w1[0] = v1.x, w1[1] = v1.y;
        }
#pragma unroll
        for (int i = 0; i < kWordsK; ++i) {
          uint32_t u0[4], u1[4];
          split_codes(w0[i], u0);
          split_codes(w1[i], u1);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_16816<__half>(o[4 * i + k], a, u0[k], u1[k]);
        }
      }
      __syncwarp();
      ++used;
      if (RW > 1 && lane == 0) mbar_arrive(empty + stage);
      if (producer) issue();
    }
    if (!ok && lane == 0 && atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0) atomicOr(p.status, kStatusKv4Wait);

    // This warp's sums over its lanes, and the output itself: codes' part * 2^24 (2^20 for odd nibbles) / vscale + ms. A maximum of -inf with
    // a sum that is not zero is one of NaN logits alone: it weighs NaN.
    const float unit = pow2(vexp - 6);
    constexpr float kCode = 16777216.f, kHighCode = 1048576.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
        ms[i] += __shfl_xor_sync(0xffffffffu, ms[i], d);
      }
      m[i] = m[i] == -INFINITY ? m[i] : m[i] * rscale[i];  // log2
    }
    // Values q = 16 (or 8) of group (i, k): row r + 8 i, dimensions (2 c + k) D / 8 + q.
    float weight[kTW][2];
    float mt[2] = {m[0], m[1]}, lt[2] = {l[0], l[1]};
    if constexpr (kTW > 1) {
      float* mine = merge + warp * 32 * (D / 2);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) mine[(g * kTiles + i) * 32 + lane] = fmaf(o[i][g] * (i & 1 ? kHighCode : kCode), unit, ms[g >> 1]);
      }
      if (c == 0) {
        ml_smem[warp * 16 + r] = make_float2(m[0], l[0]);
        ml_smem[warp * 16 + r + 8] = make_float2(m[1], l[1]);
      }
    }
    __syncthreads();
    const bool gone = *abort_flag != 0;
    if (kTW > 1 && !gone) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float2 v[kTW];
        mt[i] = -INFINITY;
        lt[i] = 0.f;
#pragma unroll
        for (int k = 0; k < kTW; ++k) {
          v[k] = ml_smem[(k * RW + rw) * 16 + r + 8 * i];
          mt[i] = fmaxf(mt[i], v[k].x);
        }
#pragma unroll
        for (int k = 0; k < kTW; ++k) {
          weight[k][i] = v[k].x == -INFINITY ? v[k].y * 0.f : exp2_approx(v[k].x - mt[i]);
          lt[i] = fmaf(weight[k][i], v[k].y, lt[i]);
        }
      }
    }
    // Whole items go out; parts go to the workspace and are counted.
    const bool whole = seg.s1 - seg.s0 == seg.blocks;
    const int slot = blockIdx.x * 2 + (seg.s0 > 0 ? 0 : 1);
    if (!gone) {
#pragma unroll
      for (int gg = 0; gg < 4 / kTW; ++gg) {
        const int g = kTW > 1 ? tw * (4 / kTW) + gg : gg, i = g >> 1;
        float f[kTiles];
        if constexpr (kTW > 1) {
#pragma unroll
          for (int q = 0; q < kTiles; ++q) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < kTW; ++k) {
              const float part = merge[((k * RW + rw) * 4 + g) * kTiles * 32 + q * 32 + lane];
              const float by = i == 0 ? weight[k][0] : weight[k][1];
              v = by == 0.f ? v : fmaf(by, part, v);
            }
            f[q] = v;
          }
        } else {
#pragma unroll
          for (int q = 0; q < kTiles; ++q) f[q] = fmaf(o[q][gg] * (q & 1 ? kHighCode : kCode), unit, ms[gg >> 1]);
        }
        const int in_tile = 16 * rw + r + 8 * i, row = seg.tile * kRows + in_tile;
        if (row < p.rows) {
          if (whole) {
            const float total_l = i == 0 ? lt[0] : lt[1];
            const float inv = total_l == 0.f ? 0.f : 1.f / total_l;
#pragma unroll
            for (int q = 0; q < kTiles; ++q) f[q] = total_l == 0.f ? 0.f : f[q] * inv;
            const int n = static_cast<int>(magic_div(row, p.group_magic)), head = seg.head * p.group + row - n * p.group;
            T* y = static_cast<T*>(p.o) + seg.b * p.os[0] + n * p.os[1] + head * p.os[2] + (2 * c + (g & 1)) * (D / 8);
#pragma unroll
            for (int q = 0; q < kTiles; q += 8) store8<T>(y + q, f + q);
          } else {
            float* y = p.partial + (static_cast<int64_t>(slot) * kRows + in_tile) * D + (2 * c + (g & 1)) * (D / 8);
#pragma unroll
            for (int q = 0; q < kTiles; q += 4) __stcg(reinterpret_cast<float4*>(y + q), make_float4(f[q], f[q + 1], f[q + 2], f[q + 3]));
            if (c == 0 && (g & 1) == 0) __stcg(p.partial_ml + static_cast<int64_t>(slot) * kRows + in_tile, i == 0 ? make_float2(mt[0], lt[0]) : make_float2(mt[1], lt[1]));
          }
        }
      }
    }
    if (!whole && !gone) {
      const long long item_end = item_begin + seg.blocks;
      const int first = static_cast<int>(item_begin / run), lastc = static_cast<int>((item_end - 1) / run), parts = lastc - first + 1;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) *last_flag = atomicAdd(p.counters + first, 1u) == static_cast<uint32_t>(parts - 1) ? 1u : 0u;
      __syncthreads();
      if (*last_flag != 0) {
        __threadfence();
        const int valid = min(kRows, p.rows - seg.tile * kRows);
        for (int u = threadIdx.x; u < valid * (D / 4); u += kKv4AttnThreads) {
          const int row = u / (D / 4), d = 4 * (u % (D / 4));
          float most = -INFINITY;
          for (int k = 0; k < parts; ++k) most = fmaxf(most, __ldcg(p.partial_ml + (static_cast<int64_t>(first + k) * 2 + (k == 0 ? 1 : 0)) * kRows + row).x);
          float sum = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int k = 0; k < parts; ++k) {
            const int64_t at = (static_cast<int64_t>(first + k) * 2 + (k == 0 ? 1 : 0)) * kRows + row;
            const float2 v = __ldcg(p.partial_ml + at);
            const float4 y = __ldcg(reinterpret_cast<const float4*>(p.partial + at * D + d));
            const float by = v.x == -INFINITY ? v.y * 0.f : exp2_approx(v.x - most);
            if (by != 0.f) {
              sum = fmaf(by, v.y, sum);
              acc.x = fmaf(by, y.x, acc.x);
              acc.y = fmaf(by, y.y, acc.y);
              acc.z = fmaf(by, y.z, acc.z);
              acc.w = fmaf(by, y.w, acc.w);
            }
          }
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          const int at = seg.tile * kRows + row, n = static_cast<int>(magic_div(at, p.group_magic)), head = seg.head * p.group + at - n * p.group;
          T* y = static_cast<T*>(p.o) + seg.b * p.os[0] + n * p.os[1] + head * p.os[2] + d;
          *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        }
        if (threadIdx.x == 0) p.counters[first] = 0;
      }
    }
    __syncthreads();  // merge buffer and flags
    if (gone) break;
    item_begin += seg.blocks;
    if (!kv4_next(p, seg)) break;
  }
  // A wait that ran out leaves copies in flight: they are waited for, again with a limit, before the shared memory goes.
  if (*abort_flag != 0 && producer) {
    for (; used < issued; ++used) mbar_wait(full + used % kKv4Stages, (used / kKv4Stages) & 1, abort_flag + 2);
  }
}

}  // namespace b200
