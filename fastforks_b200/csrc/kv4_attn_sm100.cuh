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
// Codes are the left operand: S^T = K Q^T has 16 tokens by 8 rows, O^T = V^T P^T 16 dimensions by 8 rows, so that eight rows (the q heads
// that share a kv head, of one query) fill a product. P^T comes out of the first product with tokens along the lanes and goes
// into the second with rows along them: one transposition of 8 x 8 in registers for each eight tokens. Codes of V multiply p vs as
// code - 8, and vl + 8 vs takes the rest in fp32: rounding p vs then errs by a part of a value, not of a code up to 15. For q in fp16 the 8 is
// taken off in the operand (exact in subnormals, four more instructions a word), for bfloat16 one more row of the product sums 8 p vs and
// is taken off at the end: over 20000 tokens the sums of codes cancel to 1 / 100 of themselves, which fp32 has room for
// beside an output of 8 bits, but not of 11 (error of fp16 outputs 1.65 times the output's own rounding, 1.4 with codes less 8; in bfloat16 the row is 2 % faster, 78.0 us against 79.5).
//
// A warp has 8 or 16 rows (queries x the q heads that share a kv head) and walks steps of 32 tokens. CTAs of four warps: up to 16 rows all
// four warps share the rows and take every fourth step, each with its own softmax state, joined at the end; up to 32 two and two; above
// that four warps have 64 rows and share each step. Blocks are contiguous in the cache, and so are the two of a step where pages hold a
// multiple of 32 tokens: bulk copies bring codes and parameters into a ring in shared memory.
//
// Work is laid on one line: sequences, row tiles, kv heads, steps. Each CTA takes an equal run of it. All steps of a sequence count for each of
// its row tiles, those behind the tile's causal limit too, which are left out when their turn comes: even for a few queries behind a long
// text, uneven for whole prompts, where the busiest CTA has about twice the mean. An
// item (sequence, row tile, head) cut by the end of a run is finished by the CTA that counts last: partial outputs, maxima and sums go to
// the workspace and are joined in their order, so the result does not depend on which CTA that is.
//
// Measured, one query of 32 heads on 8, head dim 128, bf16: 64 sequences up to 8192 tokens (290 MB of cache) 77 to 85 us by the pages' order, 52 to 58 %
// of the copy bandwidth. No unit is at its end there (issue 54 %, the integer pipe that takes codes apart 51 %, DRAM 45 % of nominal): what warps wait for
// most is the fixed latency of instructions that follow one another, at four warps a scheduler; a step has 160 instructions that take codes
// apart and some 450 beside them. One sequence of 4000 tokens 14 us, of 1000 10, of 100 6: 6 are launch, lengths, queries and first loads, the rest is parts and
// their join.
#pragma once

#include <float.h>

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
  int min_run;         // steps a CTA takes at least
  float* partial;      // [CTA][2][row][dim], unnormalised
  float2* partial_ml;  // [CTA][2][row]: maximum (log2) and sum
  uint32_t* counters;  // [CTA]
  uint32_t* status;
};

constexpr int kKv4AttnThreads = 128, kKv4Stages = 2, kKv4Step = 2 * kKv4Block;
// What an item costs beside its steps (queries, joining the warps, output), in steps: units of the line in front of its first step.
constexpr int kKv4Item = 4;
constexpr uint32_t kStatusKv4Wait = 1u << 22;

// NR: tiles of eight rows of a warp. RW: warps with rows of their own, the other 4 / RW share theirs.
template <int D, int NR, int RW>
struct Kv4AttnSmem {
  static constexpr int kTW = 4 / RW;  // warps that share rows
  static constexpr int kBlock = Kv4Layout<D>::kBytes;
  static constexpr int kRing = kTW * kKv4Stages * 2 * kBlock;
  static constexpr int kRegs = NR * D / 4;                           // accumulators of a lane
  static constexpr int kMerge = kTW > 1 ? 4 * 32 * kRegs * 4 : 0;    // each warp's
  // q's operand words are a lane's registers for one tile of rows, in shared memory for two
  static constexpr bool kQInSmem = NR > 1;
  static constexpr int kQ = kRing + kMerge;                                 // [RW][32 lanes][NR D / 8] words
  static constexpr int kMl = kQ + (kQInSmem ? RW * 32 * NR * D / 8 * 4 : 0);  // [4][8 NR] float2
  static constexpr int kBars = kMl + 4 * 8 * NR * 8;                        // full, empty
  static constexpr int kAhead = kBars + 2 * kTW * kKv4Stages * 8;           // [kTW] Kv4Ahead
  static constexpr int kFlags = kAhead + kTW * 80;
  static constexpr int kBytes = kFlags + 16;
  static constexpr int kCtasPerSm = NR == 1 ? 4 : 3;
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

__device__ __forceinline__ uint32_t half2_sum(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// An 8 x 8 matrix of 16-bit values, lane l holding columns 2 (l % 4) and the next of row l / 4, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// A CTA's place on the line: an item and the steps of it that are this CTA's.
struct Kv4Segment {
  int b, tile, head;  // head runs fastest
  int len, steps;     // of sequence b
  int s0, s1;
  int left;           // units of the run behind this segment
};

// The producer's place of a token warp, in shared memory: the segment it is in, its next step there and the end of those that are seen.
struct __align__(16) Kv4Ahead {
  Kv4Segment seg;
  int at, in, col, end;  // the step that is issued next (-1: none), its first block's place in its page, the page's column; the segment's end
  const uint8_t* base;   // the head's blocks of page 0
  const int32_t* pages;  // of the sequence
  int two_end, pad[3];   // steps from here on have one block
};
static_assert(sizeof(Kv4Ahead) == 80, "Kv4AttnSmem::kFlags");

__device__ __forceinline__ int kv4_length(const Kv4AttnParams& p, int b) {
  const int n = p.lengths[b], most = p.table_pages * p.page_blocks * kKv4Block;
  return n < 0 ? 0 : n > most ? most : n;
}

// The next segment of the run, if there is one. STEP: tokens of a step, ITEM: units of the line in front of an item's first step.
template <int STEP, int ITEM>
__device__ __forceinline__ bool kv4_next(const Kv4AttnParams& p, Kv4Segment& s) {
  if (s.left <= ITEM) return false;
  if (++s.head == p.kv_heads) {
    s.head = 0;
    if (++s.tile == p.row_tiles) {
      s.tile = 0;
      do {  // units are left on the line, so a sequence with some follows
        if (++s.b >= p.batch) return false;
        s.len = kv4_length(p, s.b);
      } while (s.len == 0);
      s.steps = (s.len + STEP - 1) / STEP;
    }
  }
  s.s0 = 0;
  s.s1 = min(s.steps, s.left - ITEM);
  s.left -= s.s1 + ITEM;
  return true;
}

// Steps of the segment that some row of its tile sees: [s0, result).
template <int ROWS, int STEP>
__device__ __forceinline__ int kv4_seen(const Kv4AttnParams& p, const Kv4Segment& s) {
  const int last = min(p.rows, (s.tile + 1) * ROWS) - 1;
  const int limit = s.len - p.queries + static_cast<int>(magic_div(last, p.group_magic)) + 1;
  return max(s.s0, min(s.s1, (limit + STEP - 1) / STEP));
}

// This CTA's run of the line and its first segment; false: it has none. For all lanes of each warp.
template <int STEP, int ITEM>
__device__ __forceinline__ bool kv4_start(const Kv4AttnParams& p, int* run, int* count, Kv4Segment* seg) {
  const int lane = threadIdx.x & 31, per = p.kv_heads * p.row_tiles;
  long long total = 0;
  for (int b = lane; b < p.batch; b += 32) {
    const int n = p.lengths[b], len = kv4_length(p, b);
    if (n != len && n > 0 && threadIdx.x < 32 && blockIdx.x == 0) atomicOr(p.status, kStatusPage);
    total += len == 0 ? 0 : (len + STEP - 1) / STEP + ITEM;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= per;
  *run = static_cast<int>(max(static_cast<long long>(p.min_run), (total + gridDim.x - 1) / gridDim.x));
  const long long begin = static_cast<long long>(*run) * blockIdx.x;
  *count = static_cast<int>(max(0ll, min(static_cast<long long>(*run), total - begin)));
  if (*count == 0) return false;
  // The sequence the run begins in: 32 lengths at a time.
  long long before = 0;
  for (int b0 = 0;; b0 += 32) {
    const int b = b0 + lane;
    const int len = b < p.batch ? kv4_length(p, b) : 0, units = len == 0 ? 0 : (len + STEP - 1) / STEP + ITEM;
    long long sum = static_cast<long long>(units) * per;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before + sum > begin);
    if (hit != 0) {  // always, at the latest with the last sequence: begin < total
      const int l = __ffs(hit) - 1;
      seg->b = b0 + l;
      seg->steps = __shfl_sync(0xffffffffu, units, l) - ITEM;
      before += __shfl_sync(0xffffffffu, sum, l) - static_cast<long long>(seg->steps + ITEM) * per;
      break;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
    if (b0 + 32 >= p.batch) return false;
  }
  seg->len = kv4_length(p, seg->b);
  const long long in = begin - before;
  const int item = static_cast<int>(in / (seg->steps + ITEM)), at = static_cast<int>(in - static_cast<long long>(item) * (seg->steps + ITEM));
  seg->tile = item / p.kv_heads;
  seg->head = item - seg->tile * p.kv_heads;
  seg->s0 = max(0, at - ITEM);
  seg->s1 = max(seg->s0, min(seg->steps, at - ITEM + *count));
  seg->left = *count - (seg->s1 + ITEM - at);
  return seg->s1 > seg->s0;  // else the run ends in front of the item's first step
}

// Whether a page lies in the cache; the status says where one does not.
__device__ __forceinline__ bool kv4_page_there(const Kv4AttnParams& p, int page) {
  if (static_cast<uint32_t>(page) < static_cast<uint32_t>(p.pages)) return true;
  atomicOr(p.status, kStatusPage);
  return false;
}
// What stands in shared memory for a block of a page that does not: tokens held as NaN, which show in the rows that see them.
template <int D>
__device__ __forceinline__ void kv4_spoil(uint8_t* block) {
  using L = Kv4Layout<D>;
#pragma unroll 1
  for (int i = 0; i < kKv4Block / 2; ++i) *reinterpret_cast<uint4*>(block + L::kV + i * L::kRowV + D) = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
  fence_proxy_async_smem();  // copies will lie there again
}

// Rows of sequences without tokens are on no CTA's run: they are zeros.
template <typename T, int D>
__device__ __forceinline__ void write_unseen(const Kv4AttnParams& p, int threads) {
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (kv4_length(p, b) != 0) continue;
    const uint32_t rows = static_cast<uint32_t>(p.queries) * p.q_heads;  // below 2^31; their words of 16 bytes may be more
    const int d = 8 * (threadIdx.x % (D / 8));
    for (uint32_t i = threadIdx.x / (D / 8); i < rows; i += threads / (D / 8)) {
      const uint32_t n = i / p.q_heads, h = i - n * p.q_heads;
      *reinterpret_cast<uint4*>(static_cast<T*>(p.o) + b * p.os[0] + n * p.os[1] + h * p.os[2] + d) = make_uint4(0, 0, 0, 0);
    }
  }
}

// Joins the parts of an item, which begins with CTA `first`, and writes `count` of its rows from `row0` on: UNITS float4 of the output at a time, each with PARTS
// parts' loads in flight. The sums are brought to a new maximum when one comes along.
template <typename T, int D, int UNITS, int PARTS>
__device__ __forceinline__ void join_parts(const Kv4AttnParams& p, const Kv4Segment& seg, int rows, int first, int parts, int row0, int count, int thread, int threads) {
  const int units = max(0, min(count, p.rows - seg.tile * rows - row0)) * (D / 4);
  for (int u0 = thread; u0 < units; u0 += UNITS * threads) {
    float most[UNITS], sum[UNITS];
    float4 acc[UNITS];
#pragma unroll
    for (int j = 0; j < UNITS; ++j) most[j] = -INFINITY, sum[j] = 0.f, acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = 0; k0 < parts; k0 += PARTS) {
      float2 v[UNITS][PARTS];
      float4 y[UNITS][PARTS];
#pragma unroll
      for (int j = 0; j < UNITS; ++j) {
        const int u = min(u0 + j * threads, units - 1), row = row0 + u / (D / 4), d = 4 * (u % (D / 4));
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const int k = min(k0 + i, parts - 1);
          const int64_t at = (static_cast<int64_t>(first + k) * 2 + (k == 0 ? 1 : 0)) * rows + row;
          v[j][i] = __ldcg(p.partial_ml + at);
          y[j][i] = __ldcg(reinterpret_cast<const float4*>(p.partial + at * D + d));
          if (k0 + i >= parts) v[j][i] = make_float2(-INFINITY, 0.f);
        }
      }
#pragma unroll
      for (int j = 0; j < UNITS; ++j) {
        float next = most[j];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) next = fmaxf(next, v[j][i].x);
        const float alpha = most[j] == -INFINITY ? (sum[j] == 0.f ? 0.f : 1.f) : exp2_approx(most[j] - next);
        most[j] = next;
        sum[j] *= alpha;
        acc[j].x *= alpha, acc[j].y *= alpha, acc[j].z *= alpha, acc[j].w *= alpha;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
          const float by = v[j][i].x == -INFINITY ? v[j][i].y * 0.f : exp2_approx(v[j][i].x - most[j]);
          if (by != 0.f) {
            sum[j] = fmaf(by, v[j][i].y, sum[j]);
            acc[j].x = fmaf(by, y[j][i].x, acc[j].x);
            acc[j].y = fmaf(by, y[j][i].y, acc[j].y);
            acc[j].z = fmaf(by, y[j][i].z, acc[j].z);
            acc[j].w = fmaf(by, y[j][i].w, acc[j].w);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
      const int u = u0 + j * threads, row = row0 + u / (D / 4), d = 4 * (u % (D / 4));
      if (u >= units) continue;
      const float inv = sum[j] == 0.f ? 0.f : 1.f / sum[j];
      const int at = seg.tile * rows + row, n = static_cast<int>(magic_div(at, p.group_magic)), head = seg.head * p.group + at - n * p.group;
      T* y = static_cast<T*>(p.o) + seg.b * p.os[0] + n * p.os[1] + head * p.os[2] + d;
      *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(acc[j].x * inv, acc[j].y * inv), pack2<T>(acc[j].z * inv, acc[j].w * inv));
    }
  }
}

template <typename T, int D, int NR, int RW>
__global__ void __launch_bounds__(kKv4AttnThreads, Kv4AttnSmem<D, NR, RW>::kCtasPerSm) kv4_attn_kernel(const Kv4AttnParams p) {
  using S = Kv4AttnSmem<D, NR, RW>;
  using L = Kv4Layout<D>;
  constexpr int kTW = S::kTW, kWarpRows = 8 * NR, kRows = kWarpRows * RW;
  constexpr int kWords = D / 32;  // words of codes in a lane, for each token of K and each two of V
  constexpr int kTiles = D / 16;  // row tiles of the output
  constexpr bool kLess8 = std::is_same<T, __half>::value;  // codes of V less 8 in the operands, or 8 p vs summed beside them
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int rw = warp % RW, tw = warp / RW;
  uint8_t* ring = smem + tw * kKv4Stages * 2 * S::kBlock;
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

  write_unseen<T, D>(p, kKv4AttnThreads);
  int run, count;
  Kv4Segment seg{};
  if (!kv4_start<kKv4Step, kKv4Item>(p, &run, &count, &seg)) return;

  // The producer runs kKv4Stages steps ahead, over the ends of items: lane 0 of the first row warp of each token warp.
  const bool producer = rw == 0;
  Kv4Ahead& ahead = *reinterpret_cast<Kv4Ahead*>(smem + S::kAhead + tw * sizeof(Kv4Ahead));
  uint32_t issued = 0, used = 0;  // steps of this token warp, in order
  bool ok = true;
  const bool joined = (p.page_blocks & 1) == 0;  // the blocks of a step follow one another
  const int64_t page_bytes = static_cast<int64_t>(p.kv_heads) * p.page_blocks * S::kBlock;
  int next_page[2] = {0, 0};
  // The pages of step `at` of the producer's segment, so that their load is over when the step is issued.
  const auto fetch = [&](const int32_t* pages, int at, int in, int col, int two_end) {
    next_page[0] = pages[col];
    if (!joined && at < two_end) next_page[1] = pages[in + 1 == p.page_blocks ? col + 1 : col];
  };
  const auto enter = [&](Kv4Segment next) {  // a segment of the producer's, or the first one behind it that has steps for this warp
    int at = next.s0 + tw, end = kv4_seen<kRows, kKv4Step>(p, next);
    while (at >= end) {
      if (!kv4_next<kKv4Step, kKv4Item>(p, next)) {
        ahead.at = -1;
        return;
      }
      at = next.s0 + tw;
      end = kv4_seen<kRows, kKv4Step>(p, next);
    }
    ahead.seg = next;
    ahead.at = at;
    ahead.end = end;
    ahead.col = static_cast<int>(magic_div(2 * at, p.bpp_magic));
    ahead.in = 2 * at - ahead.col * p.page_blocks;
    ahead.base = p.cache + static_cast<int64_t>(next.head) * p.page_blocks * S::kBlock;
    ahead.pages = p.page_table + next.b * p.table_stride;
    ahead.two_end = (next.len + kKv4Block - 1) / kKv4Step;
    fetch(ahead.pages, at, ahead.in, ahead.col, ahead.two_end);
  };
  const int by_col = 2 * kTW / p.page_blocks, by_in = 2 * kTW - by_col * p.page_blocks;
  const auto issue = [&]() {
    const int at = ahead.at;
    if (at < 0) return;
    int in = ahead.in, col = ahead.col;
    const int end = ahead.end, two_end = ahead.two_end;
    const uint8_t* base = ahead.base;
    const uint32_t stage = issued % kKv4Stages, round = issued / kKv4Stages;
    if (RW > 1 && round > 0 && !mbar_wait(empty + stage, (round - 1) & 1, abort_flag)) {
      ahead.at = -1;
      ok = false;
      return;
    }
    const bool two = at < two_end;  // the second block may hold nothing: what lies there is then masked
    uint8_t* to = ring + stage * 2 * S::kBlock;
    const auto block_at = [&](int page, int place) { return base + page * page_bytes + static_cast<int64_t>(place) * S::kBlock; };
    const uint32_t pages = p.pages, page0 = next_page[0], page1 = two && !joined ? next_page[1] : page0;
    const auto load_second = [&]() { bulk_load(to + S::kBlock, block_at(page1, in + 1 == p.page_blocks ? 0 : in + 1), S::kBlock, full + stage); };
    if (page0 < pages && page1 < pages) {
      mbar_arrive_expect_tx(full + stage, two ? 2 * S::kBlock : S::kBlock);
      bulk_load(to, block_at(page0, in), two && joined ? 2 * S::kBlock : S::kBlock, full + stage);
      if (two && !joined) load_second();
    } else {
      atomicOr(p.status, kStatusPage);
      if (page0 >= pages) kv4_spoil<D>(to);
      if (page1 >= pages) kv4_spoil<D>(to + S::kBlock);
      mbar_arrive_expect_tx(full + stage, page0 < pages || page1 < pages ? S::kBlock : 0);
      if (page0 < pages) bulk_load(to, block_at(page0, in), S::kBlock, full + stage);
      if (page1 < pages) load_second();
    }
    ++issued;
    if (at + kTW >= end) {
      Kv4Segment next = ahead.seg;
      if (kv4_next<kKv4Step, kKv4Item>(p, next)) enter(next);
      else ahead.at = -1;
      return;
    }
    in += by_in;
    col += by_col;
    if (in >= p.page_blocks) {
      in -= p.page_blocks;
      ++col;
    }
    ahead.at = at + kTW;
    ahead.in = in;
    ahead.col = col;
    fetch(ahead.pages, at + kTW, in, col, two_end);
  };
  if (producer && lane == 0) {
    enter(seg);
    for (int i = 0; i < kKv4Stages; ++i) issue();
  }
  __syncwarp();

  for (;;) {
    // Row r of each tile of eight: its queries as operand words, in the order of a lane's codes. What belongs to a row of the products
    // is kept by the lanes that hold the products' columns, rows 2 c and 2 c + 1.
    const int row0 = seg.tile * kRows + kWarpRows * rw;
    uint32_t qb[S::kQInSmem ? 1 : NR][4 * kWords];
    uint4* q_smem = reinterpret_cast<uint4*>(smem + S::kQ) + rw * 32 * NR * kWords;  // [NR][kWords][32 lanes]; the warps that share rows write the same
    // off: the maximum that the sums are relative to (log2); limit: logits above need a larger one, -inf: nothing is seen yet.
    float rscale[NR][2], qsum[NR][2], off[NR][2], l[NR][2], ms[NR][2], limit[NR][2];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const int row = min(row0 + 8 * t + r, p.rows - 1);
      const int n = static_cast<int>(magic_div(row, p.group_magic)), g = row - n * p.group;
      const T* x = static_cast<const T*>(p.q) + seg.b * p.qs[0] + n * p.qs[1] + (seg.head * p.group + g) * p.qs[2] + c * (D / 4);
      float most = 0.f;
      Raw8<T> raw[kWords];
#pragma unroll
      for (int w = 0; w < kWords; ++w) raw[w].load(x + 8 * w);
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
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
      for (int w = 0; w < kWords; ++w) {
        float f[8];
        raw[w].unpack(f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          f[k] *= up;
          sum += f[k];
        }
        uint32_t words[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float by = k & 1 ? 0.0625f : 1.f;
          words[k] = pack2<__half>(f[k] * by, f[k + 4] * by);
          if (!S::kQInSmem) qb[S::kQInSmem ? 0 : t][4 * w + k] = words[k];
        }
        if (S::kQInSmem) q_smem[(t * kWords + w) * 32 + lane] = make_uint4(words[0], words[1], words[2], words[3]);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // Logits of this row are in units of 2^(e - 10) 2^24; their factor may be neither 0 (masked logits) nor infinite (zeros).
      const float scale = fminf(fmaxf(p.scale_log2 * pow2(min(e + 14, 127)) * pow2(max(e - 113, 0)), FLT_MIN), FLT_MAX);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int from = 4 * (2 * c + i);
        qsum[t][i] = __shfl_sync(0xffffffffu, sum, from) * 5.9604644775390625e-08f;
        rscale[t][i] = __shfl_sync(0xffffffffu, scale, from);
        limit[t][i] = -INFINITY;
        off[t][i] = l[t][i] = ms[t][i] = 0.f;
      }
    }
    // Position of a row; a row past the last one is taken for it.
    const auto position = [&](int row) { return seg.len - p.queries + static_cast<int>(magic_div(min(row, p.rows - 1), p.group_magic)); };
    const int lowest = position(row0);
    float o[NR][kTiles][4], eights[NR][4];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
      eights[t][0] = eights[t][1] = eights[t][2] = eights[t][3] = 0.f;
    }
    int vexp = -120;     // steps of V are taken times 2^(6 - vexp)
    float vscale = 0.f;  // 2^(6 - vexp); 0: no step seen yet
    float vlimit = 0.f;  // steps from here on need a larger vexp

    const int seen = kv4_seen<kRows, kKv4Step>(p, seg);
#pragma unroll 1
    for (int s = seg.s0 + tw; s < seen; s += kTW) {
      const uint32_t stage = used % kKv4Stages, round = used / kKv4Stages;
      ok = ok && mbar_wait(full + stage, round & 1, abort_flag);  // one that ran out is noticed at the vote below
      const uint8_t* step = ring + stage * 2 * S::kBlock;
      const int base = s * kKv4Step;
      const bool masked = base + kKv4Step - 1 > lowest;
      constexpr int kChains = NR == 1 ? 2 : 1;  // sums of a logit, so that the products do not wait for one another (two tiles are two chains)
      float x[2][NR][4], odd[2][NR][4];  // blocks; tokens r and r + 8, rows 2 c and 2 c + 1
      float vs[2][2], vl[2][2];
      {
        uint32_t w[2][2][kWords];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint8_t* at = step + h * S::kBlock + (8 * k + r) * L::kRowK + c * (D / 8);
            if constexpr (D == 128) {
              const uint4 v = *reinterpret_cast<const uint4*>(at);
              w[h][k][0] = v.x, w[h][k][1] = v.y, w[h][k][2] = v.z, w[h][k][3] = v.w;
            } else {
              const uint2 v = *reinterpret_cast<const uint2*>(at);
              w[h][k][0] = v.x, w[h][k][1] = v.y;
            }
          }
#pragma unroll
          for (int t = 0; t < NR; ++t) {
            x[h][t][0] = x[h][t][1] = x[h][t][2] = x[h][t][3] = 0.f;
            odd[h][t][0] = odd[h][t][1] = odd[h][t][2] = odd[h][t][3] = 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          uint32_t q[NR][4];
#pragma unroll
          for (int t = 0; t < NR; ++t) {
            if constexpr (S::kQInSmem) {
              const uint4 v = q_smem[(t * kWords + i) * 32 + lane];
              q[t][0] = v.x, q[t][1] = v.y, q[t][2] = v.z, q[t][3] = v.w;
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) q[t][k] = qb[t][4 * i + k];
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t u0[4], u1[4];
            split_codes(w[h][0][i], u0);
            split_codes(w[h][1][i], u1);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t a[4] = {u0[2 * k], u1[2 * k], u0[2 * k + 1], u1[2 * k + 1]};
#pragma unroll
              for (int t = 0; t < NR; ++t) mma_16816<__half>(k == 0 || kChains == 1 ? x[h][t] : odd[h][t], a, q[t][2 * k], q[t][2 * k + 1]);
            }
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* block = step + h * S::kBlock;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint2 v = *reinterpret_cast<const uint2*>(block + L::kV + ((8 * k + r) >> 1) * L::kRowV + D + (r & 1) * 8);
          const float ks = __uint_as_float(v.x << 16), kl = __uint_as_float(v.x & 0xffff0000u);
          vs[h][k] = __uint_as_float(v.y << 16);
          vl[h][k] = fmaf(8.f, vs[h][k], __uint_as_float(v.y & 0xffff0000u));
#pragma unroll
          for (int t = 0; t < NR; ++t) {
#pragma unroll
            for (int i = 0; i < 2; ++i) x[h][t][2 * k + i] = fmaf(ks, kChains == 1 ? x[h][t][2 * k + i] : x[h][t][2 * k + i] + odd[h][t][2 * k + i], kl * qsum[t][i]);
          }
        }
      }
      if (masked) {
        // Tokens that a row does not see weigh nothing, whatever they hold; those behind the sequence's end hold whatever the page held.
        // A value that is not finite is put into the logits of the rows that see it, so that it cannot reach the others through 0 * NaN.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int at = base + h * kKv4Block + 8 * k + r;
            const bool spoilt = !(fabsf(vl[h][k]) < INFINITY);
#pragma unroll
            for (int t = 0; t < NR; ++t) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float& y = x[h][t][2 * k + i];
                if (spoilt) y = NAN;
                if (at > position(row0 + 8 * t + 2 * c + i)) y = -INFINITY;
              }
            }
            if (spoilt || at >= seg.len) vs[h][k] = vl[h][k] = 0.f;
          }
        }
      }
      bool raise = !ok;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          raise = raise || vs[h][k] >= vlimit;
#pragma unroll
          for (int t = 0; t < NR; ++t) raise = raise || x[h][t][2 * k] > limit[t][0] || x[h][t][2 * k + 1] > limit[t][1];
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        // New maxima for the rows and for the steps of V. Infinite and NaN steps are left out: they show in the rows that see them.
        float big = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int k = 0; k < 2; ++k) big = fmaxf(big, vs[h][k] < INFINITY ? vs[h][k] : 0.f);
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
        const int e = max(vexp, min(static_cast<int>(__float_as_uint(big) >> 23) - 127, 126));
        const float shrink = e == vexp || vscale == 0.f ? 1.f : pow2(max(vexp - e, -126));
        vexp = e;
        vscale = pow2(6 - e);
        vlimit = e >= 126 ? INFINITY : pow2(e + 1);
#pragma unroll
        for (int t = 0; t < NR; ++t) {
          float alpha[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float most = fmaxf(fmaxf(x[0][t][i], x[0][t][2 + i]), fmaxf(x[1][t][i], x[1][t][2 + i]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            alpha[i] = 0.f;
            if (most != -INFINITY) {
              const float next = limit[t][i] == -INFINITY ? most * rscale[t][i] : fmaxf(off[t][i], most * rscale[t][i]);
              alpha[i] = limit[t][i] == -INFINITY ? 0.f : exp2_approx(off[t][i] - next);
              off[t][i] = next;
              limit[t][i] = (next + 8.f) / rscale[t][i];
            } else if (limit[t][i] != -INFINITY) {
              alpha[i] = 1.f;
            }
            l[t][i] *= alpha[i];
            ms[t][i] *= alpha[i];
            alpha[i] *= shrink;
          }
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            o[t][i][0] *= alpha[0];
            o[t][i][1] *= alpha[1];
            o[t][i][2] *= alpha[0];
            o[t][i][3] *= alpha[1];
          }
          eights[t][0] *= alpha[0];
          eights[t][1] *= alpha[1];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* block = step + h * S::kBlock;
        uint32_t pb[NR][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float by = vs[h][k] * vscale;
#pragma unroll
          for (int t = 0; t < NR; ++t) {
            float e[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float y = x[h][t][2 * k + i];
              const float pk = exp2_approx(fmaf(y, rscale[t][i], -off[t][i]));
              l[t][i] += pk;
              ms[t][i] = fmaf(pk, vl[h][k], ms[t][i]);
              e[i] = pk * by;
            }
            pb[t][k] = transpose_8x8(pack2<__half>(e[0], e[1]));
          }
        }
        uint32_t w0[kWords], w1[kWords];
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
        const uint32_t eight[4] = {0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u};
#pragma unroll
        for (int t = 0; t < NR && !kLess8; ++t) mma_16816<__half>(eights[t], eight, pb[t][0], pb[t][1]);
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          uint32_t u0[4], u1[4];
          split_codes(w0[i], u0);
          split_codes(w1[i], u1);
          if constexpr (kLess8) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // 8 as either nibble has it
              u0[k] = half2_sum(u0[k], k & 1 ? 0x80808080u : 0x80088008u);
              u1[k] = half2_sum(u1[k], k & 1 ? 0x80808080u : 0x80088008u);
            }
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t a[4] = {u0[2 * k], u0[2 * k + 1], u1[2 * k], u1[2 * k + 1]};
#pragma unroll
            for (int t = 0; t < NR; ++t) mma_16816<__half>(o[t][2 * i + k], a, pb[t][0], pb[t][1]);
          }
        }
      }
      __syncwarp();
      ++used;
      if (RW > 1 && lane == 0) mbar_arrive(empty + stage);
      if (producer && lane == 0) issue();
      __syncwarp();
    }
    if (!ok && lane == 0 && atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0) atomicOr(p.status, kStatusKv4Wait);

    // This warp's sums over its lanes, and the output itself: (codes' part * 2^24 (2^20 for odd nibbles) - eights * 2^24) / vscale + ms.
    // A maximum of -inf with a sum that is not zero is one of NaN logits alone: it weighs NaN.
    const float unit = pow2(vexp - 6);
    constexpr float kCode = 16777216.f, kHighCode = 1048576.f;
    float mt[NR][2], lt[NR][2], weight[kTW][NR][2];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], d);
          ms[t][i] += __shfl_xor_sync(0xffffffffu, ms[t][i], d);
        }
        mt[t][i] = limit[t][i] == -INFINITY ? limit[t][i] : off[t][i];
        lt[t][i] = l[t][i];
#pragma unroll
        for (int q = 0; q < kTiles; ++q) {
          o[t][q][i] = fmaf(fmaf(o[t][q][i], kCode, -kCode * eights[t][i]), unit, ms[t][i]);
          o[t][q][2 + i] = fmaf(fmaf(o[t][q][2 + i], kHighCode, -kCode * eights[t][i]), unit, ms[t][i]);
        }
      }
    }
    if constexpr (kTW > 1) {
      float* mine = merge + warp * 32 * S::kRegs;
#pragma unroll
      for (int t = 0; t < NR; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int q = 0; q < 2 * kTiles; ++q) mine[((2 * t + i) * 2 * kTiles + q) * 32 + lane] = o[t][q >> 1][2 * (q & 1) + i];
          if (r == 0) ml_smem[warp * kWarpRows + 8 * t + 2 * c + i] = make_float2(mt[t][i], lt[t][i]);
        }
      }
    }
    __syncthreads();
    const bool gone = *abort_flag != 0;
    if (kTW > 1 && !gone) {
#pragma unroll
      for (int t = 0; t < NR; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float2 v[kTW];
          mt[t][i] = -INFINITY;
          lt[t][i] = 0.f;
#pragma unroll
          for (int k = 0; k < kTW; ++k) {
            v[k] = ml_smem[(k * RW + rw) * kWarpRows + 8 * t + 2 * c + i];
            mt[t][i] = fmaxf(mt[t][i], v[k].x);
          }
#pragma unroll
          for (int k = 0; k < kTW; ++k) {
            weight[k][t][i] = v[k].x == -INFINITY ? v[k].y * 0.f : exp2_approx(v[k].x - mt[t][i]);
            lt[t][i] = fmaf(weight[k][t][i], v[k].y, lt[t][i]);
          }
        }
      }
    }
    // Whole items go out; parts go to the workspace and are counted. A lane has dimensions r D / 8 + q of rows 2 c + i of each tile;
    // four at a time, dealt to the warps that share the rows.
    const bool whole = seg.s1 - seg.s0 == seg.steps;
    const int slot = blockIdx.x * 2 + (seg.s0 > 0 ? 0 : 1);
    if (!gone) {
#pragma unroll
      for (int t = 0; t < NR; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int in_tile = kWarpRows * rw + 8 * t + 2 * c + i, row = seg.tile * kRows + in_tile;
          const float inv = lt[t][i] == 0.f ? 0.f : 1.f / lt[t][i];
          const int n = static_cast<int>(magic_div(row, p.group_magic)), head = seg.head * p.group + row - n * p.group;
#pragma unroll
          for (int q4 = 0; q4 < kTiles / 2; ++q4) {
            if (kTW > 1 && ((2 * t + i) * (kTiles / 2) + q4) % kTW != tw) continue;
            float f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int q = 4 * q4 + k;
              if constexpr (kTW > 1) {
                float v = 0.f;
#pragma unroll
                for (int j = 0; j < kTW; ++j) {
                  const float part = merge[(j * RW + rw) * 32 * S::kRegs + ((2 * t + i) * 2 * kTiles + q) * 32 + lane];
                  v = weight[j][t][i] == 0.f ? v : fmaf(weight[j][t][i], part, v);
                }
                f[k] = v;
              } else {
                f[k] = o[t][q >> 1][2 * (q & 1) + i];
              }
            }
            if (row >= p.rows) continue;
            const int d = r * (D / 8) + 4 * q4;
            if (whole) {
#pragma unroll
              for (int k = 0; k < 4; ++k) f[k] = lt[t][i] == 0.f ? 0.f : f[k] * inv;
              T* y = static_cast<T*>(p.o) + seg.b * p.os[0] + n * p.os[1] + head * p.os[2] + d;
              *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]));
            } else {
              __stcg(reinterpret_cast<float4*>(p.partial + (static_cast<int64_t>(slot) * kRows + in_tile) * D + d), make_float4(f[0], f[1], f[2], f[3]));
              if (r == 0 && q4 == 0) __stcg(p.partial_ml + static_cast<int64_t>(slot) * kRows + in_tile, make_float2(mt[t][i], lt[t][i]));
            }
          }
        }
      }
    }
    if (!whole && !gone) {
      const long long item = static_cast<long long>(run) * blockIdx.x + count - seg.left - seg.s1;  // where its steps begin on the line
      const int first = static_cast<int>(item / run), parts = static_cast<int>((item + seg.steps - 1) / run) - first + 1;
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) *last_flag = atomicAdd(p.counters + first, 1u) == static_cast<uint32_t>(parts - 1) ? 1u : 0u;
      __syncthreads();
      if (*last_flag != 0) {
        __threadfence();
        join_parts<T, D, 1, 8>(p, seg, kRows, first, parts, 0, kRows, threadIdx.x, kKv4AttnThreads);
        if (threadIdx.x == 0) p.counters[first] = 0;
      }
    }
    __syncthreads();  // merge buffer and flags
    if (gone) break;
    if (!kv4_next<kKv4Step, kKv4Item>(p, seg)) break;
  }
  // A wait that ran out leaves copies in flight: they are waited for, again with a limit, before the shared memory goes.
  if (*abort_flag != 0 && producer && lane == 0) {
    for (; used < issued; ++used) mbar_wait(full + used % kKv4Stages, (used / kKv4Stages) & 1, abort_flag + 2);
  }
}

}  // namespace b200
