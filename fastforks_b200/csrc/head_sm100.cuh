// The output layer of a model and its loss, on sm_100a, without the logits. For rows x [T, D], a weight w [V, D] and logits l = x w^T (+ bias [V]):
//
//   cross entropy   loss_t = lse(l_t) - l_t,y                                    dl_t = g_t (softmax(l_t) - onehot_y)
//   distillation    loss_t = tau^2 sum_k p_k (log p_k - z_t,id(k) + lse(z_t))    dl_t = g_t tau (softmax(z_t) - sum_k p_k onehot_id(k))
//                   z = l / tau, p = softmax of the teacher's logits / tau over the row's entries
//   dx = dl w,  dw = dl^T x,  dbias = sum_t dl_t
//
// Cross entropy is the second form with one entry of weight 1 and tau = 1; the kernels know that form alone. Rows that do not count (no
// target, no entry) are left out of every product: where there are any, the others are copied together (head_rows_kernel) and the
// row tiles are counted on the device.
//
//   head_entries_kernel  distillation: a row's p, its entropy, its entries in order of their tokens
//   head_count_kernel    many rows: how many of each CTA's count
//   head_rows_kernel     which rows count, where they go, their copy
//   head_stats_kernel    logits of 256 x bn tiles in tensor memory; leaves a maximum and a sum of exponentials per row and half
//                        of a tile's columns, and the logits of the row's entries
//   head_few_kernel      the same of up to 64 rows
//   head_loss_kernel     joins those to lse and loss (head_loss_many_kernel, where a row has little to join)
//   head_coef_kernel     gradients that differ from row to row: one power of two for all
//   head_grads_kernel    a piece of the vocabulary: the logits again, their gradient in 16 bits
//   head_sums_kernel     dx += G w and dw = G^T x of that piece in one launch
//   head_db_kernel       dbias of that piece
//   head_dx_kernel       sums of dx (and of dw in parts), which are held in fp32, rounded; rows of dx put where they came from
//
// Bound by the tensor cores: 2 T D V operations forward, 6 T D V more for the gradients, 2 T D V of which compute the logits again
// instead of keeping them. The products are those of CTA pairs (cta_group::2, plain TMA loads, 256 x 256 tiles, two accumulators
// in tensor memory); head_products() below is the one pipeline that statistics, gradients of logits and sums run on.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstddef>
#include <type_traits>

#include "gemm_sm100.cuh"
#include "sm100_ptx.cuh"

namespace b200 {

constexpr uint32_t kStatusTarget = 1u << 23, kStatusHeadWait = 1u << 24;
constexpr int kHeadThreads = 320;  // warp 0 loader, warp 1 MMA, warps 2..9 epilogue
constexpr int kHeadRingBytes = 160 * 1024, kHeadMaxStages = 8;
constexpr int kHeadChunkBytes = 4096;  // what an epilogue warp stages at a time: 32 rows of 128 bytes
constexpr int kHeadBlock = 64 * 64 * 2;  // 64 values of the contiguous axis by 64 of k, an operand whose k is not contiguous
constexpr int kNoEntry = 0x7fffffff;

struct HeadSmem {
  alignas(1024) uint8_t ring[kHeadRingBytes];          // per stage: A, 16 KB, then B
  alignas(1024) uint8_t stage[8][2][kHeadChunkBytes];  // per epilogue warp, two deep
  uint64_t full[kHeadMaxStages];   // the leader's: both CTAs' tiles of the stage have landed  (TMA of both CTAs)
  uint64_t empty[kHeadMaxStages];  // the stage has been read by its products                  (MMA commit, both CTAs)
  uint64_t acc_full[2];            // accumulator finished                                     (MMA commit, both CTAs)
  uint64_t acc_empty[2];           // the leader's: read by the epilogue warps of both CTAs    (16 warps)
  uint64_t drain;                  // abort path: the leader's products have finished          (MMA commit, both CTAs)
  uint32_t tmem_base;
  uint32_t abort;
};
constexpr int kHeadBarriers = 2 * kHeadMaxStages + 2 + 2 + 1;
static_assert(offsetof(HeadSmem, drain) == offsetof(HeadSmem, full) + (kHeadBarriers - 1) * sizeof(uint64_t), "the set-up walks the barriers as one array");
static_assert(sizeof(HeadSmem) + 1024 <= 227 * 1024, "shared memory of one CTA");

// One tile of a product: rows row0 .. row0 + 255 of A, columns of B from col0 on, k-blocks kb0 .. kb1 - 1.
struct HeadItem {
  int kind, slot;
  int row0, col0;
  int kb0, kb1;
};

// k-blocks of an accumulator of logits. The tensor cores cut off what of a product lies below the last place of the running sum: over 4096
// products the loss of 64 rows came out 2.1e-6 off (products and sums in fp32 arithmetic: 3.7e-7). Longer sums are taken 1024 products at a
// time and added in fp32, which rounds: 4.7e-7. The accumulators alternate as they do between tiles, so the epilogue's additions run under
// the next products (4096 x 128000 x 4096: 2570 us; one accumulator, as in head_grads_kernel, 2546). 512 at a time halve the error once more and cost up to 6 %
// of a loss with its gradients (4096 x 64000 x 2048, rows that count 3/4: 2330 -> 2469 us), 256 up to 15 %.
constexpr int kHeadSumBlocks = 16;

// The pipeline of gemm_pair_kernel with the operands' layouts, the list of tiles and the epilogue left to `job`:
//   begin()                      reads what only the kernels in front know (after the wait for them)
//   items(pair), item(pair, i)   this pair's tiles, the same for both CTAs and all warps
//   stages(), stage_bytes()      the ring
//   bytes(t), load(t, kb, ...)   one k-block of either CTA's A and B
//   idesc(t), a_desc(), b_desc(), a_step(t), b_step(t)   what the products take; steps: 16 k-values on, in units of 16 bytes
//   Epilogue e(job, ...); e.ask(t); e.take(t, acc, hand_back)   by each epilogue warp: before the wait for the accumulator, and after it.
//                                `hand_back` is called once per tile, when the warp has read all it needs of the accumulator
template <typename Job>
__device__ __forceinline__ void head_products(Job& job, HeadSmem& sm, uint32_t* status) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_cta_rank()), pair = blockIdx.x >> 1;

  if (warp == 0) {
    uint64_t* const first = &sm.full[0];
    for (int i = lane; i < kHeadBarriers; i += 32) mbar_init(first + i, first + i == &sm.acc_empty[0] || first + i == &sm.acc_empty[1] ? 16 : 1);
    if (lane == 0) sm.abort = 0;
    mbar_init_fence();
    __syncwarp();
  }
  cluster_arrive_relaxed();
  if (warp == 0) {
    named_barrier_arrive(1, kHeadThreads);
  } else {
    if (warp == 1) {
      tmem_alloc_pair(&sm.tmem_base, 512);
      tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    named_barrier_sync(1, kHeadThreads);
    tc_fence_after_sync();
  }
  cluster_wait();  // the other CTA's barriers exist before anything of this one reaches for them
  const uint32_t tmem = sm.tmem_base;  // (not the loader's)
  volatile uint32_t* abort_flag = &sm.abort;
  const int stages = job.stages();
  const uint32_t stage_size = job.stage_bytes();

  if (warp == 0) {
    // ======================= loader (the whole warp, one lane issues) =================================
    grid_dependency_wait();
    job.begin();
    const int n = job.items(pair);
    bool ok = true;
    int g = 0, st = 0;
    uint32_t ph = 1;  // parity of the empty barriers: a ring that was never used is empty
    for (int i = 0; i < n && ok; ++i) {
      const HeadItem t = job.item(pair, i);
      const uint32_t bytes = job.bytes(t);
      for (int kb = t.kb0; kb < t.kb1; ++kb, ++g) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sm.empty[st], ph, abort_flag));
        if (!ok) break;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(&sm.full[st], bytes);
          job.load(t, kb, rank, sm.ring + st * stage_size, cluster_map(smem_u32(&sm.full[st]), 0));  // both CTAs count on the leader's barrier
        }
        if (++st == stages) {
          st = 0;
          ph ^= 1;
        }
      }
    }
    if (!ok && lane == 0 && atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0) atomicOr(status, kStatusHeadWait);
    if (__any_sync(0xffffffffu, *abort_flag != 0) && rank == 0) {  // let every copy that was issued land
      uint32_t no_abort = 0;
      for (int j = (g > stages ? g - stages : 0); j < g; ++j) mbar_wait(&sm.full[j % stages], (j / stages) & 1, &no_abort);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ======================= MMA issuer (leader only) =================================================
    // The next kernel may start from here on: this warp's CTA holds its tensor memory.
    grid_dependency_wait();
    grid_launch_dependents();
    if (rank == 0) {
      job.begin();
      const int n = job.items(pair);
      bool ok = true;
      int st = 0, it = 0;
      uint32_t ph = 0;
      bool landed = false;
      for (; it < n && ok; ++it) {
        const HeadItem t = job.item(pair, it);
        if (it >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&sm.acc_empty[it & 1], ((it >> 1) - 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t acc = tmem + (it & 1) * 256, idesc = job.idesc(t);
        const uint64_t a0 = job.a_desc(t, smem_u32(sm.ring)), b0 = job.b_desc(t, smem_u32(sm.ring) + kGemmTileBytes);
        const int a_step = job.a_step(t), b_step = job.b_step(t);
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          ok = __all_sync(0xffffffffu, landed || mbar_wait(&sm.full[st], ph, abort_flag));
          if (!ok) break;
          tc_fence_after_sync();
          const int next = st + 1 == stages ? 0 : st + 1;
          const uint32_t next_ph = st + 1 == stages ? ph ^ 1 : ph;
          landed = mbar_test_wait(&sm.full[next], next_ph);
          const uint64_t a = a0 + static_cast<uint64_t>(st) * (stage_size >> 4);
          const uint64_t b = b0 + static_cast<uint64_t>(st) * (stage_size >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kGemmBK / 16; ++kk) umma_ss_pair(acc, a + kk * a_step, b + kk * b_step, idesc, (kb != t.kb0 || kk != 0) ? 1u : 0u);
            umma_commit_pair(&sm.empty[st]);
            if (kb == t.kb1 - 1) umma_commit_pair(&sm.acc_full[it & 1]);
          }
          st = next;
          ph = next_ph;
        }
      }
      // The other CTA's epilogue warps signal `acc_empty` here: those of the last two items are waited for by nobody else.
      if (ok) ok = __all_sync(0xffffffffu, lane >= min(it, 2) || mbar_wait(&sm.acc_empty[lane], ((it - 1 - lane) / 2) & 1, abort_flag));
      if (!ok && lane == 0 && atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0) atomicOr(status, kStatusHeadWait);
      if (__any_sync(0xffffffffu, *abort_flag != 0)) {  // no product may be running when tensor memory is freed
        uint32_t no_abort = 0;
        if (elect_one()) umma_commit_pair(&sm.drain);
        mbar_wait(&sm.drain, 0, &no_abort);
      }
    }
    __syncwarp();
  } else {
    // ======================= epilogue warps ==========================================================
    grid_dependency_wait();
    job.begin();
    const int n = job.items(pair);
    const int e = warp - 2, part = e >> 2, quarter = warp & 3;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t acc_empty_at[2] = {cluster_map(smem_u32(&sm.acc_empty[0]), 0), cluster_map(smem_u32(&sm.acc_empty[1]), 0)};
    typename Job::Epilogue epilogue(job, smem_u32(sm.stage[e][0]), sm.stage[e][0], rank * 128 + quarter * 32, part);
    bool ok = true;
    for (int it = 0; it < n; ++it) {
      const HeadItem t = job.item(pair, it);
      epilogue.ask(t);
      if (!__all_sync(0xffffffffu, mbar_wait(&sm.acc_full[it & 1], (it >> 1) & 1, abort_flag))) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      epilogue.take(t, tmem + lane_addr + (it & 1) * 256, [&] {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc_empty_at[it & 1]);
      });
    }
    if (!ok && lane == 0 && atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0) atomicOr(status, kStatusHeadWait);
    if (lane == 0) tma_store_wait_read<0>();
    __syncwarp();
  }

  tc_fence_before_sync();
  __syncthreads();
  // Neither CTA goes while the other may still multiply into its tensor memory or signal its barriers; see gemm_pair_kernel.
  cluster_arrive_relaxed();
  cluster_wait();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem, 512);
  }
}

// The map of tiles to an order in which what runs at the same time shares operands: groups of `group` row tiles, rows fastest.
__device__ __forceinline__ void head_raster(int tile, int tiles_m, int tiles_n, int group, int* tm, int* tn) {
  const int per_group = group * tiles_n, g = tile / per_group, in = tile - g * per_group;
  const int rows = min(group, tiles_m - g * group);
  *tn = in / rows;
  *tm = g * group + (in - *tn * rows);
}

// A tile of shared memory added to global memory (fp32); one launch adds to a place once, so the order is that of the launches.
__device__ __forceinline__ void head_tma_add_2d(const CUtensorMap* map, const void* smem_src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
               :
               : "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(smem_src)), "r"(x), "r"(y)
               : "memory");
}

__device__ __forceinline__ float head_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- logits: statistics, and gradients -------------------------------------------------------------------------------------------
struct HeadLogitsParams {
  const int* count;     // rows that count
  const int* idx;       // [count]: which row of the caller's each is; what is indexed by rows below is by the caller's
  int all_rows;         // rows of the caller
  int dim, vocab;
  int v0, tiles_n;      // first column and column tiles of this launch
  int bn, stages, group;
  int top;              // entries of a row
  const int* ids;       // [all_rows, top], ascending, kNoEntry behind the last
  const float* p;       // [all_rows, top] their weights, or null: 1
  float log2_scale;     // log2(e) / tau
  const void* bias;     // [vocab] or null
  // statistics
  float2* parts;        // [2 tiles_n][parts_stride]: maximum of z in units of ln 2, and the sum of 2^(z - maximum)
  int64_t parts_stride;
  float* picks;         // [all_rows, top]: logits of the entries
  // gradients
  const float* lse2;    // [all_rows], in units of ln 2
  const float* coef;    // [all_rows] or null: 1
  float g_scale;        // a power of two
  int rest_at;          // G's row where what its rounding took is kept, or 0: it is not
  uint32_t* status;
};

// Adds the bias of 32 columns from `base` on, a multiple of 32: the same for all lanes.
template <typename T>
__device__ __forceinline__ void head_add_bias(float (&v)[32], const void* bias, int base, int vocab) {
  const T* const b = static_cast<const T*>(bias) + base;
  if (base + 32 <= vocab) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(b) + q);
      const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = gemm_unpack2<T>(words[i]);
        v[8 * q + 2 * i] += f.x;
        v[8 * q + 2 * i + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (base + i < vocab) v[i] += static_cast<float>(b[i]);
  }
}

// G = 2^s coef_t (softmax(z_t) - p) is held in 16 bits, the operands' type: off by half a step at most, 2^-8 of a value (fp16 2^-11). s = 15 for
// fp16, whose smallest normal number is 2^-14: a softmax of 2^-29 keeps all its bits; bfloat16 has fp32's range, s = 0. Over many rows that adds up to 1.1 to 1.45 times the error that
// the results' own rounding has; of a few rows each hangs on one or two roundings, and 1.7 times came out. Few rows and small products (head_grad_work in
// b200_training.cu), and all others where the caller asks for it, therefore keep what the rounding took, in as many rows more, and both go through the
// products: the error is that of the results' rounding.
template <typename T, bool GRADS>
struct HeadLogitsJob {
  const HeadLogitsParams& p;
  const CUtensorMap *x, *x_copy, *w, *g;
  int rows, tiles_m, k_blocks, sums;  // sums: accumulators of a tile, one after the other

  __device__ __forceinline__ HeadLogitsJob(const HeadLogitsParams& p_, const CUtensorMap* x_, const CUtensorMap* xc, const CUtensorMap* w_, const CUtensorMap* g_)
      : p(p_), x(x_), x_copy(xc), w(w_), g(g_), rows(0), tiles_m(0), k_blocks((p_.dim + kGemmBK - 1) / kGemmBK), sums(GRADS ? 1 : (k_blocks + kHeadSumBlocks - 1) / kHeadSumBlocks) {}
  __device__ __forceinline__ void begin() {
    rows = __ldg(p.count);
    tiles_m = (rows + 255) >> 8;
    if (rows < p.all_rows) x = x_copy;
  }
  __device__ __forceinline__ int items(int pair) const {
    const int tiles = tiles_m * p.tiles_n, pairs = gridDim.x >> 1;
    return tiles > pair ? (tiles - pair + pairs - 1) / pairs * sums : 0;
  }
  __device__ __forceinline__ HeadItem item(int pair, int i) const {
    int tm, tn, part = 0;
    if (!GRADS && sums > 1) {
      part = i % sums;
      i /= sums;
    }
    head_raster(pair + i * (gridDim.x >> 1), tiles_m, p.tiles_n, min(p.group, tiles_m), &tm, &tn);
    return {0, tn, tm * 256, p.v0 + tn * p.bn, k_blocks * part / sums, k_blocks * (part + 1) / sums};
  }
  __device__ __forceinline__ int stages() const { return p.stages; }
  __device__ __forceinline__ uint32_t stage_bytes() const { return kGemmTileBytes + static_cast<uint32_t>(p.bn) * kGemmBK; }
  __device__ __forceinline__ uint32_t bytes(const HeadItem&) const { return 2u * stage_bytes(); }
  __device__ __forceinline__ void load(const HeadItem& t, int kb, int rank, uint8_t* at, uint32_t bar) const {
    tma_load_2d_pair(at, x, bar, kb * kGemmBK, t.row0 + rank * 128);
    tma_load_2d_pair(at + kGemmTileBytes, w, bar, kb * kGemmBK, t.col0 + rank * (p.bn >> 1));
  }
  __device__ __forceinline__ uint32_t idesc(const HeadItem&) const {
    return umma_idesc_f16(std::is_same<T, __half>::value ? UMMA_F16 : UMMA_BF16, 256, p.bn, 0, 0);
  }
  __device__ __forceinline__ uint64_t a_desc(const HeadItem&, uint32_t at) const { return umma_smem_desc_sw128(at, 1024, 16); }
  __device__ __forceinline__ uint64_t b_desc(const HeadItem&, uint32_t at) const { return umma_smem_desc_sw128(at, 1024, 16); }
  __device__ __forceinline__ int a_step(const HeadItem&) const { return 2; }
  __device__ __forceinline__ int b_step(const HeadItem&) const { return 2; }

  // A thread has a row, a warp every second 64 columns of it.
  struct Epilogue {
    const HeadLogitsJob& job;
    const uint32_t stage;
    uint8_t* const stage_ptr;
    const int row_in, part, lane;
    int row, src;     // this thread's row of the product, and of the caller
    int next, pos;    // the row's first entry that has not been passed: its token, its place
    float lse2, coef;
    int buf;
    float sum[GRADS ? 1 : 64];  // the accumulators of a tile so far, where there are several: of the first 64 columns; the others' are staged

    __device__ __forceinline__ Epilogue(const HeadLogitsJob& j, uint32_t s, uint8_t* sp, int r, int pt)
        : job(j), stage(s), stage_ptr(sp), row_in(r), part(pt), lane(threadIdx.x & 31), row(0), src(-1), next(kNoEntry), pos(0), lse2(0.f), coef(0.f), buf(0) {}

    __device__ __forceinline__ int entry(int at) const { return at < job.p.top ? __ldg(job.p.ids + static_cast<int64_t>(src) * job.p.top + at) : kNoEntry; }

    __device__ __forceinline__ void ask(const HeadItem& t) {
      const HeadLogitsParams& p = job.p;
      if (t.kb1 < job.k_blocks) return;  // the last accumulator of a tile is asked for
      row = t.row0 + row_in + lane;
      src = row < job.rows ? __ldg(p.idx + row) : -1;
      next = kNoEntry;
      pos = 0;
      if (src < 0) return;
      int hi = p.top;  // the first entry that is not in front of the tile
      if (p.top > 1) {
        while (pos < hi) {
          const int mid = (pos + hi) >> 1;
          if (entry(mid) < t.col0) pos = mid + 1;
          else hi = mid;
        }
      }
      next = entry(pos);
      if (p.top == 1 && next < t.col0) next = kNoEntry;
      if constexpr (GRADS) {
        lse2 = __ldg(p.lse2 + src);
        coef = p.coef != nullptr ? __ldg(p.coef + src) * p.g_scale : p.g_scale;
      }
    }

    // This thread's sums of 32 columns in the warp's staging area: sixteen bytes of every lane side by side, 512 to the next sixteen.
    __device__ __forceinline__ uint32_t staged(int which) const { return stage + which * kHeadChunkBytes + lane * 16; }
    __device__ __forceinline__ void add_staged(float (&v)[32], int which) const {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const uint4 had = ld_shared_v4(staged(which) + q * 512);
        v[4 * q] += __uint_as_float(had.x);
        v[4 * q + 1] += __uint_as_float(had.y);
        v[4 * q + 2] += __uint_as_float(had.z);
        v[4 * q + 3] += __uint_as_float(had.w);
      }
    }

    // f(j, entry) for the row's entries among the 32 columns from `base` on. Entries of the other warp's columns are passed over.
    template <typename F>
    __device__ __forceinline__ void for_entries(int base, F&& f) {
      while (__any_sync(0xffffffffu, next < base + 32)) {
        if (next < base + 32) {
          if (next >= base) f(next - base, static_cast<int64_t>(src) * job.p.top + pos);
          next = entry(++pos);
        }
      }
    }

    template <typename HandBack>
    __device__ __forceinline__ void take(const HeadItem& t, uint32_t acc, HandBack&& hand_back) {
      const HeadLogitsParams& p = job.p;
      const int pieces = p.bn >> 6;
      if constexpr (!GRADS) {
        if (t.kb1 < job.k_blocks) {
#pragma unroll 1
          for (int c = part; c < pieces; c += 2) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float v[32];
              tmem_ld_x32(acc + c * 64 + half * 32, reinterpret_cast<uint32_t*>(v));
              if (c == part) {
#pragma unroll
                for (int j = 0; j < 32; ++j) sum[half * 32 + j] = t.kb0 == 0 ? v[j] : sum[half * 32 + j] + v[j];
              } else {
                if (t.kb0 > 0) add_staged(v, half);
                const uint32_t at = staged(half);
#pragma unroll
                for (int q = 0; q < 8; ++q)
                  st_shared_v4(at + q * 512, make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]), __float_as_uint(v[4 * q + 3])));
              }
            }
          }
          hand_back();
          return;
        }
        float m = -INFINITY, s = 0.f;
#pragma unroll 1
        for (int c = part; c < pieces; c += 2) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int base = t.col0 + c * 64 + half * 32;
            if (base >= p.vocab) continue;
            float v[32];
            tmem_ld_x32(acc + c * 64 + half * 32, reinterpret_cast<uint32_t*>(v));
            if (t.kb0 > 0) {
              if (c == part) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] += sum[half * 32 + j];
              } else {
                add_staged(v, half);
              }
            }
            if (p.bias != nullptr) head_add_bias<T>(v, p.bias, base, p.vocab);
            for_entries(base, [&](int j, int64_t at) {
              float got = 0.f;
#pragma unroll
              for (int i = 0; i < 32; ++i) got = i == j ? v[i] : got;
              p.picks[at] = got;
            });
            if (base + 32 > p.vocab) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = base + i < p.vocab ? v[i] : -INFINITY;
            }
            float top = v[0];
#pragma unroll
            for (int i = 1; i < 32; ++i) top = fmaxf(top, v[i]);
            const float m_new = fmaxf(m, top * p.log2_scale), from = m_new == -INFINITY ? 0.f : m_new;
            const float2 scale2 = make_float2(p.log2_scale, p.log2_scale), from2 = make_float2(-from, -from);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 z = ffma2(make_float2(v[i], v[i + 1]), scale2, from2);
              sum = fadd2(sum, make_float2(head_ex2(z.x), head_ex2(z.y)));
            }
            s = s * head_ex2(m - from) + (sum.x + sum.y);
            m = m_new;
          }
        }
        hand_back();
        if (row < job.rows) p.parts[(2 * t.slot + part) * p.parts_stride + row] = make_float2(m, s);
      } else {
        const bool partial = t.row0 + row_in + 32 > job.rows;  // rows behind the last are zeros: the products over rows read them
#pragma unroll 1
        for (int c = part; c < pieces; c += 2) {
          const int col = t.col0 + c * 64;
          const bool here = col < p.vocab;
          if (lane == 0) {  // the store that used this buffer last has read it
            if (p.rest_at > 0) tma_store_wait_read<0>();
            else tma_store_wait_read<1>();
          }
          __syncwarp();
          if (here) {
            const uint32_t at_row = stage + buf * kHeadChunkBytes + lane * 128, at_rest = stage + (buf ^ 1) * kHeadChunkBytes + lane * 128;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int base = col + half * 32;
              float v[32];
              tmem_ld_x32(acc + c * 64 + half * 32, reinterpret_cast<uint32_t*>(v));
              if (p.bias != nullptr && base < p.vocab) head_add_bias<T>(v, p.bias, base, p.vocab);
              const float2 scale2 = make_float2(p.log2_scale, p.log2_scale), from2 = make_float2(-lse2, -lse2), coef2 = make_float2(coef, coef);
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const float2 z = ffma2(make_float2(v[i], v[i + 1]), scale2, from2);
                v[i] = head_ex2(z.x);
                v[i + 1] = head_ex2(z.y);
              }
              for_entries(base, [&](int j, int64_t at) {
                const float weight = p.p != nullptr ? __ldg(p.p + at) : 1.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] -= i == j ? weight : 0.f;
              });
              if (base + 32 > p.vocab) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = base + i < p.vocab ? v[i] : 0.f;
              }
              uint32_t out[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 y = fmul2(make_float2(v[2 * i], v[2 * i + 1]), coef2);
                out[i] = gemm_pack2<T>(y.x, y.y);
              }
              if (partial) {
#pragma unroll
                for (int i = 0; i < 16; ++i) out[i] = row < job.rows ? out[i] : 0u;
              }
#pragma unroll
              for (int q = 0; q < 4; ++q)
                st_shared_v4(at_row + (((4 * half + q) ^ (lane & 7)) << 4), make_uint4(out[4 * q], out[4 * q + 1], out[4 * q + 2], out[4 * q + 3]));
              if (p.rest_at > 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float2 y = fmul2(make_float2(v[2 * i], v[2 * i + 1]), coef2), held = gemm_unpack2<T>(out[i]);
                  // (what is not finite has no rest: it is whole already)
                  const float2 rest = make_float2(isfinite(held.x) ? y.x - held.x : 0.f, isfinite(held.y) ? y.y - held.y : 0.f);
                  out[i] = row < job.rows ? gemm_pack2<T>(rest.x, rest.y) : 0u;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  st_shared_v4(at_rest + (((4 * half + q) ^ (lane & 7)) << 4), make_uint4(out[4 * q], out[4 * q + 1], out[4 * q + 2], out[4 * q + 3]));
              }
            }
            fence_proxy_async_smem();
          }
          if (c + 2 >= pieces) hand_back();
          else __syncwarp();
          if (lane == 0) {
            if (here) tma_store_2d(job.g, stage_ptr + buf * kHeadChunkBytes, col - p.v0, t.row0 + row_in);
            if (here && p.rest_at > 0) tma_store_2d(job.g, stage_ptr + (buf ^ 1) * kHeadChunkBytes, col - p.v0, p.rest_at + t.row0 + row_in);
            tma_store_commit();
          }
          buf ^= 1;
        }
        if (part >= pieces) hand_back();
      }
    }
  };
};

// ---- logits of few rows: statistics ----------------------------------------------------------------------------------------------------
// Up to 64 rows leave most of a 256 x 256 tile of the pairs empty and its tiles unevenly dealt, where only the weight's way from HBM counts. Here the
// vocabulary is the M side: a CTA takes `height` rows of w, at most 128 and such that every SM gets the same number of tiles, against all rows of x (N, a
// multiple of 16). Sums of products go to several accumulators side by side in tensor memory (few_plan in b200_training.cu). A warp of the epilogue has 32 rows
// of w; it turns 32 x 32 logits through shared memory, after which a lane has a row of x. us of a loss, by pairs -> here: 1 x 32000 x 4096 79.6 -> 56.9 (the
// weight alone 40.1), 16 rows 61.9 -> 55.3, 64 rows 64.7 -> 61.1, 64 x 128000 x 4096 206 -> 190 (160), 1 x 1000 x 768 13.4 -> 12.2; but of 128 rows 62.9 and
// 64.9, of 256 x 32000 x 2048 38.5 and 52.1: every CTA reads all of x. Bound by HBM behind a ramp: 77 % of its peak over 1 GB, 63 % over 262 MB.
struct HeadFewParams {
  HeadLogitsParams l;    // (v0, tiles_n, bn, stages, group are not looked at)
  int tiles, height;
  int n, cols;           // columns of a product, and of an accumulator: a multiple of 32, which is what a load of the epilogue takes
  int stages;
  int sums, buffers;     // accumulators of a tile; tiles that fit tensor memory side by side, 1 or 2
};
constexpr int kFewThreads = 320;  // warp 0 loader, warp 1 MMA, warps 2..9 epilogue
constexpr int kFewRows = 64, kFewMostStages = 12;
struct FewSmem {
  float turned[8][32][33];  // of each epilogue warp: [row of x][row of w]
  uint64_t full[kFewMostStages], empty[kFewMostStages], acc_full[2], acc_empty[2], drain;
  uint32_t tmem_base;
  uint32_t abort;
};
constexpr int kFewRing = (static_cast<int>(sizeof(FewSmem)) + 1023) & ~1023;  // where the ring begins
constexpr int kFewSmemBytes = 226 * 1024;  // with the 1024 bytes of alignment
__host__ __device__ constexpr uint32_t few_stage_bytes(int n) { return kGemmTileBytes + static_cast<uint32_t>(n) * 128; }

template <typename T>
__device__ __forceinline__ void head_few(const CUtensorMap* x, const CUtensorMap* x_copy, const CUtensorMap* w, const HeadFewParams& p, uint8_t* memory) {
  FewSmem& sm = *reinterpret_cast<FewSmem*>(memory);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    for (int i = lane; i < kFewMostStages; i += 32) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 1);
    }
    if (lane < 2) {
      mbar_init(&sm.acc_full[lane], 1);
      mbar_init(&sm.acc_empty[lane], 8);
    }
    if (lane == 0) {
      mbar_init(&sm.drain, 1);
      sm.abort = 0;
    }
    mbar_init_fence();
    __syncwarp();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sm.tmem_base;
  volatile uint32_t* abort_flag = &sm.abort;
  const int k_blocks = (p.l.dim + kGemmBK - 1) / kGemmBK;
  uint8_t* const ring = memory + kFewRing;
  const uint32_t stage_size = few_stage_bytes(p.n);
  const uint32_t bytes = static_cast<uint32_t>(p.height) * 128 + static_cast<uint32_t>(p.n) * 128;
  int early = 0;  // stages whose part of w is on its way before the wait: the kernel in front (head_rows_kernel) does not write it, and when this one
                  // starts, whatever wrote it is done
  if (warp == 0 && static_cast<int>(blockIdx.x) < p.tiles) {
    for (; early < p.stages && early < k_blocks; ++early) {
      if (elect_one()) {
        mbar_arrive_expect_tx(&sm.full[early], bytes);
        tma_load_2d(ring + early * stage_size, w, &sm.full[early], early * kGemmBK, blockIdx.x * p.height);
      }
    }
  }
  grid_dependency_wait();
  grid_launch_dependents();
  const int rows = __ldg(p.l.count);
  const int tiles = p.tiles;

  if (warp == 0) {
    // ======================= loader ==================================================================
    const CUtensorMap* const from = rows < p.l.all_rows ? x_copy : x;
    bool ok = true;
    int g = 0, st = 0;
    uint32_t ph = 1;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      for (int kb = 0; kb < k_blocks; ++kb, ++g) {
        if (g < early) {
          if (elect_one()) tma_load_2d(ring + st * stage_size + kGemmTileBytes, from, &sm.full[st], kb * kGemmBK, 0);
        } else {
          ok = __all_sync(0xffffffffu, mbar_wait(&sm.empty[st], ph, abort_flag));
          if (!ok) break;
          if (elect_one()) {
            mbar_arrive_expect_tx(&sm.full[st], bytes);
            tma_load_2d(ring + st * stage_size, w, &sm.full[st], kb * kGemmBK, tile * p.height);
            tma_load_2d(ring + st * stage_size + kGemmTileBytes, from, &sm.full[st], kb * kGemmBK, 0);
          }
        }
        if (++st == p.stages) {
          st = 0;
          ph ^= 1;
        }
      }
    }
    if (!ok && lane == 0 && atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0) atomicOr(p.l.status, kStatusHeadWait);
    if (__any_sync(0xffffffffu, *abort_flag != 0)) {  // let every copy that was issued land
      uint32_t no_abort = 0;
      for (int j = (g > p.stages ? g - p.stages : 0); j < g; ++j) mbar_wait(&sm.full[j % p.stages], (j / p.stages) & 1, &no_abort);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ======================= MMA issuer ==============================================================
    const uint32_t idesc = umma_idesc_f16(std::is_same<T, __half>::value ? UMMA_F16 : UMMA_BF16, 128, p.n, 0, 0);
    const uint64_t a0 = umma_smem_desc_sw128(smem_u32(ring), 1024, 16), b0 = umma_smem_desc_sw128(smem_u32(ring) + kGemmTileBytes, 1024, 16);
    bool ok = true, landed = false;
    int st = 0, it = 0;
    uint32_t ph = 0;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++it) {
      const int buf = p.buffers == 2 ? it & 1 : 0, turn = p.buffers == 2 ? it >> 1 : it;
      if (turn > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sm.acc_empty[buf], (turn - 1) & 1, abort_flag));
      if (!ok) break;
      tc_fence_after_sync();
      for (int sum = 0; sum < p.sums && ok; ++sum) {
        const uint32_t acc = tmem + (buf * p.sums + sum) * p.cols;
        const int kb0 = k_blocks * sum / p.sums, kb1 = k_blocks * (sum + 1) / p.sums;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = __all_sync(0xffffffffu, landed || mbar_wait(&sm.full[st], ph, abort_flag));
          if (!ok) break;
          tc_fence_after_sync();
          const int next = st + 1 == p.stages ? 0 : st + 1;
          const uint32_t next_ph = st + 1 == p.stages ? ph ^ 1 : ph;
          landed = mbar_test_wait(&sm.full[next], next_ph);
          const uint64_t a = a0 + static_cast<uint64_t>(st) * (stage_size >> 4), b = b0 + static_cast<uint64_t>(st) * (stage_size >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kGemmBK / 16; ++kk) umma_ss(acc, a + 2 * kk, b + 2 * kk, idesc, (kb != kb0 || kk != 0) ? 1u : 0u);
            umma_commit(&sm.empty[st]);
            if (kb == k_blocks - 1) umma_commit(&sm.acc_full[buf]);
          }
          st = next;
          ph = next_ph;
        }
      }
    }
    if (!ok && lane == 0 && atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0) atomicOr(p.l.status, kStatusHeadWait);
    if (__any_sync(0xffffffffu, *abort_flag != 0)) {  // no product may be running when tensor memory is freed
      uint32_t no_abort = 0;
      if (elect_one()) umma_commit(&sm.drain);
      mbar_wait(&sm.drain, 0, &no_abort);
    }
    __syncwarp();
  } else {
    // ======================= epilogue warps ==========================================================
    const int quarter = warp & 3, part = (warp - 2) >> 2;  // rows of w; every second 32 rows of x
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    float(*const turned)[33] = sm.turned[warp - 2];
    const int row = part * 32 + lane, src = row < rows ? __ldg(p.l.idx + row) : -1;
    const int* const ids = p.l.ids + static_cast<int64_t>(src) * p.l.top;
    bool ok = true;
    int it = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++it) {
      const int buf = p.buffers == 2 ? it & 1 : 0, turn = p.buffers == 2 ? it >> 1 : it;
      const int v0 = tile * p.height + quarter * 32, v1 = min(min(v0 + 32, (tile + 1) * p.height), p.l.vocab);  // this warp's rows of w
      int pos = 0, next = kNoEntry;  // the row's first entry from v0 on, searched for before the wait
      if (src >= 0) {
        for (int width = p.l.top > 1 ? 1 << (31 - __clz(p.l.top)) : 0; width > 0; width >>= 1)
          if (pos + width <= p.l.top && __ldg(ids + pos + width - 1) < v0) pos += width;
        if (pos < p.l.top) next = __ldg(ids + pos);
        if (next < v0) next = kNoEntry;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&sm.acc_full[buf], turn & 1, abort_flag))) {
        ok = false;
        break;
      }
      tc_fence_after_sync();
      if (part * 32 < rows) {
        const uint32_t acc = tmem + lane_addr + buf * p.sums * p.cols + part * 32;
        float v[32];
        tmem_ld_x32(acc, reinterpret_cast<uint32_t*>(v));
        for (int sum = 1; sum < p.sums; ++sum) {
          float more[32];
          tmem_ld_x32(acc + sum * p.cols, reinterpret_cast<uint32_t*>(more));
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += more[j];
        }
        const float bias = p.l.bias != nullptr && v0 + lane < v1 ? static_cast<float>(static_cast<const T*>(p.l.bias)[v0 + lane]) : 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) turned[j][lane] = v[j] + bias;
        __syncwarp();
        const float* const mine = turned[lane];
        const int n = v1 - v0;
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          v[j] = j < n ? mine[j] : -INFINITY;
          m = fmaxf(m, v[j]);
        }
        m *= p.l.log2_scale;
        const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int j = 0; j < 32; ++j) s += head_ex2(fmaf(v[j], p.l.log2_scale, -from));
        while (next < v1) {
          p.l.picks[static_cast<int64_t>(src) * p.l.top + pos] = mine[next - v0];
          next = ++pos < p.l.top ? __ldg(ids + pos) : kNoEntry;
        }
        if (src >= 0) p.l.parts[(tile * 4 + quarter) * p.l.parts_stride + row] = make_float2(m, n > 0 ? s : 0.f);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.acc_empty[buf]);
    }
    if (!ok && lane == 0 && atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0) atomicOr(p.l.status, kStatusHeadWait);
    __syncwarp();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// ---- sums: dx and dw of a piece ------------------------------------------------------------------------------------------------------
// What the sums are multiplied by: everything that is the same for all rows.
struct HeadScale {
  const float* grad;  // gradient of a loss that is one number, or null
  const float* norm;  // what head_coef_kernel divided the rows' gradients by, or null
  const int* count;   // mean: rows that count, else null
  float constant;     // tau / 2^s
};
__device__ __forceinline__ float head_scale(const HeadScale& s) {
  float v = s.constant;
  if (s.grad != nullptr) v *= __ldg(s.grad);
  if (s.norm != nullptr) v *= __ldg(s.norm);
  if (s.count != nullptr) v /= static_cast<float>(max(__ldg(s.count), 1));
  return v;
}

// Parts that dw is summed over: none without a k-block, whose product would never finish.
__device__ __forceinline__ int head_dw_parts(int rows, int twice, int splits) { return min(splits, max(1, (rows + 63) / 64) * twice); }

struct HeadSumsParams {
  const int* count;
  int all_rows, dim, vocab;
  int v0, cols;       // the piece: columns v0 .. v0 + cols - 1, cols a multiple of 256 or up to the last
  int splits;         // parts of the piece's columns that dx is summed over, 0: no dx
  int want_dw;
  int dw_splits;      // parts of the rows that dw is summed over; more than one, where a piece is all of the vocabulary: fp32 sums in place of dw
  int dw_slot_rows;   // rows of a part of those
  int bn, stages;
  int first;          // the first piece: dx begins
  int rest_at;        // see HeadLogitsParams
  int64_t slot_rows;  // rows of a part's sums, a multiple of 256
  HeadScale scale;
  uint32_t* status;
};

// kind 0: dx rows (tile of G, k along the piece's columns) x w (k not contiguous), fp32 sums that later pieces are added to;
// kind 1: dw rows (G as the left operand, its rows as k: not contiguous) x rows of x (not contiguous), final;
// kind 2: the same over a part of the rows, fp32 sums.
// An operand whose k is not contiguous comes as blocks of 64 k by 64 values, 128-byte rows with the swizzle: 8 KB from one block of
// values to the next, 1 KB from eight k to the next.
//
// The tiles of dx are long (k is the piece) and those of dw short (k counts rows): every pair takes its share of the long ones first, and the
// pairs with one fewer take so many short ones ahead of the others. Where a small vocabulary leaves few tiles of dw, each as long as there are rows, they
// are cut along the rows (forward and all gradients in us, one part -> cut: 8192 x 100 x 256 111 -> 50, 8192 x 10 x 64 100 -> 40, 2048 x 1000 x 1024 69 -> 51,
// 65536 x 256 x 512 517 -> 234).
template <typename T>
struct HeadSumsJob {
  const HeadSumsParams& p;
  const CUtensorMap *g_k, *g_mn, *w, *x, *x_copy, *dx, *dw;
  int rows, row_tiles, col_tiles, v_tiles, dx_items, n_dw, dw_parts, pairs;
  int twice;  // 2: k goes over G and then over what its rounding took

  __device__ __forceinline__ HeadSumsJob(const HeadSumsParams& p_, const CUtensorMap* gk, const CUtensorMap* gm, const CUtensorMap* w_, const CUtensorMap* x_,
                                         const CUtensorMap* xc, const CUtensorMap* dx_, const CUtensorMap* dw_)
      : p(p_), g_k(gk), g_mn(gm), w(w_), x(x_), x_copy(xc), dx(dx_), dw(dw_), twice(p_.rest_at > 0 ? 2 : 1) {}
  __device__ __forceinline__ void begin() {
    rows = __ldg(p.count);
    if (rows < p.all_rows) x = x_copy;
    pairs = gridDim.x >> 1;
    row_tiles = (rows + 255) >> 8;
    col_tiles = (p.dim + p.bn - 1) / p.bn;
    v_tiles = (p.cols + 255) >> 8;
    dx_items = row_tiles * col_tiles * p.splits;
    dw_parts = head_dw_parts(rows, twice, p.dw_splits);
    n_dw = p.want_dw ? v_tiles * col_tiles * dw_parts : 0;
  }
  // Short tiles that a pair with one long tile fewer takes first, of `behind` pairs.
  __device__ __forceinline__ void ahead(int* behind, int* each) const {
    const int rest = dx_items % pairs;
    *behind = rest == 0 ? 0 : pairs - rest;
    const int long_k = (p.cols + 63) / 64 / max(p.splits, 1), short_k = max(1, (rows + 63) / 64 / dw_parts);
    *each = *behind == 0 ? 0 : long_k / short_k;
  }
  __device__ __forceinline__ int items(int pair) const {
    int n = dx_items > pair ? (dx_items - pair + pairs - 1) / pairs : 0;
    int behind, each;
    ahead(&behind, &each);
    const int early = min(n_dw, behind * each), mine = pair - (pairs - behind);
    if (mine >= 0 && early > mine) n += (early - mine + behind - 1) / behind;
    const int late = n_dw - early;
    return n + (late > pair ? (late - pair + pairs - 1) / pairs : 0);
  }
  __device__ __forceinline__ HeadItem item(int pair, int i) const {
    const int long_ones = dx_items > pair ? (dx_items - pair + pairs - 1) / pairs : 0;
    if (i < long_ones) {
      const int at = pair + i * pairs, tiles = row_tiles * col_tiles, slot = at / tiles;
      int tm, tn;
      head_raster(at - slot * tiles, row_tiles, col_tiles, min(8, row_tiles), &tm, &tn);
      const int kbs = (p.cols + 63) / 64 * twice;
      return {0, slot, tm * 256, tn * p.bn, static_cast<int>(static_cast<int64_t>(kbs) * slot / p.splits), static_cast<int>(static_cast<int64_t>(kbs) * (slot + 1) / p.splits)};
    }
    i -= long_ones;
    int behind, each;
    ahead(&behind, &each);
    const int early = min(n_dw, behind * each), mine = pair - (pairs - behind);
    const int my_early = mine >= 0 && early > mine ? (early - mine + behind - 1) / behind : 0;
    const int at = i < my_early ? mine + i * behind : early + pair + (i - my_early) * pairs;
    const int tiles = v_tiles * col_tiles, slot = at / tiles;
    int tm, tn;
    head_raster(at - slot * tiles, v_tiles, col_tiles, min(8, v_tiles), &tm, &tn);
    const int64_t kbs = max(1, (rows + 63) / 64) * twice;  // (no row counts: a product all the same, of whatever is there, and zeros stored)
    return {p.dw_splits > 1 ? 2 : 1, slot, tm * 256, tn * p.bn, static_cast<int>(kbs * slot / dw_parts), static_cast<int>(kbs * (slot + 1) / dw_parts)};
  }
  __device__ __forceinline__ int stages() const { return p.stages; }
  __device__ __forceinline__ uint32_t stage_bytes() const { return kGemmTileBytes + static_cast<uint32_t>(p.bn) * kGemmBK; }
  __device__ __forceinline__ uint32_t bytes(const HeadItem&) const { return 2u * stage_bytes(); }
  __device__ __forceinline__ void load(const HeadItem& t, int kb, int rank, uint8_t* at, uint32_t bar) const {
    const int half = p.bn >> 1, once = t.kind == 0 ? (p.cols + 63) / 64 : max(1, (rows + 63) / 64);
    const bool rest = kb >= once;
    const int k = (rest ? kb - once : kb) * kGemmBK, g_row = rest ? p.rest_at : 0;
    if (t.kind == 0) {
      tma_load_2d_pair(at, g_k, bar, k, g_row + t.row0 + rank * 128);
    } else {
      tma_load_2d_pair(at, g_mn, bar, t.row0 + rank * 128, g_row + k);
      tma_load_2d_pair(at + kHeadBlock, g_mn, bar, t.row0 + rank * 128 + 64, g_row + k);
    }
    const CUtensorMap* b = t.kind == 0 ? w : x;
    const int b_k = t.kind == 0 ? p.v0 + k : k;
    for (int i = 0; i < half; i += 64) tma_load_2d_pair(at + kGemmTileBytes + i / 64 * kHeadBlock, b, bar, t.col0 + rank * half + i, b_k);
  }
  __device__ __forceinline__ uint32_t idesc(const HeadItem& t) const {
    return umma_idesc_f16(std::is_same<T, __half>::value ? UMMA_F16 : UMMA_BF16, 256, p.bn, t.kind != 0, 1);
  }
  __device__ __forceinline__ uint64_t a_desc(const HeadItem& t, uint32_t at) const { return umma_smem_desc_sw128(at, 1024, t.kind == 0 ? 16 : kHeadBlock); }
  __device__ __forceinline__ uint64_t b_desc(const HeadItem&, uint32_t at) const { return umma_smem_desc_sw128(at, 1024, kHeadBlock); }
  __device__ __forceinline__ int a_step(const HeadItem& t) const { return t.kind == 0 ? 2 : 128; }
  __device__ __forceinline__ int b_step(const HeadItem&) const { return 128; }

  struct Epilogue {
    const HeadSumsJob& job;
    const uint32_t stage;
    uint8_t* const stage_ptr;
    const int row_in, part, lane;
    int buf;
    const float scale;

    __device__ __forceinline__ Epilogue(const HeadSumsJob& j, uint32_t s, uint8_t* sp, int r, int pt)
        : job(j), stage(s), stage_ptr(sp), row_in(r), part(pt), lane(threadIdx.x & 31), buf(0), scale(head_scale(j.p.scale)) {}
    __device__ __forceinline__ void ask(const HeadItem&) {}

    template <typename HandBack>
    __device__ __forceinline__ void take(const HeadItem& t, uint32_t acc, HandBack&& hand_back) {
      const HeadSumsParams& p = job.p;
      const int width = t.kind != 1 ? 32 : 64, pieces = p.bn / width;  // 128 bytes of a row: fp32 sums, 16 bits of dw
#pragma unroll 1
      for (int c = part; c < pieces; c += 2) {
        const int col = t.col0 + c * width;
        const bool here = col < p.dim;
        if (lane == 0) tma_store_wait_read<1>();
        __syncwarp();
        if (here) {
          const uint32_t at_row = stage + buf * kHeadChunkBytes + lane * 128;
          if (t.kind != 1) {
            uint32_t v[32];
            tmem_ld_x32(acc + c * 32, v);
#pragma unroll
            for (int q = 0; q < 8; ++q) st_shared_v4(at_row + ((q ^ (lane & 7)) << 4), make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
          } else {
            const float2 scale2 = make_float2(scale, scale);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float v[32];
              tmem_ld_x32(acc + c * 64 + half * 32, reinterpret_cast<uint32_t*>(v));
              uint32_t out[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 y = fmul2(make_float2(v[2 * i], v[2 * i + 1]), scale2);
                out[i] = gemm_pack2<T>(y.x, y.y);
              }
              if (job.rows == 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i) out[i] = 0;
              }
#pragma unroll
              for (int q = 0; q < 4; ++q)
                st_shared_v4(at_row + (((4 * half + q) ^ (lane & 7)) << 4), make_uint4(out[4 * q], out[4 * q + 1], out[4 * q + 2], out[4 * q + 3]));
            }
          }
          fence_proxy_async_smem();
        }
        if (c + 2 >= pieces) hand_back();
        else __syncwarp();
        if (lane == 0) {
          if (here) {
            uint8_t* const from = stage_ptr + buf * kHeadChunkBytes;
            const int row = t.row0 + row_in;
            if (t.kind != 0) tma_store_2d(job.dw, from, col, t.slot * p.dw_slot_rows + p.v0 + row);
            else if (p.first) tma_store_2d(job.dx, from, col, static_cast<int>(t.slot * p.slot_rows) + row);
            else head_tma_add_2d(job.dx, from, col, static_cast<int>(t.slot * p.slot_rows) + row);
          }
          tma_store_commit();
        }
        buf ^= 1;
      }
    }
  };
};

// ---- kernels -----------------------------------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kHeadThreads, 1)
head_stats_kernel(const __grid_constant__ CUtensorMap x, const __grid_constant__ CUtensorMap x_copy, const __grid_constant__ CUtensorMap w,
                  const __grid_constant__ HeadLogitsParams p) {
  extern __shared__ uint8_t smem_raw[];
  HeadLogitsJob<T, false> job(p, &x, &x_copy, &w, nullptr);
  head_products(job, *reinterpret_cast<HeadSmem*>(smem_align_1024(smem_raw)), p.status);
}

template <typename T>
__global__ void __launch_bounds__(kFewThreads, 1)
head_few_kernel(const __grid_constant__ CUtensorMap x, const __grid_constant__ CUtensorMap x_copy, const __grid_constant__ CUtensorMap w, const __grid_constant__ HeadFewParams p) {
  extern __shared__ uint8_t smem_raw[];
  head_few<T>(&x, &x_copy, &w, p, smem_align_1024(smem_raw));
}

template <typename T>
__global__ void __launch_bounds__(kHeadThreads, 1)
head_grads_kernel(const __grid_constant__ CUtensorMap x, const __grid_constant__ CUtensorMap x_copy, const __grid_constant__ CUtensorMap w,
                  const __grid_constant__ CUtensorMap g, const __grid_constant__ HeadLogitsParams p) {
  extern __shared__ uint8_t smem_raw[];
  HeadLogitsJob<T, true> job(p, &x, &x_copy, &w, &g);
  head_products(job, *reinterpret_cast<HeadSmem*>(smem_align_1024(smem_raw)), p.status);
}

template <typename T>
__global__ void __launch_bounds__(kHeadThreads, 1)
head_sums_kernel(const __grid_constant__ CUtensorMap g_k, const __grid_constant__ CUtensorMap g_mn, const __grid_constant__ CUtensorMap w,
                 const __grid_constant__ CUtensorMap x, const __grid_constant__ CUtensorMap x_copy, const __grid_constant__ CUtensorMap dx,
                 const __grid_constant__ CUtensorMap dw, const __grid_constant__ HeadSumsParams p) {
  extern __shared__ uint8_t smem_raw[];
  HeadSumsJob<T> job(p, &g_k, &g_mn, &w, &x, &x_copy, &dx, &dw);
  head_products(job, *reinterpret_cast<HeadSmem*>(smem_align_1024(smem_raw)), p.status);
}

// Distillation: the entries of a row, a warp each. Entries whose token is negative do not count; one whose token is past the vocabulary makes NaN
// of its row. p = softmax(teacher / tau) over the others; entropy = sum p log p (0 where p is 0).
struct HeadEntriesParams {
  const void* ids;       // [rows, top] of id_bytes each, rows ids_stride apart
  const void* teacher;   // [rows, top], rows teacher_stride apart
  int64_t ids_stride, teacher_stride;
  int id_bytes, teacher_type;  // B200_ATTN_F16, _BF16 or _F32
  int rows, top, vocab;
  float inverse_tau;
  int* sorted;       // [rows, top]
  float* p;          // [rows, top]
  float* entropy;    // [rows]
  int8_t* counts;    // [rows]: whether any entry counts
  uint32_t* status;
};
constexpr int kEntriesWarps = 8, kEntriesMost = 256;

__device__ __forceinline__ float head_warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__global__ void __launch_bounds__(kEntriesWarps * 32) head_entries_kernel(const HeadEntriesParams p) {
  __shared__ int tokens[kEntriesWarps][kEntriesMost];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  grid_launch_dependents();
  const int row = blockIdx.x * kEntriesWarps + warp;
  if (row >= p.rows) return;
  constexpr int kEach = kEntriesMost / 32;
  int id[kEach];
  float z[kEach];
  float most = -INFINITY;
  bool any = false, bad = false;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int k = lane + 32 * i;
    id[i] = kNoEntry;
    z[i] = -INFINITY;
    if (k < p.top) {
      const int64_t at = row * p.ids_stride + k;
      const int64_t token = p.id_bytes == 8 ? static_cast<const int64_t*>(p.ids)[at] : static_cast<const int32_t*>(p.ids)[at];
      if (token >= 0) {
        any = true;
        const int64_t from = row * p.teacher_stride + k;
        z[i] = p.teacher_type == 0   ? __half2float(static_cast<const __half*>(p.teacher)[from])
               : p.teacher_type == 1 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.teacher)[from])
                                     : static_cast<const float*>(p.teacher)[from];
        z[i] *= p.inverse_tau;
        if (token >= p.vocab) bad = true;
        else id[i] = static_cast<int>(token);
      }
      tokens[warp][k] = id[i];
      most = fmaxf(most, z[i]);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
  any = __any_sync(0xffffffffu, any);
  bad = __any_sync(0xffffffffu, bad);
  __syncwarp();
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += z[i] == -INFINITY ? 0.f : expf(z[i] - most);  // a logit of -inf weighs nothing; NaN and +inf give NaN
  sum = head_warp_sum(sum);
  const float log_sum = logf(sum);
  float entropy = 0.f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int k = lane + 32 * i;
    if (k >= p.top) continue;
    int rank = 0;  // entries in front of this one: of lower tokens, and of the same token further left
    for (int j = 0; j < p.top; ++j) {
      const int other = tokens[warp][j];
      rank += other < id[i] || (other == id[i] && j < k) ? 1 : 0;
    }
    const float log_p = z[i] - most - log_sum;
    float weight = z[i] == -INFINITY ? 0.f : expf(log_p);
    if (any && most == -INFINITY) weight = NAN;  // entries count, but all at -inf: no distribution
    if (weight > 0.f) entropy += weight * log_p;
    if (isnan(weight) || bad) entropy = NAN;
    p.sorted[static_cast<int64_t>(row) * p.top + rank] = id[i];
    p.p[static_cast<int64_t>(row) * p.top + rank] = weight;
  }
  entropy = head_warp_sum(entropy);
  if (lane == 0) {
    p.entropy[row] = entropy;
    p.counts[row] = any ? 1 : 0;
    if (bad) atomicOr(p.status, kStatusTarget);
  }
}

// Which rows count, in the caller's order, and, where not all do, those rows of x together, with zeros behind the last up to the next
// multiple of 64 (k of the products over rows). Every CTA counts the rows in front of its own, a few kilobytes out of L2; where there are more
// (kCountedRows), head_count_kernel has left each CTA's number (a loss
// with the other kernels as they are now, without -> with it: 8192 x 10 x 64 11.6 -> 12.0 us, 24576 x 10 x 64 17.2 -> 14.1).
struct HeadRowsParams {
  const void* targets;   // [rows] of target_bytes each, or null: `counts`
  const int8_t* counts;  // distillation: whether a row has an entry
  int target_bytes;
  int64_t ignore;
  int rows, per_cta, vocab, dim;
  int top;
  const void* x;         // [rows, dim], rows ldx apart
  int64_t ldx;
  uint4* x_copy;         // [rows up to a multiple of 64, dim]
  int* count;
  unsigned* finished;    // zeroed: head_loss_kernel's CTAs count on it
  int* idx;              // [rows]
  int* place;            // [rows]: where a row went, -1: it does not count
  int* ids;              // [rows] targets as 32-bit entries (not for distillation)
  float* picks;          // [rows, top]: NaN for a target outside the vocabulary, which no tile writes
  float* loss;           // [rows] or null: 0 for rows that do not count
  int* cta_counts;       // [CTAs] or null
  uint32_t* status;
};
constexpr int kRowsThreads = 256, kRowsMost = 1024, kRowsAtOnce = 8, kCountedRows = 8192;

__device__ __forceinline__ int64_t head_target(const HeadRowsParams& p, int r) {
  return p.target_bytes == 8 ? static_cast<const int64_t*>(p.targets)[r] : static_cast<int64_t>(static_cast<const int32_t*>(p.targets)[r]);
}
__device__ __forceinline__ bool head_counted(const HeadRowsParams& p, int r) { return p.targets == nullptr ? p.counts[r] != 0 : head_target(p, r) != p.ignore; }

__global__ void __launch_bounds__(kRowsThreads) head_count_kernel(const HeadRowsParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int r0 = blockIdx.x * p.per_cta, r1 = min(p.rows, r0 + p.per_cta);
  int n = 0;
  for (int base = r0; base < r1; base += kRowsThreads) n += __syncthreads_count(base + static_cast<int>(threadIdx.x) < r1 && head_counted(p, base + threadIdx.x));
  if (threadIdx.x == 0) p.cta_counts[blockIdx.x] = n;
}

__global__ void __launch_bounds__(kRowsThreads) head_rows_kernel(const HeadRowsParams p) {
  __shared__ int from[kRowsMost], before_all, count_all, warp_sums[kRowsThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) before_all = count_all = 0;
  grid_dependency_wait();
  grid_launch_dependents();
  __syncthreads();
  const int r0 = blockIdx.x * p.per_cta, r1 = min(p.rows, r0 + p.per_cta);
  int before = 0, all = 0;
  if (p.cta_counts != nullptr) {
    for (int i = tid; i < static_cast<int>(gridDim.x); i += kRowsThreads) {
      const int c = p.cta_counts[i];
      all += c;
      before += i < static_cast<int>(blockIdx.x) ? c : 0;
    }
  } else {
#pragma unroll 8
    for (int r = tid; r < p.rows; r += kRowsThreads) {
      const int c = head_counted(p, r) ? 1 : 0;
      all += c;
      before += r < r0 ? c : 0;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, d);
    before += __shfl_xor_sync(0xffffffffu, before, d);
  }
  if (lane == 0) {
    atomicAdd(&before_all, before);
    atomicAdd(&count_all, all);
  }
  __syncthreads();
  int at = before_all;
  const int count = count_all;
  for (int base = r0; base < r1; base += kRowsThreads) {
    const int r = base + tid;
    const bool c = r < r1 && head_counted(p, r);
    const unsigned mask = __ballot_sync(0xffffffffu, c);
    if (lane == 0) warp_sums[warp] = __popc(mask);
    __syncthreads();
    int off = at;
    for (int i = 0; i < kRowsThreads / 32; ++i) {
      if (i < warp) off += warp_sums[i];
      at += warp_sums[i];
    }
    const int to = off + __popc(mask & ((1u << lane) - 1));
    if (r < r1) {
      from[r - r0] = c ? to : -1;
      p.place[r] = c ? to : -1;
      if (c) p.idx[to] = r;
      if (!c && p.loss != nullptr) p.loss[r] = 0.f;
      if (p.targets != nullptr) {
        const int64_t y = head_target(p, r);
        const bool inside = y >= 0 && y < p.vocab;
        p.ids[r] = c && inside ? static_cast<int>(y) : kNoEntry;
        if (c && !inside) {
          p.picks[r] = NAN;
          atomicOr(p.status, kStatusTarget);
        }
      }
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) {
    *p.count = count;
    *p.finished = 0;
  }
  if (count == p.rows) return;
  const int words = p.dim >> 3;
  for (int r = r0 + warp; r < r1; r += kRowsThreads / 32) {
    const int to = from[r - r0];
    if (to < 0) continue;
    const uint4* const in = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + r * p.ldx);
    uint4* const out = p.x_copy + static_cast<int64_t>(to) * words;
    for (int i = lane; i < words; i += 32 * kRowsAtOnce) {
      uint4 v[kRowsAtOnce];
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j)
        if (i + 32 * j < words) v[j] = in[i + 32 * j];
#pragma unroll
      for (int j = 0; j < kRowsAtOnce; ++j)
        if (i + 32 * j < words) out[i + 32 * j] = v[j];
    }
  }
  if (blockIdx.x == gridDim.x - 1)
    for (int64_t i = static_cast<int64_t>(count) * words + tid; i < static_cast<int64_t>((count + 63) & ~63) * words; i += kRowsThreads) p.x_copy[i] = make_uint4(0, 0, 0, 0);
}

// head_loss_kernel: lse and loss of 32 rows a CTA: a lane has a row and a warp every 32nd part; then a warp has a row and a lane every 32nd entry.
// head_loss_many_kernel: a thread has a row, where rows have one entry and few parts (a loss in us, without -> with it: 2 parts, 1024 x 10 x 64 11.5 -> 9.6,
// 8192 x 10 x 64 16.9 -> 11.6; 16 to 64 parts, 4096 x 1000 x 256 17.0 -> 17.4, 8192 x 1000 x 256 24.7 -> 20.2). The last CTA adds up the CTAs' sums in their order.
struct HeadLossParams {
  const int* count;
  const int* idx;
  const float2* parts;
  int64_t parts_stride;
  int n_parts, top;
  const float* picks;
  const float* p;        // [rows, top] or null: 1
  const float* entropy;  // [rows] or null: 0
  float log2_scale, tau;
  float* lse2;           // [rows]
  float* loss;           // [rows] or null
  float* total;          // the sum or the mean, or null
  int mean;
  float* sums;           // [CTAs]
  unsigned* finished;
};
constexpr int kLossThreads = 1024, kLossAtOnce = 8, kLossManyThreads = 256, kLossManyParts = 64, kLossManyRows = 8192, kLossFewParts = 8;

// Joins every so-manieth part of a row, from `i` on, to a maximum and a sum.
__device__ __forceinline__ void head_join_parts(const HeadLossParams& p, int row, int i, int step, float* m_out, float* s_out) {
  float m = -INFINITY, s = 0.f;
  for (; i < p.n_parts; i += step * kLossAtOnce) {  // so many loads in flight, one maximum for them
    float2 v[kLossAtOnce];
#pragma unroll
    for (int j = 0; j < kLossAtOnce; ++j) v[j] = i + step * j < p.n_parts ? __ldg(p.parts + (i + step * j) * p.parts_stride + row) : make_float2(-INFINITY, 0.f);
    float m_new = m;
#pragma unroll
    for (int j = 0; j < kLossAtOnce; ++j) m_new = fmaxf(m_new, v[j].x);
    const float from = m_new == -INFINITY ? 0.f : m_new;
    s *= head_ex2(m - from);
#pragma unroll
    for (int j = 0; j < kLossAtOnce; ++j) s = fmaf(v[j].y, head_ex2(v[j].x - from), s);
    m = m_new;
  }
  *m_out = m;
  *s_out = s;
}

// What an entry adds to its row's loss. The maximum first, and the product unrounded, as it is behind the exponentials: where the entry is the maximum what
// is left is the maximum's own rounding, which the sum holds too, and a small loss keeps its digits. An entry that does not count has no weight, and its logit
// was never written.
__device__ __forceinline__ float head_entry_loss(const HeadLossParams& p, int64_t at, float m, float log2_s) {
  const float weight = p.p != nullptr ? __ldg(p.p + at) : 1.f;
  return weight != 0.f ? weight * ((fmaf(-__ldg(p.picks + at), p.log2_scale, m) + log2_s) * 0.693147180559945f) : 0.f;
}

// The end of a row: its loss without the entropy -> as it is.
__device__ __forceinline__ float head_finish_row(const HeadLossParams& p, int src, float loss, float lse2, bool write) {
  if (p.entropy != nullptr) loss += __ldg(p.entropy + src);
  loss *= p.tau * p.tau;
  if (write) {
    p.lse2[src] = isnan(loss) ? NAN : lse2;  // a row without a loss has no gradient either
    if (p.loss != nullptr) p.loss[src] = loss;
  }
  return loss;
}

// The sum or the mean, of every CTA's sum, which thread 0 brings.
template <int THREADS>
__device__ __forceinline__ void head_total(const HeadLossParams& p, float sum, int count) {
  __shared__ double cta_sums[THREADS / 32];
  __shared__ bool last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    p.sums[blockIdx.x] = sum;
    __threadfence();
    last = atomicAdd(p.finished, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double all = 0.;
  for (unsigned i = threadIdx.x; i < gridDim.x; i += THREADS) all += static_cast<double>(__ldcg(p.sums + i));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
  if (lane == 0) cta_sums[warp] = all;
  __syncthreads();
  if (warp == 0) {
    all = lane < THREADS / 32 ? cta_sums[lane] : 0.;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
    if (lane == 0) *p.total = static_cast<float>(p.mean ? all / max(count, 1) : all);
  }
}

__global__ void __launch_bounds__(kLossManyThreads) head_loss_many_kernel(const HeadLossParams p) {
  __shared__ float warp_loss[kLossManyThreads / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int count = *p.count, row = blockIdx.x * kLossManyThreads + threadIdx.x;
  float loss = 0.f;
  if (row < count) {
    const int src = __ldg(p.idx + row);
    float m, s;
    head_join_parts(p, row, 0, 1, &m, &s);
    const float log2_s = log2f(s);
    loss = head_finish_row(p, src, head_entry_loss(p, src, m, log2_s), m + log2_s, true);
  }
  if (p.total == nullptr) return;
  const float sum = head_warp_sum(loss);
  if ((threadIdx.x & 31) == 0) warp_loss[threadIdx.x >> 5] = sum;
  __syncthreads();
  float all = 0.f;
  if (threadIdx.x == 0)
#pragma unroll
    for (int i = 0; i < kLossManyThreads / 32; ++i) all += warp_loss[i];
  head_total<kLossManyThreads>(p, all, count);
}

__global__ void __launch_bounds__(kLossThreads) head_loss_kernel(const HeadLossParams p) {
  __shared__ float2 part[32][33];
  __shared__ float row_loss[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  grid_launch_dependents();
  const int count = *p.count, row0 = blockIdx.x * 32;
  float m = -INFINITY, s = 0.f;
  if (row0 + lane < count) head_join_parts(p, row0 + lane, warp, 32, &m, &s);
  part[warp][lane] = make_float2(m, s);
  __syncthreads();
  const int row = row0 + warp;
  float loss = 0.f;
  if (row < count) {
    const float2 v = part[lane][warp];
    m = v.x;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    s = head_warp_sum(v.y * head_ex2(v.x - (m == -INFINITY ? 0.f : m)));
    const float log2_s = log2f(s);
    const int src = __ldg(p.idx + row);
    for (int k = lane; k < p.top; k += 32) loss += head_entry_loss(p, static_cast<int64_t>(src) * p.top + k, m, log2_s);
    loss = head_finish_row(p, src, head_warp_sum(loss), m + log2_s, lane == 0);
  }
  if (p.total == nullptr) return;
  if (lane == 0) row_loss[warp] = loss;
  __syncthreads();
  head_total<kLossThreads>(p, warp == 0 ? head_warp_sum(row_loss[lane]) : 0.f, count);
}

// Gradients that differ from row to row, divided by the power of two above the largest: what goes into 16 bits is then at most 1. One CTA reads them twice
// (65536 x 256 x 512 with gradients 171 -> 187 us; up to 8192 rows no difference).
struct HeadCoefParams {
  const int* count;
  const int* idx;
  const float* g;
  int64_t stride;
  float* coef;  // [rows], by the caller's rows
  float* norm;
};
constexpr int kCoefThreads = 1024;

__global__ void __launch_bounds__(kCoefThreads) head_coef_kernel(const HeadCoefParams p) {
  __shared__ float warp_most[32];
  __shared__ float norm_all;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  grid_launch_dependents();
  const int count = *p.count;
  float most = 0.f;
  for (int i = threadIdx.x; i < count; i += kCoefThreads) {
    const float g = fabsf(__ldg(p.g + __ldg(p.idx + i) * p.stride));
    if (g < INFINITY) most = fmaxf(most, g);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
  if (lane == 0) warp_most[warp] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 32; ++i) most = fmaxf(most, warp_most[i]);
    // 2^-126 .. 2^126: both it and its inverse are normal numbers
    norm_all = most > 0.f ? exp2f(fminf(fmaxf(static_cast<float>(ilogbf(most)) + 1.f, -126.f), 126.f)) : 1.f;
    *p.norm = norm_all;
  }
  __syncthreads();
  const float inverse = 1.f / norm_all;
  for (int i = threadIdx.x; i < count; i += kCoefThreads) {
    const int src = __ldg(p.idx + i);
    p.coef[src] = __ldg(p.g + src * p.stride) * inverse;
  }
}

// dbias of a piece: columns of G (and of what its rounding took) summed over the rows, 64 columns a CTA, eight a thread, every 32nd row each, the
// threads' sums in their order. One pass over G between the launch that writes it and the one that multiplies it, by as many CTAs as there are 64 columns, each of
// which walks all rows: a loss with its gradients in us, without a bias -> with it: 8192 x 10 x 64 35 -> 118, 8192 x 100 x 256 45 -> 123, 65536 x 256 x 512 171 -> 520,
// 2048 x 1000 x 1024 51 -> 73, 256 x 1000 x 768 38 -> 44, 4096 x 32000 x 1024 765 -> 950. Bound by the chain of loads of a CTA where columns are few.
struct HeadDbParams {
  const int* count;
  const void* g;    // [.., stride]
  int64_t stride;
  int rest_at, v0, cols, vocab;
  void* db;         // [vocab]
  HeadScale scale;
};
constexpr int kDbThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kDbThreads) head_db_kernel(const HeadDbParams p) {
  __shared__ float sums[kDbThreads / 8][65];
  grid_dependency_wait();
  grid_launch_dependents();
  const int count = __ldg(p.count), group = threadIdx.x & 7, first = threadIdx.x >> 3;
  float s[8] = {};
  for (int at = 0; at <= p.rest_at; at += max(p.rest_at, 1)) {  // (once without a rest)
    const T* const g = static_cast<const T*>(p.g) + at * p.stride + blockIdx.x * 64 + group * 8;
#pragma unroll 4
    for (int r = first; r < count; r += kDbThreads / 8) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(g + r * p.stride));
      const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = gemm_unpack2<T>(words[i]);
        s[2 * i] += f.x;
        s[2 * i + 1] += f.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[first][group * 8 + i] = s[i];
  __syncthreads();
  const int col = blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x >= 64 || col >= p.cols) return;
  float sum = 0.f;
  for (int i = 0; i < kDbThreads / 8; ++i) sum += sums[i][threadIdx.x];
  static_cast<T*>(p.db)[p.v0 + col] = static_cast<T>(count > 0 ? sum * head_scale(p.scale) : 0.f);  // (nothing is added up: 0 under any gradient, as dx and dw)
}

// dx, and dw where it was summed in parts: the parts' sums added in their order, scaled, rounded; zeros for rows that do not count. Eight values a thread.
struct HeadDxParams {
  const float* sums;     // [splits][slot_rows, dim]
  int splits;
  int64_t slot_rows;
  int rows, dim;         // rows 0: no dx
  const int* place;
  void* dx;              // [rows, dim]
  const float* dw_sums;  // [dw_splits][dw_slot_rows, dim]
  int dw_splits, dw_slot_rows, vocab, twice;  // vocab 0: dw is there already
  const int* count;
  void* dw;              // [vocab, dim]
  HeadScale scale;
};
constexpr int kDxThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kDxThreads) head_dx_kernel(const HeadDxParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int words = p.dim >> 3;
  const int64_t all = static_cast<int64_t>(p.rows + p.vocab) * words;
  const float scale = head_scale(p.scale);
  const int count = __ldg(p.count), dw_parts = head_dw_parts(count, p.twice, p.dw_splits);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kDxThreads + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * kDxThreads) {
    const int row = static_cast<int>(i / words), word = static_cast<int>(i - static_cast<int64_t>(row) * words);
    const bool is_dw = row >= p.rows;
    const int at = !is_dw ? __ldg(p.place + row) : count > 0 ? row - p.rows : -1, parts = is_dw ? dw_parts : p.splits;
    const int64_t slot_rows = is_dw ? p.dw_slot_rows : p.slot_rows;
    const float* const sums = is_dw ? p.dw_sums : p.sums;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (at >= 0) {
#pragma unroll 4
      for (int s = 0; s < parts; ++s) {
        const float4* const from = reinterpret_cast<const float4*>(sums + (s * slot_rows + at) * p.dim) + 2 * word;
        const float4 u = __ldg(from), v = __ldg(from + 1);
        a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
        b.x += v.x; b.y += v.y; b.z += v.z; b.w += v.w;
      }
    }
    uint4 out = make_uint4(0, 0, 0, 0);
    if (at >= 0)
      out = make_uint4(gemm_pack2<T>(a.x * scale, a.y * scale), gemm_pack2<T>(a.z * scale, a.w * scale), gemm_pack2<T>(b.x * scale, b.y * scale),
                       gemm_pack2<T>(b.z * scale, b.w * scale));
    if (is_dw) static_cast<uint4*>(p.dw)[i - static_cast<int64_t>(p.rows) * words] = out;
    else static_cast<uint4*>(p.dx)[i] = out;
  }
}

}  // namespace b200
