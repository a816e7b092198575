// Causal attention over the paged 4-bit cache for many rows: the products of kv4_attn_sm100.cuh on tcgen05.
//
// A CTA has two tiles of 128 rows (queries x the q heads that share a kv head) of one kv head and walks steps of 128 tokens. Both tiles'
// products take the same K and V, unpacked once for 256 rows to fp16. A code less 8 (three bits and a sign, or 8) times a step (eight bits) is
// exact in fp16, after powers of two that put the largest value of K of the step, and of V so far, below 2^15 (a token whose step
// is 2^26 times smaller than that loses bits). The rest of a value, least + 8 step, is treated by the type of q: in bfloat16 it is added in
// fp16 (a value is then off by at most 2^-11 of itself and 2^-11 of the rest, a quarter each of what rounding the output costs; the rest is the
// larger where a value cancels), in fp16 the softmax threads put it in in fp32: logit = q . (ks (u - 8)) + (kl + 8 ks) sum(q), o = sum p vs (w - 8) + sum p (vl + 8 vs).
//
// Roles: eight softmax warps (a thread has a row: S from tensor memory to registers, maximum, exponentials, P as fp16 over S's own
// columns), four warps that unpack K and V tiles into three buffers in turn (128-byte swizzle; K as rows of tokens, V as rows of
// dimensions along the fast index), one that brings blocks in by bulk copies, one that issues the products: PV and the
// next S of one tile while the other's softmax runs. Tensor memory: O 2 x head dim columns, S 2 x 128. The line of work, its runs and the
// join of parts are those of the other kernel.
//
// Measured: 2 x 500 queries of 32 heads on 8 over 9000 tokens, head dim 128, bf16, 212 us, 676 TFLOP/s, 41 % of the measured dense rate (the
// kernel of few rows took 647 us); whole prompts, dealt unevenly as the other kernel's comment says: 1 x 2048 130 us, 265 TFLOP/s, 1 x 4096 367 us,
// 374. A step of 256 rows takes some 4800 clocks, where its products need 1000 and its exponentials 2000: a tile's softmax (2100), its products and the
// waits between them follow one another, and unpacking (3000 for both tiles by one warp on each scheduler) is not much shorter (clocks are of one
// instrumented run).
#pragma once

#include "kv4_attn_sm100.cuh"

namespace b200 {

constexpr int kKv4TileThreads = 512, kKv4TileStep = 128, kKv4TileItem = 2, kKv4TileRows = 256;

template <int D>
struct Kv4TilesSmem {
  static constexpr int kHalves = D / 64;                 // 128-byte columns of a tile
  static constexpr int kTile = 128 * D * 2;              // bytes of 128 rows
  static constexpr int kRawBytes = 8 * Kv4Layout<D>::kBytes;
  static constexpr int kBufs = 3, kRaws = 2;
  static constexpr int kQ = 0;                           // [2 tiles]
  static constexpr int kBuf = 2 * kTile;                 // [kBufs]
  static constexpr int kRaw = kBuf + kBufs * kTile;      // [kRaws]
  static constexpr int kPar = kRaw + kRaws * kRawBytes;  // [2][kl + 8 ks, vl + 8 vs][128] floats
  static constexpr int kBig = kPar + 2 * 2 * 128 * 4;    // [2][4] largest magnitudes of K and of V, by the warp whose tokens they are of
  static constexpr int kScales = kBig + 64;              // [2] the step's power of two of K, and that of V so far
  static constexpr int kBars = kScales + 32;
  static constexpr int kFlags = kBars + 32 * 8;          // gave up, (unused), zero, tensor memory
  static constexpr int kBytes = kFlags + 16 + 1024;      // the tiles start on 1024
};

// Positions of the barriers.
enum Kv4TileBars { kBarRawFull = 0, kBarRawFree = 2, kBarBufFull = 4, kBarBufFree = 7, kBarParFull = 10, kBarParFree = 12, kBarQFull = 14, kBarSFull = 16, kBarPFull = 18, kBarOFull = 20, kBarDrain = 22, kBarCount = 23 };

// A CTA barrier (id 1) of 256 threads; whether any of them says so.
__device__ __forceinline__ bool softmax_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred.aligned q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(v ? 1u : 0u)
      : "memory");
  return r != 0;
}

// The same for the 128 threads that unpack (id 2).
__device__ __forceinline__ bool unpack_any(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred.aligned q, 2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(v ? 1u : 0u)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ uint32_t half2_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// The eight codes of a word less 8, as pairs (nibble i, nibble i + 4), by the published conversion of small integers through the low bits of 1024 in
// fp16: a code put there (or 16 times the code) makes 1024 plus it, and one multiply-add takes off 1024 + 8 (of a sixteenth: 64 + 8).
__device__ __forceinline__ void centre_codes(uint32_t w, uint32_t* pairs) {
  constexpr uint32_t kOne = 0x3c003c00u, kSixteenth = 0x2c002c00u, kLow = 0xe408e408u, kHigh = 0xd480d480u;  // 1, 1 / 16, -1032, -72
  const uint32_t h = w >> 8;
  pairs[0] = half2_fma((w & 0x000f000fu) | 0x64006400u, kOne, kLow);
  pairs[1] = half2_fma((w & 0x00f000f0u) | 0x64006400u, kSixteenth, kHigh);
  pairs[2] = half2_fma((h & 0x000f000fu) | 0x64006400u, kOne, kLow);
  pairs[3] = half2_fma((h & 0x00f000f0u) | 0x64006400u, kSixteenth, kHigh);
}
// 2^(14 - e) for the exponent e of `big`: it brings big below 2^15.
__device__ __forceinline__ int tile_exponent(float big, int least) { return max(least, min(static_cast<int>(__float_as_uint(big) >> 23) - 127, 126)); }

template <typename T, int D>
__global__ void __launch_bounds__(kKv4TileThreads, 1) kv4_tiles_kernel(const Kv4AttnParams p) {
  using S = Kv4TilesSmem<D>;
  using L = Kv4Layout<D>;
  constexpr bool kApart = std::is_same<T, __half>::value;  // least + 8 step is put in by the softmax threads
  constexpr int kStep = kKv4TileStep, kItem = kKv4TileItem;
  constexpr int kColS = 256;  // tensor memory: O at 0 and 128, S at 256 and 384
  extern __shared__ uint8_t tiles_smem_raw[];
  uint8_t* smem = smem_align_1024(tiles_smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + S::kFlags);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + kBarRawFull + i, 1);
      mbar_init(bars + kBarRawFree + i, 4);
      mbar_init(bars + kBarParFull + i, 4);
      mbar_init(bars + kBarParFree + i, 8);
      mbar_init(bars + kBarQFull + i, 4);
      mbar_init(bars + kBarSFull + i, 1);
      mbar_init(bars + kBarPFull + i, 4);
      mbar_init(bars + kBarOFull + i, 1);
    }
    for (int i = 0; i < S::kBufs; ++i) {
      mbar_init(bars + kBarBufFull + i, 4);
      mbar_init(bars + kBarBufFree + i, 1);
    }
    mbar_init(bars + kBarDrain, 1);
    abort_flag[0] = abort_flag[1] = abort_flag[2] = 0;
    mbar_init_fence();
    fence_proxy_async_smem();
  }
  if (warp == 13) {
    tmem_alloc(reinterpret_cast<uint32_t*>(smem + S::kFlags) + 3, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = abort_flag[3];
  grid_dependency_wait();
  grid_launch_dependents();
  write_unseen<T, D>(p, kKv4TileThreads);
  int run, count;  // of units
  Kv4Segment seg{};
  const bool any = kv4_start<kStep, kItem>(p, &run, &count, &seg);
  bool ok = true;
  const auto wait = [&](int bar, uint32_t parity) { return mbar_wait(bars + bar, parity, abort_flag); };
  const auto give_up = [&]() {
    if (lane == 0 && atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0) atomicOr(p.status, kStatusKv4Wait);
  };

  if (warp < 8) {
    // ---- softmax: thread `row` of tile t ----
    reg_alloc<184>();
    if (any) {
      const int t = warp >> 2, row = threadIdx.x & 127;
      const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // the warp's lanes of tensor memory, 32 (warp % 4) in the upper half
      const uint32_t s_tm = tmem + lanes + kColS + t * 128, o_tm = tmem + lanes + t * 128;
      uint32_t steps = 0, mine = 0, items = 0;  // of the CTA; of this tile
      for (;;) {
        const int seen = kv4_seen<kKv4TileRows, kStep>(p, seg);
        const int row0 = seg.tile * kKv4TileRows + 128 * t, last = min(row0 + row, p.rows - 1);
        const bool active = row0 < p.rows && seen > seg.s0;
        float l = 0.f, ms = 0.f, off = 0.f, rscale = 0.f, qsum = 0.f;  // off: log2 of what the sums are relative to, 2^-7 of the largest weight or so
        bool seen_any = false;
        float vunit = 0.f;  // O is in units of this
        const int n = static_cast<int>(magic_div(last, p.group_magic)), g = last - n * p.group, pos = seg.len - p.queries + n;
        const int lowest = seg.len - p.queries + static_cast<int>(magic_div(min(row0, p.rows - 1), p.group_magic));
        if (active) {
          const T* x = static_cast<const T*>(p.q) + seg.b * p.qs[0] + n * p.qs[1] + (seg.head * p.group + g) * p.qs[2];
          float most = 0.f;
#pragma unroll 4
          for (int w = 0; w < D / 8; ++w) {
            Raw8<T> raw;
            float f[8];
            raw.load(x + 8 * w);
            raw.unpack(f);
#pragma unroll
            for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(f[k]));
          }
          const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100), 126);
          const float up = pow2(10 - e);
#pragma unroll 4
          for (int w = 0; w < D / 8; ++w) {
            Raw8<T> raw;
            float f[8];
            raw.load(x + 8 * w);
            raw.unpack(f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              f[k] *= up;
              qsum += f[k];
            }
            // in the order in which a word of codes is split
            *reinterpret_cast<uint4*>(smem + S::kQ + t * S::kTile + (w >> 3) * 16384 + row * 128 + (((w & 7) ^ (row & 7)) << 4)) =
                make_uint4(pack2<__half>(f[0], f[4]), pack2<__half>(f[1], f[5]), pack2<__half>(f[2], f[6]), pack2<__half>(f[3], f[7]));
          }
          rscale = p.scale_log2 * pow2(e - 10);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kBarQFull + t);
        }
        for (int s = seg.s0; s < seen; ++s, ++steps) {
          const int st = steps & 1;
          if (!active) {  // keeps in step with the parameters
            ok = ok && wait(kBarParFull + st, (steps >> 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            if (lane == 0) mbar_arrive(bars + kBarParFree + st);
            continue;
          }
          ok = ok && wait(kBarParFull + st, (steps >> 1) & 1) && wait(kBarSFull + t, mine & 1);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          ++mine;
          tc_fence_after_sync();
          const float* par = reinterpret_cast<const float*>(smem + S::kPar) + st * 256;
          const float2 scales = *reinterpret_cast<const float2*>(smem + S::kScales + st * 8);
          float x[128];
          uint32_t* xu = reinterpret_cast<uint32_t*>(x);
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_x32_nowait(s_tm + 32 * c, xu + 32 * c);
          tmem_ld_wait_pin(xu);
#pragma unroll
          for (int c = 1; c < 4; ++c) tmem_ld_pin(xu + 32 * c);
          if constexpr (kApart) {
            const float2 qs2 = make_float2(qsum, qsum);
#pragma unroll
            for (int i = 0; i < 128; i += 4) {
              const float4 kl = *reinterpret_cast<const float4*>(par + i);
              const float2 a = ffma2(make_float2(kl.x, kl.y), qs2, make_float2(x[i], x[i + 1])), b = ffma2(make_float2(kl.z, kl.w), qs2, make_float2(x[i + 2], x[i + 3]));
              x[i] = a.x, x[i + 1] = a.y, x[i + 2] = b.x, x[i + 3] = b.y;
            }
          }
          const int base = s * kStep;
          if (base + kStep - 1 > lowest) {
            const int sees = pos - base;
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (i > sees) x[i] = -INFINITY;
          }
          float most = -INFINITY;
#pragma unroll
          for (int i = 0; i < 128; i += 2) most = fmaxf(most, fmaxf(x[i], x[i + 1]));
          // A row of zeros times a step of zeros leaves the range of fp32: 0 and infinity would make NaN of masked logits and of zeros. The
          // products are below 2^33, so at the least factor they are as good as zero.
          const float by = fminf(fmaxf(rscale * scales.x, FLT_MIN), FLT_MAX);
          most *= by;  // log2; by is positive
          if (__any_sync(0xffffffffu, (most > off + 15.f || !seen_any) && most != -INFINITY) || scales.y != vunit) {
            // New reference: weights are below 2^7 when it is set and below 2^15 as long as it stays.
            const float to = most != -INFINITY && (!seen_any || most > off + 7.f) ? most - 7.f : off;
            const float alpha = seen_any ? exp2_approx(off - to) : 0.f;
            seen_any = seen_any || most != -INFINITY;
            off = to;
            l *= alpha;
            ms *= alpha;
            if (s > seg.s0) {
              const float shrink = alpha * (vunit / scales.y);  // powers of two
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                uint32_t o[16];
                tmem_ld_x16(o_tm + c, o);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
                tmem_st_x16(o_tm + c, o);
              }
            }
            vunit = scales.y;
          }
          const float2 r2 = make_float2(by, by), off2 = make_float2(-off, -off);
          float2 l2 = make_float2(0.f, 0.f), ms2 = make_float2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float4 vl = make_float4(0.f, 0.f, 0.f, 0.f);
              if constexpr (kApart) vl = *reinterpret_cast<const float4*>(par + 128 + 32 * c + i);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int at = 32 * c + i + 2 * h;
                const float2 y = ffma2(make_float2(x[at], x[at + 1]), r2, off2);
                const float2 w = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                l2 = fadd2(l2, w);
                if constexpr (kApart) ms2 = ffma2(w, h == 0 ? make_float2(vl.x, vl.y) : make_float2(vl.z, vl.w), ms2);
                pk[(i + 2 * h) >> 1] = pack2<__half>(w.x, w.y);
              }
            }
            tmem_st_x16(s_tm + 16 * c, pk);
          }
          l += l2.x + l2.y;
          ms += ms2.x + ms2.y;
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bars + kBarPFull + t);
            mbar_arrive(bars + kBarParFree + st);
          }
        }
        if (active && ok) ok = wait(kBarOFull + t, items & 1);
        if (active) ++items;
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          give_up();
        }
        const bool gone = softmax_any(!ok || *abort_flag != 0);
        if (gone) break;
        // Whole items go out, parts to the workspace. O and the sums are in the same units, which cancel.
        const bool whole = seg.s1 - seg.s0 == seg.steps;
        const int slot = blockIdx.x * 2 + (seg.s0 > 0 ? 0 : 1), in_tile = 128 * t + row;
        const bool there = row0 + row < p.rows;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        tc_fence_after_sync();
        T* y = static_cast<T*>(p.o) + seg.b * p.os[0] + n * p.os[1] + (seg.head * p.group + g) * p.os[2];
        float* part = p.partial + (static_cast<int64_t>(slot) * kKv4TileRows + in_tile) * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          float f[16];
          if (active) {
            tmem_ld_x16(o_tm + c, reinterpret_cast<uint32_t*>(f));
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = fmaf(f[i], vunit, ms);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = 0.f;
          }
          if (!there) continue;
          if (whole) {
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = l == 0.f ? 0.f : f[i] * inv;
            store8<T>(y + c, f);
            store8<T>(y + c + 8, f + 8);
          } else {
#pragma unroll
            for (int i = 0; i < 16; i += 4) __stcg(reinterpret_cast<float4*>(part + c + i), make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]));
          }
        }
        tc_fence_before_sync();
        if (!whole) {
          if (there) __stcg(p.partial_ml + static_cast<int64_t>(slot) * kKv4TileRows + in_tile, make_float2(seen_any ? off : -INFINITY, l));
        }
        if (!kv4_next<kStep, kItem>(p, seg)) break;
      }
    }
  } else if (warp < 12) {
    // ---- unpacking ----
    reg_dealloc<72>();
    if (any) {
      const int thread = threadIdx.x & 127;
      uint32_t steps = 0;
      int v_exp = -100;
      for (;;) {
        const int seen = kv4_seen<kKv4TileRows, kStep>(p, seg);
        for (int s = seg.s0; s < seen; ++s, ++steps) {
          const int rs = steps & 1;
          const uint32_t kb = 2 * steps % 3, vb = (2 * steps + 1) % 3, k_use = 2 * steps / 3, v_use = (2 * steps + 1) / 3;
          const uint8_t* raw = smem + S::kRaw + rs * S::kRawBytes;
          ok = ok && wait(kBarRawFull + rs, (steps >> 1) & 1) && (k_use == 0 || wait(kBarBufFree + kb, (k_use - 1) & 1)) && (steps < 2 || wait(kBarParFree + rs, ((steps >> 1) - 1) & 1));
          // Parameters of this thread's token: zeros behind the sequence's end, where the page holds whatever it held. A token with a value that
          // is not finite gets NaN as its key and zeros as its value, so that it shows in the rows that see it alone.
          uint32_t k_pair, v_pair;  // (step, step), (step, rest) as halves
          uint32_t k_rest;
          {
            const uint2 v = *reinterpret_cast<const uint2*>(raw + (thread >> 4) * L::kBytes + L::kV + ((thread & 15) >> 1) * L::kRowV + D + (thread & 1) * 8);
            float ks = __uint_as_float(v.x << 16), kl = __uint_as_float(v.x & 0xffff0000u), vs = __uint_as_float(v.y << 16), vl = __uint_as_float(v.y & 0xffff0000u);
            if (s * kStep + thread >= seg.len) ks = kl = vs = vl = 0.f;
            kl = fmaf(8.f, ks, kl);
            vl = fmaf(8.f, vs, vl);
            float most_k = 8.f * ks + fabsf(kl), most_v = 8.f * vs + fabsf(vl);
            const bool fine = most_k + most_v < INFINITY;
            if (!fine) ks = kl = most_k = vs = vl = most_v = 0.f;
            const uint32_t big_k = __reduce_max_sync(0xffffffffu, __float_as_uint(most_k)), big_v = __reduce_max_sync(0xffffffffu, __float_as_uint(most_v));
            float* big = reinterpret_cast<float*>(smem + S::kBig) + rs * 8;
            if (lane == 0) {
              big[warp & 3] = __uint_as_float(big_k);
              big[4 + (warp & 3)] = __uint_as_float(big_v);
            }
            ok = !unpack_any(!ok);
            if (!ok) break;
            const float4 bk = *reinterpret_cast<const float4*>(big), bv = *reinterpret_cast<const float4*>(big + 4);
            const int ek = tile_exponent(fmaxf(fmaxf(bk.x, bk.y), fmaxf(bk.z, bk.w)), -100);
            v_exp = tile_exponent(fmaxf(fmaxf(bv.x, bv.y), fmaxf(bv.z, bv.w)), s == seg.s0 ? -100 : v_exp);
            const float up_k = pow2(14 - ek), up_v = pow2(14 - v_exp);
            k_pair = pack2<__half>(ks * up_k, ks * up_k);
            k_rest = kApart ? 0u : pack2<__half>(kl * up_k, kl * up_k);
            v_pair = pack2<__half>(vs * up_v, kApart ? 0.f : vl * up_v);
            if (!fine) k_pair = k_rest = 0x7e007e00u;
            float* par = reinterpret_cast<float*>(smem + S::kPar) + rs * 256 + thread;
            if (kApart) {
              par[0] = kl * up_k;
              par[128] = vl;
            }
            if (thread == 0) *reinterpret_cast<float2*>(smem + S::kScales + rs * 8) = make_float2(pow2(ek - 14), pow2(v_exp - 14));
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kBarParFull + rs);
          // K: a token's row, 16 bytes of codes (32 dimensions) at a time
          uint8_t* to = smem + S::kBuf + kb * S::kTile;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const uint4 w = *reinterpret_cast<const uint4*>(raw + (thread >> 4) * L::kBytes + (thread & 15) * L::kRowK + 16 * i);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t u[4];
              centre_codes(words[k], u);
#pragma unroll
              for (int n = 0; n < 4; ++n) u[n] = half2_fma(u[n], k_pair, k_rest);
              const int c = 4 * i + k;
              *reinterpret_cast<uint4*>(to + (c >> 3) * 16384 + thread * 128 + (((c & 7) ^ (thread & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kBarBufFull + kb);
          ok = v_use == 0 || wait(kBarBufFree + vb, (v_use - 1) & 1);
          if (unpack_any(!ok)) {
            ok = false;
            break;
          }
          // V: 16 dimensions of two tokens at a time. Every other lane has its second token first, so that eight lanes' rows differ mod 8.
          to = smem + S::kBuf + vb * S::kTile;
          const int swap = lane & 1, first_half = swap ? 0x7632 : 0x5410, second_half = swap ? 0x5410 : 0x7632;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const int unit = (warp & 3) * (D / 32) + i;  // eight pairs of tokens (a block) by four groups of 16 dimensions
            const int block = unit / (D / 64), group = unit % (D / 64) * 4 + (lane >> 3), pair = ((lane & 7) >> 1) + 4 * (lane & 1);
            const uint4 w = *reinterpret_cast<const uint4*>(raw + block * L::kBytes + L::kV + pair * L::kRowV + 16 * group);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
            // this warp's tokens are its lanes': steps and rests of the pair
            const uint32_t first = __shfl_sync(0xffffffffu, v_pair, 16 * (block & 1) + 2 * pair), second = __shfl_sync(0xffffffffu, v_pair, 16 * (block & 1) + 2 * pair + 1);
            const uint32_t v_step = __byte_perm(first, second, 0x5410), v_rest = __byte_perm(first, second, 0x7632);
            uint32_t one[8], two[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t u[4];
              centre_codes(words[k], u);
#pragma unroll
              for (int n = 0; n < 4; ++n) u[n] = half2_fma(u[n], v_step, v_rest);
              one[2 * k] = __byte_perm(u[0], u[1], first_half);
              one[2 * k + 1] = __byte_perm(u[2], u[3], first_half);
              two[2 * k] = __byte_perm(u[0], u[1], second_half);
              two[2 * k + 1] = __byte_perm(u[2], u[3], second_half);
            }
            uint8_t* half = to + (group >> 2) * 16384;
            const int r0 = 16 * block + 2 * pair + swap, r1 = r0 ^ 1, c = 2 * (group & 3);
            *reinterpret_cast<uint4*>(half + r0 * 128 + ((c ^ (r0 & 7)) << 4)) = make_uint4(one[0], one[1], one[2], one[3]);
            *reinterpret_cast<uint4*>(half + r0 * 128 + (((c + 1) ^ (r0 & 7)) << 4)) = make_uint4(one[4], one[5], one[6], one[7]);
            *reinterpret_cast<uint4*>(half + r1 * 128 + ((c ^ (r1 & 7)) << 4)) = make_uint4(two[0], two[1], two[2], two[3]);
            *reinterpret_cast<uint4*>(half + r1 * 128 + (((c + 1) ^ (r1 & 7)) << 4)) = make_uint4(two[4], two[5], two[6], two[7]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bars + kBarBufFull + vb);
            mbar_arrive(bars + kBarRawFree + rs);
          }
        }
        if (!ok) {
          give_up();
          break;
        }
        if (!kv4_next<kStep, kItem>(p, seg)) break;
      }
    }
  } else {
    reg_dealloc<72>();
    if (any && warp == 12) {
      // ---- loads ----
      if (lane == 0) {
        uint32_t steps = 0;
        while (ok) {
          const int seen = kv4_seen<kKv4TileRows, kStep>(p, seg);
          const uint8_t* base = p.cache + static_cast<int64_t>(seg.head) * p.page_blocks * L::kBytes;
          const int32_t* pages = p.page_table + seg.b * p.table_stride;
          for (int s = seg.s0; s < seen; ++s, ++steps) {
            const int rs = steps & 1;
            if (steps >= 2 && !wait(kBarRawFree + rs, ((steps >> 1) - 1) & 1)) {
              ok = false;
              break;
            }
            int block = 8 * s;
            const int end = min(block + 8, (seg.len + kKv4Block - 1) / kKv4Block);  // what lies behind is masked
            uint8_t* to = smem + S::kRaw + rs * S::kRawBytes;
            uint32_t col = magic_div(block, p.bpp_magic);
            int in = block - static_cast<int>(col) * p.page_blocks;
            while (block < end) {  // as many at a time as follow one another in a page
              const int page = pages[col], k = min(end - block, p.page_blocks - in);
              if (kv4_page_there(p, page)) {
                mbar_expect_tx(bars + kBarRawFull + rs, k * L::kBytes);
                bulk_load(to, base + (static_cast<int64_t>(page) * p.kv_heads * p.page_blocks + in) * L::kBytes, k * L::kBytes, bars + kBarRawFull + rs);
              } else {
                for (int i = 0; i < k; ++i) kv4_spoil<D>(to + i * L::kBytes);
              }
              to += k * L::kBytes;
              block += k;
              ++col;
              in = 0;
            }
            mbar_arrive(bars + kBarRawFull + rs);
          }
          if (!ok || !kv4_next<kStep, kItem>(p, seg)) break;
        }
        if (!ok) give_up();
        // Copies may still be in flight: they end before the shared memory goes. On every path, since another warp may give up when all is asked for.
        for (uint32_t i = steps < 2 ? 0 : steps - 2; i < steps; ++i) mbar_wait(bars + kBarRawFull + (i & 1), (i >> 1) & 1, abort_flag + 2);
      }
      __syncwarp();
    } else if (any && warp == 13) {
      // ---- products ----
      constexpr uint32_t idesc_s = umma_idesc_f16(UMMA_F16, 128, 128, 0, 0), idesc_o = umma_idesc_f16(UMMA_F16, 128, 64, 0, 1);
      uint32_t steps = 0, mine[2] = {0, 0}, items[2] = {0, 0};
      uint64_t& drain = bars[kBarDrain];
      // S of tile t from K in buffer kb
      const auto issue_s = [&](int t, uint32_t kb) {
        if (elect_one()) {
          const uint64_t a = umma_smem_desc_sw128(smem_u32(smem + S::kQ + t * S::kTile), 1024, 16), b = umma_smem_desc_sw128(smem_u32(smem + S::kBuf + kb * S::kTile), 1024, 16);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) umma_ss(tmem + kColS + t * 128, a + (k >> 2) * (16384 >> 4) + 2 * (k & 3), b + (k >> 2) * (16384 >> 4) + 2 * (k & 3), idesc_s, k > 0 ? 1u : 0u);
          umma_commit(bars + kBarSFull + t);
        }
        __syncwarp();
      };
      const auto issue_o = [&](int t, uint32_t vb, bool first) {
        if (elect_one()) {
#pragma unroll
          for (int h = 0; h < S::kHalves; ++h) {
            const uint64_t b = umma_smem_desc_sw128(smem_u32(smem + S::kBuf + vb * S::kTile + h * 16384), 1024, 0);
#pragma unroll
            for (int k = 0; k < 8; ++k) umma_ts(tmem + t * 128 + h * 64, tmem + kColS + t * 128 + k * 8, b + k * (2048 >> 4), idesc_o, first && k == 0 ? 0u : 1u);
          }
        }
        __syncwarp();
      };
      const auto commit = [&](int bar) {
        if (elect_one()) umma_commit(bars + bar);
        __syncwarp();
      };
      const auto all = [&](bool v) { return __all_sync(0xffffffffu, v) != 0; };
      while (ok) {
        const int seen = kv4_seen<kKv4TileRows, kStep>(p, seg), n = seen - seg.s0;
        const int tiles = p.rows > seg.tile * kKv4TileRows + 128 ? 2 : 1;
        if (n > 0) {
          uint32_t kb = 2 * steps % 3;
          ok = all(wait(kBarBufFull + kb, 2 * steps / 3 & 1));
          for (int t = 0; ok && t < tiles; ++t) {
            ok = all(wait(kBarQFull + t, items[t] & 1));
            if (!ok) break;
            ++items[t];
            tc_fence_after_sync();
            issue_s(t, kb);
          }
          if (ok) commit(kBarBufFree + kb);
          for (int j = 0; ok && j < n; ++j, ++steps) {
            const uint32_t vb = (2 * steps + 1) % 3, kn = 2 * (steps + 1) % 3;
            for (int t = 0; t < tiles; ++t) {
              ok = all(wait(kBarPFull + t, mine[t] & 1) && (t > 0 || wait(kBarBufFull + vb, (2 * steps + 1) / 3 & 1)));
              if (!ok) break;
              ++mine[t];
              tc_fence_after_sync();
              issue_o(t, vb, j == 0);
              if (t == tiles - 1) commit(kBarBufFree + vb);
              if (j + 1 == n) {
                commit(kBarOFull + t);
                continue;
              }
              if (t == 0) {
                ok = all(wait(kBarBufFull + kn, 2 * (steps + 1) / 3 & 1));
                if (!ok) break;
                tc_fence_after_sync();
              }
              issue_s(t, kn);
              if (t == tiles - 1) commit(kBarBufFree + kn);
            }
          }
        }
        if (!ok || !kv4_next<kStep, kItem>(p, seg)) break;
      }
      if (!ok) give_up();
      // Products may still run: they end before tensor memory is freed. On every path, since another warp may give up behind a look at its flag.
      if (elect_one()) umma_commit(&drain);
      __syncwarp();
      mbar_wait(&drain, 0, abort_flag + 2);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 13) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the items that the other kernel's runs cut: 32 rows of one item a CTA (the last CTA of an item, which joins in the kernel for few
// rows, would have 256 rows of every part to itself: 1 x 64 queries over 9000 tokens, 18 parts an item, took 100 us, 2 x 500 219). `ctas`:
// of the other kernel.
constexpr int kKv4JoinThreads = 256, kKv4JoinRows = 32;
template <typename T, int D>
__global__ void __launch_bounds__(kKv4JoinThreads) kv4_join_kernel(const Kv4AttnParams p, int ctas) {
  constexpr int kStep = kKv4TileStep, kItem = kKv4TileItem, kSlices = kKv4TileRows / kKv4JoinRows;
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31, per = p.kv_heads * p.row_tiles;
  const int item = blockIdx.x / kSlices, slice = blockIdx.x % kSlices;
  Kv4Segment seg{};
  seg.b = item / per;
  seg.tile = item % per / p.kv_heads;
  seg.head = item % per % p.kv_heads;
  seg.len = kv4_length(p, seg.b);
  seg.steps = (seg.len + kStep - 1) / kStep;
  long long total = 0, before = 0;  // units of the line, and those in front of the sequence
  for (int b = lane; b < p.batch; b += 32) {
    const int len = kv4_length(p, b), units = len == 0 ? 0 : (len + kStep - 1) / kStep + kItem;
    total += units;
    if (b < seg.b) before += units;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if (seg.len == 0) return;
  const long long run = max(static_cast<long long>(p.min_run), (total * per + ctas - 1) / ctas);
  const long long begin = before * per + static_cast<long long>(item % per) * (seg.steps + kItem) + kItem;  // of the item's steps
  const int first = static_cast<int>(begin / run), parts = static_cast<int>((begin + seg.steps - 1) / run) - first + 1;
  if (parts == 1) return;
  join_parts<T, D, 4, 2>(p, seg, kKv4TileRows, first, parts, slice * kKv4JoinRows, kKv4JoinRows, threadIdx.x, kKv4JoinThreads);
}

}  // namespace b200
