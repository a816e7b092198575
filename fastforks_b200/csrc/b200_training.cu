// C entry points of layer norm with its gradients and of an output layer's loss. Declarations are in include/b200_training.h.
#include "../../include/b200_training.h"

#include <algorithm>
#include <cmath>
#include <iterator>

#include "../../include/b200_attn.h"
#include "head_sm100.cuh"
#include "host_common.h"
#include "layer_norm_sm100.cuh"

namespace b200 {

namespace {

// ---- layer norm ------------------------------------------------------------------------------------------------------------------
struct NormForm {
  const void* kernel;
  int threads;  // of a row
  int vectors, vec;
  int rows = 1;                   // at a time
  int from = 0, below = 1 << 30;  // rows of the call for each SM
};

// The first that holds the row and is for so many rows. us of bf16 with several inputs in turn (threads x vectors; two: two rows at a time):
//   2400 x 1024  32 x 4 5.9, 64 x 2 two 4.4      1200 x 1024  32 x 4 5.4, 64 x 2 3.6      19200 x 1024  32 x 4 18.1, 64 x 2 two 16.5
//   2400 x 2048  128 x 2 7.6, two 6.1            9600 x 2048  128 x 2 18.0, two 16.9
//    600 x 4096  128 x 4 6.7, 256 x 2 4.7        1200 x 4096  128 x 4 7.8, 256 x 2 8.0    9600 x 4096   128 x 4 32.0, two 30.6
//   9600 x 512   32 x 2 6.9, two 5.7
// Few rows want many threads each, many rows few of them and more bytes in flight. Up to 768 values a warp has a row, without a barrier (two at a time were 3 %
// faster at 19200 x 768 and slower below).
template <typename T, int VEC, int N, int THREADS, int ROWS = 1>
NormForm forward_form(int from = 0, int below = 1 << 30) { return {reinterpret_cast<const void*>(norm_rows_kernel<T, VEC, N, THREADS, ROWS>), THREADS, N, VEC, ROWS, from, below}; }
template <typename T>
const NormForm* forward_forms(bool wide_rows, int* count) {
  // Value by value, where rows are no whole 16-byte words. us of bf16 (threads x values): 9600 x 333 256 x 4 17.4, 128 x 4 13.2; 9600 x 1001 256 x 4 23.3, two
  // 19.7; 1200 x 1901 256 x 8 9.8, two 6.8 (fp32 9.0, 9.8); 1200 x 3743 256 x 16 24.4, 512 x 8 17.2; 2400 x 5001 1024 x 16 72, 256 x 32 52, 512 x 16 39.5.
  static const NormForm values[] = {forward_form<T, 1, 1, 32>(), forward_form<T, 1, 4, 32>(), forward_form<T, 1, 8, 32>(), forward_form<T, 1, 4, 128>(),
                                    forward_form<T, 1, 4, 256>(0, 8), forward_form<T, 1, 4, 256, 2>(8), forward_form<T, 1, 8, 256>(0, 4), forward_form<T, 1, 8, 256, sizeof(T) == 2 ? 2 : 1>(4),
                                    forward_form<T, 1, 8, 512>(), forward_form<T, 1, 16, 512>(), forward_form<T, 1, 16, 1024>(), forward_form<T, 1, 32, 1024>()};
  if (!wide_rows) {
    *count = static_cast<int>(std::size(values));
    return values;
  }
  if constexpr (sizeof(T) == 2) {
    static const NormForm vectors[] = {forward_form<T, 8, 1, 32>(), forward_form<T, 8, 2, 32>(0, 64), forward_form<T, 8, 2, 32, 2>(64), forward_form<T, 8, 3, 32>(),
                                       forward_form<T, 8, 2, 64>(0, 16), forward_form<T, 8, 2, 64, 2>(16), forward_form<T, 8, 2, 128>(0, 16), forward_form<T, 8, 2, 128, 2>(16),
                                       forward_form<T, 8, 2, 256>(0, 8), forward_form<T, 8, 4, 128>(8, 32), forward_form<T, 8, 4, 128, 2>(32), forward_form<T, 8, 3, 256>(),
                                       forward_form<T, 8, 4, 256>(), forward_form<T, 8, 4, 512>(), forward_form<T, 8, 4, 1024>()};
    *count = static_cast<int>(std::size(vectors));
    return vectors;
  } else {
    static const NormForm vectors[] = {forward_form<T, 4, 1, 32>(), forward_form<T, 4, 2, 32>(), forward_form<T, 4, 3, 32>(), forward_form<T, 4, 4, 32>(), forward_form<T, 4, 2, 128>(),
                                       forward_form<T, 4, 3, 128>(), forward_form<T, 4, 4, 128>(), forward_form<T, 4, 4, 256>(), forward_form<T, 4, 4, 512>(), forward_form<T, 4, 4, 1024>(), forward_form<T, 4, 8, 1024>()};
    *count = static_cast<int>(std::size(vectors));
    return vectors;
  }
}
// The gradients of rows that do not go through shared memory: too wide for it, or not on 16 bytes.
template <typename T, int VEC, int N, int THREADS>
NormForm grad_form() { return {reinterpret_cast<const void*>(norm_rows_grad_kernel<T, VEC, N, THREADS>), THREADS, N, VEC}; }
template <typename T>
const NormForm* grad_forms(bool wide_rows, int* count) {
  // us, 128 threads a row up to 1024 values and 16 of each up to 2048 -> these: 30000 x 333 in bf16 73 -> 40, 8192 x 1001 34 -> 29, 5000 x 1900 50 -> 40. 8 values of
  // 512 threads up to 4096: 9000 x 3743 in fp32 97 -> 120, so not.
  static const NormForm values[] = {grad_form<T, 1, 1, 32>(), grad_form<T, 1, 4, 32>(), grad_form<T, 1, 8, 32>(), grad_form<T, 1, 4, 128>(), grad_form<T, 1, 4, 256>(),
                                    grad_form<T, 1, 8, 256>(), grad_form<T, 1, 16, 256>(), grad_form<T, 1, 16, 512>(), grad_form<T, 1, 16, 1024>(), grad_form<T, 1, 32, 1024>()};
  if (!wide_rows) {
    *count = static_cast<int>(std::size(values));
    return values;
  }
  if constexpr (sizeof(T) == 2) {
    static const NormForm vectors[] = {grad_form<T, 8, 2, 1024>(), grad_form<T, 8, 4, 1024>()};
    *count = static_cast<int>(std::size(vectors));
    return vectors;
  } else {
    static const NormForm vectors[] = {grad_form<T, 4, 4, 512>(), grad_form<T, 4, 4, 1024>(), grad_form<T, 4, 8, 1024>()};
    *count = static_cast<int>(std::size(vectors));
    return vectors;
  }
}
NormForm norm_form(const B200LayerNormArgs& a, bool grad, bool wide_rows, int sms) {
  int n = 0;
  const NormForm* f = nullptr;
  if (a.dtype == B200_ATTN_F16) f = grad ? grad_forms<__half>(wide_rows, &n) : forward_forms<__half>(wide_rows, &n);
  else if (a.dtype == B200_ATTN_BF16) f = grad ? grad_forms<__nv_bfloat16>(wide_rows, &n) : forward_forms<__nv_bfloat16>(wide_rows, &n);
  else f = grad ? grad_forms<float>(wide_rows, &n) : forward_forms<float>(wide_rows, &n);
  const int64_t each = a.rows / sms;
  int i = 0;
  while (i < n - 1 && (f[i].threads * f[i].vectors * f[i].vec < a.dim || each < f[i].from || each >= f[i].below)) ++i;
  return f[i];
}

// Gradients of rows that go through shared memory: G warps a row, N vectors a thread, in order of what they hold.
struct RingForm {
  const void* kernel;
  int warps, vectors;
};
template <typename T, int N, int G>
RingForm ring_form() { return {reinterpret_cast<const void*>(norm_ring_grad_kernel<T, 16 / sizeof(T), N, G>), G, N}; }
constexpr int kMostRingForms = 9;
template <typename T>
const RingForm* ring_forms(int* count) {
  if constexpr (sizeof(T) == 2) {
    static const RingForm forms[] = {ring_form<T, 1, 1>(), ring_form<T, 2, 1>(), ring_form<T, 2, 2>(), ring_form<T, 2, 4>(), ring_form<T, 2, 8>(), ring_form<T, 3, 8>(), ring_form<T, 4, 8>()};
    *count = static_cast<int>(std::size(forms));
    return forms;
  } else {
    static const RingForm forms[] = {ring_form<T, 1, 1>(), ring_form<T, 2, 1>(), ring_form<T, 3, 1>(), ring_form<T, 4, 1>(), ring_form<T, 3, 2>(), ring_form<T, 4, 2>(), ring_form<T, 3, 4>(), ring_form<T, 4, 4>(), ring_form<T, 4, 8>()};
    *count = static_cast<int>(std::size(forms));
    return forms;
  }
}

// The form of a call, or no kernel: rows that are no whole 16-byte words, or too wide.
struct RingPlan {
  RingForm form{nullptr, 0, 0};
  int index = 0, slots = 0, ctas = 0, threads = 0, smem = 0;
};
RingPlan ring_plan(const B200LayerNormArgs& a, bool wide_rows, int sms) {
  RingPlan r;
  if (!wide_rows) return r;
  int n = 0;
  const RingForm* f = a.dtype == B200_ATTN_F16 ? ring_forms<__half>(&n) : a.dtype == B200_ATTN_BF16 ? ring_forms<__nv_bfloat16>(&n) : ring_forms<float>(&n);
  const int values = a.dtype == B200_ATTN_F32 ? 4 : 8;  // of a vector
  int i = 0;
  while (i < n && f[i].warps * f[i].vectors * 32 * values < a.dim) ++i;
  if (i == n) return r;
  r.threads = 32 * ln_ring_warps(f[i].vectors * values);
  const int groups = r.threads / 32 / f[i].warps, slot = 2 * f[i].warps * f[i].vectors * 512;  // (a vector of 32 lanes: 512 bytes)
  r.form = f[i];
  r.index = (a.dtype == B200_ATTN_F16 ? 0 : a.dtype == B200_ATTN_BF16 ? 1 : 2) * kMostRingForms + i;
  r.slots = std::min(kLnMostSlots, kLnRingBytes / (groups * slot));
  r.ctas = static_cast<int>(std::min<int64_t>((a.rows + groups - 1) / groups, static_cast<int64_t>(sms)));
  r.smem = r.slots * groups * slot;
  return r;
}

size_t element(uint32_t dtype) { return dtype == B200_ATTN_F32 ? 4 : 2; }

// Shared memory above 48 KB is allowed per kernel and device.
constexpr int kHeadForms = 8, kOptIns = kHeadForms + 3 * kMostRingForms;
int opt_in(const void* kernel, int form, int smem) {
  static std::atomic<bool> done[kMaxDevices][kOptIns];
  int device = 0;
  if (const cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (device >= kMaxDevices) return fail(B200_ATTN_UNSUPPORTED, "device %d: at most %d devices", device, kMaxDevices);
  if (done[device][form].load(std::memory_order_acquire)) return B200_ATTN_OK;
  if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(shared memory)");
  done[device][form].store(true, std::memory_order_release);
  return B200_ATTN_OK;
}
bool whole_words(const B200LayerNormArgs& a) { return static_cast<size_t>(a.dim) * element(a.dtype) % 16 == 0; }

int check_norm(const B200LayerNormArgs* a) {
  if (a == nullptr) return fail(B200_ATTN_BAD_CONFIG, "args is NULL");
  if (a->struct_size != sizeof(B200LayerNormArgs))
    return fail(B200_ATTN_BAD_CONFIG, "struct_size %u does not match this library's B200LayerNormArgs (%zu bytes)", a->struct_size, sizeof(B200LayerNormArgs));
  if (a->dtype != B200_ATTN_F16 && a->dtype != B200_ATTN_BF16 && a->dtype != B200_ATTN_F32) return fail(B200_ATTN_BAD_CONFIG, "dtype %u: fp16 (0), bf16 (1) or fp32 (2)", a->dtype);
  if (a->weight_dtype != a->dtype && a->weight_dtype != B200_ATTN_F32) return fail(B200_ATTN_BAD_CONFIG, "weight_dtype %u: that of the rows or fp32 (2)", a->weight_dtype);
  if (a->dim < 1 || a->dim > 32768) return fail(B200_ATTN_UNSUPPORTED, "dim %d must be 1 .. 32768", a->dim);
  if (a->rows < 1 || a->rows > 0x7fffffffLL) return fail(B200_ATTN_UNSUPPORTED, "rows %lld must be 1 .. 2^31 - 1", static_cast<long long>(a->rows));
  if (!(a->eps >= 0.f) || std::isinf(a->eps)) return fail(B200_ATTN_BAD_CONFIG, "eps must be finite and not negative");
  return B200_ATTN_OK;
}

// A tensor of rows or of weights: its address, whether its values and (16 bytes at a time) its rows lie on boundaries.
int check_rows(const char* name, const void* p, int64_t stride, const B200LayerNormArgs* a, uint32_t dtype, bool* wide) {
  const size_t e = element(dtype);
  if (p == nullptr) return fail(B200_ATTN_BAD_CONFIG, "%s is NULL", name);
  if (reinterpret_cast<uintptr_t>(p) % e != 0) return fail(B200_ATTN_UNSUPPORTED, "%s is not aligned to its values", name);
  if (a->rows > 1 && (stride < 0 || stride >= (int64_t(1) << 40))) return fail(B200_ATTN_UNSUPPORTED, "%s: row stride %lld", name, static_cast<long long>(stride));
  if (!aligned16(p) || (a->rows > 1 && stride * static_cast<int64_t>(e) % 16 != 0)) *wide = false;
  return B200_ATTN_OK;
}
int check_weight(const char* name, const void* p, const B200LayerNormArgs* a, bool* wide) {
  if (p == nullptr) return B200_ATTN_OK;
  if (reinterpret_cast<uintptr_t>(p) % element(a->weight_dtype) != 0) return fail(B200_ATTN_UNSUPPORTED, "%s is not aligned to its values", name);
  if (!aligned16(p)) *wide = false;
  return B200_ATTN_OK;
}

// CTAs of the gradients' kernel: as many as run at once, so that each writes one part of dw and db and joining them costs little.
int grad_ctas(const B200LayerNormArgs& a, const NormForm& f, int sms) {
  const int rows_each = f.threads == 32 ? kLnGradWarps : 1, threads = f.threads == 32 ? 32 * kLnGradWarps : f.threads;
  const int per_sm = std::max(1, (f.vectors * f.vec <= 8 ? 1024 : 512) / threads);
  return static_cast<int>(std::min<int64_t>((a.rows + rows_each - 1) / rows_each, static_cast<int64_t>(sms) * per_sm));
}

LayerNormParams norm_params(const B200LayerNormArgs& a) {
  LayerNormParams p{};
  p.x = a.x;
  p.x_stride = a.x_stride;
  p.w = a.weight;
  p.stats = reinterpret_cast<float2*>(a.stats);
  p.rows = a.rows;
  p.dim = a.dim;
  p.eps = a.eps;
  p.inverse_dim = 1.f / static_cast<float>(a.dim);
  p.wide = a.weight_dtype == B200_ATTN_F32;
  return p;
}

// ---- the output layer ------------------------------------------------------------------------------------------------------------
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// What a call's buffers hold, in order, each on 256 bytes.
struct Layout {
  int64_t bytes = 0;
  int64_t add(int64_t n) {
    const int64_t at = bytes;
    bytes += up(n, 256);
    return at;
  }
};
struct HeadState {
  int64_t count, finished, idx, place, ids, p, entropy, counts, lse2, x_copy, bytes;
};
HeadState head_state(const B200HeadArgs& a) {
  const int64_t t = a.rows, k = std::max(a.top, 1);
  Layout l;
  HeadState s{};
  s.count = l.add(8);
  s.finished = s.count + 4;
  s.idx = l.add(4 * t);
  s.place = l.add(4 * t);
  s.ids = l.add(4 * t * k);
  if (a.top > 0) {
    s.p = l.add(4 * t * k);
    s.entropy = l.add(4 * t);
    s.counts = l.add(t);
  }
  s.lse2 = l.add(4 * t);
  s.x_copy = l.add(up(t, 64) * a.dim * 2);
  s.bytes = l.bytes;
  return s;
}

// Columns of a tile of logits: what makes the shortest list, by what a k-block of so many columns takes when all SMs pull operands (as for `gemm`). us,
// the widest that leaves no pair without a tile -> this: 256 x 8000 x 768 17.5 -> 15.0, with gradients 50.6 -> 47.0; of 13 other sizes from 100 x 32000 x 1024 to
// 3000 x 10000 x 4096 none changed beyond the 5 % that two runs differ by.
int logits_bn(int64_t row_tiles, int64_t cols, int64_t k_blocks, int pairs) {
  constexpr double kBlockUs[] = {0.298, 0.25, 0.21, 0.205};
  int best = 256;
  double best_us = 1e300;
  for (int i = 0; i < 4; ++i) {
    const int bn = 256 - 64 * i;
    const int64_t tiles = row_tiles * ((cols + bn - 1) / bn);
    const double us = static_cast<double>((tiles + pairs - 1) / pairs) * (static_cast<double>(k_blocks) * kBlockUs[i] + 0.15) + bn / 180.;
    if (us < best_us) {
      best_us = us;
      best = bn;
    }
  }
  return best;
}
int ring_stages(int bn) { return std::min(kHeadMaxStages, kHeadRingBytes / (kGemmTileBytes + bn * kGemmBK)); }

// How few rows are cut (head_few_kernel), n = 0: they go by pairs.
struct FewPlan {
  int n, cols, tiles, height, stages, sums, buffers;
};
FewPlan few_plan(const B200HeadArgs& a, int sms) {
  FewPlan f{};
  const int64_t n = up(a.rows, 16), cols = up(a.rows, 32);
  // As many accumulators of a tile as tensor memory holds, of 256 products or more, and of no more than the pairs take at once: the fewer products, the
  // less the tensor cores cut off, and a single row's loss has no others to average with (1 x 72 x 2048, 1024 at a time: 2.3e-6 off; 512: 7.7e-7).
  const int k_blocks = (a.dim + kGemmBK - 1) / kGemmBK, sums = static_cast<int>(std::min<int64_t>((k_blocks + 3) / 4, 512 / cols));
  if (n > kFewRows || (k_blocks + sums - 1) / sums > kHeadSumBlocks) return f;
  f.n = static_cast<int>(n);
  f.cols = static_cast<int>(cols);
  f.sums = sums;
  f.buffers = 2 * cols * sums <= 512 ? 2 : 1;
  const int each = (a.vocab + 128 * sms - 1) / (128 * sms);  // tiles of an SM
  f.height = static_cast<int>(std::max<int64_t>(32, up((a.vocab + static_cast<int64_t>(sms) * each - 1) / (static_cast<int64_t>(sms) * each), 8)));
  f.tiles = (a.vocab + f.height - 1) / f.height;
  f.stages = std::min(kFewMostStages, (kFewSmemBytes - 1024 - kFewRing) / static_cast<int>(few_stage_bytes(f.n)));
  return f;
}

struct HeadLossWork {
  FewPlan few;
  int bn, tiles_n, n_parts;
  int64_t parts_stride;
  int64_t parts, picks, sums, cta_counts, bytes;
};
HeadLossWork head_loss_work(const B200HeadArgs& a, int sms) {
  const int pairs = std::max(1, sms / 2);
  HeadLossWork w{};
  const int64_t row_tiles = (a.rows + 255) / 256;
  w.bn = logits_bn(row_tiles, a.vocab, (a.dim + kGemmBK - 1) / kGemmBK, pairs);
  w.tiles_n = (a.vocab + w.bn - 1) / w.bn;
  w.few = few_plan(a, sms);
  w.n_parts = w.few.n > 0 ? 4 * w.few.tiles : 2 * w.tiles_n;
  w.parts_stride = up(a.rows, 32);
  Layout l;
  w.parts = l.add(8LL * w.n_parts * w.parts_stride);
  w.picks = l.add(4LL * a.rows * std::max(a.top, 1));
  w.sums = l.add(4 * ((a.rows + 31) / 32));
  w.cta_counts = l.add(a.rows > kCountedRows ? 4 * ((a.rows + 7) / 8) : 0);
  w.bytes = l.bytes;
  return w;
}

// Gradients of logits in 16 bits of as many columns at a time as kPieceBytes holds, or 2048 where that is more (above 65536 rows: 1048576 x 4000 takes 4.3 GB); up to
// 2048 columns, padded to 256, are one piece. Each piece costs the fp32 sums of dx once more
// through L2 and HBM, under the products, and the rounds of two launches that are not full. us of a loss with its gradients at 128, 256 and 512 MB:
// 2047 x 50001 x 1024 609, 596, 596; 4096 x 64000 x 2048 (three quarters of the rows) 2378, 2335, 2299; 4096 x 128000 x 4096 12240, 12110, 12030.
constexpr int64_t kPieceBytes = 256 << 20;
// Where what the rounding of logits' gradients took is kept and multiplied too: few rows, whose products wait for memory, and products that are small beside
// the host's side of a call (2^31 multiply-adds more each for dx and dw, some 5 us; a call's forward and backward pass through autograd take 75). Elsewhere the
// caller says so (`whole`): 12 T D V operations in place of 8.
constexpr int64_t kRestRows = 128, kRestProducts = int64_t(1) << 31;
struct HeadGradWork {
  int64_t slot_rows;  // rows of G and of a part of dx
  int64_t g_rows;     // with those of what G's rounding took
  int cols;           // columns of G
  int splits, dw_splits, sums_bn;
  int64_t dw_slot_rows;
  int64_t g, sums, dw_sums, coef, norm, bytes;
};
HeadGradWork head_grad_work(const B200HeadArgs& a, bool want_dx, bool want_dw, int pairs) {
  HeadGradWork w{};
  w.slot_rows = up(a.rows, 256);
  w.g_rows = a.whole != 0 || a.rows <= kRestRows || static_cast<double>(a.rows) * a.dim * a.vocab <= static_cast<double>(kRestProducts) ? 2 * w.slot_rows : w.slot_rows;
  const int64_t most = std::max<int64_t>(2048, kPieceBytes / (2 * w.g_rows) / 256 * 256);
  const int64_t pieces = (a.vocab + most - 1) / most;
  w.cols = static_cast<int>(up((a.vocab + pieces - 1) / pieces, 256));
  w.sums_bn = a.dim > 128 ? 256 : 128;
  const int64_t col_tiles = (a.dim + w.sums_bn - 1) / w.sums_bn, tiles = w.slot_rows / 256 * col_tiles;
  // Parts of k that dx and dw are summed over: what gives the shortest longest list, in k-blocks of 64 (0.3 us). A tile of fp32 sums costs some four
  // more, every part a pass over them, and dw's (only where a piece is all of the vocabulary: they are not added to) a launch where dx does not have it.
  const int64_t twice = w.g_rows / w.slot_rows, k_blocks = (std::min<int64_t>(a.vocab, w.cols) + 63) / 64, row_blocks = (a.rows + 63) / 64;
  const int64_t dw_tiles = want_dw ? w.cols / 256 * col_tiles : 0, most_dx = want_dx ? std::min<int64_t>(32, k_blocks) : 1, most_dw = want_dw && pieces == 1 ? std::min<int64_t>(32, row_blocks) : 1;
  double best = 1e300;
  for (int64_t sw = 1; sw <= most_dw; ++sw) {
    const double short_each = static_cast<double>((row_blocks * twice + sw - 1) / sw) + (sw > 1 ? 4. : 0.), short_work = static_cast<double>(dw_tiles * sw) * short_each;
    const double short_pass = sw > 1 ? static_cast<double>(sw * a.vocab) * a.dim * 8. / 6.5e6 / 0.3 + 0.3 * static_cast<double>(sw) + (want_dx ? 0. : 8.) : 0.;
    for (int64_t s = 1; s <= most_dx; ++s) {
      const double rounds = want_dx ? static_cast<double>((tiles * s + pairs - 1) / pairs) : 0., each = static_cast<double>((k_blocks * twice + s - 1) / s) + 4.;
      const double even = ((want_dx ? static_cast<double>(tiles * s) * each : 0.) + short_work) / pairs + (want_dw ? 0.5 * short_each : 0.);
      const double pass = want_dx ? static_cast<double>(s * a.rows) * a.dim * 8. / 6.5e6 / 0.3 : 0.;  // written and read
      const double cost = std::max({rounds * each, even, want_dw ? short_each : 0.}) + pass + short_pass;
      if (cost < best) {
        best = cost;
        w.splits = want_dx ? static_cast<int>(s) : 0;
        w.dw_splits = static_cast<int>(sw);
      }
    }
  }
  w.dw_slot_rows = up(a.vocab, 256);
  Layout l;
  w.g = l.add(w.g_rows * w.cols * 2);
  w.sums = l.add(w.splits * w.slot_rows * a.dim * 4);
  w.dw_sums = l.add(w.dw_splits > 1 ? w.dw_splits * w.dw_slot_rows * a.dim * 4 : 0);
  w.coef = l.add(4LL * a.rows);
  w.norm = l.add(4);
  w.bytes = l.bytes;
  return w;
}

int check_head(const B200HeadArgs* a, bool sizes_only) {
  if (a == nullptr) return fail(B200_ATTN_BAD_CONFIG, "args is NULL");
  if (a->struct_size != sizeof(B200HeadArgs))
    return fail(B200_ATTN_BAD_CONFIG, "struct_size %u does not match this library's B200HeadArgs (%zu bytes)", a->struct_size, sizeof(B200HeadArgs));
  if (a->dtype != B200_ATTN_F16 && a->dtype != B200_ATTN_BF16) return fail(B200_ATTN_BAD_CONFIG, "dtype %u: x, w, dx and dw must be fp16 (0) or bf16 (1)", a->dtype);
  if (a->rows < 1 || a->rows > 1 << 24) return fail(B200_ATTN_UNSUPPORTED, "rows %d must be 1 .. 2^24", a->rows);
  if (a->dim < 8 || a->dim > 1 << 17 || a->dim % 8 != 0) return fail(B200_ATTN_UNSUPPORTED, "dim %d must be a multiple of 8, 8 .. 2^17", a->dim);
  if (a->vocab < 1 || a->vocab > 1 << 26) return fail(B200_ATTN_UNSUPPORTED, "vocab %d must be 1 .. 2^26", a->vocab);
  if (a->top < 0 || a->top > kEntriesMost) return fail(B200_ATTN_UNSUPPORTED, "top %d must be 0 .. %d", a->top, kEntriesMost);
  if (a->reduction != B200_HEAD_NONE && a->reduction != B200_HEAD_SUM && a->reduction != B200_HEAD_MEAN) return fail(B200_ATTN_BAD_CONFIG, "reduction %d: none (0), sum (1) or mean (2)", a->reduction);
  if (a->top > 0 && (!(a->tau > 0.f) || !std::isfinite(a->tau) || !std::isfinite(1.f / a->tau) || !std::isfinite(a->tau * a->tau)))
    return fail(B200_ATTN_UNSUPPORTED, "tau must be positive and finite, its square and its inverse too");
  if ((static_cast<int64_t>(a->rows) + 255) / 256 * ((static_cast<int64_t>(a->vocab) + 63) / 64) > 0x3fffffffLL) return fail(B200_ATTN_UNSUPPORTED, "problem too large for one launch");
  if (sizes_only) return B200_ATTN_OK;
  const struct { const char* name; const void* p; int64_t ld; } operands[] = {{"x", a->x, a->ldx}, {"w", a->w, a->ldw}};
  for (const auto& o : operands) {
    if (o.p == nullptr) return fail(B200_ATTN_BAD_CONFIG, "%s is NULL", o.name);
    if (!aligned16(o.p)) return fail(B200_ATTN_UNSUPPORTED, "%s is not 16-byte aligned", o.name);
    if (o.ld < a->dim || o.ld % 8 != 0 || o.ld >= (int64_t(1) << 38)) return fail(B200_ATTN_UNSUPPORTED, "%s: row stride %lld must cover the row and be a multiple of 8", o.name, static_cast<long long>(o.ld));
  }
  if (!aligned16(a->bias)) return fail(B200_ATTN_UNSUPPORTED, "bias is not 16-byte aligned");
  if (a->state == nullptr || reinterpret_cast<uintptr_t>(a->state) % 256 != 0 || a->state_bytes < head_state(*a).bytes) return fail(B200_ATTN_BAD_CONFIG, "state: %lld bytes on a 256-byte boundary are needed", static_cast<long long>(head_state(*a).bytes));
  if (a->workspace == nullptr || reinterpret_cast<uintptr_t>(a->workspace) % 256 != 0) return fail(B200_ATTN_BAD_CONFIG, "workspace must lie on a 256-byte boundary");
  return B200_ATTN_OK;
}

int head_map(CUtensorMap* map, const void* base, uint32_t dtype, int64_t rows, int64_t cols, int64_t stride, int box_cols, int box_rows, const char* name) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (enc == nullptr) return fail(B200_ATTN_CUDA_ERROR_BASE, "cuTensorMapEncodeTiled is not available from this driver");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * element(dtype)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)}, elem[2] = {1, 1};
  const CUtensorMapDataType type = dtype == B200_ATTN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : dtype == B200_ATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const CUresult r = enc(map, type, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B200_ATTN_UNSUPPORTED, "tensor map for %s rejected by the driver (CUresult %d)", name, static_cast<int>(r));
  return B200_ATTN_OK;
}

constexpr int kHeadSmemBytes = static_cast<int>(sizeof(HeadSmem)) + 1024;

template <typename P>
P* at(void* base, int64_t offset) { return reinterpret_cast<P*>(static_cast<uint8_t*>(base) + offset); }

float log2_scale(const B200HeadArgs& a) { return a.top > 0 ? static_cast<float>(1.4426950408889634 / static_cast<double>(a.tau)) : 1.4426950408889634f; }

HeadLogitsParams logits_params(const B200HeadArgs& a, const HeadState& s, uint32_t* status) {
  HeadLogitsParams p{};
  p.count = at<int>(a.state, s.count);
  p.idx = at<int>(a.state, s.idx);
  p.all_rows = a.rows;
  p.dim = a.dim;
  p.vocab = a.vocab;
  p.group = 16;
  p.top = std::max(a.top, 1);
  p.ids = at<int>(a.state, s.ids);
  p.p = a.top > 0 ? at<float>(a.state, s.p) : nullptr;
  p.log2_scale = log2_scale(a);
  p.bias = a.bias;
  p.status = status;
  return p;
}

// A thread that has made no CUDA call yet has no context, and without one no tensor map is made: autograd runs the gradients in such threads.
int bind_context() {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaSetDevice(device);
  return e == cudaSuccess ? B200_ATTN_OK : cuda_fail(e, "cudaSetDevice");
}

int launch_loss(const B200HeadArgs& a, cudaStream_t stream) {
  DeviceState* dev = nullptr;
  if (int rc = bind_context()) return rc;
  if (int rc = device_state(&dev)) return rc;
  const int pairs = std::max(1, dev->sms / 2);
  const HeadState s = head_state(a);
  const HeadLossWork w = head_loss_work(a, dev->sms);
  if (a.workspace_bytes < w.bytes) return fail(B200_ATTN_BAD_CONFIG, "workspace: %lld bytes are needed", static_cast<long long>(w.bytes));
  CUtensorMap mx, mc, mw;
  const bool few = w.few.n > 0;
  if (int rc = head_map(&mx, a.x, a.dtype, a.rows, a.dim, a.ldx, 64, few ? w.few.n : 128, "x")) return rc;
  if (int rc = head_map(&mc, at<void>(a.state, s.x_copy), a.dtype, up(a.rows, 64), a.dim, a.dim, 64, few ? w.few.n : 128, "x")) return rc;
  if (int rc = head_map(&mw, a.w, a.dtype, a.vocab, a.dim, a.ldw, 64, few ? w.few.height : w.bn / 2, "w")) return rc;
  const bool f16 = a.dtype == B200_ATTN_F16;
  const void* few_stats = f16 ? reinterpret_cast<const void*>(head_few_kernel<__half>) : reinterpret_cast<const void*>(head_few_kernel<__nv_bfloat16>);
  const void* stats = f16 ? reinterpret_cast<const void*>(head_stats_kernel<__half>) : reinterpret_cast<const void*>(head_stats_kernel<__nv_bfloat16>);
  if (int rc = few ? opt_in(few_stats, f16 ? 6 : 7, kFewSmemBytes) : opt_in(stats, f16 ? 0 : 1, kHeadSmemBytes)) return rc;
  if (a.top > 0) {
    HeadEntriesParams e{};
    e.ids = a.targets;
    e.teacher = a.teacher;
    e.ids_stride = a.targets_stride;
    e.teacher_stride = a.teacher_stride;
    e.id_bytes = a.target_bytes;
    e.teacher_type = static_cast<int>(a.teacher_dtype);
    e.rows = a.rows;
    e.top = a.top;
    e.vocab = a.vocab;
    e.inverse_tau = 1.f / a.tau;
    e.sorted = at<int>(a.state, s.ids);
    e.p = at<float>(a.state, s.p);
    e.entropy = at<float>(a.state, s.entropy);
    e.counts = at<int8_t>(a.state, s.counts);
    e.status = dev->status;
    void* args[] = {&e};
    if (int rc = launch_kernel(reinterpret_cast<const void*>(head_entries_kernel), static_cast<unsigned>((a.rows + kEntriesWarps - 1) / kEntriesWarps), 1, kEntriesWarps * 32, 0, 1, stream, args, "head_entries kernel launch")) return rc;
  }
  HeadRowsParams r{};
  r.targets = a.top > 0 ? nullptr : a.targets;
  r.counts = a.top > 0 ? at<int8_t>(a.state, s.counts) : nullptr;
  r.target_bytes = a.target_bytes;
  r.ignore = a.ignore;
  r.rows = a.rows;
  r.vocab = a.vocab;
  r.dim = a.dim;
  r.top = std::max(a.top, 1);
  r.x = a.x;
  r.ldx = a.ldx;
  r.x_copy = at<uint4>(a.state, s.x_copy);
  r.count = at<int>(a.state, s.count);
  r.finished = at<unsigned>(a.state, s.finished);
  r.idx = at<int>(a.state, s.idx);
  r.place = at<int>(a.state, s.place);
  r.ids = at<int>(a.state, s.ids);
  r.picks = at<float>(a.workspace, w.picks);
  r.loss = a.reduction == B200_HEAD_NONE ? a.loss : nullptr;
  r.status = dev->status;
  r.per_cta = std::min(kRowsMost, std::max(8, (a.rows + 2 * dev->sms - 1) / (2 * dev->sms)));
  {
    const unsigned ctas = static_cast<unsigned>((a.rows + r.per_cta - 1) / r.per_cta);  // at most every 8 rows one
    void* args[] = {&r};
    if (a.rows > kCountedRows) {
      r.cta_counts = at<int>(a.workspace, w.cta_counts);
      if (int rc = launch_kernel(reinterpret_cast<const void*>(head_count_kernel), ctas, 1, kRowsThreads, 0, 1, stream, args, "head_count kernel launch")) return rc;
    }
    if (int rc = launch_kernel(reinterpret_cast<const void*>(head_rows_kernel), ctas, 1, kRowsThreads, 0, 1, stream, args, "head_rows kernel launch")) return rc;
  }
  HeadLogitsParams p = logits_params(a, s, dev->status);
  p.v0 = 0;
  p.bn = w.bn;
  p.tiles_n = w.tiles_n;
  p.stages = ring_stages(w.bn);
  p.parts = at<float2>(a.workspace, w.parts);
  p.parts_stride = w.parts_stride;
  p.picks = at<float>(a.workspace, w.picks);
  if (few) {
    HeadFewParams q{p, w.few.tiles, w.few.height, w.few.n, w.few.cols, w.few.stages, w.few.sums, w.few.buffers};
    void* args[] = {&mx, &mc, &mw, &q};
    if (int rc = launch_kernel(few_stats, static_cast<unsigned>(std::min(w.few.tiles, dev->sms)), 1, kFewThreads, kFewSmemBytes, 1, stream, args, "head_few kernel launch")) return rc;
  } else {
    const int64_t items = (static_cast<int64_t>(a.rows) + 255) / 256 * w.tiles_n;
    void* args[] = {&mx, &mc, &mw, &p};
    if (int rc = launch_kernel(stats, static_cast<unsigned>(2 * std::min<int64_t>(items, pairs)), 1, kHeadThreads, kHeadSmemBytes, 2, stream, args, "head_stats kernel launch")) return rc;
  }
  HeadLossParams l{};
  l.count = p.count;
  l.idx = p.idx;
  l.parts = p.parts;
  l.parts_stride = p.parts_stride;
  l.n_parts = w.n_parts;
  l.top = p.top;
  l.picks = p.picks;
  l.p = p.p;
  l.entropy = a.top > 0 ? at<float>(a.state, s.entropy) : nullptr;
  l.log2_scale = p.log2_scale;
  l.tau = a.top > 0 ? a.tau : 1.f;
  l.lse2 = at<float>(a.state, s.lse2);
  l.loss = a.reduction == B200_HEAD_NONE ? a.loss : nullptr;
  l.total = a.reduction == B200_HEAD_NONE ? nullptr : a.loss;
  l.mean = a.reduction == B200_HEAD_MEAN;
  l.sums = at<float>(a.workspace, w.sums);
  l.finished = r.finished;
  void* args[] = {&l};
  if (l.top == 1 && w.n_parts <= (a.rows >= kLossManyRows ? kLossManyParts : kLossFewParts))
    return launch_kernel(reinterpret_cast<const void*>(head_loss_many_kernel), static_cast<unsigned>((a.rows + kLossManyThreads - 1) / kLossManyThreads), 1, kLossManyThreads, 0, 1, stream, args, "head_loss_many kernel launch");
  return launch_kernel(reinterpret_cast<const void*>(head_loss_kernel), static_cast<unsigned>((a.rows + 31) / 32), 1, kLossThreads, 0, 1, stream, args, "head_loss kernel launch");
}

int launch_grad(const B200HeadArgs& a, cudaStream_t stream) {
  DeviceState* dev = nullptr;
  if (int rc = bind_context()) return rc;
  if (int rc = device_state(&dev)) return rc;
  const int pairs = std::max(1, dev->sms / 2);
  const HeadState s = head_state(a);
  const bool want_dx = a.dx != nullptr, want_dw = a.dw != nullptr, want_db = a.dbias != nullptr, f16 = a.dtype == B200_ATTN_F16;
  const HeadGradWork w = head_grad_work(a, want_dx, want_dw, pairs);
  if (a.workspace_bytes < w.bytes) return fail(B200_ATTN_BAD_CONFIG, "workspace: %lld bytes are needed", static_cast<long long>(w.bytes));
  const int64_t row_tiles = w.slot_rows / 256;
  const int bn = logits_bn(row_tiles, std::min(a.vocab, w.cols), (a.dim + kGemmBK - 1) / kGemmBK, pairs);
  void* const x_copy = at<void>(a.state, s.x_copy);
  void* const g = at<void>(a.workspace, w.g);
  CUtensorMap x_k, copy_k, w_k, g_out, g_k, g_mn, w_mn, x_mn, copy_mn, dx, dw;
  if (int rc = head_map(&x_k, a.x, a.dtype, a.rows, a.dim, a.ldx, 64, 128, "x")) return rc;
  if (int rc = head_map(&copy_k, x_copy, a.dtype, up(a.rows, 64), a.dim, a.dim, 64, 128, "x")) return rc;
  if (int rc = head_map(&w_k, a.w, a.dtype, a.vocab, a.dim, a.ldw, 64, bn / 2, "w")) return rc;
  if (int rc = head_map(&g_out, g, a.dtype, w.g_rows, w.cols, w.cols, 64, 32, "workspace")) return rc;
  if (int rc = head_map(&g_k, g, a.dtype, w.g_rows, w.cols, w.cols, 64, 128, "workspace")) return rc;
  if (int rc = head_map(&g_mn, g, a.dtype, w.g_rows, w.cols, w.cols, 64, 64, "workspace")) return rc;
  if (int rc = head_map(&w_mn, a.w, a.dtype, a.vocab, a.dim, a.ldw, 64, 64, "w")) return rc;
  if (int rc = head_map(&x_mn, a.x, a.dtype, a.rows, a.dim, a.ldx, 64, 64, "x")) return rc;
  if (int rc = head_map(&copy_mn, x_copy, a.dtype, up(a.rows, 64), a.dim, a.dim, 64, 64, "x")) return rc;
  dx = dw = g_out;
  if (want_dx)
    if (int rc = head_map(&dx, at<void>(a.workspace, w.sums), B200_ATTN_F32, w.splits * w.slot_rows, a.dim, a.dim, 32, 32, "workspace")) return rc;
  const bool dw_parts = want_dw && w.dw_splits > 1;
  if (dw_parts) {
    if (int rc = head_map(&dw, at<void>(a.workspace, w.dw_sums), B200_ATTN_F32, w.dw_splits * w.dw_slot_rows, a.dim, a.dim, 32, 32, "workspace")) return rc;
  } else if (want_dw) {
    if (int rc = head_map(&dw, a.dw, a.dtype, a.vocab, a.dim, a.dim, 64, 32, "dw")) return rc;
  }
  const void* grads = f16 ? reinterpret_cast<const void*>(head_grads_kernel<__half>) : reinterpret_cast<const void*>(head_grads_kernel<__nv_bfloat16>);
  const void* sums = f16 ? reinterpret_cast<const void*>(head_sums_kernel<__half>) : reinterpret_cast<const void*>(head_sums_kernel<__nv_bfloat16>);
  if (int rc = opt_in(grads, f16 ? 2 : 3, kHeadSmemBytes)) return rc;
  if (int rc = opt_in(sums, f16 ? 4 : 5, kHeadSmemBytes)) return rc;

  const float g_scale = f16 ? 32768.f : 1.f;
  HeadScale scale{};
  scale.constant = (a.top > 0 ? a.tau : 1.f) / g_scale;
  HeadLogitsParams p = logits_params(a, s, dev->status);
  p.lse2 = at<float>(a.state, s.lse2);
  p.g_scale = g_scale;
  p.rest_at = w.g_rows > w.slot_rows ? static_cast<int>(w.slot_rows) : 0;
  p.bn = bn;
  p.stages = ring_stages(bn);
  if (a.reduction == B200_HEAD_NONE) {
    HeadCoefParams c{};
    c.count = p.count;
    c.idx = p.idx;
    c.g = a.grad;
    c.stride = a.grad_stride;
    c.coef = at<float>(a.workspace, w.coef);
    c.norm = at<float>(a.workspace, w.norm);
    p.coef = c.coef;
    scale.norm = c.norm;
    void* args[] = {&c};
    if (int rc = launch_kernel(reinterpret_cast<const void*>(head_coef_kernel), 1, 1, kCoefThreads, 0, 1, stream, args, "head_coef kernel launch")) return rc;
  } else {
    scale.grad = a.grad;
    if (a.reduction == B200_HEAD_MEAN) scale.count = p.count;
  }
  HeadSumsParams q{};
  q.count = p.count;
  q.all_rows = a.rows;
  q.dim = a.dim;
  q.vocab = a.vocab;
  q.want_dw = want_dw;
  q.dw_splits = w.dw_splits;
  q.dw_slot_rows = static_cast<int>(w.dw_slot_rows);
  q.bn = w.sums_bn;
  q.stages = ring_stages(w.sums_bn);
  q.slot_rows = w.slot_rows;
  q.rest_at = p.rest_at;
  q.scale = scale;
  q.status = dev->status;
  const int64_t col_tiles = (a.dim + w.sums_bn - 1) / w.sums_bn;
  for (int v0 = 0; v0 < a.vocab; v0 += w.cols) {
    const int cols = std::min(w.cols, a.vocab - v0);
    p.v0 = v0;
    p.tiles_n = (cols + bn - 1) / bn;
    void* logits_args[] = {&x_k, &copy_k, &w_k, &g_out, &p};
    if (int rc = launch_kernel(grads, static_cast<unsigned>(2 * std::min<int64_t>(row_tiles * p.tiles_n, pairs)), 1, kHeadThreads, kHeadSmemBytes, 2, stream, logits_args, "head_grads kernel launch")) return rc;
    q.v0 = v0;
    q.cols = cols;
    q.first = v0 == 0;
    q.splits = std::min(w.splits, (cols + 63) / 64);  // a part without a k-block would never finish; the first piece has one for each
    const int64_t items = row_tiles * col_tiles * q.splits + (want_dw ? static_cast<int64_t>((cols + 255) / 256) * col_tiles * w.dw_splits : 0);
    if (want_db) {
      HeadDbParams d{p.count, g, w.cols, p.rest_at, v0, cols, a.vocab, a.dbias, scale};
      void* db_args[] = {&d};
      const void* kernel = f16 ? reinterpret_cast<const void*>(head_db_kernel<__half>) : reinterpret_cast<const void*>(head_db_kernel<__nv_bfloat16>);
      if (int rc = launch_kernel(kernel, static_cast<unsigned>((cols + 63) / 64), 1, kDbThreads, 0, 1, stream, db_args, "head_db kernel launch")) return rc;
    }
    if (!want_dx && !want_dw) continue;
    void* sums_args[] = {&g_k, &g_mn, &w_mn, &x_mn, &copy_mn, &dx, &dw, &q};
    if (int rc = launch_kernel(sums, static_cast<unsigned>(2 * std::min<int64_t>(items, pairs)), 1, kHeadThreads, kHeadSmemBytes, 2, stream, sums_args, "head_sums kernel launch")) return rc;
  }
  if (!want_dx && !dw_parts) return B200_ATTN_OK;
  HeadDxParams d{};
  d.sums = at<float>(a.workspace, w.sums);
  d.splits = w.splits;
  d.slot_rows = w.slot_rows;
  d.rows = want_dx ? a.rows : 0;
  d.dw_sums = at<float>(a.workspace, w.dw_sums);
  d.dw_splits = w.dw_splits;
  d.dw_slot_rows = static_cast<int>(w.dw_slot_rows);
  d.vocab = dw_parts ? a.vocab : 0;
  d.twice = p.rest_at > 0 ? 2 : 1;
  d.count = p.count;
  d.dw = a.dw;
  d.dim = a.dim;
  d.place = at<int>(a.state, s.place);
  d.dx = a.dx;
  d.scale = scale;
  const int64_t words = static_cast<int64_t>(d.rows + d.vocab) * (a.dim / 8);
  const void* kernel = f16 ? reinterpret_cast<const void*>(head_dx_kernel<__half>) : reinterpret_cast<const void*>(head_dx_kernel<__nv_bfloat16>);
  void* args[] = {&d};
  return launch_kernel(kernel, static_cast<unsigned>(std::min<int64_t>((words + kDxThreads - 1) / kDxThreads, 8LL * dev->sms)), 1, kDxThreads, 0, 1, stream, args, "head_dx kernel launch");
}

}  // namespace

}  // namespace b200

using namespace b200;

extern "C" {

int b200_layer_norm(const B200LayerNormArgs* a, void* stream_ptr) {
  if (int rc = check_norm(a)) return rc;
  bool wide = whole_words(*a);
  if (int rc = check_rows("x", a->x, a->x_stride, a, a->dtype, &wide)) return rc;
  if (int rc = check_rows("y", a->y, a->y_stride, a, a->dtype, &wide)) return rc;
  if (a->rows > 1 && a->y_stride < a->dim) return fail(B200_ATTN_UNSUPPORTED, "rows of y overlap");
  if (int rc = check_weight("weight", a->weight, a, &wide)) return rc;
  if (int rc = check_weight("bias", a->bias, a, &wide)) return rc;
  LayerNormParams p = norm_params(*a);
  p.y = a->y;
  p.y_stride = a->y_stride;
  p.b = a->bias;
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  const NormForm f = norm_form(*a, false, wide, dev->sms);
  const int64_t each = (f.threads == 32 ? kLnForwardRows : 1) * f.rows, ctas = (a->rows + each - 1) / each;
  void* args[] = {&p};
  if (int rc = launch_kernel(f.kernel, static_cast<unsigned>(ctas), 1, f.threads == 32 ? 32 * kLnForwardRows : f.threads, 0, 1, static_cast<cudaStream_t>(stream_ptr), args, "layer_norm kernel launch")) return rc;
  clear_error();
  return B200_ATTN_OK;
}

int b200_layer_norm_workspace(const B200LayerNormArgs* a, int64_t* bytes) {
  if (int rc = check_norm(a)) return rc;
  if (bytes == nullptr) return fail(B200_ATTN_BAD_CONFIG, "bytes is NULL");
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  *bytes = 0;  // of whichever form the addresses lead to
  for (const bool wide : {false, true}) {
    *bytes = std::max<int64_t>(*bytes, 8LL * a->dim * grad_ctas(*a, norm_form(*a, true, wide, dev->sms), dev->sms));
    *bytes = std::max<int64_t>(*bytes, 8LL * a->dim * ring_plan(*a, wide && whole_words(*a), dev->sms).ctas);
  }
  clear_error();
  return B200_ATTN_OK;
}

int b200_layer_norm_grad(const B200LayerNormArgs* a, void* stream_ptr) {
  if (int rc = check_norm(a)) return rc;
  bool wide = whole_words(*a);
  if (int rc = check_rows("x", a->x, a->x_stride, a, a->dtype, &wide)) return rc;
  if (int rc = check_rows("dy", a->dy, a->dy_stride, a, a->dtype, &wide)) return rc;
  if (a->dx != nullptr) {
    if (int rc = check_rows("dx", a->dx, a->dx_stride, a, a->dtype, &wide)) return rc;
    if (a->rows > 1 && a->dx_stride < a->dim) return fail(B200_ATTN_UNSUPPORTED, "rows of dx overlap");
  }
  if (a->stats == nullptr || reinterpret_cast<uintptr_t>(a->stats) % 8 != 0) return fail(B200_ATTN_BAD_CONFIG, "stats must not be NULL and lie on 8 bytes");
  if (int rc = check_weight("weight", a->weight, a, &wide)) return rc;
  for (const void* p : {a->dweight, a->dbias})
    if (reinterpret_cast<uintptr_t>(p) % element(a->weight_dtype) != 0) return fail(B200_ATTN_UNSUPPORTED, "dweight or dbias is not aligned to its values");
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  const RingPlan ring = ring_plan(*a, wide, dev->sms);
  const bool through = ring.form.kernel != nullptr;
  const NormForm f = norm_form(*a, true, wide, dev->sms);
  const int ctas = through ? ring.ctas : grad_ctas(*a, f, dev->sms);
  const bool want_dw = a->dweight != nullptr || a->dbias != nullptr;
  if (want_dw && (a->workspace == nullptr || !aligned16(a->workspace) || a->workspace_bytes < 8LL * a->dim * ctas))
    return fail(B200_ATTN_BAD_CONFIG, "workspace: %lld bytes on a 16-byte boundary are needed", 8LL * a->dim * ctas);
  LayerNormParams p = norm_params(*a);
  p.dy = a->dy;
  p.dy_stride = a->dy_stride;
  p.dx = a->dx;
  p.dx_stride = a->dx_stride;
  p.partial = static_cast<float*>(a->workspace);
  p.want_dw = want_dw;
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  void* args[] = {&p};
  if (a->dx == nullptr && !want_dw) {  // nothing is asked for
    clear_error();
    return B200_ATTN_OK;
  }
  if (through) {
    p.slots = ring.slots;
    p.status = dev->status;
    if (int rc = opt_in(ring.form.kernel, kHeadForms + ring.index, kLnRingBytes)) return rc;
    if (int rc = launch_kernel(ring.form.kernel, static_cast<unsigned>(ctas), 1, static_cast<unsigned>(ring.threads), ring.smem, 1, stream, args, "layer_norm_grad kernel launch")) return rc;
  } else if (int rc = launch_kernel(f.kernel, static_cast<unsigned>(ctas), 1, f.threads == 32 ? 32 * kLnGradWarps : f.threads, f.threads == 32 ? 8 * static_cast<size_t>(a->dim) : 0, 1, stream, args, "layer_norm_grad kernel launch")) {
    return rc;
  }
  if (want_dw) {
    NormJoinParams j{};
    j.partial = p.partial;
    j.parts = ctas;
    j.dim = a->dim;
    j.dw = a->dweight;
    j.db = a->dbias;
    void* join_args[] = {&j};
    const void* kernel = a->weight_dtype == B200_ATTN_F16    ? reinterpret_cast<const void*>(norm_join_kernel<__half>)
                         : a->weight_dtype == B200_ATTN_BF16 ? reinterpret_cast<const void*>(norm_join_kernel<__nv_bfloat16>)
                                                             : reinterpret_cast<const void*>(norm_join_kernel<float>);
    if (int rc = launch_kernel(kernel, static_cast<unsigned>((a->dim + 31) / 32), 2, 32 * kLnJoinWarps, 0, 1, stream, join_args, "layer_norm_grad kernel launch")) return rc;
  }
  clear_error();
  return B200_ATTN_OK;
}

int b200_head_sizes(const B200HeadArgs* a, int64_t* state, int64_t* loss_workspace, int64_t* grad_workspace) {
  if (int rc = check_head(a, true)) return rc;
  if (state == nullptr || loss_workspace == nullptr || grad_workspace == nullptr) return fail(B200_ATTN_BAD_CONFIG, "a result is NULL");
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  const int pairs = std::max(1, dev->sms / 2);
  *state = head_state(*a).bytes;
  *loss_workspace = head_loss_work(*a, dev->sms).bytes;
  *grad_workspace = 0;
  for (int want = 0; want < 4; ++want) *grad_workspace = std::max(*grad_workspace, head_grad_work(*a, (want & 1) != 0, (want & 2) != 0, pairs).bytes);
  clear_error();
  return B200_ATTN_OK;
}

int b200_head_loss(const B200HeadArgs* a, void* stream_ptr) {
  if (int rc = check_head(a, false)) return rc;
  if (a->targets == nullptr) return fail(B200_ATTN_BAD_CONFIG, "targets is NULL");
  if ((a->target_bytes != 4 && a->target_bytes != 8) || reinterpret_cast<uintptr_t>(a->targets) % a->target_bytes != 0) return fail(B200_ATTN_BAD_CONFIG, "targets must be of 4 or 8 bytes (got %d), aligned to them", a->target_bytes);
  if (a->top > 0) {
    if (a->teacher == nullptr) return fail(B200_ATTN_BAD_CONFIG, "teacher is NULL");
    if (a->teacher_dtype != B200_ATTN_F16 && a->teacher_dtype != B200_ATTN_BF16 && a->teacher_dtype != B200_ATTN_F32) return fail(B200_ATTN_BAD_CONFIG, "teacher_dtype %u: fp16 (0), bf16 (1) or fp32 (2)", a->teacher_dtype);
    if (reinterpret_cast<uintptr_t>(a->teacher) % element(a->teacher_dtype) != 0) return fail(B200_ATTN_UNSUPPORTED, "teacher is not aligned to its values");
    if (a->targets_stride < 0 || a->teacher_stride < 0 || a->targets_stride >= (int64_t(1) << 38) || a->teacher_stride >= (int64_t(1) << 38)) return fail(B200_ATTN_UNSUPPORTED, "row strides of targets and teacher");
  }
  if (a->loss == nullptr || reinterpret_cast<uintptr_t>(a->loss) % 4 != 0) return fail(B200_ATTN_BAD_CONFIG, "loss must not be NULL and lie on 4 bytes");
  if (int rc = launch_loss(*a, static_cast<cudaStream_t>(stream_ptr))) return rc;
  clear_error();
  return B200_ATTN_OK;
}

int b200_head_grad(const B200HeadArgs* a, void* stream_ptr) {
  if (int rc = check_head(a, false)) return rc;
  if (a->grad == nullptr || reinterpret_cast<uintptr_t>(a->grad) % 4 != 0 || a->grad_stride < 0) return fail(B200_ATTN_BAD_CONFIG, "grad must not be NULL, lie on 4 bytes and have no negative stride");
  if (!aligned16(a->dx) || !aligned16(a->dw) || !aligned16(a->dbias)) return fail(B200_ATTN_UNSUPPORTED, "dx, dw or dbias is not 16-byte aligned");
  if (a->dx != nullptr || a->dw != nullptr || a->dbias != nullptr)
    if (int rc = launch_grad(*a, static_cast<cudaStream_t>(stream_ptr))) return rc;
  clear_error();
  return B200_ATTN_OK;
}

}  // extern "C"
