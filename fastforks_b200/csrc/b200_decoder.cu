// C entry points of a token decoder's layers: rotary positions, norms of q and k, the paged 4-bit cache and its attention.
// Declarations are in include/b200_decoder.h.
#include "../../include/b200_decoder.h"

#include <algorithm>
#include <cmath>

#include "../../include/b200_attn.h"
#include "host_common.h"
#include "kv4_attn_sm100.cuh"
#include "kv4_sm100.cuh"
#include "kv4_tiles_sm100.cuh"
#include "rotary_sm100.cuh"

namespace b200 {

namespace {

constexpr int kMaxDim = 512, kRotaryCtasPerSm = 2, kKv4CtasPerSm = 4, kKv4MaxRows = 64;
constexpr int kCounterBytes = 256;

// Whether every row of a tensor of heads starts on 16 bytes.
bool rows_aligned(const void* p, const int64_t s[3], int batch, int tokens, int heads, int size) {
  return aligned16(p) && (batch == 1 || s[0] * size % 16 == 0) && (tokens == 1 || s[1] * size % 16 == 0) && (heads == 1 || s[2] * size % 16 == 0);
}

int lanes_log2_of(int dim) {
  int n = 0;
  while (16 << n < dim) ++n;
  return n;
}

constexpr int kSplitBytes = 16384;  // the rows that a CTA's groups of lanes turn, as floats: 16 dimensions a lane at most
struct RotaryForm {
  const void* kernel;
  int smem, ctas_per_sm;
};
template <typename T, int FORM, int MODE>
RotaryForm stream_form(int more) {
  using S = RotaryStream<T, MODE, FORM>;
  return {reinterpret_cast<const void*>(rotary_stream_kernel<T, FORM, MODE>), S::kBytes + more, S::kCtasPerSm};
}
template <typename T, int MODE>
RotaryForm rotary_form(int form) {
  if (form == kRowHalves) return stream_form<T, kRowHalves, MODE>(0);
  if (form == kRowPairs) return stream_form<T, kRowPairs, MODE>(0);
  if (form == kRowLoose) return stream_form<T, kRowLoose, MODE>(0);
  if (form == kRowSplit) return stream_form<T, kRowSplit, MODE>(kSplitBytes);
  return {reinterpret_cast<const void*>(rotary_any_kernel<T, MODE>), 0, 2};
}
template <typename T>
RotaryForm rotary_form_of(int form, int mode) {
  return mode == kTurn ? rotary_form<T, kTurn>(form) : mode == kNormTurn ? rotary_form<T, kNormTurn>(form) : rotary_form<T, kNormBack>(form);
}
std::atomic<bool> g_rotary_opted_in[kMaxDevices][3][kRowForms][3];

// The shared-memory opt-in of a kernel on this device, once.
int opt_in(std::atomic<bool>& done, const void* kernel, int smem, const char* what) {
  if (done.load(std::memory_order_acquire)) return B200_ATTN_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return cuda_fail(e, what);
  done.store(true, std::memory_order_release);
  return B200_ATTN_OK;
}
int current_device(int* device) {
  const cudaError_t e = cudaGetDevice(device);
  return e == cudaSuccess ? B200_ATTN_OK : cuda_fail(e, "cudaGetDevice");
}

int check_table(const char* what, const float* cs, int rot, int dim, int table_rows) {
  if (rot < 0 || rot > dim || rot % 2 != 0) return fail(B200_ATTN_UNSUPPORTED, "%s: rot %d must be even and 0 .. %d", what, rot, dim);
  if (rot == 0) return B200_ATTN_OK;
  if (cs == nullptr || table_rows < 1) return fail(B200_ATTN_BAD_CONFIG, "%s: no table of positions", what);
  if (!aligned16(cs)) return fail(B200_ATTN_UNSUPPORTED, "%s: cs is not 16-byte aligned", what);
  return B200_ATTN_OK;
}

// The cache, its page table and the lengths, as all three calls over it have them.
int check_cache(const char* what, uint32_t dtype, int batch, int tokens, int kv_heads, int head_dim, int page, int pages, int table_pages, const void* cache, const int32_t* table, const int32_t* lengths) {
  if (dtype != B200_ATTN_F16 && dtype != B200_ATTN_BF16) return fail(B200_ATTN_BAD_CONFIG, "%s: dtype %u must be fp16 (0) or bf16 (1)", what, dtype);
  if (head_dim != 64 && head_dim != 128) return fail(B200_ATTN_UNSUPPORTED, "%s: head_dim %d, only 64 and 128 are built", what, head_dim);
  if (batch < 1 || tokens < 1 || kv_heads < 1) return fail(B200_ATTN_BAD_CONFIG, "%s: batch %d, tokens %d, kv_heads %d", what, batch, tokens, kv_heads);
  if (page < kKv4Block || page % kKv4Block != 0) return fail(B200_ATTN_UNSUPPORTED, "%s: a page of %d tokens, it must be a multiple of 16", what, page);
  if (pages < 1 || table_pages < 1 || static_cast<int64_t>(table_pages) * page > INT32_MAX) return fail(B200_ATTN_BAD_CONFIG, "%s: %d pages, %d in a row of the page table", what, pages, table_pages);
  if (cache == nullptr || table == nullptr || lengths == nullptr) return fail(B200_ATTN_BAD_CONFIG, "%s: cache, page table or lengths is NULL", what);
  if (!aligned16(cache)) return fail(B200_ATTN_UNSUPPORTED, "%s: the cache is not 16-byte aligned", what);
  return B200_ATTN_OK;
}

int check_heads(const char* what, const char* name, const void* p, const int64_t s[3], int batch, int tokens, int heads) {
  if (p == nullptr) return fail(B200_ATTN_BAD_CONFIG, "%s: %s is NULL", what, name);
  if (!rows_aligned(p, s, batch, tokens, heads, 2)) return fail(B200_ATTN_UNSUPPORTED, "%s: %s must be 16-byte aligned with strides in multiples of 8 elements", what, name);
  return B200_ATTN_OK;
}

int check_rows(const char* what, int64_t rows) {
  return rows <= INT32_MAX ? B200_ATTN_OK : fail(B200_ATTN_UNSUPPORTED, "%s: %lld heads of tokens, at most 2^31 - 1 a call", what, static_cast<long long>(rows));
}

void set_cache(Kv4Params* p, const B200Kv4Args* a, DeviceState* dev) {
  p->cache = static_cast<uint8_t*>(a->cache);
  p->page_table = a->page_table;
  p->table_stride = a->table_stride;
  p->lengths = a->lengths;
  p->tokens_magic = div_magic(a->tokens);
  p->page_magic = div_magic(a->page);
  p->tokens = a->tokens;
  p->q_heads = a->q_heads;
  p->kv_heads = a->kv_heads;
  p->page = a->page;
  p->pages = a->pages;
  p->table_pages = a->table_pages;
  p->status = dev->status;
}

template <typename T, int D>
const void* append_kernel_of(int form) {
  const void* k[4] = {reinterpret_cast<const void*>(kv4_append_kernel<T, D, kRowHalves>), reinterpret_cast<const void*>(kv4_append_kernel<T, D, kRowPairs>), reinterpret_cast<const void*>(kv4_append_kernel<T, D, kRowSplit>), reinterpret_cast<const void*>(kv4_append_kernel<T, D, kRowLoose>)};
  return k[form];
}

struct AttnForm {
  const void* kernel;
  int smem, rows, ctas_per_sm, threads, step, item;
};
// Rows of one kv head from which a call goes to the tcgen05 tiles. us, tiles and warps: 1 sequence of 9000 tokens, 64 rows 41 and 74; 8 of
// 2000, 64 rows 40 and 44; 16 of 700 at head dim 64, 40 rows 36 and 29. Between 40 and 64 rows, and over short contexts, nothing was measured.
constexpr int kTileRowsLeast = 49;
constexpr int kAttnForms = 5, kTileForm = 4;
template <typename T, int D, int NR, int RW>
AttnForm attn_form() {
  using S = Kv4AttnSmem<D, NR, RW>;
  return {reinterpret_cast<const void*>(kv4_attn_kernel<T, D, NR, RW>), S::kBytes, 8 * NR * RW, S::kCtasPerSm, kKv4AttnThreads, kKv4Step, kKv4Item};
}
template <typename T, int D>
AttnForm attn_form_of(int form) {
  if (form == kTileForm) return {reinterpret_cast<const void*>(kv4_tiles_kernel<T, D>), Kv4TilesSmem<D>::kBytes, kKv4TileRows, 1, kKv4TileThreads, kKv4TileStep, kKv4TileItem};
  return form == 0 ? attn_form<T, D, 1, 1>() : form == 1 ? attn_form<T, D, 2, 1>() : form == 2 ? attn_form<T, D, 2, 2>() : attn_form<T, D, 2, 4>();
}
std::atomic<bool> g_attn_opted_in[kMaxDevices][2][2][kAttnForms];

}  // namespace

}  // namespace b200

using namespace b200;

extern "C" {

int b200_rotary_workspace(int64_t* bytes) {
  if (bytes == nullptr) return fail(B200_ATTN_BAD_CONFIG, "bytes is NULL");
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  *bytes = kCounterBytes + int64_t(2) * dev->sms * kRotaryCtasPerSm * kMaxDim * 4;
  clear_error();
  return B200_ATTN_OK;
}

int b200_rotary(const B200RotaryArgs* a, void* stream_ptr) {
  if (a == nullptr) return fail(B200_ATTN_BAD_CONFIG, "args is NULL");
  if (a->struct_size != sizeof(B200RotaryArgs)) return fail(B200_ATTN_BAD_CONFIG, "struct_size %u does not match this library's B200RotaryArgs (%zu bytes)", a->struct_size, sizeof(B200RotaryArgs));
  if (a->dtype > B200_ATTN_F32) return fail(B200_ATTN_BAD_CONFIG, "rotary: dtype %u", a->dtype);
  if (a->norm && a->weight_dtype != a->dtype && a->weight_dtype != B200_ATTN_F32) return fail(B200_ATTN_BAD_CONFIG, "rotary: weight_dtype %u must be fp32 or that of x", a->weight_dtype);
  if (a->batch < 1 || a->tokens < 1 || a->tensors < 1 || a->tensors > 2) return fail(B200_ATTN_BAD_CONFIG, "rotary: batch %d, tokens %d, tensors %d", a->batch, a->tokens, a->tensors);
  if (a->head_dim < 1 || a->head_dim > kMaxDim) return fail(B200_ATTN_UNSUPPORTED, "rotary: head_dim %d must be 1 .. %d", a->head_dim, kMaxDim);
  if (int rc = check_table("rotary", a->cs, a->rot, a->head_dim, a->table_rows)) return rc;
  if (a->norm && !(a->eps >= 0.f)) return fail(B200_ATTN_BAD_CONFIG, "rotary: eps must not be negative");
  const int size = a->dtype == B200_ATTN_F32 ? 4 : 2;
  const bool reads_x = a->norm || !a->backward;
  RotaryParams p{};
  bool vec = true, sums = false;
  int64_t rows = 0;
  int heads = 0;
  for (int k = 0; k < a->tensors; ++k) {
    const B200Heads& h = a->heads[k];
    if (h.heads < 1) return fail(B200_ATTN_BAD_CONFIG, "rotary: tensor %d has %d heads", k, h.heads);
    if (h.y == nullptr || (reads_x && h.x == nullptr) || (a->backward && h.g == nullptr)) return fail(B200_ATTN_BAD_CONFIG, "rotary: a pointer of tensor %d is NULL", k);
    if ((reinterpret_cast<uintptr_t>(h.y) | (reads_x ? reinterpret_cast<uintptr_t>(h.x) : 0) | (a->backward ? reinterpret_cast<uintptr_t>(h.g) : 0)) % size != 0)
      return fail(B200_ATTN_UNSUPPORTED, "rotary: a pointer of tensor %d is not aligned to its type", k);
    vec = vec && rows_aligned(h.y, h.y_stride, a->batch, a->tokens, h.heads, size) && (!reads_x || rows_aligned(h.x, h.x_stride, a->batch, a->tokens, h.heads, size)) &&
          (!a->backward || rows_aligned(h.g, h.g_stride, a->batch, a->tokens, h.heads, size));
    RotaryTensor& t = p.t[k];
    const bool from_g = a->backward && !a->norm;  // the gradient alone goes through
    t.x = from_g ? h.g : h.x;
    t.y = h.y;
    t.g = h.g;
    t.w = a->norm ? h.w : nullptr;
    t.dw = a->norm && a->backward ? h.dw : nullptr;
    sums = sums || t.dw != nullptr;
    for (int i = 0; i < 3; ++i) t.xs[i] = from_g ? h.g_stride[i] : h.x_stride[i], t.ys[i] = h.y_stride[i], t.gs[i] = h.g_stride[i];
    t.heads = h.heads;
    const int64_t r = static_cast<int64_t>(a->batch) * a->tokens * h.heads;
    rows += r;
    if (int rc = check_rows("rotary", rows)) return rc;
    heads += h.heads;
  }
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  p.cs = a->cs;
  p.positions = a->positions;
  p.ps[0] = a->pos_stride[0];
  p.ps[1] = a->pos_stride[1];
  p.tokens_magic = div_magic(a->tokens);
  p.all_tokens = static_cast<uint32_t>(a->batch) * static_cast<uint32_t>(a->tokens);
  p.tensors = a->tensors;
  p.table_rows = a->table_rows;
  p.tokens = a->tokens;
  p.dim = a->head_dim;
  p.rot = a->rot;
  p.lanes_log2 = lanes_log2_of(a->head_dim);
  p.inv_dim = 1.f / static_cast<float>(a->head_dim);
  p.interleaved = a->interleaved != 0;
  p.w_f32 = a->weight_dtype == B200_ATTN_F32;
  p.vec = vec;
  p.eps = a->eps;
  p.sign = a->backward ? -1.f : 1.f;
  p.status = dev->status;
  // Rows of whole words on 16 bytes are streamed; halves whose partners lie in one lane are turned there, others through shared memory.
  const bool pairs = p.interleaved || a->rot == 0;
  const int form = !vec || a->head_dim % 8 != 0 ? kRowAny : pairs ? (a->rot % 8 == 0 && a->head_dim % 16 == 0 ? kRowPairs : kRowLoose) : a->head_dim % 16 == 0 && a->rot % 16 == 0 ? kRowHalves : kRowSplit;
  const int mode = !a->norm ? kTurn : a->backward ? kNormBack : kNormTurn;
  const RotaryForm kernel = a->dtype == B200_ATTN_F16 ? rotary_form_of<__half>(form, mode) : a->dtype == B200_ATTN_BF16 ? rotary_form_of<__nv_bfloat16>(form, mode) : rotary_form_of<float>(form, mode);
  // A token's rows go to as many groups of lanes as leave each of them four rows or more; calls of few tokens use more groups than that.
  const int groups = kRotaryThreads >> p.lanes_log2;
  const int64_t most = static_cast<int64_t>(dev->sms) * kernel.ctas_per_sm;
  int64_t ctas = 1;
  for (int k = 0; k < a->tensors; ++k) {
    const int heads = a->heads[k].heads;
    int g = 0;
    while (2 << g <= std::min(groups, heads / 4)) ++g;
    while (2 << g <= groups && 1 << g < heads && static_cast<int64_t>(p.all_tokens) * (1 << g) < most * groups) ++g;
    p.steps_log2[k] = g;
    ctas = std::max(ctas, std::min(most, (static_cast<int64_t>(p.all_tokens) * (1 << g) + groups - 1) / groups));
  }
  int smem = kernel.smem;
  if (form == kRowAny) smem = groups * p.dim * 4;
  if (mode == kNormBack) {
    smem = std::max({smem, kRotaryThreads / 32 * p.dim * 4, kRotaryThreads * 16});
    if (sums) {
      if (a->workspace == nullptr || !aligned16(a->workspace) || a->workspace_bytes < kCounterBytes + 2 * ctas * line_floats(p.dim) * 4)
        return fail(B200_ATTN_BAD_CONFIG, "rotary: the gradient of the weights needs a workspace (b200_rotary_workspace)");
      p.counter = static_cast<uint32_t*>(a->workspace);
      p.partial = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + kCounterBytes);
    }
  }
  if (form != kRowAny) {
    int device = 0;
    if (int rc = current_device(&device)) return rc;
    if (int rc = opt_in(g_rotary_opted_in[device][a->dtype][form][mode], kernel.kernel, kernel.smem, "rotary: shared memory opt-in")) return rc;
  }
  void* args[] = {&p};
  if (int rc = launch_kernel(kernel.kernel, static_cast<unsigned>(ctas), 1, kRotaryThreads, smem, 1, static_cast<cudaStream_t>(stream_ptr), args, "rotary kernel launch")) return rc;
  clear_error();
  return B200_ATTN_OK;
}

int b200_kv4_append(const B200Kv4Args* a, void* stream_ptr) {
  if (a == nullptr) return fail(B200_ATTN_BAD_CONFIG, "args is NULL");
  if (a->struct_size != sizeof(B200Kv4Args)) return fail(B200_ATTN_BAD_CONFIG, "struct_size %u does not match this library's B200Kv4Args (%zu bytes)", a->struct_size, sizeof(B200Kv4Args));
  if (int rc = check_cache("kv4_append", a->dtype, a->batch, a->tokens, a->kv_heads, a->head_dim, a->page, a->pages, a->table_pages, a->cache, a->page_table, a->lengths)) return rc;
  if (int rc = check_table("kv4_append", a->cs, a->rot, a->head_dim, a->table_rows)) return rc;
  const bool with_q = a->q != nullptr;
  if (with_q && a->q_heads < 1) return fail(B200_ATTN_BAD_CONFIG, "kv4_append: %d q heads", a->q_heads);
  if (int rc = check_heads("kv4_append", "k", a->k, a->k_stride, a->batch, a->tokens, a->kv_heads)) return rc;
  if (int rc = check_heads("kv4_append", "v", a->v, a->v_stride, a->batch, a->tokens, a->kv_heads)) return rc;
  if (with_q) {
    if (int rc = check_heads("kv4_append", "q", a->q, a->q_stride, a->batch, a->tokens, a->q_heads)) return rc;
    if (int rc = check_heads("kv4_append", "q_out", a->q_out, a->q_out_stride, a->batch, a->tokens, a->q_heads)) return rc;
  }
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  Kv4Params p{};
  set_cache(&p, a, dev);
  if (!with_q) p.q_heads = 0;
  p.heads = p.q_heads + 2 * a->kv_heads;
  const int64_t rows = static_cast<int64_t>(a->batch) * a->tokens * p.heads;
  if (int rc = check_rows("kv4_append", rows)) return rc;
  p.rows = static_cast<uint32_t>(rows);
  p.heads_magic = div_magic(p.heads);
  p.cs = a->cs;
  p.rot = a->rot;
  p.table_rows = a->table_rows;
  p.interleaved = a->interleaved != 0;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.q_out = a->q_out;
  for (int i = 0; i < 3; ++i) p.qs[i] = a->q_stride[i], p.ks[i] = a->k_stride[i], p.vs[i] = a->v_stride[i], p.qos[i] = a->q_out_stride[i];
  const bool pairs = p.interleaved || a->rot == 0;
  const int form = pairs ? (a->rot % 8 == 0 ? kRowPairs : kRowLoose) : a->rot % 16 == 0 ? kRowHalves : kRowSplit;
  const bool f16 = a->dtype == B200_ATTN_F16;
  const void* kernel = a->head_dim == 64 ? (f16 ? append_kernel_of<__half, 64>(form) : append_kernel_of<__nv_bfloat16, 64>(form))
                                         : (f16 ? append_kernel_of<__half, 128>(form) : append_kernel_of<__nv_bfloat16, 128>(form));
  const int groups = kKv4Threads / (a->head_dim / 16);
  void* args[] = {&p};
  if (int rc = launch_kernel(kernel, static_cast<unsigned>((rows + groups - 1) / groups), 1, kKv4Threads, 0, 1, static_cast<cudaStream_t>(stream_ptr), args, "kv4_append kernel launch")) return rc;
  clear_error();
  return B200_ATTN_OK;
}

int b200_kv4_read(const B200Kv4Args* a, void* stream_ptr) {
  if (a == nullptr) return fail(B200_ATTN_BAD_CONFIG, "args is NULL");
  if (a->struct_size != sizeof(B200Kv4Args)) return fail(B200_ATTN_BAD_CONFIG, "struct_size %u does not match this library's B200Kv4Args (%zu bytes)", a->struct_size, sizeof(B200Kv4Args));
  if (int rc = check_cache("kv4_read", a->dtype, a->batch, a->tokens, a->kv_heads, a->head_dim, a->page, a->pages, a->table_pages, a->cache, a->page_table, a->lengths)) return rc;
  if (int rc = check_heads("kv4_read", "k_out", a->k_out, a->k_out_stride, a->batch, a->tokens, a->kv_heads)) return rc;
  if (int rc = check_heads("kv4_read", "v_out", a->v_out, a->v_out_stride, a->batch, a->tokens, a->kv_heads)) return rc;
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  Kv4Params p{};
  set_cache(&p, a, dev);
  p.heads = a->kv_heads;
  const int64_t rows = static_cast<int64_t>(a->batch) * a->tokens * p.heads;
  if (int rc = check_rows("kv4_read", rows)) return rc;
  p.rows = static_cast<uint32_t>(rows);
  p.heads_magic = div_magic(p.heads);
  p.k_out = a->k_out;
  p.v_out = a->v_out;
  for (int i = 0; i < 3; ++i) p.kos[i] = a->k_out_stride[i], p.vos[i] = a->v_out_stride[i];
  const bool f16 = a->dtype == B200_ATTN_F16;
  const void* kernel = a->head_dim == 64 ? (f16 ? reinterpret_cast<const void*>(kv4_read_kernel<__half, 64>) : reinterpret_cast<const void*>(kv4_read_kernel<__nv_bfloat16, 64>))
                                         : (f16 ? reinterpret_cast<const void*>(kv4_read_kernel<__half, 128>) : reinterpret_cast<const void*>(kv4_read_kernel<__nv_bfloat16, 128>));
  const int groups = kKv4Threads / (a->head_dim / 16);
  void* args[] = {&p};
  if (int rc = launch_kernel(kernel, static_cast<unsigned>((rows + groups - 1) / groups), 1, kKv4Threads, 0, 1, static_cast<cudaStream_t>(stream_ptr), args, "kv4_read kernel launch")) return rc;
  clear_error();
  return B200_ATTN_OK;
}

int b200_kv4_workspace(int64_t* bytes, int64_t* counter_words) {
  if (bytes == nullptr || counter_words == nullptr) return fail(B200_ATTN_BAD_CONFIG, "bytes or counter_words is NULL");
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  const int64_t most_rows = std::max(kKv4CtasPerSm * kKv4MaxRows, kKv4TileRows);  // of the CTAs of one SM
  *bytes = dev->sms * 2 * most_rows * (128 * 4 + 8);
  *counter_words = static_cast<int64_t>(dev->sms) * kKv4CtasPerSm;
  clear_error();
  return B200_ATTN_OK;
}

int b200_kv4_attention(const B200Kv4AttnArgs* a, void* stream_ptr) {
  if (a == nullptr) return fail(B200_ATTN_BAD_CONFIG, "args is NULL");
  if (a->struct_size != sizeof(B200Kv4AttnArgs)) return fail(B200_ATTN_BAD_CONFIG, "struct_size %u does not match this library's B200Kv4AttnArgs (%zu bytes)", a->struct_size, sizeof(B200Kv4AttnArgs));
  if (int rc = check_cache("kv4_attention", a->dtype, a->batch, a->queries, a->kv_heads, a->head_dim, a->page, a->pages, a->table_pages, a->cache, a->page_table, a->lengths)) return rc;
  if (a->q_heads < 1 || a->q_heads % a->kv_heads != 0) return fail(B200_ATTN_BAD_CONFIG, "kv4_attention: %d q heads are no multiple of %d kv heads", a->q_heads, a->kv_heads);
  if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return fail(B200_ATTN_UNSUPPORTED, "kv4_attention: scale must be positive and finite");
  if (int rc = check_heads("kv4_attention", "q", a->q, a->q_stride, a->batch, a->queries, a->q_heads)) return rc;
  if (int rc = check_heads("kv4_attention", "o", a->o, a->o_stride, a->batch, a->queries, a->q_heads)) return rc;
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  const int group = a->q_heads / a->kv_heads;
  const int64_t rows = static_cast<int64_t>(a->queries) * group;
  if (int rc = check_rows("kv4_attention", rows * a->kv_heads * a->batch)) return rc;
  const int which = rows <= 8 ? 0 : rows <= 16 ? 1 : rows <= 32 ? 2 : rows < kTileRowsLeast ? 3 : kTileForm;
  const bool f16 = a->dtype == B200_ATTN_F16;
  const AttnForm form = a->head_dim == 64 ? (f16 ? attn_form_of<__half, 64>(which) : attn_form_of<__nv_bfloat16, 64>(which)) : (f16 ? attn_form_of<__half, 128>(which) : attn_form_of<__nv_bfloat16, 128>(which));
  Kv4AttnParams p{};
  p.cache = static_cast<const uint8_t*>(a->cache);
  p.page_table = a->page_table;
  p.table_stride = a->table_stride;
  p.lengths = a->lengths;
  p.q = a->q;
  p.o = a->o;
  for (int i = 0; i < 3; ++i) p.qs[i] = a->q_stride[i], p.os[i] = a->o_stride[i];
  p.page_blocks = a->page / kKv4Block;
  p.group_magic = div_magic(group);
  p.bpp_magic = div_magic(p.page_blocks);
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.batch = a->batch;
  p.queries = a->queries;
  p.q_heads = a->q_heads;
  p.kv_heads = a->kv_heads;
  p.group = group;
  p.rows = static_cast<int>(rows);
  p.row_tiles = static_cast<int>((rows + form.rows - 1) / form.rows);
  p.pages = a->pages;
  p.table_pages = a->table_pages;
  p.status = dev->status;
  // The lengths are on the device: the grid is for the longest that the page table allows, CTAs without a run leave at once.
  p.min_run = (which == kTileForm ? 2 : 4) + form.item;
  const int64_t most = static_cast<int64_t>(a->batch) * p.row_tiles * a->kv_heads * ((static_cast<int64_t>(a->table_pages) * a->page + form.step - 1) / form.step + form.item);
  if (most >= (int64_t(1) << 38)) return fail(B200_ATTN_UNSUPPORTED, "kv4_attention: %lld steps and items, at most 2^38 a call", static_cast<long long>(most));
  const int64_t ctas = std::min<int64_t>(static_cast<int64_t>(dev->sms) * form.ctas_per_sm, (most + p.min_run - 1) / p.min_run);
  const int64_t partial = ctas * 2 * form.rows * a->head_dim * 4, ml = ctas * 2 * form.rows * 8;
  if (a->workspace == nullptr || !aligned16(a->workspace) || a->workspace_bytes < partial + ml || a->counters == nullptr || a->counter_words < ctas)
    return fail(B200_ATTN_BAD_CONFIG, "kv4_attention: the workspace or the counters are missing or too small (b200_kv4_workspace)");
  p.partial = static_cast<float*>(a->workspace);
  p.partial_ml = reinterpret_cast<float2*>(static_cast<char*>(a->workspace) + partial);
  p.counters = a->counters;
  int device = 0;
  if (int rc = current_device(&device)) return rc;
  if (int rc = opt_in(g_attn_opted_in[device][f16 ? 0 : 1][a->head_dim == 64 ? 0 : 1][which], form.kernel, form.smem, "kv4_attention: shared memory opt-in")) return rc;
  const int64_t joins = static_cast<int64_t>(a->batch) * p.row_tiles * a->kv_heads * (kKv4TileRows / kKv4JoinRows);
  if (which == kTileForm && joins > INT32_MAX) return fail(B200_ATTN_UNSUPPORTED, "kv4_attention: too many rows");
  void* args[] = {&p};
  if (int rc = launch_kernel(form.kernel, static_cast<unsigned>(ctas), 1, form.threads, form.smem, 1, static_cast<cudaStream_t>(stream_ptr), args, "kv4_attention kernel launch")) return rc;
  if (which == kTileForm && ctas > 1) {
    const void* join = a->head_dim == 64 ? (f16 ? reinterpret_cast<const void*>(kv4_join_kernel<__half, 64>) : reinterpret_cast<const void*>(kv4_join_kernel<__nv_bfloat16, 64>))
                                         : (f16 ? reinterpret_cast<const void*>(kv4_join_kernel<__half, 128>) : reinterpret_cast<const void*>(kv4_join_kernel<__nv_bfloat16, 128>));
    int main_ctas = static_cast<int>(ctas);
    void* join_args[] = {&p, &main_ctas};
    if (int rc = launch_kernel(join, static_cast<unsigned>(joins), 1, kKv4JoinThreads, 0, 1, static_cast<cudaStream_t>(stream_ptr), join_args, "kv4_attention: launch of the join")) return rc;
  }
  clear_error();
  return B200_ATTN_OK;
}

}  // extern "C"
