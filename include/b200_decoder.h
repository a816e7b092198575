/*
 * b200_decoder.h - entry points of libb200attn.so for the layers of a token decoder (and of blocks that norm their q and
 * k): rotary positions, norms of the heads of q and k, a paged cache of keys and values held in 4 bits, and attention
 * over it.
 *
 * Conventions are those of b200_attn.h: plain pointers and sizes, every buffer is the caller's, nothing is allocated and
 * nothing synchronises, all work is launched on `stream` of the current device, the return value is a status code.
 * A tensor of heads is addressed as element (b, n, head, d) at ptr + b*stride[0] + n*stride[1] + head*stride[2] + d
 * (strides in elements). What a kernel finds wrong in index tensors (a position past the table, a page outside the cache)
 * reads and writes nothing out of range, and a bit of the word that b200_attn_status returns says so: a token is not turned, a place is
 * not written, reads as zeros, and makes NaN of the attention of queries that see it.
 */
#ifndef B200_DECODER_H_
#define B200_DECODER_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Bits of b200_attn_status that these entry points set. */
#define B200_STATUS_POSITION (1u << 20) /* a position past the rows of the table: the token was not rotated */
#define B200_STATUS_PAGE (1u << 21)     /* a page outside the cache, or a length past the page table: nothing is read or written there */
#define B200_STATUS_KV4_WAIT (1u << 22) /* attention over the cache gave up a bounded wait; its output is invalid */

/* One tensor of heads and what belongs to it. */
typedef struct B200Heads {
  const void* x;
  void* y;          /* result: the rotated (and normed) heads, or, backward, the gradient of x; may be x itself */
  const void* g;    /* backward: gradient of the forward's result */
  const void* w;    /* norm: weight [head_dim] or NULL (all ones) */
  void* dw;         /* norm, backward: gradient of w, or NULL */
  int64_t x_stride[3];
  int64_t y_stride[3];
  int64_t g_stride[3];
  int32_t heads;
  int32_t reserved;
} B200Heads;

/*
 * Rotary positions of one or two tensors of heads, with or without the root-mean-square norm of each head in front:
 *     h = x * rsqrt(mean(x^2) + eps) * w                    (norm; else h = x)
 *     y_a = h_a cos - h_b sin,  y_b = h_b cos + h_a sin     for the rot / 2 pairs (a, b), y = h for the other dimensions
 * pairs (j, j + rot / 2), or (2 j, 2 j + 1) if `interleaved`. `cs` is fp32 [table_rows, 2, rot / 2] = cos | sin; token
 * (b, n) takes row positions[b*pos_stride[0] + n*pos_stride[1]] (NULL: row n); a negative position is not rotated.
 * backward = 1: y gets the gradient of x from g (x is read with a norm only), dw that of w. Everything is computed in
 * fp32 and rounded once. The sum over tokens behind dw is taken in a fixed order.
 */
typedef struct B200RotaryArgs {
  uint32_t struct_size;  /* sizeof(B200RotaryArgs) */
  uint32_t dtype;        /* of x, y, g: B200_ATTN_F16, B200_ATTN_BF16 or B200_ATTN_F32 */
  uint32_t weight_dtype; /* of w and dw: `dtype` or B200_ATTN_F32 */
  int32_t batch;
  int32_t tokens;
  int32_t head_dim; /* 1 .. 512 */
  int32_t rot;      /* even, 0 .. head_dim; 0: nothing is rotated */
  int32_t interleaved;
  int32_t norm;
  int32_t backward;
  int32_t tensors; /* 1 or 2 */
  float eps;
  const float* cs;
  int32_t table_rows;
  int32_t reserved;
  const int32_t* positions;
  int64_t pos_stride[2];
  B200Heads heads[2];
  void* workspace; /* norm, backward: b200_rotary_workspace bytes, the first 256 of them zero (left zero) */
  int64_t workspace_bytes;
} B200RotaryArgs;

int b200_rotary(const B200RotaryArgs* args, void* stream);
int b200_rotary_workspace(int64_t* bytes);

/*
 * The cache: uint8 [pages, kv_heads, page / 16, 16 * (head_dim + 8)], contiguous, 16-byte aligned. A block holds sixteen
 * tokens of one head: their codes of K, head_dim / 2 bytes each, dimension 2 i in the low and 2 i + 1 in the high half of
 * byte i; then for each two tokens a row of head_dim + 16 bytes: the codes of V in 16-bit words (word i: dimensions
 * 4 i .. 4 i + 3, the first in the lowest bits), the words of the even and the odd token in turn, then for either token
 * four bfloat16: step and least value of K, step and least value of V. A value is least + step * code.
 * Token p of sequence b lies in page page_table[b * table_stride + p / page]. `lengths` counts the tokens of a sequence,
 * those of the call among them: token i of `tokens` is at position lengths[b] - tokens + i; negative ones are padding.
 *
 * b200_kv4_append writes k and v, k rotated before (table and layout as above, rot = 0: not), and, q != NULL, q rotated
 * into q_out. A head's vector is a group of its own: step = bf16((max - min) / 15), least = bf16(min),
 * code = clamp(round((x - least) / step), 0, 15); a step below 2^-126 counts as 0; a group whose range is not finite is NaN.
 * b200_kv4_read writes the values of the last `tokens` tokens to k_out and v_out, [batch, tokens, kv_heads, head_dim] of
 * `dtype`, zeros for padding (q, k, v, cs are not looked at).
 */
typedef struct B200Kv4Args {
  uint32_t struct_size; /* sizeof(B200Kv4Args) */
  uint32_t dtype;       /* B200_ATTN_F16 or B200_ATTN_BF16 */
  int32_t batch;
  int32_t tokens;
  int32_t q_heads;
  int32_t kv_heads;
  int32_t head_dim; /* 64 or 128 */
  int32_t rot;
  int32_t interleaved;
  int32_t page;  /* tokens in a page, a multiple of 16 */
  int32_t pages; /* in the cache */
  int32_t table_pages; /* columns of the page table */
  void* cache;
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* lengths;
  const float* cs;
  int32_t table_rows;
  int32_t reserved;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_out;
  void* v_out;
  int64_t q_stride[3];
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t q_out_stride[3];
  int64_t k_out_stride[3];
  int64_t v_out_stride[3];
} B200Kv4Args;

int b200_kv4_append(const B200Kv4Args* args, void* stream);
int b200_kv4_read(const B200Kv4Args* args, void* stream);

/*
 * Causal attention of the last `queries` tokens of each sequence over the cache, lengths and pages as above: query i is
 * at position lengths[b] - queries + i and sees the keys up to its own; o is zero where that leaves none, and NaN where a key lies on
 * a page outside the cache. A length past the page table counts as the table's end. q_heads is a
 * multiple of kv_heads, consecutive q heads share a kv head. Logits, sums and the output's accumulator are fp32; q and the
 * softmax weights go to the tensor cores as fp16 (q scaled by a power of two for each row, so that nothing is out of range).
 * `workspace`: b200_kv4_workspace bytes for partial results; `counters`: as many zeroed 32-bit words as that call
 * says, left zero. Launches that may run at the same time need their own.
 */
typedef struct B200Kv4AttnArgs {
  uint32_t struct_size; /* sizeof(B200Kv4AttnArgs) */
  uint32_t dtype;
  int32_t batch;
  int32_t queries;
  int32_t q_heads;
  int32_t kv_heads;
  int32_t head_dim;
  int32_t page;
  int32_t pages;
  int32_t table_pages;
  float scale; /* positive */
  int32_t reserved;
  const void* cache;
  const int32_t* page_table;
  int64_t table_stride;
  const int32_t* lengths;
  const void* q;
  void* o;
  int64_t q_stride[3];
  int64_t o_stride[3];
  void* workspace;
  int64_t workspace_bytes;
  uint32_t* counters;
  int64_t counter_words;
} B200Kv4AttnArgs;

int b200_kv4_attention(const B200Kv4AttnArgs* args, void* stream);
int b200_kv4_workspace(int64_t* bytes, int64_t* counter_words);

#ifdef __cplusplus
}
#endif

#endif /* B200_DECODER_H_ */
