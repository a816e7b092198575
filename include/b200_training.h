/*
 * b200_training.h - entry points of libb200attn.so for what stands between a model's last block and its gradients: layer
 * norm with its gradients, and the loss of an output layer (softmax cross entropy, or the divergence from a teacher's largest
 * logits) with the gradients of hidden states and weight, without the logits.
 *
 * Conventions are those of b200_attn.h: plain pointers and sizes, every buffer is the caller's, nothing is allocated and
 * nothing synchronises, all work is launched on `stream` of the current device, the return value is a status code. Workspaces need
 * no initial values and hold nothing from one call to the next.
 */
#ifndef B200_TRAINING_H_
#define B200_TRAINING_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Bits of b200_attn_status that these entry points set. */
#define B200_STATUS_TARGET (1u << 23)    /* a target or an entry's token past the vocabulary: NaN of its row */
#define B200_STATUS_HEAD_WAIT (1u << 24) /* a product gave up a bounded wait; its results are invalid */

/*
 * Layer norm of rows:  h = (x - mean(x)) * rsqrt(mean((x - mean(x))^2) + eps),  y = h * weight + bias
 * and, b200_layer_norm_grad, with t = dy * weight:
 *     dx = rsqrt(..) * (t - mean(t) - h * mean(t * h)),  dweight = sum over rows of dy * h,  dbias = sum over rows of dy
 * in fp32, rounded once; the sums over rows are taken in a fixed order. Row r of x, y, dy, dx begins at r * its stride (in
 * elements); rows may begin anywhere (16-byte boundaries and multiples are fastest). weight and bias are [dim] or NULL.
 */
typedef struct B200LayerNormArgs {
  uint32_t struct_size;  /* sizeof(B200LayerNormArgs) */
  uint32_t dtype;        /* of x, y, dy, dx: B200_ATTN_F16, B200_ATTN_BF16 or B200_ATTN_F32 */
  uint32_t weight_dtype; /* of weight, bias, dweight, dbias: `dtype` or B200_ATTN_F32 */
  int32_t dim;           /* 1 .. 32768 */
  int64_t rows;          /* 1 .. 2^31 - 1 */
  float eps;
  int32_t reserved;
  const void* x;
  int64_t x_stride;
  void* y;               /* forward; may be x */
  int64_t y_stride;
  const void* weight;
  const void* bias;
  float* stats;          /* [rows, 2] mean and rsqrt(..): written by b200_layer_norm (NULL: not), read by b200_layer_norm_grad */
  const void* dy;        /* gradient */
  int64_t dy_stride;
  void* dx;              /* NULL: not asked for */
  int64_t dx_stride;
  void* dweight;         /* NULL: not asked for */
  void* dbias;           /* NULL: not asked for */
  void* workspace;       /* dweight or dbias: b200_layer_norm_workspace bytes, 16-byte aligned */
  int64_t workspace_bytes;
} B200LayerNormArgs;

int b200_layer_norm(const B200LayerNormArgs* args, void* stream);
int b200_layer_norm_grad(const B200LayerNormArgs* args, void* stream);
int b200_layer_norm_workspace(const B200LayerNormArgs* args, int64_t* bytes);

/*
 * The loss of an output layer of weight w [vocab, dim] at rows x [rows, dim], logits l = x w^T + bias (never in memory):
 *     top = 0   loss_t = logsumexp(l_t) - l_t[targets[t]]; a row whose target is `ignore` does not count
 *     top > 0   z = l / tau; p = softmax(teacher[t] / tau) over the row's entries whose token (targets[t, k]) is not negative;
 *               loss_t = tau^2 * sum_k p_k (log p_k - z[token k] + logsumexp(z)); a row without an entry does not count
 * A token past the vocabulary makes NaN of its row (loss and gradients) and sets B200_STATUS_TARGET. Rows that do not count have loss 0 and no
 * gradient, and what x holds there is not looked at. The sum and the mean are over the rows that count, 0 where none does.
 * b200_head_grad gives dx = dl w, dw = dl^T x and dbias = sum over rows of dl, with dl = grad_t * tau * (softmax(z_t) - p at its tokens) held in `dtype` on its way into
 * the products (b200_head_grad, `whole` not 0: what that rounding takes goes through the products as well, half as many operations more; up to 128 rows or
 * 2^31 products it does in any case). It reads the `state` of the forward call, which may be shared by several calls and stays as it is.
 * Products accumulate in fp32; sums are taken in a fixed order.
 */
#define B200_HEAD_NONE 0 /* loss per row */
#define B200_HEAD_SUM 1
#define B200_HEAD_MEAN 2
typedef struct B200HeadArgs {
  uint32_t struct_size; /* sizeof(B200HeadArgs) */
  uint32_t dtype;       /* of x, w, dx, dw: B200_ATTN_F16 or B200_ATTN_BF16 */
  int32_t rows;         /* 1 .. 2^24 */
  int32_t dim;          /* a multiple of 8 up to 2^17 */
  int32_t vocab;        /* 1 .. 2^26 */
  int32_t top;          /* 0: cross entropy; 1 .. 256: entries of a row */
  int32_t reduction;    /* B200_HEAD_* */
  int32_t target_bytes; /* 4 or 8: int32 or int64 targets */
  uint32_t teacher_dtype;
  float tau;            /* top > 0 */
  const void* x;        /* rows ldx elements apart; 16-byte aligned, ldx a multiple of 8 */
  int64_t ldx;
  const void* w;        /* likewise */
  int64_t ldw;
  const void* targets;  /* [rows], or [rows, top] with rows targets_stride apart */
  int64_t targets_stride;
  int64_t ignore;       /* top = 0 */
  const void* teacher;  /* [rows, top], rows teacher_stride apart */
  int64_t teacher_stride;
  float* loss;          /* [rows], or one number (sum, mean) */
  void* state;          /* 256-byte aligned, as workspace */
  int64_t state_bytes;
  void* workspace;
  int64_t workspace_bytes;
  const float* grad;    /* gradient: of the loss, rows grad_stride apart, or one number */
  int64_t grad_stride;
  void* dx;             /* [rows, dim] contiguous, or NULL: not asked for */
  void* dw;             /* [vocab, dim] contiguous, or NULL: not asked for */
  const void* bias;     /* [vocab] of `dtype`, 16-byte aligned, or NULL */
  void* dbias;          /* [vocab] of `dtype`, 16-byte aligned, or NULL: not asked for */
  int32_t whole;        /* gradient, and its workspace: see above */
  int32_t reserved;
} B200HeadArgs;

int b200_head_loss(const B200HeadArgs* args, void* stream);
int b200_head_grad(const B200HeadArgs* args, void* stream);
/* Bytes of `state`, and of `workspace` for the loss and for the gradients, whichever of them are asked for. */
int b200_head_sizes(const B200HeadArgs* args, int64_t* state, int64_t* loss_workspace, int64_t* grad_workspace);

#ifdef __cplusplus
}
#endif

#endif /* B200_TRAINING_H_ */
