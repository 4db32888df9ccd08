/*
 * rafhip_vocab.h -- C ABI of the gfx950 (MI355X) operators at the vocabulary: the token embedding
 * with its gradient, and the distillation loss against a teacher's top logits with its gradient.
 * They are the two ends of a language model's training step that produce the gradients which the
 * optimizer steps of rafhip_optim.h consume; the embedding gradient is usually the longest tensor
 * of such a list.
 *
 * The rules of rafhip_optim.h hold: plain C, device pointers, a HIP stream as void*, a
 * rafhip_status from every function unless noted, the message from rafhip_last_error(), no
 * exception, no device allocation.  Tensors and workspaces belong to the current device.  Nothing
 * is kept between calls, so calls on different streams may overlap if their workspaces differ.
 * Results do not depend on the launch, the stream or the run: every sum is taken in an order that
 * the data fixes.
 *
 * An output or workspace that shares bytes with an input, or with another output, is refused
 * (RAFHIP_ERR_INVALID_ARG): the kernels read while they write.  A matrix of rows that lie apart
 * counts from its first element to its last.
 *
 * Element types: RAFHIP_F32, RAFHIP_F16 and RAFHIP_BF16 in any mixture; indices are signed, of
 * index_bits 32 or 64.  Everything is computed in fp32 or wider and rounded once on store.
 * Pointers need their element's alignment only.
 *
 * Reference operators (paths relative to the reference tree): `raf.op.embedding(x, indices)` and
 * `raf.op.embedding_dx(dy, indices, num_weight)`, src/op/dialect/cuda/embedding.cc and
 * kernels/embedding_dx_cuda.cu.  The distillation loss has no counterpart there.
 */
#ifndef RAFHIP_VOCAB_H_
#define RAFHIP_VOCAB_H_

#include "rafhip_optim.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------------------ embedding
 *     y[t, :] = scale * x[indices[t] - first_row, :]
 * for n indices and a table x of rows x width (contiguous).  An index outside
 * [first_row, first_row + rows) -- another shard's, or a negative one that marks nothing -- gives a
 * row of zeros.  first_row >= 0 places a vocabulary shard.
 * y: n x width of y_dtype, contiguous.  n, rows and width may be 0.
 */
int rafhip_embedding(const void* x, int32_t x_dtype, int64_t rows, int64_t width, const void* indices,
                     int32_t index_bits, int64_t n, int64_t first_row, float scale, void* y,
                     int32_t y_dtype, void* stream);

/*
 * Its gradient for the table,
 *     dx[r, :] = (accumulate ? dx[r, :] : 0) + scale * sum of dy[t, :] over t with indices[t] - first_row == r,
 * over all rows x width of dx.  Tokens are sorted by row and each row's are added in an order
 * fixed by their positions, 32 (up to 256 tokens: all) in fp32 and these sums in fp64, so equal inputs give
 * equal bits.  Indices outside the table and,
 * with has_padding, indices equal to padding_index take no part (their dy is not read).  With
 * accumulate, rows without a token keep their bits.
 * dy: n x width of dy_dtype, dx: rows x width of dx_dtype, contiguous.
 * workspace: rafhip_embedding_dx_workspace_bytes(n, rows, width) bytes (0 for short calls, then it
 * may be NULL), 16-byte aligned, no initialisation needed.  That function is host arithmetic; it returns -1 for
 * sizes that are not supported: 2^21 rows or more, 2^24 columns or more, or more tokens than 512
 * sort tiles hold (8,388,608 tokens below 2^18 rows, half of that for each doubling of the rows
 * from there).
 */
int64_t rafhip_embedding_dx_workspace_bytes(int64_t n, int64_t rows, int64_t width);
int rafhip_embedding_dx(const void* dy, int32_t dy_dtype, const void* indices, int32_t index_bits, int64_t n,
                        int64_t rows, int64_t width, int64_t first_row, int32_t has_padding,
                        int64_t padding_index, float scale, void* dx, int32_t dx_dtype, int32_t accumulate,
                        void* workspace, int64_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------- top-k distillation
 * The loss of a student's logits z against the top logits of a teacher, row by row,
 *     loss = soft_weight * T^2 * KL(p || softmax(z / T)) + hard_weight * -log softmax(z)[label]
 *     KL   = sum_j p_j (log p_j - log softmax(z / T)[topk_indices[j]]),   p = softmax_j(topk_logits / T)
 * and its gradient, with the upstream gradient dloss of the row,
 *     dz = dloss * (soft_weight * T * (softmax(z / T) - p) + hard_weight * (softmax(z) - onehot(label))).
 * T = temperature.  The softmax over z runs over all `vocab` columns; p is a distribution over the
 * teacher's entries, of which those with an index outside [0, vocab) or a logit of -inf are absent.
 * The same index twice counts with both its entries.  A row without entries has no soft term, one
 * whose label is missing (labels NULL, or outside [0, vocab)) no hard term; a row with neither has
 * loss 0 and a gradient of zeros, and its logits are not read, so padded rows may hold anything.
 * Logits of -inf have probability zero; a row of nothing else, +inf and NaN give NaN.
 * Columns are summed in fp32, at most 256 one after the other, and these sums and the row's values in
 * fp32 or fp64; the gradient is rounded once.
 */
typedef struct rafhip_topk_distill_args {
  const void* logits;       /* rows x vocab, rows `row_stride` elements apart                  */
  const void* topk_indices; /* rows x topk, contiguous                                         */
  const void* topk_logits;  /* rows x topk, contiguous                                         */
  const void* labels;       /* rows, or NULL                                                   */
  int64_t rows;             /* below 2^31                                                      */
  int64_t vocab;            /* columns that take part: fewer than 2^28                         */
  int64_t row_stride;       /* >= vocab, below 2^28                                            */
  int32_t topk;             /* 0 .. RAFHIP_MAX_TOPK                                            */
  int32_t logits_dtype;
  int32_t topk_dtype;
  int32_t index_bits;       /* of topk_indices and labels                                      */
  float temperature;        /* > 0, finite                                                     */
  float soft_weight;
  float hard_weight;
} rafhip_topk_distill_args;
#define RAFHIP_MAX_TOPK 1024

/* Scratch of the forward and of the combined call (0 where a row needs no help; 16-byte aligned,
 * no initialisation); -1 for invalid sizes.  Host arithmetic. */
int64_t rafhip_topk_distill_workspace_bytes(const rafhip_topk_distill_args* args);

/* Forward: loss[rows] and, for the gradient call, stats[rows][3] (fp32 both; stats may be NULL):
 * the largest logit m, log sum exp((z - m) / T) and log sum exp(z - m); a sum that the row's loss
 * does not need is 0, and so is m in a row without targets. */
int rafhip_topk_distill(const rafhip_topk_distill_args* args, float* loss, float* stats, void* workspace,
                        int64_t workspace_bytes, void* stream);

/* Gradient from the forward call's stats (same args).  dloss: `dloss_count` fp32 values, rows of
 * them or one for all rows.  dlogits: rows x out_width of the logits' dtype, contiguous,
 * out_width >= vocab; the columns behind vocab are written as zeros. */
int rafhip_topk_distill_dx(const rafhip_topk_distill_args* args, const float* dloss, int64_t dloss_count,
                           const float* stats, void* dlogits, int64_t out_width, void* stream);

/* Both at once, for a training step that knows the upstream gradient beforehand (a weight per row
 * times the loss scale): each logit is read once from memory where a row fits the registers of a
 * workgroup (204,800 columns of 16 bits, 98,304 of fp32; 24,576 where there are 64 rows or
 * fewer: several workgroups then read a row twice sooner).  loss and dlogits as above. */
int rafhip_topk_distill_step(const rafhip_topk_distill_args* args, const float* dloss, int64_t dloss_count,
                             float* loss, void* dlogits, int64_t out_width, void* workspace,
                             int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RAFHIP_VOCAB_H_ */
