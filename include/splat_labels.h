/* splat_labels.h — features and labels of Gaussians or pixels (libsplat_b200.so): the codebook
 * (embedding) a scene's Gaussians take their features from, and the label head that classifies
 * features against a vocabulary of labels. No counterpart in the reference, which learns colour
 * only.
 *
 * The conventions are those of splat.h: every call returns an sp_status, work is enqueued in call
 * order on the context's stream and nothing here waits for it except the *_check calls; device
 * pointers are borrowed; a handle owns its workspace and is used from one host thread at a time.
 * Calls on one handle share its workspace, so they belong on its context's stream.
 *
 * Matrices are row-major with unit column stride; a row stride counts elements and is at least
 * the column count. Elements are SP_F32 or SP_BF16, one type per handle. Any element-aligned
 * pointer and any such stride is accepted; bf16 matrices whose base is 16-byte aligned and whose
 * row stride is a multiple of 8 elements are read in place by the label head, others are copied
 * first. Tokens and labels are 32- or 64-bit signed; one outside [0, entries) (or [0, labels))
 * means "none". Outputs must not overlap inputs.
 *
 * Arithmetic: sums, softmax statistics and losses are held in 32 bits or more whatever the element
 * type; results do not depend on scheduling (the same call gives the same bits). */
#ifndef SPLAT_LABELS_H
#define SPLAT_LABELS_H

#include "splat.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum sp_element { SP_F32 = 0, SP_BF16 = 1 } sp_element;
typedef enum sp_index { SP_INDEX32 = 0, SP_INDEX64 = 1 } sp_index;

/* ------------------------------------------------------------------ embedding */

/* A table of `entries` rows of `dim` features looked up by token, and the gradient of its rows.
 * `max_tokens` bounds the tokens of one call (below 2^30); entries below 2^31, dim below 2^20. */
typedef struct sp_embedding sp_embedding;
sp_status sp_embedding_create(sp_context* ctx, uint64_t entries, uint32_t dim, sp_element element,
                              uint64_t max_tokens, sp_embedding** out);
void sp_embedding_destroy(sp_embedding* e);
/* out[i] = scale * table[tokens[i]], rounded once to the element type; a zero row for a token that
 * is none. */
sp_status sp_embedding_lookup(sp_embedding* e, const void* d_table, int64_t table_stride, const void* d_tokens,
                              sp_index index, uint64_t count, float scale, void* d_out, int64_t out_stride);
/* table_gradient[v] = scale * sum over i with tokens[i] = v of out_gradient[i], for every entry v
 * (zero rows included), summed in f32 in an order fixed by the tokens alone: the (token, position)
 * pairs are sorted by the renderer's radix sort and each token's rows summed in position order within
 * fixed pieces. */
sp_status sp_embedding_gradient(sp_embedding* e, const void* d_out_gradient, int64_t out_gradient_stride,
                                const void* d_tokens, sp_index index, uint64_t count, float scale,
                                void* d_table_gradient, int64_t table_gradient_stride);
/* Waits for the stream; SP_ERR_TIMEOUT when a device wait of an earlier gradient gave up (that
 * gradient is NaN throughout), and clears it. */
sp_status sp_embedding_check(sp_embedding* e);

/* ----------------------------------------------------------------- label head */

/* Logits z[i][v] = logit_scale * <features[i], weight[v]> over `labels` labels, never stored: the
 * products run in tiles on the tensor cores, and each tile is reduced (or turned into its gradient)
 * where it was made. f32 operands are split into three bf16 parts each (24 bits for
 * magnitudes from 2^-110 on, any finite or infinite value) and their six largest partial products are
 * summed; an infinite feature that meets an infinite weight gives NaN.
 * The tensor cores truncate their f32 sums, 16 products an addition. Of each addition's loss, 2^-23 of the sum at
 * most, an eighth of 2^-23 is given back for up to 257 additions, the mean for terms of both signs: logits over 512
 * such columns are good to 5e-7 of their size, exact ones (features of a single 1) are off by 5e-7 at 512 columns
 * and 3.8e-6 from 4096 on, and sums of one sign by up to a 2^-24 an addition. Wider features' sums lose an eighth
 * of 2^-23 for each 16 columns past 4096. `max_rows` bounds the rows of one call;
 * it and labels are below 2^31 - 512, dim below 2^20. `training` != 0 also reserves the gradient's workspace. */
typedef struct sp_label_head sp_label_head;
sp_status sp_label_head_create(sp_context* ctx, uint64_t labels, uint32_t dim, sp_element element, uint64_t max_rows,
                               int training, sp_label_head** out);
void sp_label_head_destroy(sp_label_head* h);
/* Cross entropy of each row's target: losses[i] = log_normalizers[i] - z[i][targets[i]] with
 * log_normalizers[i] = log sum_v exp z[i][v] (f64: a confident row's slope is the small difference of
 * its target's logit and this); *mean = the mean over the rows with a target (0 when
 * there is none). A row without a target is skipped, whatever its features hold: 0 in both
 * outputs. A label whose logit is -inf, or as low as the element type goes, has probability 0 beside
 * others; a row with a logit of NaN or +inf, or with all of them -inf, gets NaN. logit_scale > 0 and
 * finite. */
sp_status sp_label_head_loss(sp_label_head* h, const void* d_features, int64_t feature_stride, const void* d_weight,
                             int64_t weight_stride, const void* d_targets, sp_index index, uint64_t rows,
                             float logit_scale, float* d_mean, float* d_losses, double* d_log_normalizers);
/* The gradient of sum_i g[i] losses[i], g = d_row_gradient (rows floats), or with NULL of the mean
 * (g[i] = 1 / rows with a target). Both gradients are overwritten; a row without a target gets a
 * zero row and adds nothing to the weight's. `d_log_normalizers` are those of this
 * handle's sp_label_head_loss for the same features, weight, targets and scale: a confident row's slope is the
 * difference of its logit and its normalizer, which have to come from logits of the same rounding (another
 * handle, not made for training, may sum them in another order). Needs a handle made for training. Before the
 * second products the softmax slopes are kept to 24 bits (f32) or rounded to bf16, without the mean's factor;
 * the weight's gradient takes them to 16 bits where rows are at most 128, or rows times labels at most 2^21, or
 * with d_row_gradient. */
sp_status sp_label_head_gradient(sp_label_head* h, const void* d_features, int64_t feature_stride,
                                 const void* d_weight, int64_t weight_stride, const void* d_targets, sp_index index,
                                 uint64_t rows, float logit_scale, const double* d_log_normalizers,
                                 const float* d_row_gradient, void* d_feature_gradient,
                                 int64_t feature_gradient_stride, void* d_weight_gradient,
                                 int64_t weight_gradient_stride);
/* Each row's most probable label (the lowest of equal ones) and its log-probability. A row with a logit of NaN or
 * +inf, or with all of them -inf, gets the label of its largest that is a number (0 without one) and NaN. */
sp_status sp_label_head_predict(sp_label_head* h, const void* d_features, int64_t feature_stride,
                                const void* d_weight, int64_t weight_stride, uint64_t rows, float logit_scale,
                                int32_t* d_labels, float* d_log_probabilities);
/* Waits for the stream; SP_ERR_TIMEOUT when a device wait of an earlier call gave up (that call's
 * losses, log-probabilities and gradients are NaN), and clears it. */
sp_status sp_label_head_check(sp_label_head* h);

#ifdef __cplusplus
}
#endif

#endif /* SPLAT_LABELS_H */
