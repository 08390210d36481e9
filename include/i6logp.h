/*
 * C ABI of libi6train.so, third part: log probabilities of given classes, entropy and best alternatives of every frame, from the
 * scores of all classes.  Conventions, types and status codes are those of i6train.h.
 *
 * With p = softmax(logits[b, t]), for every frame t < seq_lens[b]:
 *   log_prob[b, t]     = log p_y, y = targets[b, t]; 0 where y < 0 (no target); NaN, and a report, where y >= F
 *   entropy[b, t]      = - sum_f p_f log p_f
 *   top_class[b, t, j] = the class with the j-th largest score, j < k, the lowest index first among equal ones; top[b, t, j] = its log p
 * Frames behind the end (seq_lens is clamped to [0, T]) are not looked at: 0, 0, 0 and class -1.
 * Scores of -inf are classes without probability.  A frame of nothing else has no distribution: its log probabilities are -inf, its entropy
 * is 0, its alternatives are the first k classes, and its gradient is 0.  A frame that holds NaN or +inf: NaN and class -1.
 *
 *   logits [B, T, F] of `dtype` with strides, the last one 1;  targets int32 [B, T] with strides;  seq_lens int32 [B]
 *   log_prob, entropy float [B, T];  top float, top_class int32 [B, T, k], k <= 64 and k <= F; all contiguous
 *
 * Gradient, for the incoming gl of log_prob, ge of entropy and gt of top (float, contiguous; each may be null):
 *   grad_logits_f = gl [f = y] + sum_j gt_j [f = top_class_j] - p_f (gl + sum_j gt_j + ge (log p_f + entropy))
 * written completely, contiguous, of `dtype`, zeros behind the end, NaN where y >= F.  Sums and statistics are held in 32 bits; shares below 2^-126 of a
 * frame's largest are 0.
 * Sizes: F up to 2^28; B T below 2^22, below 2^26 where F is 512 or less; larger ones are I6TRAIN_ERR_TOO_LARGE.
 */
#ifndef I6LOGP_H
#define I6LOGP_H

#include "i6train.h"

#ifdef __cplusplus
extern "C" {
#endif

#define I6LOGP_MOST_ALTERNATIVES 64

typedef struct {
    int B, T, F, k, dtype;
    const void* logits;  int64_t logits_stride_b, logits_stride_t;
    const int32_t* targets;  int64_t targets_stride_b, targets_stride_t;
    const int32_t* seq_lens;
} i6logp_problem;

/* `statistics` float [B, T, 4], 16-byte aligned (may be null): what the backward call needs besides the problem, entropy and top_class. */
int i6logp_forward(const i6logp_problem* p, float* log_prob, float* entropy, float* top, int32_t* top_class, float* statistics, void* stream);
int i6logp_backward(const i6logp_problem* p, const float* statistics, const int32_t* top_class, const float* grad_log_prob,
                    const float* grad_entropy, const float* grad_top, void* grad_logits, void* stream);

#ifdef __cplusplus
}
#endif
#endif
