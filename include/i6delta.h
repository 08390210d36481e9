/*
 * C ABI of libi6train.so, second part: a recurrence over the frames of a batch whose state is a matrix for each head.
 * Conventions, types and status codes are those of i6train.h.
 *
 * With f = 1 / (1 + exp(-gate)), w = 1 / (1 + exp(-beta)) and q, k scaled to length one (q / sqrt(q.q + 1e-6)), for every
 * sequence b, head h and t < seq_lens[b]:
 *   S'     = f[t] S[t-1]                                  S: K rows, V columns;  S[-1] = initial (0 without)
 *   S[t]   = S' + k[t] (w[t] (v[t] - S'^T k[t]))^T        what the key holds is replaced by v to the share w
 *   o[t]   = S[t]^T q[t]
 * o is 0 behind the end of a sequence; last is the state after its last frame (initial if it has none).  What frames behind
 * the end hold is not looked at.  seq_lens null: all sequences have T frames; it is clamped to [0, T].
 *
 *   q, k [B, T, G, K], v [B, T, H, V], gate, beta [B, T, H], all of `dtype`, with strides (q, k, v: the last one is 1); H is a multiple
 *   of G, and head h has keys and queries h / (H / G).  initial, last float [B, H, K, V] contiguous;  o [B, T, H, V] contiguous, of `dtype`.
 *
 * States, sums and decays are held in 32 bits.  Of bfloat16 inputs, products take their 32-bit operands in three bfloat16 parts (24 bits) where results are of 32 bits and in two (16 bits) where
 * they are of bfloat16, and a forward call for training keeps states and written rows in two such parts for the gradients.  Sums of squares of q and of k have to be below 2^127.  Sizes: B and H up to 65 535, K and V up to 128, B H ceil(T / 32) up to 2^23; larger ones
 * are I6TRAIN_ERR_TOO_LARGE.
 *
 * A forward call for training leaves in `kept` what i6delta_backward needs (null otherwise).  Gradients: grad_o (strided, last stride 1, `dtype`)
 * and grad_last (float, contiguous) may be null; grad_q, grad_k [B, T, G, K], grad_v [B, T, H, V], grad_gate and grad_beta [B, T, H] of `dtype`
 * and grad_initial float [B, H, K, V] (may be null) are contiguous and written completely, zeros behind the end.
 * Results do not depend on the run.
 */
#ifndef I6DELTA_H
#define I6DELTA_H

#include "i6train.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    int B, T, H, G, K, V, dtype;
    const void* q;  int64_t q_stride_b, q_stride_t, q_stride_g;
    const void* k;  int64_t k_stride_b, k_stride_t, k_stride_g;
    const void* v;  int64_t v_stride_b, v_stride_t, v_stride_h;
    const void* gate;  int64_t gate_stride_b, gate_stride_t, gate_stride_h;
    const void* beta;  int64_t beta_stride_b, beta_stride_t, beta_stride_h;
    const int32_t* seq_lens;
    const float* initial;
} i6delta_problem;

/* Bytes of `kept` and of the workspaces of a forward call, with `train` or without, and of a backward call; each may be 0.  They are those of calls with this very problem: with
 * other places and strides of q, k and v they may be others. */
int i6delta_sizes(const i6delta_problem* p, int train, size_t* kept_bytes, size_t* forward_bytes, size_t* backward_bytes);
int i6delta_forward(const i6delta_problem* p, void* o, float* last, void* kept, size_t kept_bytes, void* workspace, size_t workspace_bytes,
                    void* stream);
int i6delta_backward(const i6delta_problem* p, const void* grad_o, int64_t grad_stride_b, int64_t grad_stride_t, int64_t grad_stride_h,
                     const float* grad_last, const void* kept, size_t kept_bytes, void* grad_q, void* grad_k, void* grad_v, void* grad_gate,
                     void* grad_beta, float* grad_initial, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
