/*
 * C ABI of libi6train.so: the operators an emission model needs around the sequence losses of i6fbw.h, hand-written
 * for gfx950.  Three of them:
 *
 *   i6train_ce_*       output layer and frame-wise cross entropy of an alignment, without the (B, T, F) logits
 *   i6train_rec_*      gated recurrence over the frames of a batch, its gradient, and single frames with a state
 *   i6train_adamw      AdamW update of many tensors, states in 32 bits or in 8
 *
 * The conventions are those of i6fbw.h: all pointers are device pointers owned by the caller, every call is
 * asynchronous on `stream` (a hipStream_t), allocates no device memory and returns I6TRAIN_OK or a negative status
 * before anything is launched.  Workspaces are 256-byte aligned and not shared between calls in flight.  Strides are
 * in elements; innermost dimensions are contiguous.  No exception leaves the library.
 */
#ifndef I6TRAIN_H
#define I6TRAIN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. */
#define I6TRAIN_OK 0
#define I6TRAIN_ERR_INVALID_ARGUMENT (-1)
#define I6TRAIN_ERR_WORKSPACE_TOO_SMALL (-2)
#define I6TRAIN_ERR_LAUNCH (-3)
#define I6TRAIN_ERR_TOO_LARGE (-4)
/* device-side, reported by i6train_poll_status */
#define I6TRAIN_ERR_BAD_TARGET (-11)

/* Types of features, weights, gates, parameters and gradients. */
#define I6TRAIN_F32 0
#define I6TRAIN_BF16 1

const char* i6train_strerror(int code);

/*
 * What kernels of earlier calls on the current device have reported: *code is I6TRAIN_OK or a device-side code, *seq
 * the sequence it was seen on; the report is forgotten.  Reports are written to pinned host memory by the kernel that
 * sees the problem, so polling costs a read; it sees what has arrived and waits for nothing.
 */
int i6train_poll_status(int* code, int* seq);

/*
 * Cross entropy of an output layer.  For every frame t < seq_lens[b] with target y = targets[b, t] >= 0:
 *   z = weight . hidden[b, t] + bias,    loss[b, t] = log(sum_f exp z_f) - z_y
 * and 0 for every other frame (behind the end, or target < 0: no target); what such frames hold is not looked at.
 * A target >= F gives NaN in the frame's loss and in its row of grad_hidden, nothing in the gradients of the layer,
 * and a report.  seq_lens is clamped to [0, T].
 *
 *   hidden [B, T, D], weight [F, D], bias [F] or null, all of `dtype`;  targets int32 [B, T];  seq_lens int32 [B]
 *   loss   float [B, T]
 *
 * The forward call leaves in `workspace` what the backward call needs: keep it until then (it may be used for several
 * backward calls; hidden, weight and bias have to be what they were).  Logits exist in registers only; the backward call forms them again, in pieces of the
 * vocabulary.  Sums and statistics are held in 32 bits.
 * bfloat16: logits are formed from the operands as they are.  The gradient with respect to the logits is rounded to 11 bits before
 * it is multiplied, with operands that are exact down to 2^-29 of their tensor's largest value.
 * 32 bits: operands and the gradient with respect to the logits are held in 22 bits, down to 2^-29 of the largest value of a tensor.
 * Where that is too little for a row (of hidden or weight: a geometric mean of the values other than 0 below 2^-26 of the tensor's largest value, in
 * bfloat16 2^-20, or an incoming gradient below 2^-22 of the largest, 2^-16), which the device finds out, 32-bit products are formed from the values as they are, and
 * bfloat16 ones with the gradient with respect to the logits rounded to bfloat16.  Rows of zeros do not count.  So what a frame, a class or a feature holds changes
 * the precision of the others' results, at most within these bounds, and 32-bit calls become up to five times slower.
 * grad_loss is float [B, T] with strides; grad_hidden [B, T, D], grad_weight [F, D] and grad_bias [F] are of `dtype`,
 * contiguous, and written completely; each of them may be null.  Both
 * calls read hidden and weight.
 * Sizes: B T and F up to 2^22, ceil(B T / 128) ceil(F / 256) below 2^24, D up to 2^14; larger ones are I6TRAIN_ERR_TOO_LARGE.
 */
typedef struct {
    int B, T, F, D, dtype;
    const void* hidden;  int64_t hidden_stride_b, hidden_stride_t;
    const void* weight;  int64_t weight_stride_f;
    const void* bias;
    const int32_t* targets;  int64_t targets_stride_b, targets_stride_t;
    const int32_t* seq_lens;
} i6train_ce_problem;

int i6train_ce_workspace_size(const i6train_ce_problem* p, size_t* forward_bytes, size_t* backward_bytes);
int i6train_ce_forward(const i6train_ce_problem* p, float* loss, void* workspace, size_t workspace_bytes, void* stream);
int i6train_ce_backward(const i6train_ce_problem* p, const float* grad_loss, int64_t grad_stride_b, int64_t grad_stride_t,
                        void* grad_hidden, void* grad_weight, void* grad_bias,
                        const void* forward_workspace, size_t forward_bytes,
                        void* workspace, size_t workspace_bytes, void* stream);

/*
 * Gated recurrence.  With f = 1 / (1 + exp(-gate)), for t < seq_lens[b]:
 *   h[b, t] = f[b, t] h[b, t-1] + (1 - f[b, t]) x[b, t],    h[b, -1] = initial[b] (0 without)
 * h is 0 behind the end of a sequence; last[b] is the state after its last frame (initial[b] if it has none).  The
 * state is held in 32 bits; h is rounded to `dtype` as it is written.  seq_lens null: all sequences have T frames.
 * x, gate [B, T, D] of `dtype` with strides; h [B, T, D] contiguous; initial, last float [B, D] contiguous.
 * Sizes: B up to 65 535, T up to 2^30, D below 2^29.
 *
 * `states` (may be null) receives what i6train_rec_backward needs: the state in front of every span of frames, float,
 * i6train_rec_states_size bytes.  `workspace` is used where one sequence is worked on by several workgroups.
 * Backward: grad_h (strided, `dtype`) and grad_last (float [B, D] contiguous) may be null; grad_x, grad_gate [B, T, D]
 * of `dtype` and grad_initial float [B, D] are written completely, zeros behind the end; grad_initial may be null.
 */
typedef struct {
    int B, T, D, dtype;
    const void* x;  int64_t x_stride_b, x_stride_t;
    const void* gate;  int64_t gate_stride_b, gate_stride_t;
    const int32_t* seq_lens;
    const float* initial;
} i6train_rec_problem;

int i6train_rec_states_size(const i6train_rec_problem* p, size_t* bytes);
int i6train_rec_workspace_size(const i6train_rec_problem* p, size_t* bytes);
int i6train_rec_forward(const i6train_rec_problem* p, void* h, float* last, float* states, void* workspace,
                        size_t workspace_bytes, void* stream);
int i6train_rec_backward(const i6train_rec_problem* p, const void* grad_h, int64_t grad_stride_b, int64_t grad_stride_t,
                         const float* grad_last, const float* states, void* grad_x, void* grad_gate, float* grad_initial,
                         void* workspace, size_t workspace_bytes, void* stream);

/*
 * One AdamW step over n_tensors tensors.  For every value, in 32 bits:
 *   m = beta1 m + (1 - beta1) g,    v = beta2 v + (1 - beta2) g^2
 *   p = p (1 - lr weight_decay) - lr / (1 - beta1^step)  m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 *
 * state_bits 32: exp_avg and exp_avg_sq are float.  state_bits 8: exp_avg holds m and exp_avg_sq the square root of v,
 * both in the 8-bit floating-point format with 4 exponent and 3 mantissa bits (bias 7, no infinities), each block of
 * I6TRAIN_BLOCK consecutive values with a float scale of its own, largest finite magnitude / 448 (2^-100 at least).  What is
 * not finite is held as NaN, and the others of its block are as without it.  Values are rounded up
 * or down so that m and v keep their means over the steps: with the place j in the block and s = step, the two turns
 *   um = ((j PHI + s ROOT) mod 2^32) >> 16,  uv = ((j ROOT + s PHI) mod 2^32) >> 16,  PHI 2654435769, ROOT 1779033703
 * are compared, as fractions of 2^16, with where the value stands between its neighbours.  A root that is not zero does not
 * become zero.
 */
#define I6TRAIN_BLOCK 256
typedef struct {
    void* param;             /* dtype */
    const void* grad;        /* dtype */
    void* exp_avg;           /* float, or 8-bit values */
    void* exp_avg_sq;
    float* exp_avg_scale;    /* state_bits 8: ceil(n / I6TRAIN_BLOCK) floats each */
    float* exp_avg_sq_scale;
    int64_t n;               /* values, fewer than 2^36; 0 is allowed */
} i6train_adamw_tensor;

/* `tensors` is a host array. */
int i6train_adamw(const i6train_adamw_tensor* tensors, int n_tensors, int dtype, int state_bits, int64_t step, double lr,
                  double beta1, double beta2, double eps, double weight_decay, void* stream);

#ifdef __cplusplus
}
#endif
#endif
