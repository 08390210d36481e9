/*
 * C ABI of libi6train.so, fourth part: the orthogonal factor of matrices by Newton-Schulz products, and the step of an optimiser on it.
 * Conventions, types and status codes are those of i6train.h.
 *
 * X = u / max(|u|, 1e-7), |u| the root of the sum of squares; `iterations` times
 *   A = X X^T,   X = 3.4445 X + (-4.7750 A + 2.0315 A A) X
 * (u transposed where it has more rows than columns, and the result back).  Singular values of X end near one.
 * X, A and the factors are held in 22 bits relative to the largest value they can have (2^-39 at least), sums in 32.  For 16-bit results the
 * last product takes 11 bits of its operands.
 *
 * Where `momentum` is given, u comes from the gradient g and is applied to the parameter p:
 *   m = mu m + (1 - mu) g,   u = nesterov ? mu m + (1 - mu) g : m,   p = p keep - rate X
 * with `keep` and `rate` for each tensor.
 */
#ifndef I6ORTH_H
#define I6ORTH_H

#include "i6train.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    const void* update;      /* u, or g where there is a momentum: [rows][cols] contiguous, dtype */
    void* result;            /* X, or p, which is read too: [rows][cols] contiguous, dtype */
    float* momentum;         /* m [rows][cols], or null: for all tensors of a call that have values, or none */
    int rows, cols;          /* up to 2^15 each; 0 is allowed */
    float keep, rate;
} i6orth_tensor;

/* `tensors` is a host array; `workspace` has i6orth_workspace_size bytes.  That is 12 to 20 bytes a value (rows and columns rounded up to 64) of as many matrices as are worked on at the same time: up to 34 and 4 GB of it, or one matrix that
 * has more alone, and up to 32 MB that they share.  Other matrices of the call follow in the same memory. */
int i6orth_workspace_size(const i6orth_tensor* tensors, int n_tensors, int dtype, size_t* bytes);
int i6orth_step(const i6orth_tensor* tensors, int n_tensors, int dtype, int iterations, double mu, int nesterov, void* workspace,
                size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
