/*
 * minigo_ops.h - C ABI of the training operators of a move-sequence policy:
 * embedding lookup, linear layer and linear cross entropy, each with its
 * gradient.  Exported by libminigo_cuda.so next to the evaluation engine
 * (minigo_cuda.h).  The reference trains in Python (scripts/train.py) and has
 * no native counterpart of these.
 *
 * Calls are stateless: every pointer is device memory of args->device, work
 * is enqueued on `stream` (a cudaStream_t of that device, NULL for its
 * default stream) and the call returns without waiting.  No call allocates
 * device memory; one that needs scratch is given it as `workspace`
 * (256-byte aligned, at least the bytes that the matching *_workspace call
 * reports for the same arguments), which must stay untouched until the
 * enqueued work has finished.  Calls on different streams may overlap if
 * their workspaces and outputs differ.  Calls can be captured into a CUDA
 * graph after one call on the device outside a capture.
 *
 * Each call returns MG_OK or a negative MG_E_* code (minigo_cuda.h);
 * mg_op_error() then describes the calling thread's last failure.  Nothing
 * throws across this boundary.  Arguments are checked before anything is
 * enqueued; token and target values are data and never fault: a value
 * outside its vocabulary is padding (tokens) or not counted (targets).
 *
 * Results do not depend on the order in which thread blocks run: the same
 * call on the same inputs gives the same bits.
 *
 * Strides count elements.  Matrices are [rows][cols] with any row and column
 * strides (a column stride of 1 with a row stride that is a multiple of 8
 * and a 16-byte aligned base is read in place; the transposed form too;
 * others are first copied to the workspace).  Outputs are dense row-major.
 * Every pointer is aligned to its elements.
 */
#ifndef MINIGO_OPS_H
#define MINIGO_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "minigo_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types reuse MG_PREC_BF16 / MG_PREC_FP16 / MG_PREC_FP32. */

/* Activations of mg_linear. */
#define MG_ACT_NONE 0
#define MG_ACT_RELU 1
#define MG_ACT_SILU 2 /* z / (1 + exp(-z))              */
#define MG_ACT_GELU 3 /* z (1 + erf(z / sqrt 2)) / 2    */

/* Message describing the calling thread's last failed mg_* operator call. */
const char* mg_op_error(void);

/* Waits for `stream` and returns MG_E_DEVICE if a kernel of these operators
 * gave up a bounded wait on `device` since the last such call (its outputs
 * are then invalid), MG_E_CUDA if the stream reports an error, else MG_OK. */
int mg_op_synchronize(int device, void* stream);

/* y[i] = scale * table[tokens[i]] for n tokens and rows of dim elements;
 * a zero row where tokens[i] is outside [0, vocab). */
typedef struct mg_embed_args {
    const void* tokens;  /* [n] int64 (or int32), element stride token_stride */
    const void* table;   /* [vocab][dim], row stride table_row, column stride 1 */
    void* out;           /* [n][dim] dense */
    int64_t n, vocab, dim;
    int64_t token_stride, table_row;
    float scale;
    int32_t dtype;        /* MG_PREC_* of table and out */
    int32_t token_bytes;  /* 8 or 4 */
    int32_t device;
} mg_embed_args;
int mg_embed(const mg_embed_args* args, void* stream);

/* d_table[v] = scale * sum of grad[i] over the i with tokens[i] == v, zero
 * for entries that no token names; summed in 32 bits, in an order given by
 * the tokens alone, rounded once. */
typedef struct mg_embed_backward_args {
    const void* tokens;  /* [n] */
    const void* grad;    /* [n][dim], row stride grad_row, column stride 1 */
    void* d_table;       /* [vocab][dim] dense */
    int64_t n, vocab, dim;
    int64_t token_stride, grad_row;
    float scale;
    int32_t dtype;        /* MG_PREC_* of grad and d_table */
    int32_t token_bytes;  /* 8 or 4 */
    int32_t device;
} mg_embed_backward_args;
int mg_embed_backward_workspace(const mg_embed_backward_args* args, size_t* bytes);
int mg_embed_backward(const mg_embed_backward_args* args, void* workspace, size_t workspace_bytes,
                      void* stream);

/* z = x weight^T + bias;  y = act(z) + residual_scale * residual.
 * x [m][k], weight [n][k], bias [n] dense or NULL, residual [m][n] or NULL;
 * y [m][n]; z [m][n] or NULL (kept for the backward pass).  Sums in 32 bits,
 * y and z each rounded once.  BF16 or FP16; m may be 0, n and k may not. */
typedef struct mg_linear_args {
    const void* x;
    const void* weight;
    const void* bias;
    const void* residual;
    void* y;
    void* z;
    int64_t m, n, k;
    int64_t x_row, x_col, w_row, w_col, r_row, r_col;
    float residual_scale;
    int32_t activation; /* MG_ACT_* */
    int32_t dtype;
    int32_t device;
} mg_linear_args;
int mg_linear_workspace(const mg_linear_args* args, size_t* bytes);
int mg_linear(const mg_linear_args* args, void* workspace, size_t workspace_bytes, void* stream);

/* Gradients of mg_linear from grad = dL/dy [m][n] and the kept z:
 * g = grad * act'(z), rounded to the operands' type (unless there is no
 * activation); dx = g weight [m][k], dw = g^T x [n][k], db = sum of g over
 * rows [n] or NULL.  dx and dw may be NULL to leave them out.  act' of RELU
 * is 0 at z = 0, and where it is 0 so is g, whatever grad holds.  The
 * residual's gradient is residual_scale * grad and needs no kernel. */
typedef struct mg_linear_backward_args {
    const void* grad;
    const void* x;
    const void* weight;
    const void* z; /* [m][n]; unused for MG_ACT_NONE */
    void* dx;
    void* dw;
    void* db;
    int64_t m, n, k;
    int64_t g_row, g_col, x_row, x_col, w_row, w_col, z_row, z_col;
    int32_t activation;
    int32_t dtype;
    int32_t device;
    int32_t reserved; /* 0 */
} mg_linear_backward_args;
int mg_linear_backward_workspace(const mg_linear_backward_args* args, size_t* bytes);
int mg_linear_backward(const mg_linear_backward_args* args, void* workspace, size_t workspace_bytes,
                       void* stream);

/* Softmax cross entropy of l = x weight^T + bias against target indices,
 * without keeping the logits: x [n][dim], weight [vocab][dim], bias [vocab]
 * dense or NULL (-inf bans an entry).
 *   row_loss[i] = logsumexp(l[i]) - l[i][t_i], 0 where t_i is outside
 *                 [0, vocab) (a row that is not counted);
 *   loss        = sum of row_loss / number of counted rows, 0 if none is.
 * A counted row whose logits are all -inf, or whose target is banned, has
 * row_loss +inf.
 * With dx, dw (and db where there is a bias) set, also the gradients of
 * grad_scale * loss: d = (softmax(l) - onehot(t)) * grad_scale / counted
 * (softmax 0 where every logit is -inf), dx = d weight, dw = d^T x, db = sum
 * of d over rows; rows that are not counted give nothing, whatever x holds
 * there (an infinity or NaN in weight shows in every row's dx).  d is rounded
 * to the operands' type once; before that, probabilities are held to 2^-14 of
 * themselves, and to 2^-28 of the largest of up to 128 neighbouring classes
 * where they are below 2^-14 of it.  FP16 gradients are small: give a grad_scale
 * that keeps them in range.  All three gradients, or none, except that db
 * is NULL without a bias.  n may be 0; vocab and dim may not.  n, vocab and dim
 * are below 2^31 - 1024. */
typedef struct mg_cross_entropy_args {
    const void* x;
    const void* weight;
    const void* bias;
    const void* targets; /* [n] int64 (or int32), element stride target_stride */
    float* loss;         /* [1] */
    float* row_loss;     /* [n] */
    void* dx;            /* [n][dim] or NULL */
    void* dw;            /* [vocab][dim] or NULL */
    void* db;            /* [vocab] or NULL */
    int64_t n, vocab, dim;
    int64_t x_row, x_col, w_row, w_col, target_stride;
    float grad_scale;
    int32_t dtype;
    int32_t target_bytes; /* 8 or 4 */
    int32_t device;
} mg_cross_entropy_args;
int mg_cross_entropy_workspace(const mg_cross_entropy_args* args, size_t* bytes);
int mg_cross_entropy(const mg_cross_entropy_args* args, void* workspace, size_t workspace_bytes,
                     void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MINIGO_OPS_H */
