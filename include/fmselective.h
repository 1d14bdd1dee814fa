/*
 * fmselective.h -- C ABI of libfmscan_hip.so, second part: the operators of a selective state space
 * layer for AMD MI355X (gfx950), for training, for prompts and for single tokens.
 *
 *   short convolution   y[b,d,t] = act(bias[d] + sum_j weight[d,j] x[b,d,t-W+1+j]),  W taps, depthwise
 *   selective scan      dt = softplus(delta + delta_bias),  h[n] = exp(dt A[d,n]) h[n] + dt u write[n],
 *                       out = (sum_n read[n] h[n] + skip[d] u) * silu(gate)
 *   norm                r = inputs + residual,  out = r / sqrt(mean r^2 + eps) * weight, optionally in 8 bits
 *
 * The conventions are those of fmscan.h: device pointers on the current GPU, kernels enqueued on `stream`
 * (a hipStream_t), nothing kept between calls, no memory owned, 0 or an FMSCAN_E_* code or a positive
 * hipError_t back, the text from fmscan_last_error(). The reference has no counterpart of these operators.
 *
 * Sequences are time last. Inputs (B, D, L) may have any batch and channel stride (in elements, >= 0); the
 * time stride is 1. Outputs are dense. Parameters (weight, bias, skip, delta_bias) are float32 or of the
 * inputs' element type, one FMSELECTIVE_NARROW_* flag each for the latter.
 *
 * lengths (B) int32 or NULL: the steps that count of each row of a padded batch, clamped to [0, L]. Beyond
 * them inputs are not read, outputs and gradients are zero, and the final state is that after the last
 * step that counts (the initial state where none does).
 *
 * slots (B) int32 or int64, or NULL (row b has slot b, and there are B slots): where in the pool of states a
 * row of a single-token call has its state. A row whose slot is outside [0, S) is skipped: it gives zeros and
 * touches no state. Where a slot is named more than once the first row takes it and the later ones are
 * skipped in the same way.
 */
#ifndef FMSELECTIVE_H_
#define FMSELECTIVE_H_

#include "fmscan.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FMSELECTIVE_SOFTPLUS        0x1u  /* scan, step: dt = softplus(delta + delta_bias), else the sum itself */
#define FMSELECTIVE_SILU            0x2u  /* convolution: silu of the sum */
#define FMSELECTIVE_SLOTS_64        0x4u  /* slots are int64 */
#define FMSELECTIVE_NARROW_WEIGHT   0x10u /* weight has the inputs' element type */
#define FMSELECTIVE_NARROW_BIAS     0x20u /* so has bias or delta_bias */
#define FMSELECTIVE_NARROW_SKIP     0x40u /* so has skip */

/* ---- short convolution --------------------------------------------------------------------------------
 * W is 2, 3 or 4. bias, initial_state, lengths and final_state may be NULL.
 *   inputs (B, D, L) strided, weight (D, W), bias (D), initial_state (B, D, W-1): the inputs before the first
 *   out (B, D, L), final_state (B, D, W-1): the last W-1 inputs that count (out) */
int fmselective_conv_forward(const void* inputs, int64_t batch_stride, int64_t channel_stride, const void* weight,
                             const void* bias, const void* initial_state, const int32_t* lengths, void* out,
                             void* final_state, int64_t B, int64_t D, int64_t L, int64_t W, int dtype,
                             unsigned flags, void* stream);

/* Bytes of workspace that the backward call needs (its partial sums of the parameters' gradients); 0 where the
 * sizes are not valid. */
size_t fmselective_conv_workspace_bytes(int64_t B, int64_t D, int64_t L, int64_t W, int dtype);

/* Gradients. out_grad (B, D, L) strided; final_state_grad (B, D, W-1) or NULL; inputs_grad (B, D, L) dense;
 * weight_grad (D, W), bias_grad (D) or NULL, of the types of weight and bias; initial_state_grad (B, D, W-1) or
 * NULL. `bias` is needed for the silu. */
int fmselective_conv_backward(const void* inputs, int64_t batch_stride, int64_t channel_stride, const void* out_grad,
                              int64_t grad_batch_stride, int64_t grad_channel_stride, const void* weight,
                              const void* bias, const void* initial_state, const void* final_state_grad,
                              const int32_t* lengths, void* inputs_grad, void* weight_grad, void* bias_grad,
                              void* initial_state_grad, int64_t B, int64_t D, int64_t L, int64_t W, int dtype,
                              unsigned flags, void* workspace, size_t workspace_bytes, void* stream);

/* One token of every row. inputs (B, D) with a row stride, state and state_out (S, D, W-1) dense; state_out may be
 * state (updated in place) or another pool, of which the named slots alone are written. out (B, D) dense. */
int fmselective_conv_step(const void* inputs, int64_t batch_stride, const void* state, void* state_out,
                          const void* weight, const void* bias, const void* slots, void* out, int64_t B, int64_t D,
                          int64_t W, int64_t S, int dtype, unsigned flags, void* stream);

/* ---- selective scan ------------------------------------------------------------------------------------
 *   dt = softplus(delta + delta_bias),  h[b,d,n] <- exp(dt A[d,n]) h[b,d,n] + dt tokens[b,d,t] write[b,g,n,t]
 *   out[b,d,t] = (sum_n read[b,g,n,t] h[b,d,n] + skip[d] tokens[b,d,t]) * silu(gate[b,d,t])
 * with channel d in group g = d / (D / G). tokens, delta, gate (B, D, L) and write, read (B, G, N, L) have one
 * element type and any strides but the time's, which is 1; A (D, N), states and their gradients are float32.
 * gate, skip, delta_bias, initial_state and lengths may be NULL. 1 <= N <= FMSELECTIVE_MAX_STATES, G divides D.
 * Products of decays over many steps are taken: where A is positive they must stay finite in float32. A may be minus
 * infinity: such a state holds the last step's term alone, and a step of length zero leaves it as it is. */
#define FMSELECTIVE_MAX_STATES 256
#define FMSELECTIVE_MARK 128 /* steps between the states that forward saves for backward */

typedef struct fmselective_scan_inputs {
    const void *tokens, *delta, *gate, *write, *read, *skip, *delta_bias;
    const float *A, *initial_state;
    const int32_t* lengths;
    int64_t tokens_strides[2], delta_strides[2], gate_strides[2]; /* batch, channel */
    int64_t write_strides[3], read_strides[3];                    /* batch, group, state */
    int64_t B, D, L, N, G;
    int32_t dtype;
    uint32_t flags;
} fmselective_scan_inputs;

/* Rows that are too few to fill the GPU are cut along time; what passes between the pieces goes through a workspace.
 * The forward call takes NULL (rows are then scanned in one piece, the same results up to rounding), the backward
 * call needs its own, which holds its partial sums too. Bytes that a call of these sizes can use; 0 where none or
 * where the sizes are not valid.
 * Backward's is mostly the partial sums of write's and read's gradients, 1 KiB for every 16 channels of a group, state and
 * FMSELECTIVE_MARK steps, begun ones included: about B D L N / 2 bytes, so 269 MB at (8, 2048, 2048) with N = 16 and one group; as
 * much for a group of one channel as for one of 16, for one step as for 128. */
size_t fmselective_scan_workspace_bytes(int64_t B, int64_t D, int64_t L, int64_t N, int64_t G, int dtype, int backward);

/* out (B, D, L); final_state (B, D, N) or NULL; marks (B, D, ceil(L / FMSELECTIVE_MARK), N) float32 or NULL: the
 * states before every FMSELECTIVE_MARK steps, which the backward call needs (those at or beyond a row's length
 * are not specified). */
int fmselective_scan_forward(const fmselective_scan_inputs* in, void* out, float* final_state, float* marks, void* workspace,
                             size_t workspace_bytes, void* stream);

typedef struct fmselective_scan_grads {
    const void* out_grad;           /* (B, D, L), strided */
    int64_t out_grad_strides[2];
    const float* final_state_grad;  /* (B, D, N) or NULL */
    const float* marks;             /* as forward wrote them */
    void *tokens, *delta, *gate;    /* (B, D, L) dense; gate NULL where the inputs' is */
    void *write, *read;             /* (B, G, N, L) dense */
    float *A, *initial_state;       /* (D, N); (B, D, N) or NULL */
    void *skip, *delta_bias;        /* (D), of the parameters' types, NULL where the inputs' are */
} fmselective_scan_grads;

int fmselective_scan_backward(const fmselective_scan_inputs* in, const fmselective_scan_grads* grads, void* workspace,
                              size_t workspace_bytes, void* stream);

/* One token of every row. tokens, delta, gate (B, D) with a row stride (tokens_strides[0], ...), write and read
 * (B, G, N) with a batch and a group stride (the first two), L and lengths unused, initial_state the pool
 * (S, D, N) dense. state_out may be the pool (updated in place) or another, of which the named slots alone are
 * written. out (B, D) dense. */
int fmselective_scan_step(const fmselective_scan_inputs* in, float* state_out, const void* slots, int64_t S, void* out,
                          void* stream);

/* ---- root-mean-square norm with the residual's addition ------------------------------------------------
 *   r = inputs + residual (rounded to the element type, as it is stored), inv = 1 / sqrt(mean r^2 + eps)
 *   out = r inv weight
 * over `rows` dense rows of D elements, 1 <= D <= FMSELECTIVE_MAX_NORM. residual may be NULL (r is inputs, nothing
 * is stored). Squares are summed in float32. With eps = 0 a row whose mean square is zero there (zeros, or a root mean
 * square below 2^-75) has inv 0 and gives zeros; so does a row of finite values whose sum is infinite (from 2^128 on).
 * inv_rms (rows) float32 may be NULL; the backward call needs it. With scales (rows) float32 the output
 * is 8-bit e4m3 instead, one byte an element: scales = max |out| / 448 of the row, values out / scale, in float32, rounded
 * to nearest even: where the quotient of unrounded numbers is halfway, float32's own roundings decide (a row of zeros, or
 * of values below 2^-100, has scale 0 and zeros; one with a NaN among its outputs has a NaN scale). */
#define FMSELECTIVE_MAX_NORM 16384
int fmselective_norm_forward(const void* inputs, const void* residual, const void* weight, void* residual_out, void* out,
                             float* scales, float* inv_rms, int64_t rows, int64_t D, int dtype, unsigned flags, float eps,
                             void* stream);

size_t fmselective_norm_workspace_bytes(int64_t rows, int64_t D, int dtype);

/* stream_in: r as forward stored it (the inputs without a residual). residual_grad: the gradient that arrives at r
 * from elsewhere, or NULL. grad: that of inputs and of residual, which is the same. */
int fmselective_norm_backward(const void* out_grad, const void* residual_grad, const void* stream_in, const void* weight,
                              const float* inv_rms, void* grad, void* weight_grad, int64_t rows, int64_t D, int dtype,
                              unsigned flags, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
