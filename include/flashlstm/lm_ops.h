/* Operators around the recurrent layers of a language model, for MI355X (gfx950): layer norm on a residual stream.
 * They have no counterpart in the reference, which is an LSTM layer alone.
 *
 * All pointers are device pointers.  Every function only enqueues work on `stream`: it allocates nothing, waits for nothing and
 * reads nothing back, so it may be recorded into a graph.  Tensors hold one of the types of flstm_op_dtype; parameters,
 * statistics, states and losses are fp32, and all sums are.  Nothing is required of the alignment of tensors beyond that of
 * their element type.  Offsets are 64 bits wide.
 * Every function returns 0 on success, a hipError_t value on a HIP failure, or a FLSTM_E_* code (lstm_core.h); nothing is
 * enqueued when an argument is refused.  Sizes of zero are no error: there is then nothing to do but what is documented.
 */
#ifndef FLASHLSTM_LM_OPS_H_
#define FLASHLSTM_LM_OPS_H_

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { FLSTM_OP_F32 = 0, FLSTM_OP_F16 = 1, FLSTM_OP_BF16 = 2 } flstm_op_dtype;

/* ---- layer norm on a residual stream
 *
 * total = x + residual, rounded to the tensors' type (residual null: total = x, and `total` is not written);
 * mean, rstd = 1 / sqrt(var + eps) over a row of total; y = (total - mean) * rstd * weight + bias.
 * weight and bias may be null (ones, zeros).  Rows of x and residual are ldx and ldr elements apart, total and y are contiguous.
 * total, mean and rstd are what the backward pass reads; mean and rstd may be null where there will be none.
 * total and y may lie in x's or residual's place where that one is contiguous.  width is at most 16384.
 *
 * Backward, of the gradients dy of y and d_total of total (null: none):
 *   h = dy * weight;  n = (total - mean) * rstd;
 *   dx = rstd * (h - mean(h) - n * mean(h n)) + d_total   (the gradient of x and of residual alike)
 *   dweight = sum over rows of dy n;  dbias = sum over rows of dy   (each may be null)
 * dx is contiguous and may lie in the place of a contiguous dy or d_total.  The sums over rows are made in an order that depends on the
 * sizes alone.  `workspace` has flstm_layer_norm_workspace_bytes() bytes, 16-byte aligned; it may be null where dweight and
 * dbias are. */
int flstm_layer_norm_forward(size_t rows, size_t width, const void* x, size_t ldx, const void* residual, size_t ldr,
                             flstm_op_dtype dtype, const float* weight, const float* bias, float eps, void* total, void* y,
                             float* mean, float* rstd, void* stream);
size_t flstm_layer_norm_workspace_bytes(size_t rows, size_t width);
int flstm_layer_norm_backward(size_t rows, size_t width, const void* dy, size_t lddy, const void* total, size_t ldt,
                              const void* d_total, size_t lddt, flstm_op_dtype dtype, const float* weight, const float* mean,
                              const float* rstd, void* dx, float* dweight, float* dbias, void* workspace, void* stream);

#ifdef __cplusplus
}
#endif
#endif  /* FLASHLSTM_LM_OPS_H_ */
