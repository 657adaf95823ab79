/* Operators around the recurrent layers of a language model, for MI355X (gfx950): layer norm on a residual stream, attention
 * whose memory is a decaying state of fixed size, and the distillation loss against a teacher's top logits.
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

/* ---- attention with a decaying state
 *
 * For every sequence and head, with a decay g = exp(log_decay[head]) of the head's own (log_decay <= 0; minus infinity: no
 * memory), over the sequence's tokens t:
 *   S_t = g S_{t-1} + k_t v_t^T   (dk x dv, S before the first token = state_in or zeros)
 *   o_t = scale * S_t^T q_t
 * heads must be a multiple of kv_heads; query head h reads key and value head h / (heads / kv_heads).
 * 8 <= dk, dv <= 256.  States are contiguous fp32 (sequences, heads, dk, dv).
 *
 * A tensor's element (sequence, token, head, i) lies at data + sequence * .sequence + token * .token + head * .head + i elements.
 * With cu_seqlens (sequences + 1 int32 on the device) sequences are packed along the token axis: sequence n is tokens
 * [cu_seqlens[n], cu_seqlens[n + 1]) of `tokens` in all, and .sequence is not used.  A tensor's tokens may be any distance apart up to 2^23 elements
 * (FLSTM_E_TOO_LARGE beyond; from 2^21 pairs of a sequence and a head on it may also be the answer, where their workgroups are
 * more than a launch can have).  cu_seqlens must ascend from 0.  Bounds are clamped to 0 .. tokens, so that nothing
 * outside the tensors is touched whatever they are, but where they do not ascend outputs are not specified.  Tokens behind the last
 * bound get zeros.  An empty sequence's final state is its initial one.
 * What a NaN or an infinity of an input reaches by these formulas is not finite, and nothing else is changed by it.  In all but
 * flstm_decay_attention_step it may be a NaN where the formulas have an infinity: values are added to the state in parts and heads are
 * padded with zeros.
 * Outputs and gradients are those of 32 bits, rounded once.  fp16: a state is held under a power of two and fades below 2^-100; what is
 * added to it (a value times its decay to the end of its chunk of 64 tokens) is held to 2^-22 of the largest of the chunk, whatever keys
 * it meets, or of the state. */
typedef struct {
    void* data;
    ptrdiff_t sequence, token, head;
} flstm_rows;

typedef struct {
    size_t sequences, tokens;
    const int* cu_seqlens;
    int heads, kv_heads, dk, dv;
    flstm_op_dtype dtype;
    float scale;
    const float* log_decay;
} flstm_decay_attention;

/* state_in (null: zeros) and state_out may be null; they must not be one buffer.
 * `workspace` has flstm_decay_attention_workspace_bytes(shape, 0) bytes (16-byte aligned; null where that is 0). */
int flstm_decay_attention_forward(const flstm_decay_attention* shape, const flstm_rows* q, const flstm_rows* k, const flstm_rows* v,
                                  const float* state_in, const flstm_rows* o, float* state_out, void* workspace, void* stream);
/* Gradients, of d_o and d_state_out (null: zeros): dq, dk and dv (type and head counts of q, k and v; each may be null) and
 * d_state_in (may be null).  None of them may lie in an input.  `workspace`: flstm_decay_attention_workspace_bytes(shape, 1).
 * log_decay is a constant of the model and has no gradient. */
int flstm_decay_attention_backward(const flstm_decay_attention* shape, const flstm_rows* d_o, const flstm_rows* q, const flstm_rows* k,
                                   const flstm_rows* v, const float* state_in, const float* d_state_out, const flstm_rows* dq,
                                   const flstm_rows* dk, const flstm_rows* dv, float* d_state_in, void* workspace, void* stream);
size_t flstm_decay_attention_workspace_bytes(const flstm_decay_attention* shape, int backward);
/* One token of every sequence (shape->tokens and cu_seqlens are not read), the state updated in place. */
int flstm_decay_attention_step(const flstm_decay_attention* shape, const flstm_rows* q, const flstm_rows* k, const flstm_rows* v,
                               const flstm_rows* o, float* state, void* stream);

/* ---- distillation from a teacher's top logits
 *
 * Row r of the student's logits z (rows x vocabulary, ld elements apart) is held against `top` entries (teacher_logits,
 * teacher_index) of the teacher's, at temperature t > 0:
 *   p = softmax(teacher_logits / t) over the row's entries;  q = softmax(z / t) over the vocabulary
 *   loss = t^2 * sum over entries of p * (log p - log q[index])
 *   dlogits[j] = d_loss * t * (q[j] - sum of p over the entries whose index is j)
 * Entries whose index lies outside 0 .. vocabulary - 1 and entries of minus infinity do not count.  A row without any other
 * entry has loss 0 and a gradient of zeros, whatever its logits hold.  1 <= top <= 1024, vocabulary below 2^31 - 65536.
 * teacher_logits: teacher_dtype; teacher_index: int32, or int64 where index_64 is not 0; both contiguous.
 * d_loss's elements are d_stride apart (0: one for all rows).  dlogits may be logits (same place and ld).
 */
typedef struct {
    size_t rows, vocabulary;
    const void* logits;
    size_t ld;
    flstm_op_dtype dtype;
    int top;
    const void* teacher_logits;
    flstm_op_dtype teacher_dtype;
    const void* teacher_index;
    int index_64;
    float temperature;
} flstm_distillation;

/* stats (rows x 2, 8-byte aligned, may be null): a row's largest logit m, and log2 of the sum of exp((z - m) / t).  The backward
 * pass takes them apart because their sum would lose the second in a row whose logits all lie at the lowest value of their type. */
int flstm_distillation_forward(const flstm_distillation* problem, float* loss, float* stats, void* stream);
int flstm_distillation_backward(const flstm_distillation* problem, const float* stats, const float* d_loss, size_t d_stride,
                                void* dlogits, size_t ldd, void* stream);
/* Both in one call, for a d_loss known beforehand (a mean over rows, say): a row's logits are read from memory once, as
 * long as they fit a workgroup's registers (65536).  `workspace`:
 * flstm_distillation_workspace_bytes() bytes, 16-byte aligned (null where that is 0). */
size_t flstm_distillation_workspace_bytes(const flstm_distillation* problem);
int flstm_distillation_train(const flstm_distillation* problem, const float* d_loss, size_t d_stride, float* loss,
                             void* dlogits, size_t ldd, void* workspace, void* stream);

#ifdef __cplusplus
}
#endif
#endif  /* FLASHLSTM_LM_OPS_H_ */
