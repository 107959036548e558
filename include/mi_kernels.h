/*
 * mi_kernels.h — C ABI of the MI355X (gfx950) fused non-GEMM layer kernels.
 *
 * Every compute entry point replaces one free function of the reference's
 * C++ kernel interface, FINAL_CLEAN_CODE/include/kernels.h (cited per
 * function as kernels.h:line), with the same argument meaning, the same
 * overwrite-versus-accumulate contract and the same aliasing rules.  The
 * differences are the ones a C ABI needs:
 *
 *  - C linkage and an "mi_" prefix (the C++ names with the reference's exact
 *    signatures live in kernels.h of this directory and forward here);
 *  - an explicit stream (a hipStream_t passed as void*; NULL = the legacy
 *    default stream);
 *  - an int status instead of exit(): 0 on success, a hipError_t value for
 *    a runtime failure, or one of the MI_ERR_* codes below; mi_last_error()
 *    returns the message of the most recent failure on the calling thread.
 *
 * All pointers are device pointers owned by the caller, fp32 row-major
 * contiguous (ids int32).  Calls are asynchronous on `stream` and perform no
 * host synchronisation.  The column reductions (dgamma/dbeta/dbias) and the
 * embedding gradients are deterministic (no float atomics), so repeated calls
 * on identical inputs give identical bits.  The column reductions are
 * two-pass and use a library-owned device workspace; it is allocated on first
 * use (or by mi_workspace_reserve) and may not grow while the stream is being
 * captured into a graph.  Growth never frees or synchronises: the buffer it
 * replaces stays allocated (queued kernels, a launch on another thread or an
 * instantiated graph may still use it) until mi_workspace_release().
 * Workspaces are kept per device and per slot.  Calls on an explicit stream
 * or on the null stream share the device's slot: they must not run
 * concurrently on different streams of the same device (one stream
 * serialises them).  Calls on the per-thread default stream
 * (hipStreamPerThread, which the include/kernels.h entry points use, as the
 * reference's `--default-stream per-thread` build does) use a slot of the
 * calling thread's own, so host threads may issue them concurrently.  A
 * thread's slot is kept after the thread exits, until mi_workspace_release().
 */
#ifndef MI_KERNELS_H
#define MI_KERNELS_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MI_OK 0
#define MI_ERR_INVALID_ARG (-1)    /* bad size, NULL pointer, unsupported shape */
#define MI_ERR_CAPTURE_ALLOC (-2)  /* workspace growth needed during capture */

/* ----- runtime helpers (so a ctypes driver needs no other library) ------ */

const char* mi_last_error(void);
const char* mi_version(void);
int mi_device_count(int* count);
int mi_set_device(int device);
int mi_malloc(void** ptr, size_t bytes);
int mi_free(void* ptr);
int mi_memcpy_h2d(void* dst, const void* src, size_t bytes);
int mi_memcpy_d2h(void* dst, const void* src, size_t bytes);
int mi_memset_zero(void* ptr, size_t bytes, void* stream);
int mi_stream_sync(void* stream);
int mi_device_sync(void);
/* Grow the shared workspace slot of the current device (the one calls on
 * explicit streams and the null stream use) to >= bytes now (call before
 * graph capture).  mi_workspace_bytes() reports its current size. */
int mi_workspace_reserve(size_t bytes);
size_t mi_workspace_bytes(void);
/* The same for the slot that calls on `stream` from the calling thread use:
 * the thread's own slot for hipStreamPerThread, else the shared slot.  For a
 * caller that captures the per-thread stream into a graph.  Refused with
 * MI_ERR_CAPTURE_ALLOC while `stream` is capturing. */
int mi_workspace_reserve_stream(size_t bytes, void* stream);
size_t mi_workspace_bytes_stream(void* stream);
/* Synchronise the current device, then free its workspace buffers (every
 * slot's current buffer and every one a growth retired).  Only for a caller
 * who will not replay a graph captured with workspace-using calls; the next
 * call that needs a workspace allocates a new one. */
int mi_workspace_release(void);
/* Workspace an entry point needs for the given shape (bytes).  The token
 * embedding backward needs none: mi_embedding_backward_workspace returns 0. */
size_t mi_layernorm_backward_workspace(int rows, int cols);
size_t mi_bias_backward_workspace(int rows, int cols);
size_t mi_embedding_backward_workspace(int batch_seq);

/* ----- LayerNorm --------------------------------------------------------- */

/* y = (x - mean) * inv_std * gamma + beta per row, biased variance,
 * inv_std = 1/sqrt(var + eps).  Replaces layernorm_forward (kernels.h:53-54,
 * FINAL_CLEAN_CODE/src/kernels/layernorm.cu:60-66). */
int mi_layernorm_forward(const float* x, const float* gamma, const float* beta,
                         float* out, int rows, int cols, float eps, void* stream);

/* As mi_layernorm_forward and also writes mean[rows], inv_std[rows].
 * Replaces layernorm_forward_save (kernels.h:56-58, layernorm.cu:111-119). */
int mi_layernorm_forward_save(const float* x, const float* gamma, const float* beta,
                              float* out, float* mean, float* inv_std,
                              int rows, int cols, float eps, void* stream);

/* residual_out = a + b; out = LN(residual_out) with saved stats.  Replaces
 * residual_layernorm_forward_save (kernels.h:60-64, layernorm.cu:173-183). */
int mi_residual_layernorm_forward_save(const float* a, const float* b,
                                       const float* gamma, const float* beta,
                                       float* residual_out, float* out,
                                       float* mean, float* inv_std,
                                       int rows, int cols, float eps, void* stream);

/* grad_x = dx (overwrite); dgamma += sum_r g*xhat; dbeta += sum_r g.
 * Replaces layernorm_backward (kernels.h:66-70, layernorm.cu:273-289). */
int mi_layernorm_backward(const float* grad_out, const float* x,
                          const float* mean, const float* inv_std, const float* gamma,
                          float* grad_x, float* dgamma, float* dbeta,
                          int rows, int cols, void* stream);

/* grad_residual += dx; dgamma, dbeta accumulate.  Replaces
 * layernorm_backward_residual (kernels.h:72-76, layernorm.cu:291-308). */
int mi_layernorm_backward_residual(const float* grad_out, const float* x,
                                   const float* mean, const float* inv_std,
                                   const float* gamma, float* grad_residual,
                                   float* dgamma, float* dbeta,
                                   int rows, int cols, void* stream);

/* Allocation-free variant of mi_layernorm_backward (same arguments, same
 * results bit for bit: it runs the same kernels).  No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code
 * under graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  Its partial rows live in a static device array of
 * MI_LN_BWD_NOALLOC_MAX_BYTES per device instead of the library workspace;
 * the call makes no hipMalloc / hipFree.  The array is part of the
 * library's code object, so every process that loads the library holds it
 * (16 MiB + 256 B) on each device where the library's code is loaded, until
 * the process ends, whether or not this entry point is ever called.
 * A shape whose partial rows need more (mi_layernorm_backward_workspace
 * reports the need) is rejected with MI_ERR_INVALID_ARG.  Every call on a
 * device shares that device's array: calls that overlap on one device (two
 * streams, or two threads) race and must be serialised by the caller. */
#define MI_LN_BWD_NOALLOC_MAX_BYTES ((size_t)16 * 1024 * 1024 + 256)
int mi_layernorm_backward_noalloc(const float* grad_out, const float* x,
                                  const float* mean, const float* inv_std,
                                  const float* gamma, float* grad_x,
                                  float* dgamma, float* dbeta,
                                  int rows, int cols, void* stream);

/* ----- RMS norm ------------------------------------------------------------ */
/* Beside the LayerNorm calls above; the reference has no RMS norm.  With h = x, or
 * a + b, and r = 1 / sqrt(mean(h^2) + eps) per row:  out = h r gamma.  Rows are fp32,
 * fp16 or bf16 (`type`, MI_TYPE_* below), passed as void*; gamma, inv_rms (r) and dgamma
 * are fp32.  Everything is computed in fp32 (the squares' sum and h gamma have to stay in
 * that range) and rounded to its type at the end; out is that of the unrounded sum a + b,
 * residual_out the rounded sum.  cols is 1 to 2^24, eps finite and not negative; no alignment
 * beyond the element's is needed.  inv_rms may be NULL.  out may be x, residual_out may be a
 * or b; other buffers that are written must not overlap any.  Every result is the same bits on
 * every call. */
int mi_rmsnorm_forward(const void* x, const float* gamma, void* out, float* inv_rms, int rows,
                       int cols, float eps, int type, void* stream);
int mi_residual_rmsnorm_forward(const void* a, const void* b, const float* gamma,
                                void* residual_out, void* out, float* inv_rms, int rows, int cols,
                                float eps, int type, void* stream);

/* The same with y = h r gamma in 8 bits, for a product that takes scaled operands: q [rows,
 * cols] (bytes) holds the codes of y / s, s the fp32 scale that a row's columns share
 * (block = 0: scales is [rows]) or that 128 consecutive ones do (block = MI_ROW8_BLOCK:
 * [rows, ceil(cols / 128)], the last one of what is left).  With m the largest magnitude among
 * them, and no less than 2^-100:
 *   MI_ROW8_INT8: s = m / 127, code = the integer nearest to y 127 / m;
 *   MI_ROW8_E4M3: s = m / 448, code = the OCP e4m3 number nearest to y 448 / m.
 * Half values round to even.  Where a NaN or an infinity is among them, s is NaN and the codes
 * are 0.  A code is that of h gamma times one factor, so y's own roundings are not in it.  out
 * (y as rows; NULL: not wanted) may be x. */
#define MI_ROW8_BLOCK 128
#define MI_ROW8_INT8 0
#define MI_ROW8_E4M3 1
int mi_rmsnorm_forward_row8(const void* x, const float* gamma, void* q, float* scales, void* out,
                            float* inv_rms, int rows, int cols, float eps, int block, int format,
                            int type, void* stream);
int mi_residual_rmsnorm_forward_row8(const void* a, const void* b, const float* gamma,
                                     void* residual_out, void* q, float* scales, void* out,
                                     float* inv_rms, int rows, int cols, float eps, int block,
                                     int format, int type, void* stream);

/* With n = x inv_rms and g = grad_out gamma:  dx = inv_rms (g - n mean(g n)), in grad_x
 * (overwritten; it may be grad_out) or added to grad_residual;  dgamma += sum over the rows of
 * grad_out n (fp32, deterministic, through the library workspace).  x is the forward call's
 * x or residual_out. */
int mi_rmsnorm_backward(const void* grad_out, const void* x, const float* inv_rms,
                        const float* gamma, void* grad_x, float* dgamma, int rows, int cols,
                        int type, void* stream);
int mi_rmsnorm_backward_residual(const void* grad_out, const void* x, const float* inv_rms,
                                 const float* gamma, void* grad_residual, float* dgamma, int rows,
                                 int cols, int type, void* stream);
size_t mi_rmsnorm_backward_workspace(int rows, int cols, int type);

/* ----- residual / bias / ReLU ------------------------------------------- */

/* out = a + b over n elements; out may alias a or b.  Replaces residual_add
 * (kernels.h:88, FINAL_CLEAN_CODE/src/kernels/activations.cu:70-82). */
int mi_residual_add(const float* a, const float* b, float* out, long long n, void* stream);

/* out = (residual + x) + bias[c].  Replaces residual_add_with_bias
 * (kernels.h:90-92, activations.cu:119-137). */
int mi_residual_add_with_bias(const float* residual, const float* x, const float* bias,
                              float* out, int rows, int cols, void* stream);

/* out[r, c] += bias[c] in place.  Replaces bias_add (kernels.h:104,
 * activations.cu:146-151). */
int mi_bias_add(float* out, const float* bias, int rows, int cols, void* stream);

/* out = max(in, 0).  Replaces relu_forward (kernels.h:78,
 * activations.cu:10-14). */
int mi_relu_forward(const float* in, float* out, long long n, void* stream);

/* grad_in = in > 0 ? grad_out : 0.  Replaces relu_backward (kernels.h:79,
 * activations.cu:38-50). */
int mi_relu_backward(const float* in, const float* grad_out, float* grad_in,
                     long long n, void* stream);

/* out = max(in + bias[c], 0).  Replaces bias_relu_forward (kernels.h:106-107,
 * activations.cu:181-197). */
int mi_bias_relu_forward(const float* in, const float* bias, float* out,
                         int rows, int cols, void* stream);

/* grad_in = mask > 0 ? grad_out : 0; dbias += column sums of grad_in
 * (deterministic).  Replaces relu_backward_with_bias_backward
 * (kernels.h:81-83, activations.cu:274-283). */
int mi_relu_backward_with_bias_backward(const float* mask, const float* grad_out,
                                        float* grad_in, float* dbias,
                                        int rows, int cols, void* stream);

/* dbias += column sums of grad (deterministic).  Replaces bias_backward
 * (kernels.h:111, activations.cu:234-240). */
int mi_bias_backward(const float* grad, float* dbias, int rows, int cols, void* stream);

/* ----- bias + tanh-GELU (new operators in the slots of bias_relu_forward
 * and relu_backward_with_bias_backward; the reference has no GELU) ------- */

/* out = gelu_tanh(in + bias[c]). */
int mi_bias_gelu_forward(const float* in, const float* bias, float* out,
                         int rows, int cols, void* stream);

/* u = in + bias[c] (recomputed); grad_in = grad_out * gelu_tanh'(u);
 * dbias += column sums of grad_in (deterministic). */
int mi_gelu_backward_with_bias_backward(const float* in, const float* bias,
                                        const float* grad_out, float* grad_in,
                                        float* dbias, int rows, int cols, void* stream);

/* ----- embedding --------------------------------------------------------- */

/* out[i, :] = table[tokens[i], :].  vocab > 0 bounds the ids: an id outside
 * [0, vocab) yields a zero row instead of a read out of bounds; vocab <= 0
 * trusts the ids as the reference does.  Replaces embedding_forward
 * (kernels.h:131-132, FINAL_CLEAN_CODE/src/kernels/embedding.cu:13-20). */
int mi_embedding_forward(const float* table, const int* tokens, float* out,
                         int batch_seq, int dim, int vocab, void* stream);

/* grad_table[tokens[i], :] += grad_out[i, :], each table row accumulated in
 * increasing i (deterministic, same order as the CPU loop); one kernel, no
 * workspace.  vocab > 0 skips ids outside [0, vocab); vocab <= 0 trusts the
 * ids (negative ids are skipped).  Replaces embedding_backward
 * (kernels.h:133-134, embedding.cu:33-40). */
int mi_embedding_backward(const float* grad_out, const int* tokens, float* grad_table,
                          int batch_seq, int dim, int vocab, void* stream);

/* embeddings[b, t, :] += pos_table[t, :] in place.  Replaces
 * pos_embedding_forward (kernels.h:135-136, embedding.cu:52-59). */
int mi_pos_embedding_forward(const float* pos_table, float* embeddings,
                             int batch, int seq, int dim, void* stream);

/* grad_pos[t, :] += sum over b (in increasing b) of grad_out[b, t, :].
 * Replaces pos_embedding_backward (kernels.h:137-138, embedding.cu:72-79). */
int mi_pos_embedding_backward(const float* grad_out, float* grad_pos_table,
                              int batch, int seq, int dim, void* stream);

/* Fused token + position gather: out[b, t, :] = table[id, :] + pos[t, :].
 * Bit-identical to mi_embedding_forward followed by mi_pos_embedding_forward
 * (one fp32 add per element), in one pass.  The reference issues the two
 * calls back to back (FINAL_CLEAN_CODE/src/model/transformer.cu:345-346). */
int mi_embedding_pos_forward(const float* table, const float* pos_table,
                             const int* tokens, float* out,
                             int batch, int seq, int dim, int vocab, void* stream);

/* Fused token + position backward: mi_embedding_backward(grad_out, tokens,
 * grad_table, batch * seq, dim, vocab) and mi_pos_embedding_backward(grad_out,
 * grad_pos_table, batch, seq, dim) in one launch, bit-identical to the two
 * calls (same accumulation orders).  The reference issues the two calls back
 * to back (FINAL_CLEAN_CODE/src/model/transformer.cu:581-584). */
int mi_embedding_pos_backward(const float* grad_out, const int* tokens,
                              float* grad_table, float* grad_pos_table,
                              int batch, int seq, int dim, int vocab, void* stream);

/* ----- softmax and cross-entropy ----------------------------------------- */

/* out[r, :] = exp(x[r, :] - max) / sum, per row.  Replaces softmax_forward
 * (kernels.h:122, FINAL_CLEAN_CODE/src/kernels/activations.cu:394-435). */
int mi_softmax_forward(const float* x, float* out, int rows, int cols, void* stream);

/* Softmax cross-entropy with the reference kernel's arithmetic
 * (activations.cu:438-477): p = e * (1 / (sum + 1e-9)),
 * loss[b] = -log(p[target] + 1e-9), grad = p - onehot(target).  Waits for
 * the stream, copies the per-row losses back and stores their mean, summed
 * in row order on the host, in *loss.  A target outside [0, vocab) gives a
 * NaN loss and leaves that row's gradient at p.  Replaces
 * cross_entropy_forward (kernels.h:124-125, activations.cu:479-499), which
 * returns the loss; uses the library workspace for the per-row losses. */
int mi_cross_entropy_forward(const float* logits, const int* targets, float* grad,
                             int batch, int vocab, float* loss, void* stream);

/* As above with grad scaled by 1 / batch, per-row losses in losses[batch]
 * and their mean written to the device scalar *loss_out, summed in a fixed
 * order (no host sync, no memset, no atomics; graph-capturable).  Replaces
 * cross_entropy_forward_v2 (kernels.h:127-129, activations.cu:517-532). */
int mi_cross_entropy_forward_v2(const float* logits, const int* targets, float* grad,
                                float* losses, float* loss_out, int batch, int vocab,
                                void* stream);

/* Workspace bytes mi_cross_entropy_forward needs for `batch` rows. */
size_t mi_cross_entropy_workspace(int batch);

/* ----- optimizer step over the flat parameter buffer ---------------------- */

/* buf[i] *= scale.  Replaces scale_buffer (kernels.h:113,
 * FINAL_CLEAN_CODE/src/kernels/activations.cu:349-358). */
int mi_scale_buffer(float* buf, float scale, long long n, void* stream);

/* *d_result += sum of buf[i]^2, with a deterministic two-pass sum (per-block
 * partials in the library workspace, then a fixed-order total) instead of
 * the reference's per-block float atomicAdd.  Replaces buffer_norm_sq_acc
 * (kernels.h:118, activations.cu:360-381). */
int mi_buffer_norm_sq_acc(const float* buf, long long n, float* d_result, void* stream);

/* *d_clip_scale = sqrt(*d_norm_sq) > max_norm ? max_norm / sqrt(*d_norm_sq)
 * : 1.  Replaces compute_clip_scale (kernels.h:120, activations.cu:383-392). */
int mi_compute_clip_scale(const float* d_norm_sq, float* d_clip_scale, float max_norm,
                          void* stream);

/* One clipped Adam step, the arithmetic of adam_clipped_kernel
 * (FINAL_CLEAN_CODE/src/model/transformer.cu:598-617) evaluated as written:
 * g = grad * grad_scale * (*d_clip_scale); m = beta1 m + (1 - beta1) g;
 * v = beta2 v + (1 - beta2) g g; param -= lr (m / bc1) / (sqrt(v / bc2) + eps). */
int mi_adam_clipped(float* param, const float* grad, float* m, float* v,
                    const float* d_clip_scale, float lr, float beta1, float beta2, float eps,
                    float bc1, float bc2, float grad_scale, long long n, void* stream);

/* TransformerModel::update_adam (transformer.cu:619-636) in one call: bias
 * corrections 1 - beta^step on the host, the gradient norm² into *d_norm_sq
 * (overwritten, no memset), the clip scale for max norm 1 / grad_scale (1
 * when grad_scale <= 0) into *d_clip_scale, then the Adam step.  Three
 * kernels, graph-capturable; step >= 1. */
int mi_adam_update(float* param, const float* grad, float* m, float* v, long long n, float lr,
                   float beta1, float beta2, float eps, int step, float grad_scale,
                   float* d_norm_sq, float* d_clip_scale, void* stream);

/* Workspace bytes mi_buffer_norm_sq_acc / mi_adam_update need for n floats. */
size_t mi_norm_sq_workspace(long long n);

/* ----- gradients in many tensors ------------------------------------------- */
/* A model's gradients as `count` tensors: tensors[i] points to sizes[i] elements of types[i]
 * (MI_TYPE_* below; types NULL: all fp32).  tensors, outs, sizes and types are host arrays,
 * read before the call returns; their entries are baked into a captured graph.  A tensor of
 * no elements may be NULL.  No alignment beyond the element's is needed.  Squares and sums are
 * formed in fp32, and the last sum in 64 bits, in an order fixed by the sizes and types. */

/* *d_result += sum of all elements' squares (fp32). */
int mi_tensors_norm_sq_acc(const void* const* tensors, const long long* sizes, const int* types,
                           int count, float* d_result, void* stream);

/* Every element times *d_scale: in place, rounded to its type (outs NULL; nothing is read
 * or written where the scale is 1), or as fp32 in outs[i] (e.g. pieces of the flat buffer that
 * mi_adam_clipped takes).  Tensors to be scaled in place must not overlap each other, outs
 * neither each other nor the tensors; *d_scale lies in none of them. */
int mi_tensors_scale(const void* const* tensors, void* const* outs, const long long* sizes,
                     const int* types, int count, const float* d_scale, void* stream);

/* Clipping by the global norm: *d_norm_sq = sum of all elements' squares (overwritten),
 * *d_clip_scale as mi_compute_clip_scale's, then mi_tensors_scale with it.  An infinite norm
 * gives the scale 0, a NaN the scale 1, as there.  *d_norm_sq and *d_clip_scale lie apart, in
 * none of the tensors and outs. */
int mi_tensors_clip(const void* const* tensors, void* const* outs, const long long* sizes,
                    const int* types, int count, float max_norm, float* d_norm_sq,
                    float* d_clip_scale, void* stream);

/* Workspace bytes mi_tensors_norm_sq_acc / mi_tensors_clip need, at most, for `count`
 * tensors. */
size_t mi_tensors_workspace(int count);

/* ----- 16-bit activation storage ----------------------------------------- */
/* Half buffers hold IEEE binary16 values, bf16 buffers the upper 16 bits of
 * fp32; both are passed as void* (2 bytes per element).  Conversions round
 * to nearest even. */

/* out16[i] = half(in[i]).  Replaces float_to_half_buffer (kernels.h:115,
 * FINAL_CLEAN_CODE/src/kernels/activations.cu:325-329,337-341). */
int mi_float_to_half(const float* in, void* out16, long long n, void* stream);

/* out[i] = float(in16[i]).  Replaces half_to_float_buffer (kernels.h:116,
 * activations.cu:331-335,343-347). */
int mi_half_to_float(const void* in16, float* out, long long n, void* stream);

/* bf16 counterparts (no reference counterpart: the bf16 storage variant of
 * the same path). */
int mi_float_to_bf16(const float* in, void* out16, long long n, void* stream);
int mi_bf16_to_float(const void* in16, float* out, long long n, void* stream);

/* out16 = half(max(in + bias, 0)).  Replaces bias_relu_forward_to_half
 * (kernels.h:108-109, activations.cu:199-217). */
int mi_bias_relu_forward_to_half(const float* in, const float* bias, void* out16, int rows,
                                 int cols, void* stream);

/* out16 = half / bf16 (gelu(in + bias)): the bias+GELU forward with 16-bit
 * activation storage (no reference counterpart; takes the slot of
 * bias_relu_forward_to_half for the GELU path). */
int mi_bias_gelu_forward_to_half(const float* in, const float* bias, void* out16, int rows,
                                 int cols, void* stream);
int mi_bias_gelu_forward_to_bf16(const float* in, const float* bias, void* out16, int rows,
                                 int cols, void* stream);

/* grad_in = float(mask16) > 0 ? grad_out : 0; dbias += column sums
 * (deterministic).  Replaces relu_backward_with_bias_backward_half_mask
 * (kernels.h:84-86, activations.cu:285-323). */
int mi_relu_backward_with_bias_backward_half_mask(const void* mask16, const float* grad_out,
                                                  float* grad_in, float* dbias, int rows,
                                                  int cols, void* stream);

/* ----- mixture-of-experts layer: router, rows to their experts and back --- */
/* No counterpart in the reference, whose feed-forward layer is dense.  Rows
 * are fp32, fp16 or bf16 (MI_TYPE_*), passed as void*; weights and their
 * gradients are fp32, sums are formed in fp32 and rounded once, to nearest
 * even.  Slot t * k + j is choice j of token t; k is 1 to 16, experts 1 to
 * 1024 (k <= experts), tokens * k at most INT_MAX, cols at most 2^22.  Every
 * result is the same bits on every call.  No row needs an alignment beyond its
 * element's.  Buffers must not overlap, except where it says so. */
#define MI_TYPE_F32 0
#define MI_TYPE_F16 1
#define MI_TYPE_BF16 2

/* The k experts of each token with the largest logits [tokens, experts], in
 * falling order, equal logits by rising expert: ids [tokens, k].  weights
 * [tokens, k] are their softmax over the chosen ones (renormalise != 0) or over
 * all experts (0).  A logit of -inf is never chosen: where too few others are
 * left, id -1 and weight 0.  NaN ranks above every number; a row with a NaN or
 * +inf that takes part in its sum has NaN weights. */
int mi_moe_gate_forward(const void* logits, int* ids, float* weights, int tokens, int experts,
                        int k, int renormalise, int type, void* stream);

/* dlogits (overwritten, all of [tokens, experts]) from dweights [tokens, k],
 * with ids and weights as the forward call returned them.  Slots with an id
 * outside [0, experts) take no part; slots of one expert add up.  logits may be
 * NULL if renormalise != 0. */
int mi_moe_gate_backward(const void* logits, const int* ids, const float* weights,
                         const float* dweights, void* dlogits, int tokens, int experts, int k,
                         int renormalise, int type, void* stream);

/* The router's balance loss.  Of the tokens with valid[t] != 0 (bytes; NULL: all), n in number:
 * counts[e] = their slots with id e (slots with an id outside [0, experts) are not counted) and
 * counts[experts] = n; probs[e] = the mean of their p_te, the softmax of their logits over all
 * experts (0 for a row of -inf alone); *loss = coef experts / (k n) sum_e counts[e] probs[e],
 * 0 where n is 0.  counts is [experts + 1].  All three are overwritten; sums over the tokens
 * are formed in fp32 in a fixed order, through the library workspace, the loss's over the
 * experts in 64 bits: its relative error does not grow where it is small. */
int mi_moe_balance_forward(const void* logits, const int* ids, const unsigned char* valid,
                           int* counts, float* probs, float* loss, int tokens, int experts, int k,
                           float coef, int type, void* stream);

/* The loss's gradient times *dloss (device; NULL: 1):
 * dlogits[t, e] = dloss coef experts / (k n^2) p_te (counts[e] - sum_f p_tf counts[f]), with
 * counts as the forward call wrote them, or summed over several processes.  accumulate != 0:
 * added to what dlogits holds (as mi_moe_gate_backward left it), else dlogits is overwritten,
 * with 0 where a token is not valid. */
int mi_moe_balance_backward(const void* logits, const unsigned char* valid, const int* counts,
                            const float* dloss, void* dlogits, int tokens, int experts, int k,
                            float coef, int accumulate, int type, void* stream);
size_t mi_moe_balance_workspace(int tokens, int experts);

/* Sorts `slots` expert ids, stably.  offsets [experts + 1]: expert e's rows are
 * offsets[e] .. offsets[e + 1] - 1; position [slots]: the row of each slot, -1
 * for an id outside [0, experts); order [slots] (NULL: not wanted): the slot of
 * each row; entries from offsets[experts] on are left as they were.  Above 4096
 * slots it uses the library workspace. */
int mi_moe_sort(const int* ids, int* offsets, int* order, int* position, int slots, int experts,
                void* stream);
size_t mi_moe_sort_workspace(int slots, int experts);

/* out[position[t * k + j], :] = x[t, :].  x is [tokens, cols], out [rows,
 * cols]; a slot whose position is outside [0, rows) is dropped, and rows that no
 * slot has are left as they were.  No two slots may have the same row. */
int mi_moe_dispatch_forward(const void* x, const int* position, void* out, int tokens, int k,
                            int rows, int cols, int type, void* stream);

/* dx[t, :] = sum over j, in order, of dout[position[t * k + j], :]; 0 for a
 * token without rows. */
int mi_moe_dispatch_backward(const void* dout, const int* position, void* dx, int tokens, int k,
                             int rows, int cols, int type, void* stream);

/* out[t, :] = sum over j, in order, of weights[t, j] y[position[t * k + j], :];
 * 0 for a token without rows. */
int mi_moe_combine_forward(const void* y, const int* position, const float* weights, void* out,
                           int tokens, int k, int rows, int cols, int type, void* stream);

/* dy[position[t * k + j], :] = weights[t, j] dout[t, :] (other rows are left as
 * they were); dweights[t, j] = the product of dout[t, :] and y[position[t * k +
 * j], :], 0 for a dropped slot.  dy may be y: dy is the same bits then, dweights
 * may be added in another order.  No two slots may have the same row (the two sums
 * above read rows only and take the same row twice). */
int mi_moe_combine_backward(const void* dout, const void* y, const int* position,
                            const float* weights, void* dy, float* dweights, int tokens, int k,
                            int rows, int cols, int type, void* stream);

/* ----- activations kept in 8 bits for the backward pass ------------------- */
/* A checkpoint of [rows, cols] is q [rows, cols] (bytes) and scales [rows,
 * ceil(cols / 32)] (bytes): 32 consecutive columns of a row share a power of
 * two.  With e = max(floor(log2 of the block's largest magnitude), -118) the
 * scale byte is e + 127, and an element x is held as
 *   MI_CKPT8_INT8: the integer rint(x 2^(6-e)), cut at 127, of value q 2^(e-6);
 *   MI_CKPT8_E4M3: the OCP e4m3 number nearest to x 2^(8-e), cut at +-448, of
 *                  value q 2^(e-8).
 * A block with a NaN or an infinity has scale byte 255 and reads as NaN.  Half
 * values round to even.  The lowest integer is -128, of value -2^(e+1), which
 * mi_ckpt8_to_float rounds to -inf where it is beyond the type: fp16 elements from
 * -65280 down, fp32 and bf16 ones from -2^128 (1 - 2^-8) down (their gelu and its
 * slope vanish either way).  rows at most 2^30, cols at most 2^24; no alignment
 * beyond the element's is needed. */
#define MI_CKPT8_BLOCK 32
#define MI_CKPT8_INT8 0
#define MI_CKPT8_E4M3 1

/* The checkpoint of `in`, and what it stands for, as MI_TYPE_* rows. */
int mi_float_to_ckpt8(const void* in, void* q, void* scales, int rows, int cols, int format,
                      int type, void* stream);
int mi_ckpt8_to_float(const void* q, const void* scales, void* out, int rows, int cols, int format,
                      int type, void* stream);

/* out = gelu(in + bias[g]) and the checkpoint of in.  Rows belong to `groups`
 * (1 to 1024) consecutive segments, g's being offsets[g] .. offsets[g + 1] - 1
 * (as mi_moe_sort writes them; a rising list of groups + 1 device ints); bias is
 * [groups, cols], fp32.  Rows outside the segments are left as they were, in
 * out, q and scales.  offsets may be NULL for one group: all rows.  out may be
 * in. */
int mi_bias_gelu_forward_ckpt8(const void* in, const float* bias, const int* offsets, void* out,
                               void* q, void* scales, int rows, int cols, int groups, int format,
                               int type, void* stream);

/* From the checkpoint of in: u = value + bias[g]; grad_in = grad_out *
 * gelu_tanh'(u); act = gelu(u) (NULL: not wanted), the activation as the next
 * product's weight gradient needs it; dbias [groups, cols] += column sums of
 * the unrounded grad_in over each segment (fp32, deterministic, through the
 * library workspace).  Rows outside the segments are left as they were.
 * grad_in may be grad_out. */
int mi_gelu_backward_with_bias_backward_ckpt8(const void* q, const void* scales, const float* bias,
                                              const int* offsets, const void* grad_out,
                                              void* grad_in, void* act, float* dbias, int rows,
                                              int cols, int groups, int format, int type,
                                              void* stream);
size_t mi_gelu_backward_ckpt8_workspace(int rows, int cols, int groups);

#ifdef __cplusplus
}
#endif

#endif /* MI_KERNELS_H */
