/*
 * snntc.h -- C ABI of the MI355X (gfx950) implementation of the four SNN-TC custom ops.
 *
 * One entry point per reference op; each replaces the op's OpKernel::Compute (shape rules, error
 * checks) together with its GPU functor (device work).  Paths below are relative to the
 * reference checkout.
 *
 *   snntc_fc_forward   <- SnnFcOp::Compute      snntc/snnfc_kernels.cc:160-207
 *                         SnnFcFunctor<GPU>     snntc/snnfc_kernels.cu.cc:93-194
 *                         REGISTER_OP("SnnFc")  snntc/snnfc_ops.cc:6-27
 *   snntc_fc_backward  <- SnnFcGradOp::Compute  snntc/snnfcgrad_kernels.cc:93-131
 *                         SnnFcGradFunctor<GPU> snntc/snnfcgrad_kernels.cu.cc:137-225
 *                         REGISTER_OP("SnnFcGrad") snntc/snnfcgrad_ops.cc:6-20
 *   snntc_cv_forward   <- SnnCvOp::Compute      snntc/snncv_kernels.cc:191-242
 *                         SnnCvFunctor<GPU>     snntc/snncv_kernels.cu.cc:95-210
 *                         REGISTER_OP("SnnCv")  snntc/snncv_ops.cc:6-32
 *   snntc_cv_backward  <- SnnCvGradOp::Compute  snntc/snncvgrad_kernels.cc:131-183
 *                         SnnCvGradFunctor<GPU> snntc/snncvgrad_kernels.cu.cc:164-263
 *                         REGISTER_OP("SnnCvGrad") snntc/snncvgrad_ops.cc:6-20
 *
 * Conventions
 *  - All tensors are float32 (the operators over tokens and choices take 16-bit types where they say so),
 *    row-major (images NHWC), and live in DEVICE memory, except `params`, which is a HOST pointer (the reference pins it with HostMemory("params"),
 *    snntc/snnfc_kernels.cc:224, snntc/snncv_kernels.cc:259).
 *  - The caller owns every buffer, including the scratch `workspace` (device memory, 256-byte
 *    aligned, at least snntc_*_workspace_bytes() long).  The library allocates nothing, keeps no
 *    state between calls and is re-entrant.
 *  - Work is enqueued on `stream` (a hipStream_t passed as void*; NULL = the default stream) and
 *    the call returns without synchronising.
 *  - Every function returns SNNTC_OK (0) or one of the codes below; snntc_last_error() returns a
 *    thread-local text for the last failure.  Invalid-argument codes mirror the reference's
 *    OP_REQUIRES(... InvalidArgument) conditions one to one.
 *
 * Params vectors (float32, exactly as the reference's Python layers build them)
 *  dense [6]  (SNN_TC_Modules.py:48-49):   {MAX_SPIKE_TIME, Epsilon, Spike_Threshold,
 *                                           Thread_per_Block, Blocks, biasvolt}
 *  conv  [12] (SNN_TC_Modules.py:121-123): {MAX_SPIKE_TIME, Thread_per_Block, Blocks, Epsilon,
 *                                           Spike_Threshold, cudaflag, Kh, Kw, Sh, Sw,
 *                                           padding==SAME, biasvolt}
 *  biasvolt > 1e-8 means the weight matrix carries one extra (last) bias row.  Epsilon,
 *  Thread_per_Block, Blocks and cudaflag are accepted and ignored (launch shapes are chosen for
 *  gfx950 by the library; the reference's GPU scan does not read Epsilon either).
 */
#ifndef SNNTC_H_
#define SNNTC_H_

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define SNNTC_API __attribute__((visibility("default")))
#else
#define SNNTC_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

enum {
    SNNTC_OK = 0,
    SNNTC_ERR_DIM_MISMATCH = 1,   /* weight rows vs input size (+bias); grad rows != 2*batch    */
    SNNTC_ERR_TOO_LARGE = 2,      /* a tensor (or the patch matrix) exceeds INT32_MAX elements  */
    SNNTC_ERR_BAD_ARGUMENT = 3,   /* null pointer, negative size, kernel larger than the image  */
    SNNTC_ERR_WORKSPACE = 4,      /* workspace missing, misaligned or too small                  */
    SNNTC_ERR_UNSUPPORTED = 5,    /* segment longer than the largest supported one (2^24 inputs) */
    SNNTC_ERR_HIP = 6             /* a HIP runtime call or kernel launch failed                  */
};

/* Library identification: "snntc-hip gfx950 <version>". */
SNNTC_API const char* snntc_version(void);
/* Text of the last error raised on the calling thread ("" if none). */
SNNTC_API const char* snntc_last_error(void);
/* Fixed text for a status code. */
SNNTC_API const char* snntc_status_string(int status);

/* ---------------------------------------------------------------------------------------------
 * One-time set-up of a device (no counterpart in the reference, whose kernels need none).  Raises the
 * dynamic-LDS limit of every kernel instantiation and looks up the device's copy of the library's
 * static scratch array.  device < 0 means the current device.  Optional: every entry point performs
 * the same set-up on its first call on a device -- but that first call must then not happen while a
 * stream is being captured into a HIP graph (hipFuncSetAttribute is not allowed there).  A caller
 * that captures graphs calls snntc_init() once per device beforehand, or runs one un-captured call.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_init(int device);

/* ---------------------------------------------------------------------------------------------
 * Dense layer (SNN_dense).   x[B,I]   w[w_rows,J] with w_rows == I + (biasvolt > 1e-8)
 * ------------------------------------------------------------------------------------------- */

/* Scratch sizes.  Replaces the reference's allocate_temp calls (snntc/snnfc_kernels.cu.cc:110-137,
 * snntc/snnfcgrad_kernels.cu.cc:159-164).  Inputs longer than 8192 per segment (I here, Kh*Kw*C
 * for conv layers) are sorted in pieces and merged in device memory; the forward size then includes
 * two key buffers for the merge passes.  Segments beyond 2^24 inputs -> UNSUPPORTED. */
SNNTC_API int snntc_fc_forward_workspace_bytes(int64_t B, int64_t I, int64_t J, size_t* bytes);
SNNTC_API int snntc_fc_backward_workspace_bytes(int64_t B, int64_t I, int64_t J, size_t* bytes);

/* out[2B,J]: rows [0,B) = output spike times y (MAX_SPIKE_TIME for a neuron that never fires),
 * rows [B,2B) = 1/(sum_{causal set} w - Spike_Threshold) (0 for a neuron that never fires).
 * Errors: w_rows not in {I, I+1} or inconsistent with biasvolt -> DIM_MISMATCH
 *         (snntc/snnfc_kernels.cc:171-172); B*I, w_rows*J or 2*B*J > INT32_MAX -> TOO_LARGE
 *         (snntc/snnfc_kernels.cc:194-203).
 * Layers with a handful of outputs (fewer work items than compute units) run a kernel whose
 * wavefronts hand each other running sums through LDS behind a bounded wait; should that wait ever
 * run out, the affected (sample, neuron) entries of both halves of `out` are NaN and the call still
 * returns SNNTC_OK (the library never synchronises with the device).  It has not been observed.
 * snntc_scan_status() below reports it without a pass over the outputs. */
SNNTC_API int snntc_fc_forward(const float* x, const float* w, const float* params_host, float* out,
                     int64_t B, int64_t I, int64_t J, int64_t w_rows,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Same as snntc_fc_forward with optional side outputs (any may be NULL):
 *   sorted_z[B,I]  each input row sorted ascending (stable: equal values keep index order)
 *   perm[B,I]      int32 source column of every sorted element
 *   causal_k[B,J]  int32 number of sorted inputs in the causal set, -1 if the neuron never fired
 * These are the reference's temporaries d_in / order (snntc/snnfc_kernels.cu.cc:110-155) and the
 * loop counter k at exit of SnnFcCudaOutKernel (snntc/snnfc_kernels.cu.cc:43-62). */
SNNTC_API int snntc_fc_forward_ex(const float* x, const float* w, const float* params_host, float* out,
                        float* sorted_z, int32_t* perm, int32_t* causal_k,
                        int64_t B, int64_t I, int64_t J, int64_t w_rows,
                        void* workspace, size_t workspace_bytes, void* stream);

/* snntc_fc_forward for callers that cannot allocate device memory or carry a workspace: code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc.  It has no counterpart
 * in the reference (whose ops allocate their temporaries through the framework on every call).
 * Same results as snntc_fc_forward, bit for bit; the scratch (sorted rows, permutation, counts)
 * lives in a static device array of SNNTC_STATIC_SCRATCH_BYTES inside the library, which every GPU
 * the library runs on holds until the process ends.  The call allocates and frees nothing.
 * Limits: snntc_fc_forward_workspace_bytes(B, I, J) must not exceed SNNTC_STATIC_SCRATCH_BYTES
 * (e.g. B = 1024 rows of I = 784), else SNNTC_ERR_WORKSPACE.  All calls on one GPU share that GPU's
 * array: calls that overlap in time on the same GPU (two streams, two threads) race; serialise them. */
#define SNNTC_STATIC_SCRATCH_BYTES (8u << 20)
SNNTC_API size_t snntc_static_scratch_bytes(void);
SNNTC_API int snntc_fc_forward_static(const float* x, const float* w, const float* params_host, float* out,
                            int64_t B, int64_t I, int64_t J, int64_t w_rows, void* stream);

/* grad[grad_rows,J] (only rows [0,B) are read, so a buffer holding just those rows may be passed with
 * grad_rows still declared as 2B), oldout[2B,J] = the forward output.
 * dx[B,I], dw[w_rows,J], dparams[6] (device; written with zeros).  Any of the three outputs may be
 * NULL: that gradient is then not computed (the reference always computes all of them).
 * Domain: inputs are spike times; dw is exact for x >= -MAX_SPIKE_TIME (it is formed from the
 * differences y - x, which the kernels keep within 2 * MAX_SPIKE_TIME; the same holds for
 * snntc_cv_backward).
 * Errors: grad_rows != 2B -> DIM_MISMATCH (snntc/snnfcgrad_kernels.cc:119-120); sizes as above. */
SNNTC_API int snntc_fc_backward(const float* grad, const float* x, const float* w, const float* params_host,
                      const float* oldout, float* dx, float* dw, float* dparams,
                      int64_t B, int64_t I, int64_t J, int64_t w_rows, int64_t grad_rows,
                      void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Convolutional layer (SNN_conv).  xpad[B,H,W,C] is the input AFTER the Python layer's padding /
 * cropping (SNN_TC_Modules.py:144-166); w[w_rows,Kc] with w_rows == Kh*Kw*C + (biasvolt > 1e-8);
 * Nh = (H-Kh)/Sh + 1, Nw = (W-Kw)/Sw + 1 (snntc/snncv_kernels.cc:215).
 * ------------------------------------------------------------------------------------------- */

/* Output spatial size for a padded input, from the params vector. */
SNNTC_API int snntc_cv_output_dims(int64_t H, int64_t W, const float* params_host, int64_t* Nh, int64_t* Nw);

SNNTC_API int snntc_cv_forward_workspace_bytes(int64_t B, int64_t H, int64_t W, int64_t C, int64_t Kc,
                                     const float* params_host, size_t* bytes);
SNNTC_API int snntc_cv_backward_workspace_bytes(int64_t B, int64_t H, int64_t W, int64_t C, int64_t Kc,
                                      const float* params_host, size_t* bytes);

/* out[2B,Nh,Nw,Kc], halves as in the dense op.
 * Errors: w_rows != Kh*Kw*C + bias -> DIM_MISMATCH (snntc/snncv_kernels.cc:218); input, weight,
 *         output or B*Nh*Nw*w_rows > INT32_MAX -> TOO_LARGE (snntc/snncv_kernels.cc:231-238). */
SNNTC_API int snntc_cv_forward(const float* xpad, const float* w, const float* params_host, float* out,
                     int64_t B, int64_t H, int64_t W, int64_t C, int64_t Kc, int64_t w_rows,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Side outputs per patch s=(b*Nh+nh)*Nw+nw, element order (kh,kw,c):
 *   sorted_z[B*Nh*Nw, Kh*Kw*C], perm[B*Nh*Nw, Kh*Kw*C], causal_k[B*Nh*Nw, Kc]. */
SNNTC_API int snntc_cv_forward_ex(const float* xpad, const float* w, const float* params_host, float* out,
                        float* sorted_z, int32_t* perm, int32_t* causal_k,
                        int64_t B, int64_t H, int64_t W, int64_t C, int64_t Kc, int64_t w_rows,
                        void* workspace, size_t workspace_bytes, void* stream);

/* snntc_cv_forward that also leaves the spike times where the next layer reads them: next_xpad is the
 * next SNN_conv's padded input, [B, next_h, next_w, Kc], and the time of output pixel (nh, nw) is
 * written to its pixel (nh + next_top, nw + next_left) as well as to `out`.  The border of next_xpad
 * (the layer's MAX_SPIKE_TIME padding, SNN_TC_Modules.py:147-161) is the caller's: it is constant, so it
 * is filled once when the buffer is made, not per call.  This replaces the tf.pad between two conv
 * layers of the reference's models (snntc/snntc-cifar10.py:73-106 stacks SNN_conv layers directly).
 * Errors: as snntc_cv_forward; an output that does not fit the destination at that offset -> BAD_ARGUMENT. */
SNNTC_API int snntc_cv_forward_chained(const float* xpad, const float* w, const float* params_host, float* out,
                             float* next_xpad, int64_t next_h, int64_t next_w, int64_t next_top, int64_t next_left,
                             int64_t B, int64_t H, int64_t W, int64_t C, int64_t Kc, int64_t w_rows,
                             void* workspace, size_t workspace_bytes, void* stream);

/* grad[grad_rows,Nh,Nw,Kc] (rows [0,B) read), oldout[2B,Nh,Nw,Kc].
 * dxpad[B,H,W,C] (gradient w.r.t. the padded input), dw[w_rows,Kc], dparams[12]; any may be NULL
 * (not computed).
 * Errors: grad_rows != 2B -> DIM_MISMATCH; sizes as in the forward op. */
SNNTC_API int snntc_cv_backward(const float* grad, const float* xpad, const float* w, const float* params_host,
                      const float* oldout, float* dxpad, float* dw, float* dparams,
                      int64_t B, int64_t H, int64_t W, int64_t C, int64_t Kc, int64_t w_rows,
                      int64_t grad_rows, void* workspace, size_t workspace_bytes, void* stream);

/* snntc_cv_backward that stores only a window of the padded input's gradient:
 *   dx[B, dx_h, dx_w, C] = dxpad[:, dx_top : dx_top + dx_h, dx_left : dx_left + dx_w, :].
 * With the window of the un-padded image this is the gradient the layer before expects, i.e. the
 * backward of the tf.pad in SNN_conv.__call__ (SNN_TC_Modules.py:147-161) folded into the op.
 * Errors: as snntc_cv_backward; a window that does not lie inside the padded image -> BAD_ARGUMENT. */
SNNTC_API int snntc_cv_backward_cropped(const float* grad, const float* xpad, const float* w, const float* params_host,
                              const float* oldout, float* dx, int64_t dx_h, int64_t dx_w, int64_t dx_top,
                              int64_t dx_left, float* dw, float* dparams, int64_t B, int64_t H, int64_t W, int64_t C,
                              int64_t Kc, int64_t w_rows, int64_t grad_rows, void* workspace, size_t workspace_bytes,
                              void* stream);

/* ---------------------------------------------------------------------------------------------
 * Loss of the example networks, loss_func (SNN_TC_Modules.py:286-288): categorical cross-entropy of
 * label[B,J] (one-hot, or any non-negative weights) against softmax(-times[B,J]).
 *   sample_loss[B]  per-sample loss  -sum_j label_j * log softmax(-times)_j        (may be NULL)
 *   dtimes[B,J]     gradient of the batch MEAN of sample_loss w.r.t. times         (may be NULL)
 * The batch mean itself is left to the caller (mean of sample_loss).  No workspace.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_softmax_time_loss(const float* times, const float* label, float* sample_loss, float* dtimes,
                            int64_t B, int64_t J, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Earliest-spike pooling of NHWC spike times, SNN_maxpool2d (SNN_TC_Modules.py:215-246: pad with
 * padvalue = 1e5, then -maxpool(-x) with VALID windows).  The padding is implicit here:
 *   y[b,nh,nw,c] = min over kh < Kh, kw < Kw of x[b, nh*Sh - pad_top + kh, nw*Sw - pad_left + kw, c],
 * where positions outside the H x W image count as pad_value.  The caller passes the layer's
 * geometry: pad_top / pad_left (0 for VALID; the reference's SAME split puts int(total/2) before)
 * and Nh, Nw = the number of whole windows of the padded image.
 *   arg[b,nh,nw,c]  int32, kh*Kw + kw of the first window position (kh-major order) that attains
 *                   the minimum -- the position a max pooling of -x that replaces its running
 *                   maximum only on a strictly greater value ends on.  May be NULL (no backward).
 * Backward: dx[b,h,w,c] = sum of grad_y over the windows whose recorded position is pixel (h,w)
 * (a window whose minimum lies in the padding passes nothing on), added in (kh, kw) order.
 * No workspace.  Errors: a size < 0, Kh/Kw/Sh/Sw < 1, a pad < 0 or >= the kernel size, a window
 * that does not fit the padded image -> BAD_ARGUMENT; more than INT32_MAX elements -> TOO_LARGE.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_min_pool_forward(const float* x, float* y, int32_t* arg, int64_t B, int64_t H, int64_t W,
                           int64_t C, int64_t Kh, int64_t Kw, int64_t Sh, int64_t Sw, int64_t pad_top,
                           int64_t pad_left, int64_t Nh, int64_t Nw, float pad_value, void* stream);
/* snntc_min_pool_forward that also leaves the pooled times inside the padded input of the SNN_conv that
 * follows (next_xpad[B, next_h, next_w, C], pixel offset (next_top, next_left), border filled by the
 * caller): see snntc_cv_forward_chained. */
SNNTC_API int snntc_min_pool_forward_chained(const float* x, float* y, int32_t* arg, float* next_xpad, int64_t next_h,
                                   int64_t next_w, int64_t next_top, int64_t next_left, int64_t B, int64_t H, int64_t W,
                                   int64_t C, int64_t Kh, int64_t Kw, int64_t Sh, int64_t Sw, int64_t pad_top,
                                   int64_t pad_left, int64_t Nh, int64_t Nw, float pad_value, void* stream);
SNNTC_API int snntc_min_pool_backward(const float* grad_y, const int32_t* arg, float* dx, int64_t B, int64_t H,
                            int64_t W, int64_t C, int64_t Kh, int64_t Kw, int64_t Sh, int64_t Sw,
                            int64_t pad_top, int64_t pad_left, int64_t Nh, int64_t Nw, void* stream);

/* ---------------------------------------------------------------------------------------------
 * SAME padding of SNN_conv (SNN_TC_Modules.py:147-161: tf.pad with MAX_SPIKE_TIME) in one pass:
 *   xpad[b,hp,wp,c] = x[b, hp - top, wp - left, c] inside the H x W image, `value` outside,
 * xpad being [B,Hp,Wp,C] with Hp >= top + H, Wp >= left + W.  snntc_pad_time_backward is the
 * gradient: dx[b,h,w,c] = dxpad[b, h + top, w + left, c].  No workspace.
 * Errors: a negative size or offset, Hp < top + H, Wp < left + W -> BAD_ARGUMENT; more than
 * INT32_MAX elements -> TOO_LARGE.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_pad_time_forward(const float* x, float* xpad, int64_t B, int64_t H, int64_t W, int64_t C,
                           int64_t top, int64_t left, int64_t Hp, int64_t Wp, float value, void* stream);
SNNTC_API int snntc_pad_time_backward(const float* dxpad, float* dx, int64_t B, int64_t H, int64_t W, int64_t C,
                            int64_t top, int64_t left, int64_t Hp, int64_t Wp, void* stream);

/* ---------------------------------------------------------------------------------------------
 * SGD update of a training step: w[t][e] -= lr * dw[t][e] for e in [0, n[t]), t in [0, count).
 * The reference leaves the update to the framework's optimizer (snntc/snntc-mnist.py:70,92-93);
 * here all weight tensors of a network are updated by one launch (per 32 tensors).
 * w, dw and n are HOST arrays of `count` entries holding device pointers / element counts; they
 * are read before the call returns.  Tensors with n[t] == 0 are skipped.
 * Errors: count < 0, n[t] < 0, a NULL array or a NULL tensor with n[t] > 0 -> BAD_ARGUMENT.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_sgd_update(float* const* w, const float* const* dw, const int64_t* n, int64_t count, float lr,
                     void* stream);

/* ---------------------------------------------------------------------------------------------
 * Glue of the example training recipe (snntc-mnist.py:55-96).
 *   snntc_encode_time        z[e] = exp(1 - image[e]) for e in [0, n)
 *   snntc_label_loss         the loss above for integer labels[B] (int64): sample_loss[B], dtimes[B,J] (may be
 *                            NULL) and correct[B] = 1 where the earliest output (the lowest index of equal ones)
 *                            is the label.  A label outside [0, J) leaves NaN in its loss and gradient.
 *   snntc_weight_cost_*      K * sum_l mean_j max(0, 1 - sum_i w_ij) + K2 * sum_l mean(w^2) over `count` weight
 *                            tensors w[l][rows[l], cols[l]]: _sums reads the weights into the workspace, _grad
 *                            writes (accumulate = 0) or adds (1) upstream * d cost / d w[l] into grad[l] (a NULL
 *                            grad[l] is skipped; upstream: a device scalar, NULL = 1), both one launch per 24 tensors.
 *   snntc_recipe_total       total = mean(sample_loss) + cost (sample_loss may be NULL: the cost alone) and, where
 *                            correct is given, n_correct = the sum of it; after _sums, same workspace.
 * w, grad, rows and cols are HOST arrays of `count` entries, read before the call returns; total and n_correct are
 * device scalars.  Errors: a negative size, rows or cols < 1, a NULL required pointer -> BAD_ARGUMENT; sizes beyond
 * INT32_MAX elements -> TOO_LARGE; a workspace below _workspace_bytes -> WORKSPACE.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_encode_time(const float* image, float* z, int64_t n, void* stream);
SNNTC_API int snntc_label_loss(const float* times, const int64_t* labels, float* sample_loss, float* dtimes, int32_t* correct,
                     int64_t B, int64_t J, void* stream);
SNNTC_API int snntc_weight_cost_workspace_bytes(const int64_t* rows, const int64_t* cols, int64_t count, size_t* bytes);
SNNTC_API int snntc_weight_cost_sums(const float* const* w, const int64_t* rows, const int64_t* cols, int64_t count,
                           void* workspace, size_t workspace_bytes, void* stream);
SNNTC_API int snntc_weight_cost_grad(const float* const* w, float* const* grad, const int64_t* rows, const int64_t* cols,
                           int64_t count, float k, float k2, const float* upstream, int accumulate, void* workspace,
                           size_t workspace_bytes, void* stream);
SNNTC_API int snntc_recipe_total(const int64_t* rows, const int64_t* cols, int64_t count, float k, float k2,
                       const float* sample_loss, const int32_t* correct, int64_t B, float* total, int64_t* n_correct,
                       void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Element types of the tensors below that need not be float32 (tables, gates, the losses' times and the gradients of
 * each).  Arithmetic is float32 or wider; a result is rounded to its type once, to nearest even.
 * ------------------------------------------------------------------------------------------- */
enum { SNNTC_F32 = 0, SNNTC_BF16 = 1, SNNTC_F16 = 2 };

/* ---------------------------------------------------------------------------------------------
 * Spike times of tokens: tokens[N] (token_bytes 4: int32, 8: int64), table[V,D] of table_type.
 *   z[n,:] = scale table[tokens[n],:], or exp(1 - scale table[tokens[n],:]) with encode != 0 (float32; the encoding of
 *   snntc_encode_time).  A token outside [0, V) leaves NaN in its row.
 *   dtable[v,:] = k_v sum over { n : tokens[n] = v } of grad[n,:], k_v = scale, or -scale exp(1 - scale table[v,:]): every
 *   row of dtable is written, rows are added in the order of their positions, with the same sums on every call.  Positions
 *   whose token lies outside the table add nothing.  table may be NULL in the backward call where encode is 0.
 * Errors: a negative size, a token_bytes or table_type that is none of the above, a NULL required pointer, V = 0 with N > 0
 * -> BAD_ARGUMENT; N or D above 2^30, V above INT32_MAX -> TOO_LARGE (products may exceed it); a workspace below
 * _workspace_bytes -> WORKSPACE.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_embed_forward(const void* tokens, int token_bytes, const void* table, int table_type, float* z, int64_t N,
                        int64_t V, int64_t D, float scale, int encode, void* stream);
SNNTC_API int snntc_embed_backward_workspace_bytes(int64_t N, int64_t V, int64_t D, size_t* bytes);
SNNTC_API int snntc_embed_backward(const float* grad, const void* tokens, int token_bytes, const void* table, int table_type,
                         void* dtable, int64_t N, int64_t V, int64_t D, float scale, int encode, void* workspace,
                         size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Gated running mean of spike times along a sequence, x[B,T,D], gate[B,T,D] of gate_type:
 *   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t,  h_0 = state[B,D] (NULL: zeros)
 * h is carried in 64 bits: y_t lies between the smallest and the largest of h_0 and x_1 .. x_t, to the last digit in sequences of up
 * to 10^6 steps and within a step of it in longer ones.
 * lengths[B] (int64, NULL: all T; values outside [0, T] count as the nearer end): steps behind a sequence's length are
 * not read, y there is 0, and final_state[B,D] (may be NULL) is h at the sequence's length (the initial state for
 * length 0).
 * Backward, with y the forward output and u_t the gradient that reaches h_t:
 *   u_t = dy_t + a_{t+1} u_{t+1} (dfinal at a sequence's end),  dx_t = (1 - a_t) u_t,
 *   dgate_t = u_t (h_{t-1} - x_t) a_t (1 - a_t),  dstate = a_1 u_1
 * dy, dfinal, state: NULL counts as zeros.  dx, dgate (of gate_type), dstate: NULL is not computed.  dx and dgate are 0
 * behind a sequence's length, dy there is not read.  One workspace size serves both directions.
 * snntc_gated_step is one step of n independent channels: out = a state + (1 - a) x (state NULL: zeros; out may be state).
 * Errors: a negative size, a gate_type that is none of the above, a NULL required pointer -> BAD_ARGUMENT; B, T or D
 * above 2^30, B ceil(D / 64) of 2^20 and more, or n of 2^32 and more -> TOO_LARGE; a workspace below _workspace_bytes -> WORKSPACE.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_gated_scan_workspace_bytes(int64_t B, int64_t T, int64_t D, size_t* bytes);
SNNTC_API int snntc_gated_scan_forward(const float* x, const void* gate, int gate_type, const float* state, const int64_t* lengths,
                             float* y, float* final_state, int64_t B, int64_t T, int64_t D, void* workspace,
                             size_t workspace_bytes, void* stream);
SNNTC_API int snntc_gated_scan_backward(const float* dy, const float* dfinal, const float* x, const void* gate, int gate_type,
                              const float* y, const float* state, const int64_t* lengths, float* dx, void* dgate,
                              float* dstate, int64_t B, int64_t T, int64_t D, void* workspace, size_t workspace_bytes,
                              void* stream);
SNNTC_API int snntc_gated_step(const float* x, const void* gate, int gate_type, const float* state, float* out, int64_t n,
                     void* stream);

/* ---------------------------------------------------------------------------------------------
 * Losses over choices: every row times[r,:] of J spike times stands for softmax(-times), and one output of it was chosen
 * (tokens[r], int64).  logp[r] = log softmax(-times[r])[tokens[r]]; a token outside [0, J) leaves NaN in its row.
 * A row of weight 0 is not read: its logp and loss are 0 and its gradient is 0.
 *   snntc_time_logp           logp[rows] and, for the backward call, stats[rows,2] (8-byte aligned; may be NULL).
 *   snntc_time_logp_backward  dtimes[r,j] = upstream coef[r] (softmax(-times[r])[j] - [j = tokens[r]]), of times' type, the
 *                             gradient where coef[r] is a loss's derivative by logp[r] (upstream: a device scalar, NULL = 1).  A row whose
 *                             coef is 0 is not read.  (coef of a row with a token outside [0, J) is NaN in every loss here.)
 *   snntc_policy_loss         clipped policy loss with a KL term, ratio = exp(logp - old_logp), d = ref_logp - logp:
 *       row_loss = kl_coef (exp(d) - d - 1) - min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A),  A = advantage[r]
 *       (ref_logp NULL: no KL term).  The objective is sum_r weight[r] row_loss[r], weight NULL: the mean.  stats, coef[rows]
 *       and dtimes: its saved values for the backward call, its derivative by each logp, its gradient; each may be NULL, logp too.
 *   snntc_preference_loss     P pairs of sequences of T rows each, the preferred ones first (times[2P,T,J], tokens and
 *       weight[2P,T], ref_logp[2P] = log-probability of each sequence under the reference):
 *       seq_logp[q] = sum_t weight[q,t] logp[q,t],  m = beta ((seq_logp - ref_logp)[p] - (seq_logp - ref_logp)[P + p])
 *       pair_loss[p] = -(1 - smoothing) log sigmoid(m) - smoothing log sigmoid(-m)
 *       The objective is the mean of pair_loss.  weight NULL: all 1.  stats, coef[2P,T], dtimes as above.  A term of factor 0
 *       (smoothing 0 or 1) is none, also where a sequence that cannot occur makes m infinite.
 *   snntc_loss_total          total = sum_i weight[i] loss[i] (weight NULL: the mean), added in a fixed order.
 * Errors: a negative size, a times_type that is none of the above, a NULL required pointer, J = 0 with rows, a clip below 0
 * or a clip_low above 1, smoothing outside [0, 1], a beta or kl_coef that is not finite -> BAD_ARGUMENT; more than 2^24 - 1
 * rows, J above 2^30 -> TOO_LARGE; a workspace below snntc_choice_workspace_bytes (time_logp,
 * policy_loss; 0 where J <= 16384) or snntc_preference_workspace_bytes -> WORKSPACE.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_choice_workspace_bytes(int64_t rows, int64_t J, size_t* bytes);
SNNTC_API int snntc_preference_workspace_bytes(int64_t P, int64_t T, int64_t J, size_t* bytes);
SNNTC_API int snntc_time_logp(const void* times, int times_type, const int64_t* tokens, const float* weight, float* logp,
                    float* stats, int64_t rows, int64_t J, void* workspace, size_t workspace_bytes, void* stream);
SNNTC_API int snntc_time_logp_backward(const void* times, int times_type, const int64_t* tokens, const float* stats,
                             const float* coef, const float* upstream, void* dtimes, int64_t rows, int64_t J, void* stream);
SNNTC_API int snntc_policy_loss(const void* times, int times_type, const int64_t* actions, const float* old_logp,
                      const float* advantage, const float* ref_logp, const float* weight, float clip_low, float clip_high,
                      float kl_coef, float* row_loss, float* logp, float* stats, float* coef, void* dtimes, int64_t rows,
                      int64_t J, void* workspace, size_t workspace_bytes, void* stream);
SNNTC_API int snntc_preference_loss(const void* times, int times_type, const int64_t* tokens, const float* ref_logp,
                          const float* weight, float beta, float smoothing, float* pair_loss, float* seq_logp, float* stats,
                          float* coef, void* dtimes, int64_t P, int64_t T, int64_t J, void* workspace,
                          size_t workspace_bytes, void* stream);
SNNTC_API int snntc_loss_total(const float* loss, const float* weight, float* total, int64_t n, void* stream);

/* ---------------------------------------------------------------------------------------------
 * Choices by rules: what changes a row of spike times times[r,:] before a token is drawn from softmax(-times) or a loss over it is
 * taken.  history[history_rows, history_len] (int64) are sequences of tokens; row r belongs to sequence r / (rows / history_rows) and
 * sees its first lengths[r] tokens (NULL: all; values outside count as the nearer end), of which the first prompts[sequence] (NULL: 0)
 * are a prompt.  c_j: occurrences of j among what the row sees, o_j: those behind the prompt; tokens outside [0, J) are none.
 *     a_j = times_j repetition (times_j > 0), times_j / repetition (else)    where c_j > 0, times_j elsewhere
 *     b_j = a_j + (presence + frequency o_j)                                 where o_j > 0, a_j elsewhere
 *     out_j = b_j + delay_j  where bit j % 32 of allowed[j / 32] is set, +infinity elsewhere
 * in float32, product by product and sum by sum, rounded to times' type once.  repetition, presence, frequency: device arrays with a
 * number for each sequence, or NULL and *_all for all.  delay[J] or [rows,J] (delay_rows 1 or rows; NULL: none), allowed[ceil(J/32)] or
 * [rows,ceil(J/32)] likewise; what a masked element holds, or bits behind J, do not matter.  history NULL: no penalties.
 *   snntc_rule_times           out[rows,J], of times' type; must not overlap times.
 *   snntc_rule_times_backward  dtimes_j = grad_j times repetition, over it, or as it is, as times_j was; 0 where not allowed.  times may be
 *                              NULL where history is, or no sequence's repetition differs from 1.  presence, frequency, prompts and delay are not read.
 *                              dtimes must not overlap grad or times.
 *   snntc_choose               tokens[r] (int64): with p = softmax(-out[r] / T), the first j whose running sum of p exceeds uniform[r] of the
 *                              whole (uniform below 0 or NaN counts as 0; from 1 on: the last possible j), logp[r] = log p_j.  T = temperature[r], or
 *                              NULL and temperature_all.  T below 1e-30: the earliest output, the lowest index of equal ones, with its
 *                              log-probability at T = 1; uniform may be NULL where this holds for temperature_all.  Times are taken as differences
 *                              from the row's earliest, so that their quotient by T may be of any size; a difference beyond float32, like a time
 *                              of +infinity, has no chance.  Where nothing is possible (all masked or infinite), a time that is allowed is NaN or
 *                              -infinity, or T is negative or no finite number: token -1 and logp NaN.  rules may be NULL.
 * Errors: a negative size, an unknown type, a NULL required pointer, J = 0 with rows, history_rows that do not divide rows, delay_rows or
 * allowed_rows neither 1 nor rows, a result of the first two that overlaps times or grad, a repetition_all that is not positive, penalties or a temperature_all that are not finite or (this) below 0 -> BAD_ARGUMENT;
 * more than 2^24 - 1 rows, J or history_len above 2^30 -> TOO_LARGE; a workspace below snntc_choose_workspace_bytes -> WORKSPACE.
 * ------------------------------------------------------------------------------------------- */
typedef struct snntc_rules {
    const int64_t* history;
    int64_t history_rows, history_len;
    const int64_t* lengths;
    const int64_t* prompts;
    const float* repetition;
    const float* presence;
    const float* frequency;
    float repetition_all, presence_all, frequency_all;
    const float* delay;
    int64_t delay_rows;
    const int32_t* allowed;
    int64_t allowed_rows;
} snntc_rules;
SNNTC_API int snntc_rule_times(const void* times, int times_type, const snntc_rules* rules, void* out, int64_t rows, int64_t J, void* stream);
SNNTC_API int snntc_rule_times_backward(const void* grad, const void* times, int times_type, const snntc_rules* rules, void* dtimes,
                              int64_t rows, int64_t J, void* stream);
SNNTC_API int snntc_choose_workspace_bytes(int64_t rows, int64_t J, size_t* bytes);
SNNTC_API int snntc_choose(const void* times, int times_type, const float* uniform, const float* temperature, float temperature_all,
                 const snntc_rules* rules, int64_t* tokens, float* logp, int64_t rows, int64_t J, void* workspace, size_t workspace_bytes,
                 void* stream);

/* ---------------------------------------------------------------------------------------------
 * One AdamW step over many tensors, w[t] with gradients dw[t] (both of types[t]) of n[t] elements.  g = dw, scaled down to max_norm where
 * `norm`, the gradients' norm on the device, is given and larger:
 *     m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2,
 *     w = w (1 - lr weight_decay) - lr / (1 - beta1^step) m / (sqrt(v / (1 - beta2^step)) + eps)
 * A norm that is no finite number leaves w, first and second as they are.  The step's number is `step` (from 1), or, where `steps` is
 * given, one more than that device number, which the call advances (also of a step that is left out): a captured call counts by itself.
 * first, second: m and v as float32[n], or, where first_scale and second_scale are given, as uint8[n] with a float32 for every 256
 * elements (the last may be fewer), ceil(n / 256) of them: its largest magnitude s.  Code c (of m: its low 7 bits, the 8th its sign) stands for
 *     s value(c) / value(largest code),   value(c) = c (c < 8),  (8 + c % 8) 2^(c / 8 - 1) (else)
 * A state's zero is code 0 and scale 0.  A value between two codes becomes the upper one with the chance of its place between them, a weight of
 * 16 bits likewise one of its two neighbours; the random bits follow from seed, step, t and the element alone.  paired: 0, or (any other) a first
 * moment whose second moment's code is 0 is held as 0 too.  Rounded apart, each moment is right on average but not their quotient: an element
 * far below its block's largest that has kept a first moment and lost its second moves by lr first / eps, hundreds of lr, once its gradient is 0.
 *   snntc_grad_norm       norm = sqrt of the sum of squares of all gradients (float32 on the device, the sum in 64 bits, the same on
 *                         every call).
 *   snntc_adamw_moments   first_out[t], second_out[t] (float32[n]) = what the codes stand for.
 * All arrays but `steps` and `norm` are HOST arrays of `count` entries, read before the call returns; tensors of n[t] = 0 are skipped.  No two of
 * the written tensors (steps is one) may overlap, nor a gradient or norm one of them.  The workspace of snntc_adamw_update (SNNTC_ADAMW_WORKSPACE_BYTES) is needed with `steps` only.
 * Errors: a negative count or size, an unknown type, a NULL required pointer, one scale array without the other, lr or weight_decay not
 * finite or negative, a beta outside [0, 1), an eps below the smallest normal float32, a step below 1, a max_norm that is not positive -> BAD_ARGUMENT; n[t] above
 * 2^34 -> TOO_LARGE; a workspace that is missing or too small -> WORKSPACE.
 * ------------------------------------------------------------------------------------------- */
#define SNNTC_STATE_BLOCK 256
#define SNNTC_ADAMW_WORKSPACE_BYTES 256
typedef struct snntc_adamw {
    double lr, beta1, beta2, eps, weight_decay;
    int64_t step;
    int64_t* steps;
    const float* norm;
    double max_norm;
    uint64_t seed;
    int paired;
} snntc_adamw;
SNNTC_API int snntc_grad_norm_workspace_bytes(const int64_t* n, int64_t count, size_t* bytes);
SNNTC_API int snntc_grad_norm(const void* const* grads, const int* types, const int64_t* n, int64_t count, float* norm, void* workspace,
                    size_t workspace_bytes, void* stream);
SNNTC_API int snntc_adamw_update(void* const* w, const void* const* dw, void* const* first, void* const* second, float* const* first_scale,
                       float* const* second_scale, const int* types, const int64_t* n, int64_t count, const snntc_adamw* how, void* workspace,
                       size_t workspace_bytes, void* stream);
SNNTC_API int snntc_adamw_moments(const uint8_t* const* first, const uint8_t* const* second, const float* const* first_scale,
                        const float* const* second_scale, float* const* first_out, float* const* second_out, const int64_t* n, int64_t count,
                        void* stream);

/* ---------------------------------------------------------------------------------------------
 * Health of the bounded wait described at snntc_fc_forward (no counterpart in the reference, whose scan
 * has one thread per neuron and nothing to wait for).
 *   snntc_scan_status(&giveups, stream)  number of wavefronts, on the current device since the process
 *       started, whose wait ran out (each poisons the outputs of its work item with NaN).  0 = every scan
 *       result so far is what the kernels computed.  The count is a 4-byte device word read with a copy on
 *       `stream` followed by a wait for that stream: call it where the caller synchronises anyway (after a
 *       training step's loss has been read, at the end of a batch of requests).
 *   snntc_debug_set_scan_wait_polls(polls)  test hook: the number of polls a waiting wavefront spends from
 *       the next launch on (process-wide; polls < 0 restores the default of 2^20).  With 0 every wait that
 *       is not already satisfied at its first poll gives up, which drives the give-up path while every
 *       kernel still runs to its end.
 *   snntc_debug_order_tile(B,H,W,C,params,aligned,tile)  test hook, host code only: how a conv layer's patches
 *       are put in order on 256 CUs when Xpad is 16-byte aligned (aligned != 0) or not.  tile[4] = patches of a
 *       tile down and across, pixels of its region that get a bitmap of their own (0: none), bytes of LDS; all
 *       zero for a layer whose patches are sorted one by one.
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_scan_status(int64_t* giveups, void* stream);
SNNTC_API int snntc_debug_set_scan_wait_polls(int polls);
SNNTC_API int snntc_debug_order_tile(int64_t B, int64_t H, int64_t W, int64_t C, const float* params_host, int aligned,
                                     int64_t* tile);

/* ---------------------------------------------------------------------------------------------
 * Per-kernel timing (no counterpart in the reference, which only times whole scripts with
 * time.time()).  While enabled, every kernel the library launches is bracketed by a pair of HIP
 * events on its launch stream; this is the only process-wide state the library keeps and it is
 * off by default.
 *   snntc_profile_enable(1|0)  clear the totals and switch timing on / off
 *   snntc_profile_collect()    wait for the recorded events, fold them into per-kernel totals and
 *                              return the number of distinct kernels seen (>= 0)
 *   snntc_profile_entry(i,...) name, launch count and summed duration (ms) of kernel i; `name`
 *                              stays valid until the next collect/enable call
 * ------------------------------------------------------------------------------------------- */
SNNTC_API int snntc_profile_enable(int on);
SNNTC_API int snntc_profile_collect(void);
SNNTC_API int snntc_profile_entry(int index, const char** name, int64_t* launches, double* total_ms);

#ifdef __cplusplus
}
#endif
#endif /* SNNTC_H_ */
