/*
 * dgnn_train.h -- C ABI of libdgnn_spmm.so for what a training step computes beside the aggregation: the dense layer
 * transform with its epilogue and gradients, and the optimiser step. Same conventions as dgnn_spmm.h: plain device
 * pointers and sizes, an explicit HIP stream passed as void*, an int status with dgnn_last_error(); nothing allocates
 * device memory, nothing synchronises, every call can be captured in a HIP graph.
 */
#ifndef DGNN_TRAIN_H
#define DGNN_TRAIN_H

#include "dgnn_spmm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DGNN_F32  0
#define DGNN_BF16 1
#define DGNN_F16  2

/*
 * The layer transform  y = act(x W + b) + r  and its gradients. All matrices row-major with `ld*` elements between rows
 * (>= the row's width) and element-aligned, of one type (DGNN_F32 | DGNN_BF16 | DGNN_F16): x [M x K], W [K x N], b [N] or
 * NULL, r [M x N] or NULL, y [M x N]. Products and sums in fp32 (fp32 operands: six products of bf16 pieces, as close to
 * the exact sum as a chain of fp32 operations), one rounding at the end. relu(NaN) is NaN. M up to 2^31 - 1, K and N up to 2^24,
 * outputs up to 2^23 tiles of 128 x 32 to 128 x 256 (by N); more is refused.
 *   act    DGNN_ACT_*: none, relu, gelu (0.5 t (1 + erf(t / sqrt 2))), silu (t / (1 + e^-t))
 *   save   NULL, or what dgnn_linear_slope needs: for relu uint32 [M][lds], bit n % 32 of word n / 32 set where x W + b is
 *          not <= 0 (lds >= ceil(N / 32), bits past N zero); for gelu and silu x W + b as float (lds >= N)
 * With a gradient dy of y:
 *   dgnn_linear_slope         p = dy act'(x W + b) (p may be NULL), dbias[n] = sum over m of p[m][n] (may be NULL); p may be
 *                             dy itself. act DGNN_ACT_NONE: p is a copy of dy. p is rounded to its type; dbias is not made from
 *                             the rounded values
 *   dgnn_linear_grad_input    dx = p W^T + add    (add [M x K] or NULL: what else reaches x, a skip connection's gradient)
 *   dgnn_linear_grad_weight   dw = x^T p      (M = 0: zeros)
 *   dgnn_linear_backward      all of them in one call, p in the workspace (where 16-bit p of gelu or silu is rounded to its type, dw
 *                             of narrow layers takes what the rounding left as well, and dx of few values and small layers take
 *                             p in fp32); dx, dw and dbias may be NULL (x, w and save are then
 *                             only needed for what is asked for). Its workspace: dgnn_linear_backward_workspace
 * workspace: device memory of dgnn_linear_workspace(pass, ...) bytes, 16-byte aligned (0 bytes: may be NULL), free to be used
 * again once the call's kernels have run. Sums over many rows are cut by a rule of the sizes alone and joined in a fixed
 * order: the same bits every run. What a call writes must not overlap what it reads or else writes (p alone may be dy itself):
 * such a call is refused before anything is launched. Columns of one buffer, whose rows take turns, do not overlap.
 */
#define DGNN_ACT_NONE 0
#define DGNN_ACT_RELU 1
#define DGNN_ACT_GELU 2
#define DGNN_ACT_SILU 3
#define DGNN_LINEAR_FORWARD     0   /* passes of dgnn_linear_workspace */
#define DGNN_LINEAR_SLOPE       1
#define DGNN_LINEAR_GRAD_INPUT  2
#define DGNN_LINEAR_GRAD_WEIGHT 3
int dgnn_linear_workspace(int32_t pass, int64_t M, int64_t K, int64_t N, int32_t dtype, int64_t* bytes);
int dgnn_linear_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                        const void* residual, int64_t ldr, void* y, int64_t ldy, void* save, int64_t lds,
                        int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t act,
                        void* workspace, int64_t workspace_bytes, void* stream);
int dgnn_linear_slope(const void* dy, int64_t ldd, const void* save, int64_t lds, void* p, int64_t ldp, void* dbias,
                      int64_t M, int64_t N, int32_t dtype, int32_t act, void* workspace, int64_t workspace_bytes, void* stream);
int dgnn_linear_grad_input(const void* p, int64_t ldp, const void* w, int64_t ldw, const void* add, int64_t lda,
                           void* dx, int64_t ldx, int64_t M, int64_t K, int64_t N, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream);
int dgnn_linear_grad_weight(const void* x, int64_t ldx, const void* p, int64_t ldp, void* dw, int64_t ldw,
                            int64_t M, int64_t K, int64_t N, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream);
int dgnn_linear_backward_workspace(int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t act, int64_t* bytes);
int dgnn_linear_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* dy, int64_t ldd,
                         const void* save, int64_t lds, void* dx, int64_t lddx, void* dw, int64_t lddw, void* dbias,
                         int64_t M, int64_t K, int64_t N, int32_t dtype, int32_t act,
                         void* workspace, int64_t workspace_bytes, void* stream);

/*
 * One AdamW step over `count` tensors (a handful of launches for hundreds of them). With g a tensor's gradient, t the
 * number of its step:
 *     m <- b1 m + (1 - b1) g                 v <- b2 v + (1 - b2) g^2
 *     p <- p decay - rate m / (sqrt(v) root + eps)
 *     decay = 1 - lr * weight_decay,  rate = lr / (1 - b1^t),  root = 1 / sqrt(1 - b2^t)
 * all in fp32, each operation rounded once and in this order, p rounded to its type at the end.
 *
 *   param, grad   device, numel elements of `dtype` (DGNN_F32 | DGNN_BF16 | DGNN_F16), element-aligned, contiguous
 *   start         first element of the tensor in the state buffers, a multiple of 256
 *   index         the tensor's entry of `steps` / `factors`, one for each tensor (only read when they are given)
 *   decay, rate, root, turn    the factors above and t mod 2^32 (unused when `steps` is given)
 *
 * State buffers (device, 16-byte aligned, shared by all tensors of the call):
 *   master        NULL, or the fp32 values that are updated in place of param; param receives them rounded. An element of
 *                 param that is not its master rounded replaces it first (somebody else wrote it)
 *   state_bits 32: exp_avg, exp_avg_sq are float; the scales are NULL
 *   state_bits 8:  exp_avg holds m and exp_avg_sq holds sqrt(v) as e4m3 codes, one float scale per 256 elements
 *     (value = code * scale). A block's scale is max(largest value, 2^-100) / 448. A value x is rounded at the e4m3 step s
 *     of its magnitude (2^(e-3), at least 2^-9) to s floor(|x| / s + u), u in [0, 1) a 16-bit fraction that depends on
 *     the element's index in its tensor and on t alone (two Weyl sequences), so that a slow average does not stick to one
 *     code; a root above zero keeps at least 2^-9, so no denominator vanishes. A value that is not finite makes its
 *     block's values NaN from the next step on.
 * In all buffers elements between a tensor's end and the next multiple of 256 are free to be written.
 *
 * steps (device int64[], or NULL) and factors (device float[4 * entries]): when given, a first launch advances
 * steps[index] of every tensor and derives rate, root and t from it on the device with lr, beta1, beta2 -- what a captured
 * graph needs, whose host arguments are frozen; lr and weight_decay stay those of the capture.
 */
struct dgnn_adamw_tensor {
  void* param;
  const void* grad;
  int64_t numel, start;
  float decay, rate, root;
  uint32_t turn;
  int32_t index, reserved;
};

struct dgnn_adamw_state {
  void* exp_avg;
  void* exp_avg_sq;
  float* exp_avg_scale;
  float* exp_avg_sq_scale;
  float* master;
  int64_t* steps;
  float* factors;
};

int dgnn_adamw(const struct dgnn_adamw_tensor* tensors, int32_t count, int32_t dtype, int32_t state_bits,
               const struct dgnn_adamw_state* state, double lr, double beta1, double beta2, double eps, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* DGNN_TRAIN_H */
