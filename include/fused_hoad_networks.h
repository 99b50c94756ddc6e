/*
 * fused_hoad C ABI, operators of larger networks on MI355X (gfx950): the gated linear layer, the
 * norms around a block with its gate and scaled residual, and AdamW over many tensors.
 *
 * The conventions are those of fused_hoad.h: device pointers to contiguous memory on the calling
 * thread's current device unless stated, `stream` a hipStream_t (NULL = the default stream), calls
 * asynchronous to the host, no device memory allocated, an fhoad_status returned. A message for
 * the last failed call of this header on the calling thread comes from fhoad_net_last_error().
 * Element types are fhoad_dtype; every sum, statistic and moment is held in float32.
 *
 * These operators have no counterpart in the reference, whose kernels cover one fixed network.
 */
#ifndef FUSED_HOAD_NETWORKS_H_
#define FUSED_HOAD_NETWORKS_H_

#include <stddef.h>
#include <stdint.h>

#include "fused_hoad.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum fhoad_dtype { FHOAD_FLOAT32 = 0, FHOAD_BFLOAT16 = 1 } fhoad_dtype;

typedef enum fhoad_activation {
  FHOAD_SILU = 0,    /* g / (1 + exp(-g)) */
  FHOAD_TANH = 1,
  FHOAD_GELU = 2,    /* g Phi(g), with the error function */
  FHOAD_SIGMOID = 3
} fhoad_activation;

typedef enum fhoad_norm { FHOAD_RMS_NORM = 0, FHOAD_LAYER_NORM = 1 } fhoad_norm;

/* Message of the last failed call of this header on the calling thread ("" if none). */
const char* fhoad_net_last_error(void);

/* Widest row of fhoad_residual_norm_forward / _backward. */
#define FHOAD_NORM_MAX_WIDTH 16384

/*
 * Residual, gate and norms between two blocks, for each of `rows` rows of `width` values:
 *   n      = post_weight ? norm(block) * post_weight (+ post_bias) : block
 *   hidden = residual_scale * residual + gate * n
 *   normed = norm(hidden) * weight (+ bias)
 * norm is x / sqrt(mean(x^2) + eps) (FHOAD_RMS_NORM) or (x - mean) / sqrt(var + eps) with the
 * biased variance (FHOAD_LAYER_NORM). block == NULL leaves the second term out, and hidden may then
 * be NULL (not written) as well.
 * gate: NULL (one), or [rows / rows_per_gate][width]: row r uses gate row r / rows_per_gate, so
 * rows_per_gate == rows is a gate for each channel, 1 one for each element. rows must be a
 * multiple of rows_per_gate when there is a gate.
 * statistics: [rows][4] floats for the backward, or NULL.
 * All tensors of one type. rows == 0 enqueues nothing. Pointers need their elements' alignment
 * only; 16-byte aligned ones with rows of whole 16 bytes are read and written 16 bytes at a time.
 */
int fhoad_residual_norm_forward(const void* residual, const void* block, const void* gate,
                                const void* weight, const void* bias, const void* post_weight,
                                const void* post_bias, void* hidden, void* normed,
                                float* statistics, int64_t rows, int64_t width,
                                int64_t rows_per_gate, int kind, int dtype, double residual_scale,
                                double eps, void* stream);

/* Bytes of workspace of the backward (16-byte aligned). 0 for rows <= 0. */
size_t fhoad_residual_norm_backward_workspace_size(int64_t rows, int64_t width,
                                                   int64_t rows_per_gate);

/*
 * Backward of fhoad_residual_norm_forward from its inputs and statistics. grad_hidden may be NULL
 * (zero), as may grad_normed. Written, each unless NULL: grad_residual, grad_block [rows][width],
 * grad_gate like gate, grad_weight, grad_bias, grad_post_weight, grad_post_bias [width]. The sums
 * over rows run in a fixed order: results are bitwise reproducible. rows == 0 writes zeros to the
 * sums.
 */
int fhoad_residual_norm_backward(const void* residual, const void* block, const void* gate,
                                 const void* weight, const void* post_weight,
                                 const void* post_bias, const float* statistics,
                                 const void* grad_hidden, const void* grad_normed,
                                 void* grad_residual, void* grad_block, void* grad_gate,
                                 void* grad_weight, void* grad_bias, void* grad_post_weight,
                                 void* grad_post_bias, void* workspace, size_t workspace_bytes,
                                 int64_t rows, int64_t width, int64_t rows_per_gate, int kind,
                                 int dtype, double residual_scale, void* stream);

/* Elements of packed optimizer state that share a scale; tensors start at multiples of it. */
#define FHOAD_ADAMW_BLOCK 256

/* One tensor of an AdamW step. `offset` is where its state starts in the packed buffers and
 * `index` which entry of `steps` it counts in. */
typedef struct fhoad_adamw_tensor {
  void* parameter;
  const void* gradient;
  int64_t numel;
  int64_t offset;
  int64_t index;
} fhoad_adamw_tensor;

/* Bytes of workspace of fhoad_adamw_step for `count` tensors (16-byte aligned). */
size_t fhoad_adamw_workspace_size(int64_t count);

/*
 * One AdamW step (decoupled weight decay) over `count` tensors of one type. `tensors` is a host
 * array and is read during the call only. For each element, t being steps[index] + 1:
 *   m <- beta1 m + (1 - beta1) g,  v <- beta2 v + (1 - beta2) g^2
 *   p <- p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * each operation rounded to float32 by itself, and steps[index] is incremented on the device, so
 * the call can be captured in a HIP graph.
 * bits == 32: exp_avg and exp_avg_sq are packed float32 buffers, and the scales are NULL.
 * bits == 8: packed bytes, and one float32 scale for each FHOAD_ADAMW_BLOCK elements of each.
 *   The first moment is a sign, 4 exponent and 3 mantissa bits, the second moment's square root 4
 *   exponent and 4 mantissa bits, over the block's scale (its largest magnitude over 1.875 and
 *   1.9375). Values are rounded up with the probability that their remainder says, by bits mixed
 *   from `seed`, t and the element's place. A non-zero second moment never becomes zero; blocks
 *   whose magnitudes are all below 2^-100 do. A block with a non-finite moment decodes to
 *   non-finite values throughout.
 * Offsets must be multiples of FHOAD_ADAMW_BLOCK, and the packed buffers 16-byte aligned; between
 * a tensor's end and the next block's start 32-bit states are not touched and codes become zero.
 */
int fhoad_adamw_step(const fhoad_adamw_tensor* tensors, int64_t count, int dtype, int bits,
                     void* exp_avg, void* exp_avg_sq, float* exp_avg_scale,
                     float* exp_avg_sq_scale, int32_t* steps, void* workspace,
                     size_t workspace_bytes, double lr, double beta1, double beta2, double eps,
                     double weight_decay, uint32_t seed, void* stream);

/*
 * The values that 8-bit states stand for: moments[i] for i < count from codes and scales
 * (count a multiple of FHOAD_ADAMW_BLOCK). second != 0 decodes second moments (the square of the
 * stored root).
 */
int fhoad_adamw_decode(const uint8_t* codes, const float* scales, float* moments, int64_t count,
                       int second, void* stream);

/*
 * Gated linear layer, for x [rows][width] and weights [hidden][width]:
 *   g = x gate_weight^T + gate_bias,  u = x up_weight^T + up_bias,  h = activation(g) * u
 * h is [rows][hidden]; either bias may be NULL. pre: NULL, or fhoad_gated_linear_saved_size bytes,
 * 16-byte aligned, that keep g and u in float32 for the backward. workspace:
 * fhoad_gated_linear_forward_workspace_size bytes, 16-byte aligned (NULL when that is 0).
 * float32 products are formed on the 16-bit matrix cores from split operands with float32
 * accumulation. Smaller layers take three bf16 parts of a value, which hold it but for 2^-126, and
 * products of them that are good to 2^-24. Larger layers take two float16 parts of rows scaled to
 * their largest value: errors of 2^-23 of a value or 2^-51 of its row's largest, whichever is more,
 * and of 2^-22 of a product beside it (a row runs along the contraction: of x and of the weights,
 * in the backward of the gradients and columns that are contracted). bfloat16 products are formed
 * directly. All tensors of one type, with their elements' alignment. rows == 0 enqueues nothing.
 * Projections and gradients formed from an infinite or NaN operand are non-finite, NaN where float32
 * arithmetic may give an infinity.
 */
size_t fhoad_gated_linear_saved_size(int64_t rows, int64_t hidden);
size_t fhoad_gated_linear_forward_workspace_size(int64_t rows, int64_t width, int64_t hidden,
                                                 int dtype);
int fhoad_gated_linear_forward(const void* x, const void* gate_weight, const void* up_weight,
                               const void* gate_bias, const void* up_bias, void* h, float* pre,
                               void* workspace, size_t workspace_bytes, int64_t rows,
                               int64_t width, int64_t hidden, int activation, int dtype,
                               void* stream);

/* Bytes of workspace of the backward (16-byte aligned). */
size_t fhoad_gated_linear_backward_workspace_size(int64_t rows, int64_t width, int64_t hidden,
                                                  int dtype);

/*
 * Backward of fhoad_gated_linear_forward from x, the weights, pre and grad_h [rows][hidden].
 * Written, each unless NULL: grad_x, grad_gate_weight and grad_up_weight (both or neither),
 * grad_gate_bias, grad_up_bias. Sums run in a fixed order: results are bitwise reproducible.
 * bfloat16: the gradients of g and u are rounded to bfloat16 once, as operands of the products.
 */
int fhoad_gated_linear_backward(const void* x, const void* gate_weight, const void* up_weight,
                                const float* pre, const void* grad_h, void* grad_x,
                                void* grad_gate_weight, void* grad_up_weight, void* grad_gate_bias,
                                void* grad_up_bias, void* workspace, size_t workspace_bytes,
                                int64_t rows, int64_t width, int64_t hidden, int activation,
                                int dtype, void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* FUSED_HOAD_NETWORKS_H_ */
