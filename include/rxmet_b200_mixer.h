/* Operators of a decaying recurrent token mixer: residual addition with a root-mean-square norm and 8-bit output, products of 8-bit
 * codes with an epilogue, linear attention with a fixed decay for each head.  They have no counterpart in the reference.
 *
 * Conventions as in rxmet_b200.h: device pointers, a stream, a caller's workspace where one is named, status < 0 and
 * rxmet_last_error() on failure.  Every call only enqueues work; none allocates device memory. */
#ifndef RXMET_B200_MIXER_H_
#define RXMET_B200_MIXER_H_

#include <stddef.h>
#include <stdint.h>

#include "rxmet_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations. */
enum { RXMET_TYPE_F32 = 0, RXMET_TYPE_BF16 = 1, RXMET_TYPE_F16 = 2 };

/* 1 in *gave_up once a bounded device-side wait of one of these operators' kernels has run out on the current device (the results of that call are
 * not to be used: some may be missing, some wrong),
 * else 0.  Synchronises the device.  No wait runs out in a working program. */
RXMET_API int rxmet_wait_status(int *gave_up);

/* ---- residual addition and root-mean-square norm -----------------------------------------------
 * total = x + residual;  y = total * rsqrt(mean(total^2) + eps) * weight, row by row, sums in 32 bits; y is taken from the unrounded
 * total.  Rows of x and residual start `*_pitch` elements apart; total and y are contiguous.  residual may be null (total is x then and
 * is not written).  1 <= width <= 16384.  weight has weight_type. */
RXMET_API int rxmet_add_rms_norm(int64_t rows, int width, int type, const void *x_dev, int64_t x_pitch, const void *residual_dev,
                                 int64_t residual_pitch, const void *weight_dev, int weight_type, float eps, void *total_dev,
                                 void *y_dev, float *rms_dev /* optional [rows]: rsqrt(mean + eps), for the backward */, void *stream);
/* The same with an output in 8 bits: scale = max|y| / 127 of the row, codes = rne(y / scale) in [-127, 127]; a row of zeros has scale 0
 * and codes 0, a row whose largest magnitude is not finite has that value for its scale and codes that mean nothing.  codes rows start codes_pitch
 * bytes apart.  weight null: no norm (y = total), which codes the rows of any array, of up to 131071
 * elements.  A scale below the normal
 * numbers is as exact as those are; the codes are of y over that scale, and zeros where it rounds to zero.  No output may overlap an input. */
RXMET_API int rxmet_add_rms_norm_codes(int64_t rows, int width, int type, const void *x_dev, int64_t x_pitch, const void *residual_dev,
                                       int64_t residual_pitch, const void *weight_dev, int weight_type, float eps, void *total_dev,
                                       int8_t *codes_dev, int64_t codes_pitch, float *scale_dev, void *stream);
/* dx = dtotal + rms * (weight * dy - u * mean(weight * dy * u)) with u = (x + residual) * rms, the gradient of x and of residual alike;
 * dweight [width] = sum over the rows of dy * u in a fixed order (null: not computed, no workspace needed).  dtotal and residual may be null. */
RXMET_API size_t rxmet_add_rms_norm_backward_workspace_bytes(int64_t rows, int width, int type);
RXMET_API int rxmet_add_rms_norm_backward(int64_t rows, int width, int type, const void *dy_dev, const void *dtotal_dev,
                                          const void *x_dev, int64_t x_pitch, const void *residual_dev, int64_t residual_pitch,
                                          const float *rms_dev, const void *weight_dev, int weight_type, void *dx_dev, void *dweight_dev,
                                          void *workspace_dev, size_t workspace_bytes, void *stream);

/* ---- product of 8-bit codes with an epilogue ----------------------------------------------------
 * out[m][n] = activation(sum_k codes[m][k] * weight[n][k] * scale[m] * weight_scale[n] + bias[n]) + residual[m][n]
 * The sum is exact in 32-bit integers (1 <= inner <= 131071).  Rows of codes and weight start their pitches (bytes) apart, rows of
 * residual residual_pitch elements apart; out is contiguous.  bias (32 bits) and residual (type of out) may be null. */
enum { RXMET_ACTIVATION_NONE = 0, RXMET_ACTIVATION_RELU = 1, RXMET_ACTIVATION_SILU = 2, RXMET_ACTIVATION_GELU = 3 /* erf form */ };
RXMET_API int rxmet_coded_linear(int64_t rows, int inner, int outer, const int8_t *codes_dev, int64_t codes_pitch, const float *scale_dev,
                                 const int8_t *weight_dev, int64_t weight_pitch, const float *weight_scale_dev, const float *bias_dev,
                                 int activation, const void *residual_dev, int64_t residual_pitch, int out_type, void *out_dev,
                                 void *stream);

/* ---- linear attention with a decay for each head ------------------------------------------------
 * S_t = exp(log_decay[h]) S_{t-1} + k_t v_t',  out_t = scale q_t S_t  for t < lengths[b]; out is zero beyond.
 * What is not finite reaches nothing in front of it: from an infinity or a NaN in v on, its column of out and state is not finite (a NaN where the sum
 * may be an infinity), from one in k on all of a head's out.
 * A tensor of `heads` heads: element (b, t, h, d) at b * stride_b + t * stride_t + h * stride_h + d.  The operator has `heads` heads;
 * q, k and v have a number of heads that divides it, and head h reads head h / (heads / own heads) of them.  log_decay <= 0 (32 bits, -inf: no memory).
 * state [batch][heads][key_dim][value_dim] in 32 bits, null for zeros.  1 <= key_dim, value_dim <= 128; batch and heads at most
 * 65535, tokens at most 2^30. */
typedef struct rxmet_head_tensor {
    const void *data;
    int64_t stride_b, stride_t, stride_h;
    int32_t heads;
} rxmet_head_tensor;
typedef struct rxmet_decayed_attention {
    int32_t batch, tokens, heads, key_dim, value_dim, type;
    rxmet_head_tensor q, k, v;
    const float *log_decay;   /* [heads] */
    const int32_t *lengths;   /* [batch] on the device, null: all tokens; values are clamped to [0, tokens] */
    float scale;              /* finite and not zero */
} rxmet_decayed_attention;
/* out [batch][tokens][heads][value_dim]; final_state (may be null, may be `state` itself) has the layout of state.  out may be null. */
RXMET_API size_t rxmet_decayed_attention_workspace_bytes(const rxmet_decayed_attention *problem, int backward);
RXMET_API int rxmet_decayed_attention_forward(const rxmet_decayed_attention *problem, const float *state_dev, void *out_dev,
                                              float *final_state_dev, void *workspace_dev, size_t workspace_bytes, void *stream);
/* Gradients of q, k, v (contiguous, with the heads of q, k, v; gradients of shared heads are summed in 32 bits) and of state, each null
 * where it is not wanted.  dout (heads = problem->heads; it or its data) or dfinal_state may be null: zeros; without dout the gradients of k and v go token by token. */
RXMET_API int rxmet_decayed_attention_backward(const rxmet_decayed_attention *problem, const float *state_dev,
                                               const rxmet_head_tensor *dout, const float *dfinal_state_dev, void *dq_dev, void *dk_dev,
                                               void *dv_dev, float *dstate_dev, void *workspace_dev, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* RXMET_B200_MIXER_H_ */
