/* Operators of a gated recurrent token mixer and of its training with activations kept in 8 bits: a linear recurrence whose gates come from the
 * tokens, codes of activations, the product of an activated gate with its partner, and the gradient of a weight from kept codes.  They have no
 * counterpart in the reference.
 *
 * Conventions as in rxmet_b200_mixer.h: device pointers, a stream, a caller's workspace where one is named, status < 0 and rxmet_last_error() on
 * failure.  Every call only enqueues work; none allocates device memory.  No output may overlap an input unless it is said to. */
#ifndef RXMET_B200_GATED_H_
#define RXMET_B200_GATED_H_

#include "rxmet_b200_mixer.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- gated linear recurrence --------------------------------------------------------------------
 * h_t = f h_{t-1} + z c   with f = sigmoid(forget), c = value or tanh(value), z = sigmoid(input), or 1 - f without an input gate, for every
 * channel by itself and t < lengths[b]; out_t = h_t, and zero beyond.  States, gates and products are held in 32 bits.
 * Element (b, t, d) of a tensor at b * stride_b + t * stride_t + d.  tokens at most 2^30. */
typedef struct rxmet_token_tensor {
    const void *data;
    int64_t stride_b, stride_t;
} rxmet_token_tensor;
typedef struct rxmet_gated_recurrence {
    int32_t batch, tokens, width, type;
    int32_t tanh_value;                     /* c = tanh(value) where it is not zero */
    rxmet_token_tensor forget, value, input; /* input.data null: z = 1 - f */
    const int32_t *lengths;                 /* [batch] on the device, null: all tokens; values are clamped to [0, tokens] */
} rxmet_gated_recurrence;
/* states that the forward pass leaves for the backward pass (32-bit floats; 0: none) */
RXMET_API size_t rxmet_gated_recurrence_marks(const rxmet_gated_recurrence *problem);
RXMET_API size_t rxmet_gated_recurrence_workspace_bytes(const rxmet_gated_recurrence *problem);
/* out [batch][tokens][width] in the inputs' type (null: not wanted); state [batch][width] in 32 bits, null for zeros; final_state the same, may be null, may be
 * `state` itself; marks null where there will be no backward pass. */
RXMET_API int rxmet_gated_recurrence_forward(const rxmet_gated_recurrence *problem, const float *state_dev, void *out_dev, float *final_state_dev,
                                             float *marks_dev, void *workspace_dev, size_t workspace_bytes, void *stream);
/* Gradients of forget, value, input (contiguous) and state, each null where it is not wanted, from those of out and of the final state (null, or
 * null data: zeros); marks from the forward pass of the same problem. */
RXMET_API int rxmet_gated_recurrence_backward(const rxmet_gated_recurrence *problem, const float *state_dev, const float *marks_dev,
                                              const rxmet_token_tensor *dout, const float *dfinal_state_dev, void *dforget_dev, void *dvalue_dev,
                                              void *dinput_dev, float *dstate_dev, void *workspace_dev, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* RXMET_B200_GATED_H_ */
