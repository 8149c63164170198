/* C ABI of the optimiser for dense parameters: AdamW over many tensors in one launch, with moments in 32 or in 8 bits,
 * and the global norm of their gradients. Same library and context as trips_splat.h.
 *
 * The reference steps its network with libtorch's own optimiser (src/lib/models/Pipeline.cpp:870-882); its point
 * optimiser, whose elements count their own steps and stand still without a gradient (MyAdam.cu:41-88), is
 * trips_adam_step_fused in trips_splat.h. Here every element of a tensor is stepped every time.
 *
 * Every call is stream-ordered, allocates nothing, does not synchronise and may be captured into a HIP graph. Pointers
 * need the alignment of their elements only. Launches go to the context's device, whichever is current.
 */
#ifndef TRIPS_OPTIM_H
#define TRIPS_OPTIM_H

#include <stddef.h>
#include <stdint.h>

#include "trips_splat.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types beside TRIPS_DTYPE_F32 (trips_splat.h). TRIPS_DTYPE_F64 is not supported here. */
enum { TRIPS_DTYPE_BF16 = 2, TRIPS_DTYPE_F16 = 3 };

/* Elements that share a scale where moments are held in 8 bits: element i of a tensor belongs to block i / 256. */
#define TRIPS_MOMENT_BLOCK 256
#define TRIPS_GRAD_NORM_WORKSPACE_BYTES 8192

/* One tensor. With a gradient factor f, step count t (from 1), all else per tensor:
 *
 *   g = f * grads;   m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
 *   weights = weights (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 *
 * state_bits 32: first_moment, second_moment are float arrays of n elements; the scales are not read and may be NULL.
 * state_bits 8: first_moment holds n floats of 8 bits with 4 exponent and 3 mantissa bits (largest 448), second_moment
 * n of 5 and 2 bits (largest 57344), first_scale and second_scale one float per block; an element is code * scale. A new
 * scale is the smallest 2^k, -118 <= k <= 111, that 448 (57344) times covers the finite elements of the block. Codes are
 * rounded stochastically, so that the moments' small changes are kept on average (nearest rounding would lose them: a step
 * changes v by a few parts in 1000, its codes are a quarter of their value apart): |y| = |moment| / scale becomes
 * floor(|y| / q + u) q, q the distance of the codes there, u = (r + 0.5) / 65536, with r the low (first moment) or high
 * (second moment) half of mix(p ^ mix(seed + t * 0x9E3779B9)). p is the element's place (mod 2^32) when the tensors of the
 * call lie one behind the other, each from a multiple of 256; mix(x) is, on 32 bits, x ^= x >> 16, x *= 0x9E3779B9,
 * x ^= x >> 15, x *= 0xB504F333, x ^= x >> 16. A positive v is never rounded to zero. The update uses the moments before
 * they are rounded. A moment that is not finite takes the code of NaN and leaves its block's scale alone.
 *
 * Moments and scales are zero before the first step. */
typedef struct TripsAdamWTensor {
    void* weights;       /* [n] weight_dtype, updated in place */
    const void* grads;   /* [n] grad_dtype */
    void* first_moment;  /* [n] */
    void* second_moment; /* [n] */
    float* first_scale;  /* [ceil(n / 256)] or NULL */
    float* second_scale; /* [ceil(n / 256)] or NULL */
    void* copy;          /* [n] copy_dtype: the new weights in another type, before they are rounded to weight_dtype; or NULL */
    int32_t* step;       /* [1] device: steps taken; one more after the call, unless it was skipped. One of its own per tensor */
    int64_t n;
    int32_t weight_dtype, grad_dtype, copy_dtype; /* TRIPS_DTYPE_F32, _BF16 or _F16 */
    int32_t state_bits;                           /* 32 or 8 */
    double lr, beta1, beta2, eps, weight_decay;
} TripsAdamWTensor;

typedef struct TripsAdamWOptions {
    int32_t abi_version; /* TRIPS_ABI_VERSION */
    uint32_t seed;       /* of the rounding to 8 bits */
    /* NULL: f = 1 / loss_scale, and every step is taken. Else two device floats, the norm of the gradients and f (see
     * trips_grad_norm): written by the call for the gradients of all its tensors where compute_norm is nonzero, and only
     * read otherwise (a norm over several calls or ranks). Where f is not finite the step is skipped: weights, copies,
     * moments and step counts stay as they are. */
    float* grad_norm;
    int32_t compute_norm;
    float max_norm;   /* <= 0: no clipping */
    float loss_scale; /* the loss was multiplied by this */
} TripsAdamWOptions;

/* `tensors` is a HOST array. All tensors of one combination of types (weights, gradients, state bits) are stepped by one
 * launch, after a small one per 40 of them, and one or two before those that take the norm. `workspace`:
 * trips_adamw_workspace_size bytes, 256-byte aligned, of any content; calls that share it must not overlap. */
int trips_adamw_workspace_size(int n_tensors, size_t* bytes);
int trips_adamw_step(TripsCtx* ctx, const TripsAdamWTensor* tensors, int n_tensors, const TripsAdamWOptions* options,
                     void* workspace, size_t workspace_bytes, void* stream);

typedef struct TripsGradTensor {
    const void* grads;
    int64_t n;
    int32_t dtype;
} TripsGradTensor;

/* grad_norm[0] = sqrt(sum of all squares) / loss_scale, grad_norm[1] = min(1, max_norm / (grad_norm[0] + 1e-6)) / loss_scale
 * (1 / loss_scale where max_norm <= 0; NaN where the norm is not finite). Squares are summed in double, in an order that
 * depends on the sizes alone. `grad_norm`: two device floats. `workspace`: TRIPS_GRAD_NORM_WORKSPACE_BYTES, 256-byte
 * aligned, of any content; calls that share it must not overlap. */
int trips_grad_norm(TripsCtx* ctx, const TripsGradTensor* tensors, int n_tensors, float max_norm, float loss_scale,
                    float* grad_norm, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TRIPS_OPTIM_H */
