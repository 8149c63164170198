/* C ABI of the softmax cross entropy of rows against all entries of a table, with its gradients, and of dropout by a
 * counter-based generator. Same library and context as trips_splat.h.
 *
 * Every call is stream-ordered, allocates nothing, does not synchronise and may be captured into a HIP graph. Pointers
 * need the alignment of their elements only. Launches go to the context's device, whichever is current. The reference has
 * neither operator: its losses are of images (src/lib/models/Pipeline.cpp), its dropout of points is drawn and stored
 * (src/lib/rendering/PointRenderer.cu:516-521).
 */
#ifndef TRIPS_LOSS_H
#define TRIPS_LOSS_H

#include <stddef.h>
#include <stdint.h>

#include "trips_lookup.h"
#include "trips_optim.h"
#include "trips_splat.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { TRIPS_REDUCE_NONE = 0, TRIPS_REDUCE_SUM = 1, TRIPS_REDUCE_MEAN = 2 };

/* N rows and T entries of a table of C channels each, a target per row:
 *
 *   l_ij = scale <rows_i, table_j>;   lse_i = log sum_j exp l_ij;   loss_i = lse_i - l_i,target_i
 *
 * N T C is bounded by the units of work of a launch, 2^31 of some 10^4 products: what is refused for it would take minutes.
 * Rows whose target is outside [0, T) do not count: loss 0, gradient 0, whatever they hold. Strides are the elements between
 * two rows of memory; within a row elements are adjacent. A stride may be 0 where the call only reads. */
typedef struct TripsTableLossDesc {
    int32_t abi_version;  /* TRIPS_ABI_VERSION */
    int32_t dtype;        /* of rows, table and their gradients: TRIPS_DTYPE_F32, _BF16 or _F16 */
    int32_t index_dtype;  /* TRIPS_INDEX_* */
    int32_t reduction;    /* TRIPS_REDUCE_*: loss is [N], or [1]: the sum, or the mean over the rows that count (0 if none does) */
    int64_t num_rows;     /* N, at most 2^28 - 16 */
    int64_t num_entries;  /* T, below 2^31 - 256 */
    int32_t num_channels; /* C, below 2^17 */
    float scale;          /* up to 2.3e38 either way: times log2 e it is a number of 32 bits too */
    int64_t rows_stride;
    int64_t table_stride;
    int64_t d_rows_stride;  /* backward */
    int64_t d_table_stride; /* backward */
} TripsTableLossDesc;

/* kept: trips_table_loss_kept_size bytes, 256-byte aligned, what the backward call takes: the rows that count, one behind the other, and
 * of each its target, its largest product with an entry and the sum of exponentials. Logits and sums are held in 32 bits.
 * `workspace`: trips_table_loss_workspace_size bytes (backward: 0 for the forward call), 256-byte aligned, of any content;
 * calls that share one must not overlap. */
int trips_table_loss_kept_size(const TripsTableLossDesc* desc, size_t* bytes);
int trips_table_loss_workspace_size(const TripsTableLossDesc* desc, int backward, size_t* bytes);
int trips_table_loss_forward(TripsCtx* ctx, const TripsTableLossDesc* desc, const void* rows, const void* table, const void* target, float* loss,
                             void* kept, size_t kept_bytes, void* workspace, size_t workspace_bytes, void* stream);

/* The same desc (but for the strides, those of what is written among them) and table as the forward call that filled `kept`, which is
 * only read and may be used again. d_loss: [N], or [1], as the loss. d_rows [N, C] and d_table [T, C] are written, rows that do not count with
 * zeros; either may be NULL. The logits are computed again, in pieces of the table; their gradient is held in the tensors' type
 * within a piece, sums over it in 32 bits, in an order that the sizes and the number of rows that count alone determine. */
int trips_table_loss_backward(TripsCtx* ctx, const TripsTableLossDesc* desc, const void* table, const void* kept, size_t kept_bytes, const float* d_loss,
                              void* d_rows, void* d_table, void* workspace, size_t workspace_bytes, void* stream);

/* out_i = (kept_i ? x_i factor : 0) + residual_i, factor = 65536 / (65536 - border), border = round(65536 p) (ties to even): of
 * element i, half i % 2 (0: the low one) of word i % 8 / 2 of Philox-4x32-10 is its 16 random bits, and it is kept where those
 * are not below the border. The generator's key is the seed (low half first), its counter the 64 bits of i / 8, then call, then
 * step. The gradient of x is the same call on the gradient of out, without a residual. */
typedef struct TripsDropoutDesc {
    int32_t abi_version; /* TRIPS_ABI_VERSION */
    int32_t dtype;       /* of x, residual and out: TRIPS_DTYPE_F32, _BF16 or _F16 */
    int64_t n;           /* elements, one behind the other, below 2^40 */
    double p;            /* 0 to 1 */
    uint64_t seed;
    uint32_t call;
    uint32_t step;       /* where step_at is NULL */
} TripsDropoutDesc;

/* residual: [n] or NULL. step_at: a word on the device that holds the step, or NULL; step_used: a word on the device that the
 * step is written to for the gradient's call, or NULL. out may be x or the residual. */
int trips_dropout(TripsCtx* ctx, const TripsDropoutDesc* desc, const void* x, const void* residual, const uint32_t* step_at, uint32_t* step_used,
                  void* out, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TRIPS_LOSS_H */
