/* C ABI of table lookups: the entries of a table (a scene's texels, a model's embeddings) by index, scaled, and their
 * gradient, summed in the order of the indexes. Same library and context as trips_splat.h.
 *
 * The reference looks a point's descriptor up inside its render kernels (texture [C,T] by t_index,
 * src/lib/rendering/RenderForward.cu:875-899) and adds its gradient with float atomics (RenderBackward.cu:262-302), which
 * leaves the order of a texel's sum to chance where points share it. Here the order is that of the points.
 *
 * Every call is stream-ordered, allocates nothing, does not synchronise and may be captured into a HIP graph. Launches go
 * to the context's device, whichever is current.
 */
#ifndef TRIPS_LOOKUP_H
#define TRIPS_LOOKUP_H

#include <stddef.h>
#include <stdint.h>

#include "trips_optim.h"
#include "trips_splat.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { TRIPS_TABLE_COLUMNS = 0, TRIPS_TABLE_ROWS = 1 };
enum { TRIPS_INDEX_I64 = 0, TRIPS_INDEX_I32 = 1 };

/* COLUMNS: the table is [num_channels, num_texels], what is looked up [num_channels, num_points] (the scene's texture).
 * ROWS: [num_texels, num_channels] and [num_points, num_channels]. Strides are the elements between two rows of memory
 * (two channels, or two texels or points); within a row elements are adjacent. A stride may be 0 where the call only reads. */
typedef struct TripsLookupDesc {
    int32_t abi_version; /* TRIPS_ABI_VERSION */
    int32_t layout;      /* TRIPS_TABLE_* */
    int32_t dtype;       /* of table, values and gradients: TRIPS_DTYPE_F32, _BF16 or _F16 */
    int32_t index_dtype; /* TRIPS_INDEX_* */
    int64_t num_texels;  /* T, below 2^31 - 1 */
    int64_t num_points;  /* N, below 2^31 - 1 */
    int32_t num_channels; /* C, below 2^17 */
    int32_t accumulate;   /* backward: 0 = d_table is written, zeros where no point refers to; 1 = added to */
    int64_t table_stride;  /* of table and d_table */
    int64_t values_stride; /* of values and d_values */
    float scale;
} TripsLookupDesc;

/* values of point i = scale * (entry index[i] of the table), rounded once; zeros where index[i] is outside [0, T).
 * `workspace`: trips_lookup_workspace_size bytes (0 in the rows layout), 256-byte aligned, of any content, like those below;
 * calls that share one must not overlap. */
int trips_lookup_workspace_size(const TripsLookupDesc* desc, size_t* bytes);
int trips_lookup_forward(TripsCtx* ctx, const TripsLookupDesc* desc, const void* table, const void* index, void* values,
                         void* workspace, size_t workspace_bytes, void* stream);

/* The points in the order of their indexes: order [N] lists the points by (index, point), those with an index outside [0, T)
 * last; those of texel t are order[starts[t]] to order[starts[t + 1] - 1], starts [T + 1]. */
int trips_lookup_plan_workspace_size(int64_t num_texels, int64_t num_points, size_t* bytes);
int trips_lookup_plan(TripsCtx* ctx, int64_t num_texels, int64_t num_points, const void* index, int index_dtype, int32_t* order,
                      int32_t* starts, void* workspace, size_t workspace_bytes, void* stream);

/* d_table of texel t = (accumulate: d_table +) scale * sum of d_values over the points of texel t, summed in 32 bits in an
 * order that depends on `order`, `starts` and the sizes alone, and rounded once. `order` and `starts` as trips_lookup_plan
 * leaves them (points outside [0, N) in `order` are passed over). */
int trips_lookup_backward_workspace_size(const TripsLookupDesc* desc, size_t* bytes);
int trips_lookup_backward(TripsCtx* ctx, const TripsLookupDesc* desc, const void* d_values, const int32_t* order,
                          const int32_t* starts, void* d_table, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TRIPS_LOOKUP_H */
