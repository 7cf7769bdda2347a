/* vegs_embedding.h -- C ABI of the row lookup: rows of a shared, learnable table by index, scaled, and its gradients.  Same
 * library and conventions as vegs_rast.h.
 *
 *     out[i] = s_i * table[ids[i]]              s_i = scale * row_scale[i];  zeros where ids[i] is outside [0, rows)
 *     d_table[k] = sum over i with ids[i] == k, in order of i, of s_i * grad[i]
 *     d_row_scale[i] = scale * <grad[i], table[ids[i]]>        0 where ids[i] is outside [0, rows)
 */
#ifndef VEGS_EMBEDDING_H
#define VEGS_EMBEDDING_H

#include "vegs_optim.h"   /* VrDataType */

#ifdef __cplusplus
extern "C" {
#endif

typedef struct VrLookup {
    const void* table;       /* device [rows, width], rows table_stride elements apart */
    const void* ids;         /* device [n], int32 or int64; any value (outside [0, rows): "no row") */
    const float* row_scale;  /* device [n]; NULL: ones */
    int64_t n;               /* < 2^30 */
    int64_t rows;            /* < 2^31 - 1 */
    int64_t width;           /* 1 .. 2^22 */
    int64_t table_stride;    /* >= width */
    int32_t table_dtype;     /* VrDataType */
    int32_t out_dtype;       /* VrDataType of out and grad: table_dtype, or VR_F32 */
    int32_t ids_64;          /* 0: int32, 1: int64 */
    float scale;
} VrLookup;

/* out [n, width], rows one after the other. */
int vr_lookup_forward(const VrLookup* lookup, void* out, void* stream);

/* Bytes of device scratch that vr_lookup_backward needs for the table's gradient (0: none -- few entries -- or bad sizes). */
int64_t vr_lookup_scratch_bytes(int64_t n, int64_t rows, int64_t width);

/* grad [n, width], rows grad_stride elements apart.  d_table [rows, width] in the table's type, every element written; NULL:
 * not wanted (scratch may be NULL then, and where no scratch is needed).  d_row_scale [n] fp32; NULL: not wanted
 * (no value of the table is read then).  Sums are fp32 (in pieces of a fixed size that are
 * joined in order: the same inputs give the same bits) and rounded once. */
int vr_lookup_backward(const VrLookup* lookup, const void* grad, int64_t grad_stride, void* d_table, float* d_row_scale,
                       void* scratch, int64_t scratch_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
