/* grouped_args.h — operands of a product by expert, from the entry points
 * (hip_kernels.c) to its launchers:
 *   y[p] = epi(x[src(p)] W[e(p)]^T + bias[e(p)]).
 * w holds 16-bit values [E][N][K], or 4-bit codes [E][N][K / 2] with group > 0;
 * strides are in elements (codes: bytes). */
#ifndef PYC_GROUPED_ARGS_H
#define PYC_GROUPED_ARGS_H

#include <stdint.h>

typedef struct {
    const uint16_t* x;
    int64_t x_stride;
    int x_rows;
    const int32_t* rows;    /* src(p) = rows[p] / fan; NULL: p */
    int fan;
    const int32_t* offsets; /* [E + 1]; NULL: one expert has every row */
    int E, P;               /* P: rows of y */
    const void* w;
    int64_t w_stride;       /* from an expert's weights to the next one's */
    int N, K;
    const uint16_t* scale;  /* 4-bit: [E][N][K / group] */
    const uint8_t* zeros;   /* the same, or NULL: 8 */
    int group;
    const float* bias;      /* [E][N] or NULL */
    uint16_t* y;
    int64_t y_stride;
    int epi;                /* PYC_HIP_EPI_* */
} pyc_grouped;

#endif
