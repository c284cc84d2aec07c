/*
 * ops_launch.h -- plain-C interface between the host side (ops_engine.c) and the kernels of the operators on device
 * memory: routing, norms around a block and the block-scaled FP8 quantiser (ops_rows.cu), the FP8 products (ops_f8.cu).
 * Arguments have been checked by the host side; every launcher returns a cudaError_t as int.
 */
#ifndef FOMOE_B200_OPS_LAUNCH_H
#define FOMOE_B200_OPS_LAUNCH_H

#include <stdint.h>

#include "../../include/fomoe_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define OPS_MAX_E 512  /* experts of a layer */
#define OPS_MAX_K 16   /* experts of a token */
#define OPS_MAX_N 16384 /* columns of a normalised row */

typedef struct {
    fomoe_b200_route_config_t cfg;
    int n_tokens, logits_bf16;
    const void *logits;
    int64_t row_stride;
    const float *bias;
    const uint8_t *valid;
    int *ids;
    float *weights;
} ops_route_t;

/* Where kernels store 1 when FB_ST_.. `st` happens: a word each, so that neither hides the other. */
#define OPS_STATUS_WORD(st) ((st) - 1)
#define OPS_STATUS_WORDS 2

int ops_rows_init(void); /* loads the kernels on the current device */
int ops_launch_route(const ops_route_t *a, void *stream);
int ops_launch_norm(const fomoe_b200_norm_args_t *a, void *stream);
int ops_launch_f8_quantize(int rows, int cols, const void *x, int x_bf16, int64_t x_stride, uint8_t *q, int64_t q_stride,
                           float *scales, int64_t scales_stride, void *stream);

/* Where the parts of the experts' workspace lie, in bytes from its start (all 256-byte aligned). */
typedef struct {
    uint64_t counts, block_counts, pairs, pos, xp, xp_scales, act_q, act_scales, dots, bytes;
    int n_pairs; /* routed and shared pairs */
} ops_experts_ws_t;

/* What the product launchers go by on a device. */
typedef struct {
    int n_sm;
    int clusters[4]; /* clusters of 1, 2, 4, 8 blocks of the split product that the device runs at the same time */
} ops_device_t;

int ops_f8_init(ops_device_t *d); /* loads the kernels on the current device; n_sm is given */
int ops_launch_f8_matmul(const fomoe_b200_f8_matmul_args_t *a, int *status, const ops_device_t *d, int *launches, void *stream);
void ops_experts_layout(const fomoe_b200_f8_experts_args_t *a, ops_experts_ws_t *w);
int ops_launch_f8_experts(const fomoe_b200_f8_experts_args_t *a, uint8_t *ws, int *status, const ops_device_t *d,
                          int *launches, void *stream);

#ifdef __cplusplus
}
#endif
#endif
