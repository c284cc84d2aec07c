/*
 * ops_engine.c -- host side of the operators on device memory: the handle, the checks of every argument that the host
 * can see, and the switch to the handle's device and back.  Nothing here allocates device memory after create, and
 * nothing synchronises.
 */
#include <cuda_runtime_api.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/fomoe_b200.h"
#include "launch.h"
#include "ops_launch.h"

struct fomoe_b200_ops {
    int device;
    ops_device_t dev;
    int *status; /* OPS_STATUS_WORDS of mapped host memory: kernels store into them, the host reads them without a copy */
    int *status_dev;
    uint64_t launches;
    char err[256];
};

static int oerr(fomoe_b200_ops_t *o, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(o->err, sizeof(o->err), fmt, ap);
    va_end(ap);
    fprintf(stderr, "fomoe_b200 (ops): %s\n", o->err);
    return -1;
}

#define NEED(o, cond, ...) \
    do {                   \
        if (!(cond)) return oerr((o), __VA_ARGS__); \
    } while (0)

fomoe_b200_ops_t *fomoe_b200_ops_create(int device) {
    int was = 0, n = 0, major = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n || cudaGetDevice(&was) != cudaSuccess) {
        fprintf(stderr, "fomoe_b200_ops_create: no CUDA device %d\n", device);
        return NULL;
    }
    fomoe_b200_ops_t *o = (fomoe_b200_ops_t *)calloc(1, sizeof(*o));
    if (!o) return NULL;
    o->device = device;
    int ok = cudaSetDevice(device) == cudaSuccess &&
             cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device) == cudaSuccess && major == 10 &&
             cudaDeviceGetAttribute(&o->dev.n_sm, cudaDevAttrMultiProcessorCount, device) == cudaSuccess &&
             cudaHostAlloc((void **)&o->status, 64, cudaHostAllocMapped) == cudaSuccess &&
             cudaHostGetDevicePointer((void **)&o->status_dev, o->status, 0) == cudaSuccess &&
             ops_rows_init() == 0 && ops_f8_init(&o->dev) == 0;
    if (ok) {
        memset(o->status, 0, OPS_STATUS_WORDS * sizeof(int));
    } else {
        fprintf(stderr, "fomoe_b200_ops_create: device %d cannot be used: %s\n", device, cudaGetErrorString(cudaGetLastError()));
        if (o->status) cudaFreeHost(o->status);
        free(o);
        o = NULL;
    }
    cudaSetDevice(was);
    return o;
}

/* The status words stay for the life of the process: calls in flight and graphs that hold some of this handle's go on
 * storing into them.  They are no later handle's either, which would hear of what is not its own. */
void fomoe_b200_ops_destroy(fomoe_b200_ops_t *o) { free(o); }

const char *fomoe_b200_ops_last_error(fomoe_b200_ops_t *o) { return o ? o->err : "no handle"; }

int fomoe_b200_ops_status(fomoe_b200_ops_t *o) {
    if (!o) return -1;
    /* the worse first; read and cleared in one step, so that nothing stored in between is lost */
    for (int st = OPS_STATUS_WORDS; st > FB_ST_OK; st--)
        if (__atomic_exchange_n(&o->status[OPS_STATUS_WORD(st)], 0, __ATOMIC_ACQ_REL)) return st;
    return FB_ST_OK;
}

uint64_t fomoe_b200_ops_kernel_launches(fomoe_b200_ops_t *o) { return o ? o->launches : 0; }

/* run `expr` (a launcher's return code) on the handle's device */
#define ON_DEVICE(o, what, n_launch, expr)                                                              \
    do {                                                                                               \
        int was_ = -1, rc_;                                                                            \
        if (cudaGetDevice(&was_) != cudaSuccess) return oerr((o), "%s: no current CUDA device", what); \
        if (was_ != (o)->device && cudaSetDevice((o)->device) != cudaSuccess)                          \
            return oerr((o), "%s: device %d cannot be made current", what, (o)->device);               \
        rc_ = (expr);                                                                                  \
        if (was_ != (o)->device) cudaSetDevice(was_);                                                  \
        if (rc_ != 0) return oerr((o), "%s: launch failed: %s", what, cudaGetErrorString((cudaError_t)rc_)); \
        (o)->launches += (uint64_t)(n_launch);                                                         \
    } while (0)

#define OPS_MOST (1 << 30) /* rows, columns: index arithmetic in 32 bits goes a little past them */

static int is_float(int type) { return type == FOMOE_B200_F32 || type == FOMOE_B200_BF16; }
static int fits(const void *p, int type) { /* aligned to its own type */
    return ((uintptr_t)p & (type == FOMOE_B200_F32 ? 3u : 1u)) == 0;
}

int fomoe_b200_ops_route(fomoe_b200_ops_t *o, const fomoe_b200_route_config_t *c, int n_tokens, const void *logits,
                         int logits_type, int64_t row_stride, const float *bias, const uint8_t *valid, int *ids,
                         float *weights, void *stream) {
    if (!o) return -1;
    NEED(o, c && c->n_experts > 0 && c->n_experts <= OPS_MAX_E, "route: 1 to %d experts", OPS_MAX_E);
    NEED(o, c->top_k > 0 && c->top_k <= OPS_MAX_K && c->top_k <= c->n_experts, "route: top_k is 1 to %d and at most n_experts", OPS_MAX_K);
    NEED(o, c->score == FOMOE_B200_SOFTMAX || c->score == FOMOE_B200_SIGMOID, "route: unknown score %d", c->score);
    NEED(o, c->n_group > 0 && c->n_group <= 32 && c->n_experts % c->n_group == 0, "route: n_group is 1 to 32 and divides n_experts");
    NEED(o, c->topk_group > 0 && c->topk_group <= c->n_group, "route: topk_group is 1 to n_group");
    NEED(o, c->group_best == 1 || c->group_best == 2, "route: group_best is 1 or 2");
    NEED(o, is_float(logits_type), "route: logits are F32 or BF16");
    NEED(o, n_tokens >= 0 && n_tokens <= OPS_MOST, "route: %d tokens", n_tokens);
    if (n_tokens == 0) return 0;
    NEED(o, logits && ids && weights, "route: a pointer is NULL");
    NEED(o, fits(logits, logits_type) && fits(bias, FOMOE_B200_F32) && fits(ids, FOMOE_B200_F32) && fits(weights, FOMOE_B200_F32), "route: a pointer is not aligned to its type");
    NEED(o, row_stride >= c->n_experts || n_tokens == 1, "route: row_stride %lld is below n_experts", (long long)row_stride);
    ops_route_t a;
    a.cfg = *c;
    a.n_tokens = n_tokens;
    a.logits = logits;
    a.logits_bf16 = logits_type == FOMOE_B200_BF16;
    a.row_stride = row_stride;
    a.bias = bias;
    a.valid = valid;
    a.ids = ids;
    a.weights = weights;
    ON_DEVICE(o, "route", 1, ops_launch_route(&a, stream));
    return 0;
}

int fomoe_b200_ops_norm(fomoe_b200_ops_t *o, const fomoe_b200_norm_args_t *a, void *stream) {
    if (!o) return -1;
    NEED(o, a && a->n > 0 && a->n <= OPS_MAX_N, "norm: 1 to %d columns", OPS_MAX_N);
    NEED(o, a->n_tokens >= 0 && a->n_tokens <= OPS_MOST, "norm: %d tokens", a->n_tokens);
    if (a->n_tokens == 0) return 0;
    NEED(o, a->x && is_float(a->x_type) && fits(a->x, a->x_type), "norm: x is F32 or BF16, aligned to its type");
    NEED(o, a->x_stride >= a->n || a->n_tokens == 1, "norm: x_stride is below n");
    if (a->block) {
        NEED(o, is_float(a->block_type) && fits(a->block, a->block_type), "norm: the block is F32 or BF16, aligned to its type");
        NEED(o, a->block_stride >= 0, "norm: a stride is negative");
        NEED(o, fits(a->post, FOMOE_B200_F32) && fits(a->gate, a->block_type), "norm: a pointer is not aligned to its type");
        NEED(o, !a->gate || (a->gate_stride >= 0 && (a->gate_step == 0 || a->gate_step == 1)), "norm: gate_stride is not negative, gate_step 0 or 1");
    } else {
        NEED(o, !a->post && !a->gate, "norm: post and gate need a block");
    }
    NEED(o, a->x_out || a->pre, "norm: neither x_out nor pre: nothing to write");
    if (a->x_out) {
        NEED(o, fits(a->x_out, a->x_type), "norm: x_out is not aligned to its type");
        NEED(o, a->x_out_stride >= a->n || a->n_tokens == 1, "norm: x_out_stride is below n");
        NEED(o, a->x_out != a->x || a->x_out_stride == a->x_stride || a->n_tokens == 1, "norm: x_out is x: the strides have to be the same");
    }
    if (a->pre) {
        NEED(o, fits(a->pre, FOMOE_B200_F32), "norm: a pointer is not aligned to its type");
        NEED(o, a->h && (a->h_type == FOMOE_B200_F8 || (is_float(a->h_type) && fits(a->h, a->h_type))), "norm: h is F32, BF16 or F8, aligned to its type");
        NEED(o, a->h_stride >= a->n || a->n_tokens == 1, "norm: h_stride is below n");
        if (a->h_type == FOMOE_B200_F8) {
            NEED(o, a->h_scales && fits(a->h_scales, FOMOE_B200_F32), "norm: h_scales is NULL or not aligned");
            NEED(o, a->h_scales_stride >= (a->n + 127) / 128 || a->n_tokens == 1, "norm: h_scales_stride is below the number of blocks");
        }
    }
    ON_DEVICE(o, "norm", 1, ops_launch_norm(a, stream));
    return 0;
}

int fomoe_b200_ops_f8_quantize(fomoe_b200_ops_t *o, int rows, int cols, const void *x, int x_type, int64_t x_stride,
                               uint8_t *q, int64_t q_stride, float *scales, int64_t scales_stride, void *stream) {
    if (!o) return -1;
    NEED(o, rows >= 0 && rows <= OPS_MOST && cols > 0 && cols <= OPS_MOST, "f8_quantize: %d x %d", rows, cols);
    if (rows == 0) return 0;
    NEED(o, x && q && scales, "f8_quantize: a pointer is NULL");
    NEED(o, is_float(x_type) && fits(x, x_type) && fits(scales, FOMOE_B200_F32), "f8_quantize: x is F32 or BF16, pointers aligned to their types");
    NEED(o, rows == 1 || (x_stride >= 0 && q_stride >= cols && scales_stride >= ((int64_t)cols + 127) / 128), "f8_quantize: a stride is too small");
    ON_DEVICE(o, "f8_quantize", 1, ops_launch_f8_quantize(rows, cols, x, x_type == FOMOE_B200_BF16, x_stride, q, q_stride, scales, scales_stride, stream));
    return 0;
}

int fomoe_b200_ops_f8_matmul(fomoe_b200_ops_t *o, const fomoe_b200_f8_matmul_args_t *args, void *stream) {
    if (!o) return -1;
    NEED(o, args && args->m >= 0 && args->m <= OPS_MOST && args->n >= 0 && args->n <= OPS_MOST / 2, "f8_matmul: m is 0 to 2^30, n 0 to 2^29"); /* (bytes of a row of out go into a signed coordinate) */
    NEED(o, args->k > 0 && args->k <= OPS_MOST && args->k % 16 == 0, "f8_matmul: k is a positive multiple of 16");
    if (args->m == 0 || args->n == 0) return 0;
    fomoe_b200_f8_matmul_args_t own = *args, *a = &own;
    if (a->m == 1) a->a_stride = a->k; /* a single row's stride means nothing */
    if (a->n == 1) a->b_stride = a->k;
    const int64_t nb = ((int64_t)a->k + 127) / 128;
    NEED(o, a->a && a->a_scales && a->b && a->b_scales && a->out, "f8_matmul: a pointer is NULL");
    NEED(o, ((uintptr_t)a->a & 15) == 0 && ((uintptr_t)a->b & 15) == 0 && a->a_stride % 16 == 0 && a->b_stride % 16 == 0, "f8_matmul: a and b are 16-byte aligned and their strides multiples of 16");
    NEED(o, a->a_stride >= a->k && a->b_stride >= a->k, "f8_matmul: a stride is below k");
    NEED(o, (a->a_scales_stride >= nb || a->m == 1) && (a->b_scales_stride >= nb || a->n <= 128), "f8_matmul: a stride of the scales is below the number of blocks");
    NEED(o, is_float(a->out_type) && fits(a->out, a->out_type) && fits(a->a_scales, FOMOE_B200_F32) && fits(a->b_scales, FOMOE_B200_F32), "f8_matmul: out is F32 or BF16, pointers aligned to their types");
    NEED(o, a->out_stride >= a->n || a->m == 1, "f8_matmul: out_stride is below n");
    int n = 0;
    ON_DEVICE(o, "f8_matmul", n, ops_launch_f8_matmul(a, o->status_dev, &o->dev, &n, stream));
    return 0;
}

static int experts_sizes_ok(const fomoe_b200_f8_experts_args_t *a) {
    return a && a->n_tokens >= 0 && a->n_embd > 0 && a->n_embd <= OPS_MAX_N && a->n_embd % 128 == 0 && a->n_inter > 0 &&
           a->n_inter <= OPS_MAX_N && a->n_inter % 128 == 0 && a->n_experts > 0 && a->n_experts <= OPS_MAX_E && a->top_k > 0 &&
           a->top_k <= OPS_MAX_K && (a->has_shared == 0 || a->has_shared == 1) &&
           (int64_t)a->n_tokens * (a->top_k + 1) <= (1 << 22);
}

uint64_t fomoe_b200_ops_f8_experts_workspace(const fomoe_b200_f8_experts_args_t *a) {
    if (!experts_sizes_ok(a)) return 0;
    ops_experts_ws_t w;
    ops_experts_layout(a, &w);
    return w.bytes;
}

int fomoe_b200_ops_f8_experts(fomoe_b200_ops_t *o, const fomoe_b200_f8_experts_args_t *args, void *workspace,
                              uint64_t workspace_bytes, void *stream) {
    if (!o) return -1;
    NEED(o, experts_sizes_ok(args), "f8_experts: n_embd and n_inter are multiples of 128 up to %d, 1 to %d experts, top_k 1 to %d, at most 2^22 pairs", OPS_MAX_N, OPS_MAX_E, OPS_MAX_K);
    if (args->n_tokens == 0) return 0;
    fomoe_b200_f8_experts_args_t own = *args, *a = &own;
    if (a->n_tokens == 1) a->x_stride = a->n_embd; /* a single row's stride means nothing */
    NEED(o, a->x && a->x_scales && a->ids && a->weights && a->gate_up && a->gate_up_scales && a->down && a->down_scales && a->out, "f8_experts: a pointer is NULL");
    NEED(o, ((uintptr_t)a->x & 15) == 0 && ((uintptr_t)a->gate_up & 15) == 0 && ((uintptr_t)a->down & 15) == 0 && a->x_stride % 16 == 0, "f8_experts: x and the tables are 16-byte aligned, x_stride a multiple of 16");
    NEED(o, fits(a->x_scales, FOMOE_B200_F32) && fits(a->gate_up_scales, FOMOE_B200_F32) && fits(a->down_scales, FOMOE_B200_F32) && fits(a->ids, FOMOE_B200_F32) && fits(a->weights, FOMOE_B200_F32) && fits(a->out, FOMOE_B200_BF16), "f8_experts: a pointer is not aligned to its type");
    NEED(o, a->n_tokens == 1 || (a->x_stride >= a->n_embd && a->x_scales_stride >= a->n_embd / 128 && a->out_stride >= a->n_embd), "f8_experts: a stride is too small");
    NEED(o, workspace && ((uintptr_t)workspace & 255) == 0, "f8_experts: the workspace is NULL or not 256-byte aligned");
    NEED(o, workspace_bytes >= fomoe_b200_ops_f8_experts_workspace(a), "f8_experts: the workspace has %llu bytes, %llu are needed", (unsigned long long)workspace_bytes, (unsigned long long)fomoe_b200_ops_f8_experts_workspace(a));
    int n = 0;
    ON_DEVICE(o, "f8_experts", n, ops_launch_f8_experts(a, (uint8_t *)workspace, o->status_dev, &o->dev, &n, stream));
    return 0;
}
