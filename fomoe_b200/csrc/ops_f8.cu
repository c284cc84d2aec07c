/*
 * ops_f8.cu -- products of FP8 (e4m3) rows with FP8 weight matrices, both with block scales: the plain product and the
 * experts of a layer.
 */
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "launch.h"
#include "ops_launch.h"
#include "ops_quant.cuh"

#ifndef FULL
#define FULL 0xffffffffu
#endif

/* ------------------------------------------------------------------ bucket: the pairs of every expert, in pair order
 * One block.  Warp w owns a contiguous run of pairs; a first walk counts each warp's pairs of every expert, a prefix over
 * (expert, warp) gives every warp its first place, a second walk places the pairs.  The order inside an expert is the
 * order of the pairs, so results do not depend on timing.  The shared expert's pairs (n_routed + t) come last. */
#define BK_THREADS 1024
#define BK_WARPS 32

__global__ void __launch_bounds__(BK_THREADS) k_ops_bucket(const int *ids, int n_routed, int n_tokens, int n_experts,
                                                          int has_shared, int *counts, int *pairs, int4 *items,
                                                          int *status) {
    extern __shared__ int s_cnt[]; /* [n_experts][BK_WARPS] */
    __shared__ int s_tot[BK_WARPS], s_til[BK_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < n_experts * BK_WARPS; i += BK_THREADS) s_cnt[i] = 0;
    __syncthreads();
    const int run = ((n_routed + BK_THREADS - 1) / BK_THREADS) * 32; /* pairs of a warp */
    const int p0 = warp * run, p1 = min(n_routed, p0 + run);
    for (int pass = 0; pass < 2; pass++) {
        for (int b = p0; b < p1; b += 32) {
            const int p = b + lane;
            int e = p < p1 ? ids[p] : -1;
            if (e < -1 || e >= n_experts) {
                if (pass == 0) *status = FB_ST_BAD_ID;
                e = -1;
            }
            const unsigned same = __match_any_sync(FULL, e);
            if (e >= 0) {
                const int rank = __popc(same & ((1u << lane) - 1u)), at = s_cnt[e * BK_WARPS + warp];
                if (pass == 1) pairs[at + rank] = p;
            }
            __syncwarp();
            if (e >= 0 && lane == __ffs(same) - 1) s_cnt[e * BK_WARPS + warp] += __popc(same);
            __syncwarp();
        }
        if (pass == 1) break;
        __syncthreads();
        /* thread e: the expert's total, then exclusive prefixes of pairs and of 128-row tiles over the experts */
        int tot = 0;
        if (tid < n_experts)
            for (int w = 0; w < BK_WARPS; w++) tot += s_cnt[tid * BK_WARPS + ((w + tid) & 31)];
        const int til = (tot + 127) / 128;
        int a = tot, c = til;
        for (int s = 1; s < 32; s <<= 1) {
            const int oa = __shfl_up_sync(FULL, a, s), oc = __shfl_up_sync(FULL, c, s);
            if (lane >= s) {
                a += oa;
                c += oc;
            }
        }
        if (lane == 31) {
            s_tot[warp] = a;
            s_til[warp] = c;
        }
        __syncthreads();
        int base = a - tot, tbase = c - til;
        for (int w = 0; w < warp; w++) {
            base += s_tot[w];
            tbase += s_til[w];
        }
        if (tid < n_experts) {
            int at = base;
            for (int w = 0; w < BK_WARPS; w++) {
                const int n = s_cnt[tid * BK_WARPS + w];
                s_cnt[tid * BK_WARPS + w] = at;
                at += n;
            }
            for (int m = 0; m < til; m++) items[tbase + m] = make_int4(tid, base + 128 * m, min(128, tot - 128 * m), 0);
        }
        if (tid == BK_THREADS - 1) { /* no expert's thread: n_experts <= 512 */
            const int sh = has_shared ? (n_tokens + 127) / 128 : 0;
            for (int m = 0; m < sh; m++)
                items[tbase + m] = make_int4(n_experts, base + 128 * m, min(128, n_tokens - 128 * m), 0);
            counts[0] = tbase + sh; /* tiles */
            counts[1] = base;       /* routed pairs that are left */
        }
        __syncthreads();
    }
    if (has_shared) {
        int base = 0;
        for (int w = 0; w < BK_WARPS; w++) base += s_tot[w];
        for (int t = tid; t < n_tokens; t += BK_THREADS) pairs[base + t] = n_routed + t;
    }
}

/* ------------------------------------------------------------------ products: 64 x 64 tiles on the FP32 pipes */
enum { F8_DENSE = 0, F8_GATE_UP = 1, F8_DOWN = 2 };

typedef struct {
    int m, n, k; /* n: rows of b, of one half (gate or up) for F8_GATE_UP */
    const uint8_t *a;
    int64_t a_stride;
    const float *a_scales;
    int64_t as_stride;
    const uint8_t *b;
    int64_t b_stride, b_rec; /* bytes of a row, of a record */
    const float *b_scales;
    int64_t bs_stride, bs_rec;
    void *out;
    int out_bf16;
    int64_t out_stride;
    const int *counts, *pairs;
    const int4 *items;
    int n_routed, top_k;
} f8_args_t;

__device__ __forceinline__ float f8_val(uint8_t v) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(v, __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half *>(&h));
}

template <int MODE>
__global__ void __launch_bounds__(256) k_f8_tile(f8_args_t P) {
    __shared__ float s_a[32][65], s_b[2][32][65];
    __shared__ int s_row[64];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    int e = 0, r0, rows;
    if (MODE == F8_DENSE) {
        r0 = blockIdx.x * 64;
        rows = min(64, P.m - r0);
    } else {
        if ((int)(blockIdx.x >> 1) >= P.counts[0]) return;
        const int4 it = P.items[blockIdx.x >> 1];
        e = it.x;
        r0 = it.y + 64 * (blockIdx.x & 1);
        rows = min(64, it.z - 64 * (int)(blockIdx.x & 1));
        if (rows <= 0) return;
    }
    const int n0 = blockIdx.y * 64, kb_n = (P.k + 127) / 128;
    if (tid < 64) {
        int r = r0 + min(tid, rows - 1);
        if (MODE == F8_GATE_UP) {
            const int p = P.pairs[r];
            r = p < P.n_routed ? p / P.top_k : p - P.n_routed;
        }
        s_row[tid] = r;
    }
    const uint8_t *b = P.b + e * P.b_rec;
    const float *bs = P.b_scales + e * P.bs_rec;
    const int halves = MODE == F8_GATE_UP ? 2 : 1;
    float acc[2][4][4] = {};
    for (int kb = 0; kb < kb_n; kb++) {
        float part[2][4][4] = {};
        for (int k0 = kb * 128; k0 < min(P.k, kb * 128 + 128); k0 += 32) {
            __syncthreads();
            for (int i = tid; i < 64 * 32; i += 256) {
                const int r = i >> 5, k = k0 + (i & 31);
                s_a[i & 31][r] = k < P.k ? f8_val(P.a[s_row[r] * P.a_stride + k]) : 0.0f;
                for (int h = 0; h < halves; h++)
                    s_b[h][i & 31][r] =
                        k < P.k && n0 + r < P.n ? f8_val(b[(int64_t)(h * P.n + n0 + r) * P.b_stride + k]) : 0.0f;
            }
            __syncthreads();
            for (int k = 0; k < 32; k++)
                for (int h = 0; h < halves; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            part[h][i][j] = fmaf(s_a[k][ty + 16 * i], s_b[h][k][tx + 16 * j], part[h][i][j]);
        }
        for (int i = 0; i < 4; i++) {
            const float sa = P.a_scales[s_row[ty + 16 * i] * P.as_stride + kb];
            for (int h = 0; h < halves; h++)
                for (int j = 0; j < 4; j++) {
                    const int n = min(n0 + tx + 16 * j, P.n - 1);
                    acc[h][i][j] = fmaf(part[h][i][j], sa * bs[(int64_t)((h * P.n + n) >> 7) * P.bs_stride + kb], acc[h][i][j]);
                }
        }
    }
    for (int i = 0; i < 4; i++) {
        const int r = ty + 16 * i;
        if (r >= rows) continue;
        const int64_t o = (MODE == F8_DOWN ? P.pairs[r0 + r] : r0 + r) * P.out_stride;
        for (int j = 0; j < 4; j++) {
            const int n = n0 + tx + 16 * j;
            if (n >= P.n) continue;
            float v = acc[0][i][j];
            if (MODE == F8_GATE_UP) v = v / (1.0f + expf(-v)) * acc[1][i][j];
            if (P.out_bf16) reinterpret_cast<__nv_bfloat16 *>(P.out)[o + n] = __float2bfloat16_rn(v);
            else reinterpret_cast<float *>(P.out)[o + n] = v;
        }
    }
}

extern "C" int ops_launch_f8_matmul(const fomoe_b200_f8_matmul_args_t *a, int *status, int n_sm, int *launches,
                                    void *stream) {
    (void)status;
    (void)n_sm;
    f8_args_t p = {};
    p.m = a->m, p.n = a->n, p.k = a->k;
    p.a = a->a, p.a_stride = a->a_stride, p.a_scales = a->a_scales, p.as_stride = a->a_scales_stride;
    p.b = a->b, p.b_stride = a->b_stride, p.b_scales = a->b_scales, p.bs_stride = a->b_scales_stride;
    p.out = a->out, p.out_bf16 = a->out_type == FOMOE_B200_BF16, p.out_stride = a->out_stride;
    k_f8_tile<F8_DENSE><<<dim3((a->m + 63) / 64, (a->n + 63) / 64), 256, 0, (cudaStream_t)stream>>>(p);
    *launches += 1;
    return (int)cudaGetLastError();
}

/* ------------------------------------------------------------------ out[t] = sum over the slots, in slot order */
__global__ void __launch_bounds__(256) k_ops_combine(const float *dots, const int *ids, const float *weights, int n_embd,
                                                    int n_experts, int top_k, int n_routed, int has_shared,
                                                    __nv_bfloat16 *out, int64_t out_stride) {
    const int t = blockIdx.x;
    for (int c = threadIdx.x; c < n_embd; c += 256) {
        float v = 0.0f;
        for (int j = 0; j < top_k; j++) {
            const int p = t * top_k + j;
            if ((unsigned)ids[p] < (unsigned)n_experts) v = fmaf(weights[p], dots[(int64_t)p * n_embd + c], v);
        }
        if (has_shared) v += dots[(int64_t)(n_routed + t) * n_embd + c];
        out[t * out_stride + c] = __float2bfloat16_rn(v);
    }
}

extern "C" void ops_experts_layout(const fomoe_b200_f8_experts_args_t *a, ops_experts_ws_t *w) {
    const uint64_t np = (uint64_t)a->n_tokens * (a->top_k + (a->has_shared ? 1 : 0));
    const uint64_t items = np / 128 + a->n_experts + 1;
    uint64_t at = 0;
#define PART(name, n) w->name = at, at += ((uint64_t)(n) + 255) & ~255ull
    w->n_pairs = (int)np;
    PART(counts, 256 + 16 * items); /* {tiles, pairs}, then the tiles */
    PART(pairs, 4 * np);
    PART(act_q, np * a->n_inter);
    PART(act_scales, np * (a->n_inter / 128) * 4);
    PART(act, np * a->n_inter * 4);
    PART(dots, np * a->n_embd * 4);
#undef PART
    w->bytes = at;
}

extern "C" int ops_launch_f8_experts(const fomoe_b200_f8_experts_args_t *a, uint8_t *ws, int *status, int n_sm,
                                     int *launches, void *stream) {
    (void)n_sm;
    cudaStream_t st = (cudaStream_t)stream;
    ops_experts_ws_t w;
    ops_experts_layout(a, &w);
    const int n_routed = a->n_tokens * a->top_k, H = a->n_embd, I = a->n_inter;
    int *counts = (int *)(ws + w.counts), *pairs = (int *)(ws + w.pairs);
    int4 *items = (int4 *)(ws + w.counts + 256);
    k_ops_bucket<<<1, BK_THREADS, (size_t)a->n_experts * BK_WARPS * 4, st>>>(a->ids, n_routed, a->n_tokens, a->n_experts,
                                                                            a->has_shared, counts, pairs, items, status);
    f8_args_t p = {};
    p.counts = counts, p.pairs = pairs, p.items = items, p.n_routed = n_routed, p.top_k = a->top_k;
    p.n = I, p.k = H;
    p.a = a->x, p.a_stride = a->x_stride, p.a_scales = a->x_scales, p.as_stride = a->x_scales_stride;
    p.b = a->gate_up, p.b_stride = H, p.b_rec = (int64_t)2 * I * H;
    p.b_scales = a->gate_up_scales, p.bs_stride = H / 128, p.bs_rec = (int64_t)(2 * I / 128) * (H / 128);
    p.out = ws + w.act, p.out_stride = I;
    const int tiles = (w.n_pairs + 127) / 128 + a->n_experts + 1;
    k_f8_tile<F8_GATE_UP><<<dim3(2 * tiles, I / 64), 256, 0, st>>>(p);
    ops_launch_f8_quantize(w.n_pairs, I, ws + w.act, 0, I, ws + w.act_q, I, (float *)(ws + w.act_scales), I / 128, stream);
    p.n = H, p.k = I;
    p.a = ws + w.act_q, p.a_stride = I, p.a_scales = (const float *)(ws + w.act_scales), p.as_stride = I / 128;
    p.b = a->down, p.b_stride = I, p.b_rec = (int64_t)H * I;
    p.b_scales = a->down_scales, p.bs_stride = I / 128, p.bs_rec = (int64_t)(H / 128) * (I / 128);
    p.out = ws + w.dots, p.out_stride = H;
    k_f8_tile<F8_DOWN><<<dim3(2 * tiles, H / 64), 256, 0, st>>>(p);
    k_ops_combine<<<a->n_tokens, 256, 0, st>>>((const float *)(ws + w.dots), a->ids, a->weights, H, a->n_experts, a->top_k,
                                              n_routed, a->has_shared, (__nv_bfloat16 *)a->out, a->out_stride);
    *launches += 5;
    return (int)cudaGetLastError();
}

extern "C" int ops_f8_init(void) {
    cudaFuncAttributes f;
    int rc = 0;
#define RK(k) rc |= (int)cudaFuncGetAttributes(&f, (k))
    RK(k_f8_tile<F8_DENSE>); RK(k_f8_tile<F8_GATE_UP>); RK(k_f8_tile<F8_DOWN>); RK(k_ops_combine); RK(k_ops_bucket);
#undef RK
    rc |= (int)cudaFuncSetAttribute(k_ops_bucket, cudaFuncAttributeMaxDynamicSharedMemorySize, OPS_MAX_E * BK_WARPS * 4);
    return rc;
}
