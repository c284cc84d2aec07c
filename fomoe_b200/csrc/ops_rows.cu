/*
 * ops_rows.cu -- row-wise operators on device memory: routing of tokens to experts, the norms around a block, and the
 * block-scaled FP8 quantiser.
 */
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "launch.h"
#include "ops_launch.h"
#include "ops_quant.cuh"

#ifndef FULL
#define FULL 0xffffffffu
#endif

/* ------------------------------------------------------------------ routing: one warp per token
 * Lane l holds experts l, l + 32, ... .  Everything that decides an order is computed in 64 bits. */
#define RT_WARPS 4

__device__ __forceinline__ bool rt_better(double v, int i, double w, int j) { return v > w || (v == w && i < j); }

__device__ __forceinline__ void rt_warp_best(double &v, int &i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double ov = __shfl_xor_sync(FULL, v, o);
        const int oi = __shfl_xor_sync(FULL, i, o);
        if (rt_better(ov, oi, v, i)) {
            v = ov;
            i = oi;
        }
    }
}

template <int NPL>
__global__ void __launch_bounds__(32 * RT_WARPS) k_ops_route(ops_route_t A) {
    __shared__ double s_c[RT_WARPS][OPS_MAX_E];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int t = blockIdx.x * RT_WARPS + warp;
    if (t >= A.n_tokens) return;
    const int E = A.cfg.n_experts, K = A.cfg.top_k, G = A.cfg.n_group;
    const bool shut = A.valid && A.valid[t] == 0;
    const double NINF = -INFINITY;
    float x[NPL];
#pragma unroll
    for (int j = 0; j < NPL; j++) {
        const int e = j * 32 + lane;
        x[j] = -INFINITY;
        if (e < E && !shut) {
            const int64_t at = (int64_t)t * A.row_stride + e;
            const float v = A.logits_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(A.logits)[at])
                                          : reinterpret_cast<const float *>(A.logits)[at];
            if (v > -INFINITY) x[j] = fminf(v, FLT_MAX);
        }
    }
    /* p, and the order key o: the choice, or without a bias the logit itself */
    double p[NPL], o[NPL];
    if (A.cfg.score == FOMOE_B200_SOFTMAX) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < NPL; j++) mx = fmaxf(mx, x[j]);
        for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, s));
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NPL; j++) {
            p[j] = x[j] > -INFINITY ? exp((double)x[j] - (double)mx) : 0.0;
            sum += p[j];
        }
        for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(FULL, sum, s);
#pragma unroll
        for (int j = 0; j < NPL; j++) p[j] = sum > 0.0 ? p[j] / sum : 0.0;
    } else {
#pragma unroll
        for (int j = 0; j < NPL; j++) p[j] = x[j] > -INFINITY ? 1.0 / (1.0 + exp(-(double)x[j])) : 0.0;
    }
#pragma unroll
    for (int j = 0; j < NPL; j++) {
        const int e = j * 32 + lane;
        o[j] = NINF;
        if (x[j] > -INFINITY) {
            const double c = A.bias ? p[j] + (double)A.bias[e] : p[j];
            if (c > NINF) o[j] = A.bias ? c : (double)x[j];
            if (G > 1) s_c[warp][e] = c > NINF ? c : NINF;
        } else if (G > 1 && e < E) {
            s_c[warp][e] = NINF;
        }
    }
    if (G > 1) { /* lane g scores group g; then the topk_group best stay */
        __syncwarp();
        const int per = E / G;
        double g1 = NINF, g2 = NINF;
        if (lane < G)
            for (int i = 0; i < per; i++) {
                const double c = s_c[warp][lane * per + i];
                if (c > g1) {
                    g2 = g1;
                    g1 = c;
                } else if (c > g2) {
                    g2 = c;
                }
            }
        double gs = A.cfg.group_best == 2 && g2 > NINF ? g1 + g2 : g1;
        bool taken = lane >= G;
        uint32_t keep = 0;
        for (int r = 0; r < A.cfg.topk_group; r++) {
            double v = taken ? NINF : gs;
            int i = taken ? 64 : lane;
            rt_warp_best(v, i);
            if (lane == i) taken = true;
            if (i < 32) keep |= 1u << i;
        }
#pragma unroll
        for (int j = 0; j < NPL; j++) {
            const int e = j * 32 + lane;
            if (e < E && !((keep >> (e / per)) & 1u)) o[j] = NINF;
        }
    }
    double my_p = 0.0;
    int my_id = -1;
    for (int r = 0; r < K; r++) {
        double v = NINF, pv = 0.0;
        int i = OPS_MAX_E;
#pragma unroll
        for (int j = 0; j < NPL; j++)
            if (o[j] > v) {
                v = o[j];
                i = j * 32 + lane;
                pv = p[j];
            }
        const int mine = i;
        rt_warp_best(v, i);
        if (i == OPS_MAX_E) break; /* no open expert left */
        const double wp = __shfl_sync(FULL, pv, i & 31);
        if (mine == i) {
#pragma unroll
            for (int j = 0; j < NPL; j++)
                if (j == (i >> 5)) o[j] = NINF;
        }
        if (lane == r) {
            my_id = i;
            my_p = wp;
        }
    }
    if (A.cfg.renorm) {
        double s = my_p;
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
        my_p = my_p / (s + 1e-20);
    }
    if (lane < K) {
        A.ids[(int64_t)t * K + lane] = my_id;
        A.weights[(int64_t)t * K + lane] = (float)(my_p * (double)A.cfg.scale);
    }
}

extern "C" int ops_launch_route(const ops_route_t *a, void *stream) {
    const int grid = (a->n_tokens + RT_WARPS - 1) / RT_WARPS, E = a->cfg.n_experts;
    cudaStream_t st = (cudaStream_t)stream;
    if (E <= 32) k_ops_route<1><<<grid, 32 * RT_WARPS, 0, st>>>(*a);
    else if (E <= 64) k_ops_route<2><<<grid, 32 * RT_WARPS, 0, st>>>(*a);
    else if (E <= 128) k_ops_route<4><<<grid, 32 * RT_WARPS, 0, st>>>(*a);
    else if (E <= 256) k_ops_route<8><<<grid, 32 * RT_WARPS, 0, st>>>(*a);
    else k_ops_route<16><<<grid, 32 * RT_WARPS, 0, st>>>(*a);
    return (int)cudaGetLastError();
}

/* ------------------------------------------------------------------ norms around a block
 * G threads share a row; every thread holds IT runs of 8 neighbouring columns in registers, so the row is read once and
 * written once whatever the number of norms.  16 neighbouring threads hold one block of 128, whose amax is a shuffle
 * reduction.  VEC: all pointers and strides allow 16-byte accesses and n is a multiple of 8; otherwise the same code
 * goes element by element. */
#define NM_THREADS 256

template <bool VEC>
__device__ __forceinline__ void nm_load8(const void *p, int bf16, int64_t at, int left, float (&v)[8]) {
    if (VEC) {
        if (bf16) {
            const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(p) + at);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else {
            const float4 a = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + at);
            const float4 b = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + at + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            v[i] = i >= left ? 0.0f
                   : bf16    ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[at + i])
                             : reinterpret_cast<const float *>(p)[at + i];
    }
}

template <bool VEC>
__device__ __forceinline__ void nm_store8(void *p, int bf16, int64_t at, int left, const float (&v)[8]) {
    if (VEC) {
        if (bf16) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&b);
            }
            *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + at) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) {
                if (bf16) reinterpret_cast<__nv_bfloat16 *>(p)[at + i] = __float2bfloat16_rn(v[i]);
                else reinterpret_cast<float *>(p)[at + i] = v[i];
            }
    }
}

/* 8 values of one row as e4m3 at column c of q; the 16 threads of a 128-block call it together */
template <bool VEC>
__device__ __forceinline__ void nm_quant8(uint8_t *q, float *scales, int c, int n, const float (&v)[8]) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) amax = ops_amax(amax, v[i]);
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) amax = ops_amax(amax, __shfl_xor_sync(FULL, amax, s));
    const float sc = ops_f8_scale(amax);
    if (c < n) {
        if ((c & 127) == 0) scales[c >> 7] = sc;
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; h++)
            w[h] = ops_f8_pack4(__fdiv_rn(v[4 * h], sc), __fdiv_rn(v[4 * h + 1], sc), __fdiv_rn(v[4 * h + 2], sc),
                                __fdiv_rn(v[4 * h + 3], sc));
        if (VEC) {
            *reinterpret_cast<uint2 *>(q + c) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c + i < n) q[c + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
        }
    }
}

/* sum over the G threads of a row; s_red: one float per warp of the block */
template <int G>
__device__ __forceinline__ float nm_row_sum(float v, float *s_red) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(FULL, v, s);
    if (G == 32) return v;
    const int warp = threadIdx.x >> 5;
    __syncthreads(); /* the last sum's readers are done */
    if ((threadIdx.x & 31) == 0) s_red[warp] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int w = 0; w < NM_THREADS / 32; w++) t += s_red[w];
    return t;
}

template <bool VEC, int G, int IT>
__global__ void __launch_bounds__(NM_THREADS) k_ops_norm(fomoe_b200_norm_args_t A) {
    __shared__ float s_red[NM_THREADS / 32];
    const int gt = threadIdx.x % G;
    const int row = blockIdx.x * (NM_THREADS / G) + threadIdx.x / G;
    if (row >= A.n_tokens) return; /* whole warps (G = 32), or nobody (G = the block) */
    const int n = A.n;
    float x[IT][8], b[IT][8];
#pragma unroll
    for (int it = 0; it < IT; it++) {
        const int c = (it * G + gt) * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) x[it][i] = b[it][i] = 0.0f;
        if (c < n) {
            nm_load8<VEC>(A.x, A.x_type, (int64_t)row * A.x_stride + c, n - c, x[it]);
            if (A.block) nm_load8<VEC>(A.block, A.block_type, (int64_t)row * A.block_stride + c, n - c, b[it]);
        }
    }
    if (A.block) {
        float inv = 1.0f;
        if (A.post) {
            float ss = 0.0f;
#pragma unroll
            for (int it = 0; it < IT; it++)
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(b[it][i], b[it][i], ss);
            ss = nm_row_sum<G>(ss, s_red);
            inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)n) + A.eps));
        }
#pragma unroll
        for (int it = 0; it < IT; it++) {
            const int c = (it * G + gt) * 8;
            if (c < n) {
                float w[8], g[8];
                if (A.post) {
                    nm_load8<VEC>(A.post, 0, c, n - c, w);
#pragma unroll
                    for (int i = 0; i < 8; i++) b[it][i] *= inv * (w[i] + A.offset);
                }
                if (A.gate) {
                    if (A.gate_step) {
                        nm_load8<VEC>(A.gate, A.block_type, (int64_t)row * A.gate_stride + c, n - c, g);
                    } else {
                        const int64_t at = (int64_t)row * A.gate_stride;
                        const float s = A.block_type ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(A.gate)[at])
                                                     : reinterpret_cast<const float *>(A.gate)[at];
#pragma unroll
                        for (int i = 0; i < 8; i++) g[i] = s;
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) b[it][i] *= g[i];
                }
#pragma unroll
                for (int i = 0; i < 8; i++) x[it][i] = fmaf(A.scale, b[it][i], x[it][i]);
                if (!VEC)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (c + i >= n) x[it][i] = 0.0f; /* columns behind the row: a gate there may have been read as 0 * inf */
            }
        }
    }
    if (A.x_out) {
#pragma unroll
        for (int it = 0; it < IT; it++) {
            const int c = (it * G + gt) * 8;
            if (c < n) nm_store8<VEC>(A.x_out, A.x_type, (int64_t)row * A.x_out_stride + c, n - c, x[it]);
        }
    }
    if (!A.pre) return;
    float ss = 0.0f;
#pragma unroll
    for (int it = 0; it < IT; it++)
#pragma unroll
        for (int i = 0; i < 8; i++) ss = fmaf(x[it][i], x[it][i], ss);
    ss = nm_row_sum<G>(ss, s_red);
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)n) + A.eps));
#pragma unroll
    for (int it = 0; it < IT; it++) {
        const int c = (it * G + gt) * 8;
        float h[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (c < n) {
            float w[8];
            nm_load8<VEC>(A.pre, 0, c, n - c, w);
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = (VEC || c + i < n) ? x[it][i] * inv * (w[i] + A.offset) : 0.0f;
        }
        if (A.h_type == FOMOE_B200_F8)
            nm_quant8<VEC>(reinterpret_cast<uint8_t *>(A.h) + (int64_t)row * A.h_stride,
                           A.h_scales + (int64_t)row * A.h_scales_stride, c, n, h);
        else if (c < n)
            nm_store8<VEC>(A.h, A.h_type, (int64_t)row * A.h_stride + c, n - c, h);
    }
}

static bool nm_al(const void *p, int64_t stride, int bytes) {
    return p == nullptr || (((uintptr_t)p & 15) == 0 && (stride * bytes) % 16 == 0);
}

template <bool VEC>
static void nm_launch(const fomoe_b200_norm_args_t &a, cudaStream_t st) {
    const int rw = (a.n_tokens + 7) / 8, T = a.n_tokens, n = a.n;
    /* a warp to a row as long as the row fits its registers with enough rows to fill the card; else a block to a row */
    if (n <= 256) k_ops_norm<VEC, 32, 1><<<rw, NM_THREADS, 0, st>>>(a);
    else if (n <= 512) k_ops_norm<VEC, 32, 2><<<rw, NM_THREADS, 0, st>>>(a);
    else if (n <= 2048) k_ops_norm<VEC, 256, 1><<<T, NM_THREADS, 0, st>>>(a);
    else if (n <= 4096) k_ops_norm<VEC, 256, 2><<<T, NM_THREADS, 0, st>>>(a);
    else if (n <= 8192) k_ops_norm<VEC, 256, 4><<<T, NM_THREADS, 0, st>>>(a);
    else k_ops_norm<VEC, 256, 8><<<T, NM_THREADS, 0, st>>>(a);
}

extern "C" int ops_launch_norm(const fomoe_b200_norm_args_t *a, void *stream) {
    const int bs = a->block_type ? 2 : 4, hs = a->h_type == FOMOE_B200_F32 ? 4 : a->h_type == FOMOE_B200_BF16 ? 2 : 1;
    const int xs = a->x_type ? 2 : 4;
    const int many = a->n_tokens > 1; /* a single row's stride means nothing */
    const bool vec = a->n % 8 == 0 && nm_al(a->x, many * a->x_stride, xs) && nm_al(a->x_out, many * a->x_out_stride, xs) &&
                     nm_al(a->block, many * a->block_stride, bs) && nm_al(a->post, 0, 4) && nm_al(a->pre, 0, 4) &&
                     (!a->gate_step || nm_al(a->gate, many * a->gate_stride, bs)) &&
                     nm_al(a->pre ? a->h : nullptr, many * a->h_stride, hs);
    if (vec) nm_launch<true>(*a, (cudaStream_t)stream);
    else nm_launch<false>(*a, (cudaStream_t)stream);
    return (int)cudaGetLastError();
}

/* ------------------------------------------------------------------ rows to FP8: 16 threads per block of 128 */
template <bool VEC>
__global__ void __launch_bounds__(256) k_ops_quantize(int rows, int cols, int nb, const void *x, int bf16, int64_t x_stride,
                                                     uint8_t *q, int64_t q_stride, float *scales, int64_t s_stride) {
    const int64_t blk = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
    const int64_t row = blk / nb;
    const int b = (int)(blk - row * nb), c = b * 128 + (threadIdx.x & 15) * 8;
    const bool in = row < rows && c < cols;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (in) nm_load8<VEC>(x, bf16, row * x_stride + c, cols - c, v);
    nm_quant8<VEC>(q + row * q_stride, scales + row * s_stride, in ? c : cols, cols, v);
}

extern "C" int ops_launch_f8_quantize(int rows, int cols, const void *x, int x_bf16, int64_t x_stride, uint8_t *q,
                                      int64_t q_stride, float *scales, int64_t scales_stride, void *stream) {
    const int nb = (cols + 127) / 128;
    const int64_t grid = ((int64_t)rows * nb + 15) / 16;
    const bool vec = cols % 8 == 0 && nm_al(x, rows > 1 ? x_stride : 0, x_bf16 ? 2 : 4) && ((uintptr_t)q & 7) == 0 &&
                     (rows == 1 || q_stride % 8 == 0);
    if (vec)
        k_ops_quantize<true><<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(rows, cols, nb, x, x_bf16, x_stride, q, q_stride,
                                                                             scales, scales_stride);
    else
        k_ops_quantize<false><<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(rows, cols, nb, x, x_bf16, x_stride, q,
                                                                              q_stride, scales, scales_stride);
    return (int)cudaGetLastError();
}

/* every kernel of this file loaded on the current device, so that no call loads one inside a stream capture */
extern "C" int ops_rows_init(void) {
    cudaFuncAttributes f;
    int rc = 0;
#define RK(k) rc |= (int)cudaFuncGetAttributes(&f, (k))
    RK(k_ops_route<1>); RK(k_ops_route<2>); RK(k_ops_route<4>); RK(k_ops_route<8>); RK(k_ops_route<16>);
    RK((k_ops_norm<true, 32, 1>)); RK((k_ops_norm<true, 32, 2>)); RK((k_ops_norm<true, 256, 1>));
    RK((k_ops_norm<true, 256, 2>)); RK((k_ops_norm<true, 256, 4>)); RK((k_ops_norm<true, 256, 8>));
    RK((k_ops_norm<false, 32, 1>)); RK((k_ops_norm<false, 32, 2>)); RK((k_ops_norm<false, 256, 1>));
    RK((k_ops_norm<false, 256, 2>)); RK((k_ops_norm<false, 256, 4>)); RK((k_ops_norm<false, 256, 8>));
    RK(k_ops_quantize<true>); RK(k_ops_quantize<false>);
#undef RK
    return rc;
}
