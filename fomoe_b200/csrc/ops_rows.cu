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
#include "ops_launch.cuh"
#include "ops_launch.h"
#include "ops_quant.cuh"
#include "stream.cuh"

#ifndef FULL
#define FULL 0xffffffffu
#endif

/* ------------------------------------------------------------------ routing: one warp per token
 * Lane l holds experts l, l + 32, ... .  The order is the order of exact values.  Without a bias that is the logits' order,
 * which fp32 holds exactly; choices p + bias and scores of groups are computed in fp32, and where two that a decision hangs on
 * are closer than their errors allow (RT_NEAR) the warp repeats that decision in 64 bits.
 *
 * Error of a choice: p is an exp of an argument d rounded to |d| U (U = 2^-24; |d| e^-d < 0.4) by way of 2^x (3 U), a sum
 * and a quotient, 1e-6 of at most 1; the addition of the bias half a step of the choice, 6e-8 |c|.  Twice that for a
 * difference, four times for sums of two: RT_NEAR covers both with a factor of two to spare.
 *
 * The best K + 1 keys: each lane's best key first; the (K + 1)-th best of those is a bound that every one of the best K + 1
 * keys reaches, and few others do.  The keys that reach it are put side by side in shared memory, one to a lane, and each
 * counts how many are better.  (16,384 tokens x 384 experts, sigmoid + bias, top 8: 87 us in 64 bits with a round over all
 * keys for every slot, 18 us so: 810 instructions a token at 66 % of the issue slots, 28 of 64 warps on an SM; 256 experts in 8
 * groups 25 us, 1060 at 70 %)
 *
 * How often 64 bits are needed goes by the logits.  16,384 x 256 in 8 groups, logits of 1.5, 5, 8, 16 x normal: softmax 25, 27,
 * 32, 46 us, sigmoid 24, 32, 51, 50 us (groups' scores that saturate); with a bias of 0.1 x normal 25 to 27 us throughout. */
#define RT_WARPS 4
#define RT_BLOCKS 8 /* an SM: registers for so many (16,384 x 512, bias, top 16: 35 us, unbounded 36, for ten 44) */
#define RT_NEAR(a, b) (8e-6f + 1e-6f * (fabsf(a) + fabsf(b)))

/* floats as unsigned numbers in the same order; 0 stands for "closed" (below -inf) */
__device__ __forceinline__ uint32_t rt_key(float v) {
    const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v); /* (-0 is 0) */
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float rt_val(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

/* The best and the second best of every group, by the 32 / 2^ceil(log2 G) lanes that share a group; the group's first lane
 * (g << shift) has them.  c: the choices, -inf where closed. */
template <typename T>
__device__ __forceinline__ T rt_group_score(const T *c, int G, int per, int best, int shift) {
    const int lane = threadIdx.x & 31, g = lane >> shift, L = 1 << shift;
    const T NINF = -INFINITY;
    T a = NINF, b = NINF;
    if (g < G)
        for (int i = lane & (L - 1); i < per; i += L) {
            const T v = c[g * per + i];
            b = v > a ? a : v > b ? v : b;
            a = v > a ? v : a;
        }
    for (int s = L >> 1; s > 0; s >>= 1) {
        const T oa = __shfl_xor_sync(FULL, a, s), ob = __shfl_xor_sync(FULL, b, s);
        b = a > oa ? (oa > b ? oa : b) : (a > ob ? a : ob);
        a = a > oa ? a : oa;
    }
    return best == 2 && b > NINF ? a + b : a;
}

/* The groups that stay: those with fewer than topk better ones (lower group first among equals), bit g << shift for group g.
 * Group g's score is in the lane of that number. */
template <typename T>
__device__ __forceinline__ uint32_t rt_groups_stay(T gs, int G, int topk, int shift) {
    const int lane = threadIdx.x & 31, g = lane >> shift;
    int rank = 0;
    for (int h = 0; h < G; h++) {
        const T o = __shfl_sync(FULL, gs, h << shift);
        rank += o > gs || (o == gs && h < g);
    }
    return __ballot_sync(FULL, (lane & ((1 << shift) - 1)) == 0 && g < G && rank < topk);
}
/* expert e's bit of it; mul: 2^20 / per, rounded up (exact for e < 512) */
#define RT_STAYS(stay, e, mul, shift) (((stay) >> ((((uint32_t)(e) * (mul)) >> 20) << (shift))) & 1u)

__device__ __forceinline__ float rt_logit(const ops_route_t &A, int t, int e) {
    const int64_t at = (int64_t)t * A.row_stride + e;
    return A.logits_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(A.logits)[at])
                         : reinterpret_cast<const float *>(A.logits)[at];
}

/* The choices in 64 bits, to c[0 .. E) (-inf where closed).  Rare: written for size. */
__device__ __noinline__ void rt_exact_choices(const ops_route_t &A, int t, float mx, double *c) {
    const int lane = threadIdx.x & 31, E = A.cfg.n_experts;
    double sum = 0.0;
    for (int e = lane; e < E; e += 32) {
        const float v = rt_logit(A, t, e);
        const bool open = v > -INFINITY;
        const double x = fmin((double)v, (double)FLT_MAX);
        double p = 0.0;
        if (open) p = A.cfg.score == FOMOE_B200_SOFTMAX ? exp(x - (double)mx) : 1.0 / (1.0 + exp(-x));
        sum += p;
        c[e] = open ? p : -INFINITY;
    }
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(FULL, sum, s);
    for (int e = lane; e < E; e += 32) {
        double v = c[e];
        if (v > -INFINITY) {
            if (A.cfg.score == FOMOE_B200_SOFTMAX) v /= sum;
            if (A.bias) v += (double)A.bias[e];
            c[e] = v > -INFINITY ? v : -INFINITY;
        }
    }
    __syncwarp();
}

/* The choice of expert e in 64 bits (the whole warp calls it: softmax needs the sum over all experts). */
__device__ __noinline__ double rt_exact_choice(const ops_route_t &A, int t, float mx, int e) {
    const int lane = threadIdx.x & 31, E = A.cfg.n_experts;
    const bool softmax = A.cfg.score == FOMOE_B200_SOFTMAX;
    double sum = 0.0;
    if (softmax) {
        for (int i = lane; i < E; i += 32) {
            const float v = rt_logit(A, t, i);
            if (v > -INFINITY) sum += exp(fmin((double)v, (double)FLT_MAX) - (double)mx);
        }
        for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(FULL, sum, s);
    }
    if (e < 0) return -INFINITY;
    const double x = fmin((double)rt_logit(A, t, e), (double)FLT_MAX);
    return (softmax ? exp(x - (double)mx) / sum : 1.0 / (1.0 + exp(-x))) + (double)A.bias[e];
}

/* the top_k of c by rounds over all of it; closed: what is never chosen; lane r gets the id of slot r */
template <typename T>
__device__ __noinline__ int rt_top(T *c, T closed, int E, int K, uint32_t keep, uint32_t mul, int shift) {
    const int lane = threadIdx.x & 31;
    int my_id = -1;
    for (int r = 0; r < K; r++) {
        T v = closed;
        int i = OPS_MAX_E;
        for (int e = lane; e < E; e += 32)
            if (c[e] > v && RT_STAYS(keep, e, mul, shift)) {
                v = c[e];
                i = e;
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const T ov = __shfl_xor_sync(FULL, v, o);
            const int oi = __shfl_xor_sync(FULL, i, o);
            if (ov > v || (ov == v && oi < i)) {
                v = ov;
                i = oi;
            }
        }
        if (i == OPS_MAX_E) break;
        if (lane == r) my_id = i;
        __syncwarp();
        if (lane == 0) c[i] = closed;
        __syncwarp();
    }
    return my_id;
}

__device__ __forceinline__ float rt_sigmoid(float x) { /* (x = -inf: 0) */
    const float e = __expf(-fabsf(x)), q = __fdividef(1.0f, 1.0f + e);
    return x >= 0.0f ? q : e * q;
}

/* the same for a choice, whose absolute error is what counts: 1 / (1 + 2^(-x log2 e)), and 0 where that power overflows */
__device__ __forceinline__ float rt_sigmoid_choice(float x) {
    float e, p;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(1.0f + e));
    return p;
}

/* NPL: experts of a lane; LOW: as many as every lane has for certain (the size before in RT_SIZES) */
template <int NPL, int LOW>
__global__ void __launch_bounds__(32 * RT_WARPS, RT_BLOCKS) k_ops_route(const __grid_constant__ ops_route_t A) {
    __shared__ double s_c[RT_WARPS][OPS_MAX_E];
    __shared__ uint2 s_best[RT_WARPS][32]; /* candidates: choice, expert */
    __shared__ __align__(16) uint32_t s_key[RT_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int t = blockIdx.x * RT_WARPS + warp;
    if (t >= A.n_tokens) return;
    const int E = A.cfg.n_experts, K = A.cfg.top_k, G = A.cfg.n_group;
    const bool softmax = A.cfg.score == FOMOE_B200_SOFTMAX;
    if (A.valid && A.valid[t] == 0) { /* padding: every expert is closed */
        if (lane < K) {
            A.ids[(int64_t)t * K + lane] = -1;
            A.weights[(int64_t)t * K + lane] = 0.0f;
        }
        return;
    }
    float x[NPL];
#define RT_AT(j) ((j) < LOW ? (j) * 32 + lane : min((j) * 32 + lane, E - 1)) /* an expert that is there */
    if (A.logits_bf16) { /* (all loads first) */
        const uint16_t *p = reinterpret_cast<const uint16_t *>(A.logits) + (int64_t)t * A.row_stride;
#pragma unroll
        for (int j = 0; j < NPL; j++) x[j] = __uint_as_float((uint32_t)__ldg(p + RT_AT(j)) << 16);
    } else {
        const float *p = reinterpret_cast<const float *>(A.logits) + (int64_t)t * A.row_stride;
#pragma unroll
        for (int j = 0; j < NPL; j++) x[j] = __ldg(p + RT_AT(j));
    }
    /* closed experts: -inf.  (fmaxf takes a NaN to -inf, fminf +inf to FLT_MAX) */
    float mx = -INFINITY, inv = 1.0f;
#pragma unroll
    for (int j = 0; j < NPL; j++) {
        x[j] = fminf(fmaxf(x[j], -INFINITY), FLT_MAX);
        if (j >= LOW && j * 32 + lane >= E) x[j] = -INFINITY;
    }
    if (softmax) {
#pragma unroll
        for (int j = 0; j < NPL; j++) mx = fmaxf(mx, x[j]);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, s));
        float sum = 0.0f;
        const float m0 = mx > -INFINITY ? mx : 0.0f;
#pragma unroll
        for (int j = 0; j < NPL; j++) sum += __expf(x[j] - m0);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(FULL, sum, s);
        inv = sum > 0.0f ? __fdiv_rn(1.0f, sum) : 0.0f;
    }
    /* what decides the order: the choice, or without a bias the logit itself; -inf where closed */
    float v[NPL];
    if (A.bias || G > 1) {
        if (softmax) {
            const float m0 = mx > -INFINITY ? mx : 0.0f;
#pragma unroll
            for (int j = 0; j < NPL; j++) v[j] = __expf(x[j] - m0) * inv;
        } else {
#pragma unroll
            for (int j = 0; j < NPL; j++) v[j] = rt_sigmoid_choice(x[j]);
        }
        if (A.bias) {
#pragma unroll
            for (int j = 0; j < NPL; j++) v[j] += __ldg(A.bias + RT_AT(j)); /* (NaN: no comparison below finds it) */
        }
#pragma unroll
        for (int j = 0; j < NPL; j++) v[j] = x[j] > -INFINITY ? v[j] : -INFINITY;
        if (G > 1) {
#pragma unroll
            for (int j = 0; j < NPL; j++)
                if (j < LOW || j * 32 + lane < E) reinterpret_cast<float *>(s_c[warp])[j * 32 + lane] = v[j];
        }
        if (!A.bias) {
#pragma unroll
            for (int j = 0; j < NPL; j++) v[j] = x[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < NPL; j++) v[j] = x[j];
    }
    uint32_t keep = 0xffffffffu, mul = 0;
    int shift = 0;
    if (G > 1) {
        const int per = E / G;
        __syncwarp();
        mul = ((1u << 20) + per - 1) / per;
        shift = 5 - (32 - __clz(G - 1)); /* lanes of a group, as a power of two */
        const float gs = rt_group_score(reinterpret_cast<const float *>(s_c[warp]), G, per, A.cfg.group_best, shift);
        keep = rt_groups_stay(gs, G, A.cfg.topk_group, shift);
        /* does the cut pass between two scores that are too close?  The lowest that stays and the highest that does not are
         * the closest two; the largest of all is taken for the size that their error goes by. */
        const bool head = (lane & ((1 << shift) - 1)) == 0 && (lane >> shift) < G, in = (keep >> lane) & 1u;
        const uint32_t out = __reduce_max_sync(FULL, head && !in ? rt_key(gs) : 0u), low = __reduce_min_sync(FULL, head && in ? rt_key(gs) : 0xffffffffu);
        if (out > rt_key(-INFINITY)) {
            const float a = rt_val(low), b = rt_val(out);
            const float size = __uint_as_float(__reduce_max_sync(FULL, head && gs > -INFINITY ? __float_as_uint(fabsf(gs)) : 0u));
            if (!(a - b > 2.0f * RT_NEAR(size, size))) {
                rt_exact_choices(A, t, mx, s_c[warp]);
                keep = rt_groups_stay(rt_group_score(s_c[warp], G, per, A.cfg.group_best, shift), G, A.cfg.topk_group, shift);
            }
        }
#pragma unroll
        for (int j = 0; j < NPL; j++)
            if (!RT_STAYS(keep, j * 32 + lane, mul, shift)) v[j] = -INFINITY; /* (behind the last expert: closed already) */
    }
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < NPL; j++) most = fmaxf(most, v[j]);
    uint32_t best = most > -INFINITY ? rt_key(most) : 0u;
    uint32_t w = 0;
#pragma unroll 3
    for (int r = 0; r <= K; r++) { /* (equal ones of several lanes go together: the bound is only lower for it) */
        w = __reduce_max_sync(FULL, best);
        best = best == w ? 0u : best;
    }
    float bound = w ? rt_val(w) : -FLT_MAX; /* (all that is open; a value below it would be an infinite bias) */
    if (A.bias) { /* and those that may be as good for all fp32 can say */
        const float low = bound - RT_NEAR(bound, bound);
        bound = low >= -FLT_MAX ? low : -FLT_MAX; /* (infinite choices: all that is open) */
    }
    int n = 0;
#pragma unroll
    for (int j = 0; j < NPL; j++) {
        const bool in = v[j] >= bound;
        const uint32_t m = __ballot_sync(FULL, in);
        if (m) { /* (most have none) */
            const int at = n + __popc(m & ((1u << lane) - 1u));
            if (in && at < 32) s_best[warp][at] = make_uint2(__float_as_uint(v[j]), (uint32_t)(j * 32 + lane));
            n += __popc(m);
        }
    }
    __syncwarp();
    int slot = lane, id = -1; /* this lane writes slot `slot`, if there is one */
    float lx = 0.0f;          /* the logit of `id` */
    bool exact = false;
    if (n <= 32) {
        uint32_t own = 0;
        if (lane < n) {
            const uint2 c = s_best[warp][lane];
            own = rt_key(__uint_as_float(c.x));
            id = (int)c.y;
            lx = fminf(rt_logit(A, t, id), FLT_MAX); /* (holding all of x this far costs occupancy) */
        }
        s_key[warp][lane] = own;
        __syncwarp();
        int rank = 0; /* (candidates lie in the order of their ids: of equal ones the earlier is the better) */
        for (int i = 0; i < n; i += 4) {
            const uint4 o = *reinterpret_cast<const uint4 *>(&s_key[warp][i]);
            rank += (o.x + (i < lane) > own) + (o.y + (i + 1 < lane) > own) + (o.z + (i + 2 < lane) > own) + (o.w + (i + 3 < lane) > own);
        }
        slot = lane < n ? rank : lane;
        if (A.bias) { /* neighbours among the best K + 1 that are too close? */
            __syncwarp();
            if (lane < n) s_key[warp][rank] = own;
            __syncwarp();
            bool near = false;
            if (lane < K && lane + 1 < n) {
                const float a = rt_val(s_key[warp][lane]), b = rt_val(s_key[warp][lane + 1]);
                near = !(a - b > RT_NEAR(a, b));
            }
            if (__any_sync(FULL, near)) { /* rank the candidates again, by their exact choices */
                const double c = rt_exact_choice(A, t, mx, id);
                rank = 0;
                for (int i = 0; i < n; i++) {
                    const double oc = __shfl_sync(FULL, c, i);
                    const int oi = __shfl_sync(FULL, id, i);
                    rank += oc > c || (oc == c && oi < id);
                }
                slot = lane < n ? rank : lane;
            }
        }
    } else if (!A.bias) { /* more equal keys than lanes */
        uint32_t *c = reinterpret_cast<uint32_t *>(s_c[warp]);
#pragma unroll
        for (int j = 0; j < NPL; j++)
            if (j * 32 + lane < E) c[j * 32 + lane] = v[j] > -INFINITY ? rt_key(v[j]) : 0u;
        __syncwarp();
        id = rt_top<uint32_t>(c, 0u, E, K, keep, mul, shift);
    } else {
        exact = true;
    }
    if (exact) {
        rt_exact_choices(A, t, mx, s_c[warp]);
        slot = lane;
        id = rt_top<double>(s_c[warp], (double)-INFINITY, E, K, keep, mul, shift);
    }
    if (n > 32 && id >= 0) lx = fminf(rt_logit(A, t, id), FLT_MAX);
    float p = 0.0f;
    if (slot < K && id >= 0) p = softmax ? __expf(lx - mx) * inv : rt_sigmoid(lx);
    if (A.cfg.renorm) {
        float s = p;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
        p = __fdiv_rn(p, s + 1e-20f);
    }
    if (slot < K) {
        A.ids[(int64_t)t * K + slot] = id;
        A.weights[(int64_t)t * K + slot] = p * A.cfg.scale;
    }
}

#define RT_SIZES(X) X(1, 0) X(2, 1) X(4, 2) X(6, 4) X(8, 6) X(12, 8) X(16, 12) /* experts of a lane, at most and at least */

extern "C" int ops_launch_route(const ops_route_t *a, void *stream) {
    const int grid = (a->n_tokens + RT_WARPS - 1) / RT_WARPS, E = a->cfg.n_experts;
#define RT_GO(N, LOW) \
    if (E <= 32 * N) return ops_launch(k_ops_route<N, LOW>, grid, 32 * RT_WARPS, 0, (cudaStream_t)stream, *a);
    RT_SIZES(RT_GO)
#undef RT_GO
    return (int)cudaErrorInvalidValue;
}

/* ------------------------------------------------------------------ norms around a block
 * r = block / rms(block) (w_post + offset) g;  x' = x + scale r;  h = x' / rms(x') (w_pre + offset)
 * G threads share a row; every thread holds IT runs of 8 neighbouring columns in registers, so the row is read once and
 * written once whatever the number of norms.  The threads of a block of 128 are neighbours: its amax is one reduction.
 * VEC: all pointers and strides allow 16-byte accesses and n is a multiple of 8; otherwise neighbouring lanes take
 * neighbouring columns and the values change hands in shared memory, so that each thread has the same ones.
 *
 * What bounds it (8192 x 4096, fp32 residual, bf16 block, FP8 out): 69 us, 5.3 TB/s of 6.5.  The chain of a row -- load, two
 * sums over the block, two square roots, the scale of a block -- is long, so it takes many rows at once on an SM: blocks of 256
 * threads whose registers let five share one, and the next rows asked into L2.  Rings of rows in shared memory under persistent
 * blocks (108 us and more: they take the L1 that holds the weights) and 128 threads with four runs each (85 us) were slower;
 * values in pairs (fma.rn.f32x2) saved 2 us, one scale for 16 values a thread the quantiser a quarter of its time.
 * Rows without alignment (8192 x 4095: 160 us) take twice the instructions, 91 M for 43 M, from three blocks an SM (72
 * registers for 48): narrow accesses and the exchange in shared memory. */
#define NM_THREADS(G) ((G) == 32 ? 256 : (G))
#define NM_AHEAD 148 /* rows: what a later block reads is asked into L2 (8192 x 4096: 74 us, without 82, 296 rows ahead 74) */
#define NM_BLOCKS 5  /* of 256 threads, an SM (8192 x 4096: 68 us, with 4 74, with 6 and spills 93) */
#define NM_FEW 1184  /* rows: eight an SM */

/* Values go in pairs: one instruction (fma.rn.f32x2 and its like) rounds two of them as two would. */
#define NM_PAIR(op, d, a, b)                                                                                     \
    asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\n" op ".rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}" \
        : "=f"((d).x), "=f"((d).y)                                                                               \
        : "f"((a).x), "f"((a).y), "f"((b).x), "f"((b).y))

__device__ __forceinline__ float2 nm_mul(float2 a, float2 b) {
    float2 d;
    NM_PAIR("mul", d, a, b);
    return d;
}
__device__ __forceinline__ float2 nm_add(float2 a, float2 b) {
    float2 d;
    NM_PAIR("add", d, a, b);
    return d;
}
__device__ __forceinline__ float2 nm_fma(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 nm_both(float v) { return make_float2(v, v); }

/* Where a thread's runs of 8 columns lie.  One run: 16 threads share a block of 128; two, 64 columns apart: 8 threads, so that
 * the block's scale is made once for 16 values.  A row's sums come in the same order whether its accesses are wide or not. */
template <int IT>
__device__ __forceinline__ int nm_col(int thread, int it) {
    constexpr int S = IT == 2 ? 8 : 16; /* threads of a block */
    return thread / S * 128 + it * 64 + thread % S * 8;
}

/* 8 columns from `at`, STEP apart; VEC: neighbours, 16-byte accesses */
template <bool VEC, int STEP = 1>
__device__ __forceinline__ void nm_load8(const void *p, int bf16, int64_t at, int left, float2 (&v)[4]) {
    if (VEC) {
        if (bf16) {
            const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(p) + at);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        } else {
            const float4 a = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + at);
            const float4 b = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + at + 4);
            v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w), v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
        }
    } else {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            f[i] = STEP * i >= left ? 0.0f
                   : bf16              ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[at + STEP * i])
                                       : reinterpret_cast<const float *>(p)[at + STEP * i];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = make_float2(f[2 * i], f[2 * i + 1]);
    }
}

__device__ __forceinline__ void nm_store8(void *p, int bf16, int64_t at, const float2 (&v)[4]) {
    if (bf16) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 b = __float22bfloat162_rn(v[i]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + at) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + at + 4) = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
}

/* A warp's run `it` by narrow accesses: neighbouring lanes take neighbouring columns, and the 256 values change hands in
 * shared memory (s_w, the warp's).  nm_place: the column of value i of the warp's. */
template <int IT>
__device__ __forceinline__ int nm_place(int thread, int it, int i) {
    return thread / 32 * (IT * 256) + (IT == 2 ? i / 64 * 128 + it * 64 + i % 64 : i);
}

/* a thread's run `it` of the row of n values from p[at] on; !VEC: the whole warp calls it, and columns behind the row are 0 */
template <bool VEC, int IT>
__device__ __forceinline__ void nm_get(const void *p, int bf16, int64_t at, int n, int thread, int it, float2 (&v)[4], float *s_w) {
    if (VEC) {
        nm_load8<true>(p, bf16, at + nm_col<IT>(thread, it), 8, v);
    } else {
        const int lane = thread & 31;
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = nm_place<IT>(thread, it, 32 * i + lane);
            f[i] = c >= n ? 0.0f : bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[at + c]) : reinterpret_cast<const float *>(p)[at + c];
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; i++) s_w[32 * i + lane] = f[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = *reinterpret_cast<const float2 *>(s_w + 8 * lane + 2 * i);
    }
}

template <bool VEC, int IT>
__device__ __forceinline__ void nm_put(void *p, int bf16, int64_t at, int n, int thread, int it, const float2 (&v)[4], float *s_w) {
    if (VEC) {
        nm_store8(p, bf16, at + nm_col<IT>(thread, it), v);
    } else {
        const int lane = thread & 31;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<float2 *>(s_w + 8 * lane + 2 * i) = v[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = nm_place<IT>(thread, it, 32 * i + lane);
            if (c >= n) continue;
            if (bf16) reinterpret_cast<__nv_bfloat16 *>(p)[at + c] = __float2bfloat16_rn(s_w[32 * i + lane]);
            else reinterpret_cast<float *>(p)[at + c] = s_w[32 * i + lane];
        }
    }
}

/* a thread's runs of one row as e4m3; the 16 / IT threads of a block of 128 call it together */
template <bool VEC, int IT, int STEP = 1>
__device__ __forceinline__ void nm_quant(uint8_t *q, float *scales, int thread, int c0, int n, const float2 (&v)[IT][4], uint32_t *s_w = nullptr) {
    float amax = 0.0f;
#pragma unroll
    for (int it = 0; it < IT; it++)
#pragma unroll
        for (int i = 0; i < 4; i++) amax = ops_amax(ops_amax(amax, v[it][i].x), v[it][i].y);
    /* numbers without a sign are ordered as their bits are, with NaN above infinity */
    const unsigned block = IT == 2 ? 0xffu << (threadIdx.x & 24) : 0xffffu << (threadIdx.x & 16);
    amax = __uint_as_float(__reduce_max_sync(block, __float_as_uint(amax)));
    const float sc = ops_f8_scale(amax), inv = __frcp_rn(sc);
    if ((c0 & 127) == 0 && c0 < n) scales[c0 >> 7] = sc;
#pragma unroll
    for (int it = 0; it < IT; it++) {
        const int c = c0 + 64 * it;
        if ((VEC || STEP > 1) && c >= n) continue;
        float2 r[4];
#pragma unroll
        for (int i = 0; i < 4; i++) { /* (ops_f8_quot) */
            const float2 t = nm_mul(v[it][i], nm_both(inv));
            r[i] = nm_fma(nm_fma(t, nm_both(-sc), v[it][i]), nm_both(inv), t);
        }
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; h++) w[h] = ops_f8_pack4(r[2 * h].x, r[2 * h].y, r[2 * h + 1].x, r[2 * h + 1].y);
        if (VEC) {
            *reinterpret_cast<uint2 *>(q + c) = make_uint2(w[0], w[1]);
        } else if (STEP > 1) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c + STEP * i < n) q[c + STEP * i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
        } else { /* (as nm_put) */
            const int lane = threadIdx.x & 31;
            __syncwarp();
            s_w[2 * lane] = w[0], s_w[2 * lane + 1] = w[1];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int to = nm_place<IT>(thread, it, 32 * i + lane);
                if (to < n) q[to] = reinterpret_cast<const uint8_t *>(s_w)[32 * i + lane];
            }
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
    for (int w = 0; w < G / 32; w++) t += s_red[w];
    return t;
}

/* 1 / rms of the row */
template <int G, int IT>
__device__ __forceinline__ float nm_inv(const float2 (&v)[IT][4], int n, float eps, float *s_red) {
    float2 ss = nm_both(0.0f);
#pragma unroll
    for (int it = 0; it < IT; it++)
#pragma unroll
        for (int i = 0; i < 4; i++) ss = nm_fma(v[it][i], v[it][i], ss);
    return __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(nm_row_sum<G>(ss.x + ss.y, s_red), (float)n) + eps));
}

template <bool VEC, int G, int IT>
__global__ void __launch_bounds__(NM_THREADS(G), VEC && G == 256 ? NM_BLOCKS : 1) k_ops_norm(fomoe_b200_norm_args_t A) {
    __shared__ float s_red[NM_THREADS(G) / 32];
    __shared__ __align__(16) float s_turn[VEC ? 1 : NM_THREADS(G) / 32][256];
    float *s_w = s_turn[VEC ? 0 : threadIdx.x / 32];
    const int gt = threadIdx.x % G;
    const int row = blockIdx.x * (NM_THREADS(G) / G) + threadIdx.x / G;
    if (row >= A.n_tokens) return; /* whole warps (G = 32), or nobody (G = the block) */
    const int n = A.n;
    if (VEC && G > 32 && threadIdx.x == 0 && row + NM_AHEAD < A.n_tokens) { /* a row that a later block will read, into L2 */
        const int64_t r = row + NM_AHEAD;
        const int xb = A.x_type ? 2 : 4, bb = A.block_type ? 2 : 4;
        fb_prefetch_l2(reinterpret_cast<const uint8_t *>(A.x) + r * A.x_stride * xb, (uint32_t)(n * xb));
        if (A.block) fb_prefetch_l2(reinterpret_cast<const uint8_t *>(A.block) + r * A.block_stride * bb, (uint32_t)(n * bb));
    }
    float2 x[IT][4], b[IT][4];
#pragma unroll
    for (int it = 0; it < IT; it++) {
        const int c = nm_col<IT>(gt, it);
#pragma unroll
        for (int i = 0; i < 4; i++) x[it][i] = b[it][i] = nm_both(0.0f);
        if (!VEC || c < n) {
            nm_get<VEC, IT>(A.x, A.x_type, (int64_t)row * A.x_stride, n, gt, it, x[it], s_w);
            if (A.block) nm_get<VEC, IT>(A.block, A.block_type, (int64_t)row * A.block_stride, n, gt, it, b[it], s_w);
        }
    }
    if (A.block) {
        float inv = 1.0f;
        if (A.post) inv = nm_inv<G, IT>(b, n, A.eps, s_red);
#pragma unroll
        for (int it = 0; it < IT; it++) {
            const int c = nm_col<IT>(gt, it);
            if (!VEC || c < n) {
                float2 w[4];
                if (A.post) {
                    nm_get<VEC, IT>(A.post, 0, 0, n, gt, it, w, s_w);
#pragma unroll
                    for (int i = 0; i < 4; i++) b[it][i] = nm_mul(b[it][i], nm_mul(nm_both(inv), nm_add(w[i], nm_both(A.offset))));
                }
                if (A.gate) {
                    if (A.gate_step) {
                        nm_get<VEC, IT>(A.gate, A.block_type, (int64_t)row * A.gate_stride, n, gt, it, w, s_w);
                    } else {
                        const int64_t at = (int64_t)row * A.gate_stride;
                        const float s = A.block_type ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(A.gate)[at])
                                                     : reinterpret_cast<const float *>(A.gate)[at];
#pragma unroll
                        for (int i = 0; i < 4; i++) w[i] = nm_both(s);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) b[it][i] = nm_mul(b[it][i], w[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) x[it][i] = nm_fma(nm_both(A.scale), b[it][i], x[it][i]);
                if (!VEC)
#pragma unroll
                    for (int i = 0; i < 4; i++) { /* columns behind the row: a gate there may have been read as 0 * inf */
                        if (c + 2 * i >= n) x[it][i].x = 0.0f;
                        if (c + 2 * i + 1 >= n) x[it][i].y = 0.0f;
                    }
            }
        }
    }
    if (A.x_out) {
#pragma unroll
        for (int it = 0; it < IT; it++) {
            const int c = nm_col<IT>(gt, it);
            if (!VEC || c < n) nm_put<VEC, IT>(A.x_out, A.x_type, (int64_t)row * A.x_out_stride, n, gt, it, x[it], s_w);
        }
    }
    if (!A.pre) return;
    const float inv = nm_inv<G, IT>(x, n, A.eps, s_red);
#pragma unroll
    for (int it = 0; it < IT; it++) { /* (x becomes h) */
        const int c = nm_col<IT>(gt, it);
        if (VEC && c >= n) continue; /* (x is 0 there) */
        float2 w[4];
        nm_get<VEC, IT>(A.pre, 0, 0, n, gt, it, w, s_w);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[it][i] = nm_mul(nm_mul(x[it][i], nm_both(inv)), nm_add(w[i], nm_both(A.offset)));
            if (!VEC) {
                if (c + 2 * i >= n) x[it][i].x = 0.0f;
                if (c + 2 * i + 1 >= n) x[it][i].y = 0.0f;
            }
        }
        if (A.h_type != FOMOE_B200_F8) nm_put<VEC, IT>(A.h, A.h_type, (int64_t)row * A.h_stride, n, gt, it, x[it], s_w);
    }
    if (A.h_type == FOMOE_B200_F8)
        nm_quant<VEC, IT>(reinterpret_cast<uint8_t *>(A.h) + (int64_t)row * A.h_stride, A.h_scales + (int64_t)row * A.h_scales_stride,
                          gt, nm_col<IT>(gt, 0), n, x, reinterpret_cast<uint32_t *>(s_w));
}

static bool nm_al(const void *p, int64_t stride, int bytes) {
    return p == nullptr || (((uintptr_t)p & 15) == 0 && (stride * bytes) % 16 == 0);
}

template <bool VEC>
static int nm_launch(const fomoe_b200_norm_args_t &a, cudaStream_t st) {
    const int rw = (a.n_tokens + 7) / 8, T = a.n_tokens, n = a.n;
    /* one run of columns a thread while the rows do not fill the card (1 x 4096: 3.2 us, with two runs 3.9), two and more
     * blocks to an SM when they do (8192 x 4096: 76 us, with one run 80) */
    const bool few = T <= NM_FEW;
    return n <= 256          ? ops_launch(k_ops_norm<VEC, 32, 1>, rw, 256, 0, st, a)
           : n <= 512         ? ops_launch(k_ops_norm<VEC, 32, 2>, rw, 256, 0, st, a)
           : n <= 1024        ? ops_launch(k_ops_norm<VEC, 128, 1>, T, 128, 0, st, a)
           : n <= 2048        ? ops_launch(k_ops_norm<VEC, 256, 1>, T, 256, 0, st, a)
           : n <= 4096 && few ? ops_launch(k_ops_norm<VEC, 512, 1>, T, 512, 0, st, a)
           : n <= 4096        ? ops_launch(k_ops_norm<VEC, 256, 2>, T, 256, 0, st, a)
           : n <= 8192 && few ? ops_launch(k_ops_norm<VEC, 1024, 1>, T, 1024, 0, st, a)
           : n <= 8192        ? ops_launch(k_ops_norm<VEC, 512, 2>, T, 512, 0, st, a)
                              : ops_launch(k_ops_norm<VEC, 1024, 2>, T, 1024, 0, st, a);
}

extern "C" int ops_launch_norm(const fomoe_b200_norm_args_t *a, void *stream) {
    const int bs = a->block_type ? 2 : 4, hs = a->h_type == FOMOE_B200_F32 ? 4 : a->h_type == FOMOE_B200_BF16 ? 2 : 1;
    const int xs = a->x_type ? 2 : 4;
    const int many = a->n_tokens > 1; /* a single row's stride means nothing */
    const bool vec = a->n % 8 == 0 && nm_al(a->x, many * a->x_stride, xs) && nm_al(a->x_out, many * a->x_out_stride, xs) &&
                     nm_al(a->block, many * a->block_stride, bs) && nm_al(a->post, 0, 4) && nm_al(a->pre, 0, 4) &&
                     (!a->gate_step || nm_al(a->gate, many * a->gate_stride, bs)) &&
                     nm_al(a->pre ? a->h : nullptr, many * a->h_stride, hs);
    return vec ? nm_launch<true>(*a, (cudaStream_t)stream) : nm_launch<false>(*a, (cudaStream_t)stream);
}

/* ------------------------------------------------------------------ rows to FP8: 8 threads per block of 128
 * (8192 x 4096 bf16: 18.2 us, 5.5 TB/s, 75 % of the issue slots; with 16 threads a block 25 us, bound by what every thread does
 * once: the block's place, its scale, the scale's reciprocal.) */
template <bool VEC>
__global__ void __launch_bounds__(256) k_ops_quantize(int rows, int cols, int nb, uint64_t per_nb, const void *x, int bf16, int64_t x_stride,
                                                     uint8_t *q, int64_t q_stride, float *scales, int64_t s_stride) {
    const uint32_t blk = blockIdx.x * 32 + (threadIdx.x >> 3); /* (the host keeps rows * nb below 2^30) */
    const uint32_t r = nb == 1 ? blk : (uint32_t)__umul64hi(blk, per_nb); /* blk / nb: per_nb is just above 2^64 / nb */
    const int64_t row = r < (uint32_t)rows ? r : 0;
    constexpr int STEP = VEC ? 1 : 8; /* narrow accesses: neighbouring threads have neighbouring columns (4096 x 2063: 15 us, 21 without) */
    const int c0 = r < (uint32_t)rows ? (int)(blk - r * nb) * 128 + (threadIdx.x & 7) * (VEC ? 8 : 1) : cols;
    float2 v[2][4] = {};
#pragma unroll
    for (int it = 0; it < 2; it++)
        if (c0 + 64 * it < cols) nm_load8<VEC, STEP>(x, bf16, row * x_stride + c0 + 64 * it, cols - c0 - 64 * it, v[it]);
    nm_quant<VEC, 2, STEP>(q + row * q_stride, scales + row * s_stride, 0, c0, cols, v);
}

extern "C" int ops_launch_f8_quantize(int rows, int cols, const void *x, int x_bf16, int64_t x_stride, uint8_t *q,
                                      int64_t q_stride, float *scales, int64_t scales_stride, void *stream) {
    const int nb = (cols + 127) / 128;
    const uint64_t per_nb = ~0ull / (uint64_t)nb + 1; /* (nb = 1: not used) */
    const bool vec = cols % 8 == 0 && nm_al(x, rows > 1 ? x_stride : 0, x_bf16 ? 2 : 4) && ((uintptr_t)q & 7) == 0 &&
                     (rows == 1 || q_stride % 8 == 0);
    const int at_once = (1 << 30) / nb; /* rows of a launch */
    for (int64_t r0 = 0; r0 < rows; r0 += at_once) {
        const int n = rows - r0 < at_once ? (int)(rows - r0) : at_once, grid = (int)(((int64_t)n * nb + 31) / 32);
        const uint8_t *xr = reinterpret_cast<const uint8_t *>(x) + r0 * x_stride * (x_bf16 ? 2 : 4);
        const int rc = ops_launch(vec ? k_ops_quantize<true> : k_ops_quantize<false>, grid, 256, 0, (cudaStream_t)stream, n, cols, nb, per_nb,
                                  (const void *)xr, x_bf16, x_stride, q + r0 * q_stride, q_stride, scales + r0 * scales_stride,
                                  scales_stride);
        if (rc) return rc;
    }
    return 0;
}

/* every kernel of this file loaded on the current device, so that no call loads one inside a stream capture */
extern "C" int ops_rows_init(void) {
    cudaFuncAttributes f;
    int rc = 0;
#define RK(k) rc |= (int)cudaFuncGetAttributes(&f, (k))
#define RT_RK(N, LOW) RK((k_ops_route<N, LOW>));
    RT_SIZES(RT_RK)
#undef RT_RK
#define NM_RK(G, IT) RK((k_ops_norm<true, G, IT>)); RK((k_ops_norm<false, G, IT>));
    NM_RK(32, 1) NM_RK(32, 2) NM_RK(128, 1) NM_RK(256, 1) NM_RK(512, 1) NM_RK(256, 2) NM_RK(1024, 1) NM_RK(512, 2) NM_RK(1024, 2)
#undef NM_RK
    RK(k_ops_quantize<true>); RK(k_ops_quantize<false>);
#undef RK
    return rc;
}
