/*
 * ops_f8.cu -- products of FP8 (e4m3) rows with FP8 weight matrices, both with block scales: the plain product and the
 * experts of a layer.
 */
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "launch.h"
#include "ops_launch.h"
#include "ops_quant.cuh"
#include "stream.cuh"

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

/* ------------------------------------------------------------------ products on the 5th-generation tensor cores
 * D[row][col] = sum over blocks kb of sa[row][kb] sb[col / 128][kb] (sum over the 128 k of the block of a b).  The inner
 * sums are exact products added up in fp32 by tcgen05.mma (kind::f8f6f4: e4m3 x e4m3, K = 32 an instruction) into tensor
 * memory; the block scales differ from block to block, so every block's sums are read back and joined in registers:
 * acc = fma(sum, sa sb, acc).  A row is a lane of tensor memory and a weight tile has one scale a block, so a thread needs
 * one factor for all of its columns.
 *
 * One persistent block per SM, warp-specialised: warp 8 asks for the operand tiles (TMA, 128-byte swizzle, one block of
 * 128 k a stage), one thread of warp 9 issues the MMAs (M = 128 rows, N = NT columns), warps 0..7 are two warpgroups
 * that each join half of the columns.  Tensor memory holds NB buffers of NT columns, so the MMAs of the next block run
 * while this one's sums are joined: NT / 2 columns a thread are NT / 4 two-wide FMAs of 2 warps a scheduler, under the
 * 2 NT cycles that the MMAs of the block take.
 *
 *   dense    A: rows of a;                                 B: NT rows of b;                 D to out
 *   gate/up  A: the tokens of an expert's pairs (gather4); B: 128 gate rows, 128 up rows;   silu(g) u to FP8, 128 a block
 *   down     A: an expert's rows of the activations;       B: NT rows of its down matrix;   D to the pair's row of dots
 *
 * Every wait is bounded; when one runs out the status word is set, all roles stop waiting and the block drains, frees its
 * tensor memory and returns. */
enum { F8_DENSE = 0, F8_GATE_UP = 1, F8_DOWN = 2 };

#define F8_THREADS 384
#define F8_EPI_WARPS 8
#define F8_WAIT_LIMIT (1u << 22)
#define F8_A_BYTES 16384u /* 128 rows x 128 k */
#define F8_MAX_STAGES 8

typedef struct {
    CUtensorMap ta, tb;
    int m, n, k; /* n: rows of b, of one half (gate or up) for F8_GATE_UP */
    const float *a_scales;
    int64_t as_stride;
    const float *b_scales;
    int64_t bs_stride, bs_rec; /* elements of a row of blocks, of a record */
    int b_rec_rows;            /* rows of b of a record */
    void *out;
    int out_bf16, out_vec; /* out_vec: rows of out are 16-byte aligned */
    int64_t out_stride;
    uint8_t *act_q; /* F8_GATE_UP: [pairs][n] */
    float *act_scales;
    const int *counts, *pairs;
    const int4 *items;
    int n_routed, top_k;
    int *status;
} f8_args_t;

typedef struct {
    uint64_t full[F8_MAX_STAGES], empty[F8_MAX_STAGES], acc_full[4], acc_empty[4];
    uint32_t tmem_base;
    volatile int abort_flag;
    float amax[2][2][128]; /* tile parity, warpgroup, row */
} f8_ctl_t;

__device__ __forceinline__ bool f8_wait(uint32_t bar, uint32_t parity, f8_ctl_t *C) {
    for (uint32_t i = 0; i < F8_WAIT_LIMIT; i++) {
        if (fb_mbar_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u && C->abort_flag) return false;
    }
    C->abort_flag = 1;
    return false;
}

/* shared-memory matrix descriptor: K-major, 128-byte swizzle, 8-row groups 1024 bytes apart */
__device__ __forceinline__ uint64_t f8_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}

__device__ __forceinline__ void f8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void f8_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void f8_tma2(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

/* four rows of the map, anywhere */
__device__ __forceinline__ void f8_gather4(uint32_t dst, const CUtensorMap *map, int x, int4 y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void f8_tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

/* the loads of r have landed (r passes through so that nothing reads it earlier) */
__device__ __forceinline__ void f8_tmem_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

/* acc += v s, two columns at once */
__device__ __forceinline__ void f8_fma2(float2 &acc, uint32_t v0, uint32_t v1, float s) {
    unsigned long long a, v, f;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(v0), "r"(v1));
    asm("mov.b64 %0, {%1, %1};" : "=l"(f) : "f"(s));
    asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(acc.x), "f"(acc.y));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(v), "l"(f));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(acc.x), "=f"(acc.y) : "l"(a));
}

/* what tile `it` is */
typedef struct {
    int e, r0, rows, n0;
} f8_tile_t;

template <int MODE, int NT>
__device__ __forceinline__ f8_tile_t f8_tile(const f8_args_t &P, int it, int n_tiles) {
    f8_tile_t t;
    if (MODE == F8_DENSE) { /* rows first: tiles in flight at the same time share rows of b */
        const int mt = (P.m + 127) / 128, nt = it / mt;
        t.e = 0;
        t.r0 = (it - nt * mt) * 128;
        t.rows = min(128, P.m - t.r0);
        t.n0 = nt * NT;
    } else {
        const int g = it / n_tiles;
        const int4 I = P.items[g];
        t.e = I.x;
        t.r0 = I.y;
        t.rows = I.z;
        t.n0 = (it - g * n_tiles) * (MODE == F8_GATE_UP ? NT / 2 : NT);
    }
    return t;
}

template <int MODE, int NT>
struct f8_cfg {
    static constexpr int B_BYTES = NT * 128, STAGE = (int)F8_A_BYTES + B_BYTES;
    static constexpr int STAGES = NT == 256 ? 4 : NT == 128 ? 6 : 8;
    static constexpr int NB = NT == 256 ? 2 : 4;
    static constexpr int SMEM = STAGES * STAGE + 1024 + (int)sizeof(f8_ctl_t);
};

template <int MODE, int NT>
__global__ void __launch_bounds__(F8_THREADS, 1) k_f8_mma(const __grid_constant__ f8_args_t P) {
    typedef f8_cfg<MODE, NT> cfg;
    constexpr int STAGES = cfg::STAGES, NB = cfg::NB;
    extern __shared__ uint8_t dyn_raw[];
    const uint32_t dyn_u = (fb_smem_u32(dyn_raw) + 1023u) & ~1023u;
    f8_ctl_t *C = reinterpret_cast<f8_ctl_t *>(dyn_raw + (dyn_u - fb_smem_u32(dyn_raw)) + STAGES * cfg::STAGE);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per_n = MODE == F8_GATE_UP ? NT / 2 : NT;
    const int n_tiles = (P.n + per_n - 1) / per_n, kbs = (P.k + 127) / 128;
    const int tiles = MODE == F8_DENSE ? ((P.m + 127) / 128) * n_tiles : P.counts[0] * n_tiles;

    if (tid == 0) {
        for (int s = 0; s < STAGES; s++) {
            fb_mbar_init(fb_smem_u32(&C->full[s]), 1);
            fb_mbar_init(fb_smem_u32(&C->empty[s]), 1);
        }
        for (int b = 0; b < NB; b++) {
            fb_mbar_init(fb_smem_u32(&C->acc_full[b]), 1);
            fb_mbar_init(fb_smem_u32(&C->acc_empty[b]), F8_EPI_WARPS);
        }
        C->abort_flag = 0;
        fb_mbar_init_fence();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fb_smem_u32(&C->tmem_base)),
                     "r"((uint32_t)(NB * NT))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = C->tmem_base;

    if (warp >= F8_EPI_WARPS) {
        /* 384 x 168 registers at launch = 128 x 72 + 256 x 216 */
        if (NT == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 8) {
            /* ---------------- operand tiles */
            uint32_t step = 0;
            bool ok = true;
            for (int it = blockIdx.x; it < tiles && ok; it += gridDim.x) {
                const f8_tile_t t = f8_tile<MODE, NT>(P, it, n_tiles);
                int4 rows = make_int4(0, 0, 0, 0); /* gate/up: this lane's four tokens; past the end, the last pair's again */
                int groups = (t.rows + 31) / 32;
                uint32_t a_bytes = (uint32_t)groups * 4096u;
                if (MODE == F8_GATE_UP) {
                    int v[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int p = P.pairs[t.r0 + min(4 * lane + i, t.rows - 1)];
                        v[i] = p < P.n_routed ? p / P.top_k : p - P.n_routed;
                    }
                    rows = make_int4(v[0], v[1], v[2], v[3]);
                    groups = (t.rows + 3) / 4;
                    a_bytes = (uint32_t)groups * 512u;
                }
                for (int kb = 0; kb < kbs; kb++, step++) {
                    const int s = step % STAGES;
                    const uint32_t bar = fb_smem_u32(&C->full[s]), a_u = dyn_u + s * cfg::STAGE, b_u = a_u + F8_A_BYTES;
                    if (!__all_sync(FULL, f8_wait(fb_smem_u32(&C->empty[s]), ((step / STAGES) & 1) ^ 1, C))) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) {
                        fb_mbar_expect_tx(bar, a_bytes + cfg::B_BYTES);
                        if (MODE == F8_GATE_UP) {
                            f8_tma2(b_u, &P.tb, kb * 128, t.e * P.b_rec_rows + t.n0, bar);
                            f8_tma2(b_u + 16384u, &P.tb, kb * 128, t.e * P.b_rec_rows + P.n + t.n0, bar);
                        } else {
                            f8_tma2(b_u, &P.tb, kb * 128, t.e * P.b_rec_rows + t.n0, bar);
                        }
                    }
                    __syncwarp();
                    if (lane < groups) {
                        if (MODE == F8_GATE_UP) f8_gather4(a_u + lane * 512u, &P.ta, kb * 128, rows, bar);
                        else f8_tma2(a_u + lane * 4096u, &P.ta, kb * 128, t.r0 + 32 * lane, bar);
                    }
                }
            }
            /* every stage's last commit has arrived before the block, and with it the barriers' memory, goes away */
            for (int i = 0; i < STAGES && ok; i++, step++)
                ok = __all_sync(FULL, f8_wait(fb_smem_u32(&C->empty[step % STAGES]), ((step / STAGES) & 1) ^ 1, C));
        } else if (warp == 9 && lane == 0) {
            /* ---------------- MMAs: one thread */
            const uint32_t idesc = (1u << 4) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            uint32_t step = 0;
            bool ok = true;
            for (int it = blockIdx.x; it < tiles && ok; it += gridDim.x)
                for (int kb = 0; kb < kbs; kb++, step++) {
                    const int s = step % STAGES, b = step % NB;
                    if (!f8_wait(fb_smem_u32(&C->acc_empty[b]), ((step / NB) & 1) ^ 1, C) ||
                        !f8_wait(fb_smem_u32(&C->full[s]), (step / STAGES) & 1, C)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t a_u = dyn_u + s * cfg::STAGE, b_u = a_u + F8_A_BYTES;
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        f8_mma(tmem + (uint32_t)(b * NT), f8_desc(a_u + 32 * q), f8_desc(b_u + 32 * q), idesc, q > 0);
                    f8_commit(fb_smem_u32(&C->empty[s]));
                    f8_commit(fb_smem_u32(&C->acc_full[b]));
                }
        }
        __syncwarp();
    } else {
        if (NT == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        /* ---------------- join the blocks' sums: warp w reads lanes 32 (w % 4) .., warpgroup wg its half of the columns */
        constexpr int W = NT / 2, CH = W / 16;
        const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t t_row = tmem + ((uint32_t)(warp & 3) << 21);
        uint32_t step = 0, cnt = 0;
        bool ok = true;
        for (int it = blockIdx.x; it < tiles; it += gridDim.x, cnt++) {
            const f8_tile_t t = f8_tile<MODE, NT>(P, it, n_tiles);
            int sr = t.r0 + min(row, t.rows - 1); /* the row of the scales */
            if (MODE == F8_GATE_UP) {
                const int p = P.pairs[sr];
                sr = p < P.n_routed ? p / P.top_k : p - P.n_routed;
            }
            const float *sa_p = P.a_scales + (int64_t)sr * P.as_stride;
            const int c0 = t.n0 + (MODE == F8_GATE_UP ? 0 : wg * W); /* first row of b of this thread's columns */
            const float *sb_p = P.b_scales + (int64_t)t.e * P.bs_rec + (int64_t)(min(c0, P.n - 1) >> 7) * P.bs_stride;
            const float *su_p = sb_p + (int64_t)(P.n >> 7) * P.bs_stride; /* gate/up: the up rows' */
            float2 acc[W / 2];
#pragma unroll
            for (int i = 0; i < W / 2; i++) acc[i] = make_float2(0.0f, 0.0f);
            float sa = __ldg(sa_p), sb = __ldg(sb_p), su = MODE == F8_GATE_UP ? __ldg(su_p) : 0.0f;
            for (int kb = 0; kb < kbs; kb++, step++) {
                const int b = step % NB;
                const float f0 = sa * sb, f1 = MODE == F8_GATE_UP ? sa * su : f0;
                if (kb + 1 < kbs) { /* asked for before the wait */
                    sa = __ldg(sa_p + kb + 1);
                    sb = __ldg(sb_p + kb + 1);
                    if (MODE == F8_GATE_UP) su = __ldg(su_p + kb + 1);
                }
                if (ok) ok = __all_sync(FULL, f8_wait(fb_smem_u32(&C->acc_full[b]), (step / NB) & 1, C));
                if (!ok) continue;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t r[2][16];
                const uint32_t tc = t_row + (uint32_t)(b * NT);
                /* chunk c of the thread's columns: gate/up takes half of them from the gate's columns, half from the up's */
#define F8_COL(c) (uint32_t)(MODE == F8_GATE_UP ? ((c) < CH / 2 ? wg * (W / 2) + 16 * (c) : NT / 2 + wg * (W / 2) + 16 * ((c) - CH / 2)) : wg * W + 16 * (c))
                f8_tmem_ld16(tc + F8_COL(0), r[0]);
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    f8_tmem_wait(r[c & 1]);
                    if (c + 1 < CH) {
                        f8_tmem_ld16(tc + F8_COL(c + 1), r[(c + 1) & 1]);
                    } else { /* the buffer has been read: the next block's MMAs may have it */
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) fb_mbar_arrive(fb_smem_u32(&C->acc_empty[b]));
                    }
                    const float f = MODE == F8_GATE_UP && c >= CH / 2 ? f1 : f0;
#pragma unroll
                    for (int i = 0; i < 8; i++) f8_fma2(acc[8 * c + i], r[c & 1][2 * i], r[c & 1][2 * i + 1], f);
                }
            }
            if (MODE == F8_GATE_UP) {
                /* silu(g) u of this thread's 64 columns, and the amax over the row's 128 with the other warpgroup's */
                float amax = 0.0f;
#pragma unroll
                for (int i = 0; i < W / 4; i++) {
                    const float2 g = acc[i], u = acc[W / 4 + i];
                    acc[i].x = g.x / (1.0f + expf(-g.x)) * u.x;
                    acc[i].y = g.y / (1.0f + expf(-g.y)) * u.y;
                    amax = ops_amax(ops_amax(amax, acc[i].x), acc[i].y);
                }
                C->amax[cnt & 1][wg][row] = amax;
                asm volatile("bar.sync 1, 256;" ::: "memory"); /* the 8 warps meet once a tile, also after a wait that ran out */
                const float sc = ops_f8_scale(ops_amax(amax, C->amax[cnt & 1][wg ^ 1][row]));
                if (row < t.rows && ok) {
                    uint4 *q = reinterpret_cast<uint4 *>(P.act_q + (int64_t)(t.r0 + row) * P.n + t.n0 + wg * 64);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            w[i] = ops_f8_pack4(__fdiv_rn(acc[8 * j + 2 * i].x, sc), __fdiv_rn(acc[8 * j + 2 * i].y, sc),
                                                __fdiv_rn(acc[8 * j + 2 * i + 1].x, sc), __fdiv_rn(acc[8 * j + 2 * i + 1].y, sc));
                        q[j] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (wg == 0) P.act_scales[(int64_t)(t.r0 + row) * (P.n >> 7) + (t.n0 >> 7)] = sc;
                }
            } else if (row < t.rows && ok) {
                const int64_t o = (int64_t)(MODE == F8_DOWN ? P.pairs[t.r0 + row] : t.r0 + row) * P.out_stride + c0;
                const int left = P.n - c0;
                if (P.out_bf16) {
                    __nv_bfloat16 *out = reinterpret_cast<__nv_bfloat16 *>(P.out) + o;
#pragma unroll
                    for (int j = 0; j < W / 8; j++) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const __nv_bfloat162 h = __floats2bfloat162_rn(acc[4 * j + i].x, acc[4 * j + i].y);
                            w[i] = *reinterpret_cast<const uint32_t *>(&h);
                        }
                        if (P.out_vec && 8 * j + 8 <= left) {
                            *reinterpret_cast<uint4 *>(out + 8 * j) = make_uint4(w[0], w[1], w[2], w[3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; i++)
                                if (8 * j + i < left)
                                    reinterpret_cast<uint16_t *>(out)[8 * j + i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
                        }
                    }
                } else {
                    float *out = reinterpret_cast<float *>(P.out) + o;
#pragma unroll
                    for (int j = 0; j < W / 4; j++) {
                        const float4 v = make_float4(acc[2 * j].x, acc[2 * j].y, acc[2 * j + 1].x, acc[2 * j + 1].y);
                        if (P.out_vec && 4 * j + 4 <= left) {
                            *reinterpret_cast<float4 *>(out + 4 * j) = v;
                        } else {
                            if (4 * j < left) out[4 * j] = v.x;
                            if (4 * j + 1 < left) out[4 * j + 1] = v.y;
                            if (4 * j + 2 < left) out[4 * j + 2] = v.z;
                            if (4 * j + 3 < left) out[4 * j + 3] = v.w;
                        }
                    }
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (C->abort_flag) {
        if (tid == 0) *P.status = FB_ST_WAIT_TIMEOUT;
        for (int i = 0; i < 100; i++) __nanosleep(1000); /* copies and MMAs under way land before their memory is released */
        __syncthreads();
    }
    if (warp == 9)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(NB * NT)) : "memory");
}

/* ------------------------------------------------------------------ tensor maps */
typedef CUresult (*f8_encode_t)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static f8_encode_t f8_encode; /* the driver's encoder, looked up once (ops_f8_init) */

/* rows of `k` bytes, `stride` apart; boxes of 128 bytes x box_rows */
static int f8_map(CUtensorMap *m, const void *p, uint64_t k, uint64_t rows, uint64_t stride, uint32_t box_rows) {
    const cuuint64_t dim[2] = {k, rows}, st[1] = {stride};
    const cuuint32_t box[2] = {128, box_rows}, one[2] = {1, 1};
    return f8_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(p), dim, st, box, one,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0
               : (int)cudaErrorInvalidValue;
}

template <int MODE, int NT>
static int f8_launch(f8_args_t &p, int64_t most_tiles, int n_sm, int *launches, cudaStream_t st) {
    const int grid = (int)(most_tiles < n_sm ? most_tiles : n_sm);
    k_f8_mma<MODE, NT><<<grid, F8_THREADS, f8_cfg<MODE, NT>::SMEM, st>>>(p);
    *launches += 1;
    return (int)cudaGetLastError();
}

extern "C" int ops_launch_f8_matmul(const fomoe_b200_f8_matmul_args_t *a, int *status, int n_sm, int *launches,
                                    void *stream) {
    f8_args_t p = {};
    p.m = a->m, p.n = a->n, p.k = a->k;
    p.a_scales = a->a_scales, p.as_stride = a->a_scales_stride;
    p.b_scales = a->b_scales, p.bs_stride = a->b_scales_stride;
    p.out = a->out, p.out_bf16 = a->out_type == FOMOE_B200_BF16, p.out_stride = a->out_stride;
    p.out_vec = ((uintptr_t)a->out & 15) == 0 && (a->out_stride * (p.out_bf16 ? 2 : 4)) % 16 == 0;
    p.status = status;
    /* columns of a tile: 256 keep the tensor cores' operand traffic lowest; fewer when that would leave SMs without one */
    const int64_t mt = (a->m + 127) / 128;
    const int nt = mt * ((a->n + 255) / 256) >= n_sm ? 256 : mt * ((a->n + 127) / 128) >= n_sm ? 128 : 64;
    int rc = f8_map(&p.ta, a->a, a->k, a->m, a->a_stride, 32) | f8_map(&p.tb, a->b, a->k, a->n, a->b_stride, nt);
    if (rc) return rc;
    const int64_t tiles = mt * ((a->n + nt - 1) / nt);
    cudaStream_t st = (cudaStream_t)stream;
    return nt == 256   ? f8_launch<F8_DENSE, 256>(p, tiles, n_sm, launches, st)
           : nt == 128 ? f8_launch<F8_DENSE, 128>(p, tiles, n_sm, launches, st)
                       : f8_launch<F8_DENSE, 64>(p, tiles, n_sm, launches, st);
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
    PART(dots, np * a->n_embd * 4);
#undef PART
    w->bytes = at;
}

extern "C" int ops_launch_f8_experts(const fomoe_b200_f8_experts_args_t *a, uint8_t *ws, int *status, int n_sm,
                                     int *launches, void *stream) {
    cudaStream_t st = (cudaStream_t)stream;
    ops_experts_ws_t w;
    ops_experts_layout(a, &w);
    const int n_routed = a->n_tokens * a->top_k, H = a->n_embd, I = a->n_inter;
    int *counts = (int *)(ws + w.counts), *pairs = (int *)(ws + w.pairs);
    int4 *items = (int4 *)(ws + w.counts + 256);
    k_ops_bucket<<<1, BK_THREADS, (size_t)a->n_experts * BK_WARPS * 4, st>>>(a->ids, n_routed, a->n_tokens, a->n_experts,
                                                                            a->has_shared, counts, pairs, items, status);
    *launches += 1;
    int rc = (int)cudaGetLastError();
    if (rc) return rc;
    /* a tile of pairs holds at most 128 of one expert: no more tiles than this (the device knows how many there are) */
    const int64_t tiles = w.n_pairs / 128 + a->n_experts + 1, recs = a->n_experts + (a->has_shared ? 1 : 0);
    f8_args_t p = {};
    p.counts = counts, p.pairs = pairs, p.items = items, p.n_routed = n_routed, p.top_k = a->top_k, p.status = status;
    p.n = I, p.k = H;
    p.a_scales = a->x_scales, p.as_stride = a->x_scales_stride;
    p.b_scales = a->gate_up_scales, p.bs_stride = H / 128, p.bs_rec = (int64_t)(2 * I / 128) * (H / 128), p.b_rec_rows = 2 * I;
    p.act_q = ws + w.act_q, p.act_scales = (float *)(ws + w.act_scales);
    rc = f8_map(&p.ta, a->x, H, a->n_tokens, a->x_stride, 1) | f8_map(&p.tb, a->gate_up, H, recs * 2 * I, H, 128);
    if (!rc) rc = f8_launch<F8_GATE_UP, 256>(p, tiles * (I / 128), n_sm, launches, st);
    if (rc) return rc;
    p.n = H, p.k = I;
    p.a_scales = p.act_scales, p.as_stride = I / 128;
    p.b_scales = a->down_scales, p.bs_stride = I / 128, p.bs_rec = (int64_t)(H / 128) * (I / 128), p.b_rec_rows = H;
    p.out = ws + w.dots, p.out_stride = H, p.out_vec = 1;
    rc = f8_map(&p.ta, ws + w.act_q, I, w.n_pairs, I, 32) | f8_map(&p.tb, a->down, I, recs * H, I, 256);
    if (!rc) rc = f8_launch<F8_DOWN, 256>(p, tiles * ((H + 255) / 256), n_sm, launches, st);
    if (rc) return rc;
    k_ops_combine<<<a->n_tokens, 256, 0, st>>>((const float *)(ws + w.dots), a->ids, a->weights, H, a->n_experts, a->top_k,
                                              n_routed, a->has_shared, (__nv_bfloat16 *)a->out, a->out_stride);
    *launches += 1;
    return (int)cudaGetLastError();
}

extern "C" int ops_f8_init(void) {
    cudaFuncAttributes f;
    int rc = 0;
    if (!f8_encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return (int)cudaErrorUnknown;
        f8_encode = (f8_encode_t)fn;
    }
#define RK(k) rc |= (int)cudaFuncGetAttributes(&f, (k))
#define RM(MODE, NT) \
    rc |= (int)cudaFuncSetAttribute(k_f8_mma<MODE, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, f8_cfg<MODE, NT>::SMEM)
    RK(k_ops_combine); RK(k_ops_bucket);
    RM(F8_DENSE, 256); RM(F8_DENSE, 128); RM(F8_DENSE, 64); RM(F8_GATE_UP, 256); RM(F8_DOWN, 256);
#undef RM
#undef RK
    rc |= (int)cudaFuncSetAttribute(k_ops_bucket, cudaFuncAttributeMaxDynamicSharedMemorySize, OPS_MAX_E * BK_WARPS * 4);
    return rc;
}
