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
#include "ops_launch.cuh"
#include "ops_launch.h"
#include "ops_quant.cuh"
#include "stream.cuh"

#ifndef FULL
#define FULL 0xffffffffu
#endif

/* ------------------------------------------------------------------ kernels of one call, one after the other
 * Launched with the programmatic-serialization attribute a kernel may start while the one before it in the stream ends:
 * what it does before f8_after() overlaps that end and must not touch anything the kernel before it writes; f8_after()
 * returns when that kernel has completed and its writes are visible.  f8_next() in the kernel before lets the next one start
 * that early (else it starts as the blocks exit). */
__device__ __forceinline__ void f8_after() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void f8_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
static int f8_launch_after(void (*k)(P...), dim3 grid, int threads, int smem, cudaStream_t st, A... args) {
    cudaLaunchAttribute at[1] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    return ops_launch(k, grid, threads, smem, st, at, 1, args...);
}

/* ------------------------------------------------------------------ bucket: the pairs of every expert, in pair order
 * Block b owns a run of pairs, warp w a run of the block's.  A first walk counts each warp's pairs of every expert, prefixes
 * over (expert, block, warp) give every warp its first place, a second walk places the pairs.  The order inside an expert is
 * the order of the pairs, so results do not depend on timing.  The shared expert's pairs (n_routed + t) come last.  With more
 * than one block a first launch (COUNT) leaves each block's counts in `block_counts`.  Eight ids a lane are in flight at
 * once.  (65,536 pairs in 64 experts: one block 150 us, eight ids a lane 100 us, bound by one SM's scattered stores; by 16
 * blocks in two launches 19 us.) */
#define BK_THREADS 1024
#define BK_WARPS 32
#define BK_AHEAD 8
#define BK_RUN 4096   /* pairs of a block, unless that makes more than ... */
#define BK_BLOCKS 64  /* ... this many blocks */

template <bool COUNT>
__global__ void __launch_bounds__(BK_THREADS) k_ops_bucket(const int *ids, int n_routed, int block_run, int n_tokens,
                                                          int n_experts, int has_shared, int *block_counts, int *counts,
                                                          int *pairs, int *pos, int4 *items, int *status) {
    extern __shared__ int s_cnt[]; /* [n_experts][BK_WARPS], then [n_experts]: the block's first place */
    __shared__ int s_tot[BK_WARPS], s_til[BK_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    f8_next();
    for (int i = tid; i < n_experts * BK_WARPS; i += BK_THREADS) s_cnt[i] = 0;
    if (!COUNT) f8_after();
    __syncthreads();
    const int run = ((block_run + BK_THREADS - 1) / BK_THREADS) * 32; /* pairs of a warp */
    const int q1 = min(n_routed, ((int)blockIdx.x + 1) * block_run);
    const int p0 = min(q1, (int)blockIdx.x * block_run + warp * run), p1 = min(q1, p0 + run);
    for (int b0 = p0; b0 < p1; b0 += 32 * BK_AHEAD) {
        int e[BK_AHEAD];
#pragma unroll
        for (int u = 0; u < BK_AHEAD; u++) e[u] = b0 + 32 * u + lane < p1 ? ids[b0 + 32 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < BK_AHEAD; u++) {
            if ((unsigned)e[u] < (unsigned)n_experts) atomicAdd(&s_cnt[e[u] * BK_WARPS + warp], 1);
            else if (e[u] != -1) status[OPS_STATUS_WORD(FB_ST_BAD_ID)] = 1;
        }
    }
    __syncthreads();
    /* thread e: the expert's total and what the blocks before this one have of it */
    int tot = 0, before = 0;
    if (tid < n_experts) {
        if (COUNT || gridDim.x == 1)
            for (int w = 0; w < BK_WARPS; w++) tot += s_cnt[tid * BK_WARPS + ((w + tid) & 31)];
        else
            for (int b = 0; b < (int)gridDim.x; b++) {
                const int n = block_counts[b * n_experts + tid];
                tot += n;
                before += b < (int)blockIdx.x ? n : 0;
            }
    }
    if (COUNT) {
        if (tid < n_experts) block_counts[blockIdx.x * n_experts + tid] = tot;
        return;
    }
    /* exclusive prefixes of pairs and of 128-row tiles over the experts */
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
    int base = a - tot, tbase = c - til, all = 0;
    for (int w = 0; w < BK_WARPS; w++) {
        all += s_tot[w];
        if (w < warp) {
            base += s_tot[w];
            tbase += s_til[w];
        }
    }
    if (blockIdx.x == 0) {
        if (tid < n_experts) {
            for (int m = 0; m < til; m++) items[tbase + m] = make_int4(tid, base + 128 * m, min(128, tot - 128 * m), 0);
        } else if (tid == BK_THREADS - 1) { /* no expert's thread: n_experts <= 512 */
            const int sh = has_shared ? (n_tokens + 127) / 128 : 0;
            for (int m = 0; m < sh; m++)
                items[tbase + m] = make_int4(n_experts, base + 128 * m, min(128, n_tokens - 128 * m), 0);
            counts[0] = tbase + sh; /* tiles */
            counts[1] = base;       /* routed pairs that are left */
        }
    }
    /* the first place of every (expert, warp): a warp to an expert, a lane to a warp's count */
    if (tid < n_experts) s_cnt[n_experts * BK_WARPS + tid] = base + before;
    __syncthreads();
    for (int e = warp; e < n_experts; e += BK_WARPS) {
        const int n = s_cnt[e * BK_WARPS + lane];
        int x = n;
        for (int s = 1; s < 32; s <<= 1) {
            const int o = __shfl_up_sync(FULL, x, s);
            if (lane >= s) x += o;
        }
        s_cnt[e * BK_WARPS + lane] = s_cnt[n_experts * BK_WARPS + e] + x - n;
    }
    __syncthreads();
    for (int b0 = p0; b0 < p1; b0 += 32 * BK_AHEAD) {
        int e[BK_AHEAD];
#pragma unroll
        for (int u = 0; u < BK_AHEAD; u++) e[u] = b0 + 32 * u + lane < p1 ? ids[b0 + 32 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < BK_AHEAD; u++) {
            const bool in = (unsigned)e[u] < (unsigned)n_experts;
            const unsigned same = __match_any_sync(FULL, in ? e[u] : -1);
            int at = 0;
            if (in) {
                at = s_cnt[e[u] * BK_WARPS + warp] + __popc(same & ((1u << lane) - 1u));
                pairs[at] = b0 + 32 * u + lane;
                pos[b0 + 32 * u + lane] = at;
            }
            __syncwarp();
            if (in && lane == 31 - __clz(same)) s_cnt[e[u] * BK_WARPS + warp] = at + 1;
            __syncwarp();
        }
    }
    if (has_shared)
        for (int t = blockIdx.x * BK_THREADS + tid; t < n_tokens; t += gridDim.x * BK_THREADS) {
            pairs[all + t] = n_routed + t;
            pos[n_routed + t] = all + t;
        }
}

/* ------------------------------------------------------------------ products on the 5th-generation tensor cores
 * D[row][col] = sum over blocks kb of sa[row][kb] sb[col / 128][kb] (sum over the 128 k of the block of a b).  The inner
 * sums are exact products added up in fp32 by tcgen05.mma (kind::f8f6f4: e4m3 x e4m3, K = 32 an instruction) into tensor
 * memory; the block scales differ from block to block, so every block's sums are read back and joined in registers:
 * acc = fma(sum, sa sb, acc).  A row is a lane of tensor memory and a weight tile has one scale a block, so a thread needs
 * one factor for all of its columns.
 *
 * Persistent blocks, one per SM, warp-specialised: warp 8 asks for the operand tiles (TMA, 128-byte swizzle, one block of
 * 128 k a stage), one thread of warp 9 issues the MMAs (M = 128 rows, NT columns), warps 10 and 11 bring the scales, and
 * warps 0..7 are two warpgroups that each join half of the columns.  Tensor memory holds NB buffers of NT columns, so the
 * MMAs of the next block run while this one's sums are joined.
 *
 * F8_PAIR: two SMs work on one tile of 256 x 256 (cta_group::2).  Each loads its own 128 rows and half of the weights'
 * rows, 32 KB a block of k instead of 48, one thread of the first issues the MMAs of both, and each joins its own rows.  Six
 * stages leave 2 KB of staging a warp, so rows leave in runs of 64 bytes by plain stores.
 *
 * What bounds it (4096 x 8192 x 4096): one SM a tile 144.5 us, 1.90 PFLOP/s -- the MMAs with nothing but their barriers take
 * 121 us, the operands of 128 x 256 tiles pass shared memory twice, 192 bytes a cycle at the tensor cores' full rate; the
 * joining FMAs and the way out are the rest --, pairs 136 us, 2.02 PFLOP/s (their bare MMAs 102).  Under the power cap, where a
 * long step runs, 175 and 159 us at 1.66 GHz.  Pairs with four stages and TMA stores out took 179 us there, with stores of 32
 * bytes from registers 172, with runs of 64 bytes 166, all three with scales read past the L1: that alone costs 7 us.  Handing
 * the columns over in two halves (180 us) and 16 joining warps (158 us) were slower: every barrier is shared-memory traffic too.
 *
 *   dense    A: rows of a;                               B: rows of b;                        D to out
 *   gate/up  A: the tokens of an expert's pairs;         B: 128 gate rows, 128 up rows;       silu(g) u to FP8, 128 a block
 *   down     A: the activations of an expert's pairs;    B: rows of its down matrix;          D in fp32
 *
 * Every wait is bounded; when one runs out the status word is set, all roles stop waiting and the block drains, frees its
 * tensor memory and returns. */
enum { F8_DENSE = 0, F8_GATE_UP = 1, F8_DOWN = 2 };
/* a tile belongs to one SM, to the SMs of a cluster that share its blocks of k, or to two SMs that multiply together */
enum { F8_ONE = 0, F8_SPLIT = 1, F8_PAIR = 2 };

#define F8_THREADS 384
#define F8_EPI_WARPS 8
#define F8_WAIT_LIMIT (1u << 22)
#define F8_A_BYTES 16384u /* 128 rows x 128 k */
#define F8_MAX_STAGES 8
#define F8_SC 4 /* blocks of k whose scales are handed over at once */

typedef struct {
    CUtensorMap ta, tb, to; /* to: where D goes, boxes of 128 bytes x 32 rows (out_tma) */
    int m, n, k; /* n: rows of b, of one half (gate or up) for F8_GATE_UP */
    const float *a_scales;
    int64_t as_stride;
    const float *b_scales;
    int64_t bs_stride, bs_rec; /* elements of a row of blocks, of a record */
    int b_rec_rows;            /* rows of b of a record */
    void *out;
    int out_bf16, out_tma; /* out_tma: rows of out are 16-byte aligned, D leaves as boxes */
    int64_t out_stride;
    uint8_t *act_q; /* F8_GATE_UP: [pairs][n] */
    float *act_scales;
    const int *counts;
    const int4 *items;
    int *status;
} f8_args_t;

typedef struct {
    uint64_t full[F8_MAX_STAGES], empty[F8_MAX_STAGES], acc_full[4], acc_empty[4], sc_full[2], sc_empty[2];
    uint32_t tmem_base;
    volatile int abort_flag;
    float amax[2][2][128];              /* tile parity, warpgroup, row */
    float scale[2][F8_SC][2][128];      /* group parity, block of k in the group, column half, row: sa sb */
} f8_ctl_t;

__device__ __forceinline__ bool f8_wait(uint32_t bar, uint32_t parity, f8_ctl_t *C) {
    for (uint32_t i = 0; i < F8_WAIT_LIMIT; i++) {
        if (fb_mbar_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u && C->abort_flag) return false;
    }
    C->abort_flag = 1;
    return false;
}

/* one look, whose answer may be used later: on a busy SM it takes a quarter of a thousand cycles to come back */
__device__ __forceinline__ uint32_t f8_look(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok;
}

__device__ __forceinline__ bool f8_wait_all(uint32_t bar, uint32_t parity, f8_ctl_t *C) {
    return __all_sync(FULL, f8_wait(bar, parity, C));
}

/* one lane of a converged warp: the instructions that take warp-uniform operands (tcgen05, TMA) are issued under it; under
 * `lane == 0` the compiler does not know them to be uniform, and the issue of a block's MMAs took 460 cycles */
__device__ __forceinline__ bool f8_elect() {
    uint32_t p;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(p));
    return p != 0;
}

/* shared-memory matrix descriptor: K-major, 128-byte swizzle, 8-row groups 1024 bytes apart */
__device__ __forceinline__ uint64_t f8_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}

template <bool PAIR>
__device__ __forceinline__ void f8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (PAIR)
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
            "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "setp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
            "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}

/* all MMAs so far, then an arrival at `bar`, in a pair at both SMs' */
template <bool PAIR>
__device__ __forceinline__ void f8_commit(uint32_t bar) {
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

/* the same shared-memory address in the pair's first SM */
__device__ __forceinline__ uint32_t f8_leader(uint32_t addr) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}

__device__ __forceinline__ uint32_t f8_cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}

__device__ __forceinline__ uint32_t f8_cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

/* (not a bounded wait: every thread of every block of the cluster comes here, whatever ran out before) */
__device__ __forceinline__ void f8_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

/* a box of the map to this SM's shared memory; in a pair the barrier may be the first SM's */
template <bool PAIR>
__device__ __forceinline__ void f8_tma2(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    if (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
            "[%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}

__device__ __forceinline__ void f8_tmem_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}

/* the loads have landed (32 registers pass through so that nothing reads them earlier) */
__device__ __forceinline__ void f8_tmem_wait(uint32_t *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
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

__device__ __forceinline__ float f8_silu_mul(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

template <int MODE, int NT, int KIND>
struct f8_cfg {
    static constexpr bool PAIR = KIND == F8_PAIR, SPLIT = KIND == F8_SPLIT;
    static constexpr int ROWS = PAIR ? 256 : 128;              /* of a tile */
    static constexpr int B_BYTES = (PAIR ? NT / 2 : NT) * 128; /* of one SM's share */
    static constexpr int STAGE = (int)F8_A_BYTES + B_BYTES;
    static constexpr int STAGES = PAIR ? 6 : NT == 256 ? (MODE == F8_GATE_UP ? 4 : 3) : 5;
    static constexpr int NB = NT == 256 ? 2 : 4;
    static constexpr int BUFS = NT == 256 ? 2 : 1; /* a warp's staging buffers of 32 rows x 128 bytes */
    static constexpr int OUT = F8_EPI_WARPS * (MODE == F8_GATE_UP ? 0 : PAIR ? 2048 : BUFS * 4096);
    static constexpr int SMEM = STAGES * STAGE + OUT + 1024 + (int)sizeof(f8_ctl_t);
};

/* what tile `it` is */
typedef struct {
    int e, r0, rows, n0;
} f8_tile_t;

template <int MODE, int NT, int ROWS>
__device__ __forceinline__ f8_tile_t f8_tile(const f8_args_t &P, int it, int n_tiles) {
    f8_tile_t t;
    if (MODE == F8_DENSE) { /* rows first: tiles in flight at the same time share rows of b */
        const int mt = (P.m + ROWS - 1) / ROWS, nt = it / mt;
        t.e = 0;
        t.r0 = (it - nt * mt) * ROWS;
        t.rows = min(ROWS, P.m - t.r0);
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

/* 128 bytes of each of a warp's 32 rows to its staging buffer, as a TMA box with 128-byte swizzle has them: the 16-byte piece
 * q of row r at q ^ r % 8, so that a warp's stores have no bank conflicts either */
__device__ __forceinline__ void f8_stage(uint32_t buf, const uint32_t *w) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (uint32_t q = 0; q < 8; q++)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(buf + lane * 128u + ((q ^ (lane & 7u)) << 4)), "r"(w[4 * q]),
                     "r"(w[4 * q + 1]), "r"(w[4 * q + 2]), "r"(w[4 * q + 3])
                     : "memory");
}

/* staged boxes are about to be read by the copy engine */
__device__ __forceinline__ void f8_staged() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

/* a staged box to global memory, whole */
__device__ __forceinline__ void f8_box_out(uint32_t buf, const CUtensorMap *map, int x, int y) {
    if (f8_elect()) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
                     "r"(buf)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    __syncwarp();
}

/* the first `rows` rows of a staged box, by the warp.  row0: where the first row's 128 bytes go, stride: bytes from row to
 * row, left: bytes of the box's rows that are inside out (bytes of a whole row may not fit an int), elem: bytes of a value */
__device__ __forceinline__ void f8_rows_out(uint32_t buf, uint8_t *row0, int64_t stride, int rows, int left, int elem) {
    const int lane = threadIdx.x & 31, per = 128 / elem;
    for (int i = lane; i < rows * per; i += 32) {
        const int r = i / per, c = i - r * per;
        if (c * elem >= left) continue;
        const uint32_t at = buf + r * 128u + (uint32_t)((((c * elem) >> 4) ^ (r & 7)) << 4) + ((c * elem) & 15);
        if (elem == 4) {
            uint32_t v;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
            *reinterpret_cast<uint32_t *>(row0 + r * stride + c * 4) = v;
        } else {
            uint16_t v;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
            *reinterpret_cast<uint16_t *>(row0 + r * stride + c * 2) = v;
        }
    }
    __syncwarp();
}

/* 32 bytes of a row (a whole sector) */
__device__ __forceinline__ void f8_st32(void *p, const uint32_t *w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

/* A warp's 32 rows of BYTES bytes through 2 KB of shared memory, 64 bytes of a row at a time (the 16-byte piece q of row r at
 * q ^ (r / 2) % 4, so that neither side has bank conflicts): they leave as runs of 64 bytes.  Arguments as f8_rows_out's; vec:
 * rows are 16-byte aligned. */
template <int BYTES>
__device__ __forceinline__ void f8_runs_out(uint32_t buf, const uint32_t *w, uint8_t *row0, int64_t stride, int rows, int left, int elem, int vec) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int c = 0; c < BYTES / 64; c++) {
        __syncwarp();
#pragma unroll
        for (uint32_t q = 0; q < 4; q++)
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(buf + lane * 64u + ((q ^ ((lane >> 1) & 3u)) << 4)), "r"(w[16 * c + 4 * q]),
                         "r"(w[16 * c + 4 * q + 1]), "r"(w[16 * c + 4 * q + 2]), "r"(w[16 * c + 4 * q + 3])
                         : "memory");
        __syncwarp();
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const int r = (int)(8 * i + (lane >> 2)), at = 64 * c + 16 * (int)(lane & 3);
            const uint4 v = fb_lds128(buf + r * 64u + (((lane & 3u) ^ ((r >> 1) & 3u)) << 4));
            if (r >= rows || at >= left) continue;
            uint8_t *to = row0 + r * stride + at;
            if (vec && at + 16 <= left) {
                *reinterpret_cast<uint4 *>(to) = v;
            } else {
                const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (elem == 4) {
                        if (at + 4 * k < left) *reinterpret_cast<uint32_t *>(to + 4 * k) = x[k];
                    } else {
                        if (at + 4 * k < left) *reinterpret_cast<uint16_t *>(to + 4 * k) = (uint16_t)x[k];
                        if (at + 4 * k + 2 < left) *reinterpret_cast<uint16_t *>(to + 4 * k + 2) = (uint16_t)(x[k] >> 16);
                    }
                }
            }
        }
    }
}

/* the warp's boxes have left its staging buffers */
__device__ __forceinline__ void f8_box_wait() {
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}

template <int MODE, int NT, int KIND>
__global__ void __launch_bounds__(F8_THREADS, 1) k_f8_mma(const __grid_constant__ f8_args_t P) {
    typedef f8_cfg<MODE, NT, KIND> cfg;
    constexpr int STAGES = cfg::STAGES, NB = cfg::NB, ROWS = cfg::ROWS;
    constexpr bool PAIR = cfg::PAIR, SPLIT = cfg::SPLIT;
    extern __shared__ uint8_t dyn_raw[];
    const uint32_t dyn_u = (fb_smem_u32(dyn_raw) + 1023u) & ~1023u;
    const uint32_t out_u = dyn_u + STAGES * cfg::STAGE;
    f8_ctl_t *C = reinterpret_cast<f8_ctl_t *>(dyn_raw + (dyn_u - fb_smem_u32(dyn_raw)) + STAGES * cfg::STAGE + cfg::OUT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per_n = MODE == F8_GATE_UP ? NT / 2 : NT;
    const int n_tiles = (P.n + per_n - 1) / per_n;
    if (MODE != F8_DENSE) f8_next();
    /* this block's blocks of k: all, or (SPLIT) its rank's share; the cluster's blocks have one tile */
    const uint32_t ranks = SPLIT ? f8_cluster_size() : PAIR ? 2 : 1, rank = KIND != F8_ONE ? f8_cluster_rank() : 0;
    const int kb_all = (P.k + 127) / 128, kb_lo = SPLIT ? (int)(rank * kb_all / ranks) : 0;
    const int kbs = SPLIT ? (int)((rank + 1) * kb_all / ranks) - kb_lo : kb_all;
    const int first = (int)(blockIdx.x / ranks), stride = (int)(gridDim.x / ranks);
    const int up = PAIR ? 128 * (int)rank : 0; /* where this SM's rows of a tile begin */
    int tiles = MODE == F8_DENSE ? (P.m + ROWS - 1) / ROWS * n_tiles : 0;

    if (tid == 0) {
        for (int s = 0; s < STAGES; s++) {
            fb_mbar_init(fb_smem_u32(&C->full[s]), 1);
            fb_mbar_init(fb_smem_u32(&C->empty[s]), 1);
        }
        for (int b = 0; b < NB; b++) {
            fb_mbar_init(fb_smem_u32(&C->acc_full[b]), 1);
            fb_mbar_init(fb_smem_u32(&C->acc_empty[b]), PAIR ? 2 * F8_EPI_WARPS : F8_EPI_WARPS);
        }
        for (int g = 0; g < 2; g++) {
            fb_mbar_init(fb_smem_u32(&C->sc_full[g]), 2);
            fb_mbar_init(fb_smem_u32(&C->sc_empty[g]), F8_EPI_WARPS);
        }
        C->abort_flag = 0;
        fb_mbar_init_fence();
    }
    if (warp == 9) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fb_smem_u32(&C->tmem_base)),
                         "r"((uint32_t)(NB * NT))
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(fb_smem_u32(&C->tmem_base)),
                         "r"((uint32_t)(NB * NT))
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (PAIR) f8_cluster_sync();
    else __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = C->tmem_base;
    if (MODE != F8_DENSE) f8_after();
    if (MODE != F8_DENSE) tiles = P.counts[0] * n_tiles;

    if (warp >= F8_EPI_WARPS) {
        /* 384 x 168 registers at launch = 128 x 72 + 256 x 216 */
        if (NT == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 8) {
            /* ---------------- operand tiles */
            uint32_t st = 0, ph = 0; /* stage, and the parity of its phase */
            bool ok = true;
            for (int it = first; it < tiles && ok; it += stride) {
                const f8_tile_t t = f8_tile<MODE, NT, ROWS>(P, it, n_tiles);
                /* boxes of 32 rows, as many as the rows need; what is behind the tile's rows is never stored */
                const int groups = PAIR ? min(4, max(0, (t.rows - up + 31) / 32)) : (t.rows + 31) / 32;
                const int y = t.e * P.b_rec_rows + t.n0 + (PAIR && rank ? NT / 2 : 0);
                const uint32_t bytes = (uint32_t)((t.rows + 31) / 32) * 4096u + (PAIR ? 2u : 1u) * cfg::B_BYTES; /* of both SMs */
                for (int kb = 0; kb < kbs; kb++) {
                    const uint32_t a_u = dyn_u + st * cfg::STAGE, b_u = a_u + F8_A_BYTES;
                    if (!f8_wait_all(fb_smem_u32(&C->empty[st]), ph ^ 1, C)) {
                        ok = false;
                        break;
                    }
                    if (f8_elect()) {
                        const uint32_t own = fb_smem_u32(&C->full[st]), bar = PAIR ? f8_leader(own) : own;
                        const int x = (kb_lo + kb) * 128;
                        if (!PAIR || rank == 0) fb_mbar_expect_tx(own, bytes);
                        f8_tma2<PAIR>(b_u, &P.tb, x, y, bar);
                        if (MODE == F8_GATE_UP) f8_tma2<PAIR>(b_u + 16384u, &P.tb, x, y + P.n, bar);
                        for (int g = 0; g < groups; g++) f8_tma2<PAIR>(a_u + g * 4096u, &P.ta, x, t.r0 + up + 32 * g, bar);
                    }
                    __syncwarp();
                    if (++st == STAGES) {
                        st = 0;
                        ph ^= 1;
                    }
                }
            }
            /* every stage's last commit has arrived before the block, and with it the barriers' memory, goes away */
            for (int i = 0; i < STAGES && ok; i++) {
                ok = f8_wait_all(fb_smem_u32(&C->empty[st]), ph ^ 1, C);
                if (++st == STAGES) {
                    st = 0;
                    ph ^= 1;
                }
            }
        } else if (warp == 9 && (!PAIR || rank == 0)) {
            /* ---------------- MMAs: one thread, in a pair one for both SMs */
            const uint32_t idesc = (1u << 4) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
            uint32_t st = 0, ph = 0, b = 0, bph = 0, have_ab = 0, have_acc = 0;
            bool ok = true;
            for (int it = first; it < tiles && ok; it += stride)
                for (int kb = 0; kb < kbs; kb++) {
                    if ((!__all_sync(FULL, have_ab) && !f8_wait_all(fb_smem_u32(&C->full[st]), ph, C)) ||
                        (!__all_sync(FULL, have_acc) && !f8_wait_all(fb_smem_u32(&C->acc_empty[b]), bph ^ 1, C))) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t a_u = dyn_u + st * cfg::STAGE, b_u = a_u + F8_A_BYTES;
                    if (f8_elect()) {
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            f8_mma<PAIR>(tmem + b * NT, f8_desc(a_u + 32 * q), f8_desc(b_u + 32 * q), idesc, q > 0);
                        f8_commit<PAIR>(fb_smem_u32(&C->acc_full[b]));
                        f8_commit<PAIR>(fb_smem_u32(&C->empty[st]));
                    }
                    __syncwarp();
                    if (++st == STAGES) {
                        st = 0;
                        ph ^= 1;
                    }
                    if (++b == NB) {
                        b = 0;
                        bph ^= 1;
                    }
                    have_ab = f8_look(fb_smem_u32(&C->full[st]), ph);
                    have_acc = f8_look(fb_smem_u32(&C->acc_empty[b]), bph ^ 1);
                }
        } else if (warp >= 10) {
            /* ---------------- scales: 64 threads, rows i and i + 64; asked for a group of blocks ahead.  (Read by the joining
             * threads themselves they missed the L1 beside 200 KB of shared memory and cost an L2 latency every block.) */
            const int i = tid - 320;
            uint32_t g = 0;
            bool ok = true;
            for (int it = first; it < tiles && ok; it += stride) {
                const f8_tile_t t = f8_tile<MODE, NT, ROWS>(P, it, n_tiles);
                const float *a0 = P.a_scales + (int64_t)(t.r0 + min(up + i, t.rows - 1)) * P.as_stride;
                const float *a1 = P.a_scales + (int64_t)(t.r0 + min(up + i + 64, t.rows - 1)) * P.as_stride;
                const float *rec = P.b_scales + (int64_t)t.e * P.bs_rec;
                const float *b0 = rec + (int64_t)(min(t.n0, P.n - 1) >> 7) * P.bs_stride;
                const float *b1 = rec + (int64_t)((MODE == F8_GATE_UP ? P.n + t.n0 : min(t.n0 + NT / 2, P.n - 1)) >> 7) * P.bs_stride;
                for (int kb = 0; kb < kbs; kb += F8_SC, g++) {
                    float va[2][F8_SC], vb[2][F8_SC];
#pragma unroll
                    for (int q = 0; q < F8_SC; q++) {
                        const int k = kb_lo + min(kb + q, kbs - 1);
                        va[0][q] = a0[k]; /* (no __ldg: the kernel before this one may have written them as this one started) */
                        va[1][q] = a1[k];
                        vb[0][q] = __ldg(b0 + k);
                        vb[1][q] = __ldg(b1 + k);
                    }
                    ok = f8_wait_all(fb_smem_u32(&C->sc_empty[g & 1]), ((g >> 1) & 1) ^ 1, C);
                    if (!ok) break;
#pragma unroll
                    for (int q = 0; q < F8_SC; q++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            C->scale[g & 1][q][h][i] = va[0][q] * vb[h][q];
                            C->scale[g & 1][q][h][i + 64] = va[1][q] * vb[h][q];
                        }
                    __syncwarp();
                    if (lane == 0) fb_mbar_arrive(fb_smem_u32(&C->sc_full[g & 1]));
                }
            }
        }
        __syncwarp();
    } else {
        if (NT == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        /* ---------------- join the blocks' sums: warp w reads lanes 32 (w % 4) .., warpgroup wg its half of the columns */
        constexpr int W = NT / 2;
        const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t t_row = tmem + ((uint32_t)(warp & 3) << 21);
        uint32_t step = 0, cnt = 0, grp = 0, have = 0;
        bool ok = true;
        for (int it = first; it < tiles; it += stride, cnt++) {
            f8_tile_t t = f8_tile<MODE, NT, ROWS>(P, it, n_tiles);
            t.r0 += up, t.rows -= up; /* of this SM (a pair's second may have none) */
            float2 acc[W / 2];
#pragma unroll
            for (int i = 0; i < W / 2; i++) acc[i] = make_float2(0.0f, 0.0f);
            /* the group's scales have come: this block's factors; the last block of a group gives the group back */
#define F8_FACTORS(kb)                                                                               \
    do {                                                                                             \
        const int q_ = (kb) % F8_SC;                                                                 \
        if (ok && q_ == 0) ok = f8_wait_all(fb_smem_u32(&C->sc_full[grp & 1]), (grp >> 1) & 1, C);   \
        n0 = C->scale[grp & 1][q_][MODE == F8_GATE_UP ? 0 : wg][row];                                \
        if (MODE == F8_GATE_UP) n1 = C->scale[grp & 1][q_][1][row];                                  \
        if (q_ == F8_SC - 1 || (kb) == kbs - 1) {                                                    \
            __syncwarp();                                                                            \
            if (ok && lane == 0) fb_mbar_arrive(fb_smem_u32(&C->sc_empty[grp & 1]));                 \
            grp++;                                                                                   \
        }                                                                                            \
    } while (0)
            float n0, n1 = 0.0f;
            F8_FACTORS(0);
            /* Chunks of 32 columns through two register buffers: while one is joined the next is on its way, also across
             * blocks.  (gate/up: the first half of a thread's columns are the gate's, the second the up's) */
#define F8_COL(buffer, c) \
    (t_row + (uint32_t)((buffer) * NT + (MODE == F8_GATE_UP ? (c) / (CH / 2) * (NT / 2) + wg * (W / 2) + (c) % (CH / 2) * 32 : wg * W + (c) * 32)))
            constexpr int CH = W / 32;
            uint32_t r[2][32];
            if (ok && !__all_sync(FULL, have)) ok = f8_wait_all(fb_smem_u32(&C->acc_full[step % NB]), (step / NB) & 1, C);
            if (ok) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                f8_tmem_ld32(F8_COL(step % NB, 0), r[0]);
            }
            for (int kb = 0; kb < kbs; kb++, step++) {
                const int b = step % NB;
                const float f0 = n0, f1 = MODE == F8_GATE_UP ? n1 : n0;
                if (!ok) continue;
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    const int w = c & 1;
                    f8_tmem_wait(r[w]);
                    if (c + 1 < CH) {
                        f8_tmem_ld32(F8_COL(b, c + 1), r[w ^ 1]);
                    } else { /* the buffer has been read: the next block's MMAs may have it */
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) {
                            if (PAIR) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(f8_leader(fb_smem_u32(&C->acc_empty[b]))) : "memory");
                            else fb_mbar_arrive(fb_smem_u32(&C->acc_empty[b]));
                        }
                        if (kb + 1 < kbs) {
                            if (!__all_sync(FULL, have)) ok = f8_wait_all(fb_smem_u32(&C->acc_full[(step + 1) % NB]), ((step + 1) / NB) & 1, C);
                            if (ok) {
                                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                                f8_tmem_ld32(F8_COL((step + 1) % NB, 0), r[w ^ 1]);
                            }
                            F8_FACTORS(kb + 1);
                        } else {
                            have = f8_look(fb_smem_u32(&C->acc_full[(step + 1) % NB]), ((step + 1) / NB) & 1);
                        }
                    }
                    const float f = c >= CH / 2 ? f1 : f0;
#pragma unroll
                    for (int i = 0; i < 16; i++) f8_fma2(acc[16 * c + i], r[w][2 * i], r[w][2 * i + 1], f);
                    /* the next block's barrier is asked for a chunk ahead of its use */
                    if (c == CH - 2) have = f8_look(fb_smem_u32(&C->acc_full[(step + 1) % NB]), ((step + 1) / NB) & 1);
                }
            }
            const uint32_t buf = out_u + warp * (uint32_t)(cfg::OUT / F8_EPI_WARPS);
            if (MODE == F8_GATE_UP) {
                /* silu(g) u of this thread's 64 columns, and the amax over the row's 128 with the other warpgroup's */
                float amax = 0.0f;
#pragma unroll
                for (int i = 0; i < W / 4; i++) {
                    acc[i].x = f8_silu_mul(acc[i].x, acc[W / 4 + i].x);
                    acc[i].y = f8_silu_mul(acc[i].y, acc[W / 4 + i].y);
                    amax = ops_amax(ops_amax(amax, acc[i].x), acc[i].y);
                }
                C->amax[cnt & 1][wg][row] = amax;
                asm volatile("bar.sync 1, 256;" ::: "memory"); /* the 8 warps meet once a tile, also after a wait that ran out */
                const float sc = ops_f8_scale(ops_amax(amax, C->amax[cnt & 1][wg ^ 1][row]));
                const float inv = __frcp_rn(sc);
                const bool mine = row < t.rows && ok;
                if (mine) {
                    uint4 *q = reinterpret_cast<uint4 *>(P.act_q + (int64_t)(t.r0 + row) * P.n + t.n0 + wg * 64);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            w[k] = ops_f8_pack4(ops_f8_quot(acc[8 * i + 2 * k].x, sc, inv), ops_f8_quot(acc[8 * i + 2 * k].y, sc, inv),
                                                ops_f8_quot(acc[8 * i + 2 * k + 1].x, sc, inv), ops_f8_quot(acc[8 * i + 2 * k + 1].y, sc, inv));
                        q[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (wg == 0) P.act_scales[(int64_t)(t.r0 + row) * (P.n >> 7) + (t.n0 >> 7)] = sc;
                }
            } else if (SPLIT) {
                /* this rank's part of the tile, over the operand stages (every MMA has read them): 512 bytes a row, its
                 * 16-byte piece q at q ^ row % 32 */
#pragma unroll
                    for (uint32_t q = 0; q < W / 4; q++)
                        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dyn_u + row * 512u + (((wg * (W / 4) + q) ^ (row & 31u)) << 4)),
                                     "f"(acc[2 * q].x), "f"(acc[2 * q].y), "f"(acc[2 * q + 1].x), "f"(acc[2 * q + 1].y)
                                     : "memory");
            } else {
                /* rows of this warp that are the tile's; a box may only leave whole if none of its rows is another expert's */
                const int w0 = (warp & 3) * 32, rows = ok ? max(0, min(32, t.rows - w0)) : 0, c0 = t.n0 + wg * W;
                const bool tma = !PAIR && P.out_tma && (MODE == F8_DENSE ? rows > 0 : rows == 32);
                if (MODE == F8_DOWN && !tma) { /* (61 tokens of 8 in 256 experts: 156 us by staged rows, 143 so) */
                    if (lane < rows && c0 < P.n) {
                        float *o = reinterpret_cast<float *>(P.out) + (int64_t)(t.r0 + row) * P.out_stride + c0;
#pragma unroll
                        for (int i = 0; i < W / 8; i++) f8_st32(o + 8 * i, reinterpret_cast<const uint32_t *>(acc) + 8 * i);
                    }
                } else if (MODE == F8_DENSE && P.out_bf16) {
                    uint32_t w[W / 2];
#pragma unroll
                    for (int i = 0; i < W / 2; i++) {
                        const __nv_bfloat162 v = __floats2bfloat162_rn(acc[i].x, acc[i].y);
                        w[i] = *reinterpret_cast<const uint32_t *>(&v);
                    }
                    if (PAIR) {
                        f8_runs_out<2 * W>(buf, w, reinterpret_cast<uint8_t *>(P.out) + 2 * ((int64_t)(t.r0 + w0) * P.out_stride + c0),
                                           2 * P.out_stride, rows, 2 * min(P.n - c0, W), 2, P.out_tma);
                        continue;
                    }
                    f8_box_wait();
#pragma unroll
                    for (int c = 0; c < W / 64; c++) f8_stage(buf + c * 4096u, w + 32 * c); /* boxes of 64 columns */
                    f8_staged();
#pragma unroll
                    for (int c = 0; c < W / 64; c++) {
                        const int x = c0 + 64 * c;
                        if (x >= P.n) continue;
                        if (tma) f8_box_out(buf + c * 4096u, &P.to, 2 * x, t.r0 + w0);
                        else
                            f8_rows_out(buf + c * 4096u, reinterpret_cast<uint8_t *>(P.out) + 2 * ((int64_t)(t.r0 + w0) * P.out_stride + x),
                                        2 * P.out_stride, rows, 2 * min(P.n - x, 64), 2);
                    }
                } else if (PAIR) {
                    f8_runs_out<4 * W>(buf, reinterpret_cast<const uint32_t *>(acc),
                                       reinterpret_cast<uint8_t *>(P.out) + 4 * ((int64_t)(t.r0 + w0) * P.out_stride + c0),
                                       4 * P.out_stride, rows, 4 * min(P.n - c0, W), 4, P.out_tma);
                } else {
#pragma unroll
                    for (int c = 0; c < W / 32; c++) { /* boxes of 32 columns, through the buffers there are */
                        const int x = c0 + 32 * c;
                        if (c % cfg::BUFS == 0) f8_box_wait();
                        f8_stage(buf + c % cfg::BUFS * 4096u, reinterpret_cast<const uint32_t *>(acc) + 32 * c);
                        f8_staged();
                        if (x >= P.n) continue;
                        if (tma) f8_box_out(buf + c % cfg::BUFS * 4096u, &P.to, 4 * x, t.r0 + w0);
                        else
                            f8_rows_out(buf + c % cfg::BUFS * 4096u,
                                        reinterpret_cast<uint8_t *>(P.out) + 4 * ((int64_t)(t.r0 + w0) * P.out_stride + x),
                                        4 * P.out_stride, rows, 4 * min(P.n - x, 32), 4);
                    }
                }
            }
        }
        if (MODE != F8_GATE_UP && KIND == F8_ONE) f8_box_wait(); /* the staging buffers go away with the block */
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (C->abort_flag) {
        if (tid == 0) P.status[OPS_STATUS_WORD(FB_ST_WAIT_TIMEOUT)] = 1;
        for (int i = 0; i < 100; i++) __nanosleep(1000); /* copies and MMAs under way land before their memory is released */
    }
    if (SPLIT) {
        /* the parts meet: rank r sums rows r, r + ranks, ... in rank order, a warp a row */
        f8_cluster_sync();
        const f8_tile_t t = f8_tile<MODE, NT, ROWS>(P, first, n_tiles);
        for (int row = (int)rank + (int)ranks * warp; row < t.rows; row += (int)ranks * (F8_THREADS / 32)) {
            const uint32_t at = dyn_u + row * 512u + (((uint32_t)lane ^ (row & 31u)) << 4);
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t s = 0; s < ranks; s++) {
                float x[4];
                uint32_t ra;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(at), "r"(s));
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                             : "r"(ra)
                             : "memory");
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] += x[i];
            }
            const int c = t.n0 + 4 * lane;
            const int64_t o = (int64_t)(t.r0 + row) * P.out_stride + c;
            if (P.out_bf16) {
                __nv_bfloat16 *out = reinterpret_cast<__nv_bfloat16 *>(P.out) + o;
                if (P.out_tma && c + 4 <= P.n) {
                    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
                    *reinterpret_cast<uint2 *>(out) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (c + i < P.n) out[i] = __float2bfloat16_rn(v[i]);
                }
            } else {
                float *out = reinterpret_cast<float *>(P.out) + o;
                if (P.out_tma && c + 4 <= P.n) {
                    *reinterpret_cast<float4 *>(out) = make_float4(v[0], v[1], v[2], v[3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (c + i < P.n) out[i] = v[i];
                }
            }
        }
        f8_cluster_sync(); /* nobody leaves while its part is being read */
    }
    if (PAIR) f8_cluster_sync(); /* neither SM goes while the other's MMAs or arrivals may reach it */
    else __syncthreads();
    if (warp == 9) {
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(NB * NT)) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(NB * NT)) : "memory");
    }
}

/* ------------------------------------------------------------------ few rows: the weights' bytes are all that counts
 * Up to 16 rows of a, or single pairs of an expert.  A block of 8 warps takes 16 weight rows; warp w takes the units
 * (blocks of k; of all slots of a token for the down product) w, w + 8, ..., and the eight partial sums meet in shared
 * memory, in warp order.  A unit, 16 rows x 128 k, goes to the registers of mma.sync (m16n8k32, e4m3: the weight rows are
 * its 16 rows, the activations its columns) through a ring of FR_RING units a warp: each lane copies (cp.async) exactly the
 * four 16-byte pieces that it will read, so no lane waits for another.  The k inside a block come in the order that this
 * gives: lane (g, t) holds bytes 16 t .. of rows g and g + 8, the activations likewise.  16 weight rows a block spread small
 * matrices over all SMs, and nothing has to be set up first: 1 x 4096 x 4096 5.4 us (on tcgen05 11), 16 rows 7.4, 1 x 8192 x
 * 8192 16 us, 1 x 4096 x 16,384 14.5 us, 4.6 TB/s; what is left are start and end of a block, and of large matrices that 256
 * or 512 equal blocks do not come out even on 148 SMs. */
#define FR_WARPS 8
#define FR_RING 2
#define FR_SMEM (FR_WARPS * FR_RING * 2048)

__device__ __forceinline__ void fr_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

/* asks for a unit: the lane's four 16-byte pieces {row g, row g + 8} x {first, second 64 bytes} into its places of the slot;
 * nothing behind k is read (zeros) */
__device__ __forceinline__ void fr_ask(uint32_t slot, const uint8_t *r0, const uint8_t *r1, int at, int k) {
    const uint32_t dst = slot + (threadIdx.x & 31) * 16u;
    const uint32_t in0 = at < k ? 16u : 0u, in1 = at + 64 < k ? 16u : 0u;
    const int a0 = at < k ? at : 0, a1 = at + 64 < k ? at + 64 : 0;
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(r0 + a0), "r"(in0) : "memory");
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst + 512u), "l"(r1 + a0), "r"(in0) : "memory");
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst + 1024u), "l"(r0 + a1), "r"(in1) : "memory");
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst + 1536u), "l"(r1 + a1), "r"(in1) : "memory");
}

__device__ __forceinline__ void fr_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

/* the oldest of RING units in flight has landed: the lane's pieces */
template <int RING>
__device__ __forceinline__ void fr_take(uint4 (&w)[4], uint32_t slot) {
    asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = fb_lds128(slot + (threadIdx.x & 31) * 16u + 512u * i);
}

/* the block's sum of products for 8 columns */
__device__ __forceinline__ void fr_block(float (&c)[4], const uint4 (&w)[4], uint4 x0, uint4 x1) {
    c[0] = c[1] = c[2] = c[3] = 0.0f;
    fr_mma(c, w[0].x, w[1].x, w[0].y, w[1].y, x0.x, x0.y);
    fr_mma(c, w[0].z, w[1].z, w[0].w, w[1].w, x0.z, x0.w);
    fr_mma(c, w[2].x, w[3].x, w[2].y, w[3].y, x1.x, x1.y);
    fr_mma(c, w[2].z, w[3].z, w[2].w, w[3].w, x1.z, x1.w);
}

typedef struct {
    int m, n, k;
    const uint8_t *a;
    int64_t a_stride;
    const float *a_scales;
    int64_t as_stride;
    const uint8_t *b;
    int64_t b_stride;
    const float *b_scales;
    int64_t bs_stride;
    void *out;
    int out_bf16;
    int64_t out_stride;
} fr_args_t;

/* out = a b^T, m <= 8 C8 */
template <int C8>
__global__ void __launch_bounds__(32 * FR_WARPS) k_f8_few(const fr_args_t P) {
    __shared__ float s_part[FR_WARPS][16][8 * C8 + 1];
    extern __shared__ __align__(16) uint8_t ring[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t ring_u = fb_smem_u32(ring) + warp * (FR_RING * 2048u);
    const int n0 = blockIdx.x * 16, kbs = (P.k + 127) / 128;
    const uint8_t *r0 = P.b + (int64_t)min(n0 + g, P.n - 1) * P.b_stride, *r1 = P.b + (int64_t)min(n0 + g + 8, P.n - 1) * P.b_stride;
    const float *bs = P.b_scales + (int64_t)(n0 >> 7) * P.bs_stride;
#pragma unroll
    for (int i = 0; i < FR_RING; i++) {
        const int kb = warp + FR_WARPS * i;
        if (kb < kbs) fr_ask(ring_u + i * 2048u, r0, r1, kb * 128 + 16 * t, P.k);
        fr_commit();
    }
    uint4 nx[C8][2];
    float n0s[C8], n1s[C8], nb = 0.0f;
    auto ahead = [&](int kb) { /* the rows' values and the scales of a block, a block ahead of their use */
        const int at = kb * 128 + 16 * t;
        const uint4 z = make_uint4(0, 0, 0, 0);
        if (kb >= kbs) return;
        nb = __ldg(bs + kb);
#pragma unroll
        for (int h = 0; h < C8; h++) {
            const uint8_t *xp = P.a + (int64_t)min(8 * h + g, P.m - 1) * P.a_stride + at;
            nx[h][0] = at < P.k ? __ldg(reinterpret_cast<const uint4 *>(xp)) : z;
            nx[h][1] = at + 64 < P.k ? __ldg(reinterpret_cast<const uint4 *>(xp + 64)) : z;
            n0s[h] = __ldg(P.a_scales + (int64_t)min(8 * h + 2 * t, P.m - 1) * P.as_stride + kb);
            n1s[h] = __ldg(P.a_scales + (int64_t)min(8 * h + 2 * t + 1, P.m - 1) * P.as_stride + kb);
        }
    };
    ahead(warp);
    float acc[C8][4] = {};
    int slot = 0;
    for (int kb = warp; kb < kbs; kb += FR_WARPS) {
        uint4 x[C8][2];
        float s0[C8], s1[C8];
        const float sb = nb;
#pragma unroll
        for (int h = 0; h < C8; h++) x[h][0] = nx[h][0], x[h][1] = nx[h][1], s0[h] = n0s[h], s1[h] = n1s[h];
        ahead(kb + FR_WARPS);
        uint4 w[4];
        fr_take<FR_RING>(w, ring_u + slot * 2048u);
#pragma unroll
        for (int h = 0; h < C8; h++) {
            float c[4];
            fr_block(c, w, x[h][0], x[h][1]);
            acc[h][0] = fmaf(c[0], sb * s0[h], acc[h][0]);
            acc[h][1] = fmaf(c[1], sb * s1[h], acc[h][1]);
            acc[h][2] = fmaf(c[2], sb * s0[h], acc[h][2]);
            acc[h][3] = fmaf(c[3], sb * s1[h], acc[h][3]);
        }
        const int next = kb + FR_WARPS * FR_RING;
        if (next < kbs) fr_ask(ring_u + slot * 2048u, r0, r1, next * 128 + 16 * t, P.k);
        fr_commit();
        slot = (slot + 1) % FR_RING;
    }
#pragma unroll
    for (int h = 0; h < C8; h++) {
        s_part[warp][g][8 * h + 2 * t] = acc[h][0];
        s_part[warp][g][8 * h + 2 * t + 1] = acc[h][1];
        s_part[warp][g + 8][8 * h + 2 * t] = acc[h][2];
        s_part[warp][g + 8][8 * h + 2 * t + 1] = acc[h][3];
    }
    __syncthreads();
    const int n = threadIdx.x & 15, row = threadIdx.x >> 4;
    if (row < P.m && n0 + n < P.n) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < FR_WARPS; w++) v += s_part[w][n][row];
        const int64_t o = row * P.out_stride + n0 + n;
        if (P.out_bf16) reinterpret_cast<__nv_bfloat16 *>(P.out)[o] = __float2bfloat16_rn(v);
        else reinterpret_cast<float *>(P.out)[o] = v;
    }
}

typedef struct {
    int n_embd, n_inter, n_experts, top_k, has_shared;
    const uint8_t *x;
    int64_t x_stride;
    const float *x_scales;
    int64_t xs_stride;
    const int *ids;
    const float *weights;
    const uint8_t *gate_up, *down;
    const float *gu_scales, *dn_scales;
    uint8_t *act_q; /* [pairs][n_inter] */
    float *act_scales;
    __nv_bfloat16 *out;
    int64_t out_stride;
    int *status;
} fr_experts_t;

/* pair slot j of token t: its expert, or -1 */
__device__ __forceinline__ int fr_expert(const fr_experts_t &P, int t, int j) {
    if (j == P.top_k) return P.n_experts;
    const int e = P.ids[t * P.top_k + j];
    return (unsigned)e < (unsigned)P.n_experts ? e : -1;
}

/* act[pair][128 rows] = silu(gate x) (up x) in FP8; block (128 rows, slot, token) of 16 warps: warp w has rows
 * 16 (w % 8) .. of the 128 and every other block of k, both matrices.  One block holds a whole block of activations, so its
 * amax meets in shared memory; 192 KB an SM are in flight from the start to the end of a block.  (One token with 11 experts of
 * 4096 x 1024: 21 us, 4.3 TB/s from 88 blocks.  Blocks of 64 rows in clusters of two that tell one another their amax, 176 of
 * them: 28 us, two share an SM.) */
#define FG_WARPS 16
#define FG_RING 6
#define FG_SMEM (FG_WARPS * FG_RING * 2048)

__global__ void __launch_bounds__(32 * FG_WARPS) k_f8_few_gate_up(const __grid_constant__ fr_experts_t P) {
    __shared__ __align__(16) float s_part[2][128];
    extern __shared__ __align__(16) uint8_t ring[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3, khalf = warp >> 3;
    const uint32_t ring_u = fb_smem_u32(ring) + warp * (FG_RING * 2048u);
    const int t = blockIdx.z, j = blockIdx.y, n0 = blockIdx.x * 128, r0 = 16 * (warp & 7), H = P.n_embd, I = P.n_inter, kbs = H / 128;
    const int e = fr_expert(P, t, j);
    f8_next(); /* (the down product's weights may be asked for while this one runs) */
    if (e < 0) {
        if (threadIdx.x == 0 && P.ids[t * P.top_k + j] != -1) P.status[OPS_STATUS_WORD(FB_ST_BAD_ID)] = 1;
        return;
    }
    const uint8_t *w0 = P.gate_up + ((int64_t)e * 2 * I + n0 + r0 + g) * H;
    const int64_t up = (int64_t)I * H, low = (int64_t)8 * H;
    const float *gs = P.gu_scales + ((int64_t)e * 2 * (I / 128) + (n0 >> 7)) * kbs, *us = gs + (int64_t)(I / 128) * kbs;
    const uint8_t *x = P.x + t * P.x_stride + 16 * t4;
    const float *xs = P.x_scales + t * P.xs_stride;
    const int its = (kbs - khalf + 1) / 2; /* this warp's blocks of k: khalf, khalf + 2, ... */
    /* units in turn: gate and up of a block of k */
#pragma unroll
    for (int i = 0; i < FG_RING; i++) {
        const uint8_t *r = w0 + (i & 1 ? up : 0);
        if (i / 2 < its) fr_ask(ring_u + i * 2048u, r, r + low, (khalf + 2 * (i / 2)) * 128 + 16 * t4, H);
        fr_commit();
    }
    /* all factors at once, an iteration's in the lane of its number: one latency for them, not one a block */
    float fg[2] = {}, fu[2] = {};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int kb = khalf + 2 * (lane + 32 * h);
        if (kb < kbs) {
            const float sx = __ldg(xs + kb);
            fg[h] = sx * __ldg(gs + kb);
            fu[h] = sx * __ldg(us + kb);
        }
    }
    float acc[2][2] = {}; /* {gate, up} x {row g, row g + 8} (every column holds the same token) */
    int slot = 0;
    uint4 nx0 = __ldg(reinterpret_cast<const uint4 *>(x + min(khalf, kbs - 1) * 128));
    uint4 nx1 = __ldg(reinterpret_cast<const uint4 *>(x + min(khalf, kbs - 1) * 128 + 64));
    for (int it = 0; it < its; it++) {
        const uint4 x0 = nx0, x1 = nx1;
        const int nk = min(khalf + 2 * (it + 1), kbs - 1);
        nx0 = __ldg(reinterpret_cast<const uint4 *>(x + nk * 128));
        nx1 = __ldg(reinterpret_cast<const uint4 *>(x + nk * 128 + 64));
#pragma unroll
        for (int m = 0; m < 2; m++) {
            uint4 w[4];
            float c[4];
            fr_take<FG_RING>(w, ring_u + slot * 2048u);
            fr_block(c, w, x0, x1);
            const float f = __shfl_sync(FULL, m ? (it < 32 ? fu[0] : fu[1]) : (it < 32 ? fg[0] : fg[1]), it & 31);
            acc[m][0] = fmaf(c[0], f, acc[m][0]);
            acc[m][1] = fmaf(c[2], f, acc[m][1]);
            const int next = it + FG_RING / 2;
            const uint8_t *r = w0 + (m ? up : 0);
            if (next < its) fr_ask(ring_u + slot * 2048u, r, r + low, (khalf + 2 * next) * 128 + 16 * t4, H);
            fr_commit();
            slot = slot + 1 == FG_RING ? 0 : slot + 1;
        }
    }
    /* the two halves of k, then the rows of the block */
    if (khalf && t4 == 0) {
        s_part[0][r0 + g] = acc[0][0];
        s_part[0][r0 + g + 8] = acc[0][1];
        s_part[1][r0 + g] = acc[1][0];
        s_part[1][r0 + g + 8] = acc[1][1];
    }
    __syncthreads();
    if (!khalf && t4 == 0) {
        s_part[0][r0 + g] = f8_silu_mul(acc[0][0] + s_part[0][r0 + g], acc[1][0] + s_part[1][r0 + g]);
        s_part[0][r0 + g + 8] = f8_silu_mul(acc[0][1] + s_part[0][r0 + g + 8], acc[1][1] + s_part[1][r0 + g + 8]);
    }
    __syncthreads();
    if (warp == 0) {
        const float4 v = *reinterpret_cast<const float4 *>(&s_part[0][4 * lane]);
        float amax = ops_amax(ops_amax(ops_amax(ops_amax(0.0f, v.x), v.y), v.z), v.w);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) amax = ops_amax(amax, __shfl_xor_sync(FULL, amax, s));
        const float sc = ops_f8_scale(amax), inv = __frcp_rn(sc);
        const int64_t row = (int64_t)t * (P.top_k + P.has_shared) + j;
        *reinterpret_cast<uint32_t *>(P.act_q + row * I + n0 + 4 * lane) =
            ops_f8_pack4(ops_f8_quot(v.x, sc, inv), ops_f8_quot(v.y, sc, inv), ops_f8_quot(v.z, sc, inv), ops_f8_quot(v.w, sc, inv));
        if (lane == 0) P.act_scales[row * (I / 128) + (n0 >> 7)] = sc;
    }
}

/* out[t][16 rows] = sum over the slots of weight (down act); block (rows, token).
 * The warps share the (slot, block of k) units of the token. */
#define FD_RING 6
#define FD_SMEM (FR_WARPS * FD_RING * 2048)
#define FD_SMEM_MOST (FD_SMEM + 96 * 1024) /* with the activations of a token */

__global__ void __launch_bounds__(32 * FR_WARPS) k_f8_few_down(const __grid_constant__ fr_experts_t P) {
    __shared__ float s_part[FR_WARPS][16];
    __shared__ int s_e[OPS_MAX_K + 1];
    extern __shared__ __align__(16) uint8_t ring[]; /* the rings, then the token's activations in FP8, then their scales */
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const uint32_t ring_u = fb_smem_u32(ring) + warp * (FD_RING * 2048u);
    const int t = blockIdx.y, n0 = blockIdx.x * 16, H = P.n_embd, I = P.n_inter, kbs = I / 128;
    const int slots = P.top_k + P.has_shared, units = slots * kbs;
    uint8_t *s_q = ring + FD_SMEM;
    float *s_f = reinterpret_cast<float *>(s_q + slots * I); /* [units]: activation scale x weight scale x slot weight */
    if (threadIdx.x < slots) s_e[threadIdx.x] = fr_expert(P, t, threadIdx.x);
    __syncthreads();
    auto ask = [&](int un, int slot) {
        if (un < units) {
            const int j = un / kbs, kb = un - j * kbs, e = s_e[j];
            const uint8_t *r0 = P.down + ((int64_t)max(e, 0) * H + n0 + g) * I;
            if (e >= 0) fr_ask(ring_u + slot * 2048u, r0, r0 + (int64_t)8 * I, kb * 128 + 16 * t4, I);
        }
        fr_commit();
    };
#pragma unroll
    for (int i = 0; i < FD_RING; i++) ask(warp + FR_WARPS * i, i);
    f8_after(); /* the activations are there */
    /* the token's activations (16 bytes a thread) and each unit's factor */
    const int64_t row0 = (int64_t)t * slots;
    for (int i = threadIdx.x; i < units * 8; i += 32 * FR_WARPS)
        if (s_e[i / (kbs * 8)] >= 0)
            reinterpret_cast<uint4 *>(s_q)[i] = *reinterpret_cast<const uint4 *>(P.act_q + row0 * I + 16 * i);
    for (int un = threadIdx.x; un < units; un += 32 * FR_WARPS) {
        const int j = un / kbs, kb = un - j * kbs, e = s_e[j];
        if (e >= 0)
            s_f[un] = (j < P.top_k ? P.weights[t * P.top_k + j] : 1.0f) * P.act_scales[row0 * kbs + un] *
                      __ldg(P.dn_scales + ((int64_t)e * (H / 128) + (n0 >> 7)) * kbs + kb);
    }
    __syncthreads();
    float acc[2] = {};
    int slot = 0;
    for (int un = warp; un < units; un += FR_WARPS) {
        if (s_e[un / kbs] >= 0) {
            const uint4 x0 = *reinterpret_cast<const uint4 *>(s_q + un * 128 + 16 * t4);
            const uint4 x1 = *reinterpret_cast<const uint4 *>(s_q + un * 128 + 64 + 16 * t4);
            const float f = s_f[un];
            uint4 w[4];
            float c[4];
            fr_take<FD_RING>(w, ring_u + slot * 2048u);
            fr_block(c, w, x0, x1);
            acc[0] = fmaf(c[0], f, acc[0]);
            acc[1] = fmaf(c[2], f, acc[1]);
        } else {
            asm volatile("cp.async.wait_group %0;" ::"n"(FD_RING - 1) : "memory");
        }
        ask(un + FR_WARPS * FD_RING, slot);
        slot = slot + 1 == FD_RING ? 0 : slot + 1;
    }
    if (t4 == 0) {
        s_part[warp][g] = acc[0];
        s_part[warp][g + 8] = acc[1];
    }
    __syncthreads();
    if (threadIdx.x < 16) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < FR_WARPS; w++) v += s_part[w][threadIdx.x];
        P.out[t * P.out_stride + n0 + threadIdx.x] = __float2bfloat16_rn(v);
    }
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

/* most_tiles: no more than this; at_once: tiles that the device works at at the same time */
template <int MODE, int NT, int KIND>
static int f8_launch(f8_args_t &p, int64_t most_tiles, int ranks, int at_once, int *launches, cudaStream_t st) {
    cudaLaunchAttribute at[2] = {};
    int n = 0;
    if (KIND != F8_ONE) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = ranks;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        n++;
    }
    if (MODE != F8_DENSE) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    *launches += 1;
    const dim3 grid((unsigned)((KIND == F8_SPLIT || most_tiles < at_once ? most_tiles : at_once) * ranks));
    return ops_launch(k_f8_mma<MODE, NT, KIND>, grid, F8_THREADS, f8_cfg<MODE, NT, KIND>::SMEM, st, at, n, p);
}

/* Microseconds of a tile: so much a block of k and so much around them, fitted to k of 1024 and 4096 (4096 x 8192 x 4096 by
 * pairs 136 us, by single SMs 144.5; 4096 x 4096 x 1024 29.5 and 28; 64 x 4096 x 4096 in tiles of 256 columns 22, of 128 15.7, of
 * 128 split over 2 SMs 12.7, over 4 10.7; 640 x 4096 x 4096 split over 4, in five waves, 48). */
#define F8_PAIR_US(kb) (0.517 * (kb) + 2.5)
#define F8_256_US(kb) (0.56 * (kb) + 1.8)
#define F8_128_US(kb) (0.33 * (kb) + 2.1)
#define F8_SPLIT_US(kb) (0.33 * (kb) + 4.7)
static double f8_waves(int64_t tiles, int at_once) { return (double)((tiles + at_once - 1) / at_once); }

extern "C" int ops_launch_f8_matmul(const fomoe_b200_f8_matmul_args_t *a, int *status, const ops_device_t *d, int *launches,
                                    void *stream) {
    const int n_sm = d->n_sm;
    if (a->m <= 16) {
        const fr_args_t f = {a->m, a->n, a->k, a->a, a->a_stride, a->a_scales, a->a_scales_stride, a->b, a->b_stride, a->b_scales,
                             a->b_scales_stride, a->out, a->out_type == FOMOE_B200_BF16, a->out_stride};
        const int grid = (a->n + 15) / 16;
        *launches += 1;
        return ops_launch(a->m <= 8 ? k_f8_few<1> : k_f8_few<2>, grid, 32 * FR_WARPS, FR_SMEM, (cudaStream_t)stream, f);
    }
    f8_args_t p = {};
    p.m = a->m, p.n = a->n, p.k = a->k;
    p.a_scales = a->a_scales, p.as_stride = a->a_scales_stride;
    p.b_scales = a->b_scales, p.bs_stride = a->b_scales_stride;
    p.out = a->out, p.out_bf16 = a->out_type == FOMOE_B200_BF16, p.out_stride = a->out_stride;
    const int eb = p.out_bf16 ? 2 : 4;
    const int64_t os = a->out_stride * eb;
    p.out_tma = ((uintptr_t)a->out & 15) == 0 && os % 16 == 0;
    p.status = status;
    cudaStream_t st = (cudaStream_t)stream;
    const int64_t m = a->m, n = a->n, mt = (m + 127) / 128;
    /* Two SMs on 256 x 256 read the least, one on 128 x 256 wastes fewer rows, tiles of 128 columns reach more SMs, and the
     * blocks of k of few tiles are split over the SMs of a cluster: the least of waves x time of a tile. */
    const int64_t kb = (a->k + 127) / 128, pairs = (m + 255) / 256 * ((n + 255) / 256), t256 = mt * ((n + 255) / 256), t128 = mt * ((n + 127) / 128);
    double best = f8_waves(t256, n_sm) * F8_256_US(kb);
    int nt = 256, ranks = 1, pair = 0;
    for (int i = 0, r = 1; i < 4 && r <= kb; i++, r *= 2) {
        if (d->clusters[i] < 1) continue;
        const int64_t part = (kb + r - 1) / r;
        const double c = f8_waves(t128, d->clusters[i]) * (r > 1 ? F8_SPLIT_US(part) : F8_128_US(part));
        if (c < best) best = c, nt = 128, ranks = r;
    }
    if (d->clusters[1] > 0 && f8_waves(pairs, d->clusters[1]) * F8_PAIR_US(kb) < best) pair = 1, nt = 256;
    int rc = f8_map(&p.ta, a->a, a->k, a->m, a->a_stride, 32) | f8_map(&p.tb, a->b, a->k, a->n, a->b_stride, pair ? 128 : nt);
    if (p.out_tma) rc |= f8_map(&p.to, a->out, (uint64_t)a->n * eb, a->m, os, 32);
    if (rc) return rc;
    return pair         ? f8_launch<F8_DENSE, 256, F8_PAIR>(p, pairs, 2, d->clusters[1], launches, st)
           : nt == 256  ? f8_launch<F8_DENSE, 256, F8_ONE>(p, t256, 1, n_sm, launches, st)
           : ranks == 1 ? f8_launch<F8_DENSE, 128, F8_ONE>(p, t128, 1, n_sm, launches, st)
                        : f8_launch<F8_DENSE, 128, F8_SPLIT>(p, t128, ranks, n_sm, launches, st);
}

/* ------------------------------------------------------------------ the pairs' rows of x side by side: one warp a row
 * so that the products' operand tiles are plain boxes (fetching 128 scattered rows as 32 gathers a stage took 2.7
 * thousand cycles a stage, five times the MMAs). */
__global__ void __launch_bounds__(256) k_ops_permute(const uint8_t *x, int64_t x_stride, const float *xs, int64_t xs_stride, int H,
                                                     const int *counts, const int *pairs, int n_routed, int top_k, int n_shared,
                                                     uint8_t *xp, float *xps) {
    const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    f8_next();
    f8_after();
    if (r >= counts[1] + n_shared) return;
    const int p = pairs[r], t = p < n_routed ? p / top_k : p - n_routed;
    const uint4 *src = reinterpret_cast<const uint4 *>(x + t * x_stride);
    uint4 *dst = reinterpret_cast<uint4 *>(xp + (int64_t)r * H);
    for (int i = lane; i < H / 16; i += 32) dst[i] = __ldg(src + i);
    for (int i = lane; i < H / 128; i += 32) xps[(int64_t)r * (H / 128) + i] = __ldg(xs + t * xs_stride + i);
}

/* ------------------------------------------------------------------ out[t] = sum over the slots, in slot order
 * A thread has 8 columns; a token's rows of dots lie where its pairs were bucketed. */
__global__ void __launch_bounds__(256) k_ops_combine(const float *dots, const int *pos, const int *ids, const float *weights,
                                                    int n_embd, int n_experts, int top_k, int n_routed, int has_shared,
                                                    __nv_bfloat16 *out, int64_t out_stride, int vec) {
    const int t = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * 8;
    f8_after();
    if (c >= n_embd) return;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int j = 0; j < top_k + has_shared; j++) {
        const int p = j < top_k ? t * top_k + j : n_routed + t;
        if (j < top_k && (unsigned)ids[p] >= (unsigned)n_experts) continue;
        const float w = j < top_k ? weights[p] : 1.0f;
        const float4 *d = reinterpret_cast<const float4 *>(dots + (int64_t)pos[p] * n_embd + c);
        const float4 a = d[0], b = d[1];
        const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = fmaf(w, x[i], v[i]);
    }
    __nv_bfloat16 *o = out + t * out_stride + c;
    if (vec) {
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            x[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        *reinterpret_cast<uint4 *>(o) = make_uint4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = __float2bfloat16_rn(v[i]);
    }
}

/* Each pair by itself, or bucketed by expert: microseconds of either.  Few pairs stream their experts' weights once a pair, at
 * 5.3 TB/s and with 8 us around it and a block's start a pair; bucketed they are read once an expert, but five kernels and
 * their tiles come first.  (By themselves | bucketed: one token with 11 experts of 4096 x 1024 36 | 57 us, 27 pairs of it
 * 77 | 90, 45 pairs 117 | 101; 2048 x 768, 32 pairs 40 | 59, 64 pairs 65 | 66; 192 pairs in 17 experts of 512 x 256 30 | 24.)
 * How many different experts there will be is known on the device only: the expectation of equally likely ones stands for it. */
static int experts_few(const fomoe_b200_f8_experts_args_t *a, int n_pairs) {
    const double bytes = 3.0 * a->n_embd * a->n_inter, routed = (double)a->n_tokens * a->top_k;
    const double hit = a->n_experts * (1.0 - exp(-routed / a->n_experts)) + (a->has_shared ? 1.0 : 0.0);
    return n_pairs <= 256 && 8.0 + n_pairs * (0.05 + bytes / 5.3e6) <= 22.0 + hit * bytes / 5.5e6;
}

extern "C" void ops_experts_layout(const fomoe_b200_f8_experts_args_t *a, ops_experts_ws_t *w) {
    const uint64_t np = (uint64_t)a->n_tokens * (a->top_k + (a->has_shared ? 1 : 0));
    const uint64_t items = np / 128 + a->n_experts + 1;
    uint64_t at = 0;
#define PART(name, n) w->name = at, at += ((uint64_t)(n) + 255) & ~255ull
    w->n_pairs = (int)np;
    PART(counts, 256 + 16 * items); /* {tiles, routed pairs}, then the tiles */
    PART(block_counts, 4ull * BK_BLOCKS * a->n_experts);
    PART(pairs, 4 * np);
    PART(pos, 4 * np);
    PART(xp, np * a->n_embd);
    PART(xp_scales, np * (a->n_embd / 128) * 4);
    PART(act_q, np * a->n_inter);
    PART(act_scales, np * (a->n_inter / 128) * 4);
    PART(dots, np * a->n_embd * 4);
#undef PART
    w->bytes = at;
}

extern "C" int ops_launch_f8_experts(const fomoe_b200_f8_experts_args_t *a, uint8_t *ws, int *status, const ops_device_t *d,
                                     int *launches, void *stream) {
    const int n_sm = d->n_sm;
    cudaStream_t st = (cudaStream_t)stream;
    ops_experts_ws_t w;
    ops_experts_layout(a, &w);
    const int few_slots = a->top_k + (a->has_shared ? 1 : 0);
    const int few_smem = FD_SMEM + few_slots * a->n_inter + few_slots * (a->n_inter / 128) * 4; /* of the down product */
    if (experts_few(a, w.n_pairs) && few_smem <= FD_SMEM_MOST) {
        const fr_experts_t f = {a->n_embd, a->n_inter, a->n_experts, a->top_k, a->has_shared ? 1 : 0, a->x,
                                a->x_stride, a->x_scales, a->x_scales_stride, a->ids, a->weights, a->gate_up, a->down,
                                a->gate_up_scales, a->down_scales, ws + w.act_q, (float *)(ws + w.act_scales), (__nv_bfloat16 *)a->out, a->out_stride, status};
        const int rc = ops_launch(k_f8_few_gate_up, dim3(a->n_inter / 128, few_slots, a->n_tokens), 32 * FG_WARPS, FG_SMEM, st, f);
        *launches += 2;
        return rc ? rc : f8_launch_after(k_f8_few_down, dim3(a->n_embd / 16, a->n_tokens), 32 * FR_WARPS, few_smem, st, f);
    }
    const int n_routed = a->n_tokens * a->top_k, n_shared = a->has_shared ? a->n_tokens : 0, H = a->n_embd, I = a->n_inter;
    const int64_t recs = a->n_experts + (a->has_shared ? 1 : 0);
    int *counts = (int *)(ws + w.counts), *pairs = (int *)(ws + w.pairs), *pos = (int *)(ws + w.pos);
    int *block_counts = (int *)(ws + w.block_counts);
    int4 *items = (int4 *)(ws + w.counts + 256);
    f8_args_t gu = {}, dn;
    gu.counts = counts, gu.items = items, gu.status = status;
    dn = gu;
    gu.n = I, gu.k = H;
    gu.a_scales = (const float *)(ws + w.xp_scales), gu.as_stride = H / 128;
    gu.b_scales = a->gate_up_scales, gu.bs_stride = H / 128, gu.bs_rec = (int64_t)(2 * I / 128) * (H / 128), gu.b_rec_rows = 2 * I;
    gu.act_q = ws + w.act_q, gu.act_scales = (float *)(ws + w.act_scales);
    dn.n = H, dn.k = I;
    dn.a_scales = gu.act_scales, dn.as_stride = I / 128;
    dn.b_scales = a->down_scales, dn.bs_stride = I / 128, dn.bs_rec = (int64_t)(H / 128) * (I / 128), dn.b_rec_rows = H;
    dn.out = ws + w.dots, dn.out_stride = H, dn.out_tma = 1;
    int rc = f8_map(&gu.ta, ws + w.xp, H, w.n_pairs, H, 32) | f8_map(&gu.tb, a->gate_up, H, recs * 2 * I, H, 128) |
             f8_map(&dn.ta, ws + w.act_q, I, w.n_pairs, I, 32) | f8_map(&dn.tb, a->down, I, recs * H, I, 256) |
             f8_map(&dn.to, ws + w.dots, 4ull * H, w.n_pairs, 4ull * H, 32);
    if (rc) return rc;
    int run = (n_routed + BK_BLOCKS - 1) / BK_BLOCKS;
    run = run < BK_RUN ? BK_RUN : run;
    const int nb = (n_routed + run - 1) / run, bk_smem = a->n_experts * (BK_WARPS + 1) * 4;
    const int *ids = a->ids;
    if (nb > 1) {
        rc = ops_launch(k_ops_bucket<true>, nb, BK_THREADS, bk_smem, st, ids, n_routed, run, a->n_tokens, a->n_experts, a->has_shared,
                        block_counts, counts, pairs, pos, items, status);
        if (!rc)
            rc = f8_launch_after(k_ops_bucket<false>, dim3(nb), BK_THREADS, bk_smem, st, ids, n_routed, run, a->n_tokens, a->n_experts,
                                 a->has_shared, block_counts, counts, pairs, pos, items, status);
        *launches += 1;
    } else {
        rc = ops_launch(k_ops_bucket<false>, nb, BK_THREADS, bk_smem, st, ids, n_routed, run, a->n_tokens, a->n_experts, a->has_shared,
                        block_counts, counts, pairs, pos, items, status);
    }
    if (!rc)
        rc = f8_launch_after(k_ops_permute, dim3((w.n_pairs + 7) / 8), 256, 0, st, a->x, a->x_stride, a->x_scales, a->x_scales_stride, H,
                             (const int *)counts, (const int *)pairs, n_routed, a->top_k, n_shared, ws + w.xp, (float *)(ws + w.xp_scales));
    *launches += 2;
    /* no more tiles than this (the device knows how many there are).  Tiles of 32 rows, with more weights in flight and a
     * joining warp of each warpgroup, were tried for few pairs an expert: 61 tokens of 8 in 256 experts 155 us as with 128;
     * tiles of 256 by pairs of SMs for many: 8192 tokens of 8 + 1 in 64 experts 1.59 ms under the power cap, 1.55 with 128,
     * half a tile of every expert being padding (all of these with an expert's output in fp16, which saves 10 % of the last but
     * rounds what the sum over the experts may cancel). */
    const int64_t tiles = w.n_pairs / 128 + recs;
    if (!rc) rc = f8_launch<F8_GATE_UP, 256, F8_ONE>(gu, tiles * (I / 128), 1, n_sm, launches, st);
    if (!rc) rc = f8_launch<F8_DOWN, 256, F8_ONE>(dn, tiles * ((H + 255) / 256), 1, n_sm, launches, st);
    if (rc) return rc;
    const int vec = ((uintptr_t)a->out & 15) == 0 && (a->n_tokens == 1 || a->out_stride % 8 == 0);
    /* (the grid's y goes to 65535) */
    for (int t0 = 0; t0 < a->n_tokens; t0 += 65535) {
        const int nt = a->n_tokens - t0 < 65535 ? a->n_tokens - t0 : 65535, p0 = t0 * a->top_k;
        rc = f8_launch_after(k_ops_combine, dim3((H / 8 + 255) / 256, nt), 256, 0, st, (const float *)(ws + w.dots),
                             (const int *)pos + p0, ids + p0, a->weights + p0, H, a->n_experts, a->top_k, n_routed + t0 - p0,
                             a->has_shared, (__nv_bfloat16 *)a->out + t0 * a->out_stride, a->out_stride, vec);
        if (rc) return rc;
        *launches += 1;
    }
    return 0;
}

extern "C" int ops_f8_init(ops_device_t *d) {
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
#define RM(MODE, NT, KIND)                                                                                             \
    rc |= (int)cudaFuncSetAttribute((k_f8_mma<MODE, NT, KIND>), cudaFuncAttributeMaxDynamicSharedMemorySize, f8_cfg<MODE, NT, KIND>::SMEM)
    RK(k_ops_combine); RK(k_ops_permute);
#define RF(k, smem) rc |= (int)cudaFuncSetAttribute((k), cudaFuncAttributeMaxDynamicSharedMemorySize, (smem))
    RF(k_f8_few<1>, FR_SMEM); RF(k_f8_few<2>, FR_SMEM); RF(k_f8_few_gate_up, FG_SMEM); RF(k_f8_few_down, FD_SMEM_MOST);
#undef RF
    RM(F8_DENSE, 256, F8_PAIR); RM(F8_DENSE, 256, F8_ONE); RM(F8_DENSE, 128, F8_ONE); RM(F8_DENSE, 128, F8_SPLIT);
    RM(F8_GATE_UP, 256, F8_ONE); RM(F8_DOWN, 256, F8_ONE);
#undef RM
#undef RK
    d->clusters[0] = d->n_sm;
    for (int i = 1; i < 4; i++) {
        cudaLaunchConfig_t c = {};
        cudaLaunchAttribute at[1];
        c.gridDim = dim3(1u << i);
        c.blockDim = dim3(F8_THREADS);
        c.dynamicSmemBytes = f8_cfg<F8_DENSE, 128, F8_SPLIT>::SMEM;
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 1u << i;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        c.attrs = at;
        c.numAttrs = 1;
        rc |= (int)cudaOccupancyMaxActiveClusters(&d->clusters[i], k_f8_mma<F8_DENSE, 128, F8_SPLIT>, &c);
    }
    rc |= (int)cudaFuncSetAttribute(k_ops_bucket<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, OPS_MAX_E * (BK_WARPS + 1) * 4);
    rc |= (int)cudaFuncSetAttribute(k_ops_bucket<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, OPS_MAX_E * (BK_WARPS + 1) * 4);
    return rc;
}
