/*
 * Cross attention for few query rows: a decoding step's one token a head, the hypotheses of a beam
 * (which share their sentence's encoder states), the query heads that share a key head. The rows of
 * one key head are gathered into one or two 16-row tiles, so that k and v are read once for all of
 * them; the call is bound by those reads.
 *
 * A CTA takes a part of one key head's keys, in tiles of 64 through a ring of TMA copies; each of its
 * four warps works on 16 keys of every tile with mma.sync (16 x 8 x 16: the row count that fits;
 * a tcgen05 tile would be 128 rows, mostly empty, and the tensor pipe is idle most of the time either
 * way). The weights go from the first product's accumulators straight into the second's A operand.
 * Warps join their sums through shared memory, the CTAs of a cluster (1 to 8) through
 * distributed shared memory, in a fixed order: one launch, no workspace, no atomics. 8 x 8 key heads, four query
 * heads each, 16384 keys of 128: 67 us, 403 MB at 6.0 TB/s (93 % of a copy's rate). One sentence's step (8 heads,
 * 23 keys of 64) is 3.2 us on the device, launch and latency.
 *
 * XattnGradStepKernel is the backward pass of such calls (training on short targets): every warp makes dk and dv of
 * its 16 keys whole, from the same registers that give its share of dq, so k and v are read once and their
 * gradients written once, by TMA from the place of the tiles they came in. The weights' transposes are taken in
 * registers (movmatrix). The kernels of ntb_xattn_grad.cu would pad the rows to 128 and read everything twice. Bound
 * by k, v and their gradients where keys are many (20 x 16 heads, 16 rows, 2000 keys of 128: 124 us, 5.3 TB/s), by a
 * CTA's first loads and last sums where they are few (44 x 16 heads, 15 rows, 243 keys of 104: 47 us, 3.2 TB/s).
 */
#include "ntb_xattn.cuh"

namespace ntb {

namespace {

constexpr int ST_KEYS = 64;               /* keys of a tile */
constexpr int ST_BOX = ST_KEYS * ROW_BYTES;
constexpr int ST_THREADS = 160;           /* four working warps and the producer */

struct StepParams {
    XattnShape sh;
    HeadsAddr aK, aV;
    const __half * q;
    __half * out;
    ntb_heads_layout lQ, lOut;
    float * lse;
    int rows;                 /* group * lenQ */
    int splits;
    float scaleLog2;
    int * status;
};

template <int D, int MT> struct StepSmem {
    static constexpr int DC = D / 64;
    static constexpr int TILE = DC * ST_BOX;          /* k or v of one tile */
    static constexpr int STAGES = 3;
    static constexpr int RING_BYTES = STAGES * 2 * TILE;
    static constexpr int PART_BYTES = 4 * MT * 16 * D * 4;       /* the four warps' sums, in the ring's place */
    static constexpr int TOTAL = (RING_BYTES > PART_BYTES ? RING_BYTES : PART_BYTES) + 1024;
};

template <int D, int MT>
__global__ void __launch_bounds__(ST_THREADS)
XattnStepKernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const StepParams p)
{
    using SM = StepSmem<D, MT>;
    constexpr int DC = SM::DC, STAGES = SM::STAGES;
    extern __shared__ uint8_t smemRaw[];
    __shared__ __align__(8) uint64_t barFull[STAGES], barEmpty[STAGES];
    __shared__ int abortFlag;
    __shared__ float sM[4][MT * 16], sL[4][MT * 16];       /* per warp; [0] becomes the CTA's */
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = (SmemAddr(smemRaw) + 1023u) & ~1023u;
    volatile int * abortPtr = &abortFlag;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 128) {
        PrefetchTensorMap(&tmK);
        PrefetchTensorMap(&tmV);
        for (int i = 0; i < STAGES; i++) {
            MbarInit(SmemAddr(&barFull[i]), 1);
            MbarInit(SmemAddr(&barEmpty[i]), 4);
        }
        abortFlag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int rank = p.splits > 1 ? (int)ClusterRank() : 0;
    const int item = (int)blockIdx.x / p.splits;
    const int b = item / p.sh.headsKV, kvHead = item - b * p.sh.headsKV;
    const int nq = ClampLen(p.sh.queryLens, b, p.sh.lenQ);
    const int nk = nq > 0 ? ClampLen(p.sh.keyLens, b, p.sh.lenK) : 0;
    const int tiles = (nk + ST_KEYS - 1) / ST_KEYS;
    const int perSplit = (tiles + p.splits - 1) / p.splits;
    const int tile0 = rank * perSplit < tiles ? rank * perSplit : tiles;
    const int tile1 = tile0 + perSplit < tiles ? tile0 + perSplit : tiles;
    const int n = tile1 - tile0;

    float m[MT][2], l[MT][2];
    float o[MT][D / 8][4];
    if (warp == 4) {
        if (lane == 0) {
            bool ok = true;
            for (int j = 0; ok && j < n; j++) {
                const int st = j % STAGES;
                if (j >= STAGES)
                    ok = MbarWait(SmemAddr(&barEmpty[st]), (uint32_t)(j / STAGES + 1) & 1u, abortPtr, p.status);
                if (!ok)
                    break;
                const uint32_t bar = SmemAddr(&barFull[st]), dst = ring + st * 2 * SM::TILE;
                const int row = (tile0 + j) * ST_KEYS;
                MbarExpectTx(bar, 2 * SM::TILE);
#pragma unroll
                for (int dc = 0; dc < DC; dc++) {
                    TmaLoad4D(dst + dc * ST_BOX, &tmK, bar, dc * 64, row, kvHead * p.aK.mulHead, b * p.aK.mulBatch);
                    TmaLoad4D(dst + SM::TILE + dc * ST_BOX, &tmV, bar, dc * 64, row, kvHead * p.aV.mulHead, b * p.aV.mulBatch);
                }
            }
        }
        __syncwarp();
    }
    else {
        /* the query rows as A fragments: lane holds rows lane / 4 and lane / 4 + 8 of each tile */
        uint32_t qa[MT][D / 16][4];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int r = mt * 16 + hf * 8 + (lane >> 2);
                const int g = r < p.rows ? r / p.sh.lenQ : 0, i = r < p.rows ? r - g * p.sh.lenQ : 0;
                const bool rowOk = r < p.rows && i < nq;               /* rows behind the end are not looked at */
                const __half * src = p.q + b * p.lQ.batch + (kvHead * p.sh.group + g) * p.lQ.head + i * p.lQ.row;
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++)
#pragma unroll
                    for (int part = 0; part < 2; part++) {
                        const int c = ks * 16 + part * 8 + (lane & 3) * 2;
                        qa[mt][ks][part * 2 + hf] = rowOk && c < p.sh.dim ? *(const uint32_t *)(src + c) : 0u;
                    }
            }
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 8; i++)
                o[mt][i][0] = o[mt][i][1] = o[mt][i][2] = o[mt][i][3] = 0.f;
        }
        bool ok = true;
        const int key0 = warp * 16;
        /* ldmatrix addresses: matrix lane / 8, its row lane % 8 */
        const int mat = lane >> 3, mrow = lane & 7;
        const int kRow = key0 + (mat >> 1) * 8 + mrow, kChunk = mat & 1;      /* k: (keys 0-7, d 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15) */
        const int vRow = key0 + (mat & 1) * 8 + mrow, vChunk = mat >> 1;      /* v: (keys 0-7, d 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15) */
        for (int j = 0; j < n; j++) {
            const int st = j % STAGES;
            ok = MbarWaitWarp(SmemAddr(&barFull[st]), (uint32_t)(j / STAGES) & 1u, abortPtr, p.status, 200);
            if (!ok)
                break;
            /* the first lane waited; every lane observes the copy's completion itself before it reads what was copied */
            (void)MbarTryWait(SmemAddr(&barFull[st]), (uint32_t)(j / STAGES) & 1u, 0);
            const uint32_t kT = ring + st * 2 * SM::TILE, vT = kT + SM::TILE;
            const int valid = nk - (tile0 + j) * ST_KEYS - key0;              /* of this warp's 16 keys */
            if (valid > 0) {
                float s[MT][2][4];
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        s[mt][i >> 2][i & 3] = 0.f;
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++) {
                    uint32_t kb[4];
                    LdMatrix4(kb, kT + (ks / 4) * ST_BOX + kRow * ROW_BYTES + ((((ks & 3) * 2 + kChunk) ^ mrow) << 4));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        Mma16816(s[mt][0], qa[mt][ks], kb[0], kb[1]);
                        Mma16816(s[mt][1], qa[mt][ks], kb[2], kb[3]);
                    }
                }
                if (valid < 16) {
#pragma unroll
                    for (int nb = 0; nb < 2; nb++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (nb * 8 + (lane & 3) * 2 + (e & 1) >= valid)
#pragma unroll
                                for (int mt = 0; mt < MT; mt++)
                                    s[mt][nb][e] = -INFINITY;
                    /* values of v past the end of the sequence: cleared, 0 * NaN would reach the sums */
                    for (int i = lane; i < (16 - valid) * 8 * DC; i += 32) {
                        const int dc = i / ((16 - valid) * 8), rest = i - dc * (16 - valid) * 8;
                        StoreShared16(vT + dc * ST_BOX + (key0 + valid) * ROW_BYTES + rest * 16, 0u, 0u, 0u, 0u);
                    }
                    __syncwarp();
                }
                uint32_t pa[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    float top[2];
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        float t = fmaxf(fmaxf(s[mt][0][hf * 2], s[mt][0][hf * 2 + 1]), fmaxf(s[mt][1][hf * 2], s[mt][1][hf * 2 + 1]));
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                        top[hf] = t * p.scaleLog2;
                    }
                    /* the reference follows the maximum once it is far behind, in each row by its own scores alone */
                    if (__any_sync(0xffffffffu, top[0] > m[mt][0] + XATTN_AHEAD || top[1] > m[mt][1] + XATTN_AHEAD)) {
                        float f[2];
#pragma unroll
                        for (int hf = 0; hf < 2; hf++) {
                            f[hf] = 1.f;
                            if (top[hf] > m[mt][hf] + XATTN_AHEAD) {
                                f[hf] = Exp2(m[mt][hf] - (top[hf] - XATTN_BELOW));
                                m[mt][hf] = top[hf] - XATTN_BELOW;
                            }
                            l[mt][hf] *= f[hf];
                        }
#pragma unroll
                        for (int i = 0; i < D / 8; i++) {
                            o[mt][i][0] *= f[0]; o[mt][i][1] *= f[0];
                            o[mt][i][2] *= f[1]; o[mt][i][3] *= f[1];
                        }
                    }
                    float w[2][4];
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        const float ref = m[mt][hf] == -INFINITY ? 0.f : m[mt][hf];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            w[hf][e] = Exp2(fmaf(s[mt][e >> 1][hf * 2 + (e & 1)], p.scaleLog2, -ref));
                            l[mt][hf] += w[hf][e];
                        }
                    }
                    pa[mt][0] = PackHalf2(w[0][0], w[0][1]);
                    pa[mt][1] = PackHalf2(w[1][0], w[1][1]);
                    pa[mt][2] = PackHalf2(w[0][2], w[0][3]);
                    pa[mt][3] = PackHalf2(w[1][2], w[1][3]);
                }
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    uint32_t vb[4];
                    LdMatrix4Trans(vb, vT + (i / 4) * ST_BOX + vRow * ROW_BYTES + ((((i & 3) * 2 + vChunk) ^ mrow) << 4));
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        Mma16816(o[mt][2 * i], pa[mt], vb[0], vb[1]);
                        Mma16816(o[mt][2 * i + 1], pa[mt], vb[2], vb[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0)
                MbarArrive(SmemAddr(&barEmpty[st]));
        }
        /* a row's sum is spread over the four lanes that hold its columns */
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                l[mt][hf] += __shfl_xor_sync(0xffffffffu, l[mt][hf], 1);
                l[mt][hf] += __shfl_xor_sync(0xffffffffu, l[mt][hf], 2);
                if ((lane & 3) == 0) {
                    sM[warp][mt * 16 + hf * 8 + (lane >> 2)] = m[mt][hf];
                    sL[warp][mt * 16 + hf * 8 + (lane >> 2)] = l[mt][hf];
                }
            }
    }
    if (*abortPtr) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }
    }
    __syncthreads();                          /* the ring is idle: every tile loaded was waited for by all four warps */
    float * part = (float *)(smemRaw + (ring - SmemAddr(smemRaw)));       /* [warp][row][D] */
    if (warp < 4) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < D / 8; i++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int r = mt * 16 + hf * 8 + (lane >> 2);
                    *(float2 *)(part + (warp * MT * 16 + r) * D + i * 8 + (lane & 3) * 2) = make_float2(o[mt][i][hf * 2], o[mt][i][hf * 2 + 1]);
                }
    }
    __syncthreads();
    /* the CTA's sums: into warp 0's place (each thread reads and writes its own elements) */
    const int rows = p.rows;
    for (int i = threadIdx.x; i < rows * (D / 4); i += ST_THREADS) {
        const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
        const float top = fmaxf(fmaxf(sM[0][r], sM[1][r]), fmaxf(sM[2][r], sM[3][r])), ref = top == -INFINITY ? 0.f : top;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            /* a warp whose scores are all NaN has a reference of minus infinity and sums of NaN: 0 times those is NaN still */
            const float f = Exp2(sM[w][r] - ref);
            const float4 v = *(const float4 *)(part + (w * MT * 16 + r) * D + c);
            a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
        }
        *(float4 *)(part + r * D + c) = a;
    }
    __syncthreads();
    if (threadIdx.x < rows) {
        const int r = threadIdx.x;
        const float top = fmaxf(fmaxf(sM[0][r], sM[1][r]), fmaxf(sM[2][r], sM[3][r])), ref = top == -INFINITY ? 0.f : top;
        float t = 0.f;
        for (int w = 0; w < 4; w++)
            t += Exp2(sM[w][r] - ref) * sL[w][r];
        sM[0][r] = top;
        sL[0][r] = t;
    }
    if (p.splits > 1)
        ClusterSync();
    else
        __syncthreads();
    /* the item's rows, eight columns a thread, dealt over the cluster's threads */
    const int chunks = D / 8;
    for (int i = rank * ST_THREADS + threadIdx.x; i < rows * chunks; i += p.splits * ST_THREADS) {
        const int r = i / chunks, c = (i - r * chunks) * 8;
        const int g = r / p.sh.lenQ, iq = r - g * p.sh.lenQ, h = kvHead * p.sh.group + g;
        float acc[8], total = 0.f, top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; e++)
            acc[e] = 0.f;
        if (p.splits == 1) {
            top = sM[0][r];
            total = sL[0][r];
#pragma unroll
            for (int e = 0; e < 8; e++)
                acc[e] = part[r * D + c + e];
        }
        else {
            for (int t = 0; t < p.splits; t++)
                top = fmaxf(top, LoadRemote(MapShared(SmemAddr(&sM[0][r]), t)));
            const float ref = top == -INFINITY ? 0.f : top;
            for (int t = 0; t < p.splits; t++) {
                const float f = Exp2(LoadRemote(MapShared(SmemAddr(&sM[0][r]), t)) - ref);
                total += f * LoadRemote(MapShared(SmemAddr(&sL[0][r]), t));
                const uint32_t src = MapShared(ring + (r * D + c) * 4, t);
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const float4 v = LoadRemote4(src + hf * 16);
                    acc[hf * 4 + 0] += f * v.x; acc[hf * 4 + 1] += f * v.y;
                    acc[hf * 4 + 2] += f * v.z; acc[hf * 4 + 3] += f * v.w;
                }
            }
        }
        /* the lengths alone say which rows are empty: a sum of NaN, or of 0 where all scores are minus infinity, makes a live
           row NaN, as the formula has it */
        const bool rowLive = iq < nq && nk > 0;
        const float inv = 1.f / total;
        if (c < p.sh.dim) {
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (rowLive)
                w = make_uint4(PackHalf2(acc[0] * inv, acc[1] * inv), PackHalf2(acc[2] * inv, acc[3] * inv),
                               PackHalf2(acc[4] * inv, acc[5] * inv), PackHalf2(acc[6] * inv, acc[7] * inv));
            *(uint4 *)(p.out + b * p.lOut.batch + h * p.lOut.head + iq * p.lOut.row + c) = w;
        }
        if (c == 0 && p.lse != nullptr)
            p.lse[((long long)b * p.sh.headsQ + h) * p.sh.lenQ + iq] = rowLive ? (top + log2f(total)) * LN2 : -INFINITY;
    }
    if (p.splits > 1)
        ClusterSync();
}

template <int D, int MT>
int LaunchStep(const XattnCall & call, const StepParams & base, cudaStream_t stream)
{
    StepParams p = base;
    CUtensorMap tmK, tmV;
    int rc;
    if (p.sh.lenK > 0) {
        if ((rc = EncodeHeads(&tmK, &p.aK, call.k, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.lK, ST_KEYS)) != NTB_OK ||
            (rc = EncodeHeads(&tmV, &p.aV, call.v, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.lV, ST_KEYS)) != NTB_OK)
            return rc;
    }
    else {
        /* without keys neither map is read */
        if ((rc = EncodeHeads(&tmK, &p.aK, call.q, p.sh.dim, p.sh.lenQ, p.sh.headsQ, p.sh.batch, call.lQ, ST_KEYS)) != NTB_OK)
            return rc;
        tmV = tmK;
    }
    using SM = StepSmem<D, MT>;
    static SmemOptIn optIn;
    if (!optIn.Ensure((const void *)XattnStepKernel<D, MT>, SM::TOTAL))
        return NTB_ERR_CUDA;
    const unsigned grid = (unsigned)((long long)p.sh.batch * p.sh.headsKV * p.splits);
    const cudaError_t err = LaunchClusterPdl(XattnStepKernel<D, MT>, grid, ST_THREADS, SM::TOTAL, p.splits, stream, tmK, tmV, p);
    CountLaunch();
    return (err == cudaSuccess && cudaGetLastError() == cudaSuccess) ? NTB_OK : NTB_ERR_CUDA;
}


/* ---------------------------------------------------------------- gradients */

struct StepGradParams {
    XattnShape sh;
    HeadsAddr aK, aV;
    const __half * q;
    const __half * out;
    const __half * dout;
    __half * dq;
    __half * dk;
    __half * dv;
    ntb_heads_layout lQ, lOut, lDO, lDQ, lDK, lDV;
    const float * lse;
    int rows, splits;
    float scale, scaleLog2;
    int * status;
};

/* Four warps, one of which also starts the loads: a fifth would leave the sub-partition that gets two of them to set
   the registers of all (168 for two CTAs an SM instead of 255). */
constexpr int SG_THREADS = 128;

template <int D, int MT> struct StepGradSmem {
    static constexpr int DC = D / 64;
    static constexpr int ROWS_BYTES = DC * MT * 16 * ROW_BYTES;       /* q, or do */
    static constexpr int TILE = DC * ST_BOX;
    static constexpr int STAGES = 2;
    static constexpr int RESIDENT = 2;
    static constexpr int RING_BYTES = STAGES * 2 * TILE;
    static constexpr int PART_BYTES = 4 * MT * 16 * D * 4;
    static constexpr int TOTAL = 2 * ROWS_BYTES + (RING_BYTES > PART_BYTES ? RING_BYTES : PART_BYTES) + 1024;
};

template <int D, int MT>
__global__ void __launch_bounds__(SG_THREADS, MT == 1 ? 3 : 2)
XattnGradStepKernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDK,
                    const __grid_constant__ CUtensorMap tmDV, const StepGradParams p)
{
    using SM = StepGradSmem<D, MT>;
    constexpr int DC = SM::DC, STAGES = SM::STAGES, R = MT * 16;
    constexpr float P_SCALE = 4096.f, P_SCALE_INV = 1.f / 4096.f;     /* of p in dv's product, as in the kernels for many rows */
    extern __shared__ uint8_t smemRaw[];
    __shared__ __align__(8) uint64_t barFull[STAGES], barEmpty[STAGES];
    __shared__ int abortFlag;
    __shared__ float sDelta[R], sLse[R], sSum[4][R];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (SmemAddr(smemRaw) + 1023u) & ~1023u;
    const uint32_t ring = base, qS = base + (SM::TOTAL - 1024 - 2 * SM::ROWS_BYTES), doS = qS + SM::ROWS_BYTES;
    volatile int * abortPtr = &abortFlag;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        PrefetchTensorMap(&tmK);
        PrefetchTensorMap(&tmV);
        PrefetchTensorMap(&tmDK);
        PrefetchTensorMap(&tmDV);
        for (int i = 0; i < STAGES; i++) {
            MbarInit(SmemAddr(&barFull[i]), 1);
            MbarInit(SmemAddr(&barEmpty[i]), 4);
        }
        abortFlag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int rank = p.splits > 1 ? (int)ClusterRank() : 0;
    const int item = (int)blockIdx.x / p.splits;
    const int b = item / p.sh.headsKV, kvHead = item - b * p.sh.headsKV;
    const int nq = ClampLen(p.sh.queryLens, b, p.sh.lenQ);
    const int nk = nq > 0 ? ClampLen(p.sh.keyLens, b, p.sh.lenK) : 0;
    const int tiles = (nk + ST_KEYS - 1) / ST_KEYS;
    const int perSplit = (tiles + p.splits - 1) / p.splits;
    const int tile0 = rank * perSplit < tiles ? rank * perSplit : tiles;
    const int tile1 = tile0 + perSplit < tiles ? tile0 + perSplit : tiles;
    const int n = tile1 - tile0;
    /* all keys in this CTA's ring: delta from the weights (ntb_xattn_grad.cu says why) */
    const bool resident = tiles <= SM::RESIDENT && p.splits == 1;

    /* the first thread's: tile j into its stage */
    auto load = [&](int j) {
        const int st = j % STAGES, row = (tile0 + j) * ST_KEYS;
        const uint32_t bar = SmemAddr(&barFull[st]), dst = ring + st * 2 * SM::TILE;
        MbarExpectTx(bar, 2 * SM::TILE);
#pragma unroll
        for (int dc = 0; dc < DC; dc++) {
            TmaLoad4D(dst + dc * ST_BOX, &tmK, bar, dc * 64, row, kvHead * p.aK.mulHead, b * p.aK.mulBatch);
            TmaLoad4D(dst + SM::TILE + dc * ST_BOX, &tmV, bar, dc * 64, row, kvHead * p.aV.mulHead, b * p.aV.mulBatch);
        }
    };
    if (threadIdx.x == 0)
        for (int j = 0; j < STAGES && j < n; j++)
            load(j);
    __syncwarp();
    {
        /* the rows of q and do into swizzled tiles, delta and lse beside them */
        for (int r = threadIdx.x >> 3; r < R; r += SG_THREADS / 8) {
            const int part = threadIdx.x & 7;                          /* eight threads a row, 16 bytes each */
            const int g = r / p.sh.lenQ, i = r - g * p.sh.lenQ, h = kvHead * p.sh.group + g;
            const bool live = r < p.rows && i < nq && nk > 0;
            float sum = 0.f;
#pragma unroll
            for (int dc = 0; dc < DC; dc++) {
                const int col = dc * 64 + part * 8;
                uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x, z = x;
                if (live && col < p.sh.dim) {
                    x = *(const uint4 *)(p.q + b * p.lQ.batch + h * p.lQ.head + i * p.lQ.row + col);
                    y = *(const uint4 *)(p.dout + b * p.lDO.batch + h * p.lDO.head + i * p.lDO.row + col);
                    z = *(const uint4 *)(p.out + b * p.lOut.batch + h * p.lOut.head + i * p.lOut.row + col);
                }
                const uint32_t at = dc * R * ROW_BYTES + r * ROW_BYTES + ((part ^ (r & 7)) << 4);
                StoreShared16(qS + at, x.x, x.y, x.z, x.w);
                StoreShared16(doS + at, y.x, y.y, y.z, y.w);
                const uint32_t ys[4] = { y.x, y.y, y.z, y.w }, zs[4] = { z.x, z.y, z.z, z.w };
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 yf = __half22float2(*(const __half2 *)&ys[e]), zf = __half22float2(*(const __half2 *)&zs[e]);
                    sum = fmaf(yf.x, zf.x, sum);
                    sum = fmaf(yf.y, zf.y, sum);
                }
            }
#pragma unroll
            for (int off = 1; off < 8; off <<= 1)
                sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if (part == 0) {
                sDelta[r] = sum;
                /* plus infinity makes every weight of an empty row 0 */
                sLse[r] = live ? p.lse[((long long)b * p.sh.headsQ + h) * p.sh.lenQ + i] * LOG2E : INFINITY;
            }
        }
    }
    __syncthreads();

    float dq[MT][D / 8][4];
    float factor[MT][2];                      /* of each row's ds in this warp's dq (ntb_xattn.cuh) */
    {
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            factor[mt][0] = factor[mt][1] = DS_UNSET;
#pragma unroll
            for (int i = 0; i < D / 8; i++)
                dq[mt][i][0] = dq[mt][i][1] = dq[mt][i][2] = dq[mt][i][3] = 0.f;
        }
        float lse2[MT][2], delta[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                lse2[mt][hf] = sLse[mt * 16 + hf * 8 + (lane >> 2)];
                delta[mt][hf] = sDelta[mt * 16 + hf * 8 + (lane >> 2)];
            }
        bool ok = true;
        const int key0 = warp * 16;
        const int mat = lane >> 3, mrow = lane & 7;
        const int kRow = key0 + (mat >> 1) * 8 + mrow, kChunk = mat & 1;      /* keys as columns: (0-7, d 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15) */
        const int tRow = (mat & 1) * 8 + mrow, tChunk = mat >> 1;             /* 16 rows x 16 columns: (0-7, 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15) */
        /* p and dp of this warp's 16 keys of a tile, keys past the end 0 */
        auto weights = [&](uint32_t kT, uint32_t vT, int valid, float (&w)[MT][2][4], float (&g)[MT][2][4]) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 8; i++)
                    w[mt][i >> 2][i & 3] = g[mt][i >> 2][i & 3] = 0.f;
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++) {
                uint32_t kb[4], vb[4];
                const uint32_t at = (ks / 4) * ST_BOX + kRow * ROW_BYTES + ((((ks & 3) * 2 + kChunk) ^ mrow) << 4);
                LdMatrix4(kb, kT + at);
                LdMatrix4(vb, vT + at);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    uint32_t qa[4], da[4];
                    const uint32_t ra = (ks / 4) * R * ROW_BYTES + (mt * 16 + tRow) * ROW_BYTES + ((((ks & 3) * 2 + tChunk) ^ mrow) << 4);
                    LdMatrix4(qa, qS + ra);
                    LdMatrix4(da, doS + ra);
                    Mma16816(w[mt][0], qa, kb[0], kb[1]);
                    Mma16816(w[mt][1], qa, kb[2], kb[3]);
                    Mma16816(g[mt][0], da, vb[0], vb[1]);
                    Mma16816(g[mt][1], da, vb[2], vb[3]);
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nb = 0; nb < 2; nb++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool in = nb * 8 + (lane & 3) * 2 + (e & 1) < valid;
                        w[mt][nb][e] = in ? Exp2(fmaf(w[mt][nb][e], p.scaleLog2, -lse2[mt][e >> 1])) : 0.f;
                        g[mt][nb][e] = in ? g[mt][nb][e] : 0.f;
                    }
        };
        if (resident) {
            float sum[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
                sum[mt][0] = sum[mt][1] = 0.f;
            for (int j = 0; j < n; j++) {
                ok = MbarWaitWarp(SmemAddr(&barFull[j]), 0, abortPtr, p.status, 200) && ok;
                (void)MbarTryWait(SmemAddr(&barFull[j]), 0, 0);
                const uint32_t kT = ring + j * 2 * SM::TILE;
                float w[MT][2][4], g[MT][2][4];
                weights(kT, kT + SM::TILE, nk - (tile0 + j) * ST_KEYS - key0, w, g);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int nb = 0; nb < 2; nb++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            sum[mt][e >> 1] = fmaf(w[mt][nb][e], g[mt][nb][e], sum[mt][e >> 1]);
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    sum[mt][hf] += __shfl_xor_sync(0xffffffffu, sum[mt][hf], 1);
                    sum[mt][hf] += __shfl_xor_sync(0xffffffffu, sum[mt][hf], 2);
                    if ((lane & 3) == 0)
                        sSum[warp][mt * 16 + hf * 8 + (lane >> 2)] = sum[mt][hf];
                }
            __syncthreads();
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int r = mt * 16 + hf * 8 + (lane >> 2);
                    delta[mt][hf] = (sSum[0][r] + sSum[1][r]) + (sSum[2][r] + sSum[3][r]);
                }
        }
        for (int j = 0; ok && j < n; j++) {
            const int st = j % STAGES;
            if (warp == 0 && j > 0 && j - 1 + STAGES < n) {
                /* the tile before has been left by all: the one STAGES behind it takes its place */
                const int before = j - 1;
                if (lane == 0 && MbarWait(SmemAddr(&barEmpty[before % STAGES]), (uint32_t)(before / STAGES) & 1u, abortPtr, p.status))
                    load(before + STAGES);
                __syncwarp();
            }
            ok = MbarWaitWarp(SmemAddr(&barFull[st]), (uint32_t)(j / STAGES) & 1u, abortPtr, p.status, 200);
            if (!ok)
                break;
            (void)MbarTryWait(SmemAddr(&barFull[st]), (uint32_t)(j / STAGES) & 1u, 0);
            const uint32_t kT = ring + st * 2 * SM::TILE, vT = kT + SM::TILE;
            const int row0 = (tile0 + j) * ST_KEYS + key0, valid = nk - row0;
            if (valid < 16) {
                /* rows of k past the end: 0 * NaN would reach dq */
                const int from = valid > 0 ? valid : 0;
                for (int i = lane; i < (16 - from) * 8 * DC; i += 32) {
                    const int dc = i / ((16 - from) * 8), rest = i - dc * (16 - from) * 8;
                    StoreShared16(kT + dc * ST_BOX + (key0 + from) * ROW_BYTES + rest * 16, 0u, 0u, 0u, 0u);
                }
                __syncwarp();
            }
            float w[MT][2][4], g[MT][2][4];
            weights(kT, vT, valid, w, g);
            /* ds in the place of dp, the largest of each row, and of all */
            float top[MT][2], most = 0.f;
            bool past = false;
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    float t = 0.f;
#pragma unroll
                    for (int nb = 0; nb < 2; nb++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            /* a key past the end stays 0 where delta is not finite */
                            float & d = g[mt][nb][hf * 2 + e];
                            d = nb * 8 + (lane & 3) * 2 + e < valid ? w[mt][nb][hf * 2 + e] * (d - delta[mt][hf]) : 0.f;
                            t = fmaxf(t, fabsf(d));
                        }
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                    top[mt][hf] = t;
                    most = fmaxf(most, t);
                    past = past || DsPast(t, factor[mt][hf]);
                }
            if (__any_sync(0xffffffffu, past)) {
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    float f[2] = { 1.f, 1.f };
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
                        if (DsPast(top[mt][hf], factor[mt][hf])) {
                            const float now = PowerFor(top[mt][hf], DS_TOP);
                            f[hf] = now * PowerInverse(factor[mt][hf]);
                            factor[mt][hf] = now;
                        }
#pragma unroll
                    for (int i = 0; i < D / 8; i++) {
                        dq[mt][i][0] *= f[0]; dq[mt][i][1] *= f[0];
                        dq[mt][i][2] *= f[1]; dq[mt][i][3] *= f[1];
                    }
                }
            }
            /* dk of these keys is made whole here: one factor for the warp's ds, from their largest */
            most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
            const float factorK = most < INFINITY ? PowerFor(most, 14) : 1.f, outK = SumsFactor(PowerInverse(factorK), p.scale);
            /* halves of 2^12 p and of ds: as they are the A operand of dq's product, transposed those of dk's and dv's */
            uint32_t ds[MT][4], dsT[MT][4], pT[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int nb = 0; nb < 2; nb++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        const float da = g[mt][nb][hf * 2], dc = g[mt][nb][hf * 2 + 1];
                        ds[mt][nb * 2 + hf] = PackHalf2(da * factor[mt][hf], dc * factor[mt][hf]);
                        dsT[mt][hf * 2 + nb] = MoveTrans(PackHalf2(da * factorK, dc * factorK));
                        pT[mt][hf * 2 + nb] = MoveTrans(PackHalf2(w[mt][nb][hf * 2] * P_SCALE, w[mt][nb][hf * 2 + 1] * P_SCALE));
                    }
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                uint32_t kb[4];
                LdMatrix4Trans(kb, kT + (i / 4) * ST_BOX + (key0 + tRow) * ROW_BYTES + ((((i & 3) * 2 + tChunk) ^ mrow) << 4));
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    Mma16816(dq[mt][2 * i], ds[mt], kb[0], kb[1]);
                    Mma16816(dq[mt][2 * i + 1], ds[mt], kb[2], kb[3]);
                }
            }
            __syncwarp();
            /* dv and dk of these keys, 16 columns at a time, over the rows of v and k they belong to */
#pragma unroll
            for (int which = 0; which < 2; which++) {
                const uint32_t src = which == 0 ? doS : qS, dst = which == 0 ? vT : kT;
                const float f = which == 0 ? P_SCALE_INV : outK;
#pragma unroll
                for (int i = 0; i < D / 16; i++) {
                    float acc[2][4] = { { 0.f, 0.f, 0.f, 0.f }, { 0.f, 0.f, 0.f, 0.f } };
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        uint32_t rb[4];
                        LdMatrix4Trans(rb, src + (i / 4) * R * ROW_BYTES + (mt * 16 + tRow) * ROW_BYTES + ((((i & 3) * 2 + tChunk) ^ mrow) << 4));
                        Mma16816(acc[0], which == 0 ? pT[mt] : dsT[mt], rb[0], rb[1]);
                        Mma16816(acc[1], which == 0 ? pT[mt] : dsT[mt], rb[2], rb[3]);
                    }
#pragma unroll
                    for (int nb = 0; nb < 2; nb++)
#pragma unroll
                        for (int hf = 0; hf < 2; hf++) {
                            const int r = key0 + hf * 8 + (lane >> 2);
                            const bool live = r - key0 < valid;       /* 0 * inf of q or do is NaN */
                            const uint32_t at = dst + (i / 4) * ST_BOX + r * ROW_BYTES + ((((i & 3) * 2 + nb) ^ (r & 7)) << 4) + (lane & 3) * 4;
                            asm volatile("st.shared.b32 [%0], %1;" :: "r"(at), "r"(live ? PackHalf2(acc[nb][hf * 2] * f, acc[nb][hf * 2 + 1] * f) : 0u) : "memory");
                        }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (row0 < p.sh.lenK) {
#pragma unroll
                    for (int dc = 0; dc < DC; dc++) {
                        TmaStore4D(&tmDK, kT + dc * ST_BOX + key0 * ROW_BYTES, dc * 64, row0, kvHead, b);
                        TmaStore4D(&tmDV, vT + dc * ST_BOX + key0 * ROW_BYTES, dc * 64, row0, kvHead, b);
                    }
                }
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                MbarArrive(SmemAddr(&barEmpty[st]));
            }
            __syncwarp();
        }
    }
    if (*abortPtr) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }
    }
    __syncthreads();                          /* the ring is idle */
    float * part = (float *)(smemRaw + (ring - SmemAddr(smemRaw)));       /* [warp][row][D] */
    {
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int i = 0; i < D / 8; i++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int r = mt * 16 + hf * 8 + (lane >> 2);
                    const float power = PowerInverse(factor[mt][hf]);
                    *(float2 *)(part + (warp * R + r) * D + i * 8 + (lane & 3) * 2) = make_float2(dq[mt][i][hf * 2] * power, dq[mt][i][hf * 2 + 1] * power);
                }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.rows * (D / 4); i += SG_THREADS) {
        const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
        float4 a = *(const float4 *)(part + r * D + c);
#pragma unroll
        for (int w = 1; w < 4; w++) {
            const float4 v = *(const float4 *)(part + (w * R + r) * D + c);
            a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
        }
        *(float4 *)(part + r * D + c) = a;
    }
    if (p.splits > 1)
        ClusterSync();
    else
        __syncthreads();
    const int chunks = D / 8;
    for (int i = rank * SG_THREADS + threadIdx.x; i < p.rows * chunks; i += p.splits * SG_THREADS) {
        const int r = i / chunks, c = (i - r * chunks) * 8;
        const int g = r / p.sh.lenQ, iq = r - g * p.sh.lenQ, h = kvHead * p.sh.group + g;
        if (c >= p.sh.dim)
            continue;
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (iq < nq && nk > 0) {
            float acc[8] = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };
            for (int t = 0; t < p.splits; t++) {
                const uint32_t src = p.splits > 1 ? MapShared(ring + (r * D + c) * 4, t) : 0u;
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const float4 v = p.splits > 1 ? LoadRemote4(src + hf * 16) : *(const float4 *)(part + r * D + c + hf * 4);
                    acc[hf * 4 + 0] += v.x; acc[hf * 4 + 1] += v.y; acc[hf * 4 + 2] += v.z; acc[hf * 4 + 3] += v.w;
                }
            }
            w = make_uint4(PackHalf2(acc[0] * p.scale, acc[1] * p.scale), PackHalf2(acc[2] * p.scale, acc[3] * p.scale),
                           PackHalf2(acc[4] * p.scale, acc[5] * p.scale), PackHalf2(acc[6] * p.scale, acc[7] * p.scale));
        }
        *(uint4 *)(p.dq + b * p.lDQ.batch + h * p.lDQ.head + iq * p.lDQ.row + c) = w;
    }
    /* keys behind the last tile */
    const int behind = tiles * ST_KEYS < p.sh.lenK ? p.sh.lenK - tiles * ST_KEYS : 0, per = p.sh.dim / 8;
    for (long long i = rank * SG_THREADS + threadIdx.x; i < (long long)behind * per; i += p.splits * SG_THREADS) {
        const long long row = tiles * ST_KEYS + i / per;
        const int c = (int)(i % per) * 8;
        *(uint4 *)(p.dk + b * p.lDK.batch + kvHead * p.lDK.head + row * p.lDK.row + c) = make_uint4(0u, 0u, 0u, 0u);
        *(uint4 *)(p.dv + b * p.lDV.batch + kvHead * p.lDV.head + row * p.lDV.row + c) = make_uint4(0u, 0u, 0u, 0u);
    }
    if (p.splits > 1)
        ClusterSync();
}

template <int D, int MT>
int LaunchGradStep(const XattnGradCall & call, const StepGradParams & base, cudaStream_t stream)
{
    StepGradParams p = base;
    CUtensorMap tmK, tmV, tmDK, tmDV;
    HeadsAddr unused;
    int rc;
    if (p.sh.lenK > 0) {
        if ((rc = EncodeHeads(&tmK, &p.aK, call.k, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.l[1], ST_KEYS)) != NTB_OK ||
            (rc = EncodeHeads(&tmV, &p.aV, call.v, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.l[2], ST_KEYS)) != NTB_OK ||
            (rc = EncodeHeads(&tmDK, &unused, call.dk, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.l[6], 16)) != NTB_OK ||
            (rc = EncodeHeads(&tmDV, &unused, call.dv, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.l[7], 16)) != NTB_OK)
            return rc;
    }
    else {
        /* without keys no map is used */
        if ((rc = EncodeHeads(&tmK, &p.aK, call.q, p.sh.dim, p.sh.lenQ, p.sh.headsQ, p.sh.batch, call.l[0], ST_KEYS)) != NTB_OK)
            return rc;
        tmV = tmDK = tmDV = tmK;
    }
    using SM = StepGradSmem<D, MT>;
    static SmemOptIn optIn;
    if (!optIn.Ensure((const void *)XattnGradStepKernel<D, MT>, SM::TOTAL))
        return NTB_ERR_CUDA;
    const unsigned grid = (unsigned)((long long)p.sh.batch * p.sh.headsKV * p.splits);
    const cudaError_t err = LaunchClusterPdl(XattnGradStepKernel<D, MT>, grid, SG_THREADS, SM::TOTAL, p.splits, stream, tmK, tmV, tmDK, tmDV, p);
    CountLaunch();
    return (err == cudaSuccess && cudaGetLastError() == cudaSuccess) ? NTB_OK : NTB_ERR_CUDA;
}

/* split the keys until there are about two CTAs an SM, while a part keeps two tiles; and into parts of few enough
   instructions (one a warp and tile; ntb_xattn.cuh says why) */
constexpr int ST_PART_TILES = XATTN_PART_TILES * XT / 16;
int StepSplits(const DeviceCtx & ctx, const XattnShape & s)
{
    const long long heads = (long long)s.batch * s.headsKV;
    const int tiles = (s.lenK + ST_KEYS - 1) / ST_KEYS;
    int splits = 1;
    while (splits < 8 && ((heads * splits < 2LL * ctx.smCount && tiles >= splits * 4) || tiles > splits * ST_PART_TILES))
        splits *= 2;
    return splits;
}

}

/* Gradients: the parts with the shortest walk in tiles, over the waves that the GPU's places make of them. A CTA's
   rows, first loads and sums cost it about four tiles. (64 x 8 heads) x 16 x 1000 x 128 in two parts takes 111 us, in
   one 121; (20 x 16) x 16 x 2000 x 128 in one 123, in four 137. */
int GradStepSplits(const DeviceCtx & ctx, const XattnShape & s, int places)
{
    const long long heads = (long long)s.batch * s.headsKV;
    const int tiles = (s.lenK + ST_KEYS - 1) / ST_KEYS;
    long long best = 0;
    int splits = 1;
    for (int n = 1; n == 1 || (n <= 8 && tiles >= 2 * n); n *= 2) {
        const long long slots = (long long)places * ctx.smCount;
        const long long cost = (heads * n + slots - 1) / slots * ((tiles + n - 1) / n + 4);
        if (n == 1 || cost < best || tiles > splits * ST_PART_TILES) {
            best = cost;
            splits = n;
        }
    }
    return splits;
}

int LaunchXattnGradStep(const DeviceCtx & ctx, const XattnGradCall & call, cudaStream_t stream)
{
    const XattnShape & s = call.sh;
    StepGradParams p;
    memset(&p, 0, sizeof(p));
    p.sh = s;
    p.q = (const __half *)call.q;
    p.out = (const __half *)call.out;
    p.dout = (const __half *)call.dout;
    p.dq = (__half *)call.dq;
    p.dk = (__half *)call.dk;
    p.dv = (__half *)call.dv;
    p.lQ = call.l[0];
    p.lOut = call.l[3];
    p.lDO = call.l[4];
    p.lDQ = call.l[5];
    p.lDK = call.l[6];
    p.lDV = call.l[7];
    p.lse = call.lse;
    p.rows = s.group * s.lenQ;
    p.scale = call.scale;
    p.scaleLog2 = call.scale * LOG2E;
    p.status = ctx.status;
    p.splits = GradStepSplits(ctx, s, p.rows > 16 ? 2 : 3);
    if ((long long)s.batch * s.headsKV * p.splits > 0x7fffffffLL)
        return NTB_ERR_LIMIT;
    const bool two = p.rows > 16;
    if (s.dim <= 64)
        return two ? LaunchGradStep<64, 2>(call, p, stream) : LaunchGradStep<64, 1>(call, p, stream);
    return two ? LaunchGradStep<128, 2>(call, p, stream) : LaunchGradStep<128, 1>(call, p, stream);
}

int LaunchXattnStep(const DeviceCtx & ctx, const XattnCall & call, cudaStream_t stream)
{
    const XattnShape & s = call.sh;
    StepParams p;
    memset(&p, 0, sizeof(p));
    p.sh = s;
    p.q = (const __half *)call.q;
    p.out = (__half *)call.out;
    p.lQ = call.lQ;
    p.lOut = call.lOut;
    p.lse = call.lse;
    p.rows = s.group * s.lenQ;
    p.scaleLog2 = call.scale * LOG2E;
    p.status = ctx.status;
    p.splits = StepSplits(ctx, s);
    if ((long long)s.batch * s.headsKV * p.splits > 0x7fffffffLL)
        return NTB_ERR_LIMIT;
    const bool two = p.rows > 16;
    if (s.dim <= 64)
        return two ? LaunchStep<64, 2>(call, p, stream) : LaunchStep<64, 1>(call, p, stream);
    return two ? LaunchStep<128, 2>(call, p, stream) : LaunchStep<128, 1>(call, p, stream);
}

}
