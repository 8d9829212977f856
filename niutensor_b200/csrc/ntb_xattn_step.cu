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
 * Warps join their sums through shared memory, the CTAs of a cluster (1 to 8, or 16) through
 * distributed shared memory, in a fixed order: one launch, no workspace, no atomics.
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

__device__ __forceinline__ void Mma16816(float * c, const uint32_t * a, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void LdMatrix4(uint32_t * r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void LdMatrix4Trans(uint32_t * r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

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
                const bool rowOk = r < p.rows;
                const int g = rowOk ? r / p.sh.lenQ : 0, i = rowOk ? r - g * p.sh.lenQ : 0;
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
                    /* the reference follows the maximum once it is 8 (in the exponent) behind */
                    if (__any_sync(0xffffffffu, top[0] > m[mt][0] + 8.f || top[1] > m[mt][1] + 8.f)) {
                        float f[2];
#pragma unroll
                        for (int hf = 0; hf < 2; hf++) {
                            const float mNew = fmaxf(m[mt][hf], top[hf]);
                            f[hf] = mNew > m[mt][hf] ? Exp2(m[mt][hf] - mNew) : 1.f;
                            m[mt][hf] = mNew;
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
        const float top = fmaxf(fmaxf(sM[0][r], sM[1][r]), fmaxf(sM[2][r], sM[3][r]));
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        if (top != -INFINITY)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = Exp2(sM[w][r] - top);
                const float4 v = *(const float4 *)(part + (w * MT * 16 + r) * D + c);
                a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
            }
        *(float4 *)(part + r * D + c) = a;
    }
    __syncthreads();
    if (threadIdx.x < rows) {
        const int r = threadIdx.x;
        const float top = fmaxf(fmaxf(sM[0][r], sM[1][r]), fmaxf(sM[2][r], sM[3][r]));
        float t = 0.f;
        if (top != -INFINITY)
            for (int w = 0; w < 4; w++)
                t += Exp2(sM[w][r] - top) * sL[w][r];
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
            if (top != -INFINITY)
                for (int t = 0; t < p.splits; t++) {
                    const float f = Exp2(LoadRemote(MapShared(SmemAddr(&sM[0][r]), t)) - top);
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
        const bool rowLive = iq < nq && top != -INFINITY;
        const float inv = rowLive && total > 0.f ? 1.f / total : 0.f;
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
    /* split the keys until there are about two CTAs an SM, while a part keeps two tiles */
    const long long heads = (long long)s.batch * s.headsKV;
    const int tiles = (s.lenK + ST_KEYS - 1) / ST_KEYS;
    int splits = 1;
    while (splits < 8 && heads * splits < 2LL * ctx.smCount && tiles >= splits * 4)
        splits *= 2;
    p.splits = splits;
    if (heads * splits > 0x7fffffffLL)
        return NTB_ERR_LIMIT;
    const bool two = p.rows > 16;
    if (s.dim <= 64)
        return two ? LaunchStep<64, 2>(call, p, stream) : LaunchStep<64, 1>(call, p, stream);
    return two ? LaunchStep<128, 2>(call, p, stream) : LaunchStep<128, 1>(call, p, stream);
}

}
