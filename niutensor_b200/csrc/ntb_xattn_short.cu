/*
 * Gradients of cross attention (the formulas: ntb_xattn_grad.cu) to a sentence's keys, at most 128 of them. The kernels
 * on 128-row tiles spend such calls on padding and on starting and draining a CTA for every tile, twice. Here one CTA
 * takes a key head whole: its keys stay in shared memory, 16 of them a warp's, and the query rows come in chunks of 32.
 * A warp forms p and ds of its keys with mma.sync and adds to their dv and dk, which stay in its registers to the end;
 * ds goes to shared memory as halves, from which the warps, each with its own rows and columns, form the chunk's
 * dq = ds k. Everything is read once and written once, summed in a fixed order, without atomics or a workspace.
 *
 * The next chunk's rows of q and do travel to registers under the products of this one. delta comes from the weights,
 * as all keys are here (ntb_xattn_grad.cu says what that is good for). Rounding as there: ds, times powers of two (of the
 * query's row for dq, of the warp for dk), and 2^12 p to half, sums in fp32. Bound by the latency of a chunk's four steps, which other CTAs of the SM fill: hence few keys and registers
 * a CTA. 64 x 8 heads, 48 rows, 48 keys of 64: 16.5 us, 22 MB at 1.3 TB/s.
 */
#include "ntb_xattn.cuh"

namespace ntb {

namespace {

constexpr int SH_ROWS = 32;               /* query rows of a chunk */
constexpr int SH_CHUNK = SH_ROWS * ROW_BYTES;

struct ShortParams {
    XattnShape sh;
    HeadsAddr aK, aV;
    const __half * q;
    const __half * dout;
    __half * dq;
    __half * dk;
    __half * dv;
    ntb_heads_layout lQ, lDO, lDQ, lDK, lDV;
    const float * lse;
    float scale, scaleLog2;
    int * status;
};

template <int D, int WARPS> struct ShortSmem {
    static constexpr int DC = D / 64;
    static constexpr int KEYS = 16 * WARPS, THREADS = 32 * WARPS;
    static constexpr int BOX = KEYS * ROW_BYTES, TILE = DC * BOX;
    static constexpr int ROWS_BYTES = DC * SH_CHUNK;      /* q, or do, of a chunk */
    static constexpr int DS_BYTES = KEYS / 64 * SH_CHUNK;
    static constexpr int TOTAL = 2 * TILE + 2 * ROWS_BYTES + DS_BYTES + 1024;
    static constexpr int CTAS = D * WARPS == 256 ? 3 : D * WARPS == 1024 ? 1 : 2;        /* of an SM, by their registers */
};

template <int D, int WARPS>
__global__ void __launch_bounds__(ShortSmem<D, WARPS>::THREADS, ShortSmem<D, WARPS>::CTAS)
XattnGradShortKernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDK,
                     const __grid_constant__ CUtensorMap tmDV, const __grid_constant__ ShortParams p)
{
    using SM = ShortSmem<D, WARPS>;
    constexpr int DC = SM::DC, BOX = SM::BOX;
    constexpr int PASSES = SH_ROWS * 8 / SM::THREADS;     /* eight threads a row of a chunk */
    constexpr float P_SCALE = 4096.f, P_SCALE_INV = 1.f / 4096.f;
    extern __shared__ uint8_t smemRaw[];
    __shared__ __align__(8) uint64_t barFull;
    __shared__ int abortFlag;
    __shared__ float sLse[SH_ROWS], sOut[SH_ROWS];
    __shared__ float2 sSum[WARPS][SH_ROWS];                /* a warp's sum of p dp in a row, and the largest |p dp| */
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (SmemAddr(smemRaw) + 1023u) & ~1023u;
    const uint32_t kT = base, vT = kT + SM::TILE, qS = vT + SM::TILE, doS = qS + SM::ROWS_BYTES, dsS = doS + SM::ROWS_BYTES;
    volatile int * abortPtr = &abortFlag;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        PrefetchTensorMap(&tmK);
        PrefetchTensorMap(&tmV);
        PrefetchTensorMap(&tmDK);
        PrefetchTensorMap(&tmDV);
        MbarInit(SmemAddr(&barFull), 1);
        abortFlag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int b = (int)blockIdx.x / p.sh.headsKV, kvHead = (int)blockIdx.x - b * p.sh.headsKV;
    const int nq = ClampLen(p.sh.queryLens, b, p.sh.lenQ);
    const int nk = nq > 0 ? ClampLen(p.sh.keyLens, b, p.sh.lenK) : 0;
    const int perHead = (nq + SH_ROWS - 1) / SH_ROWS;        /* chunks of a query head */
    const int chunks = nk > 0 ? p.sh.group * perHead : 0;
    if (threadIdx.x == 0 && chunks > 0) {
        const uint32_t bar = SmemAddr(&barFull);
        MbarExpectTx(bar, 2 * SM::TILE);
#pragma unroll
        for (int dc = 0; dc < DC; dc++) {
            TmaLoad4D(kT + dc * BOX, &tmK, bar, dc * 64, 0, kvHead * p.aK.mulHead, b * p.aK.mulBatch);
            TmaLoad4D(vT + dc * BOX, &tmV, bar, dc * 64, 0, kvHead * p.aV.mulHead, b * p.aV.mulBatch);
        }
    }
    __syncwarp();

    /* this thread's pieces of a chunk: rows ahead / 8 of every pass, 16 bytes of each 64 columns */
    uint4 xq[PASSES][DC], xd[PASSES][DC];
    float xl[PASSES];
    const int part = threadIdx.x & 7;
    auto fetch = [&](int c) {
        const int g = c / perHead, i0 = (c - g * perHead) * SH_ROWS, h = kvHead * p.sh.group + g;
#pragma unroll
        for (int ps = 0; ps < PASSES; ps++) {
            const int i = i0 + ps * (SM::THREADS / 8) + (threadIdx.x >> 3);
            xl[ps] = INFINITY;                                 /* makes every weight of an empty row 0 */
            if (part == 0 && i < nq)
                xl[ps] = p.lse[((long long)b * p.sh.headsQ + h) * p.sh.lenQ + i] * LOG2E;
#pragma unroll
            for (int dc = 0; dc < DC; dc++) {
                const int col = dc * 64 + part * 8;
                xq[ps][dc] = xd[ps][dc] = make_uint4(0u, 0u, 0u, 0u);
                if (i < nq && col < p.sh.dim) {
                    xq[ps][dc] = *(const uint4 *)(p.q + b * p.lQ.batch + h * p.lQ.head + i * p.lQ.row + col);
                    xd[ps][dc] = *(const uint4 *)(p.dout + b * p.lDO.batch + h * p.lDO.head + i * p.lDO.row + col);
                }
            }
        }
    };
    auto put = [&]() {
#pragma unroll
        for (int ps = 0; ps < PASSES; ps++) {
            const int r = ps * (SM::THREADS / 8) + (threadIdx.x >> 3);
#pragma unroll
            for (int dc = 0; dc < DC; dc++) {
                const uint32_t at = dc * SH_CHUNK + r * ROW_BYTES + ((part ^ (r & 7)) << 4);
                StoreShared16(qS + at, xq[ps][dc].x, xq[ps][dc].y, xq[ps][dc].z, xq[ps][dc].w);
                StoreShared16(doS + at, xd[ps][dc].x, xd[ps][dc].y, xd[ps][dc].z, xd[ps][dc].w);
            }
            if (part == 0)
                sLse[r] = xl[ps];
        }
    };
    if (chunks > 0) {
        fetch(0);
        put();
    }
    const int key0 = warp * 16;
    const int mat = lane >> 3, mrow = lane & 7;
    const int kRow = key0 + (mat >> 1) * 8 + mrow, kChunk = mat & 1;      /* keys as columns: (0-7, d 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15) */
    const int tRow = (mat & 1) * 8 + mrow, tChunk = mat >> 1;             /* 16 rows x 16 columns: (0-7, 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15) */
    /* this warp's part of a chunk's dq: 16 rows, DQ_COLS columns */
    constexpr int DQ_COLS = D * 2 / WARPS;
    const int dqRow = (warp & 1) * 16, dqCol = (warp >> 1) * DQ_COLS;

    const int valid = nk - key0;                              /* of this warp's keys, if positive */
    const int groups = (nk + 15) / 16;
    /* after a wait that ran out the work goes on with what is there: all warps meet at the barriers below */
    if (chunks > 0) {
        (void)MbarWaitWarp(SmemAddr(&barFull), 0, abortPtr, p.status, 200);
        (void)MbarTryWait(SmemAddr(&barFull), 0, 0);
    }
    if (valid > 0 && valid < 16)
        /* rows of k past the end: 0 * NaN would reach dq */
        for (int i = lane; i < (16 - valid) * 8 * DC; i += 32) {
            const int dc = i / ((16 - valid) * 8), rest = i - dc * (16 - valid) * 8;
            StoreShared16(kT + dc * BOX + (key0 + valid) * ROW_BYTES + rest * 16, 0u, 0u, 0u, 0u);
        }
    float dk[D / 8][4], dv[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            dk[i][e] = dv[i][e] = 0.f;
    float factorK = DS_UNSET;                                 /* of this warp's ds in dk (ntb_xattn.cuh) */

    for (int c = 0; c < chunks; c++) {
        __syncthreads();                                  /* the chunk's rows are there, the last chunk's ds has been read */
        const bool more = c + 1 < chunks;
        if (more)
            fetch(c + 1);
        float w[2][2][4], g[2][2][4];
#pragma unroll
        for (int i = 0; i < 16; i++)
            w[i >> 3][(i >> 2) & 1][i & 3] = g[i >> 3][(i >> 2) & 1][i & 3] = 0.f;
        if (valid > 0) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ks++) {
                uint32_t kb[4], vb[4];
                const uint32_t at = (ks / 4) * BOX + kRow * ROW_BYTES + ((((ks & 3) * 2 + kChunk) ^ mrow) << 4);
                LdMatrix4(kb, kT + at);
                LdMatrix4(vb, vT + at);
#pragma unroll
                for (int mt = 0; mt < 2; mt++) {
                    uint32_t a[4];
                    const uint32_t ra = (ks / 4) * SH_CHUNK + (mt * 16 + tRow) * ROW_BYTES + ((((ks & 3) * 2 + tChunk) ^ mrow) << 4);
                    LdMatrix4(a, qS + ra);
                    Mma16816(w[mt][0], a, kb[0], kb[1]);
                    Mma16816(w[mt][1], a, kb[2], kb[3]);
                    LdMatrix4(a, doS + ra);
                    Mma16816(g[mt][0], a, vb[0], vb[1]);
                    Mma16816(g[mt][1], a, vb[2], vb[3]);
                }
            }
        }
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const float lse2 = sLse[mt * 16 + hf * 8 + (lane >> 2)];
#pragma unroll
                for (int nb = 0; nb < 2; nb++)
#pragma unroll
                    for (int e = hf * 2; e < hf * 2 + 2; e++) {
                        const bool in = nb * 8 + (lane & 3) * 2 + (e & 1) < valid;
                        w[mt][nb][e] = in ? Exp2(fmaf(w[mt][nb][e], p.scaleLog2, -lse2)) : 0.f;
                        g[mt][nb][e] = in ? g[mt][nb][e] : 0.f;
                    }
            }
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                float sum = 0.f, top = 0.f;
#pragma unroll
                for (int nb = 0; nb < 2; nb++)
#pragma unroll
                    for (int e = hf * 2; e < hf * 2 + 2; e++) {
                        sum = fmaf(w[mt][nb][e], g[mt][nb][e], sum);
                        top = fmaxf(top, fabsf(w[mt][nb][e] * g[mt][nb][e]));
                    }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                if ((lane & 3) == 0)
                    sSum[warp][mt * 16 + hf * 8 + (lane >> 2)] = make_float2(sum, top);
            }
        __syncthreads();
        if (valid > 0) {
            /* ds in the place of dp; to shared memory as halves times the row's factor, by a bound of its ds that all warps know:
               the largest p dp and, as p is at most 1, delta */
            float most = 0.f;
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int r = mt * 16 + hf * 8 + (lane >> 2);
                    float delta = 0.f, top = 0.f;         /* the keys' sums, by all threads in the same order */
#pragma unroll
                    for (int k = 0; k < WARPS; k++) {
                        const float2 s = sSum[k][r];
                        delta += s.x;
                        top = fmaxf(top, s.y);
                    }
                    top += fabsf(delta);
                    const float factor = top < INFINITY ? PowerFor(top, 14) : 1.f;
                    if (warp == 0 && (lane & 3) == 0)
                        sOut[r] = SumsFactor(PowerInverse(factor), p.scale);
#pragma unroll
                    for (int nb = 0; nb < 2; nb++) {
                        /* a key past the end stays 0 where delta is not finite */
                        const int key = nb * 8 + (lane & 3) * 2;
                        float & a = g[mt][nb][hf * 2], & d = g[mt][nb][hf * 2 + 1];
                        a = key < valid ? w[mt][nb][hf * 2] * (a - delta) : 0.f;
                        d = key + 1 < valid ? w[mt][nb][hf * 2 + 1] * (d - delta) : 0.f;
                        most = fmaxf(most, fmaxf(fabsf(a), fabsf(d)));
                        const uint32_t at = dsS + (key0 >> 6) * SH_CHUNK + r * ROW_BYTES + (((((key0 & 63) >> 3) + nb) ^ (r & 7)) << 4) + (lane & 3) * 4;
                        asm volatile("st.shared.b32 [%0], %1;" :: "r"(at), "r"(PackHalf2(a * factor, d * factor)) : "memory");
                    }
                }
            most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
            if (DsPast(most, factorK)) {
                const float now = PowerFor(most, DS_TOP), f = now * PowerInverse(factorK);
                factorK = now;
#pragma unroll
                for (int i = 0; i < D / 8; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        dk[i][e] *= f;
            }
            /* halves of 2^12 p and of ds, transposed: the A operands of dv's and dk's products */
            uint32_t dsT[2][4], pT[2][4];
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int nb = 0; nb < 2; nb++) {
                        dsT[mt][hf * 2 + nb] = MoveTrans(PackHalf2(g[mt][nb][hf * 2] * factorK, g[mt][nb][hf * 2 + 1] * factorK));
                        pT[mt][hf * 2 + nb] = MoveTrans(PackHalf2(w[mt][nb][hf * 2] * P_SCALE, w[mt][nb][hf * 2 + 1] * P_SCALE));
                    }
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int mt = 0; mt < 2; mt++) {
                    uint32_t rb[4];
                    const uint32_t at = (i / 4) * SH_CHUNK + (mt * 16 + tRow) * ROW_BYTES + ((((i & 3) * 2 + tChunk) ^ mrow) << 4);
                    LdMatrix4Trans(rb, doS + at);
                    Mma16816(dv[2 * i], pT[mt], rb[0], rb[1]);
                    Mma16816(dv[2 * i + 1], pT[mt], rb[2], rb[3]);
                    LdMatrix4Trans(rb, qS + at);
                    Mma16816(dk[2 * i], dsT[mt], rb[0], rb[1]);
                    Mma16816(dk[2 * i + 1], dsT[mt], rb[2], rb[3]);
                }
        }
        __syncthreads();                                  /* ds is complete, q and do have been read */
        if (more)
            put();
        float dq[DQ_COLS / 8][4];
#pragma unroll
        for (int n = 0; n < DQ_COLS / 8; n++)
            dq[n][0] = dq[n][1] = dq[n][2] = dq[n][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < WARPS; kk++)
            if (kk < groups) {
                uint32_t a[4];
                LdMatrix4(a, dsS + (kk >> 2) * SH_CHUNK + (dqRow + tRow) * ROW_BYTES + ((((kk & 3) * 2 + tChunk) ^ mrow) << 4));
#pragma unroll
                for (int n = 0; n < DQ_COLS / 16; n++) {
                    uint32_t kb[4];
                    const int col = dqCol + n * 16;
                    LdMatrix4Trans(kb, kT + (col >> 6) * BOX + (kk * 16 + tRow) * ROW_BYTES + (((((col & 63) >> 3) + tChunk) ^ mrow) << 4));
                    Mma16816(dq[2 * n], a, kb[0], kb[1]);
                    Mma16816(dq[2 * n + 1], a, kb[2], kb[3]);
                }
            }
        const int gq = c / perHead, quad = lane & 3;
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const int i = (c - gq * perHead) * SH_ROWS + dqRow + hf * 8 + (lane >> 2);
            __half * row = p.dq + b * p.lDQ.batch + (kvHead * p.sh.group + gq) * p.lDQ.head + i * p.lDQ.row + dqCol;
            const float out = sOut[dqRow + hf * 8 + (lane >> 2)];
            uint32_t h[DQ_COLS / 8];
#pragma unroll
            for (int n = 0; n < DQ_COLS / 8; n++)
                h[n] = PackHalf2(dq[n][hf * 2] * out, dq[n][hf * 2 + 1] * out);
            if (DQ_COLS >= 32) {
                /* the four lanes of a row turn their pairs of four blocks of columns into a block of eight columns each */
#pragma unroll
                for (int n0 = 0; n0 < DQ_COLS / 8; n0 += 4) {
                    uint32_t o[4] = { 0u, 0u, 0u, 0u };
#pragma unroll
                    for (int s = 0; s < 4; s++) {
                        const int n = quad ^ s;
                        const uint32_t mine = n == 0 ? h[n0] : n == 1 ? h[n0 + 1] : n == 2 ? h[n0 + 2] : h[n0 + 3];
                        const uint32_t got = __shfl_xor_sync(0xffffffffu, mine, s);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            o[k] = n == k ? got : o[k];
                    }
                    if (i < nq && dqCol + n0 * 8 + quad * 8 < p.sh.dim)
                        *(uint4 *)(row + n0 * 8 + quad * 8) = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
            else {
#pragma unroll
                for (int n = 0; n < DQ_COLS / 8; n++)
                    if (i < nq && dqCol + n * 8 < p.sh.dim)
                        *(uint32_t *)(row + n * 8 + quad * 2) = h[n];
            }
        }
    }
    __syncthreads();                                      /* k has been read by all */
    const float outK = SumsFactor(PowerInverse(factorK), p.scale);
    if (valid > 0) {
        /* dv and dk in the place of v and k, and out */
#pragma unroll
        for (int i = 0; i < D / 8; i++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const int r = key0 + hf * 8 + (lane >> 2);
                const bool live = r - key0 < valid;       /* 0 * inf of q or do is NaN */
                const uint32_t at = (i / 8) * BOX + r * ROW_BYTES + (((i & 7) ^ (r & 7)) << 4) + (lane & 3) * 4;
                asm volatile("st.shared.b32 [%0], %1;" :: "r"(vT + at),
                             "r"(live ? PackHalf2(dv[i][hf * 2] * P_SCALE_INV, dv[i][hf * 2 + 1] * P_SCALE_INV) : 0u) : "memory");
                asm volatile("st.shared.b32 [%0], %1;" :: "r"(kT + at),
                             "r"(live ? PackHalf2(dk[i][hf * 2] * outK, dk[i][hf * 2 + 1] * outK) : 0u) : "memory");
            }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
#pragma unroll
            for (int dc = 0; dc < DC; dc++) {
                TmaStore4D(&tmDK, kT + dc * BOX + key0 * ROW_BYTES, dc * 64, key0, kvHead, b);
                TmaStore4D(&tmDV, vT + dc * BOX + key0 * ROW_BYTES, dc * 64, key0, kvHead, b);
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
        __syncwarp();
    }
    if (*abortPtr) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }
    }
    /* rows behind a sentence, and keys behind the last warp that had any */
    const int per = p.sh.dim / 8, rest = p.sh.lenQ - (chunks > 0 ? nq : 0);
    for (int i = threadIdx.x; i < p.sh.group * rest * per; i += SM::THREADS) {
        const int row = i / per, c = (i - row * per) * 8, g = row / rest, iq = p.sh.lenQ - rest + (row - g * rest);
        *(uint4 *)(p.dq + b * p.lDQ.batch + (kvHead * p.sh.group + g) * p.lDQ.head + iq * p.lDQ.row + c) = make_uint4(0u, 0u, 0u, 0u);
    }
    const int done = chunks > 0 ? groups * 16 : 0;
    for (int i = threadIdx.x; i < (p.sh.lenK - done) * per; i += SM::THREADS) {
        const int row = done + i / per, c = (i % per) * 8;
        *(uint4 *)(p.dk + b * p.lDK.batch + kvHead * p.lDK.head + row * p.lDK.row + c) = make_uint4(0u, 0u, 0u, 0u);
        *(uint4 *)(p.dv + b * p.lDV.batch + kvHead * p.lDV.head + row * p.lDV.row + c) = make_uint4(0u, 0u, 0u, 0u);
    }
}

template <int D, int WARPS>
int LaunchShort(const XattnGradCall & call, const ShortParams & base, cudaStream_t stream)
{
    using SM = ShortSmem<D, WARPS>;
    ShortParams p = base;
    CUtensorMap tmK, tmV, tmDK, tmDV;
    HeadsAddr unused;
    int rc;
    if ((rc = EncodeHeads(&tmK, &p.aK, call.k, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.l[1], SM::KEYS)) != NTB_OK ||
        (rc = EncodeHeads(&tmV, &p.aV, call.v, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.l[2], SM::KEYS)) != NTB_OK ||
        (rc = EncodeHeads(&tmDK, &unused, call.dk, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.l[6], 16)) != NTB_OK ||
        (rc = EncodeHeads(&tmDV, &unused, call.dv, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.l[7], 16)) != NTB_OK)
        return rc;
    static SmemOptIn optIn;
    if (!optIn.Ensure((const void *)XattnGradShortKernel<D, WARPS>, SM::TOTAL))
        return NTB_ERR_CUDA;
    const cudaError_t err = LaunchPdl(XattnGradShortKernel<D, WARPS>, p.sh.batch * p.sh.headsKV, SM::THREADS, SM::TOTAL, stream, tmK, tmV, tmDK, tmDV, p);
    CountLaunch();
    return (err == cudaSuccess && cudaGetLastError() == cudaSuccess) ? NTB_OK : NTB_ERR_CUDA;
}

}

/*
 * Which calls come here, us here / in the kernels they would otherwise go to, head size 64 and 128:
 *   up to 32 rows (otherwise ntb_xattn_step.cu): 64 x 8 heads, 16 rows, 40 keys 10.1 / 11.8 and 15.7 / 18.2; 32 rows,
 *     64 keys 10.6 / 15.9 and 16.5 / 24.5; 8 rows, 128 keys 15.1 / 16.2 and 32 / 24 (that one not). Shared key heads not:
 *     their few rows would be a chunk for every query head;
 *   two chunks (otherwise ntb_xattn_grad.cu): 8 heads, 64 rows, 64 keys 7.4 / 11.4 and 10.6 / 13.1; 64 x 8 heads 18 / 46 and
 *     26 / 53; 100 keys 24 / 47 and 50 / 56;
 *   more, as a CTA takes them one after the other, where the heads fill the GPU: 64 x 4 heads, 200 rows, 64 keys 29 / 40 and
 *     37 / 46, 128 keys 37 / 41 and 72 / 49 (not); 64 heads, 200 rows, 64 keys 21 / 15 (not); 64 x 8 heads, 1000 rows, 128 keys
 *     322 / 267 (not).
 */
bool XattnGradIsShort(const DeviceCtx & ctx, const XattnShape & s)
{
    const long long heads = (long long)s.batch * s.headsKV, rows = (long long)s.group * s.lenQ;
    const long long chunks = (long long)s.group * ((s.lenQ + SH_ROWS - 1) / SH_ROWS);
    if (s.lenQ == 0 || s.lenK == 0 || s.lenK > 128 || heads > 0x7fffffffLL)
        return false;
    const bool cheap = s.dim <= 64 || s.lenK <= 64;
    if (rows <= XATTN_STEP_ROWS)
        return s.group == 1 && (cheap || rows > 16);
    return chunks <= 2 || (chunks <= 16 && cheap && heads * 2 >= ctx.smCount * 3LL);
}

int LaunchXattnGradShort(const DeviceCtx & ctx, const XattnGradCall & call, cudaStream_t stream)
{
    const XattnShape & s = call.sh;
    ShortParams p;
    memset(&p, 0, sizeof(p));
    p.sh = s;
    p.q = (const __half *)call.q;
    p.dout = (const __half *)call.dout;
    p.dq = (__half *)call.dq;
    p.dk = (__half *)call.dk;
    p.dv = (__half *)call.dv;
    p.lQ = call.l[0];
    p.lDO = call.l[4];
    p.lDQ = call.l[5];
    p.lDK = call.l[6];
    p.lDV = call.l[7];
    p.lse = call.lse;
    p.scale = call.scale;
    p.scaleLog2 = call.scale * LOG2E;
    p.status = ctx.status;
    if (s.dim <= 64)
        return s.lenK <= 64 ? LaunchShort<64, 4>(call, p, stream) : LaunchShort<64, 8>(call, p, stream);
    return s.lenK <= 64 ? LaunchShort<128, 4>(call, p, stream) : LaunchShort<128, 8>(call, p, stream);
}

}
