/*
 * Attention of a decoder's positions to an encoder's states (half tensors, sm_100a):
 *
 *     out[b, h, i] = sum_j p_ij v[b, h', j],  p_ij = exp(s_ij - lse_i),  s_ij = scale * q_i . k_j,
 *     lse_i = log sum_j exp(s_ij),  j < keyLens[b],  i < queryLens[b],  h' = h / (headsQ / headsKV)
 *
 * in one pass over the keys: with a running reference m somewhat below the row's maximum, every key tile adds
 * exp(s - m) to the row's sum and exp(s - m) v to its accumulator, and both are rescaled when the
 * maximum has grown. It serves the sublayer of the transformer sample's decoder that looks at the
 * encoder's output (source/sample/transformer/submodel/Attention.cpp:188-243 with another length
 * on the key side); the sample pads the sentences of a batch, which the two length vectors describe.
 *
 * XattnKernel (many query rows): a CTA holds one or two 128-row query tiles ("streams") of one key
 * head and walks the key tiles. Warps 0-7 (8-15): softmax of stream 0 (1), two threads a row;
 * then the TMA producer warp and the MMA warp. Scores S = q k^T go to tensor memory, the softmax
 * writes the weights back over them as halves, and the second product takes them from there as its A
 * operand, so neither ever touches shared memory. While one stream is in its softmax the tensor
 * core works for the other. Few query tiles and many keys: the key range is split over a cluster of
 * 2, 4 or 8 CTAs whose partial sums are joined through distributed shared memory in rank order,
 * without a workspace or atomics. Bound by the exponentials and the issue of the products, which a 128 x 128 tile keeps
 * about as long as the tensor core: 4 x 16 heads, 2000 rows, 8192 keys of 128 take 462 us, 1.16 PFLOP/s (537 when the
 * GPU's power limit holds the clock down); 64 x 8 heads, 61 rows, 73 keys of 64 take 12 us, 1.1 TB/s, latency.
 *
 * XattnStepKernel (ntb_xattn_step.cu) takes the calls with at most 32 query rows a key head.
 *
 * Weights are rounded to half for the second product, after a reference is taken off that gives them the upper part of
 * half's range (ntb_xattn.cuh says which); sums, maxima and accumulators
 * are fp32. Waits are bounded as in the matrix-product kernels.
 */
#include "ntb_xattn.cuh"

namespace ntb {

int LaunchXattnStep(const DeviceCtx & ctx, const XattnCall & call, cudaStream_t stream);

namespace {

struct XattnParams {
    XattnShape sh;
    HeadsAddr aQ, aK, aV;
    __half * out;
    ntb_heads_layout lOut;
    float * lse;               /* [batch, headsQ, lenQ], or NULL */
    int tilesPerHead;          /* query tiles of one head */
    int units;                 /* query tiles of one key head: group * tilesPerHead */
    int unitsPerItem;          /* items of one key head: ceil(units / STREAMS) */
    int splits;                /* CTAs of a cluster that share an item's keys */
    int item0;                 /* first item of this launch */
    float scaleLog2;
    int * status;
};

constexpr int EVENTS = 4;         /* barriers of a stream's steps, used in turn: more than the ring's tiles run ahead */

template <int D, int STREAMS> struct XattnSmem {
    static constexpr int DC = D / 64;
    static constexpr int TILE = DC * XBOX_BYTES;
    /* two streams: one CTA per SM, ring as deep as shared memory allows; one stream: two CTAs per SM */
    static constexpr int SLOTS = STREAMS == 2 ? (D == 128 ? 5 : 8) : (D == 128 ? 2 : 4);
    static constexpr int Q_BYTES = STREAMS * TILE;
    static constexpr int RING_BYTES = SLOTS * TILE;
    static constexpr int TOTAL = Q_BYTES + RING_BYTES + 1024;
    static constexpr int THREADS = STREAMS == 2 ? 608 : 320;     /* softmax, producer, issuer; relay with two streams */
    static constexpr int TMEM_COLS = STREAMS == 2 ? 512 : 256;
    static_assert(RING_BYTES >= STREAMS * XT * D * 4, "the split's partial sums take the place of the ring");
};

/* the 256 threads of a stream: whether any of them says so; and a plain barrier */
__device__ __forceinline__ bool StreamAny(int id, bool say)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.aligned.pred p, %2, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(any) : "r"((uint32_t)say), "r"(id) : "memory");
    return any != 0;
}
__device__ __forceinline__ void StreamBarrier(int id) { asm volatile("barrier.cta.sync.aligned %0, 256;" :: "r"(id) : "memory"); }

/* one value from the two threads of every row of a stream, through one word a row */
template <typename Op>
__device__ __forceinline__ float Joint(int s, int hf, volatile float * word, float mine, Op op)
{
    if (hf == 1)
        *word = mine;
    StreamBarrier(1 + s);
    if (hf == 0) {
        mine = op(mine, *word);
        *word = mine;
    }
    StreamBarrier(1 + s);
    if (hf == 1)
        mine = *word;
    return mine;
}

template <int D, int STREAMS>
__global__ void __launch_bounds__(XattnSmem<D, STREAMS>::THREADS, STREAMS == 2 ? 1 : 2)
XattnKernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
            const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const XattnParams p)
{
    using SM = XattnSmem<D, STREAMS>;
    constexpr int DC = SM::DC, TILE = SM::TILE, SLOTS = SM::SLOTS;
    constexpr int TMEM_S = 0, TMEM_O = STREAMS * 128;
    extern __shared__ uint8_t smemRaw[];
    __shared__ __align__(8) uint64_t barFull[SLOTS], barDone[STREAMS][EVENTS], barQ[STREAMS], barS[STREAMS], barP[STREAMS], barO[STREAMS], barFix;
    __shared__ uint32_t tmemBaseSlot;
    __shared__ int abortFlag;
    __shared__ float sHalf[STREAMS][XT];                 /* what the two threads of a row tell each other */
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t smemBase = (SmemAddr(smemRaw) + 1023u) & ~1023u;
    const uint32_t qS = smemBase, ringS = qS + SM::Q_BYTES;
    /* a split item's references and sums, in the place of its queries once those have been read */
    float * sM = (float *)(smemRaw + (smemBase - SmemAddr(smemRaw))), * sL = sM + STREAMS * XT;
    volatile int * abortPtr = &abortFlag;
    constexpr int PRODUCER = STREAMS * 8, ISSUER = STREAMS * 8 + 1, RELAY = STREAMS * 8 + 2;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == PRODUCER && lane == 0) {
        PrefetchTensorMap(&tmQ);
        PrefetchTensorMap(&tmK);
        PrefetchTensorMap(&tmV);
        PrefetchTensorMap(&tmO);
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < SLOTS; i++) {
            MbarInit(SmemAddr(&barFull[i]), 1);
        }
        for (int s = 0; s < STREAMS; s++) {
            for (int i = 0; i < EVENTS; i++)
                MbarInit(SmemAddr(&barDone[s][i]), 1);
            MbarInit(SmemAddr(&barQ[s]), 1);
            MbarInit(SmemAddr(&barS[s]), 1);
            MbarInit(SmemAddr(&barP[s]), STREAMS == 2 ? 9 : 8);            /* the softmax warps and the relay */
            MbarInit(SmemAddr(&barO[s]), 1);
        }
        MbarInit(SmemAddr(&barFix), 1);
        abortFlag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(SmemAddr(&tmemBaseSlot)), "r"((uint32_t)SM::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmemBase = *(volatile uint32_t *)&tmemBaseSlot;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    /* this CTA's item, and its part of the item's keys */
    const int rank = p.splits > 1 ? (int)ClusterRank() : 0;
    const int item = p.item0 + (int)blockIdx.x / p.splits;
    const int headItem = item / p.unitsPerItem;
    const int unit0 = (item - headItem * p.unitsPerItem) * STREAMS;
    const int b = headItem / p.sh.headsKV, kvHead = headItem - b * p.sh.headsKV;
    const int nq = ClampLen(p.sh.queryLens, b, p.sh.lenQ), nk = ClampLen(p.sh.keyLens, b, p.sh.lenK);
    int head[STREAMS], q0[STREAMS];
    bool exists[STREAMS], live[STREAMS];
    bool any = false;
#pragma unroll
    for (int s = 0; s < STREAMS; s++) {
        const int u = unit0 + s;
        const int g = u / p.tilesPerHead;
        exists[s] = u < p.units;
        head[s] = kvHead * p.sh.group + g;
        q0[s] = (u - g * p.tilesPerHead) * XT;
        live[s] = exists[s] && q0[s] < nq;
        any = any || live[s];
    }
    const int keyTiles = any ? (nk + XT - 1) / XT : 0;
    const int perSplit = (keyTiles + p.splits - 1) / p.splits;
    const int tile0 = rank * perSplit < keyTiles ? rank * perSplit : keyTiles;
    const int tile1 = tile0 + perSplit < keyTiles ? tile0 + perSplit : keyTiles;
    const int n = tile1 - tile0;
    /* the last tile reaches past the sequence's keys into rows that exist: their values of v are cleared */
    const bool fix = n > 0 && tile1 * XT > nk && nk < p.sh.lenK;

    /* v of tile j and k of the next have arrived, and the rows of v past the sequence's end are cleared */
    auto CopiesThere = [&](int j) {
        const int iv = 2 * j + 1, ik = iv + 1;
        return MbarWait(SmemAddr(&barFull[iv % SLOTS]), (uint32_t)(iv / SLOTS) & 1u, abortPtr, p.status, 0) &&
               (j + 1 == n || MbarWait(SmemAddr(&barFull[ik % SLOTS]), (uint32_t)(ik / SLOTS) & 1u, abortPtr, p.status, 0)) &&
               (!fix || j + 1 < n || MbarWait(SmemAddr(&barFix), 0, abortPtr, p.status, 0));
    };
    if (warp == PRODUCER) {
        bool ok = true;
        if (lane == 0 && n > 0) {
#pragma unroll
            for (int s = 0; s < STREAMS; s++) {
                if (!live[s])
                    continue;
                MbarExpectTx(SmemAddr(&barQ[s]), TILE);
#pragma unroll
                for (int dc = 0; dc < DC; dc++)
                    TmaLoad4D(qS + s * TILE + dc * XBOX_BYTES, &tmQ, SmemAddr(&barQ[s]), dc * 64, q0[s],
                              head[s] * p.aQ.mulHead, b * p.aQ.mulBatch);
            }
            /* tiles in the order of their use: k 0, v 0, k 1, v 1, ... */
            for (int i = 0; ok && i < 2 * n; i++) {
                /* the slot's last tile, number i - SLOTS (k of tile t or v of tile t - 1), was done with when every stream
                   had its scores of tile t */
                if (i >= SLOTS) {
                    const int t = (i - SLOTS + 1) / 2;
#pragma unroll
                    for (int s = 0; s < STREAMS; s++)
                        if (live[s])
                            ok = ok && MbarWait(SmemAddr(&barDone[s][t % EVENTS]), (uint32_t)(t / EVENTS) & 1u, abortPtr, p.status);
                }
                if (!ok)
                    break;
                const int row = (tile0 + (i >> 1)) * XT;
                const uint32_t dst = ringS + (i % SLOTS) * TILE, bar = SmemAddr(&barFull[i % SLOTS]);
                MbarExpectTx(bar, TILE);
                if ((i & 1) == 0) {
#pragma unroll
                    for (int dc = 0; dc < DC; dc++)
                        TmaLoad4D(dst + dc * XBOX_BYTES, &tmK, bar, dc * 64, row, kvHead * p.aK.mulHead, b * p.aK.mulBatch);
                }
                else {
#pragma unroll
                    for (int dc = 0; dc < DC; dc++)
                        TmaLoad4D(dst + dc * XBOX_BYTES, &tmV, bar, dc * 64, row, kvHead * p.aV.mulHead, b * p.aV.mulBatch);
                }
            }
        }
        __syncwarp();
        if (fix) {
            const int i = 2 * n - 1;
            if (WaitNowWarp(SmemAddr(&barFull[i % SLOTS]), (uint32_t)(i / SLOTS) & 1u, abortPtr, p.status)) {
                ZeroTileRows(ringS + (i % SLOTS) * TILE, DC, nk - (tile1 - 1) * XT, lane);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0)
                    MbarArrive(SmemAddr(&barFix));
            }
        }
    }
    else if (warp == ISSUER) {
        if (lane == 0 && n > 0) {
            constexpr uint32_t descS = XattnDesc(XT, 0), descO = XattnDesc(D, 1);
            auto scores = [&](int s, uint32_t kTile) {
#pragma unroll
                for (int dc = 0; dc < DC; dc++)
#pragma unroll
                    for (int ks = 0; ks < 4; ks++)
                        TcMma<0>(tmemBase + TMEM_S + s * XT,
                                 SmemDesc(qS + s * TILE + dc * XBOX_BYTES + ks * UMMA_K_BYTES, 16, 1024, 2),
                                 SmemDesc(kTile + dc * XBOX_BYTES + ks * UMMA_K_BYTES, 16, 1024, 2), descS, (dc | ks) != 0 ? 1u : 0u);
                TcCommit(SmemAddr(&barS[s]));
            };
            bool ok = WaitNow(SmemAddr(&barFull[0]), 0, abortPtr, p.status);
#pragma unroll
            for (int s = 0; s < STREAMS; s++) {
                if (!live[s])
                    continue;
                ok = ok && WaitNow(SmemAddr(&barQ[s]), 0, abortPtr, p.status);
                if (ok) {
                    TcFenceAfter();
                    scores(s, ringS);
                }
            }
            for (int j = 0; ok && j < n; j++) {
                const int iv = 2 * j + 1, ik = iv + 1;
                const uint32_t vTile = ringS + (iv % SLOTS) * TILE, kTile = ringS + (ik % SLOTS) * TILE;
                /* with a second CTA on the SM the issuing thread has time for these waits (see the relay) */
                if (STREAMS == 1)
                    ok = CopiesThere(j);
#pragma unroll
                for (int s = 0; s < STREAMS; s++) {
                    if (!ok || !live[s])
                        continue;
                    ok = WaitNow(SmemAddr(&barP[s]), (uint32_t)j & 1u, abortPtr, p.status);
                    if (!ok)
                        continue;
                    TcFenceAfter();
                    /* the weights of keys 0-63 and 64-127 lie over the two halves of the scores */
#pragma unroll
                    for (int ks = 0; ks < XT / 16; ks++)
                        TcMmaTmemA(tmemBase + TMEM_O + s * D, tmemBase + TMEM_S + s * XT + (ks >> 2) * 64 + (ks & 3) * 8,
                                   SmemDesc(vTile + ks * 16 * ROW_BYTES, XBOX_BYTES, 1024, 2), descO, (j | ks) != 0 ? 1u : 0u);
                    if (j + 1 < n)
                        scores(s, kTile);
                    else
                        TcCommit(SmemAddr(&barO[s]));
                }
            }
        }
    }
    else if (STREAMS == 2 && warp == RELAY) {
        /* The issuing thread sets the pace of two long streams: behind its own tensor-core instructions it sees a
           barrier only some 300 clocks late, and a second commit behind its instructions takes it 400. So it waits for one
           barrier and commits to one a tile: this thread's arrival says that v of the tile and k of the next are there,
           and a softmax thread tells the producer what has been read. With the issuing thread doing both itself, a step of
           both streams at head size 128 took 3770 clocks, 1200 of them in that. */
        if (lane == 0 && n > 0) {
            bool ok = true;
            for (int j = 0; ok && j < n; j++) {
                ok = CopiesThere(j);
#pragma unroll
                for (int s = 0; s < STREAMS; s++) {
                    if (!live[s])
                        continue;
                    /* not before the tile before has been handed over: its arrival would count there */
                    if (j > 0)
                        ok = ok && MbarWait(SmemAddr(&barP[s]), (uint32_t)(j - 1) & 1u, abortPtr, p.status, 20);
                    if (ok)
                        MbarArrive(SmemAddr(&barP[s]));
                }
            }
        }
    }
    else {
        const int s = STREAMS == 2 ? warp >> 3 : 0, hf = (warp >> 2) & 1, sub = warp & 3;
        const uint32_t laneBase = (uint32_t)(sub * 32) << 16;
        const uint32_t sT = tmemBase + laneBase + TMEM_S + s * XT + hf * 64;
        const uint32_t oT = tmemBase + laneBase + TMEM_O + s * D + hf * (D / 2);
        const int r = sub * 32 + lane;                      /* this thread's row of the tile; its half: keys and columns hf */
        const bool mine = STREAMS == 2 && s == 1 ? live[STREAMS - 1] : live[0];
        const bool there = STREAMS == 2 && s == 1 ? exists[STREAMS - 1] : exists[0];
        const int myHead = STREAMS == 2 && s == 1 ? head[STREAMS - 1] : head[0];
        const int myQ0 = STREAMS == 2 && s == 1 ? q0[STREAMS - 1] : q0[0];
        float m = -INFINITY, l = 0.f;                        /* reference of the exponents (times log2 e), this half's sum */
        const uint64_t scale2 = Pair(p.scaleLog2, p.scaleLog2);
        /* After a wait that ran out the loop goes on with what is there (the next waits return at once): the
           warps of a stream meet at a barrier in every step, which none of them may leave out. */
        bool ok = true;
        if (mine) {
            for (int j = 0; j < n; j++) {
                ok = WaitNowWarp(SmemAddr(&barS[s]), (uint32_t)j & 1u, abortPtr, p.status) && ok;
                /* with these scores the products before them are done, too */
                if ((warp & 7) == 0 && lane == 0)
                    MbarArrive(SmemAddr(&barDone[s][j % EVENTS]));
                TcFenceAfter();
                uint32_t x[64];
                TmemLoad32Async(sT, x);
                TmemLoad32Async(sT + 32, x + 32);
                TmemWaitLoad();
                const int valid = nk - (tile0 + j) * XT - hf * 64;
                if (valid < 64) {
#pragma unroll
                    for (int e = 0; e < 64; e++)
                        x[e] = e < valid ? x[e] : 0xff800000u;
                }
                float m4[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
                for (int e = 0; e < 64; e += 2)
                    m4[(e >> 1) & 3] = fmaxf(fmaxf(m4[(e >> 1) & 3], __uint_as_float(x[e])), __uint_as_float(x[e + 1]));
                const float top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scaleLog2;
                /* Both threads of a row use one reference. It follows the maximum once that is far ahead, which the first
                   tile settles and later ones rarely need. Rows behind the end have no say, and a row's reference moves by
                   its own scores alone, whoever called for the step: its result depends on no other row. */
                if (StreamAny(1 + s, j == 0 || (myQ0 + r < nq && top > m + XATTN_AHEAD))) {
                    const float both = Joint(s, hf, &sHalf[s][r], top, [](float a, float b) { return fmaxf(a, b); });
                    float f = 1.f;
                    if (both > m + XATTN_AHEAD) {
                        f = Exp2(m - (both - XATTN_BELOW));
                        m = both - XATTN_BELOW;
                    }
                    l *= f;
                    if (j > 0) {
                        /* the scores' commit covers the second product before it: the accumulator is current */
#pragma unroll 1
                        for (int c = 0; c < D / 2; c += 8) {      /* few registers: the scores are in the others */
                            uint32_t o[8];
                            TmemLoad8Async(oT + c, o);
                            TmemWaitLoad();
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            TmemStore4Async(oT + c, o);
                            TmemStore4Async(oT + c + 4, o + 4);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
                const uint64_t ref2 = Pair(-ref, -ref);
                uint64_t sum[2] = { 0, 0 };
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint64_t y = Fma2(Pair(__uint_as_float(x[c * 8 + 2 * e]), __uint_as_float(x[c * 8 + 2 * e + 1])), scale2, ref2);
                        float p0, p1;
                        Unpair(y, p0, p1);
                        p0 = Exp2(p0);
                        p1 = Exp2(p1);
                        sum[e & 1] = Add2(sum[e & 1], Pair(p0, p1));
                        w[e] = PackHalf2(p0, p1);
                    }
                    TmemStore4Async(sT + c * 4, w);
                }
                float la, lb;
                Unpair(Add2(sum[0], sum[1]), la, lb);
                l += la + lb;
                TmemWaitStore();
                TcFenceBefore();
                ArriveWarp(SmemAddr(&barP[s]), lane);
            }
            /* the row's sum from its two halves */
            l = Joint(s, hf, &sHalf[s][r], l, [](float a, float b) { return a + b; });
        }
        /* every stream's last product is done: its inputs in shared memory are free again */
#pragma unroll
        for (int t = 0; t < STREAMS; t++)
            if (n > 0 && live[t])
                ok = WaitNowWarp(SmemAddr(&barO[t]), 0, abortPtr, p.status) && ok;
        TcFenceAfter();
        const bool sums = mine && n > 0 && ok;
        const int row = myQ0 + r;
        /* The lengths alone say which rows are empty. In a live row a sum that is NaN or 0 (scores of NaN; all scores minus
           infinity) makes the result NaN, as the formula has it. */
        const bool rowLive = mine && row < nq && n > 0;
        const float inv = 1.f / l;
        if (p.splits > 1 && hf == 0) {
            sM[s * XT + r] = sums ? m : -INFINITY;
            sL[s * XT + r] = sums ? l : 0.f;
        }
        const uint32_t box = qS + s * TILE + sub * 32 * ROW_BYTES, part = ringS + (s * XT + r) * D * 4;
#pragma unroll
        for (int cc = 0; cc < D / 64; cc++) {
            const int c = hf * (D / 64) + cc;                /* of the row's 32-column pieces */
            uint32_t o[32];
            if (sums) {
                TmemLoad32Async(oT + cc * 32, o);
                TmemWaitLoad();
            }
            if (p.splits == 1) {
#pragma unroll
                for (int jj = 0; jj < 4; jj++) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        w[e] = sums && rowLive ? PackHalf2(__uint_as_float(o[jj * 8 + 2 * e]) * inv, __uint_as_float(o[jj * 8 + 2 * e + 1]) * inv) : 0u;
                    const int chunk = (c & 1) * 4 + jj;
                    StoreShared16(box + (c >> 1) * XBOX_BYTES + lane * ROW_BYTES + ((chunk ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
                }
            }
            else {
                /* the partial sums of this CTA's keys, 16-byte chunks of a row permuted by the row's low bits */
#pragma unroll
                for (int jj = 0; jj < 8; jj++)
                    StoreShared16(part + (((c * 8 + jj) ^ (r & 7)) << 4), sums ? o[jj * 4] : 0u, sums ? o[jj * 4 + 1] : 0u,
                                  sums ? o[jj * 4 + 2] : 0u, sums ? o[jj * 4 + 3] : 0u);
            }
        }
        if (p.splits == 1) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            StreamBarrier(1 + s);
            if (there && ok && hf == 0 && lane == 0 && myQ0 + sub * 32 < p.sh.lenQ) {
#pragma unroll
                for (int dc = 0; dc < DC; dc++)
                    TmaStore4D(&tmO, box + dc * XBOX_BYTES, dc * 64, myQ0 + sub * 32, myHead, b);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
            if (there && ok && hf == 0 && p.lse != nullptr && row < p.sh.lenQ)
                p.lse[((long long)b * p.sh.headsQ + myHead) * p.sh.lenQ + row] = rowLive ? (m + log2f(l)) * LN2 : -INFINITY;
        }
        __syncwarp();
    }

    __syncwarp();
    if (*abortPtr) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }
    }
    if (p.splits > 1) {
        ClusterSync();
        if (warp < STREAMS * 8) {
            const int rowsEach = XT / p.splits;
            const int chunks = D / 8;
            for (int i = threadIdx.x; i < STREAMS * rowsEach * chunks; i += STREAMS * 256) {
                const int c = i % chunks, rr = i / chunks;
                const int s = rr / rowsEach, r = rank * rowsEach + (rr - s * rowsEach);
                const bool second = STREAMS == 2 && s == 1;
                const int row = (second ? q0[STREAMS - 1] : q0[0]) + r;
                const int h = second ? head[STREAMS - 1] : head[0];
                if (!(second ? exists[STREAMS - 1] : exists[0]) || row >= p.sh.lenQ)
                    continue;
                float top = -INFINITY;
                for (int t = 0; t < p.splits; t++)
                    top = fmaxf(top, LoadRemote(MapShared(SmemAddr(&sM[s * XT + r]), t)));
                const bool rowLive = row < nq && nk > 0;
                /* A part whose scores are all NaN has a reference of minus infinity and a sum of NaN: weighed by 0 it still
                   makes the total NaN. A part without keys has zeros. */
                const float ref = top == -INFINITY ? 0.f : top;
                float total = 0.f, acc[8] = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };
                if (rowLive) {
                    for (int t = 0; t < p.splits; t++) {
                        const float f = Exp2(LoadRemote(MapShared(SmemAddr(&sM[s * XT + r]), t)) - ref);
                        total += f * LoadRemote(MapShared(SmemAddr(&sL[s * XT + r]), t));
                        const uint32_t base = MapShared(ringS + (s * XT + r) * D * 4, t);
#pragma unroll
                        for (int hf = 0; hf < 2; hf++) {
                            const float4 v = LoadRemote4(base + (((2 * c + hf) ^ (r & 7)) << 4));
                            acc[hf * 4 + 0] += f * v.x; acc[hf * 4 + 1] += f * v.y;
                            acc[hf * 4 + 2] += f * v.z; acc[hf * 4 + 3] += f * v.w;
                        }
                    }
                }
                const float inv = 1.f / total;
                if (c * 8 < p.sh.dim) {
                    uint4 w = make_uint4(0u, 0u, 0u, 0u);
                    if (rowLive)
                        w = make_uint4(PackHalf2(acc[0] * inv, acc[1] * inv), PackHalf2(acc[2] * inv, acc[3] * inv),
                                       PackHalf2(acc[4] * inv, acc[5] * inv), PackHalf2(acc[6] * inv, acc[7] * inv));
                    *(uint4 *)(p.out + b * p.lOut.batch + h * p.lOut.head + row * p.lOut.row + c * 8) = w;
                }
                if (c == 0 && p.lse != nullptr)
                    p.lse[((long long)b * p.sh.headsQ + h) * p.sh.lenQ + row] = rowLive ? (top + log2f(total)) * LN2 : -INFINITY;
            }
        }
        __syncwarp();
        ClusterSync();
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    if (warp == ISSUER)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                     :: "r"(tmemBase), "r"((uint32_t)SM::TMEM_COLS) : "memory");
}

template <int D, int STREAMS>
int LaunchXattn(const DeviceCtx & ctx, const XattnCall & call, const XattnParams & base, int splits, cudaStream_t stream)
{
    XattnParams p = base;
    p.unitsPerItem = (p.units + STREAMS - 1) / STREAMS;
    const long long items = (long long)p.sh.batch * p.sh.headsKV * p.unitsPerItem;
    if (items * splits > 0x7fffffffLL)
        return NTB_ERR_LIMIT;
    CUtensorMap tmQ, tmK, tmV, tmO;
    HeadsAddr unused;
    int rc;
    if ((rc = EncodeHeads(&tmQ, &p.aQ, call.q, p.sh.dim, p.sh.lenQ, p.sh.headsQ, p.sh.batch, call.lQ, XT)) != NTB_OK ||
        (rc = EncodeHeads(&tmO, &unused, call.out, p.sh.dim, p.sh.lenQ, p.sh.headsQ, p.sh.batch, call.lOut, 32)) != NTB_OK)
        return rc;
    tmK = tmV = tmQ;                                    /* without keys neither is read */
    p.aK = p.aV = p.aQ;
    if (p.sh.lenK > 0 &&
        ((rc = EncodeHeads(&tmK, &p.aK, call.k, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.lK, XT)) != NTB_OK ||
         (rc = EncodeHeads(&tmV, &p.aV, call.v, p.sh.dim, p.sh.lenK, p.sh.headsKV, p.sh.batch, call.lV, XT)) != NTB_OK))
        return rc;
    using SM = XattnSmem<D, STREAMS>;
    static SmemOptIn optIn;
    if (!optIn.Ensure((const void *)XattnKernel<D, STREAMS>, SM::TOTAL))
        return NTB_ERR_CUDA;
    /* The items of a last wave that fills at most half of the GPU are split over it, in a launch of their own, when
       they are long: 512 items of 64 key tiles are 3.46 waves and take 3.5 instead of 4. */
    const int slots = STREAMS == 2 ? ctx.smCount : 2 * ctx.smCount;
    const int keyTiles = (p.sh.lenK + XT - 1) / XT;
    long long rest = items % slots;
    int restSplits = splits;
    if (items > slots && splits == 1 && keyTiles >= 24)
        while (restSplits < 8 && rest * restSplits * 2 <= slots && keyTiles >= restSplits * 8)
            restSplits *= 2;
    if (restSplits == splits)
        rest = 0;
    for (int part = 0; part < 2; part++) {
        const long long n = part == 0 ? items - rest : rest;
        if (n == 0)
            continue;
        p.item0 = part == 0 ? 0 : (int)(items - rest);
        p.splits = part == 0 ? splits : restSplits;
        const cudaError_t err = LaunchClusterPdl(XattnKernel<D, STREAMS>, (unsigned)(n * p.splits), SM::THREADS, SM::TOTAL, p.splits, stream,
                                                 tmQ, tmK, tmV, tmO, p);
        CountLaunch();
        if (err != cudaSuccess || cudaGetLastError() != cudaSuccess)
            return NTB_ERR_CUDA;
    }
    return NTB_OK;
}

int DispatchXattn(const DeviceCtx & ctx, const XattnCall & call, cudaStream_t stream)
{
    const XattnShape & s = call.sh;
    if ((long long)s.group * s.lenQ <= XATTN_STEP_ROWS)
        return LaunchXattnStep(ctx, call, stream);
    XattnParams p;
    memset(&p, 0, sizeof(p));
    p.sh = s;
    p.out = (__half *)call.out;
    p.lOut = call.lOut;
    p.lse = call.lse;
    p.tilesPerHead = (s.lenQ + XT - 1) / XT;
    const long long units = (long long)s.group * p.tilesPerHead;
    if (units > 0x7fffffffLL / 2)
        return NTB_ERR_LIMIT;
    p.units = (int)units;
    p.scaleLog2 = call.scale * LOG2E;
    p.status = ctx.status;
    const long long heads = (long long)s.batch * s.headsKV;
    /* Two query tiles to a CTA halve the reads of k and v from L2; below one such CTA per SM, single tiles (two CTAs per
       SM) spread wider. Two / one, us: 4 x 16 heads, 2000 rows, 8192 keys of 128 458 / 490; 1 x 16 heads, 2048 rows and keys
       of 128 54 / 37; 8 x 8 heads, 256 rows, 2048 keys of 64 36 / 22. Over one or two key tiles the rule still takes two where
       it could take one: 64 x 8 heads, 256 rows, 73 and 256 keys of 64 29 / 22 and 34 / 28. */
    const bool two = units >= 2 && heads * ((units + 1) / 2) >= ctx.smCount;
    const long long items = two ? heads * ((units + 1) / 2) : heads * units;
    /* split the keys until the GPU is full, while a part keeps two tiles; and into parts of few enough instructions */
    int splits = 1;
    const int keyTiles = (s.lenK + XT - 1) / XT;
    while (splits < 8 && ((items * splits * 2 <= 2LL * ctx.smCount && keyTiles >= splits * 4) || keyTiles > splits * XATTN_PART_TILES))
        splits *= 2;
    if (s.dim <= 64)
        return two ? LaunchXattn<64, 2>(ctx, call, p, splits, stream) : LaunchXattn<64, 1>(ctx, call, p, splits, stream);
    return two ? LaunchXattn<128, 2>(ctx, call, p, splits, stream) : LaunchXattn<128, 1>(ctx, call, p, splits, stream);
}

}

}

using namespace ntb;

extern "C" int ntb_cross_attention(int devID, void * stream, const void * q, const void * k, const void * v, void * out, float * lse,
                                   int dtype, int batch, int headsQ, int headsKV, int lenQ, int lenK, int dim,
                                   const ntb_heads_layout * layouts, const int * queryLens, const int * keyLens, float scale)
{
    XattnCall call;
    memset(&call, 0, sizeof(call));
    int rc = XattnShapeOf(call.sh, dtype, batch, headsQ, headsKV, lenQ, lenK, dim, queryLens, keyLens, scale);
    if (rc != NTB_OK)
        return rc;
    if (batch == 0 || headsQ == 0 || lenQ == 0)
        return NTB_OK;
    if (!q || !out || !layouts || (lenK > 0 && (!k || !v)))
        return NTB_ERR_ARG;
    call.q = q; call.k = k; call.v = v; call.out = out; call.lse = lse;
    call.lQ = layouts[0]; call.lK = layouts[1]; call.lV = layouts[2]; call.lOut = layouts[3];
    call.scale = scale;
    if (!LayoutOk(q, call.lQ, dim, lenQ, headsQ, batch, true) || !LayoutOk(out, call.lOut, dim, lenQ, headsQ, batch, false) ||
        (lenK > 0 && (!LayoutOk(k, call.lK, dim, lenK, headsKV, batch, true) || !LayoutOk(v, call.lV, dim, lenK, headsKV, batch, true))))
        return NTB_ERR_ARG;
    XattnDevice dev(devID);
    if (!dev.ok)
        return NTB_ERR_CUDA;
    DeviceCtx * ctx = CtxFor(devID);
    if (!ctx)
        return NTB_ERR_CUDA;
    rc = DispatchXattn(*ctx, call, (cudaStream_t)stream);
    if (rc == NTB_ERR_CUDA)
        cudaGetLastError();
    return rc;
}
