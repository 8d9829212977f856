/*
 * Gradients of cross attention (ntb_xattn.cu), half tensors, sm_100a. With p_ij = exp(s_ij - lse_i)
 * recomputed from the kept lse:
 *
 *     dv_j = sum_i p_ij do_i           dp_ij = do_i . v_j        delta_i = do_i . out_i
 *     ds_ij = p_ij (dp_ij - delta_i)   dq_i = scale sum_j ds_ij k_j   dk_j = scale sum_i ds_ij q_i
 *
 * Calls with few query rows or few keys go to the kernels of ntb_xattn_step.cu and ntb_xattn_short.cu. Here:
 * two kernels, because the sums over j and over i run along different sides of the same score tiles and
 * one kernel for both would have to add to dq with atomics, in an order that changes from run to run:
 *
 * XattnGradQKernel: a CTA owns a 128-row query tile of one head and walks the key tiles: S = q k^T,
 * dP = do v^T, dQ += dS k (three products). It also forms delta and leaves it, with lse, for the other.
 * XattnGradKVKernel: a CTA owns a 128-key tile of one key head and walks the query tiles of all heads
 * that share it (so the gradients of a shared head are summed in tensor memory, in head order):
 * S^T = k q^T, dP^T = v do^T, dV += P^T do, dK += dS^T q (four products).
 *
 * Both: eight warps, two threads a row (64 columns each), a TMA producer warp, an MMA warp. P and dS go
 * back into tensor memory as halves over the tile they came from and are the A operand of the second
 * products. The products of one step run under the exponentials of the next. A relay warp hands the copies on. Tensor memory is full
 * (S, dP and two accumulators of 128 columns at head size 128), so tiles are not double buffered.
 * Few tiles: the walk is split over a cluster of up to 8 CTAs, joined in rank order through
 * distributed shared memory.
 *
 * Bound by the steps' products and the shared memory that feeds them, on long walks (2 x 16 query and 4 key heads,
 * 1777 rows, 4100 keys of 128: 432 us, 298 GFLOP of the formulas' five products, 418 of the seven done, 0.97 PFLOP/s;
 * a step takes some 2700 clocks in the first kernel and 3300 in the second), by the loads before an item's first
 * product and the stores behind its last on short ones (64 x 4 heads, 100 to 200 rows and keys of 128: 65 us).
 *
 * What a CTA runs once (the rows' way to tensor memory, the results' out of it) is kept in loops: unrolled, its
 * instructions came from L2 for every tile, 0.5 to 1 us of the 8 a short item takes (sentences 69.4 -> 65.2 us).
 *
 * Rounding: p is at most 1 and may be tiny (1 / lenK); for dv it is rounded to half as 2^12 p, exact powers
 * of two away from half's subnormals. ds is rounded to half times a power of two (ntb_xattn.cuh says why). In the first
 * kernel that is a row's and follows the row's largest ds as the walk goes on: a vote of the softmax threads in every step,
 * and where one of them calls for it, the accumulators scaled. The second kernel has one for all ds of a key head, from the
 * largest that the first has met: its exponent, a bit each, takes the place of the low bits of eight rows' delta (2^-23 of
 * delta, whose fp32 sum is off by more). A ds of the second kernel past that largest is the rounding of scores and dp, where
 * they cancel: it saturates. With a vote in the second kernel, too, documents took 467 us instead of 434. Sums are fp32.
 */
#include "ntb_xattn.cuh"

namespace ntb {

int LaunchXattnGradStep(const DeviceCtx & ctx, const XattnGradCall & call, cudaStream_t stream);
bool XattnGradIsShort(const DeviceCtx & ctx, const XattnShape & s);
int LaunchXattnGradShort(const DeviceCtx & ctx, const XattnGradCall & call, cudaStream_t stream);

namespace {

constexpr int GR_THREADS = 352;
constexpr int GR_PRODUCER = 8, GR_ISSUER = 9, GR_RELAY = 10;
constexpr int GR_EVENTS = 8;       /* barriers of the first kernel's steps, used in turn: more than the ring runs ahead */
constexpr float P_SCALE_LOG2 = 12.f, P_SCALE_INV = 1.f / 4096.f;

struct XattnGradParams {
    XattnShape sh;
    HeadsAddr aQ, aK, aV, aO, aDO;
    const float * lse;
    float * work;              /* [batch, headsQ, tilesPerHead][2][128]: lse and minus delta in the second kernel's units */
    int tilesPerHead, keyTiles;
    int splits, item0;         /* of this launch */
    float scale, scaleLog2;
    int * status;
    /* the destinations of the split form */
    __half * d0;               /* dq, or dk */
    __half * d1;               /* dv */
    ntb_heads_layout l0, l1;
};

template <int D> struct XattnGradSmem {
    static constexpr int DC = D / 64;
    static constexpr int TILE = DC * XBOX_BYTES;
    /* first kernel: a ring of k and v tiles (q and do are in tensor memory) */
    static constexpr int SLOTS = 7;
    static constexpr int Q_TOTAL = SLOTS * TILE + 1024;
    /* second kernel: k, v, rings of q, of do, and of the query rows' (lse, delta); barriers */
    static constexpr int QSLOTS = 3, DOSLOTS = 2, STATSLOTS = 2, STAT = 2 * XT * 4;
    static constexpr int KV_RING = 2 * TILE, KV_STATS = KV_RING + (QSLOTS + DOSLOTS) * TILE, KV_BARS = KV_STATS + STATSLOTS * STAT;
    static constexpr int KV_TOTAL = KV_BARS + 256;
    static_assert(SLOTS * TILE >= XT * D * 4 && (QSLOTS + DOSLOTS) * TILE >= 2 * XT * D * 4, "the split's partial sums take the place of the rings");
    static_assert(KV_TOTAL <= 232448, "shared memory of a CTA");
};

__device__ __forceinline__ void GradBarrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool GradAny(bool say)
{
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.aligned.pred p, 1, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(any) : "r"((uint32_t)say) : "memory");
    return any != 0;
}

/* 32 columns of a thread's ds as halves */
__device__ __forceinline__ void PackDs(uint32_t dsT, const uint32_t * ds)
{
    uint32_t w[16];
#pragma unroll
    for (int e = 0; e < 16; e++)
        w[e] = PackHalf2(__uint_as_float(ds[2 * e]), __uint_as_float(ds[2 * e + 1]));
    TmemStore16Async(dsT, w);
}
__device__ __forceinline__ float LargestDs(const uint32_t * ds)
{
    float m[4] = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
    for (int e = 0; e < 32; e += 2)
        m[(e >> 1) & 3] = fmaxf(fmaxf(m[(e >> 1) & 3], fabsf(__uint_as_float(ds[e]))), fabsf(__uint_as_float(ds[e + 1])));
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

/*
 * The end of a step's ds: one thread has 64 columns of its row, times the row's factor (in the first step 1), in
 * registers, of which the largest is `top`. Behind the first step they are in tensor memory already, and all threads vote
 * on whether some live row's are too large. If so, and in the first step, the two threads of a row settle on a factor,
 * scale the row's sums of the steps before, half of the columns each, and store their ds again. All 256 threads call;
 * word: one a row, in shared memory.
 */
template <int D>
__device__ __forceinline__ void SettleDs(uint32_t * ds, float top, float & factor, bool rowLive, bool first, int hf, volatile float * word,
                                         uint32_t dsT, uint32_t accT)
{
    if (first || GradAny(rowLive && DsPast(top, 1.f))) {
        if (hf == 1)
            *word = top;
        GradBarrier();
        if (hf == 0) {
            top = fmaxf(top, *word);
            *word = top;
        }
        GradBarrier();
        top = *word;
        const float f = first ? (top < INFINITY ? PowerFor(top, DS_TOP) : 1.f) : DsPast(top, 1.f) ? PowerFor(top, DS_TOP) : 1.f;
        factor *= f;
        if (!first) {
            TmemWaitStore();
#pragma unroll 1
            for (int c = hf * (D / 2); c < (hf + 1) * (D / 2); c += 8) {
                uint32_t o[8];
                TmemLoad8Async(accT + c, o);
                TmemWaitLoad();
#pragma unroll
                for (int e = 0; e < 8; e++)
                    o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                TmemStore4Async(accT + c, o);
                TmemStore4Async(accT + c + 4, o + 4);
            }
        }
#pragma unroll
        for (int e = 0; e < 64; e++)
            ds[e] = __float_as_uint(__uint_as_float(ds[e]) * f);
        PackDs(dsT, ds);
        PackDs(dsT + 16, ds + 32);
    }
    TmemWaitStore();
}

/* one thread's 32 accumulator columns times a power of two into its row of a split's partial sums, 16-byte chunks permuted
   by the row */
__device__ __forceinline__ void StorePartial(uint32_t rowBase, int r, int chunk0, const uint32_t * o, float power, bool have)
{
#pragma unroll
    for (int jj = 0; jj < 8; jj++) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            w[e] = have ? __float_as_uint(__uint_as_float(o[jj * 4 + e]) * power) : 0u;
        StoreShared16(rowBase + (((chunk0 + jj) ^ (r & 7)) << 4), w[0], w[1], w[2], w[3]);
    }
}

/* eight columns of a row summed over the cluster in rank order */
__device__ __forceinline__ uint4 SumPartials(uint32_t rowBase, int r, int c, int splits, float factor)
{
    float acc[8] = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };
    for (int t = 0; t < splits; t++) {
        const uint32_t base = MapShared(rowBase, t);
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const float4 v = LoadRemote4(base + (((2 * c + hf) ^ (r & 7)) << 4));
            acc[hf * 4 + 0] += v.x; acc[hf * 4 + 1] += v.y; acc[hf * 4 + 2] += v.z; acc[hf * 4 + 3] += v.w;
        }
    }
    return make_uint4(PackHalf2(acc[0] * factor, acc[1] * factor), PackHalf2(acc[2] * factor, acc[3] * factor),
                      PackHalf2(acc[4] * factor, acc[5] * factor), PackHalf2(acc[6] * factor, acc[7] * factor));
}

/* 64 columns of this thread's lane */
__device__ __forceinline__ void TmemLoad64U(uint32_t taddr, uint32_t * x)
{
    TmemLoad32Async(taddr, x);
    TmemLoad32Async(taddr + 32, x + 32);
    TmemWaitLoad();
}

/* 32 columns of this thread's lane, scaled, into four 16-byte chunks of its row of a swizzled box */
__device__ __forceinline__ void StageHalf32(uint32_t rowAddr, int lane, int chunk0, const uint32_t * o, float f, bool have)
{
#pragma unroll
    for (int jj = 0; jj < 4; jj++) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            w[e] = have ? PackHalf2(__uint_as_float(o[jj * 8 + 2 * e]) * f, __uint_as_float(o[jj * 8 + 2 * e + 1]) * f) : 0u;
        StoreShared16(rowAddr + (((chunk0 + jj) ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
    }
}

template <int D>
__global__ void __launch_bounds__(GR_THREADS, 1)
XattnGradQKernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmDO, const __grid_constant__ CUtensorMap tmDQ,
                 const XattnGradParams p)
{
    using SM = XattnGradSmem<D>;
    constexpr int DC = SM::DC, TILE = SM::TILE, SLOTS = SM::SLOTS;
    constexpr int TMEM_S = 0, TMEM_DP = 128, TMEM_DQ = 256, TMEM_Q = 256 + D, TMEM_DO = TMEM_Q + D / 2;
    constexpr int ROWS0 = SLOTS - 3;                         /* slots of the rows of q, do and out before the ring needs them */
    extern __shared__ uint8_t smemRaw[];
    __shared__ __align__(8) uint64_t barFull[SLOTS], barEvent[GR_EVENTS], barRows, barQ, barS, barSRead, barDP, barDS, barDone, barFix;
    __shared__ uint32_t tmemBaseSlot;
    __shared__ int abortFlag;
    __shared__ float sDelta[XT], sMost[8];

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t smemBase = (SmemAddr(smemRaw) + 1023u) & ~1023u;
    const uint32_t ringS = smemBase, outS = ringS;          /* dq is staged where the ring was */
    volatile int * abortPtr = &abortFlag;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == GR_PRODUCER && lane == 0) {
        PrefetchTensorMap(&tmQ);
        PrefetchTensorMap(&tmO);
        PrefetchTensorMap(&tmDO);
        PrefetchTensorMap(&tmK);
        PrefetchTensorMap(&tmV);
        PrefetchTensorMap(&tmDQ);
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < SLOTS; i++)
            MbarInit(SmemAddr(&barFull[i]), 1);
        for (int i = 0; i < GR_EVENTS; i++)
            MbarInit(SmemAddr(&barEvent[i]), 1);
        MbarInit(SmemAddr(&barRows), 1);
        MbarInit(SmemAddr(&barQ), 8);
        MbarInit(SmemAddr(&barS), 1);
        MbarInit(SmemAddr(&barSRead), 9);                  /* the softmax warps and the relay */
        MbarInit(SmemAddr(&barDP), 1);
        MbarInit(SmemAddr(&barDS), 9);
        MbarInit(SmemAddr(&barDone), 1);
        MbarInit(SmemAddr(&barFix), 1);
        abortFlag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == GR_ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(SmemAddr(&tmemBaseSlot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmemBase = *(volatile uint32_t *)&tmemBaseSlot;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int rank = p.splits > 1 ? (int)ClusterRank() : 0;
    const int item = p.item0 + (int)blockIdx.x / p.splits;
    const int headItem = item / p.tilesPerHead;
    const int q0 = (item - headItem * p.tilesPerHead) * XT;
    const int b = headItem / p.sh.headsQ, h = headItem - b * p.sh.headsQ, kvHead = h / p.sh.group;
    const int nq = ClampLen(p.sh.queryLens, b, p.sh.lenQ), nk = ClampLen(p.sh.keyLens, b, p.sh.lenK);
    const int keyTiles = q0 < nq ? (nk + XT - 1) / XT : 0;
    const int perSplit = (keyTiles + p.splits - 1) / p.splits;
    const int tile0 = rank * perSplit < keyTiles ? rank * perSplit : keyTiles;
    const int tile1 = tile0 + perSplit < keyTiles ? tile0 + perSplit : keyTiles;
    const int n = tile1 - tile0;
    /* All keys in one tile: delta_i = sum_j p_ij dp_ij is taken from the tile. From the rounded out it would be off by
       2^-11 of sum |do out|, which shows when few keys leave dp - delta small. */
    const bool single = keyTiles == 1;
    /* the last tile reaches past the sequence's keys into rows that exist: those rows of k are cleared */
    const bool fix = n > 0 && tile1 * XT > nk && nk < p.sh.lenK;

    float deltaLeft = 0.f;
    /* by the first warp, when all have left their largest ds in sMost: the exponent of the item's */
    auto leaveMost = [&]() {
        float most = 0.f;
        if (lane < 8)
            for (int t = 0; t < p.splits; t++)
                most = fmaxf(most, p.splits > 1 ? LoadRemote(MapShared(SmemAddr(&sMost[lane]), t)) : sMost[lane]);
        const uint32_t e = __reduce_max_sync(0xffffffffu, __float_as_uint(most)) >> 23;
        if (lane < 8)
            p.work[(long long)item * (2 * XT) + XT + lane] = __uint_as_float((__float_as_uint(deltaLeft) & ~1u) | (e >> lane & 1u));
    };

    if (warp == GR_PRODUCER) {
        if (lane == 0 && n > 0) {
            bool ok = true;
            /* tiles in the order of their use: k 0, v 0, k 1, v 1, ... The last three slots first hold this item's rows of
               q, do and out, on their way to tensor memory. */
            MbarExpectTx(SmemAddr(&barRows), (single ? 2 : 3) * TILE);
#pragma unroll
            for (int dc = 0; dc < DC; dc++) {
                TmaLoad4D(ringS + ROWS0 * TILE + dc * XBOX_BYTES, &tmQ, SmemAddr(&barRows), dc * 64, q0, h * p.aQ.mulHead, b * p.aQ.mulBatch);
                TmaLoad4D(ringS + (ROWS0 + 1) * TILE + dc * XBOX_BYTES, &tmDO, SmemAddr(&barRows), dc * 64, q0, h * p.aDO.mulHead, b * p.aDO.mulBatch);
                if (!single)
                    TmaLoad4D(ringS + (ROWS0 + 2) * TILE + dc * XBOX_BYTES, &tmO, SmemAddr(&barRows), dc * 64, q0, h * p.aO.mulHead, b * p.aO.mulBatch);
            }
            for (int i = 0; ok && i < 2 * n; i++) {
                if (i == ROWS0)
                    ok = MbarWait(SmemAddr(&barQ), 0, abortPtr, p.status);
                if (i >= SLOTS) {
                    /* v t was done with when its product was, k t when the next tile's was */
                    const int old = i - SLOTS, event = (old & 1) ? old / 2 : old / 2 + 1;
                    ok = MbarWait(SmemAddr(&barEvent[event % GR_EVENTS]), (uint32_t)(event / GR_EVENTS) & 1u, abortPtr, p.status);
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
            /* after its load and before the products that read it as rows of the sum; the scores of these keys
               may be taken from either state, their weights are set to 0 */
            const int i = 2 * n - 2;
            if (WaitNowWarp(SmemAddr(&barFull[i % SLOTS]), (uint32_t)(i / SLOTS) & 1u, abortPtr, p.status)) {
                ZeroTileRows(ringS + (i % SLOTS) * TILE, DC, nk - (tile1 - 1) * XT, lane);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0)
                    MbarArrive(SmemAddr(&barFix));
            }
        }
    }
    else if (warp == GR_ISSUER) {
        if (lane == 0 && n > 0) {
            constexpr uint32_t descS = XattnDesc(XT, 0), descQ = XattnDesc(D, 1);
            auto product = [&](uint32_t dst, uint32_t aTmem, uint32_t bTile) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++)
                    TcMmaTmemA(dst, aTmem + ks * 8, SmemDesc(bTile + (ks >> 2) * XBOX_BYTES + (ks & 3) * UMMA_K_BYTES, 16, 1024, 2), descS,
                               ks != 0 ? 1u : 0u);
            };
            bool ok = WaitNow(SmemAddr(&barQ), 0, abortPtr, p.status) && WaitNow(SmemAddr(&barFull[0]), 0, abortPtr, p.status);
            if (ok) {
                TcFenceAfter();
                product(tmemBase + TMEM_S, tmemBase + TMEM_Q, ringS);
                TcCommit(SmemAddr(&barS));
                ok = WaitNow(SmemAddr(&barFull[1]), 0, abortPtr, p.status);
            }
            if (ok) {
                TcFenceAfter();
                product(tmemBase + TMEM_DP, tmemBase + TMEM_DO, ringS + TILE);
                TcCommit(SmemAddr(&barDP));
            }
            for (int j = 0; ok && j < n; j++) {
                const bool more = j + 1 < n;
                if (more) {
                    /* the scores are in registers: the next ones, under the exponentials of these */
                    ok = WaitNow(SmemAddr(&barSRead), (uint32_t)j & 1u, abortPtr, p.status);
                    if (!ok)
                        break;
                    TcFenceAfter();
                    product(tmemBase + TMEM_S, tmemBase + TMEM_Q, ringS + ((2 * j + 2) % SLOTS) * TILE);
                    TcCommit(SmemAddr(&barS));
                }
                ok = WaitNow(SmemAddr(&barDS), (uint32_t)j & 1u, abortPtr, p.status);
                if (!ok)
                    break;
                TcFenceAfter();
#pragma unroll
                for (int ks = 0; ks < XT / 16; ks++)
                    TcMmaTmemA(tmemBase + TMEM_DQ, tmemBase + TMEM_DP + (ks >> 2) * 64 + (ks & 3) * 8,
                               SmemDesc(ringS + ((2 * j) % SLOTS) * TILE + ks * 16 * ROW_BYTES, XBOX_BYTES, 1024, 2), descQ, (j | ks) != 0 ? 1u : 0u);
                if (more) {
                    product(tmemBase + TMEM_DP, tmemBase + TMEM_DO, ringS + ((2 * j + 3) % SLOTS) * TILE);
                    TcCommit(SmemAddr(&barDP));
                }
                else
                    TcCommit(SmemAddr(&barDone));
            }
        }
    }
    else if (warp == GR_RELAY) {
        /* Behind its own tensor-core instructions a thread sees a barrier only some 300 clocks late, so the issuing
           thread waits for the softmax threads alone: this thread's arrivals among theirs say that the copies for the
           products that follow are there (and, at the end, that the rows of k past the sequence are cleared). */
        if (lane == 0 && n > 0) {
            bool ok = true;
            for (int j = 0; ok && j < n; j++) {
                const int ik = 2 * j + 2, iv = 2 * j + 3;
                if (j + 1 < n) {
                    /* not before the phase before is complete: the arrival would count there */
                    ok = WaitNow(SmemAddr(&barFull[ik % SLOTS]), (uint32_t)(ik / SLOTS) & 1u, abortPtr, p.status) &&
                         (j == 0 || WaitNow(SmemAddr(&barSRead), (uint32_t)(j - 1) & 1u, abortPtr, p.status));
                    if (ok)
                        MbarArrive(SmemAddr(&barSRead));
                    ok = ok && WaitNow(SmemAddr(&barFull[iv % SLOTS]), (uint32_t)(iv / SLOTS) & 1u, abortPtr, p.status);
                }
                else if (fix)
                    ok = WaitNow(SmemAddr(&barFix), 0, abortPtr, p.status);
                if (ok && j > 0)
                    ok = WaitNow(SmemAddr(&barDS), (uint32_t)(j - 1) & 1u, abortPtr, p.status);
                if (ok)
                    MbarArrive(SmemAddr(&barDS));
            }
        }
    }
    else {
        const int hf = warp >> 2, sub = warp & 3;
        const uint32_t laneBase = (uint32_t)(sub * 32) << 16;
        const int r = sub * 32 + lane, row = q0 + r;
        const bool rowLive = row < nq && nk > 0;
        /* q and do go to tensor memory as the A operands of the first products (from shared memory those would
           read two operands, at the rate all of shared memory has), half of a row a thread; delta on the way,
           joined through shared memory */
        float part = 0.f;
        bool ok = true;
        if (n > 0) {
            ok = WaitNowWarp(SmemAddr(&barRows), 0, abortPtr, p.status);
#pragma unroll 2
            for (int c = 0; c < D / 16; c++) {
                const int col = hf * (D / 2) + c * 8;
                const uint32_t at = ringS + ROWS0 * TILE + (col >> 6) * XBOX_BYTES + r * ROW_BYTES + ((((col >> 3) & 7) ^ (r & 7)) << 4);
                uint32_t xs[4], ys[4], zs[4];
                LoadShared16(at, zs);
                LoadShared16(at + TILE, ys);
                if (!single)
                    LoadShared16(at + 2 * TILE, xs);
#pragma unroll
                for (int e = 0; e < 4 && !single; e++) {
                    const float2 xf = __half22float2(*(const __half2 *)&xs[e]), yf = __half22float2(*(const __half2 *)&ys[e]);
                    part = fmaf(xf.x, yf.x, part);
                    part = fmaf(xf.y, yf.y, part);
                }
                TmemStore4Async(tmemBase + laneBase + TMEM_DO + col / 2, ys);
                TmemStore4Async(tmemBase + laneBase + TMEM_Q + col / 2, zs);
            }
            TmemWaitStore();
            TcFenceBefore();
            ArriveWarp(SmemAddr(&barQ), lane);
        }
        /* rows past the sequence hold anything; they are no part of any other row's sums here */
        if (!rowLive)
            part = 0.f;
        if (hf == 1)
            sDelta[r] = part;
        GradBarrier();
        if (hf == 0)
            sDelta[r] = part + sDelta[r];
        GradBarrier();
        float delta = sDelta[r];
        /* exponents of 2; plus infinity makes every weight of an empty row 0 */
        const float lse2 = rowLive ? p.lse[((long long)b * p.sh.headsQ + h) * p.sh.lenQ + row] * LOG2E : INFINITY;
        /* for the second kernel, whose exponents carry the factor of p; dP and delta its inverse */
        auto leaveRow = [&]() {
            if (hf == 0 && rank == 0) {
                float * w = p.work + (long long)item * (2 * XT);
                w[r] = lse2 - P_SCALE_LOG2;
                w[XT + r] = deltaLeft = -delta * P_SCALE_INV;
            }
        };
        if (!single)
            leaveRow();
        const uint32_t sT = tmemBase + laneBase + TMEM_S + hf * 64, dpT = tmemBase + laneBase + TMEM_DP + hf * 64;
        const uint32_t dqT = tmemBase + laneBase + TMEM_DQ;
        float factor = 1.f, most = 0.f;                      /* of this row's ds; their largest */
        /* no warp leaves out a step's barriers, whatever became of its waits (after one that ran out the next return at once) */
        for (int j = 0; j < n; j++) {
            const uint32_t ph = (uint32_t)j & 1u;
            ok = WaitNowWarp(SmemAddr(&barS), ph, abortPtr, p.status) && ok;
            TcFenceAfter();
            uint32_t x[64];
            TmemLoad64U(sT, x);
            TcFenceBefore();
            ArriveWarp(SmemAddr(&barSRead), lane);
#pragma unroll
            for (int e = 0; e < 64; e++)
                x[e] = __float_as_uint(Exp2(fmaf(__uint_as_float(x[e]), p.scaleLog2, -lse2)));
            const int valid = nk - (tile0 + j) * XT - hf * 64;
            ok = WaitNowWarp(SmemAddr(&barDP), ph, abortPtr, p.status) && ok;
            /* v of this tile and k of the one before have been read */
            if (threadIdx.x == 0)
                MbarArrive(SmemAddr(&barEvent[j % GR_EVENTS]));
            TcFenceAfter();
            if (single) {
                float sum = 0.f;
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t y[32];
                    TmemLoad32Async(dpT + c * 32, y);
                    TmemWaitLoad();
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        sum += c * 32 + e < valid ? __uint_as_float(x[c * 32 + e]) * __uint_as_float(y[e]) : 0.f;
                }
                if (hf == 1)
                    sDelta[r] = sum;
                GradBarrier();
                if (hf == 0)
                    sDelta[r] = sum + sDelta[r];
                GradBarrier();
                delta = rowLive ? sDelta[r] : 0.f;
                leaveRow();
            }
            const uint64_t factor2 = Pair(factor, factor), delta2 = Pair(-delta * factor, -delta * factor);
            float top = 0.f;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t y[32];
                TmemLoad32Async(dpT + c * 32, y);
                TmemWaitLoad();
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const uint64_t d = Fma2(Pair(__uint_as_float(y[e]), __uint_as_float(y[e + 1])), factor2, delta2);
                    float a, b;
                    Unpair(Mul2(Pair(__uint_as_float(x[c * 32 + e]), __uint_as_float(x[c * 32 + e + 1])), d), a, b);
                    x[c * 32 + e] = valid >= 64 || c * 32 + e < valid ? __float_as_uint(a) : 0u;
                    x[c * 32 + e + 1] = valid >= 64 || c * 32 + e + 1 < valid ? __float_as_uint(b) : 0u;
                }
                top = fmaxf(top, LargestDs(x + c * 32));
                if (j > 0)
                    PackDs(dpT + c * 16, x + c * 32);
            }
            most = fmaxf(most, top * PowerInverse(factor));
            /* the step before's product is done: its sums may be scaled */
            SettleDs<D>(x, top, factor, rowLive, j == 0, hf, &sDelta[r], dpT, dqT);
            TcFenceBefore();
            ArriveWarp(SmemAddr(&barDS), lane);
        }
        if (n > 0 && ok)
            ok = WaitNowWarp(SmemAddr(&barDone), 0, abortPtr, p.status);
        TcFenceAfter();
        const bool sums = n > 0 && ok;
        const float power = PowerInverse(factor), out = SumsFactor(power, p.scale);
        most = __uint_as_float(__reduce_max_sync(0xffffffffu, rowLive ? __float_as_uint(most) : 0u));
        if (lane == 0)
            sMost[warp] = most;
#pragma unroll 1
        for (int c = hf * (D / 64); c < (hf + 1) * (D / 64); c++) {       /* 32 columns a step; this half's D / 2 */
            uint32_t o[32];
            if (sums) {
                TmemLoad32Async(dqT + c * 32, o);
                TmemWaitLoad();
            }
            if (p.splits == 1)
                StageHalf32(outS + (c >> 1) * XBOX_BYTES + r * ROW_BYTES, lane, (c & 1) * 4, o, out, sums && rowLive);
            else
                StorePartial(ringS + r * D * 4, r, c * 8, o, power, sums);
        }
        if (p.splits == 1) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            GradBarrier();                       /* all eight warps come here, whatever became of their waits */
            if (warp == 0)
                leaveMost();
            if (ok && hf == 0 && lane == 0 && q0 + sub * 32 < p.sh.lenQ) {
#pragma unroll
                for (int dc = 0; dc < DC; dc++)
                    TmaStore4D(&tmDQ, outS + dc * XBOX_BYTES + sub * 32 * ROW_BYTES, dc * 64, q0 + sub * 32, h, b);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
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
        if (warp == 0 && rank == 0)
            leaveMost();
        if (warp < 8) {
            const int rowsEach = XT / p.splits, chunks = D / 8;
            for (int i = threadIdx.x; i < rowsEach * chunks; i += 256) {
                const int c = i % chunks, r = rank * rowsEach + i / chunks, row = q0 + r;
                if (row >= p.sh.lenQ || c * 8 >= p.sh.dim)
                    continue;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (row < nq && nk > 0)
                    w = SumPartials(ringS + r * D * 4, r, c, p.splits, p.scale);
                *(uint4 *)(p.d0 + b * p.l0.batch + h * p.l0.head + row * p.l0.row + c * 8) = w;
            }
        }
        __syncwarp();
        ClusterSync();
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    if (warp == GR_ISSUER)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmemBase), "r"(512u) : "memory");
}

template <int D>
__global__ void __launch_bounds__(GR_THREADS, 1)
XattnGradKVKernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmDO, const __grid_constant__ CUtensorMap tmDK, const __grid_constant__ CUtensorMap tmDV,
                  const XattnGradParams p)
{
    using SM = XattnGradSmem<D>;
    constexpr int DC = SM::DC, TILE = SM::TILE, QSLOTS = SM::QSLOTS, DOSLOTS = SM::DOSLOTS, STATSLOTS = SM::STATSLOTS;
    constexpr int TMEM_S = 0, TMEM_DP = 128, TMEM_DV = 256, TMEM_DK = 256 + D;
    /* everything in one region, on a swizzle boundary by its alignment: there is no room to move it up */
    extern __shared__ __align__(1024) uint8_t kvSmem[];
    struct Bars {
        uint64_t qFull[QSLOTS], qEmpty[QSLOTS], doFull[DOSLOTS], doEmpty[DOSLOTS], statFull[STATSLOTS], statEmpty[STATSLOTS];
        uint64_t qRaw[QSLOTS], doRaw[DOSLOTS];               /* loads of tiles with rows to be cleared */
        uint64_t k, v, s, p, dp, ds, done;
        uint32_t tmem;
        int abort;
        int most[8];                                         /* the warps' largest exponents of ds */
    };
    static_assert(sizeof(Bars) <= 256, "place of the barriers");
    Bars & bars = *(Bars *)(kvSmem + SM::KV_BARS);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t smemBase = SmemAddr(kvSmem);
    const uint32_t kS = smemBase, vS = kS + TILE, ringS = vS + TILE, doRing = ringS + QSLOTS * TILE, statRing = smemBase + SM::KV_STATS;
    volatile int * abortPtr = &bars.abort;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == GR_PRODUCER && lane == 0) {
        PrefetchTensorMap(&tmQ);
        PrefetchTensorMap(&tmK);
        PrefetchTensorMap(&tmV);
        PrefetchTensorMap(&tmDO);
        PrefetchTensorMap(&tmDK);
        PrefetchTensorMap(&tmDV);
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < QSLOTS; i++) {
            MbarInit(SmemAddr(&bars.qFull[i]), 1);
            MbarInit(SmemAddr(&bars.qEmpty[i]), 1);
            MbarInit(SmemAddr(&bars.qRaw[i]), 1);
        }
        for (int i = 0; i < DOSLOTS; i++) {
            MbarInit(SmemAddr(&bars.doFull[i]), 1);
            MbarInit(SmemAddr(&bars.doEmpty[i]), 1);
            MbarInit(SmemAddr(&bars.doRaw[i]), 1);
        }
        for (int i = 0; i < STATSLOTS; i++) {
            MbarInit(SmemAddr(&bars.statFull[i]), 1);
            MbarInit(SmemAddr(&bars.statEmpty[i]), 1);
        }
        MbarInit(SmemAddr(&bars.k), 1);
        MbarInit(SmemAddr(&bars.v), 1);
        MbarInit(SmemAddr(&bars.s), 1);
        MbarInit(SmemAddr(&bars.p), 9);                    /* the softmax warps and the relay */
        MbarInit(SmemAddr(&bars.dp), 1);
        MbarInit(SmemAddr(&bars.ds), 9);
        MbarInit(SmemAddr(&bars.done), 1);
        bars.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == GR_ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     :: "r"(SmemAddr(&bars.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    const uint32_t tmemBase = *(volatile uint32_t *)&bars.tmem;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int rank = p.splits > 1 ? (int)ClusterRank() : 0;
    const int item = p.item0 + (int)blockIdx.x / p.splits;
    const int headItem = item / p.keyTiles;
    const int k0 = (item - headItem * p.keyTiles) * XT;
    const int b = headItem / p.sh.headsKV, kvHead = headItem - b * p.sh.headsKV;
    const int nq = ClampLen(p.sh.queryLens, b, p.sh.lenQ), nk = ClampLen(p.sh.keyLens, b, p.sh.lenK);
    const int qTiles = (nq + XT - 1) / XT;
    const int steps = k0 < nk ? p.sh.group * qTiles : 0;
    const int perSplit = (steps + p.splits - 1) / p.splits;
    const int step0 = rank * perSplit < steps ? rank * perSplit : steps;
    const int step1 = step0 + perSplit < steps ? step0 + perSplit : steps;
    const int n = step1 - step0;
    /* a head's last query tile may reach into rows past the sequence */
    const bool ragged = nq < p.sh.lenQ && nq % XT != 0;
    auto edge = [&](int i) { return ragged && (step0 + i) % qTiles == qTiles - 1; };

    if (warp == GR_PRODUCER) {
        bool ok = true;
        auto loadOwn = [&](const CUtensorMap * map, const HeadsAddr & a, uint32_t dst, uint32_t bar) {
            if (lane == 0) {
                MbarExpectTx(bar, TILE);
#pragma unroll
                for (int dc = 0; dc < DC; dc++)
                    TmaLoad4D(dst + dc * XBOX_BYTES, map, bar, dc * 64, k0, kvHead * a.mulHead, b * a.mulBatch);
            }
            __syncwarp();
        };
        /* one tile of q or do into its ring; a tile with rows past the sequence arrives on a barrier of its own, and the
           relay hands it on */
        auto load = [&](const CUtensorMap * map, const HeadsAddr & a, int i, uint32_t dst, uint32_t full, uint32_t raw) {
            const int step = step0 + i, g = step / qTiles, qt = step - g * qTiles, h = kvHead * p.sh.group + g;
            const uint32_t bar = edge(i) ? raw : full;
            if (lane == 0) {
                MbarExpectTx(bar, TILE);
#pragma unroll
                for (int dc = 0; dc < DC; dc++)
                    TmaLoad4D(dst + dc * XBOX_BYTES, map, bar, dc * 64, qt * XT, h * a.mulHead, b * a.mulBatch);
            }
            __syncwarp();
        };
        auto loadQ = [&](int i) {
            if (i >= QSLOTS)
                ok = ok && MbarWaitWarp(SmemAddr(&bars.qEmpty[i % QSLOTS]), (uint32_t)(i / QSLOTS + 1) & 1u, abortPtr, p.status, 200);
            if (ok)
                load(&tmQ, p.aQ, i, ringS + (i % QSLOTS) * TILE, SmemAddr(&bars.qFull[i % QSLOTS]), SmemAddr(&bars.qRaw[i % QSLOTS]));
        };
        auto loadDO = [&](int i) {
            if (i >= DOSLOTS)
                ok = ok && MbarWaitWarp(SmemAddr(&bars.doEmpty[i % DOSLOTS]), (uint32_t)(i / DOSLOTS + 1) & 1u, abortPtr, p.status, 200);
            if (ok)
                load(&tmDO, p.aDO, i, doRing + (i % DOSLOTS) * TILE, SmemAddr(&bars.doFull[i % DOSLOTS]), SmemAddr(&bars.doRaw[i % DOSLOTS]));
        };
        auto loadStat = [&](int i) {
            if (i >= STATSLOTS)
                ok = ok && MbarWaitWarp(SmemAddr(&bars.statEmpty[i % STATSLOTS]), (uint32_t)(i / STATSLOTS + 1) & 1u, abortPtr, p.status, 200);
            if (ok && lane == 0) {
                const int step = step0 + i, g = step / qTiles, qt = step - g * qTiles, h = kvHead * p.sh.group + g;
                const float * src = p.work + (((long long)b * p.sh.headsQ + h) * p.tilesPerHead + qt) * (2 * XT);
                const uint32_t bar = SmemAddr(&bars.statFull[i % STATSLOTS]);
                MbarExpectTx(bar, SM::STAT);
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             :: "r"(statRing + (i % STATSLOTS) * SM::STAT), "l"(src), "r"((uint32_t)SM::STAT), "r"(bar) : "memory");
            }
            __syncwarp();
        };
        /* in the order of their use: q runs two steps ahead of the sums, do and the rows' numbers one */
        if (n > 0) {
            loadOwn(&tmK, p.aK, kS, SmemAddr(&bars.k));
            loadQ(0);
            loadStat(0);
            loadOwn(&tmV, p.aV, vS, SmemAddr(&bars.v));
            loadDO(0);
            if (n > 1)
                loadQ(1);
        }
        for (int i = 0; ok && i + 1 < n; i++) {
            loadDO(i + 1);
            loadStat(i + 1);
            if (i + 2 < n)
                loadQ(i + 2);
        }
    }
    else if (warp == GR_ISSUER) {
        if (lane == 0 && n > 0) {
            constexpr uint32_t descS = XattnDesc(XT, 0), descD = XattnDesc(D, 1);
            auto product = [&](uint32_t dst, uint32_t aTile, uint32_t bTile) {
#pragma unroll
                for (int dc = 0; dc < DC; dc++)
#pragma unroll
                    for (int ks = 0; ks < 4; ks++)
                        TcMma<0>(dst, SmemDesc(aTile + dc * XBOX_BYTES + ks * UMMA_K_BYTES, 16, 1024, 2),
                                 SmemDesc(bTile + dc * XBOX_BYTES + ks * UMMA_K_BYTES, 16, 1024, 2), descS, (dc | ks) != 0 ? 1u : 0u);
            };
            auto second = [&](uint32_t dst, uint32_t aTmem, uint32_t bTile, bool first) {
#pragma unroll
                for (int ks = 0; ks < XT / 16; ks++)
                    TcMmaTmemA(dst, aTmem + (ks >> 2) * 64 + (ks & 3) * 8, SmemDesc(bTile + ks * 16 * ROW_BYTES, XBOX_BYTES, 1024, 2), descD,
                               !first || ks != 0 ? 1u : 0u);
            };
            bool ok = WaitNow(SmemAddr(&bars.k), 0, abortPtr, p.status) && WaitNow(SmemAddr(&bars.qFull[0]), 0, abortPtr, p.status);
            if (ok) {
                TcFenceAfter();
                product(tmemBase + TMEM_S, kS, ringS);
                TcCommit(SmemAddr(&bars.s));
                ok = WaitNow(SmemAddr(&bars.v), 0, abortPtr, p.status) && WaitNow(SmemAddr(&bars.doFull[0]), 0, abortPtr, p.status);
            }
            if (ok) {
                TcFenceAfter();
                product(tmemBase + TMEM_DP, vS, doRing);
                TcCommit(SmemAddr(&bars.dp));
            }
            for (int i = 0; ok && i < n; i++) {
                const bool more = i + 1 < n;
                ok = WaitNow(SmemAddr(&bars.p), (uint32_t)i & 1u, abortPtr, p.status);
                if (!ok)
                    break;
                TcFenceAfter();
                second(tmemBase + TMEM_DV, tmemBase + TMEM_S, doRing + (i % DOSLOTS) * TILE, i == 0);
                if (more) {
                    product(tmemBase + TMEM_S, kS, ringS + ((i + 1) % QSLOTS) * TILE);
                    TcCommit(SmemAddr(&bars.s));
                }
                ok = WaitNow(SmemAddr(&bars.ds), (uint32_t)i & 1u, abortPtr, p.status);
                if (!ok)
                    break;
                TcFenceAfter();
                second(tmemBase + TMEM_DK, tmemBase + TMEM_DP, ringS + (i % QSLOTS) * TILE, i == 0);
                if (more) {
                    product(tmemBase + TMEM_DP, vS, doRing + ((i + 1) % DOSLOTS) * TILE);
                    TcCommit(SmemAddr(&bars.dp));
                }
                else
                    TcCommit(SmemAddr(&bars.done));
            }
        }
    }
    else if (warp == GR_RELAY) {
        /* as in the first kernel: the next step's copies are there, those with rows past the sequence cleared of them
           (their weights are 0, and 0 * NaN would reach the sums). Done by the producer, that held up the loads behind. */
        bool ok = true;
        uint32_t qRound = 0, doRound = 0;                    /* a bit a slot: the phase of its next raw load */
        auto ready = [&](int i, bool isQ) {
            const int slot = isQ ? i % QSLOTS : i % DOSLOTS;
            const uint32_t full = isQ ? SmemAddr(&bars.qFull[slot]) : SmemAddr(&bars.doFull[slot]);
            if (!edge(i))
                return MbarWaitWarp(full, (uint32_t)(isQ ? i / QSLOTS : i / DOSLOTS) & 1u, abortPtr, p.status, 0);
            const uint32_t rounds = isQ ? qRound : doRound;
            if (!WaitNowWarp(isQ ? SmemAddr(&bars.qRaw[slot]) : SmemAddr(&bars.doRaw[slot]), rounds >> slot & 1u, abortPtr, p.status))
                return false;
            if (isQ)
                qRound ^= 1u << slot;
            else
                doRound ^= 1u << slot;
            ZeroTileRows(isQ ? ringS + slot * TILE : doRing + slot * TILE, DC, nq - (qTiles - 1) * XT, lane);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            ArriveWarp(full, lane);
            return true;
        };
        if (n > 0 && edge(0))
            ok = ready(0, true) && ready(0, false);
        for (int i = 0; ok && i < n; i++) {
            if (i + 1 < n)
                ok = ready(i + 1, true);
            if (ok && i > 0)
                ok = MbarWaitWarp(SmemAddr(&bars.p), (uint32_t)(i - 1) & 1u, abortPtr, p.status, 0);
            if (ok)
                ArriveWarp(SmemAddr(&bars.p), lane);
            if (ok && i + 1 < n)
                ok = ready(i + 1, false);
            if (ok && i > 0)
                ok = MbarWaitWarp(SmemAddr(&bars.ds), (uint32_t)(i - 1) & 1u, abortPtr, p.status, 0);
            if (ok)
                ArriveWarp(SmemAddr(&bars.ds), lane);
        }
        __syncwarp();
    }
    else {
        const int hf = warp >> 2, sub = warp & 3;
        const uint32_t laneBase = (uint32_t)(sub * 32) << 16;
        const int r = sub * 32 + lane;
        const uint32_t sT = tmemBase + laneBase + TMEM_S + hf * 64, dpT = tmemBase + laneBase + TMEM_DP + hf * 64;
        /* the factor of this head's ds, by the largest that the first kernel met in its query tiles. An infinity there comes
           of a delta or dp that makes every dk of the head infinite or NaN: here NaN. */
        int e = 0;
        for (int t = threadIdx.x; t < steps; t += 256) {
            const int g = t / qTiles, qt = t - g * qTiles;
            const uint4 * w = (const uint4 *)(p.work + (((long long)b * p.sh.headsQ + kvHead * p.sh.group + g) * p.tilesPerHead + qt) * (2 * XT) + XT);
            const uint4 lo = __ldcg(w), hi = __ldcg(w + 1);
            e = max(e, (int)((lo.x & 1u) | (lo.y & 1u) << 1 | (lo.z & 1u) << 2 | (lo.w & 1u) << 3 |
                             (hi.x & 1u) << 4 | (hi.y & 1u) << 5 | (hi.z & 1u) << 6 | (hi.w & 1u) << 7));
        }
        e = __reduce_max_sync(0xffffffffu, e);
        if (lane == 0)
            bars.most[warp] = e;
        GradBarrier();
        for (int w = 0; w < 8; w++)
            e = max(e, bars.most[w]);
        const float factor = e < 255 ? PowerFor(__uint_as_float((uint32_t)e << 23), 14) : NAN;
        const uint64_t factor2 = Pair(factor, factor), unscale2 = Pair(factor * P_SCALE_INV, factor * P_SCALE_INV);
        bool ok = true;
        for (int i = 0; i < n; i++) {
            const uint32_t ph = (uint32_t)i & 1u;
            const float4 * lse4 = (const float4 *)(kvSmem + SM::KV_STATS + (i % STATSLOTS) * SM::STAT) + hf * 16, * delta4 = lse4 + XT / 4;
            /* every lane observes the copy's completion itself before it reads what was copied */
            ok = WaitNowWarp(SmemAddr(&bars.statFull[i % STATSLOTS]), (uint32_t)(i / STATSLOTS) & 1u, abortPtr, p.status) &&
                 WaitNowWarp(SmemAddr(&bars.s), ph, abortPtr, p.status);
            if (!ok)
                break;
            /* these scores were issued behind the last product that reads the step before's do */
            if (threadIdx.x == 0 && i >= 1)
                MbarArrive(SmemAddr(&bars.doEmpty[(i - 1) % DOSLOTS]));
            TcFenceAfter();
            uint32_t x[64];
            TmemLoad64U(sT, x);
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t w[16];
#pragma unroll
                for (int e4 = 0; e4 < 8; e4++) {
                    const float4 ls = lse4[c * 8 + e4];
                    const int e = c * 32 + e4 * 4;
                    const float p0 = Exp2(fmaf(__uint_as_float(x[e]), p.scaleLog2, -ls.x)), p1 = Exp2(fmaf(__uint_as_float(x[e + 1]), p.scaleLog2, -ls.y));
                    const float p2 = Exp2(fmaf(__uint_as_float(x[e + 2]), p.scaleLog2, -ls.z)), p3 = Exp2(fmaf(__uint_as_float(x[e + 3]), p.scaleLog2, -ls.w));
                    x[e] = __float_as_uint(p0); x[e + 1] = __float_as_uint(p1);
                    x[e + 2] = __float_as_uint(p2); x[e + 3] = __float_as_uint(p3);
                    w[e4 * 2] = PackHalf2(p0, p1);
                    w[e4 * 2 + 1] = PackHalf2(p2, p3);
                }
                TmemStore16Async(sT + c * 16, w);
            }
            TmemWaitStore();
            TcFenceBefore();
            ArriveWarp(SmemAddr(&bars.p), lane);
            ok = WaitNowWarp(SmemAddr(&bars.dp), ph, abortPtr, p.status);
            if (!ok)
                break;
            /* and this product behind the one that reads its q, which all softmax threads let go ahead */
            if (threadIdx.x == 0 && i >= 1) {
                MbarArrive(SmemAddr(&bars.qEmpty[(i - 1) % QSLOTS]));
                MbarArrive(SmemAddr(&bars.statEmpty[(i - 1) % STATSLOTS]));
            }
            TcFenceAfter();
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t y[32], w[16];
                TmemLoad32Async(dpT + c * 32, y);
                TmemWaitLoad();
#pragma unroll
                for (int e4 = 0; e4 < 8; e4++) {
                    const float4 de = delta4[c * 8 + e4];        /* -2^-12 delta */
                    const int e = e4 * 4, xe = c * 32 + e;
                    const uint64_t d0 = Fma2(Pair(__uint_as_float(y[e]), __uint_as_float(y[e + 1])), unscale2, Mul2(Pair(de.x, de.y), factor2));
                    const uint64_t d1 = Fma2(Pair(__uint_as_float(y[e + 2]), __uint_as_float(y[e + 3])), unscale2, Mul2(Pair(de.z, de.w), factor2));
                    float f0, f1, f2, f3;
                    Unpair(Mul2(Pair(__uint_as_float(x[xe]), __uint_as_float(x[xe + 1])), d0), f0, f1);
                    Unpair(Mul2(Pair(__uint_as_float(x[xe + 2]), __uint_as_float(x[xe + 3])), d1), f2, f3);
                    w[e4 * 2] = PackHalf2Finite(f0, f1);
                    w[e4 * 2 + 1] = PackHalf2Finite(f2, f3);
                }
                TmemStore16Async(dpT + c * 16, w);
            }
            TmemWaitStore();
            TcFenceBefore();
            ArriveWarp(SmemAddr(&bars.ds), lane);
        }
        if (n > 0 && ok)
            ok = WaitNowWarp(SmemAddr(&bars.done), 0, abortPtr, p.status);
        TcFenceAfter();
        const bool sums = n > 0 && ok, rowLive = k0 + r < nk;
        /* warps 0-3: dv, in the place of v; warps 4-7: dk, in the place of k */
        const uint32_t accT = tmemBase + laneBase + (hf == 0 ? TMEM_DV : TMEM_DK);
        const uint32_t box = (hf == 0 ? vS : kS) + sub * 32 * ROW_BYTES;
        const float power = hf == 0 ? P_SCALE_INV : PowerInverse(factor), out = SumsFactor(power, hf == 0 ? 1.f : p.scale);
        if (p.splits == 1) {
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                if (sums) {
                    TmemLoad32Async(accT + c * 32, o);
                    TmemWaitLoad();
                }
                StageHalf32(box + (c >> 1) * XBOX_BYTES + lane * ROW_BYTES, lane, (c & 1) * 4, o, out, sums && rowLive);
            }
        }
        else {
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                if (sums) {
                    TmemLoad32Async(accT + c * 32, o);
                    TmemWaitLoad();
                }
                StorePartial(ringS + (hf * XT + r) * D * 4, r, c * 8, o, power, sums);
            }
        }
        if (p.splits == 1 && ok) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && k0 + sub * 32 < p.sh.lenK) {
#pragma unroll
                for (int dc = 0; dc < DC; dc++)
                    TmaStore4D(hf == 0 ? &tmDV : &tmDK, box + dc * XBOX_BYTES, dc * 64, k0 + sub * 32, kvHead, b);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
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
        if (warp < 8) {
            const int rowsEach = XT / p.splits, chunks = D / 8;
            for (int i = threadIdx.x; i < 2 * rowsEach * chunks; i += 256) {
                const int c = i % chunks, rr = i / chunks, which = rr / rowsEach;
                const int r = rank * rowsEach + (rr - which * rowsEach), row = k0 + r;
                if (row >= p.sh.lenK || c * 8 >= p.sh.dim)
                    continue;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (row < nk && steps > 0)
                    w = SumPartials(ringS + (which * XT + r) * D * 4, r, c, p.splits, which == 0 ? 1.f : p.scale);
                if (which == 0)
                    *(uint4 *)(p.d1 + b * p.l1.batch + kvHead * p.l1.head + row * p.l1.row + c * 8) = w;
                else
                    *(uint4 *)(p.d0 + b * p.l0.batch + kvHead * p.l0.head + row * p.l0.row + c * 8) = w;
            }
        }
        __syncwarp();
        ClusterSync();
    }
    TcFenceBefore();
    __syncthreads();
    TcFenceAfter();
    if (warp == GR_ISSUER)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmemBase), "r"(512u) : "memory");
}

/* CTAs of a cluster that share one item's walk: until one wave is full, while a part keeps two steps; and parts of few
   enough instructions */
int GradSplits(long long items, int steps, int smCount)
{
    int splits = 1;
    while (splits < 8 && ((items * splits * 2 <= smCount && steps >= splits * 4) || steps > splits * XATTN_PART_TILES))
        splits *= 2;
    return splits;
}

/* one or two launches: the items of a last wave that fills at most half of the GPU are split over it when they are long */
struct GradPlan {
    int item0, splits;
    long long items;
};
int PlanGrad(long long items, int steps, int smCount, GradPlan * plan)
{
    if (items == 0)
        return 0;
    const int splits = GradSplits(items, steps, smCount);
    const long long rest = items > smCount && splits == 1 ? items % smCount : 0;
    int restSplits = 1;
    while (rest > 0 && restSplits < 8 && rest * restSplits * 2 <= smCount && steps >= restSplits * 8)
        restSplits *= 2;
    if (restSplits == 1) {
        plan[0] = { 0, splits, items };
        return 1;
    }
    plan[0] = { 0, 1, items - rest };
    plan[1] = { (int)(items - rest), restSplits, rest };
    return 2;
}

template <int D>
int LaunchGrad(const DeviceCtx & ctx, const XattnGradCall & call, cudaStream_t stream)
{
    using SM = XattnGradSmem<D>;
    const XattnShape & s = call.sh;
    XattnGradParams p;
    memset(&p, 0, sizeof(p));
    p.sh = s;
    p.lse = call.lse;
    p.work = call.work;
    p.tilesPerHead = (s.lenQ + XT - 1) / XT;
    p.keyTiles = (s.lenK + XT - 1) / XT;
    p.scale = call.scale;
    p.scaleLog2 = call.scale * LOG2E;
    p.status = ctx.status;
    const long long itemsQ = (long long)s.batch * s.headsQ * p.tilesPerHead, itemsKV = (long long)s.batch * s.headsKV * p.keyTiles;
    const long long steps = (long long)s.group * p.tilesPerHead;
    if (steps > 0x3fffffffLL || itemsQ * 8 > 0x7fffffffLL || itemsKV * 8 > 0x7fffffffLL)
        return NTB_ERR_LIMIT;
    CUtensorMap tmQ, tmK, tmV, tmO, tmDO, tmDQ, tmDK, tmDV;
    HeadsAddr unused;
    int rc;
    if (s.lenQ > 0 &&
        ((rc = EncodeHeads(&tmQ, &p.aQ, call.q, s.dim, s.lenQ, s.headsQ, s.batch, call.l[0], XT)) != NTB_OK ||
         (rc = EncodeHeads(&tmO, &p.aO, call.out, s.dim, s.lenQ, s.headsQ, s.batch, call.l[3], XT)) != NTB_OK ||
         (rc = EncodeHeads(&tmDO, &p.aDO, call.dout, s.dim, s.lenQ, s.headsQ, s.batch, call.l[4], XT)) != NTB_OK ||
         (rc = EncodeHeads(&tmDQ, &unused, call.dq, s.dim, s.lenQ, s.headsQ, s.batch, call.l[5], 32)) != NTB_OK))
        return rc;
    if (s.lenK > 0 &&
        ((rc = EncodeHeads(&tmK, &p.aK, call.k, s.dim, s.lenK, s.headsKV, s.batch, call.l[1], XT)) != NTB_OK ||
         (rc = EncodeHeads(&tmV, &p.aV, call.v, s.dim, s.lenK, s.headsKV, s.batch, call.l[2], XT)) != NTB_OK ||
         (rc = EncodeHeads(&tmDK, &unused, call.dk, s.dim, s.lenK, s.headsKV, s.batch, call.l[6], 32)) != NTB_OK ||
         (rc = EncodeHeads(&tmDV, &unused, call.dv, s.dim, s.lenK, s.headsKV, s.batch, call.l[7], 32)) != NTB_OK))
        return rc;
    /* an empty side's maps are never used: no step touches it */
    if (s.lenQ == 0) {
        tmQ = tmDO = tmK;
        p.aQ = p.aDO = p.aK;
    }
    if (s.lenK == 0) {
        tmK = tmV = tmQ;
        p.aK = p.aV = p.aQ;
    }
    static SmemOptIn optQ, optKV;
    if (!optQ.Ensure((const void *)XattnGradQKernel<D>, SM::Q_TOTAL) || !optKV.Ensure((const void *)XattnGradKVKernel<D>, SM::KV_TOTAL))
        return NTB_ERR_CUDA;
    cudaError_t err = cudaSuccess;
    GradPlan plan[2];
    p.d0 = (__half *)call.dq;
    p.l0 = call.l[5];
    int parts = PlanGrad(itemsQ, p.keyTiles, ctx.smCount, plan);
    for (int i = 0; i < parts && err == cudaSuccess; i++) {
        p.item0 = plan[i].item0;
        p.splits = plan[i].splits;
        err = LaunchClusterPdl(XattnGradQKernel<D>, (unsigned)(plan[i].items * p.splits), GR_THREADS, SM::Q_TOTAL, p.splits, stream,
                               tmQ, tmK, tmV, tmO, tmDO, tmDQ, p);
        CountLaunch();
    }
    p.d0 = (__half *)call.dk;
    p.l0 = call.l[6];
    p.d1 = (__half *)call.dv;
    p.l1 = call.l[7];
    parts = PlanGrad(itemsKV, (int)steps, ctx.smCount, plan);
    for (int i = 0; i < parts && err == cudaSuccess; i++) {
        p.item0 = plan[i].item0;
        p.splits = plan[i].splits;
        err = LaunchClusterPdl(XattnGradKVKernel<D>, (unsigned)(plan[i].items * p.splits), GR_THREADS, SM::KV_TOTAL, p.splits, stream,
                               tmQ, tmK, tmV, tmDO, tmDK, tmDV, p);
        CountLaunch();
    }
    return (err == cudaSuccess && cudaGetLastError() == cudaSuccess) ? NTB_OK : NTB_ERR_CUDA;
}

}

}

using namespace ntb;

extern "C" long long ntb_cross_attention_grad_work(int batch, int headsQ, int lenQ)
{
    if (batch < 0 || headsQ < 0 || lenQ < 0)
        return 0;
    return (long long)batch * headsQ * (((long long)lenQ + XT - 1) / XT) * (2 * XT) * (long long)sizeof(float);
}

extern "C" int ntb_cross_attention_grad(int devID, void * stream, const void * q, const void * k, const void * v,
                                        const void * out, const float * lse, const void * dout,
                                        void * dq, void * dk, void * dv, void * work, long long workBytes,
                                        int dtype, int batch, int headsQ, int headsKV, int lenQ, int lenK, int dim,
                                        const ntb_heads_layout * layouts, const int * queryLens, const int * keyLens, float scale)
{
    XattnGradCall call;
    memset(&call, 0, sizeof(call));
    int rc = XattnShapeOf(call.sh, dtype, batch, headsQ, headsKV, lenQ, lenK, dim, queryLens, keyLens, scale);
    if (rc != NTB_OK)
        return rc;
    /* without query heads dk and dv are the sums of nothing, as without queries */
    if (headsQ == 0)
        lenQ = call.sh.lenQ = 0;
    if (batch == 0 || headsKV == 0 || (lenQ == 0 && lenK == 0))
        return NTB_OK;
    if (!layouts || (lenQ > 0 && (!q || !out || !lse || !dout || !dq)) || (lenK > 0 && (!k || !v || !dk || !dv)))
        return NTB_ERR_ARG;
    if (workBytes < ntb_cross_attention_grad_work(batch, headsQ, lenQ) || (lenQ > 0 && (!work || ((uintptr_t)work & 15))))
        return NTB_ERR_ARG;
    if (lenQ > 0 && (!LayoutOk(q, layouts[0], dim, lenQ, headsQ, batch, true) || !LayoutOk(out, layouts[3], dim, lenQ, headsQ, batch, true) ||
                     !LayoutOk(dout, layouts[4], dim, lenQ, headsQ, batch, true) || !LayoutOk(dq, layouts[5], dim, lenQ, headsQ, batch, false)))
        return NTB_ERR_ARG;
    if (lenK > 0 && (!LayoutOk(k, layouts[1], dim, lenK, headsKV, batch, true) || !LayoutOk(v, layouts[2], dim, lenK, headsKV, batch, true) ||
                     !LayoutOk(dk, layouts[6], dim, lenK, headsKV, batch, false) || !LayoutOk(dv, layouts[7], dim, lenK, headsKV, batch, false)))
        return NTB_ERR_ARG;
    call.q = q; call.k = k; call.v = v; call.out = out; call.dout = dout; call.lse = lse;
    call.dq = dq; call.dk = dk; call.dv = dv;
    call.work = (float *)work;
    call.l = layouts;
    call.scale = scale;
    XattnDevice dev(devID);
    if (!dev.ok)
        return NTB_ERR_CUDA;
    DeviceCtx * ctx = CtxFor(devID);
    if (!ctx)
        return NTB_ERR_CUDA;
    if (XattnGradIsShort(*ctx, call.sh))
        rc = LaunchXattnGradShort(*ctx, call, (cudaStream_t)stream);
    else if (lenQ > 0 && (long long)call.sh.group * lenQ <= XATTN_STEP_ROWS)
        rc = LaunchXattnGradStep(*ctx, call, (cudaStream_t)stream);
    else
        rc = dim <= 64 ? LaunchGrad<64>(*ctx, call, (cudaStream_t)stream) : LaunchGrad<128>(*ctx, call, (cudaStream_t)stream);
    if (rc == NTB_ERR_CUDA)
        cudaGetLastError();
    return rc;
}
