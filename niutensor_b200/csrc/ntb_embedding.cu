/*
 * Embedding rows and their gradient (source/sample/transformer/submodel/Embedding.cpp: the rows of a word
 * matrix picked by token ids, times sqrt(d), plus the rows of the positions).
 *
 * Forward: out[t] = scale * w[ids[t]] + pos[t % posRows], one warp a token, 16-byte accesses, one rounding.
 * It is bound by its reads and writes: 32768 tokens of 1024 floats take 30 us, 171 MB at 5.7 TB/s.
 *
 * Gradient: dw[v] = beta dw[v] + scale * sum over the tokens t with ids[t] = v, t ascending, of dout[t].
 * Adding every row with atomics would sum in an order that changes from run to run and serialise on
 * frequent words, so the tokens are sorted first and equal words summed as runs:
 *
 *   TokenSortKernel   a stable radix sort of (id, t) in ONE launch: one cluster of CTAs, digits of at most
 *                     9 bits. Every CTA owns a contiguous part of the list; per pass it counts its digits, the
 *                     counts are prefixed over the cluster's CTAs through distributed shared memory, and the
 *                     part, tile by tile, is ranked (a warp its own piece, 32 tokens at a time), put in its new
 *                     order in shared memory and written out from there. The steps are separated by the
 *                     hardware's cluster barrier. Meanwhile the other CTAs of the grid clear dw (beta = 0).
 *   RunSumKernel      the sorted list cut into equal blocks, whatever the words' frequencies; a thread owns
 *                     16 bytes of the columns and adds the rows of a block one after the other. Runs inside a
 *                     block go straight to dw, pieces of runs that cross an edge to fp32 partial rows.
 *   RunJoinKernel     adds up the pieces of a crossing run, in block order.
 *
 * Up to FEW_TOKENS tokens (half as many without 16-byte accesses): FewTokensKernel, one launch without a workspace. The first token of a word finds its
 * others by looking through the list in shared memory and adds their rows; other CTAs meanwhile clear the rows
 * of dw whose words do not occur (beta = 0), known from a bit map of the list.
 *
 * Bound by the reads of dout and the writes of dw at large sizes (100000 tokens of 1024 floats, 32000 words: 133 us,
 * 541 MB at 4.1 TB/s, of which the sort is 41), by the launches' latency at small ones (4096 tokens of 512 halves: 25).
 *
 * Sums are fp32 in a fixed order. Ids outside [0, vocab) stand for no word.
 */
#include "ntb_xattn.cuh"

namespace ntb {

namespace {

constexpr int EM_THREADS = 256;
constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_MAX_BITS = 9, SORT_RADIX = 1 << SORT_MAX_BITS;
constexpr int SORT_AHEAD = 8;             /* tokens a thread holds at once */
constexpr int SORT_TILE = SORT_THREADS * SORT_AHEAD;
constexpr int SORT_CTAS = 16;             /* largest cluster */
static_assert(SORT_RADIX <= SORT_THREADS, "a thread a digit");

template <typename T> struct EmVec;
template <> struct EmVec<__half> { static constexpr int N = 8; };
template <> struct EmVec<float> { static constexpr int N = 4; };

__device__ __forceinline__ void UnpackRow(const uint4 & u, float * v, const __half *)
{
    const uint32_t x[4] = { u.x, u.y, u.z, u.w };
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*(const __half2 *)&x[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void UnpackRow(const uint4 & u, float * v, const float *)
{
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ uint4 PackRow(const float * v, const __half *)
{
    return make_uint4(PackHalf2(v[0], v[1]), PackHalf2(v[2], v[3]), PackHalf2(v[4], v[5]), PackHalf2(v[6], v[7]));
}
__device__ __forceinline__ uint4 PackRow(const float * v, const float *)
{
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ float Get(const __half * p) { return __half2float(*p); }
__device__ __forceinline__ float Get(const float * p) { return *p; }
__device__ __forceinline__ void Put(__half * p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void Put(float * p, float v) { *p = v; }

template <typename T>
__global__ void __launch_bounds__(EM_THREADS) EmbeddingKernel(const int * ids, const T * w, const T * pos, T * out, int tokens, int vocab, int dim,
                                                              long long ldw, long long ldo, int posRows, float scale, bool vec)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int N = EmVec<T>::N;
    const int lane = threadIdx.x & 31;
    const long long t = (long long)blockIdx.x * (EM_THREADS / 32) + (threadIdx.x >> 5);
    if (t >= tokens)
        return;
    const int id = ids[t];
    const bool word = id >= 0 && id < vocab;
    const T * row = w + (word ? id : 0) * ldw;
    const T * at = pos != nullptr ? pos + (t % posRows) * dim : nullptr;
    T * dst = out + t * ldo;
    if (vec) {
        const int packs = dim / N;
        for (int i0 = lane; i0 < packs; i0 += 128) {
            uint4 a[4], b[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * 32;
                a[u] = b[u] = make_uint4(0u, 0u, 0u, 0u);
                if (i < packs) {
                    if (word)
                        a[u] = ((const uint4 *)row)[i];
                    if (at != nullptr)
                        b[u] = ((const uint4 *)at)[i];
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * 32;
                if (i < packs) {
                    float x[N], y[N];
                    UnpackRow(a[u], x, (const T *)nullptr);
                    UnpackRow(b[u], y, (const T *)nullptr);
#pragma unroll
                    for (int e = 0; e < N; e++)
                        x[e] = fmaf(x[e], scale, y[e]);
                    ((uint4 *)dst)[i] = PackRow(x, (const T *)nullptr);
                }
            }
        }
    }
    else {
        for (int i = lane; i < dim; i += 32)
            Put(dst + i, fmaf(word ? Get(row + i) : 0.f, scale, at != nullptr ? Get(at + i) : 0.f));
    }
}

/* ---------------------------------------------------------------- sort */

struct SortParams {
    const int * ids;
    int2 * a;               /* ping and pong of (id or vocab, token); the last pass writes a */
    int2 * b;
    int tokens, vocab;
    int passes, bits;       /* digits of `bits` bits, lowest first */
    int ctas;               /* the cluster that sorts */
    /* rows the other CTAs clear, or NULL */
    unsigned char * clear;
    int clearRows;
    long long clearPitch, clearBytes;      /* bytes between rows, bytes of a row */
};

/* bytes [p, p + n) become zeros, by one warp */
__device__ __forceinline__ void ClearWarp(unsigned char * p, long long n, int lane)
{
    const long long head = (16 - ((uintptr_t)p & 15)) & 15;
    if (head >= n) {
        for (long long i = lane; i < n; i += 32)
            p[i] = 0;
        return;
    }
    if (lane < head)
        p[lane] = 0;
    uint4 * v = (uint4 *)(p + head);
    const long long packs = (n - head) / 16;
    for (long long i = lane; i < packs; i += 32)
        v[i] = make_uint4(0u, 0u, 0u, 0u);
    const long long done = head + packs * 16;
    if (done + lane < n)
        p[done + lane] = 0;
}

/* the lanes whose digit equals this lane's: one ballot a bit (a 32-bit match instruction took several times as long) */
__device__ __forceinline__ unsigned SameDigit(int d, int bits, bool in)
{
    unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
    for (int b = 0; b < SORT_MAX_BITS; b++) {
        if (b < bits) {
            const bool set = ((d >> b) & 1) != 0;
            const unsigned vote = __ballot_sync(0xffffffffu, set);
            same &= set ? vote : ~vote;
        }
    }
    return same;
}

/* exclusive sum over the block's first R threads' values; every thread calls */
__device__ __forceinline__ int BlockScan(int value, int * warpSums, int warp, int lane)
{
    int scan = value;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, scan, off);
        if (lane >= off)
            scan += o;
    }
    if (lane == 31)
        warpSums[warp] = scan;
    __syncthreads();
    const int lower = __reduce_add_sync(0xffffffffu, lane < warp ? warpSums[lane] : 0);
    return lower + scan - value;
}

__global__ void __launch_bounds__(SORT_THREADS) TokenSortKernel(const SortParams p)
{
    extern __shared__ __align__(16) unsigned char sortSmem[];
    __shared__ int totals[SORT_RADIX], bases[SORT_RADIX], localBases[SORT_RADIX], warpSums[2][SORT_WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if ((int)blockIdx.x >= p.ctas) {
        const long long warps = (long long)(gridDim.x - p.ctas) * SORT_WARPS;
        const long long first = (long long)(blockIdx.x - p.ctas) * SORT_WARPS + warp;
        if (p.clearPitch == p.clearBytes) {
            const long long all = p.clearPitch * p.clearRows;
            const long long piece = 4096;
            for (long long o = first * piece; o < all; o += warps * piece)
                ClearWarp(p.clear + o, all - o < piece ? all - o : piece, lane);
        }
        else {
            for (long long r = first; r < p.clearRows; r += warps)
                ClearWarp(p.clear + r * p.clearPitch, p.clearBytes, lane);
        }
        return;
    }
    const int R = 1 << p.bits;
    int2 * stage = (int2 *)sortSmem;                              /* a tile in its new order */
    int * counters = (int *)(stage + SORT_TILE);                  /* [warp][digit] */
    int * mine = counters + warp * R;
    const int rank = (int)blockIdx.x;
    /* this CTA's part of the list */
    const long long per = (p.tokens + p.ctas - 1) / p.ctas;
    const long long lo = rank * per < p.tokens ? rank * per : p.tokens;
    const long long hi = lo + per < p.tokens ? lo + per : p.tokens;
    const unsigned before = (1u << lane) - 1u;
    const bool once = hi - lo <= SORT_TILE;                       /* a part of one tile is loaded once a pass */

    for (int pass = 0; pass < p.passes; pass++) {
        const int shift = pass * p.bits;
        /* the last pass writes a */
        int2 * dst = ((p.passes - 1 - pass) & 1) == 0 ? p.a : p.b;
        const int2 * src = dst == p.a ? p.b : p.a;
        auto load = [&](long long i) -> int2 {
            if (pass == 0) {
                const int id = p.ids[i];
                return make_int2(id >= 0 && id < p.vocab ? id : p.vocab, (int)i);
            }
            return __ldcg(src + i);
        };
        auto digit = [&](const int2 & x) { return (x.x >> shift) & (R - 1); };
        /* a warp's tokens lie one behind the other: ranks within a digit follow the list's order */
        int2 x[SORT_AHEAD];
        int count = 0, each = 0;                                  /* of a tile; steps of 32 a warp */
        auto loadTile = [&](long long tile) {
            count = hi - tile < SORT_TILE ? (int)(hi - tile) : SORT_TILE;
            each = (count + SORT_WARPS * 32 - 1) / (SORT_WARPS * 32);
#pragma unroll
            for (int u = 0; u < SORT_AHEAD; u++) {
                const int i = (warp * each + u) * 32 + lane;
                x[u] = u < each && i < count ? load(tile + i) : make_int2(0, 0);
            }
        };
        int place[SORT_AHEAD];
        /* ranks of the tile's tokens among those of their digit in the warp's piece, and those of all pieces before it
           (counters); returns how many tokens the tile has of the thread's digit */
        auto rankTile = [&]() {
            for (int i = threadIdx.x; i < SORT_WARPS * R / 4; i += SORT_THREADS)
                ((int4 *)counters)[i] = make_int4(0, 0, 0, 0);
            __syncthreads();
#pragma unroll
            for (int u = 0; u < SORT_AHEAD; u++) {
                if (u < each) {
                    const bool in = (warp * each + u) * 32 + lane < count;
                    const int d = digit(x[u]);
                    const unsigned same = SameDigit(d, p.bits, in);
                    place[u] = mine[d] + __popc(same & before);
                    __syncwarp();
                    if (in && (same & before) == 0)
                        mine[d] += __popc(same);
                    __syncwarp();
                }
            }
            __syncthreads();
            int run = 0;
            if ((int)threadIdx.x < R) {
                int c[SORT_WARPS];
#pragma unroll
                for (int w = 0; w < SORT_WARPS; w++)
                    c[w] = counters[w * R + threadIdx.x];
#pragma unroll
                for (int w = 0; w < SORT_WARPS; w++) {
                    counters[w * R + threadIdx.x] = run;
                    run += c[w];
                }
            }
            return run;
        };
        int run = 0;
        if (once) {
            /* the ranking counts the digits, too */
            loadTile(lo);
            run = rankTile();
            if ((int)threadIdx.x < R)
                totals[threadIdx.x] = run;
        }
        else {
            if ((int)threadIdx.x < R)
                totals[threadIdx.x] = 0;
            __syncthreads();
            for (long long i0 = lo + threadIdx.x; i0 < hi; i0 += SORT_TILE) {
                int d[SORT_AHEAD];
#pragma unroll
                for (int u = 0; u < SORT_AHEAD; u++)
                    d[u] = i0 + u * SORT_THREADS < hi ? digit(load(i0 + u * SORT_THREADS)) : -1;
#pragma unroll
                for (int u = 0; u < SORT_AHEAD; u++)
                    if (d[u] >= 0)
                        atomicAdd(totals + d[u], 1);
            }
        }
        ClusterSync();
        /* where a digit's tokens start: all smaller digits, then the same digit in the CTAs before this one */
        int all = 0, ahead = 0;
        if ((int)threadIdx.x < R) {
            int n[SORT_CTAS];
#pragma unroll
            for (int c = 0; c < SORT_CTAS; c++) {
                n[c] = 0;
                if (c < p.ctas)
                    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n[c]) : "r"(MapShared(SmemAddr(totals + threadIdx.x), c)) : "memory");
            }
#pragma unroll
            for (int c = 0; c < SORT_CTAS; c++) {
                all += n[c];
                ahead += c < rank ? n[c] : 0;
            }
        }
        const int start = BlockScan(all, warpSums[0], warp, lane) + ahead;
        if ((int)threadIdx.x < R)
            bases[threadIdx.x] = start;

        for (long long tile = lo; tile < hi; tile += SORT_TILE) {
            if (!once) {
                loadTile(tile);
                run = rankTile();
            }
            const int local = BlockScan(run, warpSums[1], warp, lane);
            if ((int)threadIdx.x < R)
                localBases[threadIdx.x] = local;
            __syncthreads();
#pragma unroll
            for (int u = 0; u < SORT_AHEAD; u++)
                if (u < each && (warp * each + u) * 32 + lane < count) {
                    const int d = digit(x[u]);
                    stage[localBases[d] + mine[d] + place[u]] = x[u];
                }
            __syncthreads();
            /* in the new order neighbours go to neighbouring places: whole lines instead of one store a token */
            for (int i = threadIdx.x; i < count; i += SORT_THREADS) {
                const int2 y = stage[i];
                const int d = digit(y);
                __stcg(dst + bases[d] + i - localBases[d], y);
            }
            __syncthreads();
            if ((int)threadIdx.x < R)
                bases[threadIdx.x] += run;
        }
        /* the list in its new order is complete, and the totals have been read, before the next pass */
        ClusterSync();
    }
}

/* ---------------------------------------------------------------- runs */

struct RunParams {
    const int2 * sorted;
    const void * dout;
    void * dw;
    float * head;           /* [block][dim]: the piece of a run that began before the block */
    float * tail;           /* [block][dim]: the piece of a run that begins in the block and goes on behind it */
    int tokens, vocab, dim, block, blocks;
    long long ldo, ldw;
    float scale;
    int accumulate;
};

/* one column of a run's sum into dw */
template <typename TW>
__device__ __forceinline__ void WriteColumn(const RunParams & p, int id, int col, float acc)
{
    TW * dst = (TW *)p.dw + id * p.ldw + col;
    Put(dst, fmaf(acc, p.scale, p.accumulate ? Get(dst) : 0.f));
}

/*
 * VEC: 16-byte loads of dout, 16-byte accesses to dw; else one column a thread. ACC: the old rows of dw are added.
 * A thread walks its block's tokens with the loads of U of them in flight together (with ACC those of the old
 * rows where a word ends, too: loaded at the point of use, 100000 tokens of 512 halves took 140 us instead of 85);
 * the adds stay in order. Narrow rows have few bytes in flight: with 16 loads instead of 8 (4 without wide accesses) and as
 * many pieces of a frequent word at a time, 48420 tokens of 256 halves take 31.7 us instead of 34, 60000 of 513 floats 76 instead of 81.
 */
template <typename TO, typename TW, bool VEC, bool ACC>
__global__ void RunSumKernel(const RunParams p)
{
    constexpr int N = VEC ? EmVec<TO>::N : 1;
    constexpr int WN = VEC ? N / EmVec<TW>::N : 1;            /* 16-byte pieces of dw a thread owns */
    extern __shared__ int2 items[];                           /* the block's tokens, with the words before and behind it */
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long begin = (long long)blockIdx.x * p.block;
    const int n = p.tokens - begin < p.block ? (int)(p.tokens - begin) : p.block;
    for (int i = threadIdx.x; i < n + 2; i += blockDim.x) {
        const long long at = begin + i - 1;
        items[i] = at >= 0 && at < p.tokens ? p.sorted[at] : make_int2(-1, 0);
    }
    __syncthreads();
    const int col = (blockIdx.y * blockDim.x + threadIdx.x) * N;
    if (col >= p.dim)
        return;
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; e++)
        acc[e] = 0.f;
    bool fromBefore = items[0].x == items[1].x;
    const int2 * it = items + 1;
    constexpr int U = VEC && !ACC ? 16 : 8;
    for (int i0 = 0; i0 < n; i0 += U) {
        uint4 raw[VEC ? U : 1], oldRaw[VEC && ACC ? U * WN : 1];
        float one[VEC ? 1 : U], oldOne[!VEC && ACC ? U : 1];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u < n ? i0 + u : n - 1;
            const TO * src = (const TO *)p.dout + it[i].y * p.ldo + col;
            if (VEC)
                raw[u] = __ldcs((const uint4 *)src);
            else
                one[u] = Get(src);
            if (ACC) {
                const int id = it[i].x;
                const bool ends = id != it[i + 1].x && id != p.vocab;
                const TW * dst = (const TW *)p.dw + (ends ? id : 0) * p.ldw + col;
                if (VEC) {
#pragma unroll
                    for (int k = 0; k < WN; k++)
                        if (ends)
                            oldRaw[u * WN + k] = ((const uint4 *)dst)[k];
                }
                else
                    oldOne[u] = ends ? Get(dst) : 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u;
            if (i < n) {
                if (VEC) {
                    float v[EmVec<TO>::N];
                    UnpackRow(raw[u], v, (const TO *)nullptr);
#pragma unroll
                    for (int e = 0; e < N; e++)
                        acc[e] += v[e];
                }
                else
                    acc[0] += one[u];
                const int id = it[i].x, next = it[i + 1].x;
                if (id != next || i == n - 1) {
                    if (id != p.vocab) {
                        const bool goesOn = id == next;             /* only behind the block's last token */
                        if (fromBefore || goesOn) {
                            float * dst = (fromBefore ? p.head : p.tail) + (long long)blockIdx.x * p.dim + col;
#pragma unroll
                            for (int e = 0; e < N; e++)
                                dst[e] = acc[e];
                        }
                        else if (VEC) {
                            TW * dst = (TW *)p.dw + id * p.ldw + col;
                            constexpr int PN = EmVec<TW>::N;
#pragma unroll
                            for (int k = 0; k < WN; k++) {
                                float v[PN];
                                if (ACC)
                                    UnpackRow(oldRaw[u * WN + k], v, (const TW *)nullptr);
#pragma unroll
                                for (int e = 0; e < PN; e++)
                                    v[e] = fmaf(acc[(k * PN + e) % N], p.scale, ACC ? v[e] : 0.f);
                                ((uint4 *)dst)[k] = PackRow(v, (const TW *)nullptr);
                            }
                        }
                        else
                            Put((TW *)p.dw + id * p.ldw + col, fmaf(acc[0], p.scale, ACC ? oldOne[u] : 0.f));
                    }
#pragma unroll
                    for (int e = 0; e < N; e++)
                        acc[e] = 0.f;
                    fromBefore = false;
                }
            }
        }
    }
}

/* ---------------------------------------------------------------- few tokens */

/* Whole gradient, us in graph replay, few-tokens kernel / sort and runs, vocabulary 32000 of 512 halves and 5000 of
   1024: 256 tokens 7.2 / 14.4 and 5.3; 1000 8.8 / 16.0 and 7.9; 2048 11.4 / 18.0 and 14.7; 4096 19.8 / 19.4 and
   30.6 / 23.8 (the search grows with the square of the list). Rows without wide accesses (300 halves, 20000 words of
   513 floats): 1000 tokens 13 / 19 and 16 / 21, 2048 20 / 19 and 26 / 21, so half as many there. */
constexpr int FEW_TOKENS = 2048;
constexpr int FEW_THREADS = 256, FEW_WARPS = FEW_THREADS / 32;
constexpr int FEW_LIST = 24;              /* tokens of a word up to which one warp adds them all */
constexpr int FEW_CLEAR_ROWS = 4096;      /* rows of dw a clearing CTA looks after at a time: its bit map */

/* columns of a CTA: 16 bytes a lane, or four columns a lane one at a time */
template <int N> constexpr int FEW_COLS = N > 1 ? 32 * N : 128;

struct FewParams {
    const int * ids;
    const void * dout;
    void * dw;
    int tokens, vocab, dim;
    long long ldo, ldw;
    float scale;
    int accumulate;
    int sumCtas, colBlocks;   /* sumCtas x colBlocks CTAs sum; the others clear */
};

/* the rows at[0 .. n) of dout, one after the other, into N columns of dw's row id */
template <typename TO, typename TW, bool VEC>
__device__ __forceinline__ void AddRows(const FewParams & p, const unsigned short * at, int n, int col, float * acc)
{
    constexpr int N = VEC ? EmVec<TO>::N : 1;
    constexpr int U = 8;
    for (int i0 = 0; i0 < n; i0 += U) {
        uint4 raw[VEC ? U : 1];
        float one[VEC ? 1 : U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const TO * src = (const TO *)p.dout + (long long)at[i0 + u < n ? i0 + u : n - 1] * p.ldo + col;
            if (VEC)
                raw[u] = *(const uint4 *)src;
            else
                one[u] = Get(src);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i0 + u < n) {
                if (VEC) {
                    float v[EmVec<TO>::N];
                    UnpackRow(raw[u], v, (const TO *)nullptr);
#pragma unroll
                    for (int e = 0; e < N; e++)
                        acc[e] += v[e];
                }
                else
                    acc[0] += one[u];
            }
    }
}

template <typename TO, typename TW, bool VEC>
__device__ __forceinline__ void PutRow(const FewParams & p, int id, int col, const float * acc)
{
    constexpr int N = VEC ? EmVec<TO>::N : 1;
    TW * dst = (TW *)p.dw + id * p.ldw + col;
    if (VEC) {
        constexpr int PN = EmVec<TW>::N;
#pragma unroll
        for (int k = 0; k < N; k += PN) {
            float v[PN];
#pragma unroll
            for (int e = 0; e < PN; e++)
                v[e] = 0.f;
            if (p.accumulate)
                UnpackRow(*(const uint4 *)(dst + k), v, (const TW *)nullptr);
#pragma unroll
            for (int e = 0; e < PN; e++)
                v[e] = fmaf(acc[(k + e) % N], p.scale, v[e]);
            *(uint4 *)(dst + k) = PackRow(v, (const TW *)nullptr);
        }
    }
    else
        Put(dst, fmaf(acc[0], p.scale, p.accumulate ? Get(dst) : 0.f));
}

template <typename TO, typename TW, bool VEC>
__global__ void __launch_bounds__(FEW_THREADS) FewTokensKernel(const FewParams p)
{
    constexpr int N = VEC ? EmVec<TO>::N : 1;
    __shared__ __align__(16) int words[FEW_TOKENS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int block = blockIdx.x % (p.sumCtas > 0 ? p.sumCtas : 1);
    if ((int)blockIdx.x >= p.sumCtas * p.colBlocks) {
        /* clear the rows of the words that do not occur */
        unsigned * seen = (unsigned *)words;
        const int ctas = gridDim.x - p.sumCtas * p.colBlocks;
        const int each = (int)(((long long)p.vocab + ctas - 1) / ctas);
        const long long first = (long long)(blockIdx.x - p.sumCtas * p.colBlocks) * each;
        const int end = first + each < p.vocab ? (int)(first + each) : p.vocab;
        for (long long lo64 = first; lo64 < end; lo64 += FEW_CLEAR_ROWS) {
            const int lo = (int)lo64, hi = end - lo < FEW_CLEAR_ROWS ? end : lo + FEW_CLEAR_ROWS;
            __syncthreads();
            for (int i = threadIdx.x; i < FEW_CLEAR_ROWS / 32; i += FEW_THREADS)
                seen[i] = 0u;
            __syncthreads();
            for (int i = threadIdx.x; i < p.tokens; i += FEW_THREADS) {
                const int id = p.ids[i];
                if (id >= lo && id < hi)
                    atomicOr(seen + ((id - lo) >> 5), 1u << ((id - lo) & 31));
            }
            __syncthreads();
            for (long long v = lo + warp; v < hi; v += FEW_WARPS)           /* it passes hi, which may be 2^31 - 2 */
                if (((seen[(v - lo) >> 5] >> ((v - lo) & 31)) & 1u) == 0u)
                    ClearWarp((unsigned char *)((TW *)p.dw + v * p.ldw), (long long)p.dim * sizeof(TW), lane);
        }
        return;
    }
    __shared__ unsigned short lists[FEW_WARPS][FEW_LIST];
    __shared__ int counts[FEW_WARPS];
    __shared__ float parts[FEW_WARPS][32 * (VEC ? EmVec<TO>::N : 1)];
    /* whole steps of 256: what lies behind the list is no word */
    for (int i = threadIdx.x; i < (p.tokens + 255) / 256 * 256; i += FEW_THREADS)
        words[i] = i < p.tokens ? p.ids[i] : -1;
    __syncthreads();
    /* a warp a token: if the word has no earlier token, how many it has, and the first of them. Frequent words occur
       early: neighbours in the list go to different CTAs. */
    const unsigned before = (1u << lane) - 1u;
    const int t = warp * p.sumCtas + block;
    const int colLo = blockIdx.x / p.sumCtas * FEW_COLS<N>, colHi = colLo + FEW_COLS<N> < p.dim ? colLo + FEW_COLS<N> : p.dim;
    int count = 0;
    if (t < p.tokens) {
        const int id = words[t];
        if (id >= 0 && id < p.vocab) {
            /* four tokens a lane at a time: most steps find nothing */
            bool earlier = false;
            for (int i0 = 0; i0 < t && !earlier; i0 += 256) {
                const int i = i0 + lane * 4;
                const int4 a = *(const int4 *)(words + i), b = *(const int4 *)(words + i + 128);
                const bool hit = (a.x == id && i < t) || (a.y == id && i + 1 < t) || (a.z == id && i + 2 < t) || (a.w == id && i + 3 < t) ||
                                 (b.x == id && i + 128 < t) || (b.y == id && i + 129 < t) || (b.z == id && i + 130 < t) || (b.w == id && i + 131 < t);
                earlier = __any_sync(0xffffffffu, hit);
            }
            if (!earlier)
                for (int i0 = t & ~127; i0 < p.tokens; i0 += 128) {
                    const int i = i0 + lane * 4;
                    const int4 a = *(const int4 *)(words + i);
                    const bool h[4] = { a.x == id && i >= t, a.y == id && i + 1 >= t, a.z == id && i + 2 >= t, a.w == id && i + 3 >= t };
                    if (!__any_sync(0xffffffffu, h[0] || h[1] || h[2] || h[3]))
                        continue;
                    int place = count;
                    unsigned votes = 0;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const unsigned vote = __ballot_sync(0xffffffffu, h[k]);
                        place += __popc(vote & before);
                        votes += __popc(vote);
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (h[k]) {
                            if (place < FEW_LIST)
                                lists[warp][place] = (unsigned short)(i + k);
                            place++;
                        }
                    count += votes;
                }
        }
    }
    if (lane == 0)
        counts[warp] = count;
    __syncwarp();
    if (count > 0 && count <= FEW_LIST)
        for (int col = colLo + lane * N; col < colHi; col += 32 * N) {
            float acc[N];
#pragma unroll
            for (int e = 0; e < N; e++)
                acc[e] = 0.f;
            AddRows<TO, TW, VEC>(p, lists[warp], count, col, acc);
            PutRow<TO, TW, VEC>(p, words[t], col, acc);
        }
    __syncthreads();
    /* frequent words, one after the other: the CTA's warps share the list in equal pieces */
    for (int w = 0; w < FEW_WARPS; w++) {
        if (counts[w] <= FEW_LIST)
            continue;
        const int id = words[w * p.sumCtas + block];
        const int each = ((p.tokens + FEW_WARPS - 1) / FEW_WARPS + 31) / 32 * 32;
        const int lo = warp * each, hi = lo + each < p.tokens ? lo + each : p.tokens;
        for (int col0 = colLo; col0 < colHi; col0 += 32 * N) {
            const int col = col0 + lane * N;
            float acc[N];
#pragma unroll
            for (int e = 0; e < N; e++)
                acc[e] = 0.f;
            int have = 0;
            for (int i0 = lo; i0 < hi || have > 0; i0 += 32) {
                unsigned vote = 0u;
                if (i0 < hi) {
                    const int i = i0 + lane;
                    const bool hit = i < hi && words[i] == id;
                    vote = __ballot_sync(0xffffffffu, hit);
                }
                /* the list takes 24: a step of 32 tokens is taken in two halves */
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const unsigned bits = half == 0 ? vote & 0xffffu : vote >> 16;
                    if (have + __popc(bits) > FEW_LIST || (i0 >= hi && have > 0)) {
                        __syncwarp();
                        if (col < colHi)
                            AddRows<TO, TW, VEC>(p, lists[warp], have, col, acc);
                        have = 0;
                        __syncwarp();
                    }
                    if (lane < 16 && ((bits >> lane) & 1u))
                        lists[warp][have + __popc(bits & ((1u << lane) - 1u))] = (unsigned short)(i0 + half * 16 + lane);
                    have += __popc(bits);
                }
            }
#pragma unroll
            for (int e = 0; e < N; e++)
                parts[warp][lane * N + e] = acc[e];
            __syncthreads();
            if (warp == 0 && col < colHi) {
                for (int k = 1; k < FEW_WARPS; k++)
#pragma unroll
                    for (int e = 0; e < N; e++)
                        acc[e] += parts[k][lane * N + e];
                PutRow<TO, TW, VEC>(p, id, col, acc);
            }
            __syncthreads();
        }
    }
}

template <typename TO, typename TW>
cudaError_t LaunchFew(FewParams p, bool vec, int clearing, cudaStream_t stream)
{
    const int cols = vec ? FEW_COLS<EmVec<TO>::N> : FEW_COLS<1>;
    p.colBlocks = (p.dim + cols - 1) / cols;
    const long long grid = (long long)p.sumCtas * p.colBlocks + clearing;
    const cudaError_t err = vec ? LaunchPdl(FewTokensKernel<TO, TW, true>, (int)grid, FEW_THREADS, 0, stream, p)
                                : LaunchPdl(FewTokensKernel<TO, TW, false>, (int)grid, FEW_THREADS, 0, stream, p);
    CountLaunch();
    return err;
}

/* block i: the run, if any, that begins in block i of the list and goes on behind it */
template <typename TW>
__global__ void RunJoinKernel(const RunParams p)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int i = blockIdx.x;
    const long long end = (long long)(i + 1) * p.block;       /* the list goes on: the last block has no CTA here */
    const int id = p.sorted[end - 1].x;
    if (id == p.vocab || p.sorted[end].x != id)
        return;
    const long long begin = (long long)i * p.block;
    if (i > 0 && p.sorted[begin - 1].x == id)
        return;                                                /* it began in an earlier block */
    /* the first of the following blocks whose last token is another word (the list is sorted), or the last block:
       32 probes at a time, so that a long list takes two rounds of memory latency and not ten */
    int lo = i + 1, hi = p.blocks - 1;
    const int lane = threadIdx.x & 31;
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32;
        const int probe = lo + lane * step;
        bool goesOn = false;
        if (probe < hi)
            goesOn = p.sorted[(long long)(probe + 1) * p.block - 1].x == id;
        const int n = __popc(__ballot_sync(0xffffffffu, goesOn));         /* probes 0 .. n - 1 go on */
        const int from = n == 0 ? lo : lo + (n - 1) * step + 1;
        const int to = lo + n * step < hi ? lo + n * step : hi;
        lo = from;
        hi = n == 0 ? lo : to;
    }
    /* block lo begins with the run, or is behind a run that ended with block lo - 1 */
    const int stop = p.sorted[(long long)lo * p.block].x == id ? lo : lo - 1;
    for (int col = blockIdx.y * blockDim.x + threadIdx.x; col < p.dim; col += gridDim.y * blockDim.x) {
        float acc = p.tail[(long long)i * p.dim + col];
        int j = i + 1;
        for (; j + 15 <= stop; j += 16) {
            float v[16];
#pragma unroll
            for (int u = 0; u < 16; u++)
                v[u] = p.head[(long long)(j + u) * p.dim + col];
#pragma unroll
            for (int u = 0; u < 16; u++)
                acc += v[u];
        }
        for (; j <= stop; j++)
            acc += p.head[(long long)j * p.dim + col];
        WriteColumn<TW>(p, id, col, acc);
    }
}

/* tokens of one block of the sorted list: about four blocks an SM, few enough pieces of a frequent word to join */
int RunBlock(int tokens)
{
    int block = 8;
    while (block < 256 && (long long)block * 592 < tokens)
        block *= 2;
    return block;
}

/* CTAs that sort. Whole call on a B200 with 512 halves a row, us in graph replay with 4 / 8 / 16 CTAs: 4096 tokens
   22.6 / 19.8 / 20.2, 8192 27 / 22 / 22, 20000 48 / 33 / 32, 100000 185 / 109 / 85. */
int SortCtas(int tokens)
{
    return tokens <= 16384 ? 8 : SORT_CTAS;
}

/* column indices run up to a CTA's columns past the end in 32 bits */
constexpr int EM_MOST_COLS = 0x7fffff00;

bool RowsAligned(const void * p, long long pitch, int dim, int size)
{
    return ((uintptr_t)p & 15) == 0 && (pitch * size) % 16 == 0 && (dim * (long long)size) % 16 == 0;
}

template <typename TO, typename TW>
bool WideRows(const void * dout, long long ldo, const void * dw, long long ldw, int dim)
{
    return RowsAligned(dout, ldo, dim, sizeof(TO)) && RowsAligned(dw, ldw, dim, sizeof(TW)) && dim % EmVec<TO>::N == 0;
}

template <typename TO, typename TW>
cudaError_t LaunchRuns(const RunParams & p, bool vec, cudaStream_t stream)
{
    const int threadsNeeded = vec ? p.dim / EmVec<TO>::N : p.dim;
    const int block = threadsNeeded >= 256 ? 256 : (threadsNeeded + 31) / 32 * 32;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.blocks, (unsigned)((threadsNeeded + block - 1) / block), 1);
    cfg.blockDim = dim3((unsigned)block, 1, 1);
    cfg.dynamicSmemBytes = (p.block + 2) * sizeof(int2);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PdlEnabled() ? 1 : 0;
    cudaError_t err = p.accumulate
        ? (vec ? cudaLaunchKernelEx(&cfg, RunSumKernel<TO, TW, true, true>, p) : cudaLaunchKernelEx(&cfg, RunSumKernel<TO, TW, false, true>, p))
        : (vec ? cudaLaunchKernelEx(&cfg, RunSumKernel<TO, TW, true, false>, p) : cudaLaunchKernelEx(&cfg, RunSumKernel<TO, TW, false, false>, p));
    CountLaunch();
    if (err != cudaSuccess || p.blocks == 1)
        return err;
    cfg.gridDim = dim3((unsigned)(p.blocks - 1), (unsigned)((p.dim + 255) / 256 < 8 ? (p.dim + 255) / 256 : 8), 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.dynamicSmemBytes = 0;
    err = cudaLaunchKernelEx(&cfg, RunJoinKernel<TW>, p);
    CountLaunch();
    return err;
}

}

}

using namespace ntb;

extern "C" int ntb_embedding(int devID, void * stream, const int * ids, const void * w, const void * pos, void * out,
                             int dtype, int tokens, int vocab, int dim, long long ldw, long long ldo, int posRows, float scale)
{
    if (tokens < 0 || vocab < 0 || dim < 0 || ldw < dim || ldo < dim || (pos != nullptr && posRows < 1))
        return NTB_ERR_ARG;
    if (dtype != NTB_X_FLOAT16 && dtype != NTB_X_FLOAT)
        return NTB_ERR_DTYPE;
    if (tokens == 0 || dim == 0)
        return NTB_OK;
    if (!ids || !out || (vocab > 0 && !w))
        return NTB_ERR_ARG;
    if (dim > EM_MOST_COLS)
        return NTB_ERR_LIMIT;
    XattnDevice dev(devID);
    if (!dev.ok)
        return NTB_ERR_CUDA;
    cudaStream_t st = (cudaStream_t)stream;
    const int es = dtype == NTB_X_FLOAT16 ? 2 : 4;
    const bool vec = RowsAligned(w, ldw, dim, es) && RowsAligned(out, ldo, dim, es) && (pos == nullptr || RowsAligned(pos, dim, dim, es));
    const int grid = (int)(((long long)tokens + EM_THREADS / 32 - 1) / (EM_THREADS / 32));
    const cudaError_t err = dtype == NTB_X_FLOAT16
        ? LaunchPdl(EmbeddingKernel<__half>, grid, EM_THREADS, 0, st, ids, (const __half *)w, (const __half *)pos, (__half *)out, tokens, vocab, dim,
                    ldw, ldo, posRows, scale, vec)
        : LaunchPdl(EmbeddingKernel<float>, grid, EM_THREADS, 0, st, ids, (const float *)w, (const float *)pos, (float *)out, tokens, vocab, dim,
                    ldw, ldo, posRows, scale, vec);
    CountLaunch();
    if (err == cudaSuccess && cudaGetLastError() == cudaSuccess)
        return NTB_OK;
    cudaGetLastError();
    return NTB_ERR_CUDA;
}

extern "C" long long ntb_embedding_grad_work(int tokens, int dim)
{
    if (tokens < 0 || dim < 0)
        return 0;
    const long long block = RunBlock(tokens), blocks = (tokens + block - 1) / block;
    return (long long)tokens * 2 * (long long)sizeof(int2) + blocks * dim * 2 * (long long)sizeof(float);
}

extern "C" int ntb_embedding_grad(int devID, void * stream, const int * ids, const void * dout, void * dw, int dtypeOut, int dtypeW,
                                  int tokens, int vocab, int dim, long long ldo, long long ldw, float scale, float beta,
                                  void * work, long long workBytes)
{
    if (tokens < 0 || vocab < 0 || dim < 0 || ldo < dim || ldw < dim || !(beta == 0.f || beta == 1.f))
        return NTB_ERR_ARG;
    if (!((dtypeOut == NTB_X_FLOAT16 && (dtypeW == NTB_X_FLOAT16 || dtypeW == NTB_X_FLOAT)) || (dtypeOut == NTB_X_FLOAT && dtypeW == NTB_X_FLOAT)))
        return NTB_ERR_DTYPE;
    if (vocab == 0 || dim == 0 || (tokens == 0 && beta == 1.f))
        return NTB_OK;
    if (!dw || (tokens > 0 && (!ids || !dout)))
        return NTB_ERR_ARG;
    if (workBytes < ntb_embedding_grad_work(tokens, dim) || (tokens > 0 && (!work || ((uintptr_t)work & 15))))
        return NTB_ERR_ARG;
    /* the sort packs a token's number and its word into 32 bits each, with one value past the last word */
    if (vocab == 0x7fffffff || tokens > 0x7fffff00 || dim > EM_MOST_COLS)
        return NTB_ERR_LIMIT;
    const bool halves = dtypeOut == NTB_X_FLOAT16, halfW = dtypeW == NTB_X_FLOAT16;
    const bool wide = !halves ? WideRows<float, float>(dout, ldo, dw, ldw, dim)
        : !halfW ? WideRows<__half, float>(dout, ldo, dw, ldw, dim) : WideRows<__half, __half>(dout, ldo, dw, ldw, dim);
    const bool few = tokens <= (wide ? FEW_TOKENS : FEW_TOKENS / 2);
    /* CTAs along a launch's x where one launch does it all, blocks of columns along y where the list is sorted */
    const long long threads = wide ? dim / (halves ? EmVec<__half>::N : EmVec<float>::N) : dim;
    if (few ? (long long)((tokens + FEW_WARPS - 1) / FEW_WARPS) * (dim / (wide && halves ? 256 : 128) + 1) > 0x7fff0000LL : (threads + 255) / 256 > 65535)
        return NTB_ERR_LIMIT;
    XattnDevice dev(devID);
    if (!dev.ok)
        return NTB_ERR_CUDA;
    DeviceCtx * ctx = CtxFor(devID);
    if (!ctx)
        return NTB_ERR_CUDA;
    cudaStream_t st = (cudaStream_t)stream;
    if (few) {
        FewParams f;
        memset(&f, 0, sizeof(f));
        f.ids = ids;
        f.dout = dout;
        f.dw = dw;
        f.tokens = tokens; f.vocab = vocab; f.dim = dim;
        f.ldo = ldo; f.ldw = ldw;
        f.scale = scale;
        f.accumulate = beta == 1.f;
        f.sumCtas = (tokens + FEW_WARPS - 1) / FEW_WARPS;
        int clearing = 0;
        if (beta == 0.f) {
            const int most = 4 * ctx->smCount, want = (int)(((long long)vocab + FEW_WARPS - 1) / FEW_WARPS);
            clearing = want < most ? want : most;
        }
        const cudaError_t e = !halves ? LaunchFew<float, float>(f, wide, clearing, st)
            : !halfW ? LaunchFew<__half, float>(f, wide, clearing, st) : LaunchFew<__half, __half>(f, wide, clearing, st);
        if (e == cudaSuccess && cudaGetLastError() == cudaSuccess)
            return NTB_OK;
        cudaGetLastError();
        return NTB_ERR_CUDA;
    }
    SortParams s;
    memset(&s, 0, sizeof(s));
    s.ids = ids;
    s.a = (int2 *)work;
    s.b = s.a + tokens;
    s.tokens = tokens;
    s.vocab = vocab;
    int keyBits = 1;
    while ((vocab >> keyBits) != 0)
        keyBits++;
    s.passes = (keyBits + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
    s.bits = (keyBits + s.passes - 1) / s.passes;
    s.bits = s.bits < 2 ? 2 : s.bits;                       /* counters are cleared four at a time */
    s.ctas = SortCtas(tokens);
    int grid = s.ctas;
    const int size = dtypeW == NTB_X_FLOAT16 ? 2 : 4;
    if (beta == 0.f) {
        s.clear = (unsigned char *)dw;
        s.clearRows = vocab;
        s.clearPitch = ldw * size;
        s.clearBytes = (long long)dim * size;
        /* whole clusters up to one CTA an SM */
        const int extra = (ctx->smCount - grid) / s.ctas * s.ctas;
        grid += extra > s.ctas ? extra : s.ctas;
    }
    const int smem = SORT_TILE * (int)sizeof(int2) + SORT_WARPS * (1 << s.bits) * (int)sizeof(int);
    static SmemOptIn optIn;
    if (!optIn.Ensure((const void *)TokenSortKernel, SORT_TILE * (int)sizeof(int2) + SORT_WARPS * SORT_RADIX * (int)sizeof(int)))
        return NTB_ERR_CUDA;
    /* clusters of more than 8 CTAs are an opt-in of the kernel's on the device */
    static ClusterOptIn large;
    if (s.ctas > 8 && !large.Ensure((const void *)TokenSortKernel))
        return NTB_ERR_CUDA;
    cudaError_t err = LaunchClusterPdl(TokenSortKernel, (unsigned)grid, SORT_THREADS, smem, s.ctas, st, s);
    CountLaunch();
    if (err == cudaSuccess) {
        RunParams p;
        memset(&p, 0, sizeof(p));
        p.sorted = s.a;
        p.dout = dout;
        p.dw = dw;
        p.tokens = tokens; p.vocab = vocab; p.dim = dim;
        p.block = RunBlock(tokens);
        p.blocks = (int)(((long long)tokens + p.block - 1) / p.block);
        p.head = (float *)(s.b + tokens);
        p.tail = p.head + (long long)p.blocks * dim;
        p.ldo = ldo; p.ldw = ldw;
        p.scale = scale;
        p.accumulate = beta == 1.f;
        err = !halves ? LaunchRuns<float, float>(p, wide, st)
            : !halfW ? LaunchRuns<__half, float>(p, wide, st) : LaunchRuns<__half, __half>(p, wide, st);
    }
    if (err == cudaSuccess && cudaGetLastError() == cudaSuccess)
        return NTB_OK;
    cudaGetLastError();
    return NTB_ERR_CUDA;
}
