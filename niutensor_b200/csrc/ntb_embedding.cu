/*
 * Embedding rows and their gradient (source/sample/transformer/submodel/Embedding.cpp: the rows of a word
 * matrix picked by token ids, times sqrt(d), plus the rows of the positions).
 *
 * Forward: out[t] = scale * w[ids[t]] + pos[t % posRows], one warp a token, 16-byte accesses, one rounding.
 * It is bound by its reads and writes.
 *
 * Gradient: dw[v] = beta dw[v] + scale * sum over the tokens t with ids[t] = v, t ascending, of dout[t].
 * Adding every row with atomics would sum in an order that changes from run to run and serialise on
 * frequent words, so the tokens are sorted first and equal words summed as runs:
 *
 *   TokenSortKernel   a stable radix sort of (id, t) in ONE launch: one cluster of CTAs, digits of at most
 *                     9 bits. Every warp owns a contiguous piece of the list; per pass it counts its digits,
 *                     the counts are prefixed over warps and (through distributed shared memory) over the
 *                     cluster's CTAs, and it walks its piece again, 32 tokens at a time, to scatter them. The
 *                     steps are separated by the hardware's cluster barrier. Meanwhile the other CTAs of
 *                     the grid clear dw (beta = 0), which takes longer than the sort for large vocabularies.
 *   RunSumKernel      the sorted list cut into equal blocks, whatever the words' frequencies; a thread owns
 *                     16 bytes of the columns and adds the rows of a block one after the other. Runs inside a
 *                     block go straight to dw, pieces of runs that cross an edge to fp32 partial rows.
 *   RunJoinKernel     adds up the pieces of a crossing run, in block order.
 *
 * Sums are fp32 in a fixed order. Ids outside [0, vocab) stand for no word.
 */
#include "ntb_xattn.cuh"

namespace ntb {

namespace {

constexpr int EM_THREADS = 256;
constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_MAX_BITS = 9;

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

__global__ void __launch_bounds__(SORT_THREADS) TokenSortKernel(const SortParams p)
{
    extern __shared__ int counters[];                          /* [warp][digit], then [digit] totals, [digit] bases */
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if ((int)blockIdx.x >= p.ctas) {
        const long long warps = (long long)(gridDim.x - p.ctas) * SORT_WARPS;
        const long long first = (long long)(blockIdx.x - p.ctas) * SORT_WARPS + warp;
        if (p.clearPitch == p.clearBytes) {
            /* rows back to back: equal pieces of a multiple of 512 bytes */
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
    int * totals = counters + SORT_WARPS * R, * bases = totals + R;
    __shared__ int warpSums[SORT_WARPS];
    const int rank = (int)blockIdx.x;
    /* this warp's piece of the list, a multiple of 32 tokens long but for the last */
    const long long pieces = (long long)p.ctas * SORT_WARPS;
    const long long per = ((p.tokens + pieces - 1) / pieces + 31) / 32 * 32;
    const long long begin = ((long long)rank * SORT_WARPS + warp) * per;
    const long long lo = begin < p.tokens ? begin : p.tokens;
    const long long hi = lo + per < p.tokens ? lo + per : p.tokens;
    int * mine = counters + warp * R;
    const unsigned before = (1u << lane) - 1u;

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
        for (int d = threadIdx.x; d < SORT_WARPS * R; d += SORT_THREADS)
            counters[d] = 0;
        __syncthreads();
        for (long long i0 = lo; i0 < hi; i0 += 32) {
            const long long i = i0 + lane;
            const bool in = i < hi;
            const int d = in ? (load(i).x >> shift) & (R - 1) : R;
            const unsigned same = __match_any_sync(0xffffffffu, d);
            if (in && (same & before) == 0)
                mine[d] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        if ((int)threadIdx.x < R) {
            int run = 0;
            for (int w = 0; w < SORT_WARPS; w++) {
                const int c = counters[w * R + threadIdx.x];
                counters[w * R + threadIdx.x] = run;
                run += c;
            }
            totals[threadIdx.x] = run;
        }
        if (p.ctas > 1)
            ClusterSync();
        else
            __syncthreads();
        /* where a digit's tokens start: all smaller digits, then the same digit in the CTAs before this one */
        int all = 0, ahead = 0;
        if ((int)threadIdx.x < R) {
            for (int c = 0; c < p.ctas; c++) {
                int n;
                if (p.ctas > 1)
                    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n) : "r"(MapShared(SmemAddr(totals + threadIdx.x), c)) : "memory");
                else
                    n = totals[threadIdx.x];
                all += n;
                ahead += c < rank ? n : 0;
            }
        }
        int scan = all;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, scan, off);
            if (lane >= off)
                scan += o;
        }
        if (lane == 31)
            warpSums[warp] = scan;
        __syncthreads();
        int lower = 0;
        for (int w = 0; w < warp; w++)
            lower += warpSums[w];
        if ((int)threadIdx.x < R)
            bases[threadIdx.x] = lower + scan - all + ahead;
        __syncthreads();
        for (long long i0 = lo; i0 < hi; i0 += 32) {
            const long long i = i0 + lane;
            const bool in = i < hi;
            const int2 x = in ? load(i) : make_int2(0, 0);
            const int d = in ? (x.x >> shift) & (R - 1) : R;
            const unsigned same = __match_any_sync(0xffffffffu, d);
            int at = 0;
            if (in)
                at = bases[d] + mine[d] + __popc(same & before);
            __syncwarp();
            if (in && (same & before) == 0)
                mine[d] += __popc(same);
            __syncwarp();
            if (in)
                __stcg(dst + at, x);
        }
        /* the scattered list is complete, and the totals have been read, before the next pass */
        if (p.ctas > 1)
            ClusterSync();
        else
            __syncthreads();
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

/* N columns of a run's sum into dw */
template <typename TW, int N>
__device__ __forceinline__ void WriteRow(const RunParams & p, int id, int col, const float * acc)
{
    TW * dst = (TW *)p.dw + id * p.ldw + col;
    float v[N];
#pragma unroll
    for (int e = 0; e < N; e++)
        v[e] = fmaf(acc[e], p.scale, p.accumulate ? Get(dst + e) : 0.f);
#pragma unroll
    for (int e = 0; e < N; e++)
        Put(dst + e, v[e]);
}
template <typename TW, int N>
__device__ __forceinline__ void WriteRowVec(const RunParams & p, int id, int col, const float * acc)
{
    TW * dst = (TW *)p.dw + id * p.ldw + col;
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
            v[e] = fmaf(acc[k + e], p.scale, v[e]);
        *(uint4 *)(dst + k) = PackRow(v, (const TW *)nullptr);
    }
}

/* VEC: 16-byte loads of dout, 16-byte accesses to dw; else one column a thread */
template <typename TO, typename TW, bool VEC>
__global__ void RunSumKernel(const RunParams p)
{
    constexpr int N = VEC ? EmVec<TO>::N : 1;
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
    constexpr int U = VEC ? 8 : 4;
    for (int i0 = 0; i0 < n; i0 += U) {
        /* the loads of U rows in flight together; the adds stay in order */
        uint4 raw[VEC ? U : 1];
        float one[VEC ? 1 : U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u < n ? i0 + u : n - 1;
            const TO * src = (const TO *)p.dout + it[i].y * p.ldo + col;
            if (VEC)
                raw[u] = __ldcs((const uint4 *)src);
            else
                one[u] = Get(src);
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
                        else if (VEC)
                            WriteRowVec<TW, N>(p, id, col, acc);
                        else
                            WriteRow<TW, N>(p, id, col, acc);
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
    /* the last block the run reaches: the first of the following ones whose last token is another word (lists are sorted) */
    int lo = i + 1, hi = p.blocks - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        const long long last = (long long)(mid + 1) * p.block - 1;
        if (p.sorted[last < p.tokens ? last : p.tokens - 1].x == id)
            lo = mid + 1;
        else
            hi = mid;
    }
    /* block lo begins with the run, or is behind a run that ended with block lo - 1 */
    const int stop = p.sorted[(long long)lo * p.block].x == id ? lo : lo - 1;
    for (int col = blockIdx.y * blockDim.x + threadIdx.x; col < p.dim; col += gridDim.y * blockDim.x) {
        float acc = p.tail[(long long)i * p.dim + col];
        int j = i + 1;
        for (; j + 7 <= stop; j += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; u++)
                v[u] = p.head[(long long)(j + u) * p.dim + col];
#pragma unroll
            for (int u = 0; u < 8; u++)
                acc += v[u];
        }
        for (; j <= stop; j++)
            acc += p.head[(long long)j * p.dim + col];
        WriteRow<TW, 1>(p, id, col, &acc);
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

bool RowsAligned(const void * p, long long pitch, int dim, int size)
{
    return ((uintptr_t)p & 15) == 0 && (pitch * size) % 16 == 0 && (dim * (long long)size) % 16 == 0;
}

template <typename TO, typename TW>
cudaError_t LaunchRuns(const RunParams & p, cudaStream_t stream)
{
    const bool vec = RowsAligned(p.dout, p.ldo, p.dim, sizeof(TO)) && RowsAligned(p.dw, p.ldw, p.dim, sizeof(TW)) &&
                     (p.dim % EmVec<TO>::N) == 0;
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
    cudaError_t err = vec ? cudaLaunchKernelEx(&cfg, RunSumKernel<TO, TW, true>, p) : cudaLaunchKernelEx(&cfg, RunSumKernel<TO, TW, false>, p);
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
    if (vocab == 0x7fffffff || tokens > 0x7fffff00)
        return NTB_ERR_LIMIT;
    XattnDevice dev(devID);
    if (!dev.ok)
        return NTB_ERR_CUDA;
    DeviceCtx * ctx = CtxFor(devID);
    if (!ctx)
        return NTB_ERR_CUDA;
    cudaStream_t st = (cudaStream_t)stream;
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
    /* one CTA sorts a thousand tokens a pass in about the time of a cluster barrier */
    s.ctas = tokens <= 2048 ? 1 : tokens <= 8192 ? 4 : 8;
    int grid = tokens > 0 ? s.ctas : 0;
    if (tokens == 0)
        s.ctas = 0;
    const int size = dtypeW == NTB_X_FLOAT16 ? 2 : 4;
    if (beta == 0.f) {
        s.clear = (unsigned char *)dw;
        s.clearRows = vocab;
        s.clearPitch = ldw * size;
        s.clearBytes = (long long)dim * size;
        /* whole clusters up to one CTA an SM */
        const int unit = s.ctas > 0 ? s.ctas : 1;
        const int extra = (ctx->smCount - grid) / unit * unit;
        grid += extra > unit ? extra : unit;
    }
    const int smem = (SORT_WARPS + 2) * (1 << s.bits) * (int)sizeof(int);
    static SmemOptIn optIn;
    if (!optIn.Ensure((const void *)TokenSortKernel, (SORT_WARPS + 2) * (1 << SORT_MAX_BITS) * (int)sizeof(int)))
        return NTB_ERR_CUDA;
    cudaError_t err = LaunchClusterPdl(TokenSortKernel, (unsigned)grid, SORT_THREADS, smem, s.ctas > 0 ? s.ctas : 1, st, s);
    CountLaunch();
    if (err == cudaSuccess && tokens > 0) {
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
        err = dtypeOut == NTB_X_FLOAT ? LaunchRuns<float, float>(p, st)
            : dtypeW == NTB_X_FLOAT ? LaunchRuns<__half, float>(p, st) : LaunchRuns<__half, __half>(p, st);
    }
    if (err == cudaSuccess && cudaGetLastError() == cudaSuccess)
        return NTB_OK;
    cudaGetLastError();
    return NTB_ERR_CUDA;
}
