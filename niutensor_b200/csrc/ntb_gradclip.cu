/*
 * The norm of a whole list of gradients and their clipping to it:
 *
 *     norm = sqrt(sum over all elements of g^2),   out = g * min(1, maxNorm / norm)
 *
 * Two launches whatever the number of tensors (up to 1000; longer lists go in groups): the tensors' addresses
 * travel in the launch parameters, so there is no table to copy to the device and the call can be captured.
 * The list is cut into chunks of equal size.
 *
 * NormKernel: squares summed in fp64 for floats (a norm that fits a float may have squares that do not), in
 * fp32 over eight exact products and then fp64 for halves; one partial sum a CTA. ClipKernel: every CTA adds
 * up the partial sums in the same order (so all have the same norm; no atomics, no third launch), then scales
 * its chunks, walking the list backwards: what the first pass read last is still in L2. Both are bound by
 * their reads and writes: the list has to be read to the end before the first element can be written. 209 M
 * floats in 253 tensors take 374 us for both: 2.5 GB read twice and written once, 6.7 TB/s with what L2 gives.
 */
#include "ntb_xattn.cuh"
#include <algorithm>
#include <new>

namespace ntb {

namespace {

constexpr int CL_THREADS = 512;
constexpr int CL_CHUNK = 32768;           /* bytes */
constexpr int CL_FEW = 64, CL_MANY = 1000;     /* tensors a launch; kernel parameters end at 32764 bytes */

struct ClipTensor {
    const void * in;
    void * out;
    long long n;
    int firstChunk;
    int half;
};

template <int MAX> struct ClipList {
    ClipTensor t[MAX];
    int count;
    int chunks;
    double * partial;
    int partial0;             /* this launch's first partial sum */
    int partials;             /* all of them */
    float maxNorm;
    float * norm;             /* written by the first CTA of the first group, or NULL */
};
static_assert(sizeof(ClipList<CL_MANY>) <= 32700, "kernel parameters");

/* the chunk's tensor: the last one that starts at or before it and is not empty */
template <int MAX>
__device__ __forceinline__ int TensorOf(const ClipList<MAX> & l, int chunk)
{
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (l.t[mid].firstChunk <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double Squares(const uint4 & u, bool half)
{
    const uint32_t x[4] = { u.x, u.y, u.z, u.w };
    if (half) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*(const __half2 *)&x[i]);
            s = fmaf(f.x, f.x, s);
            s = fmaf(f.y, f.y, s);
        }
        return (double)s;
    }
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const double d = (double)__uint_as_float(x[i]);
        s = fma(d, d, s);
    }
    return s;
}

__device__ __forceinline__ float Element(const void * p, long long i, bool half)
{
    return half ? __half2float(((const __half *)p)[i]) : ((const float *)p)[i];
}

__device__ __forceinline__ void SetElement(void * p, long long i, bool half, float v)
{
    if (half)
        ((__half *)p)[i] = __float2half_rn(v);
    else
        ((float *)p)[i] = v;
}

/* the elements of a chunk: [lo, hi) of its tensor, of which [lo + head, lo + head + 16-byte packs) are aligned */
struct ChunkRange {
    long long lo, hi, body;
    int packs, perPack;
};
__device__ __forceinline__ ChunkRange RangeOf(const ClipTensor & t, int chunk)
{
    const int size = t.half ? 2 : 4, per = 16 / size;
    const long long each = CL_CHUNK / size;
    ChunkRange r;
    r.lo = (long long)(chunk - t.firstChunk) * each;
    r.hi = r.lo + each < t.n ? r.lo + each : t.n;
    const long long head = (long long)((16 - (((uintptr_t)t.in + r.lo * size) & 15)) & 15) / size;
    r.body = r.lo + head < r.hi ? r.lo + head : r.hi;
    r.packs = (int)((r.hi - r.body) / per);
    r.perPack = per;
    return r;
}

template <int MAX>
__global__ void __launch_bounds__(CL_THREADS) NormKernel(const __grid_constant__ ClipList<MAX> l)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    double sum = 0.0;
    for (int chunk = blockIdx.x; chunk < l.chunks; chunk += gridDim.x) {
        const ClipTensor & t = l.t[TensorOf(l, chunk)];
        const ChunkRange r = RangeOf(t, chunk);
        const bool half = t.half != 0;
        const uint4 * v = (const uint4 *)((const char *)t.in + r.body * (half ? 2 : 4));
        constexpr int U = CL_CHUNK / 16 / CL_THREADS;
        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = u * CL_THREADS + threadIdx.x;
            x[u] = i < r.packs ? v[i] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            sum += Squares(x[u], half);
        /* what lies before and behind the aligned packs: fewer than eight elements each */
        const long long tail = r.body + (long long)r.packs * r.perPack;
        if (threadIdx.x < r.body - r.lo) {
            const double d = Element(t.in, r.lo + threadIdx.x, half);
            sum = fma(d, d, sum);
        }
        if (threadIdx.x < r.hi - tail) {
            const double d = Element(t.in, tail + threadIdx.x, half);
            sum = fma(d, d, sum);
        }
    }
    __shared__ double sums[CL_THREADS / 32];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
        sum += __shfl_down_sync(0xffffffffu, sum, off);
    if ((threadIdx.x & 31) == 0)
        sums[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < CL_THREADS / 32; w++)
            sum += sums[w];
        l.partial[l.partial0 + blockIdx.x] = sum;
    }
}

template <int MAX>
__global__ void __launch_bounds__(CL_THREADS) ClipKernel(const __grid_constant__ ClipList<MAX> l)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ double sums[CL_THREADS / 32];
    double sum = 0.0;
    for (int i = threadIdx.x; i < l.partials; i += CL_THREADS)
        sum += l.partial[i];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
        sum += __shfl_down_sync(0xffffffffu, sum, off);
    if ((threadIdx.x & 31) == 0)
        sums[threadIdx.x >> 5] = sum;
    __syncthreads();
    double total = 0.0;
    for (int w = 0; w < CL_THREADS / 32; w++)
        total += sums[w];
    const double norm = sqrt(total);
    if (blockIdx.x == 0 && threadIdx.x == 0 && l.norm != nullptr)
        *l.norm = (float)norm;
    const bool clip = norm > (double)l.maxNorm && !isinf((float)norm);       /* as the caller sees it */
    /* A factor below a float's normal range would lose its bits, or all of them, where a clipped value is an ordinary float:
       a power of two goes first then, exactly where the result is not below a float's normal range itself. (The factor as a
       double, and all registers that takes, cost every call 3 %.) */
    double ratio = (double)l.maxNorm / norm;
    float f0 = 1.f;
    if (clip && ratio < 7.8886090522101181e-31) {                            /* 2^-100 */
        const bool least = ratio < 9.273015376718553e-69;                   /* 2^-226 */
        f0 = least ? 2.9387358770557188e-39f : 7.8886090522101181e-31f;      /* 2^-128, 2^-100 */
        ratio *= least ? 3.4028236692093846e38 : 1.2676506002282294e30;
    }
    const float f = clip ? (float)ratio : 1.f;
    for (int k = blockIdx.x; k < l.chunks; k += gridDim.x) {
        const int chunk = l.chunks - 1 - k;
        const ClipTensor & t = l.t[TensorOf(l, chunk)];
        if (!clip && t.in == t.out)
            continue;                             /* nothing changes */
        const ChunkRange r = RangeOf(t, chunk);
        const bool half = t.half != 0;
        const int size = half ? 2 : 4;
        if ((((uintptr_t)t.in ^ (uintptr_t)t.out) & 15) != 0) {
            for (long long i = r.lo + threadIdx.x; i < r.hi; i += CL_THREADS)
                SetElement(t.out, i, half, Element(t.in, i, half) * f0 * f);
            continue;
        }
        const uint4 * v = (const uint4 *)((const char *)t.in + r.body * size);
        uint4 * o = (uint4 *)((char *)t.out + r.body * size);
        constexpr int U = CL_CHUNK / 16 / CL_THREADS;
        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = u * CL_THREADS + threadIdx.x;
            if (i < r.packs)
                x[u] = __ldcs(v + i);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = u * CL_THREADS + threadIdx.x;
            if (i < r.packs) {
                uint32_t w[4] = { x[u].x, x[u].y, x[u].z, x[u].w };
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (half) {
                        const float2 g = __half22float2(*(const __half2 *)&w[e]);
                        w[e] = PackHalf2(g.x * f0 * f, g.y * f0 * f);
                    }
                    else
                        w[e] = __float_as_uint(__uint_as_float(w[e]) * f0 * f);
                }
                __stcs(o + i, make_uint4(w[0], w[1], w[2], w[3]));
            }
        }
        const long long tail = r.body + (long long)r.packs * r.perPack;
        if (threadIdx.x < r.body - r.lo)
            SetElement(t.out, r.lo + threadIdx.x, half, Element(t.in, r.lo + threadIdx.x, half) * f0 * f);
        if (threadIdx.x < r.hi - tail)
            SetElement(t.out, tail + threadIdx.x, half, Element(t.in, tail + threadIdx.x, half) * f0 * f);
    }
}

/* CTAs of the norm, each with a partial sum: 16 an SM. The clipping takes a CTA a chunk. 209 M floats, both passes,
   us: 4 CTAs an SM in both 429; 4 and a CTA a chunk 387; 16 and 64 an SM 383; 16 and a CTA a chunk 374. Many
   short CTAs keep reads and writes of different chunks in flight together where a persistent CTA alternates. */
constexpr int CL_CTAS = 16;
int Ctas(const DeviceCtx & ctx, int chunks)
{
    const int most = ctx.smCount * CL_CTAS;
    return chunks < 1 ? 1 : chunks < most ? chunks : most;
}

/*
 * Whether what is written for one entry overlaps what is written for another, or what an entry is read from, but for an
 * entry in place: CTAs read and write in no order, so such a call's result would depend on timing. The spans of a list that
 * lies in a pool are in order already.
 */
struct ClipSpan {
    uintptr_t lo, hi;
};
bool ClipOverlaps(int count, const void * const * grads, void * const * out, const int * dtypes, const long long * counts, ClipSpan * spans)
{
    auto span = [&](const void * p, int i) {
        const uintptr_t lo = (uintptr_t)p;
        return ClipSpan{ lo, lo + (uintptr_t)counts[i] * (dtypes[i] == NTB_X_FLOAT16 ? 2 : 4) };
    };
    auto before = [](const ClipSpan & a, const ClipSpan & b) { return a.lo < b.lo; };
    int n = 0;
    for (int i = 0; i < count; i++)
        if (counts[i] > 0)
            spans[n++] = span(out[i], i);
    if (!std::is_sorted(spans, spans + n, before))
        std::sort(spans, spans + n, before);
    for (int i = 1; i < n; i++)
        if (spans[i].lo < spans[i - 1].hi)
            return true;
    for (int i = 0; i < count; i++)
        if (counts[i] > 0 && grads[i] != out[i]) {
            const ClipSpan g = span(grads[i], i);
            const ClipSpan * s = std::upper_bound(spans, spans + n, g, before);        /* the first written behind g's start */
            if ((s < spans + n && s->lo < g.hi) || (s > spans && s[-1].hi > g.lo))
                return true;
        }
    return false;
}

template <int MAX>
int ClipGroups(const DeviceCtx & ctx, int count, const void * const * grads, void * const * out, const int * dtypes, const long long * counts,
               float maxNorm, float * norm, double * partial, cudaStream_t stream)
{
    for (int pass = 0; pass < 2; pass++) {
        int partials = 0;
        if (pass == 1)                            /* as many as the first pass wrote */
            for (int g0 = 0; g0 < count || g0 == 0; g0 += MAX) {
                long long chunks = 0;
                for (int i = g0; i < count && i < g0 + MAX; i++)
                    chunks += (counts[i] * (dtypes[i] == NTB_X_FLOAT16 ? 2 : 4) + CL_CHUNK - 1) / CL_CHUNK;
                partials += Ctas(ctx, (int)chunks);
            }
        int at = 0;
        for (int g0 = 0; g0 < count || g0 == 0; g0 += MAX) {
            ClipList<MAX> l;
            l.count = 0;
            long long chunks = 0;
            for (int i = g0; i < count && i < g0 + MAX; i++) {
                if (counts[i] == 0)
                    continue;
                ClipTensor & t = l.t[l.count++];
                t.in = grads[i];
                t.out = out[i];
                t.n = counts[i];
                t.half = dtypes[i] == NTB_X_FLOAT16;
                t.firstChunk = (int)chunks;
                chunks += (counts[i] * (t.half ? 2 : 4) + CL_CHUNK - 1) / CL_CHUNK;
            }
            l.chunks = (int)chunks;
            l.partial = partial;
            l.partial0 = at;
            l.partials = partials;
            l.maxNorm = maxNorm;
            l.norm = g0 == 0 ? norm : nullptr;
            const int grid = Ctas(ctx, l.chunks);
            at += grid;
            const cudaError_t err = pass == 0 ? LaunchPdl(NormKernel<MAX>, grid, CL_THREADS, 0, stream, l)
                                              : LaunchPdl(ClipKernel<MAX>, l.chunks < 1 ? 1 : l.chunks, CL_THREADS, 0, stream, l);
            CountLaunch();
            if (err != cudaSuccess || cudaGetLastError() != cudaSuccess) {
                cudaGetLastError();
                return NTB_ERR_CUDA;
            }
        }
    }
    return NTB_OK;
}

}

}

using namespace ntb;

extern "C" long long ntb_clip_grad_norm_work(int count)
{
    /* partial sums: a group of tensors at a time, on at most 256 SMs */
    const long long groups = count <= CL_MANY ? 1 : (count + CL_MANY - 1) / CL_MANY;
    return groups * 256 * CL_CTAS * (long long)sizeof(double);
}

extern "C" int ntb_clip_grad_norm(int devID, void * stream, int count, const void * const * grads, void * const * out,
                                  const int * dtypes, const long long * counts, float maxNorm, float * norm,
                                  void * work, long long workBytes)
{
    if (count < 0 || !(maxNorm >= 0.f) || !norm || !work || ((uintptr_t)work & 7) || workBytes < ntb_clip_grad_norm_work(count))
        return NTB_ERR_ARG;
    if (count > 0 && (!grads || !out || !dtypes || !counts))
        return NTB_ERR_ARG;
    long long chunks = 0;
    for (int i = 0; i < count; i++) {
        if (dtypes[i] != NTB_X_FLOAT16 && dtypes[i] != NTB_X_FLOAT)
            return NTB_ERR_DTYPE;
        const int size = dtypes[i] == NTB_X_FLOAT16 ? 2 : 4;
        if (counts[i] < 0 || (counts[i] > 0 && (!grads[i] || !out[i] || (((uintptr_t)grads[i] | (uintptr_t)out[i]) & (size - 1)))))
            return NTB_ERR_ARG;
        if (counts[i] > (1LL << 44))
            return NTB_ERR_LIMIT;
        chunks += (counts[i] * size + CL_CHUNK - 1) / CL_CHUNK;
        if (chunks > 0x7fff0000LL)
            return NTB_ERR_LIMIT;
    }
    ClipSpan few[CL_FEW], * spans = count <= CL_FEW ? few : new (std::nothrow) ClipSpan[count];
    if (!spans)
        return NTB_ERR_LIMIT;
    const bool overlaps = ClipOverlaps(count, grads, out, dtypes, counts, spans);
    if (spans != few)
        delete[] spans;
    if (overlaps)
        return NTB_ERR_ARG;
    XattnDevice dev(devID);
    if (!dev.ok)
        return NTB_ERR_CUDA;
    DeviceCtx * ctx = CtxFor(devID);
    if (!ctx)
        return NTB_ERR_CUDA;
    if (ctx->smCount > 256)
        return NTB_ERR_LIMIT;
    return count <= CL_FEW
        ? ClipGroups<CL_FEW>(*ctx, count, grads, out, dtypes, counts, maxNorm, norm, (double *)work, (cudaStream_t)stream)
        : ClipGroups<CL_MANY>(*ctx, count, grads, out, dtypes, counts, maxNorm, norm, (double *)work, (cudaStream_t)stream);
}
