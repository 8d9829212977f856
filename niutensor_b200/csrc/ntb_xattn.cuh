/*
 * Pieces shared by the cross-attention kernels (forward, single-token step, gradients):
 * tensor maps over [batch, heads, rows, dim] operands of any strides, 4-D TMA copies,
 * tensor-memory transfers, and the rule by which queries and keys past a sequence's end
 * are kept out of the sums.
 */
#ifndef NTB_XATTN_CUH
#define NTB_XATTN_CUH

#include "ntb_internal.h"
#include "ntb_ptx.cuh"
#include <cuda_fp16.h>
#include <cstring>

namespace ntb {

struct XattnShape {
    int batch, headsQ, headsKV, group, lenQ, lenK, dim;
    const int * queryLens;
    const int * keyLens;
};

/* a forward call after its checks */
struct XattnCall {
    XattnShape sh;
    const void * q;
    const void * k;
    const void * v;
    void * out;
    float * lse;
    ntb_heads_layout lQ, lK, lV, lOut;
    float scale;
};

/* a gradient call after its checks */
struct XattnGradCall {
    XattnShape sh;
    const void * q;
    const void * k;
    const void * v;
    const void * out;
    const void * dout;
    const float * lse;
    void * dq;
    void * dk;
    void * dv;
    float * work;
    const ntb_heads_layout * l;      /* q, k, v, out, dout, dq, dk, dv */
    float scale;
};

/* Query rows a key head up to which the kernels of 16-row tiles are used: two tiles are what a warp's registers hold.
   The others pad to 128 rows. Gradients of 32 rows, us, here / there: 64 x 8 heads, 200 keys of 128
   48 / 86; 1000 of 128 122 / 282; one head, 8192 keys of 64 31 / 24 (here at most eight CTAs share a head). */
constexpr int XATTN_STEP_ROWS = 32;

namespace {

constexpr int XT = 128;                               /* rows of a query tile and keys of a key tile */
constexpr int XBOX_BYTES = XT * ROW_BYTES;            /* 128 rows x 64 halves: one swizzled box of an operand tile */
/* Tiles of a walk that one part takes before it is split, as far as 8 parts go, whatever the GPU's load. The tensor core's
   fp32 accumulator rounds toward zero at every instruction of 16 keys, which costs a sum some 2^-23.5 of itself each: 2^-12.5 over
   256 tiles (measured: 1024 tiles fall short by 7e-4, more than a half's rounding). */
constexpr int XATTN_PART_TILES = 256;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

/* The reference that the forward kernels take off the exponents (of 2): XATTN_BELOW under the row's maximum when it
   is set, and set again once the maximum is more than XATTN_AHEAD over it. Weights, which are halves in the second product,
   so reach 2^15, below half's 65504; those of 2^-14 and more, 2^-21 of the largest at least, are normal and off by
   2^-11 of themselves, lighter ones by 2^-25, 2^-32 of the largest. With the maximum itself as the reference the tail of
   131072 keys, each 2^-25 of the first, would be lost: 0.4 % of the sum. */
constexpr float XATTN_BELOW = 7.f, XATTN_AHEAD = 15.f;

/* how an operand's tensor map is addressed: a broadcast extent (stride 0) is mapped with one
   element and its coordinate multiplied by 0 */
struct HeadsAddr {
    int mulBatch, mulHead;
};

__device__ __forceinline__ int ClampLen(const int * lens, int b, int longest)
{
    if (lens == nullptr)
        return longest;
    const int n = lens[b];
    return n < 0 ? 0 : n > longest ? longest : n;
}

/*
 * The waits on the critical path between the softmax warps and the MMA thread: without a suspend hint (a
 * parked thread sees the barrier several hundred clocks late, as much as half a tile's products take), all lanes
 * polling; bounded as MbarWait.
 */
__device__ __forceinline__ bool WaitNow(uint32_t bar, uint32_t parity, volatile int * abortFlag, int * status)
{
    return MbarWait(bar, parity, abortFlag, status, 0);
}
__device__ __forceinline__ bool WaitNowWarp(uint32_t bar, uint32_t parity, volatile int * abortFlag, int * status)
{
    if (__all_sync(0xffffffffu, MbarTryWait(bar, parity, 0) != 0))
        return true;
    const long long t0 = clock64();
    for (uint32_t it = 1; ; ++it) {
        if (__all_sync(0xffffffffu, MbarTryWait(bar, parity, 0) != 0))
            return true;
        if ((it & 63u) == 0) {
            const bool late = clock64() - t0 > WaitLimit(status);
            if (late) {
                *abortFlag = 1;
                atomicExch(status, NTB_ERR_DEVICE_WAIT);
            }
            if (__any_sync(0xffffffffu, late || *abortFlag != 0))
                return false;
        }
    }
}

/* One arrival for a warp whose lanes have ordered what they did to tensor memory (TcFenceBefore): one for every
   thread would be hundreds of shared-memory operations a tile, against the tensor core's operand reads. */
__device__ __forceinline__ void ArriveWarp(uint32_t bar, int lane)
{
    __syncwarp();
    if (lane == 0)
        MbarArrive(bar);
}

__device__ __forceinline__ void TmaLoad4D(uint32_t dst, const CUtensorMap * map, uint32_t bar, int c0, int c1, int c2, int c3)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 :: "r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}

__device__ __forceinline__ void TmaStore4D(const CUtensorMap * map, uint32_t src, int c0, int c1, int c2, int c3)
{
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
                 :: "l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}

/* D += A * B with A in tensor memory (two halves per 32-bit column) and B in shared memory */
__device__ __forceinline__ void TcMmaTmemA(uint32_t dTmem, uint32_t aTmem, uint64_t bDesc, uint32_t iDesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(dTmem), "r"(aTmem), "l"(bDesc), "r"(iDesc), "r"(accumulate) : "memory");
}

/* 32 columns of this thread's lane, without waiting for completion */
__device__ __forceinline__ void TmemLoad32Async(uint32_t taddr, uint32_t * r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void TmemLoad8Async(uint32_t taddr, uint32_t * r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void TmemWaitLoad() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void TmemWaitStore() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

/* 16 registers into 16 columns of this thread's lane, without waiting for completion */
__device__ __forceinline__ void TmemStore16Async(uint32_t taddr, const uint32_t * v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                    "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}

__device__ __forceinline__ void TmemStore4Async(uint32_t taddr, const uint32_t * v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};"
                 :: "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

__device__ __forceinline__ float Exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

/* pairs of floats in one 64-bit register: sm_100 adds and multiplies both in one instruction */
__device__ __forceinline__ uint64_t Pair(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void Unpair(uint64_t v, float & lo, float & hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t Fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t Add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ uint64_t Mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

/*
 * The gradient kernels' ds = p (dp - delta) go into their products as halves. They are smaller than what they are
 * summed to by p, about 1 / lenK, and left as they are would be subnormal or 0 where dq and dk are ordinary halves, or,
 * with large v and a small scale, infinite. So the ds of a product carry a power of two, taken out of its sums in fp32:
 * where they are met one after the other a row's, that brings its largest to [2^DS_TOP, 2^(DS_TOP + 1)) when it is set and is
 * set again when ds have grown past DS_MOST; where the largest is known before, one that brings that to [2^14, 2^15). ds down to
 * 2^-21 of the largest are then off by 2^-11 of themselves, smaller ones by 2^-32 of the largest.
 */
constexpr float DS_MOST = 32768.f, DS_UNSET = 1208925819614629174706176.f;      /* 2^15; 2^80: nothing but zeros so far */
constexpr int DS_TOP = 7;

/* the power of two that brings `top` to [2^e, 2^(e + 1)), at most 2^80: ds, which are less than 2^41, times it are
   finite as floats */
__device__ __forceinline__ float PowerFor(float top, int e)
{
    const int b = 254 + e - (int)(__float_as_uint(top) >> 23);
    return __uint_as_float((uint32_t)(b < 207 ? b : 207) << 23);
}
/* 1 / power, for powers of two that are normal both ways */
__device__ __forceinline__ float PowerInverse(float power) { return __uint_as_float(0x7f000000u - __float_as_uint(power)); }
/* What a row's sums of ds, which carry a factor, are multiplied by at last: its inverse and the scale. Where that is past a
   float the sums are 0 or their results past a half: 0 stays 0, the others become infinite. Where it is below a float's
   range the results, from sums below 2^62, are below a half's. */
__device__ __forceinline__ float SumsFactor(float power, float scale) { return fminf(power * scale, 3.402823466e38f); }
/* whether the factor has to be set again for a row with this largest |ds| (an infinity makes the row's sums infinite
   or NaN, whatever the factor) */
__device__ __forceinline__ bool DsPast(float top, float factor) { return top * factor > DS_MOST && top < INFINITY; }

__device__ __forceinline__ uint32_t PackHalf2(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t *)&h;
}

/* the same with the largest half for what is larger (NaN stays NaN) */
__device__ __forceinline__ uint32_t PackHalf2Finite(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ void LoadShared16(uint32_t addr, uint32_t * v)
{
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void StoreShared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

/* rows [from, 128) of an operand tile of `boxes` boxes become zeros, by the calling warp; the caller
   fences before the tensor core reads them. Rows past a sequence's end hold whatever the caller's
   buffer holds there; their weights are 0, and 0 * NaN would still reach every sum. */
__device__ __forceinline__ void ZeroTileRows(uint32_t tile, int boxes, int from, int lane)
{
    const int n = (XT - from) * 8;
    for (int box = 0; box < boxes; box++)
        for (int i = lane; i < n; i += 32)
            StoreShared16(tile + box * XBOX_BYTES + from * ROW_BYTES + i * 16, 0u, 0u, 0u, 0u);
}

/* D += A B of one warp, 16 x 8 x 16 halves, and the loads of its operands */
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

/* an 8 x 8 block of halves over a warp's lanes, transposed */
__device__ __forceinline__ uint32_t MoveTrans(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ void ClusterSync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t ClusterRank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ uint32_t MapShared(uint32_t addr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ float LoadRemote(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ float4 LoadRemote4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

/* one MMA instruction descriptor: fp16 operands, fp32 accumulator, 128 rows, n columns */
__device__ constexpr uint32_t XattnDesc(int n, int bMN)
{
    return (1u << 4) | ((uint32_t)bMN << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}

/*
 * The map of a [batch, heads, rows, dim] operand as (dim, rows, heads, batch) with boxes of 64
 * columns x boxRows rows. Strides in elements. Columns past dim read as zeros and are not
 * written. An extent of one takes any stride; a stride of 0 is a broadcast (inputs only).
 */
int EncodeHeads(CUtensorMap * map, HeadsAddr * addr, const void * base, int dim, int rows, int heads, int batch,
                const ntb_heads_layout & l, int boxRows)
{
    EncodeTiledFn enc = GetEncodeTiled();
    if (!enc)
        return NTB_ERR_CUDA;
    addr->mulBatch = l.batch == 0 ? 0 : 1;
    addr->mulHead = l.head == 0 ? 0 : 1;
    const int nb = addr->mulBatch ? batch : 1, nh = addr->mulHead ? heads : 1;
    const long long any = 16;                 /* the stride of an extent of one */
    cuuint64_t dims[4] = { (cuuint64_t)dim, (cuuint64_t)rows, (cuuint64_t)nh, (cuuint64_t)nb };
    cuuint64_t strides[3] = { (cuuint64_t)(rows > 1 ? l.row * 2 : any), (cuuint64_t)(nh > 1 ? l.head * 2 : any),
                              (cuuint64_t)(nb > 1 ? l.batch * 2 : any) };
    cuuint32_t box[4] = { 64, (cuuint32_t)boxRows, 1, 1 };
    cuuint32_t estr[4] = { 1, 1, 1, 1 };
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, (void *)base, dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? NTB_OK : NTB_ERR_ARG;
}

/* what TMA can address: 16-byte base and strides, strides below 2^40 bytes; broadcast only where allowed */
inline bool LayoutOk(const void * base, const ntb_heads_layout & l, int dim, int rows, int heads, int batch, bool broadcast)
{
    if ((uintptr_t)base & 15)
        return false;
    const long long limit = 1LL << 39;        /* elements */
    if (rows > 1 && (l.row < dim || l.row % 8 != 0 || l.row >= limit))
        return false;
    if (heads > 1 && !(broadcast && l.head == 0) && (l.head < dim || l.head % 8 != 0 || l.head >= limit))
        return false;
    if (batch > 1 && !(broadcast && l.batch == 0) && (l.batch < dim || l.batch % 8 != 0 || l.batch >= limit))
        return false;
    return true;
}

/* the checks both entry points share; fills the shape */
inline int XattnShapeOf(XattnShape & s, int dtype, int batch, int headsQ, int headsKV, int lenQ, int lenK, int dim,
                        const int * queryLens, const int * keyLens, float scale)
{
    if (batch < 0 || headsQ < 0 || headsKV < 0 || lenQ < 0 || lenK < 0 || dim < 0)
        return NTB_ERR_ARG;
    if (dtype != NTB_X_FLOAT16)
        return NTB_ERR_DTYPE;
    if (!(scale > 0.f) || scale > 2.0e38f)                       /* times log2 e it is finite, too */
        return NTB_ERR_ARG;
    if (headsQ > 0 && (headsKV == 0 || headsQ % headsKV != 0))
        return NTB_ERR_SHAPE;
    if (dim < 8 || dim > 128 || dim % 8 != 0)
        return NTB_ERR_LIMIT;
    /* row and key indices run up to a tile past the end in 32 bits */
    if (lenQ > 0x7fffff00 || lenK > 0x7fffff00)
        return NTB_ERR_LIMIT;
    s.batch = batch; s.headsQ = headsQ; s.headsKV = headsKV; s.group = headsKV ? headsQ / headsKV : 1;
    s.lenQ = lenQ; s.lenK = lenK; s.dim = dim;
    s.queryLens = queryLens; s.keyLens = keyLens;
    return NTB_OK;
}

/* launch in clusters of `cluster` CTAs along x, with programmatic stream serialisation as LaunchPdl */
template <typename... Params, typename... Args>
cudaError_t LaunchClusterPdl(void (*kern)(Params...), unsigned grid, int block, int smem, int cluster, cudaStream_t stream, Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3((unsigned)block, 1, 1);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PdlEnabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

/* makes a device current for the length of a call */
struct XattnDevice {
    int prev;
    bool ok;
    explicit XattnDevice(int dev) : prev(-1), ok(false)
    {
        if (cudaGetDevice(&prev) != cudaSuccess) {
            prev = -1;
            cudaGetLastError();
            return;
        }
        ok = prev == dev || cudaSetDevice(dev) == cudaSuccess;
        if (!ok) {
            prev = -1;
            cudaGetLastError();
        }
    }
    ~XattnDevice()
    {
        int cur = -1;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev)
            cudaSetDevice(prev);
    }
};

}

}

#endif
