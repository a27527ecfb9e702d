// How the kernels of the 4-bit linear layer share out their work.
//
// The product is a list of items (128 rows of W x a tile of rows of x), each of ku units along K (int4.cuh).  When the items fill
// the SMs evenly a thread block takes whole items; otherwise all units are laid end to end and every thread block takes an equal
// share.  Partial sums of items that are cut go to the workspace (two slots a thread block: an item it starts in the middle of, and
// one it leaves in the middle of) and int4_join_kernel adds them in order of k: no atomics, the same bits every time.
#pragma once
#include "int4.cuh"
#include "sm100.cuh"

namespace spb {
namespace {
using namespace sm100;

constexpr int kUnit = 2;   // k-tiles of a unit

struct Params {
    Int4Args a;
    int ku, ncol, items;   // units along K, column tiles, items
    int share, extra;      // thread block i takes `share` units, one more if i < extra; whole: items instead of units
    int whole;
    int split;             // > 1: the thread blocks of a cluster of this size share out one item
    int* status;
};
// First unit of thread block i's share of the list (items in order, ku units each), and the thread block that has unit x.
__device__ __forceinline__ int share_begin(const Params& p, int i) { return (i * p.share + min(i, p.extra)) * (p.whole ? p.ku : 1); }
__device__ __forceinline__ int share_of(const Params& p, int x)   // not whole
{
    const int big = p.extra * (p.share + 1);
    return x < big ? x / (p.share + 1) : p.extra + (x - big) / p.share;
}
__device__ __forceinline__ float finish(const Int4Args& a, float y, float bias, uint16_t residual)
{
    y += bias;
    if (a.activation) y = y < 0.f ? 0.f : y;   // NaN stays NaN
    return y + __half2float(__ushort_as_half(residual));
}
__device__ __forceinline__ float finish(const Int4Args& a, float y, long long m, long long n)
{
    return finish(a, y, a.bias ? __half2float(__ushort_as_half(a.bias[m])) : 0.f, a.residual ? a.residual[n * a.M + m] : (unsigned short)0);
}

// A run of k-tiles of one item.
struct Run {
    int mb, n0, u0, nkt;
    bool first, last;   // starts / ends the item
};
struct Walk {
    int x, hi, item, u;
    __device__ __forceinline__ Walk(const Params& p)
    {
        if (p.split > 1) {
            item = blockIdx.x / p.split;
            const int rank = blockIdx.x - item * p.split;
            u = p.ku * rank / p.split;
            x = item * p.ku + u;
            hi = item * p.ku + p.ku * (rank + 1) / p.split;
        } else {
            x = share_begin(p, blockIdx.x);
            hi = share_begin(p, blockIdx.x + 1);
            item = x / p.ku;
            u = x - item * p.ku;
        }
    }
    template <int NPAD>
    __device__ __forceinline__ bool next(const Params& p, Run& r)
    {
        if (x >= hi) return false;
        const int n = min(p.ku - u, hi - x);
        r.mb = item / p.ncol;
        r.n0 = (item - r.mb * p.ncol) * NPAD;
        r.u0 = u;
        r.nkt = n * kUnit;
        r.first = u == 0;
        r.last = u + n == p.ku;
        x += n;
        u = 0;
        ++item;
        return true;
    }
};

// Four rows of one column, finished and stored.
__device__ __forceinline__ void store4(const Int4Args& a, float4 sum, long long m, long long n)
{
    if (m >= a.M) return;   // M is a multiple of 64
    const float y[4] = {sum.x, sum.y, sum.z, sum.w};
    uint2 res = make_uint2(0, 0), bias = res;
    if (a.residual) res = *reinterpret_cast<const uint2*>(a.residual + n * a.M + m);
    if (a.bias) bias = *reinterpret_cast<const uint2*>(a.bias + m);
    const uint16_t *rh = reinterpret_cast<const uint16_t*>(&res), *bh = reinterpret_cast<const uint16_t*>(&bias);
    __half o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __float2half_rn(finish(a, y[i], __half2float(__ushort_as_half(bh[i])), rh[i]));
    *reinterpret_cast<uint2*>(a.out + n * a.M + m) = *reinterpret_cast<uint2*>(o);
}
// The parts [column][128 rows] that a cluster's thread blocks have at `addr`, added in order of k: a warp takes a column, every
// split-th stretch of columns a thread block.
template <int NPAD>
__device__ __forceinline__ void cluster_finish(const Params& p, uint32_t addr)
{
    cluster_sync();
    const int rank = blockIdx.x % p.split, item = blockIdx.x / p.split, n0 = item % p.ncol * NPAD, warps = blockDim.x / 32, lane = threadIdx.x & 31;
    for (int col = rank + p.split * (int)(threadIdx.x / 32); col < NPAD && n0 + col < p.a.N; col += p.split * warps) {
        float4 v[8], sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = cluster_load4(addr + (col * 128 + 4 * lane) * 4, i < p.split ? i : rank);   // all under way together
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < p.split) sum.x += v[i].x, sum.y += v[i].y, sum.z += v[i].z, sum.w += v[i].w;
        store4(p.a, sum, (long long)(item / p.ncol) * 128 + 4 * lane, n0 + col);
    }
    cluster_sync();   // nobody leaves while its part is being read
}

// Adds the partial sums of the items that were cut, in order; blockIdx.x: item, blockIdx.y: column, or columns by 8.  A warp takes a
// column; with many parts (`spread`) a thread block does, its warps share out the parts.
template <int NPAD>
__global__ void __launch_bounds__(256) int4_join_kernel(const __grid_constant__ Params p, int spread)
{
    const int x0 = blockIdx.x * p.ku, c0 = share_of(p, x0), c1 = share_of(p, x0 + p.ku - 1);
    grid_wait();
    if (c0 == c1) return;
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, col = spread ? blockIdx.y : blockIdx.y * 8 + warp;
    const long long n = (long long)(blockIdx.x % p.ncol) * NPAD + col, m = (long long)(blockIdx.x / p.ncol) * 128 + 4 * lane;
    if (n >= p.a.N) return;
    // the first part may be either slot of its thread block, the later ones start a thread block's share
    const float4* src = reinterpret_cast<const float4*>(p.a.ws + col * 128) + lane;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    const int step = spread ? 8 : 1;
#pragma unroll 4
    for (int i = c0 + (spread ? warp : 0); i <= c1; i += step) {
        const float4 v = src[(2 * (size_t)i + (i == c0)) * (NPAD * 32)];
        sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    if (spread) {
        __shared__ float4 part[8][32];
        part[warp][lane] = sum;
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            const float4 v = part[i][lane];
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
    }
    store4(p.a, sum, m, n);
}

int sm_count()
{
    static int n[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return 148;
    }
    if (!n[dev] && cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    return n[dev];
}
// How a shape is dealt out: thread blocks, whether they take whole items, and how many of them share one through a cluster.
struct Plan {
    int npad, ncol;
    long long items;
    int ku, ctas, split;
    bool whole;
};
Plan plan_for(int M, int N, int K)
{
    Plan q;
    q.npad = N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : N <= 64 ? 64 : N <= 128 ? 128 : 256;
    q.ncol = (N + q.npad - 1) / q.npad;
    q.items = (M + 127ll) / 128 * q.ncol;
    q.ku = (K + 127) / 128;
    q.split = 1;
    const int sms = sm_count();
    const long long rounds = (q.items + sms - 1) / sms, units = q.items * q.ku;
    q.whole = q.items >= 0.92 * rounds * sms;
    if (2 * q.items <= sms) {
        // Few items: the thread blocks of a cluster share one and add up through shared memory, without a second launch (5120 x 5120,
        // one row of x: 7.4 us against 9.9; 1024 x 1024: 3.6 against 4.8).  The streaming kernel does eight units at a time,
        // one per warp; the other one a unit after the other, so that with few clusters (they have eight thread blocks at most)
        // an equal share for every SM and a join is faster again: the join costs what eight units do.  All clusters have to fit at
        // once: sixteen of eight did not, and 2048 x 8192 took 10.2 us in two rounds.
        const bool stream = N <= kInt4StreamRows;
        const long long most = sms / q.items, worth = stream ? (q.ku + 7) / 8 : (q.ku + 1) / 2;
        int c = (int)(most < worth ? most : worth);
        if (c > 8) c = 8;
        while (c > 1 && int4_stream_clusters(c) < q.items) --c;
        if (stream || (q.ku + c - 1) / c <= units / sms + 8) {
            q.split = c;
            q.whole = c > 1 || worth == 1;
        }
    }
    q.ctas = (int)(q.split > 1 ? q.items * q.split : q.whole ? (sms < q.items ? (long long)sms : q.items) : units < 2 ? 1ll : units / 2 < sms ? units / 2 : (long long)sms);   // at least two units a thread block
    return q;
}
Params make_params(const Int4Args& a, const Plan& q, int* status)
{
    Params p;
    p.a = a;
    p.ku = q.ku;
    p.ncol = q.ncol;
    p.items = (int)q.items;
    p.whole = q.whole;
    p.split = q.split;
    const int all = (int)(q.whole ? q.items : q.items * q.ku);
    p.share = all / q.ctas;
    p.extra = all % q.ctas;
    p.status = status;
    return p;
}
// The product's launch and, when items are cut, the join's; both may be set up before what precedes them has ended.
template <int NPAD, class Kernel, class... More>
cudaError_t launch_product(cudaStream_t s, Kernel kernel, int threads, size_t smem, const Params& p, const Plan& q, const More&... more)
{
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = q.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(q.ctas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = q.split > 1 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p, more...);
    count_launch();
    if (e != cudaSuccess || q.whole) return e;
    const int cols = p.a.N < NPAD ? p.a.N : NPAD, spread = q.ctas > 8 * q.items;
    cfg.gridDim = dim3((unsigned)q.items, spread ? cols : (cols + 7) / 8);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, int4_join_kernel<NPAD>, p, spread);
    count_launch();
    return e;
}

}  // namespace
}  // namespace spb
