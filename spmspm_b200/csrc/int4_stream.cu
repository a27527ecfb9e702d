// Linear layer over 4-bit weights (layout: int4.cuh) for up to 16 rows of x:
//
//   out[n][m] = residual + act(bias + sum over groups of s (sum_k c x - z sum_k x))      summed in fp32, rounded once
//
// Bound by the bytes of the codes for few rows and by the rate of mma.sync for 16 (28672 x 7168: 26 us with one row, 4.2 TB/s; 42 us
// with 16 and groups of 64, tensor pipe and issue slots each waiting for the other; 17 us at copy rate).  The codes enter mma.sync.m16n8k16 as they are: a nibble masked out of its word is an fp16
// subnormal, c 2^-24 (low nibble of a byte) or c 2^-20 (high), which the instruction multiplies exactly, so unpacking costs 1.25
// instructions per two weights (3.25 when they are expanded to fp16, as the kernel for more rows does).  Low and high nibbles are
// summed apart; scale and zero point are applied to a group's fp32 sums, with sum_k x from one more matrix instruction on ones.
// No weight is rounded.
//
// A thread block is eight independent warps: each streams units of its own (128 rows x 128 k, 8.7 KB, one bulk copy) into its own
// two-stage ring and keeps the sums of all 128 rows in registers, so that a unit's x is loaded once, straight into operand
// registers, and nobody waits for anybody until the run of units ends and the warps' sums are added in shared memory, in order.
#include "int4_work.cuh"

namespace spb {
namespace {

constexpr int kWarps = 8, kStages = 2;

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT tiles of 8 rows of x.
template <int NT, int kGroup>
struct StreamSmem {
    uint8_t ring[kWarps][kStages][int4_unit_bytes(kGroup)];
    float sums[kWarps][8 * 4][32];   // [warp][row tile, register][lane], one tile of 8 rows of x at a time
    alignas(16) float total[8 * NT][128];   // cluster: this thread block's part of the item
    uint64_t full[kWarps][kStages];
    int abort;
};

template <int NT, int kGroup>
__global__ void __launch_bounds__(32 * kWarps, 1) int4_stream_kernel(const __grid_constant__ Params p)
{
    constexpr int kBytes = int4_unit_bytes(kGroup), kPer = 128 / kGroup;
    extern __shared__ __align__(128) uint8_t raw[];
    StreamSmem<NT, kGroup>& sm = *reinterpret_cast<StreamSmem<NT, kGroup>*>(raw);
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, t = lane % 4;
    volatile int* abort_flag = &sm.abort;
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(smem_u32(&sm.full[warp][i]), 1);
        if (warp == 0) sm.abort = 0;
        mbar_init_fence();
    }
    __syncthreads();
    if (threadIdx.x == 0) {   // the first units on their way to L2 while what ran before ends
        Walk first(p);
        Run f;
        if (first.next<8 * NT>(p, f)) bulk_prefetch(p.a.units + ((long long)f.mb * p.ku + f.u0) * kBytes, min(kWarps * kStages, f.nkt / kUnit) * kBytes);
    }
    grid_wait();
    grid_release();   // the join may be set up while this kernel runs; it waits for its end

    const int kt_all = p.a.K / 64;
    const uint16_t* xr[NT];
    bool have[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        have[nt] = nt * 8 + g < p.a.N;
        xr[nt] = p.a.x + (long long)(have[nt] ? nt * 8 + g : 0) * p.a.K + 8 * t;
    }
    auto load_x = [&](uint4 (&v)[NT][4], int u) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 4; ++h)
                v[nt][h] = have[nt] && 2 * u + h / 2 < kt_all ? *reinterpret_cast<const uint4*>(xr[nt] + u * 128 + 32 * h) : make_uint4(0, 0, 0, 0);
    };
    // copies: this warp's units in order, kStages ahead of the sums
    Walk ahead(p);
    Run ar;
    int ai = 0, an = 0, issued = 0, done = 0;
    bool alive = true;
    auto refill = [&](int upto) {
        while (alive && issued < upto) {
            while (ai >= an) {
                if (!ahead.next<8 * NT>(p, ar)) return;
                ai = warp, an = ar.nkt / kUnit;
            }
            if (lane == 0) {
                const uint32_t bar = smem_u32(&sm.full[warp][issued % kStages]);
                mbar_expect_tx(bar, kBytes);
                bulk_g2s(smem_u32(sm.ring[warp][issued % kStages]), p.a.units + ((long long)ar.mb * p.ku + ar.u0 + ai) * kBytes, kBytes, bar);
            }
            ai += kWarps;
            ++issued;
        }
    };
    refill(kStages);

    Walk walk(p);
    Run r;
    while (walk.next<8 * NT>(p, r)) {
        float out[8][NT][4] = {};
        uint4 xv[NT][4], xn[NT][4];
        const int n = r.nkt / kUnit;
        if (warp < n) load_x(xn, r.u0 + warp);
        for (int i = warp; i < n; i += kWarps, ++done) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int h = 0; h < 4; ++h) xv[nt][h] = xn[nt][h];
            if (i + kWarps < n) load_x(xn, r.u0 + i + kWarps);
            float xs[kPer][NT][2];   // sum of x over a group, in units of the code sums
#pragma unroll
            for (int q = 0; q < kPer; ++q)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float v[4] = {};
#pragma unroll
                    for (int h = q * kGroup / 32; h < (q + 1) * kGroup / 32; ++h) {
                        mma(v, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, xv[nt][h].x, xv[nt][h].y);
                        mma(v, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, xv[nt][h].z, xv[nt][h].w);
                    }
                    xs[q][nt][0] = v[0] * -0x1p-20f, xs[q][nt][1] = v[1] * -0x1p-20f;
                }
            if (alive) alive = mbar_wait(smem_u32(&sm.full[warp][done % kStages]), (done / kStages) & 1, abort_flag, 1024);
            if (!alive) continue;
            const uint8_t* unit = sm.ring[warp][done % kStages];
            const uint4* code = reinterpret_cast<const uint4*>(unit) + int4_chunk(g, t);
            const __half2* par = reinterpret_cast<const __half2*>(unit + 2 * kInt4CodeBytes) + g;
#pragma unroll
            for (int rt = 0; rt < 8; ++rt) {
                const uint4 c[2] = {code[rt * 32], code[rt * 32 + kInt4CodeBytes / 16]};
                float low[NT][4] = {}, high[NT][4] = {};
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const uint32_t u = h & 1 ? c[h / 2].y : c[h / 2].x, v = h & 1 ? c[h / 2].w : c[h / 2].z, us = u >> 8, vs = v >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma(low[nt], u & 0x000f000fu, v & 0x000f000fu, us & 0x000f000fu, vs & 0x000f000fu, xv[nt][h].x, xv[nt][h].y);
                        mma(high[nt], u & 0x00f000f0u, v & 0x00f000f0u, us & 0x00f000f0u, vs & 0x00f000f0u, xv[nt][h].z, xv[nt][h].w);
                    }
                    if ((h + 1) * 32 % kGroup == 0) {   // a group is complete: scale and zero point
                        constexpr int kRows = 128;
                        const int q = h * 32 / kGroup;
                        const float2 p0 = __half22float2(par[q * kRows + rt * 16]), p1 = __half22float2(par[q * kRows + rt * 16 + 8]);
                        const float s0 = p0.x * 0x1p20f, s1 = p1.x * 0x1p20f;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float dot = fmaf(low[nt][j], 16.f, high[nt][j]);
                                out[rt][nt][j] = fmaf(j < 2 ? s0 : s1, fmaf(j < 2 ? p0.y : p1.y, xs[q][nt][j & 1], dot), out[rt][nt][j]);
                                low[nt][j] = high[nt][j] = 0.f;
                            }
                    }
                }
            }
            __syncwarp();
            refill(done + 1 + kStages);
        }
        // sums of the eight warps, in order
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (nt * 8 >= p.a.N) break;
            __syncthreads();
#pragma unroll
            for (int rt = 0; rt < 8; ++rt)
#pragma unroll
                for (int j = 0; j < 4; ++j) sm.sums[warp][rt * 4 + j][lane] = out[rt][nt][j];
            __syncthreads();
#pragma unroll
            for (int e = threadIdx.x; e < 1024; e += 32 * kWarps) {
                const int row = e & 127, col = e >> 7;
                const int v = row / 16 * 4 + (row >> 3 & 1) * 2 + (col & 1), l = (row & 7) * 4 + col / 2;
                float y = sm.sums[0][v][l];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) y += sm.sums[w][v][l];
                const long long m = (long long)r.mb * 128 + row, nn = nt * 8 + col;
                if (nn >= p.a.N) continue;
                if (p.split > 1) {
                    sm.total[nn][row] = y;
                    continue;
                }
                if (!(r.first && r.last)) p.a.ws[((2 * (size_t)blockIdx.x + r.first) * (8 * NT) + nn) * 128 + row] = y;
                else if (m < p.a.M) p.a.out[nn * p.a.M + m] = __half_as_ushort(__float2half_rn(finish(p.a, y, m, nn)));
            }
        }
    }
    if (p.split > 1) cluster_finish<8 * NT>(p, smem_u32(&sm.total[0][0]));
    if (!alive) {   // a wait ran out: report, and give the copies still under way one more bounded wait
        if (lane == 0) atomicOr(p.status, (int)kStatusWaitTimeout);
        for (int i = 0; i < kStages; ++i)
            for (uint32_t spin = 0; spin < 4096; ++spin)
                if (mbar_try(smem_u32(&sm.full[warp][i]), 0) || mbar_try(smem_u32(&sm.full[warp][i]), 1)) break;
    }
}

template <int NT, int kGroup>
cudaError_t launch_stream(cudaStream_t s, const Int4Args& a, const Plan& q, int* status)
{
    static bool prepared[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    constexpr size_t smem = sizeof(StreamSmem<NT, kGroup>);
    if (!prepared[dev]) {
        e = cudaFuncSetAttribute(int4_stream_kernel<NT, kGroup>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        prepared[dev] = true;
    }
    return launch_product<8 * NT>(s, int4_stream_kernel<NT, kGroup>, 32 * kWarps, smem, make_params(a, q, status), q);
}

}  // namespace

int int4_stream_clusters(int split)
{
    static int cached[64][9] = {};   // count + 1
    int dev = 0;
    if (split < 2 || split > 8 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return 0;
    }
    if (!cached[dev][split]) {
        using Smem = StreamSmem<2, 32>;   // the variant that needs most
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = split;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(split * 64);
        cfg.blockDim = dim3(32 * kWarps);
        cfg.dynamicSmemBytes = sizeof(Smem);
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(int4_stream_kernel<2, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem)) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, int4_stream_kernel<2, 32>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        cached[dev][split] = n + 1;
    }
    return cached[dev][split] - 1;
}

cudaError_t int4_stream_launch(cudaStream_t s, const Int4Args& a, int* status)
{
    const Plan q = plan_for(a.M, a.N, a.K);
    if (q.items * q.ku > 0x7fffffff) return cudaErrorInvalidValue;
    if (q.npad == 8)
        return a.group == 128 ? launch_stream<1, 128>(s, a, q, status) : a.group == 64 ? launch_stream<1, 64>(s, a, q, status) : launch_stream<1, 32>(s, a, q, status);
    return a.group == 128 ? launch_stream<2, 128>(s, a, q, status) : a.group == 64 ? launch_stream<2, 64>(s, a, q, status) : launch_stream<2, 32>(s, a, q, status);
}

}  // namespace spb
