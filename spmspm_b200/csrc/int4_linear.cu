// Linear layer over 4-bit weights (layout: int4.cuh) for few rows of x, and the kernels that bring weights into the layout.
//
//   y[n][m] = residual + act(bias + sum over groups of s (sum_k c x - z sum_k x))      summed in fp32, rounded once
//
// int4_small_kernel: bound by the bytes of the codes while N is small.  The codes enter mma.sync.m16n8k16 as they are: a
// nibble masked out of its word is an fp16 subnormal, c 2^-24 (low nibble of a byte) or c 2^-20 (high), multiplied
// exactly, so unpacking costs 1.25 instructions per two weights; low and high nibbles are summed apart, and scale and zero
// point are applied to the fp32 sums of a group, with sum_k x from one more matrix instruction on ones.  No weight is
// rounded.  The warps of a thread block, and the thread blocks of a cluster, share out K; partial sums meet in shared
// memory, in a fixed order.  Codes and x go from memory to registers with 16-byte loads, kDepth units ahead.
#include "../../include/spmm_b200.h"
#include "int4.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace spb {
namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_stream(const uint4* p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// RT row tiles of 16, NT column tiles of 8 rows of x per warp.
template <int RT, int NT, int kGroup>
__global__ void __launch_bounds__(32 * kWarps) int4_small_kernel(Int4Args a)
{
    constexpr int kDepth = RT == 1 ? 3 : 2;          // units whose codes and parameters are on their way
    constexpr int kPer = 128 / kGroup;               // groups per unit
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, t = lane % 4;
    const int ku = (a.K + 127) / 128, rt_all = a.M / 16, kt_all = a.K / 64;
    const int parts = gridDim.y * kWarps, part = blockIdx.y * kWarps + warp;
    const int u0 = (int)((long long)ku * part / parts), u1 = (int)((long long)ku * (part + 1) / parts);
    const int rt0 = blockIdx.x * RT, n0 = blockIdx.z * 8 * NT;

    const uint8_t* unit[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int rt = min(rt0 + r, rt_all - 1);   // past the end: a row tile that is there, its result is not stored
        unit[r] = a.units + (long long)(rt / 8) * ku * int4_unit_bytes(kGroup) + rt % 8 * 512;
    }
    const uint16_t* xr[NT];
    bool have[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        have[nt] = n0 + nt * 8 + g < a.N;
        xr[nt] = a.x + (long long)(have[nt] ? n0 + nt * 8 + g : 0) * a.K + 8 * t;
    }
    float out[RT][NT][4] = {};
    float low[RT][NT][4] = {}, high[RT][NT][4] = {}, xsum[NT][4] = {};
    uint4 w[kDepth][RT][2], xv[kDepth][NT][4];
    __half2 par[kDepth][RT][kPer][2];
    auto fetch = [&](int slot, int u) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const uint8_t* p = unit[r] + (long long)u * int4_unit_bytes(kGroup);
#pragma unroll
            for (int i = 0; i < 2; ++i) w[slot][r][i] = load_stream(reinterpret_cast<const uint4*>(p + i * kInt4CodeBytes) + int4_chunk(g, t));
            const __half2* q = reinterpret_cast<const __half2*>(p - (rt0 + r < rt_all ? (rt0 + r) % 8 : (rt_all - 1) % 8) * 512 + 2 * kInt4CodeBytes) +
                               (rt0 + r < rt_all ? (rt0 + r) % 8 : (rt_all - 1) % 8) * 16 + g;
#pragma unroll
            for (int i = 0; i < kPer; ++i) par[slot][r][i][0] = q[i * 128], par[slot][r][i][1] = q[i * 128 + 8];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 4; ++h)
                xv[slot][nt][h] = have[nt] && 2 * u + h / 2 < kt_all ? *reinterpret_cast<const uint4*>(xr[nt] + u * 128 + 32 * h) : make_uint4(0, 0, 0, 0);
    };
    auto apply = [&](const __half2 (&pv)[RT][kPer][2], int grp) {   // a group is complete: scale and zero point
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const float2 p0 = __half22float2(pv[r][grp][0]), p1 = __half22float2(pv[r][grp][1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float dot = fmaf(low[r][nt][i], 16.f, high[r][nt][i]) * 1048576.f;
                    const float2 p = i < 2 ? p0 : p1;
                    out[r][nt][i] = fmaf(p.x, fmaf(-p.y, xsum[nt][i & 1], dot), out[r][nt][i]);
                    low[r][nt][i] = high[r][nt][i] = 0.f;
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) xsum[nt][0] = xsum[nt][1] = xsum[nt][2] = xsum[nt][3] = 0.f;
    };
    auto step = [&](const uint4 (&wv)[RT][2], const uint4 (&xw)[NT][4], const __half2 (&pv)[RT][kPer][2]) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {   // 32 k each
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma(xsum[nt], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, xw[nt][h].x, xw[nt][h].y);
                mma(xsum[nt], 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u, xw[nt][h].z, xw[nt][h].w);
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const uint4 c = wv[r][h / 2];
                const uint32_t u = h & 1 ? c.y : c.x, v = h & 1 ? c.w : c.z;
                const uint32_t us = u >> 8, vs = v >> 8;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma(low[r][nt], u & 0x000f000fu, v & 0x000f000fu, us & 0x000f000fu, vs & 0x000f000fu, xw[nt][h].x, xw[nt][h].y);
                    mma(high[r][nt], u & 0x00f000f0u, v & 0x00f000f0u, us & 0x00f000f0u, vs & 0x00f000f0u, xw[nt][h].z, xw[nt][h].w);
                }
            }
            if ((h + 1) * 32 % kGroup == 0) apply(pv, h * 32 / kGroup);
        }
    };
#pragma unroll
    for (int i = 0; i < kDepth; ++i)
        if (u0 + i < u1) fetch(i, u0 + i);
    int u = u0;
    for (; u + kDepth <= u1; u += kDepth) {
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
            step(w[i], xv[i], par[i]);
            if (u + i + kDepth < u1) fetch(i, u + i + kDepth);
        }
    }
#pragma unroll
    for (int i = 0; i < kDepth; ++i)
        if (u + i < u1) step(w[i], xv[i], par[i]);

    // sums of the warps, then of the cluster's thread blocks (blockIdx.y), in order
    __shared__ float part_sum[kWarps][RT * NT * 4][32];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) part_sum[warp][(r * NT + nt) * 4 + i][lane] = out[r][nt][i];
    __syncthreads();
    constexpr int kVals = RT * NT * 4 * 32;
    float* flat = &part_sum[0][0][0];
    for (int v = threadIdx.x; v < kVals; v += 32 * kWarps) {
        float sum = flat[v];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) sum += flat[i * kVals + v];
        flat[v] = sum;
    }
    auto store = [&](int v, float y) {
        const int l = v & 31, i = (v >> 5) & 3, nt = (v >> 7) % NT, r = (v >> 7) / NT;
        const int m = (rt0 + r) * 16 + l / 4 + 8 * (i >> 1), n = n0 + nt * 8 + 2 * (l & 3) + (i & 1);
        if (rt0 + r >= rt_all || n >= a.N) return;
        if (a.bias) y += __half2float(__ushort_as_half(a.bias[m]));
        if (a.activation) y = y < 0.f ? 0.f : y;   // NaN stays NaN
        if (a.residual) y += __half2float(__ushort_as_half(a.residual[(long long)n * a.M + m]));
        a.out[(long long)n * a.M + m] = __half_as_ushort(__float2half_rn(y));
    };
    if (gridDim.y == 1) {
        for (int v = threadIdx.x; v < kVals; v += 32 * kWarps) store(v, flat[v]);
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int ranks = gridDim.y, rank = blockIdx.y;
    for (int v = rank * (32 * kWarps) + threadIdx.x; v < kVals; v += ranks * 32 * kWarps) {
        float sum = 0.f;
        for (int i = 0; i < ranks; ++i) sum += *cluster.map_shared_rank(flat + v, i);
        store(v, sum);
    }
    cluster.sync();   // nobody leaves while its sums are being read
}

// Word i of the codes (eight codes of one row): its place in the units, its row and first k.
__device__ __forceinline__ long long word_place(int K, int group, long long i, long long& row, long long& k)
{
    const int ku = (K + 127) / 128;
    const int q = (int)(i & 3), chunk = (int)(i >> 2 & 31), g = chunk / 4, t = (chunk & 3) ^ (g >> 1);
    const int in_unit = (int)(i & 2047), rt = in_unit / 128 % 8, kt = in_unit / 1024;
    const long long unit = i / 2048;
    row = unit / ku * 128 + rt * 16 + g + 8 * (q >> 1);
    k = unit % ku * 128 + kt * 64 + 32 * (q & 1) + 8 * t;
    return unit * (int4_unit_bytes(group) / 4) + in_unit;
}
// Parameter word of (row, group), rows and k past the end included.
__device__ __forceinline__ long long param_place(int K, int group, long long row, long long k)
{
    const long long unit = row / 128 * ((K + 127) / 128) + k / 128;
    return unit * (int4_unit_bytes(group) / 4) + 2048 + k % 128 / group * 128 + row % 128;
}
__global__ void int4_pack_kernel(const uint8_t* codes, uint32_t* units, int M, int K, int group)
{
    const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
    if (i >= int4_units(M, K) * 2048) return;
    long long row, k;
    const long long at = word_place(K, group, i, row, k);
    uint32_t w = 0;
    if (row < M && k < K) {
        const uint2 b = *reinterpret_cast<const uint2*>(codes + row * K + k);
#pragma unroll
        for (int r = 0; r < 8; ++r) w |= ((r < 4 ? b.x >> 8 * r : b.y >> 8 * (r - 4)) & 15u) << 4 * int4_nibble(r);
    }
    units[at] = w;
}
__global__ void int4_pack_params_kernel(const uint16_t* scales, const uint8_t* zeros, uint32_t* units, int M, int K, int group)
{
    const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
    const int per = (K + 127) / 128 * (128 / group), groups = K / group;
    if (i >= (long long)(M + 127) / 128 * 128 * per) return;
    const long long row = i / per, grp = i % per;
    const bool in = row < M && grp < groups;
    const __half2 v = __halves2half2(__ushort_as_half(in ? scales[row * groups + grp] : (unsigned short)0),
                                     __ushort2half_rn((unsigned short)(in ? zeros[row * groups + grp] & 15 : 0)));
    units[param_place(K, group, row, grp * group)] = *reinterpret_cast<const uint32_t*>(&v);
}
// The value of a weight: s (c - z), rounded once to fp16.
__global__ void int4_decode_kernel(const uint32_t* units, uint16_t* dense, int M, int K, int group)
{
    const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
    if (i >= int4_units(M, K) * 2048) return;
    long long row, k;
    const uint32_t w = units[word_place(K, group, i, row, k)];
    if (row >= M || k >= K) return;
    const __half2 p = reinterpret_cast<const __half2*>(units)[param_place(K, group, row, k)];
    __half y[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
        y[r] = __hmul(__hsub(__uint2half_rn(w >> 4 * int4_nibble(r) & 15u), __high2half(p)), __low2half(p));
    *reinterpret_cast<uint4*>(dense + row * K + k) = *reinterpret_cast<uint4*>(y);
}
// Quantises one group of one row per 8 lanes x (group / 64) values: lo = min(0, min), hi = max(0, max), s = fp16((hi - lo) / 15),
// z = round(-lo / s), c = clamp(round(x / s) + z, 0, 15).  Zero is always a value of the group, as pruned weights need it.
__global__ void int4_encode_kernel(const uint16_t* dense, uint8_t* codes, uint16_t* scales, uint8_t* zeros, int M, int K, int group)
{
    const long long i = blockIdx.x * (long long)(blockDim.x / 32) + threadIdx.x / 32;   // one warp per group
    const int lane = threadIdx.x & 31, groups = K / group;
    if (i >= (long long)M * groups) return;
    const long long row = i / groups, k0 = (i % groups) * group;
    float lo = 0.f, hi = 0.f;
    bool finite = true;
    for (int k = lane; k < group; k += 32) {
        const float x = __half2float(__ushort_as_half(dense[row * K + k0 + k]));
        lo = fminf(lo, x), hi = fmaxf(hi, x);
        finite = finite && fabsf(x) <= 65504.f;
    }
#pragma unroll
    for (int o = 16; o; o /= 2) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    finite = __all_sync(0xffffffffu, finite);
    const __half s = finite ? __float2half_rn(__fdiv_rn(hi - lo, 15.f)) : __ushort_as_half((unsigned short)0x7fff);
    const float sf = __half2float(s);
    const float z = sf > 0.f ? fminf(rintf(__fdiv_rn(-lo, sf)), 15.f) : 0.f;
    for (int k = lane; k < group; k += 32) {
        const float x = __half2float(__ushort_as_half(dense[row * K + k0 + k]));
        const float c = sf > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x, sf)) + z, 0.f), 15.f) : 0.f;
        codes[row * K + k0 + k] = (uint8_t)c;
    }
    if (lane == 0) {
        scales[i] = __half_as_ushort(s);
        zeros[i] = (uint8_t)z;
    }
}

int sm_count()
{
    static int n[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!n[dev] && cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    return n[dev];
}

template <int RT, int NT, int kGroup>
cudaError_t launch_small(cudaStream_t s, const Int4Args& a)
{
    const int gx = (a.M / 16 + RT - 1) / RT, gz = (a.N + 8 * NT - 1) / (8 * NT);
    // thread blocks that share K: enough to put about two on every SM, at least two 128-k steps for every warp
    int split = 1;
    while (split < 8 && (long long)gx * gz * split < 2 * sm_count() && a.K / 128 >= 2 * kWarps * 2 * split) split *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(gx, split, gz);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = split;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, int4_small_kernel<RT, NT, kGroup>, a);
    count_launch();
    return e;
}
template <int kGroup>
cudaError_t launch_group(cudaStream_t s, const Int4Args& a)
{
    const bool many = a.M / 16 >= 8 * sm_count();   // rows enough to fill the device with four row tiles a warp
    return many ? launch_small<4, 1, kGroup>(s, a) : launch_small<1, 1, kGroup>(s, a);
}

bool check_weight(const char* who, int M, int K, int group)
{
    if (M <= 0 || K <= 0 || M % 64 || K % 64) {
        set_error("%s: M and K must be positive multiples of 64 (M=%d K=%d)", who, M, K);
        return false;
    }
    if ((group != 32 && group != 64 && group != 128) || K % group) {
        set_error("%s: the group must be 32, 64 or 128 and divide K (group=%d K=%d)", who, group, K);
        return false;
    }
    return true;
}
unsigned blocks(long long items, int per) { return (unsigned)((items + per - 1) / per); }

}  // namespace

static cudaError_t int4_small_launch(cudaStream_t s, const Int4Args& a)
{
    return a.group == 128 ? launch_group<128>(s, a) : a.group == 64 ? launch_group<64>(s, a) : launch_group<32>(s, a);
}

}  // namespace spb

extern "C" {

size_t spb_int4_bytes(int M, int K, int group)
{
    if (M <= 0 || K <= 0 || M % 64 || K % 64 || (group != 32 && group != 64 && group != 128) || K % group) return 0;
    return (size_t)spb::int4_units(M, K) * spb::int4_unit_bytes(group);
}
size_t spb_int4_workspace_bytes(int M, int N, int K) { return M > 0 && N > 0 && K > 0 ? 4 * spb::int4_wide_ws_floats(M, N, K) : 0; }

int spb_int4_pack(void* stream, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int M, int K, int group, void* packed)
{
    using namespace spb;
    if (!check_weight("int4_pack", M, K, group)) return (int)cudaErrorInvalidValue;
    if (!codes || !scales || !zeros || !packed || !aligned16(codes) || !aligned16(packed) || (reinterpret_cast<uintptr_t>(scales) & 1)) {
        set_error("int4_pack: null or misaligned device pointer (codes and packed: 16 bytes)");
        return (int)cudaErrorInvalidValue;
    }
    cudaStream_t s = (cudaStream_t)stream;
    int4_pack_kernel<<<blocks(int4_units(M, K) * 2048, 256), 256, 0, s>>>(codes, (uint32_t*)packed, M, K, group);
    int4_pack_params_kernel<<<blocks(int4_units(M, K) * 128 * (128 / group), 256), 256, 0, s>>>(scales, zeros, (uint32_t*)packed, M, K, group);
    count_launch(2);
    return (int)cudaGetLastError();
}

int spb_int4_encode(void* stream, const uint16_t* dense, int M, int K, int group, uint8_t* codes, uint16_t* scales, uint8_t* zeros)
{
    using namespace spb;
    if (!check_weight("int4_encode", M, K, group)) return (int)cudaErrorInvalidValue;
    if (!dense || !codes || !scales || !zeros || ((reinterpret_cast<uintptr_t>(dense) | reinterpret_cast<uintptr_t>(scales)) & 1)) {
        set_error("int4_encode: null or misaligned device pointer");
        return (int)cudaErrorInvalidValue;
    }
    int4_encode_kernel<<<blocks((long long)M * (K / group), 8), 256, 0, (cudaStream_t)stream>>>(dense, codes, scales, zeros, M, K, group);
    count_launch();
    return (int)cudaGetLastError();
}

int spb_int4_decode(void* stream, const void* packed, int M, int K, int group, uint16_t* dense)
{
    using namespace spb;
    if (!check_weight("int4_decode", M, K, group)) return (int)cudaErrorInvalidValue;
    if (!packed || !dense || !aligned16(packed) || !aligned16(dense)) {
        set_error("int4_decode: null or misaligned device pointer (16 bytes)");
        return (int)cudaErrorInvalidValue;
    }
    int4_decode_kernel<<<blocks(int4_units(M, K) * 2048, 256), 256, 0, (cudaStream_t)stream>>>((const uint32_t*)packed, dense, M, K, group);
    count_launch();
    return (int)cudaGetLastError();
}

int spb_linear_int4(void* stream, const void* packed, int M, int K, int group, const uint16_t* x, uint16_t* out,
                    int N, const uint16_t* bias, const uint16_t* residual, int activation, void* workspace, size_t workspace_bytes)
{
    using namespace spb;
    if (!check_weight("linear_int4", M, K, group)) return (int)cudaErrorInvalidValue;
    if (N <= 0) {
        set_error("linear_int4: N must be positive (N=%d)", N);
        return (int)cudaErrorInvalidValue;
    }
    if (activation != 0 && activation != 1) {
        set_error("linear_int4: activation must be 0 (none) or 1 (ReLU), got %d", activation);
        return (int)cudaErrorInvalidValue;
    }
    if (!packed || !x || !out) {
        set_error("linear_int4: null device pointer");
        return (int)cudaErrorInvalidValue;
    }
    if (!aligned16(packed) || !aligned16(x) || !aligned16(out) || !aligned16(bias) || !aligned16(residual)) {
        set_error("linear_int4: the weight, x, out, bias and residual must be 16-byte aligned");
        return (int)cudaErrorMisalignedAddress;
    }
    const size_t need = spb_int4_workspace_bytes(M, N, K);
    if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need)) {
        set_error("linear_int4: needs a 16-byte aligned workspace of %zu bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
        return (int)cudaErrorInvalidValue;
    }
    int* status = nullptr;
    cudaError_t e = device_status_ptr(&status);
    if (e != cudaSuccess) return (int)e;
    Int4Args a;
    a.units = (const uint8_t*)packed;
    a.M = M, a.K = K, a.group = group;
    a.x = x, a.bias = bias, a.residual = residual, a.out = out;
    a.N = N, a.activation = activation;
    a.ws = (float*)workspace, a.ws_floats = workspace_bytes / 4;
    e = N <= kInt4SmallRows ? int4_small_launch((cudaStream_t)stream, a) : int4_wide_launch((cudaStream_t)stream, a, status);
    if (e != cudaSuccess) set_error("linear_int4: %s", cudaGetErrorString(e));
    return (int)e;
}

}  // extern "C"
