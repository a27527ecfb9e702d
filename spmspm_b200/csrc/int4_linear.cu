// 4-bit weights (layout: int4.cuh): bringing them into the layout and back, and the entry point of the linear layer over them.
#include "../../include/spmm_b200.h"
#include "int4.cuh"

namespace spb {
namespace {

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

}  // namespace spb

extern "C" {

size_t spb_int4_bytes(int M, int K, int group)
{
    if (M <= 0 || K <= 0 || M % 64 || K % 64 || (group != 32 && group != 64 && group != 128) || K % group) return 0;
    return (size_t)spb::int4_units(M, K) * spb::int4_unit_bytes(group);
}
size_t spb_int4_workspace_bytes(int M, int N, int K) { return M > 0 && N > 0 && K > 0 ? 4 * spb::int4_ws_floats(M, N, K) : 0; }

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
    const size_t out_bytes = 2 * (size_t)N * M;
    if (overlap(out, out_bytes, x, 2 * (size_t)N * K) || overlap(out, out_bytes, bias, 2 * (size_t)M) ||
        (residual != out && overlap(out, out_bytes, residual, out_bytes))) {
        set_error("linear_int4: out overlaps x, the bias or, without being the same, the residual");
        return (int)cudaErrorInvalidValue;
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
    e = N <= kInt4StreamRows ? int4_stream_launch((cudaStream_t)stream, a, status) : int4_wide_launch((cudaStream_t)stream, a, status);
    if (e != cudaSuccess) set_error("linear_int4: %s", cudaGetErrorString(e));
    return (int)e;
}

}  // extern "C"
