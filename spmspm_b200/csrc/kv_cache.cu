// Writing and reading the paged 4-bit key/value cache (layout: kv_int4.cuh).
//
// kv_append: one pass over the new tokens.  A vector (one head of one token) is held by D/4 lanes, four channels each;
// keys and queries are turned by their position's angles, the minimum and maximum of every 32 channels are found with
// three shuffles among eight lanes, and the codes go straight to their places in the block.
//
//   rotation   y = (a cos - b sin, b cos + a sin), in 64 bits and rounded once to fp16: a product of an fp16 and an fp32
//              value is exact there, so the result is the correctly rounded one and the codes that follow do not depend on
//              how the sum was taken (in 32 bits one value in some thousands would land on the other fp16 neighbour).
//   entry      m = min, s = largest fp16 not above (max - min) / 15, code = round-to-even((y - m) / s) in 0..15.  s is
//              rounded down so that m + 15 s never passes the maximum (rounded to nearest it could overflow fp16); what
//              that costs is less than s / 64 at the top of the range.  A group with a value that is not finite reads
//              back as NaN as a whole (s = m = NaN).
//
// Bound by memory: 4 D bytes in and 1.25 D out per token and head; there is no reuse, so the kernel is one load, the
// arithmetic in registers and the stores.
#include "kv_int4.cuh"

namespace spb {
namespace {

constexpr int kWarps = 8;

// Sequence of packed row `tok`, its position in the cache (negative: before the start) -> false when the row belongs to
// no sequence (behind the last one).
__device__ __forceinline__ bool locate(const KvView& c, long long tok, int& b, long long& pos)
{
    if (c.cu) {
        if (tok < c.cu[0] || tok >= c.cu[c.B]) return false;
        int lo = 0, hi = c.B;   // last b with cu[b] <= tok
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (c.cu[mid] <= tok) lo = mid;
            else hi = mid;
        }
        b = lo;
        if (tok >= c.cu[b + 1]) return false;   // offsets that are not ascending
        pos = (long long)c.lens[b] - c.cu[b + 1] + tok;
    } else {
        const long long per = c.n_tokens / c.B;
        b = (int)(tok / per);
        pos = c.lens[b] - per + tok % per;
    }
    return true;
}

__device__ __forceinline__ void load4(const uint16_t* p, __half (&x)[4])
{
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    *reinterpret_cast<uint2*>(x) = r;
}
// a * c + b * d in 64 bits, rounded once to fp16
__device__ __forceinline__ __half turn(__half a, float c, __half b, float d)
{
    return __double2half(fma((double)__half2float(a), (double)c, (double)__half2float(b) * (double)d));
}

// The vector's channels c0 .. c0 + 3, turned by the angles of position pos.
__device__ __forceinline__ void load_turned(const uint16_t* vec, int c0, const KvAppendArgs& a, long long pos, __half (&x)[4])
{
    load4(vec + c0, x);
    if (c0 >= a.rot) return;
    const int half_rot = a.rot / 2;
    const float* cs = a.cosv + pos * half_rot;
    const float* sn = a.sinv + pos * half_rot;
    if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float c = cs[c0 / 2 + i], s = sn[c0 / 2 + i];
            const __half u = x[2 * i], w = x[2 * i + 1];
            x[2 * i] = turn(u, c, w, -s);
            x[2 * i + 1] = turn(w, c, u, s);
        }
    } else {
        const bool upper = c0 >= half_rot;   // half_rot is a multiple of 4: all four channels on one side
        const int i0 = upper ? c0 - half_rot : c0;
        __half o[4];
        load4(vec + (upper ? c0 - half_rot : c0 + half_rot), o);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = turn(x[i], cs[i0 + i], o[i], upper ? sn[i0 + i] : -sn[i0 + i]);
    }
}

// One vector per D/4 lanes; the vectors of a token are its keys, its values and, when q is given, its queries.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) kv_append_kernel(KvAppendArgs a, int* status)
{
    using L = KvLayout<D>;
    constexpr int kLanes = D / 4, kPer = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, c0 = 4 * sub;
    const int vecs = 2 * a.c.kv_heads + (a.q ? a.q_heads : 0);
    const long long item = ((long long)blockIdx.x * kWarps + threadIdx.x / 32) * kPer + lane / kLanes;
    const bool inside = item < a.c.n_tokens * vecs;
    const long long tok = inside ? item / vecs : 0;
    const int vec = (int)(item % vecs);
    int b = 0;
    long long pos = -1;
    const bool mine = inside && locate(a.c, tok, b, pos) && pos >= 0;
    bool write = mine;
    const bool is_q = vec >= 2 * a.c.kv_heads, is_v = !is_q && vec >= a.c.kv_heads;
    const int head = is_q ? vec - 2 * a.c.kv_heads : is_v ? vec - a.c.kv_heads : vec;
    if (mine && a.cosv && !is_v && pos >= a.max_pos) {   // no angles for this position
        if (sub == 0) atomicOr(status, kStatusBadCache);
        write = false;
    }
    __half x[4] = {};
    if (write) {
        if (is_v) load4(a.v + tok * a.v_tok + head * a.v_head + c0, x);
        else {
            const uint16_t* src = is_q ? a.q + tok * a.q_tok + head * a.q_head : a.k + tok * a.k_tok + head * a.k_head;
            if (a.cosv) load_turned(src, c0, a, pos, x);
            else load4(src + c0, x);
        }
    }
    if (is_q) {
        if (write) *reinterpret_cast<uint2*>(a.q_out + (tok * a.q_heads + head) * D + c0) = *reinterpret_cast<uint2*>(x);
        write = false;
    }
    // minimum and maximum of the eight lanes that hold a group; every lane of the warp takes part
    float f[4], lo, hi;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __half2float(x[i]);
    lo = fminf(fminf(f[0], f[1]), fminf(f[2], f[3]));
    hi = fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) finite = finite && fabsf(f[i]) <= 65504.f;
#pragma unroll
    for (int o = 1; o < 8; o *= 2) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        finite = finite & (bool)__shfl_xor_sync(0xffffffffu, (int)finite, o);
    }
    // every step rounded down: 15 times an fp16 value is an fp32 value, so nothing falls below the largest fp16 that fits
    __half s = __float2half_rd(__fdiv_rd(__fsub_rd(hi, lo), 15.f)), m = __float2half_rn(lo);
    const float sf = __half2float(s);
    uint32_t code[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float t = sf > 0.f ? rintf(__fdiv_rn(__fsub_rn(f[i], lo), sf)) : 0.f;
        code[i] = finite ? (uint32_t)fminf(t, 15.f) : 0u;
    }
    if (!finite) s = m = __ushort_as_half((unsigned short)0x7fff);
    // two lanes, four apart, share a word of key codes
    const uint32_t kbits = code[0] | code[1] << 16 | code[2] << 8 | code[3] << 24;
    const uint32_t other = __shfl_xor_sync(0xffffffffu, kbits, 4);
    if (!write) return;
    const long long off = kv_block_offset<D>(a.c, b, head, pos);
    if (off < 0) {
        if (sub == 0) atomicOr(status, kStatusBadCache);
        return;
    }
    uint8_t* blk = a.c.pool + off;
    const int t16 = (int)(pos % kKvBlock), grp = sub / 8;
    if (!is_v) {
        if (!(sub & 4)) {
            const int t = sub & 3;
            reinterpret_cast<uint32_t*>(blk + L::kKCodes)[t16 * (D / 8) + t * L::kGroups + grp] = kbits | other << 4;
        }
        if ((sub & 7) == 0)
            reinterpret_cast<__half2*>(blk + L::kKParams)[t16 * L::kGroups + grp] = __halves2half2(s, m);
    } else {
        const int j = t16 / 8, t = (t16 % 8) / 2, e = t16 & 1;
        const int g = c0 / (D / 8), k = (c0 % (D / 8)) / 4;
        *reinterpret_cast<uint16_t*>(blk + L::kVCodes + j * 4 * D + (4 * g + t) * (D / 8) + 4 * k + 2 * e) =
            (uint16_t)(code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12);
        if ((sub & 7) == 0) {
            __half* p = reinterpret_cast<__half*>(blk + L::kVParams) + ((t16 / 2) * L::kGroups + grp) * 4 + e;
            p[0] = s;
            p[2] = m;
        }
    }
}

// The values of one vector, four channels a lane: m + code * s with one rounding.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) kv_read_kernel(KvReadArgs a, int* status)
{
    using L = KvLayout<D>;
    constexpr int kLanes = D / 4, kPer = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, c0 = 4 * sub, grp = sub / 8;
    const int vecs = 2 * a.c.kv_heads;
    const long long item = ((long long)blockIdx.x * kWarps + threadIdx.x / 32) * kPer + lane / kLanes;
    if (item >= a.c.n_tokens * vecs) return;
    const long long tok = item / vecs;
    const int vec = (int)(item % vecs);
    const bool is_v = vec >= a.c.kv_heads;
    const int head = is_v ? vec - a.c.kv_heads : vec;
    int b;
    long long pos;
    if (!locate(a.c, tok, b, pos)) return;
    uint16_t* dst = (is_v ? a.v : a.k) + (tok * a.c.kv_heads + head) * D + c0;
    const long long off = pos >= 0 ? kv_block_offset<D>(a.c, b, head, pos) : -1;
    if (off < 0) {
        if (pos >= 0 && sub == 0) atomicOr(status, kStatusBadCache);
        *reinterpret_cast<uint2*>(dst) = make_uint2(0, 0);
        return;
    }
    const uint8_t* blk = a.c.pool + off;
    const int t16 = (int)(pos % kKvBlock);
    uint32_t c[4];
    __half s, m;
    if (!is_v) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(blk + L::kKCodes)[t16 * (D / 8) + (sub & 3) * L::kGroups + grp] >>
                           ((sub & 4) ? 4 : 0);
        c[0] = w & 15, c[1] = w >> 16 & 15, c[2] = w >> 8 & 15, c[3] = w >> 24 & 15;
        const __half2 p = reinterpret_cast<const __half2*>(blk + L::kKParams)[t16 * L::kGroups + grp];
        s = __low2half(p), m = __high2half(p);
    } else {
        const int j = t16 / 8, t = (t16 % 8) / 2, e = t16 & 1, g = c0 / (D / 8), k = (c0 % (D / 8)) / 4;
        const uint32_t w = *reinterpret_cast<const uint16_t*>(blk + L::kVCodes + j * 4 * D + (4 * g + t) * (D / 8) + 4 * k + 2 * e);
        c[0] = w & 15, c[1] = w >> 4 & 15, c[2] = w >> 8 & 15, c[3] = w >> 12;
        const __half* p = reinterpret_cast<const __half*>(blk + L::kVParams) + ((t16 / 2) * L::kGroups + grp) * 4 + e;
        s = p[0], m = p[2];
    }
    __half y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __hfma(__uint2half_rn(c[i]), s, m);
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(y);
}

template <int D>
unsigned blocks_for(long long vectors)
{
    const long long per = kWarps * (32 / (D / 4));
    return (unsigned)((vectors + per - 1) / per);
}

}  // namespace

cudaError_t kv_append_launch(cudaStream_t s, int D, const KvAppendArgs& a, int* status)
{
    const long long vectors = a.c.n_tokens * (2ll * a.c.kv_heads + (a.q ? a.q_heads : 0));
    if (D == 128) kv_append_kernel<128><<<blocks_for<128>(vectors), 32 * kWarps, 0, s>>>(a, status);
    else kv_append_kernel<64><<<blocks_for<64>(vectors), 32 * kWarps, 0, s>>>(a, status);
    count_launch();
    return cudaGetLastError();
}

cudaError_t kv_read_launch(cudaStream_t s, int D, const KvReadArgs& a, int* status)
{
    const long long vectors = a.c.n_tokens * 2ll * a.c.kv_heads;
    if (D == 128) kv_read_kernel<128><<<blocks_for<128>(vectors), 32 * kWarps, 0, s>>>(a, status);
    else kv_read_kernel<64><<<blocks_for<64>(vectors), 32 * kWarps, 0, s>>>(a, status);
    count_launch();
    return cudaGetLastError();
}

}  // namespace spb
