// Writing and reading the paged 4-bit key/value cache (layout: kv_int4.cuh).
//
// kv_append: one pass over the new tokens.  A vector (one head of one token) is held by D/8 lanes, eight channels each;
// keys and queries are turned by their position's angles, the minimum and maximum of every 32 channels are found with
// two shuffles among four lanes, and the codes go straight to their places in the block.
//
//   rotation   y = (a cos - b sin, b cos + a sin), exact up to 2^-48 and rounded once to fp16, so that the codes that follow do
//              not depend on how the sum was taken (in 32 bits one value in some thousands would land on the other
//              fp16 neighbour).
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
__device__ __forceinline__ bool locate(const KvView& c, int tok, int& b, int& pos)
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
        const int end = min(c.cu[b + 1], c.n_tokens);   // as kv_rows takes it
        if (tok >= end) return false;   // offsets that are not ascending
        pos = c.lens[b] - (end - tok);
    } else {
        b = (unsigned)tok / (unsigned)c.per_seq;
        pos = c.lens[b] - c.per_seq + (tok - b * c.per_seq);
    }
    return true;
}

// Tokens of the packed input one after the other, with the place of each in the cache; searched for once per sequence.
struct Cursor {
    int b = 0, pos = -1, end = 0;   // end: first row behind the sequence
    long long off = -1;             // offset of the token's block in the pool, -1: none
    __device__ __forceinline__ bool move_to(const KvView& c, int tok)
    {
        if (tok < end) {
            ++pos;
            return true;
        }
        const bool found = tok < c.n_tokens && locate(c, tok, b, pos);
        end = !found ? 0 : c.cu ? min(c.cu[b + 1], c.n_tokens) : (b + 1) * c.per_seq;
        off = -1;
        return found;
    }
    template <int D>
    __device__ __forceinline__ bool find_block(const KvView& c, int head)
    {
        if (off < 0 || pos % kKvBlock == 0) off = kv_block_offset<D>(c, b, head, pos);
        return off >= 0;
    }
};

__device__ __forceinline__ void load4(const uint16_t* p, __half (&x)[4]) { *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(p); }

// a * c + b * d rounded once to fp16.  Both products are taken exactly as pairs of fp32 values, and so is the sum, up to 2^-48 of its
// larger term; the last step to fp32 rounds to odd (an inexact result gets its last bit set), which keeps the rounding
// to fp16 right.  Fp32 throughout: the conversions that 64-bit arithmetic needs run at an eighth of its rate.
__device__ __forceinline__ __half turn_exactly(float a, float c, float b, float d)
{
    const float p = __fmul_rn(a, c), q = __fmul_rn(b, d);
    const float pl = __fmaf_rn(a, c, -p), ql = __fmaf_rn(b, d, -q);
    const float s = __fadd_rn(p, q), z = __fsub_rn(s, p);
    const float e = __fadd_rn(__fsub_rn(p, __fsub_rn(s, z)), __fsub_rn(q, z));   // s + e = p + q
    const float t = __fadd_rn(e, __fadd_rn(pl, ql));
    const float f = __fadd_rn(s, t), rest = __fsub_rn(t, __fsub_rn(f, s));
    if (!(fabsf(s) <= 3e38f)) return __float2half_rn(s);   // infinities and NaN as the plain sum has them
    uint32_t bits = __float_as_uint(f);
    if (rest != 0.f && !(bits & 1u)) bits += (rest > 0.f) == (f > 0.f) ? 1u : 0xffffffffu;
    return __float2half_rn(__uint_as_float(bits));
}
// Four of them.  In plain fp32 a sum is off by less than 2^-23 of |b d| + |sum|: when both ends of that range round to the same fp16
// value it is the right one, and only otherwise (one value in a thousand) is the exact form worked out.
__device__ __forceinline__ void turn4(const float (&a)[4], const float (&c)[4], const float (&b)[4], const float (&d)[4], __half (&y)[4])
{
    uint32_t differ = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = b[i] * d[i], s = fmaf(a[i], c[i], p), e = (fabsf(p) + fabsf(s)) * 0x1p-23f;
        const __half2 ends = __floats2half2_rn(s - e, s + e);
        y[i] = __low2half(ends);
        const uint32_t bits = *reinterpret_cast<const uint32_t*>(&ends);
        differ |= (bits ^ bits >> 16) & 0xffffu;
    }
    if (differ)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = turn_exactly(a[i], c[i], b[i], d[i]);
}

// The vector's channels c0 .. c0 + 3, turned by the angles of position pos.
__device__ __forceinline__ void load_turned(const uint16_t* vec, int c0, const KvAppendArgs& a, int pos, __half (&x)[4])
{
    load4(vec + c0, x);
    if (c0 >= a.rot) return;
    const int half_rot = a.rot / 2;
    float u[4], w[4], c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __half2float(x[i]);
    if (a.interleaved) {
        const float2 cc = *reinterpret_cast<const float2*>(a.cosv + (long long)pos * half_rot + c0 / 2);
        const float2 ss = *reinterpret_cast<const float2*>(a.sinv + (long long)pos * half_rot + c0 / 2);
        c[0] = c[1] = cc.x, c[2] = c[3] = cc.y;
        s[0] = -ss.x, s[1] = ss.x, s[2] = -ss.y, s[3] = ss.y;
        w[0] = u[1], w[1] = u[0], w[2] = u[3], w[3] = u[2];
    } else {
        const bool upper = c0 >= half_rot;   // half_rot is a multiple of 4: all four channels on one side
        const int i0 = upper ? c0 - half_rot : c0;
        __half o[4];
        load4(vec + (upper ? c0 - half_rot : c0 + half_rot), o);
        *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(a.cosv + (long long)pos * half_rot + i0);
        *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(a.sinv + (long long)pos * half_rot + i0);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __half2float(o[i]), s[i] = upper ? s[i] : -s[i];
    }
    turn4(u, c, w, s, x);
}

// One vector per D/8 lanes, eight channels each; the vectors of a token are its keys, its values and, when q is given, its queries.  A
// warp goes through `rows` consecutive tokens of the packed input for its vectors: one for a few tokens, more for many, so
// that finding the token's place is paid once.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) kv_append_kernel(KvAppendArgs a, int rows, int* status)
{
    using L = KvLayout<D>;
    constexpr int kLanes = D / 8, kPer = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, c0 = 8 * sub;
    const unsigned vecs = 2 * a.c.kv_heads + (a.q ? a.q_heads : 0);
    const unsigned item = (blockIdx.x * kWarps + threadIdx.x / 32) * kPer + lane / kLanes;
    const unsigned chunk = item / vecs, vec = item - chunk * vecs;
    const bool is_q = vec >= 2 * a.c.kv_heads, is_v = !is_q && vec >= a.c.kv_heads;
    const int head = is_q ? vec - 2 * a.c.kv_heads : is_v ? vec - a.c.kv_heads : vec;
    const uint16_t* src = is_q ? a.q + head * a.q_head : is_v ? a.v + head * a.v_head : a.k + head * a.k_head;
    const long long step = is_q ? a.q_tok : is_v ? a.v_tok : a.k_tok;
    const bool turned = a.cosv && !is_v;
    Cursor at;
    for (int i = 0; i < rows; ++i) {
        const int tok = (int)chunk * rows + i;
        bool write = at.move_to(a.c, tok) && at.pos >= 0;
        if (write && turned && at.pos >= a.max_pos) {   // no angles for this position
            if (sub == 0) atomicOr(status, kStatusBadCache);
            write = false;
        }
        __half x[2][4] = {};
        if (write) {
            const uint16_t* p = src + tok * step;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (turned) load_turned(p, c0 + 4 * k, a, at.pos, x[k]);
                else load4(p + c0 + 4 * k, x[k]);
            }
        }
        __syncwarp();   // q_out may be q: all lanes of a vector have read it
        if (is_q) {
            if (write) *reinterpret_cast<uint4*>(a.q_out + ((long long)tok * a.q_heads + head) * D + c0) = *reinterpret_cast<uint4*>(x);
            write = false;
        }
        if (!__any_sync(0xffffffffu, write)) continue;
        // minimum and maximum of the four lanes that hold a group, as {min, -max}; NaN spreads, every lane of the warp takes part
        const __half2* h2 = reinterpret_cast<const __half2*>(x);
        const __half2 lo2 = __hmin2_nan(__hmin2_nan(h2[0], h2[1]), __hmin2_nan(h2[2], h2[3]));
        const __half2 hi2 = __hmax2_nan(__hmax2_nan(h2[0], h2[1]), __hmax2_nan(h2[2], h2[3]));
        __half2 ends = __hmin2_nan(__lows2half2(lo2, __hneg2(hi2)), __highs2half2(lo2, __hneg2(hi2)));
#pragma unroll
        for (int o = 1; o < 4; o *= 2) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<uint32_t*>(&ends), o);
            ends = __hmin2_nan(ends, *reinterpret_cast<const __half2*>(&other));
        }
        const float lo = __low2float(ends), hi = -__high2float(ends);
        const bool finite = lo >= -65504.f && hi <= 65504.f;
        // s: the largest fp16 value with 15 s <= hi - lo.  A factor a little above 1/15 cannot fall below it and is one value too high at
        // most; 15 s is exact in fp32, and so is the comparison with the difference rounded down.
        const float span = __fsub_rd(hi, lo);
        __half s = __float2half_rd(span * 0x1.111116p-4f);
        if (15.f * __half2float(s) > span) s = __ushort_as_half((unsigned short)(__half_as_ushort(s) - 1));
        const float sf = __half2float(s), inv = __fdividef(1.f, sf);
        uint32_t code[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            // The quotient by the reciprocal is off by less than 2^-18; only next to a border of two codes is it divided out.
            const float d = __fsub_rn(__half2float(x[k / 4][k % 4]), lo);
            float q = d * inv, n = rintf(q);
            if (fabsf(fabsf(q - n) - 0.5f) < 0x1p-16f) n = rintf(__fdiv_rn(d, sf));
            code[k] = (uint32_t)fminf(n, 15.f);
        }
        __half m = __float2half_rn(lo);
        const bool plain = finite && sf > 0.f;   // a constant group has no codes
        if (!finite) s = m = __ushort_as_half((unsigned short)0x7fff);
        // Keys: words t and t + 1 of the group; this lane has the nibbles of one of their two halves, the lane two away those of the
        // other.  Values: a byte for each of four channel pairs, whose other byte of the halfword that lane has.
        uint32_t mine[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t* c = code + 4 * k;
            mine[k] = !plain ? 0u : is_v ? c[0] | c[1] << 4 | (c[2] | c[3] << 4) << 16 : c[0] | c[1] << 16 | c[2] << 8 | c[3] << 24;
        }
        const bool upper = sub & 2;
        const uint32_t other = __shfl_xor_sync(0xffffffffu, mine[upper ? 0 : 1], 2), kept = mine[upper ? 1 : 0];
        const uint32_t word = upper ? other | kept << (is_v ? 8 : 4) : kept | other << (is_v ? 8 : 4);
        if (!write) continue;
        if (!at.find_block<D>(a.c, head)) {
            if (sub == 0) atomicOr(status, kStatusBadCache);
            continue;
        }
        uint8_t* blk = a.c.pool + at.off;
        const int t16 = at.pos % kKvBlock, grp = sub / 4, pair = 2 * (sub & 1) + upper;   // the word or the two channel pairs this lane stores
        if (!is_v) {
            reinterpret_cast<uint32_t*>(blk + L::kKCodes)[t16 * (D / 8) + pair * L::kGroups + grp] = word;
            if ((sub & 3) == 0) reinterpret_cast<__half2*>(blk + L::kKParams)[t16 * L::kGroups + grp] = __halves2half2(s, m);
        } else {
            const int j = t16 / 8, t = (t16 % 8) / 2, e = t16 & 1;
            uint8_t* p = blk + L::kVCodes + j * 4 * D + (4 * 2 * pair + t) * (D / 8) + 4 * grp + 2 * e;
            *reinterpret_cast<uint16_t*>(p) = (uint16_t)word;
            *reinterpret_cast<uint16_t*>(p + 4 * (D / 8)) = (uint16_t)(word >> 16);
            if ((sub & 3) == 0) {
                __half* q = reinterpret_cast<__half*>(blk + L::kVParams) + ((t16 / 2) * L::kGroups + grp) * 4 + e;
                q[0] = s;
                q[2] = m;
            }
        }
    }
}

// The values of one vector, eight channels a lane: m + code * s with one rounding.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) kv_read_kernel(KvReadArgs a, int rows, int* status)
{
    using L = KvLayout<D>;
    constexpr int kLanes = D / 8, kPer = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, c0 = 8 * sub, grp = sub / 4;
    const unsigned vecs = 2 * a.c.kv_heads;
    const unsigned item = (blockIdx.x * kWarps + threadIdx.x / 32) * kPer + lane / kLanes;
    const unsigned chunk = item / vecs, vec = item - chunk * vecs;
    const bool is_v = vec >= a.c.kv_heads;
    const int head = is_v ? vec - a.c.kv_heads : vec;
    uint16_t* out = (is_v ? a.v : a.k) + head * D + c0;
    Cursor at;
    for (int i = 0; i < rows; ++i) {
        const int tok = (int)chunk * rows + i;
        if (!at.move_to(a.c, tok)) continue;
        uint16_t* dst = out + (long long)tok * a.c.kv_heads * D;
        if (at.pos < 0 || !at.find_block<D>(a.c, head)) {
            if (at.pos >= 0 && sub == 0) atomicOr(status, kStatusBadCache);
            *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(dst + 4) = make_uint2(0, 0);
            continue;
        }
        const uint8_t* blk = a.c.pool + at.off;
        const int t16 = at.pos % kKvBlock;
        uint32_t pair[4];   // two codes each, in the low nibbles of the halves
        __half s, m;
        if (!is_v) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(blk + L::kKCodes) + t16 * (D / 8) + 2 * (sub & 1) * L::kGroups + grp;
            const int shift = (sub & 2) ? 4 : 0;
#pragma unroll
            for (int k = 0; k < 2; ++k) pair[2 * k] = w[k * L::kGroups] >> shift & 0x000f000fu, pair[2 * k + 1] = w[k * L::kGroups] >> (8 + shift) & 0x000f000fu;
            const __half2 p = reinterpret_cast<const __half2*>(blk + L::kKParams)[t16 * L::kGroups + grp];
            s = __low2half(p), m = __high2half(p);
        } else {
            const int j = t16 / 8, t = (t16 % 8) / 2, e = t16 & 1;
            const uint8_t* p = blk + L::kVCodes + j * 4 * D + (4 * 4 * (sub & 1) + t) * (D / 8) + 4 * grp + 2 * e + (sub >> 1 & 1);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t c = p[4 * k * (D / 8)];
                pair[k] = (c & 15) | (c & 240) << 12;
            }
            const __half* q = reinterpret_cast<const __half*>(blk + L::kVParams) + ((t16 / 2) * L::kGroups + grp) * 4 + e;
            s = q[0], m = q[2];
        }
        __half2 y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t c = pair[k] | 0x64006400u;   // 1024 + code
            y[k] = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), __half2half2(__ushort_as_half((unsigned short)0x6400))), __half2half2(s), __half2half2(m));
        }
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(y);
        *reinterpret_cast<uint2*>(dst + 4) = *reinterpret_cast<uint2*>(y + 2);
    }
}

// Tokens a warp goes through: eight when that still leaves the device full (64 warps on each of some 150 SMs), else one.
int rows_for(long long vectors) { return vectors >= 8ll * 64 * 150 ? 8 : 1; }
template <int D>
unsigned blocks_for(int n_tokens, int rows, int vecs)
{
    const long long items = (n_tokens + rows - 1ll) / rows * vecs, per = kWarps * (32 / (D / 8));
    return (unsigned)((items + per - 1) / per);
}

}  // namespace

cudaError_t kv_append_launch(cudaStream_t s, int D, const KvAppendArgs& a, int* status)
{
    const int vecs = 2 * a.c.kv_heads + (a.q ? a.q_heads : 0), rows = rows_for((long long)a.c.n_tokens * vecs);
    if (D == 128) kv_append_kernel<128><<<blocks_for<128>(a.c.n_tokens, rows, vecs), 32 * kWarps, 0, s>>>(a, rows, status);
    else kv_append_kernel<64><<<blocks_for<64>(a.c.n_tokens, rows, vecs), 32 * kWarps, 0, s>>>(a, rows, status);
    count_launch();
    return cudaGetLastError();
}

cudaError_t kv_read_launch(cudaStream_t s, int D, const KvReadArgs& a, int* status)
{
    const int vecs = 2 * a.c.kv_heads, rows = rows_for((long long)a.c.n_tokens * vecs);
    if (D == 128) kv_read_kernel<128><<<blocks_for<128>(a.c.n_tokens, rows, vecs), 32 * kWarps, 0, s>>>(a, rows, status);
    else kv_read_kernel<64><<<blocks_for<64>(a.c.n_tokens, rows, vecs), 32 * kWarps, 0, s>>>(a, rows, status);
    count_launch();
    return cudaGetLastError();
}

}  // namespace spb
