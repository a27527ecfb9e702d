// Writing and reading the paged 4-bit key/value cache (layout: kv_int4.cuh).
//
// kv_append: one pass over the new tokens.  A vector (one head of one token) is held by D/4 lanes, four channels each;
// keys and queries are turned by their position's angles, the minimum and maximum of every 32 channels are found with
// three shuffles among eight lanes, and the codes go straight to their places in the block.
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
        const int end = c.cu[b + 1];
        if (tok >= end) return false;   // offsets that are not ascending
        pos = c.lens[b] - (end - tok);
    } else {
        b = (unsigned)tok / (unsigned)c.per_seq;
        pos = c.lens[b] - c.per_seq + (tok - b * c.per_seq);
    }
    return true;
}

__device__ __forceinline__ void load4(const uint16_t* p, __half (&x)[4])
{
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    *reinterpret_cast<uint2*>(x) = r;
}
// a * c + b * d rounded once to fp16.  Both products are taken exactly as pairs of fp32 values, and so is the sum, up to 2^-48 of its
// larger term; the last step to fp32 rounds to odd (an inexact result gets its last bit set), which keeps the rounding
// to fp16 right.  Fp32 throughout: the conversions that 64-bit arithmetic needs run at an eighth of its rate.
__device__ __forceinline__ __half turn(__half ah, float c, __half bh, float d)
{
    const float a = __half2float(ah), b = __half2float(bh);
    const float p = __fmul_rn(a, c), q = __fmul_rn(b, d);
    const float pl = __fmaf_rn(a, c, -p), ql = __fmaf_rn(b, d, -q);
    const float s = __fadd_rn(p, q), z = __fsub_rn(s, p);
    const float e = __fadd_rn(__fsub_rn(p, __fsub_rn(s, z)), __fsub_rn(q, z));   // s + e = p + q
    const float t = __fadd_rn(e, __fadd_rn(pl, ql));
    const float f = __fadd_rn(s, t), rest = __fsub_rn(t, __fsub_rn(f, s));
    uint32_t bits = __float_as_uint(f);
    if (rest != 0.f && !(bits & 1u)) bits += (rest > 0.f) == (f > 0.f) ? 1u : 0xffffffffu;
    return __float2half_rn(__uint_as_float(bits));
}

// The vector's channels c0 .. c0 + 3, turned by the angles of position pos.
__device__ __forceinline__ void load_turned(const uint16_t* vec, int c0, const KvAppendArgs& a, int pos, __half (&x)[4])
{
    load4(vec + c0, x);
    if (c0 >= a.rot) return;
    const int half_rot = a.rot / 2;
    const float* cs = a.cosv + (long long)pos * half_rot;
    const float* sn = a.sinv + (long long)pos * half_rot;
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

// One vector per D/4 lanes; the vectors of a token are its keys, its values and, when q is given, its queries.  A warp goes through
// `rows` consecutive tokens of the packed input for its vectors: one for a few tokens, more for many, so that finding the token's
// place is paid once.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) kv_append_kernel(KvAppendArgs a, int rows, int* status)
{
    using L = KvLayout<D>;
    constexpr int kLanes = D / 4, kPer = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, c0 = 4 * sub;
    const unsigned vecs = 2 * a.c.kv_heads + (a.q ? a.q_heads : 0);
    const unsigned item = (blockIdx.x * kWarps + threadIdx.x / 32) * kPer + lane / kLanes;
    const unsigned chunk = item / vecs, vec = item - chunk * vecs;
    const bool is_q = vec >= 2 * a.c.kv_heads, is_v = !is_q && vec >= a.c.kv_heads;
    const int head = is_q ? vec - 2 * a.c.kv_heads : is_v ? vec - a.c.kv_heads : vec;
    int b = 0, pos = -1, end = 0;   // end: first row behind the sequence
    for (int i = 0; i < rows; ++i) {
        const int tok = (int)chunk * rows + i;
        bool write = tok < a.c.n_tokens;
        if (write) {
            if (tok < end) ++pos;
            else {
                write = locate(a.c, tok, b, pos);
                end = !write ? 0 : a.c.cu ? a.c.cu[b + 1] : (b + 1) * a.c.per_seq;
            }
        }
        write = write && pos >= 0;
        if (write && a.cosv && !is_v && pos >= a.max_pos) {   // no angles for this position
            if (sub == 0) atomicOr(status, kStatusBadCache);
            write = false;
        }
        __half x[4] = {};
        if (write) {
            if (is_v) load4(a.v + (long long)tok * a.v_tok + head * a.v_head + c0, x);
            else {
                const uint16_t* src = is_q ? a.q + (long long)tok * a.q_tok + head * a.q_head : a.k + (long long)tok * a.k_tok + head * a.k_head;
                if (a.cosv) load_turned(src, c0, a, pos, x);
                else load4(src + c0, x);
            }
        }
        if (is_q) {
            if (write) *reinterpret_cast<uint2*>(a.q_out + ((long long)tok * a.q_heads + head) * D + c0) = *reinterpret_cast<uint2*>(x);
            write = false;
        }
        if (!__any_sync(0xffffffffu, write)) continue;
        // minimum and maximum of the eight lanes that hold a group; every lane of the warp takes part
        float f[4], lo, hi;
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = __half2float(x[k]);
        lo = fminf(fminf(f[0], f[1]), fminf(f[2], f[3]));
        hi = fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
        // a value that is not finite makes this NaN, and the sum of the group's
        float bad = (f[0] - f[0]) + (f[1] - f[1]) + (f[2] - f[2]) + (f[3] - f[3]);
#pragma unroll
        for (int o = 1; o < 8; o *= 2) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            bad += __shfl_xor_sync(0xffffffffu, bad, o);
        }
        const bool finite = bad == 0.f;
        // every step rounded down: 15 times an fp16 value is an fp32 value, so nothing falls below the largest fp16 that fits
        __half s = __float2half_rd(__fdiv_rd(__fsub_rd(hi, lo), 15.f)), m = __float2half_rn(lo);
        const float sf = __half2float(s), inv = __frcp_rn(sf);
        uint32_t code[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            // The quotient by the reciprocal is off by less than 2^-19; only next to a border of two codes is it divided out.
            const float d = __fsub_rn(f[k], lo);
            float q = d * inv, n = rintf(q);
            if (fabsf(fabsf(q - n) - 0.5f) < 0x1p-16f) n = rintf(__fdiv_rn(d, sf));
            code[k] = finite && sf > 0.f ? (uint32_t)fminf(n, 15.f) : 0u;
        }
        if (!finite) s = m = __ushort_as_half((unsigned short)0x7fff);
        // keys: two lanes, four apart, share a word; values: they exchange the bytes of neighbouring channel pairs
        const uint32_t kbits = code[0] | code[1] << 16 | code[2] << 8 | code[3] << 24;
        const uint32_t low = code[0] | code[1] << 4, high = code[2] | code[3] << 4;
        const bool upper = sub & 4;
        const uint32_t other = __shfl_xor_sync(0xffffffffu, is_v ? (upper ? low : high) : kbits, 4);
        if (!write) continue;
        const long long off = kv_block_offset<D>(a.c, b, head, pos);
        if (off < 0) {
            if (sub == 0) atomicOr(status, kStatusBadCache);
            continue;
        }
        uint8_t* blk = a.c.pool + off;
        const int t16 = pos % kKvBlock, grp = sub / 8;
        if (!is_v) {
            if (!upper) reinterpret_cast<uint32_t*>(blk + L::kKCodes)[t16 * (D / 8) + (sub & 3) * L::kGroups + grp] = kbits | other << 4;
            if ((sub & 7) == 0) reinterpret_cast<__half2*>(blk + L::kKParams)[t16 * L::kGroups + grp] = __halves2half2(s, m);
        } else {
            const int j = t16 / 8, t = (t16 % 8) / 2, e = t16 & 1, g = 2 * (sub & 3) + upper;
            *reinterpret_cast<uint16_t*>(blk + L::kVCodes + j * 4 * D + (4 * g + t) * (D / 8) + 4 * grp + 2 * e) = (uint16_t)(upper ? other | high << 8 : low | other << 8);
            if ((sub & 7) == 0) {
                __half* p = reinterpret_cast<__half*>(blk + L::kVParams) + ((t16 / 2) * L::kGroups + grp) * 4 + e;
                p[0] = s;
                p[2] = m;
            }
        }
    }
}

// The values of one vector, four channels a lane: m + code * s with one rounding.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) kv_read_kernel(KvReadArgs a, int rows, int* status)
{
    using L = KvLayout<D>;
    constexpr int kLanes = D / 4, kPer = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, c0 = 4 * sub, grp = sub / 8;
    const unsigned vecs = 2 * a.c.kv_heads;
    const unsigned item = (blockIdx.x * kWarps + threadIdx.x / 32) * kPer + lane / kLanes;
    const unsigned chunk = item / vecs, vec = item - chunk * vecs;
    const bool is_v = vec >= a.c.kv_heads;
    const int head = is_v ? vec - a.c.kv_heads : vec;
    int b = 0, pos = -1, end = 0;
    for (int i = 0; i < rows; ++i) {
        const int tok = (int)chunk * rows + i;
        if (tok >= a.c.n_tokens) return;
        if (tok < end) ++pos;
        else {
            if (!locate(a.c, tok, b, pos)) continue;
            end = a.c.cu ? a.c.cu[b + 1] : (b + 1) * a.c.per_seq;
        }
        uint16_t* dst = (is_v ? a.v : a.k) + ((long long)tok * a.c.kv_heads + head) * D + c0;
        const long long off = pos >= 0 ? kv_block_offset<D>(a.c, b, head, pos) : -1;
        if (off < 0) {
            if (pos >= 0 && sub == 0) atomicOr(status, kStatusBadCache);
            *reinterpret_cast<uint2*>(dst) = make_uint2(0, 0);
            continue;
        }
        const uint8_t* blk = a.c.pool + off;
        const int t16 = pos % kKvBlock;
        uint32_t pair[2];   // codes as fp16: 1024 + code
        __half s, m;
        if (!is_v) {
            const uint32_t w = reinterpret_cast<const uint32_t*>(blk + L::kKCodes)[t16 * (D / 8) + (sub & 3) * L::kGroups + grp] >> ((sub & 4) ? 4 : 0);
            pair[0] = w & 0x000f000fu, pair[1] = w >> 8 & 0x000f000fu;
            const __half2 p = reinterpret_cast<const __half2*>(blk + L::kKParams)[t16 * L::kGroups + grp];
            s = __low2half(p), m = __high2half(p);
        } else {
            const int j = t16 / 8, t = (t16 % 8) / 2, e = t16 & 1, g = 2 * (sub & 3);
            const uint8_t* at = blk + L::kVCodes + j * 4 * D + (4 * g + t) * (D / 8) + 4 * grp + 2 * e + (sub >> 2 & 1);
            const uint32_t low = at[0], high = at[4 * (D / 8)];
            pair[0] = (low & 15) | (low & 240) << 12, pair[1] = (high & 15) | (high & 240) << 12;
            const __half* p = reinterpret_cast<const __half*>(blk + L::kVParams) + ((t16 / 2) * L::kGroups + grp) * 4 + e;
            s = p[0], m = p[2];
        }
        __half2 y[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const uint32_t c = pair[k] | 0x64006400u;
            y[k] = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), __half2half2(__ushort_as_half((unsigned short)0x6400))), __half2half2(s), __half2half2(m));
        }
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(y);
    }
}

// Tokens a warp goes through: eight when that still leaves the device full (64 warps on each of some 150 SMs), else one.
int rows_for(long long vectors) { return vectors >= 8ll * 64 * 150 ? 8 : 1; }
template <int D>
unsigned blocks_for(int n_tokens, int rows, int vecs)
{
    const long long items = (n_tokens + rows - 1ll) / rows * vecs, per = kWarps * (32 / (D / 4));
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
