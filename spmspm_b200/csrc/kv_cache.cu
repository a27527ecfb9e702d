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
// Bound by latency and by the instructions of exact rounding, not by its bytes (4 D in and 1.25 D out per token and head): a warp takes up
// to eight turns of vectors of one kind of one token, whose place and angles it then finds once, and loads a turn ahead.  Prompts of
// 7300 tokens, 8 key heads and 32 query heads, half of each turned, with kv_read of them: 64.5 us (82 when a warp went through the
// tokens of one head; 7 more without the loads ahead), 31 at copy rate; issue slots 69 % busy in the append, 57 % in the read, the rest waits
// for loads.  64 single tokens, 8 and 64 heads: 7.3 us, launches and the dependent loads that find a token's place.
#include "kv_int4.cuh"
#include "sm100.cuh"

namespace spb {
namespace {
using namespace sm100;

constexpr int kWarps = 4;

// Sequence of packed row `tok`, its position in the cache (negative: before the start) and the first row behind the sequence -> false when
// the row belongs to no sequence (behind the last one).  The whole warp asks for the same row: 32 offsets are looked at together, since
// a search that halves the range is one load's latency after the other.
__device__ __forceinline__ bool locate(const KvView& c, int tok, int& b, int& pos, int& end)
{
    if (c.cu) {
        const int lane = threadIdx.x & 31;
        int lo = 0, n = c.B;   // the last b with cu[b] <= tok is one of n from lo on
        do {
            const int step = (n + 31) / 32, i = lane * step;
            const uint32_t below = __ballot_sync(0xffffffffu, i < n && c.cu[lo + min(i, n - 1)] <= tok);
            if (!below) return false;   // before the first sequence
            const int k = 31 - __clz(below);
            lo += k * step;
            n = min(step, n - k * step);
        } while (n > 1);
        b = lo;
        end = min(c.cu[b + 1], c.n_tokens);   // as kv_rows takes it
        if (tok >= end) return false;
        pos = c.lens[b] - (end - tok);
    } else {
        b = (unsigned)tok / (unsigned)c.per_seq;
        end = (b + 1) * c.per_seq;
        pos = c.lens[b] - (end - tok);
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
        const bool found = tok < c.n_tokens && locate(c, tok, b, pos, end);
        if (!found) end = 0;
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
// Eight of them, in place of a.  In plain fp32 a sum is off by less than 2^-23 of |b d| + |sum|: when both ends of that range round to the
// same fp16 value it is the right one, and only otherwise (one value in a thousand) is the exact form worked out.
__device__ __forceinline__ void turn8(__half (&a)[2][4], const float (&c)[8], const __half (&b)[2][4], const float (&d)[8])
{
    __half2 low[4], high[4];
    uint32_t differ = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float lo[2], hi[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = i + e;
            const float p = __half2float(b[j / 4][j % 4]) * d[j], s = fmaf(__half2float(a[j / 4][j % 4]), c[j], p), m = fabsf(p) + fabsf(s);
            lo[e] = fmaf(m, -0x1p-23f, s), hi[e] = fmaf(m, 0x1p-23f, s);
        }
        low[i / 2] = __floats2half2_rn(lo[0], lo[1]), high[i / 2] = __floats2half2_rn(hi[0], hi[1]);
        differ |= *reinterpret_cast<const uint32_t*>(&low[i / 2]) ^ *reinterpret_cast<const uint32_t*>(&high[i / 2]);
    }
    if (differ) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const __half2 l = low[j / 2], h = high[j / 2];
            const __half lj = j & 1 ? __high2half(l) : __low2half(l), hj = j & 1 ? __high2half(h) : __low2half(h);
            __half y = lj;
            if (__half_as_ushort(lj) != __half_as_ushort(hj)) y = turn_exactly(__half2float(a[j / 4][j % 4]), c[j], __half2float(b[j / 4][j % 4]), d[j]);
            low[j / 2] = j & 1 ? __halves2half2(__low2half(l), y) : __halves2half2(y, __high2half(l));
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) *reinterpret_cast<uint2*>(a[k]) = *reinterpret_cast<const uint2*>(low + 2 * k);
}

// Cosines and signed sines of position pos for the eight channels from c0 on: y = x c + partner s.
__device__ __forceinline__ void load_angles(const KvAppendArgs& a, int pos, int c0, float (&c)[8], float (&s)[8])
{
    const int half_rot = a.rot / 2;
    const float *cp = a.cosv + (long long)pos * half_rot, *sp = a.sinv + (long long)pos * half_rot;
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
        if (a.interleaved) {
            const float2 cc = *reinterpret_cast<const float2*>(cp + (c0 + k) / 2), ss = *reinterpret_cast<const float2*>(sp + (c0 + k) / 2);
            c[k] = c[k + 1] = cc.x, c[k + 2] = c[k + 3] = cc.y;
            s[k] = -ss.x, s[k + 1] = ss.x, s[k + 2] = -ss.y, s[k + 3] = ss.y;
        } else {
            const bool upper = c0 + k >= half_rot;   // half_rot is a multiple of 4: all four channels on one side
            const int i0 = c0 + k - (upper ? half_rot : 0);
            *reinterpret_cast<float4*>(c + k) = *reinterpret_cast<const float4*>(cp + i0);
            *reinterpret_cast<float4*>(s + k) = *reinterpret_cast<const float4*>(sp + i0);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[k + i] = upper ? s[k + i] : -s[k + i];
        }
    }
}

enum Kind { kKeys, kValues, kQueries };

// Sum of c[i] 2^shift(i) of the codes in the low bits of the floats 1.5 2^23 + c: the floats' other bits are a constant, taken off.
template <int S0, int S1, int S2, int S3>
__device__ __forceinline__ uint32_t pack_codes(const float* t)
{
    constexpr uint32_t kBits = 0x4b400000u, kOff = kBits * ((1u << S0) + (1u << S1) + (1u << S2) + (1u << S3));
    const uint32_t x = __float_as_uint(t[0]) * (1u << S0) + __float_as_uint(t[1]) * (1u << S1);
    return x + __float_as_uint(t[2]) * (1u << S2) + __float_as_uint(t[3]) * (1u << S3) - kOff;
}

constexpr float kRound = 12582912.f;   // 1.5 2^23: a small number added to it is rounded to even in the sum's last bits
// The code of x, as kRound + code: the quotient (x - lo) / s rounded to even.  The quotient by the reciprocal, and of the rounded
// difference, is off by less than 2^-18; next to a border b of two codes it is asked on which side of b s the exact difference lies:
// b s has 16 bits, d - b s is exact, and what the difference lost is the second term.
__device__ __noinline__ float border_code(float x, float lo, float s, float inv)
{
    const float d = __fsub_rn(x, lo), y = __fmaf_rn(d, inv, kRound), r = __fmaf_rn(d, inv, kRound - y);
    if (!(fabsf(r) > 0.5f - 0x1p-16f)) return fminf(y, kRound + 15.f);
    const float b = y - kRound + copysignf(0.5f, r), z = __fsub_rn(d, x), lost = __fadd_rn(__fsub_rn(x, __fsub_rn(d, z)), __fsub_rn(-lo, z));
    const float side = __fadd_rn(__fsub_rn(d, b * s), lost);
    return fminf(side > 0.f ? b + 0.5f : side < 0.f ? b - 0.5f : rintf(b), 15.f) + kRound;
}

// Heads head0, head0 + 32 / (D / 8), .. of one token: `turns` of them for every D/8 lanes, which hold a head's vector.
template <int D, Kind KIND>
__device__ __forceinline__ void append_vectors(const KvAppendArgs& a, int tok, int b, int pos, int head, int turns, int* status)
{
    using L = KvLayout<D>;
    constexpr int kLanes = D / 8, kPer = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, c0 = 8 * sub;
    const int heads = KIND == kQueries ? a.q_heads : a.c.kv_heads;
    bool turning = false;
    float cs[8], sn[8];
    if (a.cosv) {
        if (pos >= a.max_pos) {   // no angles for this position: the whole token is skipped, its values too
            if (lane == 0) atomicOr(status, kStatusBadCache);
            return;
        }
        turning = KIND != kValues && c0 < a.rot;
        if (turning) load_angles(a, pos, c0, cs, sn);
    }
    uint8_t* blk = nullptr;
    const long long head_bytes = (long long)(a.c.page_size / kKvBlock) * L::kBlockBytes;
    if (KIND != kQueries) {
        const long long off = kv_block_offset<D>(a.c, b, 0, pos);
        if (off < 0) {
            if (lane == 0) atomicOr(status, kStatusBadCache);
            return;
        }
        blk = a.c.pool + off + head * head_bytes;
    }
    const long long head_step = KIND == kQueries ? a.q_head : KIND == kValues ? a.v_head : a.k_head;
    const uint16_t* src = KIND == kQueries ? a.q + tok * a.q_tok : KIND == kValues ? a.v + tok * a.v_tok : a.k + tok * a.k_tok;
    src += head * head_step + c0;
    uint16_t* dst = KIND == kQueries ? a.q_out + ((long long)tok * a.q_heads + head) * D + c0 : nullptr;
    const int half_rot = a.rot / 2, t16 = pos % kKvBlock;
    uint2 next[2] = {make_uint2(0, 0), make_uint2(0, 0)};   // the next turn's channels
    if (head < heads) next[0] = reinterpret_cast<const uint2*>(src)[0], next[1] = reinterpret_cast<const uint2*>(src)[1];
    for (int i = 0; i < turns; ++i, head += kPer, src += kPer * head_step, blk += kPer * head_bytes, dst += kPer * D) {
        const bool there = head < heads;
        __half x[2][4];
        *reinterpret_cast<uint2*>(x[0]) = next[0], *reinterpret_cast<uint2*>(x[1]) = next[1];
        if (i + 1 < turns && head + kPer < heads) {
            const uint2* p = reinterpret_cast<const uint2*>(src + kPer * head_step);
            next[0] = p[0], next[1] = p[1];
        }
        if (there) {
            if (KIND != kValues && turning) {
                __half w[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (a.interleaved) w[k][0] = x[k][1], w[k][1] = x[k][0], w[k][2] = x[k][3], w[k][3] = x[k][2];
                    else load4(src + 4 * k + (c0 + 4 * k >= half_rot ? -half_rot : half_rot), w[k]);
                }
                turn8(x, cs, w, sn);
            }
        }
        if (KIND == kQueries) {
            __syncwarp();   // q_out may be q: all lanes of a vector have read it
            if (there) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(x);
            continue;
        }
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
        // kRound + code, by the reciprocal; border_code where that might not decide
        float t[8];
        bool near = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float d = __fsub_rn(__half2float(x[k / 4][k % 4]), lo), y = __fmaf_rn(d, inv, kRound);
            near = near || fabsf(__fmaf_rn(d, inv, kRound - y)) > 0.5f - 0x1p-16f;
            t[k] = fminf(y, kRound + 15.f);
        }
        if (near)
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = border_code(__half2float(x[k / 4][k % 4]), lo, sf, inv);
        __half m = __float2half_rn(lo);
        const bool plain = finite && sf > 0.f;   // a constant group has no codes
        if (!finite) s = m = __ushort_as_half((unsigned short)0x7fff);
        // Keys: words t and t + 1 of the group; this lane has the nibbles of one of their two halves, the lane two away those of the
        // other.  Values: a byte for each of four channel pairs, whose other byte of the halfword that lane has.
        uint32_t mine[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) mine[k] = !plain ? 0u : KIND == kValues ? pack_codes<0, 4, 16, 20>(t + 4 * k) : pack_codes<0, 16, 8, 24>(t + 4 * k);
        const bool upper = sub & 2;
        const uint32_t other = __shfl_xor_sync(0xffffffffu, mine[upper ? 0 : 1], 2), kept = mine[upper ? 1 : 0];
        constexpr int kShift = KIND == kValues ? 8 : 4;
        const uint32_t word = upper ? other | kept << kShift : kept | other << kShift;
        if (!there) continue;
        const int grp = sub / 4, pair = 2 * (sub & 1) + upper;   // the word or the two channel pairs this lane stores
        if (KIND == kKeys) {
            reinterpret_cast<uint32_t*>(blk + L::kKCodes)[t16 * (D / 8) + pair * L::kGroups + grp] = word;
            if ((sub & 3) == 0) reinterpret_cast<__half2*>(blk + L::kKParams)[t16 * L::kGroups + grp] = __halves2half2(s, m);
        } else {
            const int j = t16 / 8, t2 = (t16 % 8) / 2, e = t16 & 1;
            uint8_t* p = blk + L::kVCodes + j * 4 * D + (4 * 2 * pair + t2) * (D / 8) + 4 * grp + 2 * e;
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

// A warp takes some vectors of one kind of one token, so that the token's place and its angles are found once: kv_turns (q_turns) times as
// many keys or values (queries) as it holds at once, kv_warps (q_warps) warps for all of them.
struct AppendPlan {
    int kv_turns, kv_warps, q_turns, q_warps;
};
// Registers for 8 thread blocks an SM: 7 took 68 us, 9 took 66 where these took 63.
template <int D>
__global__ void __launch_bounds__(32 * kWarps, 8) kv_append_kernel(KvAppendArgs a, AppendPlan plan, int* status)
{
    constexpr int kPer = 32 / (D / 8);
    grid_wait();
    grid_release();
    const int per = 2 * plan.kv_warps + plan.q_warps, sub_head = (threadIdx.x & 31) / (D / 8);
    const unsigned item = blockIdx.x * kWarps + threadIdx.x / 32, tok = item / per;
    const int part = item - tok * per;
    int b, pos, end;
    if (tok >= (unsigned)a.c.n_tokens || !locate(a.c, (int)tok, b, pos, end) || pos < 0) return;
    if (part < plan.kv_warps) append_vectors<D, kKeys>(a, tok, b, pos, part * plan.kv_turns * kPer + sub_head, plan.kv_turns, status);
    else if (part < 2 * plan.kv_warps) append_vectors<D, kValues>(a, tok, b, pos, (part - plan.kv_warps) * plan.kv_turns * kPer + sub_head, plan.kv_turns, status);
    else append_vectors<D, kQueries>(a, tok, b, pos, (part - 2 * plan.kv_warps) * plan.q_turns * kPer + sub_head, plan.q_turns, status);
}

// The values of one vector, eight channels a lane: m + code * s with one rounding.
template <int D>
__global__ void __launch_bounds__(32 * kWarps) kv_read_kernel(KvReadArgs a, int rows, int* status)
{
    using L = KvLayout<D>;
    constexpr int kLanes = D / 8, kPer = 32 / kLanes;
    grid_wait();
    grid_release();
    const int lane = threadIdx.x & 31, sub = lane % kLanes, c0 = 8 * sub, grp = sub / 4;
    const unsigned vecs = 2 * a.c.kv_heads, warps = (vecs + kPer - 1) / kPer;   // of a token
    const unsigned item = blockIdx.x * kWarps + threadIdx.x / 32, chunk = item / warps, vec = (item - chunk * warps) * kPer + lane / kLanes;
    const bool is_v = vec >= a.c.kv_heads;
    const int head = is_v ? vec - a.c.kv_heads : vec;
    uint16_t* out = (is_v ? a.v : a.k) + head * D + c0;
    Cursor at;
    for (int i = 0; i < rows; ++i) {
        const int tok = (int)chunk * rows + i;
        if (!at.move_to(a.c, tok) || vec >= vecs) continue;
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

// Vectors of a token, or tokens, that a warp goes through: up to eight when that still leaves the device full (64 warps on each of some 150
// SMs), else one.
bool many(long long vectors) { return vectors >= 8ll * 64 * 150; }
// Both kernels may be set up before what precedes them has ended.
template <class Args, class... More>
cudaError_t start(cudaStream_t s, void (*kernel)(Args, More...), long long warps, const Args& a, More... more)
{
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((warps + kWarps - 1) / kWarps));
    cfg.blockDim = dim3(32 * kWarps);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, more...);
    count_launch();
    return e;
}

}  // namespace

cudaError_t kv_append_launch(cudaStream_t s, int D, const KvAppendArgs& a, int* status)
{
    const int at_once = 256 / D, kv = (a.c.kv_heads + at_once - 1) / at_once, q = a.q ? (a.q_heads + at_once - 1) / at_once : 0;
    const int most = many((long long)a.c.n_tokens * (2 * a.c.kv_heads + (a.q ? a.q_heads : 0))) ? 8 : 1;
    AppendPlan plan;
    plan.kv_warps = (kv + most - 1) / most, plan.kv_turns = (kv + plan.kv_warps - 1) / plan.kv_warps;
    plan.q_warps = (q + most - 1) / most, plan.q_turns = q ? (q + plan.q_warps - 1) / plan.q_warps : 0;
    const long long warps = (long long)a.c.n_tokens * (2 * plan.kv_warps + plan.q_warps);
    return D == 128 ? start(s, kv_append_kernel<128>, warps, a, plan, status) : start(s, kv_append_kernel<64>, warps, a, plan, status);
}

cudaError_t kv_read_launch(cudaStream_t s, int D, const KvReadArgs& a, int* status)
{
    const int vecs = 2 * a.c.kv_heads, rows = many((long long)a.c.n_tokens * vecs) ? 8 : 1;
    const long long warps = (a.c.n_tokens + rows - 1ll) / rows * ((vecs + 256 / D - 1) / (256 / D));
    return D == 128 ? start(s, kv_read_kernel<128>, warps, a, rows, status) : start(s, kv_read_kernel<64>, warps, a, rows, status);
}

}  // namespace spb
