// Attention over the paged 4-bit cache (layout: kv_int4.cuh):  out = softmax(q K^T scale) V  with K = m + s c, V likewise.
//
// kv_attention_split_kernel: few query rows a key head (decoding, drafts).  Everything is transposed, keys and channels on
// the 16-row side of mma.sync.m16n8k16 and query rows on its 8-column side, so that a single row wastes 7/8 of a cheap
// operand and not of the cache's.  Codes are never expanded: a nibble masked out of its word is an fp16 subnormal, c 2^-24 (low
// nibble of a byte) or c 2^-20 (high), which the instruction multiplies exactly, so unpacking costs 1.25 instructions per pair
// of codes.  Scales and minima are applied around the products, in fp32 for the keys and on the weights for the values:
//
//   scores   S^T = K Q^T per group of 32 channels, z = sum over groups of s (q.c) + m sum(q); the second term is one more matrix
//            instruction on the group sums of q, split into two fp16 values.  The high nibbles' share of q is divided by 16
//            beforehand; q is first multiplied by a power of two that brings its row's largest magnitude to [2^8, 2^9), so that the
//            division loses nothing above 2^-25 of that magnitude.
//   softmax  running maximum and sum in fp32 per row, in base 2.  The accumulators are only rescaled when a maximum grows by more
//            than 2^8; weights are kept 2^7 too large, so that in fp16 they span 2^-31 .. 1 relative to the largest.
//   values   O^T = sum over tokens of (P s) c + P m: P^T comes from S^T with two 8 x 8 transposes in registers and is multiplied
//            by the tokens' scales, one product per group, rounded to fp16 like P itself; the minima are one more matrix
//            instruction per 16 tokens.  The scales of a group are first brought to 1 .. 2 by the power of two of the largest one so far,
//            so that the products, too, span 2^-31 .. 1 relative to the largest (down to scales of 2^-15, whose values are next to the
//            smallest of fp16); when a larger one comes, the group's accumulators are scaled down.  The roundings of P and of P s average out over many keys; over
//            few they would make outputs half again as far from the exact ones (five keys: 3.0e-4, the rounding of the output alone
//            2.0e-4).  Row tiles whose first row sees at most 128 keys take a second product with what the roundings took away.
//
// Work: the context is cut in units of 128 tokens (four warps, two 16-token blocks each); all units of all (sequence, key
// head, row tile) are laid end to end and every thread block takes an equal share, found from the lengths on the device.
// A share that covers a whole row tile is finished where it is; the others leave fp32 (O, max, sum) in the workspace,
// two slots a thread block, and kv_attention_join_kernel adds them in order: no atomics, the same bits every time.
// Every warp streams its own blocks: bulk copies into its own ring, nobody waits for another warp except at
// the end of a row tile.
//
// Bound: the cache's bytes when there are enough of them, else the launches, a unit's latency and the join.  One row, 32 query heads on 8,
// 262139 tokens: 79 us, 4.25 TB/s; 32 sequences of up to 8191 tokens, 64 heads on 8: 65 us, 3.9 TB/s (issue slots 56-57 % busy, tensor pipe
// 22-25 %).  One sequence of 131 tokens: 9.3 us, a third of it launch at most (a linear layer with its launch takes 3.6); the rest is one
// dependent step after the other: lengths, list, table, the first copy, and two units of 128 tokens in a row on 40 thread blocks.
#include "kv_int4.cuh"
#include "sm100.cuh"

namespace spb {
namespace {
using namespace sm100;

constexpr int kWarps = 4;
constexpr float kShift = 7.f, kSlack = 8.f;
// 16-token blocks a warp takes per step (they share the operands of q and the softmax's bookkeeping: two measured 105 -> 82 us at
// 262139 tokens) and steps in flight per warp.
constexpr int TT = 2, kStages = 2;
constexpr int kUnit = kKvBlock * kWarps * TT;   // tokens a thread block advances per step
// Tiles of 8 query rows a thread block takes: one, or two for more than 8 rows.  Four (32 rows) left two thread blocks of 255
// registers per SM and took 210 us where two take 122 (16 sequences of 8000, 32 rows); one took 156, reading the cache twice as often.
int pick_nt(long long rows) { return rows <= 8 ? 1 : 2; }
__host__ __device__ constexpr int blocks_per_sm(int nt) { return nt == 1 ? 3 : 2; }
__device__ __forceinline__ bool wait_full(uint32_t bar, uint32_t parity)
{
    for (uint32_t i = 0; i < kSpinLimit; ++i) {
        if (mbar_try(bar, parity)) return true;
        if (i > 1024) __nanosleep(40);
    }
    return false;
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }

__device__ __forceinline__ float power(int exponent) { return __int_as_float((127 + exponent) << 23); }
__device__ __forceinline__ int exponent_of(__half2 power_of_two) { return (int)(h2_bits(power_of_two) >> 26) - 15; }

// Sequence b of the work list.
struct Seq {
    int b = 0;
    int len = 0, qlen = 0, tiles = 0;   // tokens in the cache, new tokens, row tiles
    int first = 0;                      // first packed row
    int units = 0;                      // units of one row tile
    int begin = 0, total = 0;           // its range of the list
};
template <int ROWS>
__device__ __forceinline__ void load_seq(Seq& s, const KvView& c, int b, int group, int tall)
{
    kv_rows(c, b, s.first, s.qlen);
    s.b = b;
    s.len = max(c.lens[b], 0);
    s.tiles = s.qlen * group >= tall ? 0 : (s.qlen * group + ROWS - 1) / ROWS;
    // tokens past the table's width have no page: they are not walked over
    const int held = (int)min((long long)s.len, (long long)c.table_stride * c.page_size);
    s.units = max((held - 1) / kUnit + 1, 1);
    s.total = (int)min((long long)c.kv_heads * s.tiles * s.units, 0x7fffffffll);   // as much makes the list too long
}
// The list as a warp sees it: its length, and of up to 32 sequences lane b's, so that finding one needs no second look at memory.
template <int ROWS>
struct List {
    Seq mine;
    int total;       // units of the list
    bool too_long;   // 2^31 units or next to it: refused, here, where the lengths are known (a table may be far wider than they need)
    __device__ __forceinline__ List(const KvView& c, int group, int tall)
    {
        const int lane = threadIdx.x & 31;
        long long sum = 0;
        for (int b = lane; b < c.B; b += 32) {
            load_seq<ROWS>(mine, c, b, group, tall);
            sum += mine.total;
        }
        total = (int)__reduce_add_sync(0xffffffffu, (unsigned)sum);
        too_long = __reduce_add_sync(0xffffffffu, (unsigned)min((sum + (1 << 20) - 1) >> 20, 1ll << 20)) >= 1u << 11;   // rounded up in each lane
    }
    // The sequence that holds unit x of the list (x inside the list); every lane gets the same.
    __device__ __forceinline__ void find(Seq& s, const KvView& c, int group, int tall, int x)
    {
        const int lane = threadIdx.x & 31;
        int before = 0;
        for (int b0 = 0; b0 < c.B; b0 += 32) {
            Seq t;
            if (c.B <= 32) t = mine;
            else if (b0 + lane < c.B) load_seq<ROWS>(t, c, b0 + lane, group, tall);
            int incl = t.total;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + incl > x);
            if (past) {
                const int l = __ffs(past) - 1;
                s.b = b0 + l;
                s.len = __shfl_sync(0xffffffffu, t.len, l), s.qlen = __shfl_sync(0xffffffffu, t.qlen, l);
                s.tiles = __shfl_sync(0xffffffffu, t.tiles, l), s.first = __shfl_sync(0xffffffffu, t.first, l);
                s.units = __shfl_sync(0xffffffffu, t.units, l), s.total = __shfl_sync(0xffffffffu, t.total, l);
                s.begin = before + __shfl_sync(0xffffffffu, incl - t.total, l);
                return;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
};
template <int ROWS>
__device__ __forceinline__ void next_seq(Seq& s, const KvView& c, int group, int tall)
{
    do {
        const int end = s.begin + s.total;
        load_seq<ROWS>(s, c, s.b + 1, group, tall);
        s.begin = end;
    } while (s.total == 0 && s.b + 1 < c.B);
}
// Thread block i of n takes total / n units, the first total % n of them one more.
struct Shares {
    int share, extra;
    __device__ __forceinline__ Shares(int total, int n) : share(total / n), extra(total - total / n * n) {}
    __device__ __forceinline__ int begin(int i) const { return i * share + min(i, extra); }
    __device__ __forceinline__ int of(int x) const   // thread block that has unit x
    {
        const int big = extra * (share + 1);
        return x < big ? x / (share + 1) : extra + (x - big) / share;
    }
};

// ws: slot n (two per thread block): [rows][D] sums, then [rows] maxima and [rows] sums of weights
template <int D, int ROWS>
__host__ __device__ constexpr size_t slot_floats() { return (size_t)ROWS * (D + 2); }

// Keys that row r of a sequence's rows may see.
__device__ __forceinline__ int visible_keys(const Seq& s, int row, int group)
{
    return max(s.len - s.qlen + row / group + 1, 0);
}

template <int D, int NT>
struct Smem {
    alignas(128) uint8_t ring[kWarps][kStages][TT * KvLayout<D>::kBlockBytes];
    alignas(16) float merge[kWarps - 1][NT * (D / 16) * 4 * 32 + 4 * NT * 32];
    uint2 qfrag[NT][D / 16][32];   // q operand, [tile of 8 rows][k-step][lane]
    uint32_t qsum[NT][32];         // group sums of q as an operand: lane 4 g + t holds groups 2 (t & 1), + 1 of row g, high (t < 2) or low part
    float factor[NT][8];           // score sums -> base-2 scores
    uint64_t full[kWarps][kStages];
    int ok[kWarps][kStages];    // blocks of the step that are there
};

// What a warp has of a row tile.
template <int D, int NT>
struct Sums {
    float o[NT][D / 16][4];    // sum of P s c in units of the group, rows of the high nibbles 2^-20, of the low ones 2^-24 of it
    float om[NT][4];           // sum of P m, row = group
    float mx[NT][2], sum[NT][2];
    __half2 unit[D / kKvGroup];   // 2^-e of a group, e the exponent of its largest scale so far, -15 at least
};
// A warp's two blocks of a unit and how the tile's rows see them.
struct Unit {
    const uint8_t* blocks;
    int there, pos;            // bits of the blocks that are there, first token
    int kmin, kmax;            // keys that the first and the last row see
    int before, row0, group;   // row r of the tile sees before + (row0 + r) / group keys, if that is positive
};
// FINE: the second product is taken.
template <int D, int NT, bool FINE>
__device__ __forceinline__ void attend(Sums<D, NT>& x, const Smem<D, NT>& sm, const Unit& u)
{
    using L = KvLayout<D>;
    constexpr int G = L::kGroups, MT = D / 16;
    const int lane = threadIdx.x & 31, g = lane / 4, t = lane % 4, there = u.there, pos0 = u.pos;
    const uint8_t* blk0 = u.blocks;
    auto &o = x.o;
    auto &om = x.om;
    auto &mx = x.mx, &sum = x.sum;
    auto &unit = x.unit;
    auto rescale = [&](int nt, float r0, float r1, const float (&down)[G]) {   // rows by r0, r1, groups by down
        sum[nt][0] *= r0, sum[nt][1] *= r1;
        om[nt][0] *= r0, om[nt][1] *= r1;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const float d0 = r0 * down[i / 2], d1 = r1 * down[i / 2];
            o[nt][i][0] *= d0, o[nt][i][1] *= d1, o[nt][i][2] *= d0, o[nt][i][3] *= d1;
        }
    };
        // some row does not see all of these tokens, or a block is not there: it counts as unseen
        const bool edge = pos0 + TT * kKvBlock > u.kmin || there != (1 << TT) - 1;
        auto seen_by = [&](int row, int k) {   // tokens of block k that a row of the tile sees
            return (there >> k & 1) ? max(u.before + (u.row0 + row) / u.group, 0) - (pos0 + k * kKvBlock) : 0;
        };
        // ---- scores.  keys: one word of codes per group for tokens g and g + 8
        uint32_t k0[TT][G], k1[TT][G], p0[TT][G], p1[TT][G];
#pragma unroll
        for (int k = 0; k < TT; ++k) {
            const uint32_t* kc = reinterpret_cast<const uint32_t*>(blk0 + k * L::kBlockBytes + L::kKCodes);
            const uint32_t* kp = reinterpret_cast<const uint32_t*>(blk0 + k * L::kBlockBytes + L::kKParams);
            if constexpr (G == 4) {
                *reinterpret_cast<uint4*>(k0[k]) = *reinterpret_cast<const uint4*>(kc + g * 16 + t * 4);
                *reinterpret_cast<uint4*>(k1[k]) = *reinterpret_cast<const uint4*>(kc + (g + 8) * 16 + t * 4);
                *reinterpret_cast<uint4*>(p0[k]) = *reinterpret_cast<const uint4*>(kp + g * 4);
                *reinterpret_cast<uint4*>(p1[k]) = *reinterpret_cast<const uint4*>(kp + (g + 8) * 4);
            } else {
                *reinterpret_cast<uint2*>(k0[k]) = *reinterpret_cast<const uint2*>(kc + g * 8 + t * 2);
                *reinterpret_cast<uint2*>(k1[k]) = *reinterpret_cast<const uint2*>(kc + (g + 8) * 8 + t * 2);
                *reinterpret_cast<uint2*>(p0[k]) = *reinterpret_cast<const uint2*>(kp + g * 2);
                *reinterpret_cast<uint2*>(p1[k]) = *reinterpret_cast<const uint2*>(kp + (g + 8) * 2);
            }
        }
        float z[TT][NT][4];
        {
            // minima of the lane's two groups, as an operand (lanes without a group: zero)
            uint32_t qs[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) qs[nt] = sm.qsum[nt][lane];
#pragma unroll
            for (int k = 0; k < TT; ++k) {
                uint32_t am[4] = {0u, 0u, 0u, 0u};
                if constexpr (G == 4) {
                    const bool odd = t & 1;
                    am[0] = __byte_perm(odd ? p0[k][2] : p0[k][0], odd ? p0[k][3] : p0[k][1], 0x7632);
                    am[1] = __byte_perm(odd ? p1[k][2] : p1[k][0], odd ? p1[k][3] : p1[k][1], 0x7632);
                } else if (!(t & 1)) {
                    am[0] = __byte_perm(p0[k][0], p0[k][1], 0x7632);
                    am[1] = __byte_perm(p1[k][0], p1[k][1], 0x7632);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    z[k][nt][0] = z[k][nt][1] = z[k][nt][2] = z[k][nt][3] = 0.f;
                    mma(z[k][nt], am, qs[nt], 0u);
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[k][nt][i] *= 0x1p-24f;
                }
            }
        }
#pragma unroll
        for (int w = 0; w < G; ++w) {
            uint2 ql[NT], qh[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) ql[nt] = sm.qfrag[nt][2 * w][lane], qh[nt] = sm.qfrag[nt][2 * w + 1][lane];
#pragma unroll
            for (int k = 0; k < TT; ++k) {
                const uint32_t u = k0[k][w], v = k1[k][w], us = u >> 8, vs = v >> 8;
                const uint32_t alow[4] = {u & 0x000f000fu, v & 0x000f000fu, us & 0x000f000fu, vs & 0x000f000fu};
                const uint32_t ahigh[4] = {u & 0x00f000f0u, v & 0x00f000f0u, us & 0x00f000f0u, vs & 0x00f000f0u};
                const float s0 = __low2float(as_h2(p0[k][w])), s1 = __low2float(as_h2(p1[k][w]));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                    mma(acc, alow, ql[nt].x, ql[nt].y);
                    mma(acc, ahigh, qh[nt].x, qh[nt].y);
                    z[k][nt][0] = fmaf(s0, acc[0], z[k][nt][0]);
                    z[k][nt][1] = fmaf(s0, acc[1], z[k][nt][1]);
                    z[k][nt][2] = fmaf(s1, acc[2], z[k][nt][2]);
                    z[k][nt][3] = fmaf(s1, acc[3], z[k][nt][3]);
                }
            }
        }
        // ---- scales of the values of tokens 2t, 2t+1 (j = 0) and 2t+8, 2t+9 (j = 1), all groups; minima of group g
        uint32_t vs[TT][2][G], vm[TT][2], large = 0;   // large: bit 14 of an fp16 value, 2 or more
        __half2 most[G];   // of a group's scales here
#pragma unroll
        for (int k = 0; k < TT; ++k) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t* vp = reinterpret_cast<const uint32_t*>(blk0 + k * L::kBlockBytes + L::kVParams) + (t + 4 * j) * 2 * G;
                if constexpr (G == 4) {
                    const uint4 u = *reinterpret_cast<const uint4*>(vp), w = *reinterpret_cast<const uint4*>(vp + 4);
                    vs[k][j][0] = u.x, vs[k][j][1] = u.z, vs[k][j][2] = w.x, vs[k][j][3] = w.z;
                } else {
                    const uint4 u = *reinterpret_cast<const uint4*>(vp);
                    vs[k][j][0] = u.x, vs[k][j][1] = u.z;
                }
                vm[k][j] = g < G ? vp[2 * (g & (G - 1)) + 1] : 0u;
            }
        }
        if (edge) {
            // Tokens that no row sees count as zero, whatever the page holds there.  A token that some rows see and
            // others do not may be NaN for the first and must not touch the others: it is taken out of the products
            // and put back row by row.
#pragma unroll
            for (int k = 0; k < TT; ++k) {
                uint32_t nan_tokens[G] = {};
                bool any = false;
                const int in_sight = (there >> k & 1) ? u.kmax - (pos0 + k * kKvBlock) : 0;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int tok = 2 * t + 8 * j + e;
                        const uint32_t keep = e ? 0x0000ffffu : 0xffff0000u;
                        const bool unseen = tok >= in_sight;
#pragma unroll
                        for (int w = 0; w < G; ++w) {
                            const bool bad = ((vs[k][j][w] >> 16 * e) & 0x7c00u) == 0x7c00u;
                            if (bad && !unseen) nan_tokens[w] |= 1u << tok, any = true;
                            if (bad || unseen) vs[k][j][w] &= keep;
                        }
                        if (unseen || ((vm[k][j] >> 16 * e) & 0x7c00u) == 0x7c00u) vm[k][j] &= keep;
                    }
                if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                    for (int w = 0; w < G; ++w) {   // the quad holds all 16 tokens
                        nan_tokens[w] |= __shfl_xor_sync(0xffffffffu, nan_tokens[w], 1);
                        nan_tokens[w] |= __shfl_xor_sync(0xffffffffu, nan_tokens[w], 2);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int seen = seen_by(nt * 8 + 2 * t + e, k);
                            const uint32_t mask = seen >= 16 ? 0xffffu : seen <= 0 ? 0u : (1u << seen) - 1;
#pragma unroll
                            for (int i = 0; i < MT; ++i)
                                if (nan_tokens[i / 2] & mask) o[nt][i][e] = o[nt][i][2 + e] = __int_as_float(0x7fffffff);
                        }
                }
            }
        }
#pragma unroll
        for (int w = 0; w < G; ++w) {
            most[w] = __hmax2(as_h2(vs[0][0][w]), as_h2(vs[0][1][w]));
#pragma unroll
            for (int k = 1; k < TT; ++k) most[w] = __hmax2(most[w], __hmax2(as_h2(vs[k][0][w]), as_h2(vs[k][1][w])));
            large |= h2_bits(__hmul2(most[w], unit[w]));
        }
        // ---- softmax
        bool grow = (large & 0x40004000u) != 0;
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float2 f = *reinterpret_cast<const float2*>(&sm.factor[nt][2 * t]);
#pragma unroll
            for (int k = 0; k < TT; ++k) {
                z[k][nt][0] *= f.x, z[k][nt][2] *= f.x;
                z[k][nt][1] *= f.y, z[k][nt][3] *= f.y;
                if (edge) {
                    const int s0 = seen_by(nt * 8 + 2 * t, k), s1 = seen_by(nt * 8 + 2 * t + 1, k);
                    if (g >= s0) z[k][nt][0] = -INFINITY;
                    if (g >= s1) z[k][nt][1] = -INFINITY;
                    if (g + 8 >= s0) z[k][nt][2] = -INFINITY;
                    if (g + 8 >= s1) z[k][nt][3] = -INFINITY;
                }
                const float n0 = fmaxf(z[k][nt][0], z[k][nt][2]), n1 = fmaxf(z[k][nt][1], z[k][nt][3]);
                top[nt][0] = k ? fmaxf(top[nt][0], n0) : n0;
                top[nt][1] = k ? fmaxf(top[nt][1], n1) : n1;
            }
            grow = grow || top[nt][0] > mx[nt][0] + kSlack || top[nt][1] > mx[nt][1] + kSlack;
        }
        if (__any_sync(0xffffffffu, grow)) {
            float down[G];
#pragma unroll
            for (int w = 0; w < G; ++w) {
                // the largest scale by its bits; an infinity or NaN, and what no fp16 range of values has, asks for nothing
                const uint32_t x = h2_bits(most[w]), hi = max(x & 0x7fffu, x >> 16 & 0x7fffu), e = __reduce_max_sync(0xffffffffu, hi) >> 10;
                const __half2 was = unit[w];
                if (e < 30) unit[w] = __hmin2(was, __half2half2(__ushort_as_half((unsigned short)((30 - e) << 10))));
                down[w] = power(exponent_of(unit[w]) - exponent_of(was));
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float n0 = top[nt][0], n1 = top[nt][1];
#pragma unroll
                for (int d = 4; d < 32; d *= 2) {
                    n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, d));
                    n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, d));
                }
                n0 = fmaxf(n0, mx[nt][0]), n1 = fmaxf(n1, mx[nt][1]);
                const float r0 = mx[nt][0] == -INFINITY ? 0.f : exp2_approx(mx[nt][0] - n0);
                const float r1 = mx[nt][1] == -INFINITY ? 0.f : exp2_approx(mx[nt][1] - n1);
                mx[nt][0] = n0, mx[nt][1] = n1;
                rescale(nt, r0, r1, down);
            }
        }
        uint32_t b0[TT][NT], b1[TT][NT], r0[TT][NT], r1[TT][NT];   // r: what rounding to fp16 took away, for short contexts
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float m0 = (mx[nt][0] == -INFINITY ? 0.f : mx[nt][0]) - kShift;
            const float m1 = (mx[nt][1] == -INFINITY ? 0.f : mx[nt][1]) - kShift;
#pragma unroll
            for (int k = 0; k < TT; ++k) {
                const float w0 = exp2_approx(z[k][nt][0] - m0), w1 = exp2_approx(z[k][nt][1] - m1);
                const float w2 = exp2_approx(z[k][nt][2] - m0), w3 = exp2_approx(z[k][nt][3] - m1);
                sum[nt][0] += w0 + w2;
                sum[nt][1] += w1 + w3;
                b0[k][nt] = transpose8x8(h2_bits(__floats2half2_rn(w0, w1)));
                b1[k][nt] = transpose8x8(h2_bits(__floats2half2_rn(w2, w3)));
                if constexpr (FINE) {
                    r0[k][nt] = transpose8x8(h2_bits(__floats2half2_rn(w0 - __half2float(__float2half_rn(w0)), w1 - __half2float(__float2half_rn(w1)))));
                    r1[k][nt] = transpose8x8(h2_bits(__floats2half2_rn(w2 - __half2float(__float2half_rn(w2)), w3 - __half2float(__float2half_rn(w3)))));
                }
            }
        }
        // ---- weighted values
#pragma unroll
        for (int k = 0; k < TT; ++k) {
            uint32_t vw[2][G];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint8_t* vc = blk0 + k * L::kBlockBytes + L::kVCodes + j * 4 * D + lane * (D / 8);
                if constexpr (G == 4) *reinterpret_cast<uint4*>(vw[j]) = *reinterpret_cast<const uint4*>(vc);
                else *reinterpret_cast<uint2*>(vw[j]) = *reinterpret_cast<const uint2*>(vc);
            }
            const uint32_t am[4] = {vm[k][0], 0u, vm[k][1], 0u};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma(om[nt], am, b0[k][nt], b1[k][nt]);
                if constexpr (FINE) mma(om[nt], am, r0[k][nt], r1[k][nt]);
            }
#pragma unroll
            for (int w = 0; w < G; ++w) {
                const uint32_t x0 = vw[0][w], x1 = vw[1][w], y0 = x0 >> 8, y1 = x1 >> 8;
                const uint32_t even[4] = {x0 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x000f000fu, x1 & 0x00f000f0u};
                const uint32_t odd[4] = {y0 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x000f000fu, y1 & 0x00f000f0u};
                const __half2 v0 = __hmul2(as_h2(vs[k][0][w]), unit[w]), v1 = __hmul2(as_h2(vs[k][1][w]), unit[w]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint32_t c0 = h2_bits(__hmul2(as_h2(b0[k][nt]), v0)), c1 = h2_bits(__hmul2(as_h2(b1[k][nt]), v1));
                    mma(o[nt][2 * w], even, c0, c1);
                    mma(o[nt][2 * w + 1], odd, c0, c1);
                    if constexpr (FINE) {   // P s less its rounded product
                        const uint32_t d0 = h2_bits(__hfma2(as_h2(r0[k][nt]), v0, __hfma2(as_h2(b0[k][nt]), v0, __hneg2(as_h2(c0)))));
                        const uint32_t d1 = h2_bits(__hfma2(as_h2(r1[k][nt]), v1, __hfma2(as_h2(b1[k][nt]), v1, __hneg2(as_h2(c1)))));
                        mma(o[nt][2 * w], even, d0, d1);
                        mma(o[nt][2 * w + 1], odd, d0, d1);
                    }
                }
            }
        }
}
// A function of its own, on a copy of the sums: in the kernel's loop, as a branch or as a second loop, it made long contexts up to 10 %
// slower by the registers it took (8 sequences of up to 1087 tokens, 40 heads: 25.2 us as a second loop, 23.8 so, 23.2 without).
template <int D, int NT>
__device__ __noinline__ void attend_fine(Sums<D, NT>& x, const Smem<D, NT>& sm, const Unit& u)
{
    attend<D, NT, true>(x, sm, u);
}

// SHORT: the table holds no more than one unit, so that every row tile is fine: no call for it (9.0 us against 10.2: 25 sequences of 5
// tokens, 12 heads).  The arithmetic is the same.
template <int D, int NT, bool SHORT>
__global__ void __launch_bounds__(32 * kWarps, blocks_per_sm(NT)) kv_attention_split_kernel(KvAttnArgs a, int whole_tiles, int* status)
{
    using L = KvLayout<D>;
    constexpr int G = L::kGroups, KS = D / 16, MT = D / 16, ROWS = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem<D, NT>& sm = *reinterpret_cast<Smem<D, NT>*>(smem_raw);
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane / 4, t = lane % 4;
    const KvView& c = a.c;
    const int group = a.q_heads / c.kv_heads;

    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(smem_u32(&sm.full[warp][i]), 1);
        mbar_init_fence();
    }
    __syncthreads();
    grid_wait();
    grid_release();   // the join may be set up while this kernel runs; it waits for its end

    List<ROWS> list(c, group, a.tall);
    if (list.too_long) {
        if (threadIdx.x == 0) atomicOr(status, kStatusBadCache);
        return;
    }
    const Shares shares(list.total, gridDim.x);
    int lo = shares.begin(blockIdx.x), hi = shares.begin(blockIdx.x + 1);
    Seq s;
    if (whole_tiles) {   // short contexts: the ends of a share move up to the next row tile, nothing is cut
        auto next_tile = [&](int x) {
            if (x >= list.total) return list.total;
            list.find(s, c, group, a.tall, x);
            return s.begin + (x - s.begin + s.units - 1) / s.units * s.units;
        };
        lo = next_tile(lo), hi = next_tile(hi);
    }
    const int count = hi - lo;
    if (count <= 0) return;
    list.find(s, c, group, a.tall, lo);

    // ---- segments: runs of units of one row tile
    struct Segment {
        int h, rt, rows, kmin, kmax, tile_begin, begin, end;
        bool whole;
    } seg;
    auto set_segment = [&](int x) {
        while (x >= s.begin + s.total) next_seq<ROWS>(s, c, group, a.tall);
        const int pair = (x - s.begin) / s.units;
        seg.h = pair / s.tiles;
        seg.rt = pair - seg.h * s.tiles;
        seg.tile_begin = s.begin + pair * s.units;
        seg.begin = x;
        seg.end = min(hi, seg.tile_begin + s.units);
        seg.whole = x == seg.tile_begin && seg.end == seg.tile_begin + s.units;
        seg.rows = min(ROWS, s.qlen * group - seg.rt * ROWS);   // rows of this tile
        seg.kmin = visible_keys(s, seg.rt * ROWS, group), seg.kmax = visible_keys(s, seg.rt * ROWS + seg.rows - 1, group);
    };
    uint2 raw[KS];   // q of the next segment's rows, warps below NT: 8 rows each
    auto load_q = [&]() {
        const int row = warp * 8 + g, abs_row = seg.rt * ROWS + row;
        const bool have = row < seg.rows;
        const uint16_t* src = a.q + (long long)(s.first + (have ? abs_row / group : 0)) * a.q_tok + (seg.h * group + (have ? abs_row % group : 0)) * a.q_head;
        if (warp < NT)
#pragma unroll
            for (int j = 0; j < KS; ++j) raw[j] = have ? *reinterpret_cast<const uint2*>(src + 16 * j + 4 * t) : make_uint2(0, 0);
    };
    set_segment(lo);
    load_q();

    // ---- this warp's copies: lane l looks after every 32nd unit of the share
    Seq ps = s;   // the lane's own place in the list
    long long my_off[TT];           // pool offsets of this warp's blocks of the lane's unit; -1: nothing to fetch
    auto find_blocks = [&](int x) {
        while (x >= ps.begin + ps.total) next_seq<ROWS>(ps, c, group, a.tall);
        const int r = x - ps.begin, pair = r / ps.units, h = pair / ps.tiles, rt = pair - h * ps.tiles;
        const int pos = ((r - pair * ps.units) * kWarps + warp) * (kKvBlock * TT);
        const int seen = visible_keys(ps, min((rt + 1) * ROWS, ps.qlen * group) - 1, group);
#pragma unroll
        for (int k = 0; k < TT; ++k) {
            my_off[k] = -1;
            if (pos + k * kKvBlock < seen) {
                my_off[k] = kv_block_offset<D>(c, ps.b, h, pos + k * kKvBlock);
                if (my_off[k] < 0) atomicOr(status, kStatusBadCache);
            }
        }
    };
    const uint32_t ring = smem_u32(sm.ring[warp]), bars = smem_u32(sm.full[warp]);
    int issued = 0, istage = 0;     // units whose copy is under way or done
    bool alive = true;              // no wait has run out
    auto refill = [&]() {           // whole warp
        if (!alive || issued >= count) return;
        if ((issued & 31) == 0 && issued + lane < count) find_blocks(lo + issued + lane);
        if (lane == (issued & 31)) {
            const uint32_t bar = bars + 8 * istage, dst = ring + istage * (TT * L::kBlockBytes);
            int there = 0;
#pragma unroll
            for (int k = 0; k < TT; ++k) there |= (my_off[k] >= 0) << k;
            sm.ok[warp][istage] = there;
            mbar_expect_tx(bar, __popc(there) * L::kBlockBytes);
            if (there == 3 && my_off[TT - 1] == my_off[0] + L::kBlockBytes) {
                bulk_g2s(dst, c.pool + my_off[0], 2 * L::kBlockBytes, bar);
            } else {
#pragma unroll
                for (int k = 0; k < TT; ++k)
                    if (my_off[k] >= 0) bulk_g2s(dst + k * L::kBlockBytes, c.pool + my_off[k], L::kBlockBytes, bar);
            }
        }
        ++issued;
        if (++istage == kStages) istage = 0;
    };
    for (int i = 0; i < kStages; ++i) refill();

    // ---- consumer
    int stage = 0, waited = 0;   // waited: units whose copy has been waited for
    uint32_t parity = 0;
    for (bool more = true; more;) {
        if ((long long)s.len > (long long)c.table_stride * c.page_size && threadIdx.x == 0) atomicOr(status, kStatusBadCache);
        // q of the tile
        __syncthreads();
        if (warp < NT) {
            const int nt = warp;
            float big = 0.f;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const float2 u = __half22float2(as_h2(raw[j].x)), w = __half22float2(as_h2(raw[j].y));
                big = fmaxf(big, fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(w.x), fabsf(w.y))));
            }
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            int e = 0;   // q is used as q 2^e, its largest magnitude in [2^8, 2^9)
            if (big > 0.f && big <= 65504.f) e = 8 - ilogbf(big);
            const float up = exp2f((float)e);
            float sum[G] = {};
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const float k = up * ((j & 1) ? 0.0625f : 1.f);
                const float2 u = __half22float2(as_h2(raw[j].x)), w = __half22float2(as_h2(raw[j].y));
                sum[j / 2] += (u.x + u.y) + (w.x + w.y);
                sm.qfrag[nt][j][lane] = make_uint2(h2_bits(__floats2half2_rn(u.x * k, u.y * k)), h2_bits(__floats2half2_rn(w.x * k, w.y * k)));
            }
            float mine[2] = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < G; ++w) {
                sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 1);
                sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 2);
                if (w / 2 == (t & 1)) mine[w & 1] = sum[w] * up;
            }
            const __half2 high = __floats2half2_rn(mine[0], mine[1]);
            const float2 back = __half22float2(high);
            sm.qsum[nt][lane] = h2_bits(t < 2 ? high : __floats2half2_rn(mine[0] - back.x, mine[1] - back.y));
            if (t == 0) sm.factor[nt][g] = a.scale * 1.4426950408889634f * exp2f((float)(24 - e));
        }
        __syncthreads();

        Sums<D, NT> x;
        auto &o = x.o;
        auto &om = x.om;
        auto &mx = x.mx, &sum = x.sum;
        auto &unit = x.unit;
#pragma unroll
        for (int w = 0; w < G; ++w) unit[w] = __half2half2(__ushort_as_half((unsigned short)(30 << 10)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
            om[nt][0] = om[nt][1] = om[nt][2] = om[nt][3] = 0.f;
            mx[nt][0] = mx[nt][1] = -INFINITY;
            sum[nt][0] = sum[nt][1] = 0.f;
        }
        // by what the rows see and not by how wide the table is
        const bool fine = seg.kmin <= kUnit;
        int pos0 = ((seg.begin - seg.tile_begin) * kWarps + warp) * (kKvBlock * TT);
        for (int left = seg.end - seg.begin; left > 0; --left, pos0 += kUnit) {
            if (alive) {
                alive = __all_sync(0xffffffffu, wait_full(bars + 8 * stage, parity));
                if (alive) ++waited;
                else if (lane == 0) atomicOr(status, kStatusWaitTimeout);   // the rest counts as unseen
            }
            const int there = alive ? sm.ok[warp][stage] : 0;
            if (there) {
                const Unit u{sm.ring[warp][stage], there, pos0, seg.kmin, seg.kmax, s.len - s.qlen + 1, seg.rt * ROWS, group};
                if constexpr (SHORT) {
                    attend<D, NT, true>(x, sm, u);
                } else if (fine) {
                    Sums<D, NT> copy = x;
                    const Unit at = u;
                    attend_fine<D, NT>(copy, sm, at);
                    x = copy;
                } else {
                    attend<D, NT, false>(x, sm, u);
                }
            }
            __syncwarp();
            if (++stage == kStages) stage = 0, parity ^= 1;
            refill();
        }
        const Segment done = seg;
        const int first = s.first;
        more = seg.end < hi;
        if (more) {   // q of the next segment is on its way while this one is finished
            set_segment(seg.end);
            load_q();
        }

        // ---- join the four warps
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int d = 4; d < 32; d *= 2) sum[nt][e] += __shfl_xor_sync(0xffffffffu, sum[nt][e], d);
#pragma unroll
                for (int w = 0; w < G; ++w) {
                    const float m = __shfl_sync(0xffffffffu, om[nt][e], 4 * w + t), back = power(20 - exponent_of(unit[w]));
#pragma unroll
                    for (int i = 2 * w; i < 2 * w + 2; ++i) {
                        o[nt][i][e] = fmaf(o[nt][i][e], 16.f * back, m);
                        o[nt][i][2 + e] = fmaf(o[nt][i][2 + e], back, m);
                    }
                }
            }
        }
        if (warp) {
            float* dst = sm.merge[warp - 1];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float4 ms = make_float4(mx[nt][0], mx[nt][1], sum[nt][0], sum[nt][1]);
                reinterpret_cast<float4*>(dst)[(NT * MT + nt) * 32 + lane] = ms;
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    reinterpret_cast<float4*>(dst)[(nt * MT + i) * 32 + lane] = make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]);
            }
        }
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float4 ms[kWarps - 1];
                float n0 = mx[nt][0], n1 = mx[nt][1];
#pragma unroll
                for (int w = 0; w < kWarps - 1; ++w) {
                    ms[w] = reinterpret_cast<const float4*>(sm.merge[w])[(NT * MT + nt) * 32 + lane];
                    n0 = fmaxf(n0, ms[w].x), n1 = fmaxf(n1, ms[w].y);
                }
                const float z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
                float r0 = exp2_approx(mx[nt][0] - z0), r1 = exp2_approx(mx[nt][1] - z1);
                float t0 = sum[nt][0] * r0, t1 = sum[nt][1] * r1;
#pragma unroll
                for (int i = 0; i < MT; ++i) o[nt][i][0] *= r0, o[nt][i][1] *= r1, o[nt][i][2] *= r0, o[nt][i][3] *= r1;
#pragma unroll
                for (int w = 0; w < kWarps - 1; ++w) {
                    r0 = exp2_approx(ms[w].x - z0), r1 = exp2_approx(ms[w].y - z1);
                    t0 = fmaf(ms[w].z, r0, t0), t1 = fmaf(ms[w].w, r1, t1);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const float4 v = reinterpret_cast<const float4*>(sm.merge[w])[(nt * MT + i) * 32 + lane];
                        o[nt][i][0] = fmaf(v.x, r0, o[nt][i][0]), o[nt][i][1] = fmaf(v.y, r1, o[nt][i][1]);
                        o[nt][i][2] = fmaf(v.z, r0, o[nt][i][2]), o[nt][i][3] = fmaf(v.w, r1, o[nt][i][3]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = nt * 8 + 2 * t + e;
                    if (row >= done.rows) continue;
                    const float total_w = e ? t1 : t0;
                    if (done.whole) {
                        const float inv = total_w == 0.f ? 0.f : 1.f / total_w;   // no visible key: zeros
                        const int r = done.rt * ROWS + row;
                        uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + ((long long)(first + r / group) * a.q_heads + done.h * group + r % group) * D) + g;
#pragma unroll
                        for (int i = 0; i < MT; ++i) dst[8 * i] = h2_bits(__floats2half2_rn(o[nt][i][e] * inv, o[nt][i][2 + e] * inv));
                    } else {
                        float* slot = a.ws + (2 * (size_t)blockIdx.x + (done.begin == done.tile_begin)) * slot_floats<D, ROWS>();
                        float2* dst = reinterpret_cast<float2*>(slot + row * D) + g;
#pragma unroll
                        for (int i = 0; i < MT; ++i) dst[8 * i] = make_float2(o[nt][i][e], o[nt][i][2 + e]);
                        if (g == 0) {
                            slot[ROWS * D + row] = e ? n1 : n0;
                            slot[ROWS * D + ROWS + row] = total_w;
                        }
                    }
                }
            }
        }
    }
    // only after a wait that ran out: give the copies still under way one more bounded wait before the memory goes away
    for (; waited < issued; ++waited) wait_full(bars + 8 * (waited % kStages), (waited / kStages) & 1);
}

// Adds the parts of the row tiles that were cut between thread blocks, in order.  blockIdx.x: thread block of the split kernel, for the tile
// that starts in its share and goes on behind it, if there is one; and row if there are as many thread blocks (`spread`).  With many row
// tiles each has few parts: a warp takes a row.  With few, a thread block takes a row and its warps share out the parts (one key head, 444
// parts: 207 -> 28 us).  A grid over sequences, heads and row tiles, each of whose warps walked over all lengths, took 47 ms for 1024 single
// tokens with offsets and no bound, where the attention itself takes 0.4.
constexpr int kJoinWarps = 8;
template <int D, int NT>
__global__ void __launch_bounds__(32 * kJoinWarps) kv_attention_join_kernel(KvAttnArgs a, int ctas, int spread)
{
    constexpr int ROWS = 8 * NT, V = D / 32;
    __shared__ float part_sum[kJoinWarps][D], part_weight[kJoinWarps], part_max[kJoinWarps];
    const KvView& c = a.c;
    const int group = a.q_heads / c.kv_heads, lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    // the lengths are none of the preceding kernel's results, and what wrote them had ended before that kernel let this one start
    const int row0 = spread ? blockIdx.x % spread : warp, step = spread ? spread : kJoinWarps, c0 = spread ? blockIdx.x / spread : blockIdx.x;
    Seq s;
    List<ROWS> list(c, group, a.tall);
    const Shares shares(list.total, ctas);
    const int lo = shares.begin(c0), hi = shares.begin(c0 + 1);
    bool cut = false;
    int h = 0, rt = 0, c1 = 0;
    if (!list.too_long && lo < hi && hi < list.total) {
        list.find(s, c, group, a.tall, hi - 1);
        const int pair = (hi - 1 - s.begin) / s.units, p0 = s.begin + pair * s.units, p1 = p0 + s.units;
        cut = p0 >= lo && p1 > hi;
        h = pair / s.tiles, rt = pair - h * s.tiles;
        c1 = shares.of(p1 - 1);
    }
    if (!cut && blockIdx.x) return;
    grid_wait();   // one thread block at least: the kernel must not end before what it was launched behind
    if (!cut) return;
    const int rows = min(ROWS, s.qlen * group - rt * ROWS);
    // the first part is the end of its thread block's share, the later ones start theirs (slot 0)
    auto slot = [&](int i) { return a.ws + (2 * (size_t)i + (i == c0)) * slot_floats<D, ROWS>(); };
    for (int row = row0; row < rows; row += step) {
        // four parts at a time, all their loads under way together
        float m = -INFINITY, acc[V] = {}, w = 0.f;
        const int stride = spread ? kJoinWarps : 1;
        for (int i0 = c0 + (spread ? warp : 0); i0 <= c1; i0 += 4 * stride) {
            float pm[4], pw[4], v[4][V];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = min(i0 + j * stride, c1);
                const float* p = slot(i);
                const bool in = i0 + j * stride <= c1;
                pm[j] = in ? p[ROWS * D + row] : -INFINITY;
                pw[j] = in ? p[ROWS * D + ROWS + row] : 0.f;
                if constexpr (V == 4) *reinterpret_cast<float4*>(v[j]) = *reinterpret_cast<const float4*>(p + row * D + lane * V);
                else *reinterpret_cast<float2*>(v[j]) = *reinterpret_cast<const float2*>(p + row * D + lane * V);
            }
            const float n = fmaxf(m, fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]))), z = n == -INFINITY ? 0.f : n, r = exp2_approx(m - z);
            m = n;
            w *= r;
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] *= r;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i0 + j * stride <= c1) {
                    const float q = exp2_approx(pm[j] - z);
                    w = fmaf(pw[j], q, w);
#pragma unroll
                    for (int k = 0; k < V; ++k) acc[k] = fmaf(v[j][k], q, acc[k]);
                }
        }
        const int r = rt * ROWS + row;
        uint16_t* dst = a.out + ((long long)(s.first + r / group) * a.q_heads + h * group + r % group) * D;
        if (!spread) {
            const float inv = w == 0.f ? 0.f : 1.f / w;
            __half2 y[V / 2];
#pragma unroll
            for (int k = 0; k < V / 2; ++k) y[k] = __floats2half2_rn(acc[2 * k] * inv, acc[2 * k + 1] * inv);
            if constexpr (V == 4) *reinterpret_cast<uint2*>(dst + lane * V) = *reinterpret_cast<uint2*>(y);
            else *reinterpret_cast<uint32_t*>(dst + lane * V) = *reinterpret_cast<uint32_t*>(y);
            continue;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) part_sum[warp][lane * V + k] = acc[k];
        if (lane == 0) part_weight[warp] = w, part_max[warp] = m;
        __syncthreads();
        const int ch = threadIdx.x;
        if (ch < D) {
            float y = 0.f, all = 0.f, n = part_max[0];
#pragma unroll
            for (int i = 1; i < kJoinWarps; ++i) n = fmaxf(n, part_max[i]);
            const float z = n == -INFINITY ? 0.f : n;
#pragma unroll
            for (int i = 0; i < kJoinWarps; ++i) {
                const float q = exp2_approx(part_max[i] - z);
                y = fmaf(part_sum[i][ch], q, y), all = fmaf(part_weight[i], q, all);
            }
            dst[ch] = __half_as_ushort(__float2half_rn(all == 0.f ? 0.f : y / all));
        }
        __syncthreads();
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


// Thread blocks that fit on the device at once (shared memory and registers).
template <int D, int NT, bool SHORT>
cudaError_t prepare(int* ctas)
{
    static int cached[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!cached[dev]) {
        e = cudaFuncSetAttribute(kv_attention_split_kernel<D, NT, SHORT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem<D, NT>));
        int n = 0;
        if (e == cudaSuccess)
            e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv_attention_split_kernel<D, NT, SHORT>, 32 * kWarps, sizeof(Smem<D, NT>));
        if (e != cudaSuccess) return e;
        cached[dev] = (n < 1 ? 1 : n) * sm_count();
    }
    *ctas = cached[dev];
    return cudaSuccess;
}

template <int D, int NT>
cudaError_t launch(cudaStream_t s, const KvAttnArgs& a, int* status)
{
    constexpr int ROWS = 8 * NT;
    const int group = a.q_heads / a.c.kv_heads;
    const long long units = ((long long)a.c.table_stride * a.c.page_size - 1) / kUnit + 1;
    // A tile of up to four units is done whole: cutting it saves a unit's time or two (1.5 us each), the join costs 3.5 us.
    const bool whole = units <= 4;
    int ctas = 0;
    cudaError_t e = units == 1 ? prepare<D, NT, true>(&ctas) : prepare<D, NT, false>(&ctas);
    if (e != cudaSuccess) return e;
    const long long fit = (long long)(a.ws_floats / (2 * slot_floats<D, ROWS>()));
    if (fit < 1) return cudaErrorInvalidValue;
    if (fit < ctas) ctas = (int)fit;
    // never more thread blocks than units there can be: every table entry used, every packed row in a tile of its own at worst
    const long long tiles = ((long long)a.max_q * group + ROWS - 1) / ROWS;
    const long long most = (long long)a.c.B * a.c.kv_heads * (tiles > 0 ? tiles : 1) * units;
    if (whole ? most / units < ctas : most < ctas) ctas = (int)(whole ? most / units : most);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(32 * kWarps);
    cfg.dynamicSmemBytes = sizeof(Smem<D, NT>);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = units == 1 ? cudaLaunchKernelEx(&cfg, kv_attention_split_kernel<D, NT, true>, a, (int)whole, status)
                   : cudaLaunchKernelEx(&cfg, kv_attention_split_kernel<D, NT, false>, a, (int)whole, status);
    count_launch();
    if (e != cudaSuccess || whole) return e;
    const long long rows = (long long)a.max_q * group, pairs = a.c.kv_heads * (tiles > 0 ? tiles : 1);
    const long long spread = pairs * a.c.B * 4 > ctas ? 0 : rows < 1 ? 1 : rows < ROWS ? rows : ROWS;   // five parts and more
    cfg.gridDim = dim3((unsigned)(ctas * (spread ? spread : 1)));
    cfg.blockDim = dim3(32 * kJoinWarps);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, kv_attention_join_kernel<D, NT>, a, ctas, (int)spread);
    count_launch();
    return e;
}

template <int D>
cudaError_t launch_d(cudaStream_t s, const KvAttnArgs& a, int* status)
{
    switch (pick_nt((long long)a.max_q * (a.q_heads / a.c.kv_heads))) {
        case 1: return launch<D, 1>(s, a, status);
        default: return launch<D, 2>(s, a, status);
    }
}

}  // namespace

// Rows a key head from which a sequence goes to the tcgen05 kernel, whose row tiles have 128 rows; and how many of its thread
// blocks there have to be, each of which walks over a whole context by itself (the split kernel shares one out among all SMs).
constexpr int kTallRows = 64, kTallItems = 24;

cudaError_t kv_attention_launch(cudaStream_t s, int D, const KvAttnArgs& args, int* status)
{
    KvAttnArgs a = args;
    const int group = a.q_heads / a.c.kv_heads;
    if (!a.c.cu) a.max_q = a.c.per_seq;
    a.tall = 0x7fffffff;
    if ((long long)a.max_q * group >= kTallRows && (((long long)a.c.n_tokens * group + 255) / 256) * a.c.kv_heads >= kTallItems) {
        a.tall = kTallRows;
        const cudaError_t e = kv_prefill_launch(s, D, a, a.tall, status);
        if (e != cudaSuccess) return e;
        if (!a.c.cu) return cudaSuccess;   // all sequences are alike
    }
    return D == 128 ? launch_d<128>(s, a, status) : launch_d<64>(s, a, status);
}

// Workspace for the largest grid: two slots for each thread block that fits.
size_t kv_attention_ws_floats(int D, int B, int q_heads, int kv_heads, int max_q)
{
    (void)B;
    const int rows = 8 * pick_nt((long long)max_q * (q_heads / kv_heads));
    return (size_t)2 * blocks_per_sm(rows / 8) * sm_count() * rows * (D + 2);
}

}  // namespace spb
