// Attention over the paged 4-bit cache for many query rows a key head (prompts and chunks of prompts), on tcgen05.
//
// A thread block takes up to 256 rows (two tiles of 128) of one sequence and key head and walks over the keys in tiles of 64:
//
//   warp 0        copies the 4 blocks of a key tile (4-bit keys and values) into a four-stage ring
//   warp 1        issues tcgen05.mma, one elected thread
//   warps 4-7, 8-11   softmax of row tile 0 and 1, thread = row: scores from tensor memory, running maximum and sum in fp32 and
//                 base 2, weights back to tensor memory as fp16 where the next product takes its left operand from
//   warps 12-19   expand one block each, four warps the even key tiles and four the odd: keys [key][channel] and values transposed,
//                 [channel][key], as 128-byte-swizzled tiles (m + s c with one rounding, the values that kv_read returns)
//
// S = Q K^T (both operands in shared memory) has two buffers per row tile in tensor memory, P lies over S, and O += P V (V^T in shared
// memory) is followed by the scores of the key tile after the next in the buffer it has read: the softmax warps always
// find their next scores done.  (Key tiles of 128 leave room for one buffer; softmax and products then wait for each
// other, 6700 cycles per 256 x 128 scores whatever the softmax took.)  The accumulators are rescaled, by the softmax
// warps, only when a row's maximum has grown by more than 2^8; weights are kept 2^7 too large so that fp16 holds 2^-31 .. 1.
// Weights, keys and values enter the products as fp16, each rounded once: chunks over 2043 tokens come out 2.1e-4 from the exact result, fp32
// sums 2.0e-4; prompts of a few tens of tokens 2.4 to 2.6e-4 against 2.1e-4.  There is no second product here as in kv_attention.cu: it would double
// half of the matrix instructions, which are the bound.
//
// Bound: 4 D flops a row and key on the tensor core, 16 exponentials a cycle (as many cycles at D = 128), and the
// instructions of softmax and expansion, which the 256 rows share.  What it meets is the rate of issuing narrow products: 64-column
// scores cost as much as 128-column ones, 80 cycles, so 256 rows x 128 keys take 4100 cycles of them at least and 6000 in fact.  Two chunks of
// up to 1021 tokens over 2043, 40 heads of 128: 117 us, 430 TFLOP/s (30 us at the library's dense rate).
#include "kv_int4.cuh"
#include "sm100.cuh"

namespace spb {
namespace {
using namespace sm100;

constexpr int kRows = 256, kKeys = 64, kBlocks = kKeys / kKvBlock, kRaw = 4, kInfo = 16;
constexpr int kEdge = 6;   // 256 rows see at most 255 keys apart: five tiles
constexpr int kThreads = 32 * 20, kExpand = 12;   // first expanding warp
constexpr float kShift = 7.f, kSlack = 8.f;

template <int D>
struct Smem {
    uint8_t q[2][D / 64][128 * 128];          // [row tile][64 channels][row][128 bytes], swizzled
    uint8_t k[2][D / 64][kKeys * 128];        // [key tile & 1][64 channels][key][128 bytes]
    uint8_t v[2][D * 128];                    // [key tile & 1][channel][64 keys]
    uint8_t raw[kRaw][kBlocks][KvLayout<D>::kBlockBytes];
    uint64_t raw_full[kRaw], raw_empty[kRaw], k_ready[2], k_free[2], v_ready[2], v_free[2], s_full[2][2], p_ready[2][2], pv_done[2], o_full[2];
    uint32_t holder;
    int abort;
    int blocks[kInfo];                        // blocks of the key tile that are there
    alignas(8) uint16_t nan[kEdge][D / kKvGroup][kBlocks];   // tokens whose values are NaN, taken out of the products (tiles at the causal edge)
};

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t swizzled(uint32_t base, int row, int chunk) { return base + row * 128 + ((chunk ^ (row & 7)) << 4); }

// Two fp32 values an instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// What a stretch of 16 scores needs: nothing (all rows of the warp see all of it), a look at each, or nobody sees it.
enum class Care { kNone, kEach, kUnseen };
// Keys of the tile that the rows of a warp see, and blocks that are there.
struct Sight {
    int mine, least, most;   // of this row, the least and most of the warp's
    uint32_t there;
    __device__ __forceinline__ Care of(int q) const   // stretch 16 q ..
    {
        if (!(there >> q & 1) || 16 * q >= most) return Care::kUnseen;
        return 16 * q + 16 <= least ? Care::kNone : Care::kEach;
    }
};
// The largest of 64 scores, in base 2.
__device__ __forceinline__ float row_top(const uint32_t (&v)[kKeys], float f, const Sight& s)
{
    float top = -INFINITY;
    if (s.there == (1u << kBlocks) - 1 && s.least >= kKeys && f >= 0.f) {
        float m[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = __uint_as_float(v[16 * k + 15]);
#pragma unroll
        for (int e = 0; e < 14; e += 2)
#pragma unroll
            for (int k = 0; k < 4; ++k) m[k] = max3(m[k], __uint_as_float(v[16 * k + e]), __uint_as_float(v[16 * k + e + 1]));
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = fmaxf(m[k], __uint_as_float(v[16 * k + 14]));
        return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * f;
    }
#pragma unroll
    for (int q = 0; q < kBlocks; ++q)
        if (s.of(q) != Care::kUnseen)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, 16 * q + e < s.mine ? __uint_as_float(v[16 * q + e]) * f : -INFINITY);
    return top;
}
// The scores' weights 2^(f s - base), to tensor memory as fp16; their sum.
__device__ __forceinline__ float row_weights(uint32_t addr, uint32_t (&v)[kKeys], float f, float base, const Sight& s)
{
    const uint64_t ff = pack2(f, f), bb = pack2(-base, -base);
    uint64_t sum = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint32_t p[16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int q = 2 * half + h;
            const Care care = s.of(q);
            if (care == Care::kUnseen) {
#pragma unroll
                for (int e = 0; e < 8; ++e) p[8 * h + e] = 0;
            } else {
                float x[16];
#pragma unroll
                for (int e = 0; e < 16; e += 2) unpack2(fma2(pack2(__uint_as_float(v[16 * q + e]), __uint_as_float(v[16 * q + e + 1])), ff, bb), x[e], x[e + 1]);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = exp2_approx(x[e]);
                if (care == Care::kEach)
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = 16 * q + e < s.mine ? x[e] : 0.f;
                uint64_t a = pack2(x[0], x[1]), b = pack2(x[2], x[3]);
#pragma unroll
                for (int e = 4; e < 16; e += 4) a = add2(a, pack2(x[e], x[e + 1])), b = add2(b, pack2(x[e + 2], x[e + 3]));
                sum = add2(sum, add2(a, b));
#pragma unroll
                for (int e = 0; e < 8; ++e) p[8 * h + e] = h2_bits(__floats2half2_rn(x[2 * e], x[2 * e + 1]));
            }
        }
        tc_st16(addr + 16 * half, p);
    }
    float x, y;
    unpack2(sum, x, y);
    return x + y;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) kv_prefill_kernel(KvAttnArgs a, int tall, int* status)
{
    using L = KvLayout<D>;
    constexpr int G = L::kGroups, KSteps = D / 16;
    constexpr uint32_t kS = 0, kO = 256;   // tensor memory columns: scores of row tile t and key tile i at 128 t + 64 (i & 1), outputs at 256 + D t
    extern __shared__ uint8_t smem_raw[];
    Smem<D>& sm = *reinterpret_cast<Smem<D>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const KvView& c = a.c;
    const int group = a.q_heads / c.kv_heads;
    volatile int* abort_flag = &sm.abort;

    grid_wait();
    // ---- the item: key head blockIdx.x % heads, row tile number blockIdx.x / heads of the sequences with `tall` rows and more;
    // in a sequence the last rows, which see most, come first
    const int h = blockIdx.x % c.kv_heads, want = blockIdx.x / c.kv_heads;
    int b = -1, rt = 0, first = 0, qlen = 0;
    for (int b0 = 0, before = 0; b0 < c.B && b < 0; b0 += 32) {
        int f = 0, n = 0;
        if (b0 + lane < c.B) kv_rows(c, b0 + lane, f, n);
        const int t = n * group >= tall ? (n * group + kRows - 1) / kRows : 0;
        int incl = t;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + incl > want);
        if (past) {
            const int l = __ffs(past) - 1;
            b = b0 + l;
            rt = before + __shfl_sync(0xffffffffu, incl, l) - 1 - want;
            first = __shfl_sync(0xffffffffu, f, l);
            qlen = __shfl_sync(0xffffffffu, n, l);
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (b < 0) return;
    const int rows_all = qlen * group;
    const int len = max(c.lens[b], 0), row0 = rt * kRows, rows = min(kRows, rows_all - row0);
    auto visible = [&](int row) { return max(len - qlen + row / group + 1, 0); };   // keys that row sees
    const int held = (int)min((long long)len, (long long)c.table_stride * c.page_size);
    if (held < len && threadIdx.x == 0) atomicOr(status, kStatusBadCache);
    const int ntile = rows > 128 ? 2 : 1;
    const int kmin = visible(row0), kmax = min(visible(row0 + rows - 1), held);
    const int n1 = (kmax + kKeys - 1) / kKeys;                                             // key tiles of the last row tile
    const int edge0 = kmin / kKeys;                                                        // first tile that some row does not see all of
    const int n0 = ntile == 1 ? n1 : (min(visible(row0 + 127), held) + kKeys - 1) / kKeys;   // of row tile 0

    if (threadIdx.x == 0) {
        for (int i = 0; i < kRaw; ++i) mbar_init(smem_u32(&sm.raw_full[i]), 1), mbar_init(smem_u32(&sm.raw_empty[i]), 4);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sm.k_ready[i]), 4), mbar_init(smem_u32(&sm.k_free[i]), 1);
            mbar_init(smem_u32(&sm.v_ready[i]), 4), mbar_init(smem_u32(&sm.v_free[i]), 1);
            mbar_init(smem_u32(&sm.s_full[i][0]), 1), mbar_init(smem_u32(&sm.s_full[i][1]), 1);
            mbar_init(smem_u32(&sm.p_ready[i][0]), 4), mbar_init(smem_u32(&sm.p_ready[i][1]), 4), mbar_init(smem_u32(&sm.pv_done[i]), 1), mbar_init(smem_u32(&sm.o_full[i]), 1);
        }
        sm.abort = 0;
        mbar_init_fence();
    }
    if (warp == 1) tc_alloc(smem_u32(&sm.holder), 512);   // all columns: the allocation starts at 0
    // q of both tiles, rows past the end as zeros
    if (warp >= 4 && warp < 12) {   // one thread a row
        const int tile = (warp - 4) / 4, r = (warp & 3) * 32 + lane, row = tile * 128 + r;
        const bool have = row < rows;
        const int abs_row = row0 + (have ? row : 0);
        const uint16_t* src = a.q + (long long)(first + abs_row / group) * a.q_tok + (h * group + abs_row % group) * a.q_head;
        if (tile < ntile)
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                uint2 x = make_uint2(0, 0), y = x;
                if (have) x = reinterpret_cast<const uint2*>(src)[2 * i], y = reinterpret_cast<const uint2*>(src)[2 * i + 1];
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(swizzled(smem_u32(sm.q[tile][i / 8]), r, i % 8)), "r"(x.x), "r"(x.y), "r"(y.x), "r"(y.y) : "memory");
            }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Only now that this block has its tensor memory: a kernel that follows may take some before it waits for this one, and would have it
    // while a block here waited for all of it.
    grid_release();

    bool ok = true;
    if (warp == 0) {
        // ---- copies: lane = block of the tile
        long long off = -1;
        auto find = [&](int i) -> long long {
            const int pos = i * kKeys + lane * kKvBlock;
            if (lane >= kBlocks || pos >= kmax) return -1;
            const long long o = kv_block_offset<D>(c, b, h, pos);
            if (o < 0) atomicOr(status, kStatusBadCache);
            return o;
        };
        if (n1 > 0) off = find(0);
        for (int i = 0; i < n1 && ok; ++i) {
            const int s = i % kRaw;
            const long long at = off;
            if (i + 1 < n1) off = find(i + 1);
            if (i >= kRaw) ok = mbar_wait(smem_u32(&sm.raw_empty[s]), (i / kRaw - 1) & 1, abort_flag);
            if (!ok) break;
            const uint32_t there = __ballot_sync(0xffffffffu, at >= 0), bar = smem_u32(&sm.raw_full[s]);
            if (lane == 0) {
                sm.blocks[i % kInfo] = there;
                mbar_expect_tx(bar, __popc(there) * L::kBlockBytes);
            }
            __syncwarp();
            if (at >= 0) bulk_g2s(smem_u32(sm.raw[s][lane]), c.pool + at, L::kBlockBytes, bar);
        }
    } else if (warp == 1) {
        // ---- matrix instructions
        const uint32_t q0 = kmajor_desc_low(smem_u32(sm.q)), k0 = kmajor_desc_low(smem_u32(sm.k)), v0 = kmajor_desc_low(smem_u32(sm.v));
        auto scores = [&](int i, int t) {   // of key tile i, row tile t
            if (elect_one()) {
                const uint32_t kd = k0 + (i & 1) * (uint32_t)(sizeof(sm.k[0]) >> 4), qd = q0 + t * (uint32_t)(sizeof(sm.q[0]) >> 4), d = kS + t * 128 + (i & 1) * 64;
#pragma unroll
                for (int j = 0; j < KSteps; ++j)
                    tc_mma_ss(d, qd + j / 4 * 1024 + 2 * (j % 4), kd + j / 4 * (kKeys * 8) + 2 * (j % 4), kKMajorDescHigh, f16_idesc(128, kKeys), j > 0);
                tc_commit(smem_u32(&sm.s_full[t][i & 1]));
                if (t == ntile - 1) tc_commit(smem_u32(&sm.k_free[i & 1]));   // the last row tile sees most: it is never the first to end
            }
            __syncwarp();
        };
        for (int i = 0; i < 2 && i < n1 && ok; ++i) {
            ok = mbar_wait(smem_u32(&sm.k_ready[i]), 0, abort_flag);
            if (!ok) break;
            tc_fence_after();
            if (i < n0) scores(i, 0);
            if (ntile == 2) scores(i, 1);
        }
        for (int i = 0; i < n1 && ok; ++i) {
            bool have_v = false, have_k = false;
            for (int t = 0; t < ntile && ok; ++t) {
                const int n = t == 0 ? n0 : n1;
                if (i >= n) continue;
                ok = mbar_wait(smem_u32(&sm.p_ready[t][i & 1]), i / 2 & 1, abort_flag);   // per buffer: the softmax may be two tiles ahead
                if (ok && !have_v) ok = have_v = mbar_wait(smem_u32(&sm.v_ready[i & 1]), i / 2 & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t vd = v0 + (i & 1) * (uint32_t)(sizeof(sm.v[0]) >> 4), pa = kS + t * 128 + (i & 1) * 64, d = kO + t * D;
#pragma unroll
                    for (int j = 0; j < kKeys / 16; ++j) tc_mma_ts(d, pa + 8 * j, vd + 2 * j, kKMajorDescHigh, f16_idesc(128, D), i > 0 || j > 0);
                    tc_commit(smem_u32(&sm.pv_done[t]));
                    if (i == n - 1) tc_commit(smem_u32(&sm.o_full[t]));
                    if (t == ntile - 1) tc_commit(smem_u32(&sm.v_free[i & 1]));
                }
                __syncwarp();
                if (i + 2 < n) {
                    if (!have_k) ok = have_k = mbar_wait(smem_u32(&sm.k_ready[i & 1]), (i / 2 + 1) & 1, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    scores(i + 2, t);
                }
            }
        }
    } else if (warp >= kExpand) {
        // ---- expansion: warp = block of the tile, lane 4 g + t as in the layout
        const int blk = (warp - kExpand) % 4, odd = (warp - kExpand) / 4, g = lane / 4, t = lane % 4;
        uint32_t mask_low, mask_high, bits_low, bits_high;   // kept in registers for and_or
        asm volatile("mov.b32 %0, 0x000f000f;\n\tmov.b32 %1, 0x00f000f0;\n\tmov.b32 %2, 0x64006400;\n\tmov.b32 %3, 0x54005400;"
                     : "=r"(mask_low), "=r"(mask_high), "=r"(bits_low), "=r"(bits_high));
        auto low = [&](uint32_t w, __half2 s, __half2 m) { return h2_bits(__hfma2(__hsub2(as_h2(and_or(w, mask_low, bits_low)), as_h2(bits_low)), s, m)); };
        auto high = [&](uint32_t w, __half2 s, __half2 m) { return h2_bits(__hfma2(__hsub2(as_h2(and_or(w, mask_high, bits_high)), as_h2(bits_high)), s, m)); };
        // where the lane's values go, up to constants: keys by 16-byte chunk (2 u of each half of a 64-channel row), values by channel & 1
        // and half of the block
        uint32_t k_at[4], v_at[2][2];
#pragma unroll
        for (int u = 0; u < 4; ++u) k_at[u] = swizzled(smem_u32(sm.k[odd]), blk * kKvBlock + g, 2 * u + (t >> 1)) + (t & 1) * 8;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int j = 0; j < 2; ++j) v_at[r][j] = swizzled(smem_u32(sm.v[odd]), 2 * g + r, blk * 2 + j) + 4 * t;
        // a group of four warps has every other tile, and with it every other stage and one of each two buffers: it waits for every phase
        for (int i = odd; i < n1 && ok; i += 2) {
            const int s = i % kRaw, pos = i * kKeys + blk * kKvBlock;
            ok = mbar_wait(smem_u32(&sm.raw_full[s]), (i / kRaw) & 1, abort_flag);
            if (!ok) break;
            const bool there = sm.blocks[i % kInfo] >> blk & 1;
            const uint8_t* src = sm.raw[s][blk];
            if (i >= 2) ok = mbar_wait(smem_u32(&sm.k_free[odd]), (i / 2 - 1) & 1, abort_flag);
            if (!ok) break;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int w = 0; w < G; ++w) {
                    const uint32_t x = reinterpret_cast<const uint32_t*>(src + L::kKCodes)[(g + 8 * e) * (D / 8) + t * G + w], y = x >> 8;
                    const __half2 p = as_h2(there ? reinterpret_cast<const uint32_t*>(src + L::kKParams)[(g + 8 * e) * G + w] : 0u);
                    const __half2 sc = __low2half2(p), mn = __high2half2(p);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t v0 = u ? high(x, sc, mn) : low(x, sc, mn), v1 = u ? high(y, sc, mn) : low(y, sc, mn);
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(k_at[2 * (w & 1) + u] + w / 2 * (kKeys * 128) + e * 1024), "r"(v0), "r"(v1) : "memory");
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.k_ready[odd]));
            if (i >= 2) ok = mbar_wait(smem_u32(&sm.v_free[odd]), (i / 2 - 1) & 1, abort_flag);
            if (!ok) break;
            const bool edge = i >= edge0;
#pragma unroll
            for (int w = 0; w < G; ++w) {
                uint32_t bad = 0;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t x = reinterpret_cast<const uint32_t*>(src + L::kVCodes + j * 4 * D)[lane * G + w], y = x >> 8;
                    uint2 p = make_uint2(0, 0);
                    if (there) p = *reinterpret_cast<const uint2*>(src + L::kVParams + ((t + 4 * j) * G + w) * 8);
                    if (edge) {
                        // Tokens that no row sees count as zero, whatever the page holds there; NaN that only some rows see is taken
                        // out here and put back by the softmax warps
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int tok = 8 * j + 2 * t + e;
                            const bool unseen = pos + tok >= kmax, nan = (p.x >> 16 * e & 0x7c00u) == 0x7c00u || (p.y >> 16 * e & 0x7c00u) == 0x7c00u;
                            if (nan && !unseen) bad |= 1u << tok;
                            if (nan || unseen) {
                                const uint32_t keep = e ? 0x0000ffffu : 0xffff0000u;
                                p.x &= keep, p.y &= keep;
                            }
                        }
                    }
                    const __half2 sc = as_h2(p.x), mn = as_h2(p.y);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t z = u ? y : x, rows = (32 * w + 16 * u) * 128;
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(v_at[0][j] + rows), "r"(low(z, sc, mn)) : "memory");
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(v_at[1][j] + rows), "r"(high(z, sc, mn)) : "memory");
                    }
                }
                if (edge) {
                    bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
                    bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
                    if (lane == 0) sm.nan[i - edge0][w][blk] = (uint16_t)bad;
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&sm.v_ready[odd]));
                mbar_arrive(smem_u32(&sm.raw_empty[s]));
            }
        }
    } else if (warp >= 4) {
        // ---- softmax, thread = row
        const int tile = (warp - 4) / 4, row = tile * 128 + (warp & 3) * 32 + lane, abs_row = row0 + row;
        const bool have = row < rows;
        const int mine = have ? min(visible(abs_row), held) : 0, n = tile == 0 ? n0 : ntile == 2 ? n1 : 0;
        const int least = __reduce_min_sync(0xffffffffu, mine), most = __reduce_max_sync(0xffffffffu, mine);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21, o_addr = kO + tile * D + lanes;
        const float f = a.scale * 1.4426950408889634f;
        float mx = -INFINITY, sum = 0.f;
        for (int i = 0; i < n && ok; ++i) {
            ok = mbar_wait(smem_u32(&sm.s_full[tile][i & 1]), i / 2 & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_addr = kS + tile * 128 + (i & 1) * 64 + lanes;
            const Sight sight{mine - i * kKeys, least - i * kKeys, most - i * kKeys, (uint32_t)sm.blocks[i % kInfo]};
            uint32_t v[kKeys];
            tc_ld32(s_addr, v);
            tc_ld32(s_addr + 32, v + 32);
            tc_wait_ld();
            const float top = row_top(v, f, sight);
            if (__any_sync(0xffffffffu, top > mx + kSlack)) {
                const float now = fmaxf(top, mx), c = mx == -INFINITY ? 0.f : exp2_approx(mx - now);
                mx = now;
                sum *= c;
                if (i > 0) {
                    // The accumulators rest when P V of the tile before has ended.  S of this one was issued behind P V (i - 2): at most
                    // that one is still to come, and the phase's parity tells.
                    ok = mbar_wait(smem_u32(&sm.pv_done[tile]), (i - 1) & 1, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int q = 0; q < D; q += 16) {
                        uint32_t x[16];
                        tc_ld16(o_addr + q, x);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * c);
                        tc_st16(o_addr + q, x);
                    }
                }
            }
            sum += row_weights(s_addr, v, f, (mx == -INFINITY ? 0.f : mx) - kShift, sight);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.p_ready[tile][i & 1]));
        }
        if (tile < ntile && ok) {
            if (n > 0) ok = mbar_wait(smem_u32(&sm.o_full[tile]), 0, abort_flag);
            if (ok) {
                tc_fence_after();
                uint32_t poison = 0;   // groups of channels that are NaN for this row
                for (int i = edge0; i < n; ++i)
                    for (int w = 0; w < G; ++w) {
                        const uint64_t bits = *reinterpret_cast<const uint64_t*>(sm.nan[i - edge0][w]);
                        const int seen = mine - i * kKeys;
                        const uint64_t mask = seen >= 64 ? ~0ull : seen <= 0 ? 0ull : (1ull << seen) - 1;
                        if (bits & mask) poison |= 1u << w;
                    }
                const float inv = sum == 0.f ? 0.f : 1.f / sum;   // no visible key: zeros
                uint16_t* dst = a.out + ((long long)(first + abs_row / group) * a.q_heads + h * group + abs_row % group) * D;
#pragma unroll 1
                for (int q = 0; q < D; q += 16) {
                    uint32_t x[16];
                    if (n > 0) {
                        tc_ld16(o_addr + q, x);
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = 0;
                    }
                    uint32_t y[8];
                    const bool bad = poison >> (q / kKvGroup) & 1;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        y[e] = bad ? 0x7fff7fffu : h2_bits(__floats2half2_rn(__uint_as_float(x[2 * e]) * inv, __uint_as_float(x[2 * e + 1]) * inv));
                    if (have) {
                        reinterpret_cast<uint4*>(dst + q)[0] = make_uint4(y[0], y[1], y[2], y[3]);
                        reinterpret_cast<uint4*>(dst + q)[1] = make_uint4(y[4], y[5], y[6], y[7]);
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*abort_flag) {
        if (threadIdx.x == 0) {
            atomicOr(status, kStatusWaitTimeout);
            for (int i = 0; i < kRaw; ++i)   // copies still under way get a bounded chance to land
                for (uint32_t spin = 0; spin < 4096; ++spin)
                    if (mbar_try(smem_u32(&sm.raw_full[i]), 0) || mbar_try(smem_u32(&sm.raw_full[i]), 1)) break;
        }
        __syncthreads();
    }
    if (warp == 1) tc_dealloc(sm.holder, 512);
}

template <int D>
cudaError_t launch(cudaStream_t s, const KvAttnArgs& a, int tall, int* status)
{
    static bool prepared[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    constexpr size_t smem = sizeof(Smem<D>) + 1024;
    if (!prepared[dev]) {
        e = cudaFuncSetAttribute(kv_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        prepared[dev] = true;
    }
    // as many row tiles as there can be: whole ones, and a last one in every sequence that is tall enough
    const long long rows = (long long)a.c.n_tokens * (a.q_heads / a.c.kv_heads), seqs = rows / tall < a.c.B ? rows / tall : a.c.B;
    const long long items = (rows / kRows + seqs) * a.c.kv_heads;
    if (items <= 0) return cudaSuccess;
    if (items > 0x7fffffff) return cudaErrorInvalidValue;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)items);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kv_prefill_kernel<D>, a, tall, status);
    count_launch();
    return e;
}

}  // namespace

cudaError_t kv_prefill_launch(cudaStream_t s, int D, const KvAttnArgs& a, int tall, int* status)
{
    return D == 128 ? launch<128>(s, a, tall, status) : launch<64>(s, a, tall, status);
}

}  // namespace spb
