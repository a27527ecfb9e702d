// Linear layer over 4-bit weights (layout: int4.cuh) for more than 16 rows of x, on tcgen05:
//
//   out[n][m] = residual + act(bias + sum_k w[m][k] x[n][k]),   w = s (c - z) rounded to fp16 (the value int4_decode returns)
//
// The rounding of w costs accuracy: 2.8e-4 from the exact result where fp32 sums of unrounded weights are 2.1e-4 (int4_stream.cu).
// Rows of W are the 128-row side of the matrix instruction, rows of x its 32..256-column side.  Codes become fp16 on the way
// into tensor memory, where the instruction takes its left operand from; x comes as 128-byte-swizzled tiles by tensor copies.
//
// Bound: 9216 x 36864, 509 rows: 262 us in a burst at 1965 MHz, 1320 TFLOP/s, 79 % of the library's dense rate in a burst; 301 to 315 us kept up
// under the power cap at 1430 MHz, 1100 to 1150 TFLOP/s, 79 to 82 % of the library's kept up.  Tensor pipe 69 % busy; every 128 rows of W read
// all of x from L2, 2.8 GB or 10 TB/s, which is near what L2 gives.  With 32 to 64 rows the product is bound by the 8 instructions of a
// unit, which cost the same 80 cycles for 32 columns as for 128 (16384 x 16384, 40 rows: 52 us, 22 at copy rate).  Scaling a group's sums in
// fp32 instead of the weights, so that these need no rounding, was built and measured: 405 us and 64 us for these two with groups of
// 128, and two and a half times as long with groups of 32, whose accumulators change hands four times a unit.
//
//   warps 0, 2    copies: per stage of kKT 64-k tiles one bulk copy of codes and parameters (warp 0), one tensor copy of x
//                 (warp 2).  Issuing a copy holds a warp up for a few hundred cycles, so there are few and two warps share them
//                 (one warp issuing six copies a stage capped the kernel at 0.26 us a k-tile, three times what memory needs)
//   warp 1        issues tcgen05.mma, one elected thread
//   warps 4-7     epilogue: accumulators -> bias, activation, residual, one rounding -> out; or fp32 partial sums -> workspace
//   warps 8..     kGroups groups of four, thread = row of W: per 64-k tile 8 words of codes -> 32 registers of fp16 pairs (per pair
//                 one AND/OR, one exact subtraction of offset and zero point, one multiplication by the scale) -> tcgen05.st
#include "int4_work.cuh"
#include <cuda.h>
#include <mutex>

namespace spb {
namespace {

template <int NPAD> struct Cfg {
    static constexpr int kGroups = 4;                                    // dequantising groups of four warps
    static constexpr int kThreads = 32 * (8 + 4 * kGroups);
    static constexpr int kABlocks = kGroups;                             // left-operand blocks in tensor memory, one unit (64 columns) per group
    static constexpr int kKT = NPAD <= 64 ? 4 : 2;                       // k-tiles per stage
    static constexpr int kUS = kKT / kUnit;                              // units per stage: groups share out kTurn stages
    static constexpr int kTurn = kGroups / kUS;
    static constexpr int kAcc = NPAD <= 32 ? 4 : NPAD <= 64 ? 2 : 1;     // accumulators the k-steps take in turn (short ones are latency)
    static constexpr int kAhead = 2;                                     // stages between a prefetch into L2 and the copy from there (277 -> 264 us for
                                                                         // 9216 x 36864 with 509 rows, 46 -> 43 for 28672 x 7168 with 32; 4 and 8: 1 to 3 % slower)
    static constexpr uint32_t kX = NPAD * 128;                           // bytes of x per k-tile
    static constexpr uint32_t kStage = kKT * kX + kKT / kUnit * (2 * kInt4CodeBytes + 4 * 512);   // x, units (at most four groups)
    static constexpr int kStages = (int)((222u * 1024) / kStage) < 8 ? (int)((222u * 1024) / kStage) : 8;
    static constexpr uint32_t kSmem = 1024 + 1024 + kStages * kStage;    // header, alignment
    static constexpr uint32_t kTmemCols = 512, kTmemA = 512 - 64 * kABlocks;   // accumulators from 0, operand blocks at the end
    static_assert(kAcc * NPAD <= (int)kTmemA, "accumulators and operand blocks overlap");
};

template <int NPAD, int kGroup>
__global__ void __launch_bounds__(Cfg<NPAD>::kThreads, 1) int4_wide_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap xmap)
{
    using C = Cfg<NPAD>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
    uint32_t* holder = reinterpret_cast<uint32_t*>(smem + 512);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 516);
    const uint32_t full = smem_u32(bars), empty = smem_u32(bars + 8), ready = smem_u32(bars + 16), afree = smem_u32(bars + 24),
                   acc_full = smem_u32(bars + 32), acc_empty = smem_u32(bars + 33);
    const uint32_t stage0 = smem_u32(smem + 1024);
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) mbar_init(full + 8 * i, 2), mbar_init(empty + 8 * i, 1);
        for (int i = 0; i < C::kABlocks; ++i) mbar_init(ready + 8 * i, 4), mbar_init(afree + 8 * i, 1);
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 4);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 1) tc_alloc(smem_u32(holder), C::kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0, tmem_a = C::kTmemA;   // all columns: the allocation starts at 0
    if (warp == 0) {   // the first codes on their way to L2 while what ran before ends
        Walk first(p);
        Run f;
        if (first.next<NPAD>(p, f) && elect_one())
            bulk_prefetch(p.a.units + ((long long)f.mb * p.ku + f.u0) * int4_unit_bytes(kGroup), min(C::kAhead * C::kUS, f.nkt / kUnit) * int4_unit_bytes(kGroup));
    }
    grid_wait();      // x, residual, out and the workspace belong to what ran before
    grid_release();   // the join may be set up while this kernel runs; it waits for its end

    Walk walk(p);
    Run r;
    if (warp == 0 || warp == 2) {
        // ---- copies
        constexpr int unit_bytes = int4_unit_bytes(kGroup);
        const int rows = p.items / p.ncol;
        uint32_t s = 0, round = 0;
        bool ok = true;
        while (ok && walk.next<NPAD>(p, r)) {
            for (int k = 0; k < r.nkt && ok; k += C::kKT) {
                if (round) ok = mbar_wait(empty + 8 * s, (round - 1) & 1, abort_flag);
                if (!ok) break;
                if (elect_one()) {
                    const int u = r.u0 + k / kUnit, n = min(C::kKT, r.nkt - k) / kUnit;
                    const uint32_t st = stage0 + s * C::kStage, bar = full + 8 * s;
                    if (warp == 0) {
                        mbar_expect_tx(bar, n * unit_bytes);
                        const uint8_t* src = p.a.units + ((long long)r.mb * p.ku + u) * unit_bytes;
                        bulk_g2s(st + C::kKT * C::kX, src, n * unit_bytes, bar);
                        const int more = r.nkt - k - C::kAhead * C::kKT;
                        if (more > 0) bulk_prefetch(src + C::kAhead * C::kUS * unit_bytes, min(C::kKT, more) / kUnit * unit_bytes);
                    } else {
                        mbar_expect_tx(bar, C::kKT * C::kX);   // k-tiles past K come as zeros
                        tma_load_3d(st, &xmap, 0, r.n0, u * kUnit, bar);
                        // of the thread blocks that read the same x, one fetches it for all
                        const int next = u + C::kAhead * C::kUS;
                        if (k + C::kAhead * C::kKT < r.nkt && next / C::kUS % rows == r.mb) tma_prefetch_3d(&xmap, 0, r.n0, next * kUnit);
                    }
                }
                __syncwarp();
                if (++s == (uint32_t)C::kStages) s = 0, ++round;
            }
        }
    } else if (warp == 1) {
        // ---- matrix instructions
        constexpr uint32_t idesc = f16_idesc(128, NPAD);
        uint32_t s = 0, turn = 0, item = 0, phase = 0;   // phase: bit b, parity of operand block b's next use
        bool ok = true;
        while (ok && walk.next<NPAD>(p, r)) {
            if (item) ok = mbar_wait(acc_empty, (item - 1) & 1, abort_flag, 4);
            tc_fence_after();
            for (int k = 0; k < r.nkt && ok; k += C::kKT) {
                // the groups only report a unit after the stage's copies have landed, x included
#pragma unroll
                for (int i = 0; i < C::kUS; ++i) {
                    if (k + i * kUnit >= r.nkt || !ok) break;
                    const uint32_t blk = turn * C::kUS + i;
                    ok = mbar_wait(ready + 8 * blk, phase >> blk & 1, abort_flag);
                    if (!ok) break;
                    phase ^= 1u << blk;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t b = kmajor_desc_low(stage0 + s * C::kStage + i * kUnit * C::kX), more = k > 0 || i > 0;
#pragma unroll
                        for (int c = 0; c < C::kTurn; ++c)   // the block as a constant: see tc_mma_ts
                            if (turn == c)
#pragma unroll
                                for (int j = 0; j < 4 * kUnit; ++j)
                                    tc_mma_ts(j % C::kAcc * NPAD, C::kTmemA + (c * C::kUS + i) * 64 + 8 * j, b + (j / 4) * (C::kX >> 4) + 2 * (j % 4), kKMajorDescHigh,
                                              idesc, j >= C::kAcc ? 1u : more);
                        tc_commit(afree + 8 * blk);
                        if (i + 1 == C::kUS || k + (i + 1) * kUnit >= r.nkt) tc_commit(empty + 8 * s);
                    }
                    __syncwarp();
                }
                if (++s == (uint32_t)C::kStages) s = 0;
                if (++turn == (uint32_t)C::kTurn) turn = 0;
            }
            if (ok && elect_one()) tc_commit(acc_full);
            __syncwarp();
            ++item;
        }
    } else if (warp >= 8) {
        // ---- codes to fp16, thread = row
        // the units of kTurn consecutive stages go to the groups in order; group's operand block: its own
        const int grp = (warp - 8) / 4, quad = warp & 3, g = lane % 8, high8 = lane / 8 & 1;
        const int my_turn = grp / C::kUS, my_unit = grp % C::kUS;
        constexpr uint32_t unit_bytes = int4_unit_bytes(kGroup);
        const uint32_t code_off = C::kKT * C::kX + my_unit * unit_bytes + (2 * quad + lane / 16) * 512 + high8 * 8;
        const uint32_t par_off = C::kKT * C::kX + my_unit * unit_bytes + 2 * kInt4CodeBytes + 4 * (32 * quad + lane);
        const uint32_t a_addr = tmem_a + grp * 64 + ((uint32_t)quad << 21);
        uint32_t mask_low, mask_high, bits_low, bits_high;   // kept in registers for and_or
        asm volatile("mov.b32 %0, 0x000f000f;\n\tmov.b32 %1, 0x00f000f0;\n\tmov.b32 %2, 0x64006400;\n\tmov.b32 %3, 0x54005400;"
                     : "=r"(mask_low), "=r"(mask_high), "=r"(bits_low), "=r"(bits_high));
        uint32_t s = 0, round = 0, used = 0;
        int turn = 0;
        bool ok = true;
        while (ok && walk.next<NPAD>(p, r)) {
            for (int k = 0; k < r.nkt && ok; k += C::kKT) {
                // every stage's copies are waited for, also where the group has no unit: a parity only tells neighbouring phases
                // apart, so a group that skipped a stage could take the phase before for the one it needs
                ok = mbar_wait(full + 8 * s, round & 1, abort_flag);
                if (ok && turn == my_turn && k + my_unit * kUnit < r.nkt) {
                    if (used) ok = mbar_wait(afree + 8 * grp, (used - 1) & 1, abort_flag);
                    ++used;
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t st = stage0 + s * C::kStage;
                    uint32_t pw = 0;
                    __half2 sc, zl, zh;
                    uint32_t w[4][2];
#pragma unroll
                    for (int h = 0; h < 2 * kUnit; ++h) {   // 32 k each
                        if (h * 32 % kGroup == 0) {
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(pw) : "r"(st + par_off + h * 32 / kGroup * 512));
                            const __half2 sz = *reinterpret_cast<__half2*>(&pw), z = __high2half2(sz);
                            sc = __low2half2(sz);
                            zl = __hadd2(z, *reinterpret_cast<__half2*>(&bits_low));     // 1024 + z
                            zh = __hadd2(z, *reinterpret_cast<__half2*>(&bits_high));    // 64 + z
                        }
                        if (h % 2 == 0) {
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[q][0]), "=r"(w[q][1])
                                             : "r"(st + code_off + h / 2 * kInt4CodeBytes + 16 * int4_chunk(g, q)));
                        }
                        uint32_t o[16];
#pragma unroll
                        for (int q = 0; q < 4; ++q)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {   // k = 8 q + 2 e, + 1
                                const uint32_t u = e & 1 ? w[q][h % 2] >> 8 : w[q][h % 2];
                                const uint32_t v = e < 2 ? and_or(u, mask_low, bits_low) : and_or(u, mask_high, bits_high);
                                const __half2 c = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&v), e < 2 ? zl : zh), sc);
                                o[4 * q + e] = *reinterpret_cast<const uint32_t*>(&c);
                            }
                        tc_st16(a_addr + 16 * h, o);
                    }
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(ready + 8 * grp);
                }
                if (++s == (uint32_t)C::kStages) s = 0, ++round;
                if (++turn == C::kTurn) turn = 0;
            }
        }
    } else if (warp >= 4) {
        // ---- epilogue, thread = row
        const int quad = warp & 3;
        uint32_t item = 0;
        bool ok = true;
        while (ok && walk.next<NPAD>(p, r)) {
            ok = mbar_wait(acc_full, item & 1, abort_flag, 4);
            if (!ok) break;
            tc_fence_after();
            const bool cut = !(r.first && r.last);
            float* slot = p.a.ws + (2 * (size_t)blockIdx.x + r.first) * NPAD * 128 + 32 * quad + lane;
            const long long m = (long long)r.mb * 128 + 32 * quad + lane;
            const float bias = p.a.bias && m < p.a.M ? __half2float(__ushort_as_half(p.a.bias[m])) : 0.f;
            float* part = reinterpret_cast<float*>(smem + 1024);
            const uint32_t base = tmem + ((uint32_t)quad << 21);
#pragma unroll 1
            for (int c = 0; c < NPAD && r.n0 + c < p.a.N; c += 16) {
                uint32_t v[16];
                float y[16];
                tc_ld16(base + c, v);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(v[i]);
#pragma unroll
                for (int q = 1; q < C::kAcc; ++q) {
                    tc_ld16(base + q * NPAD + c, v);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] += __uint_as_float(v[i]);
                }
                if (p.split > 1) {   // the stages are idle: this run is the thread block's only one
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[(c + i) * 128 + 32 * quad + lane] = y[i];
                } else if (cut) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) slot[(c + i) * 128] = y[i];
                } else if (m < p.a.M) {
                    // all residuals first: they may be the output itself, and loads do not pass stores (one after the other they
                    // cost 9216 x 36864 with 509 rows 90 us)
                    const long long at = (r.n0 + c) * (long long)p.a.M + m;
                    uint16_t res[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) res[i] = p.a.residual && r.n0 + c + i < p.a.N ? p.a.residual[at + (long long)i * p.a.M] : (unsigned short)0;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (r.n0 + c + i < p.a.N) p.a.out[at + (long long)i * p.a.M] = __half_as_ushort(__float2half_rn(finish(p.a, y[i], bias, res[i])));
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty);
            ++item;
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (p.split > 1) cluster_finish<NPAD>(p, stage0);
    if (*abort_flag) {
        if (threadIdx.x == 0) {
            atomicOr(p.status, (int)kStatusWaitTimeout);
            for (int i = 0; i < C::kStages; ++i)   // copies still under way get a bounded chance to land
                for (uint32_t spin = 0; spin < 4096; ++spin)
                    if (mbar_try(full + 8 * i, 0) || mbar_try(full + 8 * i, 1)) break;
        }
        __syncthreads();
    }
    if (warp == 1) tc_dealloc(*holder, C::kTmemCols);
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled()
{
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(sym);
    });
    return fn;
}
template <int NPAD, int kGroup>
cudaError_t launch(cudaStream_t s, const Int4Args& a, const Plan& q, int* status)
{
    using C = Cfg<NPAD>;
    static bool prepared[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!prepared[dev]) {
        e = cudaFuncSetAttribute(int4_wide_kernel<NPAD, kGroup>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
        if (e != cudaSuccess) return e;
        prepared[dev] = true;
    }
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return cudaErrorNotSupported;
    CUtensorMap map;
    // x as [K / 64][N][64]: the k-tiles of a stage are one copy
    const cuuint64_t dims[3] = {64, (cuuint64_t)a.N, (cuuint64_t)a.K / 64};
    const cuuint64_t strides[2] = {(cuuint64_t)a.K * 2, 128};
    const cuuint32_t box[3] = {64, (cuuint32_t)NPAD, (cuuint32_t)C::kKT}, estr[3] = {1, 1, 1};
    if (enc(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<uint16_t*>(a.x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    return launch_product<NPAD>(s, int4_wide_kernel<NPAD, kGroup>, C::kThreads, C::kSmem, make_params(a, q, status), q, map);
}

template <int kGroup>
cudaError_t launch_group(cudaStream_t s, const Int4Args& a, const Plan& q, int* status)
{
    switch (q.npad) {
        case 32: return launch<32, kGroup>(s, a, q, status);
        case 64: return launch<64, kGroup>(s, a, q, status);
        case 128: return launch<128, kGroup>(s, a, q, status);
        default: return launch<256, kGroup>(s, a, q, status);
    }
}

}  // namespace

size_t int4_ws_floats(int M, int N, int K)
{
    const Plan q = plan_for(M, N, K);
    return q.whole ? 0 : (size_t)2 * q.ctas * q.npad * 128;
}

cudaError_t int4_wide_launch(cudaStream_t s, const Int4Args& a, int* status)
{
    const Plan q = plan_for(a.M, a.N, a.K);
    if (q.items * q.ku > 0x7fffffff) return cudaErrorInvalidValue;
    return a.group == 128 ? launch_group<128>(s, a, q, status) : a.group == 64 ? launch_group<64>(s, a, q, status) : launch_group<32>(s, a, q, status);
}

}  // namespace spb
