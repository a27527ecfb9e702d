// Weights in 4 bits: layout shared by the kernels of the 4-bit linear layer.
//
// Value of weight (row, k): s (c - z), with code c and zero point z in 0..15 and s fp16 per row and group of 32, 64 or 128 k.
//
// codes   tiles of 16 rows x 64 k, 512 bytes each, [M/16][K/64]; a tile is the left operand of four m16n8k16 matrix instructions:
//         16 bytes a lane (lane = 4 g + t), words {row g, k 0..31}, {row g, k 32..63}, {row g + 8, ..}, {row g + 8, ..}; a
//         word holds k = 8 t + 4 p + e of its 32, in nibble p + 4 (e & 1) + 2 (e >> 1).  Two neighbouring k are then one AND
//         with 0x000f000f (p = 0) or 0x00f000f0 (p = 1), after a shift by 8 for e >= 2.
// params  [M/16][K/group][16 rows] {s, z}, both fp16.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace spb {

struct Int4Args {
    const uint32_t* codes;
    const __half2* params;
    int M, K, group;
    const uint16_t* x;          // [N][K]
    const uint16_t* bias;       // [M] or null
    const uint16_t* residual;   // [N][M] or null
    uint16_t* out;              // [N][M]
    int N, activation;
};
cudaError_t int4_linear_launch(cudaStream_t s, const Int4Args& a, int* status);

__host__ __device__ __forceinline__ int int4_nibble(int r)   // nibble of k = r (0..7) in the word of its lane
{
    return (r >> 2) + 4 * (r & 1) + 2 * ((r >> 1) & 1);
}

}  // namespace spb
