// Weights in 4 bits: layout shared by the kernels of the 4-bit linear layer.
//
// Value of weight (row, k): s (c - z), with code c and zero point z in 0..15 and s fp16 per row and group of 32, 64 or 128 k.
//
// Rows are padded to a multiple of 128 and K to one of 128, with weights of value zero.
//
// A unit is 128 rows x 128 k, one contiguous piece: [2 k-tiles of 64][8 row tiles of 16][512 bytes of codes], then
// [128 / group][128 rows] {s, z} (both fp16).  Units lie [M/128][K/128], so that any run of k of 128 rows is one bulk copy.
// The 512 bytes of a 16 x 64 tile are the left operand of four m16n8k16 matrix instructions, 16 bytes a lane (lane = 4 g + t):
// words {row g, k 0..31}, {row g, k 32..63}, {row g + 8, ..}, {row g + 8, ..}; a word holds k = 8 t + 4 p + e of its 32, in
// nibble p + 4 (e & 1) + 2 (e >> 1), so two neighbouring k are one AND with 0x000f000f (p = 0) or 0x00f000f0 (p = 1), after a
// shift by 8 for e >= 2.  The lane's 16 bytes are chunk 4 g + (t ^ (g >> 1)) of the tile: threads that each read one row's
// words of the same t then touch all shared-memory banks.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace spb {

struct Int4Args {
    const uint8_t* units;
    int M, K, group;
    const uint16_t* x;          // [N][K]
    const uint16_t* bias;       // [M] or null
    const uint16_t* residual;   // [N][M] or null
    uint16_t* out;              // [N][M]
    int N, activation;
    float* ws;                  // partial sums of tiles that are cut between thread blocks
    size_t ws_floats;
};
constexpr int kInt4StreamRows = 16;   // up to this many rows of x the mma.sync kernel runs, above it the tcgen05 one
cudaError_t int4_stream_launch(cudaStream_t s, const Int4Args& a, int* status);
cudaError_t int4_wide_launch(cudaStream_t s, const Int4Args& a, int* status);
int int4_stream_clusters(int split);   // clusters of `split` thread blocks of the streaming kernel that the device holds at once
size_t int4_ws_floats(int M, int N, int K);
__host__ __device__ __forceinline__ int int4_chunk(int g, int t) { return 4 * g + (t ^ (g >> 1)); }

constexpr int kInt4CodeBytes = 128 * 64 / 2;   // codes of one 64-k tile of 128 rows
__host__ __device__ constexpr int int4_unit_bytes(int group) { return 2 * kInt4CodeBytes + 512 * (128 / group); }
__host__ __device__ __forceinline__ long long int4_units(int M, int K) { return (long long)((M + 127) / 128) * ((K + 127) / 128); }
__host__ __device__ __forceinline__ int int4_nibble(int r)   // nibble of k = r (0..7) in the word of its lane
{
    return (r >> 2) + 4 * (r & 1) + 2 * ((r >> 1) & 1);
}

}  // namespace spb
