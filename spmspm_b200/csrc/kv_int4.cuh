// The paged 4-bit key/value cache: layout and the pieces that its kernels share.
//
// A page holds page_size tokens (a multiple of 16) of every key/value head; page p, head h is one contiguous run of
// page_size / 16 blocks of 16 tokens.  A block is one contiguous piece of 20 D bytes,
//     [K codes 16 x D/2][K parameters 16 x D/32 x 4][V codes 16 x D/2][V parameters 16 x D/32 x 4],
// so that the attention kernel fetches 16 tokens of one head, keys and values, with one bulk copy.
//
// Value of channel c of a token: m + code * s, with s and m (fp16) shared by 32 consecutive channels.
//
// Inside a block everything lies as the matrix instruction's operand registers want it (m16n8k16, lane = 4 g + t):
//   K codes   token-major rows; word t * (D/32) + w of a row holds the 8 channels of group w that lane t feeds to the
//             two k-steps of that group: channel 32 w + 16 p + 4 t + e sits in nibble p + 4 (e & 1) + 2 (e >> 1).  A lane
//             reads its row with one 16-byte (D = 128) or 8-byte load; and with 0x000f000f / 0x00f000f0 masks every
//             register of the operand is one AND (after one shift for e >= 2).
//   K params  [token][group] {s, m}
//   V codes   the operand is V^T (channels x tokens) in tiles of 16 channels: lane 4 g + t takes channels 16 i + 2 g and 16 i + 2 g + 1 of
//             every tile i, tokens 2t, 2t+1 (first half, j = 0) and 2t + 8, 2t + 9 (j = 1).  Word k of a lane is group k, tiles
//             2 k and 2 k + 1; halfword (token & 1) of it, byte (tile & 1), nibble (channel & 1).
//             Byte address j * 4 D + (4 g + t) * D/8 + 4 k + 2 (token & 1) + (tile & 1).
//   V params  [token pair][group] {s of the even token, s of the odd, m of the even, m of the odd}
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace spb {

constexpr int kKvBlock = 16;   // tokens a block holds
constexpr int kKvGroup = 32;   // channels that share scale and minimum

template <int D>
struct KvLayout {
    static constexpr int kGroups = D / kKvGroup;
    static constexpr int kCodes = 16 * D / 2;            // bytes of one operand's codes
    static constexpr int kParams = 16 * kGroups * 4;     // bytes of one operand's parameters
    static constexpr int kKCodes = 0, kKParams = kCodes, kVCodes = kCodes + kParams, kVParams = 2 * kCodes + kParams;
    static constexpr int kBlockBytes = 2 * (kCodes + kParams);   // 20 D
};

// What every kernel of the cache gets: the pool and where each sequence's tokens are.
struct KvView {
    uint8_t* pool;
    const int* table;        // [B][table_stride] page numbers
    const int* lens;         // [B] tokens of each sequence in the cache, the new ones included
    const int* cu;           // [B + 1] first row of each sequence among the new tokens, or null: n_tokens / B each
    int n_tokens;            // rows of the packed new tokens
    int per_seq;             // n_tokens / B
    int table_stride;        // entries a row of the table has
    int num_pages, page_size, kv_heads, B;
};

struct KvAppendArgs {
    KvView c;
    const uint16_t *k, *v, *q;   // [n_tokens][heads][D], innermost contiguous; q null: none
    long long k_tok, v_tok, q_tok, k_head, v_head, q_head;   // strides in elements
    uint16_t* q_out;             // [n_tokens][q_heads][D] contiguous
    const float *cosv, *sinv;    // [max_pos][rot / 2], null: no rotation
    int q_heads, rot, max_pos, interleaved;
};
struct KvReadArgs {
    KvView c;
    uint16_t *k, *v;   // [n_tokens][kv_heads][D] contiguous
};
struct KvAttnArgs {
    KvView c;
    const uint16_t* q;
    long long q_tok, q_head;
    uint16_t* out;     // [n_tokens][q_heads][D] contiguous
    int q_heads, max_q;
    float scale;
    float* ws;
    size_t ws_floats;
    int tall;          // sequences with this many rows a key head (new tokens times query heads that share it) go to kv_prefill
};
cudaError_t kv_append_launch(cudaStream_t s, int D, const KvAppendArgs& a, int* status);
cudaError_t kv_read_launch(cudaStream_t s, int D, const KvReadArgs& a, int* status);
cudaError_t kv_attention_launch(cudaStream_t s, int D, const KvAttnArgs& a, int* status);
cudaError_t kv_prefill_launch(cudaStream_t s, int D, const KvAttnArgs& a, int tall, int* status);
size_t kv_attention_ws_floats(int D, int B, int q_heads, int kv_heads, int max_q);

// New tokens of sequence b: first row and count.  cu is the caller's: clamped, so that bad offsets cannot index outside.
__device__ __forceinline__ void kv_rows(const KvView& c, int b, int& first, int& count)
{
    if (c.cu) {
        first = min(max(c.cu[b], 0), c.n_tokens);
        count = min(max(c.cu[b + 1], first), c.n_tokens) - first;
    } else {
        count = c.per_seq;
        first = count * b;
    }
}

// Byte offset in the pool of the 16-token block that holds token `pos` of sequence b, head h; -1 when the table has no
// usable page there (past its width, negative or not below num_pages).
template <int D>
__device__ __forceinline__ long long kv_block_offset(const KvView& c, int b, int h, int pos)
{
    const unsigned pi = (unsigned)pos / (unsigned)c.page_size, in_page = (unsigned)pos - pi * c.page_size;
    if (pi >= (unsigned)c.table_stride) return -1;
    const int page = c.table[(long long)b * c.table_stride + pi];
    if (page < 0 || page >= c.num_pages) return -1;
    return (((long long)page * c.kv_heads + h) * (c.page_size / kKvBlock) + in_page / kKvBlock) * KvLayout<D>::kBlockBytes;
}

}  // namespace spb
