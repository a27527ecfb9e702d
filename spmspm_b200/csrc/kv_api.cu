// extern "C" entry points of the paged 4-bit key/value cache (declared in include/spmm_b200.h): argument checks and launches.
#include "../../include/spmm_b200.h"
#include "kv_int4.cuh"

namespace spb {
namespace {

constexpr long long kMaxInt = 0x7fffffffll;

// Shape, null and alignment checks that the three entry points share; false: message set.
bool check_cache(const char* who, const void* pool, int num_pages, int page_size, int kv_heads, int head_dim, const void* table,
                 int table_stride, const void* lens, const void* cu, int B, long long n_tokens)
{
    if (head_dim != 64 && head_dim != 128) {
        set_error("%s: head_dim must be 64 or 128, got %d", who, head_dim);
        return false;
    }
    if (num_pages <= 0 || page_size <= 0 || page_size % kKvBlock || page_size > 65536 || kv_heads <= 0 || kv_heads > 65536) {
        set_error("%s: num_pages and kv_heads must be positive and page_size a positive multiple of 16 up to 65536 "
                  "(num_pages=%d kv_heads=%d page_size=%d)", who, num_pages, kv_heads, page_size);
        return false;
    }
    if (B <= 0 || B > 65535 || table_stride <= 0 || n_tokens < 0 || n_tokens > kMaxInt / kv_heads / 2) {
        set_error("%s: batch must be 1..65535, table_stride positive and n_tokens * kv_heads below 2^30 (batch=%d table_stride=%d "
                  "n_tokens=%lld)", who, B, table_stride, n_tokens);
        return false;
    }
    if (!cu && n_tokens % B) {
        set_error("%s: without cu_q every sequence has the same number of new tokens: %lld rows do not divide by %d", who, n_tokens, B);
        return false;
    }
    if (!pool || !table || !lens) {
        set_error("%s: null device pointer", who);
        return false;
    }
    if (!aligned16(pool) || ((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(lens) | reinterpret_cast<uintptr_t>(cu)) & 3)) {
        set_error("%s: the pool must be 16-byte aligned, page_table, kv_lens and cu_q 4-byte aligned", who);
        return false;
    }
    return true;
}
// Vectors read four channels at a time.
bool check_vectors(const char* who, const char* name, const void* p, long long tok, long long head)
{
    if (!p) {
        set_error("%s: null device pointer (%s)", who, name);
        return false;
    }
    if ((reinterpret_cast<uintptr_t>(p) & 7) || tok % 4 || head % 4 || tok < 0 || head < 0) {
        set_error("%s: %s must be 8-byte aligned with strides that are non-negative multiples of 4 elements", who, name);
        return false;
    }
    return true;
}
// Bytes from the first to the last element of [n][heads][dim] fp16.
size_t span_bytes(long long n, long long tok, int heads, long long head, int dim)
{
    return n > 0 ? 2 * ((size_t)(n - 1) * tok + (size_t)(heads - 1) * head + dim) : 0;
}
// An output [n][heads][dim] may lie on the input `in` row by row (in place), but not otherwise on it.
bool check_in_place(const char* who, const char* names, const void* out, const void* in, long long n, long long tok, int heads, long long head, int dim)
{
    const bool same = out == in && head == dim && (n < 2 || tok == (long long)heads * dim);
    if (same || !overlap(out, span_bytes(n, (long long)heads * dim, heads, dim, dim), in, span_bytes(n, tok, heads, head, dim))) return true;
    set_error("%s: %s overlap without being the same rows", who, names);
    return false;
}
KvView view(void* pool, int num_pages, int page_size, int kv_heads, const int* table, int table_stride, const int* lens, const int* cu,
            int B, long long n_tokens)
{
    KvView c;
    c.pool = static_cast<uint8_t*>(pool);
    c.table = table;
    c.lens = lens;
    c.cu = cu;
    c.n_tokens = (int)n_tokens;
    c.per_seq = (int)(n_tokens / B);
    c.table_stride = table_stride;
    c.num_pages = num_pages;
    c.page_size = page_size;
    c.kv_heads = kv_heads;
    c.B = B;
    return c;
}

}  // namespace
}  // namespace spb

extern "C" {

size_t spb_kv_cache_bytes(int num_pages, int page_size, int kv_heads, int head_dim)
{
    if (num_pages <= 0 || page_size <= 0 || page_size % spb::kKvBlock || kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)num_pages * kv_heads * (page_size / spb::kKvBlock) * 20 * head_dim;
}

int spb_kv_append(void* stream, void* pool, int num_pages, int page_size, int kv_heads, int head_dim, const int* page_table,
                  int table_stride, const int* kv_lens, const int* cu_q, int batch, long long n_tokens, const uint16_t* k,
                  long long k_token_stride, long long k_head_stride, const uint16_t* v, long long v_token_stride,
                  long long v_head_stride, const uint16_t* q, long long q_token_stride, long long q_head_stride, int q_heads,
                  uint16_t* q_out, const float* cos_table, const float* sin_table, int max_pos, int rot_dim, int interleaved)
{
    using namespace spb;
    const char* who = "kv_append";
    if (!check_cache(who, pool, num_pages, page_size, kv_heads, head_dim, page_table, table_stride, kv_lens, cu_q, batch, n_tokens))
        return (int)cudaErrorInvalidValue;
    if (!check_vectors(who, "k", k, k_token_stride, k_head_stride) || !check_vectors(who, "v", v, v_token_stride, v_head_stride))
        return (int)cudaErrorInvalidValue;
    if ((cos_table == nullptr) != (sin_table == nullptr)) {
        set_error("%s: cos_table and sin_table are given together", who);
        return (int)cudaErrorInvalidValue;
    }
    if (cos_table && (rot_dim <= 0 || rot_dim > head_dim || rot_dim % 8 || max_pos <= 0)) {
        set_error("%s: rot_dim must be a multiple of 8 up to head_dim and max_pos positive (rot_dim=%d max_pos=%d)", who, rot_dim, max_pos);
        return (int)cudaErrorInvalidValue;
    }
    if (cos_table && ((reinterpret_cast<uintptr_t>(cos_table) | reinterpret_cast<uintptr_t>(sin_table)) & 15)) {
        set_error("%s: cos_table and sin_table must be 16-byte aligned", who);
        return (int)cudaErrorInvalidValue;
    }
    if (q) {
        if (!aligned16(q_out)) {
            set_error("%s: q_out must be 16-byte aligned", who);
            return (int)cudaErrorInvalidValue;
        }
        if (!check_vectors(who, "q", q, q_token_stride, q_head_stride) || !check_vectors(who, "q_out", q_out, 0, 0)) return (int)cudaErrorInvalidValue;
        if (!cos_table) {
            set_error("%s: q is only taken to be rotated: cos_table and sin_table are missing", who);
            return (int)cudaErrorInvalidValue;
        }
        if (q_heads <= 0 || q_heads > 65536 || n_tokens > kMaxInt / (2ll * kv_heads + q_heads)) {
            set_error("%s: q_heads must be positive and n_tokens * heads below 2^31 (q_heads=%d)", who, q_heads);
            return (int)cudaErrorInvalidValue;
        }
        if (!check_in_place(who, "q and q_out", q_out, q, n_tokens, q_token_stride, q_heads, q_head_stride, head_dim)) return (int)cudaErrorInvalidValue;
        const size_t bytes = span_bytes(n_tokens, (long long)q_heads * head_dim, q_heads, head_dim, head_dim);
        if (overlap(q_out, bytes, k, span_bytes(n_tokens, k_token_stride, kv_heads, k_head_stride, head_dim)) ||
            overlap(q_out, bytes, v, span_bytes(n_tokens, v_token_stride, kv_heads, v_head_stride, head_dim))) {
            set_error("%s: q_out overlaps the keys or values", who);
            return (int)cudaErrorInvalidValue;
        }
    }
    if (n_tokens == 0) return 0;
    int* status = nullptr;
    cudaError_t e = device_status_ptr(&status);
    if (e != cudaSuccess) return (int)e;
    KvAppendArgs a;
    a.c = view(pool, num_pages, page_size, kv_heads, page_table, table_stride, kv_lens, cu_q, batch, n_tokens);
    a.k = k, a.v = v, a.q = q;
    a.k_tok = k_token_stride, a.v_tok = v_token_stride, a.q_tok = q_token_stride;
    a.k_head = k_head_stride, a.v_head = v_head_stride, a.q_head = q_head_stride;
    a.q_out = q_out;
    a.cosv = cos_table, a.sinv = sin_table;
    a.q_heads = q_heads, a.rot = cos_table ? rot_dim : 0, a.max_pos = max_pos, a.interleaved = interleaved;
    e = kv_append_launch((cudaStream_t)stream, head_dim, a, status);
    if (e != cudaSuccess) set_error("%s: %s", who, cudaGetErrorString(e));
    return (int)e;
}

int spb_kv_read(void* stream, const void* pool, int num_pages, int page_size, int kv_heads, int head_dim, const int* page_table,
                int table_stride, const int* kv_lens, const int* cu_q, int batch, long long n_tokens, uint16_t* k, uint16_t* v)
{
    using namespace spb;
    const char* who = "kv_read";
    if (!check_cache(who, pool, num_pages, page_size, kv_heads, head_dim, page_table, table_stride, kv_lens, cu_q, batch, n_tokens) ||
        !check_vectors(who, "k", k, 0, 0) || !check_vectors(who, "v", v, 0, 0))
        return (int)cudaErrorInvalidValue;
    if (n_tokens == 0) return 0;
    const size_t bytes = 2 * (size_t)n_tokens * kv_heads * head_dim;
    if (overlap(k, bytes, v, bytes)) {
        set_error("%s: k and v overlap", who);
        return (int)cudaErrorInvalidValue;
    }
    int* status = nullptr;
    cudaError_t e = device_status_ptr(&status);
    if (e != cudaSuccess) return (int)e;
    KvReadArgs a;
    a.c = view(const_cast<void*>(pool), num_pages, page_size, kv_heads, page_table, table_stride, kv_lens, cu_q, batch, n_tokens);
    a.k = k, a.v = v;
    e = kv_read_launch((cudaStream_t)stream, head_dim, a, status);
    if (e != cudaSuccess) set_error("%s: %s", who, cudaGetErrorString(e));
    return (int)e;
}

size_t spb_kv_attention_workspace_bytes(int head_dim, int batch, int q_heads, int kv_heads, int max_q)
{
    if ((head_dim != 64 && head_dim != 128) || batch <= 0 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || max_q < 0) return 0;
    return 4 * spb::kv_attention_ws_floats(head_dim, batch, q_heads, kv_heads, max_q);
}

int spb_kv_attention(void* stream, const void* pool, int num_pages, int page_size, int kv_heads, int head_dim, const int* page_table,
                     int table_stride, const int* kv_lens, const int* cu_q, int batch, long long n_tokens, const uint16_t* q,
                     long long q_token_stride, long long q_head_stride, int q_heads, int max_q, float scale, uint16_t* out,
                     void* workspace, size_t workspace_bytes)
{
    using namespace spb;
    const char* who = "kv_attention";
    if (!check_cache(who, pool, num_pages, page_size, kv_heads, head_dim, page_table, table_stride, kv_lens, cu_q, batch, n_tokens) ||
        !check_vectors(who, "q", q, q_token_stride, q_head_stride))
        return (int)cudaErrorInvalidValue;
    if (q_heads <= 0 || q_heads % kv_heads || n_tokens > kMaxInt / q_heads) {
        set_error("%s: q_heads must be a positive multiple of kv_heads and n_tokens * q_heads below 2^31 (q_heads=%d kv_heads=%d)", who, q_heads, kv_heads);
        return (int)cudaErrorInvalidValue;
    }
    if (max_q < 0 || max_q > n_tokens) {
        set_error("%s: max_q must be in 0..n_tokens, got %d", who, max_q);
        return (int)cudaErrorInvalidValue;
    }
    if (!out || !aligned16(out) || !workspace || !aligned16(workspace)) {
        set_error("%s: out and the workspace must be given and 16-byte aligned", who);
        return (int)cudaErrorInvalidValue;
    }
    if (!check_in_place(who, "q and out", out, q, n_tokens, q_token_stride, q_heads, q_head_stride, head_dim)) return (int)cudaErrorInvalidValue;
    if (workspace_bytes < spb_kv_attention_workspace_bytes(head_dim, batch, q_heads, kv_heads, max_q)) {
        set_error("%s: the workspace has %zu bytes, spb_kv_attention_workspace_bytes asks for %zu", who, workspace_bytes,
                  spb_kv_attention_workspace_bytes(head_dim, batch, q_heads, kv_heads, max_q));
        return (int)cudaErrorInvalidValue;
    }
    if (n_tokens == 0) return 0;
    int* status = nullptr;
    cudaError_t e = device_status_ptr(&status);
    if (e != cudaSuccess) return (int)e;
    KvAttnArgs a;
    a.c = view(const_cast<void*>(pool), num_pages, page_size, kv_heads, page_table, table_stride, kv_lens, cu_q, batch, n_tokens);
    a.q = q, a.q_tok = q_token_stride, a.q_head = q_head_stride;
    a.out = out;
    a.q_heads = q_heads, a.max_q = max_q;
    a.scale = scale;
    a.ws = static_cast<float*>(workspace);
    a.ws_floats = workspace_bytes / 4;
    e = kv_attention_launch((cudaStream_t)stream, head_dim, a, status);
    if (e != cudaSuccess) set_error("%s: %s", who, cudaGetErrorString(e));
    return (int)e;
}

}  // extern "C"
