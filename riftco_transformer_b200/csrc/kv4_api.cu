// C entry points of the 4-bit paged K/V cache: argument checks in the manner of the FP32 cache's
// (check_paged_dims, api.cu), workspaces, and which kernel serves a call.
#include "kv4.cuh"
#include "b2_kernels.h"

#include <cmath>

namespace b2 {
namespace {

bool misaligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) != 0; }

// Whether [a, a + a_bytes) and [b, b + b_bytes) share a byte (null shares none).
bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
    if (a == nullptr || b == nullptr) return false;
    const uint64_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y ? y - x < a_bytes : x - y < b_bytes;
}

int32_t make_view(const b2_kv4_cache* cache, Kv4View* view, uint64_t* pool_bytes) {
    if (cache == nullptr) return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache must not be null");
    if (cache->reserved != 0) return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache reserved field must be zero");
    if (cache->n_seq == 0 || cache->kv_heads == 0 || cache->head_width == 0 || cache->block_size == 0 ||
        cache->physical_blocks == 0 || cache->max_blocks == 0) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache dimensions must be positive");
    }
    if (cache->head_width != 64 && cache->head_width != 128 && cache->head_width != 256) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache head width must be 64, 128 or 256, got %u", cache->head_width);
    }
    if (cache->block_size % kKv4Tile != 0) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache block size must be a multiple of 16, got %u", cache->block_size);
    }
    if (cache->physical_blocks - 1 > 0xFFFFFFFFull) {
        return fail(B2_STATUS_OVERFLOW, "4-bit cache physical block IDs exceed uint32_t");
    }
    // physical_blocks <= 2^32, block_size / 16 < 2^28: only the product with the heads can pass 64 bits
    const uint64_t tiles = cache->physical_blocks * (cache->block_size / kKv4Tile);
    const uint64_t per_tile = static_cast<uint64_t>(cache->kv_heads) * kv4_tile_bytes(cache->head_width);
    if (tiles > UINT64_MAX / 2 / per_tile) return fail(B2_STATUS_OVERFLOW, "4-bit cache pool size overflows");
    if (cache->pages == nullptr || cache->block_tables == nullptr) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache pages and block tables must not be null");
    }
    if (misaligned(cache->pages, 16)) return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache pages must be 16-byte aligned");
    if (misaligned(cache->block_tables, 4)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache block tables must be 4-byte aligned");
    }
    *pool_bytes = tiles * per_tile;
    *view = Kv4View{static_cast<uint8_t*>(cache->pages), cache->block_tables, cache->physical_blocks, cache->n_seq,
                    cache->max_blocks, cache->kv_heads, cache->head_width, cache->block_size / kKv4Tile};
    return B2_STATUS_OK;
}

// rows * heads * width * element, refused where it passes 2^62.
int32_t tensor_bytes(uint64_t rows, uint64_t heads, uint64_t width, uint64_t element, uint64_t* out) {
    const unsigned __int128 n = static_cast<unsigned __int128>(rows) * heads * width * element;
    if (n > (static_cast<unsigned __int128>(1) << 62)) return fail(B2_STATUS_OVERFLOW, "4-bit cache tensor size overflows");
    *out = static_cast<uint64_t>(n);
    return B2_STATUS_OK;
}

int32_t check_tokens(const Kv4View& view, uint32_t n_tokens, const uint32_t* positions, const uint32_t* token_seq) {
    if (n_tokens == 0) return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache needs at least one token");
    if (n_tokens > 0x7FFFFFFFu) return fail(B2_STATUS_OVERFLOW, "4-bit cache token count too large");
    if (positions == nullptr) return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache positions must not be null");
    if (misaligned(positions, 4) || misaligned(token_seq, 4)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache positions and token sequences must be 4-byte aligned");
    }
    if (token_seq == nullptr && n_tokens != view.n_seq) {
        return fail(B2_STATUS_INVALID_ARGUMENT,
                    "without token sequences the 4-bit cache takes one token per sequence: got %u tokens, %u sequences",
                    n_tokens, view.n_seq);
    }
    return B2_STATUS_OK;
}

struct AttentionCall {
    const b2_kv4_cache* cache;
    const b2_kv4_score_rules* rules;
    const uint32_t* prefix_lens;
    const float* q;
    const uint32_t* seq_lens;
    const uint32_t* chunk_starts;
    float* ctx;
    void* ctx_bf16;
    uint32_t rows, q_heads, max_chunk, max_seq_len;
    void* workspace;
    size_t workspace_bytes;
    uint32_t* status;
};

int32_t attention_args(const AttentionCall& c, Kv4AttentionArgs* args) {
    Kv4View view;
    uint64_t pool_bytes = 0;
    B2_TRY(make_view(c.cache, &view, &pool_bytes));
    if (c.q_heads == 0 || c.rows == 0 || c.max_seq_len == 0 || c.max_chunk == 0) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention dimensions must be positive");
    }
    if (c.q_heads % view.kv_heads != 0) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention query heads must be a multiple of KV heads");
    }
    if (c.max_seq_len > 0x7FFFFFFFu) return fail(B2_STATUS_OVERFLOW, "paged attention sequence too long");
    const uint64_t required = (static_cast<uint64_t>(c.max_seq_len) - 1) / c.cache->block_size + 1;
    if (required > view.max_blocks) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention block table size does not match the sequence");
    }
    if (c.q == nullptr || c.seq_lens == nullptr || (c.ctx == nullptr && c.ctx_bf16 == nullptr)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention pointers must not be null");
    }
    if (misaligned(c.q, 16) || misaligned(c.ctx, 16) || misaligned(c.ctx_bf16, 16)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention queries and contexts must be 16-byte aligned");
    }
    if (misaligned(c.seq_lens, 4) || misaligned(c.chunk_starts, 4) || misaligned(c.prefix_lens, 4) || misaligned(c.status, 4)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention lengths and status must be 4-byte aligned");
    }
    uint64_t bytes = 0;
    B2_TRY(tensor_bytes(c.rows, c.q_heads, view.head_width, 4, &bytes));
    if (overlap(c.ctx, bytes, c.q, bytes) || overlap(c.ctx_bf16, bytes / 2, c.q, bytes) ||
        overlap(c.ctx, bytes, c.ctx_bf16, bytes / 2) || overlap(c.ctx, bytes, view.pages, pool_bytes) ||
        overlap(c.ctx_bf16, bytes / 2, view.pages, pool_bytes)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention output must not alias an input");
    }
    Kv4ScoreRules rules;
    if (c.rules != nullptr) {
        // (beyond these 1 / cap or cap * log2(e) and their products with scores leave FP32)
        if (c.rules->softcap != 0.0f && !(c.rules->softcap >= 1e-6f && c.rules->softcap <= 1e18f)) {
            return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention score cap must be 0 or between 1e-6 and 1e18");
        }
        if (misaligned(c.rules->alibi_slopes, 4)) {
            return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention slopes must be 4-byte aligned");
        }
        rules.softcap = c.rules->softcap;
        rules.window = c.rules->window;
        rules.alibi_slopes = c.rules->alibi_slopes;
    }
    rules.prefix_lens = c.prefix_lens;
    *args = Kv4AttentionArgs{view, rules, c.q, c.seq_lens, c.chunk_starts, c.ctx, c.ctx_bf16,
                             c.rows, c.q_heads, c.max_seq_len, c.max_chunk, c.status};
    return B2_STATUS_OK;
}

// The caller's workspace, or the library's arena where there is none.
int32_t take_workspace(DeviceContext* ctx, size_t need, void** workspace, size_t* bytes, cudaStream_t stream) {
    if (need == 0) return B2_STATUS_OK;
    if (*workspace == nullptr) {
        B2_TRY(reserve_arena(ctx, need, stream));
        *workspace = ctx->arena;
        *bytes = ctx->arena_bytes;
    }
    if (misaligned(*workspace, 16)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention workspace must be 16-byte aligned");
    }
    if (*bytes < need) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention workspace too small: need %zu bytes, got %zu", need, *bytes);
    }
    return B2_STATUS_OK;
}

// A size query takes the same dimensions as the call; 0 for ones the call refuses.
DeviceContext* query_context(uint32_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t head_width, uint32_t max_seq_len) {
    int32_t status = B2_STATUS_OK;
    DeviceContext* ctx = device_context(&status);
    clear_error();
    if (rows == 0 || q_heads == 0 || kv_heads == 0 || q_heads % kv_heads != 0 || max_seq_len == 0 ||
        (head_width != 64 && head_width != 128 && head_width != 256)) {
        return nullptr;
    }
    return ctx;
}

int32_t chunk_workspace(const DeviceContext& ctx, uint32_t n_seq, uint32_t n_tokens, uint32_t q_heads, uint32_t kv_heads,
                        uint32_t head_width, uint32_t max_chunk, uint32_t max_seq_len, size_t* bytes) {
    if (!kv4_chunk_pays(n_seq, n_tokens, q_heads, kv_heads, max_chunk, max_seq_len)) {
        return kv4_decode_workspace_bytes(ctx, n_tokens, q_heads, kv_heads, head_width, max_seq_len, bytes);
    }
    *bytes = kv4_chunk_workspace_bytes(ctx.sm_count, n_seq, n_tokens, q_heads, kv_heads, head_width, max_chunk, max_seq_len);
    return B2_STATUS_OK;
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int32_t b2_rope_append_kv4(const b2_kv4_cache* cache, const float* q, float* q_out, const float* k, const float* v,
                           const uint32_t* positions, const uint32_t* token_seq, uint32_t n_tokens, uint32_t q_heads,
                           float theta, uint32_t* status_word, void* stream) {
    clear_error();
    int32_t status = B2_STATUS_OK;
    DeviceContext* ctx = device_context(&status);
    if (ctx == nullptr) return status;
    Kv4View view;
    uint64_t pool_bytes = 0;
    B2_TRY(make_view(cache, &view, &pool_bytes));
    B2_TRY(check_tokens(view, n_tokens, positions, token_seq));
    if (q_heads == 0) return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache append needs at least one query head");
    if (!(theta > 0.0f) || !std::isfinite(theta)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "rotary embedding theta must be finite and positive");
    }
    if (q == nullptr || q_out == nullptr || k == nullptr || v == nullptr) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache append pointers must not be null");
    }
    if (misaligned(q, 16) || misaligned(q_out, 16) || misaligned(k, 16) || misaligned(v, 16) || misaligned(status_word, 4)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache append tensors must be 16-byte aligned");
    }
    uint64_t q_bytes = 0, kv_bytes = 0;
    B2_TRY(tensor_bytes(n_tokens, q_heads, view.head_width, 4, &q_bytes));
    B2_TRY(tensor_bytes(n_tokens, view.kv_heads, view.head_width, 4, &kv_bytes));
    if ((q_out != q && overlap(q_out, q_bytes, q, q_bytes)) || overlap(q_out, q_bytes, k, kv_bytes) ||
        overlap(q_out, q_bytes, v, kv_bytes) || overlap(view.pages, pool_bytes, q, q_bytes) ||
        overlap(view.pages, pool_bytes, q_out, q_bytes) || overlap(view.pages, pool_bytes, k, kv_bytes) ||
        overlap(view.pages, pool_bytes, v, kv_bytes)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache append outputs must not alias an input (q_out may be q)");
    }
    const Kv4AppendArgs args{view, q, q_out, k, v, positions, token_seq, n_tokens, q_heads, theta, status_word};
    return launch_kv4_append(*ctx, args, static_cast<cudaStream_t>(stream));
}

int32_t b2_kv4_dequantize(const b2_kv4_cache* cache, const uint32_t* positions, const uint32_t* token_seq,
                          uint32_t n_tokens, float* k_out, float* v_out, uint32_t* status_word, void* stream) {
    clear_error();
    int32_t status = B2_STATUS_OK;
    DeviceContext* ctx = device_context(&status);
    if (ctx == nullptr) return status;
    Kv4View view;
    uint64_t pool_bytes = 0;
    B2_TRY(make_view(cache, &view, &pool_bytes));
    B2_TRY(check_tokens(view, n_tokens, positions, token_seq));
    if (k_out == nullptr || v_out == nullptr) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache outputs must not be null");
    }
    if (misaligned(k_out, 16) || misaligned(v_out, 16) || misaligned(status_word, 4)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache outputs must be 16-byte aligned");
    }
    uint64_t bytes = 0;
    B2_TRY(tensor_bytes(n_tokens, view.kv_heads, view.head_width, 4, &bytes));
    if (overlap(k_out, bytes, v_out, bytes) || overlap(view.pages, pool_bytes, k_out, bytes) ||
        overlap(view.pages, pool_bytes, v_out, bytes)) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "4-bit cache outputs must not alias");
    }
    const Kv4ReadArgs args{view, positions, token_seq, k_out, v_out, n_tokens, status_word};
    return launch_kv4_read(*ctx, args, static_cast<cudaStream_t>(stream));
}

size_t b2_paged_decode_kv4_workspace_bytes(uint32_t n_seq, uint32_t q_heads, uint32_t kv_heads, uint32_t head_width,
                                           uint32_t max_seq_len) {
    DeviceContext* ctx = query_context(n_seq, q_heads, kv_heads, head_width, max_seq_len);
    size_t bytes = 0;
    if (ctx == nullptr || kv4_decode_workspace_bytes(*ctx, n_seq, q_heads, kv_heads, head_width, max_seq_len, &bytes) != B2_STATUS_OK) {
        bytes = 0;
    }
    clear_error();
    return bytes;
}

int32_t b2_paged_decode_attention_kv4(const b2_kv4_cache* cache, const b2_kv4_score_rules* rules, const float* q,
                                      const uint32_t* seq_lens, float* ctx_out, void* ctx_bf16, uint32_t q_heads,
                                      uint32_t max_seq_len, void* workspace, size_t workspace_bytes,
                                      uint32_t* status_word, void* stream_ptr) {
    clear_error();
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    int32_t status = B2_STATUS_OK;
    DeviceContext* ctx = device_context(&status);
    if (ctx == nullptr) return status;
    const AttentionCall call{cache, rules, nullptr, q, seq_lens, nullptr, ctx_out, ctx_bf16,
                             cache == nullptr ? 0u : cache->n_seq, q_heads, 1u, max_seq_len, workspace, workspace_bytes,
                             status_word};
    Kv4AttentionArgs args;
    B2_TRY(attention_args(call, &args));
    size_t need = 0;
    B2_TRY(kv4_decode_workspace_bytes(*ctx, args.rows, q_heads, args.cache.kv_heads, args.cache.head_width, max_seq_len, &need));
    B2_TRY(take_workspace(ctx, need, &workspace, &workspace_bytes, stream));
    note_route(B2_ROUTE_ATTENTION_KV4);
    return launch_kv4_decode(*ctx, args, workspace, workspace_bytes, stream);
}

size_t b2_paged_chunk_kv4_workspace_bytes(uint32_t n_seq, uint32_t n_tokens, uint32_t q_heads, uint32_t kv_heads,
                                          uint32_t head_width, uint32_t max_chunk, uint32_t max_seq_len) {
    if (n_seq == 0 || max_chunk == 0) return 0;
    DeviceContext* ctx = query_context(n_tokens, q_heads, kv_heads, head_width, max_seq_len);
    size_t bytes = 0;
    if (ctx == nullptr ||
        chunk_workspace(*ctx, n_seq, n_tokens, q_heads, kv_heads, head_width, max_chunk, max_seq_len, &bytes) != B2_STATUS_OK) {
        bytes = 0;
    }
    clear_error();
    return bytes;
}

int32_t b2_paged_chunk_attention_kv4(const b2_kv4_cache* cache, const b2_kv4_score_rules* rules,
                                     const uint32_t* prefix_lens, const float* q, const uint32_t* seq_lens,
                                     const uint32_t* chunk_starts, void* ctx_bf16, uint32_t n_tokens, uint32_t q_heads,
                                     uint32_t max_chunk, uint32_t max_seq_len, void* workspace, size_t workspace_bytes,
                                     uint32_t* status_word, void* stream_ptr) {
    clear_error();
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    int32_t status = B2_STATUS_OK;
    DeviceContext* ctx = device_context(&status);
    if (ctx == nullptr) return status;
    if (chunk_starts == nullptr) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention pointers must not be null");
    }
    const AttentionCall call{cache, rules, prefix_lens, q, seq_lens, chunk_starts, nullptr, ctx_bf16, n_tokens, q_heads,
                             max_chunk, max_seq_len, workspace, workspace_bytes, status_word};
    Kv4AttentionArgs args;
    B2_TRY(attention_args(call, &args));
    if (max_chunk > max_seq_len || max_chunk > n_tokens) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention chunk is longer than its sequence or the call's tokens");
    }
    const uint32_t kv_heads = args.cache.kv_heads, head_width = args.cache.head_width;
    size_t need = 0;
    B2_TRY(chunk_workspace(*ctx, args.cache.n_seq, n_tokens, q_heads, kv_heads, head_width, max_chunk, max_seq_len, &need));
    B2_TRY(take_workspace(ctx, need, &workspace, &workspace_bytes, stream));
    if (kv4_chunk_pays(args.cache.n_seq, n_tokens, q_heads, kv_heads, max_chunk, max_seq_len)) {
        note_route(B2_ROUTE_ATTENTION_KV4_TILES);
        return launch_kv4_chunk(*ctx, args, workspace, workspace_bytes, stream);
    }
    note_route(B2_ROUTE_ATTENTION_KV4);
    return launch_kv4_decode(*ctx, args, workspace, workspace_bytes, stream);
}

}  // extern "C"
