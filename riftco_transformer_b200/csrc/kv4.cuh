// The 4-bit paged K/V cache: its layout, and the argument blocks shared by the kernels that append to
// it, read it back and attend over it.
//
// One uint8 pool [physical_blocks, kv_heads, block_size / 16, 18 * d]. A tile holds 16 consecutive
// slots of one K/V head: 9d bytes of keys, then 9d bytes of values, each
//   codes  [d / 32][16 slots][16 bytes]   byte j = channels 2j (low nibble) and 2j + 1 of the 32
//   pairs  [16 slots][d / 64] of (fp16 scale, fp16 base), one for 64 channels
// and a value is base + scale * code. Keys and values of a tile lie side by side so that one bulk copy
// fetches both (2304 bytes at d = 128); a 16-byte code row is what one lane of ldmatrix addresses, so
// that a warp reads 16 rows of 64 channels with one instruction and no bank conflict, and transposed
// (`.trans`) the values come out paired by token, the order the second matrix product contracts over.
#pragma once

#include "b2_common.cuh"

namespace b2 {

constexpr uint32_t kKv4Tile = 16;          // slots of a tile
constexpr uint32_t kKv4Group = 64;         // channels that share one (scale, base)
constexpr uint32_t kKv4Pad = 0xFFFFFFFFu;  // position of a padding token

__host__ __device__ constexpr uint32_t kv4_half_bytes(uint32_t d) { return 9u * d; }
__host__ __device__ constexpr uint32_t kv4_tile_bytes(uint32_t d) { return 18u * d; }

struct Kv4View {
    uint8_t* pages;
    const uint32_t* block_tables;   // [n_seq, max_blocks]
    uint64_t physical_blocks;
    uint32_t n_seq, max_blocks, kv_heads, head_width;
    uint32_t tiles_per_block;       // block_size / 16
};

struct Kv4ScoreRules {
    float softcap = 0.0f;                  // 0: none
    uint32_t window = 0;                   // 0: none
    const float* alibi_slopes = nullptr;   // [q_heads] or null
    const uint32_t* prefix_lens = nullptr; // [n_seq] or null (several query tokens only)
};

struct Kv4AppendArgs {
    Kv4View cache;
    const float* q;
    float* q_out;
    const float* k;
    const float* v;
    const uint32_t* positions;
    const uint32_t* token_seq;   // may be null: token index = sequence
    uint32_t n_tokens, q_heads;
    float theta;
    uint32_t* status;
};

struct Kv4ReadArgs {
    Kv4View cache;
    const uint32_t* positions;
    const uint32_t* token_seq;
    float* k_out;
    float* v_out;
    uint32_t n_tokens;
    uint32_t* status;
};

struct Kv4AttentionArgs {
    Kv4View cache;
    Kv4ScoreRules rules;
    const float* q;               // [rows, q_heads, d]
    const uint32_t* seq_lens;     // [n_seq]
    const uint32_t* chunk_starts; // null: one row per sequence; else [n_seq + 1], rows of each sequence
    float* ctx;                   // either may be null, not both
    void* ctx16;
    uint32_t rows, q_heads, max_seq_len;
    uint32_t max_chunk;           // 1 without chunk_starts
    uint32_t* status;
};

// kv4_cache.cu
int32_t launch_kv4_append(const DeviceContext& ctx, const Kv4AppendArgs& args, cudaStream_t stream);
int32_t launch_kv4_read(const DeviceContext& ctx, const Kv4ReadArgs& args, cudaStream_t stream);

// kv4_decode.cu - every row on its own: one token per sequence, or a few tokens of each.
size_t kv4_decode_workspace_bytes(int sm_count, uint64_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t head_width,
                                  uint32_t max_seq_len);
int32_t launch_kv4_decode(const DeviceContext& ctx, const Kv4AttentionArgs& args, void* workspace,
                          size_t workspace_bytes, cudaStream_t stream);

#if defined(__CUDACC__)

// Adds `bits` to the caller's status word.
__device__ __forceinline__ void kv4_flag(uint32_t* status, uint32_t bits) {
    if (status != nullptr) atomicOr(status, bits);
}

// Byte offset of tile `tile` (of a sequence) of head `head` when its page is `phys`.
__device__ __forceinline__ uint64_t kv4_tile_offset(const Kv4View& c, uint64_t phys, uint32_t head, uint32_t tile_in_page) {
    return ((phys * c.kv_heads + head) * c.tiles_per_block + tile_in_page) * kv4_tile_bytes(c.head_width);
}

// Where one token lives: false (and a page that is never dereferenced) when the sequence, the position
// or the block id lies outside what the cache holds.
__device__ __forceinline__ bool kv4_locate(const Kv4View& c, uint32_t seq, uint32_t position, uint64_t* phys,
                                           uint32_t* tile_in_page, uint32_t* slot) {
    const uint32_t block_size = c.tiles_per_block * kKv4Tile;
    const uint32_t logical = position / block_size, in_page = position % block_size;
    *tile_in_page = in_page / kKv4Tile;
    *slot = in_page % kKv4Tile;
    *phys = 0;
    if (seq >= c.n_seq || logical >= c.max_blocks) return false;
    *phys = c.block_tables[static_cast<uint64_t>(seq) * c.max_blocks + logical];
    return *phys < c.physical_blocks;
}

#endif  // __CUDACC__

}  // namespace b2
