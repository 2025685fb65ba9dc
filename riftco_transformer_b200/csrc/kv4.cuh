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

#if defined(__CUDACC__)
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#endif

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
int32_t kv4_decode_workspace_bytes(const DeviceContext& ctx, uint64_t rows, uint32_t q_heads, uint32_t kv_heads,
                                   uint32_t head_width, uint32_t max_seq_len, size_t* bytes);
int32_t launch_kv4_decode(const DeviceContext& ctx, const Kv4AttentionArgs& args, void* workspace,
                          size_t workspace_bytes, cudaStream_t stream);

// kv4_chunk.cu - tiles of 128 query rows on the tcgen05 tensor cores, bf16 contexts. `pays`: rather than row by row.
bool kv4_chunk_pays(uint32_t n_seq, uint64_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t max_chunk, uint32_t max_seq_len);
size_t kv4_chunk_workspace_bytes(int sm_count, uint32_t n_seq, uint64_t rows, uint32_t q_heads, uint32_t kv_heads,
                                 uint32_t head_width, uint32_t max_chunk, uint32_t max_seq_len);
int32_t launch_kv4_chunk(const DeviceContext& ctx, const Kv4AttentionArgs& args, void* workspace,
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


// ---- shared by the two attention kernels ------------------------------------------------------

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -FLT_MAX;    // running maximum before the first score (log2 units)

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// fp16 numbers 1024 + code (or 1024 + 16 code) of two codes of a word, 16 bits apart: (word & MASK) | k1024 in one
// instruction. k1024 comes from opaque_1024() once per thread: an instruction holds one immediate, and given two
// constants the compiler takes an AND and an OR (a sixth of the decode kernel's instructions).
template <uint32_t MASK>
__device__ __forceinline__ uint32_t codes_1024(uint32_t word, uint32_t k1024) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(word), "n"(MASK), "r"(k1024));
    return r;
}
__device__ __forceinline__ uint32_t opaque_1024() {
    uint32_t r;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(r));
    return r;
}
__device__ __forceinline__ float low_half(uint32_t pair) { return __low2float(*reinterpret_cast<__half2*>(&pair)); }
__device__ __forceinline__ float high_half(uint32_t pair) { return __high2float(*reinterpret_cast<__half2*>(&pair)); }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void bulk_load(uint32_t dst32, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst32), "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
                 : "memory");
}

// For one thread of the grid: BAD_BLOCK where chunks end behind the call's rows (chunk_starts rises, its last entry tells).
// The caller raises it at its end, so that nobody waits for the load.
__device__ __forceinline__ uint32_t chunk_starts_flag(const Kv4AttentionArgs& a) {
    if (blockIdx.x != 0u || threadIdx.x != 0u || a.chunk_starts == nullptr) return 0u;
    return __ldg(a.chunk_starts + a.cache.n_seq) > a.rows ? B2_ATTN_STATUS_BAD_BLOCK : 0u;
}

// What a row sees: tokens [begin, end) of sequence `seq`, its own position, and whether the caller's
// lengths were out of bounds.
struct RowSpan {
    uint32_t seq, position, begin, end;
    bool bad;
    bool owned;   // false: a row behind the last sequence, which is left as it was
};
__device__ __forceinline__ RowSpan row_span(const Kv4AttentionArgs& a, uint32_t row) {
    RowSpan r{row, 0, 0, 0, false, true};
    uint32_t back = 0;   // tokens after this one
    if (a.chunk_starts != nullptr) {
        uint32_t lo = 0, hi = a.cache.n_seq;   // the last sequence that starts at or before `row`
        while (lo + 1u < hi) {
            const uint32_t mid = (lo + hi) / 2u;
            if (__ldg(a.chunk_starts + mid) <= row) lo = mid; else hi = mid;
        }
        r.seq = lo;
        const uint32_t first = __ldg(a.chunk_starts + lo), last = __ldg(a.chunk_starts + lo + 1u);
        r.owned = row >= first && row < last;
        if (!r.owned) return r;
        back = last - 1u - row;
        r.bad = last - first > a.max_chunk;
    }
    uint32_t len = __ldg(a.seq_lens + r.seq);
    if (len > a.max_seq_len) {
        len = a.max_seq_len;
        r.bad = true;
    }
    if (back >= len) {
        r.bad = r.bad || a.chunk_starts != nullptr;   // more new tokens than the sequence holds
        return r;
    }
    r.position = len - 1u - back;
    r.end = r.position + 1u;
    if (a.rules.prefix_lens != nullptr) r.end = max(r.end, min(len, __ldg(a.rules.prefix_lens + r.seq)));
    if (a.rules.window != 0u && r.position >= a.rules.window) r.begin = r.position - a.rules.window + 1u;
    return r;
}

// Four channels of a context, o / l; zeros where nothing was seen (l = 0).
template <int D>
__device__ __forceinline__ void put_context(const Kv4AttentionArgs& a, uint64_t out_head, uint32_t c, float4 o, float l) {
    o = l == 0.0f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
    if (a.ctx != nullptr) *reinterpret_cast<float4*>(a.ctx + out_head * D + c) = o;
    if (a.ctx16 != nullptr) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(o.x, o.y), hi = __floats2bfloat162_rn(o.z, o.w);
        uint2 packed;
        packed.x = *reinterpret_cast<const uint32_t*>(&lo);
        packed.y = *reinterpret_cast<const uint32_t*>(&hi);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.ctx16) + out_head * D + c) = packed;
    }
}

struct Joined {
    float m, l;   // maximum (log2 units), sum of weights
    float4 o;     // sums of four channels
};
// Joins `n` partial results of one (row, query head), each [m, l, -, -, sums of the channels], for the channels
// c .. c + 3 of this thread, in order: the first at `first`, the others `stride` floats apart from `rest`.
__device__ __forceinline__ Joined join_run(const float* first, const float* rest, uint64_t stride, uint32_t n, uint32_t c) {
    Joined j{kNoMax, 0.0f, make_float4(0.f, 0.f, 0.f, 0.f)};
    for (uint32_t s0 = 0; s0 < n; s0 += 8u) {
        float2 ml[8];
        float4 x[8];
#pragma unroll
        for (uint32_t u = 0; u < 8u; ++u) {   // all loads before the first use
            const bool live = s0 + u < n;
            const float* part = s0 + u == 0u ? first : rest + (s0 + u - 1u) * stride;
            ml[u] = live ? *reinterpret_cast<const float2*>(part) : make_float2(kNoMax, 0.0f);
            x[u] = live ? *reinterpret_cast<const float4*>(part + 4u + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float top = j.m;
#pragma unroll
        for (uint32_t u = 0; u < 8u; ++u) top = fmaxf(top, ml[u].x);
        const float keep = ex2(j.m - top);
        j.m = top;
        j.l *= keep;
        j.o = make_float4(j.o.x * keep, j.o.y * keep, j.o.z * keep, j.o.w * keep);
#pragma unroll
        for (uint32_t u = 0; u < 8u; ++u) {
            const float f = ex2(ml[u].x - j.m);
            j.l = fmaf(ml[u].y, f, j.l);
            j.o.x = fmaf(x[u].x, f, j.o.x);
            j.o.y = fmaf(x[u].y, f, j.o.y);
            j.o.z = fmaf(x[u].z, f, j.o.z);
            j.o.w = fmaf(x[u].w, f, j.o.w);
        }
    }
    return j;
}
template <int D>
__device__ __forceinline__ void finish(const Kv4AttentionArgs& a, const Joined& j, uint64_t out_head, uint32_t c, bool sees_any) {
    if (j.l == 0.0f && sees_any && c == 0u) kv4_flag(a.status, B2_ATTN_STATUS_ALL_NEG_INF);
    put_context<D>(a, out_head, c, j.o, j.l);
}

#endif  // __CUDACC__

}  // namespace b2
