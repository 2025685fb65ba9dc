// Attention of several new tokens per sequence over the 4-bit paged cache, on the tcgen05 tensor cores.
//
// A row is (new token, query head of one K/V head): token i and head h of the group are row i * rep + h, so
// that any number of query heads per K/V head fills whole tiles. A CTA takes 256 rows (two tiles of 128
// = two M of tcgen05.mma) of one K/V head and walks the cached tokens they see in blocks of 64:
//   S = Q K^T          [128 x 64], A and B in shared memory, FP32 in tensor memory
//   P = 2^(S - m)      fp16, written over S
//   O += P V           A = P in tensor memory, B = V^T in shared memory, FP32 in tensor memory
// Unlike in the single-row kernel (kv4_decode.cu) a block of K and V serves 256 rows, so its codes are expanded
// to fp16 once, by four warps, into swizzled shared-memory tiles: value = scale * code + base with one rounding.
// The contraction order inside eight channels follows the nibbles (0 4 1 5 2 6 3 7; Q is staged to match); V is
// transposed on the way, since its contraction is over tokens: two tokens' words are merged so that one
// AND-OR yields two tokens' codes of one channel.
//
// Roundings: Q, K, V and P are fp16 (by at most 2^-11 of each value; Q is first scaled by a power of two per row), sums,
// maxima and O are FP32, and the context is bf16 (2^-8), which is the larger error. P is measured against m, 7 below the
// largest score (log2 units) when it is set, and m is moved, and O rescaled in tensor memory, only when a score passes it
// by 15: P reaches from 2^15, as high as fp16 goes, down to its subnormal step, so that no weight is off by more than
// 2^-32 of the largest, or 2^-11 of itself. (Against the largest score itself weights below 2^-25 vanished from O but not
// from the sum: 131071 equal ones under a peak 25 above them were lost.) A row sum of 2^15 * 2^31 tokens stays far inside
// FP32.
//
// What bounds it: per 64 tokens and row tile (D = 128) the two products take 400 + 256 cycles of the tensor core
// (N = 64 reads Q faster than it multiplies) and the exponentials 512 of the 16-per-cycle unit, that is 1312 and 1024
// for the CTA. A row tile has two S buffers, so that the next scores are made while these are weighed: with blocks of
// 128 tokens, whose S and O fill tensor memory, softmax and products of a tile took turns and a 4096-token prompt
// 203 us, when it took 179 as it is (now 163 to 178, by clock and card).
//
// With heads of 256 there is one row tile (128 rows): O takes 256 columns of tensor memory and Q, as A operand of the
// first product, 128, since shared memory holds only two stages of K and V of that width. The second tile's softmax warps
// expand too: three groups of four warps take half blocks of keys and values in turn, 147 against 160 us for 2000
// tokens after 4000 of 16 / 2 heads.
//
// Roles (20 warps): 0-3 and 4-7 softmax and epilogue of the two tiles (thread = row = tensor-memory lane), 8-11
// and 12-15 expansion (of keys and of values), 16 bulk copies of raw tiles, 17 and 18 the tcgen05 issue of a
// tile each (19 completes the warpgroup whose registers go to the softmax). Every wait is bounded.
#include "kv4.cuh"

#include <cmath>

namespace b2 {
namespace {

using namespace sm100;

constexpr uint32_t kBlock = 64;   // tokens of a block
// Rows of a CTA: two tiles of 128; one where heads of 256 fill tensor memory with its O.
__host__ __device__ constexpr uint32_t rows_of(uint32_t d) { return d == 256u ? 128u : 256u; }
constexpr uint32_t kBlockTiles = kBlock / kKv4Tile;
constexpr uint32_t kExpandWarps = 4;   // of a group
constexpr uint32_t kExpandWarp = 8, kLoadWarp = 16, kIssueWarp = 17;   // and 18
constexpr uint32_t kThreads = 20 * 32;
// Registers of a thread by warpgroup, against 96 at the launch (the most that 20 warps of 640 threads can have):
// softmax 2 x 128 x 136 + expansion 2 x 128 x 80 + the last 128 x 48 = 640 x 96, what the launch holds; with three
// warpgroups that expand and one tile's softmax less.
constexpr int kSoftmaxRegisters = 136, kExpandRegisters = 80, kOtherRegisters = 48;
static_assert(256 * kSoftmaxRegisters + 256 * kExpandRegisters + 128 * kOtherRegisters <= 640 * 96, "more than the launch holds");
constexpr uint32_t kRawSlots = 3;
constexpr uint32_t kMostStages = 4;
constexpr uint32_t kTmemColumns = 512, kTmemTile = 256, kTmemO = 128;   // a tile's two S (and P) of 64 columns, its O
constexpr uint32_t kTmemQ = 384;   // heads of 256: Q, for which shared memory has no room, beside the one tile's O
constexpr float kHeadroom = 7.0f;   // log2 of the largest weight when the reference m is set, for the sake of the smallest
constexpr float kSlack = 15.0f;     // P may reach 2^kSlack before m is moved
// From this magnitude of m on (log2 units) a score's rounding counts: the steps of FP32 are 1/8 and more, so that a fused
// product minus a rounded m may be off by powers of two, and m + kSlack by a step. Such rows' scores are rounded first, the
// way their maximum is, and m follows every block's.
constexpr float kFar = 1048576.0f;

template <int D>
struct Layout {
    static constexpr bool kQInTmem = D == 256;
    static constexpr uint32_t kRows = rows_of(D), kStages = D == 256 ? 2 : kMostStages;   // of expanded keys and of values
    // Channels that a group of four warps expands in one go. Heads of 256 have halves, four to a block, which three groups
    // take in turn; the others one group for keys and one for values.
    static constexpr uint32_t kPart = D == 256 ? 128 : D, kHalves = D / kPart;
    static constexpr uint32_t kQ = kQInTmem ? 0u : kRows * D * 2, kKStage = kBlock * D * 2, kVStage = kBlock * D * 2;
    // 16 bytes apart, so that the same word of four tiles lies in different banks
    static constexpr uint32_t kRawTile = kv4_tile_bytes(D) + 16u;
    static constexpr uint32_t kRawSlot = kBlockTiles * kRawTile;
    static constexpr uint32_t kTotal = kQ + kStages * (kKStage + kVStage) + kRawSlots * kRawSlot + (kQInTmem ? 4u * 4096u : 0u) + 1024u;
};

struct Barriers {
    uint64_t raw_full[kRawSlots], raw_empty[kRawSlots];
    uint64_t k_full[kMostStages], k_empty[kMostStages], v_full[kMostStages], v_empty[kMostStages];
    uint64_t s_full[2][2], p_full[2][2];   // [tile][buffer]
    // P V of a block and of the last one. Whoever waits for o_done knows that the one before has completed (the
    // scores it has seen were issued after it), so that a parity tells; at the end only two before that is known.
    uint64_t o_done[2], o_full[2];
    uint64_t q_full[2];   // a tile's rows of Q are staged
    uint64_t pair_full;   // paired: the second tile's maxima and sums are in `pair`
    float2 pair[128];
    uint32_t tmem_base;
    uint32_t abort;
};

struct ChunkPlan {
    uint32_t row_tiles;         // CTAs a sequence's rows may need
    uint32_t paired;            // 1: at most 128 rows, whose blocks the two row tiles take in turn
    uint32_t splits;            // most splits of the blocks of one of them
    uint32_t blocks_per_split;
};

// What a CTA's rows, from `row0` on, of a sequence's n * rep rows see together.
struct TileSpan {
    uint32_t first;          // row of q of the sequence's first new token
    uint32_t tokens;         // new tokens n
    uint32_t rows;           // n * rep
    uint32_t len;
    uint32_t prefix;
    int64_t position0;       // position of new token 0: negative where the chunk is longer than the sequence
    uint32_t begin, end;     // tokens any row sees
    bool bad;
};
__device__ __forceinline__ TileSpan tile_span(const Kv4AttentionArgs& a, uint32_t seq, uint32_t rep, uint32_t row0, uint32_t cta_rows) {
    TileSpan s{};
    const uint32_t first = __ldg(a.chunk_starts + seq), last = __ldg(a.chunk_starts + seq + 1u);
    s.first = min(first, a.rows);
    const uint32_t end_row = min(last, a.rows);
    s.tokens = end_row > s.first ? end_row - s.first : 0u;   // those that the call has rows for
    s.bad = last > first && last - first > a.max_chunk;
    s.tokens = min(s.tokens, a.max_chunk);   // the grid holds max_chunk of them
    s.rows = s.tokens * rep;
    if (row0 >= s.rows) return s;
    s.len = __ldg(a.seq_lens + seq);
    if (s.len > a.max_seq_len) {
        s.len = a.max_seq_len;
        s.bad = true;
    }
    s.position0 = static_cast<int64_t>(s.len) - (last - first);
    s.bad = s.bad || s.position0 < 0;
    s.prefix = a.rules.prefix_lens != nullptr ? min(s.len, __ldg(a.rules.prefix_lens + seq)) : 0u;
    const uint32_t token_lo = row0 / rep, token_hi = min(s.tokens - 1u, (row0 + cta_rows - 1u) / rep);
    const int64_t lowest = max(static_cast<int64_t>(0), s.position0 + token_lo), highest = s.position0 + token_hi;
    if (highest < 0) return s;
    s.end = max(static_cast<uint32_t>(highest) + 1u, s.prefix);
    if (a.rules.window != 0u && lowest >= a.rules.window) s.begin = static_cast<uint32_t>(lowest) - a.rules.window + 1u;
    return s;
}

template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// Named barriers of two warps, one that waits for its turn and one that passes it.
__device__ __forceinline__ void turn_wait(uint32_t barrier, bool first) {
    if (!first) asm volatile("bar.sync %0, 64;" ::"r"(barrier) : "memory");
}
__device__ __forceinline__ void turn_pass(uint32_t barrier) { asm volatile("bar.arrive %0, 64;" ::"r"(barrier) : "memory"); }
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.u32 %0, 1, 0, p; }" : "=r"(pred));
    return pred != 0;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void tmem_st_32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
          "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
          "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// kind::f16, fp16 x fp16 -> FP32, both operands K-major, M = 128.
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((128u >> 4) << 24); }

// scale * code + base of the two codes that nibble N of both halves of `word` holds; the scales and bases
// are those of the two. 1024 + code and 1024 + 16 code are exact, so is taking the 1024 off.
template <int N>
__device__ __forceinline__ uint32_t expand(uint32_t word, __half2 scale, __half2 base, uint32_t k1024) {
    if (N >= 2) word >>= 8;
    __half2 c;
    if (N % 2 == 0) {
        uint32_t x = codes_1024<0x000F000Fu>(word, k1024);
        c = __hadd2(*reinterpret_cast<__half2*>(&x), __half2half2(__ushort_as_half(0xE400)));   // -1024
    } else {
        uint32_t x = codes_1024<0x00F000F0u>(word, k1024);
        c = __hfma2(*reinterpret_cast<__half2*>(&x), __half2half2(__ushort_as_half(0x2C00)),    // 1/16
                    __half2half2(__ushort_as_half(0xD400)));                                     // -64
    }
    c = __hfma2(c, scale, base);
    return *reinterpret_cast<const uint32_t*>(&c);
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
// Nonzero where the scale or the base of a pair is an infinity or a NaN.
__device__ __forceinline__ uint32_t not_finite(uint32_t pair) { return ((pair & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }

// A block of keys: 32 channels of one token per step and thread, rows of the tile in token order. `whole`: every
// one of the tokens is seen by some row.
template <int D>
__device__ __forceinline__ void expand_keys(uint32_t raw32, uint32_t stage32, uint32_t half, uint32_t tid, uint32_t token0, bool whole,
                                            uint32_t begin, uint32_t end, uint32_t k1024) {
    constexpr uint32_t G = D / 64, kSteps = kBlock * (Layout<D>::kPart / 32) / (kExpandWarps * 32u);
    const uint32_t n0 = half * kSteps;
    const uint32_t tk = tid % kBlock;   // lanes: consecutive tokens
    const uint32_t tile32 = raw32 + (tk / 16u) * Layout<D>::kRawTile;
    const uint32_t row32 = stage32 + tk * 128u;
    uint32_t pair[kSteps];
    uint4 raw[kSteps];
#pragma unroll
    for (uint32_t n = 0; n < kSteps; ++n) {   // chunk of 32 channels j = tid / 64 + 2 (n0 + n), group j / 2 = n0 + n
        pair[n] = lds32(tile32 + 8u * D + (tk % 16u) * (4u * G) + (n0 + n) * 4u);
        raw[n] = lds128(tile32 + (tid / kBlock + 2u * (n0 + n)) * 256u + (tk % 16u) * 16u);
    }
    // A value that is not finite must not meet the zero weight of a row that does not see it: its group is
    // expanded as zeros (expand_values), and the token's scores, which such a row masks, become NaN.
    if (half == 0u && tid < kBlock) {
#pragma unroll
        for (uint32_t gr = 0; gr < G; ++gr) {
            if (not_finite(lds32(tile32 + kv4_half_bytes(D) + 8u * D + (tk % 16u) * (4u * G) + gr * 4u))) pair[0] = 0x7FFF7FFFu;
        }
    }
    if (!whole && (token0 + tk < begin || token0 + tk >= end)) {
#pragma unroll
        for (uint32_t n = 0; n < kSteps; ++n) pair[n] = 0u;
    }
#pragma unroll
    for (uint32_t n = 0; n < kSteps; ++n) {
        const __half2 scale = __half2half2(__low2half(as_half2(pair[n]))), base = __half2half2(__high2half(as_half2(pair[n])));
        const uint32_t words[4] = {raw[n].x, raw[n].y, raw[n].z, raw[n].w};
#pragma unroll
        for (uint32_t w = 0; w < 4u; ++w) {
            const uint32_t unit = (tid / kBlock) * 4u + w;
            sts128(row32 + (n0 + n) * (kBlock * 128u) + ((unit ^ (tk & 7u)) << 4), expand<0>(words[w], scale, base, k1024),
                   expand<1>(words[w], scale, base, k1024), expand<2>(words[w], scale, base, k1024), expand<3>(words[w], scale, base, k1024));
        }
    }
}

// A block of values, transposed: eight channels of eight tokens per thread, rows of the tile are channels.
template <int D>
__device__ __forceinline__ void expand_values(uint32_t raw32, uint32_t stage32, uint32_t half, uint32_t tid, uint32_t token0, bool whole,
                                              uint32_t begin, uint32_t end, uint32_t k1024) {
    constexpr uint32_t G = D / 64;
    if (tid >= Layout<D>::kPart) return;
    const uint32_t octet = tid % 8u, word = half * (Layout<D>::kPart / 8u) + tid / 8u;   // tokens 8 octet.., channels 8 word..
    const uint32_t j = word / 4u;
    const uint32_t tile32 = raw32 + (octet / 2u) * Layout<D>::kRawTile + kv4_half_bytes(D);
    const uint32_t slot0 = (octet & 1u) * 8u;
    uint32_t pair[8], code[8];
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e) {
        pair[e] = lds32(tile32 + 8u * D + (slot0 + e) * (4u * G) + (j / 2u) * 4u);
        code[e] = lds32(tile32 + j * 256u + (slot0 + e) * 16u + (word % 4u) * 4u);
    }
    uint32_t bad = whole ? 0u : 1u;
#pragma unroll
    for (uint32_t e = 0; e < 8u; ++e) bad |= not_finite(pair[e]);
    if (bad != 0u) {
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
            const uint32_t token = token0 + octet * 8u + e;
            if (token < begin || token >= end || not_finite(pair[e])) pair[e] = 0u;
        }
    }
    uint32_t scale[4], base[4], lo[4], hi[4];
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k) {
        scale[k] = __byte_perm(pair[2 * k], pair[2 * k + 1], 0x5410);
        base[k] = __byte_perm(pair[2 * k], pair[2 * k + 1], 0x7632);
        lo[k] = __byte_perm(code[2 * k], code[2 * k + 1], 0x5410);   // channels 0..3 of both tokens
        hi[k] = __byte_perm(code[2 * k], code[2 * k + 1], 0x7632);   // channels 4..7
    }
    const uint32_t column32 = stage32 + word * 1024u;
    auto put = [&](uint32_t n, uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3) {
        sts128(column32 + n * 128u + ((octet ^ n) << 4), x0, x1, x2, x3);
    };
#define B2_KV4_PUT(N, SRC)                                                                                    \
    put(N, expand<(N) % 4>(SRC[0], as_half2(scale[0]), as_half2(base[0]), k1024),                                    \
        expand<(N) % 4>(SRC[1], as_half2(scale[1]), as_half2(base[1]), k1024),                                       \
        expand<(N) % 4>(SRC[2], as_half2(scale[2]), as_half2(base[2]), k1024),                                       \
        expand<(N) % 4>(SRC[3], as_half2(scale[3]), as_half2(base[3]), k1024))
    B2_KV4_PUT(0, lo);
    B2_KV4_PUT(1, lo);
    B2_KV4_PUT(2, lo);
    B2_KV4_PUT(3, lo);
    B2_KV4_PUT(4, hi);
    B2_KV4_PUT(5, hi);
    B2_KV4_PUT(6, hi);
    B2_KV4_PUT(7, hi);
#undef B2_KV4_PUT
}

// Two FP32 operations in one instruction.
__device__ __forceinline__ uint64_t two(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void parts(uint64_t r, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Waits for this thread's tensor-memory loads; x is what the last of them wrote, named so that no use of it is
// moved before the wait.
__device__ __forceinline__ void tmem_ld_ready(uint32_t* x) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]),
                   "+r"(x[8]), "+r"(x[9]), "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]),
                   "+r"(x[15]), "+r"(x[16]), "+r"(x[17]), "+r"(x[18]), "+r"(x[19]), "+r"(x[20]), "+r"(x[21]),
                   "+r"(x[22]), "+r"(x[23]), "+r"(x[24]), "+r"(x[25]), "+r"(x[26]), "+r"(x[27]), "+r"(x[28]),
                   "+r"(x[29]), "+r"(x[30]), "+r"(x[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_32(uint32_t taddr, uint32_t* x) { tmem_ld_32x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(x)); }

// cap * tanh(x * f) for 64 values. Up to |y| = 0.6, where capped scores mostly are, y times a polynomial in y^2
// (least-squares fit of tanh y with weights that even out its largest error: 6e-7, for a cap of 50 a thirtieth of what
// rounding the keys to fp16 moves a score); beyond, 1 - 2 / (1 + e^2y). On the exponential unit alone a capped block
// would take three times as long as its matrix products.
__device__ __forceinline__ void cap_scores(uint32_t (&x)[64], float f, float cap) {
    float most = 0.0f;
#pragma unroll
    for (int e = 0; e < 64; e += 2) {
        most = fmaxf(most, fmaxf(fabsf(__uint_as_float(x[e])), fabsf(__uint_as_float(x[e + 1]))));
    }
    if (__any_sync(0xFFFFFFFFu, !(most * f <= 0.6f))) {
#pragma unroll
        for (int e = 0; e < 64; ++e) {
            const float y = ex2(__uint_as_float(x[e]) * (f * (2.0f * kLog2e)));
            x[e] = __float_as_uint(fmaf(-2.0f * cap, rcp(1.0f + y), cap));
        }
        return;
    }
    const uint64_t f2 = two(f, f);
    const float c[4] = {0.9999909996986389f * cap, -0.33298975229263306f * cap, 0.1297455132007599f * cap,
                        -0.03961123898625374f * cap};
#pragma unroll
    for (int e = 0; e < 64; e += 2) {
        const uint64_t y = mul2(two(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f2), z = mul2(y, y);
        uint64_t r = two(c[3], c[3]);
#pragma unroll
        for (int k = 2; k >= 0; --k) r = fma2(r, z, two(c[k], c[k]));
        float lo, hi;
        parts(mul2(r, y), lo, hi);
        x[e] = __float_as_uint(lo);
        x[e + 1] = __float_as_uint(hi);
    }
}

// The softmax loop's speed hangs on what else the kernel holds, so forms that a launch can tell apart are kernels of their
// own. PAIRED (see below): in one kernel what joins the tiles made a prompt a tenth slower (191 us against 171 before
// and 166 apart). RULES: score caps or distance biases; without their code drafted tokens take 33 instead of 35 us and
// heads of 256 36 instead of 39. Unpaired tiles of smaller heads have the one form with it: that loop, as compiled, is the
// faster one for plain scores too (163 us; without that code 182, or 173 with no turns).
template <int D, bool PAIRED, bool RULES>
__global__ void __launch_bounds__(kThreads, 1)
kv4_chunk_kernel(const Kv4AttentionArgs a, float* __restrict__ partials, const ChunkPlan plan) {
    using L = Layout<D>;
    constexpr uint32_t kRows = L::kRows, kStages = L::kStages;
    constexpr uint32_t kChannels8 = D / 8;
    pdl_launch_dependents();
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) Barriers bars;

    const uint32_t starts_flag = chunk_starts_flag(a);
    const uint32_t rep = a.q_heads / a.cache.kv_heads;
    uint32_t block = blockIdx.x;
    const uint32_t split = block % plan.splits;
    block /= plan.splits;
    const uint32_t kvh = block % a.cache.kv_heads;
    block /= a.cache.kv_heads;
    const uint32_t seq = block % a.cache.n_seq;
    // the last rows see the most tokens: they start first
    const uint32_t row0 = (plan.row_tiles - 1u - block / a.cache.n_seq) * kRows;
    const TileSpan span = tile_span(a, seq, rep, row0, kRows);
    if (row0 >= span.rows) {
        if (starts_flag != 0u) kv4_flag(a.status, starts_flag);
        return;
    }
    const uint32_t rows = min(kRows, span.rows - row0);
    const uint32_t tile0 = span.begin / kKv4Tile;
    const uint32_t tiles = span.end > span.begin ? (span.end - 1u) / kKv4Tile + 1u - tile0 : 0u;
    const uint32_t blocks = (tiles + kBlockTiles - 1u) / kBlockTiles;
    const uint32_t n_splits = max(1u, (blocks + plan.blocks_per_split - 1u) / plan.blocks_per_split);
    if (split >= n_splits) return;
    const uint32_t block0 = split * plan.blocks_per_split;
    const uint32_t n_blocks = min(plan.blocks_per_split, blocks - block0);   // 0 where nothing is seen
    const uint32_t first_tile = tile0 + block0 * kBlockTiles;
    const uint32_t end_tile = min(tile0 + tiles, first_tile + n_blocks * kBlockTiles);
    // Row tiles at work. Paired, both hold the same rows, tile i of them blocks i, i + 2, ..., joined at the end: a tile's
    // chain of products and softmax is twice as long as its share of either unit, and with one tile nothing else
    // would run beside it.
    constexpr bool paired = PAIRED;
    constexpr uint32_t step = paired ? 2u : 1u;
    const uint32_t n_tiles = paired || rows > 128u ? 2u : 1u;

    const uint32_t smem32 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q32 = smem32, k32 = q32 + L::kQ, v32 = k32 + kStages * L::kKStage, raw32 = v32 + kStages * L::kVStage;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    volatile uint32_t* abort = &bars.abort;
    uint32_t flags = span.bad ? B2_ATTN_STATUS_BAD_BLOCK : starts_flag;

    if (warp == kIssueWarp) {
        if (lane == 0) {
            for (uint32_t i = 0; i < kRawSlots; ++i) {
                mbar_init(&bars.raw_full[i], 1);
                mbar_init(&bars.raw_empty[i], 2u * L::kHalves * kExpandWarps);
            }
            for (uint32_t i = 0; i < kStages; ++i) {
                mbar_init(&bars.k_full[i], L::kHalves * kExpandWarps);
                mbar_init(&bars.v_full[i], L::kHalves * kExpandWarps);
                mbar_init(&bars.k_empty[i], paired ? 1u : n_tiles);
                mbar_init(&bars.v_empty[i], paired ? 1u : n_tiles);
            }
            for (uint32_t i = 0; i < 2u; ++i) {
                for (uint32_t b = 0; b < 2u; ++b) {
                    mbar_init(&bars.s_full[i][b], 1);
                    mbar_init(&bars.p_full[i][b], 4);
                }
                mbar_init(&bars.o_done[i], 1);
                mbar_init(&bars.o_full[i], 1);
                mbar_init(&bars.q_full[i], 4);
            }
            mbar_init(&bars.pair_full, 4);
            bars.abort = 0;
            mbar_fence_init();
        }
        if (L::kQInTmem) {
            __syncwarp();
            tmem_alloc(&bars.tmem_base, kTmemColumns);
            tcgen05_fence_before_sync();
        }
    }
    __syncthreads();
    if (L::kQInTmem) tcgen05_fence_after_sync();

    // (a warpgroup's four warps take its registers with one instruction, ahead of their own branches)
    if (warp >= kLoadWarp) {
        registers_down<kOtherRegisters>();
        if (warp == kLoadWarp) {
            // ---- raw tiles ----
            const uint32_t* table = a.cache.block_tables + static_cast<uint64_t>(seq) * a.cache.max_blocks;
            uint64_t offset = 0;
            for (uint32_t jb = 0; jb < n_blocks; ++jb) {
                const uint32_t first = first_tile + jb * kBlockTiles;
                if (jb % 8u == 0u) {   // one lane for each of the next 32 tiles
                    const uint32_t tile = first + lane;
                    if (tile < end_tile) {
                        uint64_t phys = __ldg(table + tile / a.cache.tiles_per_block);
                        if (phys >= a.cache.physical_blocks) {
                            phys = 0;
                            flags |= B2_ATTN_STATUS_BAD_BLOCK;
                        }
                        offset = kv4_tile_offset(a.cache, phys, kvh, tile % a.cache.tiles_per_block);
                    }
                }
                const uint32_t slot = jb % kRawSlots;
                if (jb >= kRawSlots) mbar_wait(&bars.raw_empty[slot], (jb / kRawSlots - 1u) & 1u, abort);
                const uint32_t live = min(kBlockTiles, end_tile - first);
                if (lane == 0) mbar_expect_tx(&bars.raw_full[slot], live * kv4_tile_bytes(D));
                __syncwarp();
                const uint32_t mine = lane - (jb % 8u) * kBlockTiles;   // wraps for lanes of other blocks
                if (mine < live) {
                    fence_proxy_async_smem();
                    bulk_load(raw32 + slot * L::kRawSlot + mine * L::kRawTile, a.cache.pages + offset, kv4_tile_bytes(D),
                              &bars.raw_full[slot]);
                }
                __syncwarp();
            }
        } else if (warp - kIssueWarp < n_tiles) {
            // ---- tcgen05 issue: round n makes the scores of a tile's n-th block, then P V of the one before ----
            // One warp for each tile: an issued MMA is hardly queued, so that what one warp spends on its barriers (75
            // cycles a wait) would leave the tensor core idle, were it not for the other's MMAs. Tensor memory starts at
            // column 0, this CTA holds all of it.
            const uint32_t i = warp - kIssueWarp;
            if (i == 0u && !L::kQInTmem) tmem_alloc(&bars.tmem_base, kTmemColumns);
            // the other tile's warp must not be ahead of the allocation
            asm volatile("bar.sync 1, %0;" ::"r"(n_tiles * 32u) : "memory");
            tcgen05_fence_after_sync();
            mbar_wait(&bars.q_full[i], 0u, abort);
            tcgen05_fence_after_sync();
            const uint64_t dq = umma_desc_k_major_sw128(q32 + i * (128u * D * 2u));
            const uint64_t dk = umma_desc_k_major_sw128(k32), dv = umma_desc_k_major_sw128(v32);
            const uint32_t first_block = paired ? i : 0u;
            const uint32_t mine = n_blocks > first_block ? (n_blocks - first_block + step - 1u) / step : 0u;   // its blocks
            for (uint32_t n = 0; n <= mine && mine != 0u; ++n) {
                if (n < mine) {
                    const uint32_t jb = first_block + n * step, stage = jb % kStages;
                    mbar_wait(&bars.k_full[stage], (jb / kStages) & 1u, abort);
                    tcgen05_fence_after_sync();
                    const uint64_t kb = dk + (stage * L::kKStage >> 4);
                    const uint32_t d = i * kTmemTile + (n & 1u) * kBlock;   // its P was read by P V two of its blocks ago
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t kk = 0; kk < D / 16u; ++kk) {
                            const uint64_t b = kb + (kk / 4u) * (kBlock * 128u >> 4) + (kk % 4u) * 2u;
                            if (L::kQInTmem) {
                                umma_ts(d, kTmemQ + kk * 8u, b, idesc_f16(kBlock), kk != 0u ? 1u : 0u);
                            } else {
                                umma_ss(d, dq + (kk / 4u) * (16384u >> 4) + (kk % 4u) * 2u, b, idesc_f16(kBlock), kk != 0u ? 1u : 0u);
                            }
                        }
                        umma_commit(&bars.s_full[i][n & 1u]);
                        umma_commit(&bars.k_empty[stage]);
                    }
                    __syncwarp();
                }
                if (n > 0u) {
                    const uint32_t before = n - 1u, jb = first_block + before * step, stage = jb % kStages;
                    mbar_wait(&bars.v_full[stage], (jb / kStages) & 1u, abort);
                    mbar_wait(&bars.p_full[i][before & 1u], (before / 2u) & 1u, abort);
                    tcgen05_fence_after_sync();
                    const uint64_t b = dv + (stage * L::kVStage >> 4);
                    const uint32_t w = i * kTmemTile + (before & 1u) * kBlock;
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t kk = 0; kk < kBlock / 16u; ++kk) {
                            umma_ts(i * kTmemTile + kTmemO, w + kk * 8u, b + kk * 2u, idesc_f16(D), kk != 0u ? 1u : before);
                        }
                        umma_commit(n == mine ? &bars.o_full[i] : &bars.o_done[i]);
                        umma_commit(&bars.v_empty[stage]);
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp >= kExpandWarp || (L::kQInTmem && warp >= 4u)) {
        // ---- expansion: part `part` of a block, its keys' (or their halves) before its values' ----
        registers_down<kExpandRegisters>();
        const uint32_t k1024 = opaque_1024();
        constexpr uint32_t kParts = 2u * L::kHalves, kGroups = L::kQInTmem ? 3u : 2u;
        const uint32_t group = warp >= kExpandWarp ? (warp - kExpandWarp) / kExpandWarps : 2u, et = tid % (kExpandWarps * 32u);
        for (uint32_t part = group, jb = 0; jb < n_blocks;) {
            const bool keys = part < L::kHalves;
            const uint32_t half = part % L::kHalves;
            const uint32_t stage = jb % kStages, use = jb / kStages, slot = jb % kRawSlots;
            const uint32_t token0 = (first_tile + jb * kBlockTiles) * kKv4Tile;
            const bool whole = token0 >= span.begin && token0 + kBlock <= span.end;
            if (use > 0) mbar_wait(keys ? &bars.k_empty[stage] : &bars.v_empty[stage], (use - 1u) & 1u, abort);
            mbar_wait(&bars.raw_full[slot], (jb / kRawSlots) & 1u, abort);
            if (keys) {
                expand_keys<D>(raw32 + slot * L::kRawSlot, k32 + stage * L::kKStage, half, et, token0, whole, span.begin, span.end, k1024);
            } else {
                expand_values<D>(raw32 + slot * L::kRawSlot, v32 + stage * L::kVStage, half, et, token0, whole, span.begin, span.end, k1024);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&bars.raw_empty[slot]);
                mbar_arrive(keys ? &bars.k_full[stage] : &bars.v_full[stage]);
            }
            part += kGroups;
            if (part >= kParts) {
                part -= kParts;
                ++jb;
            }
        }
    } else if (warp / 4u < n_tiles) {
        // ---- softmax: a thread is a row ----
        registers_up<kSoftmaxRegisters>();
        const uint32_t i = warp / 4u;
        const uint32_t tile_rows = paired ? 0u : i * 128u;   // rows before the tile's
        const uint32_t r = tile_rows + (warp % 4u) * 32u + lane, gr = row0 + r;
        const bool live = r < rows;
        const uint32_t lane_base = i * kTmemTile + (((warp % 4u) * 32u) << 16);
        const int64_t position64 = span.position0 + gr / rep;
        uint32_t position = 0, begin = 0, end = 0;
        if (live && position64 >= 0) {
            position = static_cast<uint32_t>(position64);
            end = max(position + 1u, span.prefix);
            if (a.rules.window != 0u && position >= a.rules.window) begin = position - a.rules.window + 1u;
        }
        // every row of the warp sees tokens [all_begin, all_end); rows that are not live do not count
        const uint32_t all_begin = __reduce_max_sync(0xFFFFFFFFu, live ? begin : 0u);
        const uint32_t all_end = __reduce_min_sync(0xFFFFFFFFu, live ? end : 0xFFFFFFFFu);
        const bool capped = RULES && a.rules.softcap != 0.0f, biased = RULES && a.rules.alibi_slopes != nullptr;
        const float cap_log2 = a.rules.softcap * kLog2e;
        const float slope = biased && live ? __ldg(a.rules.alibi_slopes + kvh * rep + gr % rep) * kLog2e : 0.0f;
        // Q: scaled to a largest magnitude in [2^9, 2^10) per row, fp16, in the order the codes come out. A warp stages
        // its own 32 rows, four lanes a row, so that two exchanges find a row's largest.
        const float to_unit = (capped ? 1.0f / a.rules.softcap : kLog2e) / sqrtf(static_cast<float>(D));
        constexpr uint32_t kRowsAtOnce = 32u / kChannels8, kSteps = 32u / kRowsAtOnce;
        const uint32_t warp_row = tile_rows + (warp % 4u) * 32u, c8 = lane % kChannels8;
        const uint32_t my_out = static_cast<uint32_t>(gr / rep), my_head = gr % rep;
        float row_factor = 0.0f;
        // 2^e with a row's largest magnitude * 2^e in [2^9, 2^10), and what takes a product back
        auto row_scale = [&](float top, float* up, float* down) {
            int e = 9 - (static_cast<int>((__float_as_uint(top) >> 23) & 255u) - 127);
            e = min(100, e);   // a row of zeros keeps a bounded factor; the largest rows have e = -119, still a normal 2^e
            *up = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
            *down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23) * to_unit;
        };
        if constexpr (L::kQInTmem) {
            // Into each row's lane of tensor memory, by way of shared memory, 64 channels of the warp's rows at a time: a
            // thread that read its own row would take 16 bytes of 32 different ones. First the rows' largest magnitudes.
            float my_up = 0.0f;
#pragma unroll 1
            for (uint32_t n0 = 0; n0 < 32u; n0 += 8u) {
                float top8[8];
#pragma unroll
                for (uint32_t n = 0; n < 8u; ++n) {
                    const uint32_t token = __shfl_sync(0xFFFFFFFFu, my_out, n0 + n), head = __shfl_sync(0xFFFFFFFFu, my_head, n0 + n);
                    float4 u0 = make_float4(0.f, 0.f, 0.f, 0.f), u1 = u0;
                    if (warp_row + n0 + n < rows) {
                        const float* src = a.q + (static_cast<uint64_t>(span.first + token) * a.q_heads + kvh * rep + head) * D + lane * 8u;
                        u0 = __ldg(reinterpret_cast<const float4*>(src));
                        u1 = __ldg(reinterpret_cast<const float4*>(src) + 1);
                    }
                    top8[n] = fmaxf(fmaxf(fmaxf(fabsf(u0.x), fabsf(u0.y)), fmaxf(fabsf(u0.z), fabsf(u0.w))),
                                    fmaxf(fmaxf(fabsf(u1.x), fabsf(u1.y)), fmaxf(fabsf(u1.z), fabsf(u1.w))));
                }
#pragma unroll
                for (uint32_t n = 0; n < 8u; ++n) {
                    const float top = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top8[n])));   // not negative
                    float up, down;
                    row_scale(top, &up, &down);
                    if (lane == n0 + n) {
                        my_up = up;
                        row_factor = down;
                    }
                }
            }
            const uint32_t turn32 = raw32 + kRawSlots * L::kRawSlot + (warp % 4u) * 4096u;
#pragma unroll 1
            for (uint32_t c = 0; c < D / 64u; ++c) {
#pragma unroll
                for (uint32_t n = 0; n < 8u; ++n) {   // eight lanes a row
                    const uint32_t which = n * 4u + lane / 8u;
                    const uint32_t token = __shfl_sync(0xFFFFFFFFu, my_out, which), head = __shfl_sync(0xFFFFFFFFu, my_head, which);
                    const float up = __shfl_sync(0xFFFFFFFFu, my_up, which);
                    float4 u0 = make_float4(0.f, 0.f, 0.f, 0.f), u1 = u0;
                    if (warp_row + which < rows) {
                        const float* src = a.q + (static_cast<uint64_t>(span.first + token) * a.q_heads + kvh * rep + head) * D + c * 64u + lane % 8u * 8u;
                        u0 = __ldg(reinterpret_cast<const float4*>(src));
                        u1 = __ldg(reinterpret_cast<const float4*>(src) + 1);
                    }
                    sts128(turn32 + which * 128u + (((lane % 8u) ^ (which & 7u)) << 4), pack_half(u0.x * up, u1.x * up),
                           pack_half(u0.y * up, u1.y * up), pack_half(u0.z * up, u1.z * up), pack_half(u0.w * up, u1.w * up));
                }
                __syncwarp();
                uint32_t w[32];
#pragma unroll
                for (uint32_t n = 0; n < 8u; ++n) {
                    const uint4 v = lds128(turn32 + lane * 128u + ((n ^ (lane & 7u)) << 4));
                    w[4 * n] = v.x; w[4 * n + 1] = v.y; w[4 * n + 2] = v.z; w[4 * n + 3] = v.w;
                }
                tmem_st_32(lane_base + kTmemQ + c * 32u, w);
                __syncwarp();
            }
            tmem_st_wait();
            tcgen05_fence_before_sync();
        }
        constexpr uint32_t kUnits = L::kQInTmem ? 1u : D / 32u;   // of eight channels, of a lane
        constexpr uint32_t kAtOnce = L::kQInTmem ? 1u : 8u / kUnits;   // times eight rows: 64 registers of loads
#pragma unroll 1
        for (uint32_t n0 = 0; n0 < 4u && !L::kQInTmem; n0 += kAtOnce) {
            float y[kAtOnce][kUnits][8];
#pragma unroll
            for (uint32_t n = 0; n < kAtOnce; ++n) {
                const uint32_t mine = (n0 + n) * 8u + lane / 4u;   // of the warp's 32 rows
                const uint32_t token = __shfl_sync(0xFFFFFFFFu, my_out, mine), head = __shfl_sync(0xFFFFFFFFu, my_head, mine);
                const float* src = a.q + (static_cast<uint64_t>(span.first + token) * a.q_heads + kvh * rep + head) * D + lane % 4u * 8u;
#pragma unroll
                for (uint32_t u = 0; u < kUnits; ++u) {
                    float4 u0 = make_float4(0.f, 0.f, 0.f, 0.f), u1 = u0;
                    if (warp_row + mine < rows) {
                        u0 = __ldg(reinterpret_cast<const float4*>(src + u * 32u));
                        u1 = __ldg(reinterpret_cast<const float4*>(src + u * 32u) + 1);
                    }
                    y[n][u][0] = u0.x; y[n][u][1] = u0.y; y[n][u][2] = u0.z; y[n][u][3] = u0.w;
                    y[n][u][4] = u1.x; y[n][u][5] = u1.y; y[n][u][6] = u1.z; y[n][u][7] = u1.w;
                }
            }
#pragma unroll
            for (uint32_t n = 0; n < kAtOnce; ++n) {
                float top = 0.0f, up, down;
#pragma unroll
                for (uint32_t u = 0; u < kUnits; ++u)
#pragma unroll
                    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[n][u][e]));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                row_scale(top, &up, &down);
                const float f = __shfl_sync(0xFFFFFFFFu, down, lane % 8u * 4u);   // to the lane whose row it is
                if (lane / 8u == n0 + n) row_factor = f;
                const uint32_t tile_row = (warp % 4u) * 32u + (n0 + n) * 8u + lane / 4u;
                const uint32_t dst = q32 + i * (128u * D * 2u) + tile_row * 128u;
#pragma unroll
                for (uint32_t u = 0; u < kUnits; ++u) {
                    const uint32_t unit = u * 4u + lane % 4u;
                    const float(&z)[8] = y[n][u];
                    sts128(dst + (unit / 8u) * 16384u + (((unit % 8u) ^ (tile_row & 7u)) << 4), pack_half(z[0] * up, z[4] * up),
                           pack_half(z[1] * up, z[5] * up), pack_half(z[2] * up, z[6] * up), pack_half(z[3] * up, z[7] * up));
                }
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_full[i]);
        float m = kNoMax, l = 0.0f;
        float limit = kNoMax;   // largest score for which m stays: m + kSlack, or none

        const uint32_t first_block = paired ? i : 0u;
        const uint32_t mine = n_blocks > first_block ? (n_blocks - first_block + step - 1u) / step : 0u;   // the tile's blocks
        const bool turns = !PAIRED && n_tiles == 2u;
        for (uint32_t n = 0; n < mine; ++n) {
            const uint32_t token0 = (first_tile + (first_block + n * step) * kBlockTiles) * kKv4Tile;
            const uint32_t buffer = lane_base + (n & 1u) * kBlock;
            mbar_wait(&bars.s_full[i][n & 1u], (n / 2u) & 1u, abort);
            tcgen05_fence_after_sync();
            const bool masked = token0 < all_begin || token0 + kBlock > all_end;   // the same for the whole warp
            uint32_t x[64];
            tmem_ld_32(buffer, x);
            tmem_ld_32(buffer + 32u, x + 32);
            tmem_ld_ready(x);
            tmem_ld_ready(x + 32);
            float factor = row_factor;
            if (capped || biased) {   // scores in log2 units instead of raw products
                factor = 1.0f;
                if (capped) {
                    cap_scores(x, row_factor, cap_log2);
                } else {
#pragma unroll
                    for (int e = 0; e < 64; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * row_factor);
                }
                if (biased) {
                    const float away0 = static_cast<float>(static_cast<int>(position - token0));
#pragma unroll
                    for (int e = 0; e < 64; ++e) {
                        x[e] = __float_as_uint(fmaf(-slope, fabsf(away0 - static_cast<float>(e)), __uint_as_float(x[e])));
                    }
                }
            }
            if (masked) {
#pragma unroll
                for (int e = 0; e < 64; ++e) {
                    if (token0 + e < begin || token0 + e >= end) x[e] = 0xFF800000u;   // -infinity
                }
            }
            // The weights are made against the reference so far, while the block's maximum is found; where it passes that
            // by more than kSlack (the first block, hardly ever later) they are made again.
            uint32_t p[32];
            float sum, top;
            auto weigh = [&]() {
                const uint64_t factor2 = two(factor, factor), minus_m = two(-m, -m);
                uint64_t sums[2] = {0ull, 0ull};
                float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 64; e += 2) {
                    float a0, a1;
                    parts(fma2(two(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), factor2, minus_m), a0, a1);
                    a0 = ex2(a0);
                    a1 = ex2(a1);
                    top4[(e / 2) & 3] = fmaxf(fmaxf(top4[(e / 2) & 3], __uint_as_float(x[e])), __uint_as_float(x[e + 1]));
                    sums[(e / 2) & 1] = add2(sums[(e / 2) & 1], two(a0, a1));
                    p[e / 2] = pack_half(a0, a1);
                }
                float s0, s1;
                parts(add2(sums[0], sums[1]), s0, s1);
                sum = s0 + s1;
                top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * factor;
            };
            // The warps of the two tiles that share a scheduler take turns with their exponentials, so that one's run under
            // the other's loads and stores instead of both at half speed (four capped chunks of 300 to 700 tokens 118 us, 124
            // without; tiles of the same rows, whose blocks come in turn anyway, lose 1 of 40 to it).
            if (turns) turn_wait(2u + (warp % 4u) * 2u + i, i == 0u && n == 0u);
            weigh();
            if (turns && (i == 0u || n + 1u < mine)) turn_pass(2u + (warp % 4u) * 2u + (i ^ 1u));
            if (__any_sync(0xFFFFFFFFu, top > limit)) {
                const float moved = fmaxf(m, top - kHeadroom);
                const float shrink = ex2(m - moved);
                m = moved;
                l *= shrink;
                const bool far = m != kNoMax && fabsf(m) > kFar;
                limit = far ? -INFINITY : m + kSlack;
                if (__any_sync(0xFFFFFFFFu, far)) {
#pragma unroll
                    for (int e = 0; e < 64; ++e) x[e] = __float_as_uint(__fmul_rn(__uint_as_float(x[e]), factor));
                    factor = 1.0f;
                }
                if (n > 0u) {
                    mbar_wait(&bars.o_done[i], (n - 1u) & 1u, abort);   // P V of the block before: O is at rest
                    tcgen05_fence_after_sync();
#pragma unroll 1
                    for (uint32_t c = 0; c < D / 32u; ++c) {
                        tmem_ld_32(lane_base + kTmemO + c * 32u, p);
                        tmem_ld_ready(p);
#pragma unroll
                        for (int e = 0; e < 32; ++e) p[e] = __float_as_uint(__uint_as_float(p[e]) * shrink);
                        tmem_st_32(lane_base + kTmemO + c * 32u, p);
                    }
                }
                weigh();
            }
            l += sum;
            tmem_st_32(buffer, p);
            tmem_st_wait();
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_full[i][n & 1u]);
        }

        // ---- epilogue ----
        if (live && isnan(l)) flags |= B2_ATTN_STATUS_NAN_OR_POS_INF;
        if (paired && i == 1u) {   // the first tile's warps join both: they reach the same lanes of tensor memory
            bars.pair[r] = make_float2(m, l);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.pair_full);
        } else {
            const bool both = paired && n_blocks > 1u;   // the second tile had blocks
            float keep = 1.0f, other = 0.0f;             // factors of the tiles' sums
            if (mine != 0u) {
                mbar_wait(&bars.o_full[i], 0u, abort);
                if (both) {
                    mbar_wait(&bars.o_full[1], 0u, abort);
                    mbar_wait(&bars.pair_full, 0u, abort);
                    const float2 its = bars.pair[r];
                    const float top = fmaxf(m, its.x);
                    keep = ex2(m - top);
                    other = ex2(its.x - top);
                    m = top;
                    l = l * keep + its.y * other;
                }
                tcgen05_fence_after_sync();
            } else {
                mbar_wait(&bars.q_full[i], 0u, abort);   // the other warps' staging, which the rows below are written over
            }
            if (lane == 0 && *abort != 0) flags |= B2_ATTN_STATUS_TIMEOUT;
            const uint64_t out_head = static_cast<uint64_t>(span.first + my_out) * a.q_heads + kvh * rep + my_head;
            const bool whole = n_splits == 1u;
            if (whole && live && l == 0.0f && end > begin) flags |= B2_ATTN_STATUS_ALL_NEG_INF;
            float* part = partials + (out_head * plan.splits + split) * (D + 4u);
            if (!whole && live) *reinterpret_cast<float2*>(part) = make_float2(m, l);
            const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
            keep *= inv;
            other *= inv;
            // The tile's Q (heads of 256: the keys' stages) is not needed any more: 2 D bytes a row take the warp's bf16 rows, so
            // that they leave in whole rows instead of 16 bytes of 32 different ones.
            static_assert(L::kQ + kStages * L::kKStage >= kRows * D * 2u, "room for the rows");
            const uint32_t stage32 = q32 + i * (128u * D * 2u) + (warp % 4u) * (32u * D * 2u);
#pragma unroll 1
            for (uint32_t c = 0; c < D / 32u; ++c) {
                uint32_t o[32];
                if (mine != 0u) {
                    tmem_ld_32(lane_base + kTmemO + c * 32u, o);
                    tmem_ld_ready(o);
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = l == 0.0f ? 0u : __float_as_uint(__uint_as_float(o[e]) * keep);
                if (both) {
                    uint32_t its[32];
                    tmem_ld_32(lane_base + kTmemTile + kTmemO + c * 32u, its);
                    tmem_ld_ready(its);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        o[e] = l == 0.0f ? 0u : __float_as_uint(fmaf(__uint_as_float(its[e]), other, __uint_as_float(o[e])));
                    }
                }
                if (whole) {
#pragma unroll
                    for (uint32_t e = 0; e < 4u; ++e) {
                        uint32_t w[4];
#pragma unroll
                        for (uint32_t k = 0; k < 4u; ++k) {
                            const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(o[8 * e + 2 * k]), __uint_as_float(o[8 * e + 2 * k + 1]));
                            w[k] = *reinterpret_cast<const uint32_t*>(&b);
                        }
                        sts128(stage32 + lane * (D * 2u) + (((c * 4u + e) ^ (lane & 7u)) << 4), w[0], w[1], w[2], w[3]);
                    }
                } else if (live) {
                    float4* dst = reinterpret_cast<float4*>(part + 4u + c * 32u);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        dst[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                                             __uint_as_float(o[4 * e + 3]));
                    }
                }
            }
            if (whole) {
                __syncwarp();
#pragma unroll 4
                for (uint32_t n = 0; n < kSteps; ++n) {
                    const uint32_t which = n * kRowsAtOnce + lane / kChannels8;
                    const uint64_t head = __shfl_sync(0xFFFFFFFFu, out_head, which);
                    const uint4 v = lds128(stage32 + which * (D * 2u) + ((c8 ^ (which & 7u)) << 4));
                    if (warp_row + which < rows) {
                        reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.ctx16) + head * D)[c8] = v;
                    }
                }
            }
        }
    }
    if (flags != 0u) kv4_flag(a.status, flags);
    tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == kIssueWarp) tmem_dealloc(bars.tmem_base, kTmemColumns);
}

// Joins the splits of every (row, query head) that has more than one.
template <int D>
__global__ void __launch_bounds__(D / 4)
kv4_chunk_merge_kernel(const Kv4AttentionArgs a, const float* __restrict__ partials, const ChunkPlan plan) {
    pdl_launch_dependents();
    const uint64_t out_head = blockIdx.x;
    const uint32_t row = static_cast<uint32_t>(out_head / a.q_heads), rep = a.q_heads / a.cache.kv_heads;
    const uint32_t head = static_cast<uint32_t>(out_head % a.q_heads) % rep;
    const RowSpan mine = row_span(a, row);   // inputs of the call, not of the kernel before
    uint32_t n_splits = 0;
    bool ours = false;
    if (mine.owned) {
        const uint32_t first = min(__ldg(a.chunk_starts + mine.seq), a.rows);
        const TileSpan span = tile_span(a, mine.seq, rep, ((row - first) * rep + head) / rows_of(D) * rows_of(D), rows_of(D));
        ours = row - first < span.tokens;
        if (ours) {
            const uint32_t tile0 = span.begin / kKv4Tile;
            const uint32_t tiles = span.end > span.begin ? (span.end - 1u) / kKv4Tile + 1u - tile0 : 0u;
            n_splits = ((tiles + kBlockTiles - 1u) / kBlockTiles + plan.blocks_per_split - 1u) / plan.blocks_per_split;
        }
    }
    pdl_wait();   // every CTA waits, so that this grid never ends before the one it follows
    if (!ours || n_splits <= 1u) return;
    const float* first = partials + out_head * plan.splits * (D + 4u);
    const uint32_t c = threadIdx.x * 4u;
    finish<D>(a, join_run(first, first + (D + 4u), D + 4u, n_splits, c), out_head, c, mine.end > mine.begin);
}

// One CTA holds an SM. Where the row tiles are fewer than the SMs, the blocks of each are split over as many CTAs as
// make the waves shortest: a CTA's set-up and epilogue take about as long as six blocks, joining as four. With more row
// tiles the longer ones start first and the shorter ones fill in; splitting those too made four chunks of 300 to 700
// tokens, 192 CTAs, slower (132 against 166 us: the FP32 partial results of so many rows).
ChunkPlan chunk_plan(int sm_count, uint32_t n_seq, uint32_t q_heads, uint32_t kv_heads, uint32_t head_width, uint32_t max_chunk, uint32_t max_tokens) {
    const uint64_t rep = q_heads / kv_heads;
    const uint64_t sms = sm_count > 0 ? static_cast<uint64_t>(sm_count) : 148u;
    const uint64_t row_tiles = (max_chunk * rep + rows_of(head_width) - 1u) / rows_of(head_width);
    const uint64_t blocks = (static_cast<uint64_t>(max_tokens) + kBlock - 1u) / kBlock + 1u;   // a window may start inside a tile
    const uint64_t ctas = row_tiles * n_seq * kv_heads;
    uint64_t best = 1;
    if (ctas < sms) {
        uint64_t shortest = UINT64_MAX;
        for (uint64_t splits = 1; splits <= 64u && (splits == 1u || blocks >= 4u * splits); ++splits) {
            const uint64_t waves = (ctas * splits + sms - 1u) / sms;
            const uint64_t time = waves * ((blocks + splits - 1u) / splits + 6u) + (splits > 1u ? 4u : 0u);
            if (time < shortest) {
                shortest = time;
                best = splits;
            }
        }
    }
    const uint64_t per = (blocks + best - 1u) / best;
    return ChunkPlan{static_cast<uint32_t>(row_tiles), rows_of(head_width) == 256u && max_chunk * rep <= 128u ? 1u : 0u,
                     static_cast<uint32_t>((blocks + per - 1u) / per), static_cast<uint32_t>(per)};
}

template <int D, bool PAIRED, bool RULES>
int32_t launch_one(const DeviceContext& ctx, const Kv4AttentionArgs& a, float* partials, const ChunkPlan& plan,
                   cudaStream_t stream) {
    static PerDeviceOnce configured;
    B2_TRY(once_per_device(configured, ctx.device, []() -> int32_t {
        B2_CUDA_TRY(cudaFuncSetAttribute(kv4_chunk_kernel<D, PAIRED, RULES>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kTotal));
        return B2_STATUS_OK;
    }));
    const uint64_t ctas = static_cast<uint64_t>(plan.row_tiles) * a.cache.n_seq * a.cache.kv_heads * plan.splits;
    const uint64_t merges = static_cast<uint64_t>(a.rows) * a.q_heads;
    if (ctas > 0x7FFFFFFFull || merges > 0x7FFFFFFFull) return fail(B2_STATUS_OVERFLOW, "paged attention batch too large");
    kv4_chunk_kernel<D, PAIRED, RULES><<<static_cast<unsigned>(ctas), kThreads, Layout<D>::kTotal, stream>>>(a, partials, plan);
    B2_CUDA_TRY(cudaGetLastError());
    if (plan.splits <= 1u) return B2_STATUS_OK;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(merges));
    config.blockDim = dim3(D / 4);
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    B2_CUDA_TRY(cudaLaunchKernelEx(&config, kv4_chunk_merge_kernel<D>, a, const_cast<const float*>(partials), plan));
    return B2_STATUS_OK;
}

template <int D>
int32_t launch_form(const DeviceContext& ctx, const Kv4AttentionArgs& a, float* partials, const ChunkPlan& plan, cudaStream_t stream) {
    const bool rules = a.rules.softcap != 0.0f || a.rules.alibi_slopes != nullptr;
    if constexpr (D == 256) {
        return rules ? launch_one<D, false, true>(ctx, a, partials, plan, stream) : launch_one<D, false, false>(ctx, a, partials, plan, stream);
    } else {
        if (plan.paired == 0u) return launch_one<D, false, true>(ctx, a, partials, plan, stream);
        return rules ? launch_one<D, true, true>(ctx, a, partials, plan, stream) : launch_one<D, true, false>(ctx, a, partials, plan, stream);
    }
}

}  // namespace

// Row by row every token's lists (kv4_decode.cu) read all it sees, as tiles a sequence's tokens read it together. 16
// sequences at 2000 tokens, 8 query and K/V heads of 128: 34, 40, 44, 77 and 138 us row by row for 2, 3, 4, 8 and 16 new
// tokens, 34 to 36 as tiles; heads of 64 26, 31, 36, 56 and 101 against 30 to 32, heads of 256 47, 63, 73, 137 and 242
// against 48 to 55. So from three lists a sequence and K/V head on. But a call of tiles takes 12 to 23 us however small
// it is, and row by row 10 to 12 and what its lists (of 32 tokens a step; each costs eleven steps to begin and end) add.
// Over 216 calls of 1 to 64 sequences, 2 to 16 new tokens and up to 8000 cached ones tiles from 6000 steps on give the
// shortest times (geometric mean 23.4 us; from 0 or 12000 on 23.8, never 28.6).
bool kv4_chunk_pays(uint32_t n_seq, uint64_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t max_chunk, uint32_t max_seq_len) {
    const uint64_t rep = q_heads / kv_heads, chunks = (rep + 7u) / 8u;
    if (max_chunk * rep > 0x7FFFFF00u) return false;
    const double lists = static_cast<double>(rows) * static_cast<double>(chunks);   // of a K/V head
    return lists >= 3.0 * n_seq && lists * kv_heads * (max_seq_len / 32u + 12u) >= 6000.0;
}

size_t kv4_chunk_workspace_bytes(int sm_count, uint32_t n_seq, uint64_t rows, uint32_t q_heads, uint32_t kv_heads,
                                 uint32_t head_width, uint32_t max_chunk, uint32_t max_seq_len) {
    const ChunkPlan plan = chunk_plan(sm_count, n_seq, q_heads, kv_heads, head_width, max_chunk, max_seq_len);
    if (plan.splits <= 1u) return 0;
    return static_cast<size_t>(rows) * q_heads * plan.splits * (head_width + 4u) * sizeof(float);
}

int32_t launch_kv4_chunk(const DeviceContext& ctx, const Kv4AttentionArgs& a, void* workspace, size_t workspace_bytes,
                         cudaStream_t stream) {
    const size_t need = kv4_chunk_workspace_bytes(ctx.sm_count, a.cache.n_seq, a.rows, a.q_heads, a.cache.kv_heads,
                                                  a.cache.head_width, a.max_chunk, a.max_seq_len);
    if (need > workspace_bytes) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention workspace too small: need %zu bytes, got %zu", need,
                    workspace_bytes);
    }
    const ChunkPlan plan = chunk_plan(ctx.sm_count, a.cache.n_seq, a.q_heads, a.cache.kv_heads, a.cache.head_width, a.max_chunk,
                                      a.max_seq_len);
    float* partials = static_cast<float*>(workspace);
    switch (a.cache.head_width) {
        case 64u: return launch_form<64>(ctx, a, partials, plan, stream);
        case 128u: return launch_form<128>(ctx, a, partials, plan, stream);
        default: return launch_form<256>(ctx, a, partials, plan, stream);
    }
}

}  // namespace b2
