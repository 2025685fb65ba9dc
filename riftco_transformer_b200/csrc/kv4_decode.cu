// Attention over the 4-bit paged cache, each query row on its own: the single-token decode step, and a
// few new tokens of a sequence (kv4_chunk.cu takes over where there are enough to fill a tile of rows).
//
// For one row of head h, over the cached tokens t it sees:
//   s_t = q . k_t / sqrt(d)      cap:  s = cap * tanh(s / cap)      bias:  s -= slope_h * |position - t|
//   ctx = sum_t softmax(s)_t v_t
// With value = base + scale * code in groups of 64 channels,
//   q . k_t     = sum_g scale_tg (sum_{c in g} q_c code_tc) + base_tg (sum_{c in g} q_c)
//   sum_t p_t v = sum_t (p_t scale_tg) a_tc + sum_t p_t (base_tg + o scale_tg),   a = code - o
// both sums over codes are matrix products with numbers that the tensor core takes exactly, and no value is ever rounded
// to 16 bits.
//
// Keys: codes become bytes with one AND (of the word, and of the word shifted by a nibble: three instructions for eight
// codes) and meet q in integers, mma.m16n8k32. q is rounded to 23 bits of its head's largest and split into three signed
// bytes, whose sums (exact, below 2^17) are joined in FP32: 41 instructions a tile less than the form that values have.
//
// Values cannot do so: the sums of three bytes would need three accumulators for each channel and head, and registers
// hold two. Their codes become fp16 numbers a = code - o (o = 8 and 7 in turn): one AND-OR makes 1024 + code (or
// 1024 + 16 code of the next nibble) of two codes at once, one fp16 add (or multiply-add) takes the offset off, both
// exact; nine instructions for eight codes. Simpler forms of a lose accuracy, because the tensor core cuts its sums off
// instead of rounding them: fp16 subnormals (an AND alone, five instructions for eight) are aligned to the nominal
// exponent and drop ten bits of the accumulator, 4e-5 off; 1 + code / 64 (seven) has an offset whose cut-off part adds
// up over the tokens, 1.5e-4 off at 2049 tokens of zero mean; and code - 8 throughout leaves half a code on average,
// 8.5e-6 at 29000 tokens. Centred, the sums stay small and so does what is cut off. The other operand, p * scale, is
// split into two fp16 parts, 22 bits, that sit in adjacent columns of the eight of mma.m16n8k16 (up to four query heads:
// the second part costs nothing) or in a second instruction (five to eight heads). Scores, softmax statistics and
// accumulators are FP32, and the result agrees with FP32 arithmetic to about 1e-6.
//
// HBM is the floor: 9d/8 bytes per token and K/V head against 8d of the FP32 cache. What bounds it is instructions: 330
// for 16 tokens of a K/V head at d = 128, issued in 59% of the cycles (16 warps an SM, each a chain of its own; 20 warps
// spill). One sequence of 131071 tokens at 32 / 8 heads takes 43 us (3.5 TB/s), the loads alone 30 us. mma.sync rather
// than tcgen05: a row tile has at most 8 live rows, M = 64 or 128 would be idle lanes, and the operands come from
// registers without a trip through shared or tensor memory.
#include "kv4.cuh"
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

namespace b2 {
namespace {

constexpr int kWarps = 4;
constexpr int kPair = 2;              // tiles a warp works on at once: 32 tokens, one for each lane to guard
// Pairs a warp holds in shared memory, one being worked on and the rest in flight.
__host__ __device__ constexpr int slots_of(int d) { return d == 64 ? 4 : 2; }
constexpr float kSlack = 2.0f;        // p may reach 2^kSlack before the maximum is moved

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm(   // not volatile: registers only, free to be scheduled between the loads
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// N consecutive words (N = 1, 2, 4 or 8), `addr` aligned to min(N, 4) words.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&v)[N], uint32_t addr) {
    if constexpr (N == 1) {
        v[0] = lds32(addr);
    } else if constexpr (N == 2) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
                         : "r"(addr + 4u * i)
                         : "memory");
        }
    }
}
// c = kOffset + a * b in integers, c read as FP32 being kMagic + a * b; or c += a * b.
constexpr uint32_t kMagicBits = 0x4B400000u;   // 1.5 * 2^23: sums below 2^22 in magnitude keep the exponent
constexpr float kMagic = 12582912.0f;
template <bool FIRST>
__device__ __forceinline__ void mma16832(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    if constexpr (FIRST) {
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(kMagicBits));
    } else {
        asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}
// Two codes of a word, 16 bits apart, as fp16 numbers code - LOW (the lower one) and code - HIGH, exactly: 1024 + 16 * 15
// fits 11 bits.
__host__ __device__ constexpr uint32_t minus_offsets(int base, int low, int high) {   // -(base + low), -(base + high) in fp16
    // base 1024: ulp 1 at exponent 10; base 64: ulp 1/16 at exponent 6
    return base == 1024 ? (0xE400u + low) | (0xE400u + high) << 16 : (0xD400u + 16u * low) | (0xD400u + 16u * high) << 16;
}
template <int NIBBLE, int LOW, int HIGH>
__device__ __forceinline__ uint32_t codes_of(uint32_t word, uint32_t k1024) {
    if (NIBBLE >= 2) word >>= 8;
    if (NIBBLE % 2 == 0) {
        uint32_t x = codes_1024<0x000F000Fu>(word, k1024), off = minus_offsets(1024, LOW, HIGH);
        const __half2 y = __hadd2(*reinterpret_cast<__half2*>(&x), *reinterpret_cast<__half2*>(&off));
        return *reinterpret_cast<const uint32_t*>(&y);
    }
    uint32_t x = codes_1024<0x00F000F0u>(word, k1024), off = minus_offsets(64, LOW, HIGH);
    const __half2 y = __hfma2(*reinterpret_cast<__half2*>(&x), __half2half2(__ushort_as_half(0x2C00)),   // 1/16
                              *reinterpret_cast<__half2*>(&off));
    return *reinterpret_cast<const uint32_t*>(&y);
}
// The two of a word are an even token's and the next one's: 8 and 7 in turn take their mean of 7.5 off.
template <int NIBBLE>
__device__ __forceinline__ uint32_t value_codes(uint32_t word, uint32_t k1024) { return codes_of<NIBBLE, 8, 7>(word, k1024); }
// The first 11 bits of x; x minus it is exact.
__device__ __forceinline__ float first_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFFE000u); }

// How the work is cut. A list is what one K/V head of one row reads for up to HC query heads, in pairs of tiles; the
// lists of all rows, one behind the other, are cut into equal ranges, one for each CTA, whose partial results
// (one or two a CTA: of the list its range begins in and of the one it ends in) a second kernel joins. Equal ranges
// keep the card full whatever the lengths. Where every list is short, or there are so many rows that lists alone fill
// the card, a CTA takes one whole list and there is nothing to join.
constexpr uint32_t kMaxRows = 1024;   // rows a CTA finds its range among
constexpr uint32_t kMinPairs = 8;     // pairs of a range: below two a warp a CTA is mostly set-up
// Pairs of a range (were all rows of full length) from which there are more ranges than the card holds at once. More
// ranges shorten the time in which an SM's last warps run alone, and cost set-up: 64 sequences of 512 to 8192 tokens take
// 119, 107, 104, 103 and 106 us (96 now, at 160) with at most 32, 64, 96, 160 and any number of pairs, others are fastest
// from 160 on.
constexpr uint32_t kMostPairs = 160;
struct WorkPlan {
    uint32_t ctas;
    uint32_t whole_lists;   // 1: CTA i takes list i
};

// Where a list's partial results are: those of CTAs first .. last, of the first one number `slot`, of the others 0.
struct ListParts {
    uint32_t first, last, slot;
};

// Pairs of tiles of a row's lists: none for a row that is nobody's, one (of no token) for a row that sees nothing.
__device__ __forceinline__ uint32_t row_pairs(const RowSpan& span) {
    if (!span.owned) return 0u;
    if (span.end <= span.begin) return 1u;
    const uint32_t tiles = (span.end - 1u) / kKv4Tile + 1u - span.begin / kKv4Tile;
    return (tiles + kPair - 1u) / kPair;
}
// CTAs that share `total` pairs, the first pair of CTA c, and the last CTA whose range begins at or before a pair. Never
// more CTAs than pairs: `lists` counts rows that are nobody's too, which have no pairs, and a CTA with an empty range
// between a list's first and last would leave a partial result unwritten that the join reads.
__device__ __forceinline__ uint32_t live_ctas(const WorkPlan& plan, uint32_t lists, uint32_t total) {
    return min(plan.ctas, max(min(lists, total), (total + kMinPairs - 1u) / kMinPairs));
}
__device__ __forceinline__ uint32_t first_pair(uint32_t c, uint32_t total, uint32_t ctas) {
    return static_cast<uint32_t>(static_cast<uint64_t>(c) * total / ctas);
}
__device__ __forceinline__ uint32_t owner_of(uint32_t pair, uint32_t total, uint32_t ctas) {   // c * total / ctas < pair + 1
    return static_cast<uint32_t>(((static_cast<uint64_t>(pair) + 1u) * ctas - 1u) / total);
}

// CTAs that an SM's registers are to hold. (Heads of 64: as many as shared memory does; six with smaller rings spill, 44
// against 42 us for 16 sequences of 700 to 4100 tokens with a distance bias.)
__host__ __device__ constexpr int ctas_of(int d, int hc) { return d == 64 ? 5 : d == 128 ? (hc == 4 ? 4 : 3) : 2; }

// HC: query heads of one K/V head worked on together (4 or 8). RULES: score caps or distance biases; plain scores are up
// to 2% faster in a kernel without them.
template <int D, int HC, bool RULES>
__global__ void __launch_bounds__(kWarps * 32, ctas_of(D, HC))
kv4_decode_kernel(const Kv4AttentionArgs a, ListParts* __restrict__ list_parts, float* __restrict__ partials, const WorkPlan plan) {
    using namespace sm100;
    pdl_launch_dependents();
    uint32_t flags = chunk_starts_flag(a);
    constexpr int G = D / 64, kChunks = D / 32;
    constexpr int HL = HC / 4;            // heads of a lane in the score layout
    constexpr uint32_t kTileBytes = kv4_tile_bytes(D);
    constexpr float kWTop = 8192.0f;      // p * scale is scaled to at most 4 kWTop, below 65504

    extern __shared__ __align__(128) uint8_t ring_raw[];
    constexpr int kSlots = slots_of(D);
    constexpr uint32_t kPairBytes = kPair * kTileBytes;
    __shared__ __align__(8) uint64_t bars[kWarps][kSlots];
    __shared__ uint32_t s_abort;
    __shared__ float s_m[kWarps][HC], s_l[kWarps][HC];

    __shared__ uint32_t s_rows[kMaxRows + 1];   // pairs of one list of all rows before a row
    __shared__ uint32_t s_scan[kWarps];

    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t g = lane >> 2, t = lane & 3u;
    volatile uint32_t* abort = &s_abort;
    const uint32_t rep = a.q_heads / a.cache.kv_heads;
    const uint32_t head_chunks = (rep + HC - 1u) / HC, row_lists = a.cache.kv_heads * head_chunks;

    if (threadIdx.x == 0) s_abort = 0;
    if (lane == 0) {
        for (int i = 0; i < kSlots; ++i) mbar_init(&bars[warp][i], 1);
        mbar_fence_init();
    }

    // ---- this CTA's range of pairs ----
    uint32_t at = 0, at_end = 0, total = 0, ctas = 0, row = 0;
    if (plan.whole_lists != 0u) {
        row = blockIdx.x / row_lists;
        const uint32_t pairs = row_pairs(row_span(a, row));
        at = blockIdx.x % row_lists * pairs;
        at_end = at + pairs;
        __syncthreads();
    } else {
        const uint32_t per = (a.rows + kWarps * 32u - 1u) / (kWarps * 32u);   // rows of a thread
        const uint32_t r0 = min(a.rows, threadIdx.x * per), r1 = min(a.rows, r0 + per);
        uint32_t mine = 0;
        for (uint32_t r = r0; r < r1; ++r) {
            s_rows[r] = mine;
            mine += row_pairs(row_span(a, r));
        }
        uint32_t before = mine;
#pragma unroll
        for (uint32_t o = 1; o < 32u; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, before, o);
            if (lane >= o) before += up;
        }
        if (lane == 31u) s_scan[warp] = before;
        __syncthreads();
        uint32_t all = 0;
        before -= mine;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
            before += w < warp ? s_scan[w] : 0u;
            all += s_scan[w];
        }
        for (uint32_t r = r0; r < r1; ++r) s_rows[r] += before;
        if (threadIdx.x == 0) s_rows[a.rows] = all;
        __syncthreads();
        total = all * row_lists;
        ctas = live_ctas(plan, a.rows * row_lists, total);
        if (blockIdx.x >= ctas) {
            if (flags != 0u) kv4_flag(a.status, flags);
            return;
        }
        at = first_pair(blockIdx.x, total, ctas);
        at_end = first_pair(blockIdx.x + 1u, total, ctas);
        uint32_t lo = 0, hi = a.rows;   // the row with s_rows[row] * row_lists <= at < s_rows[row + 1] * row_lists
        while (lo + 1u < hi) {
            const uint32_t mid = (lo + hi) / 2u;
            if (s_rows[mid] * row_lists <= at) lo = mid; else hi = mid;
        }
        row = lo;
    }

    const uint32_t ring32 = smem_u32(ring_raw) + warp * (kSlots * kPairBytes);
    uint32_t used = 0;      // pairs this warp has taken through its ring
    uint32_t segment = 0;   // lists this CTA has begun
    while (at < at_end) {
    // ---- the next list of the range: its pairs [pair0, pair1) of `pairs` ----
    const uint32_t row_first = plan.whole_lists != 0u ? 0u : s_rows[row] * row_lists;
    const RowSpan span = row_span(a, row);
    const uint32_t pairs = row_pairs(span);
    if (at - row_first >= pairs * row_lists) {
        ++row;
        continue;
    }
    const uint32_t in_row = (at - row_first) / pairs, pair0 = (at - row_first) % pairs;
    const uint32_t pair1 = min(pairs, pair0 + (at_end - at));
    const uint32_t slot_of_list = segment == 0u ? 0u : 1u;   // a list that is not whole is the CTA's first or its last
    if (plan.whole_lists == 0u && pair0 == 0u && threadIdx.x == 0) {
        list_parts[row * row_lists + in_row] = ListParts{
            blockIdx.x, pair1 == pairs ? blockIdx.x : owner_of(at + pairs - 1u, total, ctas), slot_of_list};
    }
    at += pair1 - pair0;
    ++segment;
    const uint32_t kvh = in_row / head_chunks, chunk = in_row % head_chunks;
    const uint32_t first_head = kvh * rep + chunk * HC;
    const uint32_t live_heads = min(static_cast<uint32_t>(HC), rep - chunk * HC);
    if (span.bad) flags |= B2_ATTN_STATUS_BAD_BLOCK;
    const uint32_t tile0 = span.begin / kKv4Tile;
    const uint32_t tiles = span.end > span.begin ? (span.end - 1u) / kKv4Tile + 1u - tile0 : 0u;
    const uint32_t my_first = tile0 + pair0 * kPair + warp * kPair;
    const uint32_t tile_end = tile0 + min(tiles, pair1 * kPair);
    constexpr uint32_t kStride = kWarps * kPair;
    const uint32_t my_pairs = my_first < tile_end ? (tile_end - my_first + kStride - 1u) / kStride : 0u;
    const uint32_t* table = a.cache.block_tables + static_cast<uint64_t>(span.seq) * a.cache.max_blocks;

    // Byte offsets of the tiles of the warp's next 16 pairs, one per lane.
    uint64_t tile_offset = 0;
    auto look_up = [&](uint32_t i0) {
        const uint32_t tile = my_first + (i0 + lane / kPair) * kStride + lane % kPair;
        if (tile < tile_end) {
            uint64_t phys = __ldg(table + tile / a.cache.tiles_per_block);
            if (phys >= a.cache.physical_blocks) {
                phys = 0;
                flags |= B2_ATTN_STATUS_BAD_BLOCK;
            }
            tile_offset = kv4_tile_offset(a.cache, phys, kvh, tile % a.cache.tiles_per_block);
        }
    };
    // The whole warp: pair i of its list into the next slot (lanes 2(i % 16) and the next hold its offsets).
    auto issue = [&](uint32_t i) {
        if ((i & 15u) == 0u) look_up(i);
        const uint32_t slot = (used + i) % kSlots;
        if (lane / kPair == (i & 15u)) {
            const uint32_t which = lane % kPair, tile = my_first + i * kStride + which;
            fence_proxy_async_smem();
            if (which == 0u) {
                mbar_expect_tx(&bars[warp][slot], tile + 1u < tile_end ? kPairBytes : kTileBytes);
            }
            if (tile < tile_end) {
                bulk_load(ring32 + slot * kPairBytes + which * kTileBytes, a.cache.pages + tile_offset, kTileBytes,
                          &bars[warp][slot]);
            }
        }
    };
    for (uint32_t i = 0; i < kSlots && i < my_pairs; ++i) issue(i);

    // ---- q: rounded to 23 bits of its head's largest, split into three signed bytes, in the order the codes come out ----
    // HC = 4: columns 2h and 2h + 1 of the first product are the two upper bytes of head h, column 2h of the second the
    // lowest; HC = 8: a product for each byte, column n is head n. Of a chunk of 32 channels the lane's k positions are
    // channels 8t + 0, 2, 4, 6 (low nibbles), then 8t + 1, 3, 5, 7.
    const uint32_t col_head = HC == 4 ? g >> 1 : g;
    const bool col_live = col_head < live_heads;
    const float* qp = a.q + (static_cast<uint64_t>(row) * a.q_heads + first_head + (col_live ? col_head : 0u)) * D;
    constexpr int kProducts = HC == 4 ? 2 : 3;
    uint32_t qf[kChunks][2][kProducts];   // [chunk][register][product]
    float q_unscale;                  // of column head
    constexpr float kSumScale = 0.0078125f;   // 2^-7: the sum of 64 channels stays inside FP32
    float q_sum[G];                   // times kSumScale
    {
        float x[kChunks][8];
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const float4 u0 = __ldg(reinterpret_cast<const float4*>(qp + 32 * j + 8 * t));
            const float4 u1 = __ldg(reinterpret_cast<const float4*>(qp + 32 * j + 8 * t + 4));
            x[j][0] = u0.x; x[j][1] = u0.y; x[j][2] = u0.z; x[j][3] = u0.w;
            x[j][4] = u1.x; x[j][5] = u1.y; x[j][6] = u1.z; x[j][7] = u1.w;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (!col_live) x[j][e] = 0.0f;
                top = fmaxf(top, fabsf(x[j][e]));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        // 2^e with top * 2^e in [2^21, 2^22); a head of zeros keeps a bounded factor
        int e = 21 - (static_cast<int>((__float_as_uint(top) >> 23) & 255u) - 127);
        e = min(100, e);
        const float up = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
        // (an infinite q has no integers; a NaN one makes q_sum, and with it every score, NaN)
        q_unscale = top < INFINITY ? __uint_as_float(static_cast<uint32_t>(127 - e) << 23) : __uint_as_float(0x7FC00000u);
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            float s = 0.0f;
#pragma unroll
            for (int j = 2 * gr; j < 2 * gr + 2; ++j)
#pragma unroll
                for (int c = 0; c < 8; ++c) s = fmaf(x[j][c], kSumScale, s);
            s += __shfl_xor_sync(0xFFFFFFFFu, s, 1);
            s += __shfl_xor_sync(0xFFFFFFFFu, s, 2);
            q_sum[gr] = s;
        }
        const bool odd = HC == 4 && (g & 1u) != 0u;
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                uint32_t bytes[3] = {0u, 0u, 0u};   // lowest first, of the four channels
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int n = __float2int_rn(x[j][2 * b + w] * up);   // n = d2 2^16 + d1 2^8 + d0, -128 <= d0, d1 < 128
                    const int n1 = (n + 128) >> 8, n2 = (n1 + 128) >> 8;
                    bytes[0] |= (static_cast<uint32_t>(n) & 255u) << (8 * b);
                    bytes[1] |= (static_cast<uint32_t>(n1) & 255u) << (8 * b);
                    bytes[2] |= (static_cast<uint32_t>(n2) & 255u) << (8 * b);
                }
                if (HC == 4) {
                    qf[j][w][0] = odd ? bytes[1] : bytes[2];
                    qf[j][w][1] = odd ? 0u : bytes[0];
                } else {
                    qf[j][w][0] = bytes[2];
                    qf[j][w][1] = bytes[1];
                    qf[j][w][kProducts - 1] = bytes[0];
                }
            }
    }
    // Score layout: a lane holds tokens g and g + 8 of heads t (HC = 4) or 2t, 2t + 1 (HC = 8).
    const float inv_sqrt = 1.0f / sqrtf(static_cast<float>(D));
    // Scores come out in log2 units, or, where they are capped, divided by the cap.
    const bool capped = RULES && a.rules.softcap != 0.0f, biased = RULES && a.rules.alibi_slopes != nullptr;
    const float unit = capped ? 1.0f / a.rules.softcap : kLog2e;
    const float cap_log2 = a.rules.softcap * kLog2e;
    float code_factor[HL];   // unit / q's power of two / sqrt(d)
    float base_factor[HL][G];
    float slope[HL];
#pragma unroll
    for (int h = 0; h < HL; ++h) {
        const int src = HC == 4 ? static_cast<int>(t) * 8 : static_cast<int>(2 * t + h) * 4;   // lane of column head
        code_factor[h] = __shfl_sync(0xFFFFFFFFu, q_unscale, src) * (inv_sqrt * unit);
#pragma unroll
        for (int gr = 0; gr < G; ++gr) base_factor[h][gr] = __shfl_sync(0xFFFFFFFFu, q_sum[gr], src) * (inv_sqrt * unit * (1.0f / kSumScale));
        const uint32_t head = HC == 4 ? t : 2 * t + h;
        slope[h] = biased && head < live_heads ? __ldg(a.rules.alibi_slopes + first_head + head) * kLog2e : 0.0f;
    }

    float m[HL], l[HL], base_acc[HL][G];
    float acc[kChunks][2][4];
#pragma unroll
    for (int h = 0; h < HL; ++h) {
        m[h] = kNoMax;
        l[h] = 0.0f;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) base_acc[h][gr] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[j][u][c] = 0.0f;
    // p * scale is brought to fp16's range by a power of two over the largest magnitude of a value scale met so far.
    float scale_top = 0.0f;      // power of two at or above it (0: none but zeros yet)
    float weight_factor = 0.0f;  // kWTop / scale_top

    const uint32_t k1024 = opaque_1024();
    const float value_offset = (g & 1u) ? 7.0f : 8.0f;   // of tokens g and g + 8
    // This lane's part of a weight: the first 11 bits (even columns) or the rest (odd ones) of w, as
    // w * part_of + ((w & first 11 bits) ^ part_sign).
    const float part_of = (g & 1u) ? 1.0f : 0.0f;
    const uint32_t part_sign = (g & 1u) ? 0x80000000u : 0u;

    for (uint32_t i = 0; i < my_pairs; ++i) {
        const uint32_t token0 = (my_first + i * kStride) * kKv4Tile;
        const uint32_t slot = (used + i) % kSlots, slot32 = ring32 + slot * kPairBytes;
        // Only the first and the last tiles hold tokens that are not seen (or no tile at all).
        const bool whole = token0 >= span.begin && token0 + kPair * kKv4Tile <= span.end &&
                           my_first + i * kStride + kPair <= tile_end;
        mbar_wait(&bars[warp][slot], ((used + i) / kSlots) & 1u, abort);
        if (!whole) {
            // Lane l guards token l of the pair: a slot that is not seen may hold anything, NaN included.
            const uint32_t token = token0 + lane;
            if (token < span.begin || token >= span.end || token / kKv4Tile >= tile_end) {
                const uint32_t at = slot32 + (lane / kKv4Tile) * kTileBytes + 8u * D + (lane % kKv4Tile) * (4u * G);
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    sts32(at + 4u * gr, 0u);
                    sts32(at + 4u * gr + kv4_half_bytes(D), 0u);
                }
            }
            fence_proxy_async_smem();   // the slot is next written by a bulk copy
            __syncwarp();
        }

        // ---- scores ----
        float s[2 * kPair][HL];   // tokens g, g + 8 of both tiles
#pragma unroll
        for (int w = 0; w < kPair; ++w) {
            const uint32_t k32 = slot32 + w * kTileBytes;
            uint32_t kp0[G], kp1[G];
            lds_words<G>(kp0, k32 + 8u * D + g * (4u * G));
            lds_words<G>(kp1, k32 + 8u * D + (g + 8u) * (4u * G));
            float total0[HL], total1[HL], base0[HL], base1[HL];
#pragma unroll
            for (int h = 0; h < HL; ++h) total0[h] = total1[h] = base0[h] = base1[h] = 0.0f;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                uint32_t r[4];   // chunk 2gr: tokens g, g + 8; chunk 2gr + 1: the same
                ldsm4(r, k32 + gr * 512u + lane * 16u);
                uint32_t c[kProducts][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t a0 = r[2 * j] & 0x0F0F0F0Fu, a1 = r[2 * j + 1] & 0x0F0F0F0Fu;
                    const uint32_t a2 = (r[2 * j] >> 4) & 0x0F0F0F0Fu, a3 = (r[2 * j + 1] >> 4) & 0x0F0F0F0Fu;
#pragma unroll
                    for (int n = 0; n < kProducts; ++n) {
                        if (j == 0) {
                            mma16832<true>(c[n], a0, a1, a2, a3, qf[2 * gr][0][n], qf[2 * gr][1][n]);
                        } else {
                            mma16832<false>(c[n], a0, a1, a2, a3, qf[2 * gr + 1][0][n], qf[2 * gr + 1][1][n]);
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < HL; ++h) {
                    // the three bytes' sums joined; only the last two additions round, to 2^-24 of the largest possible sum
                    auto joined = [&](uint32_t high, uint32_t mid, uint32_t low) {
                        const float y = fmaf(__uint_as_float(high), 65536.0f, -kMagic * 65793.0f);   // 2^16 + 2^8 + 1
                        return fmaf(__uint_as_float(mid), 256.0f, y) + __uint_as_float(low);
                    };
                    const float y0 = HC == 4 ? joined(c[0][0], c[0][1], c[1][0]) : joined(c[0][h], c[1][h], c[kProducts - 1][h]);
                    const float y1 = HC == 4 ? joined(c[0][2], c[0][3], c[1][2]) : joined(c[0][2 + h], c[1][2 + h], c[kProducts - 1][2 + h]);
                    total0[h] = fmaf(low_half(kp0[gr]), y0, total0[h]);
                    total1[h] = fmaf(low_half(kp1[gr]), y1, total1[h]);
                    base0[h] = fmaf(high_half(kp0[gr]), base_factor[h][gr], base0[h]);
                    base1[h] = fmaf(high_half(kp1[gr]), base_factor[h][gr], base1[h]);
                }
            }
#pragma unroll
            for (int h = 0; h < HL; ++h) {
                s[2 * w][h] = fmaf(total0[h], code_factor[h], base0[h]);
                s[2 * w + 1][h] = fmaf(total1[h], code_factor[h], base1[h]);
            }
        }
        if (capped) {
#pragma unroll
            for (int k = 0; k < 2 * kPair; ++k)
#pragma unroll
                for (int h = 0; h < HL; ++h) s[k][h] = cap_log2 * tanhf(s[k][h]);
        }
        if (biased) {
#pragma unroll
            for (int k = 0; k < 2 * kPair; ++k) {
                const float away = fabsf(static_cast<float>(static_cast<int>(span.position - (token0 + g + 8u * k))));
#pragma unroll
                for (int h = 0; h < HL; ++h) s[k][h] = fmaf(-slope[h], away, s[k][h]);
            }
        }
        if (!whole) {
#pragma unroll
            for (int k = 0; k < 2 * kPair; ++k) {
                const uint32_t token = token0 + g + 8u * k;
                if (token < span.begin || token >= span.end || token / kKv4Tile >= tile_end) {
#pragma unroll
                    for (int h = 0; h < HL; ++h) s[k][h] = -INFINITY;
                }
            }
        }

        // ---- maximum: moved only when a score passes it by kSlack, or a value scale its bound ----
        uint32_t vq[2 * kPair][G];   // pairs of the values of tokens g, g + 8 of both tiles
        __half2 top2 = __half2half2(__ushort_as_half(0));   // of magnitudes: a scale is negative where its base was rounded up
#pragma unroll
        for (int k = 0; k < 2 * kPair; ++k) {
            lds_words<G>(vq[k], slot32 + (k / 2) * kTileBytes + kv4_half_bytes(D) + 8u * D + (g + 8u * (k % 2)) * (4u * G));
#pragma unroll
            for (int gr = 0; gr < G; ++gr) top2 = __hmax2(top2, __habs2(*reinterpret_cast<__half2*>(&vq[k][gr])));
        }
        float scale_max = __low2float(top2);
        bool move = scale_max > scale_top;
#pragma unroll
        for (int h = 0; h < HL; ++h) {
            // (the difference of close numbers is exact; m + kSlack may round up past the next score, and p to 2^4)
            move = move || fmaxf(fmaxf(s[0][h], s[1][h]), fmaxf(s[2][h], s[3][h])) - m[h] > kSlack;
        }
        if (__any_sync(0xFFFFFFFFu, move)) {
            scale_max = fmaxf(scale_max, __shfl_xor_sync(0xFFFFFFFFu, scale_max, 4));
            scale_max = fmaxf(scale_max, __shfl_xor_sync(0xFFFFFFFFu, scale_max, 8));
            scale_max = fmaxf(scale_max, __shfl_xor_sync(0xFFFFFFFFu, scale_max, 16));
            float shrink = 1.0f;
            if (scale_max > scale_top) {
                // the power of two at or above scale_max (fp16, so at least 2^-24 and at most 2^16)
                const float top = __uint_as_float((__float_as_uint(scale_max) + 0x007FFFFFu) & 0x7F800000u);
                shrink = scale_top / top;   // both powers of two; 0 the first time
                scale_top = top;
                weight_factor = kWTop / top;
            }
            float factor[HL];
#pragma unroll
            for (int h = 0; h < HL; ++h) {
                float top = fmaxf(m[h], fmaxf(fmaxf(s[0][h], s[1][h]), fmaxf(s[2][h], s[3][h])));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
                factor[h] = ex2(m[h] - top);
                m[h] = top;
                l[h] *= factor[h];
#pragma unroll
                for (int gr = 0; gr < G; ++gr) base_acc[h][gr] *= factor[h];
            }
            // accumulator columns 2t, 2t + 1 belong to the same heads as this lane's scores
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[j][u][c] *= factor[(c & 1) * (HL - 1)] * shrink;
        }

        // ---- weights ----
        float p[2 * kPair][HL];
#pragma unroll
        for (int k = 0; k < 2 * kPair; ++k)
#pragma unroll
            for (int h = 0; h < HL; ++h) {
                p[k][h] = ex2(s[k][h] - m[h]);
                l[h] += p[k][h];
            }
#pragma unroll
        for (int k = 0; k < 2 * kPair; ++k)
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                const float b = fmaf(value_offset, low_half(vq[k][gr]), high_half(vq[k][gr]));
#pragma unroll
                for (int h = 0; h < HL; ++h) base_acc[h][gr] = fmaf(p[k][h], b, base_acc[h][gr]);
            }
#pragma unroll
        for (int w = 0; w < kPair; ++w) {
            const uint32_t v32 = slot32 + w * kTileBytes + kv4_half_bytes(D);
            // To the layout of the second product's B operand: column g, tokens 2t, 2t + 1, 2t + 8, 2t + 9.
            float wt[4];
            {
                const int src0 = static_cast<int>(2 * t) * 4 + static_cast<int>(g >> 1), src1 = src0 + 4;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float a0 = __shfl_sync(0xFFFFFFFFu, p[2 * w + k][0], src0);
                    float a1 = __shfl_sync(0xFFFFFFFFu, p[2 * w + k][0], src1);
                    if (HC == 8) {   // heads 2t, 2t + 1 of the source lane: the odd columns take the second
                        const float o0 = __shfl_sync(0xFFFFFFFFu, p[2 * w + k][HL - 1], src0);
                        const float o1 = __shfl_sync(0xFFFFFFFFu, p[2 * w + k][HL - 1], src1);
                        if (g & 1u) {
                            a0 = o0;
                            a1 = o1;
                        }
                    }
                    wt[2 * k] = a0 * weight_factor;
                    wt[2 * k + 1] = a1 * weight_factor;
                }
            }
            // ---- values ----
            uint32_t vp_low[2 * G], vp_high[2 * G];   // pairs of tokens 2t, 2t + 1 and 2t + 8, 2t + 9
            lds_words<2 * G>(vp_low, v32 + 8u * D + (2u * t) * (4u * G));
            lds_words<2 * G>(vp_high, v32 + 8u * D + (2u * t + 8u) * (4u * G));
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                uint32_t b[2][HL];   // [register][part, HC = 8]
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint32_t p0 = k == 0 ? vp_low[gr] : vp_high[gr], p1 = k == 0 ? vp_low[G + gr] : vp_high[G + gr];
                    const float w0 = wt[2 * k] * low_half(p0), w1 = wt[2 * k + 1] * low_half(p1);
                    if (HC == 4) {
                        const float x0 = __uint_as_float((__float_as_uint(w0) & 0xFFFFE000u) ^ part_sign);
                        const float x1 = __uint_as_float((__float_as_uint(w1) & 0xFFFFE000u) ^ part_sign);
                        b[k][0] = pack_half(fmaf(w0, part_of, x0), fmaf(w1, part_of, x1));
                    } else {
                        const float h0 = first_part(w0), h1 = first_part(w1);
                        b[k][0] = pack_half(h0, h1);
                        b[k][HL - 1] = pack_half(w0 - h0, w1 - h1);
                    }
                }
                uint32_t r[4];   // chunk 2gr: tokens (2t, 2t+1), (2t+8, 2t+9); chunk 2gr + 1: the same
                ldsm4_trans(r, v32 + gr * 512u + lane * 16u);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        // rows g and g + 8 are channels 4g + 2u and 4g + 2u + 1 of the chunk
                        const uint32_t a0 = u == 0 ? value_codes<0>(r[2 * j], k1024) : value_codes<2>(r[2 * j], k1024);
                        const uint32_t a1 = u == 0 ? value_codes<1>(r[2 * j], k1024) : value_codes<3>(r[2 * j], k1024);
                        const uint32_t a2 = u == 0 ? value_codes<0>(r[2 * j + 1], k1024) : value_codes<2>(r[2 * j + 1], k1024);
                        const uint32_t a3 = u == 0 ? value_codes<1>(r[2 * j + 1], k1024) : value_codes<3>(r[2 * j + 1], k1024);
#pragma unroll
                        for (int part = 0; part < HL; ++part) {
                            mma16816(acc[2 * gr + j][u], a0, a1, a2, a3, b[0][part], b[1][part]);
                        }
                    }
            }
        }
        __syncwarp();   // every lane has read the slot
        if (i + kSlots < my_pairs) issue(i + kSlots);
    }

    // ---- join the warps (the ring is free: it holds their accumulators) ----
    used += my_pairs;
    __syncthreads();
    float* s_acc = reinterpret_cast<float*>(ring_raw);   // [warp][HC][D]
    const float undo = scale_top / kWTop;
#pragma unroll
    for (int h = 0; h < HL; ++h) {
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 4);
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 8);
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 16);
        const uint32_t head = HC == 4 ? t : 2 * t + h;
        // a NaN or +infinite score left a NaN weight, and nothing else does
        if (isnan(l[h]) && head < live_heads) flags |= B2_ATTN_STATUS_NAN_OR_POS_INF;
        if (g == 0) {
            s_m[warp][head] = m[h];
            s_l[warp][head] = l[h];
        }
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            float b = base_acc[h][gr];
            b += __shfl_xor_sync(0xFFFFFFFFu, b, 4);
            b += __shfl_xor_sync(0xFFFFFFFFu, b, 8);
            b += __shfl_xor_sync(0xFFFFFFFFu, b, 16);
#pragma unroll
            for (int j = 2 * gr; j < 2 * gr + 2; ++j) {
                float o[4];   // channels 32j + 4g + 0..3
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float even = HC == 4 ? acc[j][u][0] + acc[j][u][1] : acc[j][u][h];
                    const float odd = HC == 4 ? acc[j][u][2] + acc[j][u][3] : acc[j][u][2 + h];
                    o[2 * u] = fmaf(even, undo, b);
                    o[2 * u + 1] = fmaf(odd, undo, b);
                }
                *reinterpret_cast<float4*>(&s_acc[(warp * HC + head) * D + 32 * j + 4 * g]) =
                    make_float4(o[0], o[1], o[2], o[3]);
            }
        }
    }
    __syncthreads();
    const bool whole = pair1 - pair0 == pairs;
    float* const part = partials + static_cast<uint64_t>(blockIdx.x * 2u + slot_of_list) * HC * (D + 4u);
    for (uint32_t i = threadIdx.x; i < live_heads * (D / 4u); i += kWarps * 32u) {
        const uint32_t head = i / (D / 4u), c = (i % (D / 4u)) * 4u;
        float mm = s_m[0][head];
#pragma unroll
        for (int wv = 1; wv < kWarps; ++wv) mm = fmaxf(mm, s_m[wv][head]);
        float ll = 0.0f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int wv = 0; wv < kWarps; ++wv) {
            const float f = ex2(s_m[wv][head] - mm);
            const float4 x = *reinterpret_cast<const float4*>(&s_acc[(wv * HC + head) * D + c]);
            ll = fmaf(s_l[wv][head], f, ll);
            o.x = fmaf(x.x, f, o.x);
            o.y = fmaf(x.y, f, o.y);
            o.z = fmaf(x.z, f, o.z);
            o.w = fmaf(x.w, f, o.w);
        }
        const uint64_t out_head = static_cast<uint64_t>(row) * a.q_heads + first_head + head;
        if (!whole) {
            float* dst = part + head * (D + 4u);
            *reinterpret_cast<float4*>(dst + 4u + c) = o;
            if (c == 0) {
                dst[0] = mm;
                dst[1] = ll;
            }
            continue;
        }
        if (ll == 0.0f && tiles != 0u && c == 0) kv4_flag(a.status, B2_ATTN_STATUS_ALL_NEG_INF);
        put_context<D>(a, out_head, c, o, ll);
    }
    if (at < at_end) __syncthreads();   // the ring and the statistics are free again
    }
    if (lane == 0 && *abort != 0) flags |= B2_ATTN_STATUS_TIMEOUT;
    if (flags != 0u) kv4_flag(a.status, flags);
}

// Joins the partial results of every list that more than one CTA worked on: a CTA for each list and head, in which
// kJoiners groups of threads join a run of them each and then, in order, one another's.
constexpr uint32_t kJoiners = 8;
template <int D, int HC>
__global__ void __launch_bounds__(D / 4 * kJoiners)
kv4_merge_kernel(const Kv4AttentionArgs a, const ListParts* list_parts, const float* partials) {
    sm100::pdl_launch_dependents();
    const uint32_t rep = a.q_heads / a.cache.kv_heads;
    const uint32_t head_chunks = (rep + HC - 1u) / HC, row_lists = a.cache.kv_heads * head_chunks;
    const uint32_t list = blockIdx.x / HC, head = blockIdx.x % HC;
    const uint32_t row = list / row_lists, in_row = list % row_lists, chunk = in_row % head_chunks;
    const bool mine = head < rep - chunk * HC && (a.chunk_starts == nullptr || row_span(a, row).owned);
    sm100::pdl_wait();   // every CTA waits, so that this grid never ends before the one it follows
    if (!mine) return;
    const ListParts parts = list_parts[list];
    if (parts.first == parts.last) return;
    const uint32_t n = parts.last - parts.first + 1u;
    const uint64_t out_head = static_cast<uint64_t>(row) * a.q_heads + in_row / head_chunks * rep + chunk * HC + head;
    const uint64_t stride = 2ull * HC * (D + 4u);   // between CTAs
    const float* first = partials + ((parts.first * 2ull + parts.slot) * HC + head) * (D + 4u);
    const float* rest = partials + ((parts.first + 1ull) * 2u * HC + head) * (D + 4u);
    const uint32_t c = threadIdx.x % (D / 4u) * 4u, joiner = threadIdx.x / (D / 4u);
    const uint32_t run = (n + kJoiners - 1u) / kJoiners, i0 = min(n, joiner * run), i1 = min(n, i0 + run);
    __shared__ __align__(16) float s_part[kJoiners][D + 4];
    Joined mine_joined = join_run(i0 == 0u ? first : rest + (i0 - 1u) * stride, rest + i0 * stride, stride, i1 - i0, c);
    *reinterpret_cast<float4*>(&s_part[joiner][4u + c]) = mine_joined.o;
    if (c == 0u) {
        s_part[joiner][0] = mine_joined.m;
        s_part[joiner][1] = mine_joined.l;
    }
    __syncthreads();
    if (joiner != 0u) return;
    const Joined all = join_run(s_part[0], s_part[1], D + 4u, kJoiners, c);
    finish<D>(a, all, out_head, c, true);
}

uint32_t heads_together(uint32_t rep) { return rep <= 4u ? 4u : 8u; }

constexpr int ring_bytes(int d) { return kWarps * slots_of(d) * kPair * static_cast<int>(kv4_tile_bytes(d)); }

// Configures the forms for a width and number of heads on the current device and reports how many of its CTAs an SM holds.
template <int D, int HC>
int32_t resident_ctas(const DeviceContext& ctx, uint32_t* out) {
    static PerDeviceOnce configured;
    static uint32_t resident[kMaxDevices];
    B2_TRY(once_per_device(configured, ctx.device, [&]() -> int32_t {
        int n = 0, with_rules = 0;
        B2_CUDA_TRY(cudaFuncSetAttribute(kv4_decode_kernel<D, HC, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, ring_bytes(D)));
        B2_CUDA_TRY(cudaFuncSetAttribute(kv4_decode_kernel<D, HC, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, ring_bytes(D)));
        B2_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kv4_decode_kernel<D, HC, false>, kWarps * 32, ring_bytes(D)));
        B2_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&with_rules, kv4_decode_kernel<D, HC, true>, kWarps * 32, ring_bytes(D)));
        n = n < with_rules ? n : with_rules;   // the workspace does not depend on the rules
        resident[ctx.device] = n > 0 ? static_cast<uint32_t>(n) : 1u;
        return B2_STATUS_OK;
    }));
    *out = resident[ctx.device];
    return B2_STATUS_OK;
}

struct Sizes {
    uint32_t d, together;
    uint64_t lists;
};

int32_t work_plan(const DeviceContext& ctx, uint64_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t d,
                  uint32_t max_tokens, WorkPlan* plan, Sizes* sizes) {
    const uint32_t rep = q_heads / kv_heads, together = heads_together(rep);
    const uint64_t lists = rows * kv_heads * ((rep + together - 1u) / together);
    if (lists > 0x0FFFFFFFull) return fail(B2_STATUS_OVERFLOW, "paged attention batch too large");
    *sizes = Sizes{d, together, lists};
    uint32_t resident = 0;
    switch (d) {
    case 64: B2_TRY(together == 4u ? (resident_ctas<64, 4>(ctx, &resident)) : (resident_ctas<64, 8>(ctx, &resident))); break;
    case 128: B2_TRY(together == 4u ? (resident_ctas<128, 4>(ctx, &resident)) : (resident_ctas<128, 8>(ctx, &resident))); break;
    default: B2_TRY(together == 4u ? (resident_ctas<256, 4>(ctx, &resident)) : (resident_ctas<256, 8>(ctx, &resident))); break;
    }
    // a window's first tile may be cut: one tile more than the tokens alone
    const uint64_t pairs = (static_cast<uint64_t>(max_tokens) + kKv4Tile - 1u) / (kKv4Tile * kPair) + 1u;
    // prefix sums of the pairs are 32-bit numbers
    if (rows > kMaxRows || pairs <= kMinPairs || lists * pairs > 0xFFFFFFFFull) {
        *plan = WorkPlan{static_cast<uint32_t>(lists), 1u};
        return B2_STATUS_OK;
    }
    const uint64_t held = (ctx.sm_count > 0 ? static_cast<uint64_t>(ctx.sm_count) : 148u) * resident;
    uint64_t ctas = (lists * pairs + kMinPairs - 1u) / kMinPairs;
    if (ctas > held) ctas = held * ((lists * pairs + held * kMostPairs - 1u) / (held * kMostPairs));
    *plan = WorkPlan{static_cast<uint32_t>(ctas), 0u};
    return B2_STATUS_OK;
}

size_t table_bytes(const Sizes& s) { return (static_cast<size_t>(s.lists) * sizeof(ListParts) + 255u) & ~size_t{255}; }
size_t plan_bytes(const WorkPlan& plan, const Sizes& s) {
    if (plan.whole_lists != 0u) return 0;
    return table_bytes(s) + static_cast<size_t>(plan.ctas) * 2u * s.together * (s.d + 4u) * sizeof(float);
}

template <int D, int HC>
int32_t launch_one(const Kv4AttentionArgs& a, void* workspace, const WorkPlan& plan, const Sizes& sizes, cudaStream_t stream) {
    ListParts* lists = static_cast<ListParts*>(workspace);
    float* partials = workspace == nullptr ? nullptr
                                           : reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + table_bytes(sizes));
    if (a.rules.softcap != 0.0f || a.rules.alibi_slopes != nullptr) {
        kv4_decode_kernel<D, HC, true><<<plan.ctas, kWarps * 32, ring_bytes(D), stream>>>(a, lists, partials, plan);
    } else {
        kv4_decode_kernel<D, HC, false><<<plan.ctas, kWarps * 32, ring_bytes(D), stream>>>(a, lists, partials, plan);
    }
    B2_CUDA_TRY(cudaGetLastError());
    if (plan.whole_lists != 0u) return B2_STATUS_OK;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(sizes.lists * HC));
    config.blockDim = dim3(D / 4 * kJoiners);
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    B2_CUDA_TRY(cudaLaunchKernelEx(&config, kv4_merge_kernel<D, HC>, a, static_cast<const ListParts*>(lists),
                                   static_cast<const float*>(partials)));
    return B2_STATUS_OK;
}

}  // namespace

int32_t kv4_decode_workspace_bytes(const DeviceContext& ctx, uint64_t rows, uint32_t q_heads, uint32_t kv_heads,
                                   uint32_t head_width, uint32_t max_seq_len, size_t* bytes) {
    WorkPlan plan;
    Sizes sizes;
    B2_TRY(work_plan(ctx, rows, q_heads, kv_heads, head_width, max_seq_len, &plan, &sizes));
    *bytes = plan_bytes(plan, sizes);
    return B2_STATUS_OK;
}

int32_t launch_kv4_decode(const DeviceContext& ctx, const Kv4AttentionArgs& a, void* workspace, size_t workspace_bytes,
                          cudaStream_t stream) {
    WorkPlan plan;
    Sizes sizes;
    // A window bounds what a row sees. Fewer tokens need no more workspace, but for bounds so large that their pairs pass 32
    // bits: those are planned as whole lists, in no workspace, and so is their window then.
    const uint32_t window = a.rules.window != 0u && a.rules.prefix_lens == nullptr ? a.rules.window : UINT32_MAX;
    B2_TRY(work_plan(ctx, a.rows, a.q_heads, a.cache.kv_heads, a.cache.head_width, a.max_seq_len, &plan, &sizes));
    if (window < a.max_seq_len && plan.whole_lists == 0u) {
        B2_TRY(work_plan(ctx, a.rows, a.q_heads, a.cache.kv_heads, a.cache.head_width, window, &plan, &sizes));
    }
    const size_t need = plan_bytes(plan, sizes);
    if (need > workspace_bytes) {
        return fail(B2_STATUS_INVALID_ARGUMENT, "paged attention workspace too small: need %zu bytes, got %zu", need,
                    workspace_bytes);
    }
    switch (a.cache.head_width) {
    case 64:
        return sizes.together == 4u ? launch_one<64, 4>(a, workspace, plan, sizes, stream)
                                    : launch_one<64, 8>(a, workspace, plan, sizes, stream);
    case 128:
        return sizes.together == 4u ? launch_one<128, 4>(a, workspace, plan, sizes, stream)
                                    : launch_one<128, 8>(a, workspace, plan, sizes, stream);
    default:
        return sizes.together == 4u ? launch_one<256, 4>(a, workspace, plan, sizes, stream)
                                    : launch_one<256, 8>(a, workspace, plan, sizes, stream);
    }
}

}  // namespace b2
