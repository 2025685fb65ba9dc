// Appending to the 4-bit paged K/V cache, with the rotary embedding applied on the way, and reading
// stored tokens back. The FP32 counterparts are rope_append_kernel (decode_glue.cu) and the page loops
// of src/stages/serving/cache/page_table_cache.cpp:44-77; the rotation is rotate_forward,
// src/model/rotary_embedding.cpp:64-117.
//
// A group of 64 channels x of a rotated key or of a value is stored as
//   base = f16(min x)   scale = f16((max x - base) / 15)   code = clamp(rint((x - base) * (1 / scale)), 0, 15)
// in FP32, every operation rounded to nearest even. Codes are 0 where scale is 0, a constant group, or below 0, where
// base was rounded up past all of a nearly constant one. The codes are taken against the ROUNDED base and scale, the ones
// a reader uses, so that rounding them to 11 bits costs at most 15 * scale * 2^-11 at the top of the range, 1/137 of a
// step, instead of adding to the error of every value. A group that holds a NaN or an infinity, or a magnitude above 65000
// (fp16 spans 65504), is stored as scale = base = NaN: it reads back as NaN and the attention over it reports it.
#include "kv4.cuh"
#include "sm100_ptx.cuh"

#include <cuda_fp16.h>

#include <cmath>

namespace b2 {
namespace {

constexpr int kAppendWarps = 8;

// Over the 8 or 16 lanes that share a group.
template <int LANES>
__device__ __forceinline__ float lane_min(float v, uint32_t mask) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(mask, v, o));
    return v;
}
template <int LANES>
__device__ __forceinline__ float lane_max(float v, uint32_t mask) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o));
    return v;
}

struct GroupCode {
    float base, inverse;   // inverse 0: all codes 0
    uint32_t pair;         // fp16 scale (low half), fp16 base
};

// Largest magnitude a group may hold: base + 15 * scale, each rounded to fp16, then stays below fp16's
// 65504 (their rounding adds at most 16 + 15 * 8667 * 2^-11 = 80).
constexpr float kLargest = 65000.0f;

// `low`, `high`: extremes of the group; `finite`: no NaN or infinity in it.
__device__ __forceinline__ GroupCode group_code(float low, float high, bool finite) {
    GroupCode g;
    const __half base = __float2half_rn(low);
    g.base = __half2float(base);
    const __half scale = __float2half_rn(__fdiv_rn(__fsub_rn(high, g.base), 15.0f));
    const float step = __half2float(scale);
    finite = finite && low >= -kLargest && high <= kLargest;
    g.inverse = finite && step > 0.0f ? __fdiv_rn(1.0f, step) : 0.0f;
    g.pair = finite ? static_cast<uint32_t>(__half_as_ushort(scale)) |
                          static_cast<uint32_t>(__half_as_ushort(base)) << 16
                    : 0x7FFF7FFFu;
    return g;
}
__device__ __forceinline__ uint32_t code_of(float x, const GroupCode& g) {
    if (g.inverse == 0.0f) return 0u;
    const float c = rintf(__fmul_rn(__fsub_rn(x, g.base), g.inverse));
    return static_cast<uint32_t>(fminf(fmaxf(c, 0.0f), 15.0f));
}

// D / 8 lanes store one head vector of one token. Lane l of them holds channels 4l .. 4l + 3 of the lower half (`lo`)
// and of the upper half (`hi`) of the head: the rotation pairs (c, c + D/2), so both of a pair are in one lane.
// `mask`: those lanes. `half_tile` points at the keys' or the values' 9D bytes of the tile.
template <int D>
__device__ __forceinline__ void store_vector(const float4& lo, const float4& hi, uint8_t* half_tile, uint32_t slot,
                                             uint32_t l, uint32_t mask) {
    // Lanes that share a group: at D = 64 all 8, over both halves; else 16, one group (D = 128) or two in each half.
    constexpr int kLanes = D == 64 ? 8 : 16;
    float lo_min = fminf(fminf(lo.x, lo.y), fminf(lo.z, lo.w)), lo_max = fmaxf(fmaxf(lo.x, lo.y), fmaxf(lo.z, lo.w));
    float hi_min = fminf(fminf(hi.x, hi.y), fminf(hi.z, hi.w)), hi_max = fmaxf(fmaxf(hi.x, hi.y), fmaxf(hi.z, hi.w));
    // false for a NaN too; infinities the range check below finds
    bool lo_ok = lo.x == lo.x && lo.y == lo.y && lo.z == lo.z && lo.w == lo.w;
    bool hi_ok = hi.x == hi.x && hi.y == hi.y && hi.z == hi.z && hi.w == hi.w;
    if (D == 64) {
        lo_min = fminf(lo_min, hi_min);
        lo_max = fmaxf(lo_max, hi_max);
        lo_ok = lo_ok && hi_ok;
    }
    const uint32_t sharers = D == 256 ? 0xFFFFu << (l & 16u) : mask;
    lo_min = lane_min<kLanes>(lo_min, mask);
    lo_max = lane_max<kLanes>(lo_max, mask);
    lo_ok = (__ballot_sync(mask, lo_ok) & sharers) == sharers;
    const GroupCode gl = group_code(lo_min, lo_max, lo_ok);
    GroupCode gh = gl;
    if (D != 64) {
        hi_min = lane_min<kLanes>(hi_min, mask);
        hi_max = lane_max<kLanes>(hi_max, mask);
        hi_ok = (__ballot_sync(mask, hi_ok) & sharers) == sharers;
        gh = group_code(hi_min, hi_max, hi_ok);
    }
    // 4 codes of each half; of two lanes, one word
    uint32_t wl = code_of(lo.x, gl) | code_of(lo.y, gl) << 4 | code_of(lo.z, gl) << 8 | code_of(lo.w, gl) << 12;
    uint32_t wh = code_of(hi.x, gh) | code_of(hi.y, gh) << 4 | code_of(hi.z, gh) << 8 | code_of(hi.w, gh) << 12;
    wl |= __shfl_down_sync(mask, wl, 1) << 16;
    wh |= __shfl_down_sync(mask, wh, 1) << 16;
    if (l % 2u == 0u) {
        const uint32_t c = 4u * l;
        auto put = [&](uint32_t channel, uint32_t word) {
            *reinterpret_cast<uint32_t*>(half_tile + (channel / 32u) * 256u + slot * 16u + (channel % 32u) / 2u) = word;
        };
        put(c, wl);
        put(c + D / 2, wh);
    }
    uint32_t* pairs = reinterpret_cast<uint32_t*>(half_tile + 8u * D) + slot * (D / 64);
    if (l % 16u == 0u) {
        pairs[l / 16u] = gl.pair;
        if (D != 64) pairs[D / 128 + l / 16u] = gh.pair;
    }
}

constexpr uint32_t kMostTokens = 16;   // of a CTA

// Grid (token run, slice). A CTA takes `per_cta` consecutive tokens and, of each, every gridDim.y-th group of its lanes'
// head vectors: q heads are rotated, k heads rotated and stored, v heads stored. The angles of a token are the same for
// all its heads: they are worked out once, into shared memory (in double: position * theta^(-2c/D) passes 10^5
// radians in long contexts, where FP32 has lost the phase). A prompt is bound by HBM (24.6 KB of q, k and v in, 16.4 KB
// of q and 1.2 KB of pages out per token at 32 / 8 heads of 128): 16-byte accesses, no barrier between the vectors of a
// run, and the loads of the next two under way while one is worked on: 8191 tokens take 72 us (4.8 TB/s), 85 us with one
// vector ahead and a barrier per token. A single token, 6 us, is bound by the latency of its angle.
template <int D>
__global__ void __launch_bounds__(kAppendWarps * 32, 4)
kv4_append_kernel(const Kv4AppendArgs a, uint32_t per_cta) {
    sm100::pdl_launch_dependents();
    constexpr uint32_t kHalf = D / 2, kLanes = D / 8, kVectors = 32u / kLanes * kAppendWarps;   // vectors of a CTA at once
    __shared__ __align__(16) float s_cos[kMostTokens][kHalf], s_sin[kMostTokens][kHalf];
    struct Place {
        uint64_t phys;
        uint32_t tile, slot, good, real;   // real: not padding
    };
    __shared__ Place s_place[kMostTokens];
    const uint32_t l = threadIdx.x % kLanes;
    const uint32_t mask = D == 256 ? 0xFFFFFFFFu : ((1u << (kLanes % 32u)) - 1u) << (threadIdx.x % 32u / kLanes * kLanes);
    const uint32_t heads = a.q_heads + 2u * a.cache.kv_heads;
    const uint64_t token0 = static_cast<uint64_t>(blockIdx.x) * per_cta;
    const uint32_t tokens = static_cast<uint32_t>(min(static_cast<uint64_t>(per_cta), a.n_tokens - token0));

    // The CTA's vectors: slice blockIdx.y of every token's heads, one token behind the other.
    const uint32_t slice_first = blockIdx.y * kVectors, slice_step = gridDim.y * kVectors;
    const uint32_t slices = slice_first < heads ? (heads - slice_first + slice_step - 1u) / slice_step : 0u;
    const uint32_t groups = slices * tokens;   // of kVectors vectors
    struct Vector {
        float4 lo, hi;
    };
    auto head_of = [&](uint32_t group) { return slice_first + group % slices * slice_step + threadIdx.x / kLanes; };
    auto load = [&](uint32_t group) {   // q_out may be q: a lane reads both halves of its pairs before it writes
        Vector x{make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
        const uint32_t h = head_of(group);
        if (group < groups && h < heads) {
            const uint64_t token = token0 + group / slices;
            const float* base = h < a.q_heads ? a.q : h < a.q_heads + a.cache.kv_heads ? a.k : a.v;
            const uint32_t head = h < a.q_heads ? h : h < a.q_heads + a.cache.kv_heads ? h - a.q_heads : h - a.q_heads - a.cache.kv_heads;
            const float* src = base + (token * (h < a.q_heads ? a.q_heads : a.cache.kv_heads) + head) * D + 4u * l;
            x.lo = *reinterpret_cast<const float4*>(src);
            x.hi = *reinterpret_cast<const float4*>(src + kHalf);
        }
        return x;
    };
    Vector ahead[2] = {load(0), load(1)};

    {
        const uint32_t c = threadIdx.x % kHalf;
        const double turn = pow(static_cast<double>(a.theta), static_cast<double>(c) * -2.0 / static_cast<double>(D));
        for (uint32_t i = threadIdx.x / kHalf; i < tokens; i += kAppendWarps * 32u / kHalf) {
            double s_, c_;
            sincos(static_cast<double>(a.positions[token0 + i]) * turn, &s_, &c_);
            s_cos[i][c] = static_cast<float>(c_);
            s_sin[i][c] = static_cast<float>(s_);
        }
    }
    if (threadIdx.x < tokens) {
        const uint64_t token = token0 + threadIdx.x;
        const uint32_t position = a.positions[token], seq = a.token_seq != nullptr ? a.token_seq[token] : static_cast<uint32_t>(token);
        Place p{0, 0, 0, 0, position != kKv4Pad};
        if (p.real != 0u) {
            p.good = kv4_locate(a.cache, seq, position, &p.phys, &p.tile, &p.slot) ? 1u : 0u;
            if (p.good == 0u && blockIdx.y == 0) kv4_flag(a.status, B2_ATTN_STATUS_BAD_BLOCK);
        }
        s_place[threadIdx.x] = p;
    }
    __syncthreads();

#pragma unroll 2
    for (uint32_t group = 0; group < groups; ++group) {
        Vector x = ahead[group % 2u];
        ahead[group % 2u] = load(group + 2u);
        const uint32_t h = head_of(group), i = group / slices;
        const Place place = s_place[i];
        if (h >= heads || place.real == 0u) continue;   // the same for all lanes of a vector
        const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.cache.kv_heads;
        if (is_q || is_k) {
            const float4 cs = *reinterpret_cast<const float4*>(&s_cos[i][4u * l]), sn = *reinterpret_cast<const float4*>(&s_sin[i][4u * l]);
            auto turned = [](float p, float q, float c, float s, float* lo, float* hi) {
                *lo = __fsub_rn(__fmul_rn(p, c), __fmul_rn(q, s));
                *hi = __fadd_rn(__fmul_rn(q, c), __fmul_rn(p, s));
            };
            const Vector y = x;
            turned(y.lo.x, y.hi.x, cs.x, sn.x, &x.lo.x, &x.hi.x);
            turned(y.lo.y, y.hi.y, cs.y, sn.y, &x.lo.y, &x.hi.y);
            turned(y.lo.z, y.hi.z, cs.z, sn.z, &x.lo.z, &x.hi.z);
            turned(y.lo.w, y.hi.w, cs.w, sn.w, &x.lo.w, &x.hi.w);
        }
        if (is_q) {
            float* dst = a.q_out + ((token0 + i) * a.q_heads + h) * D + 4u * l;
            *reinterpret_cast<float4*>(dst) = x.lo;
            *reinterpret_cast<float4*>(dst + kHalf) = x.hi;
        } else if (place.good != 0u) {
            const uint32_t head = is_k ? h - a.q_heads : h - a.q_heads - a.cache.kv_heads;
            uint8_t* half_tile = a.cache.pages + kv4_tile_offset(a.cache, place.phys, head, place.tile) + (is_k ? 0u : kv4_half_bytes(D));
            store_vector<D>(x.lo, x.hi, half_tile, place.slot, l, mask);
        }
    }
}

// D / 4 threads read one stored vector back, four channels each: 2 bytes of codes and a pair in, 16 bytes out, so that
// a warp writes 512 bytes in a row. 16000 tokens of 8 heads of 128, 131 MB out and 18 MB in, take 42 us, 3.6 TB/s, and no
// other grid was faster. What bounds it is not shown: a vector's position, page and codes are loaded one after the other.
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadArgs a) {
    constexpr uint32_t kThreads = D / 4, kVectors = 256u / kThreads;
    const uint32_t c = threadIdx.x % kThreads * 4u;
    const uint64_t vectors = static_cast<uint64_t>(a.n_tokens) * a.cache.kv_heads;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * kVectors + threadIdx.x / kThreads; i < vectors;
         i += static_cast<uint64_t>(gridDim.x) * kVectors) {
        const uint32_t token = static_cast<uint32_t>(i / a.cache.kv_heads), head = static_cast<uint32_t>(i % a.cache.kv_heads);
        const uint32_t position = __ldg(a.positions + token);
        if (position == kKv4Pad) continue;
        const uint32_t seq = a.token_seq != nullptr ? __ldg(a.token_seq + token) : token;
        uint64_t phys;
        uint32_t tile, slot;
        if (!kv4_locate(a.cache, seq, position, &phys, &tile, &slot)) {
            if (c == 0u && head == 0u) kv4_flag(a.status, B2_ATTN_STATUS_BAD_BLOCK);
            continue;
        }
        const uint8_t* tile_base = a.cache.pages + kv4_tile_offset(a.cache, phys, head, tile);
        uint32_t codes[2], pair[2];
#pragma unroll
        for (uint32_t v = 0; v < 2u; ++v) {
            const uint8_t* half_tile = tile_base + v * kv4_half_bytes(D);
            codes[v] = *reinterpret_cast<const uint16_t*>(half_tile + (c / 32u) * 256u + slot * 16u + (c % 32u) / 2u);
            pair[v] = reinterpret_cast<const uint32_t*>(half_tile + 8u * D)[slot * (D / 64u) + c / kKv4Group];
        }
#pragma unroll
        for (uint32_t v = 0; v < 2u; ++v) {
            const float scale = low_half(pair[v]), base = high_half(pair[v]);
            // scale * code is exact (11 + 4 bits), so one rounding in all
            auto value = [&](int e) { return fmaf(scale, static_cast<float>((codes[v] >> (4 * e)) & 15u), base); };
            *reinterpret_cast<float4*>((v == 0u ? a.k_out : a.v_out) + i * D + c) = make_float4(value(0), value(1), value(2), value(3));
        }
    }
}

}  // namespace

int32_t launch_kv4_append(const DeviceContext& ctx, const Kv4AppendArgs& a, cudaStream_t stream) {
    const uint32_t heads = a.q_heads + 2u * a.cache.kv_heads;
    const uint32_t sms = ctx.sm_count > 0 ? static_cast<uint32_t>(ctx.sm_count) : 148u;
    const uint32_t vectors = kAppendWarps * 256u / a.cache.head_width;   // a CTA's at once
    // Few tokens: all vectors at once, spread over CTAs (each repeats the token's angles). Many: one CTA per run of
    // tokens, so that theta^(-2c/d) is worked out once for the run, as many as the card holds (2048 tokens 28 us, 30 with
    // twice as many, 33 with four times).
    uint32_t slices = (heads + vectors - 1u) / vectors;
    const uint64_t wanted = 4ull * sms;   // what the card holds at once
    while (slices > 1u && static_cast<uint64_t>(a.n_tokens) * slices > wanted) slices = (slices + 1u) / 2u;
    uint32_t per_cta = 1u;
    if (slices == 1u) per_cta = static_cast<uint32_t>((a.n_tokens + wanted - 1u) / wanted);
    if (per_cta > kMostTokens) per_cta = kMostTokens;
    const dim3 grid((a.n_tokens + per_cta - 1u) / per_cta, slices);
    const unsigned threads = kAppendWarps * 32;
    switch (a.cache.head_width) {
    case 64: kv4_append_kernel<64><<<grid, threads, 0, stream>>>(a, per_cta); break;
    case 128: kv4_append_kernel<128><<<grid, threads, 0, stream>>>(a, per_cta); break;
    default: kv4_append_kernel<256><<<grid, threads, 0, stream>>>(a, per_cta); break;
    }
    B2_CUDA_TRY(cudaGetLastError());
    return B2_STATUS_OK;
}

int32_t launch_kv4_read(const DeviceContext& ctx, const Kv4ReadArgs& a, cudaStream_t stream) {
    const uint64_t sms = ctx.sm_count > 0 ? static_cast<uint64_t>(ctx.sm_count) : 148u;
    const uint64_t at_once = 1024u / a.cache.head_width;
    uint64_t blocks = (static_cast<uint64_t>(a.n_tokens) * a.cache.kv_heads + at_once - 1u) / at_once;
    if (blocks > sms * 32u) blocks = sms * 32u;
    switch (a.cache.head_width) {
    case 64: kv4_read_kernel<64><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a); break;
    case 128: kv4_read_kernel<128><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a); break;
    default: kv4_read_kernel<256><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a); break;
    }
    B2_CUDA_TRY(cudaGetLastError());
    return B2_STATUS_OK;
}

}  // namespace b2
