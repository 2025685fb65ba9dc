// Appending to the 4-bit paged K/V cache, with the rotary embedding applied on the way, and reading
// stored tokens back. The FP32 counterparts are rope_append_kernel (decode_glue.cu) and the page loops
// of src/stages/serving/cache/page_table_cache.cpp:44-77; the rotation is rotate_forward,
// src/model/rotary_embedding.cpp:64-117.
//
// A group of 64 channels x of a rotated key or of a value is stored as
//   base = f16(min x)   scale = f16((max x - base) / 15)   code = clamp(rint((x - base) * (1 / scale)), 0, 15)
// in FP32, every operation rounded to nearest even (codes 0 where scale is 0, a constant group). The
// codes are taken against the ROUNDED base and scale, the ones a reader uses, so that rounding them to
// 11 bits costs at most 15 * scale * 2^-11 at the top of the range, 1/137 of a step, instead of adding
// to the error of every value. A group that holds a NaN or an infinity, or a magnitude above 65000
// (fp16 spans 65504), is stored as scale = base = NaN: it reads back as NaN and the attention over it reports it.
#include "kv4.cuh"
#include "sm100_ptx.cuh"

#include <cuda_fp16.h>

#include <cmath>

namespace b2 {
namespace {

constexpr int kAppendWarps = 8;

__device__ __forceinline__ float lane_min(float v, int lanes) {
    for (int o = lanes / 2; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}
__device__ __forceinline__ float lane_max(float v, int lanes) {
    for (int o = lanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

struct GroupCode {
    float base, inverse;   // inverse 0: all codes 0
    uint32_t pair;         // fp16 scale (low half), fp16 base
};

// Largest magnitude a group may hold: base + 15 * scale, each rounded to fp16, then stays below fp16's
// 65504 (their rounding adds at most 16 + 15 * 8667 * 2^-12 = 48).
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

// One warp stores one head vector of one token. Lane l holds channels E*l .. E*l + E - 1 of the lower
// half (`lo`) and of the upper half (`hi`) of the head, E = D / 64: the rotation pairs (c, c + D/2), so
// both of a pair are in one lane. `half_tile` points at the keys' or the values' 9D bytes of the tile.
template <int D>
__device__ __forceinline__ void store_vector(const float (&lo)[D / 64], const float (&hi)[D / 64],
                                             uint8_t* half_tile, uint32_t slot, uint32_t lane) {
    constexpr int E = D / 64;
    // Lanes that share a group: D = 64 has one group over both halves; D = 128 one for each half (all 32
    // lanes); D = 256 two for each half (16 lanes each).
    constexpr int kLanes = D == 256 ? 16 : 32;
    float lo_min = lo[0], lo_max = lo[0], hi_min = hi[0], hi_max = hi[0];
    bool lo_ok = true, hi_ok = true;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        lo_min = fminf(lo_min, lo[e]);
        lo_max = fmaxf(lo_max, lo[e]);
        hi_min = fminf(hi_min, hi[e]);
        hi_max = fmaxf(hi_max, hi[e]);
        lo_ok = lo_ok && fabsf(lo[e]) < INFINITY;   // false for a NaN too
        hi_ok = hi_ok && fabsf(hi[e]) < INFINITY;
    }
    if (D == 64) {
        lo_min = hi_min = fminf(lo_min, hi_min);
        lo_max = hi_max = fmaxf(lo_max, hi_max);
        lo_ok = hi_ok = lo_ok && hi_ok;
    }
    lo_min = lane_min(lo_min, kLanes);
    lo_max = lane_max(lo_max, kLanes);
    const uint32_t mine = D == 256 ? (0xFFFFu << (lane & 16u)) : 0xFFFFFFFFu;
    lo_ok = (__ballot_sync(0xFFFFFFFFu, lo_ok) & mine) == mine;
    GroupCode gl = group_code(lo_min, lo_max, lo_ok), gh = gl;
    if (D != 64) {
        hi_min = lane_min(hi_min, kLanes);
        hi_max = lane_max(hi_max, kLanes);
        hi_ok = (__ballot_sync(0xFFFFFFFFu, hi_ok) & mine) == mine;
        gh = group_code(hi_min, hi_max, hi_ok);
    }
    uint32_t wl = 0, wh = 0;   // E codes each
#pragma unroll
    for (int e = 0; e < E; ++e) {
        wl |= code_of(lo[e], gl) << (4 * e);
        wh |= code_of(hi[e], gh) << (4 * e);
    }
    // gather 8 codes (4 bytes) in every (8 / E)-th lane
    constexpr int kPerWord = 8 / E;
    uint32_t shift = 4u * E;
#pragma unroll
    for (int o = 1; o < kPerWord; o <<= 1) {
        wl |= __shfl_down_sync(0xFFFFFFFFu, wl, o) << shift;
        wh |= __shfl_down_sync(0xFFFFFFFFu, wh, o) << shift;
        shift <<= 1;
    }
    if (lane % kPerWord == 0) {
        const uint32_t channel = E * lane;   // of 8 codes, inside the half
        auto put = [&](uint32_t c, uint32_t word) {
            *reinterpret_cast<uint32_t*>(half_tile + (c / 32u) * 256u + slot * 16u + (c % 32u) / 2u) = word;
        };
        put(channel, wl);
        put(channel + D / 2, wh);
    }
    uint32_t* pairs = reinterpret_cast<uint32_t*>(half_tile + 8u * D) + slot * E;
    if (D == 64) {
        if (lane == 0) pairs[0] = gl.pair;
    } else if (D == 128) {
        if (lane == 0) pairs[0] = gl.pair;
        if (lane == 0) pairs[1] = gh.pair;
    } else if (lane % 16u == 0) {
        pairs[lane / 16u] = gl.pair;
        pairs[2 + lane / 16u] = gh.pair;
    }
}

template <int E>
__device__ __forceinline__ void load_e(float (&dst)[E], const float* src) {
    if constexpr (E == 1) {
        dst[0] = *src;
    } else if constexpr (E == 2) {
        const float2 t = *reinterpret_cast<const float2*>(src);
        dst[0] = t.x;
        dst[1] = t.y;
    } else {
        const float4 t = *reinterpret_cast<const float4*>(src);
        dst[0] = t.x;
        dst[1] = t.y;
        dst[2] = t.z;
        dst[3] = t.w;
    }
}
template <int E>
__device__ __forceinline__ void store_e(float* dst, const float (&src)[E]) {
    if constexpr (E == 1) {
        *dst = src[0];
    } else if constexpr (E == 2) {
        *reinterpret_cast<float2*>(dst) = make_float2(src[0], src[1]);
    } else {
        *reinterpret_cast<float4*>(dst) = make_float4(src[0], src[1], src[2], src[3]);
    }
}

// Grid (token run, slice). A CTA takes `per_cta` consecutive tokens and, of each, every gridDim.y-th
// group of warps' heads: q heads are rotated, k heads rotated and stored, v heads stored. The angles of
// a token are the same for all its heads: the first D/2 threads work them out once (in double: position *
// theta^(-2c/D) passes 10^5 radians in long contexts, where FP32 has lost the phase) into shared memory.
// Memory-bound for prompts (12.3 KB of q and k, v per token at 32 / 8 heads of 128 against 4.6 KB of
// 4-bit pages); a single token is bound by the latency of the double-precision angle.
template <int D>
__global__ void __launch_bounds__(kAppendWarps * 32)
kv4_append_kernel(const Kv4AppendArgs a, uint32_t per_cta) {
    sm100::pdl_launch_dependents();
    constexpr int E = D / 64, kHalf = D / 2;
    __shared__ __align__(16) float s_cos[2][kHalf], s_sin[2][kHalf];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t heads = a.q_heads + 2u * a.cache.kv_heads;
    double turn = 0.0;
    if (threadIdx.x < kHalf) {
        turn = pow(static_cast<double>(a.theta), static_cast<double>(threadIdx.x) * -2.0 / static_cast<double>(D));
    }
    uint32_t buffer = 0;
    for (uint32_t i = 0; i < per_cta; ++i) {
        const uint64_t token = static_cast<uint64_t>(blockIdx.x) * per_cta + i;
        if (token >= a.n_tokens) return;
        const uint32_t position = a.positions[token];
        if (position == kKv4Pad) continue;   // the same for every thread: no barrier is skipped by some
        float* const cosines = s_cos[buffer];
        float* const sines = s_sin[buffer];
        buffer ^= 1u;
        if (threadIdx.x < kHalf) {
            double s_, c_;
            sincos(static_cast<double>(position) * turn, &s_, &c_);
            cosines[threadIdx.x] = static_cast<float>(c_);
            sines[threadIdx.x] = static_cast<float>(s_);
        }
        const uint32_t seq = a.token_seq != nullptr ? a.token_seq[token] : static_cast<uint32_t>(token);
        uint64_t phys;
        uint32_t tile, slot;
        const bool good = kv4_locate(a.cache, seq, position, &phys, &tile, &slot);
        if (!good && threadIdx.x == 0 && blockIdx.y == 0) kv4_flag(a.status, B2_ATTN_STATUS_BAD_BLOCK);
        // One barrier a token: a buffer is written again two barriers after its readers' own.
        __syncthreads();
        float cs[E], sn[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            cs[e] = cosines[E * lane + e];
            sn[e] = sines[E * lane + e];
        }
        for (uint32_t h = blockIdx.y * kAppendWarps + warp; h < heads; h += gridDim.y * kAppendWarps) {
            const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.cache.kv_heads;
            if (!is_q && !good) continue;
            const uint32_t head = is_q ? h : (is_k ? h - a.q_heads : h - a.q_heads - a.cache.kv_heads);
            const uint64_t at = (token * (is_q ? a.q_heads : a.cache.kv_heads) + head) * D;
            const float* src = (is_q ? a.q : is_k ? a.k : a.v) + at;
            float lo[E], hi[E];
            load_e<E>(lo, src + E * lane);   // q_out may be q: a lane reads both halves of its pairs first
            load_e<E>(hi, src + kHalf + E * lane);
            if (is_q || is_k) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = lo[e], y = hi[e];
                    lo[e] = __fsub_rn(__fmul_rn(x, cs[e]), __fmul_rn(y, sn[e]));
                    hi[e] = __fadd_rn(__fmul_rn(y, cs[e]), __fmul_rn(x, sn[e]));
                }
            }
            if (is_q) {
                store_e<E>(a.q_out + at + E * lane, lo);
                store_e<E>(a.q_out + at + kHalf + E * lane, hi);
            } else {
                uint8_t* half_tile = a.cache.pages + kv4_tile_offset(a.cache, phys, head, tile) +
                                     (is_k ? 0u : kv4_half_bytes(D));
                store_vector<D>(lo, hi, half_tile, slot, lane);
            }
        }
    }
}

// Eight channels per thread: 4 bytes of codes and one pair in, 32 bytes out.
template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadArgs a) {
    constexpr uint32_t kParts = D / 8;
    const uint64_t items = static_cast<uint64_t>(a.n_tokens) * a.cache.kv_heads * 2u * kParts;
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * blockDim.x;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < items; i += stride) {
        const uint32_t part = static_cast<uint32_t>(i % kParts);
        const uint64_t vector = i / kParts;
        const uint32_t head = static_cast<uint32_t>(vector % a.cache.kv_heads);
        const uint64_t half = vector / a.cache.kv_heads;
        const uint32_t is_v = static_cast<uint32_t>(half & 1u);
        const uint64_t token = half >> 1;
        const uint32_t position = __ldg(a.positions + token);
        if (position == kKv4Pad) continue;
        const uint32_t seq = a.token_seq != nullptr ? __ldg(a.token_seq + token) : static_cast<uint32_t>(token);
        uint64_t phys;
        uint32_t tile, slot;
        if (!kv4_locate(a.cache, seq, position, &phys, &tile, &slot)) {
            if (part == 0) kv4_flag(a.status, B2_ATTN_STATUS_BAD_BLOCK);
            continue;
        }
        const uint8_t* half_tile = a.cache.pages + kv4_tile_offset(a.cache, phys, head, tile) +
                                   is_v * kv4_half_bytes(D);
        const uint32_t c = part * 8u;
        const uint32_t codes = *reinterpret_cast<const uint32_t*>(half_tile + (c / 32u) * 256u + slot * 16u + (c % 32u) / 2u);
        const __half2 pair = reinterpret_cast<const __half2*>(half_tile + 8u * D)[slot * (D / 64u) + c / kKv4Group];
        const float scale = __low2float(pair), base = __high2float(pair);
        float out[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // scale * code is exact (11 + 4 bits), so one rounding in all
            out[e] = fmaf(scale, static_cast<float>((codes >> (4 * e)) & 15u), base);
        }
        float4* dst = reinterpret_cast<float4*>((is_v ? a.v_out : a.k_out) + (token * a.cache.kv_heads + head) * D + c);
        dst[0] = make_float4(out[0], out[1], out[2], out[3]);
        dst[1] = make_float4(out[4], out[5], out[6], out[7]);
    }
}

}  // namespace

int32_t launch_kv4_append(const DeviceContext& ctx, const Kv4AppendArgs& a, cudaStream_t stream) {
    const uint32_t heads = a.q_heads + 2u * a.cache.kv_heads;
    const uint32_t sms = ctx.sm_count > 0 ? static_cast<uint32_t>(ctx.sm_count) : 148u;
    // Few tokens: a warp per head, spread over CTAs (each repeats the token's angles). Many: one CTA per
    // run of tokens, so that theta^(-2c/d) is worked out once for the run.
    uint32_t slices = (heads + kAppendWarps - 1u) / kAppendWarps;
    const uint64_t wanted = 8ull * sms;
    while (slices > 1u && static_cast<uint64_t>(a.n_tokens) * slices > wanted) slices = (slices + 1u) / 2u;
    uint32_t per_cta = 1u;
    if (slices == 1u) per_cta = static_cast<uint32_t>((a.n_tokens + wanted - 1u) / wanted);
    if (per_cta > 8u) per_cta = 8u;
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
    const uint64_t items = static_cast<uint64_t>(a.n_tokens) * a.cache.kv_heads * 2u * (a.cache.head_width / 8u);
    const uint64_t sms = ctx.sm_count > 0 ? static_cast<uint64_t>(ctx.sm_count) : 148u;
    uint64_t blocks = (items + 255u) / 256u;
    if (blocks > sms * 16u) blocks = sms * 16u;
    switch (a.cache.head_width) {
    case 64: kv4_read_kernel<64><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a); break;
    case 128: kv4_read_kernel<128><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a); break;
    default: kv4_read_kernel<256><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a); break;
    }
    B2_CUDA_TRY(cudaGetLastError());
    return B2_STATUS_OK;
}

}  // namespace b2
