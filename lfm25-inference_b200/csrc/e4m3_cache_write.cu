// Append to the 8-bit paged key/value cache, optionally with the RMS norm and rotation of queries and keys in front.
//
// A run is the longest sequence of tokens of the batch, one behind the other, whose slots are one behind the other within a
// page: one token in a decode step, up to 16 in a prompt.  The unit of work is a run, a KV head and K or V, and belongs to
// one warp: a scale needs the maximum over the run's 16 x head_dim values at most, which fits the warp's registers, so that
// every input is read once and nothing but the result is written.  With 8 values (16 bytes) a lane, a row of 64 takes 8
// lanes and a warp 4 rows at a time.  The run finds itself: every warp looks at the slots of the tokens around its own.
//
// The kernel is bound by the chain slots -> values and old scale -> maximum -> codes in a decode step, by bandwidth over
// long prompts.
//
// Arithmetic: everything in f32.  With norms, x / sqrt(mean(x^2) + eps) * w is rotated by position * inv_freq[d] in the
// pairs (d, d + head_dim / 2); the angle is formed and reduced in f64, since in f32 its error grows with the position
// (1e-3 at position 16384).  Queries are rounded once, to bf16, keys once, to E4M3.
#include "e4m3_cache.cuh"
#include "e4m3_cache.h"
#include "launch.h"

namespace lfm25 {

namespace {

constexpr uint32_t kWarpsMost = 16;
constexpr uint32_t kSpanMost = 16;                       // tokens of a CTA
constexpr uint32_t kRowsMost = kSpanMost + kPageSize - 1;   // with the rest of the last run

struct WriteParams {
    E4m3Cache cache;
    const __nv_bfloat16* key;
    const __nv_bfloat16* value;
    const int64_t* slot_mapping;
    const __nv_bfloat16* query;
    __nv_bfloat16* query_out;
    const __nv_bfloat16* query_norm;
    const __nv_bfloat16* key_norm;
    const float* inv_freq;
    const uint32_t* position_ids;
    uint64_t kv_token_stride;
    uint64_t query_token_stride;
    uint32_t num_tokens;
    uint32_t query_heads;
    uint32_t span;
    float eps;
};

__device__ __forceinline__ void unpack(uint4 raw, float (&x)[8]) {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const float2 pair = bf16x2_to_float2(words[i]);
        x[2 * i] = pair.x;
        x[2 * i + 1] = pair.y;
    }
}

// Norm and rotation of a row that LANES lanes hold, 8 values each; `turn` has (cos, sin) of the row's head_dim / 2 angles.
// Every lane of the warp takes part.
template <uint32_t DIM>
__device__ __forceinline__ void norm_rope_row(float (&x)[8], const float (&weight)[8], const float2* turn, uint32_t piece,
                                              float eps) {
    constexpr uint32_t LANES = DIM / 8;
    float sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
    for (uint32_t delta = LANES / 2; delta > 0; delta >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, delta);
    const float inverse = 1.0f / sqrtf(sum * (1.0f / DIM) + eps);
    const bool second = piece >= LANES / 2;
    const float2* angles = turn + (piece % (LANES / 2)) * 8;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const float mine = x[i] * inverse * weight[i];
        const float other = __shfl_xor_sync(0xffffffffu, mine, LANES / 2);
        const float2 t = angles[i];
        x[i] = fmaf(mine, t.x, second ? other * t.y : -other * t.y);
    }
}

template <uint32_t DIM, bool NORM_ROPE>
__global__ void __launch_bounds__(kWarpsMost * 32)
e4m3_cache_write_kernel(const WriteParams p) {
    constexpr uint32_t LANES = DIM / 8;            // lanes of a row
    constexpr uint32_t ROWS = 32 / LANES;          // rows of a pass
    constexpr uint32_t PASSES = kPageSize / ROWS;
    __shared__ float2 turns[NORM_ROPE ? kRowsMost * DIM / 2 : 1];
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t warps = blockDim.x >> 5;
    const uint32_t piece = lane % LANES;
    const uint32_t lane_row = lane / LANES;
    pdl_launch_dependents();
    pdl_wait();

    // ---- the runs that begin among this CTA's tokens: lane l looks at token begin - 1 + l ----
    const uint32_t begin = blockIdx.x * p.span;
    const int64_t mine = static_cast<int64_t>(begin) + lane - 1;
    const int64_t slot = mine >= 0 && mine < p.num_tokens ? p.slot_mapping[mine] : -2;
    const int64_t before = __shfl_up_sync(0xffffffffu, slot, 1);
    const bool valid = slot >= 0 && static_cast<uint64_t>(slot) / kPageSize < p.cache.num_pages;
    const bool continues = valid && slot % kPageSize != 0 && slot == before + 1 && lane > 0;
    const uint32_t continued = __ballot_sync(0xffffffffu, continues);
    uint32_t leaders = __ballot_sync(0xffffffffu, valid && !continues && lane > 0 && lane <= p.span);

    if (NORM_ROPE) {
        // angles of all tokens that this CTA's queries and runs have
        uint32_t rows = min(p.span, p.num_tokens - begin);
        if (leaders != 0) {
            const uint32_t last = 31 - __clz(leaders);
            const uint32_t after = last == 31 ? 0 : __ffs(~(continued >> (last + 1))) - 1;
            rows = max(rows, last + after);
        }
        for (uint32_t index = threadIdx.x; index < rows * (DIM / 2); index += blockDim.x) {
            const uint32_t row = index / (DIM / 2);
            const double angle = static_cast<double>(p.position_ids[begin + row]) * static_cast<double>(p.inv_freq[index % (DIM / 2)]);
            const double turn = rint(angle * 0.15915494309189535);
            float sine, cosine;
            sincosf(static_cast<float>(fma(turn, -6.283185307179586, angle)), &sine, &cosine);
            turns[index] = make_float2(cosine, sine);
        }
        __syncthreads();

        // ---- queries: all rows of this CTA's tokens ----
        float weight[8];
        unpack(*reinterpret_cast<const uint4*>(p.query_norm + piece * 8), weight);
        const uint32_t tokens = min(p.span, p.num_tokens - begin);
        const uint32_t query_rows = tokens * p.query_heads;
        for (uint32_t first = warp * ROWS; first < query_rows; first += warps * ROWS) {
            const uint32_t row = first + lane_row;
            const uint32_t here = min(row, query_rows - 1);
            const uint32_t token = here / p.query_heads;
            const uint32_t head = here % p.query_heads;
            float x[8];
            unpack(*reinterpret_cast<const uint4*>(p.query + (begin + token) * p.query_token_stride + head * DIM + piece * 8), x);
            norm_rope_row<DIM>(x, weight, turns + token * (DIM / 2), piece, p.eps);
            if (row < query_rows) {
                uint4 out;
                out.x = pack_bf16x2(x[0], x[1]);
                out.y = pack_bf16x2(x[2], x[3]);
                out.z = pack_bf16x2(x[4], x[5]);
                out.w = pack_bf16x2(x[6], x[7]);
                *reinterpret_cast<uint4*>(p.query_out + (static_cast<size_t>(begin + token) * p.query_heads + head) * DIM + piece * 8) = out;
            }
        }
    }

    // ---- runs ----
    const uint32_t kinds = 2 * p.cache.kv_heads;
    const uint32_t units = __popc(leaders) * kinds;
    uint32_t skipped = 0;                              // leaders taken off the mask so far
    for (uint32_t unit = warp; unit < units; unit += warps) {
        while (skipped < unit / kinds) {
            leaders &= leaders - 1;
            ++skipped;
        }
        const uint32_t leader = __ffs(leaders) - 1;
        const uint32_t count = 1 + (leader == 31 ? 0 : __ffs(~(continued >> (leader + 1))) - 1);
        const int64_t first_slot = __shfl_sync(0xffffffffu, slot, leader);
        const uint32_t first_row = leader - 1;         // of the CTA's rows
        const size_t page = static_cast<size_t>(first_slot) / kPageSize;
        const uint32_t offset = static_cast<uint32_t>(first_slot % kPageSize);
        const uint32_t kind = unit % kinds;
        const bool is_value = kind >= p.cache.kv_heads;
        const uint32_t head = is_value ? kind - p.cache.kv_heads : kind;
        const __nv_bfloat16* source = (is_value ? p.value : p.key) + static_cast<size_t>(begin + first_row) * p.kv_token_stride +
                                      head * DIM + piece * 8;
        uint8_t* codes = (is_value ? p.cache.value_codes : p.cache.key_codes) + (page * p.cache.kv_heads + head) * (kPageSize * DIM) + piece * 8;
        float* scale = (is_value ? p.cache.value_scales : p.cache.key_scales) + page * p.cache.kv_heads + head;
        const float old_scale = offset > 0 ? *scale : 0.0f;

        uint4 raw[PASSES];
#pragma unroll
        for (uint32_t pass = 0; pass < PASSES; ++pass) {
            const uint32_t row = pass * ROWS + lane_row;
            raw[pass] = make_uint4(0, 0, 0, 0);
            if (row < count) raw[pass] = *reinterpret_cast<const uint4*>(source + row * p.kv_token_stride);
        }
        float x[PASSES][8];
        float weight[8];
        if (NORM_ROPE && !is_value) unpack(*reinterpret_cast<const uint4*>(p.key_norm + piece * 8), weight);
        uint32_t largest = 0;
#pragma unroll
        for (uint32_t pass = 0; pass < PASSES; ++pass) {
            unpack(raw[pass], x[pass]);
            if (NORM_ROPE && !is_value) {
                const uint32_t row = min(pass * ROWS + lane_row, count - 1);   // rows that do not exist are zeros
                if (pass * ROWS < count) norm_rope_row<DIM>(x[pass], weight, turns + (first_row + row) * (DIM / 2), piece, p.eps);
            }
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                // infinities and NaN do not move the scale: they become the largest code and the NaN code
                const uint32_t magnitude = __float_as_uint(x[pass][i]) & 0x7fffffffu;
                largest = max(largest, magnitude < 0x7f800000u ? magnitude : 0u);
            }
        }
        largest = __reduce_max_sync(0xffffffffu, largest);
        const int32_t old_exponent = stored_exponent(old_scale);
        int32_t exponent = scale_exponent(largest);
        if (offset > 0) exponent = max(exponent, old_exponent);

        const float factor = power_of_two(-exponent);
#pragma unroll
        for (uint32_t pass = 0; pass < PASSES; ++pass) {
            const uint32_t row = pass * ROWS + lane_row;
            if (row < count) {
                uint2 out;
                out.x = e4m3x2(x[pass][0] * factor, x[pass][1] * factor) | (static_cast<uint32_t>(e4m3x2(x[pass][2] * factor, x[pass][3] * factor)) << 16);
                out.y = e4m3x2(x[pass][4] * factor, x[pass][5] * factor) | (static_cast<uint32_t>(e4m3x2(x[pass][6] * factor, x[pass][7] * factor)) << 16);
                *reinterpret_cast<uint2*>(codes + (offset + row) * DIM) = out;
            }
        }
        // what the page holds already goes over to a larger scale
        if (offset > 0 && exponent > old_exponent) {
            const float shrink = power_of_two(old_exponent - exponent);
#pragma unroll
            for (uint32_t pass = 0; pass < PASSES; ++pass) {
                const uint32_t row = pass * ROWS + lane_row;
                if (row < offset) {
                    uint2* place = reinterpret_cast<uint2*>(codes + row * DIM);
                    uint2 there = *place;
                    uint32_t* words[2] = {&there.x, &there.y};
#pragma unroll
                    for (uint32_t w = 0; w < 2; ++w) {
                        const float2 low = f16x2_to_float2(e4m3x2_to_f16x2(*words[w]));
                        const float2 high = f16x2_to_float2(e4m3x2_high_to_f16x2(*words[w]));
                        *words[w] = e4m3x2(low.x * shrink, low.y * shrink) |
                                    (static_cast<uint32_t>(e4m3x2(high.x * shrink, high.y * shrink)) << 16);
                    }
                    *place = there;
                }
            }
        }
        if (lane == 0) *scale = power_of_two(exponent);
    }
}

template <uint32_t DIM>
cudaError_t launch_dim(cudaStream_t stream, const WriteParams& params, unsigned int blocks, unsigned int threads) {
    return params.query != nullptr ? launch_kernel(e4m3_cache_write_kernel<DIM, true>, blocks, threads, 0, stream, 1, params)
                                   : launch_kernel(e4m3_cache_write_kernel<DIM, false>, blocks, threads, 0, stream, 1, params);
}

}  // namespace

cudaError_t launch_e4m3_cache_write(cudaStream_t stream, const E4m3WriteLaunch& launch) {
    WriteParams params = {};
    params.cache = launch.cache;
    params.key = static_cast<const __nv_bfloat16*>(launch.key);
    params.value = static_cast<const __nv_bfloat16*>(launch.value);
    params.slot_mapping = launch.slot_mapping;
    params.query = static_cast<const __nv_bfloat16*>(launch.query);
    params.query_out = static_cast<__nv_bfloat16*>(launch.query_out);
    params.query_norm = static_cast<const __nv_bfloat16*>(launch.query_norm);
    params.key_norm = static_cast<const __nv_bfloat16*>(launch.key_norm);
    params.inv_freq = launch.inv_freq;
    params.position_ids = launch.position_ids;
    params.kv_token_stride = launch.kv_token_stride;
    params.query_token_stride = launch.query_token_stride;
    params.num_tokens = static_cast<uint32_t>(launch.num_tokens);
    params.query_heads = launch.query_heads;
    params.eps = launch.eps;
    // few tokens: a CTA each, so that a decode step's tokens run side by side; many: 16 to a CTA, which then has the runs of
    // a page of a prompt, rather than 16 CTAs of which one finds work
    params.span = launch.num_tokens <= 512 ? 1 : kSpanMost;
    const uint32_t rows = 256 / launch.cache.head_dim;   // of a warp's pass
    const uint32_t units = 2 * launch.cache.kv_heads + params.span * launch.query_heads / rows;
    const unsigned int threads = 32 * (units < kWarpsMost ? units : kWarpsMost);
    const unsigned int blocks = static_cast<unsigned int>((launch.num_tokens + params.span - 1) / params.span);
    return launch.cache.head_dim == 64 ? launch_dim<64>(stream, params, blocks, threads)
                                       : launch_dim<128>(stream, params, blocks, threads);
}

}  // namespace lfm25
