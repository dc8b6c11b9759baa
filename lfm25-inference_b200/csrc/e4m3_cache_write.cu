// Append to the 8-bit paged key/value cache, optionally with the RMS norm and rotation of queries and keys in front.
//
// A run is the longest sequence of tokens of the batch, one behind the other, whose slots are one behind the other within a
// page: one token in a decode step, up to 16 in a prompt.  The unit of work is a run, a KV head and K or V, and belongs to
// one warp: a scale needs the maximum over the run's 16 x head_dim values at most, which fits the warp's registers, so that
// every input is read once and nothing but the result is written.  A lane has 4 dimensions of the first half of a head and the 4
// that they are rotated with, so that a row of 64 takes 8 lanes, a warp 4 rows at a time, and a rotation no exchange.  The run
// finds itself: every warp looks at the slots of the tokens around its own.
//
// The kernel is bound by chains of dependent loads (slots -> values and old scale -> maximum -> codes): in a decode step (128 tokens
// with norms 3.8 us), and over long prompts as well, where 80 registers a thread leave few warps to hide them: 3800 tokens with 32 query
// heads on 8 of 64 move 43 MB in 15.9 us (2.7 TB/s; 52 % of the issue slots used, 35 % of the ALU, 34 % of the places for warps), without
// norms 12 MB in 5.3 us.  Queries, keys and values have CTAs of their own: queries do not wait for slots, values not for
// angles, and all loads of a CTA are under way while it computes its angles.
//
// Arithmetic: everything in f32.  With norms, x / sqrt(mean(x^2) + eps) * w is rotated by position * inv_freq[d] in the
// pairs (d, d + head_dim / 2); the angle is formed and reduced in f64, since in f32 its error grows with the position
// (1e-3 at position 16384).  Queries are rounded once, to bf16, keys once, to E4M3.
#include "e4m3_cache.cuh"
#include "e4m3_cache.h"
#include "launch.h"

namespace lfm25 {

namespace {

constexpr uint32_t kAhead = 4;                           // query rows that a lane loads ahead
constexpr uint32_t kSpanMost = 16;                       // tokens of a CTA that looks for runs
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
    uint32_t query_blocks;   // CTAs in front that have queries, `query_span` tokens each
    uint32_t query_span;
    uint32_t run_blocks;     // behind them so many with keys, `span` tokens each, and as many with values
    uint32_t span;
    float eps;
};

// dimensions 4 i .. 4 i + 3 and, in the upper half, DIM / 2 + 4 i .. of a head, i the lane's place in the row
struct Values {
    float low[4];
    float high[4];
};

template <uint32_t DIM>
__device__ __forceinline__ uint4 load_values(const __nv_bfloat16* head, uint32_t place) {
    const uint2 low = *reinterpret_cast<const uint2*>(head + 4 * place);
    const uint2 high = *reinterpret_cast<const uint2*>(head + DIM / 2 + 4 * place);
    return make_uint4(low.x, low.y, high.x, high.y);
}

__device__ __forceinline__ Values unpack(uint4 raw) {
    const float2 a = bf16x2_to_float2(raw.x);
    const float2 b = bf16x2_to_float2(raw.y);
    const float2 c = bf16x2_to_float2(raw.z);
    const float2 d = bf16x2_to_float2(raw.w);
    return {{a.x, a.y, b.x, b.y}, {c.x, c.y, d.x, d.y}};
}

// Norm and rotation of a row that DIM / 8 lanes hold; `turn` has (cos, sin) of the row's DIM / 2 angles.  Every lane of the warp
// takes part.
template <uint32_t DIM>
__device__ __forceinline__ void norm_rope_row(Values& x, const Values& weight, const float2* turn, uint32_t place, float eps) {
    float sum = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) sum = fmaf(x.low[i], x.low[i], fmaf(x.high[i], x.high[i], sum));
#pragma unroll
    for (uint32_t delta = DIM / 16; delta > 0; delta >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, delta);
    const float inverse = rsqrtf(sum * (1.0f / DIM) + eps);     // 2 units off at most
    const float4 first = reinterpret_cast<const float4*>(turn + 4 * place)[0];
    const float4 second = reinterpret_cast<const float4*>(turn + 4 * place)[1];
    const float cosine[4] = {first.x, first.z, second.x, second.z};
    const float sine[4] = {first.y, first.w, second.y, second.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const float low = x.low[i] * inverse * weight.low[i];
        const float high = x.high[i] * inverse * weight.high[i];
        x.low[i] = fmaf(low, cosine[i], -high * sine[i]);
        x.high[i] = fmaf(high, cosine[i], low * sine[i]);
    }
}

__device__ __forceinline__ uint32_t four_codes(const float (&x)[4], float factor) {
    return e4m3x2(x[0] * factor, x[1] * factor) | (static_cast<uint32_t>(e4m3x2(x[2] * factor, x[3] * factor)) << 16);
}

// (cos, sin) of position * inv_freq for `rows` tokens from `first` on
template <uint32_t DIM, uint32_t kWarps>
__device__ __forceinline__ void angles(const WriteParams& p, uint32_t first, uint32_t rows, float2* turns) {
    for (uint32_t index = threadIdx.x; index < rows * (DIM / 2); index += kWarps * 32) {
        const double angle = static_cast<double>(p.position_ids[first + index / (DIM / 2)]) * static_cast<double>(p.inv_freq[index % (DIM / 2)]);
        const double turn = rint(angle * 0.15915494309189535);
        float sine, cosine;
        sincosf(static_cast<float>(fma(turn, -6.283185307179586, angle)), &sine, &cosine);
        turns[index] = make_float2(cosine, sine);
    }
}

// All queries of `query_span` tokens
template <uint32_t DIM, uint32_t kWarps>
__device__ __forceinline__ void write_queries(const WriteParams& p, float2* turns) {
    constexpr uint32_t LANES = DIM / 8;
    constexpr uint32_t ROWS = 32 / LANES;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t piece = lane % LANES;
    const uint32_t begin = blockIdx.x * p.query_span;
    const uint32_t tokens = min(p.query_span, p.num_tokens - begin);
    const uint32_t rows = tokens * p.query_heads;
    uint4 raw[kAhead];
    uint32_t token_of[kAhead];
    auto load = [&](uint32_t first) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t row = first + i * kWarps * ROWS + lane / LANES;
            raw[i] = make_uint4(0, 0, 0, 0);
            token_of[i] = min(row, rows - 1) / p.query_heads;
            if (row < rows) {
                raw[i] = load_values<DIM>(p.query + (begin + token_of[i]) * p.query_token_stride + (row - token_of[i] * p.query_heads) * DIM, piece);
            }
        }
    };
    load(warp * ROWS);
    const Values weight = unpack(load_values<DIM>(p.query_norm, piece));
    angles<DIM, kWarps>(p, begin, tokens, turns);
    __syncthreads();
    for (uint32_t first = warp * ROWS; first < rows; first += kAhead * kWarps * ROWS) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            if (first + i * kWarps * ROWS < rows) {          // for the whole warp
                const uint32_t row = first + i * kWarps * ROWS + lane / LANES;
                Values x = unpack(raw[i]);
                norm_rope_row<DIM>(x, weight, turns + token_of[i] * (DIM / 2), piece, p.eps);
                if (row < rows) {
                    __nv_bfloat16* out = p.query_out + (static_cast<size_t>(begin) * p.query_heads + row) * DIM;
                    *reinterpret_cast<uint2*>(out + 4 * piece) = make_uint2(pack_bf16x2(x.low[0], x.low[1]), pack_bf16x2(x.low[2], x.low[3]));
                    *reinterpret_cast<uint2*>(out + DIM / 2 + 4 * piece) =
                        make_uint2(pack_bf16x2(x.high[0], x.high[1]), pack_bf16x2(x.high[2], x.high[3]));
                }
            }
        }
        if (first + kAhead * kWarps * ROWS < rows) load(first + kAhead * kWarps * ROWS);
    }
}

template <uint32_t DIM, bool NORM_ROPE, uint32_t kWarps>
__global__ void __launch_bounds__(kWarps * 32, (DIM == 64 ? 24 : 16) / kWarps)
e4m3_cache_write_kernel(const WriteParams p) {
    constexpr uint32_t LANES = DIM / 8;            // lanes of a row
    constexpr uint32_t ROWS = 32 / LANES;          // rows of a pass
    constexpr uint32_t PASSES = kPageSize / ROWS;
    __shared__ __align__(16) float2 turns[NORM_ROPE ? kRowsMost * DIM / 2 : 2];
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t piece = lane % LANES;
    const uint32_t lane_row = lane / LANES;
    pdl_launch_dependents();
    pdl_wait();
    if constexpr (NORM_ROPE) {
        if (blockIdx.x < p.query_blocks) {
            write_queries<DIM, kWarps>(p, turns);
            return;
        }
    }

    // ---- the runs that begin among this CTA's tokens: lane l looks at token begin - 1 + l ----
    const bool is_value = blockIdx.x - p.query_blocks >= p.run_blocks;
    const uint32_t begin = (blockIdx.x - p.query_blocks - (is_value ? p.run_blocks : 0)) * p.span;
    const int64_t mine = static_cast<int64_t>(begin) + lane - 1;
    const int64_t slot = mine >= 0 && mine < p.num_tokens ? p.slot_mapping[mine] : -2;
    const int64_t before = __shfl_up_sync(0xffffffffu, slot, 1);
    const bool valid = slot >= 0 && static_cast<uint64_t>(slot) / kPageSize < p.cache.num_pages;
    const bool continues = valid && slot % kPageSize != 0 && slot == before + 1 && lane > 0;
    const uint32_t continued = __ballot_sync(0xffffffffu, continues);
    const uint32_t leaders = __ballot_sync(0xffffffffu, valid && !continues && lane > 0 && lane <= p.span);
    if (leaders == 0) {
        return;
    }
    auto run_length = [&](uint32_t leader) -> uint32_t {
        return 1 + (leader == 31 ? 0 : __ffs(~(continued >> (leader + 1))) - 1);
    };

    // ---- units: a head of each run ----
    const uint32_t kinds = p.cache.kv_heads;
    const uint32_t units = __popc(leaders) * kinds;
    struct Unit {
        uint8_t* codes;
        float* scale;
        float old_scale;
        uint32_t count;
        uint32_t offset;
        uint32_t first_row;     // of the CTA's rows
    } next = {};
    uint4 raw[PASSES];
    auto load = [&](uint32_t unit) {
        uint32_t rest = leaders;
        for (uint32_t skip = unit / kinds; skip > 0; --skip) rest &= rest - 1;
        const uint32_t leader = __ffs(rest) - 1;
        next.count = run_length(leader);
        const int64_t first_slot = __shfl_sync(0xffffffffu, slot, leader);
        next.first_row = leader - 1;
        const size_t page = static_cast<size_t>(first_slot) / kPageSize;
        next.offset = static_cast<uint32_t>(first_slot % kPageSize);
        const uint32_t head = unit % kinds;
        const __nv_bfloat16* source = (is_value ? p.value : p.key) + static_cast<size_t>(begin + next.first_row) * p.kv_token_stride +
                                      head * DIM;
        next.codes = (is_value ? p.cache.value_codes : p.cache.key_codes) + (page * p.cache.kv_heads + head) * (kPageSize * DIM);
        next.scale = (is_value ? p.cache.value_scales : p.cache.key_scales) + page * p.cache.kv_heads + head;
        next.old_scale = next.offset > 0 ? *next.scale : 0.0f;
#pragma unroll
        for (uint32_t pass = 0; pass < PASSES; ++pass) {
            const uint32_t row = pass * ROWS + lane_row;
            raw[pass] = make_uint4(0, 0, 0, 0);
            if (row < next.count) raw[pass] = load_values<DIM>(source + row * p.kv_token_stride, piece);
        }
    };
    if (warp < units) load(warp);
    Values weight = {};
    if (NORM_ROPE && !is_value) {
        weight = unpack(load_values<DIM>(p.key_norm, piece));
        const uint32_t last = 31 - __clz(leaders);
        angles<DIM, kWarps>(p, begin, last - 1 + run_length(last), turns);
        __syncthreads();
    }
    for (uint32_t unit = warp; unit < units; unit += kWarps) {
        const Unit now = next;
        Values x[PASSES];
        uint32_t largest = 0;
#pragma unroll
        for (uint32_t pass = 0; pass < PASSES; ++pass) {
            if (pass * ROWS < now.count) {
                x[pass] = unpack(raw[pass]);
                if (NORM_ROPE && !is_value) {
                    const uint32_t row = min(pass * ROWS + lane_row, now.count - 1);   // rows that do not exist are zeros
                    norm_rope_row<DIM>(x[pass], weight, turns + (now.first_row + row) * (DIM / 2), piece, p.eps);
                }
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    // infinities and NaN do not move the scale: they become the largest code and the NaN code
                    const uint32_t magnitude = __float_as_uint(i < 4 ? x[pass].low[i % 4] : x[pass].high[i % 4]) & 0x7fffffffu;
                    largest = max(largest, magnitude < 0x7f800000u ? magnitude : 0u);
                }
            }
        }
        if (unit + kWarps < units) load(unit + kWarps);
        largest = __reduce_max_sync(0xffffffffu, largest);
        const float old_scale = stored_scale(now.old_scale);
        int32_t exponent = scale_exponent(largest);
        if (now.offset > 0) exponent = max(exponent, exponent_above(old_scale));

        const float factor = power_of_two(-exponent);
#pragma unroll
        for (uint32_t pass = 0; pass < PASSES; ++pass) {
            const uint32_t row = pass * ROWS + lane_row;
            if (row < now.count) {
                uint8_t* place = now.codes + (now.offset + row) * DIM + 4 * piece;
                *reinterpret_cast<uint32_t*>(place) = four_codes(x[pass].low, factor);
                *reinterpret_cast<uint32_t*>(place + DIM / 2) = four_codes(x[pass].high, factor);
            }
        }
        // what the page holds already goes over to a larger scale
        const float shrink = old_scale * factor;
        if (now.offset > 0 && shrink != 1.0f) {
#pragma unroll 1
            for (uint32_t row = lane_row; row < now.offset; row += ROWS) {
                uint2* place = reinterpret_cast<uint2*>(now.codes + row * DIM + 8 * piece);
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
        if (lane == 0) *now.scale = power_of_two(exponent);
    }
}

template <uint32_t DIM, uint32_t kWarps>
cudaError_t launch_warps(cudaStream_t stream, const WriteParams& params, unsigned int blocks) {
    return params.query != nullptr ? launch_kernel(e4m3_cache_write_kernel<DIM, true, kWarps>, blocks, kWarps * 32, 0, stream, 1, params)
                                   : launch_kernel(e4m3_cache_write_kernel<DIM, false, kWarps>, blocks, kWarps * 32, 0, stream, 1, params);
}

template <uint32_t DIM>
cudaError_t launch_dim(cudaStream_t stream, const WriteParams& params, uint32_t warps, unsigned int blocks) {
    return warps == 4 ? launch_warps<DIM, 4>(stream, params, blocks) : launch_warps<DIM, 8>(stream, params, blocks);
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
    // A CTA of a prompt has one run or two, and a unit for each KV head of them: with fewer than 8 heads, 4 warps (8 prompts of 437 to 512,
    // 4 against 8 warps: 2 heads of 128 4.7 and 6.1 us, 4 of 128 5.2 and 6.6, 8 of 64 5.9 and 5.5; 200 tokens 3.3 and 3.5, 3.5 and
    // 3.7, 3.8 and 3.1; 128 single tokens 3.0 and 3.0, 3.2 and 3.0, 3.8 and 3.1).  With norms a CTA computes its angles first, for which 8 warps
    // are better until many CTAs share an SM (8 query heads on 2 of 128: 200 tokens 6.5 and 5.8 us, 600 6.5 and 6.3, 2400 9.4 and
    // 8.9, 3800 11.6 and 12.7; 16 on 4 of 128: 6.9 and 5.8, 7.2 and 6.7, 12.5 and 11.7, 18.2 and 19.9; 32 on 2 of 64: 4.7 and 4.0, 4.9
    // and 4.7, 7.9 and 8.0, 11.8 and 12.7; 128 single tokens the same to 0.2 us).
    const uint32_t warps = launch.cache.kv_heads < 8 && (launch.query == nullptr || launch.num_tokens >= 8 * 2 * 148) ? 4 : 8;
    // Tokens of a CTA that looks for runs: as many as leave 2 CTAs an SM with keys and 2 with values.  A decode step's tokens
    // then run side by side, and the tokens of a long prompt share the search (3800 tokens: 8 to a CTA 16.0 us, 4 to a CTA 17.3 us;
    // 700 tokens: 2 to a CTA 8.3 us, 1 to a CTA 9.3 us).
    params.span = 1;
    while (params.span < kSpanMost && launch.num_tokens / (2 * params.span) >= 2 * 148) params.span *= 2;
    const size_t run_blocks = (launch.num_tokens + params.span - 1) / params.span;
    size_t query_blocks = 0;
    if (params.query != nullptr) {
        // as many tokens as a CTA's lanes load at once
        const uint32_t rows = kAhead * warps * (256 / launch.cache.head_dim);
        params.query_span = rows / params.query_heads < 1 ? 1 : rows / params.query_heads;
        if (params.query_span > kSpanMost) params.query_span = kSpanMost;
        query_blocks = (launch.num_tokens + params.query_span - 1) / params.query_span;
    }
    if (2 * run_blocks + query_blocks > 0x7fffffffu) {
        return cudaErrorInvalidConfiguration;
    }
    params.query_blocks = static_cast<uint32_t>(query_blocks);
    params.run_blocks = static_cast<uint32_t>(run_blocks);
    const unsigned int blocks = static_cast<unsigned int>(2 * run_blocks + query_blocks);
    return launch.cache.head_dim == 64 ? launch_dim<64>(stream, params, warps, blocks) : launch_dim<128>(stream, params, warps, blocks);
}

}  // namespace lfm25
