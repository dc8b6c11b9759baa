// Attention of single tokens over the 8-bit paged cache: out = softmax(scale * q K^T) V over the keys that the token sees
// (e4m3_visible.cuh), K and V read as E4M3 codes with a power-of-two scale for each page and KV head.
//
// Bound by HBM: 2 * head_dim bytes and 8 / 16 of a scale a key and KV head, against 4 * head_dim flops a query head.  A CTA
// has one (token, KV head) with up to 16 of its query heads, or one share of its pages; its warps take pages in turn and each
// runs an online softmax of its own.
//
// A page (16 keys) is one step of mma.sync m16n8k16 in f16, which holds every E4M3 value:
//   S = Q K^T     A = the query heads as rows, B = K^T.  The order of the reduction is free, so lane (g, t) of the warp
//                 takes dimensions 16 t .. 16 t + 15 (of every 64) of the keys 4 (g / 2) + g % 2 and two further on: 16 bytes
//                 a load, which turn into operands by conversion alone.
//   O^T += V^T P^T   A = V^T, B = P^T, and the fragment of S is that of P^T.  Lane (g, t) takes the keys 4 t .. 4 t + 3
//                 (the order of keys that S has) and head_dim / 8 dimensions of each: two bytes of two keys side by side
//                 are one byte permutation, converted like K.
// Codes travel from global memory to registers, a few pages ahead of their use; nothing passes through shared memory until
// the warps are joined.  The query is brought to f16 by a power of two of its own (largest magnitude in [2^11, 2^12)): bf16
// carries 8 bits, so what is lost lies 2^-36 below the largest element.  Page scales multiply S in front of the exponential
// and the page's P V behind the MMA, both in f32, where a power of two rounds nothing.
//
// The maximum that weights refer to is only raised when a score exceeds it by more than 8 (weights are then at most 2^8,
// which f16 holds): most pages need no exchange between lanes.
//
// Split: with few (token, KV head) pairs the pages of one are shared by the CTAs of a cluster, joined through distributed
// shared memory: no workspace, so calls never share memory, and one launch.
#include "e4m3_cache.cuh"
#include "e4m3_cache.h"
#include "e4m3_visible.cuh"
#include "launch.h"

namespace lfm25 {

namespace {

constexpr uint32_t kWarps = 8;
constexpr uint32_t kThreads = kWarps * 32;
constexpr float kHeadroom = 8.0f;        // log2 of the largest weight against the reference maximum
constexpr float kNoResult = -1.0f;       // sum of a share that met an unassigned page

struct DecodeParams {
    E4m3Cache cache;
    const __nv_bfloat16* query;
    __nv_bfloat16* output;
    const uint32_t* block_tables;
    const uint32_t* request_slots;
    const uint32_t* position_ids;
    const uint32_t* token_order;
    uint64_t block_table_stride;
    uint64_t block_table_rows;
    uint64_t query_token_stride;
    uint32_t num_tokens;
    uint32_t query_heads;
    uint32_t group;        // query heads of a KV head
    uint32_t chunks;       // of at most 16 of them
    uint32_t splits;       // CTAs of a cluster
    uint32_t window;
    uint32_t sinks;
    float scale_log2;
};

__device__ __forceinline__ uint32_t cluster_address(uint32_t local_address, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_address), "r"(rank));
    return remote;
}
__device__ __forceinline__ float load_cluster(uint32_t address) {
    float value;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(value) : "r"(address) : "memory");
    return value;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n"
                 "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One page of one KV head as a lane holds it.
template <uint32_t DIM>
struct PageCodes {
    static constexpr uint32_t C = DIM / 64;
    uint4 key[2][C];         // [key of the pair][64 dimensions]
    uint2 value[4][C];       // [key][8 dimensions of 64 C]
    float key_scale;
    float value_scale;
};

// HEADS: query heads of the CTA, at most 8 or at most 16
template <uint32_t DIM, uint32_t HEADS, uint32_t AHEAD>
__global__ void __launch_bounds__(kThreads, 2)
e4m3_attention_kernel(const DecodeParams p) {
    constexpr uint32_t C = DIM / 64;
    constexpr uint32_t TILES = DIM / 16;         // of 16 dimensions, rows of O^T
    constexpr uint32_t NT = HEADS / 8;           // tiles of 8 heads, columns of O^T
    extern __shared__ float merge[];             // [kWarps][HEADS][DIM + 2]: sums, then maximum and sum of weights
    constexpr uint32_t STRIDE = DIM + 2;
    __shared__ uint32_t unassigned;
    __shared__ float joined[HEADS * STRIDE];     // this CTA's share, for its cluster
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t g = lane >> 2;
    const uint32_t t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();

    // ---- which token, KV head, heads and share; every early exit is one of the whole cluster ----
    const uint32_t split = blockIdx.x % p.splits;
    uint32_t item = blockIdx.x / p.splits;
    const uint32_t chunk = item % p.chunks;
    item /= p.chunks;
    const uint32_t kv_head = item % p.cache.kv_heads;
    item /= p.cache.kv_heads;
    const uint32_t token = p.token_order != nullptr ? p.token_order[item] : item;
    if (token >= p.num_tokens) {
        return;
    }
    const uint64_t table_row = p.request_slots[token];
    const uint32_t position = p.position_ids[token];
    if (table_row >= p.block_table_rows || position >= p.block_table_stride * kPageSize) {
        return;
    }
    const uint32_t* __restrict__ table = p.block_tables + table_row * p.block_table_stride;
    const uint32_t first_head = kv_head * p.group + chunk * 16;
    const uint32_t heads = min(p.group - chunk * 16, HEADS);
    const VisiblePages pages(position, position, p.window, p.sinks);
    const uint32_t share_begin = static_cast<uint32_t>(static_cast<uint64_t>(pages.count) * split / p.splits);
    const uint32_t share_end = static_cast<uint32_t>(static_cast<uint64_t>(pages.count) * (split + 1) / p.splits);
    const uint32_t my_pages = share_end - share_begin > warp ? (share_end - share_begin - warp + kWarps - 1) / kWarps : 0;
    if (threadIdx.x == 0) unassigned = 0;
    __syncthreads();

    // ---- pages: entries 32 at a time, codes AHEAD pages ahead ----
    uint32_t entries = 0;
    uint32_t bad = 0;
    auto look_up = [&](uint32_t iteration) {          // entry of this warp's page number `iteration`
        if (iteration % 32 == 0) {
            const uint32_t index = share_begin + warp + (iteration + lane) * kWarps;
            entries = index < share_end ? __ldg(table + pages.logical(index)) : 0;
            if (entries >= p.cache.num_pages) {
                bad = 1;                              // page 0 in its place; the token gets no result
                entries = 0;
            }
        }
        return __shfl_sync(0xffffffffu, entries, iteration % 32);
    };
    PageCodes<DIM> held[AHEAD];
    auto load = [&](PageCodes<DIM>& page, uint32_t iteration) {
        const size_t tile = static_cast<size_t>(look_up(iteration)) * p.cache.kv_heads + kv_head;
        const uint8_t* keys = p.cache.key_codes + tile * (kPageSize * DIM) + (4 * (g / 2) + g % 2) * DIM + t * 16;
        const uint8_t* values = p.cache.value_codes + tile * (kPageSize * DIM) + 4 * t * DIM + g * (DIM / 8);
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
#pragma unroll
            for (uint32_t c = 0; c < C; ++c) page.key[k][c] = __ldcs(reinterpret_cast<const uint4*>(keys + k * 2 * DIM + c * 64));
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            if constexpr (C == 1) {
                page.value[k][0] = __ldcs(reinterpret_cast<const uint2*>(values + k * DIM));
            } else {
                const uint4 both = __ldcs(reinterpret_cast<const uint4*>(values + k * DIM));
                page.value[k][0] = make_uint2(both.x, both.y);
                page.value[k][C - 1] = make_uint2(both.z, both.w);
            }
        }
        page.key_scale = __ldg(p.cache.key_scales + tile);
        page.value_scale = __ldg(p.cache.value_scales + tile);
    };
#pragma unroll
    for (uint32_t i = 0; i < AHEAD; ++i) {
        if (i < my_pages) load(held[i], i);
    }

    // ---- query: rows g and g + 8 of A, dimensions 64 c + 16 t + 4 ks .. + 3 in step (c, ks) ----
    uint32_t q[2][C][8];
    float query_factor[2];
#pragma unroll
    for (uint32_t half = 0; half < 2; ++half) {
        uint32_t raw[C][8];
        uint32_t largest = 0;
        const bool there = half < NT && g + 8 * half < heads;
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) {
            uint4 part[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
            if (there) {
                const uint4* row = reinterpret_cast<const uint4*>(p.query + token * p.query_token_stride +
                                                                 (first_head + g + 8 * half) * DIM + c * 64 + t * 16);
                part[0] = row[0];
                part[1] = row[1];
            }
            const uint32_t words[8] = {part[0].x, part[0].y, part[0].z, part[0].w, part[1].x, part[1].y, part[1].z, part[1].w};
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                raw[c][i] = words[i];
                const uint32_t low = words[i] & 0x7fffu;
                const uint32_t high = (words[i] >> 16) & 0x7fffu;
                largest = max(largest, max(low < 0x7f80u ? low : 0u, high < 0x7f80u ? high : 0u));
            }
        }
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // the power of two that brings the largest into [2^11, 2^12), within what f32 can multiply by
        const int32_t exponent = min(max(static_cast<int32_t>(largest >> 7) - 127 - 11, -126), 126);
        const float factor = power_of_two(-exponent);
        query_factor[half] = power_of_two(exponent) * p.scale_log2;
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const float2 pair = bf16x2_to_float2(raw[c][i]);
                q[half][c][i] = pack_f16x2(pair.x * factor, pair.y * factor);
            }
        }
    }

    float maximum[NT];          // of head g + 8 n, the reference of its weights (log2 units)
    float sum[NT];              // of this lane's weights
    float2 out[NT][TILES][2];   // [tile of heads][tile][row g or g + 8]: heads 2 t and 2 t + 1
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
        maximum[n] = -INFINITY;
        sum[n] = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < TILES; ++i) out[n][i][0] = out[n][i][1] = make_float2(0.0f, 0.0f);
    }

    auto use = [&](PageCodes<DIM>& page, uint32_t iteration) {
        const uint32_t base = pages.logical(share_begin + warp + iteration * kWarps) * kPageSize;
        // ---- scores: [tile of 8 keys][head g: keys 4 t + 2 tile, + 1; head g + 8: the same] ----
        float s[2][4] = {};
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
#pragma unroll
            for (uint32_t c = 0; c < C; ++c) {
                const uint32_t words[4] = {page.key[k][c].x, page.key[k][c].y, page.key[k][c].z, page.key[k][c].w};
#pragma unroll
                for (uint32_t ks = 0; ks < 4; ++ks) {
                    mma_f16_16816(s[k], q[0][c][2 * ks], NT > 1 ? q[1][c][2 * ks] : 0u, q[0][c][2 * ks + 1],
                                  NT > 1 ? q[1][c][2 * ks + 1] : 0u, e4m3x2_to_f16x2(words[ks]), e4m3x2_high_to_f16x2(words[ks]));
                }
            }
        }
        // ---- mask: only pages at an edge of what the token sees have one ----
        uint32_t seen = 0xfu;                            // of keys base + 4 t ..
        const bool whole = base + kPageSize - 1 <= position && (base >= pages.first_key || base + kPageSize <= p.sinks);
        if (!whole) {
            seen = 0;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t key = base + 4 * t + i;
                if (key <= position && (key >= pages.first_key || key < p.sinks)) {
                    seen |= 1u << i;
                } else {
                    // whatever lies there, a weight of 0 must not meet a NaN
#pragma unroll
                    for (uint32_t c = 0; c < C; ++c) page.value[i][c] = make_uint2(0, 0);
                }
            }
        }
        // ---- weights ----
        uint32_t weights[NT][2];
        bool above = false;
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n) {
            const float factor = page.key_scale * query_factor[n];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                float& x = s[i >> 1][2 * n + (i & 1)];
                x = (seen >> i) & 1 ? x * factor : -INFINITY;
                above = above || x > maximum[n] + kHeadroom;
            }
        }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) {
                float most = fmaxf(fmaxf(s[0][2 * n], s[0][2 * n + 1]), fmaxf(s[1][2 * n], s[1][2 * n + 1]));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                most = fmaxf(most, maximum[n]);
                // a row that has seen nothing yet keeps its sums of 0: exp2(-inf - -inf) is no factor
                const float factor = most == maximum[n] ? 1.0f : fast_exp2(maximum[n] - most);
                maximum[n] = most;
                sum[n] *= factor;
                const float low = __shfl_sync(0xffffffffu, factor, 8 * t);
                const float high = __shfl_sync(0xffffffffu, factor, 8 * t + 4);
#pragma unroll
                for (uint32_t i = 0; i < TILES; ++i) {
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) out[n][i][h] = make_float2(out[n][i][h].x * low, out[n][i][h].y * high);
                }
            }
        }
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n) {
            float w[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                w[i] = (seen >> i) & 1 ? fast_exp2(s[i >> 1][2 * n + (i & 1)] - maximum[n]) : 0.0f;
            }
            weights[n][0] = pack_f16x2(w[0], w[1]);
            weights[n][1] = pack_f16x2(w[2], w[3]);
            // the sum of the weights before their rounding to 11 bits, which averages out over the keys
            sum[n] += (w[0] + w[1]) + (w[2] + w[3]);
        }
        // ---- O^T += scale * V^T P^T ----
        const float scale = page.value_scale;
#pragma unroll
        for (uint32_t tile = 0; tile < TILES; tile += 2) {
            // dimensions 2 tile .. 2 tile + 3 of this lane's DIM / 8: one byte each of a word
            uint32_t word[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) word[k] = tile & 2 ? page.value[k][tile / 4].y : page.value[k][tile / 4].x;
            const uint32_t low[2] = {__byte_perm(word[0], word[1], 0x5140), __byte_perm(word[2], word[3], 0x5140)};
            const uint32_t high[2] = {__byte_perm(word[0], word[1], 0x7362), __byte_perm(word[2], word[3], 0x7362)};
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
                const uint32_t* pair = half ? high : low;
                const uint32_t a0 = e4m3x2_to_f16x2(pair[0]);
                const uint32_t a1 = e4m3x2_high_to_f16x2(pair[0]);
                const uint32_t a2 = e4m3x2_to_f16x2(pair[1]);
                const uint32_t a3 = e4m3x2_high_to_f16x2(pair[1]);
#pragma unroll
                for (uint32_t n = 0; n < NT; ++n) {
                    float d[4] = {};
                    mma_f16_16816(d, a0, a1, a2, a3, weights[n][0], weights[n][1]);
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        float2& o = out[n][tile + half][h];
                        o = make_float2(fmaf(d[2 * h], scale, o.x), fmaf(d[2 * h + 1], scale, o.y));
                    }
                }
            }
        }
    };

    for (uint32_t iteration = 0; iteration < my_pages; iteration += AHEAD) {
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            if (iteration + i < my_pages) {
                use(held[i], iteration + i);
                if (iteration + i + AHEAD < my_pages) load(held[i], iteration + i + AHEAD);
            }
        }
    }
    if (__any_sync(0xffffffffu, bad != 0) && lane == 0) unassigned = 1;

    // ---- join the warps: O^T of lane (g, t) has dimensions DIM / 8 * g + 2 tile + h of the heads 8 n + 2 t, + 1 ----
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
        sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 1);
        sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 2);
        float* mine = merge + warp * HEADS * STRIDE;
        if (t == 0) {
            mine[(8 * n + g) * STRIDE + DIM] = maximum[n];
            mine[(8 * n + g) * STRIDE + DIM + 1] = sum[n];
        }
#pragma unroll
        for (uint32_t i = 0; i < TILES; ++i) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                mine[(8 * n + 2 * t) * STRIDE + (DIM / 8) * g + 2 * i + h] = out[n][i][h].x;
                mine[(8 * n + 2 * t + 1) * STRIDE + (DIM / 8) * g + 2 * i + h] = out[n][i][h].y;
            }
        }
    }
    __syncthreads();
    for (uint32_t index = threadIdx.x; index < heads * DIM; index += kThreads) {
        const uint32_t head = index / DIM;
        const uint32_t dim = index % DIM;
        float most = -INFINITY;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) most = fmaxf(most, merge[(w * HEADS + head) * STRIDE + DIM]);
        const float base = most == -INFINITY ? 0.0f : most;
        float total = 0.0f;
        float value = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
            const float* record = merge + (w * HEADS + head) * STRIDE;
            const float factor = fast_exp2(record[DIM] - base);
            total = fmaf(record[DIM + 1], factor, total);
            value = fmaf(record[dim], factor, value);
        }
        if (p.splits > 1) {
            joined[head * STRIDE + dim] = value;
            if (dim == 0) {
                joined[head * STRIDE + DIM] = most;
                joined[head * STRIDE + DIM + 1] = unassigned ? kNoResult : total;
            }
        } else if (!unassigned) {
            p.output[(static_cast<size_t>(token) * p.query_heads + first_head + head) * DIM + dim] = __float2bfloat16_rn(value / total);
        }
    }
    if (p.splits == 1) {
        return;
    }
    // ---- join the cluster: every CTA writes a part of the heads' elements ----
    cluster_barrier();
    const uint32_t share = (heads * DIM + p.splits - 1) / p.splits;
    const uint32_t end = min((split + 1) * share, heads * DIM);
    const uint32_t own = smem_u32(joined);
    for (uint32_t index = split * share + threadIdx.x; index < end; index += kThreads) {
        const uint32_t head = index / DIM;
        const uint32_t dim = index % DIM;
        float most = -INFINITY;
        for (uint32_t r = 0; r < p.splits; ++r) most = fmaxf(most, load_cluster(cluster_address(own + (head * STRIDE + DIM) * 4, r)));
        const float base = most == -INFINITY ? 0.0f : most;
        float total = 0.0f;
        float value = 0.0f;
        bool valid = true;
        for (uint32_t r = 0; r < p.splits; ++r) {
            const uint32_t record = cluster_address(own + head * STRIDE * 4, r);
            const float factor = fast_exp2(load_cluster(record + DIM * 4) - base);
            const float part = load_cluster(record + (DIM + 1) * 4);
            valid = valid && part != kNoResult;
            total = fmaf(part, factor, total);
            value = fmaf(load_cluster(record + dim * 4), factor, value);
        }
        if (valid) {
            p.output[(static_cast<size_t>(token) * p.query_heads + first_head + head) * DIM + dim] = __float2bfloat16_rn(value / total);
        }
    }
    cluster_barrier();      // nobody leaves while its share is read
}

template <uint32_t DIM, uint32_t HEADS, uint32_t AHEAD>
cudaError_t launch_shape(cudaStream_t stream, const DecodeParams& params, uint64_t blocks) {
    constexpr size_t kShared = sizeof(float) * kWarps * HEADS * (DIM + 2);
    const cudaError_t status = allow_shared_memory<e4m3_attention_kernel<DIM, HEADS, AHEAD>>(kShared);
    if (status != cudaSuccess) {
        return status;
    }
    return launch_kernel(e4m3_attention_kernel<DIM, HEADS, AHEAD>, static_cast<unsigned int>(blocks), kThreads, kShared, stream,
                         params.splits, params);
}

}  // namespace

cudaError_t launch_e4m3_attention(cudaStream_t stream, const E4m3AttentionLaunch& launch) {
    DecodeParams params = {};
    params.cache = launch.cache;
    params.query = static_cast<const __nv_bfloat16*>(launch.query);
    params.output = static_cast<__nv_bfloat16*>(launch.output);
    params.block_tables = launch.block_tables;
    params.request_slots = launch.request_slots;
    params.position_ids = launch.position_ids;
    params.token_order = launch.token_order;
    params.block_table_stride = launch.block_table_stride;
    params.block_table_rows = launch.block_table_rows;
    params.query_token_stride = launch.query_token_stride;
    params.num_tokens = static_cast<uint32_t>(launch.num_tokens);
    params.query_heads = static_cast<uint32_t>(launch.query_heads);
    params.group = params.query_heads / launch.cache.kv_heads;
    params.chunks = (params.group + 15) / 16;
    params.window = launch.window;
    params.sinks = launch.sinks;
    params.scale_log2 = launch.scale * kLog2e;
    const uint64_t items = static_cast<uint64_t>(launch.num_tokens) * launch.cache.kv_heads * params.chunks;
    // pages of the longest context that a token can see
    uint64_t longest = launch.maximum_context_tokens;
    if (launch.window != 0 && longest > static_cast<uint64_t>(launch.window) + launch.sinks) {
        longest = static_cast<uint64_t>(launch.window) + launch.sinks + kPageSize;
    }
    const uint64_t pages = (longest + kPageSize - 1) / kPageSize;
    params.splits = 1;
    while (params.splits < 8 && items * params.splits < 592 && pages >= 2 * params.splits * kWarps) params.splits *= 2;
    const uint64_t blocks = items * params.splits;
    if (blocks > 0x7fffffffu) {
        return cudaErrorInvalidConfiguration;
    }
    if (launch.cache.head_dim == 64) {
        return params.group <= 8 ? launch_shape<64, 8, 3>(stream, params, blocks) : launch_shape<64, 16, 2>(stream, params, blocks);
    }
    return params.group <= 8 ? launch_shape<128, 8, 2>(stream, params, blocks) : launch_shape<128, 16, 1>(stream, params, blocks);
}

}  // namespace lfm25
