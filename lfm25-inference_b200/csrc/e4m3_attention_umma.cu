// Attention of prompts over the 8-bit paged cache on the 5th-generation tensor cores (tcgen05 + tensor memory).
//
// A CTA owns 128 rows: consecutive tokens of one segment times the query heads of one KV head (32 tokens x 4 heads), or one
// share of their keys.  Keys come in stages of 64 (4 pages):
//
//   warps 4-7   pages: E4M3 codes from global memory to registers one stage ahead, converted into the operands of the MMA in
//               shared memory (128-byte swizzle): K to f16 as it is, V to bf16 with its page's scale, both without a rounding
//   warp 8      one thread issues, per stage, S = Q K^T (kind::f16 on f16 operands) and, once the weights are there,
//               O += P V (bf16, P read from tensor memory, V as an MN-major operand); S of the next stage in front of P V of
//               this one, so that the tensor core works while the softmax does
//   warps 0-3   one thread a row: tcgen05.ld S, page scales, mask, exp2, weights back over the scores they came from
//
// O stays in tensor memory: the maximum that weights refer to is only raised when a score exceeds it by more than 8 (log2), and
// only then is O read, scaled and stored.  The query is brought to f16 by a power of two per row, which the scores get back
// together with the page's scale in the multiply-add in front of the exponential.
//
// What bounds it at 64 dimensions is the exponentials (128 rows x 64 keys at 16 a cycle and SM: 512 cycles a stage, the two
// products 256); 128 dimensions double the products.  Two CTAs share an SM, so that one's softmax fills the other's waits.
//
// Rows of a mask edge test bits of their own; a NaN among the values is replaced in the operand (a weight of 0 times NaN is
// NaN) and remembered by key: a row that sees it becomes NaN as a whole.  Few tiles: a cluster shares a tile's keys and joins
// through distributed shared memory.  Every wait is bounded; if one runs out, the tile keeps its output rows.
#include <cstddef>

#include "e4m3_cache.cuh"
#include "e4m3_cache.h"
#include "e4m3_visible.cuh"
#include "launch.h"
#include "tcgen05.cuh"

namespace lfm25 {

namespace {

constexpr uint32_t kRows = 128;
constexpr uint32_t kPagesPerStage = 4;
constexpr uint32_t kKeys = kPagesPerStage * kPageSize;     // 64
constexpr uint32_t kThreads = 288;
constexpr uint32_t kBuffers = 2;
constexpr uint32_t kTmemColumns = 256;
constexpr uint32_t kColumnS = 0;                           // two buffers of 64; weights take the first 32 columns of theirs
constexpr uint32_t kColumnO = 128;
constexpr float kHeadroom = 8.0f;
constexpr uint32_t kTile = kKeys * 128;                    // 64 keys x 64 dimensions of 2 bytes

struct PromptParams {
    E4m3Cache cache;
    const __nv_bfloat16* query;
    __nv_bfloat16* output;
    const uint32_t* block_tables;
    const uint32_t* request_slots;
    const uint32_t* position_ids;
    const uint32_t* segment_offsets;
    unsigned int* status;
    uint64_t block_table_stride;
    uint64_t block_table_rows;
    uint64_t query_token_stride;
    uint32_t num_tokens;
    uint32_t num_segments;
    uint32_t query_heads;
    uint32_t group;
    uint32_t chunk_heads;    // query heads of a tile
    uint32_t chunks;
    uint32_t tile_tokens;    // kRows / chunk_heads
    uint32_t splits;         // CTAs of a cluster
    uint32_t window;
    uint32_t sinks;
    float scale_log2;
    uint64_t wait_limit_ns;
    uint32_t selftest_drop;  // self-test of the bounded waits: one page warp never reports its first stage
};

template <uint32_t DIM>
struct Layout {
    static constexpr uint32_t kParts = DIM / 64;
    static constexpr uint32_t kQ = 0;                                         // [part][row] of 128 bytes
    static constexpr uint32_t kK = kQ + kParts * kRows * 128;                 // [buffer][part][key]
    static constexpr uint32_t kV = kK + kBuffers * kParts * kTile;
    static constexpr uint32_t kControl = kV + kBuffers * kParts * kTile;
    static constexpr uint32_t kBytes = kControl + 512 + 3 * kRows * 4;
    static constexpr uint32_t kAlloc = kBytes + 1024;
};

// beside the operands
struct Control {
    uint64_t full[kBuffers];       // operands of a stage are there
    uint64_t empty[kBuffers];      // its P V is done with them
    uint64_t scores[2];
    uint64_t weights[2];
    uint64_t product;              // P V of a stage is complete
    uint64_t drained;              // after a wait ran out: no MMA is in flight any more
    alignas(16) float key_scales[kBuffers][kPagesPerStage];   // read four at a time
    alignas(16) unsigned long long nan_keys[kBuffers][4];   // of each page warp: keys of the stage with a NaN among their values
    uint32_t bad_pages[kBuffers];  // unassigned pages of the stage, one bit each
    uint32_t tmem;
    uint32_t abort;
};
static_assert(offsetof(Control, key_scales) % 16 == 0, "scales are read 16 bytes at a time");
static_assert(sizeof(Control) <= 512, "the control block has 512 bytes");

__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void store_shared(uint32_t address, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n"
                 "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_cluster(uint32_t local_address, uint32_t rank) {
    uint32_t remote;
    float value;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local_address), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(value) : "r"(remote) : "memory");
    return value;
}

// bits of the keys base .. base + 15 that a token at `position` sees
__device__ __forceinline__ uint32_t visible_bits(uint32_t base, uint32_t position, uint32_t first_key, uint32_t sinks) {
    if (base > position) return 0;
    const uint32_t below = position - base >= 15 ? 0xffffu : (2u << (position - base)) - 1;
    const uint32_t outside = first_key <= base ? 0u : first_key - base >= 16 ? 0xffffu : (1u << (first_key - base)) - 1;
    const uint32_t kept = sinks <= base ? 0u : sinks - base >= 16 ? 0xffffu : (1u << (sinks - base)) - 1;
    return below & (~outside | kept);
}

template <uint32_t DIM>
__global__ void __launch_bounds__(kThreads, 2)
e4m3_prompt_attention_kernel(const PromptParams p) {
    using L = Layout<DIM>;
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const uint32_t lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();

    // ---- which tile: segments 32 at a time.  Later tiles have more keys: the grid runs backwards ----
    const uint32_t split = blockIdx.x % p.splits;
    uint32_t item = (gridDim.x / p.splits) - 1 - blockIdx.x / p.splits;
    const uint32_t chunk = item % p.chunks;
    item /= p.chunks;
    const uint32_t kv_head = item % p.cache.kv_heads;
    uint32_t slot = item / p.cache.kv_heads;
    uint32_t segment_begin = 0;
    uint32_t segment_end = 0;
    bool found = false;
    for (uint32_t first = 0; first < p.num_segments && !found; first += 32) {
        const uint32_t segment = first + lane;
        uint32_t begin = 0;
        uint32_t end = 0;
        if (segment < p.num_segments) {
            begin = __ldg(p.segment_offsets + segment);
            end = __ldg(p.segment_offsets + segment + 1);
            if (end <= begin || end > p.num_tokens) end = begin = 0;
        }
        const uint32_t tiles = (end - begin + p.tile_tokens - 1) / p.tile_tokens;
        uint32_t upto = tiles;
#pragma unroll
        for (uint32_t delta = 1; delta < 32; delta <<= 1) {
            const uint32_t other = __shfl_up_sync(0xffffffffu, upto, delta);
            if (lane >= delta) upto += other;
        }
        const uint32_t here = __ballot_sync(0xffffffffu, slot < upto);
        if (here != 0) {
            const uint32_t source = __ffs(here) - 1;
            segment_begin = __shfl_sync(0xffffffffu, begin, source);
            segment_end = __shfl_sync(0xffffffffu, end, source);
            slot -= __shfl_sync(0xffffffffu, upto - tiles, source);
            found = true;
        } else {
            slot -= __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    if (!found) {
        return;
    }
    const uint32_t tile_begin = segment_begin + slot * p.tile_tokens;
    const uint32_t tile_end = min(tile_begin + p.tile_tokens, segment_end);
    const uint32_t table_row = p.request_slots[segment_begin];
    const uint64_t origin = p.position_ids[segment_begin];            // position of the segment's first token
    const uint64_t first_wide = origin + (tile_begin - segment_begin);
    const uint64_t most = p.block_table_stride * kPageSize;
    if (table_row >= p.block_table_rows || first_wide >= most) {
        return;
    }
    const uint32_t first_position = static_cast<uint32_t>(first_wide);
    // tokens behind the end of the table have no result; those in front of it do
    const uint32_t last_position = static_cast<uint32_t>(min(first_wide + (tile_end - tile_begin), most) - 1);
    const VisiblePages pages(first_position, last_position, p.window, p.sinks);
    const uint32_t* __restrict__ table = p.block_tables + static_cast<uint64_t>(table_row) * p.block_table_stride;
    const uint32_t all_stages = (pages.count + kPagesPerStage - 1) / kPagesPerStage;
    const uint32_t begin_stage = static_cast<uint32_t>(static_cast<uint64_t>(all_stages) * split / p.splits);
    const uint32_t stages = static_cast<uint32_t>(static_cast<uint64_t>(all_stages) * (split + 1) / p.splits) - begin_stage;

    extern __shared__ uint8_t prompt_smem[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(prompt_smem) + 1023) & ~uintptr_t(1023));
    const uint32_t base = smem_u32(smem);
    Control* control = reinterpret_cast<Control*>(smem + L::kControl);
    volatile uint32_t* abort = &control->abort;
    float* joined = reinterpret_cast<float*>(smem + L::kControl + 512);   // maximum, sum, result of each row
    const uint32_t bar_full = smem_u32(control->full);
    const uint32_t bar_empty = smem_u32(control->empty);
    const uint32_t bar_scores = smem_u32(control->scores);
    const uint32_t bar_weights = smem_u32(control->weights);
    const uint32_t bar_product = smem_u32(&control->product);

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(bar_full + 8 * i, 4);
            mbar_init(bar_empty + 8 * i, 1);
            mbar_init(bar_scores + 8 * i, 1);
            mbar_init(bar_weights + 8 * i, 4);
        }
        mbar_init(bar_product, 1);
        mbar_init(smem_u32(&control->drained), 1);
        control->abort = 0;
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_allocate(smem_u32(&control->tmem), kTmemColumns);
    }

    // ---- rows: this thread's token and head, its query in f16 ----
    const uint32_t row = threadIdx.x;                    // of the softmax warps
    const uint32_t row_token = tile_begin + row / p.chunk_heads;
    const uint32_t head = chunk * p.chunk_heads + row % p.chunk_heads;   // of the group
    const uint64_t row_wide = first_wide + (row_token - tile_begin);
    bool live = false;
    float row_factor = 0.0f;
    if (warp < 4) {
        live = row < p.tile_tokens * p.chunk_heads && row_token < tile_end && head < p.group && row_wide < most;
        if (live) live = p.request_slots[row_token] == table_row && p.position_ids[row_token] == row_wide;
        const __nv_bfloat16* source = p.query + row_token * p.query_token_stride + static_cast<size_t>(kv_head * p.group + head) * DIM;
        // two passes over the row, so that it need not stay in registers
        uint32_t largest = 0;
#pragma unroll
        for (uint32_t c = 0; c < DIM / 8; ++c) {
            const uint4 raw = live ? reinterpret_cast<const uint4*>(source)[c] : make_uint4(0, 0, 0, 0);
            const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t low = words[i] & 0x7fffu;
                const uint32_t high = (words[i] >> 16) & 0x7fffu;
                largest = max(largest, max(low < 0x7f80u ? low : 0u, high < 0x7f80u ? high : 0u));
            }
        }
        const int32_t exponent = min(max(static_cast<int32_t>(largest >> 7) - 127 - 11, -126), 126);
        const float factor = power_of_two(-exponent);
        row_factor = power_of_two(exponent) * p.scale_log2;
#pragma unroll
        for (uint32_t c = 0; c < DIM / 8; ++c) {
            const uint4 raw = live ? reinterpret_cast<const uint4*>(source)[c] : make_uint4(0, 0, 0, 0);
            const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
            uint32_t half[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const float2 pair = bf16x2_to_float2(words[i]);
                half[i] = pack_f16x2(pair.x * factor, pair.y * factor);
            }
            store_shared(base + L::kQ + (c / 8) * (kRows * 128) + row * 128 + (((c % 8) ^ (row & 7)) << 4),
                         make_uint4(half[0], half[1], half[2], half[3]));
        }
        fence_proxy_async_smem();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = control->tmem;

    // a row's running state (softmax warps)
    float reference = -INFINITY;
    float sum = 0.0f;
    bool poisoned = false;       // sees a NaN value
    bool lost = false;           // sees an unassigned page
    bool ok = true;

    if (warp >= 4 && warp < 8) {
        // -------------------------------------------------------------------------------- pages
        constexpr uint32_t kPieces = DIM / 16;                       // of 16 codes, of a key
        constexpr uint32_t kLoads = kKeys * kPieces / 128;           // a thread, for K and for V
        const uint32_t thread = threadIdx.x - 128;
        const uint32_t page_warp = warp - 4;
        uint4 key_codes[kLoads];
        uint4 value_codes[kLoads];
        float value_scale[kLoads];
        float key_scale = 0.0f;
        uint32_t bad = 0;
        auto load = [&](uint32_t stage) {
            const uint32_t first = (begin_stage + stage) * kPagesPerStage;
            bad = 0;
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const uint32_t piece = i * 128 + thread;
                const uint32_t key = piece / kPieces;
                const uint32_t index = first + key / kPageSize;
                uint32_t entry = 0xffffffffu;
                if (index < pages.count) {
                    entry = __ldg(table + pages.logical(index));
                    if (entry >= p.cache.num_pages) bad |= 1u << (key / kPageSize);
                }
                if (entry < p.cache.num_pages) {
                    const size_t tile = static_cast<size_t>(entry) * p.cache.kv_heads + kv_head;
                    const size_t offset = tile * (kPageSize * DIM) + (key % kPageSize) * DIM + (piece % kPieces) * 16;
                    key_codes[i] = __ldg(reinterpret_cast<const uint4*>(p.cache.key_codes + offset));
                    value_codes[i] = __ldg(reinterpret_cast<const uint4*>(p.cache.value_codes + offset));
                    value_scale[i] = __ldg(p.cache.value_scales + tile);
                } else {
                    key_codes[i] = value_codes[i] = make_uint4(0, 0, 0, 0);
                    value_scale[i] = 0.0f;
                }
            }
            if (thread < kPagesPerStage) {
                const uint32_t index = first + thread;
                key_scale = 0.0f;
                if (index < pages.count) {
                    const uint32_t entry = __ldg(table + pages.logical(index));
                    if (entry < p.cache.num_pages) {
                        key_scale = __ldg(p.cache.key_scales + static_cast<size_t>(entry) * p.cache.kv_heads + kv_head);
                    }
                }
            }
        };
        if (stages > 0) load(0);
        for (uint32_t stage = 0; stage < stages; ++stage) {
            const uint32_t buffer = stage % kBuffers;
            if (stage >= kBuffers) {
                ok = *abort == 0 && mbar_wait_bounded(bar_empty + 8 * buffer, (stage / kBuffers - 1) & 1, p.wait_limit_ns);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
            }
            unsigned long long nan_keys = 0;
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const uint32_t piece = i * 128 + thread;
                const uint32_t key = piece / kPieces;
                const uint32_t dims = piece % kPieces;               // 16 dimensions: two pieces of 16 bytes
                const uint32_t place = (dims / 4) * kTile + key * 128;
                const uint32_t at[2] = {place + (((2 * dims % 8) ^ (key & 7)) << 4), place + (((2 * dims % 8 + 1) ^ (key & 7)) << 4)};
                const uint32_t k_words[4] = {key_codes[i].x, key_codes[i].y, key_codes[i].z, key_codes[i].w};
                const uint32_t k_base = base + L::kK + buffer * (L::kParts * kTile);
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    store_shared(k_base + at[h], make_uint4(e4m3x2_to_f16x2(k_words[2 * h]), e4m3x2_high_to_f16x2(k_words[2 * h]),
                                                            e4m3x2_to_f16x2(k_words[2 * h + 1]), e4m3x2_high_to_f16x2(k_words[2 * h + 1])));
                }
                uint32_t v_words[4] = {value_codes[i].x, value_codes[i].y, value_codes[i].z, value_codes[i].w};
                uint32_t odd = 0;
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) odd |= (v_words[w] & 0x7f7f7f7fu) + 0x01010101u;
                odd = (odd & 0x80808080u) != 0;
                if (__any_sync(0xffffffffu, odd)) {
                    // codes that are NaN become 0, and their keys are remembered
                    uint32_t lanes = __ballot_sync(0xffffffffu, odd);
                    const uint32_t first_key = (i * 128 + (thread & ~31u)) / kPieces;
                    while (lanes != 0) {
                        nan_keys |= 1ull << (first_key + (__ffs(lanes) - 1) / kPieces);
                        lanes &= lanes - 1;
                    }
#pragma unroll
                    for (uint32_t w = 0; w < 4; ++w) {
                        const uint32_t hit = (((v_words[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                        v_words[w] &= ~(hit * 0xffu);
                    }
                }
                const uint32_t v_base = base + L::kV + buffer * (L::kParts * kTile);
                const float scale = value_scale[i];
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    uint32_t pairs[4];
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t word = v_words[2 * h + j / 2];
                        const float2 x = f16x2_to_float2(j % 2 ? e4m3x2_high_to_f16x2(word) : e4m3x2_to_f16x2(word));
                        pairs[j] = pack_bf16x2(x.x * scale, x.y * scale);
                    }
                    store_shared(v_base + at[h], make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]));
                }
            }
            if (thread < kPagesPerStage) control->key_scales[buffer][thread] = key_scale;
            if (lane == 0) control->nan_keys[buffer][page_warp] = nan_keys;
            // bits of all four warps' pages: every warp of 64 dimensions has two pages a load, so one word a warp is joined by
            // the reader below
            const uint32_t warp_bad = __reduce_or_sync(0xffffffffu, bad);
            if (lane == 0) reinterpret_cast<uint8_t*>(&control->bad_pages[buffer])[page_warp] = static_cast<uint8_t>(warp_bad);
            if (stage + 1 < stages) load(stage + 1);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && !(p.selftest_drop != 0 && warp == 4 && stage == 0)) mbar_arrive(bar_full + 8 * buffer);
        }
        if (!ok && lane == 0 && *abort == 0) {
            *abort = 1;
            record_wait_timeout(p.status, kTagE4m3Prompt, (blockIdx.x << 2) | 1);
        }
    } else if (warp == 8) {
        // -------------------------------------------------------------------------------- MMA issuer
        if (elect_one()) {
            // f32 results of 128 rows; Q K^T: f16, both K-major, 64 keys; P V: bf16, V MN-major, 64 dimensions
            const uint32_t idesc_scores = (1u << 4) | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);
            const uint32_t idesc_product = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((64u >> 3) << 17) | ((kRows >> 4) << 24);
            const uint64_t q_desc = smem_descriptor(base + L::kQ);
            bool running = true;
            auto issue_scores = [&](uint32_t stage) -> bool {
                const uint32_t buffer = stage % kBuffers;
                if (*abort || !mbar_wait_bounded(bar_full + 8 * buffer, (stage / kBuffers) & 1, p.wait_limit_ns)) {
                    return false;
                }
                tcgen05_fence_after();
                const uint64_t k_desc = smem_descriptor(base + L::kK + buffer * (L::kParts * kTile));
#pragma unroll
                for (uint32_t ks = 0; ks < DIM / 16; ++ks) {   // 16 dimensions: 32 bytes within the swizzled row
                    umma_ss(tmem + kColumnS + buffer * kKeys, q_desc + (ks / 4) * (kRows * 128 >> 4) + (ks % 4) * 2,
                            k_desc + (ks / 4) * (kTile >> 4) + (ks % 4) * 2, idesc_scores, ks);
                }
                umma_commit(bar_scores + 8 * buffer);
                return true;
            };
            running = stages == 0 || issue_scores(0);
            for (uint32_t stage = 0; stage < stages && running; ++stage) {
                const uint32_t buffer = stage % kBuffers;
                // scores of the next stage first.  Their columns are free: the weights in them were consumed by a P V that was
                // issued before, and MMAs execute in order
                if (stage + 1 < stages && !issue_scores(stage + 1)) {
                    running = false;
                    break;
                }
                if (*abort || !mbar_wait_bounded(bar_weights + 8 * buffer, (stage >> 1) & 1, p.wait_limit_ns)) {
                    running = false;
                    break;
                }
                tcgen05_fence_after();
#pragma unroll
                for (uint32_t part = 0; part < L::kParts; ++part) {
                    const uint64_t v_desc = smem_descriptor(base + L::kV + (buffer * L::kParts + part) * kTile);
#pragma unroll
                    for (uint32_t step = 0; step < kPagesPerStage; ++step) {   // 16 keys: 8 columns of weights, 2 KiB of V
                        umma_ts(tmem + kColumnO + part * 64, tmem + kColumnS + buffer * kKeys + step * 8, v_desc + step * (2048 >> 4),
                                idesc_product, stage > 0 || step > 0);
                    }
                }
                umma_commit(bar_product);
                umma_commit(bar_empty + 8 * buffer);
            }
            if (!running && *abort == 0) {
                *abort = 1;
                record_wait_timeout(p.status, kTagE4m3Prompt, (blockIdx.x << 2) | 2);
            }
            if (*abort != 0) {
                umma_commit(smem_u32(&control->drained));
                (void)mbar_wait_bounded(smem_u32(&control->drained), 0, p.wait_limit_ns);
            }
        }
    } else {
        // -------------------------------------------------------------------------------- softmax
        const uint32_t position = live ? static_cast<uint32_t>(row_wide) : last_position;
        const uint32_t first_key = p.window != 0 && position >= p.window ? position - p.window + 1 : 0;
        const uint32_t lane_address = tmem + ((warp * 32) << 16);
        for (uint32_t stage = 0; stage < stages; ++stage) {
            const uint32_t buffer = stage & 1;
            // the scores, and the page warps' own words beside them (complete by then)
            ok = *abort == 0 && mbar_wait_bounded(bar_scores + 8 * buffer, (stage >> 1) & 1, p.wait_limit_ns) &&
                 mbar_wait_bounded(bar_full + 8 * buffer, (stage >> 1) & 1, p.wait_limit_ns);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            tcgen05_fence_after();
            const uint32_t columns = lane_address + kColumnS + buffer * kKeys;
            uint32_t raw[4][16];
#pragma unroll
            for (uint32_t part = 0; part < 4; ++part) tmem_load16_nowait(columns + part * 16, raw[part]);
            // ---- what this row sees of the stage ----
            const uint32_t index = (begin_stage + stage) * kPagesPerStage;
            const uint32_t stage_key = pages.logical(index) * kPageSize;
            const bool together = index + kPagesPerStage <= pages.count && (index >= pages.sink_pages || index + kPagesPerStage <= pages.sink_pages);
            const bool whole = together && position >= stage_key + kKeys - 1 && (first_key <= stage_key || p.sinks >= stage_key + kKeys);
            const bool fast = __all_sync(0xffffffffu, whole);
            uint32_t bits[2] = {0xffffffffu, 0xffffffffu};
            if (!fast) {
#pragma unroll
                for (uint32_t sub = 0; sub < kPagesPerStage; ++sub) {
                    const uint32_t seen = index + sub < pages.count
                                              ? visible_bits(pages.logical(index + sub) * kPageSize, position, first_key, p.sinks) : 0u;
                    bits[sub / 2] = sub % 2 ? bits[sub / 2] & ((seen << 16) | 0xffffu) : bits[sub / 2] & (seen | 0xffff0000u);
                }
            }
            const float4 scales = *reinterpret_cast<const float4*>(control->key_scales[buffer]);
            const float factor[4] = {row_factor * scales.x, row_factor * scales.y, row_factor * scales.z, row_factor * scales.w};
            {
                const unsigned long long* nan = control->nan_keys[buffer];
                const unsigned long long odd = (nan[0] | nan[1]) | (nan[2] | nan[3]);
                const uint32_t bad = control->bad_pages[buffer];
                if (odd != 0 || bad != 0) {
                    const unsigned long long seen = bits[0] | (static_cast<unsigned long long>(bits[1]) << 32);
                    poisoned = poisoned || (odd & seen) != 0;
                    const uint32_t all = (bad | (bad >> 8) | (bad >> 16) | (bad >> 24)) & 0xfu;
#pragma unroll
                    for (uint32_t sub = 0; sub < kPagesPerStage; ++sub) {
                        lost = lost || (((all >> sub) & 1) != 0 && ((seen >> (16 * sub)) & 0xffffu) != 0);
                    }
                }
            }
            tmem_load_wait();
            // ---- maximum ----
            if (!fast) {
                // masked scores, whatever they are, become -inf (the factor is positive or 0, so not by the product)
#pragma unroll
                for (uint32_t j = 0; j < kKeys; ++j) {
                    if (((bits[j / 32] >> (j % 32)) & 1) == 0) raw[j / 16][j % 16] = 0xff800000u;
                }
            }
            float most = -INFINITY;
#pragma unroll
            for (uint32_t sub = 0; sub < kPagesPerStage; ++sub) {
                float a = __uint_as_float(raw[sub][0]);
                float b = __uint_as_float(raw[sub][1]);
#pragma unroll
                for (uint32_t j = 2; j < 16; j += 4) {
                    a = max3(a, __uint_as_float(raw[sub][j]), __uint_as_float(raw[sub][j + 1]));
                    if (j + 2 < 16) b = max3(b, __uint_as_float(raw[sub][j + 2]), __uint_as_float(raw[sub][j + 3]));
                }
                const float here = fmaxf(a, b);
                most = fmaxf(most, here * factor[sub]);
            }
            const bool raise = most > reference + kHeadroom;
            if (__any_sync(0xffffffffu, raise)) {
                const float shrink = !raise ? 1.0f : reference == -INFINITY ? 0.0f : fast_exp2(reference - most);
                if (raise) reference = most;
                sum *= shrink;
                if (stage > 0) {
                    ok = *abort == 0 && mbar_wait_bounded(bar_product, (stage - 1) & 1, p.wait_limit_ns);
                    if (!__all_sync(0xffffffffu, ok)) {
                        ok = false;
                        break;
                    }
                    tcgen05_fence_after();
#pragma unroll
                    for (uint32_t c = 0; c < DIM; c += 16) {
                        uint32_t o[16];
                        tmem_load16(lane_address + kColumnO + c, o);
#pragma unroll
                        for (uint32_t j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
                        tmem_store16(lane_address + kColumnO + c, o);
                    }
                }
            }
            // ---- weights ----
            const float offset = reference == -INFINITY ? 0.0f : -reference;
            float2 part_sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
                uint32_t packed[16];
#pragma unroll
                for (uint32_t pair = 0; pair < 16; ++pair) {
                    const uint32_t j = half * 32 + pair * 2;
                    float2 w = fma_two(make_float2(__uint_as_float(raw[j / 16][j % 16]), __uint_as_float(raw[j / 16][j % 16 + 1])),
                                       factor[j / 16], offset);
                    w = make_float2(fast_exp2(w.x), fast_exp2(w.y));
                    if (!fast) {
                        w.x = (bits[j / 32] >> (j % 32)) & 1 ? w.x : 0.0f;
                        w.y = (bits[j / 32] >> (j % 32 + 1)) & 1 ? w.y : 0.0f;
                    }
                    packed[pair] = pack_bf16x2(w.x, w.y);
                    part_sum[pair & 1] = add_two(part_sum[pair & 1], w);   // unrounded: the roundings of many weights average out
                }
                tmem_store16(columns + half * 16, packed);
            }
            part_sum[0] = add_two(part_sum[0], part_sum[1]);
            sum += part_sum[0].x + part_sum[0].y;
            tmem_store_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_weights + 8 * buffer);
        }
        if (ok && stages > 0) {
            ok = *abort == 0 && mbar_wait_bounded(bar_product, (stages - 1) & 1, p.wait_limit_ns);
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok && lane == 0 && *abort == 0) {
            *abort = 1;
            record_wait_timeout(p.status, kTagE4m3Prompt, (blockIdx.x << 2) | 3);
        }
        tcgen05_fence_after();
        if (poisoned) sum = __int_as_float(0x7fc00000);
        const size_t out_row = (static_cast<size_t>(row_token) * p.query_heads + kv_head * p.group + head) * DIM;
        if (p.splits == 1) {
            const float inverse = 1.0f / sum;
#pragma unroll
            for (uint32_t c = 0; c < DIM; c += 16) {
                uint32_t o[16];
                tmem_load16(lane_address + kColumnO + c, o);
                if (ok && live && !lost && *abort == 0) {
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        uint32_t pairs[4];
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) {
                            pairs[j] = pack_bf16x2(__uint_as_float(o[h * 8 + 2 * j]) * inverse, __uint_as_float(o[h * 8 + 2 * j + 1]) * inverse);
                        }
                        *reinterpret_cast<uint4*>(p.output + out_row + c + h * 8) = make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]);
                    }
                }
            }
        }
    }

    // single-lane roles meet their warps again in front of the CTA's barrier
    __syncwarp();
    if (p.splits > 1) {
        // ---- join the cluster: unscaled sums, one column of 128 rows behind the other, where the operands were ----
        __syncthreads();                   // nobody writes operands any more, and the MMAs have been waited for
        float* sums = reinterpret_cast<float*>(smem);
        if (warp < 4) {
            const uint32_t lane_address = tmem + ((warp * 32) << 16);
            const bool valid = ok && !lost && *abort == 0;
#pragma unroll
            for (uint32_t c = 0; c < DIM; c += 16) {
                uint32_t o[16];
                tmem_load16(lane_address + kColumnO + c, o);
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) sums[(c + j) * kRows + row] = stages > 0 ? __uint_as_float(o[j]) : 0.0f;
            }
            joined[row] = reference;
            joined[kRows + row] = sum;
            joined[2 * kRows + row] = valid ? 1.0f : 0.0f;
        }
        __syncwarp();
        cluster_barrier();
        if (warp < 4) {
            const uint32_t own = smem_u32(joined) + row * 4;
            float most = -INFINITY;
            bool valid = live;
            for (uint32_t r = 0; r < p.splits; ++r) {
                most = fmaxf(most, load_cluster(own, r));
                valid = valid && load_cluster(own + 2 * kRows * 4, r) != 0.0f;
            }
            const float offset = most == -INFINITY ? 0.0f : most;
            float total = 0.0f;
            float weight[8];
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) {
                weight[r] = 0.0f;
                if (r < p.splits) {
                    weight[r] = fast_exp2(load_cluster(own, r) - offset);
                    total = fmaf(load_cluster(own + kRows * 4, r), weight[r], total);
                }
            }
            const float inverse = 1.0f / total;
            const uint32_t share = DIM / p.splits;       // 8 dimensions or more
            const size_t out_row = (static_cast<size_t>(row_token) * p.query_heads + kv_head * p.group + head) * DIM;
            for (uint32_t c = split * share; c < (split + 1) * share; c += 8) {
                float value[8] = {};
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r) {
                    if (r < p.splits) {
#pragma unroll
                        for (uint32_t j = 0; j < 8; ++j) {
                            value[j] = fmaf(load_cluster(base + ((c + j) * kRows + row) * 4, r), weight[r], value[j]);
                        }
                    }
                }
                if (valid) {
                    uint4 out;
                    out.x = pack_bf16x2(value[0] * inverse, value[1] * inverse);
                    out.y = pack_bf16x2(value[2] * inverse, value[3] * inverse);
                    out.z = pack_bf16x2(value[4] * inverse, value[5] * inverse);
                    out.w = pack_bf16x2(value[6] * inverse, value[7] * inverse);
                    *reinterpret_cast<uint4*>(p.output + out_row + c) = out;
                }
            }
        }
        __syncwarp();
        cluster_barrier();                 // nobody leaves while its sums are read
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 8) {
        tmem_free(tmem, kTmemColumns);
    }
}

template <uint32_t DIM>
cudaError_t launch_dim(cudaStream_t stream, const PromptParams& params, uint64_t blocks) {
    const cudaError_t status = allow_shared_memory<e4m3_prompt_attention_kernel<DIM>>(Layout<DIM>::kAlloc);
    if (status != cudaSuccess) {
        return status;
    }
    return launch_kernel(e4m3_prompt_attention_kernel<DIM>, static_cast<unsigned int>(blocks), kThreads, Layout<DIM>::kAlloc, stream,
                         params.splits, params);
}

}  // namespace

cudaError_t launch_e4m3_prompt_attention(cudaStream_t stream, const E4m3AttentionLaunch& launch) {
    PromptParams params = {};
    params.cache = launch.cache;
    params.query = static_cast<const __nv_bfloat16*>(launch.query);
    params.output = static_cast<__nv_bfloat16*>(launch.output);
    params.block_tables = launch.block_tables;
    params.request_slots = launch.request_slots;
    params.position_ids = launch.position_ids;
    params.segment_offsets = launch.segment_offsets;
    params.status = launch.status;
    params.block_table_stride = launch.block_table_stride;
    params.block_table_rows = launch.block_table_rows;
    params.query_token_stride = launch.query_token_stride;
    params.num_tokens = static_cast<uint32_t>(launch.num_tokens);
    params.num_segments = static_cast<uint32_t>(launch.num_segments);
    params.query_heads = static_cast<uint32_t>(launch.query_heads);
    params.group = params.query_heads / launch.cache.kv_heads;
    params.chunk_heads = params.group < kRows ? params.group : kRows;
    params.chunks = (params.group + params.chunk_heads - 1) / params.chunk_heads;
    params.tile_tokens = kRows / params.chunk_heads;
    params.window = launch.window;
    params.sinks = launch.sinks;
    params.scale_log2 = launch.scale * kLog2e;
    params.wait_limit_ns = wait_limit_ns();
    params.selftest_drop = wait_selftest_drop() ? 1 : 0;
    // at most so many tiles: full ones, and one that is not for each segment
    const uint64_t tiles = launch.num_tokens / params.tile_tokens + launch.num_segments;
    const uint64_t items = tiles * launch.cache.kv_heads * params.chunks;
    uint64_t longest = launch.maximum_context_tokens;
    if (launch.window != 0 && longest > static_cast<uint64_t>(launch.window) + launch.sinks + params.tile_tokens) {
        longest = static_cast<uint64_t>(launch.window) + launch.sinks + params.tile_tokens;
    }
    params.splits = 1;
    while (params.splits < 8 && items * params.splits * 2 <= 296 && longest >= 4 * kKeys * params.splits) params.splits *= 2;
    const uint64_t blocks = items * params.splits;
    if (blocks > 0x7fffffffu) {
        return cudaErrorInvalidConfiguration;
    }
    return launch.cache.head_dim == 64 ? launch_dim<64>(stream, params, blocks) : launch_dim<128>(stream, params, blocks);
}

}  // namespace lfm25
