// Attention of prompts over the 8-bit paged cache on the 5th-generation tensor cores (tcgen05 + tensor memory).
//
// A CTA owns two tiles of 128 rows: consecutive tokens of one segment times the query heads of one KV head (2 x 32 tokens x 4
// heads), or one share of their keys.  Keys come in stages of 64 (4 pages), converted once for both tiles:
//
//   page warps (4)      E4M3 codes by asynchronous copies two stages ahead, then converted into the operands of the MMA in shared
//                       memory (128-byte swizzle): K to f16 as it is, V to bf16 with its page's scale, both without a rounding (below
//                       2^-124 a scale leaves the smallest codes less than bf16 holds: 2^-134 off at most)
//   issuing warps (2)   one for each tile, per stage S = Q K^T (kind::f16 on f16 operands) and, once the weights are there, O += P V
//                       (bf16, P read from tensor memory, V as an MN-major operand); S of two stages on right behind P V of this
//                       one, so that the tensor core works while the softmax does
//   softmax warps (16)  one thread a row, four warps a tile, and at 64 dimensions two such sets that take stages by turns, each with
//                       a maximum, sum and O of its own, joined at the end: tcgen05.ld S, page scales, mask, exp2, weights back
//                       over the scores.  (At 128 dimensions tensor memory holds one O for each tile, and there is one set.)
//
// O stays in tensor memory: the maximum that weights refer to is only raised when a score exceeds it by more than 8 (log2), and
// only then is O read, scaled and stored.  The query is brought to f16 by a power of two per row, which the scores get back
// together with the page's scale in the multiply-add in front of the exponential.
//
// Eight portions of 512 tokens at depths of 0 to 3584, 32 heads on 8 of 64: 140 us, 0.49 PFLOP/s, where the exponentials alone (16 a
// cycle and SM) need 60.  What bounds it is the chain of a stage through its roles, 1.0 us or 1950 cycles (1.27 us at heads of 128, one
// set): no unit is busy for much more than half of that, page warps as long as softmax warps, and 11,000 cycles go to the ends of a CTA.
// 22 warps leave 80 registers a thread, and 72 bytes of each spill.  Measured while it took 142 us: one set of softmax warps 156 (166 with
// codes in registers one stage ahead), without exponentials 139, without conversions 146, without both 133, eight page warps 146.
//
// Rows of a mask edge test bits of their own; a NaN among the values is replaced in the operand (a weight of 0 times NaN is
// NaN) and remembered by key: a row that sees it becomes NaN as a whole.  Few tiles: a cluster shares a tile's keys and joins
// through distributed shared memory.  Every wait is bounded; if one runs out, the tile keeps its output rows.
#include <cstddef>
#include <type_traits>

#include "e4m3_cache.cuh"
#include "e4m3_cache.h"
#include "e4m3_visible.cuh"
#include "launch.h"
#include "ring.h"
#include "tcgen05.cuh"

namespace lfm25 {

namespace {

constexpr uint32_t kRows = 128;                            // of a tile
constexpr uint32_t kTiles = 2;                             // of a CTA
constexpr uint32_t kPagesPerStage = 4;
constexpr uint32_t kKeys = kPagesPerStage * kPageSize;     // 64
constexpr uint32_t kPageWarps = 4;
constexpr uint32_t kBuffersMost = 4;
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kColumnS = 0;                           // for each tile two buffers of 64; weights of 32 keys take the first 16 columns of theirs
constexpr uint32_t kColumnO = 256;
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
    uint32_t cta_tokens;     // kTiles of that
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
    // softmax warps of a tile take stages by turns, in sets of 4, each with an O of its own where tensor memory has room for two
    static constexpr uint32_t kSets = DIM == 64 ? 2 : 1;
    static constexpr uint32_t kSoftmaxWarps = 4 * kTiles * kSets;
    static constexpr uint32_t kThreads = (kSoftmaxWarps + kPageWarps + kTiles) * 32;
    static constexpr uint32_t kRowWords = 3 + 3 * kSets;                      // of a row: maximum, sum, factor; of each set maximum, sum, whether they hold
    static constexpr uint32_t kBuffers = DIM == 64 ? 4 : 3;                   // of operands
    static constexpr uint32_t kAhead = 2;                                     // stages of codes under way
    static constexpr uint32_t kCodes = 2 * kKeys * DIM;                       // bytes of a stage
    static constexpr uint32_t kQ = 0;                                         // [tile][part][row] of 128 bytes
    static constexpr uint32_t kK = kQ + kTiles * kParts * kRows * 128;        // [buffer][part][key]
    static constexpr uint32_t kV = kK + kBuffers * kParts * kTile;
    static constexpr uint32_t kRaw = kV + kBuffers * kParts * kTile;          // [stage][K, V][piece]
    static constexpr uint32_t kControl = kRaw + kAhead * kCodes;
    static constexpr uint32_t kBytes = kControl + 512 + kRowWords * kTiles * kRows * 4;
    static constexpr uint32_t kAlloc = kBytes + 1024;
    static_assert(kColumnO + kTiles * kSets * DIM <= kTmemColumns, "tensor memory has 512 columns");
    static_assert(kSets <= 2, "a set's stages are all even or all odd");
    static_assert(kControl >= kTiles * kRows * DIM * 4, "the sums that a cluster joins lie where the operands were");
};

// beside the operands
struct Control {
    uint64_t full[kBuffersMost];           // operands of a stage are there
    uint64_t empty[kBuffersMost];          // both tiles' P V are done with them
    uint64_t scores[kTiles][2];
    uint64_t weights[kTiles][2];
    // P V of an even / odd stage is complete.  Nothing orders the arrivals of two commits on different barriers, so each phase of
    // these is waited for.  With two sets the scores of a set's next stage, issued behind P V of the one before, say as much, and
    // only each set's last stage is reported.
    uint64_t product[kTiles][2];
    uint64_t drained[kTiles];          // after a wait ran out: no MMA is in flight any more
    alignas(16) float key_scales[kBuffersMost][kPagesPerStage];   // read four at a time
    alignas(16) unsigned long long nan_keys[kBuffersMost][kPageWarps];   // of each page warp: keys with a NaN among their values
    uint32_t bad_pages[kBuffersMost];      // unassigned pages of the stage, one bit each
    uint32_t odd[kBuffersMost];            // a byte of each page warp: whether any of the two words above is not 0
    uint32_t tmem;
    uint32_t abort;
};
static_assert(offsetof(Control, key_scales) % 16 == 0, "scales are read 16 bytes at a time");
static_assert(sizeof(Control) <= 512, "the control block has 512 bytes");

// Two f32 in a register pair, for the packed instructions: operands that many of them share are packed once.
__device__ __forceinline__ uint64_t pair_of(float low, float high) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(low), "f"(high));
    return v;
}
__device__ __forceinline__ float2 pair_out(uint64_t v) {
    float2 out;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(out.x), "=f"(out.y) : "l"(v));
    return out;
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
    uint32_t v;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(v) : "r"(a), "r"(b));
    return v;
}

// A pair of bf16 with the largest finite number in the place of an infinity: 256 * 2^120 and beyond, codes of values that bf16 holds
// rounded up to the next code, are more than f32 does.  (A weight of 0 must not meet an infinity.)
__device__ __forceinline__ uint32_t pack_finite_bf16x2(float low, float high) {
    uint32_t v;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(high), "f"(low));
    return v;
}

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
// Columns of this thread's lane of tensor memory.  Load and wait are one statement: nothing the compiler knows of keeps the first
// use of a register, and with it the end of its life, behind a wait that is a statement of its own.
__device__ __forceinline__ void load_columns(uint32_t address, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(address)
        : "memory");
}
__device__ __forceinline__ void load_columns(uint32_t address, uint32_t (&a)[16], uint32_t (&b)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]),
          "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]), "=r"(b[0]), "=r"(b[1]),
          "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]), "=r"(b[8]), "=r"(b[9]), "=r"(b[10]),
          "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15])
        : "r"(address)
        : "memory");
}
__device__ __forceinline__ void store_shared(uint32_t address, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(address), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 load_shared(uint32_t address) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ void copy_async(uint32_t shared, const void* global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <uint32_t LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }
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
__global__ void __launch_bounds__(Layout<DIM>::kThreads, 1)
e4m3_prompt_attention_kernel(const PromptParams p) {
    using L = Layout<DIM>;
    constexpr uint32_t kSoftmaxWarps = L::kSoftmaxWarps;
    constexpr uint32_t kThreads = L::kThreads;
    constexpr uint32_t kSets = L::kSets;
    constexpr uint32_t kBuffers = L::kBuffers;
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
        const uint32_t tiles = (end - begin + p.cta_tokens - 1) / p.cta_tokens;
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
    const uint32_t cta_begin = segment_begin + slot * p.cta_tokens;
    const uint32_t cta_end = min(cta_begin + p.cta_tokens, segment_end);
    const uint32_t table_row = p.request_slots[segment_begin];
    const uint64_t origin = p.position_ids[segment_begin];            // position of the segment's first token

    // ---- rows: this thread's token and head.  Their loads are under way together with those of the segment ----
    const uint32_t tile = (warp / 4) % kTiles;           // of the softmax warps
    const uint32_t set = warp / (4 * kTiles);
    const uint32_t row = threadIdx.x % kRows;            // of the tile
    const uint32_t row_token = cta_begin + tile * p.tile_tokens + row / p.chunk_heads;
    const uint32_t head = chunk * p.chunk_heads + row % p.chunk_heads;   // of the group
    const size_t out_row = (static_cast<size_t>(row_token) * p.query_heads + kv_head * p.group + head) * DIM;
    constexpr uint32_t kLanes = DIM / 8;                 // of a row of queries, 16 bytes each
    constexpr uint32_t kPasses = kLanes / kSets;         // of 32 / kLanes rows; the sets share them
    const bool inside = warp < kSoftmaxWarps && row < p.tile_tokens * p.chunk_heads && row_token < cta_end && head < p.group;
    uint32_t row_slot = 0;
    uint32_t row_position = 0;
    if (inside) {
        row_slot = p.request_slots[row_token];
        row_position = p.position_ids[row_token];
    }
    const uint64_t first_wide = origin + (cta_begin - segment_begin);
    const uint64_t most_positions = p.block_table_stride * kPageSize;
    if (table_row >= p.block_table_rows || first_wide >= most_positions) {
        return;
    }
    const uint32_t first_position = static_cast<uint32_t>(first_wide);
    // tokens behind the end of the table have no result; those in front of it do
    const uint32_t last_position = static_cast<uint32_t>(min(first_wide + (cta_end - cta_begin), most_positions) - 1);
    const VisiblePages pages(first_position, last_position, p.window, p.sinks);
    const uint32_t* __restrict__ table = p.block_tables + static_cast<uint64_t>(table_row) * p.block_table_stride;
    const uint32_t all_stages = (pages.count + kPagesPerStage - 1) / kPagesPerStage;
    const uint32_t begin_stage = all_stages * split / p.splits;               // less than 2^26 stages, at most 8 shares
    const uint32_t stages = all_stages * (split + 1) / p.splits - begin_stage;
    // stages that a tile takes part in: the first one's tokens see less, the second one may have no tokens
    auto stages_of = [&](uint32_t tile) -> uint32_t {
        if (tile * p.tile_tokens > last_position - first_position) return 0;
        const uint32_t last = min(last_position, first_position + (tile + 1) * p.tile_tokens - 1);
        const uint32_t until = (pages.sink_pages + last / kPageSize - pages.first_page + kPagesPerStage) / kPagesPerStage;
        return min(until > begin_stage ? until - begin_stage : 0u, stages);
    };

    extern __shared__ uint8_t prompt_smem[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(prompt_smem) + 1023) & ~uintptr_t(1023));
    const uint32_t base = smem_u32(smem);
    Control* control = reinterpret_cast<Control*>(smem + L::kControl);
    volatile uint32_t* abort = &control->abort;
    float* row_words = reinterpret_cast<float*>(smem + L::kControl + 512);
    const uint32_t bar_full = smem_u32(control->full);
    const uint32_t bar_empty = smem_u32(control->empty);
    const uint32_t bar_scores = smem_u32(control->scores);
    const uint32_t bar_weights = smem_u32(control->weights);
    const uint32_t bar_product = smem_u32(control->product);

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kBuffers; ++i) {
            mbar_init(bar_full + 8 * i, kPageWarps);
            mbar_init(bar_empty + 8 * i, kTiles);
        }
        for (uint32_t i = 0; i < 2 * kTiles; ++i) {
            mbar_init(bar_scores + 8 * i, 1);
            mbar_init(bar_weights + 8 * i, 4);
            mbar_init(bar_product + 8 * i, 1);
        }
        for (uint32_t i = 0; i < kTiles; ++i) mbar_init(smem_u32(control->drained) + 8 * i, 1);
        control->abort = 0;
        fence_barrier_init();
    }
    if (warp == kSoftmaxWarps + kPageWarps) {
        tmem_allocate(smem_u32(&control->tmem), kTmemColumns);
    }

    const uint64_t row_wide = first_wide + (row_token - cta_begin);
    float* own_words = row_words + tile * (L::kRowWords * kRows) + row;
    // All threads meet once the barriers, the tensor memory and the queries are there; each role first does what needs none of them.
    auto meet = [&]() -> uint32_t {
        tcgen05_fence_before();
        asm volatile("barrier.sync 1, %0;" ::"n"(kThreads) : "memory");
        tcgen05_fence_after();
        return control->tmem;
    };
    uint32_t tmem = 0;

    // a row's running state (softmax warps)
    float reference = -INFINITY;
    float sum = 0.0f;
    bool poisoned = false;       // sees a NaN value
    bool lost = false;           // sees an unassigned page
    bool live = false;           // has a result
    bool ok = true;
    bool valid = false;
    float weight[kSets];         // of each set's sums

    if (warp >= kSoftmaxWarps && warp < kSoftmaxWarps + kPageWarps) {
        // -------------------------------------------------------------------------------- pages
        constexpr uint32_t kPieces = DIM / 16;                       // of 16 codes, of a key
        constexpr uint32_t kLoads = kKeys * kPieces / 128;           // a thread, for K and for V
        constexpr uint32_t kBlock = 32 / kPagesPerStage;             // stages whose table entries the lanes hold
        const uint32_t page_warp = warp - kSoftmaxWarps;
        const uint32_t thread = page_warp * 32 + lane;
        // load i is piece i * 128 + thread: for a warp one page of the stage, and the same place within it in every stage
        const uint32_t page_bytes = p.cache.kv_heads * kPageSize * DIM;
        const uint32_t inside = kv_head * kPageSize * DIM + (thread / kPieces) % kPageSize * DIM + thread % kPieces * 16;
        const uint8_t* key_source = p.cache.key_codes + inside;
        const uint8_t* value_source = p.cache.value_codes + inside;
        auto page_of = [&](uint32_t i) -> uint32_t { return (i * 128 + page_warp * 32) / kPieces / kPageSize; };
        auto look_up = [&](uint32_t stage) -> uint32_t {             // entry of this lane's page of the stages from `stage` on
            const uint32_t index = (begin_stage + stage) * kPagesPerStage + lane;
            return index < pages.count ? __ldg(table + pages.logical(index)) : 0;
        };
        const uint32_t raw = base + L::kRaw + thread * 16;           // each thread reads what it has copied itself
        uint32_t entries = 0;
        uint32_t coming = look_up(0);
        uint32_t bad[2] = {0, 0};                                    // of the stages at hand and of those before
        float key_scale[2] = {0.0f, 0.0f};
        float value_scale[2] = {0.0f, 0.0f};
        auto load = [&](uint32_t stage) {
            if (stage % kBlock == 0) {
                entries = coming;
                coming = look_up(stage + kBlock);
                bad[1] = bad[0];
                bad[0] = __ballot_sync(0xffffffffu, entries >= p.cache.num_pages);
                const bool exists = (begin_stage + stage) * kPagesPerStage + lane < pages.count && entries < p.cache.num_pages;
                if (!exists) entries = 0;      // page 0 in its place, times 0: no row sees it, or those that do get no result
                const uint64_t at = static_cast<uint64_t>(entries) * p.cache.kv_heads + kv_head;
                key_scale[1] = key_scale[0];
                value_scale[1] = value_scale[0];
                key_scale[0] = exists ? __ldg(p.cache.key_scales + at) : 0.0f;
                value_scale[0] = exists ? __ldg(p.cache.value_scales + at) : 0.0f;
            }
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const uint64_t offset = static_cast<uint64_t>(__shfl_sync(0xffffffffu, entries, stage % kBlock * kPagesPerStage + page_of(i))) * page_bytes;
                copy_async(raw + stage % L::kAhead * L::kCodes + i * 2048, key_source + offset);
                copy_async(raw + stage % L::kAhead * L::kCodes + (kLoads + i) * 2048, value_source + offset);
            }
        };
        // where a piece's 32 bytes go: two pieces of 16 of its key's row
        const uint32_t turn = (thread / kPieces) & 7;
        uint32_t buffer = 0;
        for (uint32_t stage = 0; stage < L::kAhead; ++stage) {
            if (stage < stages) load(stage);
            copies_commit();
        }
        meet();
        for (uint32_t stage = 0; stage < stages; ++stage) {
            // the block of 8 stages that is at hand may be the next one's already
            const uint32_t older = min(stage + L::kAhead, stages) - 1 >= (stage / kBlock + 1) * kBlock ? 1 : 0;
            if (stage >= kBuffers) {
                ok = *abort == 0 && mbar_wait_bounded(bar_empty + 8 * buffer, (stage / kBuffers - 1) & 1, p.wait_limit_ns);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
            }
            copies_wait<L::kAhead - 1>();
            if (stage % kBlock == 0) {
                // A page that none of the tile's rows sees (it belongs to a token that has no result) may hold anything.  Masked scores
                // are -inf, which a negative factor would make the largest of all, and a weight of 0 must not meet an infinity or a NaN:
                // 0 in the place of what is no scale.  A NaN among the factors of keys reaches the rows that see them, and no others.
                // (Here, two stages behind the loads, and not where they are asked for.)
                const bool number = fabsf(value_scale[0]) <= 3.4028235e38f;
                if (!(key_scale[0] > 0.0f && key_scale[0] <= 3.4028235e38f)) key_scale[0] = 0.0f;
                if (!number) key_scale[0] = __int_as_float(0x7fc00000);
                if (!number) value_scale[0] = 0.0f;
            }
            uint4 k_now[kLoads];
            uint4 v_now[kLoads];
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                k_now[i] = load_shared(raw + stage % L::kAhead * L::kCodes + i * 2048);
                v_now[i] = load_shared(raw + stage % L::kAhead * L::kCodes + (kLoads + i) * 2048);
            }
            const uint32_t k_base = base + L::kK + buffer * (L::kParts * kTile);
            const uint32_t v_base = base + L::kV + buffer * (L::kParts * kTile);
            uint32_t check = 0;                                      // f16 sums of values: NaN where one of them is
            unsigned long long nan_keys = 0;
            auto convert_values = [&](uint32_t i, const uint32_t (&words)[4]) {
                const uint32_t key = (i * 128 + thread) / kPieces;
                const uint32_t dims = thread % kPieces;              // 16 dimensions
                const uint32_t place = v_base + (dims / 4) * kTile + key * 128;
                const float scale = __shfl_sync(0xffffffffu, older ? value_scale[1] : value_scale[0], stage % kBlock * kPagesPerStage + page_of(i));
                const uint64_t scales = pair_of(scale, scale);
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    uint32_t pairs[4];
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const uint32_t word = words[2 * h + j / 2];
                        const uint32_t halves = j % 2 ? e4m3x2_high_to_f16x2(word) : e4m3x2_to_f16x2(word);
                        check = add_f16x2(check, halves);
                        const float2 x = f16x2_to_float2(halves);
                        const float2 scaled = pair_out(pair_mul(pair_of(x.x, x.y), scales));
                        pairs[j] = pack_finite_bf16x2(scaled.x, scaled.y);
                    }
                    store_shared(place + (((2 * dims % 8 + h) ^ turn) << 4), make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]));
                }
            };
#pragma unroll
            for (uint32_t i = 0; i < kLoads; ++i) {
                const uint32_t key = (i * 128 + thread) / kPieces;
                const uint32_t dims = thread % kPieces;
                const uint32_t place = k_base + (dims / 4) * kTile + key * 128;
                const uint32_t words[4] = {k_now[i].x, k_now[i].y, k_now[i].z, k_now[i].w};
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    store_shared(place + (((2 * dims % 8 + h) ^ turn) << 4),
                                 make_uint4(e4m3x2_to_f16x2(words[2 * h]), e4m3x2_high_to_f16x2(words[2 * h]),
                                            e4m3x2_to_f16x2(words[2 * h + 1]), e4m3x2_high_to_f16x2(words[2 * h + 1])));
                }
                const uint32_t v_words[4] = {v_now[i].x, v_now[i].y, v_now[i].z, v_now[i].w};
                convert_values(i, v_words);
            }
            const float2 sums = f16x2_to_float2(check);
            if (__any_sync(0xffffffffu, isnan(sums.x + sums.y))) {
                // codes that are NaN become 0, and their keys are remembered
#pragma unroll
                for (uint32_t i = 0; i < kLoads; ++i) {
                    uint32_t words[4] = {v_now[i].x, v_now[i].y, v_now[i].z, v_now[i].w};
                    uint32_t odd = 0;
#pragma unroll
                    for (uint32_t w = 0; w < 4; ++w) {
                        const uint32_t hit = (((words[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                        odd |= hit;
                        words[w] &= ~(hit * 0xffu);
                    }
                    uint32_t lanes = __ballot_sync(0xffffffffu, odd != 0);
                    while (lanes != 0) {
                        nan_keys |= 1ull << ((i * 128 + page_warp * 32 + __ffs(lanes) - 1) / kPieces);
                        lanes &= lanes - 1;
                    }
                    convert_values(i, words);
                }
            }
            // 4 lanes of the first warp have the stage's key scales
            if (page_warp == 0 && lane / kPagesPerStage == stage % kBlock) {
                control->key_scales[buffer][lane % kPagesPerStage] = older ? key_scale[1] : key_scale[0];
            }
            if (lane == 0) {
                const uint32_t stage_bad = ((older ? bad[1] : bad[0]) >> (stage % kBlock * kPagesPerStage)) & 0xfu;
                control->nan_keys[buffer][page_warp] = nan_keys;
                if (page_warp == 0) control->bad_pages[buffer] = stage_bad;
                reinterpret_cast<uint8_t*>(&control->odd[buffer])[page_warp] = nan_keys != 0 || stage_bad != 0 ? 1 : 0;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && !(p.selftest_drop != 0 && page_warp == 0 && stage == 0)) mbar_arrive(bar_full + 8 * buffer);
            buffer = buffer + 1 == kBuffers ? 0 : buffer + 1;
            // into the place of the codes that have just been converted
            if (stage + L::kAhead < stages) load(stage + L::kAhead);
            copies_commit();
        }
        copies_wait<0>();
        if (!ok && lane == 0 && *abort == 0) {
            *abort = 1;
            record_wait_timeout(p.status, kTagE4m3Prompt, (blockIdx.x << 2) | 1);
        }
    } else if (warp >= kSoftmaxWarps + kPageWarps) {
        // -------------------------------------------------------------------------------- MMA issuers, one for each tile
        const uint32_t which = warp - (kSoftmaxWarps + kPageWarps);
        tmem = meet();
        // The warp stays together: all lanes wait, one of them issues, and none runs ahead of the others.  (Two builds in which one lane
        // ran the whole loop by itself ended in an illegal address now and then, in their first launches.  The cause is not known: that
        // form is legal, other kernels have it, reading found no access out of range in it, and keeping the warp together may have
        // changed no more than the timing.  It costs 2 us over eight portions of 512.)
        // f32 results of 128 rows; Q K^T: f16, both K-major, 64 keys; P V: bf16, V MN-major, 64 dimensions
        constexpr uint32_t idesc_scores = (1u << 4) | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);
        constexpr uint32_t idesc_product = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((64u >> 3) << 17) | ((kRows >> 4) << 24);
        const uint32_t my_stages = stages_of(which);
        const uint64_t q_desc = smem_descriptor(base + L::kQ + which * (L::kParts * kRows * 128));
        const uint64_t k_first = smem_descriptor(base + L::kK);
        const uint64_t v_first = smem_descriptor(base + L::kV);
        const uint32_t columns = tmem + kColumnS + 2 * which * kKeys;
        const uint32_t output_columns = tmem + kColumnO + which * DIM;
        const uint32_t my_scores = bar_scores + 16 * which;
        const uint32_t my_weights = bar_weights + 16 * which;
        const uint32_t my_product = bar_product + 16 * which;
        uint32_t next_buffer = 0;      // of the next scores
        uint32_t next_parity = 0;
        auto wait_for = [&](uint32_t barrier, uint32_t parity) -> bool {
            const bool came = *abort == 0 && mbar_wait_bounded(barrier, parity, p.wait_limit_ns);
            return __all_sync(0xffffffffu, came);
        };
        auto issue_scores = [&](uint32_t parity) -> bool {
            if (!wait_for(bar_full + 8 * next_buffer, next_parity)) {
                return false;
            }
            tcgen05_fence_after();
            if (elect_one()) {
                const uint64_t k_desc = k_first + next_buffer * (L::kParts * kTile >> 4);
#pragma unroll
                for (uint32_t ks = 0; ks < DIM / 16; ++ks) {   // 16 dimensions: 32 bytes within the swizzled row
                    umma_ss(columns + parity * kKeys, q_desc + (ks / 4) * (kRows * 128 >> 4) + (ks % 4) * 2,
                            k_desc + (ks / 4) * (kTile >> 4) + (ks % 4) * 2, idesc_scores, ks);
                }
                umma_commit(my_scores + 8 * parity);
            }
            __syncwarp();
            if (++next_buffer == kBuffers) {
                next_buffer = 0;
                next_parity ^= 1;
            }
            return true;
        };
        for (uint32_t stage = 0; stage < 2 && ok; ++stage) {
            if (stage < my_stages) ok = issue_scores(stage);
        }
        uint32_t buffer = 0;
        for (uint32_t stage = 0; stage < my_stages && ok; ++stage) {
            const uint32_t parity = stage & 1;
            ok = wait_for(my_weights + 8 * parity, (stage >> 1) & 1);
            if (!ok) break;
            tcgen05_fence_after();
            if (elect_one()) {
                const uint64_t v_desc = v_first + buffer * (L::kParts * kTile >> 4);
#pragma unroll
                for (uint32_t part = 0; part < L::kParts; ++part) {
#pragma unroll
                    for (uint32_t step = 0; step < kPagesPerStage; ++step) {   // 16 keys: 8 columns of weights, 2 KiB of V
                        umma_ts(output_columns + stage % kSets * (kTiles * DIM) + part * 64, columns + parity * kKeys + step / 2 * 32 + step % 2 * 8,
                                v_desc + part * (kTile >> 4) + step * (2048 >> 4), idesc_product, stage >= kSets || step > 0);
                    }
                }
                if (kSets == 1 || last_of_set(stage, my_stages, kSets)) umma_commit(my_product + 8 * parity);
                if (filled_again(stage, stages, kBuffers)) umma_commit(bar_empty + 8 * buffer);
            }
            __syncwarp();
            // Behind it the scores of two stages on: MMAs execute in order, so the weights in their columns have been consumed.
            if (stage + 2 < my_stages) ok = issue_scores(parity);
            if (++buffer == kBuffers) buffer = 0;
        }
        // stages that only the other tile takes part in
        for (uint32_t stage = my_stages; stage < stages && filled_again(stage, stages, kBuffers) && ok; ++stage) {
            ok = wait_for(bar_full + 8 * (stage % kBuffers), (stage / kBuffers) & 1);
            if (ok && lane == 0) mbar_arrive(bar_empty + 8 * (stage % kBuffers));
            __syncwarp();
        }
        if (!ok && lane == 0 && *abort == 0) {
            *abort = 1;
            record_wait_timeout(p.status, kTagE4m3Prompt, (blockIdx.x << 2) | 2);
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, *abort != 0)) {
            if (elect_one()) umma_commit(smem_u32(control->drained) + 8 * which);
            __syncwarp();
            (void)mbar_wait_bounded(smem_u32(control->drained) + 8 * which, 0, p.wait_limit_ns);
        }
    } else {
        // -------------------------------------------------------------------------------- softmax
        // ---- queries to f16, by a power of two per row ----
        const uint64_t row_offset = inside ? row_token * p.query_token_stride + static_cast<size_t>(kv_head * p.group + head) * DIM : 0;
        uint4 raw_query[kPasses];
#pragma unroll
        for (uint32_t pass = 0; pass < kPasses; ++pass) {
            const uint32_t source = (set * kPasses + pass) * (32 / kLanes) + lane / kLanes;
            const uint32_t low = __shfl_sync(0xffffffffu, static_cast<uint32_t>(row_offset), source);
            const uint32_t high = __shfl_sync(0xffffffffu, static_cast<uint32_t>(row_offset >> 32), source);
            // rows that do not exist read the first query of the batch, and are cleared below
            raw_query[pass] = *reinterpret_cast<const uint4*>(p.query + ((static_cast<uint64_t>(high) << 32) | low) + lane % kLanes * 8);
        }
        live = inside && row_wide < most_positions && row_slot == table_row && row_position == row_wide;
        const uint32_t live_rows = __ballot_sync(0xffffffffu, live);
        uint32_t largest[kPasses];                        // exchanges of all passes side by side
#pragma unroll
        for (uint32_t pass = 0; pass < kPasses; ++pass) {
            const uint32_t source = (set * kPasses + pass) * (32 / kLanes) + lane / kLanes;
            if (((live_rows >> source) & 1) == 0) raw_query[pass] = make_uint4(0, 0, 0, 0);
            const uint32_t words[4] = {raw_query[pass].x, raw_query[pass].y, raw_query[pass].z, raw_query[pass].w};
            largest[pass] = 0;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t low = words[i] & 0x7fffu;
                const uint32_t high = (words[i] >> 16) & 0x7fffu;
                largest[pass] = max(largest[pass], max(low < 0x7f80u ? low : 0u, high < 0x7f80u ? high : 0u));
            }
        }
#pragma unroll
        for (uint32_t delta = kLanes / 2; delta > 0; delta >>= 1) {
            uint32_t other[kPasses];
#pragma unroll
            for (uint32_t pass = 0; pass < kPasses; ++pass) other[pass] = __shfl_xor_sync(0xffffffffu, largest[pass], delta);
#pragma unroll
            for (uint32_t pass = 0; pass < kPasses; ++pass) largest[pass] = max(largest[pass], other[pass]);
        }
#pragma unroll
        for (uint32_t pass = 0; pass < kPasses; ++pass) {
            const uint32_t words[4] = {raw_query[pass].x, raw_query[pass].y, raw_query[pass].z, raw_query[pass].w};
            const int32_t exponent = min(max(static_cast<int32_t>(largest[pass] >> 7) - 127 - 11, -126), 126);
            const float factor = power_of_two(-exponent);
            uint32_t half[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const float2 pair = bf16x2_to_float2(words[i]);
                half[i] = pack_f16x2(pair.x * factor, pair.y * factor);
            }
            const uint32_t target = warp % 4 * 32 + (set * kPasses + pass) * (32 / kLanes) + lane / kLanes;   // row of the tile
            const uint32_t piece = lane % kLanes;
            if (piece == 0) row_words[(tile * L::kRowWords + 2) * kRows + target] = power_of_two(exponent) * p.scale_log2;
            store_shared(base + L::kQ + (tile * L::kParts + piece / 8) * (kRows * 128) + target * 128 + (((piece % 8) ^ (target & 7)) << 4),
                         make_uint4(half[0], half[1], half[2], half[3]));
        }
        fence_proxy_async_smem();
        tmem = meet();

        const float row_factor = own_words[2 * kRows];
        const uint32_t position = live ? static_cast<uint32_t>(row_wide) : last_position;
        const uint32_t first_key = p.window != 0 && position >= p.window ? position - p.window + 1 : 0;
        const uint32_t lane_address = tmem + ((warp % 4 * 32) << 16);
        const uint32_t output_columns = lane_address + kColumnO + (set * kTiles + tile) * DIM;
        const uint32_t my_stages = stages_of(tile);
        // weights complete, and handed over
        auto hand_over = [&](uint32_t stage) {
            tmem_store_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_weights + 8 * (2 * tile + (stage & 1)));
        };
        // The stages that every row of this warp sees as a whole, in one run: from the last window's first key on, up to the first
        // position.  (Stages of first tokens only are taken with those that have an edge.)
        const int32_t least = static_cast<int32_t>(__reduce_min_sync(0xffffffffu, position));
        const uint32_t edge = __reduce_max_sync(0xffffffffu, first_key);
        const int32_t shift = static_cast<int32_t>(pages.sink_pages) - static_cast<int32_t>(pages.first_page);   // of list against table
        const int32_t whole_first = max(static_cast<int32_t>(pages.sink_pages), static_cast<int32_t>((edge + kPageSize - 1) / kPageSize) + shift);
        const int32_t whole_last = (least + 1 - static_cast<int32_t>(kKeys)) >= 0 ? (least + 1 - static_cast<int32_t>(kKeys)) / static_cast<int32_t>(kPageSize) + shift : -1;
        const int32_t from = max((whole_first + static_cast<int32_t>(kPagesPerStage) - 1) / static_cast<int32_t>(kPagesPerStage) - static_cast<int32_t>(begin_stage), 0);
        const int32_t until = whole_last >= 0 ? whole_last / static_cast<int32_t>(kPagesPerStage) + 1 - static_cast<int32_t>(begin_stage) : 0;
        const uint32_t whole_begin = static_cast<uint32_t>(from);
        const uint32_t whole_count = static_cast<uint32_t>(max(until - from, 0));
        uint32_t buffer = set;
        uint32_t buffer_parity = 0;
        for (uint32_t stage = set; stage < my_stages; stage += kSets) {
            // ---- the page warps' words (there before the scores are) ----
            const bool fast = stage - whole_begin < whole_count;
            // the keys of the stage that this row sees, where that is asked for
            auto seen_keys = [&](uint32_t (&bits)[2]) {
                const uint32_t index = (begin_stage + stage) * kPagesPerStage;
                bits[0] = bits[1] = 0;
#pragma unroll 1
                for (uint32_t sub = 0; sub < kPagesPerStage; ++sub) {
                    if (index + sub < pages.count) {
                        const uint32_t seen = visible_bits(pages.logical(index + sub) * kPageSize, position, first_key, p.sinks) << (sub % 2 * 16);
                        if (sub < 2) bits[0] |= seen;
                        else bits[1] |= seen;
                    }
                }
            };
            ok = mbar_wait_bounded(bar_full + 8 * buffer, buffer_parity, p.wait_limit_ns);
            const float4 scales = *reinterpret_cast<const float4*>(control->key_scales[buffer]);
            const float factor[4] = {row_factor * scales.x, row_factor * scales.y, row_factor * scales.z, row_factor * scales.w};
            if (control->odd[buffer] != 0) {
                const unsigned long long* nan = control->nan_keys[buffer];
                const unsigned long long nan_keys = (nan[0] | nan[1]) | (nan[2] | nan[3]);
                const uint32_t bad = control->bad_pages[buffer];
                uint32_t bits[2];
                seen_keys(bits);
                const unsigned long long seen = bits[0] | (static_cast<unsigned long long>(bits[1]) << 32);
                poisoned = poisoned || (nan_keys & seen) != 0;
#pragma unroll 1
                for (uint32_t sub = 0; sub < kPagesPerStage; ++sub) {
                    lost = lost || (((bad >> sub) & 1) != 0 && ((seen >> (16 * sub)) & 0xffffu) != 0);
                }
            }
            buffer += kSets;
            if (buffer >= kBuffers) {
                buffer -= kBuffers;
                buffer_parity ^= 1;
            }
            ok = ok && mbar_wait_bounded(bar_scores + 8 * (2 * tile + (stage & 1)), (stage >> 1) & 1, p.wait_limit_ns);
            if (kSets == 1 && stage >= 2) {
                ok = ok && mbar_wait_bounded(bar_product + 8 * (2 * tile + (stage & 1)), ((stage >> 1) - 1) & 1, p.wait_limit_ns);
            }
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            tcgen05_fence_after();
            const uint32_t columns = lane_address + kColumnS + (2 * tile + (stage & 1)) * kKeys;
            // In two copies: tests of single keys, which the compiler would make predicates of every stage, were a quarter of all
            // instructions.
            auto weigh = [&](auto masked) -> bool {
                constexpr bool kMasked = decltype(masked)::value;
                uint32_t bits[2] = {0, 0};
                if constexpr (kMasked) seen_keys(bits);
                // Two sets leave no registers for all scores at once: 32 keys at a time, the first ones twice.
                constexpr bool kWhole = kSets == 1;
                uint32_t raw[kWhole ? 4 : 2][16];
                auto fetch = [&](uint32_t half) { load_columns(columns + half * 32, raw[kWhole ? half * 2 : 0], raw[kWhole ? half * 2 + 1 : 1]); };
                // ---- maximum ----
                float most = -INFINITY;
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half) {
                    fetch(half);
                    const uint32_t at = kWhole ? half * 2 : 0;
                    if constexpr (kMasked) {
                        // masked scores, whatever they are, become -inf (the factor is positive or 0, so not by the product)
#pragma unroll
                        for (uint32_t j = 0; j < 32; ++j) {
                            if (((bits[half] >> j) & 1) == 0) raw[at + j / 16][j % 16] = 0xff800000u;
                        }
                    }
#pragma unroll
                    for (uint32_t sub = 0; sub < 2; ++sub) {
                        float a = __uint_as_float(raw[at + sub][0]);
                        float b = __uint_as_float(raw[at + sub][1]);
#pragma unroll
                        for (uint32_t j = 2; j < 16; j += 4) {
                            a = max3(a, __uint_as_float(raw[at + sub][j]), __uint_as_float(raw[at + sub][j + 1]));
                            if (j + 2 < 16) b = max3(b, __uint_as_float(raw[at + sub][j + 2]), __uint_as_float(raw[at + sub][j + 3]));
                        }
                        const float here = fmaxf(a, b);
                        most = fmaxf(most, here * factor[half * 2 + sub]);
                    }
                }
                const bool raise = most > reference + kHeadroom;
                if (__any_sync(0xffffffffu, raise)) {
                    const float shrink = !raise ? 1.0f : reference == -INFINITY ? 0.0f : fast_exp2(reference - most);
                    if (raise) reference = most;
                    sum *= shrink;
                    if (stage >= kSets) {
                        if constexpr (kSets == 1) {
                            const uint32_t before = stage - 1;
                            ok = *abort == 0 && mbar_wait_bounded(bar_product + 8 * (2 * tile + (before & 1)), (before >> 1) & 1, p.wait_limit_ns);
                            if (!__all_sync(0xffffffffu, ok)) {
                                return false;
                            }
                            tcgen05_fence_after();
                        }
#pragma unroll 1
                        for (uint32_t c = 0; c < DIM; c += 16) {
                            uint32_t o[16];
                            load_columns(output_columns + c, o);
#pragma unroll
                            for (uint32_t j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
                            tmem_store16(output_columns + c, o);
                        }
                    }
                }
                // ---- weights, of the keys at hand first ----
                const float reference_offset = reference == -INFINITY ? 0.0f : -reference;
                const uint64_t offset = pair_of(reference_offset, reference_offset);
                uint64_t part_sum[2] = {0, 0};
#pragma unroll
                for (uint32_t turn = 0; turn < 2; ++turn) {
                    const uint32_t half = 1 - turn;
                    if (!kWhole && turn == 1) fetch(half);
                    const uint32_t at = kWhole ? half * 2 : 0;
                    uint32_t packed[16];
#pragma unroll
                    for (uint32_t sub = 0; sub < 2; ++sub) {
                        const uint64_t multiplier = pair_of(factor[half * 2 + sub], factor[half * 2 + sub]);
#pragma unroll
                        for (uint32_t pair = 0; pair < 8; ++pair) {
                            const uint32_t j = sub * 16 + pair * 2;
                            float2 w = pair_out(pair_fma(pair_of(__uint_as_float(raw[at + sub][pair * 2]), __uint_as_float(raw[at + sub][pair * 2 + 1])),
                                                         multiplier, offset));
                            w = make_float2(fast_exp2(w.x), fast_exp2(w.y));
                            if constexpr (kMasked) {
                                w.x = (bits[half] >> j) & 1 ? w.x : 0.0f;
                                w.y = (bits[half] >> (j + 1)) & 1 ? w.y : 0.0f;
                            }
                            // 8 bits, since both operands of the product have one type and values with their page's scale need
                            // bf16's range: 2^-9 a weight on average, which over many keys leaves 0.0021 to 0.0023 of the result
                            // (root of mean squares, the result's own rounding to bf16 among it) instead of 0.0016
                            packed[sub * 8 + pair] = pack_bf16x2(w.x, w.y);
                            part_sum[pair & 1] = pair_add(part_sum[pair & 1], pair_of(w.x, w.y));   // unrounded: roundings average out
                        }
                    }
                    tmem_store16(columns + half * 32, packed);
                }
                const float2 stage_sum = pair_out(pair_add(part_sum[0], part_sum[1]));
                sum += stage_sum.x + stage_sum.y;
                return true;
            };
            ok = fast ? weigh(std::false_type()) : weigh(std::true_type());
            if (!ok) break;
            hand_over(stage);
        }
        if (ok && my_stages > set) {
            ok = *abort == 0;
            if constexpr (kSets == 1) {
                if (my_stages > 1) {
                    const uint32_t before = my_stages - 2;
                    ok = ok && mbar_wait_bounded(bar_product + 8 * (2 * tile + (before & 1)), (before >> 1) & 1, p.wait_limit_ns);
                }
                const uint32_t last = my_stages - 1;
                ok = ok && mbar_wait_bounded(bar_product + 8 * (2 * tile + (last & 1)), (last >> 1) & 1, p.wait_limit_ns);
            } else {
                ok = ok && mbar_wait_bounded(bar_product + 8 * (2 * tile + set), 0, p.wait_limit_ns);   // a set's stages have its parity
            }
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok && lane == 0 && *abort == 0) {
            *abort = 1;
            record_wait_timeout(p.status, kTagE4m3Prompt, (blockIdx.x << 2) | 3);
        }
        tcgen05_fence_after();
        if (poisoned) sum = __int_as_float(0x7fc00000);
        valid = ok && !lost && *abort == 0;
        // ---- the sets' results together ----
        if constexpr (kSets > 1) {
            own_words[(3 + 3 * set) * kRows] = reference;
            own_words[(4 + 3 * set) * kRows] = sum;
            own_words[(5 + 3 * set) * kRows] = valid ? 1.0f : 0.0f;
            asm volatile("barrier.sync 2, %0;" ::"n"(kSoftmaxWarps * 32) : "memory");
            reference = fmaxf(own_words[3 * kRows], own_words[6 * kRows]);
            valid = own_words[5 * kRows] != 0.0f && own_words[8 * kRows] != 0.0f;
            const float offset = reference == -INFINITY ? 0.0f : reference;
            sum = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < kSets; ++i) {
                weight[i] = fast_exp2(own_words[(3 + 3 * i) * kRows] - offset);
                sum = fmaf(own_words[(4 + 3 * i) * kRows], weight[i], sum);
            }
        } else {
            weight[0] = 1.0f;
        }
    }

    __syncwarp();
    if (p.splits > 1) {
        // nobody writes operands any more, and the products have been waited for: the sums for the cluster lie there, one column of
        // 128 rows behind the other
        __syncthreads();
    }
    if (warp < kSoftmaxWarps) {
        if (p.splits > 1) {
            own_words[0] = reference;
            own_words[kRows] = valid ? sum : -1.0f;      // a sum is never negative
        }
        // each set has its share of the dimensions
        constexpr uint32_t kShare = DIM / kSets;
        const uint32_t my_stages = stages_of(tile);
        const uint32_t columns = tmem + ((warp % 4 * 32) << 16) + kColumnO + tile * DIM;
        float* sums = reinterpret_cast<float*>(smem) + tile * (DIM * kRows) + row;
        const float inverse = 1.0f / sum;
        const uint32_t staged = base + L::kQ + tile * (L::kParts * kRows * 128);      // the tile's queries are not needed any more
#pragma unroll
        for (uint32_t c = set * kShare; c < (set + 1) * kShare; c += 16) {
            float value[16] = {};
#pragma unroll
            for (uint32_t i = 0; i < kSets; ++i) {
                uint32_t o[16];
                __syncwarp();                  // the whole warp loads, also where only some rows are stored
                load_columns(columns + i * kTiles * DIM + c, o);
                if (my_stages > i) {           // else there are no sums
#pragma unroll
                    for (uint32_t j = 0; j < 16; ++j) value[j] = fmaf(__uint_as_float(o[j]), weight[i], value[j]);
                }
            }
            if (p.splits > 1) {
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) sums[(c + j) * kRows] = value[j];
            } else {
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    uint32_t pairs[4];
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) pairs[j] = pack_bf16x2(value[h * 8 + 2 * j] * inverse, value[h * 8 + 2 * j + 1] * inverse);
                    store_shared(staged + row * (DIM * 2) + (((c / 8 + h) ^ (row & 7)) << 4), make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]));
                }
            }
        }
        if (p.splits == 1) {
            // rows of this warp, by whole lines (one row a lane is 32 lines a store; 7 portions at heads of 128: 26.0 us instead of 24.7)
            constexpr uint32_t kPieces = kShare / 8;     // of a row's share
            __syncwarp();
            const uint32_t written = __ballot_sync(0xffffffffu, live && valid);
#pragma unroll
            for (uint32_t pass = 0; pass < kPieces; ++pass) {
                const uint32_t source = pass * (32 / kPieces) + lane / kPieces;
                const uint32_t piece = set * kPieces + lane % kPieces;
                const uint32_t low = __shfl_sync(0xffffffffu, static_cast<uint32_t>(out_row), source);
                const uint32_t high = __shfl_sync(0xffffffffu, static_cast<uint32_t>(static_cast<uint64_t>(out_row) >> 32), source);
                const uint32_t target = warp % 4 * 32 + source;
                const uint4 out = load_shared(staged + target * (DIM * 2) + ((piece ^ (target & 7)) << 4));
                if ((written >> source) & 1) {
                    *reinterpret_cast<uint4*>(p.output + ((static_cast<uint64_t>(high) << 32) | low) + piece * 8) = out;
                }
            }
        }
    }

    if (p.splits > 1) {
        // ---- join the cluster ----
        __syncwarp();
        cluster_barrier();
        if (warp < kSoftmaxWarps) {
            const uint32_t own = smem_u32(own_words);
            const uint32_t own_sums = base + (tile * (DIM * kRows) + row) * 4;
            float weight[8];
            float part_sum[8];
            float most = -INFINITY;
            bool complete = live;
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) {         // all loads under way at once
                weight[r] = r < p.splits ? load_cluster(own, r) : -INFINITY;
                part_sum[r] = r < p.splits ? load_cluster(own + kRows * 4, r) : 0.0f;
                complete = complete & !(part_sum[r] < 0.0f);
                most = fmaxf(most, weight[r]);
            }
            const float offset = most == -INFINITY ? 0.0f : most;
            float total = 0.0f;
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) {
                weight[r] = fast_exp2(weight[r] - offset);
                total = fmaf(part_sum[r], weight[r], total);
            }
            const float inverse = 1.0f / total;
            const uint32_t share = DIM / p.splits;       // 8 dimensions or more
            for (uint32_t c = split * share + set * 4; c < (split + 1) * share; c += 4 * kSets) {
                float value[4] = {};
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r) {
                    if (r < p.splits) {
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) {
                            value[j] = fmaf(load_cluster(own_sums + ((c + j) * kRows) * 4, r), weight[r], value[j]);
                        }
                    }
                }
                if (complete) {
                    *reinterpret_cast<uint2*>(p.output + out_row + c) = make_uint2(pack_bf16x2(value[0] * inverse, value[1] * inverse),
                                                                                  pack_bf16x2(value[2] * inverse, value[3] * inverse));
                }
            }
        }
        __syncwarp();
        cluster_barrier();                 // nobody leaves while its sums are read
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps + kPageWarps) {
        tmem_free(tmem, kTmemColumns);
    }
}

template <uint32_t DIM>
cudaError_t launch_dim(cudaStream_t stream, const PromptParams& params, uint64_t blocks) {
    const cudaError_t status = allow_shared_memory<e4m3_prompt_attention_kernel<DIM>>(Layout<DIM>::kAlloc);
    if (status != cudaSuccess) {
        return status;
    }
    return launch_kernel(e4m3_prompt_attention_kernel<DIM>, static_cast<unsigned int>(blocks), Layout<DIM>::kThreads, Layout<DIM>::kAlloc, stream,
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
    params.cta_tokens = kTiles * params.tile_tokens;
    params.window = launch.window;
    params.sinks = launch.sinks;
    params.scale_log2 = launch.scale * kLog2e;
    params.wait_limit_ns = wait_limit_ns();
    params.selftest_drop = wait_selftest_drop() ? 1 : 0;
    // at most so many tiles, by how the tokens lie in the segments: a segment's first token is one, and cta_tokens more each is another
    const uint64_t tiles = launch.num_segments < launch.num_tokens
                               ? (launch.num_tokens - launch.num_segments) / params.cta_tokens + launch.num_segments : launch.num_segments;
    const uint64_t items = tiles * launch.cache.kv_heads * params.chunks;
    uint64_t longest = launch.maximum_context_tokens;
    if (launch.window != 0 && longest > static_cast<uint64_t>(launch.window) + launch.sinks + params.cta_tokens) {
        longest = static_cast<uint64_t>(launch.window) + launch.sinks + params.cta_tokens;
    }
    // Shares of the keys as long as all CTAs run at once, one an SM, and each has a few stages.  A B200 holds 74, 33 and 15 clusters of 2,
    // 4 and 8 such CTAs, and those that find no room cost their whole time again.  32 heads on 8 of 64: 37 tokens behind 8000 126 us whole,
    // 2 shares 71, 4 41, 8 26.9; 2 x 64 behind 4000 (16 clusters) 8 shares 38.5, 4 26.7; 64 behind 500 1 16.6, 4 14.4, 8 15.6; 64 behind
    // 200 1 12.5, 2 14.9, 4 13.2; 512 behind 2000 1 46.3, 2 32.3, 4 42.2.  8 heads on 2 of 128: 37 behind 8000 153, 92, 53, 33.0; 512 behind
    // 2000 (16 clusters) 8 shares 41.0, 4 28.6; 64 behind 500 1 20.2, 4 19.4, 8 17.5; 64 behind 200 1 15.1, 8 16.5.  (Short segments count
    // for more tiles than they are: 4 x 64 behind 2000, 32 on 8 of 64, take 2 shares and 28.8 us, 4 would take 22.1.)
    constexpr uint32_t kResidentClusters[4] = {148, 74, 33, 15};
    uint32_t splits_log2 = 0;
    while (splits_log2 < 3 && items <= kResidentClusters[splits_log2 + 1] && longest >= ((2u << splits_log2) + 4) * kKeys) ++splits_log2;
    params.splits = 1u << splits_log2;
    const uint64_t blocks = items * params.splits;
    if (blocks > 0x7fffffffu) {
        return cudaErrorInvalidConfiguration;
    }
    return launch.cache.head_dim == 64 ? launch_dim<64>(stream, params, blocks) : launch_dim<128>(stream, params, blocks);
}

}  // namespace lfm25
