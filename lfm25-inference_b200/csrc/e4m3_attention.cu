// Attention of single tokens over the 8-bit paged cache: out = softmax(scale * q K^T) V over the keys that the token sees
// (e4m3_visible.cuh), K and V read as E4M3 codes with a power-of-two scale for each page and KV head.
//
// Bound by HBM: 2 * head_dim bytes and 8 / 16 of a scale a key and KV head, against 4 * head_dim flops a query head.  A CTA
// has one (token, KV head) with up to 16 of its query heads, or one share of its pages; its warps take pages in turn and each
// runs an online softmax of its own.
//
// A page (16 keys) is one step of mma.sync m16n8k16 in f16, which holds every E4M3 value:
//   S = Q K^T     A = the query heads as rows, B = K^T.  The order of the reduction is free, so lane (g, t) of the warp
//                 takes dimensions 16 t .. 16 t + 15 (of every 64) of two keys: 16 bytes a load, which turn into operands by
//                 conversion alone.
//   O^T += V^T P^T   A = V^T, B = P^T, and the fragment of S is that of P^T.  Lane (g, t) takes four keys, head_dim / 8
//                 dimensions of each: two bytes of two keys side by side are one byte permutation, converted like K.
// Which keys a lane has is free as well (key_of) and chosen, with the place of a row's 16-byte pieces in shared memory, so that
// both reads are free of bank conflicts.  Pages travel by asynchronous copies into a ring of each warp's own; nobody but the
// warp waits for them, and nothing polls.
//
// The query is brought to f16 by a power of two of its own (largest magnitude in [2^11, 2^12)): bf16 carries 8 bits, so what is
// lost lies 2^-36 below the largest element.  Page scales multiply S in front of the exponential and the page's P V behind the
// MMA, both in f32, where a power of two rounds nothing.
//
// The maximum that weights refer to is only raised when a score exceeds it by more than 4 (log2): most pages need no exchange between
// lanes.  Weights go to the product in f16, rounded to 11 bits: times 2^11, which the page's scale and the sum of weights take back, so
// that the largest there can be, 2^15, still fits and the smallest step is 2^-35 of the weight of the maximum.  (Without that factor and with a
// headroom of 8 the step was 2^-24: a first token that takes nearly all left nothing of the others.  Both take the same time: 128 tokens
// at contexts 128..4096 49.7 us, 3 at 20480..65536 36.7 against 36.4.)
//
// Without its arithmetic the kernel streams at the copy peak (128 tokens at contexts 128..4096: 43.3 us); with it 49.7, bound by the
// instructions of a page: about 180, 40 of them conversions.  K by the 8-bit MMA instead (its operands as they are, the query in two
// parts) took as long: that instruction unpacks to f16 itself.
//
// Split: with few (token, KV head) pairs the pages of one are shared by the CTAs of a cluster, joined through distributed
// shared memory: no workspace, so calls never share memory, and one launch.
#include <atomic>
#include <type_traits>

#include "e4m3_cache.cuh"
#include "e4m3_cache.h"
#include "e4m3_visible.cuh"
#include "launch.h"

namespace lfm25 {

namespace {

constexpr float kHeadroom = 4.0f;        // log2 of the largest weight against that of the reference maximum
constexpr float kLift = 11.0f;           // log2 of that of the reference maximum
constexpr float kUnlift = 1.0f / 2048.0f;
static_assert(kHeadroom + kLift < 16.0f, "f16 ends in front of 2^16");
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
    uint32_t splits;       // CTAs of a cluster, a power of two
    uint32_t splits_log2;
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

__device__ __forceinline__ void copy_async_16(uint32_t to, const void* from, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "l"(policy) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <uint32_t PENDING>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}
__device__ __forceinline__ uint4 load_shared_16(uint32_t address) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ uint2 load_shared_8(uint32_t address) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(address) : "memory");
    return v;
}

template <uint32_t DIM>
struct Page {
    static constexpr uint32_t kSide = kPageSize * DIM;         // bytes of K, and of V
    static constexpr uint32_t kStage = 2 * kSide;
    // Key of a page that lane (g, t) takes for column 2 t + e of the score tile k, i.e. for the reduction step 8 k + 2 t + e of
    // P V.  K is read 8 lanes at a time (two keys, e = 0 and 1, times 4 pieces), V 16 lanes at 64 dimensions (four keys, the t,
    // times two pieces) and 8 at 128 (four keys times two pieces); a row has its 16-byte pieces at piece ^ turn(row).
    //   64: two rows are 128 bytes.  Neighbours for e; for the t every second pair is swapped, and pieces turn with bit 2.
    //   128: a row is 128 bytes.  Rows 4 apart for e, 0 2 5 7 for the t: piece ^ row takes eight different values in both.
    static __device__ __forceinline__ uint32_t key_of(uint32_t k, uint32_t t, uint32_t e) {
        return DIM == 64 ? 8 * k + 2 * t + (e ^ (t & 1)) : 8 * k + ((2 * t + (t >> 1)) ^ (4 * e));
    }
    static __device__ __forceinline__ uint32_t turn(uint32_t row) { return DIM == 64 ? (row >> 1) & 2 : row & 7; }
};

// HEADS: query heads of the CTA, at most 8 or at most 16; WARPS: 4 or 8
template <uint32_t DIM, uint32_t HEADS, uint32_t WARPS>
struct Shape {
    static constexpr uint32_t kWarps = WARPS;
    static constexpr uint32_t kThreads = kWarps * 32;
    // Pages that a warp works on side by side, and warps that an SM holds with the registers this takes.  One page is one chain of
    // dependent instructions, 0.37 us for a warp by itself; two take 0.23 us each.  At 64 dimensions two pages and 16 warps beat one
    // and 24 (128 tokens at contexts 128..4096: 50.2 against 54.2 us; 16 heads: 39.8 at 12 warps against 44.8), at 128 and up to 8 heads
    // one and 12 beat two and 8 (100 tokens at contexts 500..5000: 33.9 against 38.2 us), at 128 and 16 heads two beat one at 8
    // warps each (32.4 against 35.0 us).
    static constexpr uint32_t kPages = DIM == 128 && HEADS == 8 ? 1 : 2;
    static constexpr uint32_t kWarpsPerSm = DIM == 64 ? (HEADS == 8 ? 16 : 12) : (HEADS == 8 ? 12 : 8);
    static constexpr uint32_t kPerSm = kWarpsPerSm / WARPS;
    static constexpr uint32_t kStages = 3;                     // so many groups of pages on the way
    static constexpr uint32_t kStride = DIM + 4;               // a head's sums, maximum and sum of weights
    static constexpr uint32_t kRing = kWarps * kStages * kPages * Page<DIM>::kStage;
    static constexpr uint32_t kMerge = kWarps * HEADS * kStride * 4;          // in the ring's place, once that is done with
    static constexpr uint32_t kQuery = kRing > kMerge ? kRing : kMerge;       // f16 [HEADS][DIM], then HEADS factors
    static constexpr uint32_t kJoined = kQuery + HEADS * DIM * 2 + HEADS * 4;
    static constexpr uint32_t kBytes = kJoined + HEADS * kStride * 4 + 16;
};

template <uint32_t DIM, uint32_t HEADS, uint32_t WARPS>
__global__ void __launch_bounds__(Shape<DIM, HEADS, WARPS>::kThreads, Shape<DIM, HEADS, WARPS>::kPerSm)
e4m3_attention_kernel(const DecodeParams p) {
    using S = Shape<DIM, HEADS, WARPS>;
    using P = Page<DIM>;
    constexpr uint32_t kWarps = S::kWarps;
    constexpr uint32_t kStages = S::kStages;
    constexpr uint32_t NP = S::kPages;
    constexpr uint32_t kGroup = NP * P::kStage;
    constexpr uint32_t STRIDE = S::kStride;
    constexpr uint32_t C = DIM / 64;
    constexpr uint32_t TILES = DIM / 16;         // of 16 dimensions, rows of O^T
    constexpr uint32_t NT = HEADS / 8;           // tiles of 8 heads, columns of O^T
    extern __shared__ __align__(16) uint8_t decode_smem[];
    float* merge = reinterpret_cast<float*>(decode_smem);
    float* joined = reinterpret_cast<float*>(decode_smem + S::kJoined);     // this CTA's share, for its cluster
    uint32_t* unassigned = reinterpret_cast<uint32_t*>(joined + HEADS * STRIDE);
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t g = lane >> 2;
    const uint32_t t = lane & 3;
    pdl_launch_dependents();
    pdl_wait();

    // ---- which token, KV head, heads and share; every early exit is one of the whole cluster ----
    const uint32_t split = blockIdx.x & (p.splits - 1);
    uint32_t item = blockIdx.x >> p.splits_log2;
    uint32_t chunk = 0;
    if (p.chunks > 1) {
        chunk = item % p.chunks;
        item /= p.chunks;
    }
    const uint32_t rank = item / p.cache.kv_heads;
    const uint32_t kv_head = item - rank * p.cache.kv_heads;
    const uint32_t token = p.token_order != nullptr ? p.token_order[rank] : rank;
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
    const uint32_t share_begin = static_cast<uint32_t>(static_cast<uint64_t>(pages.count) * split >> p.splits_log2);
    const uint32_t share_end = static_cast<uint32_t>(static_cast<uint64_t>(pages.count) * (split + 1) >> p.splits_log2);
    const uint32_t groups = (share_end - share_begin + NP - 1) / NP;
    const uint32_t my_groups = groups > warp ? (groups - warp + kWarps - 1) / kWarps : 0;

    // ---- pages: table entries and scales 32 pages at a time, a lane each; codes up to kStages pages ahead ----
    const uint32_t ring = smem_u32(decode_smem) + warp * kStages * kGroup;
    const uint64_t policy = l2_evict_first_policy();     // a page is read once a step
    const uint32_t page_bytes = p.cache.kv_heads * P::kSide;
    // this lane's pieces of a page are 512 bytes apart, on either side
    const uint8_t* key_source = p.cache.key_codes + static_cast<size_t>(kv_head) * P::kSide + lane * 16;
    const uint8_t* value_source = p.cache.value_codes + static_cast<size_t>(kv_head) * P::kSide + lane * 16;
    uint32_t place[P::kSide / 512];
#pragma unroll
    for (uint32_t i = 0; i < P::kSide / 512; ++i) {
        const uint32_t piece = i * 32 + lane;
        const uint32_t row = piece / (DIM / 16);
        place[i] = ring + row * DIM + (((piece % (DIM / 16)) ^ P::turn(row)) << 4);
    }
    constexpr uint32_t kBlock = 32 / NP;                   // groups whose entries the lanes hold
    auto look_up = [&](uint32_t group) -> uint32_t {       // entry of this lane's page of the groups from `group` on
        const uint32_t index = share_begin + (warp + (group + lane / NP) * kWarps) * NP + lane % NP;
        return index < share_end ? __ldg(table + pages.logical(index)) : 0;
    };
    uint32_t coming = look_up(0);
    uint32_t entries = 0;
    uint32_t bad = 0;
    uint32_t block = 0;                                  // first group of those whose entries are at hand
    float scales[2][2];                                  // of these pages and of the ones before, for K and V
    scales[0][0] = scales[0][1] = 0.0f;
    uint32_t fill = 0;                                   // ring place of the next group to come, in bytes
    auto fetch = [&](uint32_t group) {
        if (group % kBlock == 0) {
            entries = coming;
            block = group;
            coming = look_up(group + kBlock);
            if (entries >= p.cache.num_pages) {
                bad = 1;                                 // page 0 in its place; the token gets no result
                entries = 0;
            }
            // a page that is not there is masked, and its scales are 0: a weight of 0 times a stray scale could be NaN
            const bool exists = share_begin + (warp + (group + lane / NP) * kWarps) * NP + lane % NP < share_end;
            const uint64_t tile = static_cast<uint64_t>(entries) * p.cache.kv_heads + kv_head;
            scales[1][0] = scales[0][0];
            scales[1][1] = scales[0][1];
            scales[0][0] = exists ? __ldg(p.cache.key_scales + tile) : 0.0f;
            scales[0][1] = exists ? __ldg(p.cache.value_scales + tile) : 0.0f;
        }
#pragma unroll
        for (uint32_t j = 0; j < NP; ++j) {              // a page behind the share's last: page 0, masked later
            const uint64_t offset = static_cast<uint64_t>(__shfl_sync(0xffffffffu, entries, group % kBlock * NP + j)) * page_bytes;
            const uint8_t* key = key_source + offset;
            const uint8_t* value = value_source + offset;
#pragma unroll
            for (uint32_t i = 0; i < P::kSide / 512; ++i) {
                copy_async_16(place[i] + fill + j * P::kStage, key + i * 512, policy);
                copy_async_16(place[i] + fill + j * P::kStage + P::kSide, value + i * 512, policy);
            }
        }
        fill = fill + kGroup == kStages * kGroup ? 0 : fill + kGroup;
    };
#pragma unroll
    for (uint32_t i = 0; i < kStages; ++i) {
        if (i < my_groups) fetch(i);
        copies_commit();
    }

    // ---- query, in f16 by a power of two per head, for all warps: 8 elements a thread ----
    {
        constexpr uint32_t kLanes = DIM / 8;               // of a head
        uint8_t* query = decode_smem + S::kQuery;
        float* factors = reinterpret_cast<float*>(query + HEADS * DIM * 2);
        for (uint32_t piece = threadIdx.x; piece < HEADS * kLanes; piece += S::kThreads) {   // whole warps, or none of one
            const uint32_t head = piece / kLanes;
            uint4 raw = make_uint4(0, 0, 0, 0);
            if (head < heads) {
                raw = *reinterpret_cast<const uint4*>(p.query + token * p.query_token_stride + (first_head + head) * DIM + piece % kLanes * 8);
            }
            const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
            uint32_t largest = 0;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t low = words[i] & 0x7fffu;
                const uint32_t high = (words[i] >> 16) & 0x7fffu;
                largest = max(largest, max(low < 0x7f80u ? low : 0u, high < 0x7f80u ? high : 0u));
            }
#pragma unroll
            for (uint32_t delta = kLanes / 2; delta > 0; delta >>= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, delta));
            // the power of two that brings the largest into [2^11, 2^12), within what f32 can multiply by
            const int32_t exponent = min(max(static_cast<int32_t>(largest >> 7) - 127 - 11, -126), 126);
            const float scale = power_of_two(-exponent);
            uint32_t halves[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const float2 pair = bf16x2_to_float2(words[i]);
                halves[i] = pack_f16x2(pair.x * scale, pair.y * scale);
            }
            *reinterpret_cast<uint4*>(query + piece * 16) = make_uint4(halves[0], halves[1], halves[2], halves[3]);
            if (piece % kLanes == 0) factors[head] = power_of_two(exponent) * p.scale_log2;
        }
        if (threadIdx.x == 0) *unassigned = 0;
    }
    __syncthreads();
    // rows g and g + 8 of A, dimensions 64 c + 16 t + 4 ks .. + 3 in step (c, ks)
    uint32_t q[NT][C][8];
    float query_factor[NT];
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
        const uint32_t row = smem_u32(decode_smem) + S::kQuery + (g + 8 * n) * DIM * 2 + t * 32;
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint4 part = load_shared_16(row + c * 128 + h * 16);
                q[n][c][4 * h] = part.x;
                q[n][c][4 * h + 1] = part.y;
                q[n][c][4 * h + 2] = part.z;
                q[n][c][4 * h + 3] = part.w;
            }
        }
        query_factor[n] = reinterpret_cast<const float*>(decode_smem + S::kQuery + HEADS * DIM * 2)[g + 8 * n];
    }

    float maximum[NT];          // of head g + 8 n, the reference of its weights (log2 units)
    float limit[NT];            // above it the reference is raised
    float sum[NT];              // of this lane's weights
    float2 out[NT][TILES][2];   // [tile of heads][tile][row g or g + 8]: heads 2 t and 2 t + 1
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
        maximum[n] = limit[n] = -INFINITY;
        sum[n] = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < TILES; ++i) out[n][i][0] = out[n][i][1] = make_float2(0.0f, 0.0f);
    }

    // where this lane reads: K of its column (key_of(k, g / 2, g % 2)), V of its keys
    uint32_t key_at[C];
    {
        const uint32_t row = P::key_of(0, g >> 1, g & 1);
#pragma unroll
        for (uint32_t c = 0; c < C; ++c) key_at[c] = row * DIM + (((4 * c + t) ^ P::turn(row)) << 4);
    }
    uint32_t value_at[2];
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e) {
        const uint32_t row = P::key_of(0, t, e);
        value_at[e] = P::kSide + row * DIM + (DIM == 64 ? (((g >> 1) ^ P::turn(row)) << 4) + (g & 1) * 8 : (g ^ P::turn(row)) << 4);
    }

    uint32_t drain = ring;                               // ring place of the next group to use
    auto use = [&](uint32_t group, uint32_t index, auto masked) {
        float s[NP][2][4];
        uint2 value[NP][4][C];
        float value_scale[NP];
        float factor[NP][NT];
#pragma unroll
        for (uint32_t j = 0; j < NP; ++j) {
            const uint32_t stage = drain + j * P::kStage;
            // ---- scores of two tiles of 8 keys: head g, keys key_of(k, t, 0 and 1); head g + 8, the same ----
            uint4 codes[2][C];
#pragma unroll
            for (uint32_t k = 0; k < 2; ++k) {
#pragma unroll
                for (uint32_t c = 0; c < C; ++c) codes[k][c] = load_shared_16(stage + key_at[c] + k * 8 * DIM);
            }
#pragma unroll
            for (uint32_t c = 0; c < C; ++c) {
#pragma unroll
                for (uint32_t ks = 0; ks < 4; ++ks) {
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k) {
                        const uint32_t word = ks == 0 ? codes[k][c].x : ks == 1 ? codes[k][c].y : ks == 2 ? codes[k][c].z : codes[k][c].w;
                        const uint32_t a1 = NT > 1 ? q[NT - 1][c][2 * ks] : 0u;
                        const uint32_t a3 = NT > 1 ? q[NT - 1][c][2 * ks + 1] : 0u;
                        if (c == 0 && ks == 0) {
                            mma_f16_16816_first(s[j][k], q[0][c][0], a1, q[0][c][1], a3, e4m3x2_to_f16x2(word), e4m3x2_high_to_f16x2(word));
                        } else {
                            mma_f16_16816(s[j][k], q[0][c][2 * ks], a1, q[0][c][2 * ks + 1], a3, e4m3x2_to_f16x2(word), e4m3x2_high_to_f16x2(word));
                        }
                    }
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t at = stage + value_at[i & 1] + (i >> 1) * 8 * DIM;
                if constexpr (C == 1) {
                    value[j][i][0] = load_shared_8(at);
                } else {
                    const uint4 both = load_shared_16(at);
                    value[j][i][0] = make_uint2(both.x, both.y);
                    value[j][i][C - 1] = make_uint2(both.z, both.w);
                }
            }
            const uint32_t source = group % kBlock * NP + j;
            const float key_scale = __shfl_sync(0xffffffffu, group >= block ? scales[0][0] : scales[1][0], source);
            value_scale[j] = __shfl_sync(0xffffffffu, group >= block ? scales[0][1] : scales[1][1], source) * kUnlift;
            // never 0, so that -inf stays what it is (a score is below 2^28: with this factor it is 0)
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) factor[j][n] = fmaxf(key_scale * query_factor[n], 1.1754944e-38f);
            if constexpr (decltype(masked)::value) {
                const uint32_t base = pages.logical(index + j) * kPageSize;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t key = base + P::key_of(i >> 1, t, i & 1);
                    if (index + j >= share_end || key > position || (key < pages.first_key && key >= p.sinks)) {
                        // whatever lies there, a weight of 0 must not meet a NaN
#pragma unroll
                        for (uint32_t c = 0; c < C; ++c) value[j][i][c] = make_uint2(0, 0);
#pragma unroll
                        for (uint32_t n = 0; n < NT; ++n) s[j][i >> 1][2 * n + (i & 1)] = -INFINITY;
                    }
                }
            }
        }
        // ---- the reference maximum ----
        float most[NT];
        bool above = false;
#pragma unroll
        for (uint32_t n = 0; n < NT; ++n) {
            most[n] = -INFINITY;
#pragma unroll
            for (uint32_t j = 0; j < NP; ++j) {
                most[n] = fmaxf(most[n], fmaxf(max3(s[j][0][2 * n], s[j][0][2 * n + 1], s[j][1][2 * n]), s[j][1][2 * n + 1]) * factor[j][n]);
            }
            above = above || most[n] > limit[n];
        }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) {
                most[n] = fmaxf(most[n], __shfl_xor_sync(0xffffffffu, most[n], 1));
                most[n] = fmaxf(most[n], __shfl_xor_sync(0xffffffffu, most[n], 2));
                most[n] = fmaxf(most[n], maximum[n]);
                // a row that has seen nothing yet keeps its sums of 0: exp2(-inf - -inf) is no factor
                const float shrink = most[n] == maximum[n] ? 1.0f : fast_exp2(maximum[n] - most[n]);
                maximum[n] = most[n];
                limit[n] = most[n] + kHeadroom;
                sum[n] *= shrink;
                const float low = __shfl_sync(0xffffffffu, shrink, 8 * t);
                const float high = __shfl_sync(0xffffffffu, shrink, 8 * t + 4);
#pragma unroll
                for (uint32_t i = 0; i < TILES; ++i) {
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) out[n][i][h] = make_float2(out[n][i][h].x * low, out[n][i][h].y * high);
                }
            }
        }
        // ---- weights ----
        uint32_t weights[NP][NT][2];
#pragma unroll
        for (uint32_t j = 0; j < NP; ++j) {
#pragma unroll
            for (uint32_t n = 0; n < NT; ++n) {
                float w[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) w[i] = fast_exp2(fmaf(s[j][i >> 1][2 * n + (i & 1)], factor[j][n], kLift - maximum[n]));
                weights[j][n][0] = pack_f16x2(w[0], w[1]);
                weights[j][n][1] = pack_f16x2(w[2], w[3]);
                // the sum of the weights before their rounding to 11 bits, which averages out over the keys
                sum[n] += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }
        // ---- O^T += scale * V^T P^T ----
#pragma unroll
        for (uint32_t j = 0; j < NP; ++j) {
#pragma unroll
            for (uint32_t tile = 0; tile < TILES; tile += 2) {
                // dimensions 2 tile .. 2 tile + 3 of this lane's DIM / 8: one byte each of a word
                uint32_t word[4];
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) word[k] = tile & 2 ? value[j][k][tile / 4].y : value[j][k][tile / 4].x;
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
                        float d[4];
                        mma_f16_16816_first(d, a0, a1, a2, a3, weights[j][n][0], weights[j][n][1]);
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            float2& o = out[n][tile + half][h];
                            o = fma_pair(make_float2(d[2 * h], d[2 * h + 1]), value_scale[j], o);
                        }
                    }
                }
            }
        }
    };

    uint32_t index = share_begin + warp * NP;
    for (uint32_t group = 0; group < my_groups; ++group) {
        copies_wait<kStages - 1>();
        __syncwarp();                                  // every lane's pieces are there
        const uint32_t first = pages.logical(index) * kPageSize;
        // Only pages at an edge of what the token sees have a mask.  (A group that is no run of pages has an edge: it holds the last
        // page of the first tokens, or pages in front of the window's.)
        const bool whole = index + NP <= share_end && first + NP * kPageSize - 1 <= position &&
                           (first >= pages.first_key || first + NP * kPageSize <= p.sinks);
        if (whole) {
            use(group, index, std::false_type());
        } else {
            use(group, index, std::true_type());
        }
        index += kWarps * NP;
        drain = drain + kGroup == ring + kStages * kGroup ? ring : drain + kGroup;
        __syncwarp();                                  // and read by all
        if (group + kStages < my_groups) fetch(group + kStages);
        copies_commit();
    }
    if (__any_sync(0xffffffffu, bad != 0) && lane == 0) *unassigned = 1;
    copies_wait<0>();
    __syncthreads();                                   // the ring's place is free

    // ---- join the warps: O^T of lane (g, t) has dimensions DIM / 8 * g + 2 tile + h of the heads 8 n + 2 t, + 1 ----
#pragma unroll
    for (uint32_t n = 0; n < NT; ++n) {
        sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 1);
        sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 2);
        sum[n] *= kUnlift;
        float* mine = merge + warp * HEADS * STRIDE;
        if (t == 0) {
            mine[(8 * n + g) * STRIDE + DIM] = maximum[n];
            mine[(8 * n + g) * STRIDE + DIM + 1] = sum[n];
        }
        if (8 * n + 2 * t < heads) {
            float4* low = reinterpret_cast<float4*>(mine + (8 * n + 2 * t) * STRIDE + (DIM / 8) * g);
            float4* high = reinterpret_cast<float4*>(mine + (8 * n + 2 * t + 1) * STRIDE + (DIM / 8) * g);
#pragma unroll
            for (uint32_t i = 0; i < TILES; i += 2) {
                low[i / 2] = make_float4(out[n][i][0].x, out[n][i][1].x, out[n][i + 1][0].x, out[n][i + 1][1].x);
                high[i / 2] = make_float4(out[n][i][0].y, out[n][i][1].y, out[n][i + 1][0].y, out[n][i + 1][1].y);
            }
        }
    }
    __syncthreads();
    for (uint32_t index = threadIdx.x; index < heads * DIM; index += S::kThreads) {
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
                joined[head * STRIDE + DIM + 1] = *unassigned ? kNoResult : total;
            }
        } else if (*unassigned == 0) {
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
    for (uint32_t index = split * share + threadIdx.x; index < end; index += S::kThreads) {
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

// Whether the device holds a cluster of 16 CTAs of this shape, which needs as many places in one group of SMs: asked once per device.
template <uint32_t DIM, uint32_t HEADS, uint32_t WARPS>
bool clusters_of_16_fit() {
    using S = Shape<DIM, HEADS, WARPS>;
    static std::atomic<uint64_t> asked{0}, fits{0};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return false;
    const uint64_t bit = uint64_t{1} << (device & 63);
    if ((asked.load(std::memory_order_acquire) & bit) == 0) {
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(16, 1, 1);
        config.blockDim = dim3(S::kThreads, 1, 1);
        config.dynamicSmemBytes = S::kBytes;
        cudaLaunchAttribute attribute;
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim.x = 16;
        attribute.val.clusterDim.y = 1;
        attribute.val.clusterDim.z = 1;
        config.attrs = &attribute;
        config.numAttrs = 1;
        int clusters = 0;
        if (allow_shared_memory<e4m3_attention_kernel<DIM, HEADS, WARPS>, true>(S::kBytes) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&clusters, e4m3_attention_kernel<DIM, HEADS, WARPS>, &config) != cudaSuccess) {
            (void)cudaGetLastError();
            clusters = 0;
        }
        if (clusters > 0) fits.fetch_or(bit, std::memory_order_relaxed);
        asked.fetch_or(bit, std::memory_order_release);
    }
    return (fits.load(std::memory_order_relaxed) & bit) != 0;
}

template <uint32_t DIM, uint32_t HEADS, uint32_t WARPS>
cudaError_t launch_shape(cudaStream_t stream, const DecodeParams& params, uint64_t blocks) {
    using S = Shape<DIM, HEADS, WARPS>;
    const cudaError_t status = allow_shared_memory<e4m3_attention_kernel<DIM, HEADS, WARPS>, true>(S::kBytes);
    if (status != cudaSuccess) {
        return status;
    }
    return launch_kernel(e4m3_attention_kernel<DIM, HEADS, WARPS>, static_cast<unsigned int>(blocks), S::kThreads, S::kBytes, stream,
                         params.splits, params);
}

// (token, KV head, chunk of query heads) triples, and pages of the longest context that a token can see
struct DecodeWork {
    uint64_t items;
    uint64_t pages;
};

DecodeWork decode_work(const E4m3AttentionLaunch& launch) {
    const uint64_t group = launch.query_heads / launch.cache.kv_heads;
    uint64_t longest = launch.maximum_context_tokens;
    if (launch.window != 0 && longest > static_cast<uint64_t>(launch.window) + launch.sinks) {
        longest = static_cast<uint64_t>(launch.window) + launch.sinks + kPageSize;
    }
    return {static_cast<uint64_t>(launch.num_tokens) * launch.cache.kv_heads * ((group + 15) / 16), (longest + kPageSize - 1) / kPageSize};
}

// Clusters of 1, 2, 4, 8 and 16 CTAs that a B200 holds at once, with 1 to 4 CTAs an SM, as cudaOccupancyMaxActiveClusters answers: a
// cluster stays within one group of SMs.
constexpr uint32_t kResidentClusters[4][5] = {{148, 74, 33, 15, 7}, {296, 148, 71, 33, 14}, {444, 222, 104, 48, 21}, {592, 296, 142, 71, 31}};

// CTAs of 4 warps, their pages shared by a cluster of as many (up to 16) as fill the SMs once, a quarter over, while each warp
// has 8 pages or more; where all clusters run at once with CTAs of 8 warps, those.  Of 32 heads on 8 of 64, 1 token at 8000: 8 CTAs of 8
// warps 8.3, 16 of 4 8.7, 8 of 4 9.0 us; 32 at 64..400: 1 CTA of 8 warps 5.7, of 4 6.5, 2 of 4 7.3 us.  Of 8 heads on 2 of 128, 4 tokens
// at 8000..16000: 8 of 8 15.5, 16 of 4 15.0, 16 of 8 19.5 us; 100 at 500..5000: 2 of 4 34.4, 1 of 8 39.2, 1 of 4 45.5 us.
// Clusters that do not all run at once cost their whole time again for the last ones: 16 of 8 CTAs of 8 warps where 15 find room take
// 13.7 us (16 tokens at 4000, 16 heads on 1 of 64) and 16 CTAs of 4 warps 10.0, at heads of 128 20.2 us and 8 of 4 14.6.
// 16 wide CTAs from 2 pages a warp on where they do run at once (1 token at 16000, 16 on 1 of 64: 9.6 against 12.0 us with 8; 8 on 2 of
// 128: 10.8 and 14.8; 16 on 1 of 128: 13.7 and 17.7; 32 on 8 of 64: 11.5 and 11.9).
// Beyond 48 pages a warp of 8 CTAs the longest context decides, and shares as short as they get win over running at once (3 tokens at
// 20480..65536, 32 on 8 of 64: 16 CTAs of 4 warps 36.5, 8 of 8 40.4 us; 2 at 65536: 16 of 8 34.2, 8 of 8 40.2; 12 at 1250..50000, 8 on 2
// of 128: 45.0 with 16 of 4).  Not known to the host, and so not in the rule, is how unequal the contexts of a batch are: over 399
// batches of four layouts, 1 to 128 tokens at 300..65536, it is 5 % from the best form where contexts are alike and 7 % where they are
// spread from 1/40 on, 56 % at worst (64 tokens at 4000, 16 on 1 of 64: 22.2 us in clusters of 8, 14.2 in clusters of 2 wide ones).
template <uint32_t DIM, uint32_t HEADS>
E4m3DecodePlan plan_heads(const DecodeWork& work, bool clusters_of_16) {
    using S = Shape<DIM, HEADS, 4>;
    constexpr uint64_t kSms = 148;
    constexpr uint64_t kSlots = kSms * S::kPerSm;
    constexpr auto& kNarrow = kResidentClusters[S::kPerSm - 1];
    constexpr auto& kWide = kResidentClusters[Shape<DIM, HEADS, 8>::kPerSm - 1];
    const bool long_contexts = work.pages >= 48 * 8 * 8;
    auto wide_fits = [&](uint32_t splits_log2) {
        return long_contexts ? (work.items << splits_log2) * 8 <= kSms * S::kWarpsPerSm : work.items <= kWide[splits_log2];
    };
    if (clusters_of_16 && !long_contexts && work.pages >= 2 * 8 * 16 && wide_fits(4)) {
        return {8, 4};
    }
    const uint32_t most = clusters_of_16 && (long_contexts || work.items <= kNarrow[4]) ? 4 : 3;
    E4m3DecodePlan plan = {4, 0};
    while (plan.splits_log2 < most && (work.items << (plan.splits_log2 + 1)) <= kSlots + kSlots / 4 &&
           work.pages >= (8ull * 4 << plan.splits_log2)) {
        ++plan.splits_log2;
    }
    if (plan.splits_log2 == 4 && !long_contexts && wide_fits(3)) plan.splits_log2 = 3;
    if (wide_fits(plan.splits_log2)) plan.warps = 8;
    return plan;
}

template <uint32_t DIM, uint32_t HEADS>
cudaError_t launch_heads(cudaStream_t stream, DecodeParams params, const DecodeWork& work) {
    E4m3DecodePlan plan = plan_heads<DIM, HEADS>(work, true);
    if (plan.splits_log2 == 4 && !(plan.warps == 8 ? clusters_of_16_fit<DIM, HEADS, 8>() : clusters_of_16_fit<DIM, HEADS, 4>())) {
        plan = plan_heads<DIM, HEADS>(work, false);
    }
    params.splits_log2 = plan.splits_log2;
    params.splits = 1u << plan.splits_log2;
    const uint64_t blocks = work.items << plan.splits_log2;
    if (blocks > 0x7fffffffu) {
        return cudaErrorInvalidConfiguration;
    }
    return plan.warps == 8 ? launch_shape<DIM, HEADS, 8>(stream, params, blocks) : launch_shape<DIM, HEADS, 4>(stream, params, blocks);
}

}  // namespace

E4m3DecodePlan plan_e4m3_attention(const E4m3AttentionLaunch& launch, bool clusters_of_16) {
    const DecodeWork work = decode_work(launch);
    const bool few = launch.query_heads / launch.cache.kv_heads <= 8;
    if (launch.cache.head_dim == 64) {
        return few ? plan_heads<64, 8>(work, clusters_of_16) : plan_heads<64, 16>(work, clusters_of_16);
    }
    return few ? plan_heads<128, 8>(work, clusters_of_16) : plan_heads<128, 16>(work, clusters_of_16);
}

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
    const DecodeWork work = decode_work(launch);
    if (work.items > 0x7fffffffu) {
        return cudaErrorInvalidConfiguration;
    }
    if (launch.cache.head_dim == 64) {
        return params.group <= 8 ? launch_heads<64, 8>(stream, params, work) : launch_heads<64, 16>(stream, params, work);
    }
    return params.group <= 8 ? launch_heads<128, 8>(stream, params, work) : launch_heads<128, 16>(stream, params, work);
}

}  // namespace lfm25
