// Copies of pages of key/value caches, for all layers at once: sequences that fork get a copy of their last, partly filled
// page, and compaction moves the pages of a pool.
//
// The caches of a model are a list of arenas with pages of different sizes (keys, values, scales of every layer) and the same
// page numbers.  One launch copies every pair in every arena.  The unit of work is a piece of a page, or as many pages of one
// arena as make up a piece (scales of a page are a few words); a warp takes pieces by turns and moves each 16 bytes a lane with
// four loads in flight.  Pages that are no multiple of 16 bytes (scales of a few heads) go word by word.  Bound by HBM, read
// once and written once: 2048 pages of 8 KiB in 12 arenas of codes with their scales, 404 MB of traffic, in 71.3 us (5.7 TB/s,
// 0.88 of a plain copy).  Warps that take pieces by turns save the start of 50,000 CTAs (a CTA a piece: 74 to 107 us, the
// shorter the piece the longer); 4 CTAs an SM hide the two loads one behind the other, and 6 gain nothing (72.6 us).
#include "common.cuh"
#include "e4m3_cache.h"
#include "launch.h"

namespace lfm25 {

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kResident = 4;   // CTAs of an SM
constexpr uint32_t kLoads = 4;

struct CopyParams {
    PageArena arenas[kMaxPageArenas];
    uint32_t first_piece[kMaxPageArenas + 1];   // pieces of arena a: first_piece[a] .. first_piece[a + 1]
    const uint32_t* source_pages;
    const uint32_t* destination_pages;
    uint32_t num_arenas;
    uint32_t num_pairs;
};

__host__ __device__ inline bool by_16_bytes(const PageArena& a) {
    return ((a.page_bytes | reinterpret_cast<uintptr_t>(a.base)) & 15) == 0;
}

// bytes of a piece of this arena at most
__host__ __device__ inline uint32_t piece_bytes(const PageArena& a) {
    return 32 * kLoads * (by_16_bytes(a) ? 16 : 4);
}

// pairs of a piece in an arena of small pages, pieces of a pair in one of large pages
__host__ __device__ inline uint32_t pairs_of_piece(const PageArena& a) {
    return a.page_bytes < piece_bytes(a) ? piece_bytes(a) / static_cast<uint32_t>(a.page_bytes) : 1;
}

__host__ __device__ inline uint32_t pieces_of_page(const PageArena& a) {
    return static_cast<uint32_t>((a.page_bytes + piece_bytes(a) - 1) / piece_bytes(a));
}

template <typename T>
__device__ __forceinline__ void copy_piece(const CopyParams& p, const PageArena& a, uint32_t piece) {
    const uint32_t lane = threadIdx.x % 32;
    const uint32_t pieces = pieces_of_page(a);
    const uint32_t first = piece / pieces * pairs_of_piece(a);
    const uint32_t pairs = min(pairs_of_piece(a), p.num_pairs - first);
    const uint64_t begin = static_cast<uint64_t>(piece % pieces) * piece_bytes(a);
    const uint32_t width = static_cast<uint32_t>(min(a.page_bytes - begin, static_cast<uint64_t>(piece_bytes(a)))) / sizeof(T);
    uint8_t* const base = static_cast<uint8_t*>(a.base) + begin;
    T held[kLoads];
    T* to[kLoads];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
        const uint32_t index = i * 32 + lane;
        const uint32_t pair = index / width;
        to[i] = nullptr;
        if (pair < pairs) {
            const uint32_t source = p.source_pages[first + pair];
            const uint32_t destination = p.destination_pages[first + pair];
            if (source < a.num_pages && destination < a.num_pages) {
                held[i] = reinterpret_cast<const T*>(base + source * a.page_bytes)[index % width];
                to[i] = reinterpret_cast<T*>(base + destination * a.page_bytes) + index % width;
            }
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
        if (to[i] != nullptr) *to[i] = held[i];
    }
}

// a piece that is all of one page's, without a look at the place of each value
__device__ __forceinline__ void copy_whole(const CopyParams& p, const PageArena& a, uint32_t piece) {
    const uint32_t pieces = pieces_of_page(a);
    const uint32_t source = p.source_pages[piece / pieces];
    const uint32_t destination = p.destination_pages[piece / pieces];
    if (source >= a.num_pages || destination >= a.num_pages) {
        return;
    }
    uint8_t* const base = static_cast<uint8_t*>(a.base) + static_cast<uint64_t>(piece % pieces) * piece_bytes(a);
    const uint4* const from = reinterpret_cast<const uint4*>(base + source * a.page_bytes) + threadIdx.x % 32;
    uint4* const to = reinterpret_cast<uint4*>(base + destination * a.page_bytes) + threadIdx.x % 32;
    uint4 held[kLoads];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) held[i] = from[i * 32];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) to[i * 32] = held[i];
}

__global__ void __launch_bounds__(kThreads, kResident)
kv_pages_copy_kernel(const __grid_constant__ CopyParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t total = p.first_piece[p.num_arenas];
    uint32_t arena = 0;
    for (uint32_t piece = blockIdx.x * kWarps + threadIdx.x / 32; piece < total; piece += gridDim.x * kWarps) {
        while (piece >= p.first_piece[arena + 1]) ++arena;
        const PageArena& a = p.arenas[arena];
        const uint32_t own = piece - p.first_piece[arena];
        if (!by_16_bytes(a)) {
            copy_piece<uint32_t>(p, a, own);
        } else if (a.page_bytes % (32 * kLoads * 16) != 0) {
            copy_piece<uint4>(p, a, own);
        } else {
            copy_whole(p, a, own);
        }
    }
}

uint64_t pieces_of(const PageArena& arena, size_t num_pairs) {
    const uint32_t pairs = pairs_of_piece(arena);
    return (num_pairs + pairs - 1) / pairs * pieces_of_page(arena);
}

}  // namespace

cudaError_t launch_kv_pages_copy(cudaStream_t stream, const PageArena* arenas, size_t num_arenas,
                                 const uint32_t* source_pages, const uint32_t* destination_pages, size_t num_pairs) {
    for (size_t first = 0; first < num_arenas; first += kMaxPageArenas) {
        uint64_t pieces = 0;
        for (size_t index = first; index < num_arenas && index < first + kMaxPageArenas; ++index) {
            pieces += pieces_of(arenas[index], num_pairs);
        }
        if (pieces > 0x7fffffffu) {
            return cudaErrorInvalidConfiguration;   // before anything is launched
        }
    }
    for (size_t first = 0; first < num_arenas; first += kMaxPageArenas) {
        CopyParams params;
        params.num_arenas = static_cast<uint32_t>(num_arenas - first < kMaxPageArenas ? num_arenas - first : kMaxPageArenas);
        params.num_pairs = static_cast<uint32_t>(num_pairs);
        params.source_pages = source_pages;
        params.destination_pages = destination_pages;
        uint64_t pieces = 0;
        for (uint32_t index = 0; index < params.num_arenas; ++index) {
            params.arenas[index] = arenas[first + index];
            params.first_piece[index] = static_cast<uint32_t>(pieces);
            pieces += pieces_of(arenas[first + index], num_pairs);
        }
        params.first_piece[params.num_arenas] = static_cast<uint32_t>(pieces);
        const uint64_t blocks = (pieces + kWarps - 1) / kWarps;
        const unsigned int grid = static_cast<unsigned int>(blocks < kResident * 148 ? blocks : kResident * 148);
        const cudaError_t status = launch_kernel(kv_pages_copy_kernel, grid, kThreads, 0, stream, 1, params);
        if (status != cudaSuccess) {
            return status;
        }
    }
    return cudaSuccess;
}

}  // namespace lfm25
