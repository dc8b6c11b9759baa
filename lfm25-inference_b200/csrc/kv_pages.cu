// Copies of pages of key/value caches, for all layers at once: sequences that fork get a copy of their last, partly filled
// page, and compaction moves the pages of a pool.
//
// The caches of a model are a list of arenas with pages of different sizes (keys, values, scales of every layer) and the same
// page numbers.  One launch copies every pair in every arena: a CTA takes pieces of 16 KiB of (arena, pair) and moves them 16
// bytes a thread with eight loads in flight.  Pages that are no multiple of 16 bytes (scales of a few heads) go word by word.
// Bound by HBM, read once and written once.
#include "common.cuh"
#include "e4m3_cache.h"
#include "launch.h"

namespace lfm25 {

namespace {

constexpr uint32_t kThreads = 128;
constexpr uint32_t kLoads = 8;
constexpr uint32_t kPieceBytes = kThreads * 16 * kLoads;

struct CopyParams {
    PageArena arenas[kMaxPageArenas];
    uint32_t first_block[kMaxPageArenas + 1];   // blocks of arena a: first_block[a] .. first_block[a + 1]
    const uint32_t* source_pages;
    const uint32_t* destination_pages;
    uint32_t num_arenas;
    uint32_t num_pairs;
};

// `step` bytes at a time (16 or 4), pairs of one block behind the other
template <typename T>
__device__ __forceinline__ void copy_piece(const uint8_t* source, uint8_t* destination, uint32_t bytes) {
    const T* from = reinterpret_cast<const T*>(source);
    T* to = reinterpret_cast<T*>(destination);
    const uint32_t count = bytes / sizeof(T);
    for (uint32_t base = threadIdx.x; base < count; base += kThreads * kLoads) {
        T held[kLoads];
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            if (base + i * kThreads < count) held[i] = from[base + i * kThreads];
        }
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
            if (base + i * kThreads < count) to[base + i * kThreads] = held[i];
        }
    }
}

__global__ void __launch_bounds__(kThreads)
kv_pages_copy_kernel(const __grid_constant__ CopyParams p) {
    pdl_launch_dependents();
    pdl_wait();
    uint32_t arena = 0;
    while (arena + 1 < p.num_arenas && blockIdx.x >= p.first_block[arena + 1]) ++arena;
    const PageArena& a = p.arenas[arena];
    const uint32_t block = blockIdx.x - p.first_block[arena];
    const uint64_t pieces = (a.page_bytes + kPieceBytes - 1) / kPieceBytes;
    const uint32_t pair = static_cast<uint32_t>(block / pieces);
    const uint64_t begin = (block % pieces) * kPieceBytes;
    const uint32_t from = p.source_pages[pair];
    const uint32_t to = p.destination_pages[pair];
    if (from >= a.num_pages || to >= a.num_pages) {
        return;
    }
    const uint8_t* source = static_cast<const uint8_t*>(a.base) + from * a.page_bytes + begin;
    uint8_t* destination = static_cast<uint8_t*>(a.base) + to * a.page_bytes + begin;
    const uint32_t bytes = static_cast<uint32_t>(a.page_bytes - begin < kPieceBytes ? a.page_bytes - begin : kPieceBytes);
    if (((a.page_bytes | reinterpret_cast<uintptr_t>(a.base)) & 15) == 0) {
        copy_piece<uint4>(source, destination, bytes);
    } else {
        copy_piece<uint32_t>(source, destination, bytes);
    }
}

uint64_t blocks_of(const PageArena& arena, size_t num_pairs) {
    return num_pairs * ((arena.page_bytes + kPieceBytes - 1) / kPieceBytes);
}

}  // namespace

cudaError_t launch_kv_pages_copy(cudaStream_t stream, const PageArena* arenas, size_t num_arenas,
                                 const uint32_t* source_pages, const uint32_t* destination_pages, size_t num_pairs) {
    for (size_t first = 0; first < num_arenas; first += kMaxPageArenas) {
        uint64_t blocks = 0;
        for (size_t index = first; index < num_arenas && index < first + kMaxPageArenas; ++index) {
            blocks += blocks_of(arenas[index], num_pairs);
        }
        if (blocks > 0x7fffffffu) {
            return cudaErrorInvalidConfiguration;   // before anything is launched
        }
    }
    for (size_t first = 0; first < num_arenas; first += kMaxPageArenas) {
        CopyParams params;
        params.num_arenas = static_cast<uint32_t>(num_arenas - first < kMaxPageArenas ? num_arenas - first : kMaxPageArenas);
        params.num_pairs = static_cast<uint32_t>(num_pairs);
        params.source_pages = source_pages;
        params.destination_pages = destination_pages;
        uint64_t blocks = 0;
        for (uint32_t index = 0; index < params.num_arenas; ++index) {
            params.arenas[index] = arenas[first + index];
            params.first_block[index] = static_cast<uint32_t>(blocks);
            blocks += blocks_of(arenas[first + index], num_pairs);
        }
        params.first_block[params.num_arenas] = static_cast<uint32_t>(blocks);
        const cudaError_t status = launch_kernel(kv_pages_copy_kernel, static_cast<unsigned int>(blocks), kThreads, 0, stream, 1, params);
        if (status != cudaSuccess) {
            return status;
        }
    }
    return cudaSuccess;
}

}  // namespace lfm25
