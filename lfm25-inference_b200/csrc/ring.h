// Rings of buffers in shared memory that a producer fills by turns.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LFM25_RING_FUNCTION __host__ __device__ __forceinline__ constexpr
#else
#define LFM25_RING_FUNCTION constexpr inline
#endif

namespace lfm25 {

// Whether the buffer that holds item `index` of `items` is filled once more, and so whether its producer waits for it to be
// free.  The tensor core reports a free buffer by an arrival of its own (tcgen05.commit): one that nobody waits for may come
// after its CTA has ended and its shared memory is gone, so it is not asked for.
LFM25_RING_FUNCTION bool filled_again(uint32_t index, uint32_t items, uint32_t buffers) { return items - index > buffers; }

// Whether item `index` of `items` is the last that its set takes, where `sets` take items by turns.
LFM25_RING_FUNCTION bool last_of_set(uint32_t index, uint32_t items, uint32_t sets) { return items - index <= sets; }

}  // namespace lfm25
