// Which keys a token sees, and the pages that hold them: j <= position and (no window, or j > position - window, or
// j < sinks).  The pages of the first tokens come first in the list, then those from the window's first key on; pages
// between the two are never looked at (they may have been given back).
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace lfm25 {

struct VisiblePages {
    uint32_t first_key;    // of the window (0 without one)
    uint32_t sink_pages;   // pages in front of the window's that hold first tokens
    uint32_t first_page;   // of the window
    uint32_t count;        // pages in the list

    // tokens at positions first .. last, which all look through the same window rule
    __device__ __forceinline__ VisiblePages(uint32_t first, uint32_t last, uint32_t window, uint32_t sinks) {
        first_key = window != 0 && first >= window ? first - window + 1 : 0;
        first_page = first_key / kPageSize;
        sink_pages = min((sinks + kPageSize - 1) / kPageSize, first_page);
        count = sink_pages + last / kPageSize - first_page + 1;
    }
    __device__ __forceinline__ uint32_t logical(uint32_t index) const {
        return index < sink_pages ? index : first_page + (index - sink_pages);
    }
};

}  // namespace lfm25
