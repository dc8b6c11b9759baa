// The 8-bit paged key/value cache: launch arguments of its kernels (e4m3_cache_write.cu, e4m3_attention.cu,
// e4m3_attention_umma.cu) and of the page copies (kv_pages.cu).  Arguments are validated by the entry points in
// e4m3_api.cu.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace lfm25 {

// Codes [pages, kv_heads, 16, head_dim], scales [pages, kv_heads]; an element stands for code * scale.
struct E4m3Cache {
    uint8_t* key_codes;
    uint8_t* value_codes;
    float* key_scales;
    float* value_scales;
    uint32_t num_pages;
    uint32_t kv_heads;
    uint32_t head_dim;   // 64 or 128
};

struct E4m3WriteLaunch {
    E4m3Cache cache;
    const void* key;              // bf16 [tokens, kv_heads, head_dim], rows kv_token_stride elements apart
    const void* value;
    const int64_t* slot_mapping;  // [tokens]
    size_t num_tokens;
    size_t kv_token_stride;
    // with norms and rotation (query != nullptr)
    const void* query = nullptr;  // bf16 [tokens, query_heads, head_dim], rows query_token_stride elements apart
    void* query_out = nullptr;    // bf16 [tokens, query_heads, head_dim], dense
    const void* query_norm = nullptr;
    const void* key_norm = nullptr;
    const float* inv_freq = nullptr;
    const uint32_t* position_ids = nullptr;
    uint32_t query_heads = 0;
    size_t query_token_stride = 0;
    float eps = 0.0f;
};
cudaError_t launch_e4m3_cache_write(cudaStream_t stream, const E4m3WriteLaunch& launch);

struct E4m3AttentionLaunch {
    E4m3Cache cache;
    const void* query;             // bf16 [tokens, query_heads, head_dim], rows query_token_stride elements apart
    void* output;                  // bf16 [tokens, query_heads, head_dim], dense
    const uint32_t* block_tables;  // [rows, block_table_stride]
    const uint32_t* request_slots; // [tokens]
    const uint32_t* position_ids;  // [tokens]
    const uint32_t* token_order;   // single tokens only: permutation of the batch, or nullptr
    const uint32_t* segment_offsets;   // prompts only: [segments + 1]
    unsigned int* status;
    size_t num_tokens;
    size_t num_segments;
    size_t query_heads;
    size_t query_token_stride;
    size_t block_table_stride;
    size_t block_table_rows;
    size_t maximum_context_tokens; // longest context of the batch, for the choice of the split
    uint32_t window;               // 0: all keys up to the token's own
    uint32_t sinks;
    float scale;
};
cudaError_t launch_e4m3_attention(cudaStream_t stream, const E4m3AttentionLaunch& launch);

// How single tokens are shared out: warps of a CTA (4 or 8) and CTAs of a cluster, 1 << splits_log2, clusters of 16 only where the device
// holds them.
struct E4m3DecodePlan {
    uint32_t warps;
    uint32_t splits_log2;
};
E4m3DecodePlan plan_e4m3_attention(const E4m3AttentionLaunch& launch, bool clusters_of_16);
cudaError_t launch_e4m3_prompt_attention(cudaStream_t stream, const E4m3AttentionLaunch& launch);

// `bytes` per page, pages one behind the other from `base`
struct PageArena {
    void* base;
    uint64_t page_bytes;
    uint64_t num_pages;
};
constexpr size_t kMaxPageArenas = 64;   // arenas of one launch: the table travels as a kernel argument
cudaError_t launch_kv_pages_copy(cudaStream_t stream, const PageArena* arenas, size_t num_arenas,
                                 const uint32_t* source_pages, const uint32_t* destination_pages, size_t num_pairs);

}  // namespace lfm25
