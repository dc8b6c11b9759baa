// Entry points of the 8-bit paged key/value cache and of the page copies: host-side checks, then the launch.  Nothing is
// launched on error.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <limits>

#include "../../include/lfm25_b200.h"
#include "e4m3_cache.h"
#include "kernels.h"

namespace {

int32_t fail(int32_t code, const char* format, ...) {
    char message[256];
    va_list arguments;
    va_start(arguments, format);
    vsnprintf(message, sizeof message, format, arguments);
    va_end(arguments);
    return lfm25::report_error(code, message);
}

#define E4M3_ENSURE(condition, code, ...)    \
    do {                                     \
        if (!(condition)) {                  \
            return fail(code, __VA_ARGS__);  \
        }                                    \
    } while (0)

bool checked_mul(size_t a, size_t b, size_t* out) {
    if (a != 0 && b > std::numeric_limits<size_t>::max() / a) {
        return false;
    }
    *out = a * b;
    return true;
}

bool aligned(const void* pointer, size_t bytes) { return reinterpret_cast<uintptr_t>(pointer) % bytes == 0; }

int32_t cuda_result(cudaError_t status, const char* what) {
    return status == cudaSuccess ? LFM25_OK : fail(LFM25_ERR_CUDA, "%s: %s", what, cudaGetErrorString(status));
}

// Rows of heads * head_dim elements, `stride` elements apart: 16-byte loads, and the span they cover.
int32_t check_rows(const char* name, const lfm25_slice& rows, size_t count, size_t width, size_t stride) {
    size_t span = 0;
    E4M3_ENSURE(stride >= width && stride % 8 == 0, LFM25_ERR_INVALID_ARGUMENT,
                "8-bit cache: %s token stride %zu is no multiple of 8 of at least %zu elements", name, stride, width);
    E4M3_ENSURE(checked_mul(count - 1, stride, &span) && span + width >= span, LFM25_ERR_OVERFLOW, "8-bit cache: %s size overflow", name);
    E4M3_ENSURE(rows.len >= span + width, LFM25_ERR_BUFFER_TOO_SMALL, "8-bit cache: %s too small: required=%zu, actual=%zu", name,
                span + width, rows.len);
    E4M3_ENSURE(rows.ptr != nullptr, LFM25_ERR_NULL_POINTER, "8-bit cache: %s is null", name);
    E4M3_ENSURE(aligned(rows.ptr, 16), LFM25_ERR_INVALID_ARGUMENT, "8-bit cache: %s must be 16-byte aligned", name);
    return LFM25_OK;
}

int32_t check_vector(const char* name, const lfm25_slice& vector, size_t count, size_t alignment) {
    E4M3_ENSURE(vector.len >= count, LFM25_ERR_BUFFER_TOO_SMALL, "8-bit cache: %s too small: required=%zu, actual=%zu", name, count,
                vector.len);
    E4M3_ENSURE(vector.ptr != nullptr, LFM25_ERR_NULL_POINTER, "8-bit cache: %s is null", name);
    E4M3_ENSURE(aligned(vector.ptr, alignment), LFM25_ERR_INVALID_ARGUMENT, "8-bit cache: %s is not aligned to %zu bytes", name, alignment);
    return LFM25_OK;
}

#define E4M3_CHECK(call)                  \
    do {                                  \
        const int32_t status_ = (call);   \
        if (status_ != LFM25_OK) {        \
            return status_;               \
        }                                 \
    } while (0)

int32_t take_cache(const lfm25_e4m3_cache& cache, lfm25::E4m3Cache* out) {
    E4M3_ENSURE(cache.page_size == 16 || cache.page_size == 32, LFM25_ERR_INVALID_ARGUMENT, "unsupported KV page size %zu",
                cache.page_size);
    E4M3_ENSURE(cache.page_size == 16, LFM25_ERR_UNSUPPORTED, "page size 32 is not built; use 16");
    E4M3_ENSURE(cache.head_dim == 64 || cache.head_dim == 128, LFM25_ERR_UNSUPPORTED,
                "8-bit cache: heads of %zu are not built; use 64 or 128", cache.head_dim);
    E4M3_ENSURE(cache.num_pages > 0, LFM25_ERR_INVALID_ARGUMENT, "8-bit cache requires pages");
    E4M3_ENSURE(cache.num_pages <= 0xffffffffull, LFM25_ERR_INVALID_ARGUMENT, "8-bit cache pages exceed u32");
    E4M3_ENSURE(cache.kv_heads > 0 && cache.kv_heads <= 1024, LFM25_ERR_INVALID_ARGUMENT, "8-bit cache: %zu KV heads (1..=1024)",
                cache.kv_heads);
    size_t tiles = 0;
    size_t elements = 0;
    E4M3_ENSURE(checked_mul(cache.num_pages, cache.kv_heads, &tiles) && checked_mul(tiles, 16 * cache.head_dim, &elements),
                LFM25_ERR_OVERFLOW, "8-bit cache size overflow");
    E4M3_CHECK(check_vector("key codes", cache.key_codes, elements, 16));
    E4M3_CHECK(check_vector("value codes", cache.value_codes, elements, 16));
    E4M3_CHECK(check_vector("key scales", cache.key_scales, tiles, 4));
    E4M3_CHECK(check_vector("value scales", cache.value_scales, tiles, 4));
    out->key_codes = static_cast<uint8_t*>(cache.key_codes.ptr);
    out->value_codes = static_cast<uint8_t*>(cache.value_codes.ptr);
    out->key_scales = static_cast<float*>(cache.key_scales.ptr);
    out->value_scales = static_cast<float*>(cache.value_scales.ptr);
    out->num_pages = static_cast<uint32_t>(cache.num_pages);
    out->kv_heads = static_cast<uint32_t>(cache.kv_heads);
    out->head_dim = static_cast<uint32_t>(cache.head_dim);
    return LFM25_OK;
}

int32_t take_append(const lfm25_e4m3_cache& cache, const lfm25_slice& key, const lfm25_slice& value, const lfm25_slice& slot_mapping,
                    size_t num_tokens, size_t kv_token_stride, lfm25::E4m3WriteLaunch* out) {
    E4M3_ENSURE(num_tokens > 0, LFM25_ERR_INVALID_ARGUMENT, "8-bit cache write requires tokens");
    E4M3_ENSURE(num_tokens <= 0x7fffffffu, LFM25_ERR_INVALID_ARGUMENT, "8-bit cache write grid size exceeds u32");
    E4M3_CHECK(take_cache(cache, &out->cache));
    const size_t width = cache.kv_heads * cache.head_dim;
    out->kv_token_stride = kv_token_stride != 0 ? kv_token_stride : width;
    E4M3_CHECK(check_rows("keys", key, num_tokens, width, out->kv_token_stride));
    E4M3_CHECK(check_rows("values", value, num_tokens, width, out->kv_token_stride));
    E4M3_CHECK(check_vector("slot mapping", slot_mapping, num_tokens, 8));
    out->key = key.ptr;
    out->value = value.ptr;
    out->slot_mapping = static_cast<const int64_t*>(slot_mapping.ptr);
    out->num_tokens = num_tokens;
    return LFM25_OK;
}

int32_t take_attention(const lfm25_paged_attention_e4m3_launch& l, lfm25::E4m3AttentionLaunch* out) {
    E4M3_ENSURE(l.num_tokens > 0, LFM25_ERR_INVALID_ARGUMENT, "8-bit cache attention requires tokens");
    E4M3_ENSURE(l.num_tokens <= (1u << 24), LFM25_ERR_INVALID_ARGUMENT, "attention grid size exceeds u32");
    E4M3_CHECK(take_cache(l.cache, &out->cache));
    E4M3_ENSURE(l.query_heads > 0 && l.query_heads % l.cache.kv_heads == 0 && l.query_heads <= 4096, LFM25_ERR_INVALID_ARGUMENT,
                "8-bit cache attention: %zu query heads are no multiple of %zu KV heads (at most 4096)", l.query_heads, l.cache.kv_heads);
    E4M3_ENSURE(std::isfinite(l.scale) && l.scale > 0.0f, LFM25_ERR_INVALID_ARGUMENT, "attention scale must be finite and positive");
    E4M3_ENSURE(l.block_table_stride > 0, LFM25_ERR_INVALID_ARGUMENT, "block table stride must be positive");
    E4M3_ENSURE(l.block_table_stride <= 0x0fffffffu, LFM25_ERR_INVALID_ARGUMENT, "block table positions exceed u32");
    E4M3_ENSURE(l.block_tables.len % l.block_table_stride == 0, LFM25_ERR_INVALID_ARGUMENT, "block tables not row aligned");
    E4M3_CHECK(check_vector("block tables", l.block_tables, l.block_table_stride, 4));
    E4M3_CHECK(check_vector("request slots", l.request_slots, l.num_tokens, 4));
    E4M3_CHECK(check_vector("positions", l.position_ids, l.num_tokens, 4));
    const size_t width = l.query_heads * l.cache.head_dim;
    out->query_token_stride = l.query_token_stride != 0 ? l.query_token_stride : width;
    E4M3_CHECK(check_rows("query", l.query, l.num_tokens, width, out->query_token_stride));
    E4M3_CHECK(check_rows("output", l.output, l.num_tokens, width, width));
    out->query = l.query.ptr;
    out->output = l.output.ptr;
    out->block_tables = static_cast<const uint32_t*>(l.block_tables.ptr);
    out->request_slots = static_cast<const uint32_t*>(l.request_slots.ptr);
    out->position_ids = static_cast<const uint32_t*>(l.position_ids.ptr);
    out->num_tokens = l.num_tokens;
    out->query_heads = l.query_heads;
    out->block_table_stride = l.block_table_stride;
    out->block_table_rows = l.block_tables.len / l.block_table_stride;
    const size_t most = l.block_table_stride * 16;
    out->maximum_context_tokens = l.maximum_context_tokens == 0 || l.maximum_context_tokens > most ? most : l.maximum_context_tokens;
    out->window = static_cast<uint32_t>(l.window < 0xffffffffull ? l.window : 0xffffffffull);
    out->sinks = static_cast<uint32_t>(l.sinks < 0x7fffffffull ? l.sinks : 0x7fffffffull);
    out->scale = l.scale;
    return LFM25_OK;
}

}  // namespace

extern "C" {

int32_t lfm25_kv_cache_write_e4m3(void* stream, const lfm25_kv_cache_write_e4m3_launch* launch) {
    E4M3_ENSURE(launch != nullptr, LFM25_ERR_NULL_POINTER, "8-bit cache write launch is null");
    lfm25::E4m3WriteLaunch args = {};
    E4M3_CHECK(take_append(launch->cache, launch->key, launch->value, launch->slot_mapping, launch->num_tokens, launch->kv_token_stride, &args));
    return cuda_result(lfm25::launch_e4m3_cache_write(static_cast<cudaStream_t>(stream), args), "8-bit cache write launch failed");
}

int32_t lfm25_qk_norm_rope_kv_write_e4m3(void* stream, const lfm25_qk_norm_rope_kv_write_e4m3_launch* launch) {
    E4M3_ENSURE(launch != nullptr, LFM25_ERR_NULL_POINTER, "8-bit cache write launch is null");
    const lfm25_qk_norm_rope_kv_write_e4m3_launch& l = *launch;
    lfm25::E4m3WriteLaunch args = {};
    E4M3_CHECK(take_append(l.cache, l.key, l.value, l.slot_mapping, l.num_tokens, l.kv_token_stride, &args));
    E4M3_ENSURE(l.query_heads > 0 && l.query_heads <= 4096, LFM25_ERR_INVALID_ARGUMENT, "8-bit cache write: %zu query heads (1..=4096)", l.query_heads);
    E4M3_ENSURE(std::isfinite(l.eps) && l.eps >= 0.0f, LFM25_ERR_INVALID_ARGUMENT, "norm epsilon must be finite and not negative");
    const size_t width = l.query_heads * l.cache.head_dim;
    args.query_token_stride = l.query_token_stride != 0 ? l.query_token_stride : width;
    E4M3_CHECK(check_rows("query", l.query, l.num_tokens, width, args.query_token_stride));
    E4M3_CHECK(check_rows("query output", l.query_out, l.num_tokens, width, width));
    E4M3_ENSURE(l.query_out.ptr != l.query.ptr || args.query_token_stride == width, LFM25_ERR_INVALID_ARGUMENT,
                "8-bit cache write: queries rewritten in place must be dense");
    E4M3_CHECK(check_vector("query norm", l.query_norm, l.cache.head_dim, 16));
    E4M3_CHECK(check_vector("key norm", l.key_norm, l.cache.head_dim, 16));
    E4M3_CHECK(check_vector("rotation frequencies", l.inv_freq, l.cache.head_dim / 2, 4));
    E4M3_CHECK(check_vector("positions", l.position_ids, l.num_tokens, 4));
    args.query = l.query.ptr;
    args.query_out = l.query_out.ptr;
    args.query_norm = l.query_norm.ptr;
    args.key_norm = l.key_norm.ptr;
    args.inv_freq = static_cast<const float*>(l.inv_freq.ptr);
    args.position_ids = static_cast<const uint32_t*>(l.position_ids.ptr);
    args.query_heads = static_cast<uint32_t>(l.query_heads);
    args.eps = l.eps;
    return cuda_result(lfm25::launch_e4m3_cache_write(static_cast<cudaStream_t>(stream), args), "8-bit cache write launch failed");
}

int32_t lfm25_paged_attention_e4m3(void* stream, const lfm25_paged_attention_e4m3_launch* launch) {
    E4M3_ENSURE(launch != nullptr, LFM25_ERR_NULL_POINTER, "8-bit cache attention launch is null");
    lfm25::E4m3AttentionLaunch args = {};
    E4M3_CHECK(take_attention(*launch, &args));
    if (launch->token_order.ptr != nullptr) {
        E4M3_CHECK(check_vector("token order", launch->token_order, launch->num_tokens, 4));
        args.token_order = static_cast<const uint32_t*>(launch->token_order.ptr);
    }
    return cuda_result(lfm25::launch_e4m3_attention(static_cast<cudaStream_t>(stream), args), "8-bit cache attention launch failed");
}

int32_t lfm25_paged_attention_e4m3_plan(const lfm25_paged_attention_e4m3_launch* launch, int32_t clusters_of_16, uint32_t* warps,
                                        uint32_t* splits) {
    E4M3_ENSURE(launch != nullptr && warps != nullptr && splits != nullptr, LFM25_ERR_NULL_POINTER, "8-bit cache attention plan received a null pointer");
    lfm25::E4m3AttentionLaunch args = {};
    E4M3_CHECK(take_attention(*launch, &args));
    const lfm25::E4m3DecodePlan plan = lfm25::plan_e4m3_attention(args, clusters_of_16 != 0);
    *warps = plan.warps;
    *splits = 1u << plan.splits_log2;
    return LFM25_OK;
}

int32_t lfm25_paged_prompt_attention_e4m3(void* stream, const lfm25_paged_attention_e4m3_launch* launch) {
    E4M3_ENSURE(launch != nullptr, LFM25_ERR_NULL_POINTER, "8-bit cache attention launch is null");
    lfm25::E4m3AttentionLaunch args = {};
    E4M3_CHECK(take_attention(*launch, &args));
    E4M3_ENSURE(launch->num_segments > 0, LFM25_ERR_INVALID_ARGUMENT, "8-bit cache prompt attention requires segments");
    E4M3_ENSURE(launch->num_segments <= (1u << 24), LFM25_ERR_INVALID_ARGUMENT, "attention grid size exceeds u32");
    E4M3_CHECK(check_vector("segment offsets", launch->segment_offsets, launch->num_segments + 1, 4));
    args.segment_offsets = static_cast<const uint32_t*>(launch->segment_offsets.ptr);
    args.num_segments = launch->num_segments;
    args.status = lfm25::device_status_words();
    E4M3_ENSURE(args.status != nullptr, LFM25_ERR_CUDA, "device status words are not reachable");
    return cuda_result(lfm25::launch_e4m3_prompt_attention(static_cast<cudaStream_t>(stream), args), "8-bit cache attention launch failed");
}

int32_t lfm25_kv_pages_copy(void* stream, const lfm25_page_arena* arenas, size_t num_arenas, lfm25_slice source_pages,
                            lfm25_slice destination_pages, size_t num_pairs) {
    E4M3_ENSURE(arenas != nullptr, LFM25_ERR_NULL_POINTER, "page copy arenas are null");
    E4M3_ENSURE(num_arenas > 0 && num_arenas <= 65536, LFM25_ERR_INVALID_ARGUMENT, "page copy takes 1..=65536 arenas, got %zu", num_arenas);
    E4M3_ENSURE(num_pairs > 0, LFM25_ERR_INVALID_ARGUMENT, "page copy requires pages");
    E4M3_ENSURE(num_pairs <= 0x7fffffffu, LFM25_ERR_INVALID_ARGUMENT, "page copy grid size exceeds u32");
    for (size_t index = 0; index < num_arenas; ++index) {
        const lfm25_page_arena& arena = arenas[index];
        E4M3_ENSURE(arena.base != nullptr, LFM25_ERR_NULL_POINTER, "page copy arena %zu is null", index);
        E4M3_ENSURE(arena.num_pages > 0, LFM25_ERR_INVALID_ARGUMENT, "page copy arena %zu has no pages", index);
        E4M3_ENSURE(arena.page_bytes <= 0x7fffffffu, LFM25_ERR_INVALID_ARGUMENT, "page copy arena %zu: page size exceeds i32", index);
        E4M3_ENSURE(arena.page_bytes > 0 && arena.page_bytes % 4 == 0 && aligned(arena.base, 4), LFM25_ERR_INVALID_ARGUMENT,
                    "page copy arena %zu: pages of %zu bytes must be multiples of 4, 4-byte aligned", index, arena.page_bytes);
        size_t bytes = 0;
        E4M3_ENSURE(checked_mul(arena.page_bytes, arena.num_pages, &bytes), LFM25_ERR_OVERFLOW, "page copy arena %zu overflows", index);
    }
    E4M3_CHECK(check_vector("source pages", source_pages, num_pairs, 4));
    E4M3_CHECK(check_vector("destination pages", destination_pages, num_pairs, 4));
    static_assert(sizeof(lfm25_page_arena) == sizeof(lfm25::PageArena), "the C struct is the kernel's");
    return cuda_result(lfm25::launch_kv_pages_copy(static_cast<cudaStream_t>(stream), reinterpret_cast<const lfm25::PageArena*>(arenas),
                                                   num_arenas, static_cast<const uint32_t*>(source_pages.ptr),
                                                   static_cast<const uint32_t*>(destination_pages.ptr), num_pairs),
                       "page copy launch failed");
}

}  // extern "C"
