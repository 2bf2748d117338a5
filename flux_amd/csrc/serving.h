// Launchers of the serving operators: attention over a paged cache, windowed attention, cache pages, logits.
#pragma once

#include "flux_common.h"

#include <cstddef>
#include <cstdint>

namespace flux {

// Element types of the serving operators (flux_dtype in the C ABI).
enum class Type : int { kFloat32 = 0, kFloat16 = 1, kBFloat16 = 2 };

inline int type_bytes(Type type) { return type == Type::kFloat32 ? 4 : 2; }

constexpr int kServingMaxDim = 256;

// floor(n / divisor) for 0 <= n < 2^31 by one high product: magic = ceil(2^(32 + shift) / divisor) with
// 2^shift >= divisor, so the error n * (magic * divisor - 2^(32 + shift)) / 2^(32 + shift) stays below 1 / divisor.
struct Divider {
    uint32_t divisor;
    uint32_t magic;  // low 32 bits of magic: its bit 32 is always set and is added back below
    uint32_t shift;
};

inline Divider make_divider(uint32_t divisor) {
    uint32_t shift = 0;
    while ((uint64_t{1} << shift) < divisor) ++shift;
    const uint64_t magic = ((uint64_t{1} << 32) * ((uint64_t{1} << shift) - divisor)) / divisor + 1;
    return Divider{divisor, static_cast<uint32_t>(magic), shift};
}

__device__ __forceinline__ uint32_t divide(uint32_t n, const Divider& d) {
    return (__umulhi(n, d.magic) + n) >> d.shift;  // n < 2^31 and the high product is below n: the sum fits
}

// Sixteen bytes past the caches, for what is written in bulk and not read soon: dirty lines that wait for the kernel's end
// are written back all at once then.
typedef uint32_t Quad __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void store_past_caches(void* to, Quad value) {
    __builtin_nontemporal_store(value, static_cast<Quad*>(to));
}

// ---- attention ----

// Keys and values: pages behind a table (pages > 0), or one contiguous run per sequence (pages == 0).
// Strides are in elements; the head dimension's is 1 for key and value.
struct AttentionArgs {
    const void* query;
    const void* key;
    const void* value;
    void* out;               // contiguous [batch, query_heads, queries, dim]
    float* workspace;        // partials of the split over keys
    const int32_t* table;    // [rows, columns], row stride table_stride
    const int64_t* lengths;  // keys of each sequence; null: `keys`
    const int64_t* starts;   // position of each sequence's first query; null: length - queries
    const int64_t* slots;    // row of table and lengths of each sequence; null: its own index
    float scale;
    int batch;
    int query_heads;
    int kv_heads;
    int group;               // query heads per KV head
    Divider group_of;        // divides by group
    int dim;
    int queries;
    int64_t keys;            // positions a sequence can hold
    int64_t slot_count;      // rows of table and lengths
    int window;              // 0: no window
    int sinks;
    int64_t pages;
    Divider page;
    int64_t table_stride;
    int64_t query_strides[4];  // batch, head, row, dim
    int64_t key_strides[3];    // batch (page when paged), head, row
    int64_t value_strides[3];
    bool wide;               // every key and value row starts at 16 bytes and dim fills whole 16-byte quads
    bool query_wide;         // the same of query rows, with a dim stride of 1
    int blocks;              // workgroups over the keys, per KV head and column tile
    int least;               // tiles below which a sequence is not cut
};

int decode_attention_blocks(int batch, int64_t keys, int kv_heads, int group, int window, int sinks);
size_t decode_attention_workspace_floats(const AttentionArgs& args);
hipError_t launch_decode_attention(const AttentionArgs& args, Type type, hipStream_t stream);
hipError_t launch_window_attention(const AttentionArgs& args, Type type, hipStream_t stream);

// ---- cache pages ----

// The K and V pages of one or more layers; strides in elements, the head dimension's is 1.
struct PagePool {
    char* key;
    char* value;
    int64_t layers;
    int64_t pages;
    int64_t heads;
    int64_t page;  // rows
    int64_t dim;
    int64_t key_strides[4];  // layer, page, head, row
    int64_t value_strides[4];
    int element;  // bytes
    // Set by the launchers: the unit that rows are moved in, and divisions by a row's units and by the heads.
    int unit;
    Divider row_units;
    Divider of_heads;
};

// What an operator did with one request (flux_page_status in the C ABI).
enum PageStatus : int32_t { kPageDone = 0, kPageOutOfRange = 1, kPageRepeated = 2, kPageNoRoom = 3, kPageOccupied = 4 };

struct PageBooks {
    int32_t* table;
    int64_t table_stride;
    int64_t slots;
    int64_t columns;
    int64_t* lengths;
    int32_t* refcounts;
    int64_t pages;
    int64_t page;  // rows of a page
};

struct PageWriteArgs {
    const char* key;
    const char* value;
    int64_t key_strides[3];  // request, head, token
    int64_t value_strides[3];
    int64_t requests;
    int64_t tokens;
    const int32_t* table;
    int64_t table_stride;
    int64_t slots;
    int64_t columns;
    const int64_t* slot_list;
    const int64_t* positions;
    const int64_t* counts;  // null: `tokens`
};

// int32 words of scratch memory.
size_t page_reserve_workspace(int64_t requests, int64_t slots, int64_t pages);
size_t page_fork_workspace(int64_t requests, int64_t slots, int64_t pages);
size_t page_compact_workspace(int64_t pages);

hipError_t launch_page_reserve(const PageBooks& books, const int64_t* slots, const int64_t* counts, int64_t requests,
                               int64_t* positions, int32_t* status, int32_t* workspace, hipStream_t stream);
hipError_t launch_page_write(const PagePool& pool, const PageWriteArgs& args, hipStream_t stream);
hipError_t launch_page_copy(const PagePool& pool, const int64_t* source, const int64_t* target, int64_t requests,
                            int32_t* status, hipStream_t stream);
hipError_t launch_page_free(const PageBooks& books, const int64_t* slots, int64_t requests, int32_t* status,
                            hipStream_t stream);
hipError_t launch_page_fork(const PagePool& pool, const PageBooks& books, const int64_t* parents,
                            const int64_t* children, int64_t requests, int32_t* status, int32_t* workspace,
                            hipStream_t stream);
hipError_t launch_page_compact(const PagePool& pool, const PageBooks& books, int32_t* page_map, int64_t* used,
                               int32_t* workspace, hipStream_t stream);

// ---- logits ----
struct LogitsArgs {
    const void* logits;  // [rows, vocab], row stride logits_stride
    void* out;           // contiguous [rows, vocab]
    int64_t* tokens;     // [rows]
    int64_t rows;
    int64_t vocab;
    int64_t logits_stride;
    const int64_t* history;  // [rows, history_width] or null
    int64_t history_width;
    int64_t history_stride;
    const int64_t* history_lengths;  // null: history_width
    const float* repetition;         // [rows] or null
    const float* frequency;
    const float* presence;
    const float* bias;  // row stride bias_stride (0: one row for all) or null
    int64_t bias_stride;
    const int32_t* allowed;  // bits, row stride allowed_stride (0: one row for all) or null
    int64_t allowed_stride;
    void* workspace;
};

size_t logits_workspace_bytes(int64_t rows, int64_t vocab);
hipError_t launch_logits_process(const LogitsArgs& args, Type type, hipStream_t stream);

}  // namespace flux
