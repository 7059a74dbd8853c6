// Parameter blocks and launchers of the paged-cache kernels (paged.hip) and of the sampler
// (sample.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace plamo {

enum ValueType { TYPE_BF16 = 0, TYPE_F16 = 1, TYPE_F32 = 2 };

// x / d for 0 <= x < 2^31 as one 64-bit product and a shift: with l = ceil(log2 d) the factor
// floor(2^(31 + l) / d) + 1 exceeds 2^(31 + l) / d by at most 1, so the product is off by less than
// x / 2^(31 + l) < 1 / d and the floor is exact.
struct Divider {
    uint32_t mul, shift;
};
inline Divider divider(uint32_t d) {
    uint32_t l = 0;
    while ((uint64_t(1) << l) < d) ++l;
    return {uint32_t((uint64_t(1) << (31 + l)) / d + 1), 31 + l};
}

// Block tables, slot map and positions of a step (plamo_kernel_paged_tables).
struct PagedTablesParams {
    const int32_t* lengths;     // [rows]
    const int32_t* counts;      // [rows]
    int rows;
    int32_t* tables;            // [rows][width]
    int width, page_size;
    int32_t* free_pages;        // [pages]
    const int32_t* free_count;  // [1]
    int pages;
    int32_t* lengths_out;       // [rows]
    int32_t* free_out;          // [1]
    int32_t* offsets;           // [rows + 1]
    int32_t* slots;             // [capacity]
    int32_t* positions;         // [capacity]
    int capacity;
    int32_t* status;            // [1]
    Divider div;                // by page_size
};
void launch_paged_tables(const PagedTablesParams& p, hipStream_t s);

// A projection's rows normalised, rotated and written to their slots (plamo_kernel_paged_qkv).
struct PagedQkvParams {
    const void* qkv;
    int64_t stride;           // elements between rows
    int heads, kv_heads;
    const uint16_t* q_norm;   // [head_dim] of the cache's type; null: no normalisation
    const uint16_t* k_norm;
    const uint32_t* rope;     // [rope_rows][head_dim / 2] BF16 cos | sin << 16; null: no rotation
    int rope_rows;
    const int32_t* positions;
    const int32_t* slots;
    int tokens;
    uint16_t* q;
    int64_t q_stride;
    uint16_t *keys, *values;
    int64_t page_stride, slot_stride, head_stride;  // elements
    int pages, page_size;
    Divider div;
};
void launch_paged_qkv(const PagedQkvParams& p, int source, int type, int head_dim, hipStream_t s);

// Attention of one token per row over its pages (plamo_kernel_attention_paged).
struct PagedAttnParams {
    const char *keys, *values;
    int64_t page_stride, slot_stride, head_stride;  // bytes
    int pages, page_size;
    Divider div;
    int kv_heads, group;      // query heads per KV head
    int tiles;                // blocks of 16 query heads per KV head
    const uint16_t* q;
    int64_t q_stride;         // elements
    const int32_t* tables;
    int width;
    const int32_t* lengths;
    int rows;
    int32_t most;             // keys that a table row holds
    int window;               // 0: all keys
    float scale;              // times log2(e): scores are exponents of two
    uint16_t* out;
    int64_t out_stride;
    float* lse;               // [rows][heads] or null
    int target;               // parts that all rows' keys are divided into, for one KV head's tile
    int reach;                // most keys of a row's parts: those it can see, from a multiple of 16 on
    int least;                // fewest keys of a part, but for a row's last
    int division;             // how a workgroup finds its part
    int2* row_parts;          // [rows] first part and number of parts
    float2* part_ml;          // [parts][heads] maximum and sum
    float* part_o;            // [parts][heads][head_dim]
};
// Workspace bytes, and the pointers of a workspace.
size_t paged_attn_workspace(int rows, int heads, int kv_heads, int head_dim);
void paged_attn_bind(PagedAttnParams& p, void* workspace, int head_dim);
bool paged_attn_launches(const PagedAttnParams& p);  // a launch's threads along a direction are a 32-bit number
void launch_paged_attention(const PagedAttnParams& p, int type, int head_dim, hipStream_t s);

// Tokens drawn from logits (plamo_kernel_sample).
struct SampleParams {
    const void* logits;
    int64_t stride;           // elements between rows
    int n, rows;
    const float* temperature;  // [rows]; null: 1
    const int32_t* top_k;      // [rows]; null: off
    const float* top_p;        // [rows]; null: off
    const float* min_p;        // [rows]; null: off
    const float* uniform;      // [rows]
    int32_t* token;            // [rows]
    float* prob;               // [rows] or null
    void* workspace;
};
constexpr int SAMPLE_MAX_VOCAB = 1 << 20;
size_t sample_workspace(int rows, int n);
void launch_sample(const SampleParams& p, int type, hipStream_t s);

}  // namespace plamo
