// Parameter blocks and launchers of a speculative step's kernels: trees of drafted tokens, accepted paths, moved
// tokens and controls on logits (speculate.hip), attention of the trees' tokens (tree_attention.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "paged.h"

namespace plamo {

// Nodes of a request's tree, as its bits of ancestors hold them.
constexpr int TREE_MAX_WORDS = 32;

// Positions and ancestors of the trees' nodes (plamo_kernel_paged_tree).
struct TreeParams {
    const int32_t* lengths;   // [rows] with the new tokens
    const int32_t* offsets;   // [rows + 1]
    int rows;
    const int32_t* parents;   // [tokens] index in the request
    int tokens;
    int window;               // 0: all ancestors
    int32_t* positions;       // [tokens]
    uint32_t* ancestors;      // [tokens][words]
    int words;
    Divider by_words;
};
void launch_paged_tree(const TreeParams& p, hipStream_t s);

// Paths that the drawn tokens agree with (plamo_kernel_paged_accept).
struct AcceptParams {
    const int32_t *lengths, *offsets;
    int rows;
    const int32_t *parents, *tokens, *drawn;  // [capacity]
    int capacity;
    const int32_t* given;     // [rows]; null: 1
    const int32_t* tables;    // [rows][width]
    int width, page_size;
    int32_t* free_pages;      // [pages]
    const int32_t* free_count;
    int pages;
    int32_t *lengths_out, *free_out;
    int32_t* accepted;        // [rows][nodes + 1]
    int32_t *accepted_counts, *last;  // [rows]
    int nodes;
    int32_t *from, *to;       // [rows][nodes]
    int32_t* status;
    Divider div;              // by page_size
};
void launch_paged_accept(const AcceptParams& p, hipStream_t s);

// Tokens' keys and values from slot to slot, in all layers (plamo_kernel_paged_move).
constexpr int MOVE_LAYERS = 64;  // of a launch
struct MoveParams {
    uint64_t keys[MOVE_LAYERS], values[MOVE_LAYERS];
    int layers;
    int64_t page_stride, slot_stride, head_stride;  // bytes
    int pages, page_size;
    Divider div;
    int kv_heads, chunks;     // 16-byte chunks of a head
    const int32_t *from, *to; // [groups][group]
    int groups, group;
};
void launch_paged_move(const MoveParams& p, hipStream_t s);

// Penalties, biases and masks on logits (plamo_kernel_logit_controls).
constexpr int CONTROL_MAX_HISTORY = 1 << 17, CONTROL_MAX_BIAS = 4096, CONTROL_MAX_NGRAM = 64;
struct ControlParams {
    const int32_t *history, *history_lengths;
    int64_t history_stride;
    int sequences, history_width;
    const int32_t *offsets, *tokens;  // null: row r is sequence r
    const uint32_t* ancestors;
    int words;
    const float *repetition, *presence, *frequency;  // [sequences] or null
    const int32_t* ngram;
    const int32_t* bias_ids;  // [sequences][bias_width] or null
    const float* bias;
    int bias_width;
    const uint32_t* masks;    // [mask_count][mask_stride] or null
    const int32_t* mask_rows; // [rows]; null: row r has mask r
    int64_t mask_stride;
    int mask_count;
    const char* logits;
    int64_t stride;           // elements
    int n, rows;
    char* out;
    int64_t out_stride;
    bool in_place;
};
bool controls_launches(int n, int rows);  // a launch's threads are a 32-bit number
void launch_logit_controls(const ControlParams& p, int type, int out_type, hipStream_t s);

// Attention of several new tokens a request over its pages (plamo_kernel_attention_paged_tree).
struct TreeAttnParams {
    const char *keys, *values;
    int64_t page_stride, slot_stride, head_stride;  // bytes
    int pages, page_size;
    Divider div;
    int kv_heads, group;      // query heads per KV head
    Divider by_group;         // by group
    const uint16_t* q;
    int64_t q_stride;         // elements
    const int32_t* tables;
    int width;
    const int32_t *lengths, *offsets;
    int rows, tokens;
    int32_t most;             // keys that a table row holds
    const int32_t* positions; // [tokens], with ancestors
    const uint32_t* ancestors;  // [tokens][words]; null: each token sees those before it
    int words;
    int window;               // 0: all keys
    float scale;              // times log2(e): scores are exponents of two
    uint16_t* out;
    int64_t out_stride;
    float* lse;               // [tokens][heads] or null
    int share;                // waves that share a tile's keys: a tile is 32 rows of queries for each
    int target;               // parts that all tiles' keys are divided into
    int least;                // fewest keys of a part, but for a tile's last
    int run;                  // neighbouring parts that are put on one XCD
    int items;                // parts that a launch takes, for each KV head: all of requests that do not overlap
    bool joins;               // whether a tile can have several parts
    bool listed;              // rows' divisions are found by a launch before
    int* joined;              // [1] tiles of several parts
    int4* row_work;           // [rows] first item, first slot, first joined tile, parts
    int4* tile_work;          // [target][2] of the tiles of several parts
    float2* part_ml;          // [slots][kv_heads][32 share] maximum and sum
    float* part_o;            // [slots][kv_heads][share][head_dim / 8][64][4]
};
int64_t tree_attn_workspace(int rows, int tokens, int heads, int kv_heads, int head_dim);
void tree_attn_bind(TreeAttnParams& p, void* workspace, int head_dim);
void launch_tree_attention(const TreeAttnParams& p, int type, int head_dim, hipStream_t s);

}  // namespace plamo
