// Launchers of the attention over the quantised cache (attention.hip).
#pragma once

#include <type_traits>

#include "cache.h"

namespace nuq {

struct AttentionArgs {
    const void *q;
    void *out;
    uint64_t q_stride, out_stride;  // elements from a query row to the next
    const int32_t *table;           // [batch][table_stride] page numbers
    const int32_t *lengths;         // [batch] tokens held, the new ones among them
    const int32_t *starts;          // [batch + 1] first query row of each sequence; null: max_tokens each
    uint64_t table_stride;
    uint32_t rows;        // query rows in all
    uint32_t batch, max_tokens, group;
    uint32_t capacity;    // tokens a row of the table can name
    uint32_t window;      // 0: none
    float scale;          // of the scores, log2(e) among it
    // the plan
    uint32_t prompt;      // the prompt kernel's call
    uint32_t above, upto; // only of sequences of more than `above` and up to `upto` new tokens
    uint32_t row_tiles, blocks, splits;  // blocks: of the rows of a sequence
    uint64_t units;       // blocks of all sequences
    uint64_t floats;      // of workspace
    float *partial_o, *partial_ml;
};

// The prompt kernel (attention_prompt.hip): row tiles of a wave, tokens of a step.
constexpr int prompt_row_tiles(int head_dim, bool f32) {
    return head_dim == 64 ? (f32 ? 3 : 4) : head_dim == 128 ? (f32 ? 2 : 3) : f32 ? 1 : 2;
}
constexpr int prompt_tokens(int head_dim) { return head_dim == 256 ? 32 : 64; }
hipError_t launch_attention_prompt(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t d, uint32_t f32,
                                   const AttentionArgs &a);

// The most workgroups of a launch, 256 threads each (2^32 threads in all).
constexpr uint64_t MOST_GROUPS = 0x00ffffffull;

// Fills in the plan of a call: row tiles of 16, blocks of them, splits of the
// long axis with at most `max_floats` of workspace, for `cus` compute units. Returns whether sequences of few new
// tokens are a plan of their own, `few`, beside those of many in `a`.
bool plan_attention(uint32_t head_dim, uint32_t kv_heads, uint32_t f32, uint64_t max_length, uint32_t heads,
                    uint64_t max_floats, uint32_t cus, AttentionArgs *a, AttentionArgs *few);
hipError_t launch_attention(hipStream_t s, const CacheView &c, uint32_t bits, uint32_t head_dim, uint32_t f32,
                            uint32_t heads, AttentionArgs a, float *work);

}  // namespace nuq
