// Runs of several new tokens per sequence over paged caches: shapes shared by admission
// (draft_ops.cpp) and the kernels (draft.hip, run_attention.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "paged.hpp"

namespace mfh {

// A batch's runs: sequence s has tokens starts[s] .. starts[s + 1] - 1 behind its
// lengths[s] cached ones.
struct Runs {
    const float *starts = nullptr;   // [sequences + 1], null: a token each
    const float *lengths = nullptr;  // [sequences]
    uint32_t sequences = 0, tokens = 0;
};

// A run's tokens and the tokens before them; `end` below `begin`: none.
struct RunBounds {
    uint32_t begin = 0, end = 0;
};

// Whether entries i and i + 1 of the list of starts are whole numbers, in order, up to
// the batch's end.
__device__ __forceinline__ bool valid_bounds(const Runs &r, uint32_t i, RunBounds &out)
{
    const float a = r.starts[i], b = r.starts[i + 1];
    // NaN fails every comparison; the batch has at most 2^24 tokens.
    const bool ok = a >= 0.0f && a <= b && b <= float(r.tokens) && truncf(a) == a &&
                    truncf(b) == b;
    out.begin = ok ? uint32_t(a) : 0;
    out.end = ok ? uint32_t(b) : 0;
    return ok;
}

// The run of sequence s, for every lane of a wave; empty where the list of starts has
// ended before it.
__device__ __forceinline__ RunBounds run_of(const Runs &r, uint32_t s)
{
    RunBounds mine;
    if (!r.starts) {
        mine.begin = s;
        mine.end = s + 1;
        return mine;
    }
    bool ok = valid_bounds(r, s, mine);
    RunBounds other;
    for (uint32_t i = threadIdx.x & 63; i < s; i += 64)
        ok = valid_bounds(r, i, other) && ok;
    if (!__all(ok))
        mine.end = mine.begin = 0;
    return mine;
}

// A length, where it is a whole number that leaves the run's places below `limit`.
__device__ __forceinline__ bool valid_length(float length, uint32_t run, uint32_t limit)
{
    return length >= 0.0f && length < 16777216.0f && truncf(length) == length &&
           uint32_t(length) + run <= limit;
}

struct DraftLayout {
    Runs runs;
    const float *parents = nullptr;  // [tokens], may be null
    float *sequences = nullptr, *positions = nullptr, *places = nullptr;  // [tokens]
    uint8_t *mask = nullptr;         // [tokens, mask_bytes], may be null
    uint32_t mask_bytes = 0;
};
void launch_draft_layout(hipStream_t stream, const DraftLayout &p);

// One launch of settling: up to kSettleBuffers page buffers.
constexpr uint32_t kSettleBuffers = 64, kSettleColumns = 1024;
struct Settle {
    Runs runs;
    const float *parents = nullptr, *places = nullptr;   // [tokens], may be null
    const float *drafted = nullptr, *choices = nullptr;  // [tokens]
    const float *tables = nullptr;   // [sequences, max_pages]
    float *emitted = nullptr;        // [sequences, columns], null past the first launch
    float *counts = nullptr, *next = nullptr;  // [sequences]
    uint32_t max_pages = 0, pages = 0, page_shift = 0, columns = 0, buffers = 0;
    bool path_pages = false;         // the path's rows need pages: there are buffers
    void *buffer[kSettleBuffers];
    uint32_t heads[kSettleBuffers], row_bytes[kSettleBuffers];
};
void launch_settle(hipStream_t stream, const Settle &p);

struct LatentAppend {
    float *query_out = nullptr;
    void *pages = nullptr;
    const float *query = nullptr, *latent = nullptr, *key = nullptr;
    const float *weight = nullptr;     // null: no norm
    const float *rotation = nullptr;   // [rotation_rows, rope]
    const float *tables = nullptr;     // [sequences, max_pages]
    const float *sequences = nullptr;  // [tokens], null: token t is sequence t
    const float *positions = nullptr, *places = nullptr;  // [tokens]; places may be null
    PageShape shape;                   // one head of rank + rope columns
    uint32_t tokens = 0, rotation_rows = 0, sequence_count = 0, max_pages = 0;
    uint32_t query_heads = 0, rank = 0, rope = 0;
    bool interleaved = false;
    float epsilon = 0.0f;
};
void launch_latent_append(hipStream_t stream, const LatentAppend &p);

// Attention of runs.  Keys are `shape.head_dim` wide, values their first `value_dim`
// columns in the value pages (the key pages themselves for latents).  A query's
// first `value_dim` columns are in `query`, for latents the rest in `rotary_query`.
struct RunAttention {
    float *out = nullptr;  // [tokens, query_heads * value_dim]
    const float *query = nullptr, *rotary_query = nullptr;
    const void *key_pages = nullptr, *value_pages = nullptr;
    const float *tables = nullptr;   // [sequences, max_pages]
    const uint8_t *mask = nullptr;   // [tokens, mask_bytes]; null: all up to the token
    Runs runs;
    PageShape shape;
    uint32_t value_dim = 0, max_pages = 0, query_heads = 0, group = 0, mask_bytes = 0;
    uint32_t longest = 0;  // places of a table row, below 2^24
    float scale = 0.0f;    // times log2 e
    // Filled by run_attention_plan: blocks of the matrix-core kernel (0: the one of any
    // width) and of the join, query rows of an item, units besides its tiles; its workspace
    // of run_attention_scratch_bytes.
    uint32_t blocks = 0, rows = 0, joins = 0, item_units = 0;
    float *records = nullptr;
};
// Chooses the kernel and its split; false where the extents pass the index range.
bool run_attention_plan(RunAttention &p, int cu_count);
size_t run_attention_scratch_bytes(const RunAttention &p);
void launch_run_attention(hipStream_t stream, const RunAttention &p);

}  // namespace mfh
