// Paged key/value caches: shapes shared by admission (paged_ops.cpp) and the
// kernels (paged.hip, paged_gqa.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "internal.hpp"

namespace mfh {

// A page buffer is [pages, kv_heads, page_size, head_dim], head-major inside a
// page so that one head's keys of a page are one contiguous run; f32 or
// binary16 elements.
struct PageShape {
    uint32_t pages = 0, kv_heads = 0, page_shift = 0, head_dim = 0;
    bool half = false;
    __host__ __device__ uint32_t page_size() const { return 1u << page_shift; }
    // Elements of one page.
    __host__ __device__ uint64_t stride() const
    {
        return (uint64_t(kv_heads) * head_dim) << page_shift;
    }
};

// Whole numbers travel as exact f32 values, as token ids do; what is not one
// below `limit` (limit <= 2^24) is invalid.
__device__ __forceinline__ bool valid_index(float v, uint32_t limit)
{
    // NaN fails every comparison.
    return v >= 0.0f && v < 16777216.0f && truncf(v) == v && uint32_t(v) < limit;
}

// The nearest binary16 value; finite values past its range become its largest.
__device__ __forceinline__ _Float16 to_half(float v)
{
    constexpr float kLargest = 65504.0f;
    // Infinities stay (clamping them would make them finite), NaN stays.
    const float clamped = fminf(fmaxf(v, -kLargest), kLargest);
    return _Float16(isfinite(v) ? clamped : v);
}

struct RotationRule {
    uint32_t kind = 0;  // mfh_rope_scaling_kind
    double theta = 0, factor = 1, original = 0, low = 0, high = 0, magnitude = 1;
};
void launch_scaled_rotation_table(hipStream_t stream, float *table, uint64_t positions,
                                  uint32_t dim, const RotationRule &rule);

struct PagedRope {
    float *query_out = nullptr;
    void *key_pages = nullptr, *value_pages = nullptr;
    const float *query = nullptr, *key = nullptr, *value = nullptr;
    const float *query_weight = nullptr, *key_weight = nullptr;  // null: no norm
    const float *rotation = nullptr;   // [rotation_rows, rotary_dim]
    const float *tables = nullptr;     // [sequences, max_pages]
    const float *sequences = nullptr;  // [tokens], null: token t is sequence t
    const float *positions = nullptr;  // [tokens]
    const float *places = nullptr;     // [tokens], null: the positions
    PageShape shape;
    uint64_t tokens = 0;
    uint32_t rotation_rows = 0, rotary_dim = 0, sequence_count = 0, max_pages = 0;
    uint32_t query_heads = 0;
    bool interleaved = false;
    float epsilon = 0.0f;
};
void launch_paged_qk_norm_rope(hipStream_t stream, const PagedRope &p);

// One launch of a page copy: `pairs` (from, to) pages in each of `buffers`.  It is the
// kernel's argument, of 4 KB at most, which the host writes for every launch: a short
// form serves the few pages of a fork.
constexpr uint32_t kCopyBuffers = 32, kCopyPairs = 416, kCopyFewPairs = 8;
template <uint32_t PAIRS>
struct PageCopy {
    uint32_t pairs = 0, buffers = 0;
    uint64_t elements = 0;  // of one page
    void *to[kCopyBuffers];
    const void *from[kCopyBuffers];
    uint8_t to_half[kCopyBuffers], from_half[kCopyBuffers];
    uint32_t from_page[PAIRS], to_page[PAIRS];
};
template <uint32_t PAIRS>
void launch_copy_pages(hipStream_t stream, const PageCopy<PAIRS> &c);

// One new token per sequence over paged caches.
struct PagedAttention {
    float *out = nullptr;  // [sequences, query_heads * head_dim]
    const float *query = nullptr;
    const void *key_pages = nullptr, *value_pages = nullptr;
    const float *tables = nullptr;   // [sequences, max_pages]
    const float *lengths = nullptr;  // [sequences]
    PageShape shape;
    uint32_t sequences = 0, max_pages = 0, query_heads = 0, group = 0;
    float scale = 0.0f;
    // Filled by paged_gqa_plan: query rows of a key/value head that one item
    // holds, items per key/value head, keys of a unit and units that a block takes at
    // least (their logarithms), units that an item costs besides, blocks, the longest
    // length.
    uint32_t rows = 0, row_tiles = 0, unit_shift = 0, least_shift = 0, item_units = 0;
    uint32_t blocks = 0;
    float longest = 0.0f;
    float *records = nullptr;  // paged_gqa_scratch_bytes
};
// Widest head that the kernels serve.
constexpr uint32_t kMaxPagedHeadDim = 1024;
// Chooses the kernel's split; false where the extents pass its index range.
bool paged_gqa_plan(PagedAttention &p, int cu_count);
size_t paged_gqa_scratch_bytes(const PagedAttention &p);
void launch_paged_gqa(hipStream_t stream, const PagedAttention &p);

// The next token of each row from given uniforms (sample.hip).
struct Sampling {
    float *out = nullptr, *copy = nullptr;  // [rows]; copy may be null
    const float *logits = nullptr;          // [rows, width]
    const float *uniforms = nullptr;        // [rows]
    const float *params = nullptr;          // [rows or 1, 4]
    const uint8_t *mask = nullptr;          // [rows or 1, ceil(width / 8)], may be null
    uint32_t rows = 0, width = 0;
    bool one_params = false, one_mask = false;
};
void launch_sample_rows(hipStream_t stream, const Sampling &s);
// mfh_sample_rows' admission, for `uniform_count` values in `uniforms` (a row's, or
// those of several calls): fills `call`, enqueues nothing.
mfh_status admit_sample_rows(mfh_ctx *ctx, mfh_buf *output, const mfh_buf *logits,
                             const mfh_buf *uniforms, uint64_t uniform_count,
                             const mfh_buf *params, const mfh_buf *mask, Sampling *call);
// Enqueues an admitted call.
mfh_status run_sample_rows(mfh_ctx *ctx, const Sampling &call);

}  // namespace mfh
