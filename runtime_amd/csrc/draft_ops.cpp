// Runs of new tokens over paged caches: admission and launches of trees' layout, attention
// and settling, and of latent caches.
//
// As for the other paged operations, operands are validated before anything is enqueued,
// and values on the device (starts, parents, lengths, ids) by the kernels.
#include <cmath>

#include "draft.hpp"
#include "internal.hpp"
#include "kernels.hpp"
#include "paged_checks.hpp"

namespace mfh {
namespace {

// Blocks of 256 threads that a launch may have in one direction.
constexpr uint64_t kMostBlocks = uint64_t(INT32_MAX) / 256;
// Runs of a batch with a list of starts: layout's and settling's blocks look through it up to
// their own, settling's once for each buffer (1024 runs of two 9 us and 10 with a buffer, 52
// with 16; 65536 3.8 ms, 3.7 and 58).
constexpr uint64_t kMostRuns = 65536;

// The runs of a batch of `tokens`; `starts` may be null where `one_each`.
mfh_status check_runs(mfh_ctx *ctx, const mfh_buf *starts, const mfh_buf *lengths,
                      uint64_t tokens, bool one_each, Runs *out)
{
    mfh_status s = check_f32(ctx, lengths);
    if (s)
        return s;
    if (lengths->rank != 1)
        return fail(ctx, MFH_INVALID_SHAPE, "lengths must be one per sequence");
    const uint64_t sequences = lengths->dims[0];
    if (!starts && one_each) {
        if (sequences != tokens)
            return fail(ctx, MFH_INVALID_SHAPE,
                        "without starts the batch must have a token per sequence");
    } else if ((s = check_vector(ctx, starts, sequences + 1,
                                 "starts must be one per sequence and one"))) {
        return s;
    }
    if (tokens > kMostBlocks || sequences > kMostBlocks || (starts && sequences > kMostRuns))
        return fail(ctx, MFH_OVERFLOW, "token or sequence count exceeds the kernel index range");
    out->starts = starts ? dev_f32(starts) : nullptr;
    out->lengths = dev_f32(lengths);
    out->sequences = uint32_t(sequences);
    out->tokens = uint32_t(tokens);
    return MFH_OK;
}

// A mask of runs: [tokens, bytes], one byte at least.
mfh_status check_mask(mfh_ctx *ctx, const mfh_buf *mask, uint64_t tokens, uint32_t *bytes)
{
    mfh_status s = check_u8(ctx, mask);
    if (s)
        return s;
    if (mask->rank != 2 || mask->dims[0] != tokens || mask->dims[1] == 0)
        return fail(ctx, MFH_INVALID_SHAPE, "run masks must be [tokens, bytes]");
    if (mask->dims[1] > kIndexLimit / 8)
        return fail(ctx, MFH_UNSUPPORTED, "run mask exceeds the exact f32 index range");
    *bytes = uint32_t(mask->dims[1]);
    return MFH_OK;
}

// What attention over runs checks of its batch, tables and mask, and the launch.
mfh_status attend(mfh_ctx *ctx, mfh_buf *output, const mfh_buf *query,
                  const mfh_buf *rotary_query, const mfh_buf *key_pages,
                  const mfh_buf *value_pages, const mfh_buf *tables, const mfh_buf *starts,
                  const mfh_buf *lengths, const mfh_buf *mask, RunAttention &p)
{
    const uint64_t tokens = query->dims[0];
    mfh_status s = check_tables(ctx, tables);
    if (!s)
        s = check_runs(ctx, starts, lengths, tokens, true, &p.runs);
    if (!s && mask)
        s = check_mask(ctx, mask, tokens, &p.mask_bytes);
    if (s)
        return s;
    if (tables->dims[0] != p.runs.sequences)
        return fail(ctx, MFH_INVALID_SHAPE, "page tables must have a row per sequence");
    if ((s = check_output(ctx, output, query->dims, 2)))
        return s;
    if (p.shape.head_dim > kMaxPagedHeadDim)
        return fail(ctx, MFH_UNSUPPORTED, "GQA head dimension exceeds the device kernel limit");
    if (aliases(output, {query, rotary_query, key_pages, value_pages, tables, starts, lengths,
                         mask}))
        return aliased(ctx);
    const uint64_t longest = tables->dims[1] << p.shape.page_shift;
    p.longest = uint32_t(longest < kIndexLimit ? longest : kIndexLimit);
    p.max_pages = uint32_t(tables->dims[1]);
    p.mask = mask ? static_cast<const uint8_t *>(mask->dev) : nullptr;
    if (!run_attention_plan(p, ctx->cu_count))
        return fail(ctx, MFH_OVERFLOW, "paged attention extent exceeds the kernel index range");
    DeviceGuard guard(ctx->device);
    if (const size_t bytes = run_attention_scratch_bytes(p)) {
        p.records = static_cast<float *>(paged_scratch(ctx, bytes));
        if (!p.records)
            return allocation_failed(ctx);
    }
    mark_written(output);
    if (!tokens || !p.runs.sequences)
        return MFH_OK;
    p.out = dev_f32(output);
    p.query = dev_f32(query);
    p.rotary_query = rotary_query ? dev_f32(rotary_query) : nullptr;
    p.key_pages = key_pages->dev;
    p.value_pages = value_pages->dev;
    p.tables = dev_f32(tables);
    launch_run_attention(ctx->stream, p);
    return launched(ctx);
}

// Settling; `parents` and `places` may be null.
mfh_status settle(mfh_ctx *ctx, mfh_buf *emitted, mfh_buf *counts, mfh_buf *next,
                  mfh_buf *const *pages, size_t buffers, const mfh_buf *tokens,
                  const mfh_buf *choices, const mfh_buf *starts, const mfh_buf *parents,
                  const mfh_buf *places, const mfh_buf *lengths, const mfh_buf *tables)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    mfh_status s = check_operation(ctx, MFH_OP_COPY);
    if (!s)
        s = check_f32(ctx, tokens);
    if (s)
        return s;
    if (tokens->rank != 1)
        return fail(ctx, MFH_INVALID_SHAPE, "drafted tokens must be one per token");
    Settle p;
    if ((s = check_runs(ctx, starts, lengths, tokens->dims[0], false, &p.runs)) ||
        (s = check_vector(ctx, choices, tokens->dims[0], "choices must be one per token")) ||
        (parents && (s = check_vector(ctx, parents, tokens->dims[0],
                                      "parents must be one per token"))) ||
        (places && (s = check_vector(ctx, places, tokens->dims[0],
                                     "places must be one per token"))) ||
        (s = check_tables(ctx, tables)) || (s = check_f32(ctx, emitted)) ||
        (s = check_vector(ctx, counts, p.runs.sequences, "counts must be one per sequence")) ||
        (s = check_vector(ctx, next, p.runs.sequences, "next tokens must be one per sequence")))
        return s;
    if (tables->dims[0] != p.runs.sequences)
        return fail(ctx, MFH_INVALID_SHAPE, "page tables must have a row per sequence");
    if (emitted->rank != 2 || emitted->dims[0] != p.runs.sequences || emitted->dims[1] == 0)
        return fail(ctx, MFH_INVALID_SHAPE, "emitted tokens must be [sequences, columns]");
    if (emitted->dims[1] > kSettleColumns)
        return fail(ctx, MFH_UNSUPPORTED, "accepted paths are at most 1024 tokens long");
    if (buffers && !pages)
        return fail(ctx, MFH_INVALID_ARGUMENT, "page buffer list is null");
    PageShape first;
    for (size_t i = 0; i < buffers; ++i) {
        PageShape shape;
        if ((s = page_shape(ctx, pages[i], &shape)))
            return s;
        if (i == 0)
            first = shape;
        if (shape.page_shift != first.page_shift)
            return fail(ctx, MFH_INVALID_SHAPE, "page buffers differ in page size");
        // A path's pages are in every buffer.
        first.pages = shape.pages < first.pages ? shape.pages : first.pages;
        if (uint64_t(shape.kv_heads) * shape.head_dim > uint64_t(UINT16_MAX) * 256)
            return fail(ctx, MFH_OVERFLOW, "page extent exceeds the kernel index range");
        if (aliases(pages[i], {emitted, counts, next, tokens, choices, starts, parents, places,
                               lengths, tables}))
            return aliased(ctx);
        for (size_t j = 0; j < i; ++j)
            if (pages[j]->dev == pages[i]->dev)
                return fail(ctx, MFH_INVALID_ARGUMENT, "a page buffer is listed twice");
    }
    if (aliases(emitted, {counts, next, tokens, choices, starts, parents, places, lengths, tables}) ||
        aliases(counts, {next, tokens, choices, starts, parents, places, lengths, tables}) ||
        aliases(next, {tokens, choices, starts, parents, places, lengths, tables}))
        return aliased(ctx);
    DeviceGuard guard(ctx->device);
    for (mfh_buf *out : {emitted, counts, next})
        mark_written(out);
    for (size_t i = 0; i < buffers; ++i)
        mark_written(pages[i]);
    if (!p.runs.sequences)
        return MFH_OK;
    p.parents = parents ? dev_f32(parents) : nullptr;
    p.places = places ? dev_f32(places) : nullptr;
    p.drafted = dev_f32(tokens);
    p.choices = dev_f32(choices);
    p.tables = dev_f32(tables);
    p.emitted = dev_f32(emitted);
    p.counts = dev_f32(counts);
    p.next = dev_f32(next);
    p.max_pages = uint32_t(tables->dims[1]);
    p.columns = uint32_t(emitted->dims[1]);
    p.pages = first.pages;
    p.page_shift = first.page_shift;
    p.path_pages = buffers != 0;
    size_t done = 0;
    do {
        p.buffers = uint32_t(buffers - done < kSettleBuffers ? buffers - done : kSettleBuffers);
        for (uint32_t i = 0; i < p.buffers; ++i) {
            const mfh_buf *b = pages[done + i];
            p.buffer[i] = b->dev;
            p.heads[i] = uint32_t(b->dims[1]);
            p.row_bytes[i] = uint32_t(b->dims[3] * (b->dtype == MFH_DTYPE_U8 ? 1 : 4));
        }
        launch_settle(ctx->stream, p);
        p.emitted = nullptr;
        done += p.buffers;
    } while (done < buffers);
    return launched(ctx);
}

// Scores are formed times log2 e: the kernels take powers of two.
constexpr double kLog2E = 1.4426950408889634;

}  // namespace
}  // namespace mfh

using namespace mfh;

extern "C" {

mfh_status mfh_draft_layout(mfh_ctx *ctx, mfh_buf *sequences, mfh_buf *positions,
                            mfh_buf *places, mfh_buf *mask, const mfh_buf *starts,
                            const mfh_buf *parents, const mfh_buf *lengths)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    mfh_status s = check_operation(ctx, MFH_OP_COPY);
    if (!s)
        s = check_f32(ctx, sequences);
    if (s)
        return s;
    if (sequences->rank != 1)
        return fail(ctx, MFH_INVALID_SHAPE, "layout outputs must be one per token");
    const uint64_t tokens = sequences->dims[0];
    DraftLayout p;
    if ((s = check_runs(ctx, starts, lengths, tokens, false, &p.runs)) ||
        (parents &&
         (s = check_vector(ctx, parents, tokens, "parents must be one per token"))) ||
        (s = check_vector(ctx, positions, tokens, "layout outputs must be one per token")) ||
        (s = check_vector(ctx, places, tokens, "layout outputs must be one per token")) ||
        (mask && (s = check_mask(ctx, mask, tokens, &p.mask_bytes))))
        return s;
    if (aliases(sequences, {positions, places, mask, starts, parents, lengths}) ||
        aliases(positions, {places, mask, starts, parents, lengths}) ||
        aliases(places, {mask, starts, parents, lengths}) ||
        (mask && aliases(mask, {starts, parents, lengths})))
        return aliased(ctx);
    DeviceGuard guard(ctx->device);
    for (mfh_buf *out : {sequences, positions, places, mask})
        if (out)
            mark_written(out);
    if (!tokens)
        return MFH_OK;
    p.parents = parents ? dev_f32(parents) : nullptr;
    p.sequences = dev_f32(sequences);
    p.positions = dev_f32(positions);
    p.places = dev_f32(places);
    p.mask = mask ? static_cast<uint8_t *>(mask->dev) : nullptr;
    launch_draft_layout(ctx->stream, p);
    return launched(ctx);
}

mfh_status mfh_paged_tree_gqa(mfh_ctx *ctx, mfh_buf *output, const mfh_buf *query,
                              const mfh_buf *key_pages, const mfh_buf *value_pages,
                              const mfh_buf *tables, const mfh_buf *starts,
                              const mfh_buf *lengths, const mfh_buf *mask, uint32_t query_heads,
                              uint32_t key_value_heads, uint32_t head_dim)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    mfh_status s = check_heads(ctx, query_heads, key_value_heads, head_dim);
    if (!s)
        s = check_operation(ctx, MFH_OP_GROUPED_QUERY_ATTENTION);
    RunAttention p;
    if (!s)
        s = cache_shape(ctx, key_pages, value_pages, key_value_heads, head_dim, &p.shape);
    if (!s)
        s = check_f32(ctx, query);
    if (s)
        return s;
    if (query->rank != 2 || query->dims[1] != uint64_t(query_heads) * head_dim)
        return fail(ctx, MFH_INVALID_SHAPE, "queries must be [tokens, query_heads * head_dim]");
    p.value_dim = head_dim;
    p.query_heads = query_heads;
    p.group = query_heads / key_value_heads;
    p.scale = float(kLog2E / std::sqrt(double(head_dim)));
    return attend(ctx, output, query, nullptr, key_pages, value_pages, tables, starts, lengths,
                  mask, p);
}

mfh_status mfh_paged_latent_attention(mfh_ctx *ctx, mfh_buf *output,
                                      const mfh_buf *latent_query, const mfh_buf *rotary_query,
                                      const mfh_buf *pages, const mfh_buf *tables,
                                      const mfh_buf *starts, const mfh_buf *lengths,
                                      const mfh_buf *mask, uint32_t query_heads, float scale)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    mfh_status s = check_operation(ctx, MFH_OP_GROUPED_QUERY_ATTENTION);
    RunAttention p;
    if (!s)
        s = page_shape(ctx, pages, &p.shape);
    if (!s)
        s = check_f32(ctx, latent_query);
    if (!s)
        s = check_f32(ctx, rotary_query);
    if (s)
        return s;
    if (p.shape.kv_heads != 1)
        return fail(ctx, MFH_INVALID_SHAPE, "latent pages must have one head");
    if (query_heads == 0 || query_heads > UINT16_MAX)
        return fail(ctx, MFH_INVALID_ARGUMENT, "query head count must be in [1, 65535]");
    p.scale = float(kLog2E * double(scale));
    if (!positive(scale) || !positive(p.scale))
        return fail(ctx, MFH_INVALID_ARGUMENT,
                    "attention scale must be positive and below 2.35e38");
    if (latent_query->rank != 2 || rotary_query->rank != 2 ||
        latent_query->dims[0] != rotary_query->dims[0] ||
        latent_query->dims[1] % query_heads != 0 || rotary_query->dims[1] % query_heads != 0)
        return fail(ctx, MFH_INVALID_SHAPE,
                    "queries must be [tokens, query_heads * rank] and [tokens, query_heads * rope]");
    const uint64_t rank = latent_query->dims[1] / query_heads;
    if (rank == 0 || rank + rotary_query->dims[1] / query_heads != p.shape.head_dim)
        return fail(ctx, MFH_INVALID_SHAPE, "latent page width differs from rank + rope");
    p.value_dim = uint32_t(rank);
    p.query_heads = p.group = query_heads;
    return attend(ctx, output, latent_query, rotary_query, pages, pages, tables, starts, lengths,
                  mask, p);
}

mfh_status mfh_paged_latent_append(mfh_ctx *ctx, mfh_buf *query_out, mfh_buf *pages,
                                   const mfh_buf *query, const mfh_buf *latent,
                                   const mfh_buf *key, const mfh_buf *latent_weight,
                                   const mfh_buf *rotation, const mfh_buf *tables,
                                   const mfh_buf *sequences, const mfh_buf *positions,
                                   const mfh_buf *places, uint32_t query_heads, int interleaved,
                                   float epsilon)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    mfh_status s = check_operation(ctx, MFH_OP_QK_NORM_ROPE);
    if (s)
        return s;
    if (!positive(epsilon))
        return fail(ctx, MFH_INVALID_ARGUMENT, "RMS epsilon must be finite and positive");
    if (query_heads == 0 || query_heads > UINT16_MAX)
        return fail(ctx, MFH_INVALID_ARGUMENT, "query head count must be in [1, 65535]");
    LatentAppend p;
    if ((s = page_shape(ctx, pages, &p.shape)) || (s = check_f32(ctx, latent)))
        return s;
    if (p.shape.kv_heads != 1)
        return fail(ctx, MFH_INVALID_SHAPE, "latent pages must have one head");
    if (latent->rank != 2 || latent->dims[1] == 0 || latent->dims[1] > p.shape.head_dim)
        return fail(ctx, MFH_INVALID_SHAPE, "latents must be [tokens, rank]");
    const uint64_t tokens = latent->dims[0], rank = latent->dims[1];
    const uint64_t rope = p.shape.head_dim - rank;
    if (rope % 2 != 0)
        return fail(ctx, MFH_INVALID_SHAPE, "rotated width must be even");
    if ((s = check_dims(ctx, key, tokens, rope, "rotated keys must be [tokens, rope]")) ||
        (s = check_dims(ctx, query, tokens, query_heads * rope,
                        "rotated queries must be [tokens, query_heads * rope]")) ||
        (latent_weight && (s = check_vector(ctx, latent_weight, rank,
                                            "latent RMS weight must have rank entries"))) ||
        (s = check_f32(ctx, rotation)))
        return s;
    if (rotation->rank != 2 || rotation->dims[1] != rope)
        return fail(ctx, MFH_INVALID_SHAPE, "rotation table must be [positions, rope]");
    if (rotation->dims[0] > kIndexLimit)
        return fail(ctx, MFH_UNSUPPORTED, "rotation table exceeds the exact f32 index range");
    if ((s = check_tables(ctx, tables)))
        return s;
    if (sequences) {
        if ((s = check_vector(ctx, sequences, tokens, "sequence ids must be one per token")))
            return s;
    } else if (tables->dims[0] != tokens) {
        return fail(ctx, MFH_INVALID_SHAPE,
                    "without sequence ids the page tables must have a row per token");
    }
    if ((s = check_vector(ctx, positions, tokens, "positions must be one per token")) ||
        (places && (s = check_vector(ctx, places, tokens, "places must be one per token"))) ||
        (s = check_output(ctx, query_out, query->dims, 2)))
        return s;
    if (tokens > kMostBlocks)
        return fail(ctx, MFH_OVERFLOW, "token count exceeds the kernel index range");
    if (aliases(query_out, {pages, query, latent, key, latent_weight, rotation, tables, sequences,
                            positions, places}) ||
        aliases(pages, {query, latent, key, latent_weight, rotation, tables, sequences, positions,
                        places}))
        return aliased(ctx);
    DeviceGuard guard(ctx->device);
    mark_written(query_out);
    mark_written(pages);
    if (!tokens)
        return MFH_OK;
    p.query_out = dev_f32(query_out);
    p.pages = pages->dev;
    p.query = dev_f32(query);
    p.latent = dev_f32(latent);
    p.key = dev_f32(key);
    p.weight = latent_weight ? dev_f32(latent_weight) : nullptr;
    p.rotation = dev_f32(rotation);
    p.tables = dev_f32(tables);
    p.sequences = sequences ? dev_f32(sequences) : nullptr;
    p.positions = dev_f32(positions);
    p.places = places ? dev_f32(places) : nullptr;
    p.tokens = uint32_t(tokens);
    p.rotation_rows = uint32_t(rotation->dims[0]);
    p.sequence_count = uint32_t(tables->dims[0]);
    p.max_pages = uint32_t(tables->dims[1]);
    p.query_heads = query_heads;
    p.rank = uint32_t(rank);
    p.rope = uint32_t(rope);
    p.interleaved = interleaved != 0;
    p.epsilon = epsilon;
    launch_latent_append(ctx->stream, p);
    return launched(ctx);
}

mfh_status mfh_settle_drafts(mfh_ctx *ctx, mfh_buf *emitted, mfh_buf *counts, mfh_buf *next,
                             mfh_buf *const *pages, size_t buffers, const mfh_buf *tokens,
                             const mfh_buf *choices, const mfh_buf *starts,
                             const mfh_buf *parents, const mfh_buf *lengths,
                             const mfh_buf *tables)
{
    return settle(ctx, emitted, counts, next, pages, buffers, tokens, choices, starts, parents,
                  nullptr, lengths, tables);
}

mfh_status mfh_settle_drafts_at(mfh_ctx *ctx, mfh_buf *emitted, mfh_buf *counts, mfh_buf *next,
                                mfh_buf *const *pages, size_t buffers, const mfh_buf *tokens,
                                const mfh_buf *choices, const mfh_buf *starts,
                                const mfh_buf *parents, const mfh_buf *places,
                                const mfh_buf *lengths, const mfh_buf *tables)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    if (mfh_status s = check_f32(ctx, places))
        return s;
    return settle(ctx, emitted, counts, next, pages, buffers, tokens, choices, starts, parents,
                  places, lengths, tables);
}

}  // extern "C"
