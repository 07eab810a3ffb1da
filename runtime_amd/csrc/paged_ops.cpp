// Paged key/value caches and sampling: admission and launches.
//
// As for the dense operations, every operand is validated before anything is
// enqueued, a rejected call writes nothing, and values on the device are not
// inspected on the host: the kernels check every page id, length, position and
// sampling parameter themselves and answer a bad one with NaN.
#include <cmath>
#include <memory>
#include <new>

#include "internal.hpp"
#include "kernels.hpp"
#include "paged.hpp"

namespace mfh {
namespace {

const float *dev_f32(const mfh_buf *b) { return static_cast<const float *>(b->dev); }
float *dev_f32(mfh_buf *b) { return static_cast<float *>(b->dev); }

mfh_status launched(mfh_ctx *ctx)
{
    if (hipGetLastError() != hipSuccess)
        return fail(ctx, MFH_BACKEND_FAILURE, "paged kernel launch failed");
    return MFH_OK;
}

// Exact f32 values reach 2^24.
constexpr uint64_t kIndexLimit = uint64_t(1) << 24;

// The geometry of a page buffer: [pages, kv_heads, page_size, head_dim] F32, or
// U8 with twice the width.
mfh_status page_shape_of(mfh_ctx *ctx, const uint64_t (&dims)[4], bool half, PageShape *out)
{
    out->half = half;
    if (half && dims[3] % 2 != 0)
        return fail(ctx, MFH_INVALID_SHAPE, "binary16 page rows must hold an even byte count");
    const uint64_t d = half ? dims[3] / 2 : dims[3], size = dims[2];
    if (dims[0] == 0 || dims[1] == 0 || d == 0)
        return fail(ctx, MFH_INVALID_SHAPE, "page buffers must have a page, a head and a column");
    if (size < 8 || size > 4096 || (size & (size - 1)))
        return fail(ctx, MFH_INVALID_SHAPE, "page size must be a power of two in [8, 4096]");
    if (dims[0] > kIndexLimit)
        return fail(ctx, MFH_UNSUPPORTED, "page count exceeds the exact f32 index range");
    if (dims[1] > UINT16_MAX || d > UINT16_MAX)
        return fail(ctx, MFH_OVERFLOW, "page extent exceeds the kernel index range");
    out->pages = uint32_t(dims[0]);
    out->kv_heads = uint32_t(dims[1]);
    out->page_shift = uint32_t(__builtin_ctzll(size));
    out->head_dim = uint32_t(d);
    return MFH_OK;
}
mfh_status page_shape(mfh_ctx *ctx, const mfh_buf *buf, PageShape *out)
{
    mfh_status s = check_buffer(ctx, buf);
    if (s)
        return s;
    if (buf->rank != 4)
        return fail(ctx, MFH_INVALID_SHAPE,
                    "page buffers must be [pages, kv_heads, page_size, head_dim]");
    return page_shape_of(ctx, buf->dims, buf->dtype == MFH_DTYPE_U8, out);
}

// Key and value pages of one cache.
mfh_status cache_shape(mfh_ctx *ctx, const mfh_buf *key_pages, const mfh_buf *value_pages,
                       uint32_t key_value_heads, uint32_t head_dim, PageShape *out)
{
    PageShape value;
    mfh_status s = page_shape(ctx, key_pages, out);
    if (!s)
        s = page_shape(ctx, value_pages, &value);
    if (s)
        return s;
    if (key_pages->dtype != value_pages->dtype || !same_shape(key_pages, value_pages))
        return fail(ctx, MFH_INVALID_SHAPE, "key and value pages must have one shape and format");
    if (key_pages->dev == value_pages->dev)
        return fail(ctx, MFH_INVALID_ARGUMENT, "key and value caches must have distinct storage");
    if (out->kv_heads != key_value_heads || out->head_dim != head_dim)
        return fail(ctx, MFH_INVALID_SHAPE, "page buffer heads differ from descriptor");
    return MFH_OK;
}

mfh_status check_heads(mfh_ctx *ctx, uint32_t query_heads, uint32_t key_value_heads,
                       uint32_t head_dim)
{
    if (key_value_heads == 0 || query_heads == 0 || query_heads % key_value_heads != 0)
        return fail(ctx, MFH_INVALID_SHAPE,
                    "query heads must be a nonzero multiple of key/value heads");
    if (head_dim == 0)
        return fail(ctx, MFH_INVALID_ARGUMENT, "head count and head dimension must be nonzero");
    return MFH_OK;
}

// A sequence table: [sequences, max_pages] page ids.
mfh_status check_tables(mfh_ctx *ctx, const mfh_buf *tables)
{
    mfh_status s = check_f32(ctx, tables);
    if (s)
        return s;
    if (tables->rank != 2)
        return fail(ctx, MFH_INVALID_SHAPE, "page tables must be [sequences, max_pages]");
    if (tables->dims[0] > kIndexLimit || tables->dims[1] > kIndexLimit)
        return fail(ctx, MFH_UNSUPPORTED, "page table extent exceeds the exact f32 index range");
    return MFH_OK;
}

// An F32 operand of shape [dims[0], ...].
mfh_status check_dims(mfh_ctx *ctx, const mfh_buf *buf, uint64_t rows, uint64_t columns,
                      const char *message)
{
    mfh_status s = check_f32(ctx, buf);
    if (s)
        return s;
    if (buf->rank != 2 || buf->dims[0] != rows || buf->dims[1] != columns)
        return fail(ctx, MFH_INVALID_SHAPE, message);
    return MFH_OK;
}

mfh_status check_vector(mfh_ctx *ctx, const mfh_buf *buf, uint64_t count, const char *message)
{
    mfh_status s = check_f32(ctx, buf);
    if (s)
        return s;
    if (buf->rank != 1 || buf->dims[0] != count)
        return fail(ctx, MFH_INVALID_SHAPE, message);
    return MFH_OK;
}

mfh_status aliased(mfh_ctx *ctx)
{
    return fail(ctx, MFH_INVALID_ARGUMENT, "output aliases an input");
}

// The launches of a page copy, PAIRS pages and kCopyBuffers buffers at most in each.
template <uint32_t PAIRS>
void copy_pairs(hipStream_t stream, uint64_t elements, mfh_buf *const *destinations,
                const mfh_buf *const *sources, size_t buffers, const uint32_t *from_pages,
                const uint32_t *to_pages, size_t count)
{
    PageCopy<PAIRS> c;
    c.elements = elements;
    for (size_t b = 0; count && b < buffers; b += c.buffers) {
        c.buffers = uint32_t(buffers - b < kCopyBuffers ? buffers - b : kCopyBuffers);
        for (uint32_t i = 0; i < c.buffers; ++i) {
            c.to[i] = destinations[b + i]->dev;
            c.from[i] = sources[b + i]->dev;
            c.to_half[i] = destinations[b + i]->dtype == MFH_DTYPE_U8;
            c.from_half[i] = sources[b + i]->dtype == MFH_DTYPE_U8;
        }
        for (size_t n = 0; n < count; n += c.pairs) {
            c.pairs = uint32_t(count - n < PAIRS ? count - n : PAIRS);
            for (uint32_t i = 0; i < c.pairs; ++i) {
                c.from_page[i] = from_pages[n + i];
                c.to_page[i] = to_pages[n + i];
            }
            launch_copy_pages(stream, c);
        }
    }
}

// Page ids, by open addressing in a table of twice their number or more: the work
// follows the ids, whatever the cache's page count.  The few ids of a fork need no
// allocation.
class PageSet {
  public:
    explicit PageSet(size_t count)
    {
        while (size_t(1) << bits_ < 2 * count)
            ++bits_;
        if (size_t(1) << bits_ > kFew) {
            heap_.reset(new (std::nothrow) uint32_t[size_t(1) << bits_]);
            slots_ = heap_.get();
        }
        for (size_t i = 0; slots_ && i < size_t(1) << bits_; ++i)
            slots_[i] = kNone;
    }
    bool allocated() const { return slots_ != nullptr; }
    // The id's slot, or the free one that it would have.
    uint32_t &slot(uint32_t id)
    {
        // The upper bits of a product with 2^32 over the golden ratio.
        size_t at = uint32_t(id * 2654435769u) >> (32 - bits_);
        while (slots_[at] != kNone && slots_[at] != id)
            at = (at + 1) & ((size_t(1) << bits_) - 1);
        return slots_[at];
    }
    bool has(uint32_t id) { return slot(id) == id; }
    // False where it was there.
    bool add(uint32_t id)
    {
        uint32_t &to = slot(id);
        if (to == id)
            return false;
        to = id;
        return true;
    }

  private:
    static constexpr uint32_t kNone = UINT32_MAX;  // no page: ids are below 2^24
    static constexpr size_t kFew = 32;
    unsigned bits_ = 1;
    uint32_t few_[kFew];
    std::unique_ptr<uint32_t[]> heap_;
    uint32_t *slots_ = few_;
};

bool positive(float v) { return std::isfinite(v) && v > 0.0f; }

}  // namespace
}  // namespace mfh

using namespace mfh;

extern "C" {

mfh_status mfh_alloc_pages(mfh_ctx *ctx, uint64_t pages, uint32_t key_value_heads,
                           uint32_t page_size, uint32_t head_dim, int half, mfh_buf **out)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    if (!out)
        return fail(ctx, MFH_INVALID_ARGUMENT, "output handle pointer is null");
    *out = nullptr;
    const uint64_t dims[4] = {pages, key_value_heads, page_size,
                              half ? 2 * uint64_t(head_dim) : head_dim};
    PageShape shape;
    if (mfh_status s = page_shape_of(ctx, dims, half != 0, &shape))
        return s;
    return half ? alloc_zeroed_u8(ctx, dims, 4, MFH_CLASS_CACHE, out)
                : mfh_alloc_f32(ctx, dims, 4, MFH_CLASS_CACHE, 1, out);
}

mfh_status mfh_rotation_table(mfh_ctx *ctx, mfh_buf *output, float theta,
                              const mfh_rope_scaling *scaling)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    mfh_status s = check_operation(ctx, MFH_OP_ROTARY);
    if (!s)
        s = check_f32(ctx, output);
    if (s)
        return s;
    if (output->rank != 2)
        return fail(ctx, MFH_INVALID_SHAPE, "rotation table must be [positions, rotary_dim]");
    if (output->dims[1] == 0 || output->dims[1] % 2 != 0)
        return fail(ctx, MFH_INVALID_SHAPE, "rotation table width must be even and nonzero");
    if (!positive(theta))
        return fail(ctx, MFH_INVALID_ARGUMENT, "RoPE theta must be finite and positive");
    if (output->dims[0] > kIndexLimit || output->dims[1] > kIndexLimit)
        return fail(ctx, MFH_UNSUPPORTED, "rotation table exceeds the exact f32 index range");
    RotationRule rule;
    rule.theta = double(theta);
    if (scaling) {
        const uint32_t kind = scaling->kind;
        if (kind > MFH_ROPE_YARN)
            return fail(ctx, MFH_INVALID_ARGUMENT, "unknown RoPE scaling");
        if (!positive(scaling->magnitude))
            return fail(ctx, MFH_INVALID_ARGUMENT, "RoPE magnitude must be finite and positive");
        if (kind != MFH_ROPE_PLAIN && !positive(scaling->factor))
            return fail(ctx, MFH_INVALID_ARGUMENT,
                        "RoPE scaling factor must be finite and positive");
        if (kind == MFH_ROPE_NTK && output->dims[1] == 2)
            return fail(ctx, MFH_INVALID_SHAPE, "NTK scaling requires more than one pair");
        if (kind == MFH_ROPE_WAVELENGTH || kind == MFH_ROPE_YARN) {
            if (!positive(scaling->original_positions) || !positive(scaling->low) ||
                !positive(scaling->high) || !(scaling->high > scaling->low))
                return fail(ctx, MFH_INVALID_ARGUMENT,
                            "RoPE scaling needs original positions and 0 < low < high");
            if (kind == MFH_ROPE_YARN && !(theta > 1.0f))
                return fail(ctx, MFH_INVALID_ARGUMENT, "this RoPE scaling requires theta above 1");
        }
        rule.kind = kind;
        rule.factor = double(scaling->factor);
        rule.original = double(scaling->original_positions);
        rule.low = double(scaling->low);
        rule.high = double(scaling->high);
        rule.magnitude = double(scaling->magnitude);
    }
    DeviceGuard guard(ctx->device);
    mark_written(output);
    launch_scaled_rotation_table(ctx->stream, dev_f32(output), output->dims[0],
                                 uint32_t(output->dims[1]), rule);
    return launched(ctx);
}

mfh_status mfh_paged_qk_norm_rope(mfh_ctx *ctx, mfh_buf *query_out, mfh_buf *key_pages,
                                  mfh_buf *value_pages, const mfh_buf *query, const mfh_buf *key,
                                  const mfh_buf *value, const mfh_buf *query_weight,
                                  const mfh_buf *key_weight, const mfh_buf *rotation,
                                  const mfh_buf *tables, const mfh_buf *sequences,
                                  const mfh_buf *positions, uint32_t query_heads,
                                  uint32_t key_value_heads, uint32_t head_dim, int interleaved,
                                  float epsilon)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    mfh_status s = check_heads(ctx, query_heads, key_value_heads, head_dim);
    if (!s)
        s = check_operation(ctx, MFH_OP_QK_NORM_ROPE);
    if (s)
        return s;
    if (!positive(epsilon))
        return fail(ctx, MFH_INVALID_ARGUMENT, "RMS epsilon must be finite and positive");
    PagedRope p;
    if ((s = cache_shape(ctx, key_pages, value_pages, key_value_heads, head_dim, &p.shape)) ||
        (s = check_f32(ctx, query)))
        return s;
    if (query->rank != 2 || query->dims[1] != uint64_t(query_heads) * head_dim)
        return fail(ctx, MFH_INVALID_SHAPE, "packed head tensor width differs from descriptor");
    const uint64_t tokens = query->dims[0], kv_width = uint64_t(key_value_heads) * head_dim;
    if ((s = check_dims(ctx, key, tokens, kv_width, "keys must be [tokens, kv_heads * head_dim]")) ||
        (s = check_dims(ctx, value, tokens, kv_width,
                        "values must be [tokens, kv_heads * head_dim]")))
        return s;
    if (!query_weight != !key_weight)
        return fail(ctx, MFH_INVALID_ARGUMENT,
                    "query and key norm weights must be given together");
    if (query_weight &&
        ((s = check_vector(ctx, query_weight, head_dim,
                           "head RMS weight must have head_dim entries")) ||
         (s = check_vector(ctx, key_weight, head_dim,
                           "head RMS weight must have head_dim entries"))))
        return s;
    if ((s = check_f32(ctx, rotation)))
        return s;
    if (rotation->rank != 2 || rotation->dims[1] % 2 != 0 || rotation->dims[1] > head_dim)
        return fail(ctx, MFH_INVALID_SHAPE,
                    "rotation table must be [positions, even width up to head_dim]");
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
        (s = check_output(ctx, query_out, query->dims, 2)))
        return s;
    if (tokens > uint64_t(INT32_MAX) / 256 / (query_heads + 2 * uint64_t(key_value_heads)))
        return fail(ctx, MFH_OVERFLOW, "token count exceeds the kernel index range");
    if (aliases(query_out, {query, key, value, query_weight, key_weight, rotation, tables,
                            sequences, positions, key_pages, value_pages}) ||
        aliases(key_pages, {query, key, value, query_weight, key_weight, rotation, tables,
                            sequences, positions}) ||
        aliases(value_pages, {query, key, value, query_weight, key_weight, rotation, tables,
                              sequences, positions}))
        return aliased(ctx);
    DeviceGuard guard(ctx->device);
    mark_written(query_out);
    mark_written(key_pages);
    mark_written(value_pages);
    if (!tokens)
        return MFH_OK;
    p.query_out = dev_f32(query_out);
    p.key_pages = key_pages->dev;
    p.value_pages = value_pages->dev;
    p.query = dev_f32(query);
    p.key = dev_f32(key);
    p.value = dev_f32(value);
    p.query_weight = query_weight ? dev_f32(query_weight) : nullptr;
    p.key_weight = key_weight ? dev_f32(key_weight) : nullptr;
    p.rotation = dev_f32(rotation);
    p.tables = dev_f32(tables);
    p.sequences = sequences ? dev_f32(sequences) : nullptr;
    p.positions = dev_f32(positions);
    p.tokens = tokens;
    p.rotation_rows = uint32_t(rotation->dims[0]);
    p.rotary_dim = uint32_t(rotation->dims[1]);
    p.sequence_count = uint32_t(tables->dims[0]);
    p.max_pages = uint32_t(tables->dims[1]);
    p.query_heads = query_heads;
    p.interleaved = interleaved != 0;
    p.epsilon = epsilon;
    launch_paged_qk_norm_rope(ctx->stream, p);
    return launched(ctx);
}

mfh_status mfh_paged_gqa(mfh_ctx *ctx, mfh_buf *output, const mfh_buf *query,
                         const mfh_buf *key_pages, const mfh_buf *value_pages,
                         const mfh_buf *tables, const mfh_buf *lengths, uint32_t query_heads,
                         uint32_t key_value_heads, uint32_t head_dim)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    mfh_status s = check_heads(ctx, query_heads, key_value_heads, head_dim);
    if (!s)
        s = check_operation(ctx, MFH_OP_GROUPED_QUERY_ATTENTION);
    PagedAttention p;
    if (!s)
        s = cache_shape(ctx, key_pages, value_pages, key_value_heads, head_dim, &p.shape);
    if (!s)
        s = check_tables(ctx, tables);
    if (!s)
        s = check_f32(ctx, query);
    if (s)
        return s;
    const uint64_t sequences = tables->dims[0];
    if ((s = check_dims(ctx, query, sequences, uint64_t(query_heads) * head_dim,
                        "queries must be [sequences, query_heads * head_dim]")) ||
        (s = check_vector(ctx, lengths, sequences, "lengths must be one per sequence")) ||
        (s = check_output(ctx, output, query->dims, 2)))
        return s;
    if (head_dim > kMaxPagedHeadDim)
        return fail(ctx, MFH_UNSUPPORTED, "GQA head dimension exceeds the device kernel limit");
    if (aliases(output, {query, key_pages, value_pages, tables, lengths}))
        return aliased(ctx);
    p.sequences = uint32_t(sequences);
    p.max_pages = uint32_t(tables->dims[1]);
    p.query_heads = query_heads;
    p.group = query_heads / key_value_heads;
    // Scores are formed times log2 e: the kernels take powers of two.
    p.scale = float(1.4426950408889634 / std::sqrt(double(head_dim)));
    if (!paged_gqa_plan(p, ctx->cu_count))
        return fail(ctx, MFH_OVERFLOW, "paged attention extent exceeds the kernel index range");
    DeviceGuard guard(ctx->device);
    if (const size_t bytes = paged_gqa_scratch_bytes(p)) {
        p.records = static_cast<float *>(paged_scratch(ctx, bytes));
        if (!p.records)
            return allocation_failed(ctx);
    }
    mark_written(output);
    if (!sequences)
        return MFH_OK;
    p.out = dev_f32(output);
    p.query = dev_f32(query);
    p.key_pages = key_pages->dev;
    p.value_pages = value_pages->dev;
    p.tables = dev_f32(tables);
    p.lengths = dev_f32(lengths);
    launch_paged_gqa(ctx->stream, p);
    return launched(ctx);
}

mfh_status mfh_copy_pages(mfh_ctx *ctx, mfh_buf *const *destinations,
                          const mfh_buf *const *sources, size_t buffers,
                          const uint32_t *from_pages, const uint32_t *to_pages, size_t count)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    mfh_status s = check_operation(ctx, MFH_OP_COPY);
    if (s)
        return s;
    if (buffers && (!destinations || !sources))
        return fail(ctx, MFH_INVALID_ARGUMENT, "page buffer list is null");
    if (count && (!from_pages || !to_pages))
        return fail(ctx, MFH_INVALID_ARGUMENT, "page list is null");
    PageShape first;
    uint64_t least_from = UINT64_MAX, least_to = UINT64_MAX;  // pages of the smallest buffers
    bool in_place = false;
    for (size_t i = 0; i < buffers; ++i) {
        PageShape to, from;
        if ((s = page_shape(ctx, destinations[i], &to)) || (s = page_shape(ctx, sources[i], &from)))
            return s;
        if (i == 0)
            first = to;
        for (const PageShape *p : {&to, &from})
            if (p->kv_heads != first.kv_heads || p->page_shift != first.page_shift ||
                p->head_dim != first.head_dim)
                return fail(ctx, MFH_INVALID_SHAPE, "page buffers differ in page shape");
        least_to = to.pages < least_to ? to.pages : least_to;
        least_from = from.pages < least_from ? from.pages : least_from;
        in_place = in_place || destinations[i]->dev == sources[i]->dev;
    }
    for (size_t i = 0; i < buffers; ++i)
        for (size_t j = 0; j < buffers; ++j)
            if (j != i && (destinations[i]->dev == sources[j]->dev ||
                           destinations[i]->dev == destinations[j]->dev))
                return fail(ctx, MFH_INVALID_ARGUMENT,
                            "a destination is another pair's source or destination");
    for (size_t i = 0; buffers && i < count; ++i)
        if (from_pages[i] >= least_from || to_pages[i] >= least_to)
            return fail(ctx, MFH_OUT_OF_BOUNDS, "page id exceeds the page count");
    // No page is written twice, and in place none written that is read: the
    // copies run in no order.
    if (buffers && count > 1) {
        const char *message = "a page is copied to twice, or copied from and to";
        // More than every page once is a page twice; the table stays small.
        if (count > least_to)
            return fail(ctx, MFH_INVALID_ARGUMENT, message);
        PageSet targets(count);
        if (!targets.allocated())
            return fail(ctx, MFH_RESOURCE_LIMIT, "host allocation failed");
        for (size_t i = 0; i < count; ++i)
            if (!targets.add(to_pages[i]))
                return fail(ctx, MFH_INVALID_ARGUMENT, message);
        for (size_t i = 0; in_place && i < count; ++i)
            if (targets.has(from_pages[i]))
                return fail(ctx, MFH_INVALID_ARGUMENT, message);
    } else if (buffers && count == 1 && in_place && from_pages[0] == to_pages[0]) {
        return fail(ctx, MFH_INVALID_ARGUMENT, "a page is copied to twice, or copied from and to");
    }
    DeviceGuard guard(ctx->device);
    for (size_t i = 0; i < buffers; ++i)
        mark_written(destinations[i]);
    if (count <= kCopyFewPairs)
        copy_pairs<kCopyFewPairs>(ctx->stream, first.stride(), destinations, sources, buffers,
                                  from_pages, to_pages, count);
    else
        copy_pairs<kCopyPairs>(ctx->stream, first.stride(), destinations, sources, buffers,
                               from_pages, to_pages, count);
    return launched(ctx);
}

mfh_status mfh_sample_rows(mfh_ctx *ctx, mfh_buf *output, const mfh_buf *logits,
                           const mfh_buf *uniforms, const mfh_buf *params, const mfh_buf *mask)
{
    if (!ctx)
        return MFH_INVALID_ARGUMENT;
    Sampling call;
    mfh_status s = check_f32(ctx, logits);
    if (!s)
        s = admit_sample_rows(ctx, output, logits, uniforms, logits->dims[0], params, mask, &call);
    if (s)
        return s;
    mark_written(output);
    return run_sample_rows(ctx, call);
}

}  // extern "C"

namespace mfh {

mfh_status admit_sample_rows(mfh_ctx *ctx, mfh_buf *output, const mfh_buf *logits,
                             const mfh_buf *uniforms, uint64_t uniform_count,
                             const mfh_buf *params, const mfh_buf *mask, Sampling *call)
{
    mfh_status s = check_operation(ctx, MFH_OP_ARGMAX);
    if (!s)
        s = check_f32(ctx, logits);
    if (s)
        return s;
    if (logits->rank != 2)
        return fail(ctx, MFH_INVALID_SHAPE, "sampling logits must be rank two");
    const uint64_t rows = logits->dims[0], width = logits->dims[1];
    if (width == 0 || width > kIndexLimit)
        return fail(ctx, MFH_UNSUPPORTED,
                    "sampling width must be in [1, 2^24] for exact f32 indices");
    if ((s = check_vector(ctx, uniforms, uniform_count,
                          "uniform values must be one per row and step")) ||
        (s = check_f32(ctx, params)))
        return s;
    if (params->rank != 2 || params->dims[1] != 4 || (params->dims[0] != rows && params->dims[0] != 1))
        return fail(ctx, MFH_INVALID_SHAPE, "sampling parameters must be [rows or 1, 4]");
    if (mask) {
        if ((s = check_u8(ctx, mask)))
            return s;
        if (mask->rank != 2 || mask->dims[1] != (width + 7) / 8 ||
            (mask->dims[0] != rows && mask->dims[0] != 1))
            return fail(ctx, MFH_INVALID_SHAPE, "sampling mask must be [rows or 1, ceil(width / 8)]");
    }
    const uint64_t dims[1] = {rows};
    if ((s = check_output(ctx, output, dims, 1)))
        return s;
    if (aliases(output, {logits, uniforms, params, mask}))
        return aliased(ctx);
    if (rows > uint64_t(INT32_MAX) / 1024)
        return fail(ctx, MFH_OVERFLOW, "sampling row count exceeds the kernel index range");
    call->out = dev_f32(output);
    call->logits = dev_f32(logits);
    call->uniforms = dev_f32(uniforms);
    call->params = dev_f32(params);
    call->mask = mask ? static_cast<const uint8_t *>(mask->dev) : nullptr;
    call->rows = uint32_t(rows);
    call->width = uint32_t(width);
    call->one_params = params->dims[0] == 1;
    call->one_mask = mask && mask->dims[0] == 1;
    return MFH_OK;
}

mfh_status run_sample_rows(mfh_ctx *ctx, const Sampling &call)
{
    DeviceGuard guard(ctx->device);
    launch_sample_rows(ctx->stream, call);
    if (hipGetLastError() != hipSuccess)
        return fail(ctx, MFH_BACKEND_FAILURE, "sampling launch failed");
    return MFH_OK;
}

}  // namespace mfh
