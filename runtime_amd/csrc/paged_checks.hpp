// Admission that the operations over paged caches share: page buffers, tables, operand
// shapes.
#pragma once

#include <cmath>

#include "internal.hpp"
#include "paged.hpp"

namespace mfh {

inline const float *dev_f32(const mfh_buf *b) { return static_cast<const float *>(b->dev); }
inline float *dev_f32(mfh_buf *b) { return static_cast<float *>(b->dev); }

inline mfh_status launched(mfh_ctx *ctx)
{
    if (hipGetLastError() != hipSuccess)
        return fail(ctx, MFH_BACKEND_FAILURE, "paged kernel launch failed");
    return MFH_OK;
}

// Exact f32 values reach 2^24.
constexpr uint64_t kIndexLimit = uint64_t(1) << 24;

// The geometry of a page buffer: [pages, kv_heads, page_size, head_dim] F32, or
// U8 with twice the width.
inline mfh_status page_shape_of(mfh_ctx *ctx, const uint64_t (&dims)[4], bool half, PageShape *out)
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
inline mfh_status page_shape(mfh_ctx *ctx, const mfh_buf *buf, PageShape *out)
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
inline mfh_status cache_shape(mfh_ctx *ctx, const mfh_buf *key_pages, const mfh_buf *value_pages,
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

inline mfh_status check_heads(mfh_ctx *ctx, uint32_t query_heads, uint32_t key_value_heads,
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
inline mfh_status check_tables(mfh_ctx *ctx, const mfh_buf *tables)
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
inline mfh_status check_dims(mfh_ctx *ctx, const mfh_buf *buf, uint64_t rows, uint64_t columns,
                             const char *message)
{
    mfh_status s = check_f32(ctx, buf);
    if (s)
        return s;
    if (buf->rank != 2 || buf->dims[0] != rows || buf->dims[1] != columns)
        return fail(ctx, MFH_INVALID_SHAPE, message);
    return MFH_OK;
}

inline mfh_status check_vector(mfh_ctx *ctx, const mfh_buf *buf, uint64_t count, const char *message)
{
    mfh_status s = check_f32(ctx, buf);
    if (s)
        return s;
    if (buf->rank != 1 || buf->dims[0] != count)
        return fail(ctx, MFH_INVALID_SHAPE, message);
    return MFH_OK;
}

inline mfh_status aliased(mfh_ctx *ctx)
{
    return fail(ctx, MFH_INVALID_ARGUMENT, "output aliases an input");
}

inline bool positive(float v) { return std::isfinite(v) && v > 0.0f; }

}  // namespace mfh
