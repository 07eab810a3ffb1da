// Rotation tables, the entry of new tokens into paged caches, page copies.
#include "kernels.hpp"
#include "paged.hpp"

namespace mfh {
namespace {

constexpr int kBlock = 256;

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1)
        v += __shfl_xor(v, offset, 64);
    return v;
}

// ---- rotation table ------------------------------------------------------

// Angle per position of pair c of dim / 2, in 64 bits: theta^(-2c / dim),
// stretched by the rule.
__device__ double frequency(uint32_t c, uint32_t dim, const RotationRule &r)
{
    double theta = r.theta;
    if (r.kind == MFH_ROPE_NTK)
        theta *= pow(r.factor, double(dim) / (double(dim) - 2.0));
    const double f = pow(theta, -2.0 * double(c) / double(dim));
    constexpr double kTurn = 6.283185307179586476925;
    if (r.kind == MFH_ROPE_LINEAR)
        return f / r.factor;
    if (r.kind == MFH_ROPE_WAVELENGTH) {
        const double turns = r.original * f / kTurn;  // in the original context
        const double keep = fmin(fmax((turns - r.low) / (r.high - r.low), 0.0), 1.0);
        return f * (keep + (1.0 - keep) / r.factor);
    }
    if (r.kind == MFH_ROPE_YARN) {
        // The pair number that turns n times in the original context.
        const double per = double(dim) / (2.0 * log(theta));
        const double first = fmax(floor(per * log(r.original / (kTurn * r.high))), 0.0);
        const double last = fmin(ceil(per * log(r.original / (kTurn * r.low))), double(dim) - 1.0);
        const double stretch =
            fmin(fmax((double(c) - first) / (last > first ? last - first : 0.001), 0.0), 1.0);
        return f * (1.0 - stretch + stretch / r.factor);
    }
    return f;
}

// One thread per element pair: row p holds m cos(p f_c) in column c and
// m sin(p f_c) in column dim / 2 + c.  Frequencies, angles and their sine and
// cosine are 64-bit (an f32 angle of position 10^5 is off by up to 2^-8), each
// value is rounded once.
__global__ __launch_bounds__(kBlock) void rotation_table_kernel(float *__restrict__ table,
                                                                uint64_t positions, uint32_t dim,
                                                                RotationRule rule)
{
    const uint32_t pairs = dim / 2;
    const uint64_t total = positions * pairs;
    const uint64_t stride = uint64_t(gridDim.x) * kBlock;
    for (uint64_t i = uint64_t(blockIdx.x) * kBlock + threadIdx.x; i < total; i += stride) {
        const uint64_t p = i / pairs;
        const uint32_t c = uint32_t(i - p * pairs);
        double sine, cosine;
        sincos(double(p) * frequency(c, dim, rule), &sine, &cosine);
        table[p * dim + c] = float(rule.magnitude * cosine);
        table[p * dim + pairs + c] = float(rule.magnitude * sine);
    }
}

// ---- new tokens into the caches --------------------------------------------

__device__ __forceinline__ void store(void *pages, bool half, uint64_t at, float v)
{
    if (half)
        static_cast<_Float16 *>(pages)[at] = to_half(v);
    else
        static_cast<float *>(pages)[at] = v;
}

// One wave per (token, head): query heads, then key heads, then value heads.
// y = x / sqrt(mean(x^2) + epsilon) * w, then of each rotated pair (a, b) of
// the first rotary_dim columns (a cos - b sin, b cos + a sin); columns behind
// them stay.  Sums of squares are f32.
__global__ __launch_bounds__(kBlock) void paged_rope_kernel(PagedRope p)
{
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t kv = p.shape.kv_heads, d = p.shape.head_dim, pairs = p.rotary_dim / 2;
    const uint32_t heads = p.query_heads + 2 * kv;
    const uint64_t waves = uint64_t(gridDim.x) * (kBlock / 64), segments = p.tokens * heads;
    for (uint64_t s = uint64_t(blockIdx.x) * (kBlock / 64) + (threadIdx.x >> 6); s < segments;
         s += waves) {
        const uint64_t token = s / heads;
        const uint32_t head = uint32_t(s - token * heads);
        const bool is_query = head < p.query_heads;
        const bool is_value = head >= p.query_heads + kv;
        const uint32_t h = is_query ? head : is_value ? head - p.query_heads - kv
                                                      : head - p.query_heads;
        const float position = p.positions[token];
        const float sequence = p.sequences ? p.sequences[token] : float(token);
        // The page that the token enters; every head of the token agrees.
        bool ok = valid_index(position, p.rotation_rows) &&
                  valid_index(sequence, p.sequence_count);
        const uint32_t at = ok ? uint32_t(position) : 0;
        ok = ok && (at >> p.shape.page_shift) < p.max_pages;
        float page = 0.0f;
        if (ok) {
            page = p.tables[uint64_t(uint32_t(sequence)) * p.max_pages +
                            (at >> p.shape.page_shift)];
            ok = valid_index(page, p.shape.pages);
        }
        const float *in = (is_query ? p.query : is_value ? p.value : p.key) +
                          (token * (is_query ? p.query_heads : kv) + h) * uint64_t(d);
        float *out = p.query_out + (token * p.query_heads + h) * uint64_t(d);
        if (!ok) {
            // Nothing enters the caches; the query row says so.
            if (is_query)
                for (uint32_t c = lane; c < d; c += 64)
                    out[c] = __builtin_nanf("");
            continue;
        }
        const uint64_t row = uint64_t(uint32_t(page)) * p.shape.stride() +
                             ((uint64_t(h) << p.shape.page_shift) +
                              (at & (p.shape.page_size() - 1))) * d;
        if (is_value) {
            for (uint32_t c = lane; c < d; c += 64)
                store(p.value_pages, p.shape.half, row + c, in[c]);
            continue;
        }
        const float *weight = is_query ? p.query_weight : p.key_weight;
        float reciprocal = 1.0f;
        if (weight) {
            float squares = 0.0f;
            for (uint32_t c = lane; c < d; c += 64)
                squares += in[c] * in[c];
            reciprocal = 1.0f / sqrtf(wave_sum(squares) / float(d) + p.epsilon);
        }
        const auto normed = [&](uint32_t c) {
            return weight ? in[c] * reciprocal * weight[c] : in[c];
        };
        const auto put = [&](uint32_t c, float v) {
            if (is_query)
                out[c] = v;
            else
                store(p.key_pages, p.shape.half, row + c, v);
        };
        const float *turn = p.rotation + uint64_t(at) * p.rotary_dim;
        for (uint32_t c = lane; c < pairs; c += 64) {
            const uint32_t first = p.interleaved ? 2 * c : c;
            const uint32_t second = p.interleaved ? 2 * c + 1 : pairs + c;
            const float a = normed(first), b = normed(second);
            const float cosine = turn[c], sine = turn[pairs + c];
            put(first, a * cosine - b * sine);
            put(second, b * cosine + a * sine);
        }
        for (uint32_t c = 2 * pairs + lane; c < d; c += 64)
            put(c, normed(c));
    }
}

// ---- page copies ---------------------------------------------------------------

// Block (part, pair, buffer) copies a part of one page.  The host has checked
// that no page is written twice, and none written that is read.
constexpr uint64_t kCopyPart = 8192;  // elements of a block

__global__ __launch_bounds__(kBlock) void copy_pages_kernel(PageCopy c)
{
    const uint32_t pair = blockIdx.y, buffer = blockIdx.z;
    const uint64_t from = c.from_page[pair] * c.elements, to = c.to_page[pair] * c.elements;
    const uint64_t begin = blockIdx.x * kCopyPart;
    const uint64_t end = begin + kCopyPart < c.elements ? begin + kCopyPart : c.elements;
    const bool from_half = c.from_half[buffer];
    for (uint64_t i = begin + threadIdx.x; i < end; i += kBlock) {
        const float v = from_half
                            ? float(static_cast<const _Float16 *>(c.from[buffer])[from + i])
                            : static_cast<const float *>(c.from[buffer])[from + i];
        store(c.to[buffer], c.to_half[buffer], to + i, v);
    }
}

unsigned grid_for(uint64_t count, uint64_t per_block)
{
    const uint64_t blocks = (count + per_block - 1) / per_block;
    return unsigned(blocks < 262144 ? (blocks ? blocks : 1) : 262144);
}

}  // namespace

void launch_scaled_rotation_table(hipStream_t stream, float *table, uint64_t positions,
                                  uint32_t dim, const RotationRule &rule)
{
    if (!positions || !dim)
        return;
    rotation_table_kernel<<<grid_for(positions * (dim / 2), kBlock), kBlock, 0, stream>>>(
        table, positions, dim, rule);
}

void launch_paged_qk_norm_rope(hipStream_t stream, const PagedRope &p)
{
    const uint64_t segments = p.tokens * (p.query_heads + 2 * uint64_t(p.shape.kv_heads));
    if (!segments)
        return;
    paged_rope_kernel<<<grid_for(segments, kBlock / 64), kBlock, 0, stream>>>(p);
}

void launch_copy_pages(hipStream_t stream, const PageCopy &c)
{
    const uint64_t parts = (c.elements + kCopyPart - 1) / kCopyPart;
    copy_pages_kernel<<<dim3(unsigned(parts), c.pairs, c.buffers), kBlock, 0, stream>>>(c);
}

}  // namespace mfh
