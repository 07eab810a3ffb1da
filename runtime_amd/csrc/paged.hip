// Rotation tables, the entry of new tokens into paged caches, page copies.
#include "kernels.hpp"
#include "paged.hpp"

namespace mfh {
namespace {

constexpr int kBlock = 256;

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

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

// Row p holds m cos(p f_c) in column c and m sin(p f_c) in column dim / 2 + c.
// Frequencies, angles and their sine and cosine are 64-bit (an f32 angle of
// position 10^5 is off by up to 2^-8), each value is rounded once.  A thread
// forms the first of `run` positions' values and turns it by f_c for each
// further one (64-bit products: 2^-52 a step), so that the one power and sine
// are shared; threads of a wave are neighbouring columns, so a wave writes whole
// rows.  Bound by the writes: 131072 positions of 128 columns (67 MB) take 13.7
// us, 4.9 TB/s (a sine for every value: 204 us); 2048 of 64, 3.5 us, a launch.
__global__ __launch_bounds__(kBlock) void rotation_table_kernel(float *__restrict__ table,
                                                                uint64_t positions, uint32_t dim,
                                                                uint32_t run, RotationRule rule)
{
    const uint32_t pairs = dim / 2;
    const uint64_t i = uint64_t(blockIdx.x) * kBlock + threadIdx.x;
    const uint64_t first = i / pairs * run;
    const uint32_t c = uint32_t(i % pairs);
    if (first >= positions)
        return;
    const double f = frequency(c, dim, rule);
    double sine, cosine, step_sine, step_cosine;
    sincos(double(first) * f, &sine, &cosine);
    sincos(f, &step_sine, &step_cosine);
    float *at = table + first * dim + c;
    const uint64_t left = positions - first;
    const uint32_t count = left < run ? uint32_t(left) : run;
    for (uint32_t n = 0; n < count; ++n, at += dim) {
        at[0] = float(rule.magnitude * cosine);
        at[pairs] = float(rule.magnitude * sine);
        const double turned = cosine * step_cosine - sine * step_sine;
        sine = sine * step_cosine + cosine * step_sine;
        cosine = turned;
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

// Where a token goes: false where its position, its sequence or its page is none.
struct Place {
    uint32_t position;
    uint64_t row;  // element of its page's first head
};
__device__ __forceinline__ bool place_of(const PagedRope &p, uint64_t token, Place &place)
{
    const float position = p.positions[token];
    const float sequence = p.sequences ? p.sequences[token] : float(token);
    if (!valid_index(position, p.rotation_rows) || !valid_index(sequence, p.sequence_count))
        return false;
    place.position = uint32_t(position);
    uint32_t at = place.position;
    if (p.places) {
        const float given = p.places[token];
        if (!valid_index(given, 1u << 24))
            return false;
        at = uint32_t(given);
    }
    const uint32_t column = at >> p.shape.page_shift;
    if (column >= p.max_pages)
        return false;
    const float page = p.tables[uint64_t(uint32_t(sequence)) * p.max_pages + column];
    if (!valid_index(page, p.shape.pages))
        return false;
    place.row = uint64_t(uint32_t(page)) * p.shape.stride() +
                uint64_t(at & (p.shape.page_size() - 1)) * p.shape.head_dim;
    return true;
}

// y = x / sqrt(mean(x^2) + epsilon) * w, then of each rotated pair (a, b) of
// the first rotary_dim columns (a cos - b sin, b cos + a sin); columns behind
// them stay.  Sums of squares are f32.  Heads of a token are its query heads,
// then key heads, then value heads.

// Any shape: one wave per (token, head).  4099 tokens of 32 + 8 + 8 heads of 128
// into binary16 pages took 134 us with it, where the kernel below takes 37.8.
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
        const float *in = (is_query ? p.query : is_value ? p.value : p.key) +
                          (token * (is_query ? p.query_heads : kv) + h) * uint64_t(d);
        float *out = p.query_out + (token * p.query_heads + h) * uint64_t(d);
        Place place;
        if (!place_of(p, token, place)) {
            // Nothing enters the caches; the query row says so.
            if (is_query)
                for (uint32_t c = lane; c < d; c += 64)
                    out[c] = __builtin_nanf("");
            continue;
        }
        const uint64_t row = place.row + (uint64_t(h) << p.shape.page_shift) * d;
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
        const float *turn = p.rotation + uint64_t(place.position) * p.rotary_dim;
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

// Heads of whole float4s, up to 256 wide: LANES lanes (the power of two that
// holds them) take a head, four columns each, kHeads heads at a time, and the
// token's place and coefficients once.  Pairs across the halves are exchanged
// between lanes.  `parts` blocks share a token.  Bound by the bytes: those 4099
// tokens move 185 MB at 4.9 TB/s, what a large copy reaches; one token takes 4.0
// us, a launch and three dependent reads (position, table, coefficients).
constexpr int kHeads = 4;

template <int LANES>
__global__ __launch_bounds__(kBlock) void paged_rope_vector_kernel(PagedRope p, uint32_t parts)
{
    constexpr uint32_t GROUPS = kBlock / LANES;
    const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const uint32_t kv = p.shape.kv_heads, d = p.shape.head_dim, pairs = p.rotary_dim / 2;
    const uint32_t heads = p.query_heads + 2 * kv;
    const uint64_t token = blockIdx.x / parts;
    const uint32_t part = blockIdx.x % parts, step = parts * GROUPS;
    const uint32_t column = 4 * lane;
    const bool inside = column < d;
    const v4f zero = {0, 0, 0, 0};
    const auto source = [&](uint32_t head) {
        if (head < p.query_heads)
            return p.query + (token * p.query_heads + head) * d;
        head -= p.query_heads;
        return head < kv ? p.key + (token * kv + head) * d : p.value + (token * kv + head - kv) * d;
    };
    const auto load = [&](v4f (&x)[kHeads], uint32_t first) {
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const uint32_t head = first + i * step;
            x[i] = inside && head < heads ? __builtin_nontemporal_load(reinterpret_cast<const v4f *>(
                                                source(head) + column))
                                          : zero;
        }
    };
    uint32_t first = part * GROUPS + group;
    v4f x[kHeads];
    load(x, first);
    const v4f query_weight = inside && p.query_weight
                                 ? *reinterpret_cast<const v4f *>(p.query_weight + column)
                                 : zero;
    const v4f key_weight =
        inside && p.key_weight ? *reinterpret_cast<const v4f *>(p.key_weight + column) : zero;
    Place place;
    const bool placed = place_of(p, token, place);
    // The lane's coefficients: cosines, and sines with the sign that its
    // columns take them with.
    const bool turned = placed && column < 2 * pairs;
    v4f cosine = {1, 1, 1, 1}, sine = zero;
    const bool upper = !p.interleaved && column >= pairs;
    if (turned) {
        const float *turn = p.rotation + uint64_t(place.position) * p.rotary_dim;
        if (p.interleaved) {
            const v2f c = *reinterpret_cast<const v2f *>(turn + column / 2);
            const v2f s = *reinterpret_cast<const v2f *>(turn + pairs + column / 2);
            cosine = v4f{c[0], c[0], c[1], c[1]};
            sine = v4f{-s[0], s[0], -s[1], s[1]};
        } else {
            const uint32_t at = upper ? column - pairs : column;
            cosine = *reinterpret_cast<const v4f *>(turn + at);
            sine = *reinterpret_cast<const v4f *>(turn + pairs + at);
            if (!upper)
                sine = -sine;
        }
    }
    // The lane that holds the other half's columns.
    const uint32_t other = !turned ? lane : upper ? lane - pairs / 4 : lane + pairs / 4;
    for (; first < heads; first += kHeads * step) {
        v4f y[kHeads];
#pragma unroll
        for (int i = 0; i < kHeads; ++i)
            y[i] = x[i];
        if (first + kHeads * step < heads)
            load(x, first + kHeads * step);
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            // Every lane of a group has the same head, but not of the wave:
            // the exchanges run for all.
            const uint32_t head = first + i * step;
            const bool is_query = head < p.query_heads, is_value = head >= p.query_heads + kv;
            v4f v = y[i];
            if (p.query_weight) {
                float squares = v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3];
#pragma unroll
                for (int offset = LANES / 2; offset > 0; offset >>= 1)
                    squares += __shfl_xor(squares, offset, LANES);
                const float reciprocal = 1.0f / sqrtf(squares / float(d) + p.epsilon);
                if (!is_value)
                    v = v * reciprocal * (is_query ? query_weight : key_weight);
            }
            v4f across;
            if (p.interleaved) {
                across = v4f{v[1], v[0], v[3], v[2]};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    across[e] = __shfl(v[e], int(other), LANES);
            }
            if (!is_value && turned)
                v = v * cosine + across * sine;
            if (!inside || head >= heads)
                continue;
            if (is_query) {
                const float nan = __builtin_nanf("");
                *reinterpret_cast<v4f *>(p.query_out + (token * p.query_heads + head) * d + column) =
                    placed ? v : v4f{nan, nan, nan, nan};
            } else if (placed) {
                const uint32_t h = head - p.query_heads - (is_value ? kv : 0);
                const uint64_t at =
                    place.row + (uint64_t(h) << p.shape.page_shift) * d + column;
                void *pages = is_value ? p.value_pages : p.key_pages;
                if (p.shape.half)
                    *reinterpret_cast<v4h *>(static_cast<_Float16 *>(pages) + at) =
                        v4h{to_half(v[0]), to_half(v[1]), to_half(v[2]), to_half(v[3])};
                else
                    *reinterpret_cast<v4f *>(static_cast<float *>(pages) + at) = v;
            }
        }
    }
}

// ---- page copies ---------------------------------------------------------------

// Block (part, pair, buffer) copies a part of one page, 16 bytes a load, all of a
// thread's in flight at once.  The host has checked that no page is written
// twice, and none written that is read.  Page sizes are multiples of 8 rows, so a
// page is whole 8-element pieces.  Bound by the bytes: 599 pages of 16 KB in 12
// buffers (236 MB read and written) take 50 us, 4.7 TB/s, in two launches (an element a
// thread took 124); one page of 12 buffers 3.4 us, a
// launch.
constexpr uint32_t kCopyPieces = 4;  // of 8 elements, of a thread
constexpr uint64_t kCopyPart = 8 * kCopyPieces * kBlock;

template <bool FROM_HALF, bool TO_HALF>
__device__ __forceinline__ void copy_part(const void *from, void *to, uint64_t elements,
                                          uint64_t begin)
{
    constexpr int IN = FROM_HALF ? 1 : 2;  // 16-byte loads of a piece
    v4u piece[kCopyPieces][IN];
    const v4u *source = static_cast<const v4u *>(from);
    v4u *target = static_cast<v4u *>(to);
    const uint64_t pieces = elements / 8, first = begin / 8 + threadIdx.x;
#pragma unroll
    for (uint32_t i = 0; i < kCopyPieces; ++i)
#pragma unroll
        for (int e = 0; e < IN; ++e)
            if (first + i * kBlock < pieces)
                piece[i][e] = __builtin_nontemporal_load(&source[(first + i * kBlock) * IN + e]);
#pragma unroll
    for (uint32_t i = 0; i < kCopyPieces; ++i) {
        const uint64_t at = first + i * kBlock;
        if (at >= pieces)
            break;
        if constexpr (FROM_HALF == TO_HALF) {
#pragma unroll
            for (int e = 0; e < IN; ++e)
                target[at * IN + e] = piece[i][e];
        } else if constexpr (TO_HALF) {
            v8h out;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                out[e] = to_half(__uint_as_float(piece[i][e / 4][e % 4]));
            target[at] = __builtin_bit_cast(v4u, out);
        } else {
            const v8h in = __builtin_bit_cast(v8h, piece[i][0]);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                target[2 * at + e] = __builtin_bit_cast(
                    v4u, v4f{float(in[4 * e]), float(in[4 * e + 1]), float(in[4 * e + 2]),
                             float(in[4 * e + 3])});
        }
    }
}

template <uint32_t PAIRS>
__global__ __launch_bounds__(kBlock) void copy_pages_kernel(PageCopy<PAIRS> c)
{
    const uint32_t pair = blockIdx.y, buffer = blockIdx.z;
    const bool from_half = c.from_half[buffer], to_half = c.to_half[buffer];
    const char *from = static_cast<const char *>(c.from[buffer]) +
                       c.from_page[pair] * c.elements * (from_half ? 2 : 4);
    char *to = static_cast<char *>(c.to[buffer]) +
               c.to_page[pair] * c.elements * (to_half ? 2 : 4);
    const uint64_t begin = blockIdx.x * kCopyPart;
    if (from_half && to_half)
        copy_part<true, true>(from, to, c.elements, begin);
    else if (from_half)
        copy_part<true, false>(from, to, c.elements, begin);
    else if (to_half)
        copy_part<false, true>(from, to, c.elements, begin);
    else
        copy_part<false, false>(from, to, c.elements, begin);
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
    // Threads for the whole device (65536) before longer runs.
    const uint64_t pairs = dim / 2, each = positions * pairs / 65536;
    const uint32_t run = each < 1 ? 1 : each > 32 ? 32 : uint32_t(each);
    const uint64_t threads = (positions + run - 1) / run * pairs;
    rotation_table_kernel<<<unsigned((threads + kBlock - 1) / kBlock), kBlock, 0, stream>>>(
        table, positions, dim, run, rule);
}

void launch_paged_qk_norm_rope(hipStream_t stream, const PagedRope &p)
{
    const uint32_t heads = p.query_heads + 2 * p.shape.kv_heads;
    const uint64_t segments = p.tokens * heads;
    if (!segments)
        return;
    // float4 columns and coefficients (whole float4s in each half, or two pairs).
    const uint32_t d = p.shape.head_dim;
    if (d % 4 == 0 && d <= 256 && p.rotary_dim % (p.interleaved ? 4 : 8) == 0) {
        const uint32_t lanes = d <= 64 ? 16 : d <= 128 ? 32 : 64, groups = kBlock / lanes;
        // Blocks for the whole device before longer runs of heads.
        const uint32_t most = (heads + groups - 1) / groups;
        const uint64_t wanted = p.tokens < 2048 ? 2048 / p.tokens : 1;
        const uint32_t parts = wanted < most ? uint32_t(wanted) : most;
        const auto kernel = lanes == 16   ? paged_rope_vector_kernel<16>
                            : lanes == 32 ? paged_rope_vector_kernel<32>
                                          : paged_rope_vector_kernel<64>;
        kernel<<<unsigned(p.tokens * parts), kBlock, 0, stream>>>(p, parts);
        return;
    }
    paged_rope_kernel<<<grid_for(segments, kBlock / 64), kBlock, 0, stream>>>(p);
}

template <uint32_t PAIRS>
void launch_copy_pages(hipStream_t stream, const PageCopy<PAIRS> &c)
{
    const uint64_t parts = (c.elements + kCopyPart - 1) / kCopyPart;
    copy_pages_kernel<PAIRS><<<dim3(unsigned(parts), c.pairs, c.buffers), kBlock, 0, stream>>>(c);
}
template void launch_copy_pages(hipStream_t, const PageCopy<kCopyPairs> &);
template void launch_copy_pages(hipStream_t, const PageCopy<kCopyFewPairs> &);

}  // namespace mfh
