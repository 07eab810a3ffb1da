// Drafted trees: their layout, the settling of what was accepted, and the entry of tokens
// into latent caches.
#include "draft.hpp"
#include "kernels.hpp"

namespace mfh {
namespace {

constexpr int kBlock = 256;

// ---- layout ----------------------------------------------------------------

// Block s lays out the run of sequence s, block `sequences` marks the tokens in no run.
// A token's ancestors have falling numbers, so one walk writes its mask from the last
// word to the first.
constexpr uint32_t kLayoutParents = 4096;  // of a run, held in LDS

__global__ __launch_bounds__(kBlock) void draft_layout_kernel(DraftLayout p)
{
    __shared__ float held[kLayoutParents];
    const uint32_t s = blockIdx.x;
    const auto unset = [&](uint32_t t) {
        p.sequences[t] = p.positions[t] = p.places[t] = -1.0f;
        for (uint32_t b = 0; b < p.mask_bytes; ++b)
            p.mask[uint64_t(t) * p.mask_bytes + b] = 0;
    };
    if (s == p.runs.sequences) {
        // The list's first and last valid entry.
        uint32_t first = p.runs.tokens, last = p.runs.tokens;
        for (uint32_t i = 0; i < p.runs.sequences; ++i) {
            RunBounds b;
            if (!valid_bounds(p.runs, i, b))
                break;
            if (i == 0)
                first = b.begin;
            last = b.end;
        }
        for (uint32_t t = threadIdx.x; t < p.runs.tokens; t += kBlock)
            if (t < first || t >= last)
                unset(t);
        return;
    }
    const RunBounds run = run_of(p.runs, s);
    const uint32_t n = run.end - run.begin;
    const float length = p.runs.lengths[s];
    const bool fits = valid_length(length, n, 1u << 24);
    if (p.parents) {
        for (uint32_t i = threadIdx.x; i < n && i < kLayoutParents; i += kBlock)
            held[i] = p.parents[run.begin + i];
        __syncthreads();
    }
    // -2: a bad one.
    const auto parent_of = [&](uint32_t i) {
        if (!p.parents)
            return int(i) - 1;
        const float v = i < kLayoutParents ? held[i] : p.parents[run.begin + i];
        return v == -1.0f ? -1 : valid_index(v, i) ? int(v) : -2;
    };
    for (uint32_t i = threadIdx.x; i < n; i += kBlock) {
        const uint32_t t = run.begin + i;
        uint32_t depth = 0;
        int at = int(i);
        while ((at = parent_of(uint32_t(at))) >= 0)
            ++depth;
        if (at == -2 || !fits || (p.mask && i >= 8ull * p.mask_bytes)) {
            unset(t);
            continue;
        }
        p.sequences[t] = float(s);
        p.positions[t] = length + float(depth);
        p.places[t] = length + float(i);
        uint8_t *row = p.mask + uint64_t(t) * p.mask_bytes;
        at = int(i);
        for (int b = int(p.mask_bytes) - 1; b >= 0; --b) {
            uint32_t bits = 0;
            for (; at >= 8 * b; at = parent_of(uint32_t(at)))
                bits |= 1u << (at & 7);
            row[b] = uint8_t(bits);
        }
    }
}

// ---- settling ----------------------------------------------------------------

// Block (s, b, part) walks the tree of sequence s and moves a part of its accepted rows
// in buffer b: a thread has one unit (16, 4 or 2 bytes of a head's row) of every
// row and moves them in the path's order, whose sources never lie before its targets.
template <typename T>
__device__ __forceinline__ void move_rows(const Settle &p, uint32_t b, const uint64_t *from,
                                          uint32_t count)
{
    constexpr uint32_t HELD = 8;
    const uint32_t units = p.row_bytes[b] / uint32_t(sizeof(T)), heads = p.heads[b];
    const uint64_t unit = uint64_t(blockIdx.z) * kBlock + threadIdx.x;
    if (unit >= uint64_t(heads) * units)
        return;
    const uint32_t head = uint32_t(unit / units), column = uint32_t(unit - uint64_t(head) * units);
    T *pages = static_cast<T *>(p.buffer[b]);
    // A row's unit: rows are counted through pages of one head.
    const auto at = [&](uint64_t row) {
        const uint64_t page = row >> p.page_shift, slot = row & ((1u << p.page_shift) - 1);
        return pages + (((page * heads + head) << p.page_shift) + slot) * units + column;
    };
    const uint64_t *to = from + kSettleColumns;
    for (uint32_t k = 0; k < count; k += HELD) {
        T held[HELD];
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i)
            held[i] = *at(from[k + i < count ? k + i : count - 1]);
#pragma unroll
        for (uint32_t i = 0; i < HELD; ++i)
            if (k + i < count && from[k + i] != to[k + i])
                *at(to[k + i]) = held[i];
    }
}

__global__ __launch_bounds__(kBlock) void settle_kernel(Settle p)
{
    __shared__ uint64_t rows[2 * kSettleColumns];  // sources, then targets
    __shared__ float chosen[kSettleColumns];
    __shared__ int bad;
    const uint32_t s = blockIdx.x, lane = threadIdx.x & 63;
    const RunBounds run = run_of(p.runs, s);
    const uint32_t n = run.end - run.begin;
    const float length = p.runs.lengths[s];
    const bool fits = n && valid_length(length, n, 1u << 24);
    uint32_t count = 0;
    if (threadIdx.x == 0)
        bad = 0;
    if (fits) {
        // Every wave walks; the first writes the path down.
        uint32_t at = 0;
        while (true) {
            const float choice = p.choices[run.begin + at];
            if (threadIdx.x == 0) {
                rows[count] = at;
                chosen[count] = choice;
            }
            if (++count == p.columns)
                break;
            uint32_t child = n;
            for (uint32_t base = at + 1; base < n; base += 64) {
                const uint32_t i = base + lane, t = run.begin + (i < n ? i : n - 1);
                const float parent = p.parents ? p.parents[t] : float(int(i) - 1);
                const uint64_t found =
                    __ballot(i < n && parent == float(at) && p.drafted[t] == choice);
                if (found) {
                    child = base + uint32_t(__builtin_ctzll(found));
                    break;
                }
            }
            if (child == n)
                break;
            at = child;
        }
    }
    __syncthreads();
    const float *table = p.tables + uint64_t(s) * p.max_pages;
    const auto row_of = [&](uint32_t place) {
        const uint32_t column = place >> p.page_shift;
        const float id = column < p.max_pages ? table[column] : -1.0f;
        if (!valid_index(id, p.pages)) {
            bad = 1;
            return uint64_t(0);
        }
        return (uint64_t(uint32_t(id)) << p.page_shift) + (place & ((1u << p.page_shift) - 1));
    };
    for (uint32_t k = threadIdx.x; p.path_pages && k < count; k += kBlock) {
        const uint32_t base = uint32_t(length);
        rows[kSettleColumns + k] = row_of(base + k);
        rows[k] = row_of(base + uint32_t(rows[k]));
    }
    __syncthreads();
    const bool good = !bad && (fits || !n);
    if (p.emitted && blockIdx.y == 0 && blockIdx.z == 0) {
        const float nan = __builtin_nanf("");
        for (uint32_t k = threadIdx.x; k < p.columns; k += kBlock)
            p.emitted[uint64_t(s) * p.columns + k] = !good ? nan : k < count ? chosen[k] : -1.0f;
        if (threadIdx.x == 0) {
            p.counts[s] = good ? float(count) : nan;
            p.next[s] = !good ? nan : count ? chosen[count - 1] : -1.0f;
        }
    }
    const uint32_t b = blockIdx.y;
    if (!good || !count || b >= p.buffers)
        return;
    if (p.row_bytes[b] % 16 == 0)
        move_rows<uint4>(p, b, rows, count);
    else if (p.row_bytes[b] % 4 == 0)
        move_rows<uint32_t>(p, b, rows, count);
    else
        move_rows<uint16_t>(p, b, rows, count);
}

// ---- new tokens into latent caches --------------------------------------------

// Block t takes token t: the sum of its latent's squares over the block, then latent,
// key and queries, each pair of columns by a thread.
__global__ __launch_bounds__(kBlock) void latent_append_kernel(LatentAppend p)
{
    __shared__ float sums[kBlock / 64];
    const uint64_t t = blockIdx.x;
    const float nan = __builtin_nanf("");
    const uint32_t pairs = p.rope / 2, width = p.rank + p.rope;
    const float position = p.positions[t];
    const float place = p.places ? p.places[t] : position;
    const float sequence = p.sequences ? p.sequences[t] : float(t);
    bool good = valid_index(position, p.rotation_rows) && valid_index(place, 1u << 24) &&
                valid_index(sequence, p.sequence_count);
    uint64_t row = 0;
    if (good) {
        const uint32_t at = uint32_t(place), column = at >> p.shape.page_shift;
        const float page =
            column < p.max_pages
                ? p.tables[uint64_t(uint32_t(sequence)) * p.max_pages + column]
                : -1.0f;
        good = valid_index(page, p.shape.pages);
        row = good ? uint64_t(uint32_t(page)) * p.shape.stride() +
                         uint64_t(at & (p.shape.page_size() - 1)) * width
                   : 0;
    }
    if (!good) {
        for (uint32_t c = threadIdx.x; c < p.query_heads * p.rope; c += kBlock)
            p.query_out[t * p.query_heads * p.rope + c] = nan;
        return;
    }
    const auto store = [&](uint32_t c, float v) {
        if (p.shape.half)
            static_cast<_Float16 *>(p.pages)[row + c] = to_half(v);
        else
            static_cast<float *>(p.pages)[row + c] = v;
    };
    const float *latent = p.latent + t * p.rank;
    float reciprocal = 1.0f;
    if (p.weight) {
        float squares = 0.0f;
        for (uint32_t c = threadIdx.x; c < p.rank; c += kBlock)
            squares += latent[c] * latent[c];
#pragma unroll
        for (int offset = 32; offset > 0; offset >>= 1)
            squares += __shfl_xor(squares, offset, 64);
        if ((threadIdx.x & 63) == 0)
            sums[threadIdx.x >> 6] = squares;
        __syncthreads();
        squares = 0.0f;
#pragma unroll
        for (int w = 0; w < kBlock / 64; ++w)
            squares += sums[w];
        reciprocal = 1.0f / sqrtf(squares / float(p.rank) + p.epsilon);
    }
    for (uint32_t c = threadIdx.x; c < p.rank; c += kBlock)
        store(c, p.weight ? latent[c] * reciprocal * p.weight[c] : latent[c]);
    const float *turn = p.rotation + uint64_t(uint32_t(position)) * p.rope;
    const auto turned = [&](const float *in, uint32_t c, auto put) {
        const uint32_t first = p.interleaved ? 2 * c : c;
        const uint32_t second = p.interleaved ? 2 * c + 1 : pairs + c;
        const float a = in[first], b = in[second], cosine = turn[c], sine = turn[pairs + c];
        put(first, a * cosine - b * sine);
        put(second, b * cosine + a * sine);
    };
    for (uint32_t c = threadIdx.x; c < pairs; c += kBlock)
        turned(p.key + t * p.rope, c, [&](uint32_t at, float v) { store(p.rank + at, v); });
    for (uint32_t i = threadIdx.x; i < p.query_heads * pairs; i += kBlock) {
        const uint32_t head = i / pairs;
        const uint64_t base = (t * p.query_heads + head) * p.rope;
        turned(p.query + base, i - head * pairs,
               [&](uint32_t at, float v) { p.query_out[base + at] = v; });
    }
}

}  // namespace

void launch_draft_layout(hipStream_t stream, const DraftLayout &p)
{
    if (p.runs.tokens)
        draft_layout_kernel<<<p.runs.sequences + 1, kBlock, 0, stream>>>(p);
}

void launch_settle(hipStream_t stream, const Settle &p)
{
    if (!p.runs.sequences)
        return;
    uint64_t most = 1;
    for (uint32_t b = 0; b < p.buffers; ++b) {
        const uint32_t bytes = p.row_bytes[b];
        const uint64_t units = uint64_t(p.heads[b]) * (bytes % 16 == 0 ? bytes / 16
                                                       : bytes % 4 == 0 ? bytes / 4
                                                                        : bytes / 2);
        most = units > most ? units : most;
    }
    const dim3 grid(p.runs.sequences, p.buffers ? p.buffers : 1,
                    unsigned((most + kBlock - 1) / kBlock));
    settle_kernel<<<grid, kBlock, 0, stream>>>(p);
}

void launch_latent_append(hipStream_t stream, const LatentAppend &p)
{
    if (p.tokens)
        latent_append_kernel<<<p.tokens, kBlock, 0, stream>>>(p);
}

}  // namespace mfh
