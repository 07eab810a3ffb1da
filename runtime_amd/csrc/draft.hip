// Drafted trees: their layout, the settling of what was accepted, and the entry of tokens
// into latent caches.
#include "draft.hpp"
#include "kernels.hpp"

namespace mfh {
namespace {

constexpr int kBlock = 256;

// ---- layout ----------------------------------------------------------------

// Block s lays out the run of sequence s, block `sequences` marks the tokens in no run.  Runs
// of up to 64 tokens are a wave's lanes, which form their ancestors in six steps: after k of
// them a lane knows 2^k generations, and where the next one is.  Longer runs go 64 tokens at
// a time, whose ancestors before them are those of one earlier token: its depth and its
// mask row are read back.  Bound by the launch and three dependent reads: 16 tokens 4.5
// us, 96 sequences of 8 to 64 the same.  Of longer runs by the steps of 64, which follow one
// another: 2048 tokens 26 us, 295 with their 512 KB of masks, 8192 97.

// The lane's ancestors among the wave's 64 tokens and itself; `good` where it and they are.
// `parent`: a lower lane, or -1.
__device__ __forceinline__ uint64_t lane_ancestors(uint32_t lane, int parent, bool &good)
{
    uint64_t seen = 1ull << lane;
#pragma unroll
    for (int step = 0; step < 6; ++step) {
        const int from = parent < 0 ? int(lane) : parent;
        const uint32_t low = __shfl(uint32_t(seen), from, 64);
        const uint32_t high = __shfl(uint32_t(seen >> 32), from, 64);
        const int far = __shfl(parent, from, 64);
        const bool sound = __shfl(int(good), from, 64);
        seen |= uint64_t(high) << 32 | low;
        good = good && sound;
        parent = parent < 0 ? parent : far;
    }
    return seen;
}

__global__ __launch_bounds__(kBlock) void draft_layout_kernel(DraftLayout p)
{
    __shared__ uint64_t seen_of[64];  // of a long run's 64 tokens
    __shared__ int root_of[64];
    const uint32_t s = blockIdx.x, lane = threadIdx.x & 63;
    const auto put = [&](uint32_t t, float sequence, float position, float place) {
        p.sequences[t] = sequence;
        p.positions[t] = position;
        p.places[t] = place;
    };
    const auto unset = [&](uint32_t t) {
        put(t, -1.0f, -1.0f, -1.0f);
        for (uint32_t b = 0; b < p.mask_bytes; ++b)
            p.mask[uint64_t(t) * p.mask_bytes + b] = 0;
    };
    if (s == p.runs.sequences) {
        // The list's first and last valid entry.
        uint32_t first = p.runs.tokens, last = p.runs.tokens;
        for (uint32_t base = 0; base < p.runs.sequences; base += 64) {
            RunBounds b;
            const uint32_t i = base + lane;
            const bool mine = i < p.runs.sequences;
            const bool ok = mine && valid_bounds(p.runs, i, b);
            const uint64_t wrong = __ballot(mine && !ok);
            const uint64_t good = wrong ? (wrong & -wrong) - 1 : __ballot(ok);
            if (good) {
                if (base == 0)
                    first = __shfl(b.begin, 0, 64);
                last = __shfl(b.end, 63 - __builtin_clzll(good), 64);
            }
            if (wrong)
                break;
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
    if (n <= 64) {
        if (threadIdx.x >= 64 || !n)
            return;
        const uint32_t t = run.begin + (lane < n ? lane : n - 1);
        int parent = int(lane) - 1;
        bool good = lane < n;
        if (p.parents) {
            const float v = p.parents[t];
            good = good && (v == -1.0f || valid_index(v, lane));
            parent = good ? int(v) : -1;
        }
        // A token past the mask's last bit has no place.
        good = good && (!p.mask || lane < 8ull * p.mask_bytes);
        const uint64_t seen = lane_ancestors(lane, parent, good);
        if (lane >= n)
            return;
        if (!good || !fits) {
            unset(t);
            return;
        }
        put(t, float(s), length + float(__popcll(seen) - 1), length + float(lane));
        uint8_t *row = p.mask + uint64_t(t) * p.mask_bytes;
        for (uint32_t b = 0; b < p.mask_bytes; ++b)
            row[b] = b < 8 ? uint8_t(seen >> 8 * b) : 0;
        return;
    }
    const auto barred = [&](uint32_t i) { return !fits || (p.mask && i >= 8ull * p.mask_bytes); };
    if (!p.parents) {
        for (uint32_t i = threadIdx.x; i < n; i += kBlock) {
            const uint32_t t = run.begin + i;
            if (barred(i)) {
                unset(t);
                continue;
            }
            put(t, float(s), length + float(i), length + float(i));
            uint8_t *row = p.mask + uint64_t(t) * p.mask_bytes;
            for (uint32_t b = 0; b < p.mask_bytes; ++b) {
                const int left = int(i) + 1 - 8 * int(b);
                row[b] = left >= 8 ? 0xff : left <= 0 ? 0 : uint8_t((1u << left) - 1);
            }
        }
        return;
    }
    for (uint32_t base = 0; base < n; base += 64) {
        if (threadIdx.x < 64) {
            const uint32_t i = base + lane, t = run.begin + (i < n ? i : n - 1);
            const float v = p.parents[t];
            bool good = i < n && !barred(i) && (v == -1.0f || valid_index(v, i));
            const int parent = good ? int(v) : -1;
            const bool inside = parent >= int(base);
            const uint64_t seen = lane_ancestors(lane, inside ? parent - int(base) : -1, good);
            // What the first of them follows, of an earlier 64.
            const int root = __shfl(inside ? -1 : parent, __builtin_ctzll(seen), 64);
            const float before = root < 0 ? length - 1.0f : p.positions[run.begin + root];
            good = good && (root < 0 || before >= 0.0f);
            if (i < n) {
                if (good)
                    put(t, float(s), before + float(__popcll(seen)), length + float(i));
                else
                    put(t, -1.0f, -1.0f, -1.0f);
            }
            seen_of[lane] = good ? seen : 0;
            root_of[lane] = good ? root : -1;
        }
        __syncthreads();
        // A wave a row; rows before this 64 are whole, and their bytes are.
        for (uint32_t r = threadIdx.x >> 6; p.mask && r < 64 && base + r < n; r += kBlock / 64) {
            const uint64_t seen = seen_of[r];
            const uint8_t *from = p.mask + uint64_t(run.begin + root_of[r]) * p.mask_bytes;
            uint8_t *row = p.mask + uint64_t(run.begin + base + r) * p.mask_bytes;
            for (uint32_t b = lane; b < p.mask_bytes; b += 64) {
                const uint32_t in = b - base / 8;  // of the 64 tokens' bytes
                row[b] = b < base / 8 ? (root_of[r] < 0 ? 0 : from[b])
                         : in < 8     ? uint8_t(seen >> 8 * in)
                                      : 0;
            }
        }
        __syncthreads();  // rows, positions and what the waves share
    }
}

// ---- settling ----------------------------------------------------------------

// Block (s, b, part) walks the tree of sequence s and moves a part of its accepted rows
// in buffer b: a thread has one unit (16, 4 or 2 bytes of a head's row) of every
// row and moves them in the path's order, whose sources never lie before its targets.
// Bound by dependent reads: the lists, a search of the run per accepted token, page ids,
// the rows.  12 buffers of 8 heads of 64: one run of 16 tokens, f32, 7.8 us a call, 96 of 4
// to 32, binary16, 8.7 to 9.9 (two cards).  Each block walks for itself: a launch between the walk and the
// moves would add its own latency.
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
                bool next = i < n && parent == float(at) && p.drafted[t] == choice;
                // A token without a place was not stored.
                if (p.places)
                    next = next && p.places[t] == length + float(i);
                const uint64_t found = __ballot(next);
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
    // The layout refuses a run whose first token follows another.
    if (threadIdx.x == kBlock - 1 && fits &&
        ((p.parents && p.parents[run.begin] != -1.0f) ||
         (p.places && p.places[run.begin] != length)))
        bad = 1;
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

// Block t takes token t: queries and key by V columns (and the V that they turn with) a
// thread, the latent's squares summed over the block, then the latent.  V is 4 where the
// widths allow, as it does everywhere but for odd ones.  Bound by the bytes: 4099 tokens of
// 32 heads, rank 512 and rope 64 (82 MB) 16.5 us, 5.0 TB/s (a column a thread 22.3); one
// token 4.9, a launch and its dependent reads.
template <int V>
__global__ __launch_bounds__(kBlock) void latent_append_kernel(LatentAppend p)
{
    typedef float piece __attribute__((ext_vector_type(V)));
    typedef _Float16 half_piece __attribute__((ext_vector_type(V)));
    __shared__ float sums[kBlock / 64];
    const uint64_t t = blockIdx.x;
    const uint32_t pairs = p.rope / 2, width = p.rank + p.rope;
    const uint32_t turns = pairs / V;  // of a head, V pairs each
    const auto load = [](const float *at) { return *reinterpret_cast<const piece *>(at); };
    // The first of a thread's loads go out before anything that they do not need.
    const float *latent = p.latent + t * p.rank;
    piece first = {};
    if (threadIdx.x * V < p.rank)
        first = load(latent + threadIdx.x * V);
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
            p.query_out[t * p.query_heads * p.rope + c] = __builtin_nanf("");
        return;
    }
    const auto store = [&](uint32_t c, piece v) {
        if (p.shape.half) {
            half_piece h;
#pragma unroll
            for (int e = 0; e < V; ++e)
                h[e] = to_half(v[e]);
            *reinterpret_cast<half_piece *>(static_cast<_Float16 *>(p.pages) + row + c) = h;
        } else {
            *reinterpret_cast<piece *>(static_cast<float *>(p.pages) + row + c) = v;
        }
    };
    const float *turn = p.rotation + uint64_t(uint32_t(position)) * p.rope;
    // V pairs of a head: the V columns from `at` on and those behind them (interleaved), or
    // half a head further.
    const auto turned = [&](const float *in, uint32_t c, auto put) {
        const piece cosine = load(turn + c), sine = load(turn + pairs + c);
        const uint32_t low = p.interleaved ? 2 * c : c, high = p.interleaved ? low + V : pairs + c;
        const piece x = load(in + low), y = load(in + high);
        piece a = x, b = y;
        if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                a[e] = 2 * e < V ? x[2 * e % V] : y[2 * e % V];
                b[e] = 2 * e + 1 < V ? x[(2 * e + 1) % V] : y[(2 * e + 1) % V];
            }
        }
        const piece u = a * cosine - b * sine, v = b * cosine + a * sine;
        piece to_low = u, to_high = v;
        if (p.interleaved) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                to_low[e] = e % 2 ? v[e / 2] : u[e / 2];
                to_high[e] = (V + e) % 2 ? v[(V + e) / 2] : u[(V + e) / 2];
            }
        }
        put(low, to_low);
        put(high, to_high);
    };
    for (uint32_t i = threadIdx.x; i < p.query_heads * turns; i += kBlock) {
        const uint32_t head = i / turns;
        const uint64_t base = (t * p.query_heads + head) * p.rope;
        turned(p.query + base, (i - head * turns) * V, [&](uint32_t at, piece v) {
            *reinterpret_cast<piece *>(p.query_out + base + at) = v;
        });
    }
    for (uint32_t c = threadIdx.x; c < turns; c += kBlock)
        turned(p.key + t * p.rope, c * V, [&](uint32_t at, piece v) { store(p.rank + at, v); });
    float reciprocal = 1.0f;
    if (p.weight) {
        float squares = 0.0f;
        for (uint32_t c = threadIdx.x * V; c < p.rank; c += kBlock * V) {
            const piece x = c < kBlock * V ? first : load(latent + c);
#pragma unroll
            for (int e = 0; e < V; ++e)
                squares += x[e] * x[e];
        }
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
    for (uint32_t c = threadIdx.x * V; c < p.rank; c += kBlock * V) {
        const piece x = c < kBlock * V ? first : load(latent + c);
        store(c, p.weight ? x * reciprocal * load(p.weight + c) : x);
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
    if (!p.tokens)
        return;
    if (p.rank % 4 == 0 && p.rope % 8 == 0)
        latent_append_kernel<4><<<p.tokens, kBlock, 0, stream>>>(p);
    else
        latent_append_kernel<1><<<p.tokens, kBlock, 0, stream>>>(p);
}

}  // namespace mfh
