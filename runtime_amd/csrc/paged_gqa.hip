// Attention of one new token per sequence over paged key/value caches.
//
// o = sum_j p_j v_j / sum_j p_j over the first length keys of a sequence, with
// p_j = exp(s_j - max s) and s_j = q . k_j / sqrt(head_dim); query heads
// kv_head * group .. of a key/value head share its keys.
//
// The work is a line of units: `unit_keys` keys of one item, an item being
// (sequence, key/value head, tile of `rows` of its query heads), items in order.
// Lengths live on the device, so every block adds up the units of the sequences
// itself and takes an equal run of them, which balances a batch of any mix of
// lengths.  A block that holds all units of an item writes its output; the
// blocks that share an item store records (maximum, sum, unnormalised output)
// that a second launch joins in block order, so results do not depend on timing.
// A run touches at most two shared items, its first and its last: two records a
// block.
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

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1)
        v = fmaxf(v, __shfl_xor(v, offset, 64));
    return v;
}

// How an item is shared: its first record, and the records (0: a block wrote the
// output itself).  The record of a further block b is 2 b.
struct ItemShare {
    uint32_t first, count;
};

// The records buffer: [2 blocks][rows][head_dim] outputs, [2 blocks][rows][2]
// (maximum, sum), then an ItemShare per item.
__host__ __device__ inline float *record_stats(const PagedAttention &p)
{
    return p.records + 2 * uint64_t(p.blocks) * p.rows * p.shape.head_dim;
}
__host__ __device__ inline ItemShare *item_shares(const PagedAttention &p)
{
    return reinterpret_cast<ItemShare *>(record_stats(p) + 4 * uint64_t(p.blocks) * p.rows);
}

// Keys of sequence s, or UINT32_MAX where its length is not a whole number
// that its table row has room for.
__device__ __forceinline__ uint32_t length_of(const PagedAttention &p, uint32_t s)
{
    const float v = p.lengths[s];
    if (!(v >= 0.0f && v <= 16777216.0f && truncf(v) == v))
        return UINT32_MAX;
    return uint64_t(v) <= (uint64_t(p.max_pages) << p.shape.page_shift) ? uint32_t(v) : UINT32_MAX;
}

__device__ __forceinline__ uint32_t units_of(const PagedAttention &p, uint32_t length)
{
    return length == UINT32_MAX ? 0 : (length + p.unit_keys - 1) / p.unit_keys;
}

// A block's place on the line of units.
struct Run {
    uint32_t sequence, head;  // the item of the next unit
    uint32_t unit;            // of that item
    uint32_t at, end;         // on the line
    uint32_t per;             // units of a block
};

// Adds up the sequences' units (every thread a run of sequences, then a scan
// over threads) and finds the block's first unit.  False: nothing to do.
__device__ bool find_run(const PagedAttention &p, Run &run)
{
    __shared__ uint32_t sums[kBlock / 64];
    __shared__ uint32_t found[3];
    const uint32_t heads = p.shape.kv_heads * p.row_tiles;
    const uint32_t each = (p.sequences + kBlock - 1) / kBlock;
    const uint32_t first = threadIdx.x * each;
    const uint32_t last = first + each < p.sequences ? first + each : p.sequences;
    uint32_t mine = 0;
    for (uint32_t s = first; s < last; ++s)
        mine += units_of(p, length_of(p, s));
    uint32_t upto = mine;  // inclusive scan over the wave
#pragma unroll
    for (int offset = 1; offset < 64; offset <<= 1) {
        const uint32_t v = __shfl_up(upto, offset, 64);
        if (int(threadIdx.x & 63) >= offset)
            upto += v;
    }
    if ((threadIdx.x & 63) == 63)
        sums[threadIdx.x >> 6] = upto;
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kBlock / 64; ++w) {
        if (w < threadIdx.x >> 6)
            upto += sums[w];
        total += sums[w];
    }
    total *= heads;
    run.per = (total + p.blocks - 1) / p.blocks;
    run.at = blockIdx.x * run.per;
    if (run.at >= total)
        return false;  // the same for every thread
    run.end = run.at + run.per < total ? run.at + run.per : total;
    uint32_t before = upto - mine;
    if (run.at >= before * heads && run.at < upto * heads) {
        for (uint32_t s = first; s < last; ++s) {
            const uint32_t units = units_of(p, length_of(p, s));
            if (run.at < (before + units) * heads) {
                const uint32_t inside = run.at - before * heads;
                found[0] = s;
                found[1] = inside / units;
                found[2] = inside % units;
                break;
            }
            before += units;
        }
    }
    __syncthreads();
    run.sequence = found[0];
    run.head = found[1];
    run.unit = found[2];
    return true;
}

// The part of an item that a block holds.
struct Part {
    uint32_t sequence, kv_head, row_tile, item;
    uint32_t length;       // keys of the sequence
    uint32_t begin, end;   // its keys
    bool whole;            // all of the item
    uint32_t record;       // where it is not
};

// The next part of a run, false at its end.  The block that holds an item's
// first unit says how the item is shared.
__device__ bool next_part(const PagedAttention &p, Run &run, Part &part)
{
    if (run.at >= run.end)
        return false;
    const uint32_t heads = p.shape.kv_heads * p.row_tiles;
    uint32_t length = length_of(p, run.sequence);
    uint32_t units = units_of(p, length);
    while (!units) {  // at < end: another unit follows
        ++run.sequence;
        length = length_of(p, run.sequence);
        units = units_of(p, length);
    }
    const uint32_t left = units - run.unit;
    const uint32_t take = left < run.end - run.at ? left : run.end - run.at;
    part.sequence = run.sequence;
    part.kv_head = run.head / p.row_tiles;
    part.row_tile = run.head % p.row_tiles;
    part.item = run.sequence * heads + run.head;
    part.length = length;
    part.begin = run.unit * p.unit_keys;
    const uint32_t end = (run.unit + take) * p.unit_keys;
    part.end = end < length ? end : length;
    part.whole = take == units;
    part.record = 2 * blockIdx.x + (run.at == blockIdx.x * run.per ? 0 : 1);
    if (run.unit == 0 && threadIdx.x == 0) {
        const uint32_t last = (run.at + units - 1) / run.per;
        item_shares(p)[part.item] = {part.record, part.whole ? 0 : last - blockIdx.x + 1};
    }
    run.at += take;
    run.unit += take;
    if (run.unit == units) {
        run.unit = 0;
        if (++run.head == heads) {
            run.head = 0;
            ++run.sequence;
        }
    }
    return true;
}

// ---- any head width -----------------------------------------------------------
//
// A block walks its part 64 keys at a time: each wave forms the scores of every
// fourth key by dot products over its lanes, the rows' maxima and sums follow
// online, and the block's threads add the keys' values to outputs in LDS.
// Bound by the dots' shuffles; head widths that are multiples of 16 have
// kernels of their own.
constexpr uint32_t kGeneralKeys = 64;
constexpr uint32_t kGeneralLds = 4096;  // most rows * head_dim of an item

template <typename T>
__global__ __launch_bounds__(kBlock) void paged_gqa_general_kernel(PagedAttention p)
{
    extern __shared__ float lds[];
    const uint32_t d = p.shape.head_dim, rows = p.rows;
    float *q = lds;              // [rows][d]
    float *acc = q + rows * d;   // [rows][d]
    float *prob = acc + rows * d;                // [rows][kGeneralKeys]
    float *stat = prob + rows * kGeneralKeys;    // [rows] maximum, sum, rescale
    __shared__ int bad;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T *keys = static_cast<const T *>(p.key_pages);
    const T *values = static_cast<const T *>(p.value_pages);
    Run run;
    if (!find_run(p, run))
        return;
    Part part;
    while (next_part(p, run, part)) {
        __syncthreads();
        const uint32_t head0 = part.kv_head * p.group + part.row_tile * rows;
        const uint32_t left = p.group - part.row_tile * rows;
        const uint32_t mine = left < rows ? left : rows;
        const float *query = p.query + (uint64_t(part.sequence) * p.query_heads + head0) * d;
        for (uint32_t i = threadIdx.x; i < mine * d; i += kBlock) {
            q[i] = query[i];
            acc[i] = 0.0f;
        }
        for (uint32_t r = threadIdx.x; r < rows; r += kBlock) {
            stat[r] = -__builtin_inff();
            stat[rows + r] = 0.0f;
        }
        if (threadIdx.x == 0)
            bad = 0;
        __syncthreads();
        const float *table = p.tables + uint64_t(part.sequence) * p.max_pages;
        // Offset of a key's row; an entry that names no page reads page 0 and
        // poisons the item.
        const auto row_of = [&](uint32_t key) {
            const float id = table[key >> p.shape.page_shift];
            const bool ok = valid_index(id, p.shape.pages);
            if (!ok)
                bad = 1;
            return uint64_t(ok ? uint32_t(id) : 0) * p.shape.stride() +
                   ((uint64_t(part.kv_head) << p.shape.page_shift) +
                    (key & (p.shape.page_size() - 1))) * d;
        };
        for (uint32_t base = part.begin; base < part.end; base += kGeneralKeys) {
            const uint32_t count =
                part.end - base < kGeneralKeys ? part.end - base : kGeneralKeys;
            for (uint32_t j = wave; j < count; j += kBlock / 64) {
                const T *key = keys + row_of(base + j);
                for (uint32_t r = 0; r < mine; ++r) {
                    float dot = 0.0f;
                    for (uint32_t c = lane; c < d; c += 64)
                        dot += q[r * d + c] * float(key[c]);
                    dot = wave_sum(dot);
                    if (lane == 0)
                        prob[r * kGeneralKeys + j] = dot * p.scale;
                }
            }
            __syncthreads();
            for (uint32_t r = wave; r < mine; r += kBlock / 64) {
                const float s = lane < count ? prob[r * kGeneralKeys + lane] : -__builtin_inff();
                const float before = stat[r];
                const float most = fmaxf(before, wave_max(s));
                // Where every score so far is -infinity, nothing is added.
                const float base_line = most == -__builtin_inff() ? 0.0f : most;
                const float e = lane < count ? expf(s - base_line) : 0.0f;
                const float rescale = expf(before - base_line);
                prob[r * kGeneralKeys + lane] = e;
                const float sum = wave_sum(e);
                if (lane == 0) {
                    stat[r] = most;
                    stat[rows + r] = stat[rows + r] * rescale + sum;
                    stat[2 * rows + r] = rescale;
                }
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < mine * d; i += kBlock) {
                const uint32_t r = i / d, c = i - r * d;
                float sum = 0.0f;
                for (uint32_t j = 0; j < count; ++j)
                    sum += prob[r * kGeneralKeys + j] * float(values[row_of(base + j) + c]);
                acc[i] = acc[i] * stat[2 * rows + r] + sum;
            }
            __syncthreads();
        }
        const float poison = bad ? __builtin_nanf("") : 0.0f;
        if (part.whole) {
            float *out = p.out + (uint64_t(part.sequence) * p.query_heads + head0) * d;
            for (uint32_t i = threadIdx.x; i < mine * d; i += kBlock)
                out[i] = acc[i] / stat[rows + i / d] + poison;
        } else {
            float *out = p.records + uint64_t(part.record) * rows * d;
            for (uint32_t i = threadIdx.x; i < mine * d; i += kBlock)
                out[i] = acc[i];
            float *stats = record_stats(p) + uint64_t(part.record) * rows * 2;
            for (uint32_t r = threadIdx.x; r < mine; r += kBlock) {
                stats[2 * r] = stat[r];
                stats[2 * r + 1] = stat[rows + r] + poison;
            }
        }
    }
}

// ---- the join --------------------------------------------------------------------

// One block per (item, row).  Shared items: out = sum_i a_i e^(m_i - M) / sum_i l_i
// e^(m_i - M) over the records, in block order.  Sequences without a key give
// zeros, those whose length is invalid NaN.
__global__ __launch_bounds__(kBlock) void paged_gqa_join_kernel(PagedAttention p)
{
    extern __shared__ float part[];  // [parts][width]
    const uint32_t heads = p.shape.kv_heads * p.row_tiles, d = p.shape.head_dim;
    const uint32_t item = blockIdx.x / p.rows, row = blockIdx.x % p.rows;
    const uint32_t sequence = item / heads, head = item % heads;
    const uint32_t in_group = head % p.row_tiles * p.rows + row;
    if (in_group >= p.group)
        return;
    float *out = p.out + (uint64_t(sequence) * p.query_heads +
                          head / p.row_tiles * p.group + in_group) * d;
    const uint32_t length = length_of(p, sequence);
    if (length == 0 || length == UINT32_MAX) {
        for (uint32_t c = threadIdx.x; c < d; c += kBlock)
            out[c] = length ? __builtin_nanf("") : 0.0f;
        return;
    }
    const ItemShare share = item_shares(p)[item];
    if (!share.count)
        return;
    const auto record = [&](uint32_t i) {
        return uint64_t(i ? share.first / 2 * 2 + 2 * i : share.first) * p.rows + row;
    };
    const float *stats = record_stats(p);
    float most = -__builtin_inff();
    for (uint32_t i = threadIdx.x & 63; i < share.count; i += 64)
        most = fmaxf(most, stats[2 * record(i)]);
    most = wave_max(most);
    const float base_line = most == -__builtin_inff() ? 0.0f : most;
    float sum = 0.0f;
    for (uint32_t i = threadIdx.x & 63; i < share.count; i += 64)
        sum += stats[2 * record(i) + 1] * expf(stats[2 * record(i)] - base_line);
    sum = wave_sum(sum);
    // Threads: `parts` interleaved shares of the records by up to kBlock columns.
    const uint32_t width = d < kBlock ? d : kBlock, parts = kBlock / width;
    const uint32_t mine = threadIdx.x / width;
    for (uint32_t c0 = 0; c0 < d; c0 += width) {
        const uint32_t c = c0 + threadIdx.x % width;
        float a = 0.0f;
        if (mine < parts && c < d)
            for (uint32_t i = mine; i < share.count; i += parts)
                a += p.records[record(i) * d + c] * expf(stats[2 * record(i)] - base_line);
        __syncthreads();
        if (mine < parts)
            part[threadIdx.x] = a;
        __syncthreads();
        if (threadIdx.x < width && c < d) {
            for (uint32_t i = 1; i < parts; ++i)
                a += part[i * width + threadIdx.x];
            out[c] = a / sum;
        }
    }
}

}  // namespace

bool paged_gqa_plan(PagedAttention &p, int cu_count)
{
    const uint32_t d = p.shape.head_dim;
    const uint32_t most_rows = kGeneralLds / d < 16 ? kGeneralLds / d : 16;
    p.rows = p.group < most_rows ? p.group : most_rows;
    p.row_tiles = (p.group + p.rows - 1) / p.rows;
    p.unit_keys = kGeneralKeys;
    const uint64_t items = uint64_t(p.sequences) * p.shape.kv_heads * p.row_tiles;
    const uint64_t longest = uint64_t(p.max_pages) << p.shape.page_shift;
    const uint64_t per_item = (longest + p.unit_keys - 1) / p.unit_keys;
    const uint64_t limit = uint64_t(1) << 31;
    if (items * p.rows > limit || per_item > limit || (per_item && items > limit / per_item))
        return false;
    // What the block's end and the last block's start reach stays in 32 bits.
    const uint64_t most_blocks = uint64_t(cu_count) * 4, units = items * per_item;
    p.blocks = uint32_t(units < most_blocks ? units : most_blocks);
    return true;
}

size_t paged_gqa_scratch_bytes(const PagedAttention &p)
{
    const uint64_t floats = 2 * uint64_t(p.blocks) * p.rows * (p.shape.head_dim + 2);
    const uint64_t items = uint64_t(p.sequences) * p.shape.kv_heads * p.row_tiles;
    return size_t(floats * sizeof(float) + items * sizeof(ItemShare));
}

void launch_paged_gqa(hipStream_t stream, const PagedAttention &p)
{
    const uint64_t items = uint64_t(p.sequences) * p.shape.kv_heads * p.row_tiles;
    if (!items)
        return;
    if (p.blocks) {
        const size_t bytes =
            (2 * size_t(p.rows) * p.shape.head_dim + size_t(p.rows) * (kGeneralKeys + 3)) *
            sizeof(float);
        if (p.shape.half)
            paged_gqa_general_kernel<_Float16><<<p.blocks, kBlock, bytes, stream>>>(p);
        else
            paged_gqa_general_kernel<float><<<p.blocks, kBlock, bytes, stream>>>(p);
    }
    paged_gqa_join_kernel<<<unsigned(items * p.rows), kBlock, kBlock * sizeof(float), stream>>>(p);
}

}  // namespace mfh
