// Attention of one new token per sequence over paged key/value caches.
//
// o = sum_j p_j v_j / sum_j p_j over the first length keys of a sequence, with
// p_j = exp(s_j - max s) and s_j = q . k_j / sqrt(head_dim); query heads
// kv_head * group .. of a key/value head share its keys.
//
// The work is a line of units: a few keys (a power of two) of one item, an item being
// (sequence, key/value head, tile of `rows` of its query heads), items in order.
// Lengths live on the device, so every block adds up the units of the sequences
// itself and takes an equal run of them, which balances a batch of any mix of
// lengths.  A block that holds all units of an item writes its output; the
// blocks that share an item store records (maximum, sum, unnormalised output)
// that a second launch joins in block order, so results do not depend on timing.
// A run touches at most two shared items, its first and its last: two records a
// block.
//
// Bound by the reads of the cache.  Both launches, in us (and the cache's TB/s): 96
// sequences of 33 to 2048 keys, 8 key heads of 64, f32 39.8 (4.9); 48 of 17 to 8191,
// 8 of 128, binary16 52.5 (5.2); one of 131071, 8 of 64, binary16 48.7 (5.5), f32 88.1
// (6.1).  About 9 us of each are the two launches and their dependent reads, which
// is all that a short call takes: one sequence of 2047 keys 10.4.
#include <type_traits>

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

// A length, or UINT32_MAX where it is not a whole number that a table row has room
// for.
__device__ __forceinline__ uint32_t checked_length(const PagedAttention &p, float v)
{
    return v >= 0.0f && v <= p.longest && truncf(v) == v ? uint32_t(v) : UINT32_MAX;
}
__device__ __forceinline__ uint32_t length_of(const PagedAttention &p, uint32_t s)
{
    return checked_length(p, p.lengths[s]);
}

// An item's place on the line: `item_units` for what every item costs, then its
// units of keys.  Five, for the waits of an item's start and end, in the time of a
// unit: a block can be given many short items.  48 sequences of 17 to 8191 keys in
// any order take 69 to 75 us with two, 63 with three, 55.7, 53.6, 53.6 and 54 with
// four, five, six and eight (166 without).
__device__ __forceinline__ uint32_t units_of(const PagedAttention &p, uint32_t length)
{
    const uint32_t units = (length + (1u << p.unit_shift) - 1) >> p.unit_shift;
    return length == UINT32_MAX || length == 0 ? 0 : units + p.item_units;
}

// A block's place on the line of units: block b of n starts at floor(b total / n), so
// that items of one length start where blocks do wherever they can.
struct Run {
    uint32_t sequence, kv_head, row_tile;  // the item of the next unit
    uint32_t length;                       // of the sequence
    uint32_t unit;                         // of that item
    uint32_t start, at, end;               // on the line
    uint32_t total, blocks;                // of the line
};

// A block's units out of `total`, even to one, and whether it has any.
__device__ __forceinline__ bool take_units(const PagedAttention &p, uint32_t total, Run &run)
{
    const uint32_t most = (total + (1u << p.least_shift) - 1) >> p.least_shift;
    const uint32_t blocks = most < p.blocks ? most : p.blocks, b = blockIdx.x;
    if (b >= blocks)
        return false;
    run.total = total;
    run.blocks = blocks;
    // The products stay in 32 bits: blocks are at most a few for every CU.
    const uint32_t quotient = total / blocks, odd = total - quotient * blocks;
    run.start = run.at = b * quotient + b * odd / blocks;
    run.end = (b + 1) * quotient + (b + 1) * odd / blocks;
    return true;
}
// The block that has a unit: the quotient of whole numbers below 2^53, so the
// rounded one is below the next whole number where the exact one is.
__device__ __forceinline__ uint32_t block_of(const Run &run, uint32_t unit)
{
    const double after = (double(unit) + 1.0) * double(run.blocks) - 1.0;
    return uint32_t(after / double(run.total));
}

// Inclusive scan over the wave's lanes by DPP moves; lane 63 ends with the sum.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v)
{
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t lanes_scan(uint32_t v)
{
    v += moved<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);  // row 0's and 2's last lane to the next row
    v += moved<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
    return v;
}

// The item that a block's first unit is in, `inside` the units of a sequence whose
// items have `units` each.
__device__ __forceinline__ void start_run(const PagedAttention &p, Run &run, uint32_t sequence,
                                          uint32_t length, uint32_t units, uint32_t inside)
{
    const auto scalar = [](uint32_t v) { return uint32_t(__builtin_amdgcn_readfirstlane(v)); };
    const uint32_t head = scalar(inside) / scalar(units);
    run.sequence = scalar(sequence);
    run.length = scalar(length);
    run.unit = scalar(inside) - head * scalar(units);
    run.kv_head = head;
    run.row_tile = 0;
    if (p.row_tiles > 1) {
        run.kv_head = head / p.row_tiles;
        run.row_tile = head - run.kv_head * p.row_tiles;
    }
}

// Adds up the sequences' units and finds the block's first one.  Up to 256
// sequences are four for every lane of each wave, without a barrier; more are a
// run of sequences for every thread, then a scan over the block.  False, for
// every thread: nothing to do.  A call's first reads wait for this code, which runs
// once and is fetched as it runs: divisions are few and of 32 bits, scans are moves
// between lanes, and the first tile's reads go out before anything that can wait (with
// 64-bit divisions and shuffles before them calls took 0.3 to 3.6 us longer, 128
// sequences of 128 keys 22.1 for 19.5).
__device__ __forceinline__ bool find_run(const PagedAttention &p, Run &run)
{
    const uint32_t heads = p.shape.kv_heads * p.row_tiles;
    const uint32_t lane = threadIdx.x & 63;
    if (p.sequences <= 256) {
        float value[4];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            value[e] = p.lengths[4 * lane + e < p.sequences ? 4 * lane + e : p.sequences - 1];
        uint32_t length[4], upto[4], sum = 0;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            length[e] = 4 * lane + e < p.sequences ? checked_length(p, value[e]) : 0;
            upto[e] = sum += units_of(p, length[e]);
        }
        const uint32_t scan = lanes_scan(sum);
        if (!take_units(p, __builtin_amdgcn_readlane(scan, 63) * heads, run))
            return false;
        const uint32_t from = __builtin_ctzll(__ballot(run.at < scan * heads));
        const auto of = [&](uint32_t v) { return uint32_t(__builtin_amdgcn_readlane(v, from)); };
        const uint32_t before = of(scan) - of(sum);
        uint32_t e = 0, last = 0, next = of(upto[0]), keys = of(length[0]);
#pragma unroll
        for (uint32_t n = 1; n < 4; ++n)
            if (run.at >= (before + next) * heads) {
                e = n;
                last = next;
                next = of(upto[n]);
                keys = of(length[n]);
            }
        start_run(p, run, 4 * from + e, keys, next - last, run.at - (before + last) * heads);
        return true;
    }
    __shared__ uint32_t sums[kBlock / 64];
    __shared__ uint32_t found[4];
    const uint32_t each = (p.sequences + kBlock - 1) / kBlock;
    const uint32_t first = threadIdx.x * each;
    const uint32_t last = first + each < p.sequences ? first + each : p.sequences;
    uint32_t mine = 0;
    for (uint32_t s = first; s < last; ++s)
        mine += units_of(p, length_of(p, s));
    uint32_t upto = lanes_scan(mine);
    if (lane == 63)
        sums[threadIdx.x >> 6] = upto;
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kBlock / 64; ++w) {
        if (w < threadIdx.x >> 6)
            upto += sums[w];
        total += sums[w];
    }
    if (!take_units(p, __builtin_amdgcn_readfirstlane(total) * heads, run))
        return false;
    uint32_t before = upto - mine;
    if (run.at >= before * heads && run.at < upto * heads) {
        for (uint32_t s = first; s < last; ++s) {
            const uint32_t length = length_of(p, s), units = units_of(p, length);
            if (run.at < (before + units) * heads) {
                found[0] = s;
                found[1] = length;
                found[2] = units;
                found[3] = run.at - before * heads;
                break;
            }
            before += units;
        }
    }
    __syncthreads();
    start_run(p, run, found[0], found[1], found[2], found[3]);
    return true;
}

// The part of an item that a block holds.
struct Part {
    uint32_t sequence, kv_head, row_tile;
    uint32_t length;       // keys of the sequence
    uint32_t begin, end;   // its keys
    bool whole;            // all of the item
    uint32_t record;       // where it is not
    uint32_t last_unit;    // on the line, of the item; UINT32_MAX but for its first keys
};

// The next part of a run, false at its end; it may have no keys (begin == end).  The
// block that holds an item's first keys says how the item is shared.
__device__ __forceinline__ bool next_part(const PagedAttention &p, Run &run, Part &part)
{
    if (run.at >= run.end)
        return false;
    uint32_t units = units_of(p, run.length);
    while (!units) {  // at < end: another unit follows
        run.length = length_of(p, ++run.sequence);
        units = units_of(p, run.length);
    }
    const uint32_t length = run.length;
    const uint32_t left = units - run.unit;
    const uint32_t take = left < run.end - run.at ? left : run.end - run.at;
    // Units of keys, past the item's own.
    const uint32_t own = p.item_units;
    const uint32_t begin = run.unit > own ? run.unit - own : 0;
    const uint32_t end = run.unit + take > own ? run.unit + take - own : 0;
    part.sequence = run.sequence;
    part.kv_head = run.kv_head;
    part.row_tile = run.row_tile;
    part.length = length;
    part.begin = begin << p.unit_shift;
    part.end = end << p.unit_shift < length ? end << p.unit_shift : length;
    part.whole = begin == 0 && end == units - own;
    part.record = 2 * blockIdx.x + (run.at == run.start ? 0 : 1);
    part.last_unit = begin == 0 && end > 0 ? run.at - run.unit + units - 1 : UINT32_MAX;
    run.at += take;
    run.unit += take;
    if (run.unit == units) {
        run.unit = 0;
        if (++run.row_tile == p.row_tiles) {
            run.row_tile = 0;
            if (++run.kv_head == p.shape.kv_heads) {
                run.kv_head = 0;
                ++run.sequence;
                run.length = run.at < run.end ? length_of(p, run.sequence) : 0;
            }
        }
    }
    return true;
}

// Said once the part's reads are on their way.
__device__ __forceinline__ void say_share(const PagedAttention &p, const Run &run,
                                          const Part &part)
{
    if (part.last_unit == UINT32_MAX)
        return;
    const uint32_t count = part.whole ? 0 : block_of(run, part.last_unit) - blockIdx.x + 1;
    const uint32_t item =
        (part.sequence * p.shape.kv_heads + part.kv_head) * p.row_tiles + part.row_tile;
    if (threadIdx.x == 0)
        item_shares(p)[item] = {part.record, count};
}

// ---- any head width -----------------------------------------------------------
//
// A block walks its part 64 keys at a time: each wave forms the scores of every
// fourth key by dot products over its lanes, the rows' maxima and sums follow
// online, and the block's threads add the keys' values to outputs in LDS.
// Bound by the dots' shuffles: 32 sequences of 2048 keys of 4 heads of 144 take 640 us
// in f32 and 579 in binary16, of 160, which has a kernel of its own, 61 and 37.
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
        if (part.begin == part.end)
            continue;
        say_share(p, run, part);
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
                const float e = lane < count ? exp2f(s - base_line) : 0.0f;
                const float rescale = exp2f(before - base_line);
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

// ---- head widths that are multiples of 16, on matrix cores ------------------------
//
// A wave takes every fourth tile of a part: TILE = 16 NB keys.  Per tile,
// S^T = K Q^T leaves query row j in lane column j (lane 16 q + j holds the
// scores of keys 16 c + 4 q + r in register r of block c), the softmax follows
// online in the row's four lanes, and O^T += V^T P^T takes those registers as
// its second operand as they are.  Both first operands come straight from the
// cache to registers: a lane's piece of a key row is the operand of S^T, and
// its piece of a value row (the columns s j .. s j + s - 1 of a chunk of s
// 16-column tiles) is, column by column, an operand row of s tiles of O^T, whose
// rows are then columns s i + t.  No LDS and no barrier until the part ends.
//
// f32 caches run on v_mfma_f32_16x16x4_f32: exact products, f32 sums.
// Binary16 caches run on v_mfma_f32_16x16x32_f16: keys and values are operands
// as they are, queries and probabilities are the sum of two binary16 parts
// (each part the nearest to what is left, so the two are within 2^-24 of the
// value, f32's own rounding).  A query row is first scaled by a power of two to
// below 2^15, so what is cut off is below 2^-39 of its largest element;
// probabilities carry 2^15, so what is cut off is below 2^-40 of the largest.
//
// Loads of the next tile's keys are issued as soon as the products have read
// this tile's, its values' likewise: each is in flight behind the other's
// arithmetic, in the same registers.  They are read once, and said to be
// (nontemporal): with that said of neither the first three calls above took 12, 16 and
// 9 % longer, of one a time in between.
//
// A tile is 32 keys in binary16 (a product's depth) and 16 in f32: of twice that
// the registers hold fewer blocks.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kWaves = kBlock / 64;
constexpr uint32_t kItemUnits = 5;
constexpr uint32_t kRowsMost = 16;
constexpr float kProbabilityShift = 15.0f;

template <bool HALF>
constexpr int key_blocks(int)
{
    return HALF ? 2 : 1;
}

// Chunks of a value row: as many 16-column tiles as one load holds (16 bytes,
// then 8, 4, 2).
template <bool HALF>
__host__ __device__ constexpr int chunk_tiles(int left)
{
    const int most = HALF ? 8 : 4;
    int s = most;
    while (s > left)
        s /= 2;
    return s;
}

// f(first tile, tiles) for each chunk of N tiles, both as constants.
template <int N, bool HALF, int T = 0, typename F>
__device__ __forceinline__ void for_chunks(F f)
{
    if constexpr (T < N) {
        constexpr int S = chunk_tiles<HALF>(N - T);
        f(std::integral_constant<int, T>{}, std::integral_constant<int, S>{});
        for_chunks<N, HALF, T + S>(f);
    }
}

// Maximum over a row's four lanes.
__device__ __forceinline__ float lanes_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float lanes_sum(float v)
{
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// a and b as two binary16 parts each.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t &hi, uint32_t &lo)
{
    const v2h h = {_Float16(a), _Float16(b)};
    const v2h l = {_Float16(a - float(h[0])), _Float16(b - float(h[1]))};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

// Blocks of the kernel for every CU; all run at once.  Two keep 64 KB or more of
// reads in flight, which is enough, and make fewer starts, ends and records than
// what the registers hold: 32 sequences of 2048 keys, one of 65536, 64 of 20 to
// 4000, 128 of 256, with 4 to 8 key heads of 64, f32: 28.4 / 48.0 / 41.4 / 26.0 us
// with two, 29.2 / 50.2 / 41.3 / 26.1 with four; of 96 39.7 / 70.7 / 59.2 / 38.9 and
// with three 39.7 / 73.2 / 58.8 / 43.9.  Narrow heads, whose tiles are small, take
// four (width 32, binary16: 14.3 / 18.9 / 18.8 / 11.7, two 14.0 / 18.0 / 20.9 /
// 13.1), wide ones the one that their registers allow.
constexpr int resident_blocks(int d)
{
    return d > 128 ? 1 : d > 32 ? 2 : 4;
}

// D: head width.  SMALL: pages of 8 keys (else a page holds whole 16-key blocks).
template <int D, bool HALF, bool SMALL>
__global__ __launch_bounds__(kBlock, resident_blocks(D)) void paged_gqa_mfma_kernel(PagedAttention p)
{
    static_assert(D % 16 == 0 && D <= 256, "head width of the matrix-core path");
    using T = typename std::conditional<HALF, _Float16, float>::type;
    constexpr int NB = key_blocks<HALF>(D);
    constexpr uint32_t TILE = 16 * NB;
    constexpr int U = HALF ? (D + 31) / 32 : D / 16;  // 16-byte pieces of a key row per lane
    constexpr int N = D / 16;                         // 16-column tiles
    constexpr int W = HALF ? (N + 1) / 2 : N;         // dwords of a value row per lane
    extern __shared__ float lds[];
    const uint32_t rows = p.rows;
    float *part_out = lds;                               // [kWaves][rows][D]
    float *part_stat = lds + kWaves * rows * D;          // [kWaves][16][2]
    __shared__ int bad_any;

    const uint32_t lane = threadIdx.x & 63, q = lane >> 4, j = lane & 15;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t shift = p.shape.page_shift, inside = p.shape.page_size() - 1;
    const T *keys = static_cast<const T *>(p.key_pages);
    const T *values = static_cast<const T *>(p.value_pages);
    Run run;
    if (!find_run(p, run))
        return;
    Part part;
    while (next_part(p, run, part)) {
        if (part.begin == part.end)
            continue;
        const uint32_t head0 = part.kv_head * p.group + part.row_tile * rows;
        const uint32_t left = p.group - part.row_tile * rows;
        const uint32_t mine = left < rows ? left : rows;
        const float *table = p.tables + uint64_t(part.sequence) * p.max_pages;
        const uint32_t last_key = part.length - 1;
        const uint64_t head_offset = (uint64_t(part.kv_head) << shift) * D;
        int bad = 0;

        // Page ids of a tile's 16-key blocks: the one of all its keys, or with
        // small pages those of the lane's key row and of its value rows.
        struct Ids {
            float key[NB], value[SMALL ? NB : 1];
        };
        const auto load_ids = [&](uint32_t k0) {
            Ids ids;
#pragma unroll
            for (int c = 0; c < NB; ++c) {
                if (SMALL) {
                    const uint32_t a = k0 + 16 * c + j, b = k0 + 16 * c + 4 * q;
                    ids.key[c] = table[(a < last_key ? a : last_key) >> shift];
                    ids.value[c] = table[(b < last_key ? b : last_key) >> shift];
                } else {
                    const uint32_t a = k0 + 16 * c;
                    ids.key[c] = reinterpret_cast<const __attribute__((address_space(4))) float *>(
                        reinterpret_cast<uint64_t>(table))[(a < last_key ? a : last_key) >> shift];
                }
            }
            return ids;
        };
        const auto page_base = [&](float id) {
            const bool ok = valid_index(id, p.shape.pages);
            bad |= !ok;
            return uint64_t(ok ? uint32_t(id) : 0) * p.shape.stride() + head_offset;
        };

        uint32_t kr[NB][U][4];
        uint32_t vr[4 * NB][W];
        const auto load_keys = [&](const Ids &ids, uint32_t k0) {
#pragma unroll
            for (int c = 0; c < NB; ++c) {
                const uint32_t a = k0 + 16 * c + j;
                const uint32_t slot = (a < last_key ? a : last_key) & inside;
                const T *row = keys + page_base(ids.key[c]) + slot * uint32_t(D);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    // Past the head's end (its width an odd number of 16s) a
                    // lane reads columns that its query's zeros drop.
                    uint32_t column = HALF ? 32 * u + 8 * q : 16 * u + 4 * q;
                    if (D % 32 != 0 && HALF && u == U - 1 && q >= 2)
                        column -= 16;
                    const v4u piece = __builtin_nontemporal_load(reinterpret_cast<const v4u *>(row + column));
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        kr[c][u][e] = piece[e];
                }
            }
        };
        const auto load_values = [&](const Ids &ids, uint32_t k0) {
#pragma unroll
            for (int c = 0; c < NB; ++c) {
                const uint64_t base = page_base(SMALL ? ids.value[c] : ids.key[c]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t a = k0 + 16 * c + 4 * q + r;
                    const uint32_t slot = (a < last_key ? a : last_key) & inside;
                    const T *row = values + base + slot * uint32_t(D);
                    uint32_t *to = vr[4 * c + r];
                    for_chunks<N, HALF>([&](auto first_tile, auto tiles) {
                        constexpr int t = first_tile, n = tiles;
                        constexpr int bytes = n * int(sizeof(T)), w = HALF ? t / 2 : t;
                        const T *at = row + 16 * t + n * j;
                        if constexpr (bytes == 16) {
                            const v4u piece = __builtin_nontemporal_load(reinterpret_cast<const v4u *>(at));
                            to[w] = piece[0], to[w + 1] = piece[1];
                            to[w + 2] = piece[2], to[w + 3] = piece[3];
                        } else if constexpr (bytes == 8) {
                            const v2u piece = __builtin_nontemporal_load(reinterpret_cast<const v2u *>(at));
                            to[w] = piece[0], to[w + 1] = piece[1];
                        } else if constexpr (bytes == 4) {
                            to[w] = *reinterpret_cast<const uint32_t *>(at);
                        } else {
                            to[w] = *reinterpret_cast<const uint16_t *>(at);
                        }
                    });
                }
            }
        };

        // The wave's tiles; one without any takes the part's first without a key.
        const uint32_t first = part.begin + wave * TILE;
        const bool any = first < part.end;
        Ids ids = load_ids(any ? first : part.begin);
        // The lane's row of queries; rows past the group, and columns past the head's
        // end, are zero.
        const float *query =
            p.query + (uint64_t(part.sequence) * p.query_heads + head0 + (j < mine ? j : 0)) * D;
        float qf[U][HALF ? 8 : 4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < (HALF ? 8 : 4); e += 4) {
                const uint32_t column = HALF ? 32 * u + 8 * q + e : 16 * u + 4 * q + e;
                const v4f piece =
                    *reinterpret_cast<const v4f *>(query + (column < uint32_t(D) ? column : 0));
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    qf[u][e + i] = piece[i];
            }
        if (any) {
            load_keys(ids, first);
            load_values(ids, first);
        }
        say_share(p, run, part);
        float most = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < (HALF ? 8 : 4); ++i) {
                const uint32_t column = HALF ? 32 * u + 8 * q + i : 16 * u + 4 * q + i;
                qf[u][i] = j < mine && column < uint32_t(D) ? qf[u][i] : 0.0f;
                most = fmaxf(most, fabsf(qf[u][i]));
            }
        float factor = p.scale;
        uint32_t qh[HALF ? U : 1][4], ql[HALF ? U : 1][4];
        if (HALF) {
            most = lanes_max(most);
            // 2^14 <= most 2^exponent < 2^15 (0 and infinities as they are).
            int exponent = 0;
            if (most > 0.0f && most < __builtin_inff())
                exponent = 15 - (ilogbf(most) + 1);
            factor = ldexpf(p.scale, -exponent);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    split_pair(ldexpf(qf[u][2 * e], exponent), ldexpf(qf[u][2 * e + 1], exponent),
                               qh[u][e], ql[u][e]);
        }

        v4f o[N];
#pragma unroll
        for (int t = 0; t < N; ++t)
            o[t] = v4f{0, 0, 0, 0};
        float m = -__builtin_inff(), l = 0.0f;
        const auto tile = [&](uint32_t k0, auto last) {
            constexpr bool LAST = last;
            const uint32_t next = k0 + kWaves * TILE;
            if constexpr (!LAST)
                ids = load_ids(next);
            v4f s[NB];
#pragma unroll
            for (int c = 0; c < NB; ++c)
                s[c] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    const v4u piece = {kr[c][u][0], kr[c][u][1], kr[c][u][2], kr[c][u][3]};
                    if constexpr (HALF) {
                        const v4u hi = {qh[u][0], qh[u][1], qh[u][2], qh[u][3]};
                        const v4u lo = {ql[u][0], ql[u][1], ql[u][2], ql[u][3]};
                        const v8h k = __builtin_bit_cast(v8h, piece);
                        s[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            k, __builtin_bit_cast(v8h, lo), s[c], 0, 0, 0);
                        s[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            k, __builtin_bit_cast(v8h, hi), s[c], 0, 0, 0);
                    } else {
                        const v4f k = __builtin_bit_cast(v4f, piece);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], qf[u][e], s[c], 0, 0,
                                                                        0);
                    }
                }
            if constexpr (!LAST)
                load_keys(ids, next);
            float top = -__builtin_inff();
#pragma unroll
            for (int c = 0; c < NB; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = s[c][r] * factor;
                    if (LAST && k0 + 16 * c + 4 * q + r >= part.end)
                        v = -__builtin_inff();
                    s[c][r] = v;
                    top = fmaxf(top, v);
                }
            top = fmaxf(m, lanes_max(top));
            // While every score is -infinity, nothing is added.
            const float base = top == -__builtin_inff() ? 0.0f : top;
            if (__any(top > m)) {
                const float rescale = __builtin_amdgcn_exp2f(m - base);
                l *= rescale;
#pragma unroll
                for (int t = 0; t < N; ++t)
                    o[t] *= rescale;
                m = top;
            }
#pragma unroll
            for (int c = 0; c < NB; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[c][r] =
                        __builtin_amdgcn_exp2f(s[c][r] - (HALF ? base - kProbabilityShift : base));
                    l += s[c][r];
                }
            if (LAST && k0 + TILE > part.end) {
                // Rows past the end repeat the last key's: they may hold
                // what a zero weight does not drop.
#pragma unroll
                for (int i = 0; i < 4 * NB; ++i)
                    if (k0 + 16 * (i / 4) + 4 * q + i % 4 >= part.end)
#pragma unroll
                        for (int w = 0; w < W; ++w)
                            vr[i][w] = 0;
            }
            if constexpr (HALF) {
                v4u hi, lo;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    uint32_t a, b;
                    split_pair(s[h / 2][2 * (h % 2)], s[h / 2][2 * (h % 2) + 1], a, b);
                    hi[h] = a, lo[h] = b;
                }
#pragma unroll
                for (int t = 0; t < N; ++t) {
                    v4u column;
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        column[h] =
                            __builtin_amdgcn_perm(vr[2 * h + 1][t / 2], vr[2 * h][t / 2],
                                                  t % 2 ? 0x07060302u : 0x05040100u);
                    const v8h v = __builtin_bit_cast(v8h, column);
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, __builtin_bit_cast(v8h, lo),
                                                                  o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, __builtin_bit_cast(v8h, hi),
                                                                  o[t], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int c = 0; c < NB; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int t = 0; t < N; ++t)
                            o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __uint_as_float(vr[4 * c + r][t]), s[c][r], o[t], 0, 0, 0);
            }
            if constexpr (!LAST)
                load_values(ids, next);
        };
        // The last tile apart: it alone has keys past the end, and without a
        // condition on the others' loads the compiler knows how many are in flight
        // and waits for no more than it needs.
        if (any) {
            uint32_t k0 = first;
#pragma unroll 1
            for (; k0 + kWaves * TILE < part.end; k0 += kWaves * TILE)
                tile(k0, std::false_type{});
            tile(k0, std::true_type{});
        }

        // The waves' shares of the part, joined in their order.
        l = lanes_sum(l);
        __syncthreads();  // an earlier part's shares have been read
        if (threadIdx.x == 0)
            bad_any = 0;
        if (j < mine) {
            float *row = part_out + (wave * rows + j) * D;
            for_chunks<N, HALF>([&](auto first_tile, auto tiles) {
                constexpr int t0 = first_tile, n = tiles;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int t = 0; t < n; ++t)
                        row[16 * t0 + n * (4 * q + r) + t] = o[t0 + t][r];
            });
        }
        if (q == 0) {
            part_stat[(wave * 16 + j) * 2] = m;
            part_stat[(wave * 16 + j) * 2 + 1] = l;
        }
        __syncthreads();
        if (bad)
            bad_any = 1;
        __syncthreads();
        const float poison = bad_any ? __builtin_nanf("") : 0.0f;
        float *out = part.whole
                         ? p.out + (uint64_t(part.sequence) * p.query_heads + head0) * D
                         : p.records + uint64_t(part.record) * rows * D;
        for (uint32_t i = threadIdx.x; i < mine * D; i += kBlock) {
            const uint32_t r = i / D;
            float top = part_stat[r * 2];
#pragma unroll
            for (int w = 1; w < kWaves; ++w)
                top = fmaxf(top, part_stat[(w * 16 + r) * 2]);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            float a = 0.0f, sum = poison;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float weight = __builtin_amdgcn_exp2f(part_stat[(w * 16 + r) * 2] - base);
                a += weight * part_out[w * rows * D + i];
                sum += weight * part_stat[(w * 16 + r) * 2 + 1];
            }
            out[i] = part.whole ? a / sum : a;
            if (!part.whole && i % D == 0) {
                float *stats = record_stats(p) + (uint64_t(part.record) * rows + r) * 2;
                stats[0] = top;
                stats[1] = sum;
            }
        }
    }
}

// The kernel of a page shape (null: none) and the blocks of it that a CU holds.
struct MfmaKernel {
    void (*run)(PagedAttention) = nullptr;
    int resident = 0;
};
template <int D>
MfmaKernel mfma_kernel_of(bool half, bool small)
{
    if (half)
        return {small ? paged_gqa_mfma_kernel<D, true, true> : paged_gqa_mfma_kernel<D, true, false>,
                resident_blocks(D)};
    return {small ? paged_gqa_mfma_kernel<D, false, true> : paged_gqa_mfma_kernel<D, false, false>,
            resident_blocks(D)};
}
MfmaKernel mfma_kernel(const PageShape &shape)
{
    const bool half = shape.half, small = shape.page_shift < 4;
    switch (shape.head_dim) {
    case 16: return mfma_kernel_of<16>(half, small);
    case 32: return mfma_kernel_of<32>(half, small);
    case 48: return mfma_kernel_of<48>(half, small);
    case 64: return mfma_kernel_of<64>(half, small);
    case 80: return mfma_kernel_of<80>(half, small);
    case 96: return mfma_kernel_of<96>(half, small);
    case 112: return mfma_kernel_of<112>(half, small);
    case 128: return mfma_kernel_of<128>(half, small);
    case 160: return mfma_kernel_of<160>(half, small);
    case 192: return mfma_kernel_of<192>(half, small);
    case 256: return mfma_kernel_of<256>(half, small);
    default: return {};
    }
}

// ---- the join --------------------------------------------------------------------

// One wave per (item, row).  Shared items: out = sum_i a_i 2^(m_i - M) / sum_i l_i
// 2^(m_i - M) over the records.  Sequences without a key give zeros, those whose
// length is invalid NaN.  Lanes are as many shares of the records as rows of
// V-column pieces fit the wave (V = 4 where the head width allows), each summed in
// record order, and the shares in order; lane i forms the weight of record i of
// 64.  Bound by two dependent reads, of what other XCDs' blocks wrote, and by the
// code's own fetch: 4.5 to 4.7 us (0.2 to 1 more with the records read once the
// weights are formed, up to 12.8 with a condition on the loads, 5.1 to 6.1 for a
// block of 256 threads with barriers).
template <int V>
__global__ __launch_bounds__(64) void paged_gqa_join_kernel(PagedAttention p)
{
    typedef float piece __attribute__((ext_vector_type(V)));
    const uint32_t heads = p.shape.kv_heads * p.row_tiles, d = p.shape.head_dim;
    const uint32_t lane = threadIdx.x;
    const uint32_t item = blockIdx.x, row = blockIdx.y;
    const ItemShare share = item_shares(p)[item];  // unset where there is no key
    const uint32_t sequence = item / heads, head = item - sequence * heads;
    uint32_t kv_head = head, row_tile = 0;
    if (p.row_tiles > 1) {
        kv_head = head / p.row_tiles;
        row_tile = head - kv_head * p.row_tiles;
    }
    const uint32_t in_group = row_tile * p.rows + row;
    if (in_group >= p.group)
        return;
    float *out = p.out + (uint64_t(sequence) * p.query_heads + kv_head * p.group + in_group) * d;
    const uint32_t length = length_of(p, sequence);
    if (length == 0 || length == UINT32_MAX) {
        for (uint32_t c = lane; c < d; c += 64)
            out[c] = length ? __builtin_nanf("") : 0.0f;
        return;
    }
    if (!share.count)
        return;
    const auto record = [&](uint32_t i) {
        return uint64_t(i ? share.first / 2 * 2 + 2 * i : share.first) * p.rows + row;
    };
    const v2f *stats = reinterpret_cast<const v2f *>(record_stats(p));
    const uint32_t columns = d / V;
    const uint32_t width = columns < 64 ? columns : 64, shares = 64 / width;
    const uint32_t mine = lane / width;  // lanes past the last share add to none
    // kHeld records a lane in flight, the next ones behind the arithmetic: loads
    // without a condition, under which the compiler waits for each.
    constexpr uint32_t kHeld = 8;
    struct At {
        uint32_t column, group, n;  // of 64 records
    } at = {0, 0, 0};
    piece next[kHeld];
    const auto load = [&] {
        const uint32_t c = at.column + lane % width;
#pragma unroll
        for (uint32_t u = 0; u < kHeld; ++u) {
            const uint32_t i = at.group + at.n + u * shares + mine;
            next[u] = *reinterpret_cast<const piece *>(
                p.records + record(i < share.count ? i : share.count - 1) * d +
                (c < columns ? c : 0) * V);
        }
    };
    load();
    v2f stat = stats[record(lane < share.count ? lane : 0)];
    float most = stat[0];
#pragma unroll 1
    for (uint32_t i = lane + 64; i < share.count; i += 64)
        most = fmaxf(most, stats[record(i)][0]);
    most = wave_max(most);
    const float base = most == -__builtin_inff() ? 0.0f : most;
    float total = 0.0f, weight = 0.0f;
    piece a = {};
#pragma unroll 1
    while (at.column < columns) {
        const At now = at;
        const uint32_t c = now.column + lane % width;
        const uint32_t left = share.count - now.group, count = left < 64 ? left : 64;
        if (now.n == 0) {
            if (now.group || now.column)
                stat = stats[record(now.group + (lane < count ? lane : 0))];
            weight = __builtin_amdgcn_exp2f(stat[0] - base);
            if (now.column == 0)
                total += lane < count ? stat[1] * weight : 0.0f;
        }
        piece held[kHeld];
#pragma unroll
        for (uint32_t u = 0; u < kHeld; ++u)
            held[u] = next[u];
        at.n += kHeld * shares;
        if (at.n >= count) {
            at.n = 0;
            at.group += 64;
            if (at.group >= share.count) {
                at.group = 0;
                at.column += width;
            }
        }
        if (at.column < columns)
            load();
#pragma unroll
        for (uint32_t u = 0; u < kHeld; ++u) {
            const uint32_t i = now.n + u * shares + mine;
            const float w = __shfl(weight, int(i & 63), 64);
            if (i < count)
                a += w * held[u];
        }
        if (at.column == now.column)
            continue;
        if (now.column == 0)
            total = wave_sum(total);
        piece sum = a;
#pragma unroll 1
        for (uint32_t s = 1; s < shares; ++s)
#pragma unroll
            for (int e = 0; e < V; ++e)
                sum[e] += __shfl(a[e], int((lane + s * width) & 63), 64);
        if (mine == 0 && c < columns)
            *reinterpret_cast<piece *>(out + c * V) = sum / total;
        a = piece{};
    }
}

}  // namespace

bool paged_gqa_plan(PagedAttention &p, int cu_count)
{
    const uint32_t d = p.shape.head_dim;
    const MfmaKernel mfma = mfma_kernel(p.shape);
    const uint32_t most_rows =
        mfma.run || kGeneralLds / d >= kRowsMost ? kRowsMost : kGeneralLds / d;
    p.rows = p.group < most_rows ? p.group : most_rows;
    p.row_tiles = (p.group + p.rows - 1) / p.rows;
    // A unit is a wave's tile, and a block has one for each wave at least; all
    // blocks are resident at once.
    p.unit_shift = !mfma.run ? 6 : p.shape.half ? 5 : 4;
    p.least_shift = mfma.run ? 2 : 0;
    static_assert(kGeneralKeys == 1 << 6 && kWaves == 1 << 2, "shifts of a unit");
    const uint64_t items = uint64_t(p.sequences) * p.shape.kv_heads * p.row_tiles;
    const uint64_t longest = uint64_t(p.max_pages) << p.shape.page_shift;
    p.item_units = mfma.run ? kItemUnits : 0;
    p.longest = float(longest < (1u << 24) ? longest : 1u << 24);
    const uint64_t per_item = (longest >> p.unit_shift) + 1 + p.item_units;
    // Units stay in 32 bits, and so do the join's threads, 64 for each row.
    if (items * p.rows > (uint64_t(1) << 25) || items > (uint64_t(1) << 31) / per_item)
        return false;
    const uint64_t most_blocks = uint64_t(cu_count) * (mfma.run ? mfma.resident : 4);
    const uint64_t wanted = (items * per_item + (1u << p.least_shift) - 1) >> p.least_shift;
    p.blocks = uint32_t(wanted < most_blocks ? wanted : most_blocks);
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
    const MfmaKernel mfma = mfma_kernel(p.shape);
    if (p.blocks && mfma.run) {
        const size_t bytes =
            (size_t(kWaves) * p.rows * p.shape.head_dim + kWaves * 16 * 2) * sizeof(float);
        mfma.run<<<p.blocks, kBlock, bytes, stream>>>(p);
    } else if (p.blocks) {
        const size_t bytes =
            (2 * size_t(p.rows) * p.shape.head_dim + size_t(p.rows) * (kGeneralKeys + 3)) *
            sizeof(float);
        if (p.shape.half)
            paged_gqa_general_kernel<_Float16><<<p.blocks, kBlock, bytes, stream>>>(p);
        else
            paged_gqa_general_kernel<float><<<p.blocks, kBlock, bytes, stream>>>(p);
    }
    const dim3 blocks(unsigned(items), p.rows);
    if (p.shape.head_dim % 4 == 0)
        paged_gqa_join_kernel<4><<<blocks, 64, 0, stream>>>(p);
    else
        paged_gqa_join_kernel<1><<<blocks, 64, 0, stream>>>(p);
}

}  // namespace mfh
