// Attention of runs of new tokens (trees of drafted ones, or a prompt's) over paged
// caches of keys and values, or of latents.
//
// o = sum_j p_j v_j / sum_j p_j over the keys j that a token attends, with p_j =
// exp(s_j - max s) and s_j = q . k_j scale: all of the sequence's cached tokens and those
// of the run that its mask names.
#include <type_traits>

#include "digits.hpp"
#include "draft.hpp"
#include "kernels.hpp"

namespace mfh {
namespace {

// ---- any width -----------------------------------------------------------------

// A wave per (token, query head): 64 keys at a time, a lane forms one key's score, then the
// lanes are columns of the values.  Every token and head reads the cache for itself, a
// lane a row of its own: bound by the latency of scattered reads.  The cases given below
// take 37 to 300 times as long (one tree 749 us, 48 trees 14.6 ms); it is for widths that
// have no kernel there.
__global__ __launch_bounds__(64) void run_attention_general_kernel(RunAttention p)
{
    extern __shared__ float lds[];
    const uint32_t d = p.shape.head_dim, dv = p.value_dim, lane = threadIdx.x;
    const uint32_t t = uint32_t(blockIdx.x / p.query_heads);
    const uint32_t h = uint32_t(blockIdx.x - uint64_t(t) * p.query_heads), kv = h / p.group;
    float *q = lds, *acc = lds + d;
    // The token's sequence.
    uint32_t s = t, begin = t, end = t + 1;
    if (p.runs.starts) {
        s = UINT32_MAX;
        for (uint32_t base = 0; base < p.runs.sequences && s == UINT32_MAX; base += 64) {
            RunBounds b;
            const bool mine = base + lane < p.runs.sequences;
            const bool ok = !mine || valid_bounds(p.runs, base + lane, b);
            const uint64_t wrong = __ballot(!ok);
            const uint64_t found = __ballot(mine && ok && t >= b.begin && t < b.end);
            const uint32_t first = found ? uint32_t(__builtin_ctzll(found)) : 64;
            if (wrong && uint32_t(__builtin_ctzll(wrong)) < first)
                return;
            if (found) {
                s = base + first;
                begin = __shfl(b.begin, int(first), 64);
                end = __shfl(b.end, int(first), 64);
            }
        }
        if (s == UINT32_MAX)
            return;
    }
    float *out = p.out + (uint64_t(t) * p.query_heads + h) * dv;
    const float given = p.runs.lengths[s];
    if (!valid_length(given, end - begin, p.longest)) {
        for (uint32_t c = lane; c < dv; c += 64)
            out[c] = __builtin_nanf("");
        return;
    }
    const uint32_t length = uint32_t(given), number = t - begin;
    const uint32_t keys = length + (p.mask ? end - begin : number + 1);
    for (uint32_t c = lane; c < d; c += 64)
        q[c] = c < dv ? p.query[(uint64_t(t) * p.query_heads + h) * dv + c]
                      : p.rotary_query[(uint64_t(t) * p.query_heads + h) * (d - dv) + c - dv];
    for (uint32_t c = lane; c < dv; c += 64)
        acc[c] = 0.0f;
    __syncthreads();
    const float *table = p.tables + uint64_t(s) * p.max_pages;
    const uint8_t *mask = p.mask + uint64_t(t) * p.mask_bytes;
    const auto value = [&](const void *pages, uint64_t at) {
        return p.shape.half ? float(static_cast<const _Float16 *>(pages)[at])
                            : static_cast<const float *>(pages)[at];
    };
    float most = -__builtin_inff(), total = 0.0f;
    bool bad = false;
    for (uint32_t base = 0; base < keys; base += 64) {
        const uint32_t key = base + lane, i = key - length;
        bool seen = key < keys;
        if (seen && key >= length && p.mask)
            seen = i < 8ull * p.mask_bytes && (mask[i >> 3] >> (i & 7) & 1);
        uint64_t row = 0;
        if (seen) {
            const float id = table[key >> p.shape.page_shift];
            const bool ok = valid_index(id, p.shape.pages);
            bad |= !ok;
            seen = ok;
            row = ok ? uint64_t(uint32_t(id)) * p.shape.stride() +
                           ((uint64_t(kv) << p.shape.page_shift) +
                            (key & (p.shape.page_size() - 1))) * d
                     : 0;
        }
        float score = -__builtin_inff();
        if (seen) {
            float dot = 0.0f;
            for (uint32_t c = 0; c < d; ++c)
                dot += q[c] * value(p.key_pages, row + c);
            score = dot * p.scale;
        }
        float top = score;
#pragma unroll
        for (int offset = 32; offset > 0; offset >>= 1)
            top = fmaxf(top, __shfl_xor(top, offset, 64));
        top = fmaxf(top, most);
        // While every score is -infinity, nothing is added.
        const float line = top == -__builtin_inff() ? 0.0f : top;
        const float rescale = exp2f(most - line);
        const float weight = seen ? exp2f(score - line) : 0.0f;
        most = top;
        float sum = weight;
#pragma unroll
        for (int offset = 32; offset > 0; offset >>= 1)
            sum += __shfl_xor(sum, offset, 64);
        total = total * rescale + sum;
        const uint64_t some = __ballot(seen);
        for (uint32_t c0 = 0; c0 < dv; c0 += 64) {
            const uint32_t c = c0 + lane < dv ? c0 + lane : dv - 1;
            float add = 0.0f;
            for (uint64_t left = some; left; left &= left - 1) {
                const int j = __builtin_ctzll(left);
                const uint32_t low = __shfl(uint32_t(row), j, 64);
                const uint32_t high = __shfl(uint32_t(row >> 32), j, 64);
                add += __shfl(weight, j, 64) *
                       value(p.value_pages, (uint64_t(high) << 32 | low) + c);
            }
            if (c0 + lane < dv)
                acc[c] = acc[c] * rescale + add;
        }
    }
    const float poison = __any(bad) ? __builtin_nanf("") : 0.0f;
    for (uint32_t c = lane; c < dv; c += 64)
        out[c] = (total == 0.0f ? 0.0f : acc[c] / total) + poison;
}

// ---- matrix cores ---------------------------------------------------------------
//
// Query rows of a key/value head are (token, head of the group) pairs, counted through a run.
// An item is (sequence, key/value head, a tile of its rows); a block walks the item's keys a
// tile at a time, which all its waves share in LDS, a wave having 16 or 32 of the rows, or
// (SPLIT waves to the same 16) a part of the key columns for the scores and of the value
// columns for the output: one wave cannot hold queries and outputs 512 wide.  Per tile,
// S^T = K Q^T leaves query row j in lane column j (lane 16 q + j holds the scores of keys
// 16 c + 4 q + r in register r of block c), the softmax follows online in the row's four
// lanes, and O^T += V^T P^T takes those registers as its second operand, so that
// probabilities never pass through LDS; its first is put together from pieces of eight key
// rows.
//
// Binary16 caches: keys and values are operands as they are, queries (scaled by a power of
// two to below 2^15) and probabilities (times 2^12, up to 2^15) two binary16 parts each.  They
// are within 2^-23 of the value from 2^-2 on and within 2^-25 of smaller ones (a second part
// below 2^-14 has fewer bits), which is 2^-39 of a row's largest query column and 2^-37 of its
// largest probability, or less.  f32 caches: all four are three bfloat16 parts, which hold 24
// bits, and six of the nine products are formed (the others are below 2^-26).  Six
// products of 16 bits take 6/16 of the cycles of one of f32.
//
// Tiles of binary16 whose rows are whole groups of 64 columns are copied straight to LDS,
// two to four stages ahead of the products: no registers, no instructions to store them, the
// page ids of 256 runs of eight keys looked up at once.  Others pass through registers: f32
// for its parts, other widths for their padding.
//
// The work is a line of units (a tile of keys; items in order, item_units besides for each),
// which every block adds up itself, for starts and lengths live on the device, and takes
// an equal run of.  A block that holds all tiles of an item writes its rows; the others
// store records (maximum, sum, unnormalised output) that a second launch joins in block
// order, so that results do not depend on timing.
//
// What bounds it, in us of a call (the time of its bytes at a copy's 4.7 TB/s, or of its
// products at the 1083 TFLOP/s of a large one):
// - few rows over long caches, the cache's reads: 48 trees of 4 to 32 tokens over 17 to 8191
//   keys, 32 / 8 heads of 128, binary16, 90 (63); 64 tokens of 16 heads over 100 to
//   8191 latents of 512 + 64 49 (30);
// - prompts, products and the vector instructions between them, in turn: 2048 tokens over 2048,
//   32 / 8 heads of 64, 138 to 160 (95 with both parts of queries and probabilities); of
//   the SIMDs' 256 M cycles matrix cores are busy in 102 M, and the 30.7 M other vector
//   instructions take about 123 M; 1024 over 1024 latents, 32 heads, 300 to 345 (202);
// - f32 caches, six products for one and the parts of every tile: the prompt above 435 (278), 48
//   trees as above 262 (121);
// - single sequences, the chain of a launch's dependent reads (starts, page ids, queries, a
//   tile) and the join's: 16 tokens over 2047 keys of 64, f32, 20, the smallest call (a
//   tree over 127 keys) 14.  One token over the same keys takes 17 here and 11 in the
//   kernel for single tokens, whose chain is shorter.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kBlock = 256;
// An item's queries, records and rows cost about five tiles: 48 trees as above take 99 us at 4,
// 95 at 5, 92 at 6, 48 x 8 tokens over 2047 keys 101, 104 and 105, the prompt of heads of 64
// 144, 144 and 147, trees over f32 caches 257, 259 and 266.  Where a CU has three blocks, of
// tiles of 32 keys, eight (48 x 32 tokens over 2047 keys 160 us at 6, 157 to 165 at 8, 161
// at 10).
constexpr uint32_t kItemUnits = 5, kItemUnitsOfThree = 8;
// Units of a block: of more than one, a short call leaves CUs empty (one tree as above 20
// us at 1, 28 at 4).
constexpr uint32_t kLeastUnits = 1;
constexpr uint32_t kMostBlocks = 1024;
// A row's maximum is followed once it has risen by kSlack (powers of two), which the
// probabilities are below then; binary16 ones are times 2^kProbabilityShift.  Most tiles
// then leave the outputs as they are (the prompts above 161 and 333 us; with every rise
// followed 163 and 344).
constexpr float kSlack = 3.0f, kProbabilityShift = 12.0f;

// What a block's first unfinished item needs of the join.
struct Share {
    uint32_t count, record;          // records (0: none), the first one
    uint32_t begin, run, kv_head, row_tile;
};

__host__ __device__ inline float *record_stats(const RunAttention &p)
{
    return p.records + 2 * uint64_t(p.blocks) * p.rows * p.value_dim;
}
__host__ __device__ inline Share *block_shares(const RunAttention &p)
{
    return reinterpret_cast<Share *>(record_stats(p) + 4 * uint64_t(p.blocks) * p.rows);
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
__device__ __forceinline__ uint32_t scalar(uint32_t v)
{
    return uint32_t(__builtin_amdgcn_readfirstlane(v));
}

// A sequence's run: its tokens, and the keys before it, UINT32_MAX for a bad length.
struct Run {
    uint32_t begin = 0, count = 0, length = 0;
};

// Sequence i's run; false where the list of starts ends at it.
__device__ __forceinline__ bool load_run(const RunAttention &p, uint32_t i, Run &run)
{
    RunBounds b;
    b.begin = i;
    b.end = i + 1;
    const bool ok = !p.runs.starts || valid_bounds(p.runs, i, b);
    const float length = p.runs.lengths[i];
    run.begin = b.begin;
    run.count = b.end - b.begin;
    run.length = valid_length(length, run.count, p.longest) ? uint32_t(length) : UINT32_MAX;
    return ok;
}

// Units of a sequence's items, SHIFT the logarithm of a tile's keys.  Where tokens attend
// all before them, a later item has more keys: `step` tiles more after every `every` items,
// in whole numbers, so that the sum has a closed form.
template <int SHIFT>
struct Units {
    uint32_t base, step, every;  // step 0: all items alike
    __device__ __forceinline__ Units(const RunAttention &p, const Run &run)
    {
        constexpr uint32_t KEYS = 1u << SHIFT;
        base = p.item_units;
        step = 0;
        every = 1;
        if (run.length == UINT32_MAX)
            return;
        if (p.mask || run.count == 1) {
            base += (run.length + run.count + KEYS - 1) >> SHIFT;
        } else {
            step = p.rows < KEYS ? 1 : p.rows / KEYS;
            every = p.rows < KEYS ? KEYS / p.rows * p.group : p.group;
            base += ((run.length + KEYS - 1) >> SHIFT) + step;
        }
    }
    __device__ __forceinline__ uint32_t of(uint32_t tile) const
    {
        return base + (step ? tile / every * step : 0);
    }
    // Of the first `tiles` items.
    __device__ __forceinline__ uint32_t upto(uint32_t tiles) const
    {
        uint32_t sum = tiles * base;
        if (step) {
            const uint32_t whole = tiles / every, left = tiles - whole * every;
            sum += step * (every * (whole * (whole - 1) / 2) + whole * left);
        }
        return sum;
    }
};
__device__ __forceinline__ uint32_t row_tiles(const RunAttention &p, const Run &run)
{
    return (run.count * p.group + p.rows - 1) / p.rows;
}

// A block's place on the line of units: block b of n starts at floor(b total / n).
struct Line {
    uint32_t sequence, kv_head, row_tile, unit;  // the item of the next unit
    Run run;
    uint32_t start, at, end, total, blocks, block;
};

template <int SHIFT>
__device__ __forceinline__ bool find_line(const RunAttention &p, Line &line)
{
    const uint32_t lane = threadIdx.x & 63, heads = p.shape.kv_heads;
    Run run;
    uint32_t total = 0, scan = 0, mine = 0;
    const auto load = [&](uint32_t base) {
        const uint32_t i = base + lane < p.runs.sequences ? base + lane : p.runs.sequences - 1;
        const uint64_t wrong = __ballot(!load_run(p, i, run));
        if (base + lane >= p.runs.sequences || (wrong << (63 - lane)) != 0)
            run = Run();
        mine = run.count ? heads * Units<SHIFT>(p, run).upto(row_tiles(p, run)) : 0;
        scan = lanes_scan(mine);
        return wrong == 0;
    };
    for (uint32_t base = 0; base < p.runs.sequences; base += 64) {
        const bool more = load(base);
        total += __builtin_amdgcn_readlane(scan, 63);
        if (!more)
            break;
    }
    const uint32_t most = (total + kLeastUnits - 1) / kLeastUnits;
    const uint32_t blocks = most < p.blocks ? most : p.blocks;
    // Neighbours on the line share an XCD's cache where all blocks have work.
    uint32_t b = blockIdx.x;
    if (blocks == p.blocks && blocks % 8 == 0)
        b = b % 8 * (blocks / 8) + b / 8;
    line.block = b;
    if (b >= blocks)
        return false;
    line.total = total;
    line.blocks = blocks;
    const uint32_t quotient = total / blocks, odd = total - quotient * blocks;
    line.start = line.at = b * quotient + b * odd / blocks;
    line.end = (b + 1) * quotient + (b + 1) * odd / blocks;
    uint32_t before = 0, base = 0;
    for (;; base += 64) {
        if (p.runs.sequences > 64)
            load(base);
        const uint32_t sum = __builtin_amdgcn_readlane(scan, 63);
        if (line.at < before + sum)
            break;
        before += sum;
    }
    const uint32_t from = __builtin_ctzll(__ballot(line.at < before + scan));
    const auto of = [&](uint32_t v) { return uint32_t(__builtin_amdgcn_readlane(v, from)); };
    line.sequence = base + from;
    line.run.begin = of(run.begin);
    line.run.count = of(run.count);
    line.run.length = of(run.length);
    const uint32_t inside = line.at - before - of(scan) + of(mine);
    const Units<SHIFT> units(p, line.run);
    const uint32_t tiles = row_tiles(p, line.run), each = units.upto(tiles);
    line.kv_head = inside / each;
    const uint32_t left = inside - line.kv_head * each;
    // The last tile that starts at or before `left`.
    uint32_t low = 0, high = tiles;
    while (high - low > 1) {
        const uint32_t middle = (low + high) / 2;
        if (units.upto(middle) <= left)
            low = middle;
        else
            high = middle;
    }
    line.row_tile = low;
    line.unit = left - units.upto(low);
    return true;
}

// The block that has a unit: the quotient of whole numbers below 2^53, so the rounded one
// is below the next whole number where the exact one is.
__device__ __forceinline__ uint32_t block_of(const Line &line, uint32_t unit)
{
    const double after = (double(unit) + 1.0) * double(line.blocks) - 1.0;
    return uint32_t(after / double(line.total));
}

// The part of an item that a block holds.
struct Part {
    uint32_t sequence, kv_head, row_tile;
    Run run;
    uint32_t keys;         // of the item
    uint32_t first, last;  // tiles, from first to before last
    bool whole, leads;     // all of the item; its first tiles
    bool opens;            // its first unit
    bool counts;           // has a place among the item's records
    uint32_t record, last_unit;
};

template <int SHIFT>
__device__ __forceinline__ bool next_part(const RunAttention &p, Line &line, Part &part)
{
    if (line.at >= line.end)
        return false;
    while (!line.run.count) {  // at < end: another unit follows
        Run run;
        load_run(p, ++line.sequence, run);
        line.run.begin = scalar(run.begin);
        line.run.count = scalar(run.count);
        line.run.length = scalar(run.length);
    }
    const Run &run = line.run;
    const uint32_t units = Units<SHIFT>(p, run).of(line.row_tile);
    const uint32_t left = units - line.unit;
    const uint32_t take = left < line.end - line.at ? left : line.end - line.at;
    const uint32_t from = line.unit, to = line.unit + take;
    part.sequence = line.sequence;
    part.kv_head = line.kv_head;
    part.row_tile = line.row_tile;
    part.run = run;
    part.keys = 0;
    if (run.length != UINT32_MAX) {
        // The item's last row is of this token.
        const uint32_t token = (p.rows * line.row_tile + p.rows - 1) / p.group;
        part.keys = run.length + (p.mask || token >= run.count ? run.count : token + 1);
    }
    const uint32_t tiles = (part.keys + (1u << SHIFT) - 1) >> SHIFT;
    // The item's last units may be more or fewer than its tiles.
    const auto tile_at = [&](uint32_t unit) {
        const uint32_t t = unit > p.item_units ? unit - p.item_units : 0;
        return unit == units || t > tiles ? tiles : t;
    };
    part.first = tile_at(from);
    part.last = tile_at(to);
    part.leads = from <= p.item_units;
    part.opens = from == 0;
    part.counts = to > p.item_units;
    part.whole = part.leads && to == units;
    part.record = 2 * line.block + (line.at == line.start ? 0 : 1);
    part.last_unit = line.at - from + units - 1;
    line.at += take;
    line.unit = to;
    if (to == units) {
        line.unit = 0;
        if (++line.row_tile == row_tiles(p, run)) {
            line.row_tile = 0;
            if (++line.kv_head == p.shape.kv_heads) {
                line.kv_head = 0;
                line.run.count = 0;
            }
        }
    }
    return true;
}

// Chunks of a value row: as many 16-column tiles as one LDS read holds (16 bytes, then 8,
// 4, 2).
__host__ __device__ constexpr int chunk_tiles(int left, int most)
{
    int s = most;
    while (s > left)
        s /= 2;
    return s;
}
// f(first tile, tiles) for each chunk of N tiles, both as constants.
template <int N, int MOST, int T = 0, typename F>
__device__ __forceinline__ void for_chunks(F f)
{
    if constexpr (T < N) {
        constexpr int S = chunk_tiles(N - T, MOST);
        f(std::integral_constant<int, T>{}, std::integral_constant<int, S>{});
        for_chunks<N, MOST, T + S>(f);
    }
}

// Maximum and sum over a row's four lanes (q = 0..3).
__device__ __forceinline__ float quad_max(float v)
{
    const uint32_t x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t y = __float_as_uint(v);
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float v)
{
    const uint32_t x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const uint32_t y = __float_as_uint(v);
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A pair of values as PARTS operand parts, the largest first: each is the nearest to what
// the ones before it left.
template <bool HALF, int PARTS>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&out)[PARTS])
{
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        if constexpr (HALF) {
            out[i] = __builtin_bit_cast(uint32_t, v2h{_Float16(a), _Float16(b)});
            if (i + 1 < PARTS) {
                // What is left, from the packed halves as they are: a - half in one
                // instruction.
                const float x = a, y = b;
                asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]"
                    : "=v"(a) : "v"(out[i]), "v"(x));
                asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
                    : "=v"(b) : "v"(out[i]), "v"(y));
            }
        } else {
            out[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2b));
            a -= __uint_as_float(out[i] << 16);
            b -= __uint_as_float(out[i] & 0xffff0000u);
        }
    }
}

template <bool HALF>
__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c)
{
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                      __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a),
                                                       __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

// Elements between LDS rows that pass through registers, of D 16-bit columns: 16 bytes more
// than the row, so that 16 rows' pieces of one column fall on all banks, at places that
// differ by constants.
template <int D>
constexpr int kPitch = D + 8;

// The value, which the compiler takes for a new one: what rarely run code forms from it is
// formed there, not held in registers around the loop.
__device__ __forceinline__ uint32_t formed_here(uint32_t v)
{
    asm volatile("" : "+v"(v));
    return v;
}

// What a kernel of a width has in a tile, in LDS and on a CU.  A wave has GROUPS times 16
// rows; SPLIT waves share them, each with a part of the key columns for the scores and of
// the value columns for the output.
template <int DK, int DV, bool HALF, bool LATENT, int WAVES, int SPLIT, int GROUPS, int RESIDENT>
struct Shape {
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int ROWS = 16 * GROUPS * WAVES / SPLIT;
    static constexpr int PARTS = HALF ? 1 : 3;          // of keys and values
    static constexpr int QUERY_PARTS = HALF ? 2 : 3;    // of queries and probabilities
    static constexpr int SHIFT = RESIDENT < 3 && DK * GROUPS <= (HALF ? 128 : 64) ? 6 : 5;
    static constexpr int KEYS = 1 << SHIFT;
    // Copied to LDS without passing through registers: rows as they are, of which eight
    // are whole copies of a wave.
    static constexpr bool COPIED = HALF && DK % 64 == 0;
    static constexpr int PITCH = COPIED ? DK : kPitch<DK>;
    static constexpr int KEY_PLANE = KEYS * PITCH, VALUE_PLANE = LATENT ? 0 : KEY_PLANE;
    static constexpr int STAGE = PARTS * (KEY_PLANE + VALUE_PLANE);  // 16-bit elements
    // Of a CU's 160 KB of LDS, beside the scores that waves exchange.
    static constexpr int ROOM = (SPLIT > 1 ? 61440 : 73728) / RESIDENT / STAGE;
    static constexpr int STAGES = !HALF ? 1 : !COPIED || ROOM < 2 ? 2 : ROOM < 4 ? ROOM : 4;
    static constexpr int CHUNK = SPLIT > 1 ? 4 : 8;     // most tiles of a value chunk
};

// 16-byte loads of a tile's rows of D columns, by wave: each load is of one run of eight
// keys, which one page holds, so that its page is the wave's and its lanes' places in
// the run never change.
template <typename T, int D, int KEYS, int WAVES>
struct Loads {
    static constexpr int PIECE = 16 / sizeof(T);      // columns of a load
    static constexpr int CHUNKS = 8 * D / PIECE;      // of eight keys
    static constexpr int EACH = (CHUNKS + 63) / 64;   // loads of eight keys
    static constexpr int ALL = KEYS / 8 * EACH;
    static constexpr int MINE = (ALL + WAVES - 1) / WAVES;
    __device__ __forceinline__ static uint32_t number(int i, uint32_t wave)
    {
        const uint32_t n = wave + i * WAVES;
        return (i + 1) * WAVES > ALL && n >= uint32_t(ALL) ? ALL - 1 : n;
    }
    // The lane's chunk of the eight keys; past their end the last one again.
    __device__ __forceinline__ static uint32_t chunk(uint32_t n, uint32_t lane)
    {
        const uint32_t c = n % EACH * 64 + lane;
        return CHUNKS % 64 != 0 && c >= uint32_t(CHUNKS) ? CHUNKS - 1 : c;
    }
};

// Copied rows hold their 16-byte chunks in an order of their own, chunk c at c ^ turn(row) of
// its group of G, by which 16 rows' equal chunks fall on all banks.  16-byte reads are served
// for lanes 0-3, 12-15, 20-27 (and 4-11, 16-19, 28-31) together: of keys these are the
// chunks c and c + 1 of rows, of values half the chunks of two rows 4 apart, which a turn
// by the row alone would put on the same banks (a conflict each: 48 sequences of 32 tokens
// over 2047 keys of 128 173 us against 168, one of 16 over 65535 78 against 74).
template <int D>
struct Turned {
    static constexpr uint32_t G = D / 8 % 16 == 0 ? 16 : 8;
    __device__ __forceinline__ static uint32_t turn(uint32_t row)
    {
        const uint32_t r = row / (16 / G) & (G - 1);
        return G == 16 ? r ^ (r & 4) << 1 : r;
    }
    __device__ __forceinline__ static uint32_t place(uint32_t row, uint32_t chunk)
    {
        return (chunk & ~(G - 1)) + ((chunk ^ turn(row)) & (G - 1));
    }
};

// Waits until at most `count` of the wave's loads and copies are on their way.
template <int COUNT>
__device__ __forceinline__ void wait_loads()
{
    __builtin_amdgcn_s_waitcnt(0x0f70 | (COUNT & 15) | (COUNT >> 4) << 14);
}

constexpr uint32_t kHeld = 512;  // places of runs of eight keys, in LDS

template <int DK, int DV, bool HALF, bool LATENT, int WAVES, int SPLIT, int GROUPS, int RESIDENT>
__global__ __launch_bounds__(64 * WAVES, (RESIDENT * WAVES / 4))
void run_attention_kernel(RunAttention p)
{
    using S = Shape<DK, DV, HALF, LATENT, WAVES, SPLIT, GROUPS, RESIDENT>;
    using T = typename std::conditional<HALF, _Float16, float>::type;
    static_assert(DK % (SPLIT > 1 ? 32 : 16) == 0 && DV % (16 * SPLIT) == 0,
                  "widths of the matrix-core path");
    constexpr int KEYS = S::KEYS, SHIFT = S::SHIFT, PARTS = S::PARTS, QP = S::QUERY_PARTS;
    constexpr uint32_t ROWS = S::ROWS;
    constexpr int NB = KEYS / 16;                  // key blocks of a tile
    constexpr int DEPTHS = (DK + 31) / 32;         // product depths of a key row
    constexpr int U = (DEPTHS + SPLIT - 1) / SPLIT;  // of them a wave's
    constexpr int N = DV / 16 / SPLIT;             // the wave's 16-column tiles of the output
    using Load = Loads<T, DK, KEYS, WAVES>;        // values are as wide, or the keys
    __shared__ __attribute__((aligned(16))) uint16_t lds[S::STAGES * S::STAGE];
    __shared__ v4f partial[SPLIT > 1 ? WAVES * GROUPS * NB * 64 : 1];
    __shared__ uint32_t flags[3][2];  // keys of a tile that are marked, by bit
    __shared__ uint2 held[S::COPIED ? kHeld : 1];  // bytes from the cache's first; bit 63: no page
    __shared__ uint32_t any_bad;
    constexpr bool COPIED = S::COPIED;
    constexpr int STAGES = S::STAGES, PITCH = S::PITCH, THREADS = S::THREADS;
    using Order = Turned<DK>;

    const uint32_t lane = threadIdx.x & 63, q = lane >> 4, j = lane & 15;
    const uint32_t wave = scalar(threadIdx.x >> 6), split = wave % SPLIT;
    const uint32_t wave_row = 16 * GROUPS * (wave / SPLIT);  // the wave's first of the item's
    const uint32_t page_shift = p.shape.page_shift, in_page = p.shape.page_size() - 1;
    // The lane's places in a load: bytes from its first key's row, and elements in LDS,
    // which are held where they are few.
    constexpr uint32_t PER_ROW = DK / Load::PIECE;
    constexpr bool HELD = Load::MINE <= 5 && DK != 256 && !COPIED, OWN_AT = COPIED || Load::CHUNKS % 64 != 0;
    uint32_t load_at[OWN_AT ? Load::MINE : 1], store_held[HELD ? Load::MINE : 1];
    const auto place = [&](int i, uint32_t me) {
        const uint32_t n = Load::number(i, wave), c = Load::chunk(n, me);
        const uint32_t row = c / PER_ROW, piece = c - row * PER_ROW;
        return (8 * (n / Load::EACH) + row) * PITCH + piece * Load::PIECE;
    };
    const auto store_at = [&](int i) {
        return HELD ? store_held[HELD ? i : 0] : place(i, formed_here(lane));
    };
    load_at[0] = lane * 16;
#pragma unroll
    for (int i = 0; i < Load::MINE; ++i) {
        const uint32_t n = Load::number(i, wave), c = Load::chunk(n, lane);
        if (COPIED) {
            // What belongs to the chunk of LDS that the lane writes.
            const uint32_t row = c / PER_ROW;
            load_at[i] = (row * PER_ROW +
                          Order::place(8 * (n / Load::EACH) + row, c - row * PER_ROW)) * 16;
        } else if (OWN_AT) {
            load_at[i] = c * 16;
        }
        if (HELD)
            store_held[i] = place(i, lane);
    }
    const uint32_t lds_at = uint32_t(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) uint16_t *)&lds[0]));
    Line line;
    const bool any = find_line<SHIFT>(p, line);
    Share share = {};
    Part part;
    while (any && next_part<SHIFT>(p, line, part)) {
        const uint32_t rows = part.run.count * p.group, row0 = ROWS * part.row_tile;
        const bool active = row0 + wave_row < rows;
        bool real[GROUPS];
        uint32_t token[GROUPS];      // of the run
        uint64_t query_row[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            uint32_t row = row0 + wave_row + 16 * g + j;
            real[g] = row < rows;
            row = real[g] ? row : rows - 1;
            token[g] = row / p.group;
            query_row[g] = uint64_t(part.run.begin + token[g]) * p.query_heads +
                           part.kv_head * p.group + row - token[g] * p.group;
            if (part.run.length == UINT32_MAX && part.opens && real[g])
                for (uint32_t c = q + 4 * split; c < uint32_t(DV); c += 4 * SPLIT)
                    p.out[query_row[g] * DV + c] = __builtin_nanf("");
        }
        if (part.run.length == UINT32_MAX)
            continue;
        if (!part.counts)
            continue;
        const float *table = p.tables + uint64_t(part.sequence) * p.max_pages;
        const uint32_t last_key = part.keys - 1, length = part.run.length;
        const uint64_t head_bytes =
            (uint64_t(part.kv_head) << page_shift) * DK * sizeof(T);
        const uint64_t page_bytes = p.shape.stride() * sizeof(T);

        // The first key of a load, in the last eight with a key where it is past them.
        const auto key_of = [&](uint32_t tile, int i) {
            const uint32_t key = tile * KEYS + 8 * (Load::number(i, wave) / Load::EACH);
            return key <= last_key ? key : last_key & ~7u;
        };
        // A tile's page ids, lane i the one of the wave's load i: a vector load, for a scalar
        // one would be waited for with every LDS access.
        float ids;
        const auto load_ids = [&](uint32_t tile) {
            const uint32_t i = lane < uint32_t(Load::MINE) ? lane : Load::MINE - 1;
            ids = table[key_of(tile, int(i)) >> page_shift];
        };
        v4u key_reg[Load::MINE], value_reg[LATENT ? 1 : Load::MINE];
        uint32_t bad = 0;  // loads of the tile whose page is none
        const auto load_tile = [&](uint32_t tile) {
            bad = 0;
#pragma unroll
            for (int i = 0; i < Load::MINE; ++i) {
                const float id = __uint_as_float(
                    uint32_t(__builtin_amdgcn_readlane(__float_as_int(ids), i)));
                const bool ok = valid_index(id, p.shape.pages);
                bad |= ok ? 0 : 1u << i;
                const uint32_t page = scalar(ok ? uint32_t(id) : 0);
                uint64_t at = page * page_bytes + head_bytes +
                              (key_of(tile, i) & in_page) * uint32_t(DK * sizeof(T));
                if (Load::CHUNKS % 64 == 0)
                    at += Load::number(i, wave) % Load::EACH * 1024;
                const uint32_t lane_at = load_at[OWN_AT ? i : 0];
                key_reg[i] = __builtin_nontemporal_load(reinterpret_cast<const v4u *>(
                    static_cast<const char *>(p.key_pages) + at + lane_at));
                if constexpr (!LATENT)
                    value_reg[i] = __builtin_nontemporal_load(reinterpret_cast<const v4u *>(
                        static_cast<const char *>(p.value_pages) + at + lane_at));
            }
        };
        // 16 loaded bytes into the operand planes.  In a tile that not every row attends whole,
        // what is not finite becomes zero and its key is marked: only rows that attend it
        // shall see it.
        const auto store_piece = [&](v4u x, uint16_t *to, int plane, uint32_t at, bool mixed,
                                     uint32_t turn) {
            if (mixed) {
                bool odd = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (HALF) {
                        const bool low = (x[e] & 0x7c00u) == 0x7c00u;
                        const bool high = (x[e] & 0x7c000000u) == 0x7c000000u;
                        odd |= low || high;
                        x[e] &= (low ? 0xffff0000u : ~0u) & (high ? 0xffffu : ~0u);
                    } else {
                        // The largest finite ones too: their first part would be infinite.
                        const bool all = (x[e] & 0x7fffffffu) >= 0x7f7f8000u;
                        odd |= all;
                        x[e] = all ? 0 : x[e];
                    }
                }
                if (odd) {
                    const uint32_t key = formed_here(at) / PITCH;
                    atomicOr(&flags[turn][key / 32], 1u << key % 32);
                }
            }
            if constexpr (HALF) {
                *reinterpret_cast<v4u *>(to) = x;
            } else {
                uint32_t a[PARTS], b[PARTS];
                split_pair<HALF>(__uint_as_float(x[0]), __uint_as_float(x[1]), a);
                split_pair<HALF>(__uint_as_float(x[2]), __uint_as_float(x[3]), b);
#pragma unroll
                for (int i = 0; i < PARTS; ++i)
                    *reinterpret_cast<v2u *>(to + i * plane) = v2u{a[i], b[i]};
            }
        };
        // Where the kHeld / 2 runs of eight keys from one on lie.
        const auto hold_places = [&](uint32_t first) {
            for (uint32_t i = threadIdx.x; i < kHeld / 2; i += THREADS) {
                const uint32_t key = 8 * (first + i);
                const uint32_t at = key <= last_key ? key : last_key & ~7u;
                const float id = table[at >> page_shift];
                const bool ok = valid_index(id, p.shape.pages);
                const uint64_t bytes = (ok ? uint32_t(id) : 0) * page_bytes + head_bytes +
                                       (at & in_page) * uint32_t(DK * sizeof(T));
                held[(first + i) % kHeld] =
                    uint2{uint32_t(bytes), uint32_t(bytes >> 32) | (ok ? 0 : 1u << 31)};
                if (!ok)
                    any_bad = 1;
            }
        };
        const auto starts_places = [&](uint32_t tile) {
            return tile * (KEYS / 8) % (kHeld / 2) == 0;
        };
        // Starts the copies of a tile, the same number in every wave and tile.
        constexpr int COPIES = Load::MINE * (LATENT ? 1 : 2);
        const auto copy_tile = [&](uint32_t tile, uint32_t slot) {
            const uint32_t stage = lds_at + slot * (2 * S::STAGE);
            uint2 place[Load::MINE];
#pragma unroll
            for (int i = 0; i < Load::MINE; ++i)
                place[i] = held[(tile * (KEYS / 8) + Load::number(i, wave) / Load::EACH) % kHeld];
#pragma unroll
            for (int i = 0; i < Load::MINE; ++i) {
                const uint32_t n = Load::number(i, wave);
                const uint64_t at =
                    uint64_t(scalar(place[i].y) & 0x7fffffffu) << 32 | scalar(place[i].x);
                const uint32_t to = stage + n * 1024;
                copy_to_lds(static_cast<const uint8_t *>(p.key_pages) + at, load_at[OWN_AT ? i : 0],
                            to);
                if constexpr (!LATENT)
                    copy_to_lds(static_cast<const uint8_t *>(p.value_pages) + at,
                                load_at[OWN_AT ? i : 0], to + 2 * S::KEY_PLANE);
            }
        };
        // In a copied tile, as store_piece does in a loaded one.
        const auto check_tile = [&](uint16_t *stage, uint32_t turn) {
            for (uint32_t n = threadIdx.x; n < uint32_t(S::STAGE / 8); n += THREADS) {
                v4u x = *reinterpret_cast<v4u *>(stage + 8 * n);
                bool odd = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool low = (x[e] & 0x7c00u) == 0x7c00u;
                    const bool high = (x[e] & 0x7c000000u) == 0x7c000000u;
                    odd |= low || high;
                    x[e] &= (low ? 0xffff0000u : ~0u) & (high ? 0xffffu : ~0u);
                }
                if (odd) {
                    const uint32_t key = n / (PITCH / 8) % KEYS;
                    *reinterpret_cast<v4u *>(stage + 8 * n) = x;
                    atomicOr(&flags[turn][key / 32], 1u << key % 32);
                }
            }
        };
        const auto store_tile = [&](uint16_t *stage, bool mixed, uint32_t turn) {
#pragma unroll
            for (int i = 0; i < Load::MINE; ++i) {
                const uint32_t first = 8 * (Load::number(i, wave) / Load::EACH);
                if (bad >> i & 1 && lane == 0)
                    atomicOr(&flags[turn][first / 32], formed_here(0xff) << first % 32);
                const uint32_t to = store_at(i);
                store_piece(key_reg[i], stage + to, S::KEY_PLANE, to, mixed, turn);
                if constexpr (!LATENT)
                    store_piece(value_reg[i], stage + PARTS * S::KEY_PLANE + to, S::VALUE_PLANE,
                                to, mixed, turn);
            }
        };

        if constexpr (COPIED) {
            __syncthreads();  // an earlier part's tiles and places have been read
            if (threadIdx.x == 0)
                any_bad = 0;
            __syncthreads();
            hold_places(part.first * (KEYS / 8) / (kHeld / 2) * (kHeld / 2));
            __syncthreads();
#pragma unroll
            for (int ahead = 0; ahead < STAGES - 1; ++ahead)
                if (part.first + ahead < part.last) {
                    if (ahead && starts_places(part.first + ahead)) {
                        hold_places((part.first + ahead) * (KEYS / 8));
                        __syncthreads();
                    }
                    copy_tile(part.first + ahead, ahead);
                }
        } else {
            load_ids(part.first);
            if (part.first < part.last) {
                load_tile(part.first);
                load_ids(part.first + 1 < part.last ? part.first + 1 : part.first);
            }
        }
        // The wave's queries, in parts; rows past the run's are zero.
        v4u query[GROUPS][U][QP];
        float factor[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const float *at = p.query + query_row[g] * DV;
            const auto load = [&](int u, int e) {
                const uint32_t column = 32 * (split * U + u) + 8 * q + e;
                const float *from = at + (column < uint32_t(DV) ? column : 0);
                if (LATENT && column >= uint32_t(DV))
                    from = p.rotary_query + query_row[g] * (DK - DV) +
                           (column < uint32_t(DK) ? column - DV : 0);
                const v4f piece = *reinterpret_cast<const v4f *>(from);
                const bool mine = real[g] && column < uint32_t(DK);
                return mine ? piece : v4f{0, 0, 0, 0};
            };
            v4f x[2 * U];
#pragma unroll
            for (int i = 0; i < 2 * U; ++i)
                x[i] = load(i / 2, 4 * (i % 2));
            factor[g] = p.scale;
            int exponent = 0;
            if (HALF) {
                float most = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * U; ++i)
                    most = fmaxf(fmaxf(most, fmaxf(fabsf(x[i][0]), fabsf(x[i][1]))),
                                 fmaxf(fabsf(x[i][2]), fabsf(x[i][3])));
                most = quad_max(most);
                // 2^14 <= most 2^exponent < 2^15 (0 and infinities as they are; below
                // 2^-86, where no score of an ordinary scale differs from 0, by 2^100).
                if (most > 0.0f && most < __builtin_inff())
                    exponent = 15 - __builtin_amdgcn_frexp_expf(most);
                exponent = exponent < 100 ? exponent : 100;
                factor[g] = ldexpf(p.scale, -exponent);
                // Not 0 where a masked score of -infinity meets it: scores are below 2^42, and
                // times the least normal factor as good as 0.
                if (SPLIT == 1)
                    factor[g] = fmaxf(factor[g], 0x1p-126f);
            }
#pragma unroll
            for (int i = 0; i < 2 * U; ++i)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    uint32_t parts[QP];
                    split_pair<HALF>(HALF ? ldexpf(x[i][e], exponent) : x[i][e],
                                     HALF ? ldexpf(x[i][e + 1], exponent) : x[i][e + 1], parts);
#pragma unroll
                    for (int part = 0; part < QP; ++part)
                        query[g][i / 2][part][2 * (i % 2) + e / 2] = parts[part];
                }
        }

        v4f o[GROUPS][N];
        float m[GROUPS], l[GROUPS];
        bool poison[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
#pragma unroll
            for (int t = 0; t < N; ++t)
                o[g][t] = v4f{0, 0, 0, 0};
            m[g] = -__builtin_inff();
            l[g] = 0.0f;
            poison[g] = false;
        }
        // Every row attends the keys before this one.
        const uint32_t common = length + (p.mask ? 0 : row0 / p.group + 1);
        uint32_t turn = 0, slot = 0;
        __syncthreads();  // an earlier part's tiles and marks have been read
        if (threadIdx.x < 6)
            flags[threadIdx.x / 2][threadIdx.x % 2] = 0;
        __syncthreads();
#pragma unroll 1
        for (uint32_t tile = part.first; tile < part.last; ++tile) {
            const uint32_t k0 = tile * KEYS;
            const bool mixed = k0 + KEYS > common;
            uint16_t *stage = lds + slot * S::STAGE;
            // The tile before's, free once every wave is here.
            const uint32_t slot_behind = slot ? slot - 1 : STAGES - 1;
            slot = slot == STAGES - 1 ? 0 : slot + 1;
            uint64_t marks = 0;
            const uint32_t next = tile + STAGES - 1;
            if constexpr (COPIED) {
                // This tile's copies have ended, those of the ones behind it may not have.
                const uint32_t behind = part.last - 1 - tile;
                if (STAGES >= 4 && behind >= 2)
                    wait_loads<2 * COPIES>();
                else if (STAGES >= 3 && behind >= 1)
                    wait_loads<COPIES>();
                else
                    wait_loads<0>();
                if (next < part.last && starts_places(next))
                    hold_places(next * (KEYS / 8));
                __syncthreads();
                if (any_bad) {
                    const uint32_t place = tile * (KEYS / 8) + lane % (KEYS / 8);
                    uint32_t none = uint32_t(
                        __ballot(lane < KEYS / 8 && held[place % kHeld].y >> 31));
                    for (; none; none &= none - 1)
                        marks |= 0xffull << 8 * __builtin_ctz(none);
                }
                if (mixed) {
                    check_tile(stage, turn);
                    __syncthreads();
                    marks |= uint64_t(flags[turn][1]) << 32 | flags[turn][0];
                    turn ^= 1;
                    if (threadIdx.x < 2)
                        flags[turn][threadIdx.x] = 0;
                }
            } else {
                if (STAGES == 1)
                    __syncthreads();  // the tile before has been read
                store_tile(stage, mixed, turn);
                if (tile + 1 < part.last) {
                    load_tile(tile + 1);
                    load_ids(tile + 2 < part.last ? tile + 2 : tile + 1);
                }
                __syncthreads();
                marks = uint64_t(flags[turn][1]) << 32 | flags[turn][0];
                // The mark after the next one: no thread is past the next barrier.
                turn = turn == 2 ? 0 : turn + 1;
                if (threadIdx.x < 2)
                    flags[turn == 2 ? 0 : turn + 1][threadIdx.x] = 0;
            }

            v4f s[GROUPS][NB];
            if (active) {
                const uint32_t me = SPLIT > 1 ? formed_here(lane) : lane;
                // Copied rows: where the wave's depths v, v + PLACES, ... lie in their groups of
                // chunks.
                constexpr uint32_t PLACES = COPIED ? Order::G / 4 : 1;
                uint32_t key_lane[PLACES];
#pragma unroll
                for (uint32_t v = 0; v < PLACES; ++v) {
                    const uint32_t chunk = 4 * ((split * U + v) % PLACES) + (me >> 4);
                    key_lane[v] =
                        (me & 15) * PITCH + 8 * (COPIED ? Order::place(me & 15, chunk) : me >> 4);
                }
                // f32 caches: the largest product apart from the others, whose sums it would
                // round.
                v4f rest[GROUPS][HALF ? 1 : NB];
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                    for (int c = 0; c < NB; ++c)
                        s[g][c] = rest[g][HALF ? 0 : c] = v4f{0, 0, 0, 0};
                // Reads are in the order (depth, key block, part), the smallest part first.
                constexpr int READS = U * NB * PARTS, MOST = HALF ? 6 : 3;
                constexpr int AHEAD = READS < MOST ? READS : MOST;
                const auto read = [&](int n) {
                    const int u = n / (NB * PARTS), c = n / PARTS % NB;
                    const int i = PARTS - 1 - n % PARTS;
                    uint32_t depth = split * U + u;
                    if (DEPTHS % SPLIT != 0 && depth >= uint32_t(DEPTHS))
                        depth = DEPTHS - 1;  // its queries are zero
                    const uint16_t *from = stage;
                    from += key_lane[u % PLACES] + depth / PLACES * (32 * PLACES);
                    // Past the row's end a lane reads columns that the query's zeros drop.
                    if (DK % 32 != 0 && u == U - 1 && q >= 2)
                        from -= 16;
                    return *reinterpret_cast<const v4u *>(from + 16 * c * PITCH +
                                                          i * S::KEY_PLANE);
                };
                // Each is issued some products ahead of its own, where the compiler would
                // place it right before them and wait.
                v4u ahead[AHEAD];
#pragma unroll
                for (int n = 0; n < AHEAD; ++n)
                    ahead[n] = read(n);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < READS; ++n) {
                    const int u = n / (NB * PARTS), c = n / PARTS % NB;
                    const int i = PARTS - 1 - n % PARTS;
                    const v4u k = ahead[n % AHEAD];
#pragma unroll
                    for (int b = (HALF ? 1 : 2) - i; b >= 0; --b)
#pragma unroll
                        for (int g = 0; g < GROUPS; ++g)
                            if (HALF || i + b == 0)
                                s[g][c] = mfma<HALF>(k, query[g][u][b], s[g][c]);
                            else
                                rest[g][HALF ? 0 : c] =
                                    mfma<HALF>(k, query[g][u][b], rest[g][HALF ? 0 : c]);
                    if (n + AHEAD < READS)
                        ahead[n % AHEAD] = read(n + AHEAD);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (COPIED)
                    if (next < part.last)
                        copy_tile(next, slot_behind);  // beside the products
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                    for (int c = 0; c < NB; ++c) {
                        if (!HALF)
                            s[g][c] += rest[g][c];
                        if (SPLIT > 1) {
                            s[g][c] *= factor[g];
                            partial[((wave * GROUPS + g) * NB + c) * 64 + lane] = s[g][c];
                        }
                    }
            } else if constexpr (COPIED) {
                if (next < part.last)
                    copy_tile(next, slot_behind);
            }
            if (SPLIT > 1) {
                // The same sum, in the same order, in every wave of a row.
                __syncthreads();
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                    for (int c = 0; c < NB; ++c)
#pragma unroll
                        for (int w = 0; w < SPLIT; ++w) {
                            const v4f x =
                                partial[(((wave - split + w) * GROUPS + g) * NB + c) * 64 + lane];
                            s[g][c] = w ? s[g][c] + x : x;
                        }
            }
            if (!active)
                continue;
            const int first = int(k0) - int(length);  // the run's token at key 0
            const int last = int(last_key - k0);
            if (mixed) {
                const uint32_t q4 = 4 * formed_here(q);
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    // Bit 4 c + r: whether the row attends key 16 c + 4 q + r.
                    uint32_t seen = 0;
                    if (p.mask) {
                        const uint8_t *mask =
                            p.mask + uint64_t(part.run.begin + token[g]) * p.mask_bytes;
#pragma unroll 1
                        for (int n = 0; n < 4 * NB; ++n) {
                            const int at = 16 * (n / 4) + int(q4) + n % 4, i = first + at;
                            uint32_t bit = at <= last;
                            if (i >= 0 && at <= last)
                                bit = uint32_t(i) < 8 * p.mask_bytes
                                          ? mask[uint32_t(i) >> 3] >> (i & 7) & 1
                                          : 0;
                            seen |= bit << n;
                        }
                    } else {
                        const int most = int(token[g]) - first;
                        // Of each four keys, the first most + 1 - (their first) ones.
#pragma unroll
                        for (int c = 0; c < NB; ++c) {
                            int n = most + 1 - 16 * c - int(q4);
                            n = n < 0 ? 0 : n > 4 ? 4 : n;
                            seen |= ((1u << n) - 1) << (4 * c);
                        }
                    }
                    if (marks) {
                        uint32_t mine = 0;
#pragma unroll
                        for (int c = 0; c < NB; ++c)
                            mine |= uint32_t(marks >> (16 * c + q4) & 15) << (4 * c);
                        poison[g] |= (seen & mine) != 0;
                    }
#pragma unroll
                    for (int c = 0; c < NB; ++c)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            s[g][c][r] =
                                seen >> (4 * c + r) & 1 ? s[g][c][r] : -__builtin_inff();
                }
            } else if (marks) {
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
                    poison[g] = true;
            }
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const float times = SPLIT > 1 ? 1.0f : factor[g];
                float top = -__builtin_inff();
#pragma unroll
                for (int c = 0; c < NB; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        top = fmaxf(top, s[g][c][r]);
                top = fmaxf(m[g], quad_max(top) * times);
                if (__any(top > m[g] + kSlack)) {
                    const float base = top == -__builtin_inff() ? 0.0f : top;
                    const float rescale = __builtin_amdgcn_exp2f(m[g] - base);
                    l[g] *= rescale;
#pragma unroll
                    for (int t = 0; t < N; ++t)
                        o[g][t] *= rescale;
                    m[g] = top;
                }
                // While every score is -infinity, nothing is added.
                const float base = m[g] == -__builtin_inff() ? 0.0f : m[g];
                const float line_at = HALF ? base - kProbabilityShift : base;
#pragma unroll
                for (int c = 0; c < NB; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[g][c][r] =
                            __builtin_amdgcn_exp2f(__builtin_fmaf(s[g][c][r], times, -line_at));
                        l[g] += s[g][c][r];
                    }
            }
            const uint32_t me = SPLIT > 1 ? formed_here(lane) : lane;
            const uint16_t *value_stage = stage + (LATENT ? 0 : PARTS * S::KEY_PLANE);
#pragma unroll
            for (int h = 0; h < NB / 2; ++h) {  // 32 keys, a product's depth
                v4u prob[GROUPS][QP];
#pragma unroll
                for (int g = 0; g < GROUPS; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t parts[QP];
                        split_pair<HALF>(s[g][2 * h + e / 2][2 * (e % 2)],
                                         s[g][2 * h + e / 2][2 * (e % 2) + 1], parts);
#pragma unroll
                        for (int i = 0; i < QP; ++i)
                            prob[g][i][e] = parts[i];
                    }
                for_chunks<N, S::CHUNK>([&](auto first_tile, auto tiles) {
                    constexpr int t0 = first_tile, n = tiles, W = (n + 1) / 2;
#pragma unroll
                    for (int i = PARTS - 1; i >= 0; --i) {
                        uint32_t x[8][W];
                        // Columns 16 t0 + n j .. + n - 1 of the wave's, of the key 32 h + 16
                        // (e / 4) + 4 q + e % 4; copied rows have 2 or 4 orders among them.
                        constexpr uint32_t ORDERS = !COPIED ? 1 : Order::G == 16 ? 4 : 2;
                        static_assert(!COPIED || 2 * t0 % Order::G == 0, "whole groups of chunks");
                        uint32_t value_lane[ORDERS];
#pragma unroll
                        for (uint32_t v = 0; v < ORDERS; ++v) {
                            const uint32_t row = 4 * (me >> 4) + v * (4 / ORDERS);
                            const uint32_t column = split * (DV / SPLIT) + n * (me & 15);
                            value_lane[v] =
                                4 * (me >> 4) * PITCH +
                                (COPIED ? 8 * Order::place(row, column / 8) + column % 8 : column);
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint16_t *from = value_stage + i * S::KEY_PLANE +
                                                   (32 * h + 16 * (e / 4) + e % 4) * PITCH +
                                                   16 * t0 + value_lane[e % 4 * ORDERS / 4];
                            if constexpr (n == 8) {
                                const v4u piece = *reinterpret_cast<const v4u *>(from);
                                x[e][0] = piece[0], x[e][1] = piece[1];
                                x[e][2] = piece[2], x[e][3] = piece[3];
                            } else if constexpr (n == 4) {
                                const v2u piece = *reinterpret_cast<const v2u *>(from);
                                x[e][0] = piece[0], x[e][1] = piece[1];
                            } else if constexpr (n == 2) {
                                x[e][0] = *reinterpret_cast<const uint32_t *>(from);
                            } else {
                                x[e][0] = *from;
                            }
                        }
#pragma unroll
                        for (int t = 0; t < n; ++t) {
                            v4u v;
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                v[e] = __builtin_amdgcn_perm(x[2 * e + 1][t / 2], x[2 * e][t / 2],
                                                             t % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
                            for (int b = (HALF ? 1 : 2) - i; b >= 0; --b)
#pragma unroll
                                for (int g = 0; g < GROUPS; ++g)
                                    o[g][t0 + t] = mfma<HALF>(v, prob[g][b], o[g][t0 + t]);
                        }
                    }
                });
            }
        }

#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const float total = quad_sum(poison[g] ? __builtin_nanf("") : l[g]);
            if (!real[g])
                continue;
            const uint64_t record = uint64_t(part.record) * ROWS + wave_row + 16 * g + j;
            float *to = (part.whole ? p.out + query_row[g] * DV : p.records + record * DV) +
                        split * (DV / SPLIT);
            // Nothing attended: zeros.
            const float scale = !part.whole ? 1.0f : total == 0.0f ? 0.0f : 1.0f / total;
            for_chunks<N, S::CHUNK>([&](auto first_tile, auto tiles) {
                constexpr int t0 = first_tile, n = tiles;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float *at = to + 16 * t0 + n * (4 * q + r);
                    if constexpr (n % 4 == 0) {
#pragma unroll
                        for (int t = 0; t < n; t += 4)
                            *reinterpret_cast<v4f *>(at + t) =
                                v4f{o[g][t0 + t][r], o[g][t0 + t + 1][r], o[g][t0 + t + 2][r],
                                    o[g][t0 + t + 3][r]} * scale;
                    } else {
#pragma unroll
                        for (int t = 0; t < n; ++t)
                            at[t] = o[g][t0 + t][r] * scale;
                    }
                }
            });
            if (!part.whole && q == 0 && split == 0)
                reinterpret_cast<v2f *>(record_stats(p))[record] = v2f{m[g], total};
        }
        if (part.leads && !part.whole)
            share = {block_of(line, part.last_unit) - line.block + 1, part.record, part.run.begin,
                     part.run.count, part.kv_head, part.row_tile};
    }
    if (threadIdx.x == 0)
        block_shares(p)[line.block] = share;
}

// The shared items' rows: out = sum_i a_i 2^(m_i - M) / sum_i l_i 2^(m_i - M) over the
// records, in an order that their number fixes.  Every block reads how many rows each block
// of the first launch has left to join and takes every so-many-th task of them.  A lane has a
// 4-column piece; up to kFewRecords records a wave takes as many rows as its lanes hold
// and reads all of a row's records at once, of more a block takes one row (and 256
// columns), its lanes' shares every so-many-th record.  Bound by dependent reads (shares,
// then statistics and records): 5 us for one tree, 12 and 18 for the two prompts above,
// whose records it reads once.
constexpr uint32_t kFewRecords = 8, kJoinHeld = 8, kJoinsPerCu = 4;

__global__ __launch_bounds__(kBlock) void run_attention_join_kernel(RunAttention p)
{
    __shared__ uint32_t ends[kMostBlocks];  // of the tasks of each block's share
    __shared__ uint32_t wave_sums[kBlock / 64];
    __shared__ v4f sums[kBlock];
    __shared__ float weights[kMostBlocks];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t d = p.value_dim, pieces = d / 4, width = pieces < 64 ? pieces : 64;
    const uint32_t columns = (pieces + 63) / 64, shares = 64 / width;
    const uint32_t mine = lane / width, c = lane % width;
    const Share *all = block_shares(p);
    const auto rows_of = [&](const Share &s) {
        const uint32_t left = s.run * p.group - p.rows * s.row_tile;
        return left < p.rows ? left : p.rows;
    };
    // Units that a wave takes at once: their records together are kFewRecords.
    const auto rows_at_once = [](uint32_t count) { return count <= 2 ? 4 : count <= 4 ? 2 : 1; };
    // Tasks, four blocks' shares a thread.
    uint32_t upto[kMostBlocks / kBlock], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kMostBlocks / kBlock; ++i) {
        const uint32_t b = threadIdx.x * (kMostBlocks / kBlock) + i;
        if (b < p.blocks) {
            const Share s = all[b];
            const uint32_t units = rows_of(s) * columns;
            const uint32_t each = (kBlock / 64) * shares * rows_at_once(s.count);
            sum += !s.count ? 0 : s.count > kFewRecords ? units : (units + each - 1) / each;
        }
        upto[i] = sum;
    }
    const uint32_t scan = lanes_scan(sum);
    if (lane == 63)
        wave_sums[wave] = scan;
    __syncthreads();
    uint32_t before = scan - sum, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kBlock / 64; ++w) {
        before += w < wave ? wave_sums[w] : 0;
        total += wave_sums[w];
    }
#pragma unroll
    for (uint32_t i = 0; i < kMostBlocks / kBlock; ++i)
        ends[threadIdx.x * (kMostBlocks / kBlock) + i] = before + upto[i];
    __syncthreads();
    const v2f *stats = reinterpret_cast<const v2f *>(record_stats(p));
#pragma unroll 1
    for (uint32_t task = blockIdx.x; task < total; task += gridDim.x) {
        // The first block whose tasks end behind this one.
        uint32_t b = 0;
#pragma unroll
        for (uint32_t step = kMostBlocks / 2; step; step /= 2)
            if (ends[b + step - 1] <= task)
                b += step;
        Share share = all[b];
        share = {scalar(share.count), scalar(share.record), scalar(share.begin), scalar(share.run),
                 scalar(share.kv_head), scalar(share.row_tile)};
        const uint32_t number = scalar(task - (b ? ends[b - 1] : 0));
        const uint32_t units = rows_of(share) * columns;
        const auto record = [&](uint32_t i, uint32_t in_tile) {
            return uint64_t(i ? share.record / 2 * 2 + 2 * i : share.record) * p.rows + in_tile;
        };
        const auto piece_at = [&](uint64_t n, uint32_t piece) {
            return *reinterpret_cast<const v4f *>(p.records + n * d + 4 * piece);
        };
        // A record without a key has no outputs.
        const auto weighed = [](float w, v4f y) { return w != 0.0f ? y * w : v4f{0, 0, 0, 0}; };
        const auto write = [&](uint32_t in_tile, uint32_t piece, v4f a, float sum_l) {
            const uint32_t row = p.rows * share.row_tile + in_tile, token = row / p.group;
            const uint64_t at = uint64_t(share.begin + token) * p.query_heads +
                                share.kv_head * p.group + row - token * p.group;
            *reinterpret_cast<v4f *>(p.out + at * d + 4 * piece) =
                a * (sum_l == 0.0f ? 0.0f : 1.0f / sum_l);
        };
        // Up to RECORDS of them, kFewRecords / RECORDS units a wave.
        const auto join_few = [&](auto records) {
            constexpr uint32_t RECORDS = records, UNITS = kFewRecords / RECORDS;
            v4f x[UNITS][RECORDS];
            v2f stat[UNITS][RECORDS];
            uint32_t in_tile[UNITS], piece[UNITS];
            bool real[UNITS];
#pragma unroll
            for (uint32_t u = 0; u < UNITS; ++u) {
                const uint32_t unit =
                    ((number * UNITS + u) * (kBlock / 64) + wave) * shares + mine;
                real[u] = unit < units && mine < shares;
                in_tile[u] = (real[u] ? unit : 0) / columns;
                piece[u] = ((real[u] ? unit : 0) - in_tile[u] * columns) * 64 + c;
#pragma unroll
                for (uint32_t i = 0; i < RECORDS; ++i) {
                    const uint64_t n = record(i < share.count ? i : 0, in_tile[u]);
                    x[u][i] = piece_at(n, piece[u]);
                    stat[u][i] = stats[n];
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < UNITS; ++u) {
                float most = -__builtin_inff(), sum_l = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < RECORDS; ++i)
                    most = fmaxf(most, stat[u][i][0]);
                const float base = most == -__builtin_inff() ? 0.0f : most;
                v4f a = {0, 0, 0, 0};
#pragma unroll
                for (uint32_t i = 0; i < RECORDS; ++i) {
                    const float w =
                        i < share.count ? __builtin_amdgcn_exp2f(stat[u][i][0] - base) : 0.0f;
                    sum_l += i < share.count ? stat[u][i][1] * w : 0.0f;
                    a += weighed(w, x[u][i]);
                }
                if (real[u])
                    write(in_tile[u], piece[u], a, sum_l);
            }
        };
        if (share.count <= 2) {
            join_few(std::integral_constant<uint32_t, 2>{});
            continue;
        }
        if (share.count <= 4) {
            join_few(std::integral_constant<uint32_t, 4>{});
            continue;
        }
        if (share.count <= kFewRecords) {
            join_few(std::integral_constant<uint32_t, 8>{});
            continue;
        }
        const uint32_t in_tile = number / columns, piece = (number - in_tile * columns) * 64 + c;
        // The lane's records, `by` apart from its first one.
        const uint32_t first = wave * shares + (mine < shares ? mine : 0);
        const uint32_t by = (kBlock / 64) * shares;
        v4f x[kJoinHeld];
        const auto load = [&](uint32_t from) {
#pragma unroll
            for (uint32_t i = 0; i < kJoinHeld; ++i) {
                const uint32_t n = from + i * by;
                x[i] = piece_at(record(n < share.count ? n : share.count - 1, in_tile), piece);
            }
        };
        load(first);
        // Each wave forms the row's maximum and sum, the first one's weights are shared.
        float most = -__builtin_inff(), sum_l = 0.0f;
        for (uint32_t i = lane; i < share.count; i += 64)
            most = fmaxf(most, stats[record(i, in_tile)][0]);
#pragma unroll
        for (int offset = 32; offset > 0; offset >>= 1)
            most = fmaxf(most, __shfl_xor(most, offset, 64));
        const float base = most == -__builtin_inff() ? 0.0f : most;
        __syncthreads();  // the task before has been read
        for (uint32_t i = lane; i < share.count; i += 64) {
            const v2f stat = stats[record(i, in_tile)];
            const float w = __builtin_amdgcn_exp2f(stat[0] - base);
            sum_l += stat[1] * w;
            if (wave == 0)
                weights[i] = w;
        }
#pragma unroll
        for (int offset = 32; offset > 0; offset >>= 1)
            sum_l += __shfl_xor(sum_l, offset, 64);
        __syncthreads();
        v4f a = {0, 0, 0, 0};
#pragma unroll 1
        for (uint32_t n0 = 0; n0 < share.count; n0 += kJoinHeld * by) {
            v4f now[kJoinHeld];
#pragma unroll
            for (uint32_t i = 0; i < kJoinHeld; ++i)
                now[i] = x[i];
            if (n0 + kJoinHeld * by < share.count)
                load(first + n0 + kJoinHeld * by);
#pragma unroll
            for (uint32_t i = 0; i < kJoinHeld; ++i) {
                const uint32_t n = first + n0 + i * by;
                a += weighed(n < share.count && mine < shares ? weights[n] : 0.0f, now[i]);
            }
        }
        sums[threadIdx.x] = a;
        __syncthreads();
        if (threadIdx.x < width && piece < pieces) {
            a = v4f{0, 0, 0, 0};
            for (uint32_t w = 0; w < kBlock / 64; ++w)
                for (uint32_t s = 0; s < shares; ++s)
                    a += sums[64 * w + s * width + c];
            write(in_tile, piece, a, sum_l);
        }
    }
}

// The kernel of a shape (null: none), its threads and rows of an item, the blocks of it that
// a CU holds, a tile's keys.
struct MatrixKernel {
    void (*run)(RunAttention) = nullptr;
    int threads = 0, rows = 0, resident = 0, shift = 0;
};
template <int DK, int DV, bool HALF, bool LATENT, int WAVES, int SPLIT, int GROUPS, int RESIDENT>
MatrixKernel matrix_kernel_with()
{
    using S = Shape<DK, DV, HALF, LATENT, WAVES, SPLIT, GROUPS, RESIDENT>;
    return {run_attention_kernel<DK, DV, HALF, LATENT, WAVES, SPLIT, GROUPS, RESIDENT>, S::THREADS,
            S::ROWS, RESIDENT, S::SHIFT};
}
// Blocks on a CU: two waves to a SIMD, one where a wave needs all registers, three as below.
//
// `many`: more rows than one item has, on average over the sequences, for the starts live on the
// device.  Batches of a prompt and single tokens take what the two take apart, or less: 256
// tokens, and 47 of one over 2047 keys, 32 / 8 heads, binary16, of 64 columns 21 and 44 us,
// together 49, of 128 26 and 87, together 94; with 1024 over 1024 58 and 44, together 106, and 82
// and 87, together 131.  Up to 112 wide a wave
// then has 32 of them, for which each operand read from LDS serves two products: the
// prompt above 160 us against 180, and of heads 128 wide 48 sequences of 24 tokens over 2047
// (96 rows) 169 against 193, of 16 tokens (64 rows) 147 against 126.  Of 128 columns that
// is all registers of two waves and some spilled; three waves of 16 rows, with tiles of 32
// keys, take 158 there, and 168 against 189 of 32 tokens, but with few rows, where loads
// and the start count, longer than two with tiles of 64: 16 tokens over 2047 31 us against 23,
// 48 x 4 over 17 to 8191 62 against 59.
template <int D>
MatrixKernel matrix_kernel_of(bool half, bool many)
{
    constexpr int RESIDENT = D <= 128 ? 2 : 1;
    if (half) {
        if constexpr (D <= 128)
            if (many)
                return matrix_kernel_with<D, D, true, false, 4, 1, (D < 128 ? 2 : 1),
                                          (D < 128 ? 2 : 3)>();
        return matrix_kernel_with<D, D, true, false, 4, 1, 1, RESIDENT>();
    }
    // Three parts of a wide row need the registers of two waves; of 256 columns these spill 28
    // still (48 trees over 17 to 4095 keys, 16 / 4 heads, 164 us, its bytes' time 70).
    if constexpr (D < 128)
        return matrix_kernel_with<D, D, false, false, 4, 1, 1, RESIDENT>();
    else
        return matrix_kernel_with<D, D, false, false, 8, 2, 1, 1>();
}
// The fewer rows an item has, the more of a row's columns are a wave's own: items of 64
// rows (two waves to a row), of 32 (four) and of 16 (eight, whose operand reads no other
// wave shares).  Binary16, 64 sequences over 2047 latents of 512 + 64: of 32 rows 62 us in
// items of 64, 60 of 32; of 64 rows 83 and 98; the prompt above 328 and 452.  f32, the same
// of 16 rows: 121 in items of 16, 141 of 32; of 32 rows 202 and 167.  Of rank 512 the f32
// kernel for items of 32 rows spills registers (62, with 32 rotated columns 65), and so
// does the binary16 one for 64 rows and 32 rotated columns (33).  64 and 128 rows to a
// sequence, 64 sequences over 2047: binary16 88 and 138 us (36 and 67 of bytes or products),
// f32 266 and 436 (98 and 197).
template <int RANK, int ROPE>
MatrixKernel latent_kernel_of(bool half, uint64_t rows, uint64_t sequences)
{
    constexpr int DK = RANK + ROPE;
    if (half)
        return rows > 32 * sequences ? matrix_kernel_with<DK, RANK, true, true, 8, 2, 1, 1>()
                                     : matrix_kernel_with<DK, RANK, true, true, 8, 4, 1, 1>();
    if constexpr (RANK == 512)
        if (rows <= 16 * sequences)
            return matrix_kernel_with<DK, RANK, false, true, 8, 8, 1, 1>();
    return matrix_kernel_with<DK, RANK, false, true, 8, 4, 1, 1>();
}
MatrixKernel matrix_kernel(const RunAttention &p)
{
    const bool half = p.shape.half;
    const uint32_t rope = p.shape.head_dim - p.value_dim;
    const uint64_t rows = uint64_t(p.runs.tokens) * p.group;
    if (rope == 0) {
        const bool many = rows > 64 * uint64_t(p.runs.sequences);
        switch (p.value_dim) {
        case 32: return matrix_kernel_of<32>(half, many);
        case 64: return matrix_kernel_of<64>(half, many);
        case 80: return matrix_kernel_of<80>(half, many);
        case 96: return matrix_kernel_of<96>(half, many);
        case 112: return matrix_kernel_of<112>(half, many);
        case 128: return matrix_kernel_of<128>(half, many);
        case 160: return matrix_kernel_of<160>(half, many);
        case 192: return matrix_kernel_of<192>(half, many);
        case 256: return matrix_kernel_of<256>(half, many);
        default: return {};
        }
    }
    const uint64_t sequences = p.runs.sequences;
    switch (p.value_dim * 1024 + rope) {
    case 128 * 1024 + 32: return latent_kernel_of<128, 32>(half, rows, sequences);
    case 128 * 1024 + 64: return latent_kernel_of<128, 64>(half, rows, sequences);
    case 256 * 1024 + 32: return latent_kernel_of<256, 32>(half, rows, sequences);
    case 256 * 1024 + 64: return latent_kernel_of<256, 64>(half, rows, sequences);
    case 512 * 1024 + 32: return latent_kernel_of<512, 32>(half, rows, sequences);
    case 512 * 1024 + 64: return latent_kernel_of<512, 64>(half, rows, sequences);
    default: return {};
    }
}

}  // namespace

bool run_attention_plan(RunAttention &p, int cu_count)
{
    const uint64_t rows = uint64_t(p.runs.tokens) * p.query_heads;
    p.blocks = 0;
    if (rows > uint64_t(1) << 25)
        return false;
    const MatrixKernel kernel = matrix_kernel(p);
    if (!kernel.run || !rows || !p.runs.sequences)
        return true;
    p.rows = kernel.rows;
    p.item_units = kernel.resident == 3 ? kItemUnitsOfThree : kItemUnits;
    // Units stay in 32 bits.  A run that passes its table's row has no tiles; past the others'
    // keys an item has up to six units for what is rounded up.
    const uint64_t items = (uint64_t(p.runs.tokens) * p.group / p.rows + p.runs.sequences) *
                           p.shape.kv_heads;
    const uint64_t most = items * (p.item_units + 6 + (p.longest >> kernel.shift));
    if (most >= uint64_t(1) << 31)
        return false;
    const uint64_t wanted = (most + kLeastUnits - 1) / kLeastUnits;
    const uint64_t resident = uint64_t(cu_count) * kernel.resident;
    p.blocks = uint32_t(wanted < resident ? wanted : resident);
    p.blocks = p.blocks < kMostBlocks ? p.blocks : kMostBlocks;
    p.joins = uint32_t(cu_count) * kJoinsPerCu;
    return true;
}

size_t run_attention_scratch_bytes(const RunAttention &p)
{
    return size_t(p.blocks) * (2 * size_t(p.rows) * (p.value_dim + 2) * sizeof(float) +
                               sizeof(Share));
}

void launch_run_attention(hipStream_t stream, const RunAttention &p)
{
    if (p.blocks) {
        const MatrixKernel kernel = matrix_kernel(p);
        kernel.run<<<p.blocks, kernel.threads, 0, stream>>>(p);
        run_attention_join_kernel<<<p.joins, kBlock, 0, stream>>>(p);
        return;
    }
    const uint64_t blocks = uint64_t(p.runs.tokens) * p.query_heads;
    if (!blocks)
        return;
    const size_t bytes = (size_t(p.shape.head_dim) + p.value_dim) * sizeof(float);
    run_attention_general_kernel<<<unsigned(blocks), 64, bytes, stream>>>(p);
}

}  // namespace mfh
