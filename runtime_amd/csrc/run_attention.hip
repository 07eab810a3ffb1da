// Attention of runs of new tokens (trees of drafted ones, or a prompt's) over paged
// caches of keys and values, or of latents.
//
// o = sum_j p_j v_j / sum_j p_j over the keys j that a token attends, with p_j =
// exp(s_j - max s) and s_j = q . k_j scale: all of the sequence's cached tokens and those
// of the run that its mask names.
#include <type_traits>

#include "draft.hpp"
#include "kernels.hpp"

namespace mfh {
namespace {

// ---- any width -----------------------------------------------------------------

// A wave per (token, query head): 64 keys at a time, a lane forms one key's score, then the
// lanes are columns of the values.
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
// Query rows of a key/value head are (token, head of the group) pairs, counted through a run;
// an item is (sequence, key/value head, 64 of its rows), a wave of a block has 16
// of them.  The block walks the item's keys a tile at a time: all threads load a tile's rows
// to registers (the next tile's while this one is worked on) and store them to LDS as
// operands that the waves share.  Per tile, S^T = K Q^T leaves query row j in lane
// column j (lane 16 q + j holds the scores of keys 16 c + 4 q + r in register r of
// block c), the softmax follows online in the row's four lanes, and O^T += V^T P^T takes
// those registers as its second operand; its first is put together from pieces of eight
// key rows.
//
// Binary16 caches: keys and values are operands as they are, queries (scaled by a power of
// two to below 2^15) and probabilities (times 2^15) two binary16 parts each, which are
// within 2^-24 of the value.  f32 caches: all four are three bfloat16 parts, which hold 24
// bits, and six of the nine products are formed (the others are below 2^-26).
//
// The work is a line of units (a tile of keys; items in order, kItemUnits besides for each),
// which every block adds up itself, for starts and lengths live on the device, and takes
// an equal run of.  A block that holds all tiles of an item writes its rows; the others
// store records (maximum, sum, unnormalised output) that a second launch joins in block
// order, so that results do not depend on timing.
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

constexpr int kBlock = 256;
constexpr uint32_t kRows = 64;       // query rows of an item
constexpr uint32_t kItemUnits = 2;
constexpr uint32_t kLeastUnits = 4;  // of a block
constexpr float kProbabilityShift = 15.0f;

// What a block's first unfinished item needs of the join.
struct Share {
    uint32_t count, record;          // records (0: none), the first one
    uint32_t begin, run, kv_head, row_tile;
};

__host__ __device__ inline float *record_stats(const RunAttention &p)
{
    return p.records + 2 * uint64_t(p.blocks) * kRows * p.value_dim;
}
__host__ __device__ inline Share *block_shares(const RunAttention &p)
{
    return reinterpret_cast<Share *>(record_stats(p) + 4 * uint64_t(p.blocks) * kRows);
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
// all before them, a later item has more keys: (64 / group) a row tile more, counted in
// whole tiles, so that the sum has a closed form.
template <int SHIFT>
struct Units {
    uint32_t group, base, step;  // step: tiles of a run's 64 tokens; 0: the same for all
    __device__ __forceinline__ Units(const RunAttention &p, const Run &run)
    {
        constexpr uint32_t KEYS = 1u << SHIFT;
        group = p.group;
        step = 0;
        base = kItemUnits;
        if (run.length == UINT32_MAX)
            return;
        if (p.mask || run.count == 1) {
            base += (run.length + run.count + KEYS - 1) >> SHIFT;
        } else {
            step = kRows / KEYS;
            base += ((run.length + KEYS - 1) >> SHIFT) + step;
        }
    }
    __device__ __forceinline__ uint32_t of(uint32_t tile) const
    {
        return base + (step ? tile / group * step : 0);
    }
    // Of the first `tiles` items.
    __device__ __forceinline__ uint32_t upto(uint32_t tiles) const
    {
        uint32_t sum = tiles * base;
        if (step) {
            const uint32_t whole = tiles / group, left = tiles - whole * group;
            sum += step * (group * (whole * (whole - 1) / 2) + whole * left);
        }
        return sum;
    }
};
__device__ __forceinline__ uint32_t row_tiles(const RunAttention &p, const Run &run)
{
    return (run.count * p.group + kRows - 1) / kRows;
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
        const uint32_t token = (kRows * line.row_tile + kRows - 1) / p.group;
        part.keys = run.length + (p.mask || token >= run.count ? run.count : token + 1);
    }
    const uint32_t tiles = (part.keys + (1u << SHIFT) - 1) >> SHIFT;
    // The item's last units may be more or fewer than its tiles.
    const auto tile_at = [&](uint32_t unit) {
        const uint32_t t = unit > kItemUnits ? unit - kItemUnits : 0;
        return unit == units || t > tiles ? tiles : t;
    };
    part.first = tile_at(from);
    part.last = tile_at(to);
    part.leads = from <= kItemUnits;
    part.opens = from == 0;
    part.counts = to > kItemUnits;
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
__host__ __device__ constexpr int chunk_tiles(int left)
{
    int s = 8;
    while (s > left)
        s /= 2;
    return s;
}
// f(first tile, tiles) for each chunk of N tiles, both as constants.
template <int N, int T = 0, typename F>
__device__ __forceinline__ void for_chunks(F f)
{
    if constexpr (T < N) {
        constexpr int S = chunk_tiles(N - T);
        f(std::integral_constant<int, T>{}, std::integral_constant<int, S>{});
        for_chunks<N, T + S>(f);
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
            const v2h h = {_Float16(a), _Float16(b)};
            out[i] = __builtin_bit_cast(uint32_t, h);
            a -= float(h[0]);
            b -= float(h[1]);
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

// The products of a's parts (a cache's) with b's (a query's or a probability's), the
// smallest first.
template <bool HALF, int A, int B>
__device__ __forceinline__ v4f products(const v4u (&a)[A], const v4u (&b)[B], v4f c)
{
    constexpr int most = HALF ? 1 : 2;  // the sum of the parts' numbers
#pragma unroll
    for (int sum = most; sum >= 0; --sum)
#pragma unroll
        for (int i = 0; i < A; ++i)
            if (sum - i >= 0 && sum - i < B)
                c = mfma<HALF>(a[i], b[sum - i], c);
    return c;
}

// LDS rows of D 16-bit columns hold 16-byte chunks in an order of their own, by which 16
// rows' equal chunks fall on all banks.
template <int D>
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk)
{
    constexpr uint32_t C = D / 8;
    constexpr uint32_t G = C % 16 == 0 ? 16 : C % 8 == 0 ? 8 : C % 4 == 0 ? 4 : 2;
    static_assert(C % G == 0, "whole groups of chunks");
    return row * D + ((chunk ^ (row / (16 / G) & (G - 1))) * 8);
}

// What a kernel of a width has in a tile, in LDS and on a CU.
template <int DK, int DV, bool HALF, bool LATENT>
struct Shape {
    static constexpr int PARTS = HALF ? 1 : 3;          // of keys and values
    static constexpr int QUERY_PARTS = HALF ? 2 : 3;    // of queries and probabilities
    static constexpr int SHIFT = DK <= (HALF ? 128 : 64) ? 6 : 5;
    static constexpr int KEYS = 1 << SHIFT;
    static constexpr int KEY_PLANE = KEYS * DK, VALUE_PLANE = LATENT ? 0 : KEYS * DV;
    static constexpr int STAGE = PARTS * (KEY_PLANE + VALUE_PLANE);  // 16-bit elements
    static constexpr int STAGES = HALF ? 2 : 1;
    static constexpr int RESIDENT = DK <= 128 ? 2 : 1;
};

template <int DK, int DV, bool HALF, bool LATENT>
__global__ __launch_bounds__(kBlock, (Shape<DK, DV, HALF, LATENT>::RESIDENT))
void run_attention_kernel(RunAttention p)
{
    using S = Shape<DK, DV, HALF, LATENT>;
    using T = typename std::conditional<HALF, _Float16, float>::type;
    static_assert(DK % 16 == 0 && DV % 16 == 0, "widths of the matrix-core path");
    constexpr int KEYS = S::KEYS, SHIFT = S::SHIFT, PARTS = S::PARTS, QP = S::QUERY_PARTS;
    constexpr int NB = KEYS / 16;                  // key blocks of a tile
    constexpr int U = (DK + 31) / 32;              // product depths of a key row
    constexpr int N = DV / 16;                     // 16-column tiles of the output
    constexpr int PIECE = 16 / sizeof(T);          // columns of a 16-byte load
    constexpr int KC = DK / PIECE, VC = LATENT ? 0 : DV / PIECE;
    constexpr int NK = (KEYS * KC + kBlock - 1) / kBlock;
    constexpr int NV = (KEYS * VC + kBlock - 1) / kBlock;
    __shared__ __attribute__((aligned(16))) uint16_t lds[S::STAGES * S::STAGE];
    __shared__ unsigned long long flags[3];

    const uint32_t lane = threadIdx.x & 63, q = lane >> 4, j = lane & 15;
    const uint32_t wave = scalar(threadIdx.x >> 6);
    const uint32_t page_shift = p.shape.page_shift, in_page = p.shape.page_size() - 1;
    Line line;
    const bool any = find_line<SHIFT>(p, line);
    Share share = {};
    Part part;
    while (any && next_part<SHIFT>(p, line, part)) {
        const uint32_t rows = part.run.count * p.group, row0 = kRows * part.row_tile;
        const uint32_t row = row0 + 16 * wave + j;
        const bool real = row < rows;
        const uint32_t token = (real ? row : rows - 1) / p.group;  // of the run
        const uint32_t head = part.kv_head * p.group + (real ? row : rows - 1) - token * p.group;
        const uint64_t query_row = uint64_t(part.run.begin + token) * p.query_heads + head;
        if (part.run.length == UINT32_MAX) {
            if (part.opens && real)
                for (uint32_t c = q; c < uint32_t(DV); c += 4)
                    p.out[query_row * DV + c] = __builtin_nanf("");
            continue;
        }
        if (!part.counts)
            continue;
        const float *table = p.tables + uint64_t(part.sequence) * p.max_pages;
        const uint32_t last_key = part.keys - 1, length = part.run.length;
        const T *keys = static_cast<const T *>(p.key_pages);
        const T *values = static_cast<const T *>(p.value_pages);

        // A tile's page ids, lane r key r's; keys past the end are the last one.
        const auto load_id = [&](uint32_t tile) {
            const uint32_t key = tile * KEYS + (lane & (KEYS - 1));
            return table[(key < last_key ? key : last_key) >> page_shift];
        };
        v4u key_reg[NK], value_reg[NV ? NV : 1];
        uint64_t bad_pages = 0;
        const auto load_tile = [&](uint32_t tile, float id) {
            const bool ok = valid_index(id, p.shape.pages);
            bad_pages = __ballot(!ok);
            if (KEYS < 64)
                bad_pages &= (uint64_t(1) << (KEYS & 63)) - 1;
            const uint32_t page = ok ? uint32_t(id) : 0;
            const auto at = [&](const T *pages, uint32_t key_row, uint32_t chunk, uint32_t width) {
                const uint32_t key = tile * KEYS + key_row;
                const uint32_t slot = (key < last_key ? key : last_key) & in_page;
                const uint64_t base = uint64_t(uint32_t(__shfl(page, int(key_row), 64))) *
                                          p.shape.stride() +
                                      (uint64_t(part.kv_head) << page_shift) * width;
                return reinterpret_cast<const v4u *>(pages + base + slot * width + chunk * PIECE);
            };
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                uint32_t n = threadIdx.x + i * kBlock;
                if ((i + 1) * kBlock > KEYS * KC)
                    n = n < uint32_t(KEYS * KC) ? n : KEYS * KC - 1;
                key_reg[i] = __builtin_nontemporal_load(at(keys, n / KC, n % KC, DK));
            }
            if constexpr (!LATENT)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    uint32_t n = threadIdx.x + i * kBlock;
                    if ((i + 1) * kBlock > KEYS * VC)
                        n = n < uint32_t(KEYS * VC) ? n : KEYS * VC - 1;
                    value_reg[i] = __builtin_nontemporal_load(at(values, n / VC, n % VC, DV));
                }
        };
        // 16 loaded bytes into the operand planes.  In a tile of the run, what is not finite
        // becomes zero and its key is marked: only rows that attend it shall see it.
        const auto store_piece = [&](v4u x, uint16_t *plane, int plane_size, uint32_t key_row,
                                     uint32_t chunk, auto width, bool of_run, uint32_t turn) {
            constexpr int D = width;
            if (of_run) {
                bool odd = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (HALF) {
                        const bool low = (x[e] & 0x7c00u) == 0x7c00u;
                        const bool high = (x[e] & 0x7c000000u) == 0x7c000000u;
                        odd |= low || high;
                        x[e] &= (low ? 0xffff0000u : ~0u) & (high ? 0xffffu : ~0u);
                    } else {
                        const bool all = (x[e] & 0x7f800000u) == 0x7f800000u;
                        odd |= all;
                        x[e] = all ? 0 : x[e];
                    }
                }
                if (odd)
                    atomicOr(&flags[turn], 1ull << key_row);
            }
            if constexpr (HALF) {
                *reinterpret_cast<v4u *>(plane + swizzled<D>(key_row, chunk)) = x;
            } else {
                uint32_t a[PARTS], b[PARTS];
                split_pair<HALF>(__uint_as_float(x[0]), __uint_as_float(x[1]), a);
                split_pair<HALF>(__uint_as_float(x[2]), __uint_as_float(x[3]), b);
                uint16_t *to = plane + swizzled<D>(key_row, chunk / 2) + chunk % 2 * 4;
#pragma unroll
                for (int i = 0; i < PARTS; ++i)
                    *reinterpret_cast<v2u *>(to + i * plane_size) = v2u{a[i], b[i]};
            }
        };
        const auto store_tile = [&](uint16_t *stage, bool of_run, uint32_t turn) {
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                uint32_t n = threadIdx.x + i * kBlock;
                if ((i + 1) * kBlock > KEYS * KC)
                    n = n < uint32_t(KEYS * KC) ? n : KEYS * KC - 1;
                store_piece(key_reg[i], stage, S::KEY_PLANE, n / KC, n % KC,
                            std::integral_constant<int, DK>{}, of_run, turn);
            }
            if constexpr (!LATENT)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    uint32_t n = threadIdx.x + i * kBlock;
                    if ((i + 1) * kBlock > KEYS * VC)
                        n = n < uint32_t(KEYS * VC) ? n : KEYS * VC - 1;
                    store_piece(value_reg[i], stage + PARTS * S::KEY_PLANE, S::VALUE_PLANE,
                                n / VC, n % VC, std::integral_constant<int, DV>{}, of_run, turn);
                }
        };

        float id = load_id(part.first);
        // The wave's queries; rows past the run's are zero.
        float qf[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const uint32_t column = 32 * u + 8 * q + e;
                const float *from;
                if (LATENT && 32 * u >= DV)
                    from = p.rotary_query + query_row * (DK - DV) + column - DV;
                else
                    from = p.query + query_row * DV + (column < uint32_t(DV) ? column : 0);
                const v4f piece = *reinterpret_cast<const v4f *>(from);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    qf[u][e + i] = real && column < uint32_t(DK) ? piece[i] : 0.0f;
            }
        if (part.first < part.last) {
            load_tile(part.first, id);
            id = load_id(part.first + 1 < part.last ? part.first + 1 : part.first);
        }
        float factor = p.scale;
        int exponent = 0;
        if (HALF) {
            float most = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    most = fmaxf(most, fabsf(qf[u][e]));
            most = quad_max(most);
            // 2^14 <= most 2^exponent < 2^15 (0 and infinities as they are).
            if (most > 0.0f && most < __builtin_inff())
                exponent = 15 - (ilogbf(most) + 1);
            factor = ldexpf(p.scale, -exponent);
        }
        v4u query[U][QP];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float a = qf[u][2 * e], b = qf[u][2 * e + 1];
                if (HALF)
                    a = ldexpf(a, exponent), b = ldexpf(b, exponent);
                uint32_t parts[QP];
                split_pair<HALF>(a, b, parts);
#pragma unroll
                for (int i = 0; i < QP; ++i)
                    query[u][i][e] = parts[i];
            }

        v4f o[N];
#pragma unroll
        for (int t = 0; t < N; ++t)
            o[t] = v4f{0, 0, 0, 0};
        float m = -__builtin_inff(), l = 0.0f;
        bool poison = false;
        const uint8_t *mask = p.mask + uint64_t(part.run.begin + token) * p.mask_bytes;
        uint32_t turn = 0;
        __syncthreads();  // an earlier part's tiles and marks have been read
        if (threadIdx.x < 3)
            flags[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll 1
        for (uint32_t tile = part.first; tile < part.last; ++tile) {
            const uint32_t k0 = tile * KEYS;
            const bool of_run = k0 + KEYS > length;
            uint16_t *stage = lds + (S::STAGES == 2 && (tile & 1) ? S::STAGE : 0);
            if (S::STAGES == 1)
                __syncthreads();  // the tile before has been read
            store_tile(stage, of_run, turn);
            uint64_t marks = bad_pages;
            if (tile + 1 < part.last) {
                load_tile(tile + 1, id);
                id = load_id(tile + 2 < part.last ? tile + 2 : tile + 1);
            }
            __syncthreads();
            if (of_run)
                marks |= flags[turn];
            // The mark after the next one: no thread is past the next barrier.
            turn = turn == 2 ? 0 : turn + 1;
            if (threadIdx.x == 0)
                flags[turn == 2 ? 0 : turn + 1] = 0;
            if (row0 + 16 * wave >= rows)
                continue;

            v4f s[NB];
#pragma unroll
            for (int c = 0; c < NB; ++c)
                s[c] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    uint32_t chunk = 4 * u + q;
                    // Past the row's end a lane reads columns that the query's zeros drop.
                    if (DK % 32 != 0 && u == U - 1 && q >= 2)
                        chunk -= 2;
                    v4u k[PARTS];
#pragma unroll
                    for (int i = 0; i < PARTS; ++i)
                        k[i] = *reinterpret_cast<const v4u *>(stage + i * S::KEY_PLANE +
                                                              swizzled<DK>(16 * c + j, chunk));
                    s[c] = products<HALF>(k, query[u], s[c]);
                }
            float top = -__builtin_inff();
            if (of_run || marks) {
                const int first = int(k0) - int(length);  // the run's token at key 0
#pragma unroll
                for (int c = 0; c < NB; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t at = 16 * c + 4 * q + r;
                        const int i = first + int(at);
                        bool seen = k0 + at <= last_key;
                        if (p.mask) {
                            if (i >= 0)
                                seen = seen && uint32_t(i) < 8 * p.mask_bytes &&
                                       (mask[uint32_t(i) >> 3] >> (i & 7) & 1);
                        } else {
                            seen = seen && i <= int(token);
                        }
                        poison |= seen && (marks >> at & 1);
                        s[c][r] = seen ? s[c][r] * factor : -__builtin_inff();
                        top = fmaxf(top, s[c][r]);
                    }
            } else {
#pragma unroll
                for (int c = 0; c < NB; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[c][r] *= factor;
                        top = fmaxf(top, s[c][r]);
                    }
            }
            top = fmaxf(m, quad_max(top));
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
            const uint16_t *value_stage = LATENT ? stage : stage + PARTS * S::KEY_PLANE;
            constexpr int VALUE_PLANE = LATENT ? S::KEY_PLANE : S::VALUE_PLANE;
#pragma unroll
            for (int h = 0; h < NB / 2; ++h) {  // 32 keys, a product's depth
                v4u prob[QP];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t parts[QP];
                    split_pair<HALF>(s[2 * h + e / 2][2 * (e % 2)],
                                     s[2 * h + e / 2][2 * (e % 2) + 1], parts);
#pragma unroll
                    for (int i = 0; i < QP; ++i)
                        prob[i][e] = parts[i];
                }
                for_chunks<N>([&](auto first_tile, auto tiles) {
                    constexpr int t0 = first_tile, n = tiles, W = (n + 1) / 2;
                    uint32_t x[PARTS][8][W];
#pragma unroll
                    for (int i = 0; i < PARTS; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t key = 32 * h + 16 * (e / 4) + 4 * q + e % 4;
                            // Columns 16 t0 + n j .. + n - 1.
                            const uint16_t *from = value_stage + i * VALUE_PLANE +
                                                   swizzled<DK>(key, 2 * t0 + n * j / 8) +
                                                   n * j % 8;
                            if constexpr (n == 8) {
                                const v4u piece = *reinterpret_cast<const v4u *>(from);
                                x[i][e][0] = piece[0], x[i][e][1] = piece[1];
                                x[i][e][2] = piece[2], x[i][e][3] = piece[3];
                            } else if constexpr (n == 4) {
                                const v2u piece = *reinterpret_cast<const v2u *>(from);
                                x[i][e][0] = piece[0], x[i][e][1] = piece[1];
                            } else if constexpr (n == 2) {
                                x[i][e][0] = *reinterpret_cast<const uint32_t *>(from);
                            } else {
                                x[i][e][0] = *from;
                            }
                        }
#pragma unroll
                    for (int t = 0; t < n; ++t) {
                        v4u v[PARTS];
#pragma unroll
                        for (int i = 0; i < PARTS; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                v[i][e] = __builtin_amdgcn_perm(
                                    x[i][2 * e + 1][t / 2], x[i][2 * e][t / 2],
                                    t % 2 ? 0x07060302u : 0x05040100u);
                        o[t0 + t] = products<HALF>(v, prob, o[t0 + t]);
                    }
                });
            }
        }

        l = quad_sum(poison ? __builtin_nanf("") : l);
        if (real) {
            float *to = part.whole
                            ? p.out + query_row * DV
                            : p.records + (uint64_t(part.record) * kRows + 16 * wave + j) * DV;
            // Nothing attended: zeros.
            const float scale = !part.whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            for_chunks<N>([&](auto first_tile, auto tiles) {
                constexpr int t0 = first_tile, n = tiles;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float *at = to + 16 * t0 + n * (4 * q + r);
                    if constexpr (n % 4 == 0) {
#pragma unroll
                        for (int t = 0; t < n; t += 4)
                            *reinterpret_cast<v4f *>(at + t) =
                                v4f{o[t0 + t][r], o[t0 + t + 1][r], o[t0 + t + 2][r],
                                    o[t0 + t + 3][r]} * scale;
                    } else {
#pragma unroll
                        for (int t = 0; t < n; ++t)
                            at[t] = o[t0 + t][r] * scale;
                    }
                }
            });
            if (!part.whole && q == 0)
                reinterpret_cast<v2f *>(record_stats(p))[uint64_t(part.record) * kRows +
                                                         16 * wave + j] = v2f{m, l};
        }
        if (part.leads && !part.whole)
            share = {block_of(line, part.last_unit) - line.block + 1, part.record, part.run.begin,
                     part.run.count, part.kv_head, part.row_tile};
    }
    if (threadIdx.x == 0)
        block_shares(p)[line.block] = share;
}

// A wave per row of a shared item: out = sum_i a_i 2^(m_i - M) / sum_i l_i 2^(m_i - M) over
// the records, in their order.  Lanes are shares of the records, each of the row's
// 4-column pieces.
__global__ __launch_bounds__(kBlock) void run_attention_join_kernel(RunAttention p)
{
    const Share share = block_shares(p)[blockIdx.x];
    const uint32_t in_tile = blockIdx.y * (kBlock / 64) + (threadIdx.x >> 6);
    const uint32_t row = kRows * share.row_tile + in_tile;
    if (!share.count || row >= share.run * p.group)
        return;
    const uint32_t lane = threadIdx.x & 63, d = p.value_dim, pieces = d / 4;
    const uint32_t token = row / p.group, head = share.kv_head * p.group + row - token * p.group;
    float *out = p.out + (uint64_t(share.begin + token) * p.query_heads + head) * d;
    const auto record = [&](uint32_t i) {
        return uint64_t(i ? share.record / 2 * 2 + 2 * i : share.record) * kRows + in_tile;
    };
    const v2f *stats = reinterpret_cast<const v2f *>(record_stats(p));
    float most = -__builtin_inff();
    for (uint32_t i = lane; i < share.count; i += 64)
        most = fmaxf(most, stats[record(i)][0]);
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1)
        most = fmaxf(most, __shfl_xor(most, offset, 64));
    const float base = most == -__builtin_inff() ? 0.0f : most;
    const uint32_t width = pieces < 64 ? pieces : 64, shares = 64 / width, mine = lane / width;
    float total = 0.0f;
    for (uint32_t column = 0; column < pieces; column += width) {
        const uint32_t c = column + lane % width;
        v4f a = {0, 0, 0, 0};
        for (uint32_t group = 0; group < share.count; group += 64) {
            const uint32_t left = share.count - group, count = left < 64 ? left : 64;
            float weight = 0.0f;
            if (lane < count) {
                const v2f stat = stats[record(group + lane)];
                weight = __builtin_amdgcn_exp2f(stat[0] - base);
                if (column == 0)
                    total += stat[1] * weight;
            }
            for (uint32_t i = 0; i < count; i += shares) {
                const uint32_t n = i + mine;
                const float w = __shfl(weight, int(n & 63), 64);
                // A record without a key has no outputs.
                if (n < count && mine < shares && c < pieces && w != 0.0f)
                    a += w * *reinterpret_cast<const v4f *>(p.records + record(group + n) * d + 4 * c);
            }
        }
        if (column == 0) {
#pragma unroll
            for (int offset = 32; offset > 0; offset >>= 1)
                total += __shfl_xor(total, offset, 64);
        }
        v4f sum = a;
        for (uint32_t s = 1; s < shares; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sum[e] += __shfl(a[e], int((lane + s * width) & 63), 64);
        if (mine == 0 && c < pieces)
            *reinterpret_cast<v4f *>(out + 4 * c) = sum * (total == 0.0f ? 0.0f : 1.0f / total);
    }
}

// The kernel of a shape (null: none), the blocks of it that a CU holds, a tile's keys.
struct MatrixKernel {
    void (*run)(RunAttention) = nullptr;
    int resident = 0, shift = 0;
};
template <int DK, int DV, bool LATENT>
MatrixKernel matrix_kernel_of(bool half)
{
    if (half)
        return {run_attention_kernel<DK, DV, true, LATENT>, Shape<DK, DV, true, LATENT>::RESIDENT,
                Shape<DK, DV, true, LATENT>::SHIFT};
    return {run_attention_kernel<DK, DV, false, LATENT>, Shape<DK, DV, false, LATENT>::RESIDENT,
            Shape<DK, DV, false, LATENT>::SHIFT};
}
MatrixKernel matrix_kernel(const RunAttention &p)
{
    const bool half = p.shape.half;
    const uint32_t rope = p.shape.head_dim - p.value_dim;
    if (rope == 0) {
        switch (p.value_dim) {
        case 32: return matrix_kernel_of<32, 32, false>(half);
        case 64: return matrix_kernel_of<64, 64, false>(half);
        case 80: return matrix_kernel_of<80, 80, false>(half);
        case 96: return matrix_kernel_of<96, 96, false>(half);
        case 112: return matrix_kernel_of<112, 112, false>(half);
        case 128: return matrix_kernel_of<128, 128, false>(half);
        case 160: return matrix_kernel_of<160, 160, false>(half);
        case 192: return matrix_kernel_of<192, 192, false>(half);
        case 256: return matrix_kernel_of<256, 256, false>(half);
        default: return {};
        }
    }
    switch (p.value_dim * 1024 + rope) {
    case 128 * 1024 + 32: return matrix_kernel_of<160, 128, true>(half);
    case 128 * 1024 + 64: return matrix_kernel_of<192, 128, true>(half);
    case 256 * 1024 + 32: return matrix_kernel_of<288, 256, true>(half);
    case 256 * 1024 + 64: return matrix_kernel_of<320, 256, true>(half);
    case 512 * 1024 + 32: return matrix_kernel_of<544, 512, true>(half);
    case 512 * 1024 + 64: return matrix_kernel_of<576, 512, true>(half);
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
    // Units stay in 32 bits.
    const uint64_t items = (uint64_t(p.runs.tokens) * p.group / kRows + p.runs.sequences) *
                           p.shape.kv_heads;
    const uint64_t most = items * (kItemUnits + 4 + ((uint64_t(p.longest) + p.runs.tokens) >>
                                                     kernel.shift));
    if (most >= uint64_t(1) << 31)
        return false;
    const uint64_t wanted = (most + kLeastUnits - 1) / kLeastUnits;
    const uint64_t resident = uint64_t(cu_count) * kernel.resident;
    p.blocks = uint32_t(wanted < resident ? wanted : resident);
    return true;
}

size_t run_attention_scratch_bytes(const RunAttention &p)
{
    return size_t(p.blocks) * (2 * size_t(kRows) * (p.value_dim + 2) * sizeof(float) +
                               sizeof(Share));
}

void launch_run_attention(hipStream_t stream, const RunAttention &p)
{
    if (p.blocks) {
        matrix_kernel(p).run<<<p.blocks, kBlock, 0, stream>>>(p);
        run_attention_join_kernel<<<dim3(p.blocks, kRows / (kBlock / 64)), kBlock, 0, stream>>>(p);
        return;
    }
    const uint64_t blocks = uint64_t(p.runs.tokens) * p.query_heads;
    if (!blocks)
        return;
    const size_t bytes = (size_t(p.shape.head_dim) + p.value_dim) * sizeof(float);
    run_attention_general_kernel<<<unsigned(blocks), 64, bytes, stream>>>(p);
}

}  // namespace mfh
