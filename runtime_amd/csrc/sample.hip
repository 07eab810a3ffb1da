// The next token of each row of logits from a given uniform value, under
// temperature, top-k, top-p and min-p.
//
// With m the row's largest logit, w_i = exp((l_i - m) / temperature).  In
// descending order of l (equal values: lower index first) the first top_k
// tokens are kept, of those the shortest run from the start whose weight
// reaches top_p of their weight, of those the ones with w >= min_p.  The token
// is the first index j, in the vocabulary's order, at which the kept weights up
// to j pass u times their sum.
//
// Weights and sums are 64-bit: over a vocabulary of 65536, sums in f32 would
// put a token's border on the wrong side of u for about one draw in a hundred.
//
// One block takes a row and reads it once for each pass; a row stays in the L2.
// Nothing is sorted: every cut is a value and an index (kept: values above, and
// equal ones up to the index).
//
// top-k: the count's bin among equal steps of the logit (ln 2 / 32 temperatures)
// in the row's first tokens gives a value that the cut cannot lie below; one pass
// lists all tokens from there up in LDS, where the cut is found.  top-p: the
// bin in which the row's weight reaches the share is found from a histogram of
// weights (whole numbers of 2^-46 or so, so that the order of additions does not
// matter), its tokens are listed, and the cut is found among them.  The choice is
// made from a list of the kept tokens, or, where they are more than it holds,
// from sums of 256 tokens each.  Rows with more tokens about a cut than the list
// holds (many equal values, or a temperature far above the logits' spread) are
// searched digit by digit of the values' order-preserving keys.
//
// Bound by one CU's vector work per row -- an instruction for every token of 65536
// is 1024 cycles, and a 64-bit exponential about 20 of them -- and by the fetch of
// code that runs once: a pass is a small loop of its own, and what several steps
// need is a function that is called, not inlined (inlined, with loops unrolled by
// 4 to 8, one row of 65536 took 1.5 to 2 times as long).
#include "kernels.hpp"
#include "paged.hpp"

namespace mfh {
namespace {

constexpr int kBlock = 1024;
constexpr int kWaves = kBlock / 64;
constexpr uint32_t kChunk = 4 * kBlock;   // tokens of one float4 a thread
constexpr uint32_t kSegmentChunks = 64;   // chunks whose sums LDS holds
// Bins of a histogram (44 temperatures: what lies below weighs less than 2^-63 of
// the largest), tokens listed about a cut, tokens kept in a list.
constexpr uint32_t kBins = 2048, kList = 2048, kMany = 16384;
constexpr uint32_t kGroups = kSegmentChunks * kWaves;  // of 256 tokens, of a segment

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));  // rows of any width

// An order-preserving whole number for a value, both zeros alike, and back.
__device__ __forceinline__ uint32_t key_of(float v)
{
    const uint32_t bits = __float_as_uint(v + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Inclusive scans over a wave's lanes by DPP moves; lane 63 ends with the sum.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v)
{
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(v)), CTRL, ROWS, 0xf, false);
    const uint32_t hi =
        __builtin_amdgcn_update_dpp(0, int(uint32_t(v >> 32)), CTRL, ROWS, 0xf, false);
    return uint64_t(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t plus(uint64_t a, uint64_t moved_bits) { return a + moved_bits; }
__device__ __forceinline__ double plus(double a, uint64_t moved_bits)
{
    return a + __builtin_bit_cast(double, moved_bits);
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v)
{
    const auto bits = [](T x) { return __builtin_bit_cast(uint64_t, x); };
    v = plus(v, moved<0x111, 0xf>(bits(v)));  // row_shr 1, 2, 4, 8
    v = plus(v, moved<0x112, 0xf>(bits(v)));
    v = plus(v, moved<0x114, 0xf>(bits(v)));
    v = plus(v, moved<0x118, 0xf>(bits(v)));
    v = plus(v, moved<0x142, 0xa>(bits(v)));  // row 0's and 2's last lane to the next row
    v = plus(v, moved<0x143, 0xc>(bits(v)));  // lane 31 to rows 2 and 3
    return v;
}
template <typename T>
__device__ __forceinline__ T lane_value(T v, int lane)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t r =
        uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b >> 32)), lane))) << 32 |
        uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b)), lane));
    return __builtin_bit_cast(T, r);
}
template <typename T>
__device__ __forceinline__ T wave_total(T v)
{
    return lane_value(wave_scan(v), 63);
}

// A kernel's LDS, as functions take it.
struct Shared;
typedef __attribute__((address_space(3))) Shared Lds;

// Global memory, said outright: a pointer that has been in LDS is of no known kind
// to the compiler, whose loads then wait for LDS too.
template <typename T>
using Global = const __attribute__((address_space(1))) T *;

// A row and its temperature: the same for every thread.
struct Row {
    Global<float> logits;
    Global<uint8_t> mask;
    uint32_t width, chunks;
    double per_step;  // 32 / (ln 2 temperature)
    double largest;
};

struct Shared {
    double table[32];  // 2^(j / 32)
    Row row;
    union {
        uint64_t weight[kBins];
        uint32_t count[kBins];
        uint64_t votes[kSegmentChunks * kChunk / 64];
    } bins;
    uint32_t index[kMany];
    float value[kList];
    double weight[kList];
    uint32_t sub[kList];
    double group[kGroups];
    double segment[(1u << 24) / (kSegmentChunks * kChunk)];
    uint64_t scratch[kWaves];
    float floats[kWaves];
    uint32_t flags[kWaves];
    uint32_t found, below;
    uint64_t before;
    uint32_t reached;
};

// The row in scalar registers.
__device__ __forceinline__ Row row_of(Lds *sh)
{
    const auto scalar = [](uint32_t v) {
        return uint32_t(__builtin_amdgcn_readfirstlane(int(v)));
    };
    const auto wide = [&](uint64_t v) {
        return uint64_t(scalar(uint32_t(v >> 32))) << 32 | scalar(uint32_t(v));
    };
    Row row;
    row.logits = (Global<float>)wide((uint64_t)sh->row.logits);
    row.mask = (Global<uint8_t>)wide((uint64_t)sh->row.mask);
    row.width = scalar(sh->row.width);
    row.chunks = scalar(sh->row.chunks);
    row.per_step = __builtin_bit_cast(double, wide(__builtin_bit_cast(uint64_t, sh->row.per_step)));
    row.largest = __builtin_bit_cast(double, wide(__builtin_bit_cast(uint64_t, sh->row.largest)));
    return row;
}

// The thread's four tokens of a chunk, -infinity where there is none or the mask
// leaves it out.
__device__ __forceinline__ v4f load_chunk(const Row &row, uint32_t c)
{
    const uint32_t i = c * kChunk + 4 * threadIdx.x;
    constexpr float kNone = -__builtin_inff();
    v4f v;
    if ((c + 1) * kChunk <= row.width) {
        v = *(Global<v4f_any>)(row.logits + i);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = row.logits[i + e < row.width ? i + e : row.width - 1];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = i + e < row.width ? v[e] : kNone;
    }
    if (row.mask) {
        const uint32_t at = i < row.width ? i : 0;
        const uint32_t bits = row.mask[at >> 3] >> (at & 7);  // a multiple of 4
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = bits >> e & 1 ? v[e] : kNone;
    }
    return v;
}

// f(chunk, values) over chunks [begin, end), AHEAD chunks' loads in flight before
// the first is used; f is in the code AHEAD times.
template <int AHEAD, typename F>
__device__ __forceinline__ void each(const Row &row, uint32_t begin, uint32_t end, F f)
{
#pragma unroll 1
    for (uint32_t c = begin; c < end; c += AHEAD) {
        v4f v[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            v[a] = load_chunk(row, c + a < end ? c + a : end - 1);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            if (c + a < end)
                f(c + a, v[a]);
    }
}
// The same for work that hides a load: the next chunk's is in flight behind it.
template <typename F>
__device__ __forceinline__ void each_next(const Row &row, uint32_t begin, uint32_t end, F f)
{
    v4f next = load_chunk(row, begin);
#pragma unroll 1
    for (uint32_t c = begin; c < end; ++c) {
        const v4f v = next;
        if (c + 1 < end)
            next = load_chunk(row, c + 1);
        f(c, v);
    }
}

// (v - from) / temperature in steps of ln 2 / 32, -65536 at the least; and raised by
// 1.5 * 2^52, which leaves the nearest whole number in the low bits.
constexpr double kRaise = 6755399441055744.0;
__device__ __forceinline__ double steps_of(const Row &row, float v, double from)
{
    return __builtin_fmax((double(v) - from) * row.per_step, -65536.0);
}
__device__ __forceinline__ int whole_of(double raised)
{
    return int(uint32_t(__builtin_bit_cast(uint64_t, raised)));
}
// The bin of a value: whole steps below `from` (0 for what is above, kBins past the
// range).  Monotone in v.
__device__ __forceinline__ uint32_t bin_of(const Row &row, float v, double from)
{
    const int b = -whole_of(steps_of(row, v, from) + kRaise);
    return b < 0 ? 0 : b < int(kBins) ? uint32_t(b) : kBins;
}

// exp((v - largest) / temperature) as 2^(n / 32) 2^(f / 32), |f| <= 1/2, the latter by
// its series to the fifth power: within 2^-47 (the argument's own rounding, where
// a weight matters, and 2^-48 of what the series leaves).  `steps`: -n.
__device__ __forceinline__ double weight_of(Lds *sh, const Row &row, float v, int *steps)
{
    constexpr double k = 0.021660849392498290;  // ln 2 / 32
    const double t = steps_of(row, v, row.largest);
    const double raised = t + kRaise, f = t - (raised - kRaise), f2 = f * f;
    const double low = __builtin_fma(f, k, 1.0);
    const double middle = __builtin_fma(f, k * k * k / 6, k * k / 2);
    const double high = __builtin_fma(f, k * k * k * k * k / 120, k * k * k * k / 24);
    const double e = __builtin_fma(__builtin_fma(high, f2, middle), f2, low);
    const int whole = whole_of(raised);
    *steps = -whole;
    return __builtin_ldexp(sh->table[whole & 31] * e, whole >> 5);
}
__device__ __forceinline__ double weight_of(Lds *sh, const Row &row, float v)
{
    int steps;
    return weight_of(sh, row, v, &steps);
}

template <typename T>
struct Scan {
    T upto, total;
};
// Inclusive scan over the block and its total.
template <typename T>
__device__ __attribute__((noinline)) Scan<T> block_scan(Lds *sh, T v)
{
    static_assert(kWaves <= 16, "one DPP row of waves");
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63)
        sh->scratch[threadIdx.x >> 6] = __builtin_bit_cast(uint64_t, v);
    __syncthreads();
    // Of a row of lanes.
    const T waves = wave_scan(__builtin_bit_cast(T, sh->scratch[threadIdx.x % kWaves]));
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    return {wave ? v + lane_value(waves, int(wave) - 1) : v, lane_value(waves, kWaves - 1)};
}

// max(a, b, c); NaN operands are ignored.
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// The largest of a thread's values, and whether one is NaN.
struct Extremes {
    float most = -__builtin_inff();
    bool nan = false;
    __device__ __forceinline__ void take(v4f v)
    {
        most = max3(max3(most, v[0], v[1]), v[2], v[3]);
        nan = nan || __builtin_isunordered(v[0], v[1]) || __builtin_isunordered(v[2], v[3]);
    }
};
// The largest of the block's, NaN where one is NaN or +infinity.
__device__ __attribute__((noinline)) float join_extremes(Lds *sh, float most, bool nan)
{
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1)
        most = fmaxf(most, __shfl_xor(most, offset, 64));
    const bool any = __any(nan);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        sh->floats[threadIdx.x >> 6] = any ? __builtin_inff() : most;
    __syncthreads();
    most = sh->floats[threadIdx.x % kWaves];
#pragma unroll
    for (int offset = kWaves / 2; offset > 0; offset >>= 1)
        most = fmaxf(most, __shfl_xor(most, offset, 64));
    most = __uint_as_float(__builtin_amdgcn_readfirstlane(int(__float_as_uint(most))));
    return most < __builtin_inff() ? most : __builtin_nanf("");
}

__device__ __attribute__((noinline)) float row_extremes(Lds *sh, uint32_t chunks)
{
    const Row row = row_of(sh);
    Extremes extremes;
    each<4>(row, 0, chunks, [&](uint32_t, v4f v) { extremes.take(v); });
    return join_extremes(sh, extremes.most, extremes.nan);
}

// Weights as whole numbers of 2^-unit: adding 2^(52 - unit) leaves them in the
// low bits.
struct Units {
    double scale, shift;
    __device__ explicit Units(uint32_t width)
    {
        // Their sum over the row stays below 2^63.
        const int most = 62 - (32 - __builtin_clz(width)), unit = most < 46 ? most : 46;
        scale = __builtin_ldexp(1.0, -unit);
        shift = __builtin_ldexp(1.0, 52 - unit);
    }
    __device__ unsigned long long of(double w) const
    {
        return raised(w + shift);
    }
    __device__ unsigned long long raised(double w) const
    {
        return __builtin_bit_cast(uint64_t, w) - __builtin_bit_cast(uint64_t, shift);
    }
};

__device__ __forceinline__ void add_to_bin(Lds *sh, uint32_t b, unsigned long long v)
{
    (void)__hip_atomic_fetch_add(reinterpret_cast<__attribute__((address_space(3))) uint64_t *>(
                                     &sh->bins.weight[b]),
                                 uint64_t(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

__device__ __attribute__((noinline)) void clear_bins(Lds *sh)
{
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kBins; i += kBlock)
        sh->bins.weight[i] = 0;
    __syncthreads();
}

// The bins of the first chunks' tokens below `from`: how many, or (`from` being the
// largest) their weight.
__device__ __attribute__((noinline)) void histogram(Lds *sh, uint32_t chunks, double from,
                                                    bool counts)
{
    const Row row = row_of(sh);
    const Units units(row.width);
    clear_bins(sh);
    if (counts)
        each_next(row, 0, chunks, [&](uint32_t, v4f v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t b = bin_of(row, v[e], from);
                if (b < kBins)
                    add_to_bin(sh, b, 1);
            }
        });
    else
        each_next(row, 0, chunks, [&](uint32_t, v4f v) {
            // All four before the first condition, so that they overlap (the
            // compiler would move each behind its own).
            double w[4];
            int bin[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = weight_of(sh, row, v[e], &bin[e]) + units.shift;
            asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (bin[e] < int(kBins))
                    add_to_bin(sh, uint32_t(bin[e]), units.raised(w[e]));
        });
    __syncthreads();
}

// The first bin with which `goal` is reached, over + the bins before it times
// `unit` being below it (the last bin that holds any where none reaches it), and
// what is over with those before it.  A share of the bins' total takes goal's place
// where `share` is not negative.
struct Found {
    double goal, over;
    uint32_t bin;
    bool reached;
};
__device__ __attribute__((noinline)) Found find_bin(Lds *sh, double goal, double share,
                                                    double over, double unit)
{
    constexpr uint32_t kEach = kBins / kBlock;
    static_assert(kEach == 2, "neighbours of a thread");
    const uint64_t a = sh->bins.weight[2 * threadIdx.x], b = sh->bins.weight[2 * threadIdx.x + 1];
    const Scan<uint64_t> scan = block_scan(sh, a + b);
    const double total = double(scan.total) * unit;
    if (share >= 0.0)
        goal = share > 0.0 ? share * total : 0x1p-60;
    const auto look = [&](uint32_t bin, uint64_t before, uint64_t own) {
        const bool reached = over + double(before + own) * unit >= goal;
        if (own && over + double(before) * unit < goal &&
            (reached || before + own == scan.total)) {
            sh->found = bin;
            sh->before = before;
            sh->reached = reached;
        }
    };
    look(2 * threadIdx.x, scan.upto - a - b, a);
    look(2 * threadIdx.x + 1, scan.upto - b, b);
    __syncthreads();
    return {goal, over + double(sh->before) * unit, sh->found, sh->reached != 0};
}

// The smallest value of a bin up to `b`, -infinity where all finite ones are: by
// halving, from a few neighbours where the steps' rounding allows.
__device__ __attribute__((noinline)) float edge_of(Lds *sh, uint32_t b, double from)
{
    const Row row = row_of(sh);
    const double reach = (double(b) + 0.5) / row.per_step, near = from - reach;
    const double room = 1.5e-7 * __builtin_fabs(near) + 1e-12 * (__builtin_fabs(from) + reach);
    constexpr double kMost = 3.4028234663852886e38;
    uint32_t low = key_of(float(near - room > -kMost ? near - room : -kMost));
    uint32_t high = key_of(float(near + room < kMost ? near + room : kMost));
    const auto within = [&](uint32_t key) { return bin_of(row, value_of(key), from) <= b; };
    if (within(low)) {
        low = key_of(float(-kMost));
        if (within(low))
            return -__builtin_inff();
    }
    if (!within(high))
        high = key_of(float(from));
#pragma unroll 1
    while (high - low > 1) {
        const uint32_t middle = low + (high - low) / 2;
        if (within(middle))
            high = middle;
        else
            low = middle;
    }
    return value_of(high);
}

// The kept tokens: values above `value`, and equal ones up to `index`.
struct Cut {
    float value;
    uint32_t index;
    __device__ bool keeps(float v, uint32_t i) const
    {
        return (v > value) | ((v == value) & (i <= index));  // without branches
    }
};

// The votes of a chunk's tokens for low <= v < high, to LDS: tokens are taken a
// wave's 64 neighbours at a time, so that the words and their bits are in the
// tokens' order.  f(value) is called for each.
template <typename F>
__device__ __forceinline__ void vote_chunks(Lds *sh, const Row &row, uint32_t begin, uint32_t end,
                                            float low, float high, F f)
{
    constexpr uint32_t kRuns = kChunk / kBlock;  // of kBlock tokens, of a chunk
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool first_lane = (threadIdx.x & 63) == 0;
#pragma unroll 1
    for (uint32_t c = begin; c < end; c += 2) {
        float v[2 * kRuns];
#pragma unroll
        for (uint32_t e = 0; e < 2 * kRuns; ++e) {
            const uint32_t i = c * kChunk + e * kBlock + threadIdx.x;
            v[e] = row.logits[i < row.width ? i : row.width - 1];
        }
#pragma unroll
        for (uint32_t e = 0; e < 2 * kRuns; ++e) {
            const uint32_t i = c * kChunk + e * kBlock + threadIdx.x;
            v[e] = i < row.width ? v[e] : -__builtin_inff();
        }
        if (row.mask)
#pragma unroll
            for (uint32_t e = 0; e < 2 * kRuns; ++e) {
                const uint32_t i = c * kChunk + e * kBlock + threadIdx.x;
                const uint32_t at = i < row.width ? i : 0;
                v[e] = row.mask[at >> 3] >> (at & 7) & 1 ? v[e] : -__builtin_inff();
            }
        uint64_t votes[2 * kRuns];
#pragma unroll
        for (uint32_t e = 0; e < 2 * kRuns; ++e)
            votes[e] = __ballot(v[e] >= low && v[e] < high);
        f(v4f{v[0], v[1], v[2], v[3]});
        f(v4f{v[4], v[5], v[6], v[7]});
        // A chunk past the end, of an odd count, has no votes and a place.
        if (first_lane)
#pragma unroll
            for (uint32_t e = 0; e < 2 * kRuns; ++e)
                sh->bins.votes[((c - begin) * kRuns + e) * kWaves + wave] = votes[e];
    }
}

struct Listed {
    uint32_t count;
    float most;  // the row's largest, or NaN (join_extremes)
};
// Lists the indices of the tokens with low <= v < high, but -infinity, in their
// order: as many as are there, or kMany + 1, and no list, where they are more.
__device__ __attribute__((noinline)) Listed list_tokens(Lds *sh, float low, float high)
{
    const Row row = row_of(sh);
    low = fmaxf(low, -3.4028235e38f);
    Extremes extremes;
    uint32_t listed = 0;
#pragma unroll 1
    for (uint32_t begin = 0; begin < row.chunks; begin += kSegmentChunks) {
        const uint32_t end =
            row.chunks - begin < kSegmentChunks ? row.chunks : begin + kSegmentChunks;
        __syncthreads();
        vote_chunks(sh, row, begin, end, low, high, [&](v4f v) { extremes.take(v); });
        __syncthreads();
        // A thread lists the tokens of a run of words.
        const uint32_t words = (end - begin) * (kChunk / 64);
        const uint32_t each_has = (words + kBlock - 1) / kBlock;
        const uint32_t first = threadIdx.x * each_has < words ? threadIdx.x * each_has : words;
        const uint32_t last = first + each_has < words ? first + each_has : words;
        uint64_t mine = 0;
        for (uint32_t w = first; w < last; ++w)
            mine += __popcll(sh->bins.votes[w]);
        const Scan<uint64_t> scan = block_scan(sh, mine);
        if (listed + scan.total <= kMany && mine) {
            uint32_t at = listed + uint32_t(scan.upto - mine);
            for (uint32_t w = first; w < last; ++w)
                for (uint64_t votes = sh->bins.votes[w]; votes; votes &= votes - 1)
                    sh->index[at++] = begin * kChunk + 64 * w + __builtin_ctzll(votes);
        }
        listed = listed + scan.total < kMany + 1 ? uint32_t(listed + scan.total) : kMany + 1;
    }
    return {listed, join_extremes(sh, extremes.most, extremes.nan)};
}

// How many equal tokens of weight `each` fit above `above` short of `goal`: those
// whose predecessors' weight is below it.
__device__ __forceinline__ uint32_t ties_within(double goal, double above, double each)
{
    const double fit = __builtin_ceil((goal - above) / each);
    return fit < 1.0 ? 1 : fit < 1e9 ? uint32_t(fit) : 1000000000u;
}

// Where `goal` (or a share of all) is reached among the n listed tokens that
// `first` keeps: the smallest value with less than it (counts, or weights) above,
// `over` among that, and the index of the last equal token whose predecessors stay
// below it.  Bins are (steps below `from` - offset) * zoom; their tokens are few
// (unless they are equal): one wave tries the values of up to 64 at once, or
// halves the range of more.
__device__ __attribute__((noinline)) Cut list_cut(Lds *sh, uint32_t n, bool counts, double goal,
                                                  double share, double over, Cut first,
                                                  double from, double offset, double zoom)
{
    const Row row = row_of(sh);
    const Units units(row.width);
    const uint32_t lane = threadIdx.x & 63;
    const auto bin = [&](float v) {
        const double x = (-steps_of(row, v, from) - offset) * zoom;
        return x < 0.0 ? 0u : x < double(kBins - 1) ? uint32_t(x) : kBins - 1;
    };
    clear_bins(sh);
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < n; i += kBlock) {
        const float v = row.logits[sh->index[i]];
        const double w = counts ? 1.0 : weight_of(sh, row, v);
        sh->value[i] = v;
        sh->weight[i] = w;
        if (first.keeps(v, sh->index[i]))
            add_to_bin(sh, bin(v), counts ? 1ull : units.of(w));
    }
    __syncthreads();
    const Found found = find_bin(sh, goal, share, over, counts ? 1.0 : units.scale);
    // The bin's tokens in their order: a thread looks at neighbours.
    const auto in = [&](uint32_t i) {
        return i < n && first.keeps(sh->value[i], sh->index[i]) && bin(sh->value[i]) == found.bin;
    };
    static_assert(kList == 2 * kBlock, "neighbours of a thread");
    const bool a = in(2 * threadIdx.x), b = in(2 * threadIdx.x + 1);
    const Scan<uint64_t> scan = block_scan(sh, uint64_t(a) + b);
    if (a)
        sh->sub[scan.upto - a - b] = 2 * threadIdx.x;
    if (b)
        sh->sub[scan.upto - b] = 2 * threadIdx.x + 1;
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t m = __builtin_amdgcn_readfirstlane(uint32_t(scan.total));
        const auto above_of = [&](uint32_t key) {
            double above = 0.0;
            for (uint32_t i = lane; i < m; i += 64) {
                const uint32_t t = sh->sub[i];
                if (key_of(sh->value[t]) > key)
                    above += sh->weight[t];
            }
            return found.over + wave_total(above);
        };
        uint32_t high;
        if (m <= 64) {
            const uint32_t t = sh->sub[lane < m ? lane : 0];
            const float value = sh->value[t];
            const double weight = sh->weight[t];
            double above = found.over;
#pragma unroll 1
            for (uint32_t i = 0; i < m; ++i) {
                const float other = __uint_as_float(uint32_t(
                    __builtin_amdgcn_readlane(int(__float_as_uint(value)), int(i))));
                above += other > value ? lane_value(weight, int(i)) : 0.0;
            }
            // The largest always qualifies.
            high = above < found.goal ? key_of(value) : UINT32_MAX;
#pragma unroll
            for (int step = 32; step > 0; step >>= 1) {
                const uint32_t other = __shfl_xor(high, step, 64);
                high = other < high ? other : high;
            }
            high = __builtin_amdgcn_readfirstlane(high);
        } else {
            uint32_t least = UINT32_MAX, most = 0;
            for (uint32_t i = lane; i < m; i += 64) {
                const uint32_t k = key_of(sh->value[sh->sub[i]]);
                least = k < least ? k : least;
                most = k > most ? k : most;
            }
#pragma unroll
            for (int step = 32; step > 0; step >>= 1) {
                const uint32_t c = __shfl_xor(least, step, 64), d = __shfl_xor(most, step, 64);
                least = c < least ? c : least;
                most = d > most ? d : most;
            }
            uint32_t low = __builtin_amdgcn_readfirstlane(least) - 1;
            high = __builtin_amdgcn_readfirstlane(most);
#pragma unroll 1
            while (high - low > 1) {
                const uint32_t middle = low + (high - low) / 2;
                if (above_of(middle) < found.goal)
                    high = middle;
                else
                    low = middle;
            }
        }
        const float value = value_of(high);
        uint32_t ties = ties_within(found.goal, above_of(high),
                                    counts ? 1.0 : weight_of(sh, row, value));
        uint32_t index = 0;
#pragma unroll 1
        for (uint32_t base = 0; base < m; base += 64) {
            const uint32_t i = base + lane;
            uint64_t equal = __ballot(i < m && sh->value[sh->sub[i < m ? i : 0]] == value);
            const uint32_t here = __popcll(equal);
            if (!here)
                continue;
            if (here >= ties) {
                for (; ties > 1; --ties)
                    equal &= equal - 1;
                index = sh->index[sh->sub[base + __builtin_ctzll(equal)]];
                break;
            }
            ties -= here;
            index = sh->index[sh->sub[base + 63 - __builtin_clzll(equal)]];
        }
        if (lane == 0) {
            sh->floats[0] = value;
            sh->flags[0] = index;
        }
    }
    __syncthreads();
    const Cut cut = {sh->floats[0], sh->flags[0]};
    __syncthreads();
    return cut;
}

// The same over the whole row, 11 bits of the values' keys at a time: for rows with
// too many tokens about the cut to list.
__device__ __attribute__((noinline)) Cut digit_cut(Lds *sh, bool counts, double goal, double share,
                                                   Cut first)
{
    const Row row = row_of(sh);
    const Units units(row.width);
    const double unit = counts ? 1.0 : units.scale;
    double over = 0.0;
    uint32_t prefix = 0;  // the digits found, in place
    constexpr uint32_t kDigit = kBins - 1;
#pragma unroll 1
    for (int low = 21; low >= -1; low -= 11) {
        // Digits of bits 31 .. 21, 20 .. 10 and 9 .. 0.
        const uint32_t shift = low > 0 ? low : 0, above = low > 0 ? low + 11 : 10;
        const uint32_t digit = (1u << (above - shift)) - 1;
        clear_bins(sh);
        each_next(row, 0, row.chunks, [&](uint32_t c, v4f v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t key = key_of(v[e]);
                if (v[e] > -__builtin_inff() && (above > 31 || key >> above == prefix >> above) &&
                    first.keeps(v[e], c * kChunk + 4 * threadIdx.x + e))
                    add_to_bin(sh, kDigit - (key >> shift & digit),
                               counts ? 1ull : units.of(weight_of(sh, row, v[e])));
            }
        });
        __syncthreads();
        const Found found = find_bin(sh, goal, share, over, unit);
        goal = found.goal;
        over = found.over;
        share = -1.0;
        prefix |= (kDigit - found.bin) << shift;
    }
    const float value = value_of(prefix);
    uint32_t ties = ties_within(goal, over, counts ? 1.0 : weight_of(sh, row, value));
    // The index of the last of that many equal tokens, by the waves' votes.
    uint32_t last = 0;
#pragma unroll 1
    for (uint32_t begin = 0; begin < row.chunks; begin += kSegmentChunks) {
        const uint32_t end =
            row.chunks - begin < kSegmentChunks ? row.chunks : begin + kSegmentChunks;
        __syncthreads();
        // [value, value] as a range: up to the next value above.
        vote_chunks(sh, row, begin, end, value, value_of(key_of(value) + 1), [](v4f) {});
        __syncthreads();
        const uint32_t words = (end - begin) * (kChunk / 64);
        const uint32_t each_has = (words + kBlock - 1) / kBlock;
        const uint32_t from = threadIdx.x * each_has < words ? threadIdx.x * each_has : words;
        const uint32_t to = from + each_has < words ? from + each_has : words;
        uint64_t mine = 0;
        for (uint32_t w = from; w < to; ++w)
            mine += __popcll(sh->bins.votes[w]);
        const Scan<uint64_t> scan = block_scan(sh, mine);
        const uint64_t wanted = ties < scan.total ? ties : scan.total;  // the last one here, else
        if (scan.total && scan.upto >= wanted && scan.upto - mine < wanted) {
            uint64_t left = wanted - (scan.upto - mine);
            for (uint32_t w = from; w < to && left; ++w)
                for (uint64_t votes = sh->bins.votes[w]; votes && left; votes &= votes - 1, --left)
                    sh->found = begin * kChunk + 64 * w + __builtin_ctzll(votes);
        }
        __syncthreads();
        if (scan.total)
            last = sh->found;
        if (scan.total >= ties)
            break;
        ties -= uint32_t(scan.total);
    }
    __syncthreads();
    return {value, last};
}

// The weights of four tokens that a cut and min_p leave, formed side by side.
__device__ __forceinline__ void terms_of(Lds *sh, const Row &row, v4f v, uint32_t i, Cut cut,
                                         double min_p, double (&w)[4])
{
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = weight_of(sh, row, v[e]);
    asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = bool(cut.keeps(v[e], i + e) & (w[e] >= min_p)) ? w[e] : 0.0;
}

// Sums of the kept weights of each 256 tokens (a wave's float4s) of a segment, in
// sh->group: returns the thread's own and the scan of all.
struct Groups {
    double own, upto, total;
};
__device__ __attribute__((noinline)) Groups group_sums(Lds *sh, uint32_t begin, Cut cut,
                                                       double min_p)
{
    const Row row = row_of(sh);
    begin = __builtin_amdgcn_readfirstlane(begin);
    const uint32_t end =
        row.chunks - begin < kSegmentChunks ? row.chunks : begin + kSegmentChunks;
    __syncthreads();
    each_next(row, begin, end, [&](uint32_t c, v4f v) {
        double sum = 0.0;
        if (__any(max3(max3(v[0], v[1], v[2]), v[3], v[3]) >= cut.value)) {
            double w[4];
            terms_of(sh, row, v, c * kChunk + 4 * threadIdx.x, cut, min_p, w);
            sum = wave_scan((w[0] + w[1]) + (w[2] + w[3]));
        }
        if ((threadIdx.x & 63) == 63)
            sh->group[(c - begin) * kWaves + (threadIdx.x >> 6)] = sum;
    });
    __syncthreads();
    const double own = threadIdx.x < (end - begin) * kWaves ? sh->group[threadIdx.x] : 0.0;
    const Scan<double> scan = block_scan(sh, own);
    return {own, scan.upto, scan.total};
}

// ---- the kernel -------------------------------------------------------------------

__global__ __launch_bounds__(kBlock) void sample_kernel(Sampling s)
{
    __shared__ Shared shared;
    Lds *sh = (Lds *)&shared;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t r = blockIdx.x;
    const float *params = s.params + (s.one_params ? 0 : 4 * uint64_t(r));
    const float u = s.uniforms[r];
    const float temperature = params[0], top_k = params[1], top_p = params[2], min_p = params[3];
    if (threadIdx.x < 32)
        sh->table[threadIdx.x] = exp2(double(threadIdx.x) / 32.0);
    Row row;
    row.width = s.width;
    row.chunks = (s.width + kChunk - 1) / kChunk;
    row.logits = (Global<float>)(s.logits + uint64_t(r) * s.width);
    row.mask = (Global<uint8_t>)(
        s.mask ? s.mask + (s.one_mask ? 0 : uint64_t(r) * ((s.width + 7) / 8)) : nullptr);
    row.per_step = 46.166241308446828384 / double(temperature);
    row.largest = 0.0;
    if (threadIdx.x == 0) {
        sh->row.logits = row.logits;
        sh->row.mask = row.mask;
        sh->row.width = row.width;
        sh->row.chunks = row.chunks;
        sh->row.per_step = row.per_step;
    }
    const auto answer = [&](float token) {
        s.out[r] = token;
        if (s.copy)
            s.copy[r] = token;
    };
    const bool good = temperature >= 0.0f && temperature < __builtin_inff() && top_k >= 0.0f &&
                      truncf(top_k) == top_k && top_p >= 0.0f && top_p <= 1.0f && min_p >= 0.0f &&
                      min_p <= 1.0f && u >= 0.0f && u < 1.0f;
    if (!good) {
        if (threadIdx.x == 0)
            answer(__builtin_nanf(""));
        return;
    }

    if (temperature == 0.0f) {
        // The first largest: a thread's indices increase.
        float best = -__builtin_inff();
        uint32_t first = UINT32_MAX;
        Extremes extremes;
        each<4>(row, 0, row.chunks, [&](uint32_t c, v4f v) {
            extremes.take(v);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v[e] > best) {
                    best = v[e];
                    first = c * kChunk + 4 * threadIdx.x + e;
                }
        });
        const float most = join_extremes(sh, extremes.most, extremes.nan);
        first = best == most ? first : UINT32_MAX;
#pragma unroll
        for (int offset = 32; offset > 0; offset >>= 1) {
            const uint32_t other = __shfl_xor(first, offset, 64);
            first = other < first ? other : first;
        }
        if (lane == 0)
            sh->flags[wave] = first;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kWaves; ++w)
                first = sh->flags[w] < first ? sh->flags[w] : first;
            answer(most > -__builtin_inff() ? float(first) : __builtin_nanf(""));
        }
        return;
    }
    __syncthreads();

    const uint32_t k = top_k > 0.0f && top_k < float(s.width) ? uint32_t(top_k) : 0;
    const double share = top_p < 1.0f ? double(top_p) : -1.0;
    Cut cut = {-__builtin_inff(), UINT32_MAX};
    bool bounded = k || top_p < 1.0f;  // tokens below cut.value are not kept
    uint32_t listed = 0;               // tokens of the list, where it holds every kept one
    Listed list = {0, 0.0f};
    if (k) {
        // A value that the k-th largest of the row does not lie below: of the
        // first tokens, enough for about 1024 listed ones.
        float floor = -__builtin_inff();
        if (s.width > kList) {
            uint32_t chunks = uint32_t((uint64_t(row.chunks) * k + 1023) / 1024);
            chunks = chunks < row.chunks ? chunks : row.chunks;
            const float from = row_extremes(sh, chunks);
            if (from > -__builtin_inff()) {
                histogram(sh, chunks, double(from), true);
                const Found found = find_bin(sh, double(k), -1.0, 0.0, 1.0);
                // Tokens past the bins' range weigh nothing: its end bounds too.
                floor = edge_of(sh, found.reached ? found.bin : kBins - 1, double(from));
            }
        }
        list = list_tokens(sh, floor, __builtin_inff());
    } else {
        list.most = row_extremes(sh, row.chunks);
    }
    if (!(list.most > -__builtin_inff())) {
        if (threadIdx.x == 0)
            answer(__builtin_nanf(""));
        return;
    }
    const double from = row.largest = double(list.most);
    if (threadIdx.x == 0)
        sh->row.largest = from;
    __syncthreads();
    if (k && list.count <= kList) {
        listed = list.count;
        if (listed > k)
            cut = list_cut(sh, listed, true, double(k), -1.0, 0.0, cut, from, -0.5, 1.0);
        if (share >= 0.0)
            cut = list_cut(sh, listed, false, 0.0, share, 0.0, cut, from, -0.5, 1.0);
    } else if (k) {
        cut = digit_cut(sh, true, double(k), -1.0, cut);
        if (share >= 0.0)
            cut = digit_cut(sh, false, 0.0, share, cut);
    } else if (share >= 0.0) {
        histogram(sh, row.chunks, from, false);
        const Found found = find_bin(sh, 0.0, share, 0.0, Units(s.width).scale);
        const float low = edge_of(sh, found.bin, from);
        const float high = found.bin ? edge_of(sh, found.bin - 1, from) : __builtin_inff();
        const uint32_t n = list_tokens(sh, low, high).count;
        // Within the bin: its own equal steps.
        cut = n <= kList ? list_cut(sh, n, false, found.goal, -1.0, found.over, cut, from,
                                    double(found.bin) - 0.5, double(kBins))
                         : digit_cut(sh, false, found.goal, -1.0, cut);
    }
    if (min_p > 0.0f) {
        // A value whose weight is surely below min_p: a bound, with room for
        // its own rounding; the weights themselves decide.
        const float bound =
            list.most + temperature * (logf(min_p) - 0.01f) - 1e-5f * fabsf(list.most);
        if (bound > cut.value)
            cut = {bound, UINT32_MAX};
        bounded = true;
    }
    const auto term = [&](float v, uint32_t i) {
        const double w = weight_of(sh, row, v);
        return bool(cut.keeps(v, i) & (w >= double(min_p))) ? w : 0.0;
    };
    if (bounded && !listed) {
        const uint32_t n = list_tokens(sh, cut.value, __builtin_inff()).count;
        listed = n <= kMany ? n : 0;
    }

    // The choice: the first kept token at which their sum passes the target (the
    // last kept one where rounding leaves none).
    if (threadIdx.x == 0) {
        sh->found = UINT32_MAX;
        sh->below = 0;
    }
    if (listed) {
        // A thread has neighbours of the list.
        const uint32_t each_has = (listed + kBlock - 1) / kBlock;
        const uint32_t first = threadIdx.x * each_has < listed ? threadIdx.x * each_has : listed;
        const uint32_t last = first + each_has < listed ? first + each_has : listed;
        double mine = 0.0, at = 0.0, target = __builtin_inf();
        uint32_t token = 0;
        // Sums, then a walk by the thread that holds the target.
#pragma unroll 1
        for (int walk = 0; walk < 2; ++walk) {
            double sum = 0.0;
#pragma unroll 1
            for (uint32_t i = first; i < last; ++i) {
                const double t = term(row.logits[sh->index[i]], sh->index[i]);
                sum += t;
                if (walk && t > 0.0) {
                    token = sh->index[i];
                    if (at + sum > target)
                        break;
                }
            }
            if (walk) {
                answer(float(token));
                return;
            }
            mine = sum;
            const Scan<double> scan = block_scan(sh, mine);
            target = double(u) * scan.total;
            at = scan.upto - mine;
            if (mine > 0.0) {
                if (scan.upto > target)
                    atomicMin(&shared.found, threadIdx.x);
                atomicMax(&shared.below, threadIdx.x);
            }
            __syncthreads();
            if (threadIdx.x != (sh->found != UINT32_MAX ? sh->found : sh->below))
                return;
        }
    }
    // Too many for the list: sums of 256 tokens (a wave's float4s), of the segment
    // that holds the target, then that wave's lanes.
    const uint32_t segments = (row.chunks + kSegmentChunks - 1) / kSegmentChunks;
    double total = 0.0, passed = 0.0, target = 0.0;
    uint32_t begin = 0;
    Groups groups = {0.0, 0.0, 0.0};
    // Every segment's sum; then, of several, the one that holds the target again.
#pragma unroll 1
    for (uint32_t g = 0; g <= segments; ++g) {
        if (g == segments) {
            target = double(u) * total;
            if (segments == 1)
                break;
            // The first that passes the target (the last with a token where
            // rounding leaves none).
            __syncthreads();
            uint32_t chosen = 0;
            double at = 0.0;
            for (uint32_t i = 0; i < segments; ++i) {
                const double sum = sh->segment[i];
                if (sum > 0.0) {
                    chosen = i;
                    passed = at;
                }
                at += sum;
                if (sum > 0.0 && at > target)
                    break;
            }
            begin = chosen * kSegmentChunks;
        } else {
            begin = g * kSegmentChunks;
        }
        groups = group_sums(sh, begin, cut, double(min_p));
        if (g < segments) {
            if (threadIdx.x == 0)
                sh->segment[g] = groups.total;
            total += groups.total;
        }
    }
    // The first group that passes it, likewise.
    if (groups.own > 0.0) {
        if (passed + groups.upto > target)
            atomicMin(&shared.found, threadIdx.x);
        atomicMax(&shared.below, threadIdx.x);
    }
    __syncthreads();
    const uint32_t group = sh->found != UINT32_MAX ? sh->found : sh->below;
    if (threadIdx.x == group)
        sh->segment[0] = passed + (groups.upto - groups.own);
    __syncthreads();
    if (wave != group % kWaves)
        return;
    const double start = sh->segment[0];
    const uint32_t chunk = begin + group / kWaves;
    const v4f v = load_chunk(row, chunk);
    const uint32_t i = chunk * kChunk + 4 * threadIdx.x;
    double w[4];
    terms_of(sh, row, v, i, cut, double(min_p), w);
    const double own = (w[0] + w[1]) + (w[2] + w[3]);
    const double upto = wave_scan(own);
    const uint64_t some = __ballot(own > 0.0);
    const uint64_t past = __ballot(own > 0.0 && start + upto > target);
    if (!some)
        return;  // not reached: the group's sum is positive
    if (lane == (past ? uint32_t(__builtin_ctzll(past)) : 63 - uint32_t(__builtin_clzll(some)))) {
        double at = start + (upto - own);
        uint32_t token = i;
        bool passed_it = false;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (w[e] > 0.0 && !passed_it) {
                at += w[e];
                token = i + e;
                passed_it = at > target;
            }
        answer(float(token));
    }
}

}  // namespace

void launch_sample_rows(hipStream_t stream, const Sampling &s)
{
    if (s.rows)
        sample_kernel<<<s.rows, kBlock, 0, stream>>>(s);
}

}  // namespace mfh
