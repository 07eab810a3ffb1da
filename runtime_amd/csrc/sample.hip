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
// top-k: the count's bin among equal steps of the logit (ln 2 / 32 temperatures, or 64
// times that) in the row's first tokens gives a value that the cut cannot lie below; one pass
// lists all tokens from there up in LDS, where the cut is found.  top-p: the
// bin in which the row's weight reaches the share is found from a histogram of
// weights (whole numbers, of units that follow the bins, so that the order of additions
// does not matter), its tokens are listed, and the cut is found among them.  The choice is
// made from a list of the tokens down to there, or, where they are more than it
// holds, of all.  Rows with more tokens about a cut than the list
// holds (many equal values, or a temperature far above the logits' spread) are
// searched digit by digit of the values' order-preserving keys.
//
// Bound by one CU's vector work per row -- an instruction for every token of 65536
// is 1024 cycles, and a 64-bit exponential about 14 of them --, by its reads (a pass
// without work takes 9000 cycles), and by the fetch of code that runs once: a pass is
// a small loop of its own, and what several steps need is a function that is called,
// not inlined (inlined, with loops unrolled by 4 to 8, one row of 65536 took 1.5 to 2
// times as long).  One row of 65536 takes, in us: greedy 6.2, min-p 12, all
// tokens 20, top-k 50 18.1 and with top-p 21.3, top-p 0.9 at temperatures 0.6 / 1 /
// 1.5 27.6 / 32.5 / 41.3; 192 rows 11, 21, 27, 23 and 27, 38 / 47 / 54.
#include "kernels.hpp"
#include "paged.hpp"

namespace mfh {
namespace {

constexpr int kBlock = 1024;
constexpr int kWaves = kBlock / 64;
constexpr uint32_t kChunk = 4 * kBlock;   // tokens of one float4 a thread
constexpr uint32_t kSegmentChunks = 32;   // chunks whose codes LDS holds
// Bins of a histogram (44 temperatures: what lies below weighs less than 2^-63 of
// the largest), tokens listed about a cut, tokens kept in a list.
constexpr uint32_t kBins = 2048, kList = 2048, kMany = 16384;

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
template <int LANES>
__device__ __forceinline__ uint32_t lanes_scan(uint32_t v)  // of a row's 16 lanes, or all
{
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x111, 0xf, 0xf, false));
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x112, 0xf, 0xf, false));
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x114, 0xf, 0xf, false));
    v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x118, 0xf, 0xf, false));
    if constexpr (LANES == 64) {
        v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x142, 0xa, 0xf, false));
        v += uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x143, 0xc, 0xf, false));
    }
    return v;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane)
{
    return uint32_t(__builtin_amdgcn_readlane(int(v), lane));
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

// f over a wave's values, or the first row's 16 lanes, by the same moves.
template <int CTRL, int ROWS, typename F>
__device__ __forceinline__ uint32_t joined(uint32_t v, F f)
{
    return f(v, uint32_t(__builtin_amdgcn_update_dpp(int(v), int(v), CTRL, ROWS, 0xf, false)));
}
template <bool ROW, typename F>
__device__ __forceinline__ uint32_t wave_join(uint32_t v, F f)
{
    v = joined<0x111, 0xf>(v, f);
    v = joined<0x112, 0xf>(v, f);
    v = joined<0x114, 0xf>(v, f);
    v = joined<0x118, 0xf>(v, f);
    if constexpr (!ROW) {
        v = joined<0x142, 0xa>(v, f);
        v = joined<0x143, 0xc>(v, f);
    }
    return __builtin_amdgcn_readlane(int(v), ROW ? 15 : 63);
}
template <bool ROW = false>
__device__ __forceinline__ float wave_largest(float v)
{
    return __uint_as_float(wave_join<ROW>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <bool ROW = false>
__device__ __forceinline__ uint32_t wave_least(uint32_t v)
{
    return wave_join<ROW>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
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
        uint64_t weight[2 * kBins];  // the second half for Bins::two
        uint64_t codes[kSegmentChunks * kBlock / 8];  // a byte for four tokens
    } bins;
    uint32_t index[kMany];
    uint32_t pick[kList];
    float value[kList];
    double weight[kList];
    uint32_t sub[kList];
    uint64_t scratch[kWaves];
    float floats[kWaves];
    uint32_t flags[kWaves];
    uint32_t found;
    uint32_t reached;
    double over;
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

// Tokens i .. i + 3, -infinity where there is none or the mask leaves it out;
// `whole`: they are all there, for every thread.
__device__ __forceinline__ v4f load_four(const Row &row, uint32_t i, bool whole)
{
    constexpr float kNone = -__builtin_inff();
    v4f v;
    if (whole) {
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
__device__ __forceinline__ v4f load_chunk(const Row &row, uint32_t c)
{
    return load_four(row, c * kChunk + 4 * threadIdx.x, (c + 1) * kChunk <= row.width);
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
            if (c + a < end)
                v[a] = load_chunk(row, c + a);
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

// (v - from) / temperature in steps of ln 2 / 32, and its whole part (towards zero;
// what an int does not hold, -infinity too, is its least or largest).
__device__ __forceinline__ double steps_of(const Row &row, float v, double from)
{
    return (double(v) - from) * row.per_step;
}
__device__ __forceinline__ int whole_of(double steps)
{
    int whole;
    asm("v_cvt_i32_f64 %0, %1" : "=v"(whole) : "v"(steps));
    return whole;
}
// The bin of that: whole steps below `from` (0 for what is above, kBins past the
// range).  Monotone in v.
__device__ __forceinline__ uint32_t bin_of(const Row &row, float v, double from)
{
    const int n = whole_of(steps_of(row, v, from));
    const uint32_t b = 0u - uint32_t(n);
    return n > 0 ? 0 : b < kBins ? b : kBins;
}

// exp((v - largest) / temperature) as 2^(n / 32) 2^(-f / 32), 0 <= f < 1, the latter
// by the polynomial of fourth degree, 1 at 0, that is nearest to it (2^-43.3; the
// argument's own rounding is less where a weight matters).  Of no meaning for
// -infinity.  graded_of: without the power of two's whole part, so in (0.97, 1.96), and
// `steps`: n.
__device__ __forceinline__ double graded_of(Lds *sh, const Row &row, float v, int *steps)
{
    const double t = steps_of(row, v, row.largest), f = __builtin_amdgcn_fract(-t);
    const int n = whole_of(t);
    double e = __builtin_fma(f, 9.076184072276023e-09, -1.6937700541791561e-06);
    e = __builtin_fma(e, f, 0.0002345961713900732);
    e = __builtin_fma(e, f, -0.021660849389733828);
    e = __builtin_fma(e, f, 1.0);
    *steps = n;
    return sh->table[n & 31] * e;
}
__device__ __forceinline__ double weight_of(Lds *sh, const Row &row, float v)
{
    int steps;
    const double graded = graded_of(sh, row, v, &steps);
    return __builtin_ldexp(graded, steps >> 5);
}

// Of lanes with `some` of what is summed, the one that holds a target: the first that
// reaches it (`past`), or else the last.
__device__ __forceinline__ uint32_t holder(bool some, bool past)
{
    const uint64_t with = __ballot(some), over = __ballot(some && past);
    return over ? __builtin_ctzll(over) : with ? 63 - __builtin_clzll(with) : 0;
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
// The largest of some values, NaN where one is NaN or +infinity (which a wave with a
// NaN says it has).
__device__ __forceinline__ float extremes_of(float most)
{
    return most < __builtin_inff() ? most : __builtin_nanf("");
}
// The largest of the block's, or NaN (extremes_of).
__device__ __attribute__((noinline)) float join_extremes(Lds *sh, float most, bool nan)
{
    most = wave_largest(most);
    const bool any = __any(nan);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        sh->floats[threadIdx.x >> 6] = any ? __builtin_inff() : most;
    __syncthreads();
    return extremes_of(wave_largest<true>(sh->floats[threadIdx.x % kWaves]));
}

__device__ __attribute__((noinline)) float row_extremes(Lds *sh, uint32_t chunks)
{
    const Row row = row_of(sh);
    Extremes extremes;
    each<4>(row, 0, chunks, [&](uint32_t, v4f v) { extremes.take(v); });
    return join_extremes(sh, extremes.most, extremes.nan);
}

// Values below 1.96 as whole numbers of 2^-unit, of which `count` add up below 2^64:
// adding 2^(52 - unit) leaves them in the low bits.
struct Units {
    double scale, shift;
    __device__ explicit Units(uint32_t count)
    {
        const int most = 63 - (32 - __clz(int(count - 1))), unit = most < 51 ? most : 51;
        scale = __builtin_ldexp(1.0, -unit);
        shift = __builtin_ldexp(1.0, 52 - unit);
    }
    __device__ unsigned long long of(double w) const
    {
        return raised(w + shift);
    }
    // What lies behind the exponent, which is shift's.
    __device__ unsigned long long raised(double w) const
    {
        return __builtin_bit_cast(uint64_t, w) & 0xfffffffffffffull;
    }
};

// What a bin's whole number stands for.  A row's weights span 2^64, so in units that are
// fine enough for one of them another is lost: bins of steps hold graded weights, each
// bin's in units of its own power of two, and every weight keeps 38 bits or more in rows
// of 2^24 (46 at 65536).  Where a bin's weights have no power in common there are two
// words, the second of what the first's units leave.
enum class Bins { plain, steps, two };
// The power of two that weights `steps` whole steps below the largest are graded by.
__device__ __forceinline__ int grade_of(uint32_t steps)
{
    return -int(steps) >> 5;
}

// Bins stand in reverse: bin b in slot kBins - 1 - b.
__device__ __forceinline__ void add_to_slot(Lds *sh, int slot, unsigned long long v)
{
    (void)__hip_atomic_fetch_add(reinterpret_cast<__attribute__((address_space(3))) uint64_t *>(
                                     &sh->bins.weight[slot]),
                                 uint64_t(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
__device__ __forceinline__ void add_to_bin(Lds *sh, uint32_t b, unsigned long long v)
{
    add_to_slot(sh, int(kBins - 1 - b), v);
}

__device__ __attribute__((noinline)) void clear_bins(Lds *sh, Bins kind)
{
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < (kind == Bins::two ? 2 : 1) * kBins; i += kBlock)
        sh->bins.weight[i] = 0;
    __syncthreads();
}

// The bins of the first chunks' tokens below `from`: how many, or (`from` being the
// largest) their graded weights.
__device__ __attribute__((noinline)) void histogram(Lds *sh, uint32_t chunks, double from,
                                                    bool counts)
{
    const Row row = row_of(sh);
    const Units units(row.width);
    clear_bins(sh, Bins::plain);
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
                w[e] = graded_of(sh, row, v[e], &bin[e]) + units.shift;
            asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (bin[e] > -int(kBins))
                    add_to_slot(sh, int(kBins - 1) + bin[e], units.raised(w[e]));
        });
    __syncthreads();
}

// The first bin with which `goal` is reached, over + the bins before it being below it
// (the last bin that holds any where none reaches it), and what is over with those
// before it.  A whole number of a bin stands for `unit`, by `kind`.  A share of the
// bins' total takes goal's place where `share` is not negative.
struct Found {
    double goal, over;
    uint32_t bin;
    bool reached;
};
__device__ __attribute__((noinline)) Found find_bin(Lds *sh, double goal, double share,
                                                    double over, double unit, Bins kind)
{
    constexpr uint32_t kEach = kBins / kBlock;
    static_assert(kEach == 2, "neighbours of a thread");
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const auto held = [&](uint32_t bin) {
        const uint32_t slot = kBins - 1 - bin;
        double v = double(sh->bins.weight[slot]) * unit;
        if (kind == Bins::steps)
            v = __builtin_ldexp(v, grade_of(bin));
        if (kind == Bins::two)
            v += double(sh->bins.weight[kBins + slot]) * (unit * unit);
        return v;
    };
    const double a = held(2 * threadIdx.x), b = held(2 * threadIdx.x + 1);
    const double scan = wave_scan(a + b);
    if (lane == 63)
        sh->scratch[wave] = __builtin_bit_cast(uint64_t, scan);
    __syncthreads();
    // Every wave finds the one that holds the goal; that one alone goes on.
    const double own = __builtin_bit_cast(double, sh->scratch[lane % kWaves]);
    const double upto = wave_scan(own);  // a row's
    if (share >= 0.0)
        goal = share > 0.0 ? share * lane_value(upto, kWaves - 1) : 0x1p-60;
    const uint32_t here = holder(lane < kWaves && own > 0.0, over + upto >= goal);
    if (wave == here) {
        // Boundaries of the thread's bins: sums that neighbours share.
        const double base = here ? lane_value(upto, int(here) - 1) : 0.0;
        const double before =  // the lane's before, zero for the first
            __builtin_bit_cast(double, moved<0x138, 0xf>(__builtin_bit_cast(uint64_t, scan)));
        const double from = over + (base + before), to = over + (base + scan);
        const double middle = from + a;
        const bool reached = to >= goal;
        if (lane == holder(a + b > 0.0, reached)) {
            const bool first = a > 0.0 && (!(b > 0.0) || middle >= goal);
            sh->found = 2 * threadIdx.x + (first ? 0 : 1);
            sh->over = first ? from : middle;
            sh->reached = reached;
        }
    }
    __syncthreads();
    return {goal, sh->over, sh->found, sh->reached != 0};
}

// The smallest value of a bin up to `b`, -infinity where all finite ones are: by
// halving, from a few neighbours where the steps' rounding allows.
__device__ __forceinline__ float edge_of(const Row &row, uint32_t b, double from)
{
    const double reach = (double(b) + 1.0) / row.per_step, near = from - reach;
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

// The smallest values of bins up to `b` and, for all but bin 0, up to b - 1: by a wave
// each.
struct Edges {
    float low, high;
};
__device__ __attribute__((noinline)) Edges edges_of(Lds *sh, uint32_t b, double from)
{
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave < 2) {
        const Row row = row_of(sh);
        const float edge = wave > b ? __builtin_inff() : edge_of(row, b - wave, from);
        if ((threadIdx.x & 63) == 0)
            sh->floats[wave] = edge;
    }
    __syncthreads();
    return {sh->floats[0], sh->floats[1]};
}

// Bins of counts where a temperature's are too narrow: 64 times as wide.
constexpr double kWider = 1.0 / 64.0;

// The kept tokens: values above `value`, and equal ones up to `index`.
struct Cut {
    float value;
    uint32_t index;
    __device__ bool keeps(float v, uint32_t i) const
    {
        return (v > value) | ((v == value) & (i <= index));  // without branches
    }
};

// Codes of chunks to LDS, a byte for a thread's four tokens: bit e for low <= v, and
// bit 4 + e where also v < high.  f(values) is called for each.
constexpr uint64_t kListed = 0x0f0f0f0f0f0f0f0full;
template <typename F>
__device__ __forceinline__ void code_chunks(Lds *sh, const Row &row, uint32_t begin, uint32_t end,
                                            float low, float high, F f)
{
    const auto codes = reinterpret_cast<__attribute__((address_space(3))) uint8_t *>(
        &sh->bins.codes[0]);
    each<4>(row, begin, end, [&](uint32_t c, v4f v) {
        f(v);
        uint32_t code = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t both = v[e] < high ? 0x11u << e : 1u << e;
            code |= v[e] >= low ? both : 0;
        }
        codes[(c - begin) * kBlock + threadIdx.x] = uint8_t(code);
    });
}
// A thread's run of a segment's code words (eight bytes, 32 tokens).
struct Words {
    uint32_t first, last;
    __device__ __forceinline__ explicit Words(uint32_t chunks)
    {
        const uint32_t words = chunks * (kBlock / 8), each_has = (words + kBlock - 1) / kBlock;
        first = threadIdx.x * each_has < words ? threadIdx.x * each_has : words;
        last = first + each_has < words ? first + each_has : words;
    }
};
// The token of a word's lowest bit, of those in kListed.
__device__ __forceinline__ uint32_t token_of(uint32_t begin, uint32_t word, uint64_t bits)
{
    const uint32_t bit = __builtin_ctzll(bits);
    return begin * kChunk + 32 * word + 4 * (bit >> 3) + (bit & 7);
}

struct Listed {
    uint32_t count, picked;
    float most;  // the row's largest, or NaN (extremes_of), where asked for
};
// Lists the tokens with low <= v, but -infinity, in sh->index and those with also
// v < high in sh->pick, in their order; what passes the lists' ends is counted.
template <bool MOST>
__device__ __attribute__((noinline)) Listed list_tokens(Lds *sh, float low, float high)
{
    const Row row = row_of(sh);
    low = fmaxf(low, -3.4028235e38f);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Extremes extremes;
    uint32_t listed = 0, picked = 0;
#pragma unroll 1
    for (uint32_t begin = 0; begin < row.chunks; begin += kSegmentChunks) {
        const uint32_t end =
            row.chunks - begin < kSegmentChunks ? row.chunks : begin + kSegmentChunks;
        __syncthreads();
        code_chunks(sh, row, begin, end, low, high, [&](v4f v) {
            if constexpr (MOST)
                extremes.take(v);
        });
        __syncthreads();
        const Words words(end - begin);
        // Listed and picked, in two halves of a word: a wave has 8192 tokens at most.
        static_assert(kSegmentChunks * kChunk / kWaves < 65536, "a wave's tokens of a segment");
        uint32_t mine = 0;
        for (uint32_t w = words.first; w < words.last; ++w) {
            const uint64_t word = sh->bins.codes[w];
            mine += __popcll(word & kListed) + (__popcll(word >> 4 & kListed) << 16);
        }
        const uint32_t scan = lanes_scan<64>(mine), before = scan - mine;
        if (lane == 63)
            sh->flags[wave] = scan;
        if constexpr (MOST) {
            const float most = wave_largest(extremes.most);
            const bool bad = __any(extremes.nan);
            if (lane == 63)
                sh->floats[wave] = bad ? __builtin_inff() : most;
        }
        __syncthreads();
        const uint32_t in_wave = sh->flags[lane % kWaves];
        const uint32_t here = in_wave & 0xffff, picks = in_wave >> 16;
        const uint32_t here_upto = lanes_scan<16>(here), picks_upto = lanes_scan<16>(picks);
        uint32_t at = listed + lane_value(here_upto - here, wave) + (before & 0xffff);
        uint32_t pick = picked + lane_value(picks_upto - picks, wave) + (before >> 16);
        listed += lane_value(here_upto, kWaves - 1);
        picked += lane_value(picks_upto, kWaves - 1);
        // Of more than the list holds nothing is listed but what is picked.
        const bool fits = listed <= kMany;
#pragma unroll 1
        for (uint32_t w = words.first; w < words.last; ++w) {
            const uint64_t word = sh->bins.codes[w];
#pragma unroll 1
            for (uint64_t bits = (fits ? word : word >> 4) & kListed; bits; bits &= bits - 1) {
                const uint32_t token = token_of(begin, w, bits);
                if (fits)
                    sh->index[at++] = token;
                if (word >> 4 & bits & -bits) {
                    if (pick < kList)
                        sh->pick[pick] = token;
                    ++pick;
                }
            }
        }
    }
    __syncthreads();  // the lists are there
    return {listed, picked,
            MOST ? extremes_of(wave_largest<true>(sh->floats[lane % kWaves])) : 0.0f};
}

// How many equal tokens of weight `each` fit above `above` short of `goal`: those
// whose predecessors' weight is below it.
__device__ __forceinline__ uint32_t ties_within(double goal, double above, double each)
{
    const double fit = __builtin_ceil((goal - above) / each);
    return fit < 1.0 ? 1 : fit < 1e9 ? uint32_t(fit) : 1000000000u;
}

// Where `goal` (or a share of all) is reached among the n tokens of `list` that
// `first` keeps: the smallest value with less than it (counts, or weights) above,
// `over` among that, and the index of the last equal token whose predecessors stay
// below it.  Bins are (steps below `from` - offset) * zoom, the zoom being 1, that of one
// such step's bins, or for counts kWider; their tokens are few (unless they are equal): one wave tries the values of up to 64 at once, or
// halves the range of more.  `again`: the list is that of the call before.
typedef const __attribute__((address_space(3))) uint32_t *LdsList;
__device__ __attribute__((noinline)) Cut list_cut(Lds *sh, LdsList list, uint32_t n, bool counts,
                                                  double goal, double share, double over,
                                                  Cut first, double from, double offset,
                                                  double zoom, bool again)
{
    const Row row = row_of(sh);
    const Units units(n);
    const uint32_t lane = threadIdx.x & 63;
    const Bins kind = !counts && zoom == 1.0 ? Bins::steps : Bins::plain;
    const auto grade = [&](uint32_t b) { return grade_of(zoom == 1.0 ? b : uint32_t(offset)); };
    const auto bin = [&](float v) {
        const double x = (-steps_of(row, v, from) - offset) * zoom;
        return x < 0.0 ? 0u : x < double(kBins - 1) ? uint32_t(x) : kBins - 1;
    };
    clear_bins(sh, kind);
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < n; i += kBlock) {
        float v;
        if (again)
            v = sh->value[i];
        else
            sh->value[i] = v = row.logits[list[i]];
        const double w = counts ? 1.0 : weight_of(sh, row, v);
        sh->weight[i] = w;
        if (first.keeps(v, list[i])) {
            const uint32_t b = bin(v);
            add_to_bin(sh, b, counts ? 1ull : units.of(__builtin_ldexp(w, -grade(b))));
        }
    }
    __syncthreads();
    const double unit = kind == Bins::steps ? units.scale
                                            : __builtin_ldexp(units.scale, grade(0));
    const Found found = find_bin(sh, goal, share, over, counts ? 1.0 : unit, kind);
    // The bin's tokens in their order: a thread looks at neighbours.
    const auto in = [&](uint32_t i) {
        return i < n && first.keeps(sh->value[i], list[i]) && bin(sh->value[i]) == found.bin;
    };
    static_assert(kList == 2 * kBlock, "neighbours of a thread");
    const bool a = in(2 * threadIdx.x), b = in(2 * threadIdx.x + 1);
    const uint64_t some_a = __ballot(a), some_b = __ballot(b), below = (1ull << lane) - 1;
    if (lane == 0)
        sh->flags[threadIdx.x >> 6] = __popcll(some_a) + __popcll(some_b);
    __syncthreads();
    const uint32_t in_wave = sh->flags[lane % kWaves], waves = lanes_scan<16>(in_wave);
    uint32_t at = __popcll(some_a & below) + __popcll(some_b & below);
    at += lane_value(waves - in_wave, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    if (a)
        sh->sub[at] = 2 * threadIdx.x;
    if (b)
        sh->sub[at + a] = 2 * threadIdx.x + 1;
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t m = lane_value(waves, kWaves - 1);
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
            const uint32_t high =
                wave_least(lane < m && above < found.goal ? key_of(value) : UINT32_MAX);
            uint64_t equal = __ballot(lane < m && key_of(value) == high);
            const int one = __builtin_ctzll(equal);
            const uint32_t count = __popcll(equal);
            uint32_t ties = ties_within(found.goal, lane_value(above, one), lane_value(weight, one));
            for (ties = ties < count ? ties : count; ties > 1; --ties)
                equal &= equal - 1;
            if (lane == uint32_t(__builtin_ctzll(equal))) {
                sh->floats[0] = value;
                sh->flags[0] = list[t];
            }
        } else {
            const auto above_of = [&](uint32_t key) {
                double above = 0.0;
                for (uint32_t i = lane; i < m; i += 64) {
                    const uint32_t t = sh->sub[i];
                    if (key_of(sh->value[t]) > key)
                        above += sh->weight[t];
                }
                return found.over + wave_total(above);
            };
            uint32_t least = UINT32_MAX, most = 0;
            for (uint32_t i = lane; i < m; i += 64) {
                const uint32_t k = key_of(sh->value[sh->sub[i]]);
                least = k < least ? k : least;
                most = k > most ? k : most;
            }
            uint32_t low = wave_least(least) - 1, high = ~wave_least(~most);
#pragma unroll 1
            while (high - low > 1) {
                const uint32_t middle = low + (high - low) / 2;
                if (above_of(middle) < found.goal)
                    high = middle;
                else
                    low = middle;
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
                    index = list[sh->sub[base + __builtin_ctzll(equal)]];
                    break;
                }
                ties -= here;
                index = list[sh->sub[base + 63 - __builtin_clzll(equal)]];
            }
            if (lane == 0) {
                sh->floats[0] = value;
                sh->flags[0] = index;
            }
        }
    }
    __syncthreads();
    const Cut cut = {sh->floats[0], sh->flags[0]};
    __syncthreads();
    return cut;
}

// The same over the row's tokens in `range`, 11 bits of the values' keys at a time: for
// rows with too many tokens about the cut to list.  `grade` is that of the range's
// weights, or kAnyGrade where they are of any size.
constexpr int kAnyGrade = 1;
__device__ __attribute__((noinline)) Cut digit_cut(Lds *sh, bool counts, double goal, double share,
                                                   double over, Cut first, Edges range, int grade)
{
    const Row row = row_of(sh);
    const Units units(row.width);
    const Bins kind = !counts && grade == kAnyGrade ? Bins::two : Bins::plain;
    const double unit = counts               ? 1.0
                        : kind == Bins::two ? units.scale
                                            : __builtin_ldexp(units.scale, grade);
    const double finer = 1.0 / unit;
    uint32_t prefix = 0;  // the digits found, in place
    constexpr uint32_t kDigit = kBins - 1;
#pragma unroll 1
    for (int low = 21; low >= -1; low -= 11) {
        // Digits of bits 31 .. 21, 20 .. 10 and 9 .. 0.
        const uint32_t shift = low > 0 ? low : 0, above = low > 0 ? low + 11 : 10;
        const uint32_t digit = (1u << (above - shift)) - 1;
        clear_bins(sh, kind);
        each_next(row, 0, row.chunks, [&](uint32_t c, v4f v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t key = key_of(v[e]);
                if (v[e] > -__builtin_inff() && v[e] >= range.low && v[e] < range.high &&
                    (above > 31 || key >> above == prefix >> above) &&
                    first.keeps(v[e], c * kChunk + 4 * threadIdx.x + e)) {
                    const uint32_t b = kDigit - (key >> shift & digit);
                    if (counts) {
                        add_to_bin(sh, b, 1);
                        continue;
                    }
                    const double w = weight_of(sh, row, v[e]);
                    if (kind == Bins::plain) {
                        add_to_bin(sh, b, units.of(__builtin_ldexp(w, -grade)));
                        continue;
                    }
                    const double high = __builtin_floor(w * finer);
                    add_to_bin(sh, b, uint64_t(high));
                    add_to_slot(sh, int(2 * kBins - 1 - b), uint64_t((w * finer - high) * finer));
                }
            }
        });
        __syncthreads();
        const Found found = find_bin(sh, goal, share, over, unit, kind);
        goal = found.goal;
        over = found.over;
        share = -1.0;
        prefix |= (kDigit - found.bin) << shift;
    }
    const float value = value_of(prefix);
    uint32_t ties = ties_within(goal, over, counts ? 1.0 : weight_of(sh, row, value));
    // The index of the last of that many equal tokens, by their codes.
    uint32_t last = 0;
#pragma unroll 1
    for (uint32_t begin = 0; begin < row.chunks; begin += kSegmentChunks) {
        const uint32_t end =
            row.chunks - begin < kSegmentChunks ? row.chunks : begin + kSegmentChunks;
        __syncthreads();
        // [value, value] as a range: up to the next value above.
        code_chunks(sh, row, begin, end, value, value_of(key_of(value) + 1), [](v4f) {});
        __syncthreads();
        const Words words(end - begin);
        uint64_t mine = 0;
        for (uint32_t w = words.first; w < words.last; ++w)
            mine += __popcll(sh->bins.codes[w] >> 4 & kListed);
        const Scan<uint64_t> scan = block_scan(sh, mine);
        const uint64_t wanted = ties < scan.total ? ties : scan.total;  // the last one here, else
        if (scan.total && scan.upto >= wanted && scan.upto - mine < wanted) {
            uint64_t left = wanted - (scan.upto - mine);
            for (uint32_t w = words.first; w < words.last && left; ++w)
                for (uint64_t bits = sh->bins.codes[w] >> 4 & kListed; bits && left;
                     bits &= bits - 1, --left)
                    sh->found = token_of(begin, w, bits);
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

// The weights of four tokens that a cut (not of -infinity) and min_p leave, formed
// side by side; `tied(e)`: whether token e is kept where its value is the cut's.
template <typename F>
__device__ __forceinline__ void terms_of(Lds *sh, const Row &row, v4f v, Cut cut, double min_p,
                                         double (&w)[4], F tied)
{
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = weight_of(sh, row, v[e]);
    asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3]));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const bool kept = (v[e] > cut.value) | ((v[e] == cut.value) & tied(e));
        w[e] = kept & (w[e] >= min_p) ? w[e] : 0.0;
    }
}

// The first kept token, in the vocabulary's order, at which the sum of kept weights
// passes u * total (the last kept one where rounding leaves none): of all tokens,
// or of `listed` in sh->index.  Each wave sums a run of tiles of 256, a lane four
// neighbours of each; the run that holds the target is shared out again, until it
// is one tile a wave.
__device__ __attribute__((noinline)) void choose(Lds *sh, uint32_t listed, Cut cut, double min_p,
                                                 double u, float *out, float *copy)
{
    const Row row = row_of(sh);
    listed = __builtin_amdgcn_readfirstlane(listed);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t begin = 0, tiles = ((listed ? listed : row.width) + 255) / 256;
    double passed = 0.0, target = -1.0;
#pragma unroll 1
    for (;;) {
        const uint32_t each_has = (tiles + kWaves - 1) / kWaves;
        const uint32_t first = wave * each_has < tiles ? wave * each_has : tiles;
        const uint32_t last = first + each_has < tiles ? first + each_has : tiles;
        double w[4] = {0.0, 0.0, 0.0, 0.0}, own = 0.0;
        if (listed) {
#pragma unroll 1
            for (uint32_t t = begin + first; t < begin + last; ++t) {
                const uint32_t at = t * 256 + 4 * lane;
                uint32_t i[4];
                v4f v;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    i[e] = sh->index[at + e < listed ? at + e : listed - 1];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = row.logits[i[e]];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = at + e < listed ? v[e] : -__builtin_inff();
                terms_of(sh, row, v, cut, min_p, w, [&](int e) { return i[e] <= cut.index; });
                own += (w[0] + w[1]) + (w[2] + w[3]);
            }
        } else if (first < last) {
            // The next tile's loads are in flight behind this one's weights.
            const auto load = [&](uint32_t t) {
                return load_four(row, t * 256 + 4 * lane, (t + 1) * 256 <= row.width);
            };
            v4f next = load(begin + first);
#pragma unroll 1
            for (uint32_t t = begin + first; t < begin + last; ++t) {
                const v4f v = next;
                if (t + 1 < begin + last)
                    next = load(t + 1);
                const int room = int(cut.index < 0x7fffffffu ? cut.index : 0x7fffffffu) -
                                 int(t * 256);
                terms_of(sh, row, v, cut, min_p, w,
                         [&](int e) { return int(4 * lane) + e <= room; });
                own += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }
        const double upto = wave_scan(own);
        __syncthreads();
        if (lane == 63)
            sh->scratch[wave] = __builtin_bit_cast(uint64_t, upto);
        __syncthreads();
        const double run = lane < kWaves ? __builtin_bit_cast(double, sh->scratch[lane]) : 0.0;
        const double runs = wave_scan(run);
        if (target < 0.0)
            target = u * lane_value(runs, kWaves - 1);
        const uint32_t chosen =
            __builtin_amdgcn_readfirstlane(holder(run > 0.0, passed + runs > target));
        if (chosen)
            passed += lane_value(runs, int(chosen) - 1);
        if (each_has > 1) {
            begin += chosen * each_has;
            tiles = tiles - chosen * each_has < each_has ? tiles - chosen * each_has : each_has;
            continue;
        }
        if (wave == chosen && lane == holder(own > 0.0, passed + upto > target)) {
            double at = passed + (upto - own);
            uint32_t token = 0;
            bool done = false;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (w[e] > 0.0 && !done) {
                    at += w[e];
                    token = (begin + first) * 256 + 4 * lane + e;
                    done = at > target;
                }
            if (listed)
                token = sh->index[token];
            *out = float(token);
            if (copy)
                *copy = float(token);
        }
        return;
    }
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
        first = wave_least(first);
        if (lane == 0)
            sh->flags[wave] = first;
        __syncthreads();
        first = wave_least<true>(sh->flags[threadIdx.x % kWaves]);
        if (threadIdx.x == 0)
            answer(most > -__builtin_inff() ? float(first) : __builtin_nanf(""));
        return;
    }
    __syncthreads();

    const uint32_t k = top_k > 0.0f && top_k < float(s.width) ? uint32_t(top_k) : 0;
    const double share = top_p < 1.0f ? double(top_p) : -1.0;
    Cut cut = {-3.4028235e38f, UINT32_MAX};
    uint32_t listed = 0;  // tokens of the list, where it holds every kept one
    Listed list = {0, 0, 0.0f};
    float floor = -__builtin_inff();
    if (k) {
        // A value that the k-th largest of the row does not lie below: of the
        // first tokens, enough for about 1024 listed ones.
        if (s.width > kList) {
            uint32_t chunks = uint32_t((uint64_t(row.chunks) * k + 1023) / 1024);
            chunks = chunks < row.chunks ? chunks : row.chunks;
            const float from = row_extremes(sh, chunks);
            if (from > -__builtin_inff()) {
                // Where fewer than k lie in the bins (a low temperature, few tokens
                // admitted) bins 64 times as wide are tried, then all tokens are
                // listed: k are kept however little they weigh.
                bool reached = false;
#pragma unroll 1
                for (int wider = 0; wider < 2 && !reached; ++wider) {
                    if (wider) {
                        if (threadIdx.x == 0)
                            sh->row.per_step = row.per_step * kWider;
                        __syncthreads();
                    }
                    histogram(sh, chunks, double(from), true);
                    const Found found = find_bin(sh, double(k), -1.0, 0.0, 1.0, Bins::plain);
                    reached = found.reached;
                    if (reached)
                        floor = edges_of(sh, found.bin, double(from)).low;
                    if (wider) {
                        if (threadIdx.x == 0)
                            sh->row.per_step = row.per_step;
                        __syncthreads();
                    }
                }
            }
        }
        list = list_tokens<true>(sh, floor, __builtin_inff());
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
        if (listed > k) {
            // The bins reach down to the list's floor, or nearly all of it would lie in
            // the last one (T = 0.05, one row of 65536: 76 us, with this 24).
            const bool near = !(floor > -__builtin_inff()) ||
                              (from - double(floor)) * row.per_step < double(kBins);
            cut = list_cut(sh, &sh->index[0], listed, true, double(k), -1.0, 0.0, cut, from, 0.0,
                           near ? 1.0 : kWider, false);
        }
        if (share >= 0.0)
            cut = list_cut(sh, &sh->index[0], listed, false, 0.0, share, 0.0, cut, from, 0.0, 1.0,
                           listed > k);
    } else if (k) {
        const Edges all = {-__builtin_inff(), __builtin_inff()};
        cut = digit_cut(sh, true, double(k), -1.0, 0.0, cut, all, kAnyGrade);
        if (share >= 0.0)
            cut = digit_cut(sh, false, 0.0, share, 0.0, cut, all, kAnyGrade);
    } else if (share >= 0.0) {
        histogram(sh, row.chunks, from, false);
        const Found found = find_bin(sh, 0.0, share, 0.0, Units(s.width).scale, Bins::steps);
        const Edges edges = edges_of(sh, found.bin, from);
        list = list_tokens<false>(sh, edges.low, edges.high);
        // Within the bin: its own equal steps.
        cut = list.picked <= kList
                  ? list_cut(sh, &sh->pick[0], list.picked, false, found.goal, -1.0, found.over,
                             cut, from, double(found.bin), double(kBins), false)
                  : digit_cut(sh, false, found.goal, -1.0, found.over, cut, edges,
                              grade_of(found.bin));
        listed = list.count <= kMany ? list.count : 0;
    }
    if (min_p > 0.0f) {
        // A value whose weight is surely below min_p: a bound, with room for
        // its own rounding; the weights themselves decide.
        const float bound =
            list.most + temperature * (logf(min_p) - 0.01f) - 1e-5f * fabsf(list.most);
        if (bound > cut.value)
            cut = {bound, UINT32_MAX};
    }
    // A list of what a cut has left, where there is none yet.
    if (!listed && ((k && list.count > kList) || (!k && share < 0.0 && min_p > 0.0f))) {
        const uint32_t n = list_tokens<false>(sh, cut.value, __builtin_inff()).count;
        listed = n <= kMany ? n : 0;
    }
    choose(sh, listed, cut, double(min_p), double(u), s.out + r, s.copy ? s.copy + r : nullptr);
}

}  // namespace

void launch_sample_rows(hipStream_t stream, const Sampling &s)
{
    if (s.rows)
        sample_kernel<<<s.rows, kBlock, 0, stream>>>(s);
}

}  // namespace mfh
