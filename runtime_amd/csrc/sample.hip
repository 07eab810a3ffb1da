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
// equal ones up to the index).  The cut's bin among kBins equal steps of (m - l)
// / temperature is found from a histogram of counts (top-k) or weights (top-p;
// whole numbers of 2^-46 or so, so that the order of additions does not matter),
// its tokens are listed in LDS in their order, and one wave finds the cut by
// halving the range of their values.  With top-k all tokens down to the cut are
// listed and the whole choice is the wave's; else the chosen token is found from
// the sums of 256 tokens each.  Rows whose bin holds more than the list (many
// equal values, or a temperature far above the logits' spread) search the whole
// row by halving.
//
#include "kernels.hpp"
#include "paged.hpp"

namespace mfh {
namespace {

constexpr int kBlock = 1024;
constexpr int kWaves = kBlock / 64;
constexpr uint32_t kChunk = 4 * kBlock;   // tokens of one float4 a thread
constexpr uint32_t kSegmentChunks = 64;   // chunks whose sums LDS holds
constexpr uint32_t kBins = 4096, kList = 2048;
// Beyond this a weight is below 2^24 times less than 2^-45 of the largest.
constexpr float kRange = 48.0f;

typedef float v4f __attribute__((ext_vector_type(4)));

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

// Inclusive scan over the block and its total.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *scratch, T *total)
{
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63)
        scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (w == threadIdx.x >> 6)
            before = all;
        all += scratch[w];
    }
    *total = all;
    return v + before;
}

// A row's values and settings, and the passes over it.
struct Row {
    const float *logits;
    const uint8_t *mask;
    uint32_t width, chunks;
    bool aligned;
    float largest;
    double largest64, inverse;  // of the temperature
    const double *table;        // 2^(j / 32)

    __device__ float value(uint32_t i) const { return logits[i]; }  // of an admitted token
    __device__ __forceinline__ v4f load(uint32_t c) const
    {
        const uint32_t i = c * kChunk + 4 * threadIdx.x;
        constexpr float kNone = -__builtin_inff();
        v4f v = {kNone, kNone, kNone, kNone};
        if (aligned && i + 3 < width) {
            v = *reinterpret_cast<const v4f *>(logits + i);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < width)
                    v[e] = logits[i + e];
        }
        if (mask && i < width) {
            const uint32_t bits = mask[i >> 3] >> (i & 7);  // i is a multiple of 4
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!(bits >> e & 1))
                    v[e] = kNone;
        }
        return v;
    }
    // f(chunk, values) over chunks [begin, end), kAhead chunks' loads in flight.
    template <typename F>
    __device__ __forceinline__ void each(uint32_t begin, uint32_t end, F f) const
    {
        constexpr uint32_t kAhead = 4;
        for (uint32_t c = begin; c < end; c += kAhead) {
            v4f v[kAhead];
#pragma unroll
            for (uint32_t a = 0; a < kAhead; ++a)
                if (c + a < end)
                    v[a] = load(c + a);
#pragma unroll
            for (uint32_t a = 0; a < kAhead; ++a)
                if (c + a < end)
                    f(c + a, v[a]);
        }
    }
    // exp((v - largest) / temperature) to 2^-52: 2^(n / 32) e^r with |r| <= ln 2 / 64.
    __device__ __forceinline__ double weight(float v) const
    {
        const double x = (double(v) - largest64) * inverse;
        if (!(x > -740.0))
            return 0.0;
        const double n = __builtin_rint(x * 46.166241308446828384);
        double r = __builtin_fma(n, -0x1.62e42fefa0000p-6, x);
        r = __builtin_fma(n, -0x1.cf79abc9e3b3ap-45, r);
        double e = __builtin_fma(r, 1.0 / 720, 1.0 / 120);
        e = __builtin_fma(e, r, 1.0 / 24);
        e = __builtin_fma(e, r, 1.0 / 6);
        e = __builtin_fma(e, r, 0.5);
        e = __builtin_fma(e, r, 1.0);
        e = __builtin_fma(e, r, 1.0);
        const int whole = int(n);
        return __builtin_ldexp(table[whole & 31] * e, whole >> 5);
    }
};

struct Shared {
    double table[32];
    union {
        uint64_t weight[kBins];
        uint32_t count[kBins];
        uint64_t votes[kSegmentChunks * kWaves * 4];
    } bins;
    float value[kList];
    uint32_t index[kList];
    double weight[kList];
    double group[kSegmentChunks * kWaves];
    double segment[(1u << 24) / (kSegmentChunks * kChunk)];
    double doubles[kWaves];
    uint64_t wholes[kWaves];
    float floats[kWaves];
    uint32_t flags[kWaves];
    uint32_t found, below, listed;
    uint64_t before;
};

// The kept tokens: values above `value`, and equal ones up to `index`.
struct Cut {
    float value;
    uint32_t index;
    __device__ bool keeps(float v, uint32_t i) const
    {
        return v > value || (v == value && i <= index);
    }
};

// Lists the tokens for which keep(value) in their order; returns how many there
// are (the list is valid where they fit).  The waves' votes of a segment go to
// LDS; a thread then lists the tokens of one group of 256.
template <typename F>
__device__ uint32_t list_tokens(const Row &row, Shared &sh, F keep)
{
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t listed = 0;
    for (uint32_t begin = 0; begin < row.chunks; begin += kSegmentChunks) {
        const uint32_t end =
            row.chunks - begin < kSegmentChunks ? row.chunks : begin + kSegmentChunks;
        __syncthreads();
        row.each(begin, end, [&](uint32_t c, v4f v) {
            uint64_t votes[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                votes[e] = __ballot(keep(v[e]));
            if (lane < 4)
                sh.bins.votes[((c - begin) * kWaves + wave) * 4 + lane] =
                    lane & 2 ? (lane & 1 ? votes[3] : votes[2]) : (lane & 1 ? votes[1] : votes[0]);
        });
        __syncthreads();
        uint64_t votes[4] = {0, 0, 0, 0};
        if (threadIdx.x < (end - begin) * kWaves)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                votes[e] = sh.bins.votes[threadIdx.x * 4 + e];
        const uint64_t mine = __popcll(votes[0]) + __popcll(votes[1]) + __popcll(votes[2]) +
                              __popcll(votes[3]);
        uint64_t total = 0;
        uint32_t at = listed + uint32_t(block_scan(mine, sh.wholes, &total) - mine);
        if (listed + total <= kList) {
            uint64_t lanes = votes[0] | votes[1] | votes[2] | votes[3];
            const uint32_t first = (begin + threadIdx.x / kWaves) * kChunk +
                                   threadIdx.x % kWaves * 256;
            for (; lanes; lanes &= lanes - 1) {
                const uint32_t l = __builtin_ctzll(lanes);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (votes[e] >> l & 1)
                        sh.index[at++] = first + 4 * l + e;
            }
        }
        listed = listed + total < kList + 1 ? uint32_t(listed + total) : kList + 1;
    }
    __syncthreads();
    if (listed <= kList)
        for (uint32_t i = threadIdx.x; i < listed; i += kBlock) {
            sh.value[i] = row.value(sh.index[i]);
            sh.weight[i] = row.weight(sh.value[i]);
        }
    __syncthreads();
    return listed;
}

// One wave over the list.  The smallest key for which ok(key, sum of
// measure(i) over listed keys above it) holds, between the list's keys; ok has to
// hold for the largest.
template <typename M, typename F>
__device__ uint32_t list_cut(const Shared &sh, uint32_t n, M measure, F ok)
{
    const uint32_t lane = threadIdx.x & 63;
    uint32_t least = UINT32_MAX, most = 0;
    for (uint32_t i = lane; i < n; i += 64) {
        const uint32_t k = key_of(sh.value[i]);
        least = k < least ? k : least;
        most = k > most ? k : most;
    }
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1) {
        const uint32_t a = __shfl_xor(least, offset, 64), b = __shfl_xor(most, offset, 64);
        least = a < least ? a : least;
        most = b > most ? b : most;
    }
    uint32_t low = __builtin_amdgcn_readfirstlane(least) - 1;
    uint32_t high = __builtin_amdgcn_readfirstlane(most);
    while (high - low > 1) {
        const uint32_t middle = low + (high - low) / 2;
        double above = 0.0;
        for (uint32_t i = lane; i < n; i += 64)
            if (key_of(sh.value[i]) > middle)
                above += measure(i);
        if (ok(wave_total(above)))
            high = middle;
        else
            low = middle;
    }
    return high;
}

// The index of the count-th listed token (from 1) with this value, or of the last.
__device__ uint32_t list_tie(const Shared &sh, uint32_t n, float value, uint32_t count)
{
    const uint32_t lane = threadIdx.x & 63;
    uint32_t last = 0;
    for (uint32_t base = 0; base < n; base += 64) {
        const uint32_t i = base + lane;
        uint64_t equal = __ballot(i < n && sh.value[i < n ? i : 0] == value);
        if (!equal)
            continue;
        const uint32_t here = __popcll(equal);
        if (here >= count) {
            for (uint32_t skip = 1; skip < count; ++skip)
                equal &= equal - 1;
            return sh.index[base + __builtin_ctzll(equal)];
        }
        count -= here;
        last = sh.index[base + 63 - __builtin_clzll(equal)];
    }
    return last;
}

// How many equal tokens of weight `each` fit above `above` short of `wanted`: those
// whose predecessors' weight is below it.
__device__ __forceinline__ uint32_t ties_within(double wanted, double above, double each)
{
    const double fit = __builtin_ceil((wanted - above) / each);
    return fit < 1.0 ? 1 : fit < 1e9 ? uint32_t(fit) : 1000000000u;
}

// ---- the whole row by halving: rows whose bin passes the list -------------------

template <typename F>
__device__ double row_sum(const Row &row, Shared &sh, F f)
{
    double sum = 0.0;
    row.each(0, row.chunks, [&](uint32_t c, v4f v) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            sum += f(v[e], c * kChunk + 4 * threadIdx.x + e);
    });
    double total = 0.0;
    (void)block_scan(sum, sh.doubles, &total);
    return total;
}

// The index up to which `count` tokens have this value.
__device__ uint32_t row_tie(const Row &row, Shared &sh, float value, uint32_t count)
{
    uint32_t low = 0, high = row.width - 1;
    while (low < high) {
        const uint32_t middle = low + (high - low) / 2;
        const double n = row_sum(
            row, sh, [&](float v, uint32_t i) { return v == value && i <= middle ? 1.0 : 0.0; });
        if (n >= double(count))
            high = middle;
        else
            low = middle + 1;
    }
    return low;
}

__device__ Cut row_cut(const Row &row, Shared &sh, uint32_t top_k, double top_p)
{
    Cut cut = {-__builtin_inff(), UINT32_MAX};
    const uint32_t top = key_of(row.largest);
    if (top_k) {
        // The smallest key with fewer than top_k tokens above it (keys below
        // -infinity's are NaN's).
        uint32_t low = key_of(-__builtin_inff()), high = top;
        while (low < high) {
            const uint32_t middle = low + (high - low) / 2;
            const float value = value_of(middle);
            const double n =
                row_sum(row, sh, [&](float v, uint32_t) { return v > value ? 1.0 : 0.0; });
            if (n < double(top_k))
                high = middle;
            else
                low = middle + 1;
        }
        cut.value = value_of(low);
        const double above =
            row_sum(row, sh, [&](float v, uint32_t) { return v > cut.value ? 1.0 : 0.0; });
        cut.index = row_tie(row, sh, cut.value, uint32_t(double(top_k) - above));
    }
    if (top_p < 1.0) {
        const auto weight_above = [&](float value) {
            return row_sum(row, sh, [&](float v, uint32_t i) {
                return v > value && cut.keeps(v, i) ? row.weight(v) : 0.0;
            });
        };
        const double all = row_sum(
            row, sh, [&](float v, uint32_t i) { return cut.keeps(v, i) ? row.weight(v) : 0.0; });
        const double wanted = top_p > 0.0 ? top_p * all : 0x1p-60;
        // The smallest key with less than the wanted weight above it.
        uint32_t low = key_of(cut.value), high = top;
        while (low < high) {
            const uint32_t middle = low + (high - low) / 2;
            if (weight_above(value_of(middle)) < wanted)
                high = middle;
            else
                low = middle + 1;
        }
        const float value = value_of(low);
        const uint32_t ties = ties_within(wanted, weight_above(value), row.weight(value));
        const uint32_t index = row_tie(row, sh, value, ties);
        if (value > cut.value || (value == cut.value && index < cut.index))
            cut = {value, index};
    }
    return cut;
}

// ---- the kernel -------------------------------------------------------------------

__global__ __launch_bounds__(kBlock) void sample_kernel(Sampling s)
{
    __shared__ Shared sh;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t r = blockIdx.x;
    Row row;
    row.width = s.width;
    row.chunks = (s.width + kChunk - 1) / kChunk;
    row.aligned = s.width % 4 == 0;
    row.logits = s.logits + uint64_t(r) * s.width;
    row.mask = s.mask ? s.mask + (s.one_mask ? 0 : uint64_t(r) * ((s.width + 7) / 8)) : nullptr;
    row.table = sh.table;
    const float *params = s.params + (s.one_params ? 0 : 4 * uint64_t(r));
    const float u = s.uniforms[r];
    const float temperature = params[0], top_k = params[1], top_p = params[2], min_p = params[3];
    if (threadIdx.x < 32)
        sh.table[threadIdx.x] = exp2(double(threadIdx.x) / 32.0);
    const auto answer = [&](float token) {
        s.out[r] = token;
        if (s.copy)
            s.copy[r] = token;
    };

    // The largest value, and whether any is NaN or +infinity.
    float most = -__builtin_inff();
    bool poison = false;
    row.each(0, row.chunks, [&](uint32_t, v4f v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            poison = poison || !(v[e] < __builtin_inff());
            most = fmaxf(most, v[e]);
        }
    });
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1)
        most = fmaxf(most, __shfl_xor(most, offset, 64));
    const bool bad = __any(poison);
    if (lane == 0) {
        sh.floats[wave] = most;
        sh.flags[wave] = bad;
    }
    __syncthreads();
    uint32_t bads = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        most = fmaxf(most, sh.floats[w]);
        bads |= sh.flags[w];
    }
    const bool good = temperature >= 0.0f && temperature < __builtin_inff() && top_k >= 0.0f &&
                      truncf(top_k) == top_k && top_p >= 0.0f && top_p <= 1.0f && min_p >= 0.0f &&
                      min_p <= 1.0f && u >= 0.0f && u < 1.0f;
    if (bads || !good || most == -__builtin_inff()) {
        if (threadIdx.x == 0)
            answer(__builtin_nanf(""));
        return;
    }
    row.largest = most;
    row.largest64 = double(most);
    row.inverse = 1.0 / double(temperature);

    if (temperature == 0.0f) {
        uint32_t first = UINT32_MAX;
        row.each(0, row.chunks, [&](uint32_t c, v4f v) {
#pragma unroll
            for (int e = 3; e >= 0; --e) {
                const uint32_t i = c * kChunk + 4 * threadIdx.x + e;
                if (v[e] == most && i < first)
                    first = i;
            }
        });
#pragma unroll
        for (int offset = 32; offset > 0; offset >>= 1) {
            const uint32_t other = __shfl_xor(first, offset, 64);
            first = other < first ? other : first;
        }
        __syncthreads();
        if (lane == 0)
            sh.flags[wave] = first;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kWaves; ++w)
                first = sh.flags[w] < first ? sh.flags[w] : first;
            answer(float(first));
        }
        return;
    }

    const uint32_t k = top_k > 0.0f && top_k < float(s.width) ? uint32_t(top_k) : 0;
    Cut cut = {-__builtin_inff(), UINT32_MAX};
    if (k || top_p < 1.0f) {
        // Equal steps of (largest - v) / temperature; both halved, so that the
        // difference of finite values is finite.  Monotone in v.
        const float steps = fminf(2.0f * float(kBins) / kRange / temperature, 1e30f);
        const float half = 0.5f * most;
        const auto bin_of = [&](float v) {
            const float x = (half - 0.5f * v) * steps;
            return x < float(kBins) ? uint32_t(x) : kBins;
        };
        // Whole numbers of 2^-unit: their sum over the row stays below 2^63.
        const int unit = 46 < 62 - (32 - __builtin_clz(s.width)) ? 46
                                                                : 62 - (32 - __builtin_clz(s.width));
        const double shift = __builtin_ldexp(1.0, 52 - unit);
        const uint64_t shift_bits = __builtin_bit_cast(uint64_t, shift);
        for (uint32_t i = threadIdx.x; i < kBins; i += kBlock)
            sh.bins.weight[i] = 0;
        __syncthreads();
        if (k)
            row.each(0, row.chunks, [&](uint32_t, v4f v) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t b = bin_of(v[e]);
                    if (b < kBins)
                        atomicAdd(&sh.bins.count[b], 1u);
                }
            });
        else
            row.each(0, row.chunks, [&](uint32_t, v4f v) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t b = bin_of(v[e]);
                    if (b < kBins)
                        atomicAdd(reinterpret_cast<unsigned long long *>(&sh.bins.weight[b]),
                                  __builtin_bit_cast(uint64_t, row.weight(v[e]) + shift) -
                                      shift_bits);
                }
            });
        if (threadIdx.x == 0)
            sh.found = kBins;
        __syncthreads();
        // The first bin with which the count, or the weight, is reached.
        constexpr uint32_t kEach = kBins / kBlock;
        uint64_t own[kEach], mine = 0, total = 0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            own[i] = k ? sh.bins.count[threadIdx.x * kEach + i]
                       : sh.bins.weight[threadIdx.x * kEach + i];
            mine += own[i];
        }
        uint64_t upto = block_scan(mine, sh.wholes, &total) - mine;
        const double all = double(total);
        const double wanted = k ? double(k) : top_p > 0.0f ? double(top_p) * all : 0.5;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            if (double(upto) < wanted && double(upto + own[i]) >= wanted) {
                sh.found = threadIdx.x * kEach + i;
                sh.before = upto;
            }
            upto += own[i];
        }
        __syncthreads();
        const uint32_t found = sh.found;
        const uint64_t before = sh.before;
        // With top-k all tokens down to the bin (down to the range's end where
        // there are fewer), else the bin's.
        const uint32_t n = list_tokens(row, sh, [&](float v) {
            const uint32_t b = bin_of(v);
            return k ? b <= found && b < kBins : b == found && b < kBins;
        });
        if (n <= kList && (k || found < kBins)) {
            if (wave == 0) {
                const auto weight = [&](uint32_t i) { return sh.weight[i]; };
                if (k) {
                    if (n > k) {
                        const uint32_t key = list_cut(
                            sh, n, [](uint32_t) { return 1.0; },
                            [&](double above) { return above < double(k); });
                        cut.value = value_of(key);
                        uint32_t above = 0;
                        for (uint32_t i = lane; i < n; i += 64)
                            above += sh.value[i] > cut.value;
#pragma unroll
                        for (int offset = 32; offset > 0; offset >>= 1)
                            above += __shfl_xor(above, offset, 64);
                        cut.index = list_tie(sh, n, cut.value, k - above);
                    }
                    const Cut first = cut;
                    const auto kept = [&](uint32_t i) {
                        return first.keeps(sh.value[i], sh.index[i]) ? sh.weight[i] : 0.0;
                    };
                    if (top_p < 1.0f) {
                        double sum = 0.0;
                        for (uint32_t i = lane; i < n; i += 64)
                            sum += kept(i);
                        sum = wave_total(sum);
                        const double goal = top_p > 0.0f ? double(top_p) * sum : 0x1p-60;
                        const uint32_t key =
                            list_cut(sh, n, kept, [&](double above) { return above < goal; });
                        const float value = value_of(key);
                        double above = 0.0;
                        for (uint32_t i = lane; i < n; i += 64)
                            above += sh.value[i] > value ? kept(i) : 0.0;
                        above = wave_total(above);
                        const uint32_t index = list_tie(
                            sh, n, value, ties_within(goal, above, row.weight(value)));
                        if (value > cut.value || (value == cut.value && index < cut.index))
                            cut = {value, index};
                    }
                    // The choice: sums in the list's order, 64 tokens at a time.
                    const auto term = [&](uint32_t i) {
                        const bool in = i < n && cut.keeps(sh.value[i], sh.index[i]) &&
                                        sh.weight[i] >= double(min_p);
                        return in ? sh.weight[i] : 0.0;
                    };
                    double sum = 0.0;
                    for (uint32_t base = 0; base < n; base += 64)
                        sum += wave_total(term(base + lane));
                    const double target = double(u) * sum;
                    double at = 0.0;
                    uint32_t token = 0;
                    for (uint32_t base = 0; base < n; base += 64) {
                        const double t = term(base + lane);
                        const double scan = wave_scan(t);
                        const uint64_t some = __ballot(t > 0.0);
                        if (some)
                            token = sh.index[base + 63 - __builtin_clzll(some)];
                        const uint64_t past = __ballot(t > 0.0 && at + scan > target);
                        if (past) {
                            token = sh.index[base + __builtin_ctzll(past)];
                            break;
                        }
                        at += lane_value(scan, 63);
                    }
                    if (lane == 0)
                        answer(float(token));
                } else {
                    const double scale = __builtin_ldexp(1.0, -unit);
                    const double goal = wanted * scale, over = double(before) * scale;
                    const uint32_t key = list_cut(
                        sh, n, weight, [&](double above) { return over + above < goal; });
                    const float value = value_of(key);
                    double above = 0.0;
                    for (uint32_t i = lane; i < n; i += 64)
                        above += sh.value[i] > value ? sh.weight[i] : 0.0;
                    above = over + wave_total(above);
                    const uint32_t index =
                        list_tie(sh, n, value, ties_within(goal, above, row.weight(value)));
                    if (lane == 0) {
                        sh.floats[0] = value;
                        sh.flags[0] = index;
                    }
                }
            }
            if (k)
                return;
            __syncthreads();
            cut = {sh.floats[0], sh.flags[0]};
        } else {
            cut = row_cut(row, sh, k, double(top_p));
        }
    }

    // The choice among the kept tokens: sums of 256 tokens (a wave's float4s), of
    // the segment that holds the target, then that wave's lanes.
    const auto term = [&](float v, uint32_t i) {
        if (!cut.keeps(v, i))
            return 0.0;
        const double w = row.weight(v);
        return w >= double(min_p) ? w : 0.0;
    };
    const auto lane_sum = [&](uint32_t c, v4f v) {
        const uint32_t i = c * kChunk + 4 * threadIdx.x;
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            sum += term(v[e], i + e);
        return sum;
    };
    const auto group_sums = [&](uint32_t begin, uint32_t end) {
        __syncthreads();
        row.each(begin, end, [&](uint32_t c, v4f v) {
            const bool any = __any(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= cut.value);
            const double sum = any ? wave_scan(lane_sum(c, v)) : 0.0;
            if (lane == 63)
                sh.group[(c - begin) * kWaves + wave] = sum;
        });
        __syncthreads();
    };
    const uint32_t segments = (row.chunks + kSegmentChunks - 1) / kSegmentChunks;
    double total = 0.0, mine = 0.0, upto = 0.0;
    for (uint32_t g = 0; g < segments; ++g) {
        const uint32_t begin = g * kSegmentChunks;
        const uint32_t end =
            row.chunks - begin < kSegmentChunks ? row.chunks : begin + kSegmentChunks;
        group_sums(begin, end);
        mine = threadIdx.x < (end - begin) * kWaves ? sh.group[threadIdx.x] : 0.0;
        double sum = 0.0;
        upto = block_scan(mine, sh.doubles, &sum);
        if (threadIdx.x == 0)
            sh.segment[g] = sum;
        total += sum;
    }
    const double target = double(u) * total;
    double passed = 0.0;
    uint32_t begin = 0;
    if (segments > 1) {
        // The first segment that passes the target (the last with a token where
        // rounding leaves none).
        __syncthreads();
        uint32_t chosen = 0;
        double at = 0.0;
        for (uint32_t g = 0; g < segments; ++g) {
            if (sh.segment[g] > 0.0) {
                chosen = g;
                passed = at;
            }
            at += sh.segment[g];
            if (sh.segment[g] > 0.0 && at > target)
                break;
        }
        begin = chosen * kSegmentChunks;
        const uint32_t end =
            row.chunks - begin < kSegmentChunks ? row.chunks : begin + kSegmentChunks;
        group_sums(begin, end);
        mine = threadIdx.x < (end - begin) * kWaves ? sh.group[threadIdx.x] : 0.0;
        double sum = 0.0;
        upto = block_scan(mine, sh.doubles, &sum);
    }
    // The first group that passes it, likewise.
    if (threadIdx.x == 0) {
        sh.found = UINT32_MAX;
        sh.below = 0;
    }
    __syncthreads();
    if (mine > 0.0) {
        if (passed + upto > target)
            atomicMin(&sh.found, threadIdx.x);
        atomicMax(&sh.below, threadIdx.x);
    }
    __syncthreads();
    const uint32_t group = sh.found != UINT32_MAX ? sh.found : sh.below;
    if (threadIdx.x == group)
        sh.doubles[0] = passed + (upto - mine);
    __syncthreads();
    if (wave != group % kWaves)
        return;
    const double start = sh.doubles[0];
    const uint32_t chunk = begin + group / kWaves;
    const v4f v = row.load(chunk);
    const double own = lane_sum(chunk, v);
    const double scan = wave_scan(own);
    const uint64_t some = __ballot(own > 0.0);
    const uint64_t past = __ballot(own > 0.0 && start + scan > target);
    if (!some)
        return;  // not reached: the group's sum is positive
    if (lane == (past ? uint32_t(__builtin_ctzll(past)) : 63 - uint32_t(__builtin_clzll(some)))) {
        const uint32_t i = chunk * kChunk + 4 * threadIdx.x;
        double at = start + (scan - own);
        uint32_t token = i;
        for (int e = 0; e < 4; ++e) {
            const double t = term(v[e], i + e);
            if (t > 0.0) {
                at += t;
                token = i + e;
                if (at > target)
                    break;
            }
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
