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
#include "kernels.hpp"
#include "paged.hpp"

namespace mfh {
namespace {

constexpr int kBlock = 1024;
constexpr int kWaves = kBlock / 64;

// An order-preserving whole number for a value; both zeros alike.
__device__ __forceinline__ uint32_t key_of(float v)
{
    const uint32_t bits = __float_as_uint(v + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T *scratch, F join)
{
#pragma unroll
    for (int offset = 32; offset > 0; offset >>= 1)
        v = join(v, __shfl_xor(v, offset, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
        v = join(v, scratch[w]);
    return v;
}

__global__ __launch_bounds__(kBlock) void sample_kernel(Sampling s)
{
    __shared__ double doubles[kWaves];
    __shared__ uint32_t counts[kWaves];
    __shared__ uint32_t chosen;
    const uint32_t row = blockIdx.x, width = s.width;
    const float *logits = s.logits + uint64_t(row) * width;
    const uint8_t *mask =
        s.mask ? s.mask + (s.one_mask ? 0 : uint64_t(row) * ((width + 7) / 8)) : nullptr;
    const float *params = s.params + (s.one_params ? 0 : 4 * uint64_t(row));
    const float u = s.uniforms[row];
    const float temperature = params[0], top_k = params[1], top_p = params[2], min_p = params[3];
    const auto sum = [](auto a, auto b) { return a + b; };
    const auto most = [](auto a, auto b) { return a > b ? a : b; };
    const auto value = [&](uint32_t i) {
        return !mask || (mask[i >> 3] >> (i & 7) & 1) ? logits[i] : -__builtin_inff();
    };
    const auto answer = [&](float token) {
        if (threadIdx.x == 0) {
            s.out[row] = token;
            if (s.copy)
                s.copy[row] = token;
        }
    };

    uint32_t key = 0, poison = 0;
    for (uint32_t i = threadIdx.x; i < width; i += kBlock) {
        const float v = value(i);
        poison |= !(v < __builtin_inff());
        key = most(key, key_of(v));
    }
    key = block_reduce(key, counts, most);
    poison = block_reduce(poison, counts, most);
    const bool good = temperature >= 0.0f && temperature < __builtin_inff() && top_k >= 0.0f &&
                      truncf(top_k) == top_k && top_p >= 0.0f && top_p <= 1.0f && min_p >= 0.0f &&
                      min_p <= 1.0f && u >= 0.0f && u < 1.0f;
    if (poison || !good || key == key_of(-__builtin_inff())) {
        answer(__builtin_nanf(""));
        return;
    }
    const uint32_t top = key;
    const double largest =
        double(__uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top));
    const double inverse = 1.0 / double(temperature);
    const auto weight = [&](float v) { return exp((double(v) - largest) * inverse); };

    // The kept tokens: keys above `cut`, and the first `ties` of those at it.
    uint32_t cut = 0, ties = width;
    // Tokens (or their weight) above a key.
    const auto count_above = [&](uint32_t k) {
        uint32_t n = 0;
        for (uint32_t i = threadIdx.x; i < width; i += kBlock)
            n += key_of(value(i)) > k;
        return block_reduce(n, counts, sum);
    };
    if (temperature == 0.0f) {
        cut = top;
        ties = 1;
    } else {
        if (top_k > 0.0f && top_k < float(width)) {
            // The smallest key with fewer than top_k tokens above it.
            const uint32_t k = uint32_t(top_k);
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
                if (count_above((cut | bit) - 1) >= k)
                    cut |= bit;
            ties = k - count_above(cut);
        }
        if (top_p < 1.0f) {
            // Ranks among the keys at the cut are by index: the last index kept.
            uint32_t last = 0;
            if (ties < width) {
                uint32_t low = 0, high = width - 1;
                while (low < high) {
                    const uint32_t middle = (low + high) / 2;
                    uint32_t n = 0;
                    for (uint32_t i = threadIdx.x; i <= middle; i += kBlock)
                        n += key_of(value(i)) == cut;
                    if (block_reduce(n, counts, sum) >= ties)
                        high = middle;
                    else
                        low = middle + 1;
                }
                last = low;
            } else {
                last = width - 1;
            }
            const auto weight_above = [&](uint32_t k) {
                double w = 0.0;
                for (uint32_t i = threadIdx.x; i < width; i += kBlock) {
                    const float v = value(i);
                    const uint32_t at = key_of(v);
                    if (at > k && (at > cut || (at == cut && i <= last)))
                        w += weight(v);
                }
                return block_reduce(w, doubles, sum);
            };
            // The smallest key with less than the wanted weight above it.
            const double wanted = double(top_p) * weight_above(cut ? cut - 1 : 0);
            uint32_t border = 0;
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
                if (weight_above((border | bit) - 1) >= wanted)
                    border |= bit;
            if (top_p == 0.0f || border > top)
                border = top;
            const double above = weight_above(border);
            const double each = weight(
                __uint_as_float(border & 0x80000000u ? border & 0x7fffffffu : ~border));
            double fit = ceil((wanted - above) / each);
            fit = fit >= 1.0 ? fit : border == top ? 1.0 : 0.0;
            const uint32_t whole = fit < double(width) ? uint32_t(fit) : width;
            if (border > cut) {
                cut = border;
                ties = whole;
            } else if (whole < ties) {
                ties = whole;
            }
        }
    }

    // Every thread a run of tokens; the kept ones' weights in their order.
    const uint32_t each = (width + kBlock - 1) / kBlock;
    const uint32_t first = threadIdx.x * each < width ? threadIdx.x * each : width;
    const uint32_t last = first + each < width ? first + each : width;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t equal = 0;
    for (uint32_t i = first; i < last; ++i)
        equal += key_of(value(i)) == cut;
    uint32_t before = equal;
#pragma unroll
    for (int offset = 1; offset < 64; offset <<= 1) {
        const uint32_t v = __shfl_up(before, offset, 64);
        if (int(lane) >= offset)
            before += v;
    }
    __syncthreads();
    if (lane == 63)
        counts[wave] = before;
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w)
        before += counts[w];
    before -= equal;
    const auto walk = [&](auto f) {
        uint32_t rank = before;
        for (uint32_t i = first; i < last; ++i) {
            const float v = value(i);
            const uint32_t at = key_of(v);
            if (at > cut || (at == cut && rank++ < ties)) {
                const double w = temperature == 0.0f ? 1.0 : weight(v);
                if (w >= double(min_p) && w > 0.0 && f(i, w))
                    break;
            }
        }
    };
    double mine = 0.0;
    walk([&](uint32_t, double w) {
        mine += w;
        return false;
    });
    double upto = mine;
#pragma unroll
    for (int offset = 1; offset < 64; offset <<= 1) {
        const double v = __shfl_up(upto, offset, 64);
        if (int(lane) >= offset)
            upto += v;
    }
    if (lane == 63)
        doubles[wave] = upto;
    if (threadIdx.x == 0)
        chosen = UINT32_MAX;
    __syncthreads();
    double total = 0.0;
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (w == wave)
            upto += total;
        total += doubles[w];
    }
    // The first thread whose run ends past the target; within its run the first
    // token that does, or its last kept one where rounding leaves none.
    const double target = double(u) * total;
    if (mine > 0.0 && upto > target)
        atomicMin(&chosen, threadIdx.x);
    __syncthreads();
    if (threadIdx.x == chosen) {
        double at = upto - mine;
        uint32_t token = 0;
        walk([&](uint32_t i, double w) {
            at += w;
            token = i;
            return at > target;
        });
        s.out[row] = float(token);
        if (s.copy)
            s.copy[row] = float(token);
    }
}

}  // namespace

void launch_sample_rows(hipStream_t stream, const Sampling &s)
{
    if (s.rows)
        sample_kernel<<<s.rows, kBlock, 0, stream>>>(s);
}

}  // namespace mfh
