// Attention of runs of new tokens (trees of drafted ones, or a prompt's) over paged
// caches of keys and values, or of latents.
//
// o = sum_j p_j v_j / sum_j p_j over the keys j that a token attends, with p_j =
// exp(s_j - max s) and s_j = q . k_j scale: all of the sequence's cached tokens and those
// of the run that its mask names.
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

}  // namespace

void launch_run_attention(hipStream_t stream, const RunAttention &p)
{
    const uint64_t blocks = uint64_t(p.runs.tokens) * p.query_heads;
    if (!blocks)
        return;
    const size_t bytes = (size_t(p.shape.head_dim) + p.value_dim) * sizeof(float);
    run_attention_general_kernel<<<unsigned(blocks), 64, bytes, stream>>>(p);
}

}  // namespace mfh
