// Penalties, biases and token masks on logits, in front of the token pick (include/llm_amd/paged.h).
#include <algorithm>

#include "common.h"
#include "llm_amd/paged.h"

using namespace llm;

namespace {

struct PenaltyArgs {
    bf16 *out;
    const bf16 *x;
    const int *tokens, *prompt_len, *token_len;
    const float *repetition, *frequency, *presence;
    const int *bias_tokens;
    const float *bias;
    const int *bias_len;
    const uint32_t *allowed;
    int vocab, token_stride, bias_stride, allowed_stride, slice;
    int64_t out_stride, x_stride;
};

constexpr uint32_t IN_PROMPT = 1u << 31;  // above the count of a token's answers

// What a token's logit becomes. met: its prompt bit and its count of answers.
struct Row {
    bool repeats;
    float repetition, frequency, presence;
    __device__ __forceinline__ float operator()(float x, uint32_t met, float bias, bool biased, bool allowed) const {
        const uint32_t count = met & ~IN_PROMPT;
        if (met && repeats) x = x > 0.0f ? x / repetition : x * repetition;
        if (count) x = x - frequency * (float)count - presence;
        if (biased) x += bias;
        return allowed ? x : -INFINITY;
    }
};

// Calls f(i, v) for the n values at p, four at a time from the first 16-byte boundary on, several requested
// ahead.
template <int T, class F>
__device__ __forceinline__ void each(const int *p, int n, F f) {
    const int lead = min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) / 4), quads = (n - lead) / 4;
    if ((int)threadIdx.x < lead) f(threadIdx.x, gptr(p)[threadIdx.x]);
    const u32x4 *q = (const u32x4 *)(p + lead);
    constexpr int U = 4;
    for (int i = threadIdx.x; i < quads; i += U * T) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) v[u] = *gptr(q + min(i + u * T, quads - 1));
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u * T < quads)
#pragma unroll
                for (int e = 0; e < 4; e++) f(lead + 4 * (i + u * T) + e, (int)v[u][e]);
    }
    const int done = lead + 4 * quads;
    if ((int)threadIdx.x < n - done) f(done + threadIdx.x, gptr(p)[done + threadIdx.x]);
}

// One workgroup per slice of a row's vocabulary. The row's history is read once by every slice (from L2 after
// the first); the slice's tokens are counted in LDS, by whole numbers, so that the order of the additions does
// not matter, and a bias is the last entry's because the largest index of a token's entries is kept. Then
// eight logits per thread at a time, 16 bytes where the rows' alignment allows it. Bound by the logits' bytes
// where there are many rows; one row by the launch and two round trips to memory.
template <int T>
__global__ __launch_bounds__(T) void penalty_kernel(PenaltyArgs a) {
    extern __shared__ uint32_t lds[];
    const int r = blockIdx.y, t0 = blockIdx.x * a.slice, n = min(a.slice, a.vocab - t0);
    uint32_t *met = lds;                                          // per token of the slice
    int *entry = (int *)(lds + (a.tokens ? a.slice : 0));         // 1 + the index of the token's last bias
    const bf16 *from = a.x + r * a.x_stride + t0;
    bf16 *to = a.out + r * a.out_stride + t0;
    // eight logits from a multiple of 8 on; the first ones are requested before the history is read
    const bool wide = (((uintptr_t)from | (uintptr_t)to) & 15) == 0;
    const auto request = [&](int i) {
        u32x4 x = {0, 0, 0, 0};
        if (wide && i + 8 <= n) {
            x = ld16(from + i);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (i + e < n) x[e / 2] |= (uint32_t)gptr(from)[i + e] << (e % 2 * 16);
        }
        return x;
    };
    const uint32_t *allowed = a.allowed ? a.allowed + (int64_t)r * a.allowed_stride + t0 / 32 : nullptr;
    u32x4 x = {0, 0, 0, 0};
    uint32_t word = ~0u;
    if (8 * (int)threadIdx.x < n) {
        x = request(8 * threadIdx.x);
        if (allowed) word = gptr(allowed)[threadIdx.x / 4];
    }
    const int history = a.tokens ? max(0, min(a.token_stride, gptr(a.token_len)[r])) : 0;
    const int prompt = a.tokens && a.prompt_len ? gptr(a.prompt_len)[r] : 0;
    const int biases = !a.bias_tokens ? 0
                       : a.bias_len   ? max(0, min(a.bias_stride, gptr(a.bias_len)[r]))
                                      : a.bias_stride;
    const Row row = {a.repetition != nullptr, a.repetition ? gptr(a.repetition)[r] : 1.0f,
                     a.frequency ? gptr(a.frequency)[r] : 0.0f, a.presence ? gptr(a.presence)[r] : 0.0f};
    const int clear = (a.tokens ? a.slice : 0) + (a.bias_tokens ? a.slice : 0);
    for (int i = 4 * threadIdx.x; i < clear; i += 4 * T) *(u32x4 *)(lds + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    if (history)
        each<T>(a.tokens + (int64_t)r * a.token_stride, history, [&](int i, int token) {
            const unsigned t = (unsigned)token - (unsigned)t0;
            if (t < (unsigned)n) {
                if (i < prompt)
                    atomicOr(&met[t], IN_PROMPT);
                else
                    atomicAdd(&met[t], 1u);
            }
        });
    if (biases)
        each<T>(a.bias_tokens + (int64_t)r * a.bias_stride, biases, [&](int i, int token) {
            const unsigned t = (unsigned)token - (unsigned)t0;
            if (t < (unsigned)n) atomicMax(&entry[t], i + 1);
        });
    __syncthreads();
    const float *bias = a.bias_tokens ? a.bias + (int64_t)r * a.bias_stride : nullptr;
    for (int i = 8 * threadIdx.x; i < n; i += 8 * T) {
        u32x4 more = {0, 0, 0, 0};
        uint32_t next = ~0u;
        if (i + 8 * T < n) {
            more = request(i + 8 * T);
            if (allowed) next = gptr(allowed)[(i + 8 * T) / 32];
        }
        const uint32_t bits = word >> (i % 32);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t m = history ? met[i + e] : 0;
            const int k = biases ? entry[i + e] : 0;
            y[e] = row(elem(x, e), m, k ? gptr(bias)[k - 1] : 0.0f, k != 0, bits >> e & 1);
        }
        if (wide && i + 8 <= n) {
            st16(to + i, u32x4{pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(y[4], y[5]), pack2(y[6], y[7])});
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (i + e < n) gptr(to)[i + e] = (bf16)f2bf(y[e]);
        }
        x = more;
        word = next;
    }
}

}  // namespace

extern "C" void logits_penalty_forward(bf16 *out, const bf16 *logits, const int *tokens,
                                       const int *prompt_len, const int *token_len,
                                       const float *repetition, const float *frequency,
                                       const float *presence, const int *bias_tokens,
                                       const float *bias, const int *bias_len,
                                       const uint32_t *allowed, int rows, int vocab,
                                       int token_stride, int bias_stride, int allowed_stride,
                                       int64_t out_stride, int64_t logits_stride,
                                       hipStream_t stream) {
    static const char name[] = "logits_penalty";
    if (rows < 0 || rows > 65535) {
        llm_fail("%s: rows %d is not in 0..65535", name, rows);
        return;
    }
    if (vocab <= 0 || vocab > 1 << 28) {
        llm_fail("%s: vocab %d is not in 1..268435456", name, vocab);
        return;
    }
    if (rows == 0) return;
    if (!out || !logits) {
        llm_fail("%s: out and logits must not be null", name);
        return;
    }
    if (out_stride < vocab || logits_stride < vocab) {
        llm_fail("%s: rows %lld and %lld elements apart overlap (vocab %d)", name,
                 (long long)out_stride, (long long)logits_stride, vocab);
        return;
    }
    if (out == logits && out_stride != logits_stride) {
        llm_fail("%s: in place, the rows of out and logits must be the same", name);
        return;
    }
    if (tokens && (!token_len || token_stride < 0)) {
        llm_fail("%s: a history needs token_len and a token_stride that is not negative", name);
        return;
    }
    if (bias_tokens && (!bias || bias_stride < 0)) {
        llm_fail("%s: biases need their values and a bias_stride that is not negative", name);
        return;
    }
    if (allowed && allowed_stride < (vocab + 31) / 32) {
        llm_fail("%s: allowed_stride %d is under the %d words of %d tokens", name, allowed_stride,
                 (vocab + 31) / 32, vocab);
        return;
    }
    // a slice as large as the device is still filled with, so that histories are read less often (whole
    // 512s of tokens: a bias entry and a count are 8 bytes of LDS each)
    int slice = 8192;
    while (slice > 1024 && (int64_t)rows * ((vocab + slice - 1) / slice) < 512) slice /= 2;
    PenaltyArgs a = {out, logits, tokens, prompt_len, token_len, repetition, frequency, presence,
                     bias_tokens, bias, bias_len, allowed, vocab, token_stride, bias_stride,
                     allowed_stride, slice, out_stride, logits_stride};
    const dim3 grid((vocab + slice - 1) / slice, rows);
    const unsigned lds = slice * ((tokens ? 4 : 0) + (bias_tokens ? 4 : 0));
    if (slice > 2048)
        penalty_kernel<512><<<grid, 512, lds, stream>>>(a);
    else
        penalty_kernel<256><<<grid, 256, lds, stream>>>(a);
    LAUNCH_OK();
}
