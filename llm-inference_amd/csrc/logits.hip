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

// One workgroup per slice of a row's vocabulary. The row's history is read once by every slice; the
// slice's tokens are counted in LDS, by whole numbers, so that the order of the additions does not
// matter, and a bias is the last entry's because the largest index of a token's entries is kept.
__global__ __launch_bounds__(256) void penalty_kernel(PenaltyArgs a) {
    extern __shared__ uint32_t lds[];
    uint32_t *met = lds;               // a prompt bit and the answers' count per token of the slice
    int *entry = (int *)(lds + a.slice);  // 1 + the index of the token's last bias
    const int r = blockIdx.y, t0 = blockIdx.x * a.slice, n = min(a.slice, a.vocab - t0);
    const int history = a.tokens ? max(0, min(a.token_stride, gptr(a.token_len)[r])) : 0;
    const int prompt = a.tokens && a.prompt_len ? gptr(a.prompt_len)[r] : 0;
    const int biases = !a.bias_tokens ? 0
                       : a.bias_len   ? max(0, min(a.bias_stride, gptr(a.bias_len)[r]))
                                      : a.bias_stride;
    for (int i = threadIdx.x; i < n; i += 256) {
        met[i] = 0;
        if (a.bias_tokens) entry[i] = 0;
    }
    __syncthreads();
    const int *tokens = a.tokens + (int64_t)r * a.token_stride;
    for (int i = threadIdx.x; i < history; i += 256) {
        const unsigned t = (unsigned)(gptr(tokens)[i]) - (unsigned)t0;
        if (t < (unsigned)n) {
            if (i < prompt)
                atomicOr(&met[t], IN_PROMPT);
            else
                atomicAdd(&met[t], 1u);
        }
    }
    const int *bias_tokens = a.bias_tokens + (int64_t)r * a.bias_stride;
    for (int i = threadIdx.x; i < biases; i += 256) {
        const unsigned t = (unsigned)(gptr(bias_tokens)[i]) - (unsigned)t0;
        if (t < (unsigned)n) atomicMax(&entry[t], i + 1);
    }
    __syncthreads();
    const float repetition = a.repetition ? gptr(a.repetition)[r] : 1.0f;
    const float frequency = a.frequency ? gptr(a.frequency)[r] : 0.0f;
    const float presence = a.presence ? gptr(a.presence)[r] : 0.0f;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int t = t0 + i;
        float x = bf2f(gptr(a.x)[r * a.x_stride + t]);
        const uint32_t m = met[i], count = m & ~IN_PROMPT;
        if (m && a.repetition) x = x > 0.0f ? x / repetition : x * repetition;
        if (count) x = x - frequency * (float)count - presence;
        if (a.bias_tokens && entry[i]) x += gptr(a.bias)[(int64_t)r * a.bias_stride + entry[i] - 1];
        if (a.allowed && !(gptr(a.allowed)[(int64_t)r * a.allowed_stride + t / 32] >> (t % 32) & 1))
            x = -INFINITY;
        gptr(a.out)[r * a.out_stride + t] = (bf16)f2bf(x);
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
    PenaltyArgs a = {out, logits, tokens, prompt_len, token_len, repetition, frequency, presence,
                     bias_tokens, bias, bias_len, allowed, vocab, token_stride, bias_stride,
                     allowed_stride, 4096, out_stride, logits_stride};
    const dim3 grid((vocab + a.slice - 1) / a.slice, rows);
    penalty_kernel<<<grid, 256, a.slice * (bias_tokens ? 8 : 4), stream>>>(a);
    LAUNCH_OK();
}
