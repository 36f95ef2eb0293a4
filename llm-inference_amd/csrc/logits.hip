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

constexpr int T = 512;                     // threads of a workgroup
constexpr uint32_t IN_PROMPT = 1u << 31;  // above the count of a token's answers

// The values of a row, four per thread at a time where the row is 16-byte aligned: the first U times T fours
// are requested (as far as the row's `room` goes) before the row's length is known.
constexpr int U = 4;
struct Values {
    const int *p;
    int room;
    bool wide;
    u32x4 first[U];
    __device__ __forceinline__ Values(const int *p_, int room_) : p(p_), room(room_), wide(((uintptr_t)p_ & 15) == 0) {
        if (!wide || room < 4) return;
#pragma unroll
        for (int u = 0; u < U; u++) first[u] = *gptr((const u32x4 *)p + min((int)threadIdx.x + u * T, room / 4 - 1));
    }
    // f(i, value i) for the first n values, n <= room.
    template <class F>
    __device__ __forceinline__ void each(int n, F f) {
        int done = 0;
        if (wide && n >= 4) {
            const int quads = n / 4;
            const u32x4 *q = (const u32x4 *)p;
            for (int i = threadIdx.x; i < quads; i += U * T) {
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (i + u * T < quads) {
#pragma unroll
                        for (int e = 0; e < 4; e++) f(4 * (i + u * T) + e, (int)first[u][e]);
                        if (i + (u + U) * T < quads) first[u] = *gptr(q + i + (u + U) * T);
                    }
            }
            done = 4 * quads;
        }
        for (int i = done + threadIdx.x; i < n; i += T) f(i, gptr(p)[i]);
    }
};

// One workgroup per slice of a row's vocabulary. The row's history is read once by every slice (from memory by the
// first on each XCD, then from its L2); the slice's tokens are counted in LDS, by whole numbers, so that the order of
// the additions does not matter. Then eight logits per thread at a time, 16 bytes where the row's alignment allows it
// and one by one where not (64 rows of 50256 10.8 us, of 50257, where one row in eight is aligned, 16.1). 64 rows of
// 151936, up to 8192 tokens and 300 biases: 15.6 us, 2.6 TB/s, of which the history takes 1.6 and the biases 2; what
// bounds it is one phase of a workgroup waiting for the other (all logits requested in front of the history
// instead of the first eight per thread: 21.0 against 19.9 then); one row by the launch and two round trips to
// memory (4.9 us).
// NARROW: counts of 16 bits instead of 32, for histories that cannot count further.
// DENSE: a word per token for its bias, for any number of biases: entry i leaves -(i + 1) there if that is the
// least, so the last entry of a token stays, and then puts its value there. As floats those numbers are NaN,
// which no value put there is, so no other entry can take a value for its number. Otherwise, for up to T biases,
// a bit per token, and a token's last entry in the first of 2 T places from its own on that no other token has
// (in the order of the tokens instead, found by counting bits, with three barriers more, 19.9 us instead of 17.4).
template <bool NARROW, bool DENSE>
__global__ __launch_bounds__(T) void penalty_kernel(PenaltyArgs a) {
    extern __shared__ uint32_t lds[];
    constexpr int PER = NARROW ? 2 : 1;  // tokens per word of the counts
    constexpr int WORD = DENSE ? 1 : 32;  // tokens per word of the biases
    constexpr int PLACES = DENSE ? 1 : 2 * T;
    __shared__ uint32_t placed[PLACES];
    __shared__ float values[DENSE ? 1 : T];
    const int r = blockIdx.y, t0 = blockIdx.x * a.slice, n = min(a.slice, a.vocab - t0);
    uint32_t *met = lds, *biased = lds + (a.tokens ? a.slice / PER : 0);
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
    Values tokens(a.tokens + (int64_t)r * a.token_stride, a.tokens ? a.token_stride : 0);
    u32x4 x = {0, 0, 0, 0};
    uint32_t word = ~0u;
    if (8 * (int)threadIdx.x < n) {
        x = request(8 * threadIdx.x);
        if (allowed) word = gptr(allowed)[threadIdx.x / 4];
    }
    int bias_token = -1;  // this thread's entry, where there are no more than threads
    float value = 0.0f;
    if (!DENSE && a.bias_tokens && (int)threadIdx.x < a.bias_stride) {
        bias_token = gptr(a.bias_tokens)[(int64_t)r * a.bias_stride + threadIdx.x];
        value = gptr(a.bias)[(int64_t)r * a.bias_stride + threadIdx.x];
    }
    const int history = a.tokens ? max(0, min(a.token_stride, gptr(a.token_len)[r])) : 0;
    const int prompt = a.tokens && a.prompt_len ? gptr(a.prompt_len)[r] : 0;
    const int biases = !a.bias_tokens ? 0
                       : a.bias_len   ? max(0, min(a.bias_stride, gptr(a.bias_len)[r]))
                                      : a.bias_stride;
    const float repetition = a.repetition ? gptr(a.repetition)[r] : 1.0f, inverse = 1.0f / repetition;
    const float frequency = a.frequency ? gptr(a.frequency)[r] : 0.0f;
    const float presence = a.presence ? gptr(a.presence)[r] : 0.0f;
    const int *bias_tokens = a.bias_tokens + (int64_t)r * a.bias_stride;
    const float *bias = a.bias + (int64_t)r * a.bias_stride;
    const auto in_slice = [&](int token) { return (unsigned)token - (unsigned)t0 < (unsigned)n; };
    const int clear = (a.tokens ? a.slice / PER : 0) + (a.bias_tokens ? a.slice / WORD : 0);
    for (int i = 4 * threadIdx.x; i < clear; i += 4 * T) *(u32x4 *)(lds + i) = u32x4{0, 0, 0, 0};
    if (!DENSE && a.bias_tokens) placed[threadIdx.x] = placed[threadIdx.x + T] = 0;
    __syncthreads();
    if (history)
        tokens.each(history, [&](int i, int token) {
            const unsigned t = (unsigned)token - (unsigned)t0;
            if (t < (unsigned)n) {
                const int shift = NARROW ? t % 2 * 16 : 0;
                if (i < prompt)
                    atomicOr(&met[t / PER], (NARROW ? 0x8000u : IN_PROMPT) << shift);
                else
                    atomicAdd(&met[t / PER], 1u << shift);
            }
        });
    if (DENSE && biases) {
        for (int i = threadIdx.x; i < biases; i += T)
            if (in_slice(gptr(bias_tokens)[i])) atomicMin((int *)&biased[gptr(bias_tokens)[i] - t0], -(i + 1));
        __syncthreads();
        for (int i = threadIdx.x; i < biases; i += T) {
            if (!in_slice(gptr(bias_tokens)[i])) continue;
            uint32_t *at = &biased[gptr(bias_tokens)[i] - t0];
            if ((int)*at != -(i + 1)) continue;
            const float v = gptr(bias)[i];
            *at = v == v ? __float_as_uint(v) : 0x7fc00000u;
        }
    } else if ((int)threadIdx.x < biases && in_slice(bias_token)) {
        const int t = bias_token - t0;
        values[threadIdx.x] = value;
        atomicOr(&biased[t / 32], 1u << (t % 32));
        const uint32_t entry = (uint32_t)t << 16 | (threadIdx.x + 1);
        for (uint32_t at = t;; at++) {  // ends: there are more places than entries
            const uint32_t there = atomicCAS(&placed[at % PLACES], 0, entry);
            if (there && there >> 16 != (uint32_t)t) continue;
            if (there) atomicMax(&placed[at % PLACES], entry);
            break;
        }
    }
    __syncthreads();
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
            uint32_t m = history ? met[(i + e) / PER] : 0;
            if constexpr (NARROW) m = e & 1 ? m >> 16 : m & 0xffff;
            const uint32_t count = m & (NARROW ? 0x7fff : ~IN_PROMPT);
            const float z = elem(x, e), factor = z > 0.0f ? inverse : repetition;
            const float less = fmaf(frequency, (float)count, presence);
            y[e] = z * (m ? factor : 1.0f) - (count ? less : 0.0f);
        }
        if (DENSE && biases) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (biased[i + e]) y[e] += __uint_as_float(biased[i + e]);
        } else if (biases) {
            const uint32_t all = biased[i / 32];
            if (all >> (i % 32) & 0xff) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (!(all >> (i % 32 + e) & 1)) continue;
                    uint32_t at = i + e, entry = placed[at % PLACES];
                    while (entry >> 16 != (uint32_t)(i + e)) entry = placed[++at % PLACES];  // it is there
                    y[e] += values[(entry & 0xffff) - 1];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = bits >> e & 1 ? y[e] : -INFINITY;
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
    if (bias_tokens && bias_stride > 1 << 22) {  // more entries' numbers would meet the bits of -inf
        llm_fail("%s: bias_stride %d is over 4194304", name, bias_stride);
        return;
    }
    if (allowed && allowed_stride < (vocab + 31) / 32) {
        llm_fail("%s: allowed_stride %d is under the %d words of %d tokens", name, allowed_stride,
                 (vocab + 31) / 32, vocab);
        return;
    }
    const bool narrow = token_stride < 1 << 15, dense = bias_tokens && bias_stride > T;
    // a slice's counts and biases in at most 48 KB of LDS; smaller ones where there are too few workgroups (64 rows
    // of 151936, up to 8192 tokens and 300 biases, slices of 4096 / 8192 / 12288 / 16384: 17.1 / 15.6 / 16.4 / 16.9 us,
    // with up to 40000 tokens 25.6 / 21.8 / 25.1; 16 rows, 2048 / 4096 / 8192: 8.7 / 8.0 / 8.4; one, 2048 / 4096: 4.6 / 4.4)
    int slice = dense && !narrow ? 4096 : 8192;
    while (slice > 2048 && (int64_t)rows * ((vocab + slice - 1) / slice) < 512) slice /= 2;
    PenaltyArgs a = {out, logits, tokens, prompt_len, token_len, repetition, frequency, presence,
                     bias_tokens, bias, bias_len, allowed, vocab, token_stride, bias_stride,
                     allowed_stride, slice, out_stride, logits_stride};
    const dim3 grid((vocab + slice - 1) / slice, rows);
    const unsigned lds = (tokens ? slice * (narrow ? 2 : 4) : 0) + (bias_tokens ? dense ? slice * 4 : slice / 8 : 0);
    if (narrow && !dense)
        penalty_kernel<true, false><<<grid, T, lds, stream>>>(a);
    else if (narrow)
        penalty_kernel<true, true><<<grid, T, lds, stream>>>(a);
    else if (!dense)
        penalty_kernel<false, false><<<grid, T, lds, stream>>>(a);
    else
        penalty_kernel<false, true><<<grid, T, lds, stream>>>(a);
    LAUNCH_OK();
}
