// A projection of many rows with the low-rank adapters of their sequences (include/llm_amd/batch.h).
#include <algorithm>

#include "common.h"
#include "llm_amd/batch.h"

using namespace llm;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

struct LoraArgs {
    bf16 *out;
    const bf16 *x, *w, *residual;
    const bf16 *a, *b;
    const float *scale;
    const int *q_start, *adapter;
    float *low;  // [n_tokens, rank]
    int64_t out_stride, x_stride, residual_stride;
    int n_tokens, n_out, n_in, n_seqs, n_adapters, rank;
};

__device__ __forceinline__ f32x4 mfma(const u32x4 &a, const u32x4 &b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                   0, 0);
}

// The sequence of row t, or -1.
__device__ __forceinline__ int sequence_of(const LoraArgs &l, int t) {
    int lo = 0, hi = l.n_seqs;  // the first sequence that ends behind t
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (gptr(l.q_start)[mid + 1] <= t) lo = mid + 1;
        else hi = mid;
    }
    return lo < l.n_seqs && gptr(l.q_start)[lo] <= t && t < gptr(l.q_start)[lo + 1] ? lo : -1;
}
// Its adapter: -1 none, -2 no sequence.
__device__ __forceinline__ int adapter_of(const LoraArgs &l, int t) {
    if (!l.a) return -1;
    const int s = sequence_of(l, t);
    if (s < 0) return -2;
    const int a = gptr(l.adapter)[s];
    return (unsigned)a < (unsigned)l.n_adapters ? a : -1;
}

// low[t] = scale (a x[t]), a wave per row and element.
__global__ __launch_bounds__(256) void shrink_kernel(LoraArgs l) {
    const int t = blockIdx.y, j = blockIdx.x * 4 + wave_id(), lane = threadIdx.x & 63;
    const int a = adapter_of(l, t);
    if (a < 0 || j >= l.rank) return;
    const bf16 *row = l.a + ((int64_t)a * l.rank + j) * l.n_in, *x = l.x + t * l.x_stride;
    float sum = 0;
    for (int i = lane * 8; i < l.n_in; i += 512) sum = dot8(ld16(row + i), ld16(x + i), sum);
    sum = wave_sum(sum);
    if (lane == 0) l.low[(int64_t)t * l.rank + j] = sum * (l.scale ? gptr(l.scale)[a] : 1.0f);
}

// 16 rows by 16 columns per wave: lane's row l % 16, columns 4 (l / 16) .. + 3.
__global__ __launch_bounds__(256) void project_kernel(LoraArgs l) {
    const int lane = threadIdx.x & 63, n0 = (blockIdx.x * 4 + wave_id()) * 16, t0 = blockIdx.y * 16;
    if (n0 >= l.n_out) return;
    const int t = t0 + lane % 16, k0 = lane / 16 * 8;
    f32x4 acc = {0, 0, 0, 0};
    if (l.w) {
        const bf16 *w = l.w + (int64_t)min(n0 + lane % 16, l.n_out - 1) * l.n_in, *x = l.x + min(t, l.n_tokens - 1) * l.x_stride;
        for (int k = k0; k - k0 < l.n_in; k += 32) {
            u32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (k < l.n_in) a = ld16(w + k), b = ld16(x + k);
            acc = mfma(a, b, acc);
        }
    }
    if (t >= l.n_tokens) return;
    const int a = adapter_of(l, t);
    if (a == -2) return;
    for (int e = 0; e < 4; e++) {
        const int n = n0 + lane / 16 * 4 + e;
        if (n >= l.n_out) break;
        float y = acc[e];
        if (a >= 0) {
            const bf16 *b = l.b + ((int64_t)a * l.n_out + n) * l.rank;
            for (int j = 0; j < l.rank; j++) y = fmaf(l.low[(int64_t)t * l.rank + j], bf2f(gptr(b)[j]), y);
        }
        if (l.residual) y += bf2f(gptr(l.residual)[t * l.residual_stride + n]);
        gptr(l.out)[t * l.out_stride + n] = (bf16)f2bf(y);
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

bool check_sizes(const char *name, int n_tokens, int n_out, int n_in, int rank) {
    if (n_tokens < 0 || n_tokens > 1 << 20) return llm_fail("%s: n_tokens %d is not in 0..1048576", name, n_tokens);
    if (n_out <= 0 || n_out > 1 << 22) return llm_fail("%s: n_out %d is not in 1..4194304", name, n_out);
    if (n_in <= 0 || n_in > 1 << 20 || n_in % 8)
        return llm_fail("%s: n_in %d is not a multiple of 8 in 8..1048576", name, n_in);
    if (rank < 0 || rank > 256 || rank % 8) return llm_fail("%s: rank %d is not a multiple of 8 up to 256", name, rank);
    return true;
}

}  // namespace

extern "C" size_t lora_projection_workspace_floats(int n_tokens, int n_out, int n_in, int rank) {
    if (!check_sizes("lora_projection_workspace_floats", n_tokens, n_out, n_in, rank)) return 0;
    return (size_t)n_tokens * rank;
}

extern "C" void lora_projection_forward(bf16 *out, const bf16 *x, const bf16 *w, const bf16 *residual,
                                        const LoraBatch *lora, float *ws, int n_tokens, int n_out, int n_in,
                                        int64_t out_stride, int64_t x_stride, int64_t residual_stride,
                                        hipStream_t stream) {
    static const char name[] = "lora_projection";
    if (!check_sizes(name, n_tokens, n_out, n_in, lora ? lora->rank : 0)) return;
    if (lora) {
        if (lora->rank == 0 || lora->n_seqs <= 0 || lora->n_seqs > 1 << 20 || lora->n_adapters <= 0) {
            llm_fail("%s: rank %d, n_seqs %d (up to 1048576) and n_adapters %d must be positive", name, lora->rank,
                     lora->n_seqs, lora->n_adapters);
            return;
        }
        if (!lora->a || !lora->b || !lora->q_start || !lora->adapter || !aligned16(lora->a) || !aligned16(lora->b)) {
            llm_fail("%s: a, b, q_start and adapter must not be null, a and b 16-byte aligned", name);
            return;
        }
    }
    if (n_tokens == 0) return;
    if (!out || !x || !aligned16(x) || !aligned16(w)) {
        llm_fail("%s: out and x must not be null, x and w 16-byte aligned", name);
        return;
    }
    if (x_stride < n_in || x_stride % 8) {
        llm_fail("%s: the rows of x are %lld elements apart, not a multiple of 8 of at least %d", name,
                 (long long)x_stride, n_in);
        return;
    }
    if (out_stride < n_out || (residual && residual_stride < n_out)) {
        llm_fail("%s: rows %lld and %lld elements apart overlap (n_out %d)", name, (long long)out_stride,
                 (long long)residual_stride, n_out);
        return;
    }
    if (out == residual && out_stride != residual_stride) {
        llm_fail("%s: in place, the rows of out and residual must be the same", name);
        return;
    }
    if (out == x) {
        llm_fail("%s: out must not be x, which is read again", name);
        return;
    }
    if (!aligned16(ws) || (lora && !ws)) {
        llm_fail("%s: ws must be a 16-byte aligned device address", name);
        return;
    }
    LoraArgs l = {out, x, w, residual, nullptr, nullptr, nullptr, nullptr, nullptr, ws, out_stride, x_stride, residual_stride,
                  n_tokens, n_out, n_in, 0, 0, 0};
    if (lora) {
        l.a = lora->a, l.b = lora->b, l.scale = lora->scale, l.q_start = lora->q_start, l.adapter = lora->adapter;
        l.n_seqs = lora->n_seqs, l.n_adapters = lora->n_adapters, l.rank = lora->rank;
        shrink_kernel<<<dim3((l.rank + 3) / 4, n_tokens), 256, 0, stream>>>(l);
        if (!LAUNCH_OK()) return;
    }
    project_kernel<<<dim3((n_out + 63) / 64, (n_tokens + 15) / 16), 256, 0, stream>>>(l);
    LAUNCH_OK();
}
