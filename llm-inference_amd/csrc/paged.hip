// Operators over a paged KV cache: QK-norm + RoPE that writes new keys and values into pages, and the
// attention of new tokens over pages (include/llm_amd/paged.h).
#include <math.h>
#include <string.h>

#include <algorithm>

#include "common.h"
#include "llm_amd/paged.h"

using namespace llm;

namespace {

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// ------------------------------------------------------------------------------------------
// the batch on the device
// ------------------------------------------------------------------------------------------

// n / d for 0 <= n < 2^31 by a multiplication: with 2^(l-1) < d <= 2^l and m = floor(2^(31+l) / d) + 1,
// m d exceeds 2^(31+l) by at most d <= 2^l, so floor(n m / 2^(31+l)) = floor(n / d) for n < 2^31.
struct Divisor {
    uint32_t m;
    int l;
    explicit Divisor(uint32_t d = 1) : m(0), l(0) {
        while ((1ull << l) < d) l++;
        m = (uint32_t)((1ull << (31 + l)) / d + 1);
    }
};
__device__ __forceinline__ int divide(int n, uint32_t m, int l) {
    return l == 0 ? n : (int)(__umulhi((uint32_t)n, m) >> (l - 1));
}

// What the kernels read of a PagedBatch.
struct Batch {
    bf16 *kc, *vc;
    int64_t page_stride, slot_stride, head_stride;
    const int *table, *q_start, *kv_len;
    int n_seqs, n_pages, page_size, table_pages, n_tokens;
    Divisor page;
};

// The sequence whose rows hold row t, or -1: the number of sequences that end at or before t, found by
// all 64 lanes at once (64 probes per round), then checked against that sequence's first row. Whatever
// q_start holds, the result is in [-1, n_seqs).
__device__ __forceinline__ int sequence_of(const Batch &b, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = b.n_seqs;
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;
        const int64_t at = lo + (int64_t)(lane + 1) * step - 1;  // the last of the lane's share
        const bool ends = at < hi && gptr(b.q_start)[at + 1] <= t;
        const int n = __popcll(__ballot(ends));
        hi = min(hi, lo + n * step + step - 1);
        lo += n * step;
    }
    if (lo >= b.n_seqs || gptr(b.q_start)[lo] > t || gptr(b.q_start)[lo + 1] <= t) return -1;
    return lo;
}

// Lengths outside [-2^30, 2^30] are cut to it, so that positions do not overflow.
__device__ __forceinline__ int kv_length(const Batch &b, int s) {
    return max(-(1 << 30), min(1 << 30, gptr(b.kv_len)[s]));
}

// Element offset of position p of sequence s in the caches (head 0), or -1 where it is not there.
__device__ __forceinline__ int64_t place(const Batch &b, int s, int p) {
    if (p < 0) return -1;
    const int i = divide(p, b.page.m, b.page.l);
    if (i >= b.table_pages) return -1;
    const int page = gptr(b.table)[(int64_t)s * b.table_pages + i];
    if ((unsigned)page >= (unsigned)b.n_pages) return -1;
    return page * b.page_stride + (p - i * b.page_size) * b.slot_stride;
}

bool take_batch(const char *name, const PagedBatch *p, int n_tokens, int n_heads, Batch *b) {
    if (!p) return llm_fail("%s: no batch", name);
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
        return llm_fail("%s: head_dim %d is not 64, 128 or 256", name, p->head_dim);
    if (p->n_kv_heads <= 0 || n_heads <= 0 || n_heads % p->n_kv_heads != 0)
        return llm_fail("%s: n_heads %d is not a positive multiple of n_kv_heads %d", name, n_heads,
                        p->n_kv_heads);
    if (n_heads > 65535) return llm_fail("%s: n_heads %d is over 65535", name, n_heads);
    if (p->n_seqs <= 0 || p->n_pages <= 0 || p->page_size <= 0 || p->table_pages <= 0)
        return llm_fail("%s: n_seqs %d, n_pages %d, page_size %d and table_pages %d must be positive", name,
                        p->n_seqs, p->n_pages, p->page_size, p->table_pages);
    if (p->page_size > 1 << 20) return llm_fail("%s: page_size %d is over 1048576", name, p->page_size);
    if (n_tokens < 0 || n_tokens > 1 << 24)
        return llm_fail("%s: n_tokens %d is not in 0..16777216", name, n_tokens);
    if (!p->key_cache || !p->value_cache || !p->page_table || !p->q_start || !p->kv_len)
        return llm_fail("%s: the batch has a null pointer", name);
    if (!aligned16(p->key_cache) || !aligned16(p->value_cache))
        return llm_fail("%s: the caches must be 16-byte aligned", name);
    if (p->page_stride % 8 || p->slot_stride % 8 || p->head_stride % 8)
        return llm_fail("%s: cache strides %lld, %lld, %lld are not multiples of 8", name,
                        (long long)p->page_stride, (long long)p->slot_stride, (long long)p->head_stride);
    b->kc = p->key_cache;
    b->vc = p->value_cache;
    b->page_stride = p->page_stride;
    b->slot_stride = p->slot_stride;
    b->head_stride = p->head_stride;
    b->table = p->page_table;
    b->q_start = p->q_start;
    b->kv_len = p->kv_len;
    b->n_seqs = p->n_seqs;
    b->n_pages = p->n_pages;
    b->page_size = p->page_size;
    b->table_pages = p->table_pages;
    b->n_tokens = n_tokens;
    b->page = Divisor((uint32_t)p->page_size);
    return true;
}

bool check_rows(const char *name, const char *what, const void *p, int64_t stride, int64_t width) {
    if (!p) return llm_fail("%s: %s is null", name, what);
    if (!aligned16(p)) return llm_fail("%s: %s must be 16-byte aligned", name, what);
    if (stride < width || stride % 8)
        return llm_fail("%s: the rows of %s are %lld elements apart, not a multiple of 8 of at least %lld",
                        name, what, (long long)stride, (long long)width);
    return true;
}

// ------------------------------------------------------------------------------------------
// QK-norm + RoPE into pages
// ------------------------------------------------------------------------------------------

struct AppendArgs {
    Batch b;
    bf16 *q_out;
    const bf16 *q, *k, *v, *qn, *kn;
    const double *inv_freq;
    int64_t qo_stride, q_stride, k_stride, v_stride;
    int n_heads, n_kv_heads, rotary, interleaved;
    int q_groups, kv_groups, share, waves_per_token;
    float eps, scale;
};

// A wave takes `share` of a row's head groups: 64 / (D / 8) heads of q, k or v at a time, 16 bytes of a
// head per lane. The row's cos and sin are computed once per wave, a pair or two per lane, in 64 bits
// (the angle, reduced by whole turns, and its cos and sin), and read back from LDS by the lanes that hold
// the pair's elements. The norm's sum and everything after it stay in 32 bits up to the one rounding.
template <int D>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    constexpr int LH = D / 8, HPW = 64 / LH;
    __shared__ __align__(16) float2 turn[4][D / 2];
    const int lane = threadIdx.x & 63, w = wave_id();
    const int64_t wave = (int64_t)blockIdx.x * 4 + w;
    const int t = (int)(wave / a.waves_per_token);
    if (t >= a.b.n_tokens) return;
    const int part = (int)(wave - (int64_t)t * a.waves_per_token);
    const int s = sequence_of(a.b, t);
    if (s < 0) return;
    const int pos = kv_length(a.b, s) - gptr(a.b.q_start)[s + 1] + t;
    const int64_t at = place(a.b, s, pos);
    const int half = a.rotary / 2;
    for (int j = lane; j < half; j += 64) {
        // angle - 2 pi k with 2 pi in two parts: the first product is exact to the last bit of fma
        const double angle = (double)pos * gptr(a.inv_freq)[j];
        const double k = rint(angle * 0x1.45f306dc9c883p-3);
        const double r = fma(-k, 0x1.1a62633145c07p-52, fma(-k, 0x1.921fb54442d18p+2, angle));
        double sn, cs;
        sincos_d(r, &sn, &cs);
        turn[w][j] = make_float2((float)cs * a.scale, (float)sn * a.scale);
    }
    const int L = lane % LH, hg = lane / LH;
    const bool turned = 8 * L < a.rotary;
    const bool second = !a.interleaved && 8 * L >= half;
    float c[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int j = a.interleaved ? 4 * L + e / 2 : 8 * L + e - (second ? half : 0);
        const float2 cs = turned ? turn[w][j] : make_float2(1.0f, 0.0f);
        c[e] = cs.x;
        // the pair (x, y) goes to (x cos - y sin, y cos + x sin)
        sn[e] = (a.interleaved ? !(e & 1) : !second) ? -cs.y : cs.y;
    }
    const int partner = second ? lane - half / 8 : lane + half / 8;
    const int groups = a.q_groups + 2 * a.kv_groups;
    for (int g = part * a.share; g < min(groups, (part + 1) * a.share); g++) {
        const bool is_q = g < a.q_groups, is_v = g >= a.q_groups + a.kv_groups;
        const int h = (is_q ? g : is_v ? g - a.q_groups - a.kv_groups : g - a.q_groups) * HPW + hg;
        const bool there = h < (is_q ? a.n_heads : a.n_kv_heads);
        if (!is_q && at < 0) continue;
        const bf16 *src = is_q   ? a.q + t * a.q_stride
                          : is_v ? a.v + t * a.v_stride
                                 : a.k + t * a.k_stride;
        u32x4 x = {0, 0, 0, 0};
        if (there) x = ld16(src + h * D + 8 * L);
        if (is_v) {
            if (there) st16(a.b.vc + at + h * a.b.head_stride + 8 * L, x);
            continue;
        }
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = elem(x, e);
        const bf16 *weight = is_q ? a.qn : a.kn;
        if (weight) {
            const u32x4 wt = ld16(weight + 8 * L);
            const float inv = 1.0f / sqrtf(group_sum<LH>(dot8(x, x, 0.0f)) / (float)D + a.eps);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = y[e] * inv * elem(wt, e);
        }
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float other = a.interleaved ? y[e ^ 1] : __shfl(y[e], partner & 63);
            o[e] = turned ? fmaf(other, sn[e], y[e] * c[e]) : y[e];
        }
        if (!there) continue;
        const u32x4 r = {pack2(o[0], o[1]), pack2(o[2], o[3]), pack2(o[4], o[5]), pack2(o[6], o[7])};
        if (is_q)
            st16(a.q_out + t * a.qo_stride + h * D + 8 * L, r);
        else
            st16(a.b.kc + at + h * a.b.head_stride + 8 * L, r);
    }
}

}  // namespace

extern "C" float rope_frequencies(double *inv_freq, int rotary_dim, double theta, int kind,
                                  double factor, int trained) {
    if (!inv_freq || rotary_dim <= 0 || rotary_dim % 2) {
        llm_fail("rope_frequencies: rotary_dim %d is not a positive even number", rotary_dim);
        return 0.0f;
    }
    if (!(theta > 1.0) || !isfinite(theta)) {
        llm_fail("rope_frequencies: theta %g is not over 1", theta);
        return 0.0f;
    }
    if (kind != ROPE_PLAIN && kind != ROPE_LINEAR && kind != ROPE_YARN) {
        llm_fail("rope_frequencies: kind %d is not ROPE_PLAIN, ROPE_LINEAR or ROPE_YARN", kind);
        return 0.0f;
    }
    if (kind != ROPE_PLAIN && (!(factor >= 1.0) || !isfinite(factor))) {
        llm_fail("rope_frequencies: factor %g is not at least 1", factor);
        return 0.0f;
    }
    if (kind == ROPE_YARN && trained <= 0) {
        llm_fail("rope_frequencies: trained %d must be positive", trained);
        return 0.0f;
    }
    double low = 0, high = 1;
    if (kind == ROPE_YARN) {
        // the pair that turns n times over the trained length: trained theta^(-2j / R) = 2 pi n
        const auto pair_that_turns = [&](double n) {
            return rotary_dim * log(trained / (n * 2 * M_PI)) / (2 * log(theta));
        };
        low = fmax(floor(pair_that_turns(32)), 0.0);
        high = fmin(ceil(pair_that_turns(1)), (double)(rotary_dim - 1));
        if (high == low) high += 0.001;
    }
    for (int j = 0; j < rotary_dim / 2; j++) {
        const double f = pow(theta, -2.0 * j / rotary_dim);
        const double ramp = fmin(1.0, fmax(0.0, (j - low) / (high - low)));
        inv_freq[j] = kind == ROPE_PLAIN    ? f
                      : kind == ROPE_LINEAR ? f / factor
                                            : f * (1 - ramp) + f / factor * ramp;
    }
    return kind == ROPE_YARN ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
}

extern "C" void qk_norm_rope_paged(bf16 *q_out, const bf16 *q, const bf16 *k, const bf16 *v,
                                   const bf16 *q_norm_w, const bf16 *k_norm_w,
                                   const double *inv_freq, const PagedBatch *batch, int n_tokens,
                                   int n_heads, int rotary_dim, int interleaved, float eps,
                                   float rope_scale, int64_t q_out_stride, int64_t q_stride,
                                   int64_t k_stride, int64_t v_stride, hipStream_t stream) {
    static const char name[] = "qk_norm_rope_paged";
    AppendArgs a;
    if (!take_batch(name, batch, n_tokens, n_heads, &a.b)) return;
    const int D = batch->head_dim;
    if (n_tokens == 0) return;
    if (rotary_dim < 16 || rotary_dim > D || rotary_dim % 16) {
        llm_fail("%s: rotary_dim %d is not a multiple of 16 up to head_dim %d", name, rotary_dim, D);
        return;
    }
    if (!inv_freq || ((uintptr_t)inv_freq & 7)) {
        llm_fail("%s: inv_freq must be an 8-byte aligned device address", name);
        return;
    }
    if (!aligned16(q_norm_w) || !aligned16(k_norm_w)) {
        llm_fail("%s: the norm weights must be 16-byte aligned", name);
        return;
    }
    const int64_t q_width = (int64_t)n_heads * D, kv_width = (int64_t)batch->n_kv_heads * D;
    if (!check_rows(name, "q_out", q_out, q_out_stride, q_width) ||
        !check_rows(name, "q", q, q_stride, q_width) || !check_rows(name, "k", k, k_stride, kv_width) ||
        !check_rows(name, "v", v, v_stride, kv_width))
        return;
    a.q_out = q_out;
    a.q = q;
    a.k = k;
    a.v = v;
    a.qn = q_norm_w;
    a.kn = k_norm_w;
    a.inv_freq = inv_freq;
    a.qo_stride = q_out_stride;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.n_heads = n_heads;
    a.n_kv_heads = batch->n_kv_heads;
    a.rotary = rotary_dim;
    a.interleaved = interleaved != 0;
    a.eps = eps;
    a.scale = rope_scale;
    const int hpw = 512 / D;
    a.q_groups = (n_heads + hpw - 1) / hpw;
    a.kv_groups = (batch->n_kv_heads + hpw - 1) / hpw;
    a.share = 1;
    a.waves_per_token = a.q_groups + 2 * a.kv_groups;
    const int64_t blocks = ((int64_t)n_tokens * a.waves_per_token + 3) / 4;
    if (blocks > INT32_MAX) {
        llm_fail("%s: %d rows of %d heads are too many for one launch", name, n_tokens, n_heads);
        return;
    }
    if (D == 64)
        append_kernel<64><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else if (D == 128)
        append_kernel<128><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else
        append_kernel<256><<<(unsigned)blocks, 256, 0, stream>>>(a);
    LAUNCH_OK();
}

// ------------------------------------------------------------------------------------------
// attention over pages
// ------------------------------------------------------------------------------------------

namespace {

struct AttendArgs {
    Batch b;
    bf16 *out;
    const bf16 *q;
    int64_t out_stride, q_stride;
    int n_heads, n_kv_heads, window;
    float scale;
};

// One wave per row and head, one key at a time with a running maximum and sum.
template <int D>
__global__ __launch_bounds__(256) void attend_rows_kernel(AttendArgs a) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * 4 + wave_id();
    const int t = (int)(wave / a.n_heads), h = (int)(wave - (int64_t)t * a.n_heads);
    if (t >= a.b.n_tokens) return;
    const int s = sequence_of(a.b, t);
    if (s < 0) return;
    const int pos = kv_length(a.b, s) - gptr(a.b.q_start)[s + 1] + t;
    const int kv = h / (a.n_heads / a.n_kv_heads);
    float q[E], acc[E], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        q[e] = bf2f(gptr(a.q)[t * a.q_stride + h * D + lane + 64 * e]);
        acc[e] = 0.0f;
    }
    for (int p = a.window > 0 ? max(0, pos - a.window + 1) : 0; p <= pos; p++) {
        const int64_t at = place(a.b, s, p);
        if (at < 0) continue;
        const bf16 *k = a.b.kc + at + kv * a.b.head_stride, *v = a.b.vc + at + kv * a.b.head_stride;
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) dot = fmaf(q[e], bf2f(gptr(k)[lane + 64 * e]), dot);
        const float x = wave_sum(dot) * a.scale;
        if (x == -INFINITY) continue;
        const float next = fmaxf(top, x);
        const float keep = exp_f32(top - next), weight = exp_f32(x - next);
        top = next;
        sum = sum * keep + weight;
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] = acc[e] * keep + weight * bf2f(gptr(v)[lane + 64 * e]);
    }
#pragma unroll
    for (int e = 0; e < E; e++)
        gptr(a.out)[t * a.out_stride + h * D + lane + 64 * e] =
            (bf16)f2bf(top == -INFINITY ? 0.0f : acc[e] / sum);
}

}  // namespace

extern "C" size_t attention_paged_workspace_floats(int n_tokens, int n_seqs, int n_heads,
                                                   int n_kv_heads, int head_dim, int max_q_len,
                                                   int max_kv_len) {
    (void)n_tokens, (void)n_seqs, (void)n_heads, (void)n_kv_heads, (void)head_dim, (void)max_q_len;
    (void)max_kv_len;
    return 0;
}

extern "C" void attention_paged_forward(bf16 *out, const bf16 *q, const PagedBatch *batch, float *ws,
                                        int n_tokens, int n_heads, int max_q_len, int max_kv_len,
                                        int window, float scale, int64_t out_stride,
                                        int64_t q_stride, hipStream_t stream) {
    static const char name[] = "attention_paged";
    AttendArgs a;
    if (!take_batch(name, batch, n_tokens, n_heads, &a.b)) return;
    if (n_tokens == 0) return;
    if (max_q_len <= 0 || max_kv_len <= 0) {
        llm_fail("%s: max_q_len %d and max_kv_len %d must be positive", name, max_q_len, max_kv_len);
        return;
    }
    if (window < 0) {
        llm_fail("%s: window %d is negative", name, window);
        return;
    }
    if (!(scale > 0.0f) || !isfinite(scale)) {
        llm_fail("%s: scale %g is not positive and finite", name, (double)scale);
        return;
    }
    const int64_t width = (int64_t)n_heads * batch->head_dim;
    if (!check_rows(name, "out", out, out_stride, width) || !check_rows(name, "q", q, q_stride, width))
        return;
    if (!aligned16(ws)) {
        llm_fail("%s: ws must be 16-byte aligned", name);
        return;
    }
    a.out = out;
    a.q = q;
    a.out_stride = out_stride;
    a.q_stride = q_stride;
    a.n_heads = n_heads;
    a.n_kv_heads = batch->n_kv_heads;
    a.window = window;
    a.scale = scale;
    const int64_t blocks = ((int64_t)n_tokens * n_heads + 3) / 4;
    if (batch->head_dim == 64)
        attend_rows_kernel<64><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else if (batch->head_dim == 128)
        attend_rows_kernel<128><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else
        attend_rows_kernel<256><<<(unsigned)blocks, 256, 0, stream>>>(a);
    LAUNCH_OK();
}
