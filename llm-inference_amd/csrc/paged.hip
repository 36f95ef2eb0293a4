// QK-norm + RoPE that writes new keys and values into pages (include/llm_amd/paged.h).
#include <math.h>
#include <string.h>

#include "paged_batch.h"

using namespace llm;

namespace {

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
// the pair's elements. The norm's sum and everything after it stay in 32 bits up to the one rounding. Bound by the
// rows' bytes where there are many (3402 rows of 48 heads of 128: 20.4 us, 4.1 TB/s; a 2 GiB copy: 4.8), by
// three dependent lookups (sequence, its lengths, the page) and the launch where there are few (1 to 64 rows: 4.7 us).
template <int D>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    constexpr int LH = D / 8, HPW = 64 / LH;
    __shared__ __align__(16) float2 turn[4][D / 2];
    const int lane = threadIdx.x & 63, w = wave_id();
    const int64_t wave = (int64_t)blockIdx.x * 4 + w;
    const int t = (int)(wave / a.waves_per_token);
    if (t >= a.b.n_tokens) return;
    const int part = (int)(wave - (int64_t)t * a.waves_per_token);
    const int L = lane % LH, hg = lane / LH;
    const int groups = a.q_groups + 2 * a.kv_groups, last = min(groups, (part + 1) * a.share);
    // the lane's 16 bytes of its head of group g (of q, then k, then v)
    const auto request = [&](int g) {
        const bool is_q = g < a.q_groups, is_v = g >= a.q_groups + a.kv_groups;
        const int h = (is_q ? g : is_v ? g - a.q_groups - a.kv_groups : g - a.q_groups) * HPW + hg;
        const bf16 *src = is_q ? a.q + t * a.q_stride : is_v ? a.v + t * a.v_stride : a.k + t * a.k_stride;
        u32x4 x = {0, 0, 0, 0};
        if (h < (is_q ? a.n_heads : a.n_kv_heads)) x = ld16_nt(src + h * D + 8 * L);
        return x;
    };
    u32x4 ahead = request(part * a.share);
    const u32x4 wq = a.qn ? ld16(a.qn + 8 * L) : u32x4{0, 0, 0, 0}, wk = a.kn ? ld16(a.kn + 8 * L) : u32x4{0, 0, 0, 0};
    const int s = sequence_of(a.b, t);
    if (s < 0) return;
    const int pos = kv_length(a.b, s) - min(a.b.n_tokens, gptr(a.b.q_start)[s + 1]) + t;
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
    for (int g = part * a.share; g < last; g++) {
        const bool is_q = g < a.q_groups, is_v = g >= a.q_groups + a.kv_groups;
        const int h = (is_q ? g : is_v ? g - a.q_groups - a.kv_groups : g - a.q_groups) * HPW + hg;
        const bool there = h < (is_q ? a.n_heads : a.n_kv_heads) && (is_q || at >= 0);
        const u32x4 x = ahead;
        if (g + 1 < last) ahead = request(g + 1);
        if (is_v) {
            if (there) st16(a.b.vc + at + h * a.b.head_stride + 8 * L, x);
            continue;
        }
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = elem(x, e);
        if (is_q ? a.qn != nullptr : a.kn != nullptr) {
            const float inv = 1.0f / sqrtf(group_sum<LH>(dot8(x, x, 0.0f)) / (float)D + a.eps);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = y[e] * inv * elem(is_q ? wq : wk, e);
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
    if (rotary_dim <= 0 || rotary_dim % 2) {
        llm_fail("rope_frequencies: rotary_dim %d is not a positive even number", rotary_dim);
        return 0.0f;
    }
    if (!inv_freq) {
        llm_fail("rope_frequencies: inv_freq is null");
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
        if (pair_that_turns(1) <= 0)
            low = -1, high = 0;  // none turns once: all are divided
        else if (high <= low)
            high = low + 0.001;  // all turn more than 32 times
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
    if (q_out == q && q_out_stride != q_stride) {
        llm_fail("%s: in place, the rows of q_out and q must be the same", name);
        return;
    }
    // what is written must not lie on itself (as expanded tensors do)
    if ((batch->n_kv_heads > 1 && batch->head_stride < D) || (batch->n_pages > 1 && batch->page_stride < D)) {
        llm_fail("%s: pages %lld and kv heads %lld elements apart overlap (head_dim %d)", name,
                 (long long)batch->page_stride, (long long)batch->head_stride, D);
        return;
    }
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
    const int groups = a.q_groups + 2 * a.kv_groups;
    // about 6144 waves (24 to a CU), as far as the rows go: with fewer a wave's loads wait too long for each
    // other, with more the angles are computed too often (3402 rows of 48 heads of 128: one group of heads per
    // wave 36.8 us, 3 23.8, 6 20.6, 12 23.9; 411 rows: one 6.8, two 6.9, six 9.5)
    a.share = (int)std::min<int64_t>(groups, std::max<int64_t>(1, (int64_t)n_tokens * groups / 6144));
    a.waves_per_token = (groups + a.share - 1) / a.share;
    // at most n_tokens + 12288 waves, so within one launch's 2^32 threads
    const int64_t blocks = ((int64_t)n_tokens * a.waves_per_token + 3) / 4;
    if (D == 64)
        append_kernel<64><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else if (D == 128)
        append_kernel<128><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else
        append_kernel<256><<<(unsigned)blocks, 256, 0, stream>>>(a);
    LAUNCH_OK();
}
