// The next token of every row of logits by temperature, top-k, top-p and min-p (include/llm_amd/batch.h).
//
// bf16 logits have fewer than 2^16 values, so a row is counted by value, and everything after that is about
// values: weight and count of each, in the order of the values. Weights and sums are in 64 bits: a pick falls on
// the other side of a token's edge where the sums differ by more than what lies between u and the edge, and with
// sums in 32 bits that happened to one row in a few hundred.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "llm_amd/batch.h"

using namespace llm;

namespace {

struct SampleArgs {
    int *out;
    float *logprob;
    const bf16 *x;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *u;
    int vocab;
    int64_t x_stride;
};

constexpr int T = 1024, WAVES = T / 64;
constexpr int BINS = 1 << 16, CHUNK = 128, CHUNKS = BINS / CHUNK;
constexpr int MAX_VOCAB = 1 << 22, MOST_CARRIES = 128;  // over vocab / 2^16 + vocab / 2^32
constexpr int NONE = -1;

// The place of a value among the values, largest first, from its bits; NONE for what is never taken.
__device__ __forceinline__ int place_of(uint32_t b) {
    if ((b & 0x7fff) > 0x7f80 || b == 0xff80) return NONE;
    if (b == 0x8000) b = 0;
    return b & 0x8000 ? b : 0x7fff - b;
}
__device__ __forceinline__ float value_at(int place) {
    return bf2f((uint16_t)(place & 0x8000 ? place : 0x7fff - place));
}

struct Row {
    uint32_t counts[BINS / 2];   // n0 + 2^16 n1 of two values, modulo 2^32
    double mass[CHUNKS + 1];     // in front of each chunk of values
    int tokens[CHUNKS + 1];
    int carries;                 // how often a sum passed what it is held in:
    uint32_t carry[MOST_CARRIES];  // 2 w: n0 of word w passed a multiple of 2^16, 2 w + 1: the word one of 2^32
    int found[WAVES];
    int answer;
};

// f(index, bits) for the logits from `first` to `last` (a thread's eight at a time from aligned addresses on)
template <class F>
__device__ __forceinline__ void each_logit(const bf16 *x, int first, int last, F f) {
    const int head = min(last, first + (int)((16 - ((uintptr_t)(x + first) & 15)) / 2 & 7));
    const int body = head + (last - head) / 8 * 8;
    if (first + (int)threadIdx.x < head) f(first + threadIdx.x, (uint32_t)gptr(x)[first + threadIdx.x]);
    for (int i = head + 8 * threadIdx.x; i < body; i += 8 * T) {
        const u32x4 v = ld16(x + i);
#pragma unroll
        for (int e = 0; e < 8; e++) f(i + e, v[e / 2] >> (e % 2 * 16) & 0xffff);
    }
    if (body + (int)threadIdx.x < last) f(body + threadIdx.x, (uint32_t)gptr(x)[body + threadIdx.x]);
}

__device__ __forceinline__ void carried(Row &row, uint32_t what) {
    row.carry[atomicAdd(&row.carries, 1) & (MOST_CARRIES - 1)] = what;
}
__device__ __forceinline__ void count(Row &row, int place, uint32_t n) {
    const uint32_t w = place / 2, more = n << (place % 2 * 16), old = atomicAdd(&row.counts[w], more);
    if (place % 2 == 0 && (old & 0xffff) + n > 0xffff) carried(row, 2 * w);
    if (old + more < old) carried(row, 2 * w + 1);
}

// Counts of the two values of word w.
__device__ __forceinline__ void counts_of(const Row &row, uint32_t w, int &first, int &second) {
    int64_t word = row.counts[w];
    first = (int)(word & 0xffff);
    for (int i = 0; i < row.carries; i++) {
        if (row.carry[i] == 2 * w) first += 1 << 16;
        if (row.carry[i] == 2 * w + 1) word += 1ll << 32;
    }
    second = (int)((word - first) >> 16);
}

struct Scale {
    double top, by;  // the largest value, 1 / temperature
    __device__ __forceinline__ double weight(int place) const {
        const double x = (double)value_at(place);
        return x == top ? 1.0 : top > 3.5e38 ? 0.0 : exp((x - top) * by);  // beside +inf nothing else weighs
    }
};

// Within a chunk: this lane's two values, and mass and tokens in front of them.
struct Lane {
    double w0, w1, before;
    int n0, n1, tokens;
};
__device__ __forceinline__ Lane lane_of(const Row &row, const Scale &s, int chunk) {
    Lane l;
    const int lane = threadIdx.x & 63, word = chunk * 64 + lane;
    counts_of(row, word, l.n0, l.n1);
    l.w0 = l.n0 ? s.weight(2 * word) : 0.0;
    l.w1 = l.n1 ? s.weight(2 * word + 1) : 0.0;
    const double own = l.n0 * l.w0 + l.n1 * l.w1;
    const int tokens = l.n0 + l.n1;
    double upto = own;
    int n = tokens;
    for (int d = 1; d < 64; d *= 2) {
        const double a = __shfl_up(upto, d);
        const int b = __shfl_up(n, d);
        if (lane >= d) upto += a, n += b;
    }
    l.before = row.mass[chunk] + __shfl_up(upto, 1);
    if (lane == 0) l.before = row.mass[chunk];
    l.tokens = row.tokens[chunk] + n - tokens;
    return l;
}

// The last chunk whose front value is at most `at` (there is one: chunk 0's is 0).
template <class V>
__device__ __forceinline__ int chunk_at(const V *front, V at) {
    int lo = 0, hi = CHUNKS;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (front[mid] <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Mass of the first n tokens.
__device__ __forceinline__ double mass_of(const Row &row, const Scale &s, int n) {
    if (n >= row.tokens[CHUNKS]) return row.mass[CHUNKS];
    const Lane l = lane_of(row, s, chunk_at(row.tokens, n));
    const int last = __popcll(__ballot(l.tokens <= n)) - 1;
    const int a = min(l.n0, n - l.tokens), b = n - l.tokens - a;
    return __shfl(l.before + (a * l.w0 + b * l.w1), last);
}

// The number of leading tokens whose mass is not past `at`: strictly less (PAST false) or at most `at`.
template <bool EQUAL>
__device__ __forceinline__ int tokens_within(const Row &row, const Scale &s, double at) {
    int lo = 0, hi = CHUNKS;  // the last chunk with its front within
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (EQUAL ? row.mass[mid] <= at : row.mass[mid] < at) lo = mid;
        else hi = mid;
    }
    const Lane l = lane_of(row, s, lo);
    const auto fits = [&](double m) { return EQUAL ? m <= at : m < at; };
    // how many of n tokens of weight w fit behind m
    const auto part = [&](double m, double w, int n) {
        if (n == 0 || !fits(m)) return 0;
        int k = w > 0 ? (int)fmin(fmax((at - m) / w, 0.0), (double)n) : n;
        if (k > 0 && !fits(m + k * w)) k--;
        if (k < n && fits(m + (k + 1) * w)) k++;
        return k;
    };
    int mine = part(l.before, l.w0, l.n0);
    if (mine == l.n0) mine += part(l.before + l.n0 * l.w0, l.w1, l.n1);
    for (int d = 1; d < 64; d *= 2) mine += __shfl_xor(mine, d);
    return row.tokens[lo] + mine;
}

__global__ __launch_bounds__(T) void sample_kernel(SampleArgs a) {
    __shared__ Row row;
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = wave_id();
    const bf16 *x = a.x + r * a.x_stride;
    for (int i = threadIdx.x; i < BINS / 2 / 4; i += T) ((u32x4 *)row.counts)[i] = u32x4{0, 0, 0, 0};
    if (threadIdx.x == 0) row.carries = 0;
    __syncthreads();
    int least = BINS;  // the place of the largest value
    each_logit(x, 0, a.vocab, [&](int, uint32_t b) {
        const int p = place_of(b);
        if (p == NONE) return;
        least = min(least, p);
        count(row, p, 1);
    });
    for (int d = 1; d < 64; d *= 2) least = min(least, __shfl_xor(least, d));
    if (lane == 0) row.found[wave] = least;
    __syncthreads();
    for (int i = 0; i < WAVES; i++) least = min(least, row.found[i]);
    if (least == BINS) {
        if (threadIdx.x == 0) {
            a.out[r] = -1;
            if (a.logprob) a.logprob[r] = -INFINITY;
        }
        return;
    }
    const float temperature = a.temperature ? gptr(a.temperature)[r] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    const Scale s = {(double)value_at(least), 1.0 / (double)temperature};
    int place = least, nth = 0;
    double logprob = 0.0;
    if (!greedy) {
        for (int c = wave; c < CHUNKS; c += WAVES) {
            int n0, n1;
            counts_of(row, c * 64 + lane, n0, n1);
            double m = 0;
            if (n0) m += n0 * s.weight(2 * (c * 64 + lane));
            if (n1) m += n1 * s.weight(2 * (c * 64 + lane) + 1);
            int n = n0 + n1;
            for (int d = 1; d < 64; d *= 2) m += __shfl_xor(m, d), n += __shfl_xor(n, d);
            if (lane == 0) row.mass[c] = m, row.tokens[c] = n;
        }
        __syncthreads();
        if (wave == 0) {  // what lies in front of each chunk, eight chunks per lane
            constexpr int EACH = CHUNKS / 64;
            double m = 0, own[EACH];
            int n = 0, tokens[EACH];
            for (int i = 0; i < EACH; i++) {
                m += own[i] = row.mass[lane * EACH + i];
                n += tokens[i] = row.tokens[lane * EACH + i];
            }
            double m_upto = m;
            int n_upto = n;
            for (int d = 1; d < 64; d *= 2) {
                const double a = __shfl_up(m_upto, d);
                const int b = __shfl_up(n_upto, d);
                if (lane >= d) m_upto += a, n_upto += b;
            }
            m = __shfl_up(m_upto, 1);
            n = n_upto - n;
            if (lane == 0) m = 0;
            for (int i = 0; i < EACH; i++) {
                row.mass[lane * EACH + i] = m;
                row.tokens[lane * EACH + i] = n;
                m += own[i];
                n += tokens[i];
            }
            if (lane == 63) row.mass[CHUNKS] = m, row.tokens[CHUNKS] = n;
        }
        __syncthreads();
        int left = row.tokens[CHUNKS];
        double total = row.mass[CHUNKS];
        const int k = a.top_k ? gptr(a.top_k)[r] : 0;
        if (k > 0 && k < left) {
            left = k;
            total = mass_of(row, s, left);
        }
        const float p = a.top_p ? gptr(a.top_p)[r] : 1.0f;
        if (p < 1.0f) {  // those in front of the one that reaches p, and that one
            left = min(left, tokens_within<false>(row, s, (double)p * total) + 1);
            total = mass_of(row, s, left);
        }
        const float min_p = a.min_p ? gptr(a.min_p)[r] : 0.0f;
        if (min_p > 0.0f) {
            // the first place of less weight, by halves: weights do not grow along the places
            int lo = least, hi = 0xff7f + 1;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (s.weight(mid) >= (double)min_p) lo = mid;
                else hi = mid;
            }
            const Lane l = lane_of(row, s, lo / CHUNK);
            int fit = l.tokens + l.n0 + (lo % 2 ? l.n1 : 0);
            fit = max(1, __shfl(fit, lo % CHUNK / 2));
            if ((double)min_p > 1.0) fit = 1;
            if (fit < left) {
                left = fit;
                total = mass_of(row, s, left);
            }
        }
        const float u = gptr(a.u)[r];
        int rank = u != u ? 0 : min(left - 1, tokens_within<true>(row, s, (double)u * total));
        // back to the last one of positive weight
        rank = max(0, min(rank, tokens_within<false>(row, s, total)));
        const Lane l = lane_of(row, s, chunk_at(row.tokens, rank));
        const int at = __popcll(__ballot(l.tokens <= rank)) - 1;
        int mine = rank - l.tokens, which = 2 * (chunk_at(row.tokens, rank) * 64 + lane);
        double w = l.w0;
        if (mine >= l.n0) mine -= l.n0, which++, w = l.w1;
        place = __shfl(which, at);
        nth = __shfl(mine, at);
        logprob = log(__shfl(w, at) / total);
    }
    // the nth of the tokens with that value: each wave counts its part of the row, then one looks through its own
    const uint32_t bits = __float_as_uint(value_at(place)) >> 16;
    const auto same = [&](uint32_t b) { return b == bits || (bits == 0 && b == 0x8000); };
    const int part = (a.vocab + WAVES - 1) / WAVES, first = min(a.vocab, wave * part), last = min(a.vocab, first + part);
    int met = 0;
    for (int i = first; i < last; i += 64)
        met += __popcll(__ballot(i + lane < last && same(gptr(x)[min(i + lane, a.vocab - 1)])));
    __syncthreads();
    if (lane == 0) row.found[wave] = met;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < wave; i++) before += row.found[i];
    if (nth < before || nth >= before + met) return;
    nth -= before;
    for (int i = first; i < last; i += 64) {
        const uint64_t here = __ballot(i + lane < last && same(gptr(x)[min(i + lane, a.vocab - 1)]));
        const int n = __popcll(here);
        if (nth < n) {
            const bool mine = here >> lane & 1 && __popcll(here & ((1ull << lane) - 1)) == nth;
            if (mine) {
                a.out[r] = i + lane;
                if (a.logprob) a.logprob[r] = (float)logprob;
            }
            return;
        }
        nth -= n;
    }
}

constexpr int SPLIT_VOCAB = 16384, SPLIT_ROWS = 128;

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

bool check_sizes(const char *name, int rows, int vocab) {
    if (rows < 0 || rows > 1 << 20) return llm_fail("%s: rows %d is not in 0..1048576", name, rows);
    if (vocab <= 0 || vocab > MAX_VOCAB) return llm_fail("%s: vocab %d is not in 1..%d", name, vocab, MAX_VOCAB);
    return true;
}

}  // namespace

extern "C" size_t sample_rows_workspace_floats(int rows, int vocab) {
    if (!check_sizes("sample_rows_workspace_floats", rows, vocab) || vocab < SPLIT_VOCAB) return 0;
    return (size_t)std::min(rows, SPLIT_ROWS) * (vocab + 64);
}

extern "C" void sample_rows_forward(int *out, float *logprob, const bf16 *logits, const float *temperature,
                                    const int *top_k, const float *top_p, const float *min_p, const float *u,
                                    float *ws, int rows, int vocab, int64_t logits_stride, hipStream_t stream) {
    static const char name[] = "sample_rows";
    if (!check_sizes(name, rows, vocab) || rows == 0) return;
    if (!out || !logits || !u) {
        llm_fail("%s: out, logits and u must not be null", name);
        return;
    }
    if (logits_stride < vocab) {
        llm_fail("%s: rows %lld elements apart overlap (vocab %d)", name, (long long)logits_stride, vocab);
        return;
    }
    if (!aligned16(ws) || (sample_rows_workspace_floats(rows, vocab) && !ws)) {
        llm_fail("%s: ws must be a 16-byte aligned device address", name);
        return;
    }
    const SampleArgs a = {out, logprob, logits, temperature, top_k, top_p, min_p, u, vocab, logits_stride};
    sample_kernel<<<rows, T, 0, stream>>>(a);
    LAUNCH_OK();
}
