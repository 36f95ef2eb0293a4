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
    int *entries;       // [rows, slices]: how many values each slice of a row has
    uint32_t *lists;    // [rows, slices, slice]: these, place << 16 | count
    int slices, slice;  // of a row (1: none), tokens of each but the last
};

constexpr int T = 1024, WAVES = T / 64;
constexpr int BINS = 1 << 16, CHUNK = 128, CHUNKS = BINS / CHUNK;
constexpr int MAX_VOCAB = 1 << 22, MOST_CARRIES = 128;  // over vocab / 2^16 + vocab / 2^32
constexpr int NONE = -1, MOST_SLICES = 8, MOST_SLICE = 65528;  // a multiple of 8 that 16 bits count

// The place of a value among the values, largest first, from its bits; NONE for what is never taken.
__device__ __forceinline__ int place_of(uint32_t b) {
    if ((b & 0x7fff) > 0x7f80 || b == 0xff80) return NONE;
    if (b == 0x8000) b = 0;
    return b & 0x8000 ? b : 0x7fff - b;
}
__device__ __forceinline__ uint32_t bits_at(int place) { return place & 0x8000 ? place : 0x7fff - place; }

struct Row {
    uint32_t counts[BINS / 2];   // n0 + 2^16 n1 of two values, modulo 2^32
    double mass[CHUNKS + 1];     // in front of each chunk of values
    int tokens[CHUNKS + 1];
    int carries;                 // how often a sum passed what it is held in:
    uint32_t carry[MOST_CARRIES];  // 2 w: n0 of word w passed a multiple of 2^16, 2 w + 1: the word one of 2^32
    int found[WAVES];
    int entries;
};

__device__ __forceinline__ void clear(Row &row) {
    for (int i = threadIdx.x; i < BINS / 2 / 4; i += T) ((u32x4 *)row.counts)[i] = u32x4{0, 0, 0, 0};
    if (threadIdx.x == 0) row.carries = row.entries = 0;
    __syncthreads();
}

// CARRY: there may be more tokens than 16 bits count.
template <bool CARRY>
__device__ __forceinline__ void count(Row &row, int place, uint32_t n) {
    const uint32_t w = place / 2, more = n << (place % 2 * 16);
    if constexpr (CARRY) {
        const uint32_t old = atomicAdd(&row.counts[w], more);
        const bool first = place % 2 == 0 && (old & 0xffff) + n > 0xffff, word = old + more < old;
        if (first || word) {
            if (first) row.carry[atomicAdd(&row.carries, 1) & (MOST_CARRIES - 1)] = 2 * w;
            if (word) row.carry[atomicAdd(&row.carries, 1) & (MOST_CARRIES - 1)] = 2 * w + 1;
        }
    } else {
        atomicAdd(&row.counts[w], more);
    }
}

// Counts of the two values of word w, whose sum modulo 2^32 is `word`.
__device__ __forceinline__ void counts_of(const Row &row, int carries, uint32_t w, uint32_t word, int &first, int &second) {
    int64_t whole = word;
    first = (int)(whole & 0xffff);
    for (int i = 0; i < carries; i++) {
        if (row.carry[i] == 2 * w) first += 1 << 16;
        if (row.carry[i] == 2 * w + 1) whole += 1ll << 32;
    }
    second = (int)((whole - first) >> 16);
}

// f(index, bits) for the logits from `first` to `last`, eight per thread at a time from aligned addresses on, four
// times under way.
template <class F>
__device__ __forceinline__ void each_logit(const bf16 *x, int first, int last, F f) {
    constexpr int U = 4;
    const int head = min(last, first + (int)((16 - ((uintptr_t)(x + first) & 15)) / 2 & 7));
    const int body = head + (last - head) / 8 * 8;
    for (int i0 = head + 8 * (int)threadIdx.x; i0 < body; i0 += U * 8 * T) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i0 + u * 8 * T < body) v[u] = ld16(x + i0 + u * 8 * T);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i0 + u * 8 * T < body) {
#pragma unroll
                for (int e = 0; e < 8; e++) f(i0 + u * 8 * T + e, v[u][e / 2] >> (e % 2 * 16) & 0xffff);
            }
    }
    if (first + (int)threadIdx.x < head) f(first + threadIdx.x, (uint32_t)gptr(x)[first + threadIdx.x]);
    if (body + (int)threadIdx.x < last) f(body + threadIdx.x, (uint32_t)gptr(x)[body + threadIdx.x]);
}

template <int S>
__device__ __forceinline__ double xor_lane(double v) {
    return __hiloint2double(llm::xor_lane<S>(__double2hiint(v)), llm::xor_lane<S>(__double2loint(v)));
}
__device__ __forceinline__ double sum_lanes(double v) {
    v += xor_lane<1>(v), v += xor_lane<2>(v), v += xor_lane<4>(v), v += xor_lane<8>(v), v += xor_lane<16>(v);
    return v + xor_lane<32>(v);
}
__device__ __forceinline__ int sum_lanes(int v) {
    v += llm::xor_lane<1>(v), v += llm::xor_lane<2>(v), v += llm::xor_lane<4>(v), v += llm::xor_lane<8>(v), v += llm::xor_lane<16>(v);
    return v + llm::xor_lane<32>(v);
}
// Sums of the lanes in front of this one.
__device__ __forceinline__ void sum_before(double &v, int &n) {
    const int lane = threadIdx.x & 63;
    const int tokens = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double a = __shfl_up(v, d);
        const int b = __shfl_up(n, d);
        if (lane >= d) v += a, n += b;
    }
    v = __shfl_up(v, 1);  // not less its own, which would round
    if (lane == 0) v = 0.0;
    n -= tokens;
}

// The draw from a row's counts, by every wave alike.
struct Draw {
    const Row &row;
    int carries;
    double top, by;  // the largest value, 1 / temperature

    __device__ __forceinline__ double weight(int place) const {
        const double x = (double)__uint_as_float(bits_at(place) << 16);
        // beside +inf nothing else weighs
        return x == top ? 1.0 : top > 3.5e38 ? 0.0 : exp((x - top) * by);
    }

    // A chunk's values, two per lane, with mass and tokens in front of them.
    struct Lane {
        double w0, w1, before;
        int n0, n1, tokens;
    };
    __device__ __forceinline__ Lane lane_of(int chunk) const {
        Lane l;
        const int word = chunk * 64 + (threadIdx.x & 63);
        counts_of(row, carries, word, row.counts[word], l.n0, l.n1);
        l.w0 = l.n0 ? weight(2 * word) : 0.0;
        l.w1 = l.n1 ? weight(2 * word + 1) : 0.0;
        l.before = l.n0 * l.w0 + l.n1 * l.w1;
        l.tokens = l.n0 + l.n1;
        sum_before(l.before, l.tokens);
        l.before += row.mass[chunk];
        l.tokens += row.tokens[chunk];
        return l;
    }

    // The last chunk whose front passes `fits` (which the fronts stop doing, and the first does).
    template <class V, class Fits>
    __device__ __forceinline__ int chunk_at(const V *front, Fits fits) const {
        const int lane = threadIdx.x & 63, group = max(0, __popcll(__ballot(fits(front[lane * 8]))) - 1);
        return group * 8 + max(0, __popcll(__ballot(lane < 8 && fits(front[group * 8 + (lane & 7)]))) - 1);
    }

    // A place in the order of the tokens: so many in front of it and their mass; the value of the token there, how
    // many of that value are in front of it, and its weight.
    struct Spot {
        int tokens, place, nth;
        double mass, weight;
    };
    // Of this lane's two values, k0 and k1 tokens are in front of the spot: the lane where that stops.
    __device__ __forceinline__ Spot spot(int chunk, const Lane &l, int k0, int k1) const {
        const uint64_t stops = __ballot(k0 + k1 < l.n0 + l.n1);
        const int at = stops ? __builtin_ctzll(stops) : 63, lane = threadIdx.x & 63;
        const bool second = k0 == l.n0;
        Spot s = {l.tokens + k0 + k1, 2 * (chunk * 64 + lane) + (second ? 1 : 0), second ? k1 : k0,
                  l.before + (k0 * l.w0 + k1 * l.w1), second ? l.w1 : l.w0};
        s.tokens = __shfl(s.tokens, at);
        s.place = __shfl(s.place, at);
        s.nth = __shfl(s.nth, at);
        s.mass = __shfl(s.mass, at);
        s.weight = __shfl(s.weight, at);
        return s;
    }
    // The spot behind n tokens.
    __device__ __forceinline__ Spot behind(int n) const {
        const int chunk = chunk_at(row.tokens, [&](int t) { return t <= n; });
        const Lane l = lane_of(chunk);
        const int k0 = max(0, min(l.n0, n - l.tokens));
        return spot(chunk, l, k0, max(0, min(l.n1, n - l.tokens - l.n0)));
    }
    // The spot behind the last token up to which the mass is less than `at` (EQUAL: not more).
    template <bool EQUAL>
    __device__ __forceinline__ Spot within(double at) const {
        const auto fits = [&](double m) { return EQUAL ? m <= at : m < at; };
        const int chunk = chunk_at(row.mass, fits);
        const Lane l = lane_of(chunk);
        // how many of n tokens of weight w fit behind m
        const auto part = [&](double m, double w, int n) {
            if (n == 0 || !fits(m)) return 0;
            int k = w > 0 ? (int)fmin(fmax((at - m) / w, 0.0), (double)n) : n;
            if (k > 0 && !fits(m + k * w)) k--;
            if (k < n && fits(m + (k + 1) * w)) k++;
            return k;
        };
        const int k0 = part(l.before, l.w0, l.n0), k1 = k0 < l.n0 ? 0 : part(l.before + l.n0 * l.w0, l.w1, l.n1);
        // all of the chunk, where its sum falls short of the next one's front by a rounding, or it is empty
        if (!__any(k0 + k1 < l.n0 + l.n1)) return behind(row.tokens[chunk + 1]);
        return spot(chunk, l, k0, k1);
    }
};

// The smallest of the threads' places, in every thread (two barriers, with what is in LDS before them).
__device__ __forceinline__ int least_of(Row &row, int least) {
    for (int d = 1; d < 64; d *= 2) least = min(least, __shfl_xor(least, d));
    if ((threadIdx.x & 63) == 0) row.found[wave_id()] = least;
    __syncthreads();
    least = row.found[threadIdx.x % WAVES];
    for (int d = 1; d < WAVES; d *= 2) least = min(least, __shfl_xor(least, d));
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(least);
}

// Row r's token from its counts. least: the place of the largest value (BINS: none). where(place, nth, first, last)
// says among which tokens the nth of that value is, and leaves in nth how many of it are in front of it there.
template <class Where>
__device__ __forceinline__ void draw(const SampleArgs &a, Row &row, int r, int least, Where where) {
    const int lane = threadIdx.x & 63, wave = wave_id();
    if (least == BINS) {
        if (threadIdx.x == 0) {
            a.out[r] = -1;
            if (a.logprob) a.logprob[r] = -INFINITY;
        }
        return;
    }
    const float temperature = a.temperature ? gptr(a.temperature)[r] : 1.0f;
    const int top_k = a.top_k ? gptr(a.top_k)[r] : 0;
    const float top_p = a.top_p ? gptr(a.top_p)[r] : 1.0f, min_p = a.min_p ? gptr(a.min_p)[r] : 0.0f, u = gptr(a.u)[r];
    const int carries = row.carries;
    const Draw d = {row, carries, (double)__uint_as_float(bits_at(least) << 16), 1.0 / (double)temperature};
    int place = least, nth = 0;
    double logprob = 0.0;
    if (temperature > 0.0f) {
        constexpr int EACH = CHUNKS / WAVES;  // chunks of a wave, every WAVES-th one
        uint32_t words[EACH];
#pragma unroll
        for (int i = 0; i < EACH; i++) words[i] = row.counts[(i * WAVES + wave) * 64 + lane];
#pragma unroll
        for (int i = 0; i < EACH; i++) {
            const int chunk = i * WAVES + wave;
            double m = 0.0;
            int n = 0;
            if (__any(words[i] != 0) || carries) {
                int n0, n1;
                counts_of(row, carries, chunk * 64 + lane, words[i], n0, n1);
                if (n0) m = n0 * d.weight(2 * (chunk * 64 + lane));
                if (n1) m += n1 * d.weight(2 * (chunk * 64 + lane) + 1);
                m = sum_lanes(m);
                n = sum_lanes(n0 + n1);
            }
            if (lane == 0) row.mass[chunk] = m, row.tokens[chunk] = n;
        }
        __syncthreads();
        if (wave == 0) {  // what lies in front of each chunk, eight chunks per lane
            constexpr int EIGHT = CHUNKS / 64;
            double before = 0.0, own[EIGHT];
            int n = 0, tokens[EIGHT];
#pragma unroll
            for (int i = 0; i < EIGHT; i++) {
                before += own[i] = row.mass[lane * EIGHT + i];
                n += tokens[i] = row.tokens[lane * EIGHT + i];
            }
            sum_before(before, n);
#pragma unroll
            for (int i = 0; i < EIGHT; i++) {
                row.mass[lane * EIGHT + i] = before;
                row.tokens[lane * EIGHT + i] = n;
                before += own[i];
                n += tokens[i];
            }
            if (lane == 63) row.mass[CHUNKS] = before, row.tokens[CHUNKS] = n;
        }
        __syncthreads();
        int left = row.tokens[CHUNKS];
        double total = row.mass[CHUNKS];
        if (top_k > 0 && top_k < left) {
            left = top_k;
            total = d.behind(left).mass;
        }
        if (top_p < 1.0f) {  // those in front of the one that reaches p, and that one
            const Draw::Spot s = d.template within<false>((double)top_p * total);
            if (s.tokens + 1 < left) {
                left = s.tokens + 1;
                total = s.mass + s.weight;
            }
        }
        if (min_p > 0.0f) {
            // the last place of enough weight, by 64ths and then one by one of what is left: weights do not grow
            // along the places
            int lo = least, hi = 0xff7f + 1;
            while (hi - lo > 1) {
                const int step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
                const int fit = __popcll(__ballot(at < hi && d.weight(at) >= (double)min_p));
                hi = min(hi, lo + (fit + 1) * step);
                lo += fit * step;
            }
            const int chunk = lo / CHUNK;
            const Draw::Lane l = d.lane_of(chunk);
            const int k0 = lane < lo % CHUNK / 2 || 2 * lane == lo % CHUNK || 2 * lane + 1 == lo % CHUNK ? l.n0 : 0;
            const int k1 = lane < lo % CHUNK / 2 || 2 * lane + 1 == lo % CHUNK ? l.n1 : 0;
            const Draw::Spot s = d.spot(chunk, l, k0, k1);
            const bool one = min_p > 1.0f;  // more than the first one weighs
            if (one || s.tokens < left) {
                left = one ? 1 : s.tokens;
                total = one ? 1.0 : s.mass;
            }
        }
        const double at = (double)u * total;
        Draw::Spot s = u != u ? d.behind(0) : d.template within<true>(at);
        // past the last one: to that; or to the last one of positive weight
        if (s.tokens >= left) s = d.behind(left - 1);
        if (!(at < total) && u == u) {
            const Draw::Spot last = d.template within<false>(total);
            if (last.tokens < s.tokens) s = last;
        }
        place = s.place;
        nth = s.nth;
        logprob = log(s.weight / total);
    }
    int first, last;
    where(place, nth, first, last);
    // each wave counts the value in its part of these tokens, then one looks through its own
    const uint32_t bits = bits_at(place);
    const auto same = [&](uint32_t b) { return b == bits || (bits == 0 && b == 0x8000); };
    const bf16 *x = a.x + r * a.x_stride;
    // parts of whole 512 tokens from an aligned address on
    const int begin = first - (int)((uintptr_t)(x + first) % 16 / 2), part = (last - begin + 512 * WAVES - 1) / (512 * WAVES) * 512;
    const auto request = [&](int i) {  // eight tokens from i on, as a mask of those of the value
        uint32_t mask = 0;
        if (i >= first && i + 8 <= last) {
            const u32x4 v = ld16(x + i);
#pragma unroll
            for (int e = 0; e < 8; e++) mask |= same(v[e / 2] >> (e % 2 * 16) & 0xffff) ? 1u << e : 0;
        } else {
            for (int e = 0; e < 8; e++)
                if (i + e >= first && i + e < last && same(gptr(x)[i + e])) mask |= 1u << e;
        }
        return mask;
    };
    const int mine = begin + wave * part, end = min(last, mine + part);
    int met = 0;
#pragma unroll 4
    for (int i = mine; i < end; i += 512) met += __popc(request(i + 8 * lane));
    met = sum_lanes(met);
    __syncthreads();
    if (lane == 0) row.found[wave] = met;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < wave; i++) before += row.found[i];
    if (nth < before || nth >= before + met) return;
    nth -= before;
    for (int i = mine; i < end; i += 512) {
        const uint32_t mask = request(i + 8 * lane);
        int upto = __popc(mask);
        const int own = upto;
#pragma unroll
        for (int k = 1; k < 64; k *= 2) {
            const int v = __shfl_up(upto, k);
            if (lane >= k) upto += v;
        }
        const int all = __shfl(upto, 63);
        if (nth < all) {
            int rest = nth - (upto - own);
            if (rest < 0 || rest >= own) return;
            for (int e = 0; e < 8; e++)
                if (mask >> e & 1 && rest-- == 0) {
                    a.out[r] = i + 8 * lane + e;
                    if (a.logprob) a.logprob[r] = (float)logprob;
                }
            return;
        }
        nth -= all;
    }
}

// One workgroup per row.
template <bool CARRY>
__global__ __launch_bounds__(T) void sample_kernel(SampleArgs a) {
    __shared__ Row row;
    const int r = blockIdx.x;
    clear(row);
    int least = BINS;
    each_logit(a.x + r * a.x_stride, 0, a.vocab, [&](int, uint32_t b) {
        const int p = place_of(b);
        if (p == NONE) return;
        least = min(least, p);
        count<CARRY>(row, p, 1);
    });
    least = least_of(row, least);
    draw(a, row, r, least, [&](int, int &, int &first, int &last) { first = 0, last = a.vocab; });
}

// A slice of a row: its values and their counts as a list.
__global__ __launch_bounds__(T) void slice_kernel(SampleArgs a) {
    __shared__ Row row;
    const int r = blockIdx.y, lane = threadIdx.x & 63, wave = wave_id();
    const int first = blockIdx.x * a.slice, last = min(a.vocab, first + a.slice);
    clear(row);
    each_logit(a.x + r * a.x_stride, first, last, [&](int, uint32_t b) {
        const int p = place_of(b);
        if (p != NONE) count<false>(row, p, 1);  // a slice has less than 2^16 tokens
    });
    __syncthreads();
    const int at = r * a.slices + blockIdx.x;
    uint32_t *list = a.lists + (int64_t)at * a.slice;
    constexpr int EACH = CHUNKS / WAVES;
    uint32_t words[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) words[i] = row.counts[(i * WAVES + wave) * 64 + lane];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const uint64_t some0 = __ballot((words[i] & 0xffff) != 0), some1 = __ballot(words[i] >> 16 != 0);
        if (!(some0 | some1)) continue;
        int to = 0;
        if (lane == 0) to = atomicAdd(&row.entries, __popcll(some0) + __popcll(some1));
        to = __builtin_amdgcn_readfirstlane(to);
        const uint64_t before = (1ull << lane) - 1;
        const uint32_t place = 2 * ((i * WAVES + wave) * 64 + lane);
        if (words[i] & 0xffff) gptr(list)[to + __popcll(some0 & before)] = place << 16 | (words[i] & 0xffff);
        if (words[i] >> 16) gptr(list)[to + __popcll(some0) + __popcll(some1 & before)] = (place + 1) << 16 | words[i] >> 16;
    }
    __syncthreads();
    if (threadIdx.x == 0) gptr(a.entries)[at] = row.entries;
}

// The draw from a row's slices.
template <bool CARRY>
__global__ __launch_bounds__(T) void merge_kernel(SampleArgs a) {
    __shared__ Row row;
    __shared__ int of_slice[MOST_SLICES];  // how many of the drawn value
    const int r = blockIdx.x;
    int sizes[MOST_SLICES];
#pragma unroll
    for (int s = 0; s < MOST_SLICES; s++) sizes[s] = s < a.slices ? gptr(a.entries)[r * a.slices + s] : 0;
    clear(row);
    int least = BINS;
    const uint32_t *lists = a.lists + (int64_t)r * a.slices * a.slice;
    constexpr int U = 4;
#pragma unroll
    for (int s = 0; s < MOST_SLICES; s++) {
        const uint32_t *list = lists + (int64_t)s * a.slice;
        for (int i0 = threadIdx.x; i0 < sizes[s]; i0 += U * T) {
            uint32_t v[U];
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = i0 + u * T < sizes[s] ? gptr(list)[i0 + u * T] : 0;
#pragma unroll
            for (int u = 0; u < U; u++)
                if (v[u]) {
                    least = min(least, (int)(v[u] >> 16));
                    count<CARRY>(row, v[u] >> 16, v[u] & 0xffff);
                }
        }
    }
    least = least_of(row, least);
    draw(a, row, r, least, [&](int place, int &nth, int &first, int &last) {
        if (threadIdx.x < MOST_SLICES) of_slice[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < MOST_SLICES; s++) {
            const uint32_t *list = lists + (int64_t)s * a.slice;
            for (int i0 = threadIdx.x; i0 < sizes[s]; i0 += U * T) {
                uint32_t v[U];
#pragma unroll
                for (int u = 0; u < U; u++) v[u] = i0 + u * T < sizes[s] ? gptr(list)[i0 + u * T] : 0;
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (v[u] && (int)(v[u] >> 16) == place) of_slice[s] = v[u] & 0xffff;
            }
        }
        __syncthreads();
        int s = 0;
        while (s + 1 < a.slices && nth >= of_slice[s]) nth -= of_slice[s++];
        first = s * a.slice, last = min(a.vocab, first + a.slice);
    });
}

constexpr int SPLIT_VOCAB = 16384, SPLIT_ROWS = 128;  // rows of at least so many tokens, and fewer of them, are cut

// Slices of a row.
int slices_of(int rows, int vocab) {
    if (vocab < SPLIT_VOCAB || rows >= SPLIT_ROWS) return 1;
    const int slices = std::max(2, std::min({MOST_SLICES, 256 / rows, vocab / 4096}));
    return std::max(slices, (vocab + MOST_SLICE - 1) / MOST_SLICE);
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

bool check_sizes(const char *name, int rows, int vocab) {
    if (rows < 0 || rows > 1 << 20) return llm_fail("%s: rows %d is not in 0..1048576", name, rows);
    if (vocab <= 0 || vocab > MAX_VOCAB) return llm_fail("%s: vocab %d is not in 1..%d", name, vocab, MAX_VOCAB);
    return true;
}

// Floats of a row's lists, whatever its slices.
size_t list_floats(int vocab) { return (size_t)vocab + 10 * MOST_SLICES; }

}  // namespace

extern "C" size_t sample_rows_workspace_floats(int rows, int vocab) {
    if (!check_sizes("sample_rows_workspace_floats", rows, vocab) || vocab < SPLIT_VOCAB) return 0;
    return std::min(rows, SPLIT_ROWS - 1) * list_floats(std::min(vocab, MOST_SLICES * MOST_SLICE));
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
    SampleArgs a = {out, logprob, logits, temperature, top_k, top_p, min_p, u, vocab, logits_stride, nullptr, nullptr, 1, vocab};
    const int slices = slices_of(rows, vocab);
    const bool carry = vocab > 65535;
    if (slices > 1 && slices <= MOST_SLICES) {
        // from multiples of 8 on, so that slices are as aligned as their row
        a.slice = ((vocab + slices - 1) / slices + 7) / 8 * 8;
        a.slices = (vocab + a.slice - 1) / a.slice;
        a.entries = (int *)ws;
        a.lists = (uint32_t *)ws + ((size_t)rows * a.slices + 3) / 4 * 4;
        slice_kernel<<<dim3(a.slices, rows), T, 0, stream>>>(a);
        if (!LAUNCH_OK()) return;
        if (carry) merge_kernel<true><<<rows, T, 0, stream>>>(a);
        else merge_kernel<false><<<rows, T, 0, stream>>>(a);
    } else if (carry) {
        sample_kernel<true><<<rows, T, 0, stream>>>(a);
    } else {
        sample_kernel<false><<<rows, T, 0, stream>>>(a);
    }
    LAUNCH_OK();
}
