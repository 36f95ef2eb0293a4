// The next token of every row of logits by temperature, top-k, top-p and min-p (include/llm_amd/batch.h).
//
// bf16 logits have fewer than 2^16 values, so a row is counted by value, and everything after that is about
// values: weight and count of each, in the order of the values. Weights and sums are in 64 bits: a pick falls on
// the other side of a token's edge where the sums differ by more than what lies between u and the edge, and with
// sums in 32 bits that happened to one row in a few hundred.
//
// Bound by what a workgroup does one after the other, not by bytes: for one row of 151936 (22 us in two launches) 7 us
// for the slices' lists and 16 to merge and draw, of which clearing the counts takes 0.8, the weights and their sums 3, each
// filter about 1 and the search for the token 2 to 3. 64 such rows take 31 us, 200 rows of 32003 in one launch 18.
#include <math.h>

#include <algorithm>
#include <type_traits>

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
constexpr uint32_t NO_VALUE = 0xffffffffu;  // two NaN
constexpr int NONE = -1, MOST_SLICES = 8, MOST_SLICE = 65528;  // a multiple of 8 that 16 bits count

// The place of a value among the values, largest first, from its bits; NONE for what is never taken.
__device__ __forceinline__ int place_of(uint32_t b) {
    if ((b & 0x7fff) > 0x7f80 || b == 0xff80) return NONE;
    if (b == 0x8000) b = 0;
    return b & 0x8000 ? b : 0x7fff - b;
}
__device__ __forceinline__ uint32_t bits_at(int place) { return place & 0x8000 ? place : 0x7fff - place; }

struct Row {
    alignas(16) uint32_t counts[BINS / 2];  // n0 + 2^16 n1 of two values, modulo 2^32
    double mass[CHUNKS + 1];     // in front of each chunk of values
    int tokens[CHUNKS + 1];
    int carries;                 // how often a sum passed what it is held in:
    uint32_t carry[MOST_CARRIES];  // 2 w: n0 of word w passed a multiple of 2^16, 2 w + 1: the word one of 2^32
    int found[WAVES], sums[WAVES];
    int entries;
    int place, nth;              // of the token drawn: its value, and how many of that are in front of it
    double ratio;               // of its weight to the sum of what is left
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

// The logits from `first` to `last`, eight per thread at a time from aligned addresses on, the next two under way: the
// first ones are requested when this is made, in front of what else there is to do.
struct Logits {
    const bf16 *x;
    int first, last, head, body, i;
    u32x4 v, next;
    __device__ __forceinline__ u32x4 request(int at) const { return at < body ? ld16(x + at) : u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ Logits(const bf16 *x_, int first_, int last_) : x(x_), first(first_), last(last_) {
        head = min(last, first + (int)((16 - ((uintptr_t)(x + first) & 15)) / 2 & 7));
        body = head + (last - head) / 8 * 8;
        i = head + 8 * (int)threadIdx.x;
        v = request(i);
        next = request(i + 8 * T);
    }
    // f(bits) for each.
    template <class F>
    __device__ __forceinline__ void each(F f) {
#pragma unroll 1
        for (; i < body; i += 8 * T) {
            const u32x4 now = v;
            v = next;
            next = request(i + 2 * 8 * T);
#pragma unroll
            for (int e = 0; e < 8; e++) f(now[e / 2] >> (e % 2 * 16) & 0xffff);
        }
        // what is in front of the first aligned address, and behind the last one
        const int rest = (int)threadIdx.x < head - first ? first + threadIdx.x : body + (threadIdx.x - (head - first));
        if (rest < last && (rest < head || rest >= body)) f((uint32_t)gptr(x)[rest]);
    }
};

__device__ __forceinline__ int sum_lanes(int v) {
    v += llm::xor_lane<1>(v), v += llm::xor_lane<2>(v), v += llm::xor_lane<4>(v), v += llm::xor_lane<8>(v), v += llm::xor_lane<16>(v);
    return v + llm::xor_lane<32>(v);
}
__device__ __forceinline__ int least_lane(int v) {
    v = min(v, llm::xor_lane<1>(v)), v = min(v, llm::xor_lane<2>(v)), v = min(v, llm::xor_lane<4>(v));
    v = min(v, llm::xor_lane<8>(v)), v = min(v, llm::xor_lane<16>(v));
    return min(v, llm::xor_lane<32>(v));
}

// Sums of the lanes up to this one: within rows of 16 lanes of those 1, 2, 4 and 8 in front (DPP row_shr, 0 past the
// row's first), then the last one of the row in front (row_bcast15, into rows 1 and 3), then that of the first half.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
    return __hiloint2double(moved<CTRL, ROWS>(__double2hiint(v)), moved<CTRL, ROWS>(__double2loint(v)));
}
template <class V>
__device__ __forceinline__ V sum_upto(V v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    return v + moved<0x143, 0xc>(v);
}
// Of the lane in front (wave_shr:1), 0 for the first.
__device__ __forceinline__ int in_front(int v) { return __builtin_amdgcn_update_dpp(0, v, 0x138, 0xf, 0xf, true); }
__device__ __forceinline__ double in_front(double v) {
    return __hiloint2double(in_front(__double2hiint(v)), in_front(__double2loint(v)));
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ double lane_value(double v, int lane) {
    return __hiloint2double(lane_value(__double2hiint(v), lane), lane_value(__double2loint(v), lane));
}

// The smallest of the threads' places and the sum of their counts, in every thread (behind a barrier, with what is in
// LDS before it).
__device__ __forceinline__ void gather(Row &row, int &least, int &n) {
    least = least_lane(least);
    n = sum_lanes(n);
    if ((threadIdx.x & 63) == 0) row.found[wave_id()] = least, row.sums[wave_id()] = n;
    __syncthreads();
    const int lane = threadIdx.x & 63;
    least = __builtin_amdgcn_readfirstlane(least_lane(row.found[lane % WAVES]));
    n = __builtin_amdgcn_readfirstlane(sum_lanes(lane < WAVES ? row.sums[lane] : 0));
}

// In front of each chunk, from each chunk's own: the first wave, eight chunks per lane.
template <class V>
__device__ __forceinline__ void sum_chunks(V *chunks) {
    constexpr int EIGHT = CHUNKS / 64;
    const int lane = threadIdx.x & 63;
    V sum = 0, own[EIGHT];
#pragma unroll
    for (int i = 0; i < EIGHT; i++) sum += own[i] = chunks[lane * EIGHT + i];
    sum = in_front(sum_upto(sum));
#pragma unroll
    for (int i = 0; i < EIGHT; i++) {
        chunks[lane * EIGHT + i] = sum;
        sum += own[i];
    }
    if (lane == 63) chunks[CHUNKS] = sum;
}

// A wave looks at the counts four chunks at a time, a lane having four words (eight values) of one of them: group i of
// the wave's are the chunks from 4 (i WAVES + wave) on. Those that are not empty, as a mask.
constexpr int GROUPS = CHUNKS / 4 / WAVES;
__device__ __forceinline__ int word_of(int i) { return ((i * WAVES + wave_id()) * 64 + (threadIdx.x & 63)) * 4; }
__device__ __forceinline__ uint32_t groups_with_some(const Row &row) {
    uint32_t some = 0;
#pragma unroll
    for (int i = 0; i < GROUPS; i++) {
        const u32x4 v = *(const u32x4 *)(row.counts + word_of(i));
        if (__any((v[0] | v[1] | v[2] | v[3]) != 0)) some |= 1u << i;
    }
    return some;
}
// The sum over a lane's row of 16, in its last lane.
template <class V>
__device__ __forceinline__ V sum_of_row(V v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    return v + moved<0x118, 0xf>(v);
}

// The tokens in front of every chunk, and the groups of this wave that are not empty.
__device__ __forceinline__ uint32_t sum_tokens(Row &row, int carries) {
    const int lane = threadIdx.x & 63;
    if (threadIdx.x < CHUNKS) row.tokens[threadIdx.x] = 0, row.mass[threadIdx.x] = 0.0;
    const uint32_t some = carries ? (1u << GROUPS) - 1 : groups_with_some(row);
    __syncthreads();
#pragma unroll 1
    for (uint32_t rest = some; rest; rest &= rest - 1) {
        const int word = word_of(__builtin_ctz(rest));
        const u32x4 v = *(const u32x4 *)(row.counts + word);
        int n = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            int n0, n1;
            counts_of(row, carries, word + j, v[j], n0, n1);
            n += n0 + n1;
        }
        n = sum_of_row(n);
        if (lane % 16 == 15) row.tokens[word / 64] = n;
    }
    __syncthreads();
    if (wave_id() == 0) sum_chunks(row.tokens);
    __syncthreads();
    return some;
}

// e^x for x <= 0: k = rint(x log2 e), r = x - k ln 2 with ln 2 in two parts, the series of e^r to r^13 (|r| <= 0.347:
// the next term is below 2^-57), times 2^k.
__device__ __forceinline__ double exp_d(double x) {
    x = fmax(x, -1100.0);
    const double k = rint(x * 0x1.71547652b82fep+0);
    double r = fma(-k, 0x1.62e42fefa39efp-1, x);
    r = fma(-k, 0x1.abc9e3b39803fp-56, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)k);
}

// Row r's token from its counts. least: the place of the largest value (BINS: none); some: of sum_tokens.
// where(place, nth, first, last) says among which tokens the nth of that value is, and leaves in nth how many of it
// are in front of it there.
template <class Where>
__device__ __forceinline__ void draw(const SampleArgs &a, Row &row, int r, int least, uint32_t some, Where where) {
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
    const double top = (double)__uint_as_float(bits_at(least) << 16), by = 1.0 / (double)temperature;
    const auto weight = [&](int place) {
        const double x = (double)__uint_as_float(bits_at(place) << 16), y = exp_d((x - top) * by);
        // beside +inf nothing else weighs
        return x == top ? 1.0 : top > 3.5e38 ? 0.0 : y;
    };
    // a chunk's values, two per lane
    int n[2];
    double w[2];
    const auto weights = [&](int chunk) {
        const int word = chunk * 64 + lane;
        counts_of(row, carries, word, row.counts[word], n[0], n[1]);
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const double each = weight(2 * word + e);
            w[e] = n[e] ? each : 0.0;
        }
    };
    int place = least, nth = 0;
    double ratio = 1.0;
    if (temperature > 0.0f) {
        int left = row.tokens[CHUNKS];
        if (top_k > 0) left = min(left, top_k);
        // the mass of the chunks that hold some of the first top_k
#pragma unroll 1
        for (uint32_t rest = some; rest; rest &= rest - 1) {
            const int word = word_of(__builtin_ctz(rest));
            if (row.tokens[word / 256 * 4] >= left) break;  // in front of the group
            const u32x4 v = *(const u32x4 *)(row.counts + word);
            double part[8], m = 0.0;  // side by side
#pragma unroll
            for (int j = 0; j < 4; j++) {
                counts_of(row, carries, word + j, v[j], n[0], n[1]);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const double each = weight(2 * (word + j) + e);
                    part[2 * j + e] = n[e] ? n[e] * each : 0.0;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) m += part[j];
            m = sum_of_row(m);
            if (lane % 16 == 15) row.mass[word / 64] = m;
        }
        __syncthreads();
        if (wave == 0) sum_chunks(row.mass);
        __syncthreads();
    }
    if (temperature > 0.0f && wave == 0) {
        int left = row.tokens[CHUNKS];
        if (top_k > 0) left = min(left, top_k);
        double total = row.mass[CHUNKS];

        // Spots in the order of the tokens: behind a number of them, behind those up to a value, or behind the last
        // one up to which the mass is below `at` (BELOW) or not past it (WITHIN).
        enum { TOKENS, VALUES, BELOW, WITHIN };
        enum { TOP_K, TOP_P, MIN_P, PICK, BACK, DONE };
        int spot_tokens = 0;
#pragma unroll 1
        for (int step = TOP_K; step < DONE;) {
            int how = TOKENS, behind = 0;
            double at = 0.0;
            bool needed = true;
            if (step == TOP_K) {
                needed = left < row.tokens[CHUNKS];
                behind = left;
            } else if (step == TOP_P) {
                needed = top_p < 1.0f;
                how = BELOW;
                at = (double)top_p * total;
            } else if (step == MIN_P) {
                // of a u of 1 or more, which no running sum passes, the pick is the last token of positive weight: those of
                // none go here, as a sum need not show the difference
                needed = min_p > 0.0f || u >= 1.0f;
                how = VALUES;
                // the last place of enough weight, by 64ths of what is left: weights do not grow along the places
                int lo = least, hi = needed ? 0xff7f + 1 : least + 1;
#pragma unroll 1
                while (hi - lo > 1) {
                    const int by64 = (hi - lo + 63) / 64, mine = lo + (lane + 1) * by64;
                    const double each = weight(mine);
                    const int fit = __popcll(__ballot(mine < hi && each > 0.0 && !(each < (double)min_p)));
                    hi = min(hi, lo + (fit + 1) * by64);
                    lo += fit * by64;
                }
                behind = lo;
            } else if (step == PICK) {
                how = u != u ? TOKENS : WITHIN;
                at = u < 1.0f ? (double)u * total : INFINITY;  // 1 or more: all of them, so the last one
            } else {  // past the last one by a rounding: that
                needed = spot_tokens >= left;
                behind = left - 1;
            }
            if (!needed) {
                step++;
                continue;
            }
            const auto fits = [&](double m) { return how == WITHIN ? m <= at : m < at; };
            int chunk, k0, k1;
            uint64_t stops;
            double before;
            int tokens;
            for (;;) {
                // the last chunk whose front is not past the spot; fronts do not fall
                const auto front = [&](int c) { return how == TOKENS ? row.tokens[c] <= behind : fits(row.mass[c]); };
                const int group = max(0, __popcll(__ballot(front(lane * 8))) - 1);
                chunk = group * 8 + max(0, __popcll(__ballot(lane < 8 && front(group * 8 + (lane & 7)))) - 1);
                if (how == VALUES) chunk = behind / CHUNK;
                weights(chunk);
                before = row.mass[chunk] + in_front(sum_upto(n[0] * w[0] + n[1] * w[1]));
                tokens = row.tokens[chunk] + in_front(sum_upto(n[0] + n[1]));
                // how many tokens of the lane's two values are in front of the spot
                if (how == TOKENS) {
                    k0 = max(0, min(n[0], behind - tokens));
                    k1 = max(0, min(n[1], behind - tokens - n[0]));
                } else if (how == VALUES) {
                    k0 = 2 * (chunk * 64 + lane) <= behind ? n[0] : 0;
                    k1 = 2 * (chunk * 64 + lane) + 1 <= behind ? n[1] : 0;
                } else {
                    const auto part = [&](double m, double each, int most) {
                        if (most == 0 || !fits(m)) return 0;
                        // the reciprocal's 26 bits are enough for one too many or too few of up to 2^22
                        int k = each > 0 ? (int)fmin(fmax((at - m) * __builtin_amdgcn_rcp(each), 0.0), (double)most) : most;
                        if (k > 0 && !fits(m + k * each)) k--;
                        if (k < most && fits(m + (k + 1) * each)) k++;
                        return k;
                    };
                    k0 = part(before, w[0], n[0]);
                    k1 = k0 < n[0] ? 0 : part(before + n[0] * w[0], w[1], n[1]);
                }
                stops = __ballot(k0 + k1 < n[0] + n[1]);
                if (stops || how == TOKENS || how == VALUES) break;
                // all of the chunk, where its sum falls short of the next one's front by a rounding, or it is empty
                how = TOKENS;
                behind = row.tokens[chunk + 1];
            }
            const int from = stops ? (int)__builtin_ctzll(stops) : 63;
            const bool second = k0 == n[0];
            spot_tokens = lane_value(tokens + k0 + k1, from);
            const double mass = lane_value(before + (k0 * w[0] + k1 * w[1]), from);
            const double each = lane_value(second ? w[1] : w[0], from);
            if (step == TOP_K) {
                total = mass;
            } else if (step == TOP_P) {  // with the one that reaches p
                if (spot_tokens + 1 < left) left = spot_tokens + 1, total = mass + each;
            } else if (step == MIN_P) {
                if (min_p > 1.0f) left = 1, total = 1.0;  // more than the first one weighs
                else if (spot_tokens < left) left = spot_tokens, total = mass;
            } else {
                place = lane_value(2 * (chunk * 64 + lane) + (second ? 1 : 0), from);
                nth = lane_value(second ? k1 : k0, from);
                ratio = each / total;
            }
            step++;
        }
    }
    if (threadIdx.x == 0) row.place = place, row.nth = nth, row.ratio = ratio;
    __syncthreads();
    place = row.place;
    nth = row.nth;
    ratio = row.ratio;
    int first, last;
    where(place, nth, first, last);
    // each wave counts the value in its part of these tokens, 32 per lane at a time, then one looks through its own
    const uint32_t bits = bits_at(place);
    const bf16 *x = a.x + r * a.x_stride;
    constexpr int ROUND = 64 * 32;
    const int begin = first - (int)((uintptr_t)(x + first) % 16 / 2);
    const int part = (last - begin + ROUND * WAVES - 1) / (ROUND * WAVES) * ROUND, mine = begin + wave * part;
    const auto look_at = [&](int i) {  // the lane's 32 tokens from i on: which have the value
        u32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = i + 8 * j;
            v[j] = u32x4{NO_VALUE, NO_VALUE, NO_VALUE, NO_VALUE};
            if (c >= first && c + 8 <= last) {
                v[j] = ld16(x + c);
            } else if (c + 8 > first && c < last) {  // at an end that is not aligned
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c + e >= first && c + e < last)
                        v[j][e / 2] = e % 2 ? (v[j][e / 2] & 0xffff) | (uint32_t)gptr(x)[c + e] << 16
                                            : (v[j][e / 2] & 0xffff0000u) | gptr(x)[c + e];
            }
        }
        uint32_t mask = 0;
#pragma unroll
        for (int j = 0; j < 32; j++) {
            uint32_t b = v[j / 8][j % 8 / 2] >> (j % 2 * 16) & 0xffff;
            if (b == 0x8000) b = 0;
            mask |= b == bits ? 1u << j : 0;
        }
        return mask;
    };
    int met = 0, at = mine;
    uint32_t mask = 0;
#pragma unroll 1
    for (bool counted = false;;) {
        // once to count; where that takes one round, its mask is that of the second time
        if (!counted) {
            for (int i = mine; i < min(last, mine + part); i += ROUND) {
                mask = look_at(i + 32 * lane);
                met += __popc(mask);
            }
            met = sum_lanes(met);
            if (lane == 0) row.sums[wave] = met;
            __syncthreads();
            const int before = __builtin_amdgcn_readfirstlane(sum_lanes(lane < wave ? row.sums[lane] : 0));
            if (nth < before || nth >= before + met) return;
            nth -= before;
            counted = true;
            if (part > ROUND) continue;
        } else {
            mask = look_at(at + 32 * lane);
        }
        const int upto = sum_upto((int)__popc(mask)), all = lane_value(upto, 63);
        if (nth < all) {
            int rest = nth - (upto - __popc(mask));
            if (rest < 0 || rest >= __popc(mask)) return;
            for (; rest > 0; rest--) mask &= mask - 1;
            a.out[r] = at + 32 * lane + __builtin_ctz(mask);
            if (a.logprob) a.logprob[r] = (float)log(ratio);
            return;
        }
        nth -= all;
        if ((at += ROUND) >= last) return;
    }
}

// Counts with add(exact), which gives the smallest place and the number of what it counted; again, with carries, where
// the sum of the counts says that some passed 16 bits.
template <class Add>
__device__ __forceinline__ uint32_t count_all(Row &row, int &least, Add add) {
    int n = 0;
    least = BINS;
    add(std::false_type{}, least, n);
    __syncthreads();
    gather(row, least, n);
    uint32_t some = sum_tokens(row, 0);
    if (row.tokens[CHUNKS] == n) return some;
    __syncthreads();
    clear(row);
    add(std::true_type{}, least, n);
    __syncthreads();
    return sum_tokens(row, row.carries);
}

// One workgroup per row.
__global__ __launch_bounds__(T) void sample_kernel(SampleArgs a) {
    __shared__ Row row;
    const int r = blockIdx.x;
    Logits logits(a.x + r * a.x_stride, 0, a.vocab);
    clear(row);
    int least;
    const uint32_t some = count_all(row, least, [&](auto carry, int &least, int &n) {
        if (carry) logits = Logits(a.x + r * a.x_stride, 0, a.vocab);  // again
        logits.each([&](uint32_t b) {
            const int p = place_of(b);
            if (p == NONE) return;
            least = min(least, p);
            n++;
            count<decltype(carry)::value>(row, p, 1);
        });
    });
    draw(a, row, r, least, some, [&](int, int &, int &first, int &last) { first = 0, last = a.vocab; });
}

// A slice of a row: its values and their counts as a list.
__global__ __launch_bounds__(T) void slice_kernel(SampleArgs a) {
    __shared__ Row row;
    const int r = blockIdx.y, lane = threadIdx.x & 63;
    const int first = blockIdx.x * a.slice, last = min(a.vocab, first + a.slice);
    Logits logits(a.x + r * a.x_stride, first, last);
    clear(row);
    logits.each([&](uint32_t b) {
        const int p = place_of(b);
        if (p != NONE) count<false>(row, p, 1);  // a slice has less than 2^16 tokens
    });
    __syncthreads();
    const int at = r * a.slices + blockIdx.x;
    uint32_t *list = a.lists + (int64_t)at * a.slice;
    const uint32_t some = groups_with_some(row);
    const auto entries = [](const u32x4 &v) {
        int n = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) n += ((v[j] & 0xffff) != 0) + (v[j] >> 16 != 0);
        return n;
    };
    int all = 0;
#pragma unroll 1
    for (uint32_t rest = some; rest; rest &= rest - 1) all += entries(*(const u32x4 *)(row.counts + word_of(__builtin_ctz(rest))));
    const int upto = sum_upto(all);
    int to = 0;
    if (lane == 63) to = atomicAdd(&row.entries, upto);
    to = lane_value(to, 63) + upto - all;  // a lane's entries lie side by side
#pragma unroll 1
    for (uint32_t rest = some; rest; rest &= rest - 1) {
        const int word = word_of(__builtin_ctz(rest));
        const u32x4 v = *(const u32x4 *)(row.counts + word);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t place = 2 * (word + j);
            if (v[j] & 0xffff) gptr(list)[to++] = place << 16 | (v[j] & 0xffff);
            if (v[j] >> 16) gptr(list)[to++] = (place + 1) << 16 | v[j] >> 16;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) gptr(a.entries)[at] = row.entries;
}

// The draw from a row's slices.
__global__ __launch_bounds__(T) void merge_kernel(SampleArgs a) {
    __shared__ Row row;
    __shared__ int of_slice[MOST_SLICES];  // how many of the drawn value
    const int r = blockIdx.x;
    int sizes[MOST_SLICES], most = 0;
#pragma unroll
    for (int s = 0; s < MOST_SLICES; s++) sizes[s] = s < a.slices ? gptr(a.entries)[r * a.slices + s] : 0;
#pragma unroll
    for (int s = 0; s < MOST_SLICES; s++) most = max(most, sizes[s]);
    const uint32_t *lists = a.lists + (int64_t)r * a.slices * a.slice;
    // an entry of every slice at a time; the first ones stay in registers
    constexpr int KEPT = 3;
    uint32_t kept[KEPT][MOST_SLICES];
    const auto request = [&](int i, uint32_t (&v)[MOST_SLICES]) {
#pragma unroll
        for (int s = 0; s < MOST_SLICES; s++) v[s] = i < sizes[s] ? gptr(lists)[(int64_t)s * a.slice + i] : 0;
    };
#pragma unroll
    for (int k = 0; k < KEPT; k++) request(k * T + threadIdx.x, kept[k]);
    const auto each_entry = [&](auto f) {
        const auto all = [&](const uint32_t (&v)[MOST_SLICES]) {
#pragma unroll
            for (int s = 0; s < MOST_SLICES; s++)
                if (v[s]) f(s, (int)(v[s] >> 16), v[s] & 0xffff);
        };
#pragma unroll
        for (int k = 0; k < KEPT; k++)
            if (k * T < most) all(kept[k]);
#pragma unroll 1
        for (int i = KEPT * T + threadIdx.x; i < most; i += T) {
            uint32_t v[MOST_SLICES];
            request(i, v);
            all(v);
        }
    };
    clear(row);
    int least;
    const uint32_t some = count_all(row, least, [&](auto carry, int &least, int &n) {
        each_entry([&](int, int place, uint32_t m) {
            least = min(least, place);
            n += m;
            count<decltype(carry)::value>(row, place, m);
        });
    });
    draw(a, row, r, least, some, [&](int place, int &nth, int &first, int &last) {
        if (threadIdx.x < MOST_SLICES) of_slice[threadIdx.x] = 0;
        __syncthreads();
        each_entry([&](int s, int p, uint32_t m) {
            if (p == place) of_slice[s] = m;
        });
        __syncthreads();
        int which = 0;
        bool there = false;
#pragma unroll
        for (int s = 0; s < MOST_SLICES; s++) {
            there |= nth < of_slice[s];
            if (!there && s + 1 < a.slices) nth -= of_slice[s], which = s + 1;
        }
        first = which * a.slice, last = min(a.vocab, first + a.slice);
    });
}

// Rows of at least SPLIT_VOCAB tokens are cut, into as many slices as let all workgroups of a launch have a CU to themselves;
// from SPLIT_ROWS on those of LONG_VOCAB alone, and from LONG_ROWS on none. us of a captured call with temperature, top-k and
// top-p, uncut and in the slices of this rule: one row of 32000 17.4 and 20.4, of 50257 22.3 and 21.1, of 65536 24.2 and 21.2,
// of 151936 39.7 and 23.0; 64 of 50257 23.5 and 23.6, of 65536 25.3 and 24.3; 96 of 65536 25.8 and 27.4, of 100352 33.9 and
// 32.4; 127 of 151936 45.4 and 42.4, 160 45.7 and 43.1, 200 46.5 and 52.4.
constexpr int SPLIT_VOCAB = 49152, SPLIT_ROWS = 65, LONG_VOCAB = 98304, LONG_ROWS = 128;

// Slices of a row.
int slices_of(int rows, int vocab) {
    if (vocab < SPLIT_VOCAB || rows >= (vocab < LONG_VOCAB ? SPLIT_ROWS : LONG_ROWS)) return 1;
    const int slices = std::max(2, std::min(MOST_SLICES, 256 / rows));
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
    return std::min(rows, LONG_ROWS - 1) * list_floats(std::min(vocab, MOST_SLICES * MOST_SLICE));
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
    if (slices > 1 && slices <= MOST_SLICES) {
        // from multiples of 8 on, so that slices are as aligned as their row
        a.slice = ((vocab + slices - 1) / slices + 7) / 8 * 8;
        a.slices = (vocab + a.slice - 1) / a.slice;
        a.entries = (int *)ws;
        a.lists = (uint32_t *)ws + ((size_t)rows * a.slices + 3) / 4 * 4;
        slice_kernel<<<dim3(a.slices, rows), T, 0, stream>>>(a);
        if (!LAUNCH_OK()) return;
        merge_kernel<<<rows, T, 0, stream>>>(a);
    } else {
        sample_kernel<<<rows, T, 0, stream>>>(a);
    }
    LAUNCH_OK();
}
