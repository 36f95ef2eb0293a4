// Attention of new tokens over a paged KV cache (include/llm_amd/paged.h).
//
// A sequence's new rows times the query heads of one kv head are the columns of the matrix products:
// scores S^T = K Q^T (keys x columns) and outputs O^T += V^T P^T (head_dim x columns), both on
// 32x32x16 MFMAs with the columns spread over the lanes, so that the softmax runs down a lane's registers
// and P^T goes from the first product's accumulators into the second's operand without crossing lanes: of
// 16 keys, lane half h holds 4h..4h+3 and 8+4h..8+4h+3, and the second product sums over any order of keys.
#include <math.h>

#include <type_traits>

#include "paged_batch.h"

using namespace llm;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

#define LLM_LDS __attribute__((address_space(3)))
typedef LLM_LDS char lds_char;

constexpr float LOWEST = -3.402823466e+38f;
constexpr int CUS = 256;

struct AttendArgs {
    Batch b;
    bf16 *out;
    const bf16 *q;
    int64_t out_stride, q_stride;
    float *part, *stats;  // of this kernel's units: [unit][split][row][head_dim], [unit][split][row][2]
    int n_heads, n_kv_heads, group, window;
    int n_split, chunk;   // keys per split, a multiple of 128
    int which;            // the sequences whose rows these are
    float scale_log2;     // scale * log2(e)
};

// The same arguments read from the kernel's argument memory where they are used: what only rare steps need
// does not hold scalar registers through the loops.
struct LaunchArgs {
    AttendArgs few, many;
    int few_units, many_units, few_groups, many_groups;  // tiles x kv heads, and those x splits
    int many_split, mirrored;
};
#define LLM_CONST __attribute__((address_space(4)))
__device__ __forceinline__ const LLM_CONST AttendArgs *again(bool many) {
    const LLM_CONST LaunchArgs *l = (const LLM_CONST LaunchArgs *)__builtin_amdgcn_kernarg_segment_ptr();
    const LLM_CONST AttendArgs *a = many ? &l->many : &l->few;
    asm volatile("" : "+s"(a));
    return a;
}

// ------------------------------------------------------------------------------------------
// which rows and keys
// ------------------------------------------------------------------------------------------

// T rows (new tokens x query heads of a kv head) of one sequence.
struct Tile {
    int s, first, rows;      // sequence, first row among the sequence's, rows of this tile
    int q0;                  // the sequence's first token
    int before;              // position of its first token
    int begin, end, active;  // keys of any row (begin a multiple of 64), splits that have some
    int from, to, least, most;  // positions from..to are seen by every row, least..most by any
};

__device__ __forceinline__ int token_at(const Batch &b, int i) {
    return max(0, min(b.n_tokens, gptr(b.q_start)[i]));
}

// Which sequences a kernel takes.
enum { ALL_ROWS, FEW_ROWS, MANY_ROWS };  // any number of rows; at most FEW; more than FEW
constexpr int FEW = 32;                  // rows of a tile of attend_few
constexpr int MANY = 128;                // rows of a tile of attend_many

// Tile i, counted over the sequences that `which` takes, false past the last one. A sequence's tiles come
// last rows first: those see the most keys.
template <int T>
__device__ __forceinline__ bool find_tile(const AttendArgs &a, int which, int i, Tile &t) {
    const int lane = threadIdx.x & 63;
    int j = -1, tokens = 0;
    for (int s0 = 0; s0 < a.b.n_seqs; s0 += 64) {
        const int s = min(s0 + lane, a.b.n_seqs - 1);  // what the lanes read goes out together
        const int first = token_at(a.b, s), count = max(0, token_at(a.b, s + 1) - first), length = kv_length(a.b, s);
        const int64_t rows = (int64_t)count * a.group;
        int n = 0;
        if (s0 + lane < a.b.n_seqs && (which == ALL_ROWS || (rows <= FEW) == (which == FEW_ROWS)))
            n = (int)((rows + T - 1) / T);
        int upto = n;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int before = __shfl_up(upto, d);
            if (lane >= d) upto += before;
        }
        const uint64_t past = __ballot(upto > i);
        if (past) {
            const int at = __builtin_ctzll(past);
            t.s = s0 + at;
            t.q0 = __builtin_amdgcn_readlane(first, at);
            tokens = __builtin_amdgcn_readlane(count, at);
            t.before = __builtin_amdgcn_readlane(length, at) - tokens;
            j = __builtin_amdgcn_readlane(upto, at) - 1 - i;
            break;
        }
        i -= __builtin_amdgcn_readlane(upto, 63);
    }
    if (j < 0) return false;
    t.first = j * T;
    t.rows = min(T, tokens * a.group - t.first);
    const int lo = t.before + t.first / a.group, hi = t.before + (t.first + t.rows - 1) / a.group;
    t.to = lo;
    t.most = hi;
    t.from = a.window > 0 ? max(0, hi - a.window + 1) : 0;
    t.least = a.window > 0 ? max(0, lo - a.window + 1) : 0;
    const int64_t room = (int64_t)a.b.table_pages * a.b.page_size;
    t.end = (int)min((int64_t)(hi + 1), room);
    t.begin = t.least & ~63;
    t.active = t.end > t.begin ? min(a.n_split, (t.end - t.begin + a.chunk - 1) / a.chunk) : 1;
    return true;
}

// ------------------------------------------------------------------------------------------
// pages into LDS
// ------------------------------------------------------------------------------------------

// Rows of keys or values lie in LDS as they are, 16-byte chunk c of row r at chunk c ^ swizzle(r): the 16 rows
// that a product's operand reads at one chunk, and the four rows of 64 bytes that a transposing read takes,
// then lie in different banks. Linear in the bits of r.
template <int D>
__device__ __forceinline__ constexpr int swizzle(int r) {
    return D == 64 ? ((r >> 1 & 1) << 2 | (r >> 2 & 3)) : ((r & 3) << 2 | (r >> 2 & 3));
}

// 64 lanes' 16 bytes from base + offset into LDS at `to` on, without passing registers. The wave waits for
// it with wait_loads: the compiler does not know of it.
// STREAM: read non-temporally, what one workgroup alone reads (64 tokens over up to 8448 positions 216 -> 195 us).
template <bool STREAM>
__device__ __forceinline__ void load_to_lds(unsigned to, const void *base, unsigned offset) {
    if constexpr (STREAM)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(to), "v"(offset), "s"(base)
                     : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base)
                     : "memory");
}
template <bool STREAM>
__device__ __forceinline__ void load_to_lds(unsigned to, const void *at) {
    if constexpr (STREAM)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(to), "v"(at) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(at) : "memory");
}
// A wave-uniform value in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t x) {
    const int lo = __builtin_amdgcn_readfirstlane((int)x), hi = __builtin_amdgcn_readfirstlane((int)(x >> 32));
    return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}
// All but the last N vector memory operations of the wave are done.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// A wave's ROWS consecutive positions at a time, of every STEP, out of the pages into LDS. Positions that are
// not there read the pool's first rows (the scores' mask leaves them out).
// WHOLE: the 16 positions from a multiple of 16 on lie in one page, so a place is looked up once for them, 64
// at a time, one per lane; otherwise every position's place is looked up, 128 at a time, into LDS.
template <int D, int ROWS, int STEP, bool WHOLE, bool STREAM>
struct Pages {
    static constexpr int PER = 512 / D;        // rows per load
    static constexpr int LOADS = ROWS / PER;   // of keys, and as many of values
    static constexpr int GROUPS = ROWS < 16 ? 1 : ROWS / 16, GROUP_LOADS = LOADS / GROUPS;
    static constexpr int AHEAD = WHOLE ? 64 / GROUPS : 128 / ROWS;  // steps looked up at a time
    int first;                // the first step's first position
    int64_t mine;             // WHOLE: the lane's place, in bytes, with the kv head
    int present;              // WHOLE: whether it is there
    LLM_LDS int64_t *places;  // otherwise: 128 of them
    int64_t head;             // bytes to the kv head
    unsigned offset[GROUP_LOADS];  // the lane's bytes within load i: WHOLE with its row, otherwise its chunk alone

    // row0: where in the buffer the wave's rows begin, a multiple of PER
    __device__ __forceinline__ Pages(const Batch &b, int kv, int first_, int row0, LLM_LDS int64_t *places_)
        : first(first_), mine(0), present(0), places(places_), head(uniform(kv * b.head_stride * 2)) {
        const int lane = threadIdx.x & 63, r = lane / (D / 8);
#pragma unroll
        for (int i = 0; i < GROUP_LOADS; i++)
            offset[i] = (lane % (D / 8) ^ swizzle<D>(row0 + i * PER + r)) * 16 +
                        (WHOLE ? (unsigned)(i * PER + r) * (unsigned)b.slot_stride * 2 : 0);
    }

    __device__ __forceinline__ void set(int64_t at) {
        present = at >= 0;
        mine = (at < 0 ? 0 : at * 2) + head;
    }
    // Looks up steps step .. step + AHEAD - 1, when step is a multiple of AHEAD.
    __device__ __forceinline__ void look_up(bool many, int s, int step) {
        if (step % AHEAD != 0) return;
        const int lane = threadIdx.x & 63;
        const auto &b = again(many)->b;
        if constexpr (WHOLE) {
            set(place(b, s, first + (step + lane / GROUPS) * STEP + lane % GROUPS * 16));
        } else {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int n = lane + 64 * k;
                const int64_t at = place(b, s, first + (step + n / ROWS) * STEP + n % ROWS);
                places[n] = at < 0 ? -1 : at * 2 + head;
            }
            wait_lds();
        }
    }

    // Bit r: the step's position r is there.
    __device__ __forceinline__ uint32_t there(int step) const {
        if constexpr (WHOLE) {
            uint32_t bits = 0;
#pragma unroll
            for (int g = 0; g < GROUPS; g++)
                if (__builtin_amdgcn_readlane(present, step % AHEAD * GROUPS + g))
                    bits |= (ROWS < 16 ? (1u << ROWS) - 1 : 0xffffu) << (16 * g);
            return bits;
        } else {
            const int lane = threadIdx.x & 63;
            return (uint32_t)__ballot(lane < ROWS && places[step % AHEAD * ROWS + (lane & (ROWS - 1))] >= 0);
        }
    }

    // WHOLE: where 16 of the step's positions begin in a cache.
    __device__ __forceinline__ const char *base(const bf16 *cache, int step, int group = 0) const {
        if constexpr (!WHOLE) return (const char *)cache;
        const int lane = step % AHEAD * GROUPS + group;
        const int hi = __builtin_amdgcn_readlane((int)(mine >> 32), lane);
        const unsigned lo = __builtin_amdgcn_readlane((int)mine, lane);
        return (const char *)cache + (int64_t)((uint64_t)(unsigned)hi << 32 | lo);
    }
    // Load i of the step's rows into LDS at `to` (where load 0 goes); from: base() of the load's group.
    __device__ __forceinline__ void load(const char *from, int step, int i, unsigned to) const {
        if constexpr (WHOLE) {
            load_to_lds<STREAM>(to + i * 1024, from, offset[i % GROUP_LOADS]);
        } else {
            const int64_t at = places[step % AHEAD * ROWS + i * PER + (threadIdx.x & 63) / (D / 8)];
            load_to_lds<STREAM>(to + i * 1024, from + (at < 0 ? head : at) + offset[i % GROUP_LOADS]);
        }
    }
    // All loads of the step's rows of one cache.
    __device__ __forceinline__ void request(const bf16 *cache, int step, unsigned to) const {
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            const char *from = base(cache, step, g);
#pragma unroll
            for (int i = g * GROUP_LOADS; i < (g + 1) * GROUP_LOADS; i++) load(from, step, i, to);
        }
    }
};

// The wave's own rows of values in LDS, as LOADS loads of its lanes left them, from position `at` on: those that
// no row of the tile sees become zeros, since 0 times a NaN or an infinity would not be 0. Of those that some
// rows see and others do not, NaN and infinities become zeros; whether there were any (add_bad then gives
// them back to the rows that see them). seen: positions from..to are seen by every row, least..most by any.
template <int D, int LOADS>
__device__ __forceinline__ bool clear_unseen(lds_char *rows, int at, uint32_t there, int from, int to, int least,
                                             int most) {
    const int lane = threadIdx.x & 63;
    bool found = false;
#pragma unroll 1
    for (int i = 0; i < LOADS; i++) {
        const int r = i * (512 / D) + lane / (D / 8), p = at + r;
        LLM_LDS u32x4 *x = (LLM_LDS u32x4 *)(rows + i * 1024 + lane * 16);
        if (!(there >> r & 1) || p < least || p > most) {
            *x = u32x4{0, 0, 0, 0};
        } else if (p < from || p > to) {
            u32x4 v = *x;
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if ((v[j] & 0x7f80u) == 0x7f80u) v[j] &= 0xffff0000u, bad = true;
                if ((v[j] & 0x7f800000u) == 0x7f800000u) v[j] &= 0xffffu, bad = true;
            }
            if (bad) *x = v;
            found |= bad;
        }
    }
    return __any(found);
}

// ------------------------------------------------------------------------------------------
// a wave's 32 columns
// ------------------------------------------------------------------------------------------

template <int D>
struct Columns {
    f32x16 o[D / 32];      // O^T: rows 32 dt + (r & 3) + 8 (r / 4) + 4 h in register r of lane half h
    u32x4 q[D / 16];       // Q^T: elements 16 ks + 8 h .. + 7
    float top, sum;        // the running maximum (times scale_log2) and this half's part of the sum
    int position, column;  // of the lane's row (-1: no row), its index in the wave

    __device__ __forceinline__ void start(const AttendArgs &a, const Tile &t, int kv, int first) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        column = lane & 31;
        const int row = t.first + first + column;
        const bool there = first + column < t.rows;
        const int token = row / a.group;
        position = there ? t.before + token : -1;
        const bf16 *src = a.q + (t.q0 + token) * a.q_stride + (kv * a.group + row - token * a.group) * D + 8 * h;
#pragma unroll
        for (int k = 0; k < D / 16; k++) q[k] = there ? ld16(src + 16 * k) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
        top = LOWEST;
        sum = 0.0f;
    }

    // Bit k: the lane's row sees position at + k, k < 32.
    __device__ __forceinline__ uint32_t sees(int at, int window) const {
        const int last = position - at;  // the last bit
        uint32_t bits = last < 0 ? 0 : last >= 31 ? ~0u : (2u << last) - 1;
        if (window > 0) {
            const int first = last - window + 1;
            if (first > 31)
                bits = 0;
            else if (first > 0)
                bits &= ~0u << first;
        }
        return bits;
    }

    // Scores of 32 keys in LDS.
    __device__ __forceinline__ f32x16 scores(const lds_char *keys) const {
        const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
        const lds_char *row = keys + r * (2 * D);
        const int c0 = (h ^ swizzle<D>(r)) * 16;
        f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
            const u32x4 x = *(const LLM_LDS u32x4 *)(row + (c0 ^ (k * 32)));
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, x),
                                                        __builtin_bit_cast(bf16x8_t, q[k]), s, 0, 0, 0);
        }
        return s;
    }

    // Scores to weights 2^(s c - top) in two steps. The maximum moves where a column's has grown by more than a
    // factor of 2^8 (for all 32 columns then): below that the weights stay in range, and a larger maximum would
    // change no relative rounding.
    template <int KT>
    __device__ __forceinline__ float peak(const f32x16 (&s)[KT], float c) const {
        float m = s[0][0];
#pragma unroll
        for (int k = 0; k < KT; k++)
#pragma unroll
            for (int r = 0; r < 16; r++) m = fmaxf(m, s[k][r]);
        float x, y;
        swap_pair<32>(m, x, y);
        return fmaxf(x, y) * c;
    }
    __device__ __forceinline__ void raise(float m) {
        if (!__any(m > top + 8.0f)) return;
        const float next = fmaxf(top, m);
        const float keep = __builtin_amdgcn_exp2f(top - next);
        top = next;
        sum *= keep;
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] *= keep;
    }
    // Weights 2^(s c - top) of 32 keys as the second product's operands of 16 keys each, rounded to bf16 (half
    // a step each, at random; their sum adds the rounded ones), with EXACT what the rounding left as well.
    template <bool EXACT>
    __device__ __forceinline__ void weigh(f32x16 &s, float c, u32x4 (&hi)[2], u32x4 (&lo)[2]) {
        float part = 0.0f;
        const bf16x2_t ones = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[8 * t + 2 * j], c, -top));
                const float y = __builtin_amdgcn_exp2f(fmaf(s[8 * t + 2 * j + 1], c, -top));
                const uint32_t w = pack2(x, y);
                hi[t][j] = w;
                if constexpr (EXACT) {
                    lo[t][j] = pack2(x - lo_f(w), y - hi_f(w));
                    sum += x;
                    part += y;
                } else if (t == 0) {
                    sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), ones, sum, false);
                } else {
                    part = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), ones, part, false);
                }
            }
        sum += part;
    }

    // O^T += V^T P^T over 32 keys.
    template <bool EXACT>
    __device__ __forceinline__ void add(const lds_char *values, const u32x4 (&hi)[2], const u32x4 (&lo)[2]) {
        const int lane = threadIdx.x & 63, i = lane & 15, h = lane >> 5;
        const int row = 4 * h + (i >> 2);
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int d = 0; d < D / 32; d++) {
                const int c = d * 4 + (lane >> 4 & 1) * 2 + ((i & 3) >> 1);
                s16x4 v[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int r = 16 * t + 8 * u + row;
                    v[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (LLM_LDS s16x4 *)(values + r * (2 * D) + (c ^ swizzle<D>(r)) * 16 + (i & 1) * 8));
                }
                const u32x2 v0 = __builtin_bit_cast(u32x2, v[0]), v1 = __builtin_bit_cast(u32x2, v[1]);
                const bf16x8_t vt = __builtin_bit_cast(bf16x8_t, (u32x4{v0.x, v0.y, v1.x, v1.y}));
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt, __builtin_bit_cast(bf16x8_t, hi[t]), o[d], 0, 0, 0);
                if constexpr (EXACT)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt, __builtin_bit_cast(bf16x8_t, lo[t]), o[d], 0, 0, 0);
            }
    }

    // One step of 32 KT keys, the matrix products with everything else between them: the next keys' scores into
    // `next` beside the first 32 weights per two lanes and the loads of later keys and values (bring), then
    // O^T += V^T P^T beside the other weights and the maximum of `next`, which is the result. The matrix unit takes
    // an instruction every 32 cycles, and the other units' fit in between where they are spread evenly and do not
    // wait for each other: a weight's fma, exponential and rounding stand in three places. The fences keep the
    // order written.
    template <int KT, class Bring>
    __device__ __forceinline__ float step(const lds_char *keys, const lds_char *values, const f32x16 (&s)[KT],
                                          f32x16 (&next)[KT], float c, Bring bring) {
        constexpr int QK = KT * D / 16, PV = KT * D / 16, RING = 4;  // products of each kind; operands in flight
        constexpr int ALL = 16 * KT;                                 // weights of a lane
        const int lane = threadIdx.x & 63, r = lane & 31, i = lane & 15, h = lane >> 5;
        const lds_char *key_row = keys + r * (2 * D);
        const int c0 = (h ^ swizzle<D>(r)) * 16, value_row = 4 * h + (i >> 2);
        const auto key = [&](int j) {
            return __builtin_bit_cast(
                bf16x8_t, *(const LLM_LDS u32x4 *)(key_row + (j % KT) * 64 * D + (c0 ^ (j / KT * 32))));
        };
        const auto value = [&](int j) {
            const int d = j % (D / 32), t = j / (D / 32), chunk = d * 4 + (lane >> 4 & 1) * 2 + ((i & 3) >> 1);
            u32x4 v;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int row = 16 * t + 8 * u + value_row;
                const u32x2 x = __builtin_bit_cast(
                    u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LLM_LDS s16x4 *)(
                               values + row * (2 * D) + (chunk ^ swizzle<D>(row)) * 16 + (i & 1) * 8)));
                v[2 * u] = x.x;
                v[2 * u + 1] = x.y;
            }
            return __builtin_bit_cast(bf16x8_t, v);
        };
        const bf16x2_t ones = {(__bf16)1.0f, (__bf16)1.0f};
        u32x4 p[2 * KT];              // weights of 16 keys each
        float odd = 0.0f, w[4];       // the last weights
        float arg = fmaf(s[0][0], c, -top);
        const auto pair = [&](int e) {  // weights e and e + 1: rounded, and added
            const uint32_t both = pack2(w[e & 3], w[(e & 3) + 1]);
            p[e / 16 * 2 + e % 16 / 8][e % 8 / 2] = both;
            float &to = e & 2 ? odd : sum;
            to = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, both), ones, to, false);
        };
        const auto weigh_one = [&](int e) {  // weight e; the pair before it where it begins a new one
            w[e & 3] = __builtin_amdgcn_exp2f(arg);
            if (e + 1 < ALL) arg = fmaf(s[(e + 1) / 16][(e + 1) % 16], c, -top);
            if (e >= 2 && !(e & 1)) pair(e - 2);
        };
        bf16x8_t ring[RING];
#pragma unroll
        for (int j = 0; j < RING - 1; j++) ring[j] = key(j);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < QK; j++) {
            ring[(j + RING - 1) % RING] = j + RING - 1 < QK ? key(j + RING - 1) : value(j + RING - 1 - QK);
            f32x16 from = next[j % KT];
            if (j < KT)
#pragma unroll
                for (int e = 0; e < 16; e++) from[e] = 0.0f;
            next[j % KT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[j % RING], __builtin_bit_cast(bf16x8_t, q[j / KT]),
                                                                   from, 0, 0, 0);
#pragma unroll
            for (int e = 16 * j / QK; e < 16 * (j + 1) / QK; e++) weigh_one(e);
            if (j & 1) bring(j / 2);  // QK / 2 of them
            __builtin_amdgcn_sched_barrier(0);
        }
        if (KT == 1) pair(14);
        float peak = LOWEST;
        constexpr int FIRST = KT == 1 ? 0 : PV / 2;  // products beside the last weights; then the maximum
#pragma unroll
        for (int j = 0; j < PV; j++) {
            if (j + RING - 1 < PV) ring[(QK + j + RING - 1) % RING] = value(j + RING - 1);
            f32x16 &to = o[j % (D / 32)];
            to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[(QK + j) % RING], __builtin_bit_cast(bf16x8_t, p[j / (D / 32)]),
                                                         to, 0, 0, 0);
            if (j < FIRST) {
#pragma unroll
                for (int e = 32 * j / PV; e < 32 * (j + 1) / PV; e++) weigh_one(16 + e);
            } else {
                if (KT == 2 && j == FIRST) pair(30);
#pragma unroll
                for (int e = ALL * (j - FIRST) / (PV - FIRST); e < ALL * (j + 1 - FIRST) / (PV - FIRST); e++)
                    peak = fmaxf(peak, next[e / 16][e % 16]);
                asm volatile("" : "+v"(peak));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        sum += odd;
        float x, y;
        swap_pair<32>(peak, x, y);
        return fmaxf(x, y) * c;
    }

    // What clear_unseen took out, for the rows that see it: the keys first .. last, one by one, each weight from
    // its own score.
    __device__ __forceinline__ void add_bad(bool many, const Tile &t, int kv, int first, int last, int base) {
        const auto &a = *again(many);
        const int h = (threadIdx.x & 63) >> 5, row = min(base + column, t.rows - 1) + t.first, token = row / a.group;
        const bf16 *query = a.q + (t.q0 + token) * a.q_stride + (kv * a.group + row - token * a.group) * D;
#pragma unroll 1
        for (int p = first; p <= last; p++) {
            const int64_t where = place(a.b, t.s, p);
            if (where < 0) continue;
            const bf16 *k = a.b.kc + where + kv * a.b.head_stride, *v = a.b.vc + where + kv * a.b.head_stride;
            float dot = 0.0f;
#pragma unroll 1
            for (int d = 0; d < D; d += 8) dot = dot8(ld16(query + d), ld16(k + d), dot);
            const bool seen = p <= position && (a.window <= 0 || p > position - a.window);
            // what a row does not see weighs 0 even where its score is no number
            const float weight = seen ? __builtin_amdgcn_exp2f(fmaf(dot, a.scale_log2, -top)) : 0.0f;
#pragma unroll
            for (int d = 0; d < D / 32; d++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const u32x2 x = *gptr((const u32x2 *)(v + 32 * d + 8 * r + 4 * h));
                    const float e[4] = {lo_f(x.x), hi_f(x.x), lo_f(x.y), hi_f(x.y)};
#pragma unroll
                    for (int n = 0; n < 4; n++)
                        o[d][4 * r + n] = fmaf(weight, seen && !(fabsf(e[n]) < INFINITY) ? e[n] : 0.0f, o[d][4 * r + n]);
                }
        }
    }
};

// Leaves a score of what a row does not see at -inf. bits: the lane's (Columns::sees and what is there).
__device__ __forceinline__ void hide(f32x16 &s, uint32_t bits) {
    const uint32_t mine = bits >> ((threadIdx.x & 32) / 8);
#pragma unroll
    for (int r = 0; r < 16; r++)
        if (!(mine >> ((r & 3) + 8 * (r >> 2)) & 1)) s[r] = -INFINITY;
}

// Four consecutive elements of an output row.
__device__ __forceinline__ void store4(bf16 *to, float a, float b, float c, float d) {
    *gptr((u32x2 *)to) = u32x2{pack2(a, b), pack2(c, d)};
}

// A workgroup's LDS: 512 D bytes of keys and values and little else.
template <int D, bool WHOLE>
struct Space {
    __align__(1024) char rows[512 * D];
    int64_t places[WHOLE ? 1 : 8][WHOLE ? 1 : 128];  // of each wave; many: for keys, then for values
    float tops[4][32], sums[4][32];        // few: of each wave's columns
    __align__(16) uint32_t present[2][4];  // many: which of each wave's rows are there
    int bad[4];
};

// ------------------------------------------------------------------------------------------
// few rows: at most 32 per sequence and kv head
// ------------------------------------------------------------------------------------------

// One token, or a few, over a long history: bound by the bytes of the keys and values. A workgroup takes a
// split's keys, each of its four waves a quarter of them with the same 32 columns and buffers of its own, so
// nothing waits between waves until their outputs are joined. A wave keeps 32 keys' rows and 32 values' rows in
// LDS: the next keys are requested once the scores are formed and the next values once they are summed, so
// that eight waves of a CU have about 100 KB under way. The columns that hold no row are multiplied all the same: the
// matrix unit is idle most of the time here, which also pays for the weights' remainders (EXACT).
// 64 tokens over up to 8448 positions, 32 heads on 8 of 128: 192 us with the join, 5.7 TB/s of keys and values (a
// 2 GiB copy: 4.8; the library's read probe: 7.2); one token over 40960: 34 us with a join of 5; one over 261, 16 heads
// on 8: 8.7 us, which are the launch, the sequence's and the page's lookups and three steps of a wave one after the
// other. Heads of 256, 16 on 4: 199 and 36 us for the first two, of 64 113 and 22.
// EXACT: with remainders. The result is then whether an output of the workgroup came out infinite or as no number.
// A remainder may be 0 or negative, and 0 or a negative number times an infinite value makes no number where the
// weight itself makes an infinity: such a workgroup does all of it again without remainders.
template <int D, bool WHOLE, bool EXACT>
__device__ __forceinline__ bool few_rows(const AttendArgs &a, int kv, const Tile &t, int unit, int z,
                                         Space<D, WHOLE> &space) {
    constexpr int ROWS = 32, BYTES = ROWS * 2 * D;
    typedef Pages<D, ROWS, ROWS, WHOLE, true> P;
    constexpr int LOADS = P::LOADS;
    const int w = wave_id(), lane = threadIdx.x & 63;
    const int begin = t.begin + z * a.chunk;
    const int end = z == a.n_split - 1 ? t.end : min(t.end, begin + a.chunk);
    const int steps = end > begin ? (end - begin + ROWS - 1) / ROWS : 0;
    const int s0 = (int)((int64_t)steps * w / 4), n = (int)((int64_t)steps * (w + 1) / 4) - s0;

    Columns<D> c;
    c.start(a, t, kv, 0);
    P pages(a.b, kv, begin + s0 * ROWS, 0, (LLM_LDS int64_t *)space.places[WHOLE ? 0 : w]);
    lds_char *keys = (lds_char *)space.rows + w * 2 * BYTES, *values = keys + BYTES;
    const unsigned key_at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)keys), value_at = key_at + BYTES;
    uint32_t there = 0;
    if (n > 0) {
        pages.look_up(false, t.s, 0);
        there = pages.there(0);
        pages.request(a.b.kc, 0, key_at);
        pages.request(a.b.vc, 0, value_at);
    }
    bool bad = false;
    for (int i = 0; i < n; i++) {
        const int at = begin + (s0 + i) * ROWS;
        const bool more = i + 1 < n;
        const bool edge = at < t.from || at + ROWS - 1 > t.to || there != ~0u;
        const uint32_t here = there;
        wait_loads<LOADS>();
        f32x16 s[1] = {c.scores(keys)};
        if (edge) hide(s[0], c.sees(at, a.window) & here);
        wait_lds();
        if (more) {
            pages.look_up(false, t.s, i + 1);
            there = pages.there(i + 1);
            pages.request(a.b.kc, i + 1, key_at);
        }
        c.raise(c.peak(s, a.scale_log2));
        u32x4 hi[2], lo[2];
        c.template weigh<EXACT>(s[0], a.scale_log2, hi, lo);
        if (more)
            wait_loads<LOADS>();
        else
            wait_loads<0>();
        if (edge) bad |= clear_unseen<D, LOADS>(values, at, here, t.from, t.to, t.least, t.most);
        c.template add<EXACT>(values, hi, lo);
        wait_lds();
        if (more) pages.request(a.b.vc, i + 1, value_at);
    }
    if (bad) {
        const int first = begin + s0 * ROWS, last = min(first + n * ROWS, t.end) - 1;
        c.add_bad(false, t, kv, max(first, t.least), min(last, t.from - 1), 0);
        c.add_bad(false, t, kv, max(max(first, t.least), max(t.from, t.to + 1)), min(last, t.most), 0);
    }

    // join the waves: each one's output, maximum and sum through LDS
    float x, y;
    swap_pair<32>(c.sum, x, y);
    if (EXACT && threadIdx.x == 0) space.bad[0] = 0;  // the second time waves may still have to read it
    __syncthreads();
    if (lane < 32) {
        space.tops[w][lane] = c.top;
        space.sums[w][lane] = x + y;
    }
    constexpr int CHUNKS = D / 4;  // of four elements, chunk k of a column at k ^ (column & 15)
    LLM_LDS f32x4 *joined = (LLM_LDS f32x4 *)(lds_char *)space.rows;
    if (c.column < t.rows) {
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int k = 8 * d + 2 * r + (lane >> 5);
                joined[(w * 32 + c.column) * CHUNKS + (k ^ (c.column & 15))] =
                    f32x4{c.o[d][4 * r], c.o[d][4 * r + 1], c.o[d][4 * r + 2], c.o[d][4 * r + 3]};
            }
    }
    __syncthreads();
    const int64_t at = ((int64_t)unit * a.n_split + z) * FEW;
    for (int i = threadIdx.x; i < t.rows * CHUNKS; i += 256) {
        const int row = i / CHUNKS, k = i % CHUNKS;
        float top = space.tops[0][row];
#pragma unroll
        for (int v = 1; v < 4; v++) top = fmaxf(top, space.tops[v][row]);
        float sum = 0.0f;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const float f = __builtin_amdgcn_exp2f(space.tops[v][row] - top);
            sum = fmaf(f, space.sums[v][row], sum);
            const f32x4 e = joined[(v * 32 + row) * CHUNKS + (k ^ (row & 15))];
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = fmaf(f, e[j], o[j]);
        }
        if constexpr (EXACT) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (!(fabsf(o[j]) < INFINITY)) space.bad[0] = 1;
        }
        if (t.active > 1) {
            *gptr((f32x4 *)(a.part + (at + row) * D + 4 * k)) = o;
            if (k == 0) {
                gptr(a.stats)[(at + row) * 2] = top;
                gptr(a.stats)[(at + row) * 2 + 1] = sum;
            }
        } else {
            const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int r = t.first + row, token = r / a.group;
            store4(a.out + (t.q0 + token) * a.out_stride + (kv * a.group + r - token * a.group) * D + 4 * k, o[0] * f,
                   o[1] * f, o[2] * f, o[3] * f);
        }
    }
    if constexpr (!EXACT) return false;
    __syncthreads();
    return space.bad[0] != 0;
}

template <int D, bool WHOLE>
__device__ __forceinline__ void attend_few(const AttendArgs &a, int unit, int z, Space<D, WHOLE> &space) {
    const int tile = unit / a.n_kv_heads, kv = unit - tile * a.n_kv_heads;
    Tile t;
    if (!find_tile<FEW>(a, a.which, tile, t) || z >= t.active) return;
    if (few_rows<D, WHOLE, true>(a, kv, t, unit, z, space)) few_rows<D, WHOLE, false>(a, kv, t, unit, z, space);
}

// ------------------------------------------------------------------------------------------
// many rows
// ------------------------------------------------------------------------------------------

// A chunk of new tokens: bound by the matrix products. The four waves of a workgroup take 32 columns each and
// share the keys and values in LDS, two buffers of NK rows: while one is used the other is filled, a quarter by
// each wave, with one barrier per NK keys. Two workgroups share a CU (heads of 256: one), so that one's products
// run beside the other's lookups and barriers.
// 2048 tokens after 6144, 32 heads on 8 of 128: 227 to 244 us (card to card), 1.0 PFLOP/s (a product of two 8192 x 8192
// matrices: 1.2, of larger ones 1.37). What bounds it then is power: the clock falls to 1.75 GHz, and the same call on zeros takes
// 199 us at 2.35. Of the 240 us, without the loads into LDS 30 less, without the softmax 20 less. Two groups of 32
// columns per wave would halve the LDS reads, but need the second half of the register file, which vector
// instructions cannot use: 453 us. As it is six registers are spilled, outside the loop; pages of other sizes than
// multiples of 16 take 14, of which a step reads two, and a lookup's result from LDS before every load: 337 us with
// pages of 24, 347 with pages of one. Heads of 64: 143 to 152 us for the same rows, bound by the softmax's vector
// work; of 256 (16 on 4) 333, with one workgroup per CU, so nothing runs beside a wait.
template <int D, bool WHOLE>
__device__ __forceinline__ void attend_many(const AttendArgs &a, int unit, int z, Space<D, WHOLE> &space) {
    constexpr int NK = D == 256 ? 32 : 64, KT = NK / 32, BYTES = NK * 2 * D;
    typedef Pages<D, NK / 4, NK, WHOLE, false> P;
    constexpr int LOADS = P::LOADS;
    static_assert(2 * LOADS == KT * D / 32, "as many loads as Columns::step asks for");
    const int w = wave_id(), lane = threadIdx.x & 63;
    const int tile = unit / a.n_kv_heads, kv = unit - tile * a.n_kv_heads;
    Tile t;
    if (!find_tile<MANY>(a, a.which, tile, t) || z >= t.active) return;
    const int begin = t.begin + z * a.chunk;
    const int end = z == a.n_split - 1 ? t.end : min(t.end, begin + a.chunk);
    const int n = end > begin ? (end - begin + NK - 1) / NK : 0;

    Columns<D> c;
    c.start(a, t, kv, 32 * w);
    const bool any_rows = 32 * w < t.rows;
    const int first = begin + w * (NK / 4), window = a.window;
    const float scale = a.scale_log2;
    const bf16 *kc = a.b.kc, *vc = a.b.vc;
    P kp(a.b, kv, first, w * (NK / 4), (LLM_LDS int64_t *)space.places[WHOLE ? 0 : w]);
    P vp(a.b, kv, first, w * (NK / 4), (LLM_LDS int64_t *)space.places[WHOLE ? 0 : 4 + w]);
    const unsigned mine = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_char *)space.rows) + w * (BYTES / 4);
    constexpr int QUARTER = NK / 4;  // the rows that a wave brings
    lds_char *keys = (lds_char *)space.rows, *values = keys + 2 * BYTES;  // two buffers each
    f32x16 scores[2][KT];
    float peak = LOWEST;  // of the step's scores, as long as none is hidden
    bool bad = false;
    // Every row of the workgroup sees all of the steps plain0 .. plain1 - 1 as far as it is there.
    const int plain0 = max(0, t.from - begin + NK - 1) / NK, plain1 = (t.to + 1 - begin) / NK;
    int groups = 0;      // WHOLE: which quarters of the lane's step are there
    bool whole = false;  // WHOLE: all of the steps looked up that are plain
    const auto look_up_values = [&](int i) {
        if constexpr (WHOLE) {
            if (i % P::AHEAD != 0) return;
            const auto &b = again(true)->b;
            int64_t at[4];
            groups = 0;
#pragma unroll
            for (int v = 0; v < 4; v++) at[v] = place(b, t.s, begin + (i + lane) * NK + v * QUARTER);
#pragma unroll
            for (int v = 0; v < 4; v++) {
                if (at[v] >= 0) groups |= 1 << v;
                if (v == w) vp.set(at[v]);
            }
            whole = !__any(groups != 15 && i + lane >= plain0 && i + lane < plain1);
        } else {
            vp.look_up(true, t.s, i);
        }
    };
    if (n > 0) {
        look_up_values(0);
        if constexpr (WHOLE) {
            kp.mine = vp.mine;
            kp.present = vp.present;
        } else {
            kp.look_up(true, t.s, 0);
        }
        kp.request(kc, 0, mine);
        vp.request(vc, 0, mine + 2 * BYTES);
        wait_loads<LOADS>();  // the keys
        __syncthreads();
        if (n > 1) {
            kp.look_up(true, t.s, 1);
            kp.request(kc, 1, mine + BYTES);
        }
#pragma unroll
        for (int k = 0; k < KT; k++) scores[0][k] = c.scores(keys + k * 32 * 2 * D);
        peak = c.peak(scores[0], scale);
    }
    const auto step = [&](auto which, int i) {
        constexpr int B = decltype(which)::value;
        f32x16(&s)[KT] = scores[B], (&next)[KT] = scores[B ^ 1];
        const int at = begin + i * NK;
        const bool plain = whole && i >= plain0 && i < plain1;
        int there = 0;  // WHOLE: the step's quarters
        wait_loads<0>();
        if (!plain) {
            uint32_t own;
            if constexpr (WHOLE) {
                there = __builtin_amdgcn_readlane(groups, i % P::AHEAD);
                own = there >> w & 1 ? (1u << QUARTER) - 1 : 0;
            } else {
                own = vp.there(i);
                if (lane == 0) space.present[B][w] = own;
            }
            bad |= clear_unseen<D, LOADS>(values + B * BYTES + w * (BYTES / 4), at + w * QUARTER, own, t.from, t.to, t.least,
                                          t.most);
        }
        __syncthreads();
        // later steps' keys and values; past the last one its own again
        const int next_values = min(i + 1, n - 1), next_keys = min(i + 2, n - 1);
        if ((i + 1) % P::AHEAD == 0 && i + 1 < n) look_up_values(i + 1);
        if ((i + 2) % P::AHEAD == 0 && i + 2 < n) kp.look_up(true, t.s, i + 2);
        const char *key_base = kp.base(kc, next_keys), *value_base = vp.base(vc, next_values);
        const auto bring = [&](int l) {
            if (l < LOADS)
                kp.load(key_base, next_keys, l, mine + B * BYTES);
            else
                vp.load(value_base, next_values, l - LOADS, mine + (2 + (B ^ 1)) * BYTES);
        };
        if (!any_rows) {
#pragma unroll
            for (int l = 0; l < 2 * LOADS; l++) bring(l);
            return;
        }
        if (!plain) {
#pragma unroll
            for (int k = 0; k < KT; k++) {
                uint32_t here = 0;
                constexpr int PARTS = 32 / QUARTER;  // waves whose rows make 32
#pragma unroll
                for (int v = 0; v < PARTS; v++) {
                    const uint32_t rows = WHOLE ? there >> (k * PARTS + v) & 1 ? (1u << QUARTER) - 1 : 0
                                                : space.present[B][k * PARTS + v];
                    here |= rows << (v * QUARTER);
                }
                hide(s[k], c.sees(at + 32 * k, window) & here);
            }
            peak = c.peak(s, scale);
        }
        c.raise(peak);
        // the next scores' products run beside this softmax (past the last keys, on what the buffer holds)
        const lds_char *ahead = keys + (B ^ 1) * BYTES;
        peak = c.step(ahead, values + B * BYTES, s, next, scale, bring);
    };
    for (int i = 0; i < n; i += 2) {
        step(std::integral_constant<int, 0>(), i);
        if (i + 1 < n) step(std::integral_constant<int, 1>(), i + 1);
    }
    wait_loads<0>();
    if (lane == 0) space.bad[w] = bad;
    __syncthreads();
    if (space.bad[0] | space.bad[1] | space.bad[2] | space.bad[3]) {
        const int last = min(begin + n * NK, t.end) - 1;
        c.add_bad(true, t, kv, max(begin, t.least), min(last, t.from - 1), 32 * w);
        c.add_bad(true, t, kv, max(max(begin, t.least), max(t.from, t.to + 1)), min(last, t.most), 32 * w);
    }

    if (!any_rows || c.column >= t.rows - 32 * w) return;
    float x, y;
    swap_pair<32>(c.sum, x, y);
    const float sum = x + y;
    const int h = lane >> 5, row = 32 * w + c.column;
    if (t.active > 1) {
        const int64_t at = ((int64_t)unit * a.n_split + z) * MANY + row;
        if (h == 0) {
            gptr(a.stats)[at * 2] = c.top;
            gptr(a.stats)[at * 2 + 1] = sum;
        }
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *gptr((f32x4 *)(a.part + at * D + 32 * d + 8 * r + 4 * h)) =
                    f32x4{c.o[d][4 * r], c.o[d][4 * r + 1], c.o[d][4 * r + 2], c.o[d][4 * r + 3]};
        return;
    }
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int r0 = t.first + row, token = r0 / a.group;
    bf16 *to = a.out + (t.q0 + token) * a.out_stride + (kv * a.group + r0 - token * a.group) * D + 4 * h;
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            store4(to + 32 * d + 8 * r, c.o[d][4 * r] * f, c.o[d][4 * r + 1] * f, c.o[d][4 * r + 2] * f,
                   c.o[d][4 * r + 3] * f);
}

// ------------------------------------------------------------------------------------------
// the launch
// ------------------------------------------------------------------------------------------

// Workgroups of many rows first: they take longest, and those of few rows, where there are any, fill up beside
// them. (Kinds in turns put the few ones first into the places there are: two chunks beside 20 single tokens 71 us
// against 55, with warm caches; two windowed chunks, whose batch then had empty workgroups of few rows in
// between, 45 against 34.)
template <int D, bool WHOLE>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_kernel(LaunchArgs l) {
    __shared__ Space<D, WHOLE> space;
    const bool many = (int)blockIdx.x < l.many_groups;
    const int i = blockIdx.x - (many ? 0 : l.many_groups);
    if (many) {
        // A unit's splits one after the other, so that tiles that are not there come last (two chunks beside 20 single
        // tokens 61.5 us instead of 65.1); heads of 256, one workgroup to a CU, the splits' first pieces first (1024
        // tokens after 16000 in two splits 395 us instead of 412).
        // Where the device holds all of these workgroups at once, two to a CU, the second of a CU is as much
        // shorter as its first is longer
        int unit = D == 256 ? i % l.many_units : i / l.many_split;
        const int z = D == 256 ? i / l.many_units : i % l.many_split;
        if (l.mirrored && unit >= CUS) unit = l.many_units - 1 - (unit - CUS);
        attend_many<D, WHOLE>(l.many, unit, z, space);
    } else {
        attend_few<D, WHOLE>(l.few, i % l.few_units, i / l.few_units, space);
    }
}

// ------------------------------------------------------------------------------------------
// the splits' join
// ------------------------------------------------------------------------------------------

// A wave joins 256 / D rows, four elements of a row per lane, up to 8 splits' parts requested at a time and
// added in order. Few rows of many splits: the four waves of a workgroup take a quarter of the splits each and
// are joined in order through LDS; many rows of few splits: each wave takes rows of its own. The
// first parts, whose place does not depend on the sequence, requested in front of its lookup bring nothing (one token
// after 40960 / 4000, 64 after 6144: 34.8 / 12.6 / 25.7 us both ways; two chunks of 64 after 6144 36.1 instead of 34.6).
template <int D, int T>
__device__ __forceinline__ void join_tile(const AttendArgs &a, int unit, int part, int parts, f32x4 (&outs)[4][64],
                                          float (&tops)[4][64], float (&sums)[4][64]) {
    constexpr int CHUNKS = D / 4, ROWS = 64 / CHUNKS, U = 8;
    constexpr bool SHARED = T == FEW;
    const int tile = unit / a.n_kv_heads, kv = unit - tile * a.n_kv_heads;
    const int w = wave_id(), lane = threadIdx.x & 63, k = lane % CHUNKS;
    const int z0 = SHARED ? a.n_split * w / 4 : 0, upto = SHARED ? a.n_split * (w + 1) / 4 : a.n_split;
    u32x2 stats[U];
    f32x4 e[U];
    const auto request = [&](int row, int z) {
        const int64_t at = (int64_t)unit * a.n_split * T + row;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t from = at + (int64_t)min(z + u, a.n_split - 1) * T;
            stats[u] = *gptr((const u32x2 *)(a.stats + from * 2));
            e[u] = *gptr((const f32x4 *)(a.part + from * D + 4 * k));
        }
        // all of them requested before the first is waited for: otherwise each load goes where its part is added (one token
        // after 40960 36.8 us instead of 34.6, 64 after 6144 32.3 instead of 25.3)
        asm volatile(""
                     : "+v"(e[0]), "+v"(e[1]), "+v"(e[2]), "+v"(e[3]), "+v"(e[4]), "+v"(e[5]), "+v"(e[6]), "+v"(e[7]));
        static_assert(U == 8, "all of e stand there");
    };
    const int first = part * ROWS * (SHARED ? 1 : 4), own = (SHARED ? 0 : w * ROWS) + lane / CHUNKS;
    Tile t;
    if (!find_tile<T>(a, a.which, tile, t) || t.active <= 1) return;
    const int z1 = min(upto, t.active);
    for (int r0 = first; r0 < t.rows; r0 += parts * ROWS * (SHARED ? 1 : 4)) {
        const int row = r0 + own;
        float top = LOWEST, sum = 0.0f;
        f32x4 o = {0, 0, 0, 0};
        for (int z = z0; z < z1; z += U) {
            request(min(row, t.rows - 1), z);
            float m[U], n[U];
            float next = top;
#pragma unroll
            for (int u = 0; u < U; u++) {
                m[u] = z + u < z1 ? __uint_as_float(stats[u].x) : LOWEST;
                n[u] = z + u < z1 ? __uint_as_float(stats[u].y) : 0.0f;
                next = fmaxf(next, m[u]);
            }
            const float f = __builtin_amdgcn_exp2f(top - next);
            top = next;
            sum *= f;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] *= f;
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (z + u >= z1) break;
                const float g = __builtin_amdgcn_exp2f(m[u] - next);
                sum = fmaf(n[u], g, sum);
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = fmaf(e[u][j], g, o[j]);
            }
        }
        if constexpr (SHARED) {
            __syncthreads();  // the last rows' parts have been read
            outs[w][lane] = o;
            tops[w][lane] = top;
            sums[w][lane] = sum;
            __syncthreads();
            if (w != 0) continue;
            for (int v = 1; v < 4; v++) top = fmaxf(top, tops[v][lane]);
            sum = 0.0f;
            o = f32x4{0, 0, 0, 0};
            for (int v = 0; v < 4; v++) {
                const float g = __builtin_amdgcn_exp2f(tops[v][lane] - top);
                sum = fmaf(sums[v][lane], g, sum);
                const f32x4 e = outs[v][lane];
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = fmaf(e[j], g, o[j]);
            }
        }
        if (row >= t.rows) continue;
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int r = t.first + row, token = r / a.group;
        store4(a.out + (t.q0 + token) * a.out_stride + (kv * a.group + r - token * a.group) * D + 4 * k, o[0] * f,
               o[1] * f, o[2] * f, o[3] * f);
    }
}

template <int D>
__global__ __launch_bounds__(256) void attend_join_kernel(LaunchArgs l, int few_parts, int many_parts) {
    __shared__ f32x4 outs[4][64];
    __shared__ float tops[4][64], sums[4][64];
    const int few = l.few.n_split > 1 ? l.few_units * few_parts : 0;
    int i = blockIdx.x;
    if (i < few) {
        join_tile<D, FEW>(l.few, i / few_parts, i % few_parts, few_parts, outs, tops, sums);
    } else {
        i -= few;
        join_tile<D, MANY>(l.many, i / many_parts, i % many_parts, many_parts, outs, tops, sums);
    }
}

// ------------------------------------------------------------------------------------------
// the host
// ------------------------------------------------------------------------------------------

// How the work is split, from the host's sizes alone. A sequence's rows (new tokens x group) go to attend_few
// up to FEW and to attend_many above, or all to one of them where the expected lengths leave the other nothing.
struct Plan {
    bool few, many;
    int64_t few_units, many_units;  // tiles x kv heads, at most
    int few_split, few_chunk, many_split, many_chunk;
    size_t few_rows, many_rows;  // rows of partial outputs

    // Parts (units x splits) of a call that splits at most, so that the workspace stays within 68 MB and 136 MB (heads of
    // 128) however many sequences or rows there are: the device is full long before. (Single tokens of 256 / 512 / 1024
    // sequences of up to 8192, 32 heads on 8 of 128, in 4 splits 779 / 1512 / 3100 us, with 4096 parts at most 752 / 1425 /
    // 2853, with 2048 741 / 1445 / 2819; 128 sequences 394 / 394 / 412. Chunks of 2080 after 6112 / 2400 after 14000 / 6160
    // after 2000, by the estimate alone 327 / 670 / 616 us, with 4096 parts 326 / 672 / 685, with 2048 295 / 633 / 507, with
    // 1024 305 / 669 / 507; 1056 after 7136 179 / 179 / 178 / 193.)
    static constexpr int64_t FEW_PARTS = 4096, MANY_PARTS = 2048;
    static constexpr int64_t UNSPLIT = 640, MOST_SPLITS = 64;  // keys that few rows never split; splits of many rows

    // Floats of workspace that the plans of these sizes, and of any with fewer tokens or sequences or with less
    // expected of them, take at most: every term is one that does not fall as they grow.
    static size_t floats(int n_tokens, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_q_len,
                         int max_kv_len) {
        const int64_t group = n_heads / n_kv_heads, rows = n_tokens * group, seqs = std::min(n_seqs, n_tokens);
        const int64_t pieces = ((int64_t)max_kv_len + 127) / 128;
        const auto parts = [&](int64_t tile, int64_t splits, int64_t most) {
            splits = std::min(splits, pieces);
            return splits > 1 ? std::min(most, (rows + (tile - 1) * seqs) / tile * n_kv_heads * splits) : 0;
        };
        const int64_t few_most = max_kv_len <= UNSPLIT ? 1
                                 : n_seqs > 1 ? std::max<int64_t>(2 * CUS / n_kv_heads, (pieces + 7) / 8)
                                              : CUS / n_kv_heads;
        const int64_t few = parts(FEW, few_most, FEW_PARTS);
        const int64_t many = std::min(max_q_len, n_tokens) * group > FEW ? parts(MANY, MOST_SPLITS, MANY_PARTS) : 0;
        return (size_t)(few * FEW + many * MANY) * (head_dim + 2);
    }

    // A join costs 2 to 3 us, what a workgroup takes for about 600 keys alone (one token, 32 heads on 8, 511 / 639 / 1023 /
    // 4095 positions: unsplit 9.8 / 10.9 / 16.4 / 46.1 us, in pieces of 128 keys 11.1 / 11.8 / 12.2 / 13.3; 40959 positions
    // in 256 workgroups 34.5, in 512 35.7). Several sequences, which may be of
    // unequal length, take twice the workgroups (4 / 8 / 16 of up to 2000, 256 workgroups 14.0 / 16.3 / 22.7, 512 14.0 /
    // 16.5 / 22.5), in pieces of 1024 keys, or 2048 where there are enough of those (16 of up to 8000, pieces of 2048 /
    // 1024: 62.5 / 54.6; 64 of up to 8447, whole / 2048 / 1024: 217 / 195 / 195).
    static int64_t few_splits(int64_t units, int n_seqs, int64_t span) {
        if (span <= UNSPLIT) return 1;
        const int64_t target = n_seqs > 1 ? 2 * CUS : CUS, piece = units <= CUS ? 1024 : 2048;
        return std::max<int64_t>(
            1, std::min((span + 127) / 128, std::max(target / units, n_seqs > 1 ? (span + piece - 1) / piece : 1)));
    }

    // The least of an estimate in ns: a workgroup's keys (alone on a CU; beside another from CUS workgroups on; past
    // two to a CU in turns), the parts' bytes written and read, and the join. Beside workgroups of few rows at most
    // `most`. Over 123 shapes (33 to 2048 tokens after 0 to 16000, heads of 64, 128 and 256) what it chooses takes 0.4%
    // longer than the best of those measured, at most 6%. (32 heads on 8 of 128, in 1 / 2 / 4 / 8 / 16 splits: 64 tokens
    // after 6144 103 / 63 / 41 / 30 / 27 us, 512 after 6144 110 / 78 / 75 / 91 / 109, 1024 after none 28 / 38 / 53 / 51 / 51.)
    static int64_t many_splits(int64_t units, int head_dim, int64_t span, int64_t most) {
        int64_t best = 1;
        double least = 0;
        for (int64_t n = 1; n <= std::min<int64_t>(most, (span + 127) / 128); n++) {
            const double groups = (double)units * n, keys = (double)((span + n - 1) / n);
            const double shared = groups <= CUS       ? 1.0
                                  : groups <= 2 * CUS ? 1.3 + 0.55 * (groups - CUS) / CUS
                                                      : 1.85 * ceil(groups / (2 * CUS));
            const double key = head_dim == 256 ? 39.0 * ceil(groups / CUS) : 16.3 * shared * (head_dim + 64) / 192;
            const double cost = keys * key + (n > 1 ? 8000 + groups * 128 * (head_dim + 2) * 8 / 10000 : 0);
            if (n == 1 || cost < least) best = n, least = cost;
        }
        return best;
    }

    Plan(int n_tokens, int n_seqs, int n_heads, int n_kv_heads, int head_dim, int max_q_len, int max_kv_len,
         int window) {
        const int64_t group = n_heads / n_kv_heads, rows = n_tokens * group;
        const int64_t longest = std::min<int64_t>(max_q_len, n_tokens) * group;
        many = longest > FEW;
        // with sequences of at most FEW / group tokens of few rows and the others of at most max_q_len, this many
        // at least have many rows: where that is all of them, all go to attend_many (one that is short after all
        // takes longer there, and its weights have no remainders)
        const int64_t tokens = FEW / group, rest = n_tokens - n_seqs * tokens;
        few = !many || (n_seqs > 1 && rest <= (int64_t)(n_seqs - 1) * (max_q_len - tokens));
        // r rows of a sequence make at most (r + T - 1) / T tiles; one of many rows has over FEW. Empty workgroups
        // between the others would put two of those on a CU and none on another (with one tile too many 512 tokens
        // after 6144 in two splits 95 us instead of 78).
        const int64_t seqs = std::min(n_seqs, n_tokens);  // that have rows
        const int64_t few_tiles = many ? seqs : (rows + (FEW - 1) * seqs) / FEW;
        const int64_t long_seqs = few ? std::min(seqs, rows / (FEW + 1)) : seqs;
        const int64_t many_tiles = (rows + (MANY - 1) * long_seqs) / MANY;
        few_units = few ? few_tiles * n_kv_heads : 0;
        many_units = many ? many_tiles * n_kv_heads : 0;
        // a window shortens what the rows see; the workspace is asked for without it, so never more splits than then
        const auto cut = [&](int64_t tokens, auto splits, int &n, int &chunk) {
            n = INT32_MAX;
            for (const int64_t span : {(int64_t)max_kv_len, std::min<int64_t>(max_kv_len, window + tokens + 63)}) {
                const int64_t want = std::min<int64_t>(n, splits(span));
                chunk = (int)((span + want - 1) / want + 127) / 128 * 128;
                n = (int)((span + chunk - 1) / chunk);
                if (window == 0) break;
            }
        };
        // Workgroups of few rows need places of their own beside those of many. In at most 1 / 2 / 3 / 4 / 6 / 8 splits:
        // chunks of 511 and 71 after up to 4095 beside 20 single tokens, 16 heads on 8 of 128, 99 / 69 / 63 / 63 / 63 / 63
        // us; 32 on 8, 511 after 8000 beside 64 247 / 233 / 265 / 266 / 265 / 266, 128 after 4000 beside 8 81 / 52 / 43 /
        // 40 / 36 / 37, 256 after 16000 beside 16 312 / 184 / 147 / 146 / 149 / 154, two of 300 after 2000 beside 32
        // 62 / 52 / 59 / 59 / 59 / 59; 16 on 4 of 256, 256 after 8000 beside 8 339 / 183 / 129 / 105 / 93 / 92.
        const int64_t units = (rows + MANY - 1) / MANY * n_kv_heads, beside = few ? 288 / units : MOST_SPLITS;
        const int64_t few_most = std::max<int64_t>(1, FEW_PARTS / std::max<int64_t>(1, few_units));
        const int64_t many_most = std::max<int64_t>(1, std::min(beside, MANY_PARTS / std::max<int64_t>(1, many_units)));
        cut(FEW, [&](int64_t span) { return std::min(few_most, few_splits((int64_t)n_seqs * n_kv_heads, n_seqs, span)); },
            few_split, few_chunk);
        cut(MANY, [&](int64_t span) { return many_splits(units, head_dim, span, many_most); }, many_split, many_chunk);
        few_rows = few_split > 1 ? (size_t)few_units * few_split * FEW : 0;
        many_rows = many_split > 1 ? (size_t)many_units * many_split * MANY : 0;
    }
};

bool check_sizes(const char *name, int n_tokens, int n_heads, int max_q_len, int max_kv_len) {
    if (max_q_len <= 0 || max_kv_len <= 0)
        return llm_fail("%s: max_q_len %d and max_kv_len %d must be positive", name, max_q_len, max_kv_len);
    if (max_kv_len > 1 << 30) return llm_fail("%s: max_kv_len %d is over 1073741824", name, max_kv_len);
    if ((int64_t)n_tokens * n_heads > INT32_MAX / 2)
        return llm_fail("%s: %d rows of %d heads are too many", name, n_tokens, n_heads);
    return true;
}

template <int D, bool WHOLE>
void launch_attention(const AttendArgs &a, const Plan &p, float *ws, int max_q_len, hipStream_t stream) {
    LaunchArgs l;
    l.few = l.many = a;
    l.few.part = ws;
    l.few.stats = ws + p.few_rows * D;
    l.many.part = l.few.stats + p.few_rows * 2;
    l.many.stats = l.many.part + p.many_rows * D;
    l.few.n_split = p.few_split;
    l.few.chunk = p.few_chunk;
    l.many.n_split = l.many_split = p.many_split;
    l.many.chunk = p.many_chunk;
    l.few.which = p.many ? FEW_ROWS : ALL_ROWS;
    l.many.which = p.few ? MANY_ROWS : ALL_ROWS;
    l.few_units = (int)p.few_units;
    l.many_units = (int)p.many_units;
    l.few_groups = l.few_units * p.few_split;
    l.many_groups = l.many_units * p.many_split;
    l.mirrored = !p.few && p.many_split == 1 && p.many_units > CUS && p.many_units <= 2 * CUS;
    attend_kernel<D, WHOLE><<<l.few_groups + l.many_groups, 256, 0, stream>>>(l);
    if (!LAUNCH_OK()) return;
    constexpr int ROWS = 256 / D;  // of a wave of the join
    // workgroups per tile: those of few rows mostly hold one token's
    const int expected = (int)std::min<int64_t>(FEW, p.many ? a.group : (int64_t)max_q_len * a.group);
    const int few_parts = (expected + ROWS - 1) / ROWS, many_parts = MANY / (8 * ROWS);
    const int joins = (p.few_split > 1 ? l.few_units * few_parts : 0) + (p.many_split > 1 ? l.many_units * many_parts : 0);
    if (joins > 0) {
        attend_join_kernel<D><<<joins, 256, 0, stream>>>(l, few_parts, many_parts);
        LAUNCH_OK();
    }
}

}  // namespace

extern "C" size_t attention_paged_workspace_floats(int n_tokens, int n_seqs, int n_heads, int n_kv_heads, int head_dim,
                                                   int max_q_len, int max_kv_len) {
    static const char name[] = "attention_paged_workspace_floats";
    if (n_tokens < 0 || n_tokens > 1 << 24 || n_seqs <= 0 || n_seqs > 1 << 20 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads ||
        (head_dim != 64 && head_dim != 128 && head_dim != 256)) {
        llm_fail("%s: no attention of %d rows in %d sequences, %d heads on %d of %d", name, n_tokens, n_seqs, n_heads,
                 n_kv_heads, head_dim);
        return 0;
    }
    if (!check_sizes(name, n_tokens, n_heads, max_q_len, max_kv_len)) return 0;
    if (n_tokens == 0) return 0;
    return Plan::floats(n_tokens, n_seqs, n_heads, n_kv_heads, head_dim, max_q_len, max_kv_len);
}

extern "C" void attention_paged_forward(bf16 *out, const bf16 *q, const PagedBatch *batch, float *ws, int n_tokens,
                                        int n_heads, int max_q_len, int max_kv_len, int window, float scale,
                                        int64_t out_stride, int64_t q_stride, hipStream_t stream) {
    static const char name[] = "attention_paged";
    AttendArgs a;
    if (!take_batch(name, batch, n_tokens, n_heads, &a.b)) return;
    if (!check_sizes(name, n_tokens, n_heads, max_q_len, max_kv_len)) return;
    if (n_tokens == 0) return;
    if (window < 0) {
        llm_fail("%s: window %d is negative", name, window);
        return;
    }
    if (window >= 1 << 30) window = 0;  // past every position; positions less the window then stay in range
    if (!(scale > 0.0f) || !isfinite(scale * 1.44269504f)) {
        llm_fail("%s: scale %g is not positive and finite", name, (double)scale);
        return;
    }
    const int D = batch->head_dim;
    const int64_t width = (int64_t)n_heads * D;
    if (!check_rows(name, "out", out, out_stride, width) || !check_rows(name, "q", q, q_stride, width)) return;
    const Plan plan(n_tokens, batch->n_seqs, n_heads, batch->n_kv_heads, D, max_q_len, max_kv_len, window);
    // a launch has less than 2^32 threads; the join, of units that are split, stays far below
    if (plan.few_units * plan.few_split + plan.many_units * plan.many_split >= 1 << 24) {
        llm_fail("%s: %d rows in %d sequences of up to %d tokens are too many for one launch", name, n_tokens,
                 batch->n_seqs, max_kv_len);
        return;
    }
    if (!aligned16(ws) || (plan.few_rows + plan.many_rows && !ws)) {
        llm_fail("%s: ws must be a 16-byte aligned device address", name);
        return;
    }
    if (out == q) {
        llm_fail("%s: out must not be q, which is read again", name);
        return;
    }
    a.out = out;
    a.q = q;
    a.out_stride = out_stride;
    a.q_stride = q_stride;
    a.n_heads = n_heads;
    a.n_kv_heads = batch->n_kv_heads;
    a.group = n_heads / batch->n_kv_heads;
    a.window = window;
    a.scale_log2 = scale * 1.44269504f;
    const bool whole = batch->page_size % 16 == 0;
#define ATTEND(D_)                                      \
    if (D == D_) {                                      \
        if (whole)                                      \
            launch_attention<D_, true>(a, plan, ws, max_q_len, stream);  \
        else                                            \
            launch_attention<D_, false>(a, plan, ws, max_q_len, stream); \
    }
    ATTEND(64) ATTEND(128) ATTEND(256)
#undef ATTEND
}
