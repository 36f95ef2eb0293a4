// A projection of many rows with the low-rank adapters of their sequences (include/llm_amd/batch.h).
//
// out = x Wt + low Bt, low = scale x At: the second term is the first one's sum carried on over the rank, with rows
// of `low` for rows of x and an adapter's b for W. low is kept as two bf16, the value and what that leaves (16 bits
// of mantissa), side by side, so the sum goes over twice the rank.
//
// A call takes one of four ways, the first by its size, the others by the estimate in Plan:
//   one or two rows, little rank and a small W: one launch, in which each workgroup computes low for itself;
//   many rows, where the product's operations count: low, then one product whose last steps are the adapters';
//   few rows, where W's bytes and the launches count: parts of the product's sum and, in the same launch behind them,
//   of low's; then join_kernel adds the parts up, with b's product and the residual;
//   without adapters: the product, and sum_kernel where its sum is split.
// 64 rows of 4096 over 2560, each with one of 48 adapters of rank 16, take 14 us (the product alone, from a library:
// 19.3), 2582 rows of five prompts of 9728 over 2560, rank 32, 132 to 143 (115), 924 rows of 22 sequences of 2560 over 9728,
// rank 64, 80 to 84 (66).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "internal.h"
#include "llm_amd/batch.h"

using namespace llm;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

#define LLM_LDS __attribute__((address_space(3)))
typedef LLM_LDS char lds_char;

constexpr int CUS = 256, XCDS = 8;
constexpr int NO_ADAPTER = -1, NO_SEQUENCE = -2;

struct LoraArgs {
    bf16 *out;
    const bf16 *x, *w, *residual;
    const bf16 *a, *b;       // a null: no adapters, every row is of one sequence
    const float *scale;
    const int *q_start, *adapter;
    bf16 *low;               // [n_tokens, 2 rank]: value, remainder
    float *low_part;         // [low_splits, n_tokens, rank]: its parts, without the scale
    int *owner;              // [n_tokens]: the row's adapter, NO_ADAPTER or NO_SEQUENCE
    float *part;             // [splits, n_tokens, part_width], or null: straight to out
    int64_t out_stride, x_stride, residual_stride;
    int n_tokens, n_out, n_in, n_seqs, n_adapters, rank;
    int part_width;
    int splits, split_steps;  // of the product's sum, steps of 64 each
    int m_tiles, n_tiles;
    int low_groups, low_splits;  // workgroups behind the product's that compute low_part; its parts
    int wide;                // elements of out and residual that lie in aligned memory from each multiple of it on: 8, 4, 1
};

// What is loaded for places past an operand's end.
__device__ const u32x4 g_zeros = {0, 0, 0, 0};

__device__ __forceinline__ f32x4 mfma(const u32x4 &a, const u32x4 &b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                   0, 0);
}

// 64 lanes' 16 bytes into LDS at `to` on, without passing registers: the wave waits for it with wait_loads.
// (m0 is reserved: it cannot be named as written, and the compiler has no use for it in these kernels.)
template <bool STREAM = false>
__device__ __forceinline__ void load_to_lds(unsigned to, const void *base, unsigned offset) {
    if constexpr (STREAM)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(to), "v"(offset), "s"(base) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void load_to_lds(unsigned to, const void *at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(at) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// A builtin, so that the compiler knows that what was read is there and does not wait for newer reads in its place.
__device__ __forceinline__ void wait_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// ------------------------------------------------------------------------------------------
// the rows' sequences
// ------------------------------------------------------------------------------------------

__device__ __forceinline__ int start_of(const LoraArgs &l, int s) {
    return max(0, min(l.n_tokens, gptr(l.q_start)[s]));
}

// What low_part wrote for row m. Starts that decrease, which no call may have, leave rows that it wrote nothing for: what is
// there from before is kept to the adapters that there are, so that it leads to no address outside of the call's tensors.
__device__ __forceinline__ int owner_of(const LoraArgs &l, int m) {
    const int owner = gptr(l.owner)[m];
    return owner >= NO_SEQUENCE && owner < l.n_adapters ? owner : NO_SEQUENCE;
}

// R rows of one sequence at most. A sequence of n rows from f on has at most (f + n) / R - f / R + 1 tiles, so those
// of sequence s are found from f / R + s on, of n_tokens / R + n_seqs.
struct RowTile {
    int first, rows, adapter;  // rows 0: no tile
};
template <int R>
__device__ __forceinline__ RowTile row_tile(const LoraArgs &l, int i) {
    RowTile t = {0, 0, NO_ADAPTER};
    const int lane = threadIdx.x & 63;
    int s0 = 0;  // the sequence is among the 64 from s0 on, which are read at once
    if (l.n_seqs > 64) s0 = max(0, count_leading(l.n_seqs, [&](int j) { return start_of(l, j) / R + j <= i; }) - 1);
    const int s = min(s0 + lane, l.n_seqs - 1);
    const int f = start_of(l, s), n = start_of(l, s + 1) - f, adapter = gptr(l.adapter)[s];
    const uint64_t upto = __ballot(s0 + lane < l.n_seqs && f / R + s <= i);
    if (!upto) return t;
    const int at = 63 - __builtin_clzll(upto);
    const int first = __builtin_amdgcn_readlane(f, at), rows = __builtin_amdgcn_readlane(n, at), a = __builtin_amdgcn_readlane(adapter, at);
    const int j = i - (first / R + s0 + at);
    t.first = first + R * j;
    t.rows = max(0, min(R, rows - R * j));
    if ((unsigned)a < (unsigned)l.n_adapters) t.adapter = a;
    return t;
}

// ------------------------------------------------------------------------------------------
// low
// ------------------------------------------------------------------------------------------

// A part of low, over SPAN elements of its sum per wave, of 16 MT rows and 16 NT elements of the rank.
template <int MT, int NT, int WAVES, int SPAN>
__device__ __forceinline__ void low_sums(const LoraArgs &l, const RowTile &t, int r0, int split, float *sums) {
    constexpr int U = MT == 1 && NT < 4 ? SPAN / 32 : 4;  // loads of each row under way
    constexpr int ROW = 16 * NT;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const bf16 *a = l.a + (int64_t)t.adapter * l.rank * l.n_in, *x[MT], *row[NT];
#pragma unroll
    for (int i = 0; i < MT; i++) x[i] = l.x + (t.first + min(i * 16 + lane % 16, t.rows - 1)) * l.x_stride;
#pragma unroll
    for (int j = 0; j < NT; j++) row[j] = a + (int64_t)min(r0 + j * 16 + lane % 16, l.rank - 1) * l.n_in;
    const int begin = (split * WAVES + wave) * SPAN, end = min(l.n_in, begin + SPAN);
    f32x4 acc[MT][NT] = {};
    for (int k0 = begin; k0 < end; k0 += 32 * U) {
        u32x4 xs[U][MT], as[U][NT];
        const auto request = [&](const bf16 *p, int u) {
            const int k = k0 + 32 * u + lane / 16 * 8;
            return k < end ? ld16(p + k) : u32x4{0, 0, 0, 0};
        };
        // the halves of a line one after the other
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int u = 0; u < U; u++) xs[u][i] = request(x[i], u);
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int u = 0; u < U; u++) as[u][j] = request(row[j], u);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) acc[i][j] = mfma(as[u][j], xs[u][i], acc[i][j]);
    }
    // rows 16 bytes further apart: side by side those of a product's 16 would meet in the same banks
    constexpr int ALL = 16 * MT * (ROW + 4);
    float *mine = sums + wave * ALL;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) *(f32x4 *)(mine + (i * 16 + lane % 16) * (ROW + 4) + j * 16 + lane / 16 * 4) = acc[i][j];
    __syncthreads();
    float *to = l.low_part + ((int64_t)split * l.n_tokens + t.first) * l.rank + r0;
    for (int i = 4 * threadIdx.x; i < 16 * MT * ROW; i += 4 * 64 * WAVES) {
        const int m = i / ROW, r = i % ROW;
        if (m >= t.rows || r0 + r >= l.rank) continue;
        f32x4 y = {0, 0, 0, 0};
        for (int w = 0; w < WAVES; w++) y += *(const f32x4 *)(sums + w * ALL + m * (ROW + 4) + r);
        *gptr((f32x4 *)(to + (int64_t)m * l.rank + r)) = y;
    }
}
__host__ __device__ __forceinline__ int low_width(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }

// A part of low of R rows, in 32 bits and without the scale; and the rows' owners.
template <int R, int WAVES, int SPAN>
__device__ __forceinline__ void low_part(const LoraArgs &l, int block, float *lds) {
    const int width = low_width(l.rank), groups = (l.rank + width - 1) / width;
    const int split = block % l.low_splits, r0 = block / l.low_splits % groups * width;
    const int tile = block / l.low_splits / groups;
    const RowTile t = row_tile<R>(l, tile);
    if (split == 0 && r0 == 0) {
        if (tile == 0) {
            const int begin = start_of(l, 0), end = max(begin, start_of(l, l.n_seqs));
            for (int i = threadIdx.x; i < l.n_tokens; i += 64 * WAVES)
                if (i < begin || i >= end) gptr(l.owner)[i] = NO_SEQUENCE;
        }
        if ((int)threadIdx.x < t.rows) gptr(l.owner)[t.first + threadIdx.x] = t.adapter;
    }
    if (t.rows == 0 || t.adapter < 0) return;
    const auto sum = [&](auto mt) {
        constexpr int MT = decltype(mt)::value;
        if (width == 16) low_sums<MT, 1, WAVES, SPAN>(l, t, r0, split, lds);
        else if (width == 32) low_sums<MT, 2, WAVES, SPAN>(l, t, r0, split, lds);
        else low_sums<MT, 4, WAVES, SPAN>(l, t, r0, split, lds);
    };
    if (t.rows <= 16) sum(std::integral_constant<int, 1>{});
    else sum(std::integral_constant<int, R / 16>{});
}

// Bound by its round trips, launch, starts, operands: 10 us for 2582 rows over 2560 and rank 32, 13 MB of x. (Unsplit, with
// sixteen waves a sum and low_sum_kernel's work at its end, a call took as long or, at rank 128, 5 us longer.)
// Elements of the sum per workgroup: of 64 rows so few that the workgroups fill the CUs, of 16 beside the product more,
// for fewer parts to add up.
constexpr int LOW_WAVES = 4, LOW_ROWS = 64, LOW_SPAN = 512, JOIN_LOW_SPAN = 1024;
__global__ __launch_bounds__(64 * LOW_WAVES) void low_kernel(LoraArgs l) {
    __shared__ __attribute__((aligned(16))) float sums[LOW_WAVES * LOW_ROWS * 68];
    low_part<LOW_ROWS, LOW_WAVES, LOW_SPAN / LOW_WAVES>(l, blockIdx.x, sums);
}

// Element i of a row's low: the parts in order, and the scale.
__device__ __forceinline__ f32x4 low_sum(const LoraArgs &l, int64_t at, float scale) {
    f32x4 y = {0, 0, 0, 0};
    constexpr int U = 4;
    for (int s0 = 0; s0 < l.low_splits; s0 += U) {
        f32x4 part[U];
#pragma unroll
        for (int s = 0; s < U; s++)
            part[s] = s0 + s < l.low_splits ? *gptr((const f32x4 *)(l.low_part + (int64_t)(s0 + s) * l.n_tokens * l.rank + at))
                                            : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < U; s++) y += part[s];
    }
    return y * scale;
}
// Two numbers as bf16, and what that leaves of them. Of finite ones past the largest bf16 that leaves less than 2^120, which
// is rounded by 2^111 at most, 2^-16 of the value.
__device__ __forceinline__ void in_two(float y0, float y1, uint32_t &value, uint32_t &rest) {
    constexpr float MOST = 0x1.fep127f;
    const bool finite0 = fabsf(y0) < INFINITY, finite1 = fabsf(y1) < INFINITY;
    const float v0 = finite0 ? fminf(fmaxf(y0, -MOST), MOST) : y0, v1 = finite1 ? fminf(fmaxf(y1, -MOST), MOST) : y1;
    value = pack2(v0, v1);
    rest = pack2(finite0 ? y0 - round_bf(v0) : 0.0f, finite1 ? y1 - round_bf(v1) : 0.0f);
}

// low from its parts: four elements per thread.
__global__ __launch_bounds__(256) void low_sum_kernel(LoraArgs l) {
    const int per = l.rank / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int m = (int)(i / per), r = (int)(i % per) * 4;
    if (m >= l.n_tokens) return;
    const int owner = owner_of(l, m);
    if (owner < 0) return;
    const f32x4 y = low_sum(l, (int64_t)m * l.rank + r, l.scale ? gptr(l.scale)[owner] : 1.0f);
    u32x2 value, rest;
    uint32_t v, w;
    in_two(y[0], y[1], v, w);
    value.x = v, rest.x = w;
    in_two(y[2], y[3], v, w);
    value.y = v, rest.y = w;
    bf16 *low = l.low + (int64_t)m * 2 * l.rank + r;
    *gptr((u32x2 *)low) = value;
    *gptr((u32x2 *)(low + l.rank)) = rest;
}

// Four columns of a row, with the residual's.
__device__ __forceinline__ void store4(const LoraArgs &l, bf16 *to, const bf16 *res, f32x4 y, int n) {
    if (l.wide >= 4 && n + 4 <= l.n_out) {
        if (l.residual) {
            const u32x2 v = *gptr((const u32x2 *)res);
            y += f32x4{lo_f(v.x), hi_f(v.x), lo_f(v.y), hi_f(v.y)};
        }
        *gptr((u32x2 *)to) = u32x2{pack2(y[0], y[1]), pack2(y[2], y[3])};
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < l.n_out) gptr(to)[e] = (bf16)f2bf(y[e] + (l.residual ? bf2f(gptr(res)[e]) : 0.0f));
    }
}

// Eight columns of a row, past the caches: the eight lanes side by side of a wave of 64 columns write whole lines so, those of
// 32 (tiles of 64 by 128) halves, of 16 (the smaller ones) quarters. 2582 rows of 9728 over 2560 take 135 us with such
// stores, 166 with four columns a lane of 16 rows at a time, through the caches (157 past them), and 161 with whole lines
// through the caches; 64 rows of 151936, in halves of lines, 148, 158, 156 and 156.
__device__ __forceinline__ void store8(const LoraArgs &l, bf16 *to, const bf16 *res, f32x4 y, f32x4 z, int n) {
    if (l.wide == 8 && n + 8 <= l.n_out) {
        if (l.residual) {
            const u32x4 v = *(gptr((const u32x4 *)res));
            y += f32x4{lo_f(v[0]), hi_f(v[0]), lo_f(v[1]), hi_f(v[1])};
            z += f32x4{lo_f(v[2]), hi_f(v[2]), lo_f(v[3]), hi_f(v[3])};
        }
        __builtin_nontemporal_store((u32x4{pack2(y[0], y[1]), pack2(y[2], y[3]), pack2(z[0], z[1]), pack2(z[2], z[3])}), gptr((u32x4 *)to));
    } else {
        store4(l, to, res, y, n);
        if (n + 4 < l.n_out) store4(l, to + 4, res + 4, z, n + 4);
    }
}

// Whether NaN or infinities were among eight elements; they are 2^-126 of the same sign then: zero for rows whose low is
// zero, infinite where it is infinite, as the product would be, and lost beside the term of unfit_term otherwise.
__device__ __forceinline__ bool clear_unfit_of(u32x4 &v) {
    bool found = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if ((v[j] & 0x7f80u) == 0x7f80u) v[j] = (v[j] & 0xffff8000u) | 0x0080u, found = true;
        if ((v[j] & 0x7f800000u) == 0x7f800000u) v[j] = (v[j] & 0x8000ffffu) | 0x00800000u, found = true;
    }
    return found;
}
// What those that b has for column n add, with low(j).
template <class Of>
__device__ __forceinline__ float unfit_term(const LoraArgs &l, int n, int adapter, Of low) {
    const uint16_t *b = (const uint16_t *)l.b + ((int64_t)adapter * l.n_out + n) * l.rank;
    float y = 0.0f;
    for (int j = 0; j < l.rank; j++) {
        const float v = bf2f(gptr(b)[j]);
        if (!(fabsf(v) < INFINITY)) y += low(j) * v;
    }
    return y;
}

// ------------------------------------------------------------------------------------------
// the product
// ------------------------------------------------------------------------------------------

// TM rows by TN columns of a workgroup, in waves of RM by RN, on 16x16x32 MFMAs (on 32x32x16 ones 2048 rows of 6144
// over 2560 took 72 us where these took 56); BK elements of the sum a step, STAGES steps' operands in LDS, where
// they come from memory without passing registers. Chunk c (16 bytes) of row r lies at c ^ (r % chunks): the rows that
// a product reads at one chunk are in different banks then.
template <int TM_, int TN_, int RM_, int RN_, int BK_, int STAGES_, bool STREAM_ = false>
struct Shape {
    static constexpr bool STREAM = STREAM_;                          // W is read once, past the caches
    static constexpr int TM = TM_, TN = TN_, RM = RM_, RN = RN_, BK = BK_, STAGES = STAGES_;
    static constexpr int WM = TM / RM, WN = TN / RN, WAVES = WM * WN, T = 64 * WAVES, MT = RM / 16, NT = RN / 16;
    static constexpr bool JOINS = TM <= 128;                         // also in front of join_kernel
    static constexpr int CHUNKS = BK / 8, ROW = 2 * BK, PER = 64 / CHUNKS;  // of a row: chunks, bytes; rows of a load
    static constexpr int BYTES = (TM + TN) * ROW;                    // of a stage
    static_assert(TM <= T, "a thread per row looks up its owner");
    // rows of low_part beside it, whose sums are in LDS: 64 where a workgroup has a CU to itself and there are many rows
    // (924 rows of 2560 over 9728, of 22 sequences: 82 us, with 16 rows 87)
    static constexpr int LOW_ROWS = TM == 128 && TN == 256 ? 64 : 16;
    static_assert(!JOINS || STAGES * BYTES >= WAVES * LOW_ROWS * 68 * 4, "low_part's sums");
    static constexpr int X_LOADS = (TM / PER + WAVES - 1) / WAVES;   // per wave, of PER rows; the last ones may be
    static constexpr int W_LOADS = (TN / PER + WAVES - 1) / WAVES;   // loaded more than once
    static constexpr int LOADS = X_LOADS + W_LOADS;
};

// Large tiles: 2582 rows of 9728 over 2560 take 118 us, 1.09 PFLOP/s (a library product of 8192 x 8192 x 8192: 1.40), in 456
// tiles, two rounds that are 89% full, each with 6 us of first loads and stores; the matrix units are busy 42% of the time with
// operands from memory. Each step's operands come from LDS while the step before it is multiplied, and the loads of
// the step behind the stages go between the products; an XCD has tiles side by side, which share operands in its L2.
// Tiles of up to 64 rows are bound by W: 64 rows of 151936 over 2560 at 5.4 TB/s, which neither longer steps,
// more stages, another order of tiles nor another start of each tile's sum changes.
template <class G>
__global__ __launch_bounds__(G::T) void product_kernel(LoraArgs l) {
    __shared__ __attribute__((aligned(128))) char lds[G::STAGES * G::BYTES + G::TM * 8 + 8];
    int *owner = (int *)(lds + G::STAGES * G::BYTES), *list = owner + G::TM, *count = list + G::TM, *unfit = count + 1;
    const int lane = threadIdx.x & 63, wave = wave_id();
    if (G::JOINS && (int)blockIdx.x >= l.m_tiles * l.n_tiles * l.splits)
        return low_part<G::LOW_ROWS, G::WAVES, JOIN_LOW_SPAN / G::WAVES>(l, blockIdx.x - l.m_tiles * l.n_tiles * l.splits, (float *)lds);
    // the tiles of one XCD, whose workgroups every eighth one is, lie side by side
    const int tiles = l.m_tiles * l.n_tiles * l.splits, block = blockIdx.x;
    const int each = tiles / XCDS, more = tiles % XCDS, xcd = block % XCDS;
    const int at = xcd * each + min(xcd, more) + block / XCDS;
    const int m0 = at % l.m_tiles * G::TM, n0 = at / l.m_tiles % l.n_tiles * G::TN, split = at / (l.m_tiles * l.n_tiles);
    const bool join = l.part != nullptr, adapters = l.a && !l.low_groups && split == l.splits - 1;
    const bool owned = l.a && !l.low_groups;  // otherwise join_kernel looks them up
    if (owned && (int)threadIdx.x < G::TM)
        owner[threadIdx.x] = m0 + (int)threadIdx.x < l.n_tokens ? owner_of(l, m0 + threadIdx.x) : NO_SEQUENCE;
    if (threadIdx.x == 0) *unfit = *count = 0;

    // loads: lane's row and chunk of PER rows
    const unsigned base = (unsigned)(uintptr_t)(lds_char *)lds;
    const int row = lane / G::CHUNKS;
    unsigned x_at[G::X_LOADS], w_at[G::W_LOADS];   // bytes from the tile's first row
    const auto x_group = [&](int i) { return min(wave * G::X_LOADS + i, G::TM / G::PER - 1); };
    const auto w_group = [&](int i) { return min(wave * G::W_LOADS + i, G::TN / G::PER - 1); };
    const auto x_row = [&](int i) { return x_group(i) * G::PER + row; };
    const auto w_row = [&](int i) { return w_group(i) * G::PER + row; };
    const auto chunk_of = [&](int r) { return (lane % G::CHUNKS) ^ (r & (G::CHUNKS - 1)); };
#pragma unroll
    for (int i = 0; i < G::X_LOADS; i++)
        x_at[i] = (unsigned)(min(x_row(i), l.n_tokens - 1 - m0) * l.x_stride * 2) + chunk_of(x_row(i)) * 16;
#pragma unroll
    for (int i = 0; i < G::W_LOADS; i++)
        w_at[i] = (unsigned)min(w_row(i), l.n_out - 1 - n0) * (unsigned)l.n_in * 2 + chunk_of(w_row(i)) * 16;
    const char *x_from = (const char *)(l.x + m0 * l.x_stride), *w_from = (const char *)(l.w + (int64_t)n0 * l.n_in);
    const int all_steps = l.w ? (l.n_in + G::BK - 1) / G::BK : 0, whole_steps = l.w ? l.n_in / G::BK : 0;
    const int last_step = min(all_steps, (split + 1) * l.split_steps);
    int step = split * l.split_steps, next = 0, piece = 0;  // what is requested next: the product's, then adapters'
    unsigned of_adapter = 0;                                // stages that hold some of these
    const int pieces = (2 * l.rank + G::BK - 1) / G::BK;
    __syncthreads();
    if (adapters && wave == 0) {  // the adapters of the tile's rows, each once: entry 64 q + lane in entry[q]
        constexpr int Q = (G::TM + 63) / 64;
        int entry[Q], n = 0;
#pragma unroll
        for (int q = 0; q < Q; q++) entry[q] = NO_ADAPTER;
#pragma unroll 1
        for (int q = 0; q < Q; q++) {
            const int i = q * 64 + lane, mine = i < G::TM ? owner[i] : NO_SEQUENCE;
            uint64_t starts = __ballot(mine >= 0 && (i == 0 || owner[i - 1] != mine));
            while (starts) {  // of rows with one adapter, one after the other
                const int a = __builtin_amdgcn_readlane(mine, __builtin_ctzll(starts));
                starts &= starts - 1;
                bool there = false;
#pragma unroll
                for (int p = 0; p < Q; p++) there |= entry[p] == a;
                if (__any(there)) continue;
#pragma unroll
                for (int p = 0; p < Q; p++)
                    if (p * 64 + lane == n) entry[p] = a;
                n++;
            }
        }
#pragma unroll
        for (int q = 0; q < Q; q++)
            if (q * 64 + lane < n) list[q * 64 + lane] = entry[q];
        if (lane == 0) *count = n;
    }
    if (adapters) __syncthreads();
    const int listed = adapters ? __builtin_amdgcn_readfirstlane(*count) : 0;

    // Load i of a step of whole chunks into stage `to`.
    const auto load_whole = [&](int i, int to) {
        const unsigned xs = base + to * G::BYTES;
        if (i < G::X_LOADS) load_to_lds(xs + x_group(i) * 1024, x_from + (int64_t)step * G::ROW, x_at[i]);
        else load_to_lds<G::STREAM>(xs + G::TM * G::ROW + w_group(i - G::X_LOADS) * 1024, w_from + (int64_t)step * G::ROW, w_at[i - G::X_LOADS]);
    };
    // Requests the next step's operands into stage `to`; false after the last.
    const int whole_end = min(whole_steps, last_step);
    const auto request = [&](int to) {
        const unsigned xs = base + to * G::BYTES, ws = xs + G::TM * G::ROW;
        if (step < whole_end) {
#pragma unroll
            for (int i = 0; i < G::LOADS; i++) load_whole(i, to);
            step++;
            return true;
        }
        if (step < last_step) {  // the last step of a width that is no multiple of 64
            const char *x = x_from + (int64_t)step * G::ROW, *w = w_from + (int64_t)step * G::ROW;
            const auto there = [&](int r) { return step * G::BK + chunk_of(r) * 8 < l.n_in; };
#pragma unroll
            for (int i = 0; i < G::X_LOADS; i++)
                load_to_lds(xs + x_group(i) * 1024, there(x_row(i)) ? x + x_at[i] : (const char *)&g_zeros);
#pragma unroll
            for (int i = 0; i < G::W_LOADS; i++)
                load_to_lds(ws + w_group(i) * 1024, there(w_row(i)) ? w + w_at[i] : (const char *)&g_zeros);
            step++;
            return true;
        }
        if (next == listed) return false;
        const int current = __builtin_amdgcn_readfirstlane(list[next]);
        const int chunks = l.rank / 8;
        const char *low = (const char *)(l.low + (int64_t)m0 * 2 * l.rank);
        const char *b = (const char *)(l.b + ((int64_t)current * l.n_out + n0) * l.rank);
#pragma unroll
        for (int i = 0; i < G::X_LOADS; i++) {
            const int r = x_row(i), c = piece * G::CHUNKS + chunk_of(r);
            load_to_lds(xs + x_group(i) * 1024, c < 2 * chunks && owner[r] == current ? low + ((int64_t)r * 2 * chunks + c) * 16
                                                                                     : (const char *)&g_zeros);
        }
#pragma unroll
        for (int i = 0; i < G::W_LOADS; i++) {
            const int r = w_row(i), c = piece * G::CHUNKS + chunk_of(r);
            load_to_lds(ws + w_group(i) * 1024,
                        c < 2 * chunks ? b + ((int64_t)min(r, l.n_out - 1 - n0) * chunks + (c >= chunks ? c - chunks : c)) * 16
                                       : (const char *)&g_zeros);
        }
        if (++piece == pieces) piece = 0, next++;
        of_adapter |= 1u << to;
        return true;
    };
    f32x4 acc[G::MT][G::NT];
    const int mine_m = wave % G::WM * G::RM, mine_n = wave / G::WM * G::RN;
    constexpr int KS = G::BK / 32;  // products of a step, on operands in alternating registers
    static_assert(KS % 2 == 0, "registers alternate");
    u32x4 xf[2][G::MT], wf[2][G::NT];
    const auto fetch = [&](int from, int k) {
        const char *xs = lds + from * G::BYTES, *ws = xs + G::TM * G::ROW;
        const int r = lane % 16, slot = (k * 4 + lane / 16) ^ (r & (G::CHUNKS - 1));
#pragma unroll
        for (int i = 0; i < G::MT; i++) xf[k % 2][i] = *(const u32x4 *)(xs + (mine_m + i * 16 + r) * G::ROW + slot * 16);
#pragma unroll
        for (int j = 0; j < G::NT; j++) wf[k % 2][j] = *(const u32x4 *)(ws + (mine_n + j * 16 + r) * G::ROW + slot * 16);
    };
    const auto multiply = [&](int k) {
#pragma unroll
        for (int i = 0; i < G::MT; i++)
#pragma unroll
            for (int j = 0; j < G::NT; j++) acc[i][j] = mfma(wf[k % 2][j], xf[k % 2][i], acc[i][j]);
    };
    // NaN and infinities of an adapter, times the zeros of other rows or a remainder of zero, would be no numbers
    // everywhere. Where there are some, which the largest exponent tells, the tile is computed again with small numbers in
    // their place, and the rows that they belong to get them in the end.
    u16x2 largest = {0, 0};
    bool clear = false;
    const auto begin = [&](int from) {
        if (of_adapter >> from & 1 && clear) {
            for (int c = threadIdx.x; c < G::TN * G::CHUNKS; c += G::T) {
                u32x4 *at = (u32x4 *)(lds + from * G::BYTES + G::TM * G::ROW + c * 16), v = *at;
                if (clear_unfit_of(v)) *at = v;
            }
            wait_lds();
            barrier();
        }
        fetch(from, 0);
    };
    const auto look_at = [&](int from, int k) {
        if (!(of_adapter >> from & 1)) return;
#pragma unroll
        for (int j = 0; j < G::NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                largest = __builtin_elementwise_max(largest, __builtin_bit_cast(u16x2, wf[k % 2][j][e] & 0x7fff7fffu));
    };

again:
#pragma unroll
    for (int i = 0; i < G::MT; i++)
#pragma unroll
        for (int j = 0; j < G::NT; j++) acc[i][j] = {};
    int pending = 0, stage = 0;  // steps requested and not yet multiplied; the first one's stage
#pragma unroll
    for (int i = 0; i < G::STAGES - 1; i++)
        if (request(i)) pending++;
    if (pending > 0) {
        if (pending == G::STAGES - 1) wait_loads<(G::STAGES - 2) * G::LOADS>();
        else wait_loads<0>();
        barrier();
        if (pending == G::STAGES - 1 && request(G::STAGES - 1)) pending++;
        begin(0);
    }
    // the next step is there and this one read, in every wave: its stage takes another one, and the next step's first
    // operands come beside this one's last products
    while (pending == G::STAGES && step < whole_end) {
#pragma unroll
        for (int k = 0; k + 1 < KS; k++) {
            fetch(stage, k + 1);
            multiply(k);
        }
        const int free = stage;
        stage = stage == G::STAGES - 1 ? 0 : stage + 1;
        wait_lds();
        wait_loads<(G::STAGES - 2) * G::LOADS>();
        barrier();
        fetch(stage, 0);
#pragma unroll
        for (int i = 0; i < G::MT; i++) {
#pragma unroll
            for (int n = i * G::LOADS / G::MT; n < (i + 1) * G::LOADS / G::MT; n++) load_whole(n, free);
#pragma unroll
            for (int j = 0; j < G::NT; j++)
                acc[i][j] = mfma(wf[(KS - 1) % 2][j], xf[(KS - 1) % 2][i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
        step++;
    }
    while (pending > 0) {
        const int at = stage;
#pragma unroll
        for (int k = 0; k + 1 < KS; k++) {
            fetch(at, k + 1);
            look_at(at, k);
            multiply(k);
        }
        look_at(at, KS - 1);
        of_adapter &= ~(1u << at);
        if (pending > 1) {
            stage = stage == G::STAGES - 1 ? 0 : stage + 1;
            wait_lds();
            if (pending == G::STAGES) wait_loads<(G::STAGES - 2) * G::LOADS>();
            else wait_loads<0>();
            barrier();
            if (pending == G::STAGES && request(at)) pending++;
            begin(stage);
        }
        multiply(KS - 1);
        pending--;
    }
    wait_lds();
    barrier();
    if (adapters && !clear) {
        if (largest[0] >= 0x7f80 || largest[1] >= 0x7f80) *unfit = 1;
        wait_lds();
        barrier();
        clear = __builtin_amdgcn_readfirstlane(*unfit);
        if (clear) {
            step = split * l.split_steps;
            next = 0;
            goto again;
        }
    }

    // parts from the registers, a lane having four columns side by side of a row; out through LDS, a wave's 16 rows at a
    // time, so that what goes out is whole lines, or as much of them as the wave has columns
    constexpr int PITCH = G::RN + 4, EIGHTS = G::RN / 8;
    static_assert(G::WAVES * 16 * PITCH * 4 <= G::STAGES * G::BYTES, "rows on their way out");
    float *rows = (float *)lds + wave * 16 * PITCH;
#pragma unroll
    for (int i = 0; i < G::MT; i++) {
        if (join) {
            const int m = m0 + mine_m + i * 16 + lane % 16;
            if (m >= l.n_tokens) continue;
            float *part = l.part + ((int64_t)split * l.n_tokens + m) * l.part_width;
#pragma unroll
            for (int j = 0; j < G::NT; j++) {
                const int n = n0 + mine_n + j * 16 + lane / 16 * 4;
                if (n < l.n_out) *gptr((f32x4 *)(part + n)) = acc[i][j];
            }
            continue;
        }
#pragma unroll
        for (int j = 0; j < G::NT; j++) *(f32x4 *)(rows + lane % 16 * PITCH + j * 16 + lane / 16 * 4) = acc[i][j];
        wait_lds();
#pragma unroll
        for (int p = lane; p < 16 * EIGHTS; p += 64) {
            const int tile_row = mine_m + i * 16 + p / EIGHTS, m = m0 + tile_row, c = p % EIGHTS * 8, n = n0 + mine_n + c;
            if (m >= l.n_tokens || (owned && owner[tile_row] == NO_SEQUENCE) || n >= l.n_out) continue;
            const float *from = rows + p / EIGHTS * PITCH + c;
            store8(l, l.out + m * l.out_stride + n, l.residual + m * l.residual_stride + n, *(const f32x4 *)from,
                   *(const f32x4 *)(from + 4), n);
        }
        wait_lds();
    }
    if (clear) {  // the infinities and NaN, behind what was written
        __syncthreads();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "agent");
        for (int i = threadIdx.x; i < G::TM * G::TN; i += G::T) {
            const int m = m0 + i / G::TN, n = n0 + i % G::TN, a = owner[i / G::TN];
            if (a < 0 || n >= l.n_out) continue;
            const uint16_t *low = (const uint16_t *)l.low + (int64_t)m * 2 * l.rank;
            const float more = unfit_term(l, n, a, [&](int j) { return bf2f(gptr(low)[j]) + bf2f(gptr(low)[l.rank + j]); });
            if (fabsf(more) < INFINITY) continue;
            LLM_GLOBAL float *part = gptr(l.part) + ((int64_t)split * l.n_tokens + m) * l.part_width + n;
            LLM_GLOBAL bf16 *to = gptr(l.out) + m * l.out_stride + n;
            if (join) *part += more;
            else *to = (bf16)f2bf(bf2f(*to) + more);
        }
    }
}

// out of the product's parts, in their order: four columns of a row per thread. Bound by their bytes.
__global__ __launch_bounds__(256) void sum_kernel(LoraArgs l) {
    const int per = l.part_width / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int m = (int)(i / per), n = (int)(i % per) * 4;
    if (m >= l.n_tokens || (l.a && owner_of(l, m) == NO_SEQUENCE)) return;
    const float *part = l.part + (int64_t)m * l.part_width + n;
    const int64_t next = (int64_t)l.n_tokens * l.part_width;
    f32x4 y = {0, 0, 0, 0};
    constexpr int U = 4;
    for (int s0 = 0; s0 < l.splits; s0 += U) {
        f32x4 v[U];
#pragma unroll
        for (int s = 0; s < U; s++)
            v[s] = s0 + s < l.splits ? *gptr((const f32x4 *)(part + (s0 + s) * next)) : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < U; s++) y += v[s];
    }
    store4(l, l.out + m * l.out_stride + n, l.residual + m * l.residual_stride + n, y, n);
}

// ------------------------------------------------------------------------------------------
// the join: the product's parts, the adapters' terms and the residual
// ------------------------------------------------------------------------------------------

// 16 rows of a sequence by 256 columns per workgroup. Bound by its round trips for few rows (5 us for 64 rows of 4096), by
// the parts' and b's bytes for many (924 rows of 2560, three parts, rank 64: 19 us, 3.8 TB/s). What the lanes read besides the parts of low is requested in
// front of those, so that all of it comes in one round trip behind the lookup of the rows.
constexpr int FEW = 4;      // rows up to which a lane has a column, and the sum over the rank is one of vector operations

// low of the tile's rows, into LDS.
__device__ __forceinline__ void join_low(const LoraArgs &l, const RowTile &t, float scale, float *low) {
    for (int i = 4 * threadIdx.x; i < t.rows * l.rank; i += 4 * 256)
        *(f32x4 *)(low + i) = low_sum(l, (int64_t)t.first * l.rank + i, scale);
    __syncthreads();
}

// ROWS: rows of the tile at most.
template <int ROWS>
__device__ __forceinline__ void join_few(const LoraArgs &l, const RowTile &t, int n, float scale, float *low) {
    constexpr int P = ROWS == 1 ? 8 : 4, CHUNKS = 4;  // parts, and chunks of b, under way
    const int at = min(n, l.n_out - 1), rank = t.adapter >= 0 ? l.rank : 0;
    const auto part_at = [&](int i, int s) {
        return i < t.rows && s < l.splits ? gptr(l.part)[((int64_t)s * l.n_tokens + t.first + i) * l.part_width + at] : 0.0f;
    };
    float part[ROWS][P], y[ROWS];
    u32x4 v[CHUNKS];
    const bf16 *b = l.b + ((int64_t)max(t.adapter, 0) * l.n_out + at) * l.rank;
#pragma unroll
    for (int c = 0; c < CHUNKS; c++)
        if (c * 8 < rank) v[c] = ld16(b + c * 8);
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        y[i] = l.residual && i < t.rows ? bf2f(gptr(l.residual)[(t.first + i) * l.residual_stride + at]) : 0.0f;
#pragma unroll
        for (int s = 0; s < P; s++) part[i][s] = part_at(i, s);
    }
    if (rank) join_low(l, t, scale, low);
    for (int s0 = 0;;) {
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int s = 0; s < P; s++) y[i] += part[i][s];
        if ((s0 += P) >= l.splits) break;
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int s = 0; s < P; s++) part[i][s] = part_at(i, s0 + s);
    }
    for (int j0 = 0; j0 < rank; j0 += 8 * CHUNKS) {
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            if (j0 + c * 8 >= rank) break;
#pragma unroll
            for (int i = 0; i < ROWS; i++)
                if (i < t.rows)
#pragma unroll
                    for (int e = 0; e < 8; e++) y[i] = fmaf(low[i * rank + j0 + c * 8 + e], elem(v[c], e), y[i]);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; c++)
            if (j0 + (CHUNKS + c) * 8 < rank) v[c] = ld16(b + j0 + (CHUNKS + c) * 8);
    }
    if (n < l.n_out)
#pragma unroll
        for (int i = 0; i < ROWS; i++)
            if (i < t.rows) gptr(l.out)[(t.first + i) * l.out_stride + n] = (bf16)f2bf(y[i]);
}

// R: rows of a tile at most, FEW or 16. Tiles of few rows are bound by their round trips, so by how many workgroups a CU
// takes at once: with a kernel of their own, six (three where all tiles shared one), 64 single tokens take 14 us (16.6).
template <int R>
__global__ __launch_bounds__(256, R == FEW ? 6 : 3) void join_kernel(LoraArgs l) {
    constexpr int PITCH = 64 + 4;
    __shared__ __attribute__((aligned(16))) float low[R * 256], lines[R == FEW ? 1 : 4 * 16 * PITCH];
    const int lane = threadIdx.x & 63, wave = wave_id();
    const RowTile t = row_tile<R>(l, blockIdx.x);
    if (t.rows == 0) return;
    const float scale = l.scale && t.adapter >= 0 ? gptr(l.scale)[t.adapter] : 1.0f;
    if (t.rows == 1) return join_few<1>(l, t, blockIdx.y * 256 + threadIdx.x, scale, low);
    if (R == FEW || t.rows <= FEW) return join_few<FEW>(l, t, blockIdx.y * 256 + threadIdx.x, scale, low);
    // a lane has row lane % 16 and four columns of each 16
    const int n0 = (blockIdx.y * 4 + wave) * 64, mine = min(lane % 16, t.rows - 1), m = t.first + mine;
    const auto part_at = [&](int j, int s) {
        if (s >= l.splits) return f32x4{0, 0, 0, 0};
        const int n = min(n0 + j * 16 + lane / 16 * 4, l.part_width - 4);
        return *gptr((const f32x4 *)(l.part + ((int64_t)s * l.n_tokens + m) * l.part_width + n));
    };
    constexpr int P = 4;
    f32x4 part[4][P], y[4] = {};
#pragma unroll
    for (int s = 0; s < P; s++)
#pragma unroll
        for (int j = 0; j < 4; j++) part[j][s] = part_at(j, s);
    if (t.adapter >= 0) join_low(l, t, scale, low);
    if (n0 >= l.n_out) return;
    for (int s0 = 0;;) {
#pragma unroll
        for (int s = 0; s < P; s++)
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] += part[j][s];
        if ((s0 += P) >= l.splits) break;
#pragma unroll
        for (int s = 0; s < P; s++)
#pragma unroll
            for (int j = 0; j < 4; j++) part[j][s] = part_at(j, s0 + s);
    }
    f32x4 acc[4] = {};
    bool unfit = false;
    if (t.adapter >= 0) {
        const bf16 *b = l.b + (int64_t)t.adapter * l.n_out * l.rank;
        constexpr int U = 2;
        for (int c0 = 0; c0 < l.rank / 8; c0 += 4 * U) {
            u32x4 v[U][4];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int c = c0 + 4 * u + lane / 16, n = min(n0 + j * 16 + lane % 16, l.n_out - 1);
                    v[u][j] = c < l.rank / 8 ? ld16(b + (int64_t)n * l.rank + c * 8) : u32x4{0, 0, 0, 0};
                }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = c0 + 4 * u + lane / 16;
                u32x4 value = {0, 0, 0, 0}, rest = {0, 0, 0, 0};
                if (c < l.rank / 8) {
                    const float *from = low + mine * l.rank + c * 8;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t two, left;
                        in_two(from[2 * e], from[2 * e + 1], two, left);
                        value[e] = two;
                        rest[e] = left;
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    unfit |= clear_unfit_of(v[u][j]);
                    acc[j] = mfma(v[u][j], value, acc[j]);
                    acc[j] = mfma(v[u][j], rest, acc[j]);
                }
            }
        }
    }
    unfit = __any(unfit);
    // a wave's rows through LDS, so that what goes out is whole lines
    float *rows = lines + wave * 16 * PITCH;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = n0 + j * 16 + lane / 16 * 4;
        y[j] += acc[j];
        if (unfit && lane % 16 < t.rows)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < l.n_out) y[j][e] += unfit_term(l, n + e, t.adapter, [&](int i) { return low[mine * l.rank + i]; });
        *(f32x4 *)(rows + lane % 16 * PITCH + j * 16 + lane / 16 * 4) = y[j];
    }
    wait_lds();
#pragma unroll
    for (int p = lane; p < 16 * 8; p += 64) {
        const int i = p / 8, c = p % 8 * 8, n = n0 + c;
        if (i >= t.rows || n >= l.n_out) continue;
        const float *from = rows + i * PITCH + c;
        store8(l, l.out + (t.first + i) * l.out_stride + n, l.residual + (t.first + i) * l.residual_stride + n,
               *(const f32x4 *)from, *(const f32x4 *)(from + 4), n);
    }
}

// ------------------------------------------------------------------------------------------
// one or two rows with little rank: everything in one launch
// ------------------------------------------------------------------------------------------

constexpr int ONE_COLUMNS = 16, ONE_LOW = 16, ONE_SEQS = 64;  // columns of a workgroup; elements of low, sequences at most

// The adapter of row m, found among up to 64 sequences in one round trip.
__device__ __forceinline__ int owner_among(const LoraArgs &l, int first, int end, int adapter, int m) {
    const int lane = threadIdx.x & 63;
    const uint64_t mine = __ballot(lane < l.n_seqs && first <= m && m < end);
    if (!mine) return NO_SEQUENCE;
    const int a = __builtin_amdgcn_readlane(adapter, __builtin_ctzll(mine));
    return (unsigned)a < (unsigned)l.n_adapters ? a : NO_ADAPTER;
}

// A wave has four columns, and four elements of low, which every workgroup computes for itself, by vector operations in 32
// bits: at most as much is read of A as of W, and A comes from L2. Bound by two round trips, the lookup's and the operands'
// (W's first ones are requested in front of the lookup): 4.7 us for 2048 over 1024, rank 8.
template <int ROWS>
__global__ __launch_bounds__(256) void one_kernel(LoraArgs l) {
    constexpr int U = 2;
    __shared__ float low[ONE_LOW];
    const int lane = threadIdx.x & 63, wave = wave_id(), n0 = blockIdx.x * ONE_COLUMNS + wave * 4, s = min(lane, l.n_seqs - 1);
    const int first = start_of(l, s), end = start_of(l, s + 1), adapter = gptr(l.adapter)[s];
    const bf16 *w[4], *x[ROWS];
    const int chunks = l.n_in / 8;
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = l.w + (int64_t)min(n0 + j, l.n_out - 1) * l.n_in;
#pragma unroll
    for (int i = 0; i < ROWS; i++) x[i] = l.x + i * l.x_stride;
    u32x4 xs[U][ROWS], ws[U][4], as[U][4];
    const auto request = [&](const bf16 *p, int c) { return c < chunks ? ld16(p + c * 8) : u32x4{0, 0, 0, 0}; };
    const auto request_w = [&](int c0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int i = 0; i < ROWS; i++) xs[u][i] = request(x[i], c0 + 64 * u);
#pragma unroll
            for (int j = 0; j < 4; j++) ws[u][j] = l.w ? request(w[j], c0 + 64 * u) : u32x4{0, 0, 0, 0};
        }
    };
    request_w(lane);
    int owner[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) owner[i] = owner_among(l, first, end, adapter, i);
    // elements 4 wave .. 4 wave + 3 of low, which are of one row, as the rank is a multiple of 8
    const int element = wave * 4, of = element / l.rank, r = element % l.rank;
    const int mine = of == 0 ? owner[0] : of < ROWS ? owner[ROWS - 1] : NO_SEQUENCE;
    const bf16 *a = l.a + ((int64_t)max(mine, 0) * l.rank + r) * l.n_in;
    const int some = mine >= 0 ? chunks : 0;
    const auto request_a = [&](int c0) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                as[u][j] = c0 + 64 * u < some ? ld16(a + (int64_t)j * l.n_in + (c0 + 64 * u) * 8) : u32x4{0, 0, 0, 0};
    };
    request_a(lane);
    // what lane 4 i + j needs for column j of row i
    const int row = lane / 4 % ROWS, n = n0 + lane % 4, at = min(n, l.n_out - 1), its = row == 0 ? owner[0] : owner[ROWS - 1];
    const bf16 *b = l.b + ((int64_t)max(its, 0) * l.n_out + at) * l.rank;
    const u32x4 b0 = ld16(b), b1 = l.rank > 8 ? ld16(b + 8) : u32x4{0, 0, 0, 0};
    const float scale = l.scale && mine >= 0 ? gptr(l.scale)[mine] : 1.0f;
    float y = l.residual ? bf2f(gptr(l.residual)[row * l.residual_stride + at]) : 0.0f;
    float acc[ROWS][4] = {}, sum[4] = {};
    for (int c0 = lane;;) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
#pragma unroll
                    for (int i = 0; i < ROWS; i++) acc[i][j] = fmaf(elem(xs[u][i], e), elem(ws[u][j], e), acc[i][j]);
                    sum[j] = fmaf(elem(of == 0 ? xs[u][0] : xs[u][ROWS - 1], e), elem(as[u][j], e), sum[j]);
                }
        c0 += 64 * U;
        if (c0 - lane >= chunks) break;
        request_w(c0);
        request_a(c0);
    }
    const auto all = [&](float v) {
        v += xor_lane<1>(v), v += xor_lane<2>(v), v += xor_lane<4>(v), v += xor_lane<8>(v), v += xor_lane<16>(v);
        return v + xor_lane<32>(v);
    };
#pragma unroll
    for (int j = 0; j < 4; j++) {
        sum[j] = all(sum[j]) * scale;
        if (lane == 0 && element + j < ROWS * l.rank) low[element + j] = sum[j];
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            acc[i][j] = all(acc[i][j]);
            if (l.w && row == i && lane % 4 == j) y += acc[i][j];
        }
    }
    __syncthreads();
    if (its >= 0)
#pragma unroll
        for (int e = 0; e < 16; e++)
            if (e < l.rank) y = fmaf(low[row * l.rank + e], elem(e < 8 ? b0 : b1, e % 8), y);
    if (lane < 4 * ROWS && n < l.n_out && its != NO_SEQUENCE) gptr(l.out)[row * l.out_stride + n] = (bf16)f2bf(y);
}

// ------------------------------------------------------------------------------------------
// on the host
// ------------------------------------------------------------------------------------------

// Shapes of the product, with what an estimate goes by, in ns: workgroups that a CU holds at once, a step where few
// CUs have a workgroup and where all do, and a tile's first loads and stores.
struct Pace {
    int tm, tn, at_once;
    double alone, full, fixed;
};
// What the large ones are for, us of a product without adapters (beside it the best of the other shapes): 256 by 192, 1152 rows of
// 9728 over 2560 64 (71); 224 by 256, 2100 rows of 6144 over 2560 59 (70), 3200 rows of 4096 over 2560 60 (70), although it keeps
// 22 registers in scratch memory, outside of the loop over whole steps; 192 by 256, 2500 rows of 4096 over 2560 51 (54); 128 by
// 256, 700 rows of 19456 over 2560 82 (124). Of 24 drawn calls each that take 256 by 192, 224 by 256 or 128 by 128, the estimate's
// next choice takes 7%, 11% and 4% longer on average.
typedef Shape<256, 192, 64, 96, 64, 2> Wide;
typedef Shape<224, 256, 112, 64, 64, 2> High;
typedef Shape<192, 256, 96, 64, 64, 2> Square;
typedef Shape<128, 256, 64, 64, 64, 3> Half;
typedef Shape<128, 128, 32, 64, 64, 2> Quarter;
typedef Shape<64, 128, 64, 32, 64, 3, true> Few128;
typedef Shape<64, 64, 64, 16, 64, 4, true> Few64;
typedef Shape<32, 64, 32, 16, 64, 4, true> Few32;
typedef Shape<16, 64, 16, 16, 64, 4, true> Few16;
constexpr Pace PACES[] = {{256, 192, 1, 920, 1380, 5800}, {224, 256, 1, 970, 1450, 5900}, {192, 256, 1, 960, 1220, 6100},
                          {128, 256, 1, 650, 720, 3900},  {128, 128, 2, 520, 740, 3900},  {64, 128, 2, 440, 610, 1900},
                          {64, 64, 2, 460, 250, 2400},    {32, 64, 3, 310, 280, 2100},    {16, 64, 3, 270, 230, 1700}};
// And what a launch goes by.
struct Tile {
    int tm, tn, threads, low_rows;
};
template <class G>
constexpr Tile tile_of() {
    return {G::TM, G::TN, G::T, G::LOW_ROWS};
}
constexpr Tile TILES[] = {tile_of<Wide>(),   tile_of<High>(),  tile_of<Square>(), tile_of<Half>(), tile_of<Quarter>(),
                          tile_of<Few128>(), tile_of<Few64>(), tile_of<Few32>(),  tile_of<Few16>()};
constexpr int SHAPES = sizeof(PACES) / sizeof(PACES[0]);

constexpr int MOST_SPLITS = 32;
constexpr size_t MOST_PART = 1 << 23;  // floats

// For tests: a plan that is taken wherever it can be, in the calls of the thread that set it.
thread_local struct {
    int shape = -1, splits, join;
} g_forced;

// Few rows in all or of each sequence, on average: join_kernel has tiles of FEW rows. 60 rows of one sequence, 4096 over 2560
// and rank 16, take 15 us so and 19 with tiles of 16; 64 sequences of two rows 18 and 21; 120 rows of one, 6144 over 2560 and
// rank 128, 32 and 30; 128 sequences of four, 2560 over 9728 and rank 64, 95 and 89. Of 244 calls (4 to 512 rows, 1 to 256
// sequences of equal length, ranks 8 to 128) 210 are within 3% of the shorter way; the others take up to 26% longer, of low
// rank with tiles of 16 (16 sequences of 12 rows of 1024 over 1024, rank 8: 12.9 and 10.2), of high with tiles of FEW.
bool few_each(int n_tokens, int n_seqs) { return n_tokens <= std::max(128, 2 * n_seqs); }

// How a call is computed: tiles of one of the shapes, in splits; and whether the adapters' terms are steps of the
// product, or join_kernel's. The least of an estimate fitted to 107 calls (1 to 4079 rows, 1 to 128 sequences, ranks of 8
// to 128, 500 to 151936 columns), each in every shape and many splits. Of 600 other calls (1 to 4096 rows, more than half
// of the widths of models) what it chooses takes 5% longer on average than the best shape and splits, one in 20 takes 22% longer
// or more, one 60%.
struct Plan {
    int shape, splits, split_steps;
    bool join;

    static size_t part_floats(int n_tokens, int n_out) { return (size_t)n_tokens * ((n_out + 3) / 4 * 4); }
    // Of the parts, for n_tokens and for fewer.
    static size_t most_part(int n_tokens, int n_out) {
        return std::min(MOST_PART, MOST_SPLITS * part_floats(n_tokens, n_out));
    }

    Plan(int n_tokens, int n_out, int n_in, bool product, bool adapters, int rank, int n_seqs, int n_adapters) {
        const int steps = product ? (n_in + 63) / 64 : 0, pieces = (2 * rank + 63) / 64;
        const double rows = n_tokens, seqs = n_seqs, one = (double)part_floats(n_tokens, n_out);
        const bool few = few_each(n_tokens, n_seqs);
        // bytes of low's operands with tiles of so many rows, and of b with join_kernel's
        const auto low = [&](int tile) { return adapters ? (std::min(rows, rows / tile + seqs) * rank + rows) * n_in * 2 : 0; };
        const double b = adapters ? std::min(rows, rows / (few ? FEW : 16) + seqs) * n_out * rank * 2 : 0;
        // adapters of a tile's rows, each with steps of its own: between those of sequences of one length, and as many
        // as there can be, where the short ones lie side by side
        const auto own_steps = [&](const Pace &s) {
            if (!adapters) return 0.0;
            const double tile = std::min<double>(s.tm, rows), even = std::min<double>(n_adapters, 1 + seqs * tile / rows);
            return pieces * sqrt(even * std::min({(double)n_adapters, seqs, tile}));
        };
        // join_kernel's workgroups, most of which find nothing where most sequences are empty
        const bool joins = adapters && (rows / (few ? FEW : 16) + seqs) * ceil(n_out / 256.0) < 1 << 23;
        double least = 0;
        shape = -1;
        for (int i = 0; i < SHAPES; i++) {
            const Pace &s = PACES[i];
            const double m_tiles = ceil(rows / s.tm), tiles = m_tiles * ceil((double)n_out / s.tn);
            // W past the caches, for more rows of tiles (those of 128 columns have up to 16 MB of it in part from there): 1344
            // rows of 6144 over 2560 take 114 us in tiles of 64 by 64, 50 in large ones
            const double again = s.tm > 64 ? 0 : s.tn == 64 ? 0.7 * (m_tiles - 1) : 0.63 * std::min(m_tiles - 1, n_out * (double)n_in > 1 << 23 ? m_tiles : 8.0);
            const double memory = product ? 2.0 * n_out * n_in * (1 + again) / 5770 : 0;
            for (int n = 1; n <= std::min(MOST_SPLITS, std::max(steps, 1)) && (n == 1 || n * one <= (double)MOST_PART); n++) {
                const double groups = tiles * n, step = s.alone + (s.full - s.alone) * std::min(1.0, groups / CUS);
                const double rounds = ceil(groups / (s.at_once * CUS)), each = (steps + n - 1) / n, parts = one * (8 * n + 4);
                const double own = own_steps(s), rest = rounds * s.fixed;
                const double product_cost = product ? std::max(rounds * each * step, memory) : 0;
                const double cost = 1930 + product_cost + rounds * own * step + rest +
                                    (n > 1 ? 3010 + parts / 9350 : one * 2 / 9030) + (adapters ? 11100 + low(LOW_ROWS) / 8570 : 0);
                if (shape < 0 || cost < least) shape = i, splits = n, join = false, least = cost;
                if (!joins || s.tm > 128 || (product && n * one > (double)MOST_PART)) continue;
                if (!product && i < SHAPES - 1) continue;  // low alone: the smallest workgroups
                const int at_once = few ? 8 : 4;  // parts that the join has under way
                const double joined = 1930 + product_cost + (product ? rest : 0) + (few ? 3000 : 4500) + 1270 * ceil((double)n / at_once) +
                                      parts / 4960 + b / 7670 + low(TILES[i].low_rows) / 8570;
                if (joined < least) shape = i, splits = n, join = true, least = joined;
            }
        }
        if (g_forced.shape >= 0) {
            shape = g_forced.shape;
            join = g_forced.join && joins && PACES[shape].tm <= 128;
            splits = std::max(1, std::min(g_forced.splits, steps));
            if (splits * one > (double)MOST_PART) splits = 1, join = join && (one <= (double)MOST_PART || !product);
        }
        // the last split has the adapters' steps
        const double own = join ? 0 : own_steps(PACES[shape]);
        split_steps = std::min(steps, (int)((steps + own + splits - 1) / splits));
        splits = split_steps ? (steps + split_steps - 1) / split_steps : join ? 0 : 1;
    }
};

// Threads that a launch has fewer than.
constexpr int64_t MOST_THREADS = 1ll << 31;

template <class G>
bool launch_product(const LoraArgs &l, hipStream_t stream) {
    product_kernel<G><<<l.m_tiles * l.n_tiles * l.splits + l.low_groups, G::T, 0, stream>>>(l);
    return LAUNCH_OK();
}

// What one_kernel takes: sums of few round trips (of 1024 elements each; the other ways have the sum in up to 32 parts), and
// columns that the CUs take at once. us of a captured call among others, beside the other way's:
//   one row of rank 8: 2048 over 1024 4.7 (6.7), 16 over 4096 6.6 (7.1), 16 over 5120 7.7 (7.7), 16 over 9728 12.8 (8.5), 4096
//   over 4096 11.3 (11.6), 8192 over 1024 7.3 (8.5), 9728 over 1024 9.8 (9.4), 8192 over 2048 12.4 (10.7);
//   of rank 16: 4096 over 2560 8.9 (9.7), 1024 over 4096 8.1 (7.9), 2048 over 4096 10.2 (9.1);
//   two rows: 2048 over 1024 5.4 (6.8), 2048 over 2048 7.8 (7.7), 16 over 2560 6.9 (6.6), 4096 over 2048 10.1 (9.0);
//   without W, one row of rank 8: 4096 over 1024 4.1 (6.0), 2048 over 2560 6.0 (6.0), 16 over 4096 6.6 (5.5); two: 2048 over
//   1024 4.8 (6.0), 16 over 2560 6.8 (5.7).
bool takes_one(int n_tokens, int n_out, int n_in, bool product, int rank, int n_seqs) {
    const int trips = n_tokens == 2 ? 2 : product && rank == 8 ? 4 : 3;
    return n_tokens <= 2 && n_tokens * rank <= ONE_LOW && n_seqs <= ONE_SEQS && n_in <= trips * 1024 && n_out <= 8192 &&
           (int64_t)n_tokens * n_out * n_in <= (product ? (1 << 24) - 1 : 1 << 23);
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

// low and its parts, of which there are the most without a join.
int low_splits(int n_in) { return (n_in + LOW_SPAN - 1) / LOW_SPAN; }
size_t low_floats(int n_tokens, int n_in, int rank) { return (size_t)n_tokens * rank * (1 + low_splits(n_in)); }
size_t owner_floats(int n_tokens, int rank) { return rank ? ((size_t)n_tokens + 3) / 4 * 4 : 0; }

}  // namespace

extern "C" int llm_lora_force(int shape, int splits, int join) {
    g_forced.shape = shape < SHAPES ? shape : -1;
    g_forced.splits = splits;
    g_forced.join = join;
    return SHAPES;
}

extern "C" int llm_lora_plan(int n_tokens, int n_out, int n_in, int rank, int n_seqs, int n_adapters) {
    return Plan(n_tokens, n_out, n_in, true, rank > 0, rank, n_seqs, n_adapters).shape;
}

extern "C" size_t lora_projection_workspace_floats(int n_tokens, int n_out, int n_in, int rank) {
    if (!check_sizes("lora_projection_workspace_floats", n_tokens, n_out, n_in, rank)) return 0;
    return low_floats(n_tokens, n_in, rank) + owner_floats(n_tokens, rank) + Plan::most_part(n_tokens, n_out);
}

extern "C" void lora_projection_forward(bf16 *out, const bf16 *x, const bf16 *w, const bf16 *residual,
                                        const LoraBatch *lora, float *ws, int n_tokens, int n_out, int n_in,
                                        int64_t out_stride, int64_t x_stride, int64_t residual_stride,
                                        hipStream_t stream) {
    static const char name[] = "lora_projection";
    const int rank = lora ? lora->rank : 0;
    if (!check_sizes(name, n_tokens, n_out, n_in, rank)) return;
    if (lora) {
        if (rank == 0 || lora->n_seqs <= 0 || lora->n_seqs > 1 << 20 || lora->n_adapters <= 0) {
            llm_fail("%s: rank %d, n_seqs %d (up to 1048576) and n_adapters %d must be positive", name, rank,
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
    if (x_stride < n_in || x_stride % 8 || x_stride > 1 << 22) {
        llm_fail("%s: the rows of x are %lld elements apart, not a multiple of 8 of at least %d, up to 4194304", name,
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
    const Plan p(n_tokens, n_out, n_in, w != nullptr, lora != nullptr, rank, lora ? lora->n_seqs : 0,
                 lora ? lora->n_adapters : 0);
    if (!ws || !aligned16(ws)) {
        llm_fail("%s: ws must be a 16-byte aligned device address", name);
        return;
    }
    LoraArgs l = {};
    l.out = out, l.x = x, l.w = w, l.residual = residual;
    l.out_stride = out_stride, l.x_stride = x_stride, l.residual_stride = residual_stride;
    l.n_tokens = n_tokens, l.n_out = n_out, l.n_in = n_in;
    l.part_width = (n_out + 3) / 4 * 4;
    l.splits = p.splits, l.split_steps = p.split_steps;
    const auto aligned = [&](int n) {
        return out_stride % n == 0 && (uintptr_t)out % (2 * n) == 0 &&
               (!residual || (residual_stride % n == 0 && (uintptr_t)residual % (2 * n) == 0));
    };
    l.wide = aligned(8) ? 8 : aligned(4) ? 4 : 1;
    l.low = (bf16 *)ws;
    l.low_part = ws + (size_t)n_tokens * rank;
    l.low_splits = p.join ? (n_in + JOIN_LOW_SPAN - 1) / JOIN_LOW_SPAN : low_splits(n_in);
    l.owner = (int *)(ws + low_floats(n_tokens, n_in, rank));
    if (p.splits > 1 || p.join) l.part = ws + low_floats(n_tokens, n_in, rank) + owner_floats(n_tokens, rank);
    int64_t low_groups = 0;
    if (lora) {
        l.a = lora->a, l.b = lora->b, l.scale = lora->scale, l.q_start = lora->q_start, l.adapter = lora->adapter;
        l.n_seqs = lora->n_seqs, l.n_adapters = lora->n_adapters, l.rank = rank;
        if (g_forced.shape < 0 && takes_one(n_tokens, n_out, n_in, w != nullptr, rank, lora->n_seqs)) {
            const int groups = (n_out + ONE_COLUMNS - 1) / ONE_COLUMNS;
            if (n_tokens == 1) one_kernel<1><<<groups, 256, 0, stream>>>(l);
            else one_kernel<2><<<groups, 256, 0, stream>>>(l);
            LAUNCH_OK();
            return;
        }
        const int low_rows = p.join ? TILES[p.shape].low_rows : LOW_ROWS;
        low_groups = (int64_t)(n_tokens / low_rows + lora->n_seqs) * ((rank + low_width(rank) - 1) / low_width(rank)) * l.low_splits;
        if (low_groups * 64 * LOW_WAVES >= MOST_THREADS) {
            llm_fail("%s: %d sequences of rank %d over n_in %d are too many for one launch", name, lora->n_seqs, rank, n_in);
            return;
        }
        if (p.join) l.low_groups = (int)low_groups;
    }
    const Tile &tile = TILES[p.shape];
    l.m_tiles = (n_tokens + tile.tm - 1) / tile.tm;
    l.n_tiles = (n_out + tile.tn - 1) / tile.tn;
    if (((int64_t)l.m_tiles * l.n_tiles * l.splits + l.low_groups) * tile.threads >= MOST_THREADS) {
        llm_fail("%s: n_tokens %d by n_out %d is too much for one launch", name, n_tokens, n_out);
        return;
    }
    if (lora && !p.join) {
        low_kernel<<<low_groups, 64 * LOW_WAVES, 0, stream>>>(l);
        if (!LAUNCH_OK()) return;
        low_sum_kernel<<<((int64_t)n_tokens * (rank / 4) + 255) / 256, 256, 0, stream>>>(l);
        if (!LAUNCH_OK()) return;
    }
    bool ok = false;
    switch (p.shape) {
    case 0: ok = launch_product<Wide>(l, stream); break;
    case 1: ok = launch_product<High>(l, stream); break;
    case 2: ok = launch_product<Square>(l, stream); break;
    case 3: ok = launch_product<Half>(l, stream); break;
    case 4: ok = launch_product<Quarter>(l, stream); break;
    case 5: ok = launch_product<Few128>(l, stream); break;
    case 6: ok = launch_product<Few64>(l, stream); break;
    case 7: ok = launch_product<Few32>(l, stream); break;
    default: ok = launch_product<Few16>(l, stream);
    }
    if (!ok) return;
    const int n_tiles = (n_out + 255) / 256;
    if (p.join && few_each(n_tokens, lora->n_seqs)) join_kernel<FEW><<<dim3(n_tokens / FEW + lora->n_seqs, n_tiles), 256, 0, stream>>>(l);
    else if (p.join) join_kernel<16><<<dim3(n_tokens / 16 + lora->n_seqs, n_tiles), 256, 0, stream>>>(l);
    else if (p.splits > 1) sum_kernel<<<((int64_t)n_tokens * (l.part_width / 4) + 255) / 256, 256, 0, stream>>>(l);
    LAUNCH_OK();
}
