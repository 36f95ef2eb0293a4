// A projection of many rows with the low-rank adapters of their sequences (include/llm_amd/batch.h).
//
// out = x Wt + low Bt, low = scale x At: the second term is the first one's sum carried on over the rank, with rows
// of `low` for rows of x and an adapter's b for W. low is kept as two bf16, the value and what that leaves (16 bits
// of mantissa), side by side, so the sum goes over twice the rank.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "llm_amd/batch.h"

using namespace llm;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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
    int *owner;              // [n_tokens]: the row's adapter, NO_ADAPTER or NO_SEQUENCE
    float *part;             // [splits, n_tokens, part_width], or null: straight to out
    float *low_part;         // [low_splits, n_tokens, rank], where there are parts
    int64_t out_stride, x_stride, residual_stride;
    int n_tokens, n_out, n_in, n_seqs, n_adapters, rank;
    int part_width;
    int splits, split_steps;  // of the product's sum, steps of 64 each
    int m_tiles, n_tiles;
    int low_groups, low_splits;  // workgroups in front of the product's that compute low_part
    bool wide;               // out and residual take 8 bytes at a time
};

// What is loaded for places past an operand's end.
__device__ const u32x4 g_zeros = {0, 0, 0, 0};

template <int S>
struct Mfma;
template <>
struct Mfma<32> {
    typedef f32x16 Acc;
    static constexpr int K = 16, REGS = 16;
    static __device__ __forceinline__ f32x16 mul(const u32x4 &a, const u32x4 &b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    }
    // The first of the four rows that registers 4 i .. 4 i + 3 hold.
    static __device__ __forceinline__ int row(int i, int lane) { return 8 * i + 4 * (lane / 32); }
};
template <>
struct Mfma<16> {
    typedef f32x4 Acc;
    static constexpr int K = 32, REGS = 4;
    static __device__ __forceinline__ f32x4 mul(const u32x4 &a, const u32x4 &b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    }
    static __device__ __forceinline__ int row(int, int lane) { return 4 * (lane / 16); }
};

// 64 lanes' 16 bytes into LDS at `to` on, without passing registers: the wave waits for it with wait_loads.
__device__ __forceinline__ void load_to_lds(unsigned to, const void *base, unsigned offset) {
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

// 16 rows of one sequence at most. A sequence of n rows from f on has at most (f + n) / 16 - f / 16 + 1 tiles, so
// those of sequence s are found from f / 16 + s on, of n_tokens / 16 + n_seqs.
struct RowTile {
    int first, rows, adapter;  // rows 0: no tile
};
__device__ __forceinline__ RowTile row_tile(const LoraArgs &l, int i) {
    RowTile t = {16 * i, 0, NO_ADAPTER};
    if (!l.a) {
        t.rows = min(16, l.n_tokens - t.first);
        return t;
    }
    const int lane = threadIdx.x & 63;
    int s0 = 0;  // the sequence is among the 64 from s0 on, which are read at once
    if (l.n_seqs > 64) s0 = max(0, count_leading(l.n_seqs, [&](int j) { return start_of(l, j) / 16 + j <= i; }) - 1);
    const int s = min(s0 + lane, l.n_seqs - 1);
    const int f = start_of(l, s), n = start_of(l, s + 1) - f, adapter = gptr(l.adapter)[s];
    const uint64_t upto = __ballot(s0 + lane < l.n_seqs && f / 16 + s <= i);
    if (!upto) return t;
    const int at = 63 - __builtin_clzll(upto);
    const int first = __builtin_amdgcn_readlane(f, at), rows = __builtin_amdgcn_readlane(n, at), a = __builtin_amdgcn_readlane(adapter, at);
    const int j = i - (first / 16 + s0 + at);
    t.first = first + 16 * j;
    t.rows = max(0, min(16, rows - 16 * j));
    if ((unsigned)a < (unsigned)l.n_adapters) t.adapter = a;
    return t;
}

// low of 16 rows and 16 NT elements of the rank, of the sum's elements from `from` on; the waves of the workgroup
// take SPAN of them each. The sum into sums (LDS, [16][16 NT]).
template <int NT>
struct Low {
    static constexpr int U = NT == 4 ? 4 : 8;  // loads of each operand under way
    template <int WAVES>
    static __device__ __forceinline__ void sum(const LoraArgs &l, const RowTile &t, int r0, int from, int span, float *sums) {
        const int lane = threadIdx.x & 63, wave = wave_id();
        const bf16 *x = l.x + (t.first + min(lane % 16, t.rows - 1)) * l.x_stride;
        const bf16 *a = l.a + (int64_t)t.adapter * l.rank * l.n_in;
        const bf16 *row[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) row[j] = a + (int64_t)min(r0 + j * 16 + lane % 16, l.rank - 1) * l.n_in;
        const int to = min(l.n_in, from + (wave + 1) * span);
        f32x4 acc[NT] = {};
        for (int k0 = from + wave * span; k0 < to; k0 += 32 * U) {
            u32x4 xs[U], as[U][NT];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int k = k0 + 32 * u + lane / 16 * 8;
                xs[u] = k < to ? ld16(x + k) : u32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < NT; j++) as[u][j] = k < to ? ld16(row[j] + k) : u32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < NT; j++) acc[j] = Mfma<16>::mul(as[u][j], xs[u], acc[j]);
        }
        constexpr int ROW = 16 * NT;
        float *mine = sums + wave * 16 * ROW;
#pragma unroll
        for (int j = 0; j < NT; j++) *(f32x4 *)(mine + lane % 16 * ROW + j * 16 + lane / 16 * 4) = acc[j];
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * ROW; i += 64 * WAVES) {
            float y = 0.0f;
            for (int w = 0; w < WAVES; w++) y += sums[w * 16 * ROW + i];
            sums[i] = y;
        }
    }
};
constexpr int LOW_SPAN = 1024;  // elements of the sum per workgroup where a join adds their parts
__host__ __device__ __forceinline__ int low_width(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }

// For a join: part low_split of low, in 32 bits and without its scale.
template <int WAVES>
__device__ __forceinline__ void low_part(const LoraArgs &l, int block, float *lds) {
    const int width = low_width(l.rank), groups = (l.rank + width - 1) / width;
    const int split = block % l.low_splits, r0 = block / l.low_splits % groups * width;
    const RowTile t = row_tile(l, block / l.low_splits / groups);
    if (t.rows == 0 || t.adapter < 0) return;
    const int from = split * LOW_SPAN;
    if (width == 16) Low<1>::sum<WAVES>(l, t, r0, from, LOW_SPAN / WAVES, lds);
    else if (width == 32) Low<2>::sum<WAVES>(l, t, r0, from, LOW_SPAN / WAVES, lds);
    else Low<4>::sum<WAVES>(l, t, r0, from, LOW_SPAN / WAVES, lds);
    float *to = l.low_part + ((int64_t)split * l.n_tokens + t.first) * l.rank + r0;
    for (int i = threadIdx.x; i < 16 * width; i += 64 * WAVES)
        if (i / width < t.rows && r0 + i % width < l.rank) gptr(to)[(int64_t)(i / width) * l.rank + i % width] = lds[i];
}

// Otherwise: low as two bf16, and the rows' owners. 16 waves share the sum.
constexpr int LOW_WAVES = 16;
template <int NT>
__global__ __launch_bounds__(64 * LOW_WAVES) void low_kernel(LoraArgs l) {
    __shared__ __attribute__((aligned(16))) float sums[LOW_WAVES * 16 * 16 * NT];
    const int r0 = blockIdx.y * 16 * NT;
    const RowTile t = row_tile(l, blockIdx.x);
    if (blockIdx.y == 0) {
        if (blockIdx.x == 0) {
            const int begin = start_of(l, 0), end = max(begin, start_of(l, l.n_seqs));
            for (int i = threadIdx.x; i < l.n_tokens; i += 64 * LOW_WAVES)
                if (i < begin || i >= end) gptr(l.owner)[i] = NO_SEQUENCE;
        }
        if ((int)threadIdx.x < t.rows) gptr(l.owner)[t.first + threadIdx.x] = t.adapter;
    }
    if (t.rows == 0 || t.adapter < 0) return;
    const float scale = l.scale ? gptr(l.scale)[t.adapter] : 1.0f;
    Low<NT>::template sum<LOW_WAVES>(l, t, r0, 0, (l.n_in + 32 * LOW_WAVES - 1) / (32 * LOW_WAVES) * 32, sums);
    const int i = threadIdx.x, m = i / (16 * NT), r = r0 + i % (16 * NT);
    if (m >= t.rows || r >= l.rank) return;
    const float sum = sums[i] * scale;
    const float value = round_bf(sum), rest = fabsf(value) < INFINITY ? sum - value : 0.0f;
    LLM_GLOBAL uint16_t *low = gptr((uint16_t *)l.low) + (int64_t)(t.first + m) * 2 * l.rank + r;
    low[0] = (uint16_t)f2bf(value);
    low[l.rank] = (uint16_t)f2bf(rest);
}

// Four columns of a row, with the residual's.
__device__ __forceinline__ void store4(const LoraArgs &l, bf16 *to, const bf16 *res, f32x4 y, int n) {
    if (l.wide && n + 4 <= l.n_out) {
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

// Whether NaN or infinities were among eight elements; they are zeros then.
__device__ __forceinline__ bool clear_unfit_of(u32x4 &v) {
    bool found = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if ((v[j] & 0x7f80u) == 0x7f80u) v[j] &= 0xffff0000u, found = true;
        if ((v[j] & 0x7f800000u) == 0x7f800000u) v[j] &= 0xffffu, found = true;
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

// TM rows by TN columns of a workgroup, in waves of RM by RN, on MFMAs of side S; 64 elements of the sum a step,
// STAGES steps' operands in LDS. A row's 128 bytes of a step lie as eight 16-byte chunks, chunk c of row r at
// c ^ (r % 8): the rows that a product reads at one chunk then lie in different banks.
template <int TM_, int TN_, int RM_, int RN_, int S_, int STAGES_>
struct Shape {
    static constexpr int TM = TM_, TN = TN_, RM = RM_, RN = RN_, S = S_, STAGES = STAGES_;
    static constexpr int WM = TM / RM, WN = TN / RN, WAVES = WM * WN, T = 64 * WAVES, MT = RM / S, NT = RN / S;
    static constexpr int BYTES = (TM + TN) * 128;                    // of a stage
    static constexpr int X_LOADS = (TM / 8 + WAVES - 1) / WAVES;     // per wave, of eight rows; the last ones may be
    static constexpr int W_LOADS = (TN / 8 + WAVES - 1) / WAVES;     // loaded more than once
    static constexpr int LOADS = X_LOADS + W_LOADS;
    static constexpr int SUMS = WAVES * 16 * 64 * 4;                 // of low's parts
    static constexpr int LDS = STAGES * BYTES > SUMS ? STAGES * BYTES : SUMS;
};

template <class G>
__global__ __launch_bounds__(G::T) void product_kernel(LoraArgs l) {
    __shared__ __attribute__((aligned(128))) char lds[G::LDS + G::TM * 4 + 4];
    int *owner = (int *)(lds + G::LDS), *unfit = owner + G::TM;
    const int lane = threadIdx.x & 63, wave = wave_id();
    if ((int)blockIdx.x < l.low_groups) return low_part<G::WAVES>(l, blockIdx.x, (float *)lds);
    // the tiles of one XCD, whose workgroups every eighth one is, lie side by side
    const int tiles = l.m_tiles * l.n_tiles * l.splits, block = blockIdx.x - l.low_groups;
    const int each = tiles / XCDS, more = tiles % XCDS, xcd = block % XCDS;
    const int at = xcd * each + min(xcd, more) + block / XCDS;
    const int m0 = at % l.m_tiles * G::TM, n0 = at / l.m_tiles % l.n_tiles * G::TN, split = at / (l.m_tiles * l.n_tiles);
    const bool join = l.part != nullptr, adapters = l.a && !join;
    if (adapters && (int)threadIdx.x < G::TM)
        owner[threadIdx.x] = m0 + (int)threadIdx.x < l.n_tokens ? gptr(l.owner)[m0 + threadIdx.x] : NO_SEQUENCE;
    if (threadIdx.x == 0) *unfit = 0;

    // loads: lane's row lane / 8 and chunk lane % 8 of eight rows
    const unsigned base = (unsigned)(uintptr_t)(lds_char *)lds;
    const int row = lane / 8, chunk = lane % 8 ^ row;
    unsigned x_at[G::X_LOADS], w_at[G::W_LOADS];   // bytes from the tile's first row
    int x_row[G::X_LOADS];
    const auto x_group = [&](int i) { return min(wave * G::X_LOADS + i, G::TM / 8 - 1); };
    const auto w_group = [&](int i) { return min(wave * G::W_LOADS + i, G::TN / 8 - 1); };
#pragma unroll
    for (int i = 0; i < G::X_LOADS; i++) {
        x_row[i] = x_group(i) * 8 + row;
        x_at[i] = (unsigned)(min(x_row[i], l.n_tokens - 1 - m0) * l.x_stride * 2) + chunk * 16;
    }
#pragma unroll
    for (int i = 0; i < G::W_LOADS; i++)
        w_at[i] = (unsigned)min(w_group(i) * 8 + row, l.n_out - 1 - n0) * (unsigned)l.n_in * 2 + chunk * 16;
    const char *x_from = (const char *)(l.x + m0 * l.x_stride), *w_from = (const char *)(l.w + (int64_t)n0 * l.n_in);
    const int all_steps = l.w ? (l.n_in + 63) / 64 : 0, whole_steps = l.w ? l.n_in / 64 : 0;
    int step = split * l.split_steps;
    const int last_step = min(all_steps, step + l.split_steps);
    int current = NO_ADAPTER, piece = 0;  // the adapter whose part of the sum comes next
    unsigned of_adapter = 0;              // stages that hold some of it
    const int pieces = (2 * l.rank + 63) / 64;
    __syncthreads();

    // Load i of a step of whole chunks into stage `to`.
    const auto load_whole = [&](int i, int to) {
        const unsigned xs = base + to * G::BYTES;
        if (i < G::X_LOADS) load_to_lds(xs + x_group(i) * 1024, x_from + (int64_t)step * 128, x_at[i]);
        else load_to_lds(xs + G::TM * 128 + w_group(i - G::X_LOADS) * 1024, w_from + (int64_t)step * 128, w_at[i - G::X_LOADS]);
    };
    // Requests the next step's operands into stage `to`; false after the last.
    const int whole_end = min(whole_steps, last_step);
    const auto request = [&](int to) {
        const unsigned xs = base + to * G::BYTES, ws = xs + G::TM * 128;
        if (step < whole_end) {
#pragma unroll
            for (int i = 0; i < G::LOADS; i++) load_whole(i, to);
            step++;
            return true;
        }
        if (step < last_step) {  // the last step of a width that is no multiple of 64
            const char *x = x_from + (int64_t)step * 128, *w = w_from + (int64_t)step * 128;
            const bool there = step * 64 + chunk * 8 < l.n_in;
#pragma unroll
            for (int i = 0; i < G::X_LOADS; i++)
                load_to_lds(xs + x_group(i) * 1024, there ? x + x_at[i] : (const char *)&g_zeros);
#pragma unroll
            for (int i = 0; i < G::W_LOADS; i++)
                load_to_lds(ws + w_group(i) * 1024, there ? w + w_at[i] : (const char *)&g_zeros);
            step++;
            return true;
        }
        if (!adapters) return false;
        if (piece == 0) {  // the next higher adapter of the tile's rows
            int next = INT32_MAX;
#pragma unroll
            for (int i = 0; i < (G::TM + 63) / 64; i++) {
                const int o = owner[min(i * 64 + lane, G::TM - 1)];
                if (o > current) next = min(next, o);
            }
            for (int d = 1; d < 64; d *= 2) next = min(next, __shfl_xor(next, d));
            current = __builtin_amdgcn_readfirstlane(next);
        }
        if (current == INT32_MAX) return false;
        const int c = piece * 8 + chunk, chunks = l.rank / 8;
        const char *low = (const char *)(l.low + (int64_t)m0 * 2 * l.rank) + c * 16;
        const char *b = (const char *)(l.b + ((int64_t)current * l.n_out + n0) * l.rank) + (c >= chunks ? c - chunks : c) * 16;
        const bool there = c < 2 * chunks;
#pragma unroll
        for (int i = 0; i < G::X_LOADS; i++)
            load_to_lds(xs + x_group(i) * 1024, there && owner[x_row[i]] == current ? low + (int64_t)x_row[i] * 4 * l.rank
                                                                                  : (const char *)&g_zeros);
#pragma unroll
        for (int i = 0; i < G::W_LOADS; i++)
            load_to_lds(ws + w_group(i) * 1024,
                        there ? b + (int64_t)min(w_group(i) * 8 + row, l.n_out - 1 - n0) * 2 * l.rank : (const char *)&g_zeros);
        if (++piece == pieces) piece = 0;
        of_adapter |= 1u << to;
        return true;
    };
    // NaN and infinities of an adapter become zeros: times the zeros of other rows, or a remainder of zero, they
    // would be no numbers. The rows that they belong to get them in the end.
    const auto clear_unfit = [&](int from) {
        bool found = false;
        for (int c = threadIdx.x; c < G::TN * 8; c += G::T) {
            u32x4 *at = (u32x4 *)(lds + from * G::BYTES + G::TM * 128 + c * 16), v = *at;
            if (clear_unfit_of(v)) *at = v, found = true;
        }
        if (found) *unfit = 1;
        wait_lds();
        barrier();
    };

    typename Mfma<G::S>::Acc acc[G::MT][G::NT] = {};
    const int mine_m = wave % G::WM * G::RM, mine_n = wave / G::WM * G::RN;
    constexpr int KS = 64 / Mfma<G::S>::K;  // products of a step, on operands in alternating registers
    static_assert(KS % 2 == 0, "registers alternate");
    u32x4 xf[2][G::MT], wf[2][G::NT];
    const auto fetch = [&](int from, int k) {
        const char *xs = lds + from * G::BYTES, *ws = xs + G::TM * 128;
        const int r = lane % G::S, slot = (k * (64 / G::S) + lane / G::S) ^ (r & 7);
#pragma unroll
        for (int i = 0; i < G::MT; i++) xf[k % 2][i] = *(const u32x4 *)(xs + (mine_m + i * G::S + r) * 128 + slot * 16);
#pragma unroll
        for (int j = 0; j < G::NT; j++) wf[k % 2][j] = *(const u32x4 *)(ws + (mine_n + j * G::S + r) * 128 + slot * 16);
    };
    const auto multiply = [&](int k) {
#pragma unroll
        for (int i = 0; i < G::MT; i++)
#pragma unroll
            for (int j = 0; j < G::NT; j++) acc[i][j] = Mfma<G::S>::mul(wf[k % 2][j], xf[k % 2][i], acc[i][j]);
    };
    const auto begin = [&](int from) {
        if (of_adapter >> from & 1) {
            clear_unfit(from);
            of_adapter &= ~(1u << from);
        }
        fetch(from, 0);
    };

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
                acc[i][j] = Mfma<G::S>::mul(wf[(KS - 1) % 2][j], xf[(KS - 1) % 2][i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
        step++;
    }
    while (pending > 0) {
#pragma unroll
        for (int k = 0; k + 1 < KS; k++) {
            fetch(stage, k + 1);
            multiply(k);
        }
        if (pending > 1) {
            const int free = stage;
            stage = stage == G::STAGES - 1 ? 0 : stage + 1;
            wait_lds();
            if (pending == G::STAGES) wait_loads<(G::STAGES - 2) * G::LOADS>();
            else wait_loads<0>();
            barrier();
            if (pending == G::STAGES && request(free)) pending++;
            begin(stage);
        }
        multiply(KS - 1);
        pending--;
    }
    wait_lds();
    barrier();

    // a lane has four columns side by side of a row
#pragma unroll
    for (int i = 0; i < G::MT; i++) {
        const int tile_row = mine_m + i * G::S + lane % G::S, m = m0 + tile_row;
        if (m >= l.n_tokens || (adapters && owner[tile_row] == NO_SEQUENCE)) continue;
        bf16 *to = l.out + m * l.out_stride;
        const bf16 *res = l.residual + m * l.residual_stride;
        float *part = l.part + ((int64_t)split * l.n_tokens + m) * l.part_width;
#pragma unroll
        for (int j = 0; j < G::NT; j++)
#pragma unroll
            for (int r = 0; r < Mfma<G::S>::REGS / 4; r++) {
                const int n = n0 + mine_n + j * G::S + Mfma<G::S>::row(r, lane);
                if (n >= l.n_out) continue;
                const f32x4 y = {acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
                if (join) *gptr((f32x4 *)(part + n)) = y;
                else store4(l, to + n, res + n, y, n);
            }
    }
    if (adapters && *unfit) {  // infinities and NaN, behind what was written
        __syncthreads();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "agent");
        for (int i = threadIdx.x; i < G::TM * G::TN; i += G::T) {
            const int m = m0 + i / G::TN, n = n0 + i % G::TN, a = owner[i / G::TN];
            if (a < 0 || n >= l.n_out) continue;
            const uint16_t *low = (const uint16_t *)l.low + (int64_t)m * 2 * l.rank;
            const float more = unfit_term(l, n, a, [&](int j) { return bf2f(gptr(low)[j]) + bf2f(gptr(low)[l.rank + j]); });
            LLM_GLOBAL bf16 *to = gptr(l.out) + m * l.out_stride + n;
            if (!(fabsf(more) < INFINITY)) *to = (bf16)f2bf(bf2f(*to) + more);
        }
    }
}

// ------------------------------------------------------------------------------------------
// the join: the parts of the product, the adapters' term and the residual
// ------------------------------------------------------------------------------------------

// 16 rows of a sequence by 256 columns per workgroup. The rows' low is added up once, into LDS; the first parts of the
// product, and what b and the residual hold for few rows, are requested in front of that, so that all of it comes in
// one round trip behind the lookup of the rows.
constexpr int FEW = 4;      // rows up to which a lane has a column, and the sum over the rank is one of vector operations
constexpr int PARTS = 4;    // parts, and chunks of b, under way

// low of the tile's rows, from its parts.
__device__ __forceinline__ void join_low(const LoraArgs &l, const RowTile &t, float *low) {
    const float *from = l.low_part + (int64_t)t.first * l.rank;
    for (int i = threadIdx.x; i < t.rows * l.rank; i += 256) {
        float y = 0.0f;
        constexpr int U = 8;
        for (int s0 = 0; s0 < l.low_splits; s0 += U) {
            float part[U];
#pragma unroll
            for (int s = 0; s < U; s++)
                part[s] = s0 + s < l.low_splits ? gptr(from)[(int64_t)(s0 + s) * l.n_tokens * l.rank + i] : 0.0f;
#pragma unroll
            for (int s = 0; s < U; s++) y += part[s];
        }
        low[i] = y;
    }
    const float scale = l.scale ? gptr(l.scale)[t.adapter] : 1.0f;
    for (int i = threadIdx.x; i < t.rows * l.rank; i += 256) low[i] *= scale;
    __syncthreads();
}

__device__ __forceinline__ void join_few(const LoraArgs &l, const RowTile &t, int n, float *low) {
    const int at = min(n, l.n_out - 1);
    const auto part_at = [&](int i, int s) {
        return i < t.rows && s < l.splits ? gptr(l.part)[((int64_t)s * l.n_tokens + t.first + i) * l.part_width + at] : 0.0f;
    };
    float part[FEW][PARTS], res[FEW], y[FEW] = {};
    u32x4 v[PARTS];
    const bf16 *b = l.b + ((int64_t)max(t.adapter, 0) * l.n_out + at) * l.rank;
    const int rank = t.adapter >= 0 ? l.rank : 0;
#pragma unroll
    for (int c = 0; c < PARTS; c++)
        if (c * 8 < rank) v[c] = ld16(b + c * 8);
#pragma unroll
    for (int i = 0; i < FEW; i++) {
#pragma unroll
        for (int s = 0; s < PARTS; s++) part[i][s] = part_at(i, s);
        res[i] = l.residual && i < t.rows ? bf2f(gptr(l.residual)[(t.first + i) * l.residual_stride + at]) : 0.0f;
    }
    if (rank) join_low(l, t, low);
#pragma unroll
    for (int i = 0; i < FEW; i++)
#pragma unroll
        for (int s = 0; s < PARTS; s++) y[i] += part[i][s];
    for (int s0 = PARTS; s0 < l.splits; s0 += PARTS) {
#pragma unroll
        for (int i = 0; i < FEW; i++)
#pragma unroll
            for (int s = 0; s < PARTS; s++) part[i][s] = part_at(i, s0 + s);
#pragma unroll
        for (int i = 0; i < FEW; i++)
#pragma unroll
            for (int s = 0; s < PARTS; s++) y[i] += part[i][s];
    }
#pragma unroll
    for (int i = 0; i < FEW; i++) y[i] += res[i];
    for (int j0 = 0; j0 < rank; j0 += 8 * PARTS) {
        u32x4 next[PARTS];
#pragma unroll
        for (int c = 0; c < PARTS; c++)
            if (j0 + (PARTS + c) * 8 < rank) next[c] = ld16(b + j0 + (PARTS + c) * 8);
#pragma unroll
        for (int c = 0; c < PARTS; c++) {
            if (j0 + c * 8 >= rank) break;
#pragma unroll
            for (int i = 0; i < FEW; i++)
                if (i < t.rows)
#pragma unroll
                    for (int e = 0; e < 8; e++) y[i] = fmaf(low[i * rank + j0 + c * 8 + e], elem(v[c], e), y[i]);
            v[c] = next[c];
        }
    }
    if (n < l.n_out)
#pragma unroll
        for (int i = 0; i < FEW; i++)
            if (i < t.rows) gptr(l.out)[(t.first + i) * l.out_stride + n] = (bf16)f2bf(y[i]);
}

__global__ __launch_bounds__(256) void join_kernel(LoraArgs l) {
    __shared__ float low[16 * 256];
    const int lane = threadIdx.x & 63, wave = wave_id();
    const RowTile t = row_tile(l, blockIdx.x);
    if (t.rows == 0) return;
    if (t.rows <= FEW) return join_few(l, t, blockIdx.y * 256 + threadIdx.x, low);
    // a lane has row lane % 16 and four columns of each 16
    const int n0 = (blockIdx.y * 4 + wave) * 64, mine = min(lane % 16, t.rows - 1), m = t.first + mine;
    const auto part_at = [&](int j, int s) {
        if (s >= l.splits) return f32x4{0, 0, 0, 0};
        const int n = min(n0 + j * 16 + lane / 16 * 4, l.part_width - 4);
        return *gptr((const f32x4 *)(l.part + ((int64_t)s * l.n_tokens + m) * l.part_width + n));
    };
    f32x4 part[4][PARTS], y[4] = {};
#pragma unroll
    for (int s = 0; s < PARTS; s++)
#pragma unroll
        for (int j = 0; j < 4; j++) part[j][s] = part_at(j, s);
    if (t.adapter >= 0) join_low(l, t, low);
    if (n0 >= l.n_out) return;
#pragma unroll
    for (int s = 0; s < PARTS; s++)
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] += part[j][s];
    for (int s0 = PARTS; s0 < l.splits; s0 += PARTS) {
#pragma unroll
        for (int s = 0; s < PARTS; s++)
#pragma unroll
            for (int j = 0; j < 4; j++) part[j][s] = part_at(j, s0 + s);
#pragma unroll
        for (int s = 0; s < PARTS; s++)
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] += part[j][s];
    }
    f32x4 acc[4] = {};
    bool unfit = false;
    if (t.adapter >= 0) {
        const bf16 *b = l.b + (int64_t)t.adapter * l.n_out * l.rank;
        constexpr int U = 2;
        for (int c0 = 0; c0 < l.rank / 8; c0 += 4 * U) {
            u32x4 v[U][4];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
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
                        const float y0 = from[2 * e], y1 = from[2 * e + 1], v0 = round_bf(y0), v1 = round_bf(y1);
                        value[e] = pack2(y0, y1);
                        rest[e] = pack2(fabsf(v0) < INFINITY ? y0 - v0 : 0.0f, fabsf(v1) < INFINITY ? y1 - v1 : 0.0f);
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    unfit |= clear_unfit_of(v[u][j]);
                    acc[j] = Mfma<16>::mul(v[u][j], value, acc[j]);
                    acc[j] = Mfma<16>::mul(v[u][j], rest, acc[j]);
                }
            }
        }
    }
    unfit = __any(unfit);
    if (lane % 16 >= t.rows) return;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = n0 + j * 16 + lane / 16 * 4;
        if (n >= l.n_out) break;
        y[j] += acc[j];
        if (unfit)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < l.n_out) y[j][e] += unfit_term(l, n + e, t.adapter, [&](int i) { return low[mine * l.rank + i]; });
        store4(l, l.out + m * l.out_stride + n, l.residual + m * l.residual_stride + n, y[j], n);
    }
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
typedef Shape<256, 192, 64, 96, 16, 2> Wide;
typedef Shape<224, 256, 112, 64, 16, 2> High;
typedef Shape<192, 256, 96, 64, 16, 2> Square;
typedef Shape<128, 256, 64, 64, 16, 3> Half;
typedef Shape<128, 128, 32, 64, 16, 2> Quarter;
typedef Shape<64, 128, 64, 32, 16, 3> Low64;
typedef Shape<64, 64, 64, 16, 16, 4> Small;
typedef Shape<16, 64, 16, 16, 16, 4> Row;
constexpr Pace PACES[] = {{256, 192, 1, 930, 1130, 11000}, {224, 256, 1, 1050, 1250, 11000}, {192, 256, 1, 920, 1050, 11000},
                          {128, 256, 1, 620, 780, 8000},   {128, 128, 2, 560, 760, 6000},    {64, 128, 2, 400, 500, 4500},
                          {64, 64, 2, 300, 400, 4000},     {16, 64, 3, 250, 350, 3500}};
constexpr int SHAPES = sizeof(PACES) / sizeof(PACES[0]);

constexpr int MOST_SPLITS = 32, MOST_JOINED = 2048;
constexpr size_t MOST_PART = 1 << 23;  // floats

// How a call is computed: the product's tiles, its splits, and whether a join adds them and the adapters' term.
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
        const int64_t one = (int64_t)part_floats(n_tokens, n_out);
        const int most = (int)std::min<int64_t>(std::min(MOST_SPLITS, std::max(steps, 1)), MOST_PART / one);
        double least = 0;
        shape = -1;
        for (int i = 0; i < SHAPES; i++) {
            const Pace &s = PACES[i];
            const double tiles = (double)((n_tokens + s.tm - 1) / s.tm) * ((n_out + s.tn - 1) / s.tn);
            const auto consider = [&](int n, bool joined) {
                // adapters of a tile's rows, each with steps of its own
                const double own = !joined && adapters
                    ? pieces * std::min<double>(n_adapters, 1.0 + (double)n_seqs * std::min(s.tm, n_tokens) / n_tokens) : 0;
                const double groups = tiles * n, rounds = ceil(groups / (s.at_once * CUS)), busy = std::min(1.0, groups / CUS);
                const double step = s.alone + (s.full - s.alone) * busy;
                const double cost = rounds * (((steps + n - 1) / n + own) * step + s.fixed) +
                                    (joined ? 5000 + one * (n * 8.0 + 4) / 4500 : adapters ? 5000 : 0);
                if (shape < 0 || cost < least) shape = i, splits = n, join = joined, least = cost;
            };
            consider(1, false);
            for (int n = adapters || !product ? 1 : 2; n <= most && n_tokens <= MOST_JOINED; n++) consider(n, true);
        }
        split_steps = (steps + splits - 1) / splits;
        splits = split_steps ? (steps + split_steps - 1) / split_steps : join ? 0 : 1;
    }
};

template <class G>
bool launch_product(const char *name, LoraArgs l, hipStream_t stream) {
    l.m_tiles = (l.n_tokens + G::TM - 1) / G::TM;
    l.n_tiles = (l.n_out + G::TN - 1) / G::TN;
    const int64_t groups = l.low_groups + (int64_t)l.m_tiles * l.n_tiles * l.splits;
    if (groups * G::T >= 1ll << 32)  // the threads of a launch
        return llm_fail("%s: n_tokens %d by n_out %d is too much for one launch", name, l.n_tokens, l.n_out);
    if (groups) product_kernel<G><<<groups, G::T, 0, stream>>>(l);
    return LAUNCH_OK();
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

int low_splits(int n_in) { return (n_in + LOW_SPAN - 1) / LOW_SPAN; }
// Of low: as two bf16, or of its parts, which a join of at most MOST_JOINED rows adds.
size_t low_floats(int n_tokens, int n_in, int rank) {
    return (size_t)rank * std::max(n_tokens, std::min(n_tokens, MOST_JOINED) * low_splits(n_in));
}
size_t owner_floats(int n_tokens, int rank) { return rank ? ((size_t)n_tokens + 3) / 4 * 4 : 0; }

}  // namespace

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
    l.wide = out_stride % 4 == 0 && (uintptr_t)out % 8 == 0 &&
             (!residual || (residual_stride % 4 == 0 && (uintptr_t)residual % 8 == 0));
    l.low = (bf16 *)ws;
    l.low_part = ws;
    l.low_splits = low_splits(n_in);
    l.owner = (int *)(ws + low_floats(n_tokens, n_in, rank));
    float *part = ws + low_floats(n_tokens, n_in, rank) + owner_floats(n_tokens, rank);
    int tiles = (n_tokens + 15) / 16;
    if (lora) {
        l.a = lora->a, l.b = lora->b, l.scale = lora->scale, l.q_start = lora->q_start, l.adapter = lora->adapter;
        l.n_seqs = lora->n_seqs, l.n_adapters = lora->n_adapters, l.rank = rank;
        tiles = n_tokens / 16 + lora->n_seqs;
    }
    const auto product = [&](const LoraArgs &a) {
        switch (p.shape) {
        case 0: return launch_product<Wide>(name, a, stream);
        case 1: return launch_product<High>(name, a, stream);
        case 2: return launch_product<Square>(name, a, stream);
        case 3: return launch_product<Half>(name, a, stream);
        case 4: return launch_product<Quarter>(name, a, stream);
        case 5: return launch_product<Low64>(name, a, stream);
        case 6: return launch_product<Small>(name, a, stream);
        default: return launch_product<Row>(name, a, stream);
        }
    };
    if (p.join) {
        l.part = part;
        if (lora) l.low_groups = tiles * ((rank + low_width(rank) - 1) / low_width(rank)) * l.low_splits;
        if (!product(l)) return;
        join_kernel<<<dim3(tiles, (n_out + 255) / 256), 256, 0, stream>>>(l);
        LAUNCH_OK();
        return;
    }
    if (lora) {
        const int width = low_width(rank);
        const dim3 grid(tiles, (rank + width - 1) / width);
        if (width == 16) low_kernel<1><<<grid, 64 * LOW_WAVES, 0, stream>>>(l);
        else if (width == 32) low_kernel<2><<<grid, 64 * LOW_WAVES, 0, stream>>>(l);
        else low_kernel<4><<<grid, 64 * LOW_WAVES, 0, stream>>>(l);
        if (!LAUNCH_OK()) return;
    }
    product(l);
}
