// The batch of sequences over pages (include/llm_amd/paged.h) as the kernels see it, and its checks on the
// host.
#pragma once

#include <algorithm>

#include "common.h"
#include "llm_amd/paged.h"

namespace llm {
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

// The number of leading i in [0, n) with pred(i), pred not increasing: 64 probes per round, one per lane.
// Whatever pred says, the result is in [0, n] and pred is asked about [0, n) alone.
template <class Pred>
__device__ __forceinline__ int count_leading(int n, Pred pred) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;
        const int64_t at = lo + (int64_t)(lane + 1) * step - 1;  // the last of the lane's share
        const int met = __popcll(__ballot(at < hi && pred((int)at)));
        hi = min(hi, lo + met * step + step - 1);
        lo += met * step;
    }
    return lo;
}

// The sequence whose rows hold row t, or -1.
__device__ __forceinline__ int sequence_of(const Batch &b, int t) {
    const int s = count_leading(b.n_seqs, [&](int i) { return gptr(b.q_start)[i + 1] <= t; });
    if (s >= b.n_seqs || gptr(b.q_start)[s] > t || gptr(b.q_start)[s + 1] <= t) return -1;
    return s;
}

// Lengths outside [-2^30, 2^30] are cut to it, so that positions do not overflow.
__device__ __forceinline__ int kv_length(const Batch &b, int s) {
    return max(-(1 << 30), min(1 << 30, gptr(b.kv_len)[s]));
}

// Element offset of position p of sequence s in the caches (head 0), or -1 where it is not there. Without
// branches, so that several lookups' loads go out together.
template <class B>
__device__ __forceinline__ int64_t place(B &b, int s, int p) {
    const int i = divide(max(p, 0), b.page.m, b.page.l);
    const int page = gptr(b.table)[(int64_t)s * b.table_pages + min(i, b.table_pages - 1)];
    const bool there = p >= 0 && i < b.table_pages && (unsigned)page < (unsigned)b.n_pages;
    return there ? page * b.page_stride + (p - i * b.page_size) * b.slot_stride : -1;
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
    if (p->n_seqs > 1 << 20) return llm_fail("%s: n_seqs %d is over 1048576", name, p->n_seqs);
    if (n_tokens < 0 || n_tokens > 1 << 24)
        return llm_fail("%s: n_tokens %d is not in 0..16777216", name, n_tokens);
    if (!p->key_cache || !p->value_cache || !p->page_table || !p->q_start || !p->kv_len)
        return llm_fail("%s: the batch has a null pointer", name);
    if (!aligned16(p->key_cache) || !aligned16(p->value_cache))
        return llm_fail("%s: the caches must be 16-byte aligned", name);
    if (p->page_stride < 0 || p->slot_stride < 0 || p->head_stride < 0 || p->slot_stride > 1 << 26)
        return llm_fail("%s: cache strides %lld, %lld, %lld: none may be negative, nor slots over 2^26 apart", name,
                        (long long)p->page_stride, (long long)p->slot_stride, (long long)p->head_stride);
    if (p->page_stride % 8 || p->slot_stride % 8 || p->head_stride % 8)
        return llm_fail("%s: cache strides %lld, %lld, %lld are not multiples of 8", name,
                        (long long)p->page_stride, (long long)p->slot_stride, (long long)p->head_stride);
    if (p->page_size > 1 && p->slot_stride < p->head_dim)
        return llm_fail("%s: slots %lld elements apart overlap (head_dim %d)", name, (long long)p->slot_stride, p->head_dim);
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

}  // namespace
}  // namespace llm
