// paged.cuh -- index arithmetic of the paged latent cache and its batches of new tokens.
//
// Page tables, cache lengths and token offsets are device arrays (a captured graph replays with
// the values they hold then), so the host cannot check them: every kernel takes them through
// the functions below, which never return an index outside the arrays they index. What they
// find wrong is recorded in the context's error block (word 1) and reported by the next
// k3cuda_sync. The functions are plain C++ without CUDA types, so a host compiler checks them.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define K3_HD __host__ __device__ __forceinline__
#else
#define K3_HD inline
#endif

namespace k3 {

// What a kernel found wrong in the device-side tables (word 1 of the error block).
enum PagedError {
    PAGED_OK = 0,
    PAGED_OFFSETS = 1,  // cu_tokens falls, is negative or ends past the token rows: this sequence
                        // and all behind it are left out (paged_in_order)
    PAGED_LENGTH = 2,   // ctx_lens negative
    PAGED_DRAFTS = 3,   // more new tokens than the call takes per sequence
    PAGED_TABLE = 4,    // rows past the sequence's page table
    PAGED_PAGE = 5      // a page number outside the cache
};

// The cache and the batch as the kernels see them (k3cuda_paged_cache, k3cuda_token_batch).
struct PagedView {
    const int *table;   // [B][max_pages]
    int n_pages, page_size, max_pages;
    const int *lens;    // [B]
    const int *cu;      // [B + 1]
    int B, T;
    int shift;          // log2 of page_size
};

// Whether sequence b's offsets are in order. The sequences that count are those before the first
// whose offsets are not, so that no two of them have a row in common: a caller of paged_seq sees to
// that.
K3_HD bool paged_in_order(const PagedView &v, int b) {
    return v.cu[b] >= 0 && v.cu[b] <= v.cu[b + 1] && v.cu[b + 1] <= v.T;
}

// Sequence b's new tokens: rows first .. first + n - 1 of the token arrays, behind `len` cached
// rows. A sequence that breaks a rule has n = 0 and says why in `code`.
struct PagedSeq {
    int first, n, len, code;
};

K3_HD PagedSeq paged_seq(const PagedView &v, int b, int max_n) {
    PagedSeq s;
    s.first = v.cu[b];
    s.len = v.lens[b];
    s.code = PAGED_OK;
    const long long n = (long long)v.cu[b + 1] - s.first;
    if (s.first < 0 || n < 0 || s.first + n > v.T) s.code = PAGED_OFFSETS;
    else if (n > 0 && s.len < 0) s.code = PAGED_LENGTH;
    else if (n > max_n) s.code = PAGED_DRAFTS;
    else if (n > 0 && (long long)s.len + n > (long long)v.max_pages * v.page_size)
        s.code = PAGED_TABLE;
    s.n = s.code ? 0 : (int)n;
    return s;
}

// The cache row of sequence b's position pos (0 <= pos < max_pages * page_size, as paged_seq
// has checked), or -1 where the table names a page that the cache does not have.
K3_HD long long paged_row(const PagedView &v, int b, int pos) {
    const int page = v.table[(long long)b * v.max_pages + (pos >> v.shift)];
    if (page < 0 || page >= v.n_pages) return -1;
    return ((long long)page << v.shift) + (pos & (v.page_size - 1));
}

// Work line of the tree attention. Every (sequence, row tile) is a unit that takes `fixed` +
// tiles places on a line; cluster c of G takes places [total c / G, total (c + 1) / G).
K3_HD long long line_begin(long long total, int G, int c) { return total * c / G; }
// The cluster that holds place x: the last c with total c / G <= x.
K3_HD int line_cluster(long long total, int G, long long x) {
    return (int)(((x + 1) * G - 1) / total);
}

// Largest i in [0, n) with a[i] <= x, where a[0] <= x (0 where no element is).
template <typename A, typename X> K3_HD int last_at_most(const A *a, int n, X x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if ((X)a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Which of the 64 positions p0 .. p0 + 63 a draft sees, as bits: every cached position (below
// len), and the drafts j (at len + j, j < n) whose bit is set in `mask`.
K3_HD uint64_t tree_bits(uint64_t mask, int len, int n, long long p0) {
    if (n < 64) mask &= ((uint64_t)1 << n) - 1;
    const long long d = p0 - len;  // draft index of the first position
    if (d >= 64) return 0;
    if (d >= 0) return mask >> d;
    if (d <= -64) return ~(uint64_t)0;
    return (mask << -d) | (((uint64_t)1 << -d) - 1);
}

}  // namespace k3
