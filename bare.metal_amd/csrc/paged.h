/* SPDX-License-Identifier: MPL-2.0
 *
 * paged.h — what the kernels over a paged cache share (include/bm_paged.h):
 * the batch's tables and their checks.
 */
#ifndef BMK_PAGED_COMMON_H
#define BMK_PAGED_COMMON_H

#include "bmk.h"

namespace bmk {

/* Rows, sequences and strides a launch takes at most, so that row and column indexes stay inside an int. */
constexpr int PG_MAX_DIM = 1 << 30;
constexpr int PG_MAX_HD = 256, PG_MAX_SEQS = 4096;

/* A launch's workgroups, side by side and in as few rows as take them: HIP has fewer than 2^32 work-items along an axis.
 * The last row may have workgroups over, fewer than there are rows. */
inline dim3 pg_grid(int64_t groups, int lanes) {
    const int64_t most = ((1LL << 32) - 1) / lanes, rows = (groups + most - 1) / most;
    return dim3((unsigned int)((groups + rows - 1) / rows), (unsigned int)rows);
}
__device__ __forceinline__ unsigned int pg_group() { return blockIdx.y * gridDim.x + blockIdx.x; }

/* x / d for x below 2^31 by one product */
struct Div {
    unsigned int d, mul, shift;
    __device__ __forceinline__ int of(int x) const { return (int)((__umulhi((unsigned int)x, mul) + (unsigned int)x) >> shift); }
};
inline Div div_by(int d) {
    Div v = {(unsigned int)d, 0, 0};
    while ((1ull << v.shift) < (unsigned int)d) v.shift++;
    v.mul = (unsigned int)(((1ull << 32) * ((1ull << v.shift) - d)) / d + 1);
    return v;
}

/* The batch's tables and the cache's shape. */
struct PgBatch {
    const int* start; /* [S + 1] */
    const int* len;   /* [S] */
    const int* pages; /* [S][max_pages] */
    int N, S, NKV, HD;
    int shift; /* page = 1 << shift tokens */
    int n_pages, max_pages;

    /* keys that the page table has room for */
    __host__ __device__ int room() const { return max_pages << shift; }
    /* Sequence of row n, the last one that starts at or before it, or -1 where
     * the row is outside all of them.  Ends, inside the table, whatever that holds. */
    __host__ __device__ __forceinline__ int seq_of(int n) const {
        if (n < start[0] || n >= start[S]) return -1;
        int lo = 0, hi = S;
        while (hi - lo > 1) {
            const int mid = lo + ((hi - lo) >> 1);
            if (start[mid] <= n) lo = mid;
            else hi = mid;
        }
        return lo;
    }
    /* position of row n of sequence s; sums that leave an int wrap and fall out as positions without a page */
    __host__ __device__ __forceinline__ int pos_of(int s, int n) const {
        return (int)((unsigned int)len[s] - (unsigned int)start[s + 1] + (unsigned int)n);
    }
    /* page of sequence s's key j, or -1 where it is missing */
    __host__ __device__ __forceinline__ int page_of(int s, int j) const {
        if (j < 0 || j >= room()) return -1;
        const int pg = pages[(size_t)s * max_pages + (j >> shift)];
        return pg >= 0 && pg < n_pages ? pg : -1;
    }
    /* first element of a KV head's keys (part 0) or values (1) in page pg, which lies in 0 .. n_pages - 1 */
    __device__ __forceinline__ size_t base(int pg, int part, int kh) const {
        return ((((size_t)pg * 2 + part) * NKV + kh) << shift) * HD;
    }
};

/* elements of `rows` rows of `width`, ld apart */
inline size_t pg_span(int rows, size_t width, int ld) { return (size_t)(rows - 1) * (size_t)ld + width; }

inline int pg_log2(int v) { /* of a power of two, else -1 */
    return v > 0 && (v & (v - 1)) == 0 ? __builtin_ctz((unsigned)v) : -1;
}

} // namespace bmk

#define BMK_NEED_ALIGNED(a, i, by, what) \
    BMK_REQUIRE(((uintptr_t)(a)->dev[i] & ((by) - 1)) == 0, "%s: buffer %d (%s) lies off a %d-byte boundary", __func__, i, \
                what, (int)(by))

/* A matrix of `rows` rows of `width` elements of esz bytes, ld elements apart, in buffer i. */
#define BMK_NEED_ROWS(a, i, rows, width, ld, esz, what) do { \
    BMK_REQUIRE((ld) <= bmk::PG_MAX_DIM && (ld) > 0 && (size_t)(ld) >= (size_t)(width), \
                "%s: %s rows of %zu elements, stride %d", __func__, what, (size_t)(width), (int)(ld)); \
    BMK_NEED_BYTES(a, i, bmk::pg_span(rows, width, ld) * (esz), what); \
    BMK_NEED_ALIGNED(a, i, esz, what); \
} while (0)

/* The tables in buffers i, i + 1, i + 2 and the cache in buffer c, for a batch whose numbers are set. */
#define BMK_NEED_BATCH(a, b, page, i, c, esz) do { \
    (b).shift = bmk::pg_log2(page); \
    BMK_REQUIRE((b).shift >= 3 && (page) <= 65536 && (b).n_pages > 0 && (b).max_pages > 0 && \
                    (int64_t)(b).max_pages * (page) <= bmk::PG_MAX_DIM && (int64_t)(b).n_pages * (page) <= (1LL << 38), \
                "%s: bad cache: page %d, n_pages %d, max_pages %d", __func__, (int)(page), (b).n_pages, (b).max_pages); \
    BMK_REQUIRE((b).HD % 8 == 0 && (b).NKV <= 4096, "%s: cache of %d heads of %d", __func__, (b).NKV, (b).HD); \
    BMK_NEED_BYTES(a, i, ((size_t)(b).S + 1) * 4, "start"); \
    BMK_NEED_BYTES(a, (i) + 1, (size_t)(b).S * 4, "len"); \
    BMK_NEED_BYTES(a, (i) + 2, (size_t)(b).S * (b).max_pages * 4, "pages"); \
    for (int t_ = 0; t_ < 3; t_++) BMK_NEED_ALIGNED(a, (i) + t_, 4, "table"); \
    BMK_NEED_BYTES(a, c, ((size_t)(b).n_pages * 2 * (b).NKV << (b).shift) * (b).HD * (esz), "cache"); \
    BMK_NEED_ALIGNED(a, c, 16, "cache"); \
    (b).start = (const int*)(a)->dev[i]; \
    (b).len = (const int*)(a)->dev[(i) + 1]; \
    (b).pages = (const int*)(a)->dev[(i) + 2]; \
} while (0)

#endif
