/* SPDX-License-Identifier: MPL-2.0
 *
 * attn_paged.hip — attention_forward_paged (include/bm_paged.h): the new
 * tokens of several sequences over the keys in their pages,
 *   out = softmax(scale * q . K + mask) V,
 * in one pass over the keys with the running maximum and sum (fp32) of the
 * softmax.  A wave takes one head of one row: 64 keys at a time, a lane the
 * score of one of them, then a dimension (or up to four) of the output.
 */
#include "paged.h"
#include "q8_common.h"

#include <math.h>

namespace {

using namespace bmk;

struct PaArgs {
    const void* q;
    const void* cache;
    void* out;
    PgBatch b;
    int NH, R; /* R: query heads a KV head */
    int causal, window;
    size_t ldq, ldo;
    float scale;
};

template <bool BF16>
__device__ __forceinline__ float at(const void* p, size_t i) {
    return BF16 ? __uint_as_float((unsigned int)((const unsigned short*)p)[i] << 16) : ((const float*)p)[i];
}

template <bool BF16>
__global__ __launch_bounds__(64) void k_attn_paged(PaArgs a) {
    __shared__ float qs[PG_MAX_HD];
    const PgBatch& b = a.b;
    const int lane = threadIdx.x, n = blockIdx.x / a.NH, h = blockIdx.x % a.NH, HD = b.HD, kh = h / a.R;
    const int s = b.seq_of(n);
    if (s < 0) return;
    const int p = b.pos_of(s, n);
    const int last = a.causal ? p : max(b.len[s], 0) - 1; /* keys first .. last are seen */
    const int first = a.window ? max(0, p - a.window + 1) : 0;
    bool missing = last >= b.room();
    for (int d = lane; d < HD; d += 64) qs[d] = at<BF16>(a.q, (size_t)n * a.ldq + (size_t)h * HD + d);
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[PG_MAX_HD / 64] = {};
    for (int base = first; base <= min(last, b.room() - 1); base += 64) {
        const int j = base + lane;
        const bool in = j <= last && j < b.room();
        const int pg = in ? b.page_of(s, j) : -1;
        const bool there = pg >= 0;
        missing |= in && !there;
        const size_t row = there ? b.base(pg, 0, kh) + (size_t)(j & ((1 << b.shift) - 1)) * HD : 0;
        float sc = 0.0f;
        if (there)
            for (int d = 0; d < HD; d++) sc = fmaf(qs[d], at<BF16>(a.cache, row + d), sc);
        sc = there ? sc * a.scale : -INFINITY;
        const float mn = fmaxf(m, wave_max(sc)), f = m > -INFINITY ? expf(m - mn) : 0.0f;
        const float w = there ? expf(sc - (mn > -INFINITY ? mn : 0.0f)) : 0.0f;
        l = l * f + wave_sum(w);
#pragma unroll
        for (int e = 0; e < PG_MAX_HD / 64; e++) acc[e] *= f;
        m = mn;
        const size_t v = row + ((size_t)b.NKV * HD << b.shift);
        for (int k = 0; k < 64; k++) {
            const float wk = __shfl(w, k);
            const size_t vk = __shfl((unsigned long long)v, k);
            if (!__shfl((int)there, k)) continue;
#pragma unroll
            for (int e = 0; e < PG_MAX_HD / 64; e++)
                if (lane + 64 * e < HD) acc[e] = fmaf(wk, at<BF16>(a.cache, vk + lane + 64 * e), acc[e]);
        }
    }
    missing = __any(missing);
#pragma unroll
    for (int e = 0; e < PG_MAX_HD / 64; e++) {
        const int d = lane + 64 * e;
        if (d >= HD) continue;
        const float o = missing ? NAN : last < first ? 0.0f : acc[e] / l;
        const size_t i = (size_t)n * a.ldo + (size_t)h * HD + d;
        if (BF16) ((unsigned short*)a.out)[i] = bf16_bits(o);
        else ((float*)a.out)[i] = o;
    }
}

/* {q T [N][ldq], cache, out T [N][ldo], start, len, pages,
 *  params int{N, S, NH, NKV, HD, ldq, ldo, page, n_pages, max_pages, causal, window}, f32{scale}} */
int launch_attn_paged(const bmk_launch_t* l, bool bf16) {
    BMK_NEED_BYTES(l, 6, 48, "params");
    BMK_NEED_BYTES(l, 7, 4, "scale");
    const int N = bmk_pi(l, 6, 0), S = bmk_pi(l, 6, 1), NH = bmk_pi(l, 6, 2), NKV = bmk_pi(l, 6, 3), HD = bmk_pi(l, 6, 4);
    const int ldq = bmk_pi(l, 6, 5), ldo = bmk_pi(l, 6, 6), causal = bmk_pi(l, 6, 10), window = bmk_pi(l, 6, 11);
    BMK_REQUIRE(N >= 0 && N <= PG_MAX_DIM && S >= 0 && S <= PG_MAX_DIM && NH > 0 && NH <= PG_MAX_DIM && NKV > 0 &&
                    NH % NKV == 0 && HD > 0 && HD <= PG_MAX_HD,
                "attention_forward_paged: bad shape N=%d S=%d NH=%d NKV=%d HD=%d", N, S, NH, NKV, HD);
    BMK_REQUIRE((causal == 1 && window >= 0) || (causal == 0 && window == 0),
                "attention_forward_paged: bad mask causal=%d window=%d", causal, window);
    BMK_REQUIRE((int64_t)N * NH < (1LL << 31), "attention_forward_paged: %d rows of %d heads are over 2^31 heads", N, NH);
    if (N == 0 || S == 0) return 0;
    const size_t esz = bf16 ? 2 : 4;
    PaArgs a = {};
    a.b.N = N;
    a.b.S = S;
    a.b.NKV = NKV;
    a.b.HD = HD;
    a.b.n_pages = bmk_pi(l, 6, 8);
    a.b.max_pages = bmk_pi(l, 6, 9);
    BMK_NEED_BATCH(l, a.b, bmk_pi(l, 6, 7), 3, 1, esz);
    BMK_NEED_ROWS(l, 0, N, (size_t)NH * HD, ldq, esz, "q");
    BMK_NEED_ROWS(l, 2, N, (size_t)NH * HD, ldo, esz, "out");
    a.q = l->dev[0];
    a.cache = l->dev[1];
    a.out = l->dev[2];
    a.NH = NH;
    a.R = NH / NKV;
    a.causal = causal;
    a.window = window;
    a.ldq = ldq;
    a.ldo = ldo;
    a.scale = bmk_pf(l, 7, 0);
    const dim3 grid((unsigned)N * (unsigned)NH);
    if (bf16) hipLaunchKernelGGL(k_attn_paged<true>, grid, dim3(64), 0, l->stream, a);
    else hipLaunchKernelGGL(k_attn_paged<false>, grid, dim3(64), 0, l->stream, a);
    BMK_LAUNCH_CHECK();
    return 0;
}

} // namespace

/* the tables' lookups on the host: row n's sequence, its position, and the page of key j of it (-1: none) */
extern "C" void bmk_paged_lookup(const int* start, const int* len, const int* pages, int S, int page, int n_pages,
                                 int max_pages, int n, int j, int* out) {
    PgBatch b = {};
    b.start = start;
    b.len = len;
    b.pages = pages;
    b.S = S;
    b.shift = pg_log2(page);
    b.n_pages = n_pages;
    b.max_pages = max_pages;
    out[0] = b.seq_of(n);
    out[1] = out[0] < 0 ? 0 : b.pos_of(out[0], n);
    out[2] = out[0] < 0 ? -1 : b.page_of(out[0], j);
}

extern "C" int bmk_launch_attn_paged(const bmk_launch_t* a) { return launch_attn_paged(a, false); }
extern "C" int bmk_launch_attn_paged_bf16(const bmk_launch_t* a) { return launch_attn_paged(a, true); }
