/* SPDX-License-Identifier: MPL-2.0
 *
 * rope_rows.hip — rotary positions of rows of heads, norms of q and k with
 * the rotation, and appending to a paged cache (include/bm_paged.h):
 *   rope_forward_rows     out = turn(x, pos)
 *   qk_norm_rope_forward  out = turn(x / sqrt(mean x^2 + eps) * gain, pos)
 *   kv_append_paged       q out = turn([norm] q), cache = turn([norm] k), v
 * One kernel: a group of lanes takes one head of one row (an item), a lane
 * two chunks of E elements, which hold whole rotation pairs, so nothing but
 * the norm's sum passes between lanes, and a lane stores what it loaded (an
 * output may be its input's buffer).
 *
 * HBM bounds the large calls (us, MI355X): 4096 rows of 40 heads of 128 in
 * bf16 15.1 (5.6 TB/s; chunks of 4 bytes in place of 16 32), norms of them in
 * fp32 33 (5.1; with the norm's root and gains by every lane from memory 59).
 * 16 chunks of 32 + 16 heads to their pages take 24.6 (3.8 TB/s; cos and sin by
 * every head 43): 17.4 the turning, 2 to 3 the norms, 2 each the lookups of
 * sequences and of pages.  Small ones take 2 to 4, a launch and two loads on end.
 */
#include "paged.h"

#include <algorithm>

namespace {

using namespace bmk;

constexpr int NT = 512;       /* (norms of 4096 rows of 40 heads of 128 in fp32: 128 46 us, 256 40, 512 39, 1024 43) */
constexpr int MAX_ROWS = 520; /* that a workgroup touches */

struct RopeArgs {
    const void *q, *k, *v;
    void *qo, *ko; /* ko: NULL where k and v go to the cache */
    void* cache;
    const int* pos; /* NULL: positions by the batch's tables */
    const unsigned long long* turns;
    const float* gain; /* NULL: no norm */
    PgBatch b;
    int NH, NK, heads; /* q's, k's and all heads of a row; b.NKV of v where there is a cache */
    int rot, pairs;
    int units, lp_log; /* lanes with work in a group, log2 of its lanes */
    size_t ldq, ldk, ldv, ldqo, ldko;
    int items; /* heads of all rows */
    int turns_held;
    int once; /* inputs that leave no room in the cache for what follows */
    Div by_heads, by_half;
    double by_hd; /* 1 / HD */
    float mscale, eps;
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

/* E elements as they lie in memory, on a boundary of their own size */
template <bool BF16, int E> struct alignas(E * (BF16 ? 2 : 4)) Chunk {
    unsigned char raw[E * (BF16 ? 2 : 4)];
};

template <bool BF16, int E>
__device__ __forceinline__ float value(const Chunk<BF16, E>& c, int e) {
    if constexpr (BF16) {
        unsigned short u[E];
        __builtin_memcpy(u, &c, sizeof c);
        return __uint_as_float((unsigned int)u[e] << 16);
    } else {
        float x[E];
        __builtin_memcpy(x, &c, sizeof c);
        return x[e];
    }
}

template <bool BF16, int E>
__device__ __forceinline__ void store(void* p, size_t i, const float* x) {
    Chunk<BF16, E> c;
    if constexpr (BF16) { /* to nearest even */
        unsigned short u[E + 1];
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const f32x2 f = {x[e], e + 1 < E ? x[e + 1] : 0.0f};
            const bf16x2 r = __builtin_convertvector(f, bf16x2);
            __builtin_memcpy(&u[e], &r, 4);
        }
        __builtin_memcpy(&c, u, sizeof c);
    } else {
        __builtin_memcpy(&c, x, sizeof c);
    }
    *(Chunk<BF16, E>*)((char*)p + i * (BF16 ? 2 : 4)) = c;
}

/* cos and sin of t / 2^32 of a turn: the nearest quarter taken off, the
 * Taylor series of what is left (at most pi / 4 to either side, fp32: up to
 * 2^-26.3 of a turn off), whose next terms are under 2e-9; 1.7 x 2^-24 off in all. */
__device__ __forceinline__ void cos_sin(unsigned int t, float* c, float* s) {
    const unsigned int quarter = (t + 0x20000000u) >> 30;
    const float x = (float)(int)(t - (quarter << 30)) * 1.46291807926715968e-9f; /* 2 pi / 2^32 */
    const float z = x * x;
    float sn = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 0.0f);
    sn = fmaf(x, sn, x);
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const float a = quarter & 1 ? sn : cs, b = quarter & 1 ? cs : sn;
    *c = quarter == 1 || quarter == 2 ? -a : a;
    *s = quarter >= 2 ? -b : b;
}

/* Sum over 2^k neighbouring lanes, which all get it: up to 16 by moves inside a row of lanes. */
template <int CTRL>
__device__ __forceinline__ double lanes_add(double v) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    const unsigned int lo = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)(unsigned int)u, CTRL, 0xF, 0xF, false);
    const unsigned int hi = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)(unsigned int)(u >> 32), CTRL, 0xF, 0xF, false);
    return v + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double group_sum(double v, int lanes) {
    if (lanes > 1) v = lanes_add<0xB1>(v);  /* lane ^ 1 */
    if (lanes > 2) v = lanes_add<0x4E>(v);  /* lane ^ 2 */
    if (lanes > 4) v = lanes_add<0x141>(v); /* the other four of eight */
    if (lanes > 8) v = lanes_add<0x140>(v); /* the other eight of sixteen */
    if (lanes > 16) v += __shfl_xor(v, 16);
    if (lanes > 32) v += __shfl_xor(v, 32);
    return v;
}
/* 1 / sqrt(m), of the instruction's 23 bits by one Newton step; 0 of infinity */
__device__ __forceinline__ double root_inverse(double m) {
    const double r = __builtin_amdgcn_rsq(m);
    return m == INFINITY ? 0.0 : fma(r * 0.5, fma(-m * r, r, 1.0), r);
}

/* Heads of all rows in order, one to each group of 1 << lp_log lanes: positions, places, cos and sin of the few rows that a
 * workgroup touches go to LDS, while its heads are loaded.  UN: units a lane takes at most. */
template <bool BF16, int E, int UN, bool PAIRS, bool ONCE>
__global__ __launch_bounds__(NT) void k_rope_rows(RopeArgs a) {
    extern __shared__ __attribute__((aligned(16))) float turns[]; /* a.turns_held of cos, then of sin */
    float *tc = turns, *ts = turns + a.turns_held;
    __shared__ __attribute__((aligned(16))) float gains[2 * PG_MAX_HD];
    __shared__ size_t places[MAX_ROWS];
    __shared__ int where[MAX_ROWS]; /* bit 0: a row of the batch, bit 1: with a place in the cache */
    const int t = threadIdx.x, lanes = 1 << a.lp_log, lane = t & (lanes - 1), slots = NT >> a.lp_log;
    const int HD = a.b.HD, half = a.rot / 2;
    const int first = (int)pg_group() * slots, x = first + (t >> a.lp_log), items = a.items;
    if (first >= items) return;
    const int n0 = a.by_heads.of(first), rows = a.by_heads.of(min(first + slots, items) - 1) - n0 + 1;
    const int halves = PAIRS ? 0 : a.rot / (2 * E); /* units whose chunks lie half of the turned part apart */
    auto at = [&](int i, int j) { /* of the lane's unit i, chunk j: its place in a head */
        const int u = lane + (i << a.lp_log);
        return u < halves ? E * u + (j ? half : 0) : 2 * E * u + (j ? E : 0);
    };

    const int n = a.by_heads.of(min(x, items - 1));
    int h = x - n * a.heads;
    const int kind = h < a.NH ? 0 : h < a.NH + a.NK ? 1 : 2; /* q, k, v */
    h -= kind == 0 ? 0 : kind == 1 ? a.NH : a.NH + a.NK;
    Chunk<BF16, E> raw[UN][2];
    if (x < items) {
        const void* src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
        const size_t from = (size_t)n * (kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv) + (size_t)h * HD;
#pragma unroll
        for (int i = 0; i < UN; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
                if (lane + (i << a.lp_log) < a.units) {
                    if constexpr (ONCE) { /* past the caches */
                        const u32x4 u = __builtin_nontemporal_load((const u32x4*)((const char*)src + (from + at(i, j)) * (BF16 ? 2 : 4)));
                        __builtin_memcpy(&raw[i][j], &u, sizeof u);
                    } else {
                        raw[i][j] = *(const Chunk<BF16, E>*)((const char*)src + (from + at(i, j)) * (BF16 ? 2 : 4));
                    }
                }
    }

    if (a.gain)
        for (int i = t; i < 2 * HD; i += NT) gains[i] = a.gain[i];
    for (int i = t; i < rows * max(half, 1); i += NT) {
        const int row = half ? a.by_half.of(i) : i, pair = i - row * half;
        int p, in = 1;
        if (a.pos) {
            p = a.pos[n0 + row];
        } else {
            const int s = a.b.seq_of(n0 + row);
            in = s >= 0;
            p = in ? a.b.pos_of(s, n0 + row) : 0;
            if (half == 0 || pair == 0) { /* once */
                const int pg = in ? a.b.page_of(s, p) : -1;
                places[row] = pg >= 0 ? a.b.base(pg, 0, 0) + (size_t)(p & ((1 << a.b.shift) - 1)) * HD : 0;
                in |= pg >= 0 ? 2 : 0;
            }
        }
        if (half == 0 || pair == 0) where[row] = in;
        if (half) {
            const unsigned long long turn = (unsigned long long)(long long)p * a.turns[pair];
            float c, s;
            cos_sin((unsigned int)(turn >> 32), &c, &s);
            tc[i] = c * a.mscale;
            ts[i] = s * a.mscale;
        }
    }
    __syncthreads();

    const int row = n - n0, flags = where[row];
    const bool cached = kind == 2 || (kind == 1 && !a.ko);
    if (x >= items || !(flags & 1) || (cached && !(flags & 2))) return;
    float y[UN][2][E];
#pragma unroll
    for (int i = 0; i < UN; i++)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < E; e++) y[i][j][e] = lane + (i << a.lp_log) < a.units ? value<BF16, E>(raw[i][j], e) : 0.0f;
    if (a.gain && kind < 2) { /* squares and their sum in 64 bits: those of heads past 2^64 or under 2^-64 need no care */
        double sum = 0;
#pragma unroll
        for (int i = 0; i < UN; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < E; e++) sum = fma((double)y[i][j][e], (double)y[i][j][e], sum);
        const double inv = root_inverse(group_sum(sum, lanes) * a.by_hd + (double)a.eps);
        const float f = (float)inv;
        /* a factor under 2^-126 has not all of fp32's bits, one over 2^128 (heads under 2^-128 with an eps as small) is none */
        const bool far = f < 0x1p-100f || f > 0x1p100f;
        if (__builtin_expect(__any(far), 0)) {
#pragma unroll
            for (int i = 0; i < UN; i++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        asm volatile(""); /* a branch, not a choice between two values */
                        y[i][j][e] = far ? (float)((double)y[i][j][e] * inv) : y[i][j][e] * f;
                    }
        } else {
#pragma unroll
            for (int i = 0; i < UN; i++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int e = 0; e < E; e++) y[i][j][e] *= f;
        }
#pragma unroll
        for (int i = 0; i < UN; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float g[E];
                __builtin_memcpy(g, __builtin_assume_aligned(gains + (kind == 1 ? HD : 0) + min(at(i, j), HD - E), E * 4 < 8 ? 4 : 8), sizeof g);
#pragma unroll
                for (int e = 0; e < E; e++) y[i][j][e] *= g[e];
            }
    }
    void* dst = kind == 0 ? a.qo : cached ? a.cache : a.ko;
    const size_t to = kind == 0 ? (size_t)n * a.ldqo + (size_t)h * HD
                      : !cached ? (size_t)n * a.ldko + (size_t)h * HD
                                : places[row] + ((size_t)(h + (kind == 2 ? a.b.NKV : 0)) * HD << a.b.shift);
#pragma unroll
    for (int i = 0; i < UN; i++) {
        const int u = lane + (i << a.lp_log);
        if (u >= a.units) continue;
        const bool turned = kind < 2 && 2 * E * u < a.rot;
        if (BF16 && !turned && (kind == 2 || !a.gain)) { /* every bit of it: a conversion would make other NaNs */
#pragma unroll
            for (int j = 0; j < 2; j++) *(Chunk<BF16, E>*)((char*)dst + (to + at(i, j)) * 2) = raw[i][j];
            continue;
        }
        if (turned) {
            float cs[E], sn[E];
            __builtin_memcpy(cs, __builtin_assume_aligned(tc + row * half + E * u, E * 4 < 16 ? E * 4 : 16), sizeof cs);
            __builtin_memcpy(sn, __builtin_assume_aligned(ts + row * half + E * u, E * 4 < 16 ? E * 4 : 16), sizeof sn);
#pragma unroll
            for (int e = 0; e < E; e++) { /* pair E u + e: element e of both chunks, or neighbours along them */
                float &x0 = PAIRS ? y[i][2 * e / E][2 * e % E] : y[i][0][e];
                float &x1 = PAIRS ? y[i][(2 * e + 1) / E][(2 * e + 1) % E] : y[i][1][e];
                /* spelt out, so that every form gives the same bits */
                const float y0 = fmaf(x0, cs[e], -(x1 * sn[e])), y1 = fmaf(x0, sn[e], x1 * cs[e]);
                x0 = y0;
                x1 = y1;
            }
        }
#pragma unroll
        for (int j = 0; j < 2; j++) store<BF16, E>(dst, to + at(i, j), y[i][j]);
    }
}

template <bool BF16, int E, int UN>
int launch(RopeArgs& a, hipStream_t stream) {
    a.units = a.b.HD / (2 * E);
    a.lp_log = 0;
    while ((UN << a.lp_log) < a.units) a.lp_log++;
    a.by_heads = div_by(a.heads);
    a.by_half = div_by(std::max(a.rot / 2, 1));
    a.by_hd = 1.0 / a.b.HD;
    /* a workgroup's heads lie in whole rows and a part of one at either end; LDS for no more than those, so that it does not
     * keep workgroups off a CU */
    const int slots = NT >> a.lp_log, rows = (slots - 1) / a.heads + 2;
    static_assert(NT + 1 <= MAX_ROWS, "");
    a.turns_held = (rows * (a.rot / 2) + 3) & ~3;
    const size_t bytes = (size_t)a.turns_held * 8;
    const dim3 grid = pg_grid(((int64_t)a.items + slots - 1) / slots, NT);
    constexpr bool WIDE = E * (BF16 ? 2 : 4) == 16;
    if (WIDE && a.once) {
        if (a.pairs) hipLaunchKernelGGL((k_rope_rows<BF16, E, UN, true, WIDE>), grid, dim3(NT), bytes, stream, a);
        else hipLaunchKernelGGL((k_rope_rows<BF16, E, UN, false, WIDE>), grid, dim3(NT), bytes, stream, a);
    } else if (a.pairs) {
        hipLaunchKernelGGL((k_rope_rows<BF16, E, UN, true, false>), grid, dim3(NT), bytes, stream, a);
    } else {
        hipLaunchKernelGGL((k_rope_rows<BF16, E, UN, false, false>), grid, dim3(NT), bytes, stream, a);
    }
    BMK_LAUNCH_CHECK();
    return 0;
}

/* Heads' layout: shapes of q (and k, v), the rotation's table. */
int run(const bmk_launch_t* l, RopeArgs& a, bool bf16, int layout, int turns_at, const char* what) {
    const int HD = a.b.HD;
    BMK_REQUIRE(layout == 0 || layout == 1, "%s: bad layout %d", what, layout);
    BMK_REQUIRE(a.rot >= 0 && a.rot <= HD && a.rot % 2 == 0, "%s: bad rot %d of head size %d", what, a.rot, HD);
    if (a.rot > 0) {
        BMK_REQUIRE(l->bytes[turns_at] >= (size_t)a.rot * 4, "%s: turns hold %zu bytes, rot %d needs %zu", what,
                    l->bytes[turns_at], a.rot, (size_t)a.rot * 4);
        BMK_REQUIRE(((uintptr_t)l->dev[turns_at] & 7) == 0, "%s: turns lie off an 8-byte boundary", what);
    }
    BMK_REQUIRE((int64_t)a.b.N * a.heads <= PG_MAX_DIM, "%s: %d rows of %d heads are over 2^30 heads", what, a.b.N, a.heads);
    a.turns = (const unsigned long long*)l->dev[turns_at];
    a.pairs = layout;
    a.items = a.b.N * a.heads;
    /* Inputs of more than half the Infinity Cache (256 MB) are read past it, so that it keeps the outputs for who reads them:
     * norms whose outputs are the next call's inputs, 168 MB each: of bf16 75 -> 54 us, fp32 61 -> 50; 84 MB 29 -> 27 and 24 -> 25, 42 MB
     * and less the same or worse, 336 MB 120 -> 124. */
    a.once = (size_t)a.items * HD * (bf16 ? 2 : 4) > (size_t)128 << 20;
    /* Chunks of up to 16 bytes: as many elements as divide every stride and address, the turned part's halves and the rest
     * of a head. */
    const size_t esz = bf16 ? 2 : 4;
    size_t all = a.ldq | a.ldk | a.ldv | a.ldqo | a.ldko | (size_t)a.rot / 2 | (size_t)HD / 2 | 16 / esz;
    for (const void* p : {a.q, a.k, a.v, (const void*)a.qo, (const void*)a.ko}) all |= (uintptr_t)p / esz;
    switch ((all & -all) * (bf16 ? 1 : 2)) { /* of bf16's 8 */
    case 8: return bf16 ? launch<true, 8, 1>(a, l->stream) : launch<false, 4, 1>(a, l->stream);
    case 4: return bf16 ? launch<true, 4, 1>(a, l->stream) : launch<false, 2, 1>(a, l->stream);
    case 2: return bf16 ? launch<true, 2, 1>(a, l->stream) : launch<false, 1, 2>(a, l->stream);
    default: return launch<true, 1, 2>(a, l->stream);
    }
}

/* {x T [N][ldx], out T [N][ldo], pos int32 [N], turns, params int{N, NH, HD, rot, layout, ldx, ldo}, f32{mscale}} */
int launch_rope_rows(const bmk_launch_t* l, bool bf16) {
    BMK_NEED_BYTES(l, 4, 28, "params");
    BMK_NEED_BYTES(l, 5, 4, "mscale");
    const int N = bmk_pi(l, 4, 0), NH = bmk_pi(l, 4, 1), HD = bmk_pi(l, 4, 2), ldx = bmk_pi(l, 4, 5), ldo = bmk_pi(l, 4, 6);
    BMK_REQUIRE(N >= 0 && N <= PG_MAX_DIM && NH > 0 && NH <= PG_MAX_DIM && HD > 0 && HD <= PG_MAX_HD && HD % 2 == 0,
                "rope_forward_rows: bad shape N=%d NH=%d HD=%d", N, NH, HD);
    if (N == 0) return 0;
    const size_t esz = bf16 ? 2 : 4;
    BMK_NEED_ROWS(l, 0, N, (size_t)NH * HD, ldx, esz, "x");
    BMK_NEED_ROWS(l, 1, N, (size_t)NH * HD, ldo, esz, "out");
    BMK_NEED_BYTES(l, 2, (size_t)N * 4, "pos");
    BMK_NEED_ALIGNED(l, 2, 4, "pos");
    RopeArgs a = {};
    a.q = l->dev[0];
    a.qo = l->dev[1];
    a.pos = (const int*)l->dev[2];
    a.b.N = N;
    a.b.HD = HD;
    a.NH = a.heads = NH;
    a.rot = bmk_pi(l, 4, 3);
    a.ldq = ldx;
    a.ldqo = ldo;
    a.mscale = bmk_pf(l, 5, 0);
    return run(l, a, bf16, bmk_pi(l, 4, 4), 3, "rope_forward_rows");
}

/* {q, k, q out, k out, pos int32 [N], turns, gain f32 [2][HD],
 *  params int{N, NH, NKV, HD, rot, layout, ldq, ldk, ldqo, ldko}, f32{mscale, eps}} */
int launch_qk_norm_rope(const bmk_launch_t* l, bool bf16) {
    BMK_NEED_BYTES(l, 7, 40, "params");
    BMK_NEED_BYTES(l, 8, 8, "mscale, eps");
    const int N = bmk_pi(l, 7, 0), NH = bmk_pi(l, 7, 1), NKV = bmk_pi(l, 7, 2), HD = bmk_pi(l, 7, 3);
    const int ldq = bmk_pi(l, 7, 6), ldk = bmk_pi(l, 7, 7), ldqo = bmk_pi(l, 7, 8), ldko = bmk_pi(l, 7, 9);
    BMK_REQUIRE(N >= 0 && N <= PG_MAX_DIM && NH > 0 && NH <= PG_MAX_DIM / 2 && NKV > 0 && NKV <= PG_MAX_DIM / 2 && HD > 0 &&
                    HD <= PG_MAX_HD && HD % 2 == 0,
                "qk_norm_rope_forward: bad shape N=%d NH=%d NKV=%d HD=%d", N, NH, NKV, HD);
    BMK_REQUIRE(bmk_pf(l, 8, 1) >= 0, "qk_norm_rope_forward: bad eps %g", (double)bmk_pf(l, 8, 1));
    if (N == 0) return 0;
    const size_t esz = bf16 ? 2 : 4;
    BMK_NEED_ROWS(l, 0, N, (size_t)NH * HD, ldq, esz, "q");
    BMK_NEED_ROWS(l, 1, N, (size_t)NKV * HD, ldk, esz, "k");
    BMK_NEED_ROWS(l, 2, N, (size_t)NH * HD, ldqo, esz, "q out");
    BMK_NEED_ROWS(l, 3, N, (size_t)NKV * HD, ldko, esz, "k out");
    BMK_NEED_BYTES(l, 4, (size_t)N * 4, "pos");
    BMK_NEED_ALIGNED(l, 4, 4, "pos");
    BMK_NEED_BYTES(l, 6, (size_t)HD * 8, "gain");
    BMK_NEED_ALIGNED(l, 6, 4, "gain");
    RopeArgs a = {};
    a.q = l->dev[0];
    a.k = l->dev[1];
    a.qo = l->dev[2];
    a.ko = l->dev[3];
    a.pos = (const int*)l->dev[4];
    a.gain = (const float*)l->dev[6];
    a.b.N = N;
    a.b.HD = HD;
    a.NH = NH;
    a.NK = NKV;
    a.heads = NH + NKV;
    a.rot = bmk_pi(l, 7, 4);
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldqo = ldqo;
    a.ldko = ldko;
    a.mscale = bmk_pf(l, 8, 0);
    a.eps = bmk_pf(l, 8, 1);
    return run(l, a, bf16, bmk_pi(l, 7, 5), 5, "qk_norm_rope_forward");
}

/* {q, k, v, q out, cache, start, len, pages, turns, gain f32 [2][HD],
 *  params int{N, S, NH, NKV, HD, rot, layout, ldq, ldk, ldv, ldqo, page, n_pages, max_pages, norm}, f32{mscale, eps}} */
int launch_kv_append(const bmk_launch_t* l, bool bf16) {
    BMK_NEED_BYTES(l, 10, 60, "params");
    BMK_NEED_BYTES(l, 11, 8, "mscale, eps");
    const int N = bmk_pi(l, 10, 0), S = bmk_pi(l, 10, 1), NH = bmk_pi(l, 10, 2), NKV = bmk_pi(l, 10, 3), HD = bmk_pi(l, 10, 4);
    const int ldq = bmk_pi(l, 10, 7), ldk = bmk_pi(l, 10, 8), ldv = bmk_pi(l, 10, 9), ldqo = bmk_pi(l, 10, 10);
    const int norm = bmk_pi(l, 10, 14);
    BMK_REQUIRE(N >= 0 && N <= PG_MAX_DIM && S >= 0 && S <= PG_MAX_SEQS && NH >= 0 && NH <= PG_MAX_DIM / 2 && NKV > 0 &&
                    NKV <= PG_MAX_DIM / 4 && HD > 0 && HD <= PG_MAX_HD && (norm == 0 || norm == 1),
                "kv_append_paged: bad shape N=%d S=%d NH=%d NKV=%d HD=%d norm=%d", N, S, NH, NKV, HD, norm);
    BMK_REQUIRE(!norm || bmk_pf(l, 11, 1) >= 0, "kv_append_paged: bad eps %g", (double)bmk_pf(l, 11, 1));
    if (N == 0 || S == 0) return 0;
    const size_t esz = bf16 ? 2 : 4;
    RopeArgs a = {};
    a.b.N = N;
    a.b.S = S;
    a.b.NKV = NKV;
    a.b.HD = HD;
    a.b.n_pages = bmk_pi(l, 10, 12);
    a.b.max_pages = bmk_pi(l, 10, 13);
    BMK_NEED_BATCH(l, a.b, bmk_pi(l, 10, 11), 5, 4, esz);
    if (NH > 0) {
        BMK_NEED_ROWS(l, 0, N, (size_t)NH * HD, ldq, esz, "q");
        BMK_NEED_ROWS(l, 3, N, (size_t)NH * HD, ldqo, esz, "q out");
        a.q = l->dev[0];
        a.qo = l->dev[3];
        a.ldq = ldq;
        a.ldqo = ldqo;
    }
    BMK_NEED_ROWS(l, 1, N, (size_t)NKV * HD, ldk, esz, "k");
    BMK_NEED_ROWS(l, 2, N, (size_t)NKV * HD, ldv, esz, "v");
    if (norm) {
        BMK_NEED_BYTES(l, 9, (size_t)HD * 8, "gain");
        BMK_NEED_ALIGNED(l, 9, 4, "gain");
        a.gain = (const float*)l->dev[9];
    }
    a.k = l->dev[1];
    a.v = l->dev[2];
    a.cache = l->dev[4];
    a.NH = NH;
    a.NK = NKV;
    a.heads = NH + 2 * NKV;
    a.rot = bmk_pi(l, 10, 5);
    a.ldk = ldk;
    a.ldv = ldv;
    a.mscale = bmk_pf(l, 11, 0);
    a.eps = bmk_pf(l, 11, 1);
    return run(l, a, bf16, bmk_pi(l, 10, 6), 8, "kv_append_paged");
}

} // namespace

extern "C" int bmk_launch_rope_rows(const bmk_launch_t* a) { return launch_rope_rows(a, false); }
extern "C" int bmk_launch_rope_rows_bf16(const bmk_launch_t* a) { return launch_rope_rows(a, true); }
extern "C" int bmk_launch_qk_norm_rope(const bmk_launch_t* a) { return launch_qk_norm_rope(a, false); }
extern "C" int bmk_launch_qk_norm_rope_bf16(const bmk_launch_t* a) { return launch_qk_norm_rope(a, true); }
extern "C" int bmk_launch_kv_append(const bmk_launch_t* a) { return launch_kv_append(a, false); }
extern "C" int bmk_launch_kv_append_bf16(const bmk_launch_t* a) { return launch_kv_append(a, true); }
