/* SPDX-License-Identifier: MPL-2.0
 *
 * rope_rows.hip — rotary positions of rows of heads, norms of q and k with
 * the rotation, and appending to a paged cache (include/bm_paged.h):
 *   rope_forward_rows     out = turn(x, pos)
 *   qk_norm_rope_forward  out = turn(x / sqrt(mean x^2 + eps) * gain, pos)
 *   kv_append_paged       q out = turn([norm] q), cache = turn([norm] k), v
 * One kernel: a group of LP lanes takes one head of one row (an item), a lane
 * two chunks of E elements, which hold whole rotation pairs, so nothing but
 * the norm's sum passes between lanes, and a lane stores what it loaded (an
 * output may be its input's buffer).
 */
#include "paged.h"

namespace {

using namespace bmk;

constexpr int NT = 256;

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
    unsigned int items;
    float mscale, eps;
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

/* E elements as they lie in memory, on a boundary of their own size */
template <bool BF16, int E> struct alignas(E * (BF16 ? 2 : 4)) Chunk {
    unsigned char raw[E * (BF16 ? 2 : 4)];
};

template <bool BF16, int E>
__device__ __forceinline__ void load(const void* p, size_t i, float* x) {
    const Chunk<BF16, E> c = *(const Chunk<BF16, E>*)((const char*)p + i * (BF16 ? 2 : 4));
    if constexpr (BF16) {
        unsigned short u[E];
        __builtin_memcpy(u, &c, sizeof c);
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = __uint_as_float((unsigned int)u[e] << 16);
    } else {
        __builtin_memcpy(x, &c, sizeof c);
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
 * Taylor series of what is left (at most pi / 4 to either side), whose next
 * terms are under 2e-9. */
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

/* UN: units a lane takes at most */
template <bool BF16, int E, int UN>
__global__ __launch_bounds__(NT) void k_rope_rows(RopeArgs a) {
    const unsigned int lane = threadIdx.x & ((1u << a.lp_log) - 1);
    const unsigned int item = (blockIdx.x * (unsigned int)NT + threadIdx.x) >> a.lp_log;
    if (item >= a.items) return; /* whole groups */
    const int n = (int)(item / (unsigned int)a.heads);
    int h = (int)(item - (unsigned int)n * (unsigned int)a.heads);
    int p;
    size_t place = 0; /* of the row in the cache, KV head 0's keys */
    bool kept = false;
    if (a.pos) {
        p = a.pos[n];
    } else {
        const int s = a.b.seq_of(n);
        if (s < 0) return;
        p = a.b.pos_of(s, n);
        const int pg = a.b.page_of(s, p);
        kept = pg >= 0;
        if (kept) place = a.b.base(pg, 0, 0) + (size_t)(p & ((1 << a.b.shift) - 1)) * a.b.HD;
    }
    const int HD = a.b.HD;
    const size_t plane = (size_t)HD << a.b.shift; /* of one KV head's part of a page */
    const void* src;
    void* dst;
    size_t from, to;
    bool turned = true;
    const float* gain = a.gain;
    if (h < a.NH) {
        src = a.q;
        dst = a.qo;
        from = (size_t)n * a.ldq + (size_t)h * HD;
        to = (size_t)n * a.ldqo + (size_t)h * HD;
    } else if (h < a.NH + a.NK) {
        h -= a.NH;
        if (gain) gain += HD;
        src = a.k;
        from = (size_t)n * a.ldk + (size_t)h * HD;
        dst = a.ko ? a.ko : a.cache;
        to = a.ko ? (size_t)n * a.ldko + (size_t)h * HD : place + h * plane;
        if (!a.ko && !kept) return;
    } else {
        h -= a.NH + a.NK;
        gain = nullptr;
        turned = false;
        src = a.v;
        from = (size_t)n * a.ldv + (size_t)h * HD;
        dst = a.cache;
        to = place + (a.b.NKV + h) * plane;
        if (!kept) return;
    }
    /* unit u's chunks: in the turned part by halves E u and rot/2 + E u, else 2 E u and the next */
    const int halves = a.pairs ? 0 : a.rot / (2 * E); /* units that lie so */
    float x[UN][2][E];
    int at[UN][2];
#pragma unroll
    for (int i = 0; i < UN; i++) {
        const int u = (int)lane + (i << a.lp_log);
        at[i][0] = u < halves ? E * u : 2 * E * u;
        at[i][1] = u < halves ? a.rot / 2 + E * u : 2 * E * u + E;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (u < a.units) load<BF16, E>(src, from + at[i][j], x[i][j]);
            else
#pragma unroll
                for (int e = 0; e < E; e++) x[i][j][e] = 0.0f;
        }
    }
    if (gain) { /* squares and their sum in 64 bits: heads past 2^64 or under 2^-64 need no care */
        double sum = 0;
#pragma unroll
        for (int i = 0; i < UN; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < E; e++) sum = fma((double)x[i][j][e], (double)x[i][j][e], sum);
        for (int o = 1; o < 1 << a.lp_log; o <<= 1) sum += __shfl_xor(sum, o);
        const double inv = 1.0 / sqrt(sum / HD + (double)a.eps);
#pragma unroll
        for (int i = 0; i < UN; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < E; e++)
                    if ((int)lane + (i << a.lp_log) < a.units)
                        x[i][j][e] = (float)((double)x[i][j][e] * inv) * gain[at[i][j] + e];
    }
#pragma unroll
    for (int i = 0; i < UN; i++) {
        const int u = (int)lane + (i << a.lp_log);
        if (u >= a.units) continue;
        if (turned && 2 * E * u < a.rot) {
#pragma unroll
            for (int e = 0; e < E; e++) { /* pair E u + e: element e of both chunks, or neighbours along them */
                const unsigned long long t = (unsigned long long)(long long)p * a.turns[E * u + e];
                float c, s;
                cos_sin((unsigned int)(t >> 32), &c, &s);
                c *= a.mscale;
                s *= a.mscale;
                float &x0 = a.pairs ? x[i][2 * e / E][2 * e % E] : x[i][0][e];
                float &x1 = a.pairs ? x[i][(2 * e + 1) / E][(2 * e + 1) % E] : x[i][1][e];
                const float y0 = x0 * c - x1 * s, y1 = x0 * s + x1 * c;
                x0 = y0;
                x1 = y1;
            }
        }
#pragma unroll
        for (int j = 0; j < 2; j++) store<BF16, E>(dst, to + at[i][j], x[i][j]);
    }
}

template <bool BF16, int E, int UN>
int launch(RopeArgs& a, hipStream_t stream) {
    a.units = a.b.HD / (2 * E);
    a.lp_log = 0;
    while ((UN << a.lp_log) < a.units) a.lp_log++;
    const unsigned int per = NT >> a.lp_log;
    hipLaunchKernelGGL((k_rope_rows<BF16, E, UN>), dim3((a.items + per - 1) / per), dim3(NT), 0, stream, a);
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
    BMK_REQUIRE((int64_t)a.b.N * a.heads < (1LL << 31), "%s: %d rows of %d heads are over 2^31 heads", what, a.b.N, a.heads);
    a.turns = (const unsigned long long*)l->dev[turns_at];
    a.pairs = layout;
    a.items = (unsigned int)a.b.N * (unsigned int)a.heads;
    return bf16 ? launch<true, 1, 2>(a, l->stream) : launch<false, 1, 2>(a, l->stream);
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
