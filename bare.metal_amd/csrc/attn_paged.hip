/* SPDX-License-Identifier: MPL-2.0
 *
 * attn_paged.hip — attention_forward_paged (include/bm_paged.h): the new
 * tokens of several sequences over the keys in their pages,
 *   out = softmax(scale * q . K + mask) V,
 * in one pass over the keys with the running maximum and sum (fp32) of the
 * softmax.
 *
 * A unit of work is 128 rows (new token, query head of the group) of one
 * sequence and KV head, so that every key and value is read once for a whole
 * group of heads; a unit's keys may be split over workgroups, whose partial
 * results the last one of them joins.  A workgroup goes over its keys in tiles of
 * KT, which lie in LDS in pieces of bf16: bf16 as it is, fp32 as three terms
 * x = x0 + x1 + x2 (truncations, exact), whose products of at least 2^-24 are
 * taken, six of nine.  Each of its four waves has 32 rows; of fewer rows than that, each
 * wave takes a part of the tile's keys instead.  Per 32 keys a wave forms
 *   S^T (32 keys x 32 rows) = K Q^T,   O^T (HD x 32 rows) += V^T P^T
 * with v_mfma_f32_32x32x16_bf16.  A lane holds the scores of one row (lane %
 * 32) and 16 keys, exactly those whose weights the second product wants of
 * it once its sum runs over the keys in the order of the registers, so P goes
 * from the scores to the product without moving between lanes; V comes
 * transposed out of LDS (ds_read_b64_tr_b16).
 */
#include "paged.h"
#include "q8_common.h"

#include <math.h>

#include <algorithm>

namespace {

using namespace bmk;

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(1))) void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

constexpr int NT = 256, NW = 4;
constexpr int ROWS = 32 * NW;    /* of a unit */
constexpr float SLACK = 8.0f;    /* in powers of two: how far a score may pass the running maximum before that moves */
constexpr int MAX_SPLIT = 64;    /* parts of a unit's keys */
constexpr int WANTED = 1024;     /* workgroups that the splits aim at */

/* The scratch memory begins with arrival counters, each on a line of its own, that are zero between launches of any
 * kernel; the units' partial results lie behind them. */
constexpr int DONE_STRIDE = 32, MAX_UNITS = 1024;
constexpr size_t DONE_BYTES = (size_t)DONE_STRIDE * MAX_UNITS * 4;

struct PaArgs {
    const void* q;
    const void* cache;
    void* out;
    unsigned int* done;
    float* rec;
    PgBatch b;
    int NH, R; /* R: query heads a KV head */
    int causal, window;
    size_t ldq, ldo;
    float scale2; /* |scale| * log2(e) */
    unsigned int flip; /* scale's sign, for q's */
    unsigned int most; /* rows' records that fit behind the counters */
};

/* How a tile lies: HDP is the head size rounded up, with zeros behind it. */
template <bool BF16, int HDP> struct Tile {
    static constexpr int TERMS = BF16 ? 1 : 3;
    static constexpr int KT = BF16 ? (HDP == 256 ? 32 : 64) : (HDP == 64 ? 64 : 32);
    static constexpr int KB = KT / 32;
    static constexpr int ROWB = HDP * 2, CPR = HDP / 8; /* bytes and 16-byte chunks of a row's term */
    static constexpr int PLANE = KT * ROWB;
    static constexpr int BYTES = 2 * TERMS * PLANE; /* keys' terms, then values' */
    static constexpr int WAVES = HDP <= (BF16 ? 128 : 64) ? 2 : 1; /* a SIMD */
};

/* Chunk c of row r lies at c ^ key: K is read 8 rows of one chunk at a time, V 4 rows of two neighbouring ones, each
 * set on all banks. */
__device__ __forceinline__ int k_place(int r, int c) { return c ^ (r & 7); }
__device__ __forceinline__ int v_place(int r, int c) { return c ^ (2 * (r & 3)); }

__device__ const u32x4 pg_zeros = {0, 0, 0, 0}, pg_nans = {0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};

__device__ __forceinline__ void agent_store2(float* p, float x, float y) {
    const unsigned long long u = ((unsigned long long)__float_as_uint(y) << 32) | __float_as_uint(x);
    __hip_atomic_store((unsigned long long*)p, u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 agent_load2(const float* p) {
    const unsigned long long u = __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return f32x2{__uint_as_float((unsigned int)u), __uint_as_float((unsigned int)(u >> 32))};
}

/* two values' bf16, rounded to nearest even */
__device__ __forceinline__ unsigned int pack_rne(float x, float y) {
    return __builtin_bit_cast(unsigned int, __builtin_convertvector(f32x2{x, y}, bf16x2));
}
/* the upper halves of two values */
__device__ __forceinline__ unsigned int pack_top(float x, float y) {
    return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
}
__device__ __forceinline__ float top(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

/* x's three terms of two values each, packed; of an infinity or NaN the first alone */
__device__ __forceinline__ void split2(float x, float y, unsigned int* t) {
    t[0] = pack_top(x, y);
    const float rx = __builtin_isfinite(x) ? x - top(x) : 0.0f, ry = __builtin_isfinite(y) ? y - top(y) : 0.0f;
    t[1] = pack_top(rx, ry);
    t[2] = pack_top(rx - top(rx), ry - top(ry));
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float other_half(float v) {
    const u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? s[0] : s[1]);
}

/* ---------------------------------------------------------------- the work */

struct Seq {
    int n, len, T; /* new tokens, keys, tiles of keys that a unit sees at most */
    unsigned int units; /* per KV head */
};

/* What is to be done, from the tables alone: every wave finds it for itself, 64 sequences at a time, the first of them
 * kept in registers. */
template <int KT>
struct Plan {
    const PaArgs& a;
    const int lane;
    Seq first;
    int per;            /* tiles a part */
    unsigned int total; /* pieces of work; 0 where the tables are none */

    __device__ __forceinline__ Seq seq(int s) const {
        Seq q = {0, 0, 0, 0};
        if (s < a.b.S) {
            const int at = a.b.start[s], end = a.b.start[s + 1];
            q.len = max(a.b.len[s], 0);
            if (at >= 0 && at < end && end <= a.b.N) q.n = end - at;
            q.units = ((unsigned int)q.n * (unsigned int)a.R + ROWS - 1) / ROWS;
            int span = min(q.len, a.b.room());
            if (a.window) span = min(span, a.window + ROWS / a.R + 1 + KT);
            q.T = (span + KT - 1) / KT;
        }
        return q;
    }
    __device__ __forceinline__ Seq chunk(int c) const { return c ? seq(c + lane) : first; }
    __device__ __forceinline__ unsigned int parts(const Seq& q) const { return max(1, (q.T + per - 1) / per); }

    __device__ __forceinline__ Plan(const PaArgs& args) : a(args), lane(threadIdx.x & 63) {
        first = seq(lane);
        float tiles = 0, rows = 0;
        int longest = 0;
        for (int c = 0; c < a.b.S; c += 64) {
            const Seq q = chunk(c);
            tiles += (float)q.units * (float)q.T;
            rows += (float)q.n;
            longest = max(longest, q.T);
        }
        tiles = wave_sum(tiles) * a.b.NKV;
        rows = wave_sum(rows);
        for (int o = 1; o < 64; o <<= 1) longest = max(longest, __shfl_xor(longest, o));
        per = max((int)(tiles / WANTED) + 1, (longest + MAX_SPLIT - 1) / MAX_SPLIT);
        if (!a.most) per = max(longest, 1);
        per = __builtin_amdgcn_readfirstlane(per);
        total = 0;
        if (rows > (float)a.b.N * 1.0001f) return; /* sequences that overlap: no batch */
        for (;;) { /* parts as long as their records and counters need; ends at one part a unit */
            float recs = 0, units = 0;
            unsigned int w = 0;
            for (int c = 0; c < a.b.S; c += 64) {
                const Seq q = chunk(c);
                const unsigned int p = parts(q);
                w += q.units * p * a.b.NKV;
                if (p > 1) {
                    recs += (float)q.n * a.R * p * a.b.NKV;
                    units += (float)q.units * a.b.NKV;
                }
            }
            recs = wave_sum(recs);
            units = wave_sum(units);
            if (per >= longest || (recs * 1.0001f < (float)a.most && units <= (float)MAX_UNITS)) {
                for (int o = 1; o < 64; o <<= 1) w += __shfl_xor(w, o);
                total = __builtin_amdgcn_readfirstlane(w);
                return;
            }
            per = per > longest / 2 ? longest : 2 * per;
            per = __builtin_amdgcn_readfirstlane(per);
        }
    }

    struct Item {
        int s, kh, unit, part, parts;
        int n, len;
        unsigned int rec, done; /* first of the unit's records, its counter */
    };
    /* piece w < total of the work: within a sequence the KV heads side by side, the last units, which see the most keys, first */
    __device__ __forceinline__ Item item(unsigned int w) const {
        Item it = {};
        unsigned int recs = 0, units = 0;
        for (int c = 0; c < a.b.S; c += 64) {
            const Seq q = chunk(c);
            const unsigned int p = parts(q), mine = q.units * p * a.b.NKV;
            const unsigned int r = p > 1 ? (unsigned int)q.n * a.R * p * a.b.NKV : 0, u = p > 1 ? q.units * a.b.NKV : 0;
            unsigned int iw = mine, ir = r, iu = u; /* sums up to this lane */
            for (int o = 1; o < 64; o <<= 1) {
                const unsigned int x = __shfl_up(iw, o), y = __shfl_up(ir, o), z = __shfl_up(iu, o);
                if (lane >= o) {
                    iw += x;
                    ir += y;
                    iu += z;
                }
            }
            const unsigned long long past = __ballot(iw > w);
            if (past) {
                const int l = __builtin_ctzll(past);
                it.s = c + l;
                it.n = __builtin_amdgcn_readlane(q.n, l);
                it.len = __builtin_amdgcn_readlane(q.len, l);
                it.parts = __builtin_amdgcn_readlane((int)p, l);
                const unsigned int local = w - (unsigned int)__builtin_amdgcn_readlane((int)(iw - mine), l);
                const unsigned int nu = (unsigned int)__builtin_amdgcn_readlane((int)q.units, l);
                it.kh = local % a.b.NKV;
                const unsigned int rest = local / a.b.NKV;
                it.part = rest % it.parts;
                it.unit = (int)(nu - 1 - rest / it.parts);
                it.rec = recs + (unsigned int)__builtin_amdgcn_readlane((int)(ir - r), l);
                it.done = units + (unsigned int)__builtin_amdgcn_readlane((int)(iu - u), l) + it.unit * a.b.NKV + it.kh;
                return it;
            }
            w -= __builtin_amdgcn_readlane((int)iw, 63);
            recs += (unsigned int)__builtin_amdgcn_readlane((int)ir, 63);
            units += (unsigned int)__builtin_amdgcn_readlane((int)iu, 63);
        }
        it.s = -1;
        return it;
    }
};

/* keys that a row at position p sees: first .. last */
struct Seen {
    int first, last;
};
__device__ __forceinline__ Seen seen(const PaArgs& a, int p, int len) {
    Seen r;
    r.last = a.causal ? p : len - 1;
    r.first = a.window ? max(0, p - a.window + 1) : 0;
    return r;
}

template <bool BF16>
__device__ __forceinline__ void store4(const PaArgs& a, size_t row, int d, const float* o) {
    const size_t i = row + d;
    if (BF16) {
        unsigned short* p = (unsigned short*)a.out + i;
        const u32x2 v = {pack_rne(o[0], o[1]), pack_rne(o[2], o[3])};
        if (((uintptr_t)p & 7) == 0) {
            *(u32x2*)p = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] = (unsigned short)(v[e >> 1] >> (16 * (e & 1)));
        }
    } else {
        float* p = (float*)a.out + i;
        if (((uintptr_t)p & 15) == 0) {
            *(f32x4*)p = f32x4{o[0], o[1], o[2], o[3]};
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] = o[e];
        }
    }
}

/* ---------------------------------------------------------------- the kernel */

template <bool BF16, int HDP>
__global__ __launch_bounds__(NT, (Tile<BF16, HDP>::WAVES)) void k_attn_paged(PaArgs a) {
    typedef Tile<BF16, HDP> T;
    constexpr int TERMS = T::TERMS, KT = T::KT, KB = T::KB, CPR = T::CPR, PLANE = T::PLANE;
    constexpr int STEPS = HDP / 16, DT = HDP / 32; /* of the first product's sum; tiles of the output's dimensions */
    constexpr int RPI = 1024 / T::ROWB, NI = PLANE / 1024 / NW; /* rows of a wave's load into LDS, loads of keys a wave */
    /* two arrays, not one: reads of the one then wait for no load into the other */
    __shared__ __attribute__((aligned(16))) unsigned char lds0[T::BYTES], lds1[BF16 ? T::BYTES : 16];
    __shared__ float row_m[ROWS], row_l[ROWS];
    __shared__ int last_one;
    const PgBatch& b = a.b;
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
    const int col = lane & 31, half = lane >> 5;
    const int HD = b.HD;
    const Plan<KT> plan(a);

    for (unsigned int w = blockIdx.x; w < plan.total; w += gridDim.x) {
        const auto it = plan.item(w);
        if (it.s < 0) return;
        const int rows_all = it.n * a.R, r0 = it.unit * ROWS, nrows = min(ROWS, rows_all - r0);
        const int p0 = (int)((unsigned)it.len - (unsigned)it.n); /* position of the sequence's first new token */
        const int n0 = b.start[it.s];
        const int tok0 = r0 / a.R, tok1 = (r0 + nrows - 1) / a.R;
        const int room = b.room();
        /* tiles of keys that some row of the unit sees, and this part's */
        const int lo = seen(a, p0 + tok0, it.len).first, hi = min(seen(a, p0 + tok1, it.len).last + 1, room);
        const int t0 = lo / KT, t1 = hi > lo ? (hi + KT - 1) / KT : t0;
        const int parts = max(1, (t1 - t0 + plan.per - 1) / plan.per);
        if (it.part >= parts) continue;
        const int kt0 = t0 + it.part * plan.per, kt1 = min(kt0 + plan.per, t1);
        /* waves side by side on rows, the rest on parts of the tile's keys */
        const int groups = nrows <= 32 ? 1 : nrows <= 64 ? 2 : 4, kparts = min(NW / groups, KB);
        const int group = wave & (groups - 1), kpart = wave / groups;
        const bool active = kpart < kparts && 32 * group < nrows;
        const int r = r0 + 32 * group + col, tok = r / a.R, head = it.kh * a.R + (r - tok * a.R);
        const bool mine = r < r0 + nrows;
        const Seen sn = mine ? seen(a, p0 + tok, it.len) : Seen{0, -1};
        /* of the wave's rows: keys from all_first to all_last are seen by all, outside any_first .. any_last by none */
        const int gtok0 = min(r0 + 32 * group, r0 + nrows - 1) / a.R, gtok1 = min(r0 + 32 * group + 31, r0 + nrows - 1) / a.R;
        const Seen sa = seen(a, p0 + gtok0, it.len), sz = seen(a, p0 + gtok1, it.len);
        const int any_first = sa.first, any_last = sz.last, all_first = sz.first, all_last = sa.last;

        bf16x8 qf[TERMS][STEPS]; /* step s: dimensions 16 s + 8 half .. + 7 of the lane's row */
        {
            const size_t at = (size_t)(n0 + min(tok, tok1)) * a.ldq + (size_t)(mine ? head : it.kh * a.R) * HD;
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                const int d = 16 * s + 8 * half;
                unsigned int u[TERMS][4];
                if (!mine || d >= HD) {
#pragma unroll
                    for (int x = 0; x < TERMS; x++)
#pragma unroll
                        for (int e = 0; e < 4; e++) u[x][e] = 0;
                } else if constexpr (BF16) {
                    const unsigned short* p = (const unsigned short*)a.q + at + d;
                    if (((uintptr_t)p & 15) == 0) {
                        __builtin_memcpy(u[0], __builtin_assume_aligned(p, 16), 16);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) u[0][e] = p[2 * e] | (unsigned int)p[2 * e + 1] << 16;
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) u[0][e] ^= a.flip >> 16 | a.flip;
                } else {
                    const float* p = (const float*)a.q + at + d;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        unsigned int y[3];
                        split2(__uint_as_float(__float_as_uint(p[2 * e]) ^ a.flip),
                               __uint_as_float(__float_as_uint(p[2 * e + 1]) ^ a.flip), y);
#pragma unroll
                        for (int x = 0; x < TERMS; x++) u[x][e] = y[x];
                    }
                }
#pragma unroll
                for (int x = 0; x < TERMS; x++) __builtin_memcpy(&qf[x][s], u[x], 16);
            }
        }

        f32x16 acc[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[d][e] = 0.0f;
        float m = -INFINITY, l = 0.0f; /* in powers of two, of the row; this lane's keys' sum */

        const size_t kv = (size_t)HD << b.shift; /* elements of one head's keys or values in a page */
        const int mask = (1 << b.shift) - 1;
        const int* table = b.pages + (size_t)it.s * b.max_pages;
        auto page_at = [&](int key) { /* page of a key before hi, or none */
            const int pg = table[key >> b.shift];
            return pg >= 0 && pg < b.n_pages ? pg : -1;
        };

        /* 32 keys at k0, block kb of the tile in LDS at `buf` */
        auto block = [&](const unsigned char* buf, int kb, int k0) {
            f32x16 sc;
#pragma unroll
            for (int e = 0; e < 16; e++) sc[e] = 0.0f;
            const int row = 32 * kb + col;
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                bf16x8 kf[TERMS];
#pragma unroll
                for (int x = 0; x < TERMS; x++)
                    kf[x] = *(const bf16x8*)(buf + x * PLANE + row * T::ROWB + 16 * k_place(row, 2 * s + half));
                if constexpr (!BF16) { /* the small terms first */
                    sc = mfma(kf[2], qf[0][s], sc);
                    sc = mfma(kf[0], qf[2][s], sc);
                    sc = mfma(kf[1], qf[1][s], sc);
                    sc = mfma(kf[1], qf[0][s], sc);
                    sc = mfma(kf[0], qf[1][s], sc);
                }
                sc = mfma(kf[0], qf[0][s], sc);
            }
            /* lane's score e: key k0 + 8 (e / 4) + 4 half + e % 4 */
            const bool masked = k0 < all_first || k0 + 31 > all_last;
            unsigned int sees = 0xffff; /* bit e */
            if (masked) {
                sees = 0;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int key = k0 + 8 * (e >> 2) + 4 * half + (e & 3);
                    const bool in = key >= sn.first && key <= sn.last;
                    sees |= (unsigned int)in << e;
                    sc[e] = in ? sc[e] : -INFINITY;
                }
            }
            float cm = sc[0];
#pragma unroll
            for (int e = 1; e < 16; e++) cm = fmaxf(cm, sc[e]);
            cm *= a.scale2; /* -infinity times 0 is NaN, which moves nothing */
            if (__any(cm > m + SLACK)) {
                cm = fmaxf(cm, other_half(cm));
                const float mn = fmaxf(m, cm), f = mn > -INFINITY ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
                l *= f;
#pragma unroll
                for (int d = 0; d < DT; d++) acc[d] *= f;
                m = mn;
            }
            const float ms = m > -INFINITY ? m : 0.0f;
            float p[16];
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], a.scale2, -ms));
            if (masked) {
#pragma unroll
                for (int e = 0; e < 16; e++) p[e] = sees >> e & 1 ? p[e] : 0.0f;
            }
            float s4[4];
#pragma unroll
            for (int e = 0; e < 4; e++) s4[e] = (p[e] + p[e + 4]) + (p[e + 8] + p[e + 12]);
            l += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            bf16x8 pf[TERMS][2];
#pragma unroll
            for (int s = 0; s < 2; s++) {
                unsigned int u[TERMS][4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = p[8 * s + 2 * e], y = p[8 * s + 2 * e + 1];
                    if constexpr (BF16) {
                        u[0][e] = pack_rne(x, y);
                    } else {
                        unsigned int z[3];
                        split2(x, y, z);
#pragma unroll
                        for (int i = 0; i < TERMS; i++) u[i][e] = z[i];
                    }
                }
#pragma unroll
                for (int x = 0; x < TERMS; x++) __builtin_memcpy(&pf[x][s], u[x], 16);
            }
            /* dimension 32 d + col, keys 16 s + 4 half + 0 .. 3 and 8 more, of V's term x */
            auto values = [&](int x, int d, int s) {
                const int vr = 32 * kb + 16 * s + 4 * half + ((lane & 15) >> 2), dim = 32 * d + (lane & 16) + 4 * (lane & 3);
                const unsigned char* at = buf + (TERMS + x) * PLANE + vr * T::ROWB + 16 * v_place(vr, dim >> 3) + 2 * (dim & 4);
                /* the second set lies 8 rows on, in the same place of its row */
                s16x4 y[2];
                y[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lvoid*)at);
                y[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lvoid*)(at + 8 * T::ROWB));
                return __builtin_bit_cast(u32x4, y);
            };
            /* A value that is no number times a masked key's weight 0 would be NaN.  Where some row of the wave does not see
             * one of the keys, such values are taken out, and the rows that do see one get NaN by a product of their own. */
            unsigned int vis[2][4];
            if (masked) {
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const unsigned int two = sees >> (8 * s + 2 * e);
                        vis[s][e] = (two & 1 ? 0x3f80u : 0u) | (two & 2 ? 0x3f800000u : 0u); /* 1 in bf16 */
                    }
            }
#pragma unroll
            for (int d = 0; d < DT; d++) {
                u32x4 v[TERMS][2];
#pragma unroll
                for (int x = 0; x < TERMS; x++)
#pragma unroll
                    for (int s = 0; s < 2; s++) v[x][s] = values(x, d, s);
                if (masked) {
                    unsigned int odd = 0;
#pragma unroll
                    for (int s = 0; s < 2; s++)
#pragma unroll
                        for (int e = 0; e < 4; e++) /* an exponent of ones carries into bit 15 or 31 */
                            odd |= (((v[0][s][e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u);
                    if (__builtin_expect(__any(odd != 0), 0)) {
                        f32x16 hit;
#pragma unroll
                        for (int e = 0; e < 16; e++) hit[e] = 0.0f;
#pragma unroll
                        for (int s = 0; s < 2; s++) {
                            u32x4 flag, one;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const unsigned int o = ((v[0][s][e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                                const unsigned int all = (o >> 15) * 0xffffu; /* both halves' bits */
                                flag[e] = all & 0x3f803f80u;
                                one[e] = vis[s][e];
#pragma unroll
                                for (int x = 0; x < TERMS; x++) v[x][s][e] &= ~all;
                            }
                            hit = mfma(__builtin_bit_cast(bf16x8, flag), __builtin_bit_cast(bf16x8, one), hit);
                        }
#pragma unroll
                        for (int e = 0; e < 16; e++) acc[d][e] = hit[e] > 0.0f ? NAN : acc[d][e];
                    }
                }
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    bf16x8 vf[TERMS];
#pragma unroll
                    for (int x = 0; x < TERMS; x++) vf[x] = __builtin_bit_cast(bf16x8, v[x][s]);
                    if constexpr (!BF16) {
                        acc[d] = mfma(vf[2], pf[0][s], acc[d]);
                        acc[d] = mfma(vf[0], pf[2][s], acc[d]);
                        acc[d] = mfma(vf[1], pf[1][s], acc[d]);
                        acc[d] = mfma(vf[1], pf[0][s], acc[d]);
                        acc[d] = mfma(vf[0], pf[1][s], acc[d]);
                    }
                    acc[d] = mfma(vf[0], pf[0][s], acc[d]);
                }
            }
        };
        auto compute = [&](const unsigned char* buf, int kt) {
            if (!active) return;
            for (int kb = kpart; kb < KB; kb += kparts) {
                const int k0 = kt * KT + 32 * kb;
                if (k0 <= any_last && k0 + 31 >= any_first && k0 < hi) block(buf, kb, k0);
            }
        };

        if constexpr (BF16) {
            /* straight into LDS, 16 bytes a lane: load i of a wave fills rows (i NW + wave) RPI .. + RPI - 1 */
            int pg[NI];
            auto pages = [&](int kt) {
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    const int key = kt * KT + (i * NW + wave) * RPI + lane / CPR;
                    pg[i] = kt < kt1 && key < hi ? page_at(key) : -2; /* -2: behind the keys */
                }
            };
            auto request = [&](int kt, unsigned char* buf) {
#pragma unroll
                for (int i = 0; i < NI; i++) {
                    const int row = (i * NW + wave) * RPI + lane / CPR, place = lane % CPR;
                    const int kc = k_place(row, place), vc = v_place(row, place); /* their own inverses */
                    const size_t at = b.base(max(pg[i], 0), 0, it.kh) + (size_t)((kt * KT + row) & mask) * HD;
                    const unsigned short* k = (const unsigned short*)a.cache + at;
                    const unsigned short* v = k + (size_t)b.NKV * kv;
                    const void* ks = 8 * kc >= HD || pg[i] == -2 ? (const void*)&pg_zeros : pg[i] < 0 ? (const void*)&pg_nans : (const void*)(k + 8 * kc);
                    const void* vs = 8 * vc >= HD || pg[i] < 0 ? (const void*)&pg_zeros : (const void*)(v + 8 * vc);
                    unsigned char* to = buf + (i * NW + wave) * 1024;
                    __builtin_amdgcn_global_load_lds((const gvoid*)ks, (lvoid*)to, 16, 0, 0);
                    __builtin_amdgcn_global_load_lds((const gvoid*)vs, (lvoid*)(to + PLANE), 16, 0, 0);
                }
            };
            __syncthreads(); /* an item before this one is through with LDS */
            if (kt0 < kt1) {
                pages(kt0);
                request(kt0, lds0);
                pages(kt0 + 1);
            }
            auto step = [&](int kt, unsigned char* buf, unsigned char* next) {
                __builtin_amdgcn_s_waitcnt(0xF70); /* vmcnt(0): the tile has landed (and the next one's pages) */
                __syncthreads();
                if (kt + 1 < kt1) {
                    request(kt + 1, next);
                    pages(kt + 2);
                }
                compute(buf, kt);
            };
            for (int kt = kt0; kt < kt1; kt += 2) {
                step(kt, lds0, lds1);
                if (kt + 1 < kt1) step(kt + 1, lds1, lds0);
            }
        } else {
            /* through registers: thread's part i of a tile is chunk c = x % CPR of row x / CPR, x = i NT + t: eight values
             * of keys and of values, split into their terms on the way into LDS */
            constexpr int PER = KT * CPR / NT;
            static_assert(KT * CPR % NT == 0, "whole parts");
            f32x4 kr[PER][2], vr[PER][2];
            auto fetch = [&](int kt) {
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int x = i * NT + t, row = x / CPR, c = x % CPR, key = kt * KT + row;
                    const int pg = key < hi ? page_at(key) : -2;
                    const size_t at = b.base(max(pg, 0), 0, it.kh) + (size_t)(key & mask) * HD + 8 * c;
                    const bool there = pg >= 0 && 8 * c < HD;
                    const float fill = pg == -1 && 8 * c < HD ? NAN : 0.0f;
                    const f32x4* k = (const f32x4*)((const float*)a.cache + at);
                    const f32x4* v = (const f32x4*)((const float*)a.cache + at + (size_t)b.NKV * kv);
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        kr[i][e] = there ? k[e] : f32x4{fill, fill, fill, fill};
                        vr[i][e] = there ? v[e] : f32x4{0, 0, 0, 0};
                    }
                }
            };
            auto put = [&](unsigned char* buf) {
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int x = i * NT + t, row = x / CPR, c = x % CPR;
#pragma unroll
                    for (int part = 0; part < 2; part++) {
                        const f32x4* src = part ? vr[i] : kr[i];
                        unsigned int z[4][3];
#pragma unroll
                        for (int e = 0; e < 4; e++) split2(src[e >> 1][2 * (e & 1)], src[e >> 1][2 * (e & 1) + 1], z[e]);
                        unsigned char* to = buf + part * TERMS * PLANE + row * T::ROWB + 16 * (part ? v_place(row, c) : k_place(row, c));
#pragma unroll
                        for (int y = 0; y < TERMS; y++) *(u32x4*)(to + y * PLANE) = u32x4{z[0][y], z[1][y], z[2][y], z[3][y]};
                    }
                }
            };
            if (kt0 < kt1) fetch(kt0);
            for (int kt = kt0; kt < kt1; kt++) {
                __syncthreads(); /* the tile before has been read */
                put(lds0);
                __syncthreads();
                if (kt + 1 < kt1) fetch(kt + 1);
                compute(lds0, kt);
            }
        }
        l += other_half(l);

        /* the waves' parts of the tiles' keys, joined in the first one's registers */
        if constexpr (KB > 1) {
            constexpr int REGS = HDP / 2 + 2;
            static_assert(KB == 2 && REGS * 64 * 4 <= sizeof lds0, "two parts, one group at a time");
            float* mem = (float*)lds0 + lane;
            for (int g = 0; kparts > 1 && g < groups; g++) {
                __syncthreads();
                if (active && group == g && kpart == 1) {
                    mem[0] = m;
                    mem[64] = l;
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++) mem[(2 + 16 * d + e) * 64] = acc[d][e];
                }
                __syncthreads();
                if (active && group == g && kpart == 0) {
                    /* a part without a finite score has what its scores left there: 0, or NaN */
                    const float m1 = mem[0], mx = fmaxf(m, m1);
                    const float f0 = m > -INFINITY ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
                    const float f1 = m1 > -INFINITY ? __builtin_amdgcn_exp2f(m1 - mx) : 1.0f;
                    l = l * f0 + mem[64] * f1;
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++) acc[d][e] = acc[d][e] * f0 + mem[(2 + 16 * d + e) * 64] * f1;
                    m = mx;
                }
            }
        }
        const bool writes = active && kpart == 0 && mine;
        if (parts == 1) {
            if (writes) {
                const size_t row = (size_t)(n0 + tok) * a.ldo + (size_t)head * HD;
                const bool none = sn.last < sn.first, gone = sn.last >= room;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const int dim = 32 * d + 2 * e + 4 * half;
                        float o[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) o[i] = none ? 0.0f : gone ? NAN : acc[d][e + i] / l;
                        if (dim < HD) store4<BF16>(a, row, dim, o);
                    }
            }
            continue;
        }
        /* Records cross XCDs: they are written and read with agent-scope accesses, past the XCDs' own L2s, and each wave
         * waits for its stores before the barrier, so a part is counted only after its record has arrived.  A unit's
         * records: [part][row]{HDP values, maximum, sum}, from the unit's rows and KV heads before it. */
        constexpr int REC = HDP + 2;
        float* recs = a.rec + ((size_t)it.rec + (size_t)it.parts * ((size_t)rows_all * it.kh + r0)) * REC;
        if (writes) {
            float* rec = recs + ((size_t)it.part * nrows + (r - r0)) * REC;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const int dim = 32 * d + 8 * (e >> 2) + 4 * half + (e & 3);
                    if (dim < HD) agent_store2(rec + dim, acc[d][e], acc[d][e + 1]);
                }
            if (half == 0) agent_store2(rec + HDP, m, l);
        }
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0);
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __syncthreads();
        if (t == 0) {
            unsigned int* done = &a.done[it.done * DONE_STRIDE];
            const unsigned int n = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_one = n == (unsigned int)parts - 1u;
            if (last_one) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last_one) continue;
        /* the rows' maxima and sums over the parts: as many threads a row as there are */
        {
            int tpr = 64;
            while (tpr * nrows > NT) tpr >>= 1;
            const int row = t / tpr, sub = t % tpr;
            float mx = -INFINITY, sum = 0.0f;
            if (row < nrows)
                for (int i = sub; i < parts; i += tpr) {
                    const f32x2 ml = agent_load2(recs + ((size_t)i * nrows + row) * REC + HDP);
                    const float mn = fmaxf(mx, ml[0]);
                    sum = sum * (mx > -INFINITY ? __builtin_amdgcn_exp2f(mx - mn) : 1.0f) +
                          ml[1] * (ml[0] > -INFINITY ? __builtin_amdgcn_exp2f(ml[0] - mn) : 1.0f);
                    mx = mn;
                }
            for (int o = 1; o < tpr; o <<= 1) {
                const float m1 = __shfl_xor(mx, o), s1 = __shfl_xor(sum, o), mn = fmaxf(mx, m1);
                sum = sum * (mx > -INFINITY ? __builtin_amdgcn_exp2f(mx - mn) : 1.0f) +
                      s1 * (m1 > -INFINITY ? __builtin_amdgcn_exp2f(m1 - mn) : 1.0f);
                mx = mn;
            }
            if (row < nrows && sub == 0) {
                row_m[row] = mx;
                row_l[row] = sum;
            }
        }
        __syncthreads();
        for (int x = t; x < nrows * (HD / 4); x += NT) {
            const int row = x / (HD / 4), dim = 4 * (x - row * (HD / 4));
            const float mx = row_m[row];
            float o[4] = {0, 0, 0, 0};
            for (int i = 0; i < parts; i += 8) {
                f32x2 y[8][3];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float* rec = recs + ((size_t)min(i + e, parts - 1) * nrows + row) * REC;
                    y[e][0] = agent_load2(rec + dim);
                    y[e][1] = agent_load2(rec + dim + 2);
                    y[e][2] = agent_load2(rec + HDP);
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (i + e >= parts) continue;
                    const float f = y[e][2][0] > -INFINITY ? __builtin_amdgcn_exp2f(y[e][2][0] - mx) : 1.0f;
#pragma unroll
                    for (int j = 0; j < 4; j++) o[j] = fmaf(f, y[e][j >> 1][j & 1], o[j]);
                }
            }
            const int rr = r0 + row, rtok = rr / a.R;
            const Seen s = seen(a, p0 + rtok, it.len);
            const bool none = s.last < s.first, gone = s.last >= room;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = none ? 0.0f : gone ? NAN : o[j] / row_l[row];
            store4<BF16>(a, (size_t)(n0 + rtok) * a.ldo + (size_t)(it.kh * a.R + rr - rtok * a.R) * HD, dim, o);
        }
        __syncthreads(); /* before another item's rows lie there */
    }
}

template <bool BF16, int HDP>
int start(PaArgs& a, const bmk_launch_t* l) {
    constexpr int KT = Tile<BF16, HDP>::KT;
    a.most = 0;
    if (l->scratch_bytes > DONE_BYTES)
        a.most = (unsigned int)std::min<size_t>((l->scratch_bytes - DONE_BYTES) / ((HDP + 2) * 4), 1u << 30);
    a.done = (unsigned int*)l->scratch;
    a.rec = (float*)((char*)l->scratch + DONE_BYTES);
    /* pieces of work: a unit for every new token or ROWS rows, in parts of a tile at least, WANTED more at most */
    const int64_t units = a.b.NKV * std::min<int64_t>(a.b.N, a.b.S + (int64_t)a.b.N * a.R / ROWS);
    const int64_t tiles = std::min<int64_t>((a.b.room() + KT - 1) / KT, MAX_SPLIT);
    const int64_t grid = std::min<int64_t>(std::min(units * tiles, units + WANTED), 1 << 20);
    hipLaunchKernelGGL((k_attn_paged<BF16, HDP>), dim3((unsigned)grid), dim3(NT), 0, l->stream, a);
    BMK_LAUNCH_CHECK();
    return 0;
}

/* {q T [N][ldq], cache, out T [N][ldo], start, len, pages,
 *  params int{N, S, NH, NKV, HD, ldq, ldo, page, n_pages, max_pages, causal, window}, f32{scale}} */
int launch_attn_paged(const bmk_launch_t* l, bool bf16) {
    BMK_NEED_BYTES(l, 6, 48, "params");
    BMK_NEED_BYTES(l, 7, 4, "scale");
    const int N = bmk_pi(l, 6, 0), S = bmk_pi(l, 6, 1), NH = bmk_pi(l, 6, 2), NKV = bmk_pi(l, 6, 3), HD = bmk_pi(l, 6, 4);
    const int ldq = bmk_pi(l, 6, 5), ldo = bmk_pi(l, 6, 6), causal = bmk_pi(l, 6, 10), window = bmk_pi(l, 6, 11);
    BMK_REQUIRE(N >= 0 && N <= PG_MAX_DIM && S >= 0 && S <= PG_MAX_SEQS && NH > 0 && NH <= PG_MAX_DIM && NKV > 0 &&
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
    a.window = std::min(window, PG_MAX_DIM); /* keys lie below that */
    a.ldq = ldq;
    a.ldo = ldo;
    const float scale = bmk_pf(l, 7, 0);
    a.flip = std::signbit(scale) ? 0x80000000u : 0u;
    a.scale2 = fabsf(scale) * 1.44269504088896341f;
    if (HD <= 64) return bf16 ? start<true, 64>(a, l) : start<false, 64>(a, l);
    if (HD <= 128) return bf16 ? start<true, 128>(a, l) : start<false, 128>(a, l);
    return bf16 ? start<true, 256>(a, l) : start<false, 256>(a, l);
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
