/* SPDX-License-Identifier: MPL-2.0
 *
 * attn_paged.hip — attention_forward_paged (include/bm_paged.h): the new
 * tokens of several sequences over the keys in their pages,
 *   out = softmax(scale * q . K + mask) V,
 * in one pass over the keys with the running maximum and sum (fp32) of the
 * softmax.
 *
 * A unit of work is up to 128 rows (new token, query head of the group)
 * of one sequence and KV head, so that every key and
 * value is read once for a whole group of heads; a unit's keys may be split
 * over workgroups, whose partial results the last one of them joins.  The work
 * goes over the keys in tiles of 32, which the loads put straight into LDS (a
 * missing page and what lies past the end by the descriptors' bounds):
 *   up to 32 rows  each of the workgroup's waves takes tiles of its own, with no barrier
 *   more           every wave has 32 rows of each tile, through a ring of tiles
 * Per tile a wave forms
 *   S^T (32 keys x 32 rows) = K Q^T,   O^T (HD x 32 rows) += V^T P^T
 * with v_mfma_f32_32x32x16_bf16.  A lane holds the scores of one row (lane %
 * 32) and 16 keys, exactly those whose weights the second product wants of
 * it once its sum runs over the keys in the order of the registers, so P goes
 * from the scores to the product without moving between lanes; V comes
 * transposed out of LDS (ds_read_b64_tr_b16).  fp32 goes in as three terms
 * x = x0 + x1 + x2 of bf16, exactly: |x1| < 2^-7 |x|, |x2| <= 2^-16 |x|, x2 of
 * either sign.  Six of the nine products are taken; what the other three would add is at
 * most 2^-22 of a product, 0.4 x 2^-24 in the mean and of either sign (with all terms cut off
 * towards zero up to 2^-21, and 0.7 x 2^-24 too little in the mean).  In bf16
 * P goes in as two terms, 2^-17 of it, where waves go alone, which the reads hide; where rows
 * fill the waves it is rounded to bf16, half a step of the output's own type (its sum is
 * not): 1.9 to 2.1e-3 from the exact result in place of the 1.66e-3 of the output's rounding,
 * but 2048 tokens over 16384 keys in 635 us in place of 760.
 *
 * What bounds it (us a pass, MI355X).  One token a sequence: reading the
 * cache; 64 sequences of 8192 keys, 8 KV heads of 128 in bf16, 233 (5.4 TB/s), 1024 of 512
 * keys, 5 heads of 64, 124 (5.4).  Few keys: the chain of latencies (the tables 1-2, the
 * page's number and the first keys 2.5, a tile 1.5, the waves' join 0.7, records and counter
 * 0.9, the parts' join 2.1); 300 keys of one token 10 of kernel time.  Long chunks: 2048 tokens
 * over 16384 keys, 32 heads of 128, 605-640, 515 GFLOP at 0.80-0.85 PFLOP/s (the
 * library's 8192^3 product runs at 1.16): a tile takes 512 cycles of the matrix cores and
 * some 600 of exponentials and other vector instructions, one after the other in a wave, which
 * two waves a SIMD overlap in part (35% and 45% busy).  fp32: 512 tokens over 4096 keys, 15 heads of 64,
 * 59-66: 43 thousand cycles a SIMD of the matrix cores, 44 thousand of vector instructions.
 */
#include "paged.h"
#include "q8_common.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

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
typedef __attribute__((address_space(3))) void lvoid;

constexpr int KT = 32;           /* keys of a tile */
/* in powers of two: how far a score may pass the running maximum before that moves (32 sequences of 16 tokens over 1500 keys,
 * with 0 28.8 us, with 8 27.6); fp32's sums have room for more */
[[maybe_unused]] constexpr float SLACK = 8.0f;
/* A row's weights are exp2(fma(score, scale2, -m)) with m = score * scale2 of its largest score, rounded, so that score's own
 * exponent is what the rounding left: up to 32 where m is under FAR, which all weights of the row have in common, but past
 * fp32's range from 2^31 on.  From FAR on the scores of a row, numbers of 24 bits, lie 64 apart or are equal: the largest takes
 * all, also with the power of two at or over scale2 in its place, whose products with them are exact.  (The rest of m as a second
 * number, carried to the joins: 2048 rows over 16384 keys 2% slower, 24 mixed sequences 4%.) */
[[maybe_unused]] constexpr float FAR = 0x1p30f;
constexpr int MAX_SPLIT = 128;   /* parts of a unit's keys */
/* tiles a part, at least: one a wave (1 token over 300 keys, parts of 2 15.3 us, 4 15.1, 8 17.5) */
constexpr int LEAST = 4;
constexpr int MANY_LEAST = 8;    /* ... of more than 32 rows (Cut::parts) */
constexpr int CUS = 256, ROUNDS = 4, ROUND_TILES = 32; /* Cut::begin */

/* The scratch memory begins with arrival counters, each on a line of its own, that are zero between launches of any
 * kernel; a table of the work and the units' partial results lie behind them. */
constexpr int DONE_STRIDE = 32, MAX_UNITS = 1024;
constexpr size_t DONE_BYTES = (size_t)DONE_STRIDE * MAX_UNITS * 4, TABLE_BYTES = 1024;
static_assert(DONE_BYTES <= BMK_SCRATCH_COUNTERS, "");

struct PaArgs {
    const void* q;
    const void* cache;
    void* out;
    unsigned int* done;
    float* rec;
    PgBatch b;
    int R; /* query heads a KV head */
    Div by_r, by_kv;
    int q_wide; /* q's heads begin on 16-byte boundaries */
    int causal, window;
    size_t ldq, ldo;
    float scale2, far_scale2; /* |scale| * log2(e); the power of two from there on */
    unsigned int flip; /* scale's sign, for q's */
    unsigned int most; /* rows' records that fit behind the counters */
    int slots; /* workgroups that run at once */
    const struct Table* table; /* of many sequences, else NULL */
};

/* How a tile lies in LDS: keys, then values, a row behind the other, HDP elements each (the head size rounded up, with zeros
 * behind it).
 *   AS_BF16  bf16 as it is
 *   AS_F32   fp32 as it is; the wave that reads it takes it apart
 *   TERMS3   fp32's three terms, one plane each, taken apart once for the waves that read them */
enum { AS_BF16, AS_F32, TERMS3 };
template <int FORM, int HDP> struct Tile {
    static constexpr int TERMS = FORM == AS_BF16 ? 1 : 3, PLANES = FORM == TERMS3 ? 3 : 1;
    static constexpr int ESZ = FORM == AS_F32 ? 4 : 2;
    static constexpr int ROWB = HDP * ESZ, CPR = ROWB / 16; /* bytes and 16-byte chunks of a row */
    static constexpr int RPI = 1024 / ROWB;                  /* rows of a wave's load into LDS */
    static constexpr int PLANE = KT * ROWB;
    static constexpr int BYTES = 2 * PLANES * PLANE;
};

/* Chunk c of row r lies at c ^ key, key < 16, so that what lanes read at once lies on all 64 banks, 256 bytes: of K one chunk
 * of 16 rows; of V two neighbouring chunks of 4 rows and the two after them (fp32: eight of a row and of the row 4 on).  Rows of
 * 128 bytes lie in two halves of the banks already.  (2048 rows over 16384 keys, keys of 8 rows in place of 16 and V's halves
 * on the same banks: half of LDS' cycles were conflicts.) */
template <int CPR>
__device__ __forceinline__ int k_place(int r, int c) { return c ^ (CPR == 8 ? r >> 1 & 7 : r & 15); }
template <int FORM, int CPR>
__device__ __forceinline__ int v_place(int r, int c) {
    return c ^ (FORM == AS_F32 ? 2 * (r & 4) : CPR == 8 ? 2 * (r & 3) : 4 * (r & 3));
}

/* A workgroup's waves and LDS: every wave has a tile of its own while it goes alone, and where rows fill the waves all have
 * a ring of four (bf16) or two (fp32, in terms; heads over 128 have no such form: their registers spill). */
template <bool BF16, int HDP> struct Shape {
    static constexpr int NW = 4, NT = 64 * NW, ROWS = 32 * NW;
    static constexpr int ALONE = BF16 ? AS_BF16 : AS_F32;
    static constexpr bool SHARED = BF16 || HDP <= 128;
    /* a wave's own tile where both halves do not fit for four waves: the values into the keys' place, once those are read (64
     * sequences of 4000 keys, 4 heads of 256: two waves with both 689 us, four with halves 446; 512 rows of 4 heads over 4096
     * 655 and 377) */
    static constexpr bool HALVES = !BF16 && HDP == 256;
    static constexpr int ALONE_BYTES = Tile<ALONE, HDP>::BYTES / (HALVES ? 2 : 1), ARRAYS = BF16 ? 4 : 1;
    static constexpr int BYTES = NW / ARRAYS * ALONE_BYTES; /* of an array */
    /* waves a SIMD, as registers (512 a lane) and LDS allow */
    static constexpr int WAVES = BF16 ? (HDP == 64 ? 3 : HDP == 128 ? 2 : 1) : HDP == 64 ? 2 : 1;
    static constexpr int SLOTS = CUS * WAVES; /* workgroups that run at once */
};

/* eight rows of a missing page's keys: NaN in either type */
#define N4 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u
#define N64 N4, N4, N4, N4, N4, N4, N4, N4, N4, N4, N4, N4, N4, N4, N4, N4
#define N512 N64, N64, N64, N64, N64, N64, N64, N64
[[maybe_unused]] __device__ __attribute__((aligned(16))) const unsigned int pg_nans[8 * PG_MAX_HD] = {N512, N512, N512, N512};
#undef N512
#undef N64
#undef N4

/* bits 15 and 31: the half below is an infinity or NaN (an exponent of ones carries) */
__device__ __forceinline__ unsigned int no_numbers(unsigned int two) {
    return ((two & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
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

__device__ __forceinline__ float low_half(unsigned int two) { return __uint_as_float(two << 16); }
__device__ __forceinline__ float high_half(unsigned int two) { return __uint_as_float(two & 0xffff0000u); }

/* Two values' three terms, packed: the upper half, which no finite value leaves for infinity, of what is left the nearest, and
 * the rest, exactly.  An infinity's others are NaN, which leaves what sees it no number, as it should. */
__device__ __forceinline__ void split2(float x, float y, unsigned int* t) {
    t[0] = pack_top(x, y);
    const float rx = x - top(x), ry = y - top(y);
    t[1] = pack_rne(rx, ry);
    t[2] = pack_top(rx - low_half(t[1]), ry - high_half(t[1]));
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

/* of all lanes alike: in scalar registers, where a descriptor has to be (the compiler loops over the lanes' descriptors
 * otherwise) */
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const char* scalar(const char* p) {
    const unsigned long long u = (unsigned long long)p;
    return (const char*)((unsigned long long)(unsigned int)scalar((int)(u >> 32)) << 32 | (unsigned int)scalar((int)u));
}

/* a descriptor of `bytes` bytes from p on, past whose end a load gives zeros and a store is dropped */
#ifdef __HIP_DEVICE_COMPILE__ /* no type of the host's */
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const char* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)scalar(p), 0, scalar(bytes), 0x00027000);
}
#endif

/* all waves of the workgroup; memory accesses stay on their side of it */
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

__device__ __forceinline__ float other_half(float v) {
    const u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? s[0] : s[1]);
}

/* ---------------------------------------------------------------- the work */

struct Seq {
    int start, n, len, T; /* first row, new tokens, keys, tiles of keys that a unit sees at most */
    unsigned int units; /* per KV head */
};

/* Sums over the lanes up to each, and the largest of all lanes, by row shifts and broadcasts (a shuffle through LDS takes
 * ten times as long, and some forty of them stood before a small launch's first load). */
template <class V>
__device__ __forceinline__ V dpp_sums(V v) {
    unsigned int u;
#define STEP(ctrl, rows) \
    u = (unsigned int)__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xF, false); \
    v += __builtin_bit_cast(V, u);
    STEP(0x111, 0xF) /* row_shr 1, 2, 4, 8 */
    STEP(0x112, 0xF)
    STEP(0x114, 0xF)
    STEP(0x118, 0xF)
    STEP(0x142, 0xA) /* lane 15 of rows 0 and 2 to the next row */
    STEP(0x143, 0xC) /* lane 31 to rows 2 and 3 */
#undef STEP
    return v;
}
template <class V>
__device__ __forceinline__ V lane_of(V v, int l) {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
__device__ __forceinline__ int dpp_most(int v) { /* of values from 0 on */
    int u;
#define STEP(ctrl, rows) \
    u = __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xF, false); \
    v = max(v, u);
    STEP(0x111, 0xF)
    STEP(0x112, 0xF)
    STEP(0x114, 0xF)
    STEP(0x118, 0xF)
    STEP(0x142, 0xA)
    STEP(0x143, 0xC)
#undef STEP
    return __builtin_amdgcn_readlane(v, 63);
}

/* Sums of pieces of work, records and units in parts, over sequences. */
struct Sums {
    unsigned int w, recs, units;
};
/* Of more sequences than a wave has lanes, a kernel ahead lays out the work: here, of each 64 sequences, the sums up to their
 * end.  (Every wave for itself, 64 sequences at a time: 128 sequences of 512 keys 18.7 us, with the table 18.2; 512 of them 93
 * and 66, 4096 2165 and 490; 65 of 16 keys 6.9 and 9.1, which is the launch, so that up to 64, where the registers hold all,
 * there is none.) */
struct Table {
    int per;            /* tiles a part */
    unsigned int total; /* pieces of work */
    Sums upto[PG_MAX_SEQS / 64];
};
static_assert(sizeof(Table) <= TABLE_BYTES && PG_MAX_SEQS == 64 * 64, "a lane of a wave for each 64 sequences");

/* How sequences are cut into units of ROWS rows and those into parts of keys. */
template <int ROWS>
struct Cut {
    const PaArgs& a;
    int per; /* tiles a part */

    __device__ __forceinline__ Seq seq(int s) const {
        Seq q = {};
        if (s < a.b.S) {
            const int at = a.b.start[s], end = a.b.start[s + 1];
            q.len = max(a.b.len[s], 0);
            q.start = at;
            if (at >= 0 && at < end && end <= a.b.N) q.n = end - at;
            q.units = ((unsigned int)q.n * (unsigned int)a.R + ROWS - 1) / ROWS;
            int span = min(q.len, a.b.room());
            if (a.window) span = min(span, a.window + a.by_r.of(ROWS) + 1 + KT);
            q.T = (span + KT - 1) / KT;
        }
        return q;
    }
    /* of a unit of q; of more rows than one wave's, no more than pay for their records (24 mixed sequences, parts of 8 tiles on
     * 26 us, of 4 or 6 27, of 12 or 16 33) */
    __device__ __forceinline__ unsigned int parts(const Seq& q) const {
        const int p = (q.T + per - 1) / per;
        return max(1, q.n * a.R > 32 ? min(p, q.T / MANY_LEAST) : p);
    }
    __device__ __forceinline__ Sums own(const Seq& q) const {
        const unsigned int p = parts(q);
        return Sums{q.units * p * a.b.NKV, p > 1 ? (unsigned int)q.n * a.R * p * a.b.NKV : 0, p > 1 ? q.units * a.b.NKV : 0};
    }
    static __device__ __forceinline__ Sums up_to(const Sums& m) {
        return Sums{dpp_sums(m.w), dpp_sums(m.recs), dpp_sums(m.units)};
    }
    /* from the sums over all sequences: of units times their tiles and of units, and the most tiles of one */
    __device__ __forceinline__ void begin(float tiles, float units, int longest) {
        tiles *= a.b.NKV;
        units *= a.b.NKV;
        /* Parts for all workgroups that run at once, or for several rounds of them, so that ragged lengths even out, where those
         * parts still have ROUND_TILES tiles (64 ragged sequences of up to 8192 keys 265 -> 235 us); never for two or three, the
         * last of which would be part empty (4 sequences of 64 rows over 40000 keys, 2 rounds 187 us, 1 145; 2.4 rounds 178). */
        const float want = a.slots * (tiles >= (float)a.slots * ROUND_TILES * ROUNDS ? ROUNDS : 1.0f);
        auto over = [](float x, float y) { return x * __builtin_amdgcn_rcpf(y); };
        int p = (int)over(tiles, fmaxf(want - 0.5f * units, 0.25f * want)) + 1;
        /* were all as long as the longest: no parts that only just do not fit (24 sequences of 4000 keys, 8 heads of 128, in
         * three parts 81 us, in two 72) */
        const float alike = over(tiles, (float)max(longest, 1));
        if (alike * ceilf(over((float)longest, (float)p) - 0.001f) > want)
            p = (int)ceilf(over((float)longest, fmaxf(floorf(over(want, alike)), 1.0f)) - 0.001f);
        per = max(max(p, LEAST), (longest + MAX_SPLIT - 1) / MAX_SPLIT);
        if (!a.most) per = max(longest, 1); /* no memory for records */
        per = scalar(per);
    }
    /* whether the records and counters do; else the parts are longer; ends at one part a unit */
    __device__ __forceinline__ bool fits(float recs, float units, int longest) {
        if (per >= longest || (recs * 1.0001f < (float)a.most && units <= (float)MAX_UNITS)) return true;
        per = scalar(per > longest / 2 ? longest : 2 * per);
        return false;
    }
    /* no batch: sequences that overlap */
    __device__ __forceinline__ bool overlap(float rows) const { return rows > (float)a.b.N * 1.0001f; }
};

/* What is to be done: of up to 64 sequences every wave finds it for itself, a sequence a lane; of more, from the table. */
template <int ROWS>
struct Plan {
    Cut<ROWS> cut;
    const PaArgs& a;
    const int lane;
    Seq first;
    unsigned int total; /* pieces of work; 0 where the tables are none */
    Sums sums;          /* over the sequences up to the lane's; over the table's entries up to the lane's */

    __device__ __forceinline__ Plan(const PaArgs& args) : cut{args, 0}, a(args), lane(threadIdx.x & 63) {
        if (a.table) {
            cut.per = a.table->per;
            total = a.table->total;
            sums = a.table->upto[lane];
            return;
        }
        first = cut.seq(lane);
        const int longest = dpp_most(first.T);
        cut.begin(lane_of(dpp_sums((float)first.units * (float)first.T), 63), lane_of(dpp_sums((float)first.units), 63), longest);
        total = 0;
        if (cut.overlap(lane_of(dpp_sums((float)first.n), 63))) return;
        for (;;) {
            const Sums m = cut.own(first);
            sums = cut.up_to(m);
            total = lane_of(sums.w, 63);
            if (cut.fits(lane_of(dpp_sums((float)m.recs), 63), lane_of(dpp_sums((float)m.units), 63), longest)) return;
        }
    }

    struct Item {
        int s, kh, unit, part, parts;
        int start, n, len;
        unsigned int rec, done; /* first of the sequence's records, the unit's counter */
    };
    /* piece w < total of the work: within a sequence the KV heads side by side, the last units, which see the most keys, first */
    __device__ __forceinline__ Item item(unsigned int w) const {
        Item it = {};
        it.s = -1;
        Sums before = {};
        int c = 0;
        Seq q = first;
        Sums m, up = sums;
        if (a.table) {
            c = __builtin_ctzll(__ballot(sums.w > w) | 1ull << 63);
            if (c) before = Sums{lane_of(sums.w, c - 1), lane_of(sums.recs, c - 1), lane_of(sums.units, c - 1)};
            q = cut.seq(64 * c + lane);
            up = cut.up_to(cut.own(q));
            w -= before.w;
        }
        m = cut.own(q);
        const unsigned long long past = __ballot(up.w > w);
        if (!past) return it;
        const int l = __builtin_ctzll(past);
        it.s = 64 * c + l;
        it.start = lane_of(q.start, l);
        it.n = lane_of(q.n, l);
        it.len = lane_of(q.len, l);
        it.parts = (int)lane_of(cut.parts(q), l);
        const unsigned int local = w - lane_of(up.w - m.w, l), nu = lane_of(q.units, l);
        const int rest = a.by_kv.of(local);
        it.kh = (int)local - rest * a.b.NKV;
        const int back = it.parts == 1 ? rest : rest / it.parts;
        it.part = rest - back * it.parts;
        it.unit = (int)nu - 1 - back;
        it.rec = before.recs + lane_of(up.recs - m.recs, l);
        it.done = before.units + lane_of(up.units - m.units, l) + it.unit * a.b.NKV + it.kh;
        return it;
    }
};

/* The table, by one workgroup: a wave has every sixteenth 64 sequences, in registers. */
template <int ROWS>
__global__ __launch_bounds__(1024) void k_attn_paged_plan(PaArgs a, Table* table) {
    constexpr int WAVES = 16, MINE = PG_MAX_SEQS / 64 / WAVES;
    __shared__ float sum[2][3][WAVES];
    __shared__ int most[WAVES];
    __shared__ Sums of64[PG_MAX_SEQS / 64];
    const int t = threadIdx.x, wave = scalar(t >> 6), lane = t & 63;
    Cut<ROWS> cut{a, 0};
    Seq q[MINE];
    float tiles = 0, units = 0, rows = 0;
    int longest = 0;
#pragma unroll
    for (int i = 0; i < MINE; i++) {
        q[i] = cut.seq(64 * (wave + WAVES * i) + lane);
        tiles += (float)q[i].units * (float)q[i].T;
        units += (float)q[i].units;
        rows += (float)q[i].n;
        longest = max(longest, q[i].T);
    }
    /* over the workgroup, in x, y, z's places */
    auto all = [&](int turn, float x, float y, float z) __attribute__((always_inline)) {
        const float v[3] = {lane_of(dpp_sums(x), 63), lane_of(dpp_sums(y), 63), lane_of(dpp_sums(z), 63)};
        if (lane == 0)
            for (int k = 0; k < 3; k++) sum[turn][k][wave] = v[k];
        __syncthreads();
    };
    auto total = [&](int turn, int k) {
        float v = 0;
        for (int i = 0; i < WAVES; i++) v += sum[turn][k][i];
        return v;
    };
    longest = dpp_most(longest);
    if (lane == 0) most[wave] = longest;
    all(0, tiles, units, rows);
    for (int i = 0; i < WAVES; i++) longest = max(longest, most[i]);
    cut.begin(total(0, 0), total(0, 1), longest);
    const bool none = cut.overlap(total(0, 2));
    for (int turn = 1;; turn ^= 1) {
        float recs = 0;
        units = 0;
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            const Sums m = cut.own(q[i]), up = cut.up_to(m);
            recs += (float)m.recs;
            units += (float)m.units;
            if (lane == 63) of64[wave + WAVES * i] = up;
        }
        all(turn, recs, units, 0.0f);
        if (cut.fits(total(turn, 0), total(turn, 1), longest)) break;
        __syncthreads(); /* of64 has not been read; sum[turn] is not written before the next turn's barrier */
    }
    if (wave) return;
    const Sums up = cut.up_to(of64[lane]);
    table->upto[lane] = up;
    if (lane == 63) {
        table->per = cut.per;
        table->total = none ? 0 : up.w;
    }
}

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
__global__ __launch_bounds__((Shape<BF16, HDP>::NT), (Shape<BF16, HDP>::WAVES)) void k_attn_paged(PaArgs a) {
#ifdef __HIP_DEVICE_COMPILE__ /* buffer descriptors are no type of the host's, which then leaves the kernel's entry out */
    typedef Shape<BF16, HDP> W;
    constexpr int NT = W::NT, NW = W::NW, ROWS = W::ROWS, TERMS = BF16 ? 1 : 3;
    constexpr int STEPS = HDP / 16, DT = HDP / 32; /* of the first product's sum; tiles of the output's dimensions */
    /* a ring of four arrays, not one array: reads of one then wait for no load into another */
    constexpr int REST = W::ARRAYS == 4 ? W::BYTES : 16;
    __shared__ __attribute__((aligned(16))) unsigned char lds0[W::BYTES], lds1[REST], lds2[REST], lds3[REST];
    __shared__ float part_m[NW][32], part_l[NW][32];
    __shared__ int last_one;
    const PgBatch& b = a.b;
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
    const int col = lane & 31, half = lane >> 5;
    const int HD = b.HD, R = a.R;
    const Plan<ROWS> plan(a);

    const unsigned int piece = pg_group();
    if (piece >= plan.total) return;
    {
        const auto it = plan.item(piece);
        if (it.s < 0) return;
        const int rows_all = it.n * R, r0 = it.unit * ROWS, nrows = min(ROWS, rows_all - r0);
        const int p0 = (int)((unsigned)it.len - (unsigned)it.n); /* position of the sequence's first new token */
        const int n0 = it.start;
        const int tok0 = a.by_r.of(r0), tok1 = a.by_r.of(r0 + nrows - 1);
        const int room = b.room();
        /* tiles of keys that some row of the unit sees, and this part's */
        const int lo = seen(a, p0 + tok0, it.len).first, hi = min(seen(a, p0 + tok1, it.len).last + 1, room);
        const int t0 = lo / KT, t1 = hi > lo ? (hi + KT - 1) / KT : t0;
        const int parts = max(1, min(it.parts, (t1 - t0 + plan.cut.per - 1) / plan.cut.per));
        const int per = (t1 - t0 + parts - 1) / parts; /* as even as they go */
        if (it.part >= parts) return;
        const int kt0 = t0 + it.part * per, kt1 = min(kt0 + per, t1);
        /* all waves have the same 32 rows and take turns on the keys' tiles, or each has rows of its own and all tiles */
        const int groups = nrows <= 32 ? 1 : NW, kparts = NW / groups; /* (48 rows in two groups on two parts: 5% more) */
        const int group = wave & (groups - 1), kpart = wave / groups;
        const bool active = 32 * group < nrows;
        const int r = r0 + 32 * group + col, tok = a.by_r.of(r), head = it.kh * R + (r - tok * R);
        const bool mine = r < r0 + nrows;
        const Seen sn = mine ? seen(a, p0 + tok, it.len) : Seen{0, -1};
        /* of the wave's rows: keys from all_first to all_last are seen by all, outside any_first .. any_last by none */
        const int gtok0 = a.by_r.of(min(r0 + 32 * group, r0 + nrows - 1));
        const int gtok1 = a.by_r.of(min(r0 + 32 * group + 31, r0 + nrows - 1));
        const Seen sa = seen(a, p0 + gtok0, it.len), sz = seen(a, p0 + gtok1, it.len);
        const int any_first = sa.first, any_last = sz.last, all_first = sz.first, all_last = sa.last;

        const size_t kv = (size_t)HD << b.shift; /* elements of one head's keys or values in a page */
        const int mask = (1 << b.shift) - 1;
        const int* table = b.pages + (size_t)it.s * b.max_pages;

        constexpr int ESZ = BF16 ? 2 : 4;
        /* q of step s: dimensions 16 s + 8 half .. + 7 of the lane's row; of fp32 heads over 128 as they are, for their terms'
         * registers spill */
        constexpr bool LATE = !BF16 && HDP == 256;
        bf16x8 qf[TERMS][LATE ? 1 : STEPS];
        u32x4 qr[STEPS][BF16 ? 1 : 2];
        /* No lane stays out (what it has no use for it reads from a place that is q's): the compiler has put a spill of all
         * lanes' values between such branches' ends. */
        auto q_request = [&]() {
            const size_t at = (size_t)(n0 + min(tok, tok1)) * a.ldq + (size_t)(mine ? head : it.kh * R) * HD;
            if (a.q_wide) {
#pragma unroll
                for (int s = 0; s < STEPS; s++)
#pragma unroll
                    for (int i = 0; i < (BF16 ? 1 : 2); i++)
                        qr[s][i] = *(const u32x4*)((const char*)a.q + (at + min(16 * s + 8 * half, HD - 8) + 4 * i) * ESZ);
            } else {
#pragma unroll
                for (int s = 0; s < STEPS; s++)
#pragma unroll
                    for (int i = 0; i < (BF16 ? 1 : 2); i++) {
                        const char* p = (const char*)a.q + (at + min(16 * s + 8 * half, HD - 8) + 4 * i) * ESZ;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const unsigned short* two = (const unsigned short*)p + 2 * e;
                            qr[s][i][e] = BF16 ? two[0] | (unsigned int)two[1] << 16 : ((const unsigned int*)p)[e];
                        }
                    }
            }
        };
        auto q_terms = [&](int s, auto& z) __attribute__((always_inline)) {
            const bool there = 16 * s + 8 * half < HD;
            unsigned int u[TERMS][4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if constexpr (BF16) {
                    u[0][e] = there ? qr[s][0][e] ^ (a.flip >> 16 | a.flip) : 0;
                } else {
                    unsigned int y[3];
                    split2(__uint_as_float(there ? qr[s][e >> 1][2 * (e & 1)] ^ a.flip : 0),
                           __uint_as_float(there ? qr[s][e >> 1][2 * (e & 1) + 1] ^ a.flip : 0), y);
#pragma unroll
                    for (int x = 0; x < TERMS; x++) u[x][e] = y[x];
                }
            }
#pragma unroll
            for (int x = 0; x < TERMS; x++) __builtin_memcpy(&z[x], u[x], 16);
        };
        auto q_take = [&]() __attribute__((always_inline)) {
            if constexpr (LATE) return;
#pragma unroll
            for (int s = 0; s < (LATE ? 0 : STEPS); s++) {
                bf16x8 z[TERMS];
                q_terms(s, z);
#pragma unroll
                for (int x = 0; x < TERMS; x++) qf[x][s] = z[x];
            }
        };

        f32x16 acc[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[d][e] = 0.0f;
        float m = -INFINITY, l = 0.0f; /* in powers of two, of the row; this lane's keys' sum */
        float scale2 = a.scale2;       /* the row's: far_scale2 where m is far */

        /* The tile of keys k0 .. k0 + 31, in LDS at `buf`.  Reads are issued in groups ahead of the products that take
         * them, the first of V's ahead of the softmax. */
        constexpr int KG = !BF16 && HDP == 256 ? 1 : 2, VG = 1;
        auto block = [&](auto form, auto weights, const unsigned char* buf, int k0,
                         auto behind_k) __attribute__((always_inline)) {
            constexpr int PT = decltype(weights)::value; /* terms of the weights */
            constexpr int FORM = decltype(form)::value, PLANES = Tile<FORM, HDP>::PLANES, PLANE = Tile<FORM, HDP>::PLANE;
            constexpr int ROWB = Tile<FORM, HDP>::ROWB, CPR = Tile<FORM, HDP>::CPR;
            f32x16 sc;
#pragma unroll
            for (int e = 0; e < 16; e++) sc[e] = 0.0f;
            typedef __attribute__((address_space(3))) s16x4 lds4;
            bf16x8 kf[2][KG][PLANES];
            f32x4 kw[2][KG][FORM == AS_F32 ? 2 : 1];
            auto read_k = [&](int g) {
                const int row = col;
#pragma unroll
                for (int s = 0; s < KG; s++) {
                    const int at = g * KG + s;
                    if constexpr (FORM == AS_F32) {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const int place = k_place<CPR>(row, (4 * at & 15) + 2 * half + i) + (4 * at & ~15);
                            kw[g & 1][s][i] = *(const f32x4*)(buf + row * ROWB + 16 * place);
                        }
                    } else {
                        const int place = k_place<CPR>(row, (2 * at & 15) + half) + (2 * at & ~15);
#pragma unroll
                        for (int x = 0; x < PLANES; x++)
                            kf[g & 1][s][x] = *(const bf16x8*)(buf + x * PLANE + row * ROWB + 16 * place);
                    }
                }
            };
            /* dimension 32 d + col, keys 16 s + 4 half + 0 .. 3 and 8 more, of V */
            u32x4 vf[2][VG][PLANES][2];
            float vw[2][VG][2][FORM == AS_F32 ? 8 : 1];
            auto read_v = [&](int g) {
#pragma unroll
                for (int d = 0; d < VG; d++)
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        if constexpr (FORM == AS_F32) {
                            const int vr = 16 * s + 4 * half, dim = 32 * (g * VG + d) + col;
                            const unsigned char* at =
                                buf + (W::HALVES ? 0 : PLANE) + vr * ROWB + 16 * v_place<FORM, CPR>(vr, dim >> 2) + 4 * (dim & 3);
#pragma unroll
                            for (int e = 0; e < 8; e++) vw[g & 1][d][s][e] = *(const float*)(at + ((e & 3) + 2 * (e & 4)) * ROWB);
                        } else {
                            const int vr = 16 * s + 4 * half + ((lane & 15) >> 2);
                            const int dim = 32 * (g * VG + d) + (lane & 16) + 4 * (lane & 3);
#pragma unroll
                            for (int x = 0; x < PLANES; x++) {
                                const unsigned char* at = buf + (PLANES + x) * PLANE + vr * ROWB +
                                                          16 * v_place<FORM, CPR>(vr, dim >> 3) + 2 * (dim & 4);
                                s16x4 y[2]; /* the second set lies 8 rows on, in the same place of its row */
                                y[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(lvoid*)at);
                                y[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(lvoid*)(at + 8 * ROWB));
                                vf[g & 1][d][x][s] = __builtin_bit_cast(u32x4, y);
                            }
                        }
                    }
            };
            auto terms_of = [&](const float* w, u32x4* t) { /* eight values' three terms */
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    unsigned int z[3];
                    split2(w[2 * e], w[2 * e + 1], z);
#pragma unroll
                    for (int x = 0; x < 3; x++) t[x][e] = z[x];
                }
            };
            read_k(0);
#pragma unroll
            for (int g = 0; g < STEPS / KG; g++) {
                if (g + 1 < STEPS / KG) read_k(g + 1);
                else if constexpr (!W::HALVES) read_v(0);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int s = 0; s < KG; s++) {
                    const int at = g * KG + s;
                    bf16x8 k[TERMS];
                    if constexpr (FORM == AS_F32) {
                        float w[8];
                        u32x4 z[TERMS];
                        __builtin_memcpy(w, kw[g & 1][s], 32);
                        terms_of(w, z);
#pragma unroll
                        for (int x = 0; x < TERMS; x++) k[x] = __builtin_bit_cast(bf16x8, z[x]);
                    } else {
#pragma unroll
                        for (int x = 0; x < TERMS; x++) k[x] = kf[g & 1][s][x];
                    }
                    bf16x8 q[TERMS];
                    if constexpr (LATE) {
                        asm volatile("" : "+v"(qr[at][0]), "+v"(qr[at][1])); /* here, not ahead of the loop */
                        q_terms(at, q);
                    } else {
#pragma unroll
                        for (int x = 0; x < TERMS; x++) q[x] = qf[x][at];
                    }
                    if constexpr (!BF16) { /* the small terms first */
                        sc = mfma(k[2], q[0], sc);
                        sc = mfma(k[0], q[2], sc);
                        sc = mfma(k[1], q[1], sc);
                        sc = mfma(k[1], q[0], sc);
                        sc = mfma(k[0], q[1], sc);
                    }
                    sc = mfma(k[0], q[0], sc);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            behind_k();
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
            if (__any(cm * scale2 > m + SLACK)) { /* -infinity times 0 is NaN, which moves nothing */
                cm = fmaxf(cm, other_half(cm));
                /* of its own scores alone: what another row of the wave sees does not touch a row's roundings */
                const bool moves = cm * scale2 > m + SLACK;
                if (moves) scale2 = fabsf(cm * a.scale2) >= FAR ? a.far_scale2 : a.scale2;
                const float mn = moves ? cm * scale2 : m, f = mn > -INFINITY ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
                l *= f;
#pragma unroll
                for (int d = 0; d < DT; d++) acc[d] *= f;
                m = mn;
            }
            const float ms = m > -INFINITY ? m : 0.0f;
            float p[16];
#pragma unroll
            for (int e = 0; e < 16; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], scale2, -ms));
            if (masked) {
#pragma unroll
                for (int e = 0; e < 16; e++) p[e] = sees >> e & 1 ? p[e] : 0.0f;
            }
            float s4[4];
#pragma unroll
            for (int e = 0; e < 4; e++) s4[e] = (p[e] + p[e + 4]) + (p[e + 8] + p[e + 12]);
            l += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            bf16x8 pf[PT][2];
#pragma unroll
            for (int s = 0; s < 2; s++) {
                unsigned int u[PT][4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = p[8 * s + 2 * e], y = p[8 * s + 2 * e + 1];
                    if constexpr (BF16) {
                        u[0][e] = pack_rne(x, y);
                        if constexpr (PT == 2) u[1][e] = pack_rne(x - low_half(u[0][e]), y - high_half(u[0][e]));
                    } else {
                        unsigned int z[3];
                        split2(x, y, z);
#pragma unroll
                        for (int i = 0; i < TERMS; i++) u[i][e] = z[i];
                    }
                }
#pragma unroll
                for (int x = 0; x < PT; x++) __builtin_memcpy(&pf[x][s], u[x], 16);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (W::HALVES) {
                __builtin_amdgcn_s_waitcnt(0x0F70); /* vmcnt(0): the values are there */
                asm volatile("" ::: "memory");
                read_v(0);
            }
#pragma unroll
            for (int g = 0; g < DT / VG; g++) {
                if (W::HALVES ? g > 0 : g + 1 < DT / VG) read_v(W::HALVES ? g : g + 1); /* HALVES: no registers for one ahead */
                __builtin_amdgcn_sched_barrier(0);
                u32x4 v[VG][TERMS][2];
#pragma unroll
                for (int d = 0; d < VG; d++)
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        u32x4 z[TERMS];
                        if constexpr (FORM == AS_F32) {
                            terms_of(vw[g & 1][d][s], z);
                        } else {
#pragma unroll
                            for (int x = 0; x < TERMS; x++) z[x] = vf[g & 1][d][x][s];
                        }
#pragma unroll
                        for (int x = 0; x < TERMS; x++) v[d][x][s] = z[x];
                    }
                /* A value that is no number times a masked key's weight 0 would be NaN.  Where some row of the wave does not
                 * see one of the keys, such values are taken out, and the rows that do see one get NaN by a product of
                 * their own. */
                if (masked) {
                    unsigned int odd = 0;
#pragma unroll
                    for (int d = 0; d < VG; d++)
#pragma unroll
                        for (int s = 0; s < 2; s++)
#pragma unroll
                            for (int e = 0; e < 4; e++) odd |= no_numbers(v[d][0][s][e]);
                    if (__builtin_expect(__any(odd != 0), 0)) {
                        u32x4 vis[2];
#pragma unroll
                        for (int s = 0; s < 2; s++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const unsigned int two = sees >> (8 * s + 2 * e);
                                vis[s][e] = (two & 1 ? 0x3f80u : 0u) | (two & 2 ? 0x3f800000u : 0u); /* 1 in bf16 */
                            }
#pragma unroll
                        for (int d = 0; d < VG; d++) {
                            f32x16 hit;
#pragma unroll
                            for (int e = 0; e < 16; e++) hit[e] = 0.0f;
#pragma unroll
                            for (int s = 0; s < 2; s++) {
                                u32x4 flag;
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const unsigned int all = (no_numbers(v[d][0][s][e]) >> 15) * 0xffffu; /* the halves' bits */
                                    flag[e] = all & 0x3f803f80u;
#pragma unroll
                                    for (int x = 0; x < TERMS; x++) v[d][x][s][e] &= ~all;
                                }
                                hit = mfma(__builtin_bit_cast(bf16x8, flag), __builtin_bit_cast(bf16x8, vis[s]), hit);
                            }
#pragma unroll
                            for (int e = 0; e < 16; e++) acc[g * VG + d][e] = hit[e] > 0.0f ? NAN : acc[g * VG + d][e];
                        }
                    }
                }
#pragma unroll
                for (int s = 0; s < 2; s++)
#pragma unroll
                    for (int d = 0; d < VG; d++) {
                        f32x16& o = acc[g * VG + d];
                        bf16x8 y[TERMS];
#pragma unroll
                        for (int x = 0; x < TERMS; x++) y[x] = __builtin_bit_cast(bf16x8, v[d][x][s]);
                        if constexpr (!BF16) {
                            o = mfma(y[2], pf[0][s], o);
                            o = mfma(y[0], pf[2][s], o);
                            o = mfma(y[1], pf[1][s], o);
                            o = mfma(y[1], pf[0][s], o);
                            o = mfma(y[0], pf[1][s], o);
                        } else if constexpr (PT == 2) {
                            o = mfma(y[0], pf[1][s], o);
                        }
                        o = mfma(y[0], pf[0][s], o);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto compute = [&](auto form, auto weights, const unsigned char* buf, int kt,
                           auto behind_k) __attribute__((always_inline)) {
            const int k0 = kt * KT;
            if (active && (kt & (kparts - 1)) == kpart && k0 <= any_last && k0 + 31 >= any_first && k0 < hi)
                block(form, weights, buf, k0, behind_k);
        };

        /* Straight into LDS, 16 bytes a lane, a wave's load RPI rows, eight at most, which lie in one page.  Its number is read
         * into a scalar register, apart from the loads' count, so that nothing waits for the tiles that are under way; what lies
         * behind this part's keys or a head's end comes as zeros by the buffer's bounds, a missing page's keys from rows of
         * NaN. */
        typedef Tile<W::ALONE, HDP> T;
        constexpr int RPI = T::RPI, CPR = T::CPR, PLANE = T::PLANE, KINDS = 16 / RPI; /* loads whose places differ */
        const int end = min(hi, kt1 * KT), rowb = HD * ESZ;
        const size_t page_bytes = (size_t)b.NKV * kv * (2 * ESZ), kh_bytes = (size_t)it.kh * kv * ESZ;
        auto page_of = [&](int key) { /* key: a multiple of 8, or within them; wave-uniform */
            return ((const __attribute__((address_space(4))) int*)table)[scalar(max(min(key, hi - 1), 0) >> b.shift)];
        };
        /* a lane's place in the rows of a load whose first row is `first` mod 16, of keys and of values */
        auto lane_place = [&](int first, int& k, int& v) {
            const int row = lane / CPR, place = lane % CPR;
            /* their own inverses */
            const int kc = k_place<CPR>(first + row, place), vc = v_place<W::ALONE, CPR>(first + row, place);
            k = 16 * kc < rowb ? row * rowb + 16 * kc : 1 << 30;
            v = 16 * vc < rowb ? row * rowb + 16 * vc : 1 << 30;
        };
        auto load = [&](int pg, int key, unsigned char* to, int k_off, int v_off, bool keys = true,
                        bool values = true) __attribute__((always_inline)) {
            const bool there = (unsigned int)pg < (unsigned int)b.n_pages;
            const int bytes = min(max(end - key, 0), RPI) * rowb;
            const char* k = (const char*)a.cache + (there ? pg : 0) * page_bytes + kh_bytes + (unsigned int)((key & mask) * rowb);
            const auto ks = rsrc(there ? k : (const char*)pg_nans, bytes), vs = rsrc(k + page_bytes / 2, there ? bytes : 0);
            if (keys) __builtin_amdgcn_raw_ptr_buffer_load_lds(ks, (lvoid*)to, 16, k_off, 0, 0, 0);
            if (values) __builtin_amdgcn_raw_ptr_buffer_load_lds(vs, (lvoid*)(to + (W::HALVES ? 0 : PLANE)), 16, v_off, 0, 0, 0);
        };

        if (!W::SHARED || groups == 1) {
            /* Few rows: each wave goes over tiles of its own, one at a time, with no barrier; the other waves' loads are under
             * way while it computes. */
            unsigned char* buf;
            if constexpr (W::ARRAYS == 4) buf = wave == 0 ? lds0 : wave == 1 ? lds1 : wave == 2 ? lds2 : lds3;
            else buf = lds0 + wave * W::ALONE_BYTES;
            int k_off[KINDS], v_off[KINDS];
            if constexpr (KINDS <= 8)
#pragma unroll
                for (int i = 0; i < KINDS; i++) lane_place(i * RPI, k_off[i], v_off[i]);
            int pg[4]; /* of eight rows each */
            auto pages = [&](int kt) {
#pragma unroll
                for (int i = 0; i < 4; i++) pg[i] = page_of(kt * KT + 8 * i);
            };
            auto request = [&](int kt, bool values) __attribute__((always_inline)) { /* HALVES: the keys, or the values */
                if constexpr (W::HALVES) { /* 32 descriptors at once spill scalar registers */
                    static_assert(RPI == 1, "");
#pragma unroll 1
                    for (int g = 0; g < 4; g++) {
                        const int key = kt * KT + 8 * g, p = page_of(key);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            int k, v;
                            lane_place(8 * g + i, k, v);
                            load(p, key + i, buf + (8 * g + i) * 1024, k, v, !values, values);
                        }
                    }
                    return;
                }
#pragma unroll
                for (int i = 0; i < KT / RPI; i++)
                    load(pg[i * RPI / 8], kt * KT + i * RPI, buf + i * 1024, k_off[i % KINDS], v_off[i % KINDS]);
            };
            int kt = kt0 + ((kpart - kt0) & (kparts - 1)); /* tiles kpart mod kparts, as compute takes them */
            pages(kt);
            q_request();
            if constexpr (!BF16 && HDP == 256) q_take(); /* no registers for both */
            __builtin_amdgcn_sched_barrier(0);
            request(kt, false);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (BF16 || HDP < 256) q_take();
            for (; kt < kt1; kt += kparts) {
                pages(kt + kparts);
                __builtin_amdgcn_s_waitcnt(0x0F70); /* vmcnt(0) */
                asm volatile("" ::: "memory");
                auto values = [&]() __attribute__((always_inline)) {
                    if constexpr (W::HALVES) request(kt, true);
                };
                compute(std::integral_constant<int, W::ALONE>{}, std::integral_constant<int, BF16 ? 2 : 3>{}, buf, kt, values);
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                if (kt + kparts < kt1) request(kt + kparts, false);
            }
            __builtin_amdgcn_s_waitcnt(0x0F70); /* none under way */
        } else if constexpr (BF16) {
            /* Load i of a wave fills rows (i NW + wave) RPI .. + RPI - 1. */
            constexpr int NI = PLANE / 1024 / NW, KN = NW * RPI < 16 ? 16 / (NW * RPI) : 1;
            int k_off[KN], v_off[KN], pg[NI];
#pragma unroll
            for (int i = 0; i < KN; i++) lane_place((i * NW + wave) * RPI, k_off[i], v_off[i]);
            auto pages = [&](int kt) {
#pragma unroll
                for (int i = 0; i < NI; i++) pg[i] = page_of(kt * KT + (i * NW + wave) * RPI);
            };
            auto request = [&](int kt, unsigned char* buf) {
#pragma unroll
                for (int i = 0; i < NI; i++)
                    load(pg[i], kt * KT + (i * NW + wave) * RPI, buf + (i * NW + wave) * 1024, k_off[i % KN], v_off[i % KN]);
            };
            pages(kt0);
            q_request();
            __builtin_amdgcn_sched_barrier(0);
            request(kt0, lds0);
            pages(kt0 + 1);
            request(kt0 + 1, lds1);
            pages(kt0 + 2);
            request(kt0 + 2, lds2);
            pages(kt0 + 3);
            __builtin_amdgcn_sched_barrier(0);
            q_take();
            /* Three tiles are under way while one is read; a tile's array is requested again behind the barrier that all
             * waves reach when they have read it.  Tiles behind the last are zeros. */
            constexpr int AHEAD = 4 * NI; /* loads of the two tiles after the one to be read */
            auto step = [&](int kt, unsigned char* buf, unsigned char* before) __attribute__((always_inline)) {
                __builtin_amdgcn_s_waitcnt(0x0F70 | (AHEAD & 15) | ((AHEAD >> 4) << 14));
                barrier();
                request(kt + 3, before);
                pages(kt + 4);
                compute(std::integral_constant<int, AS_BF16>{}, std::integral_constant<int, 1>{}, buf, kt, []() {});
            };
            for (int kt = kt0; kt < kt1; kt += 4) {
                step(kt, lds0, lds3);
                if (kt + 1 < kt1) step(kt + 1, lds1, lds0);
                if (kt + 2 < kt1) step(kt + 2, lds2, lds1);
                if (kt + 3 < kt1) step(kt + 3, lds3, lds2);
            }
            __builtin_amdgcn_s_waitcnt(0x0F70); /* none under way */
        } else if constexpr (W::SHARED) {
            /* Through registers: piece x = i NT + t of a tile is eight values, chunk c of a row, of keys, then of values, split
             * into their terms on the way into LDS, two tiles in turn. */
            typedef Tile<TERMS3, HDP> T3;
            constexpr int C3 = T3::CPR, HALF = KT * C3, PER = 2 * HALF / NT;
            static_assert(2 * HALF % NT == 0 && HALF % 64 == 0 && 2 * T3::BYTES <= W::BYTES,
                          "whole pieces, a wave's of keys or of values, two tiles");
            constexpr int RPP = 64 / C3; /* rows of a wave's piece, in one page */
            f32x4 raw[PER][2];
            int pg[PER];
            const int off = 8 * (lane % C3) < HD ? lane / C3 * rowb + 32 * (lane % C3) : 1 << 30;
            auto row_of = [&](int i) { return (i * NT / 64 + wave) % (HALF / 64) * RPP; };
            auto part_of = [&](int i) { return (i * NT / 64 + wave) / (HALF / 64); };
            auto pages = [&](int kt) {
#pragma unroll
                for (int i = 0; i < PER; i++) pg[i] = page_of(kt * KT + row_of(i));
            };
            auto fetch = [&](int kt) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int key = kt * KT + row_of(i), part = part_of(i);
                    const bool there = (unsigned int)pg[i] < (unsigned int)b.n_pages;
                    const char* k = (const char*)a.cache + (there ? pg[i] : 0) * page_bytes + kh_bytes +
                                    (unsigned int)((key & mask) * rowb);
                    const auto from = rsrc(part ? k + page_bytes / 2 : there ? k : (const char*)pg_nans,
                                           part && !there ? 0 : min(max(end - key, 0), RPP) * rowb);
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        raw[i][e] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, off + 16 * e, 0, 0));
                }
            };
            auto put = [&](unsigned char* buf) {
#pragma unroll
                for (int i = 0; i < PER; i++) {
                    const int part = part_of(i), row = row_of(i) + lane / C3, c = lane % C3;
                    unsigned int z[4][3];
#pragma unroll
                    for (int e = 0; e < 4; e++) split2(raw[i][e >> 1][2 * (e & 1)], raw[i][e >> 1][2 * (e & 1) + 1], z[e]);
                    unsigned char* to = buf + part * 3 * T3::PLANE + row * T3::ROWB +
                                        16 * (part ? v_place<TERMS3, C3>(row, c) : k_place<C3>(row, c));
#pragma unroll
                    for (int w = 0; w < 3; w++) *(u32x4*)(to + w * T3::PLANE) = u32x4{z[0][w], z[1][w], z[2][w], z[3][w]};
                }
            };
            pages(kt0);
            q_request();
            fetch(kt0);
            pages(kt0 + 1);
            q_take();
            for (int kt = kt0; kt < kt1; kt++) {
                unsigned char* buf = lds0 + ((kt - kt0) & 1) * T3::BYTES;
                put(buf);
                __syncthreads(); /* the tile is there, and the one before has been read */
                fetch(kt + 1); /* behind the part's last: zeros */
                pages(kt + 2);
                compute(std::integral_constant<int, TERMS3>{}, std::integral_constant<int, 3>{}, buf, kt, []() {});
            }
        }
        l += other_half(l);

        constexpr int REC = HDP + 4, SC1 = 16;
        const int part_bytes = nrows * REC * 4, quads = HD / 4;
        const auto recs = rsrc((const char*)(a.rec + ((size_t)it.rec + (size_t)it.parts * ((size_t)rows_all * it.kh + r0)) * REC),
                               parts * part_bytes);
        auto four = [&](int d, int e) __attribute__((always_inline)) {
            return f32x4{acc[d][e], acc[d][e + 1], acc[d][e + 2], acc[d][e + 3]};
        };
        auto put = [&](int row, int quad, f32x4 x) __attribute__((always_inline)) {
            const int at = it.part * part_bytes + (quad * nrows + row) * 16;
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), recs, at, 0, SC1);
        };
        /* four outputs of a row, of its sums */
        auto finish = [&](int row, int quad, f32x4 x, float sum) __attribute__((always_inline)) {
            const int rr = r0 + row, rtok = a.by_r.of(rr);
            const Seen s = seen(a, p0 + rtok, it.len);
            const bool none = s.last < s.first, gone = s.last >= room;
            float out[4];
#pragma unroll
            for (int j = 0; j < 4; j++) out[j] = none ? 0.0f : gone ? NAN : x[j] / sum;
            store4<BF16>(a, (size_t)(n0 + rtok) * a.ldo + (size_t)(it.kh * R + rr - rtok * R) * HD, 4 * quad, out);
        };
        if (kparts > 1) {
            /* The waves' sums of the same rows, each in its own tile's place, joined four outputs a lane. */
            constexpr int SUMS = HDP * 128;
            static_assert(SUMS <= W::ALONE_BYTES, "");
            auto place = [&](int w) {
                return (f32x4*)(W::ARRAYS == 1 ? lds0 + w * W::ALONE_BYTES
                                : w == 0       ? lds0
                                : w == 1       ? lds1
                                : w == 2       ? lds2
                                               : lds3);
            };
            if (mine) {
                f32x4* mem = place(wave) + col;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        mem[(8 * d + e / 2 + half) * 32] = four(d, e);
                if (half == 0) {
                    part_m[wave][col] = m;
                    part_l[wave][col] = l;
                }
            }
            __syncthreads();
            for (int x = t; x < nrows * quads; x += NT) {
                const int quad = x / nrows, row = x - quad * nrows;
                float mx = part_m[0][row], sum = 0.0f;
#pragma unroll
                for (int w = 1; w < NW; w++) mx = fmaxf(mx, part_m[w][row]);
                f32x4 o = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < NW; w++) { /* a part without a finite score has what its scores left there: 0, or NaN */
                    const float mw = part_m[w][row], f = mw > -INFINITY ? __builtin_amdgcn_exp2f(mw - mx) : 1.0f;
                    const f32x4 y = place(w)[quad * 32 + row];
                    sum = fmaf(part_l[w][row], f, sum);
#pragma unroll
                    for (int j = 0; j < 4; j++) o[j] = fmaf(y[j], f, o[j]);
                }
                if (parts == 1) {
                    finish(row, quad, o, sum);
                } else {
                    put(row, quad, o);
                    if (quad == 0) put(row, HDP / 4, f32x4{mx, sum, 0.0f, 0.0f});
                }
            }
            if (parts == 1) return;
        } else if (parts == 1) {
            if (mine) {
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        if (32 * d + 2 * e + 4 * half < HD) finish(r - r0, 8 * d + e / 2 + half, four(d, e), l);
            }
            return;
        } else if (mine) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    if (32 * d + 2 * e + 4 * half < HD) put(r - r0, 8 * d + e / 2 + half, four(d, e));
            if (half == 0) put(r - r0, HDP / 4, f32x4{m, l, 0.0f, 0.0f});
        }
        /* Records cross XCDs: they are written and read past the XCDs' own L2s (sc1), and each wave waits for its stores before
         * the barrier, so a part is counted only after its record has arrived.  A unit's records: of each part, four
         * dimensions of all rows side by side, then all rows' maxima and sums, 16 bytes each. */
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
        if (!last_one) return;
        /* Four outputs (a quad of dimensions) at a time from their records.  Where a unit has more quads than there are lanes, a
         * lane keeps to one row and reads U of its quads' records and P parts at once (4 and 4: of 24 mixed sequences 26 us, two
         * quads a row for each lane 28; 8 and 4 or 4 and 8 have no registers: 30 and 34); where it has fewer, 1 << by_log lanes
         * side by side, up to 64, share a quad's parts. */
        const int across = NT / nrows, each = (quads + across - 1) / across;
        int by_log = 0;
        while (by_log < 6 && nrows * quads << (by_log + 1) <= NT && 4 << by_log < parts) by_log++;
        auto take = [&](int at) __attribute__((always_inline)) {
            return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(recs, at, 0, SC1));
        };
        auto join = [&](auto us, auto ps) __attribute__((always_inline)) {
            constexpr int U = decltype(us)::value, P = decltype(ps)::value;
            const int sub = U == 1 ? t & ((1 << by_log) - 1) : 0, x = U == 1 ? t >> by_log : t;
            /* this lane's quads: col0, col0 + apart, .. */
            const int col0 = x / nrows, row = x - col0 * nrows, apart = (NT >> by_log) / nrows;
            if (col0 >= (U == 1 ? quads : across)) return;
            for (int q0 = col0; q0 < quads; q0 += U * apart) {
                f32x4 o[U];
                float mx = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int u = 0; u < U; u++) o[u] = f32x4{0, 0, 0, 0};
                for (int i = sub; i < parts; i += P << by_log) {
                    f32x4 y[P][U], ml[P];
#pragma unroll
                    for (int e = 0; e < P; e++) { /* past the parts: the descriptor's end, zeros */
                        const int at = (i + (e << by_log)) * part_bytes + row * 16;
                        ml[e] = take(at + HDP / 4 * nrows * 16);
#pragma unroll
                        for (int u = 0; u < U; u++) {
                            const int quad = min(q0 + u * apart, quads - 1);
                            y[e][u] = take(at + quad * nrows * 16);
                        }
                    }
                    float mn = mx;
#pragma unroll
                    for (int e = 0; e < P; e++) {
                        if (i + (e << by_log) >= parts) ml[e] = f32x4{-INFINITY, 0, 0, 0};
                        mn = fmaxf(mn, ml[e][0]);
                    }
                    const float f = mx > -INFINITY ? __builtin_amdgcn_exp2f(mx - mn) : 1.0f;
                    sum *= f;
#pragma unroll
                    for (int u = 0; u < U; u++) o[u] *= f;
#pragma unroll
                    for (int e = 0; e < P; e++) { /* a part without a finite score has 0 or NaN */
                        const float g = ml[e][0] > -INFINITY ? __builtin_amdgcn_exp2f(ml[e][0] - mn) : 1.0f;
                        sum = fmaf(g, ml[e][1], sum);
#pragma unroll
                        for (int u = 0; u < U; u++)
#pragma unroll
                            for (int j = 0; j < 4; j++) o[u][j] = fmaf(g, y[e][u][j], o[u][j]);
                    }
                    mx = mn;
                }
                if constexpr (U == 1) {
                    for (int k = 0; k < by_log; k++) {
                        const float m1 = __shfl_xor(mx, 1 << k), mn = fmaxf(mx, m1);
                        const float f = mx > -INFINITY ? __builtin_amdgcn_exp2f(mx - mn) : 1.0f;
                        const float g = m1 > -INFINITY ? __builtin_amdgcn_exp2f(m1 - mn) : 1.0f;
                        sum = sum * f + __shfl_xor(sum, 1 << k) * g;
#pragma unroll
                        for (int j = 0; j < 4; j++) o[0][j] = o[0][j] * f + __shfl_xor(o[0][j], 1 << k) * g;
                        mx = mn;
                    }
                    if (sub) return;
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (q0 + u * apart >= quads) break;
                    finish(row, q0 + u * apart, o[u], sum);
                }
            }
        };
        if (each == 1) join(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
        else join(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
    }
#endif
}

template <bool BF16, int HDP>
int start(PaArgs& a, const bmk_launch_t* l) {
    typedef Shape<BF16, HDP> W;
    a.most = 0;
    if (l->scratch_bytes > DONE_BYTES + TABLE_BYTES)
        a.most = (unsigned int)std::min<size_t>((l->scratch_bytes - DONE_BYTES - TABLE_BYTES) / ((HDP + 4) * 4), 1u << 30);
    a.done = (unsigned int*)l->scratch;
    a.rec = (float*)((char*)l->scratch + DONE_BYTES + TABLE_BYTES);
    a.slots = W::SLOTS;
    if (a.b.S > 64 && !a.most) { /* no memory for the table */
        PaArgs some = a;
        for (int s = 0; s < a.b.S; s += 64) {
            some.b.S = std::min(a.b.S - s, 64);
            some.b.start = a.b.start + s;
            some.b.len = a.b.len + s;
            some.b.pages = a.b.pages + (size_t)s * a.b.max_pages;
            if (int rc = start<BF16, HDP>(some, l)) return rc;
        }
        return 0;
    }
    if (a.b.S > 64) {
        Table* table = (Table*)((char*)l->scratch + DONE_BYTES);
        hipLaunchKernelGGL((k_attn_paged_plan<W::ROWS>), dim3(1), dim3(1024), 0, l->stream, a, table);
        BMK_LAUNCH_CHECK();
        a.table = table;
    }
    /* A workgroup a piece: no more than a unit for every sequence with new tokens and every ROWS rows, each in one part more
     * than the tiles' share of the plan's want (the 8: sums rounded in fp32). */
    const int64_t units = a.b.NKV * (std::min<int64_t>(a.b.N, a.b.S) + (int64_t)a.b.N * a.R / W::ROWS);
    const int64_t tiles = (a.b.room() + KT - 1) / KT;
    const int64_t rounds = units * tiles >= (int64_t)a.slots * ROUND_TILES * ROUNDS ? ROUNDS : 1;
    const int64_t grid = std::min(units * std::min<int64_t>(tiles, MAX_SPLIT), units + a.slots * rounds + 8);
    hipLaunchKernelGGL((k_attn_paged<BF16, HDP>), pg_grid(grid, W::NT), dim3(W::NT), 0, l->stream, a);
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
    BMK_REQUIRE((int64_t)N * NH < (1LL << 30), "attention_forward_paged: %d rows of %d heads are over 2^30 heads", N, NH);
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
    a.R = NH / NKV;
    a.by_r = div_by(a.R);
    a.by_kv = div_by(NKV);
    a.q_wide = (uintptr_t)l->dev[0] % 16 == 0 && ldq * esz % 16 == 0;
    a.causal = causal;
    a.window = std::min(window, PG_MAX_DIM); /* keys lie below that */
    a.ldq = ldq;
    a.ldo = ldo;
    const float scale = bmk_pf(l, 7, 0);
    a.flip = std::signbit(scale) ? 0x80000000u : 0u;
    a.scale2 = fabsf(scale) * 1.44269504088896341f;
    int two;
    /* 0 and the powers of two are their own */
    a.far_scale2 = a.scale2 < INFINITY && frexpf(a.scale2, &two) > 0.5f ? ldexpf(1.0f, two) : a.scale2;
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

/* workgroups of a launch along x and y */
extern "C" void bmk_paged_grid(long long groups, int lanes, unsigned int* xy) {
    const dim3 g = pg_grid(groups, lanes);
    xy[0] = g.x;
    xy[1] = g.y;
}

extern "C" int bmk_launch_attn_paged(const bmk_launch_t* a) { return launch_attn_paged(a, false); }
extern "C" int bmk_launch_attn_paged_bf16(const bmk_launch_t* a) { return launch_attn_paged(a, true); }
