/* SPDX-License-Identifier: MPL-2.0
 *
 * i8_gemm.hip — the product of 8-bit codes (matmul_forward_i8, _bf16) on gfx950 int8 MFMA:
 *   out[m][n] = (sum_k a[m][k] * w[n][k]) * sa[m] * sw[n] + bias[n]
 * The sum is exact in 32-bit integers (fewer than 2^17 columns: 2^17 products
 * of at most 2^14 would pass 2^31), so neither tiles nor the split of a sum
 * change a result.  It is converted once, multiplied by the row's scale, then
 * by the column's (each rounding to fp32), the bias added, and for bf16
 * outputs rounded once more.
 *
 * All forms use v_mfma_i32_16x16x64_i8, with the weights as its first operand:
 * a lane then holds four neighbouring outputs of one row.  The 32 x 32 x 32 form
 * is slower on this part (registers only, all CUs, codes of a normal
 * distribution: 2.6 against 4.1 POP/s).
 *   k_i8_few   few rows or outputs: operands straight into registers, the sum split over four or eight waves
 *   k_i8_tile  tiles of 32 x 32 to 192 x 192 through LDS, four or eight waves
 *   k_i8_pair  256 x 256, eight waves in two groups that take turns at the matrix cores and at LDS
 * Operands go to LDS by global_load_lds, which writes 16 bytes a lane at
 * consecutive addresses, so a row's 16-byte groups are permuted on the source
 * side (group_key), such that the 16 rows of a fragment lie in different banks.
 * Rows past M or OC repeat the last one and groups past C the last one; the
 * first feed nothing stored, and the tokens' codes past C are zeroed in
 * registers (what the weights hold there is then multiplied by zero).
 */
#include "i8_common.h"

#include <climits>

namespace {

using namespace bmk;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(1))) void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

constexpr int MAX_C = (1 << 17) - 1;
constexpr int XCDS = 8;
constexpr int CUS = 256;
constexpr int MAX_GRID_X = 1 << 20;

struct GemmArgs {
    const unsigned char* a;
    const float* sa;
    const unsigned char* w;
    const float* sw;
    const float* bias;
    void* out;
    size_t lda, ldw, ldo;
    int M, C, OC, tiles_m, tiles_n;
};

__device__ __forceinline__ int workgroup() { return (int)(blockIdx.y * gridDim.x + blockIdx.x); }

/* This workgroup's tile, or false for one past the last.  Workgroups are dealt
 * to the XCDs in turn, and every XCD takes a run of neighbouring tiles (four
 * tile rows wide), which share operands in its L2. */
__device__ __forceinline__ bool tile_of(const GemmArgs& g, int& tm, int& tn) {
    const int total = g.tiles_m * g.tiles_n;
    int b = workgroup();
    if (b >= total) return false;
    const int per = total / XCDS, x = b % XCDS;
    b = x * per + min(x, total - per * XCDS) + b / XCDS;
    constexpr int GM = 4;
    const int span = GM * g.tiles_n, grp = b / span, in = b - grp * span, gm = min(GM, g.tiles_m - grp * GM);
    tm = grp * GM + in % gm;
    tn = in / gm;
    return true;
}

/* the first n bytes of a 16-byte group (all from n = 16 on), zeros behind them */
__device__ __forceinline__ i32x4 head_bytes(i32x4 v, int n) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int left = n - 4 * i;
        if (left <= 0) v[i] = 0;
        else if (left < 4) v[i] &= (1 << (8 * left)) - 1;
    }
    return v;
}

__device__ __forceinline__ unsigned int pk(float lo, float hi) {
    return __builtin_bit_cast(unsigned int, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

/* 16 or 8 bytes to an address on an output element's boundary */
template <bool BF16, class T>
__device__ __forceinline__ void store_vec(void* out, size_t at, T v) {
    if (BF16) __builtin_memcpy(__builtin_assume_aligned((unsigned short*)out + at, 2), &v, sizeof v);
    else __builtin_memcpy(__builtin_assume_aligned((float*)out + at, 4), &v, sizeof v);
}

/* Scales, bias and store of TM x TN 16 x 16 sums: lane l holds row l % 16,
 * columns 4 (l / 16) .. + 3 of each.  Pairs of bf16 tiles swap 16-lane halves
 * first, so that a lane stores 8 neighbours: 64 bytes a row and instruction. */
template <int TM, int TN, bool BF16>
__device__ __forceinline__ void store_tile(const GemmArgs& g, const i32x4 (&acc)[TM][TN], int m0, int n0) {
#pragma clang fp contract(off) /* the bias is added to a rounded product */
    const int lane = threadIdx.x & 63, q = lane >> 4;
    f32x4 sw[TN], bv[TN];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int n = min(n0 + 16 * j + 4 * q + r, g.OC - 1);
            sw[j][r] = g.sw[n];
            bv[j][r] = g.bias ? g.bias[n] : -0.0f; /* nothing to add: v + -0 is v for every v */
        }
    float sa[TM];
#pragma unroll
    for (int i = 0; i < TM; i++) sa[i] = g.sa[min(m0 + 16 * i + (lane & 15), g.M - 1)];
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const int m = m0 + 16 * i + (lane & 15);
        const size_t row = (size_t)m * g.ldo;
        f32x4 v[TN];
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) v[j][r] = (float)acc[i][j][r] * sa[i] * sw[j][r] + bv[j][r];
        if (n0 + 16 * TN <= g.OC) {
            if (BF16) {
#pragma unroll
                for (int j = 0; j + 1 < TN; j += 2) {
                    const u32x2 x = __builtin_amdgcn_permlane16_swap(pk(v[j][0], v[j][1]), pk(v[j + 1][0], v[j + 1][1]),
                                                                     false, false);
                    const u32x2 y = __builtin_amdgcn_permlane16_swap(pk(v[j][2], v[j][3]), pk(v[j + 1][2], v[j + 1][3]),
                                                                     false, false);
                    if (m < g.M)
                        store_vec<BF16>(g.out, row + n0 + 16 * (j + (q & 1)) + 8 * (q >> 1), u32x4{x[0], y[0], x[1], y[1]});
                }
                if (TN % 2 && m < g.M)
                    store_vec<BF16>(g.out, row + n0 + 16 * (TN - 1) + 4 * q,
                                    u32x2{pk(v[TN - 1][0], v[TN - 1][1]), pk(v[TN - 1][2], v[TN - 1][3])});
            } else {
#pragma unroll
                for (int j = 0; j < TN; j++)
                    if (m < g.M) store_vec<BF16>(g.out, row + n0 + 16 * j + 4 * q, v[j]);
            }
        } else if (m < g.M) {
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int n = n0 + 16 * j + 4 * q + r;
                    if (n >= g.OC) continue;
                    if (BF16) ((unsigned short*)g.out)[row + n] = __builtin_bit_cast(unsigned short, (__bf16)v[j][r]);
                    else ((float*)g.out)[row + n] = v[j][r];
                }
        }
    }
}

template <int TM, int TN>
__device__ __forceinline__ void clear(i32x4 (&acc)[TM][TN]) {
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[i][j] = i32x4{0, 0, 0, 0};
}

/* ------------------------------------------------------------------ */
/* few rows or outputs */

/* 16 x 16 outputs a workgroup; wave p of KP takes every KP-th slice of 64
 * columns from p on, two slices' loads in flight, so that a workgroup reads 64 KP
 * neighbouring bytes of a row at once.  The partial sums meet in LDS.
 * What bounds it: with many outputs reading the weights (1 x 960 -> 49152 11.0 us, 4.3 TB/s); with few, one workgroup's chain
 * of loads, the join, the scales and the store (us with the weights in the Infinity Cache / from memory: 1 x 960 -> 5120 3.5 /
 * 4.0, 1 x 2560 -> 960 on 60 CUs 3.9 / 5.9, 5 x 8192 -> 500 on 32 8.7 / 12.3; reading back one row of 576 codes, a load and
 * a store, takes 1.5).  Four waves along the sum: one took 5.2 us for 1 x 2560 -> 960, sixteen 4.2, eight 4.5, four 3.8 (in the
 * cache).  Two and four tiles of outputs a wave, and four slices in flight: slower wherever this form is the best (1 x
 * 2560 -> 960 5.3, 7.8 and 4.5 us). */
template <int KP, bool BF16>
__global__ __launch_bounds__(64 * KP) void k_i8_few(GemmArgs g) {
    constexpr int U = 2;
    __shared__ __attribute__((aligned(16))) i32x4 part[KP * 64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int tm, tn;
    if (!tile_of(g, tm, tn)) return;
    const int m0 = tm * 16, n0 = tn * 16;
    const int c = 16 * (lane >> 4), last = 16 * ((g.C - 1) >> 4), slices = (g.C + 63) >> 6;
    const unsigned char* ap = g.a + (size_t)min(m0 + (lane & 15), g.M - 1) * g.lda;
    const unsigned char* wp = g.w + (size_t)min(n0 + (lane & 15), g.OC - 1) * g.ldw;
    i32x4 acc[1][1];
    clear(acc);
    for (int s = wave; s < slices; s += KP * U) {
        i32x4 a[U], w[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = min(64 * (s + KP * u) + c, last);
            w[u] = *(const i32x4*)(wp + k);
            a[u] = *(const i32x4*)(ap + k);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int left = g.C - 64 * (s + KP * u) - c;
            if (left < 16) a[u] = head_bytes(a[u], left);
            acc[0][0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u], a[u], acc[0][0], 0, 0, 0);
        }
    }
    part[wave * 64 + lane] = acc[0][0];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int p = 1; p < KP; p++) acc[0][0] += part[p * 64 + lane];
    store_tile<1, 1, BF16>(g, acc, m0, n0);
}

/* ------------------------------------------------------------------ */
/* LDS stages */

/* Of a row of BK / 16 groups, group c lies at place c ^ group_key(row).  A
 * fragment's read takes, in each of its four passes of 16 lanes, rows r, r + 1,
 * r + 2, r + 3 of two quads at group c and of the other two at c + 1; the keys
 * put these 16 groups in 16 different places of 256 bytes (64 banks). */
template <int BK>
__device__ __forceinline__ int group_key(int row) {
    static_assert(BK == 64 || BK == 128 || BK == 256, "");
    return BK == 64 ? (0x78 >> (2 * ((row >> 2) & 3))) & 3 : BK == 128 ? (row >> 1) & 7 : row & 15;
}

/* keeps memory accesses on their side; no instruction */
__device__ __forceinline__ void fence() { asm volatile("" ::: "memory"); }

/* waits until at most VM of this wave's loads are under way (and, with LDS, none of its LDS accesses) */
template <int VM, bool LDS>
__device__ __forceinline__ void wait_loads() {
    static_assert(VM < 64, "six bits");
    __builtin_amdgcn_s_waitcnt((LDS ? 0x070 : 0xF70) | (VM & 15) | ((VM >> 4) << 14));
}

__device__ __forceinline__ void barrier() {
    fence();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    fence();
}

constexpr int RING = 3; /* stages of a tile's ring */

/* waves on each SIMD: two, of one workgroup, or of two where a CU's 160 KB hold their rings */
constexpr int tile_waves(int waves, int stage_bytes) { return waves >= 8 || RING * stage_bytes <= 80 * 1024 ? 2 : 1; }

/* MW x NW waves of TM x TN 16 x 16 tiles, stages of BK columns, a ring of
 * three: while a stage is multiplied, the first fragments of the next are read
 * and two more are on their way.  A stage's buffer is requested again at the
 * one barrier behind which every wave has read it.
 * What bounds it: a CU's loads into LDS (84 KB/us in 128-byte pieces of rows on
 * 128-byte boundaries, a fifth less off them; 128 x 128 tiles reach 60), with small tiles a
 * stage's chain of load, barrier and fragment reads (0.17 us).  us at
 * 2048 x 2048 x 2048 / 4096 x 2560 x 960 / 1024 x 4096 x 4096, tiles of 128 x 128: eight
 * waves over 128 columns a stage 12.5 / 14.1 / 21; over 64 13.4 / 16.3 / 24; four waves
 * 13.7 / 16 / 24; a ring of two 13.2 / 17.2 / 28, of four over 64 14.3 / 18 / 26. */
template <int MW, int NW, int TM, int TN, int BK, bool BF16>
__global__ __launch_bounds__(64 * MW * NW, tile_waves(MW * NW, 16 * (TM * MW + TN * NW) * BK)) void k_i8_tile(GemmArgs g) {
    constexpr int W = MW * NW, BM = 16 * TM * MW, BN = 16 * TN * NW, SB = (BM + BN) * BK;
    constexpr int CPR = BK / 16, RPI = 1024 / BK, NI = SB / 1024 / W, S = BK / 64;
    static_assert(SB % (1024 * W) == 0 && BM % (RPI * W) == 0, "whole loads, each of one operand");
    __shared__ __attribute__((aligned(16))) unsigned char s0[SB], s1[SB], s2[SB];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int tm, tn;
    if (!tile_of(g, tm, tn)) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int wm = (wave % MW) * 16 * TM, wn = (wave / MW) * 16 * TN;
    const int last16 = 16 * ((g.C - 1) >> 4), stages = (g.C + BK - 1) / BK, last = stages - 1;
    /* this lane's rows and groups of the loads: load i fills 1 KB, RPI rows */
    const unsigned char* rp[NI];
    int ck[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int row = (i * W + wave) * RPI + lane / CPR;
        ck[i] = 16 * ((lane % CPR) ^ group_key<BK>(row));
        rp[i] = i * W * RPI < BM ? g.a + (size_t)min(m0 + row, g.M - 1) * g.lda
                                 : g.w + (size_t)min(n0 + row - BM, g.OC - 1) * g.ldw;
    }
    auto request = [&](int stage, unsigned char* buf) {
#pragma unroll
        for (int i = 0; i < NI; i++)
            __builtin_amdgcn_global_load_lds((const gvoid*)(rp[i] + min(stage * BK + ck[i], last16)),
                                             (lvoid*)(buf + (i * W + wave) * 1024), 16, 0, 0);
    };
    i32x4 acc[TM][TN];
    clear(acc);
    struct Frag {
        i32x4 a[TM], b[TN];
    };
    int fo[S]; /* this lane's place in a fragment of slice s */
#pragma unroll
    for (int s = 0; s < S; s++) fo[s] = (lane & 15) * BK + (((4 * s + (lane >> 4)) ^ group_key<BK>(lane & 15)) << 4);
    auto read = [&](const unsigned char* buf, int s, Frag& f) {
#pragma unroll
        for (int j = 0; j < TN; j++) f.b[j] = *(const i32x4*)(buf + (BM + wn + 16 * j) * BK + fo[s]);
#pragma unroll
        for (int i = 0; i < TM; i++) f.a[i] = *(const i32x4*)(buf + (wm + 16 * i) * BK + fo[s]);
    };
    auto multiply = [&](const Frag& f) {
#pragma unroll
        for (int i = 0; i < TM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.b[j], f.a[i], acc[i][j], 0, 0, 0);
    };
    /* stage `stage` out of buf, its first slice in f already; leaves the next stage's first slice there */
    auto body = [&](int stage, Frag& f, unsigned char* buf, const unsigned char* next) {
        Frag h;
#pragma unroll
        for (int s = 0; s < S; s++) {
            Frag& to = s & 1 ? f : h;
            if (s + 1 < S) {
                read(buf, s + 1, to);
            } else {
                wait_loads<(RING - 2) * NI, true>(); /* the next stage has landed, this one has been read */
                barrier();
                request(stage + RING, buf);
                read(next, 0, to);
            }
            multiply(s & 1 ? h : f);
            /* the reads and requests between the MFMAs, not behind them */
#pragma unroll
            for (int i = 0; i < TM + TN; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, TM * TN > TM + TN ? TM * TN / (TM + TN) : 1, 0); /* MFMA */
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                       /* LDS read */
                if (i % 2 == 0 && i / 2 < NI) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);             /* load */
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (S & 1) f = h;
    };
    Frag f;
    request(0, s0);
    request(1, s1);
    request(2, s2);
    wait_loads<(RING - 1) * NI, false>();
    barrier();
    read(s0, 0, f);
    int stage = 0;
    for (; stage + RING <= last; stage += RING) { /* one way out: a loop left in its middle costs the sums copies */
        body(stage, f, s0, s1);
        body(stage + 1, f, s1, s2);
        body(stage + 2, f, s2, s0);
    }
    const unsigned char* end = s0;
    if (stage < last) {
        body(stage, f, s0, s1);
        end = s1;
    }
    if (stage + 1 < last) {
        body(stage + 1, f, s1, s2);
        end = s2;
    }
#pragma unroll
    for (int s = 0; s < S; s++) {
        if (s) read(end, s, f);
        const int left = g.C - last * BK - 64 * s - 16 * (lane >> 4);
        if (left < 16) {
#pragma unroll
            for (int i = 0; i < TM; i++) f.a[i] = head_bytes(f.a[i], left);
        }
        multiply(f);
    }
    wait_loads<0, true>(); /* nothing may land in the LDS of the workgroup after this one */
    store_tile<TM, TN, BF16>(g, acc, m0 + wm, n0 + wn);
}

/* ------------------------------------------------------------------ */
/* 256 x 256 */

constexpr size_t PAIR_MAX_LD = (size_t)1 << 23; /* 256 rows of it stay inside 32-bit offsets */
/* Five stages (us there / in 128 x 128 tiles: 1356 x 364 x 24934 47.4 / 47.3, 5211 x 452 x 2415 21.7 / 25.4; when it took fewer,
 * 7439 x 113 x 43794 276 / 203, 2279 x 307 x 24615 71 / 63). */
constexpr int PAIR_MIN_C = 320;

/* Eight waves of 128 x 64 (2 x 4), two on each SIMD, in two groups of four a
 * half turn apart: while one group's 16 MFMAs of a half stage run, the other
 * reads the fragments of its next, and a barrier ends each turn.
 * A stage of 64 columns is 32 KB; the ring of five fills the CU's LDS.  Stages 2t
 * and 2t + 1 share the 128-byte lines of their rows, and a CU fetches whole lines
 * (from L2 84 KB/us in 128-byte pieces of rows, 47 in 64-byte ones), so the two are
 * requested line by line, in two halves.
 * What bounds it: on every CU at once, the part's power (4096 x 4096 x 8192 takes 97 us
 * on zeros, 115 on codes of a normal distribution), then the turns (MFMAs alone 96).
 * Against those 115 us: each stage requested by itself 125, the two at once 123;
 * turns without fragments read ahead 132; four waves of 128 x 128 142; the
 * whole workgroup in step and fragments read as they are used 173. */
template <bool BF16>
__global__ __launch_bounds__(512, 2) void k_i8_pair(GemmArgs g) {
    constexpr int W = 8, MW = 2, TM = 8, TN = 4, HM = TM / 2, BM = 256, BN = 256, BK = 64, SB = (BM + BN) * BK;
    constexpr int NI = SB / 1024 / W;
    __shared__ __attribute__((aligned(16))) unsigned char s0[SB], s1[SB], s2[SB], s3[SB], s4[SB];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int tm, tn;
    if (!tile_of(g, tm, tn)) return;
    const int m0 = tm * BM, n0 = tn * BN;
    const int wm = (wave % MW) * 16 * TM, wn = (wave / MW) * 16 * TN;
    const int last16 = 16 * ((g.C - 1) >> 4), stages = (g.C + BK - 1) / BK, last = stages - 1;
    const int group = 16 * ((lane & 3) ^ group_key<BK>(lane >> 2));
    const unsigned char* ab = g.a + (size_t)m0 * g.lda;
    const unsigned char* wb = g.w + (size_t)n0 * g.ldw;
    unsigned int ro[NI]; /* this lane's rows, in bytes from the tile's first */
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int row = (i * W + wave) * 16 + (lane >> 2);
        ro[i] = i * W * 16 < BM ? min(row, g.M - 1 - m0) * (unsigned int)g.lda
                                : min(row - BM, g.OC - 1 - n0) * (unsigned int)g.ldw;
    }
    /* loads i0 .. i0 + NI / 2 - 1 of stages `stage` (even) and stage + 1 */
    auto request = [&](int stage, unsigned char* even, unsigned char* odd, int i0) {
        const unsigned int k0 = min(stage * BK + group, last16), k1 = min(stage * BK + BK + group, last16);
#pragma unroll
        for (int j = 0; j < NI / 2; j++) {
            const int i = i0 + j;
            const unsigned char* p = i * W * 16 < BM ? ab : wb;
            __builtin_amdgcn_global_load_lds((const gvoid*)(p + (ro[i] + k0)), (lvoid*)(even + (i * W + wave) * 1024), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((const gvoid*)(p + (ro[i] + k1)), (lvoid*)(odd + (i * W + wave) * 1024), 16, 0, 0);
        }
    };
    i32x4 acc[TM][TN];
    clear(acc);
    const int fo = (lane & 15) * BK + (((lane >> 4) ^ group_key<BK>(lane & 15)) << 4);
    struct Cols {
        i32x4 v[TN];
    };
    struct Rows {
        i32x4 v[HM];
    };
    Cols b0, b1; /* weights of this stage and the next, in turn */
    Rows a0, a1; /* the wave's upper and lower half of rows */
    auto read_cols = [&](const unsigned char* buf, Cols& b) {
#pragma unroll
        for (int j = 0; j < TN; j++) b.v[j] = *(const i32x4*)(buf + (BM + wn + 16 * j) * BK + fo);
    };
    auto read_rows = [&](const unsigned char* buf, int half, Rows& a) {
#pragma unroll
        for (int i = 0; i < HM; i++) a.v[i] = *(const i32x4*)(buf + (wm + 16 * (i + half * HM)) * BK + fo);
    };
    auto multiply = [&](const Rows& a, const Cols& b, int half) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < HM; i++)
#pragma unroll
            for (int j = 0; j < TN; j++)
                acc[i + half * HM][j] =
                    __builtin_amdgcn_mfma_i32_16x16x64_i8(b.v[j], a.v[i], acc[i + half * HM][j], 0, 0, 0);
        __builtin_amdgcn_s_setprio(0);
    };
    auto turn = [&](const Rows& a, const Cols& b, int half) {
        barrier();
        multiply(a, b, half);
        barrier();
    };
    /* Turns are counted by barriers: the first group reads for a stage's second
     * half in turn 4s and for the first half of stage s + 1 in turn 4s + 2, the
     * other group a turn later.  So stage s + 1 has to have landed for all before turn
     * 4s + 2 (each wave waits for its own part in its first reads of stage s),
     * and stage s has been read by all, the reads waited for, before turn 4s + 5.
     * In two(), s odd, stages s + 3 and s + 4 take the places of s - 2 and s - 1 from turn
     * 4s + 2 on.  Its waits: stage s + 1 has landed when at most the last load, of stage s + 2, is
     * under way; stage s + 2 when only the first half of the next request is. */
    auto two = [&](int s, const unsigned char* x, const unsigned char* y, const unsigned char* next, unsigned char* even,
                   unsigned char* odd) {
        read_rows(x, 1, a1);
        wait_loads<1, false>();
        turn(a0, b1, 0);
        read_cols(y, b0);
        read_rows(y, 0, a0);
        request(s + 3, even, odd, 0);
        turn(a1, b1, 1);
        read_rows(y, 1, a1);
        wait_loads<NI, false>();
        request(s + 3, even, odd, NI / 2);
        turn(a0, b0, 0);
        read_cols(next, b1);
        read_rows(next, 0, a0);
        turn(a1, b0, 1);
    };
    /* a stage without a request; the next one has landed */
    auto one = [&](const unsigned char* x, const unsigned char* next, const Cols& b, Cols& bn) {
        read_rows(x, 1, a1);
        turn(a0, b, 0);
        read_cols(next, bn);
        read_rows(next, 0, a0);
        turn(a1, b, 1);
    };
    request(0, s0, s1, 0);
    request(0, s0, s1, NI / 2);
    request(2, s2, s3, 0);
    request(2, s2, s3, NI / 2);
    wait_loads<2 * NI, false>(); /* stages 0 and 1 */
    barrier();
    read_cols(s0, b0);
    read_rows(s0, 0, a0);
    if (wave >= W / 2) barrier(); /* the half turn */
    one(s0, s1, b0, b1);
    int s = 1;
    for (; s + 10 <= last; s += 10) {
        two(s, s1, s2, s3, s4, s0);
        two(s + 2, s3, s4, s0, s1, s2);
        two(s + 4, s0, s1, s2, s3, s4);
        two(s + 6, s2, s3, s4, s0, s1);
        two(s + 8, s4, s0, s1, s2, s3);
    }
    const int rest = last - s;
    const unsigned char *end = s1, *next = s2;
    if (rest >= 2) {
        two(s, s1, s2, s3, s4, s0);
        end = s3;
        next = s4;
    }
    if (rest >= 4) {
        two(s + 2, s3, s4, s0, s1, s2);
        end = s0;
        next = s1;
    }
    if (rest >= 6) {
        two(s + 4, s0, s1, s2, s3, s4);
        end = s2;
        next = s3;
    }
    if (rest >= 8) {
        two(s + 6, s2, s3, s4, s0, s1);
        end = s4;
        next = s0;
    }
    if (rest & 1) {
        wait_loads<0, false>(); /* ahead of the first reads' barrier: the next stage, for all */
        one(end, next, b1, b0);
        end = next;
    } else {
        b0 = b1;
    }
    read_rows(end, 1, a1);
    const int left = g.C - last * BK - 16 * (lane >> 4);
    if (left < 16) {
#pragma unroll
        for (int i = 0; i < HM; i++) {
            a0.v[i] = head_bytes(a0.v[i], left);
            a1.v[i] = head_bytes(a1.v[i], left);
        }
    }
    multiply(a0, b0, 0);
    multiply(a1, b0, 1);
    if (wave < W / 2) barrier();
    wait_loads<0, true>(); /* nothing may land in the LDS of the workgroup after this one */
    store_tile<TM, TN, BF16>(g, acc, m0 + wm, n0 + wn);
}

/* ------------------------------------------------------------------ */

long tiles(long n, int t) { return (n + t - 1) / t; }

dim3 grid_of(GemmArgs& g, int bm, int bn) {
    g.tiles_m = (int)tiles(g.M, bm);
    g.tiles_n = (int)tiles(g.OC, bn);
    const long n = (long)g.tiles_m * g.tiles_n;
    return n <= MAX_GRID_X ? dim3((unsigned)n) : dim3(MAX_GRID_X, (unsigned)tiles(n, MAX_GRID_X));
}

/* Few outputs, straight from memory (us there / in tiles, eight sets of inputs in turn, which the Infinity Cache holds but for
 * the last two's; then both over enough sets to pass it): a tile
 * of 16 x 16 for each CU at most (17 x 960 x 960 3.0 / 3.4, 4.0 / 4.2; 40 x 5420 x 761 6.0 / 7.9, 7.0 / 10.3; 344 x 1792 x
 * 189, 264 of them, 6.0 / 4.2, 6.6 / 5.4), or three times as many and a short sum (68 x 99 x 1173 2.7 / 2.8, 3.6 / 3.8; 37 x
 * 198 x 2539 2.9 / 2.9, 3.7 / 3.6; 114 x 451 x 1951 3.5 / 3.3, 4.2 / 4.0), or few rows (16 x 960 x 5120 3.7 / 3.9, 4.3 /
 * 4.4; 8 x 1536 x 8192 4.7 / 4.8, 5.6 / 5.6; 8 x 4096 x 6000 8.1 / 6.6, 9.3 / 9.2; 16 x 1536 x 6000 5.1 / 4.5, 5.9 / 5.4) up
 * to where the weights' way into LDS counts (8 x 960 x 49152 12.7 / 12.0, 12.7 / 12.2; but 1 x 960 x 49152 10.9 / 11.2,
 * 11.0 / 11.4). */
bool few_outputs(const GemmArgs& g) {
    const long t32 = tiles(g.M, 32) * tiles(g.OC, 32), t16 = tiles(g.M, 16) * tiles(g.OC, 16);
    if (g.M < 4 || t16 <= CUS) return true;
    return (g.C < 1280 && t32 <= 192) || (g.M <= 16 && t32 < 448 && g.C < (g.M > 8 ? 1280 : 2048));
}

/* The kernels by the outputs of a workgroup and, where there are more than one over them, the waves or the columns of a
 * stage. */
enum Kernel {
    K_FEW_4, K_FEW_8, K_PAIR, K_192, K_256X128, K_128X192, K_128_S64, K_128_S128, K_128X64_S128, K_128X64_S256, K_64_S128,
    K_64_S256, K_32X64_S128, K_32X64_S256, K_32_S128, K_32_S256
};
struct KernelInfo {
    const char* name;
    int bm, bn;
};
constexpr KernelInfo KERNELS[] = {
    {"few 4", 16, 16}, {"few 8", 16, 16}, {"256x256", 256, 256}, {"192x192", 192, 192}, {"256x128", 256, 128},
    {"128x192", 128, 192}, {"128x128 64", 128, 128}, {"128x128 128", 128, 128}, {"128x64 128", 128, 64},
    {"128x64 256", 128, 64}, {"64x64 128", 64, 64}, {"64x64 256", 64, 64}, {"32x64 128", 32, 64}, {"32x64 256", 32, 64},
    {"32x32 128", 32, 32}, {"32x32 256", 32, 32}};

/* Eight waves where the sums are long and many CUs have a workgroup, but no more than one (us in eight / four, inputs in the
 * Infinity Cache: 1 x 8192 x 2048 6.8 / 8.9, 44 x 6711 x 405 6.8 / 7.9; 7 x 5437 x 106 5.2 / 5.1, 52 x 3122 x 565 4.3 / 4.4,
 * 8 x 8192 x 6000 16.5 / 15.3).  With weights from HBM eight are ahead before that (8.3 / 12.4, 8.2 / 10.8; 6.5 / 9.1, 5.3 /
 * 6.7; 1 x 2560 x 960 5.0 / 5.9): the border is the cache's. */
Kernel few_kernel(const GemmArgs& g) {
    const long t16 = tiles(g.M, 16) * tiles(g.OC, 16);
    return t16 >= 48 && t16 <= CUS && g.C >= 3500 ? K_FEW_8 : K_FEW_4;
}

/* The other tiles by their sides, and what the busiest CU has to move: its rounds of tiles times a tile's operands, and
 * four bytes an output for its stores and its start. */
enum { PAIR, T192, T256X128, T128X192, T128, T128X64, T64, T32X64, T32, FORMS };
constexpr int SIDES[FORMS][2] = {{256, 256}, {192, 192}, {256, 128}, {128, 192}, {128, 128},
                                 {128, 64},  {64, 64},   {32, 64},   {32, 32}};
/* The three below 256 x 256 take sums from here on, as their first loads take long (us in 128 x 192 / the best of the
 * others: 944 x 192 x 9055 18.5 / 15.4, though 192 x 192 takes 13.7, 3125 x 403 x 3131 20.2 / 19.1, 2267 x 602 x 2553 13.1 /
 * 14.3). */
constexpr int WIDE_MIN_C = 512;

long cost_of(int form, long rounds, int C) {
    const int bm = SIDES[form][0], bn = SIDES[form][1];
    return rounds * ((long)(bm + bn) * C + 4l * bm * bn);
}

struct Form {
    int form;
    long cost;
};
/* The form that costs least, of equals the largest.  Over 170 shapes with 1.5 million outputs or more and 200 .. 8192
 * columns, what is chosen is 2.3% slower than the best kernel on average, 44% at most (1134 x 338 x 7412 16.7 us, 11.6 in 192 x
 * 192, which starts at WIDE_MIN_C); over 200 shapes of all sizes 2.7%, 47% at most (455 x 894 x 289 5.1 straight from memory,
 * 3.5 in 32 x 32); the largest tile that 150 of are there, over other shapes, 4.2% and 63%.  us (eight sets of inputs in turn; the choice marked):
 *                      256x256  192x192  256x128  128x192  128x128   128x64    64x64    32x64    32x32
 *   4096 x 960 x 4096     22.0*    32.7     30.4     34.8     31.5     35.8     41.9     57.6     71.2
 *   1300 x 960 x 6000     19.3     15.3*    26.4     20.5     21.9     21.7     21.8     28.1     33.7
 *   2048 x 2560 x 4000    31.5     25.2     25.1*    34.4     28.2     31.7     39.1     55.2     68.2
 *   1024 x 960 x 5120     17.7     14.8     12.7     12.4*    14.4     14.3     15.1     19.5     23.2
 *   1024 x 4096 x 4096    40.0     27.3     24.7     23.1     21.6*    24.0     29.5     41.0     50.1
 *   512 x 960 x 5120      17.1     13.7     11.9     10.4      8.4*     9.4      9.6     11.2     12.6
 *   777 x 2500 x 1999     41.0     26.0     25.3     20.6     16.8     11.8*    15.1     19.7     21.3
 *   64 x 960 x 49152      20.6     19.3     26.0     16.1*    19.6     20.8     17.1     20.1     23.6
 *   512 x 2560 x 960      31.3     18.7     17.9     14.9     12.1      9.5      7.3      6.1*     6.7
 *   16384 x 960 x 16      15.4     11.2     11.2      8.7      7.4      6.7      6.1      5.8      5.1* */
Form form_of(const GemmArgs& g, bool pair) {
    Form best = {T32, LONG_MAX};
    for (int i = pair ? PAIR : T192; i < FORMS; i++) {
        if (i >= T192 && i <= T128X192 && g.C < WIDE_MIN_C) continue;
        const long cost = cost_of(i, tiles(tiles(g.M, SIDES[i][0]) * tiles(g.OC, SIDES[i][1]), CUS), g.C);
        if (cost < best.cost) best = {i, cost};
    }
    return best;
}

Kernel kernel_of(const GemmArgs& g, int form) {
    const bool one = tiles(g.M, SIDES[form][0]) * tiles(g.OC, SIDES[form][1]) <= CUS;
    switch (form) {
    case PAIR: return K_PAIR;
    case T192: return K_192;
    case T256X128: return K_256X128;
    case T128X192: return K_128X192;
    /* stages of 64 columns for short sums, which leave a CU room for two tiles (us in 64 / 128: 2048 x 576 x 3000 11.8 /
     * 14.5, 539 x 448 x 10861 13.3 / 15.0; one tile a CU 1586 x 640 x 1292 7.0 / 6.4, 1272 x 448 x 2594 7.1 / 7.4) */
    case T128: return g.C < (one ? 512 : 1024) ? K_128_S64 : K_128_S128;
    /* stages of 256 columns for long sums and one tile a CU at most (us in 128 / 256: 32 x 64 512 x 2560 x 960 7.0 / 6.1, 32 x
     * 32 64 x 4096 x 4096 8.6 / 6.6, 64 x 64 1000 x 8192 x 960 18.2 / 16.4; two tiles a CU 1024 x 2048 x 1500 8.7 / 11.7), 128 x
     * 64 earlier where rows straddle lines (777 x 2500 x 1999 12.7 / 11.8, 2048 x 5000 x 960 21.5 / 19.6; 777 x 1536 x 1984
     * 7.3 / 7.7) */
    case T128X64: return one && g.C >= (g.lda % 128 || g.ldw % 128 ? 1500 : 4096) ? K_128X64_S256 : K_128X64_S128;
    case T64: return one && g.C >= 2048 ? K_64_S256 : K_64_S128;
    case T32X64: return one && g.C >= 1280 ? K_32X64_S256 : K_32X64_S128;
    default: return one && g.C >= 1280 ? K_32_S256 : K_32_S128;
    }
}

template <bool BF16>
void launch_kernel(GemmArgs g, Kernel k, hipStream_t s) {
    const dim3 d = grid_of(g, KERNELS[k].bm, KERNELS[k].bn);
    switch (k) {
    case K_FEW_4: hipLaunchKernelGGL((k_i8_few<4, BF16>), d, dim3(256), 0, s, g); break;
    case K_FEW_8: hipLaunchKernelGGL((k_i8_few<8, BF16>), d, dim3(512), 0, s, g); break;
    case K_PAIR: hipLaunchKernelGGL(k_i8_pair<BF16>, d, dim3(512), 0, s, g); break;
    case K_192: hipLaunchKernelGGL((k_i8_tile<2, 4, 6, 3, 128, BF16>), d, dim3(512), 0, s, g); break;
    case K_256X128: hipLaunchKernelGGL((k_i8_tile<4, 2, 4, 4, 128, BF16>), d, dim3(512), 0, s, g); break;
    case K_128X192: hipLaunchKernelGGL((k_i8_tile<4, 2, 2, 6, 128, BF16>), d, dim3(512), 0, s, g); break;
    case K_128_S64: hipLaunchKernelGGL((k_i8_tile<4, 2, 2, 4, 64, BF16>), d, dim3(512), 0, s, g); break;
    case K_128_S128: hipLaunchKernelGGL((k_i8_tile<4, 2, 2, 4, 128, BF16>), d, dim3(512), 0, s, g); break;
    case K_128X64_S128: hipLaunchKernelGGL((k_i8_tile<4, 2, 2, 2, 128, BF16>), d, dim3(512), 0, s, g); break;
    case K_128X64_S256: hipLaunchKernelGGL((k_i8_tile<4, 2, 2, 2, 256, BF16>), d, dim3(512), 0, s, g); break;
    case K_64_S128: hipLaunchKernelGGL((k_i8_tile<2, 2, 2, 2, 128, BF16>), d, dim3(256), 0, s, g); break;
    case K_64_S256: hipLaunchKernelGGL((k_i8_tile<2, 2, 2, 2, 256, BF16>), d, dim3(256), 0, s, g); break;
    case K_32X64_S128: hipLaunchKernelGGL((k_i8_tile<2, 2, 1, 2, 128, BF16>), d, dim3(256), 0, s, g); break;
    case K_32X64_S256: hipLaunchKernelGGL((k_i8_tile<2, 2, 1, 2, 256, BF16>), d, dim3(256), 0, s, g); break;
    case K_32_S128: hipLaunchKernelGGL((k_i8_tile<2, 2, 1, 1, 128, BF16>), d, dim3(256), 0, s, g); break;
    case K_32_S256: hipLaunchKernelGGL((k_i8_tile<2, 2, 1, 1, 256, BF16>), d, dim3(256), 0, s, g); break;
    }
}

constexpr long LAUNCH_COST = 170000; /* a second launch, 2 us, at the 84 KB/us of a CU's loads into LDS */

struct Part {
    GemmArgs g;
    Kernel kernel;
};
/* The launches of a product.  One whose last round of 256 x 256 tiles is far from full goes in two, the full rounds' rows or
 * columns and what is left in the form that suits it, where that costs less (4096 x 960 x 5120, a round and a
 * quarter: 41.7 -> 35.1 us; 2048 x 4096 x 9000, 1.125: 108 -> 82). */
int parts_of(const GemmArgs& g, size_t out_size, Part (&parts)[2]) {
    parts[0].g = parts[1].g = g;
    if (few_outputs(g)) {
        parts[0].kernel = few_kernel(g);
        return 1;
    }
    const bool pair = g.C >= PAIR_MIN_C && g.lda <= PAIR_MAX_LD && g.ldw <= PAIR_MAX_LD;
    const Form one = form_of(g, pair);
    parts[0].kernel = kernel_of(g, one.form);
    const long tm = tiles(g.M, 256), tn = tiles(g.OC, 256), full = tm * tn / CUS;
    if (!pair || full == 0) return 1;
    long least = one.cost;
    int n_parts = 1;
    for (int columns = 0; columns < 2; columns++) {
        const long n = 256 * (full * CUS / (columns ? tm : tn)); /* rows or columns in the full rounds */
        if (n == 0 || n >= (columns ? g.OC : g.M)) continue;
        GemmArgs first = g, rest = g;
        if (columns) {
            first.OC = (int)n;
            rest.OC -= (int)n;
            rest.w += n * g.ldw;
            rest.sw += n;
            if (rest.bias) rest.bias += n;
            rest.out = (char*)g.out + n * out_size;
        } else {
            first.M = (int)n;
            rest.M -= (int)n;
            rest.a += n * g.lda;
            rest.sa += n;
            rest.out = (char*)g.out + n * g.ldo * out_size;
        }
        const Form f = form_of(rest, false);
        const long cost = cost_of(PAIR, full, g.C) + f.cost + LAUNCH_COST;
        if (cost < least) {
            least = cost;
            parts[0] = {first, K_PAIR};
            parts[1] = {rest, kernel_of(rest, f.form)};
            n_parts = 2;
        }
    }
    return n_parts;
}

/* {codes [BT][lda], scale f32 [BT], weight codes [OC][ldw], scale f32 [OC], bias f32 [OC], out [BT][ldo],
 *  params int{BT, C, OC, has_bias, lda, ldw, ldo}} */
int launch_matmul_i8(const bmk_launch_t* a, bool bf16) {
    BMK_NEED_BYTES(a, 6, 28, "params");
    const int BT = bmk_pi(a, 6, 0), C = bmk_pi(a, 6, 1), OC = bmk_pi(a, 6, 2), lda = bmk_pi(a, 6, 4),
              ldw = bmk_pi(a, 6, 5), ldo = bmk_pi(a, 6, 6);
    const bool bias = bmk_pi(a, 6, 3) != 0;
    BMK_REQUIRE(BT >= 0 && BT <= I8_MAX_DIM && OC > 0 && OC <= I8_MAX_DIM && C > 0 && C <= MAX_C && ldo >= OC,
                "matmul_forward_i8: bad shape BT=%d C=%d (at most %d) OC=%d ldo=%d", BT, C, MAX_C, OC, ldo);
    if (BT == 0) return 0;
    const size_t esz = bf16 ? 2 : 4;
    BMK_NEED_CODES(a, 0, BT, C, lda, "codes");
    BMK_NEED_BYTES(a, 1, (size_t)BT * 4, "scale");
    BMK_NEED_CODES(a, 2, OC, C, ldw, "weight codes");
    BMK_NEED_BYTES(a, 3, (size_t)OC * 4, "weight scale");
    if (bias) BMK_NEED_BYTES(a, 4, (size_t)OC * 4, "bias");
    BMK_NEED_BYTES(a, 5, (((size_t)BT - 1) * (size_t)ldo + (size_t)OC) * esz, "out");
    BMK_REQUIRE((((uintptr_t)a->dev[1] | (uintptr_t)a->dev[3] | (bias ? (uintptr_t)a->dev[4] : 0)) & 3) == 0 &&
                    ((uintptr_t)a->dev[5] & (esz - 1)) == 0,
                "matmul_forward_i8: misaligned scale, bias or out offset");
    GemmArgs g;
    g.a = (const unsigned char*)a->dev[0];
    g.sa = (const float*)a->dev[1];
    g.w = (const unsigned char*)a->dev[2];
    g.sw = (const float*)a->dev[3];
    g.bias = bias ? (const float*)a->dev[4] : nullptr;
    g.out = a->dev[5];
    g.lda = lda;
    g.ldw = ldw;
    g.ldo = ldo;
    g.M = BT;
    g.C = C;
    g.OC = OC;
    Part parts[2];
    const int n = parts_of(g, esz, parts);
    for (int i = 0; i < n; i++) {
        if (bf16) launch_kernel<true>(parts[i].g, parts[i].kernel, a->stream);
        else launch_kernel<false>(parts[i].g, parts[i].kernel, a->stream);
    }
    BMK_LAUNCH_CHECK();
    return 0;
}

} // namespace

extern "C" int bmk_launch_matmul_i8(const bmk_launch_t* a) { return launch_matmul_i8(a, false); }
extern "C" int bmk_launch_matmul_i8_bf16(const bmk_launch_t* a) { return launch_matmul_i8(a, true); }

/* The kernel of a product's launch `part` (from 0) and its rows and columns, or NULL past the last: for tests, so that each
 * can say which kernel it runs. */
extern "C" const char* bmk_matmul_i8_kernel(int BT, int C, int OC, int lda, int ldw, int part, int* rows, int* cols) {
    GemmArgs g = {};
    g.lda = lda;
    g.ldw = ldw;
    g.M = BT;
    g.C = C;
    g.OC = OC;
    Part parts[2];
    if (part < 0 || part >= parts_of(g, 4, parts)) return nullptr;
    *rows = parts[part].g.M;
    *cols = parts[part].g.OC;
    return KERNELS[parts[part].kernel].name;
}
