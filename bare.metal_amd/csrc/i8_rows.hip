/* SPDX-License-Identifier: MPL-2.0
 *
 * i8_rows.hip — rows to 8-bit codes with a scale each (i8_common.h), and back:
 *   quantize_rows_i8    p = src
 *   rmsnorm_forward_i8  h = x + residual (fp32, stored), p = h * weight; the row's factor
 *                       1 / sqrt(mean h^2 + eps) is positive, so it is in the scale alone and one
 *                       pass over the row gives both the maximum and the sum
 *   swiglu_forward_i8   p = gate / (1 + exp(-gate)) * up
 *   dequantize_rows_i8  dst = code * scale
 * Sums of squares are kept in 64 bits.
 */
#include "i8_common.h"

namespace {

using namespace bmk;

constexpr int MAX_GRID = 1 << 20; /* workgroups of a launch of the forms that take any row */

enum { OP_QUANT, OP_NORM, OP_SWIGLU };

struct RowArgs {
    const void* x; /* src, x or gate */
    const void* y; /* residual (NULL: none) or up */
    const float* w;
    float* h;
    unsigned char* q;
    float* s;
    size_t ldx, ldq;
    int rows, C;
    float eps;
};

template <bool BF16>
__device__ __forceinline__ float load1(const void* p, size_t i) {
    return BF16 ? __uint_as_float((unsigned int)((const unsigned short*)p)[i] << 16) : ((const float*)p)[i];
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

/* Elements a lane takes at once: 16 bytes of the source, or with fp32 operands
 * beside a bf16 source (the norm) 16 bytes of those, so that every access of a
 * wave is one span (eight elements a lane there: 70 us for 8192 x 4096 against 61). */
template <int OP, bool BF16> constexpr int G = BF16 && OP != OP_NORM ? 8 : 4;

/* Loads on an element's boundary.  Rows are read once, so past the caches
 * (nontemporal: 8192 x 4096 fp32 quantized 31.3 -> 28.0 us, SwiGLU of 4096 x 8192 58.6 -> 51.8; the norm's
 * sum written so too: 78.2 -> 69.9). */
typedef u32x4 u32x4_2 __attribute__((aligned(2)));
typedef u32x4 u32x4_4 __attribute__((aligned(4)));
typedef u32x2 u32x2_2 __attribute__((aligned(2)));
typedef f32x4 f32x4_4 __attribute__((aligned(4)));

/* E source elements as they are, in dwords */
template <bool BF16, int E> struct Raw {
    unsigned int u[BF16 ? E / 2 : E];
};
template <bool BF16, int E>
__device__ __forceinline__ Raw<BF16, E> load_raw(const void* p, size_t i) {
    Raw<BF16, E> r;
    if (BF16 && E == 4) {
        const u32x2 v = __builtin_nontemporal_load((const u32x2_2*)((const unsigned short*)p + i));
        __builtin_memcpy(&r, &v, 8);
    } else {
        const u32x4 v = BF16 ? __builtin_nontemporal_load((const u32x4_2*)((const unsigned short*)p + i))
                             : __builtin_nontemporal_load((const u32x4_4*)((const float*)p + i));
        __builtin_memcpy(&r, &v, sizeof r);
    }
    return r;
}
/* element e, as fp32 */
template <bool BF16, int E>
__device__ __forceinline__ float element(const Raw<BF16, E>& v, int e) {
    if (!BF16) return __uint_as_float(v.u[e]);
    return __uint_as_float(e & 1 ? v.u[e >> 1] & 0xffff0000u : v.u[e >> 1] << 16);
}

/* x / (1 + exp(-x)), within 1.6 units in the last place, so that few codes differ from those of other sound fp32 forms
 * (us, with one product for the exponent and the reciprocal for the quotient, within about 3 units, first: 4096 x 8192 bf16
 * 30.0 / 30.0, 8192 x 2560 20.7 / 22.9).  Under -64 within 1.8.
 * -x log2(e) is a product t and what its rounding and that of the constant left out, w: exp(-x) = 2^t (1 + w ln 2).  The quotient
 * is corrected by its remainder.  Under -64, where exp(-x) nears the end of fp32's range and 1 + exp(x) is 1: x exp(x), as
 * (x 2^-64) (2^(64 - t) (1 - w ln 2)), whose last product alone may be a subnormal number, which the instruction does not
 * give; 64 - t is exact. */
__device__ __forceinline__ float silu(float x) {
#pragma clang fp contract(off)
    const float c = -1.44269502f, c_rest = -1.92596299e-8f, ln2 = 0.693147182f;
    const float xe = fminf(x, 128.0f), t = xe * c, w = __builtin_fmaf(xe, c_rest, __builtin_fmaf(xe, c, -t));
    const float p = __builtin_amdgcn_exp2f(t), d = 1.0f + __builtin_fmaf(p, w * ln2, p);
    const float r = __builtin_amdgcn_rcpf(d), q = x * r;
    float y = __builtin_fmaf(__builtin_fmaf(-q, d, x), r, q);
    if (__builtin_expect(__any(x < -64.0f), 0)) { /* a branch of the wave: choosing a lane's value cost 4 us of those 30.0 */
        asm volatile("");
        const float xl = fmaxf(x, -256.0f), tl = xl * c, wl = __builtin_fmaf(xl, c_rest, __builtin_fmaf(xl, c, -tl));
        const float e = __builtin_amdgcn_exp2f(64.0f - tl);
        y = x < -64.0f ? x * 0x1p-64f * __builtin_fmaf(e, -wl * ln2, e) : y;
    }
    return y;
}

/* four codes of products p * inv: adding 1.5 * 2^23 rounds to a whole number, to even, which lies in the low byte */
__device__ __forceinline__ unsigned int pack4(const float* p, float inv) {
#pragma clang fp contract(off)
    unsigned int u[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float t = p[i] * inv;
        u[i] = __float_as_uint(t + 12582912.0f);
    }
    const unsigned int lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
    return lo | hi;
}

/* Maximum and sum over L = 16 or 64 neighbouring lanes (all of them get it): row rotations inside 16, then swaps. */
template <int CTRL>
__device__ __forceinline__ unsigned int dpp(unsigned int v) {
    return (unsigned int)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
template <int L, class F>
__device__ __forceinline__ unsigned int lanes_fold(unsigned int v, F f) {
    v = f(v, dpp<0x128>(v)); /* row_ror 8, 4, 2, 1 */
    v = f(v, dpp<0x124>(v));
    v = f(v, dpp<0x122>(v));
    v = f(v, dpp<0x121>(v));
    if (L >= 64) {
        u32x2 s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = f(s[0], s[1]);
        s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f(s[0], s[1]);
    }
    return v;
}
template <int L>
__device__ __forceinline__ unsigned int lanes_max(unsigned int v) {
    return lanes_fold<L>(v, [](unsigned int a, unsigned int b) { return max(a, b); });
}
__device__ __forceinline__ double dbl(unsigned int lo, unsigned int hi) {
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    return v + dbl(dpp<CTRL>((unsigned int)b), dpp<CTRL>((unsigned int)(b >> 32)));
}
template <int L>
__device__ __forceinline__ double lanes_sum(double v) {
    v = dpp_add<0x128>(v);
    v = dpp_add<0x124>(v);
    v = dpp_add<0x122>(v);
    v = dpp_add<0x121>(v);
    if (L >= 64) {
        unsigned long long b = __builtin_bit_cast(unsigned long long, v);
        u32x2 lo = __builtin_amdgcn_permlane16_swap((unsigned int)b, (unsigned int)b, false, false);
        u32x2 hi = __builtin_amdgcn_permlane16_swap((unsigned int)(b >> 32), (unsigned int)(b >> 32), false, false);
        v = dbl(lo[0], hi[0]) + dbl(lo[1], hi[1]);
        b = __builtin_bit_cast(unsigned long long, v);
        lo = __builtin_amdgcn_permlane32_swap((unsigned int)b, (unsigned int)b, false, false);
        hi = __builtin_amdgcn_permlane32_swap((unsigned int)(b >> 32), (unsigned int)(b >> 32), false, false);
        v = dbl(lo[0], hi[0]) + dbl(lo[1], hi[1]);
    }
    return v;
}

/* the norm's scale: top * rstd / 127, rounded once */
__device__ __forceinline__ float norm_scale(unsigned int top, double ss, int C, float eps) {
    return (float)((double)__uint_as_float(top) / (127.0 * sqrt(ss / C + (double)eps)));
}

/* Rows of up to LPR * NV * G columns: LPR lanes a row (16: four rows a wave;
 * 64: a wave; more: a workgroup), which read it once, 16 bytes a lane and load, all
 * loads before the first use, and keep it in registers until the codes are
 * written.  A workgroup takes several rows in turn where there are more than
 * the launch has workgroups, and keeps the norm's weights.
 * What bounds it: HBM, with many rows (TB/s of what is read and written: 49152 x
 * 960 6.0, and 5.4 with its codes' reading back between, 8192 x 4096 norm 6.3, 4096 x 8192 bf16 SwiGLU 5.6, where its
 * arithmetic is close behind; a 1 GiB copy reaches 5.1); with few, the chain of load,
 * reduction and store (the norm of one row of 576 2.3 us, 333 of 960 bf16 4.2). */
template <int OP, bool BF16, int LPR, int NV>
__global__ __launch_bounds__(LPR < 64 ? 64 : LPR) void k_rows_i8(RowArgs a) {
    constexpr int E = G<OP, BF16>, NT = LPR < 64 ? 64 : LPR, RPW = NT / LPR, WAVES = NT / 64;
    __shared__ unsigned int tops[2][WAVES];
    __shared__ double sums[2][WAVES];
    const int l = threadIdx.x % LPR, wave = threadIdx.x >> 6, C = a.C;
    const int end = (int)i8_row_bytes(C), ragged = C % E, clamp = max(C - E, 0);
    f32x4 w[NV];
    if (OP == OP_NORM && C >= E) {
#pragma unroll
        for (int v = 0; v < NV; v++) w[v] = *(const f32x4_4*)(a.w + min((v * LPR + l) * E, clamp));
    }
    int turn = 0;
    for (size_t row = (size_t)blockIdx.x * RPW + threadIdx.x / LPR; row < (size_t)a.rows; row += (size_t)gridDim.x * RPW) {
        float p[NV][E];
        unsigned int top = 0;
        double ss = 0.0;
        const size_t at = row * a.ldx, hat = row * (size_t)C;
        if (C >= E) {
            Raw<BF16, E> x[NV], y[NV];
            f32x4 r[NV];
#pragma unroll
            for (int v = 0; v < NV; v++) { /* groups past the row read its last one and count as zeros */
                const int c = min((v * LPR + l) * E, clamp);
                x[v] = load_raw<BF16, E>(a.x, at + c);
                if (OP == OP_SWIGLU) y[v] = load_raw<BF16, E>(a.y, at + c);
                if (OP == OP_NORM && a.y) r[v] = __builtin_nontemporal_load((const f32x4_4*)((const float*)a.y + hat + c));
            }
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int c = (v * LPR + l) * E;
                const bool in = v < NV - 1 || c + E <= C; /* all but the last group of a lane lie inside (launch_form) */
                f32x4 h;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float xe = element<BF16, E>(x[v], e);
                    float pe = xe;
                    if (OP == OP_SWIGLU) pe = silu(xe) * element<BF16, E>(y[v], e);
                    if (OP == OP_NORM) {
                        const float he = a.y ? xe + r[v][e & 3] : xe;
                        h[e & 3] = he;
                        pe = he * w[v][e & 3];
                        if (in) ss += (double)he * he;
                    }
                    p[v][e] = in ? pe : 0.0f;
                    top = max(top, i8_mag(p[v][e]));
                }
                if (OP == OP_NORM && a.y && in) __builtin_nontemporal_store(h, (f32x4_4*)(a.h + hat + c));
            }
        } else {
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int e = 0; e < E; e++) p[v][e] = 0.0f;
        }
        if (ragged) { /* the last group, element by element */
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int c = (v * LPR + l) * E;
                if (c >= C || c + E <= C) continue;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    if (c + e >= C) continue;
                    const float xe = load1<BF16>(a.x, at + c + e);
                    float pe = xe;
                    if (OP == OP_SWIGLU) pe = silu(xe) * load1<BF16>(a.y, at + c + e);
                    if (OP == OP_NORM) {
                        const float he = a.y ? xe + ((const float*)a.y)[hat + c + e] : xe;
                        if (a.y) a.h[hat + c + e] = he;
                        ss += (double)he * he;
                        pe = he * a.w[c + e];
                    }
                    p[v][e] = pe;
                    top = max(top, i8_mag(pe));
                }
            }
        }
        top = lanes_max<(LPR < 64 ? LPR : 64)>(top);
        if (OP == OP_NORM) ss = lanes_sum<(LPR < 64 ? LPR : 64)>(ss);
        if (WAVES > 1) { /* two places in turn: one barrier a row */
            if ((threadIdx.x & 63) == 0) {
                tops[turn][wave] = top;
                sums[turn][wave] = ss;
            }
            __syncthreads();
            top = tops[turn][0];
#pragma unroll
            for (int i = 1; i < WAVES; i++) top = max(top, tops[turn][i]);
            if (OP == OP_NORM) {
                ss = sums[turn][0];
#pragma unroll
                for (int i = 1; i < WAVES; i++) ss += sums[turn][i];
            }
            turn ^= 1;
        }
        const I8Grid g = i8_grid(top);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = (v * LPR + l) * E;
            if (c >= end) continue;
            unsigned int* q = (unsigned int*)(a.q + row * a.ldq + c);
            const unsigned int q0 = g.inv == 0.0f ? 0u : pack4(p[v], g.inv);
            if (E == 8) *(u32x2*)q = u32x2{q0, g.inv == 0.0f ? 0u : pack4(p[v] + E - 4, g.inv)};
            else *q = q0;
        }
        if (l == 0) a.s[row] = OP == OP_NORM && g.inv != 0.0f ? norm_scale(top, ss, C, a.eps) : g.step;
    }
}

/* Rows of any length, read twice, an element a lane and load.  TB/s of what has to be read and written: norm of 2048 x 16384
 * 3.0 (144 us), fp32 SwiGLU of 2048 x 28672 2.3 (233), 2048 x 40000 quantized 2.5 (165). */
template <int OP, bool BF16>
__device__ __forceinline__ float row_value(const RowArgs& a, size_t row, int c, float* h) {
    const float x = load1<BF16>(a.x, row * a.ldx + c);
    if (OP == OP_NORM) {
        *h = a.y ? x + ((const float*)a.y)[row * (size_t)a.C + c] : x;
        return *h * a.w[c];
    }
    if (OP == OP_SWIGLU) return silu(x) * load1<BF16>(a.y, row * a.ldx + c);
    return x;
}

template <int OP, bool BF16>
__global__ __launch_bounds__(1024) void k_rows_i8_long(RowArgs a) {
    constexpr int NT = 1024;
    __shared__ unsigned int tops[NT / 64];
    __shared__ double sums[NT / 64];
    const int wave = threadIdx.x >> 6;
    for (size_t row = blockIdx.x; row < (size_t)a.rows; row += gridDim.x) {
        unsigned int top = 0;
        double ss = 0.0;
        for (int c = threadIdx.x; c < a.C; c += NT) {
            float h;
            top = max(top, i8_mag(row_value<OP, BF16>(a, row, c, &h)));
            if (OP == OP_NORM) ss += (double)h * h;
        }
        top = lanes_max<64>(top);
        if (OP == OP_NORM) ss = lanes_sum<64>(ss);
        __syncthreads(); /* the row before has been read */
        if ((threadIdx.x & 63) == 0) {
            tops[wave] = top;
            sums[wave] = ss;
        }
        __syncthreads();
        top = 0;
        ss = 0.0;
        for (int i = 0; i < NT / 64; i++) {
            top = max(top, tops[i]);
            if (OP == OP_NORM) ss += sums[i];
        }
        const I8Grid g = i8_grid(top);
        if (threadIdx.x == 0) a.s[row] = OP == OP_NORM && g.inv != 0.0f ? norm_scale(top, ss, a.C, a.eps) : g.step;
        const int end = (int)i8_row_bytes(a.C);
        for (int c = threadIdx.x; c < end; c += NT) {
            float h = 0.0f;
            const float p = c < a.C ? row_value<OP, BF16>(a, row, c, &h) : 0.0f;
            if (OP == OP_NORM && a.y && c < a.C) a.h[row * (size_t)a.C + c] = h;
            a.q[row * a.ldq + c] = (unsigned char)i8_code(p, g.inv);
        }
    }
}

/* code * scale: LPR lanes a row, 8 (to bf16) or 4 codes a lane and step, so that a lane stores 16 bytes.  HBM-bound: 49152 x
 * 960 to bf16 21.7 us (6.5 TB/s) with the codes from the Infinity Cache, where they were just written, 28.0 (5.1) with them
 * from memory, to fp32 48.6 (4.9); 8192 x 4096 15.4, 20.1 and 33.5. */
template <bool BF16, int LPR>
__global__ __launch_bounds__(256) void k_rows_back(const unsigned char* q, const float* s, void* dst, size_t ldq,
                                                   size_t ldd, int rows, int C) {
    constexpr int E = BF16 ? 8 : 4, RPB = 256 / LPR;
    const int l = threadIdx.x % LPR;
    for (size_t row = (size_t)blockIdx.x * RPB + threadIdx.x / LPR; row < (size_t)rows; row += (size_t)gridDim.x * RPB) {
        const float sc = s[row];
        const unsigned char* qr = q + row * ldq;
        for (int c = l * E; c < C; c += LPR * E) {
            unsigned int u[2];
            __builtin_memcpy(u, __builtin_assume_aligned(qr + c, E), E); /* whole 16-byte groups are there */
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = (float)(signed char)(u[e >> 2] >> (8 * (e & 3))) * sc;
            if (c + E <= C) {
                u32x4 o;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    o[i] = BF16 ? __builtin_bit_cast(unsigned int, __builtin_convertvector(
                                                                       f32x2{v[(2 * i) % E], v[(2 * i + 1) % E]}, bf16x2))
                                : __float_as_uint(v[i]);
                if (BF16) __builtin_memcpy(__builtin_assume_aligned((unsigned short*)dst + row * ldd + c, 2), &o, 16);
                else __builtin_memcpy(__builtin_assume_aligned((float*)dst + row * ldd + c, 4), &o, 16);
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    if (c + e >= C) continue;
                    if (BF16) ((unsigned short*)dst)[row * ldd + c + e] = __builtin_bit_cast(unsigned short, (__bf16)v[e]);
                    else ((float*)dst)[row * ldd + c + e] = v[e];
                }
            }
        }
    }
}

/* A workgroup a row where that is one to eight waves (49152 x 960 43.5 -> 41.8 us, 4096 x 8192 SwiGLU 54.0 -> 51.8);
 * the shortest rows and the longest take what the CUs hold, in turns (1000000 x 64 66.6 -> 58.0, 2048 x 16384 35.9 -> 33.1). */
template <int OP, bool BF16, int LPR, int NV>
void go(const RowArgs& r, hipStream_t s) {
    constexpr int NT = LPR < 64 ? 64 : LPR, RPW = NT / LPR;
    constexpr long most = LPR >= 64 && LPR <= 512 ? MAX_GRID : 256 * 32 * 64 / NT;
    const long wgs = ((long)r.rows + RPW - 1) / RPW;
    hipLaunchKernelGGL((k_rows_i8<OP, BF16, LPR, NV>), dim3((unsigned)(wgs < most ? wgs : most)), dim3(NT), 0, s, r);
}

/* Past 2048 groups: sixteen waves a row, or, for the norm, whose operands do not fit their registers, the form that reads
 * twice. */
template <int OP, bool BF16>
void launch_wide(const RowArgs& r, int groups, hipStream_t s) {
    if constexpr (OP != OP_NORM) {
        if (groups <= 3 * 1024) return go<OP, BF16, 1024, 3>(r, s);
        if (groups <= 4 * 1024) return go<OP, BF16, 1024, 4>(r, s);
    }
    hipLaunchKernelGGL((k_rows_i8_long<OP, BF16>), dim3((unsigned)(r.rows < MAX_GRID ? r.rows : MAX_GRID)), dim3(1024), 0, s,
                       r);
}

/* Lanes a row and groups a lane, the fewest lanes that hold the row (8192 x 2560
 * bf16 SwiGLU, 320 groups: 27.2 us with two on each of 256 lanes, 22.9 with three on 128; 46427 x
 * 192 quantized, 48 groups: 14.0 with one on each of 64, 9.0 with three on 16; 65536 x 256 19.5 / 15.1, but the
 * norm of 32768 x 256, with three operands a group, 19.0 / 20.0).
 * NV is the smallest that does, so all but a lane's last group lie inside the row. */
template <int OP, bool BF16>
void launch_form(const RowArgs& r, hipStream_t s) {
    const int groups = (int)(i8_row_bytes(r.C) / G<OP, BF16>); /* the zeros behind a row's codes among them */
    if (groups <= 16) go<OP, BF16, 16, 1>(r, s);
    else if (groups <= 32) go<OP, BF16, 16, 2>(r, s);
    else if (groups <= 48) go<OP, BF16, 16, 3>(r, s);
    else if (groups <= 64) go<OP, BF16, OP == OP_QUANT ? 16 : 64, OP == OP_QUANT ? 4 : 1>(r, s);
    else if (groups <= 128) go<OP, BF16, 64, 2>(r, s);
    else if (groups <= 192) go<OP, BF16, 64, 3>(r, s);
    else if (groups <= 256) go<OP, BF16, 64, 4>(r, s);
    else if (groups <= 384) go<OP, BF16, 128, 3>(r, s);
    else if (groups <= 512) go<OP, BF16, 128, 4>(r, s);
    else if (groups <= 768) go<OP, BF16, 256, 3>(r, s);
    else if (groups <= 1024) go<OP, BF16, 256, 4>(r, s);
    else if (groups <= 1536) go<OP, BF16, 512, 3>(r, s);
    else if (groups <= 2048) go<OP, BF16, 512, 4>(r, s);
    else launch_wide<OP, BF16>(r, groups, s);
}

template <int OP>
int launch_rows(const RowArgs& r, bool bf16, hipStream_t s) {
    if (bf16) launch_form<OP, true>(r, s);
    else launch_form<OP, false>(r, s);
    BMK_LAUNCH_CHECK();
    return 0;
}

template <bool BF16>
void launch_back(const bmk_launch_t* a, int M, int C, int ldq, int ldd) {
    const unsigned char* q = (const unsigned char*)a->dev[0];
    const float* s = (const float*)a->dev[1];
    constexpr int E = BF16 ? 8 : 4;
    const int groups = (C + E - 1) / E;
    auto grid = [&](int rpb) {
        const long n = ((long)M + rpb - 1) / rpb;
        return dim3((unsigned)(n < MAX_GRID ? n : MAX_GRID));
    };
    void* dst = a->dev[2];
    const size_t lq = ldq, ld = ldd;
    if (groups <= 32)
        hipLaunchKernelGGL((k_rows_back<BF16, 16>), grid(16), dim3(256), 0, a->stream, q, s, dst, lq, ld, M, C);
    else if (groups <= 256)
        hipLaunchKernelGGL((k_rows_back<BF16, 64>), grid(4), dim3(256), 0, a->stream, q, s, dst, lq, ld, M, C);
    else
        hipLaunchKernelGGL((k_rows_back<BF16, 256>), grid(1), dim3(256), 0, a->stream, q, s, dst, lq, ld, M, C);
}

/* bytes of a row-major matrix of rows ld elements apart */
size_t span(int rows, int C, int ld, size_t esz) { return (((size_t)rows - 1) * (size_t)ld + (size_t)C) * esz; }

/* {src [M][lds], codes, scale f32 [M], params int{M, C, lds, ldq}} */
int launch_quantize_rows(const bmk_launch_t* a, bool bf16) {
    BMK_NEED_BYTES(a, 3, 16, "params");
    const int M = bmk_pi(a, 3, 0), C = bmk_pi(a, 3, 1), lds = bmk_pi(a, 3, 2), ldq = bmk_pi(a, 3, 3);
    BMK_REQUIRE(M >= 0 && M <= I8_MAX_DIM && C > 0 && C <= I8_MAX_DIM && lds >= C,
                "quantize_rows_i8: bad shape M=%d C=%d lds=%d", M, C, lds);
    if (M == 0) return 0;
    const size_t esz = bf16 ? 2 : 4;
    BMK_NEED_BYTES(a, 0, span(M, C, lds, esz), "src");
    BMK_NEED_CODES(a, 1, M, C, ldq, "codes");
    BMK_NEED_BYTES(a, 2, (size_t)M * 4, "scale");
    BMK_REQUIRE(((uintptr_t)a->dev[0] & (esz - 1)) == 0 && ((uintptr_t)a->dev[2] & 3) == 0,
                "quantize_rows_i8: misaligned src or scale offset");
    RowArgs r = {};
    r.x = a->dev[0];
    r.q = (unsigned char*)a->dev[1];
    r.s = (float*)a->dev[2];
    r.ldx = lds;
    r.ldq = ldq;
    r.rows = M;
    r.C = C;
    return launch_rows<OP_QUANT>(r, bf16, a->stream);
}

/* {x [N][C], residual f32 [N][C], weight f32 [C], sum f32 [N][C], codes, scale f32 [N],
 *  params int{N, C, ldq, has_residual}, eps float} */
int launch_rmsnorm_i8(const bmk_launch_t* a, bool bf16) {
    BMK_NEED_BYTES(a, 6, 16, "params");
    BMK_NEED_BYTES(a, 7, 4, "eps");
    const int N = bmk_pi(a, 6, 0), C = bmk_pi(a, 6, 1), ldq = bmk_pi(a, 6, 2);
    const bool res = bmk_pi(a, 6, 3) != 0;
    BMK_REQUIRE(N >= 0 && N <= I8_MAX_DIM && C > 0 && C <= I8_MAX_DIM, "rmsnorm_forward_i8: bad shape N=%d C=%d", N, C);
    if (N == 0) return 0;
    const size_t esz = bf16 ? 2 : 4, n = (size_t)N * (size_t)C;
    BMK_NEED_BYTES(a, 0, n * esz, "x");
    BMK_NEED_BYTES(a, 2, (size_t)C * 4, "weight");
    if (res) {
        BMK_NEED_BYTES(a, 1, n * 4, "residual");
        BMK_NEED_BYTES(a, 3, n * 4, "sum");
        BMK_REQUIRE((((uintptr_t)a->dev[1] | (uintptr_t)a->dev[3]) & 3) == 0,
                    "rmsnorm_forward_i8: misaligned residual or sum offset");
    }
    BMK_NEED_CODES(a, 4, N, C, ldq, "codes");
    BMK_NEED_BYTES(a, 5, (size_t)N * 4, "scale");
    BMK_REQUIRE(((uintptr_t)a->dev[0] & (esz - 1)) == 0 && (((uintptr_t)a->dev[2] | (uintptr_t)a->dev[5]) & 3) == 0,
                "rmsnorm_forward_i8: misaligned x, weight or scale offset");
    RowArgs r = {};
    r.x = a->dev[0];
    r.y = res ? a->dev[1] : nullptr;
    r.w = (const float*)a->dev[2];
    r.h = (float*)a->dev[3];
    r.q = (unsigned char*)a->dev[4];
    r.s = (float*)a->dev[5];
    r.ldx = C;
    r.ldq = ldq;
    r.rows = N;
    r.C = C;
    r.eps = bmk_pf(a, 7, 0);
    return launch_rows<OP_NORM>(r, bf16, a->stream);
}

/* {gate [N][ld], up [N][ld], codes, scale f32 [N], params int{N, H, ld, ldq}} */
int launch_swiglu_i8(const bmk_launch_t* a, bool bf16) {
    BMK_NEED_BYTES(a, 4, 16, "params");
    const int N = bmk_pi(a, 4, 0), H = bmk_pi(a, 4, 1), ld = bmk_pi(a, 4, 2), ldq = bmk_pi(a, 4, 3);
    BMK_REQUIRE(N >= 0 && N <= I8_MAX_DIM && H > 0 && H <= I8_MAX_DIM && ld >= H,
                "swiglu_forward_i8: bad shape N=%d H=%d ld=%d", N, H, ld);
    if (N == 0) return 0;
    const size_t esz = bf16 ? 2 : 4;
    BMK_NEED_BYTES(a, 0, span(N, H, ld, esz), "gate");
    BMK_NEED_BYTES(a, 1, span(N, H, ld, esz), "up");
    BMK_NEED_CODES(a, 2, N, H, ldq, "codes");
    BMK_NEED_BYTES(a, 3, (size_t)N * 4, "scale");
    BMK_REQUIRE((((uintptr_t)a->dev[0] | (uintptr_t)a->dev[1]) & (esz - 1)) == 0 && ((uintptr_t)a->dev[3] & 3) == 0,
                "swiglu_forward_i8: misaligned gate, up or scale offset");
    RowArgs r = {};
    r.x = a->dev[0];
    r.y = a->dev[1];
    r.q = (unsigned char*)a->dev[2];
    r.s = (float*)a->dev[3];
    r.ldx = ld;
    r.ldq = ldq;
    r.rows = N;
    r.C = H;
    return launch_rows<OP_SWIGLU>(r, bf16, a->stream);
}

/* {codes, scale f32 [M], dst [M][ldd], params int{M, C, ldq, ldd}} */
int launch_dequantize_rows(const bmk_launch_t* a, bool bf16) {
    BMK_NEED_BYTES(a, 3, 16, "params");
    const int M = bmk_pi(a, 3, 0), C = bmk_pi(a, 3, 1), ldq = bmk_pi(a, 3, 2), ldd = bmk_pi(a, 3, 3);
    BMK_REQUIRE(M >= 0 && M <= I8_MAX_DIM && C > 0 && C <= I8_MAX_DIM && ldd >= C,
                "dequantize_rows_i8: bad shape M=%d C=%d ldd=%d", M, C, ldd);
    if (M == 0) return 0;
    const size_t esz = bf16 ? 2 : 4;
    BMK_NEED_CODES(a, 0, M, C, ldq, "codes");
    BMK_NEED_BYTES(a, 1, (size_t)M * 4, "scale");
    BMK_NEED_BYTES(a, 2, span(M, C, ldd, esz), "dst");
    BMK_REQUIRE(((uintptr_t)a->dev[2] & (esz - 1)) == 0 && ((uintptr_t)a->dev[1] & 3) == 0,
                "dequantize_rows_i8: misaligned scale or dst offset");
    if (bf16) launch_back<true>(a, M, C, ldq, ldd);
    else launch_back<false>(a, M, C, ldq, ldd);
    BMK_LAUNCH_CHECK();
    return 0;
}

} // namespace

extern "C" int bmk_launch_quantize_rows_i8(const bmk_launch_t* a) { return launch_quantize_rows(a, false); }
extern "C" int bmk_launch_quantize_rows_i8_bf16(const bmk_launch_t* a) { return launch_quantize_rows(a, true); }
extern "C" int bmk_launch_dequantize_rows_i8(const bmk_launch_t* a) { return launch_dequantize_rows(a, false); }
extern "C" int bmk_launch_dequantize_rows_i8_bf16(const bmk_launch_t* a) { return launch_dequantize_rows(a, true); }
extern "C" int bmk_launch_rmsnorm_i8(const bmk_launch_t* a) { return launch_rmsnorm_i8(a, false); }
extern "C" int bmk_launch_rmsnorm_i8_bf16(const bmk_launch_t* a) { return launch_rmsnorm_i8(a, true); }
extern "C" int bmk_launch_swiglu_i8(const bmk_launch_t* a) { return launch_swiglu_i8(a, false); }
extern "C" int bmk_launch_swiglu_i8_bf16(const bmk_launch_t* a) { return launch_swiglu_i8(a, true); }
