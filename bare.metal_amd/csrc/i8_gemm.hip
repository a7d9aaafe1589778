/* SPDX-License-Identifier: MPL-2.0
 *
 * i8_gemm.hip — the product of 8-bit codes (matmul_forward_i8, _bf16) on gfx950 int8 MFMA:
 *   out[m][n] = (sum_k a[m][k] * w[n][k]) * sa[m] * sw[n] + bias[n]
 * The sum is exact in 32-bit integers (fewer than 2^17 columns: 2^17 products
 * of at most 2^14 would pass 2^31); it is converted once, multiplied by the
 * row's scale, then by the column's (each rounding to fp32), the bias added, and
 * for bf16 outputs rounded once more.
 */
#include "i8_common.h"

namespace {

using namespace bmk;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int MAX_C = (1 << 17) - 1;

struct GemmArgs {
    const unsigned char* a;
    const float* sa;
    const unsigned char* w;
    const float* sw;
    const float* bias;
    void* out;
    size_t lda, ldw, ldo;
    int M, C, OC, tiles_n;
};

template <bool BF16>
__device__ __forceinline__ void store1(const GemmArgs& g, int m, int n, int acc) {
    float v = (float)acc * g.sa[m] * g.sw[n];
    if (g.bias) v += g.bias[n];
    const size_t at = (size_t)m * g.ldo + n;
    if (BF16) ((unsigned short*)g.out)[at] = __builtin_bit_cast(unsigned short, (__bf16)v);
    else ((float*)g.out)[at] = v;
}

/* the first n bytes (1 .. 15) of a 16-byte group, zeros behind them */
__device__ __forceinline__ i32x4 head_bytes(i32x4 v, int n) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int left = n - 4 * i;
        if (left <= 0) v[i] = 0;
        else if (left < 4) v[i] &= (1 << (8 * left)) - 1;
    }
    return v;
}

constexpr int NT = 256;

/* 64 x 64 outputs a workgroup, four waves of 32 x 32, 64 columns a step through LDS. */
template <bool BF16>
__global__ __launch_bounds__(NT) void k_i8_gemm(GemmArgs g) {
    constexpr int LD = 80; /* LDS row of 64 codes, padded against bank conflicts */
    __shared__ __attribute__((aligned(16))) unsigned char lds[2][64 * LD];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int tm = blockIdx.x / g.tiles_n, tn = blockIdx.x - tm * g.tiles_n;
    const int m0 = tm * 64, n0 = tn * 64, wm = 32 * (wave & 1), wn = 32 * (wave >> 1);
    const int r = t >> 2, c = 16 * (t & 3);
    const unsigned char* ap = g.a + (size_t)min(m0 + r, g.M - 1) * g.lda;
    const unsigned char* wp = g.w + (size_t)min(n0 + r, g.OC - 1) * g.ldw;
    i32x16 acc;
#pragma unroll
    for (int i = 0; i < 16; i++) acc[i] = 0;
    for (int k = 0; k < g.C; k += 64) {
        const int left = g.C - (k + c); /* codes of this thread's group that the row has; past them zeros */
        i32x4 av = {0, 0, 0, 0}, wv = {0, 0, 0, 0};
        if (left > 0) {
            av = *(const i32x4*)(ap + k + c);
            wv = *(const i32x4*)(wp + k + c);
            if (left < 16) av = head_bytes(av, left);
        }
        __syncthreads();
        *(i32x4*)&lds[0][r * LD + c] = av;
        *(i32x4*)&lds[1][r * LD + c] = wv;
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < 64; kk += 32) {
            const int at = (lane & 31) * LD + kk + 16 * (lane >> 5);
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*(const i32x4*)&lds[0][wm * LD + at],
                                                        *(const i32x4*)&lds[1][wn * LD + at], acc, 0, 0, 0);
        }
    }
    const int n = n0 + wn + (lane & 31);
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int m = m0 + wm + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        if (m < g.M && n < g.OC) store1<BF16>(g, m, n, acc[i]);
    }
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
    g.tiles_n = (OC + 63) / 64;
    const size_t tiles = (size_t)((BT + 63) / 64) * (size_t)g.tiles_n;
    BMK_REQUIRE(tiles <= (1u << 24) - 1, "matmul_forward_i8: BT=%d x OC=%d is too large for one launch", BT, OC);
    const dim3 grid((unsigned)tiles);
    if (bf16) hipLaunchKernelGGL(k_i8_gemm<true>, grid, dim3(NT), 0, a->stream, g);
    else hipLaunchKernelGGL(k_i8_gemm<false>, grid, dim3(NT), 0, a->stream, g);
    BMK_LAUNCH_CHECK();
    return 0;
}

} // namespace

extern "C" int bmk_launch_matmul_i8(const bmk_launch_t* a) { return launch_matmul_i8(a, false); }
extern "C" int bmk_launch_matmul_i8_bf16(const bmk_launch_t* a) { return launch_matmul_i8(a, true); }
