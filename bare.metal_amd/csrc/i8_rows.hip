/* SPDX-License-Identifier: MPL-2.0
 *
 * i8_rows.hip — rows to 8-bit codes with a scale each (i8_common.h), and back:
 *   quantize_rows_i8    p = src
 *   rmsnorm_forward_i8  h = x + residual (fp32, stored), p = h * weight; the row's factor
 *                       1 / sqrt(mean h^2 + eps) is positive, so it is in the scale alone and one
 *                       pass over the row gives both the maximum and the sum
 *   swiglu_forward_i8   p = gate / (1 + exp(-gate)) * up
 *   dequantize_rows_i8  dst = code * scale
 * Sums of squares are kept in 64 bits.  A workgroup takes a row.
 */
#include "i8_common.h"

namespace {

using namespace bmk;

constexpr int NT = 256;
constexpr int MAX_GRID = 1 << 20; /* workgroups of a launch; each takes every MAX_GRID-th row past that */

template <bool BF16>
__device__ __forceinline__ float load1(const void* p, size_t i) {
    return BF16 ? __uint_as_float((unsigned int)((const unsigned short*)p)[i] << 16) : ((const float*)p)[i];
}

/* fp32 -> bf16 bits, round to nearest even */
__device__ __forceinline__ unsigned short bf16_of(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }

/* x / (1 + exp(-x)) with the exponential of -|x|, which does not overflow */
__device__ __forceinline__ float silu(float x) {
    const float e = expf(-fabsf(x));
    return (x < 0.0f ? x * e : x) / (1.0f + e);
}

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
__global__ __launch_bounds__(NT) void k_rows_i8(RowArgs a) {
    __shared__ unsigned int tops[NT / 64];
    __shared__ double sums[NT / 64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (size_t row = blockIdx.x; row < (size_t)a.rows; row += gridDim.x) {
        unsigned int top = 0;
        double ss = 0.0;
        for (int c = threadIdx.x; c < a.C; c += NT) {
            float h;
            top = max(top, i8_mag(row_value<OP, BF16>(a, row, c, &h)));
            if (OP == OP_NORM) ss += (double)h * h;
        }
        for (int off = 32; off > 0; off >>= 1) {
            top = max(top, (unsigned int)__shfl_xor((int)top, off));
            if (OP == OP_NORM) ss += __shfl_xor(ss, off);
        }
        __syncthreads(); /* the row before has been read */
        if (lane == 0) {
            tops[wave] = top;
            sums[wave] = ss;
        }
        __syncthreads();
        top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
        const I8Grid g = i8_grid(top);
        if (threadIdx.x == 0) {
            if (OP == OP_NORM) {
                ss = (sums[0] + sums[1]) + (sums[2] + sums[3]);
                const double k = 1.0 / sqrt(ss / a.C + (double)a.eps) / 127.0;
                a.s[row] = g.inv == 0.0f ? g.step : (float)(__uint_as_float(top) * k);
            } else {
                a.s[row] = g.step;
            }
        }
        const int end = (int)i8_row_bytes(a.C);
        for (int c = threadIdx.x; c < end; c += NT) {
            float h = 0.0f;
            const float p = c < a.C ? row_value<OP, BF16>(a, row, c, &h) : 0.0f;
            if (OP == OP_NORM && a.y && c < a.C) a.h[row * (size_t)a.C + c] = h;
            a.q[row * a.ldq + c] = (unsigned char)i8_code(p, g.inv);
        }
    }
}

template <bool BF16>
__global__ __launch_bounds__(NT) void k_rows_back(const unsigned char* q, const float* s, void* dst, size_t ldq,
                                                  size_t ldd, int rows, int C) {
    for (size_t row = blockIdx.x; row < (size_t)rows; row += gridDim.x) {
        const float sc = s[row];
        for (int c = threadIdx.x; c < C; c += NT) {
            const float v = (float)(signed char)q[row * ldq + c] * sc;
            if (BF16) ((unsigned short*)dst)[row * ldd + c] = bf16_of(v);
            else ((float*)dst)[row * ldd + c] = v;
        }
    }
}

template <int OP>
int launch_rows(const RowArgs& r, bool bf16, hipStream_t s) {
    const dim3 grid((unsigned)(r.rows < MAX_GRID ? r.rows : MAX_GRID));
    if (bf16) hipLaunchKernelGGL((k_rows_i8<OP, true>), grid, dim3(NT), 0, s, r);
    else hipLaunchKernelGGL((k_rows_i8<OP, false>), grid, dim3(NT), 0, s, r);
    BMK_LAUNCH_CHECK();
    return 0;
}

/* bytes of a row-major matrix of rows ld elements apart */
size_t span(int rows, int C, int ld, size_t esz) { return (((size_t)rows - 1) * (size_t)ld + (size_t)C) * esz; }

/* {src [M][lds], codes, scale f32 [M], params int{M, C, lds, ldq}} */
int launch_quantize_rows(const bmk_launch_t* a, bool bf16) {
    BMK_NEED_BYTES(a, 3, 16, "params");
    const int M = bmk_pi(a, 3, 0), C = bmk_pi(a, 3, 1), lds = bmk_pi(a, 3, 2), ldq = bmk_pi(a, 3, 3);
    BMK_REQUIRE(M >= 0 && M <= I8_MAX_DIM && C > 0 && C <= I8_MAX_DIM && lds >= C, "quantize_rows_i8: bad shape M=%d C=%d lds=%d", M, C, lds);
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
    BMK_REQUIRE(N >= 0 && N <= I8_MAX_DIM && H > 0 && H <= I8_MAX_DIM && ld >= H, "swiglu_forward_i8: bad shape N=%d H=%d ld=%d", N, H, ld);
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
    BMK_REQUIRE(M >= 0 && M <= I8_MAX_DIM && C > 0 && C <= I8_MAX_DIM && ldd >= C, "dequantize_rows_i8: bad shape M=%d C=%d ldd=%d", M, C, ldd);
    if (M == 0) return 0;
    const size_t esz = bf16 ? 2 : 4;
    BMK_NEED_CODES(a, 0, M, C, ldq, "codes");
    BMK_NEED_BYTES(a, 1, (size_t)M * 4, "scale");
    BMK_NEED_BYTES(a, 2, span(M, C, ldd, esz), "dst");
    BMK_REQUIRE(((uintptr_t)a->dev[2] & (esz - 1)) == 0 && ((uintptr_t)a->dev[1] & 3) == 0,
                "dequantize_rows_i8: misaligned scale or dst offset");
    const dim3 grid((unsigned)(M < MAX_GRID ? M : MAX_GRID));
    const unsigned char* q = (const unsigned char*)a->dev[0];
    const float* s = (const float*)a->dev[1];
    if (bf16) hipLaunchKernelGGL(k_rows_back<true>, grid, dim3(NT), 0, a->stream, q, s, a->dev[2], (size_t)ldq, (size_t)ldd, M, C);
    else hipLaunchKernelGGL(k_rows_back<false>, grid, dim3(NT), 0, a->stream, q, s, a->dev[2], (size_t)ldq, (size_t)ldd, M, C);
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
