/* SPDX-License-Identifier: MPL-2.0
 *
 * i8_common.h — what the kernels of the 8-bit integer path share: a row's
 * scale and its codes, and the checks of a matrix of codes.
 *
 * A row p of C values becomes codes q and one scale s (values q * s):
 *   top = max |p|, inv = 127 * (1 / top), q = round-to-even(p * inv), s = top / 127,
 * each step rounded to fp32.  127 / top would be one rounding for inv's two, as numpy and C compute it; torch computes a
 * number over a tensor as this product, and weights quantized there have the same codes here.
 * p * inv is at most 127 * (1 + 2^-21), so q needs no clamp: 1 / top is off by 2^-24, or by 2^-22 where it is subnormal (top
 * over 2^126), and the two products by 2^-24 each.  Two kinds of row
 * have no such grid: one that holds a NaN or an infinity gets zero codes and
 * the scale NaN (so that what is computed from it shows it), one whose top is
 * so small (under 3.73e-37, or all zero) that inv overflows gets zero codes
 * and the scale 0.
 */
#ifndef BMK_I8_COMMON_H
#define BMK_I8_COMMON_H

#include "bmk.h"

namespace bmk {

/* |v| as an integer that orders like it; NaN above infinity above every number, so a maximum keeps them */
__device__ __forceinline__ unsigned int i8_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct I8Grid {
    float inv;  /* 0: every code is 0 */
    float step; /* top / 127, or 0, or NaN */
};
__device__ __forceinline__ I8Grid i8_grid(unsigned int top_bits) {
    I8Grid g;
    const float top = __uint_as_float(top_bits);
    g.inv = 127.0f * (1.0f / top);
    g.step = top / 127.0f;
    if (top_bits >= 0x7f800000u) {
        g.inv = 0.0f;
        g.step = __uint_as_float(0x7fc00000u);
    } else if (!(g.inv <= 3.402823466e38f)) {
        g.inv = g.step = 0.0f;
    }
    return g;
}
__device__ __forceinline__ int i8_code(float p, float inv) {
    return inv == 0.0f ? 0 : (int)rintf(p * inv); /* the first keeps inf * 0 out of a row without a grid */
}

} // namespace bmk

/* Rows and columns a launch takes at most, so that tile and column indexes stay inside an int. */
static constexpr int I8_MAX_DIM = 1 << 30;

/* Columns a row of C codes occupies: whole 16-byte groups. */
static __host__ __device__ inline size_t i8_row_bytes(int C) { return ((size_t)C + 15) & ~(size_t)15; }

/* A matrix of codes in buffer i: rows on 16-byte boundaries ld bytes apart,
 * the last one in whole 16-byte groups too. */
#define BMK_NEED_CODES(a, i, rows, C, ld, what) do { \
    BMK_REQUIRE((ld) % 16 == 0 && (ld) >= (C) && ((uintptr_t)(a)->dev[i] & 15) == 0, \
                "%s: %s rows of %d codes need 16-byte aligned rows of at least as many bytes (row stride %d)", __func__, \
                what, (int)(C), (int)(ld)); \
    BMK_NEED_BYTES(a, i, ((size_t)(rows) - 1) * (size_t)(ld) + i8_row_bytes(C), what); \
} while (0)

#endif
