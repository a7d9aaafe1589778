/* SPDX-License-Identifier: MPL-2.0
 *
 * bm_paged.h — serving several sequences from a cache in pages: MI355X
 * additions beside the reference's one-sequence kernels rope_forward,
 * kv_store and attention_forward (backend.h), which have no batch, no pages
 * and fp32 alone (reference src/baremetal/scheduler.c:835-947).
 *
 * Named kernels, bound like any other through backend_encode_dispatch (the
 * grid and threadgroup sizes are not looked at).  A _bf16 name takes and
 * gives bf16 where "T" stands, the plain name f32; sums and norms are held in
 * fp32 or more and results rounded once (what attention_forward_paged rounds
 * besides stands with it).  Rows of a matrix lie ld elements apart, on an
 * element's boundary; a row holds its heads one after another, HD elements
 * each (HD even and at most 256; a multiple of 8 where there is a cache).
 * Row counts may be 0 (nothing is done).  Outputs may not overlap inputs but
 * where stated.
 *
 * The cache: T [n_pages][2][NKV][page][HD], keys then values, on a 16-byte
 * boundary; page a power of two from 8 to 65536, max_pages * page at most 2^30,
 * n_pages * page at most 2^38, NKV at most 4096.
 * A layer's cache goes in by its buffer's offset.
 * The batch: S sequences, at most 4096; start int32 [S + 1], not falling: the new tokens
 * of sequence s are rows start[s] .. start[s + 1] - 1 of N; len int32 [S]:
 * its keys, the new tokens' own included; pages int32 [S][max_pages]: the
 * pages of its keys in order.  Row i of a sequence with n new tokens stands
 * at position len - n + i.  All three are read on the device; a sequence may
 * have no new tokens, rows outside start[0] .. start[S] - 1 are left as they
 * are, entries of pages past a sequence's keys are not read.  Nothing is read or written
 * outside the buffers whatever the tables hold: a key whose page lies outside 0 .. n_pages - 1 or past the table counts as
 * missing (see the kernels).  Two sequences may share pages that neither appends to.
 *
 * Rotation: pair i of a head's first rot elements (rot even, at most HD), elements i and
 * i + rot/2 (layout 0, halves) or 2i and 2i + 1 (layout 1, neighbours), is
 * turned at position p by a = 2 pi (p * turns[i] mod 2^64) / 2^64 and
 * multiplied by mscale: (x0, x1) -> mscale (x0 cos a - x1 sin a, x0 sin a + x1
 * cos a).  turns u64 [rot/2] on an 8-byte boundary comes from bm_rope_turns; the product's fraction of a
 * turn is kept to 2^-32 (and the table's rounding, 2^-64 a position) at any position, where rope_forward's
 * fp32 product loses the fraction of far ones (so the two differ by up to about p * 2^-24 in the
 * angle).  cos and sin of it are fp32's, within 2 x 2^-24.  Elements from rot on pass unturned.  rot 0: no rotation (bind any
 * buffer as turns).
 *
 *   "rope_forward_rows", "rope_forward_rows_bf16"
 *                        {x T [N][ldx], out T [N][ldo], pos int32 [N], turns,
 *                         params int{N, NH, HD, rot, layout, ldx, ldo}, f32{mscale}}: every head
 *                         of row n turned at pos[n] (which may be negative); out may be x's own
 *                         buffer with ldo = ldx
 *   "qk_norm_rope_forward", "qk_norm_rope_forward_bf16"
 *                        {q T [N][ldq], k T [N][ldk], q out T [N][ldqo], k out T [N][ldko],
 *                         pos int32 [N], turns, gain f32 [2][HD],
 *                         params int{N, NH, NKV, HD, rot, layout, ldq, ldk, ldqo, ldko},
 *                         f32{mscale, eps}}: each head x as x / sqrt(mean x^2 + eps) * gain (gain[0]
 *                         for q, gain[1] for k), then turned; an output may be its input's own
 *                         buffer with the same stride
 *   "kv_append_paged", "kv_append_paged_bf16"
 *                        {q T [N][ldq], k T [N][ldk], v T [N][ldv], q out T [N][ldqo], cache, start,
 *                         len, pages, turns, gain f32 [2][HD], params int{N, S, NH, NKV, HD, rot,
 *                         layout, ldq, ldk, ldv, ldqo, page, n_pages, max_pages, norm},
 *                         f32{mscale, eps}}: q turned at its row's position to q out (which may be
 *                         q's own buffer with the same stride), k turned and v as it is into the
 *                         cache there; norm 1: q and k through the norm first (norm 0: bind any as
 *                         gain).  NH 0: no q (bind any).  A row before position 0 or on a missing
 *                         page is not written to the cache
 *   "attention_forward_paged", "attention_forward_paged_bf16"
 *                        {q T [N][ldq], cache, out T [N][ldo], start, len, pages,
 *                         params int{N, S, NH, NKV, HD, ldq, ldo, page, n_pages, max_pages, causal,
 *                         window}, f32{scale}}: softmax(scale * q . K) V, head h over KV head
 *                         h / (NH / NKV).  causal 1: a row at position p sees the keys up to p,
 *                         with window w > 0 the last w of them; causal 0 (window 0): all len keys.
 *                         A row that sees no key gets zeros; one that sees a missing key gets NaN.
 *                         What masked keys, values and the rest of a page hold does not matter,
 *                         infinities and NaN included; a value that a row sees and that is not
 *                         finite makes that element of the row not finite, a key its whole row
 *                         (but in bf16 a key whose score is -infinity has weight 0).
 *                         Roundings: scores and sums are fp32.  f32: operands of the products as
 *                         three terms of bf16, six products of nine, which leaves out at most 2^-22 of a
 *                         product; multiples of 2^-133 remain of an element.  bf16: of a sequence with up to 32 rows
 *                         for a KV head (new tokens x query heads) the weights keep 2^-17 of each, with
 *                         more they are rounded to bf16 (of long random sums, 2.1e-3 from the exact result in the mean
 *                         square in place of 1.7e-3).  Finite for scores up to 2^125 with values up to 2^56
 */
#ifndef BM_PAGED_H
#define BM_PAGED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* How bm_rope_turns scales the frequencies f_i = theta^(-2i/rot), radians a
 * position, of a context longer than the model's first one of `original`
 * positions:
 *   NONE    f_i
 *   LLAMA3  waves of more than original / low positions f_i / factor, of less than original / high
 *           f_i, between them (1 - t) f_i / factor + t f_i, t = (original f_i / 2 pi - low) / (high - low)
 *           (as bm_arch_t's BM_ROPE_LLAMA3)
 *   LINEAR  f_i / factor
 *   YARN    (1 - t) f_i + t f_i / factor, t rising from 0 to 1 over the pairs from a to b, those that make
 *           high and low turns over the original context, pair(x) = rot ln(original / (2 pi x)) / (2 ln theta):
 *           a = max(floor(pair(high)), 0), b = min(ceil(pair(low)), rot - 1), t = (i - a) / max(b - a, 0.001)
 *           clamped; mscale = 0.1 ln(factor) + 1
 * mscale is 1 but for YARN. */
enum { BM_TURNS_NONE = 0, BM_TURNS_LLAMA3 = 1, BM_TURNS_LINEAR = 2, BM_TURNS_YARN = 3 };

/* Fills turns[rot / 2] with f_i / 2 pi as fractions of 2^64 (whole turns a
 * position drop out), and *mscale.  0, or -1 for a rot that is odd or
 * negative, a theta that is not over 1, or with scaling a factor under 1,
 * an original not over 0 or high not over low > 0. */
int bm_rope_turns(int rot, int scaling, double theta, double factor, double low, double high, double original,
                  uint64_t* turns, float* mscale);

#ifdef __cplusplus
}
#endif

#endif /* BM_PAGED_H */
