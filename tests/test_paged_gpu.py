# SPDX-License-Identifier: MPL-2.0
"""Serving from a paged cache (include/bm_paged.h) through the backend's C ABI against the formulas in 64 bits.

Tolerances count roundings: U32 = 2^-24 and UB16 = 2^-8, half a step relative to the value."""
import ctypes

import numpy as np
import pytest

import bmhip
from paged_exactness import deviation, last_bits, last_bits_off

pytestmark = pytest.mark.gpu
U32, UB16 = 2.0 ** -24, 2.0 ** -8
MARK = 0x5A  # what lies in buffers where nothing may be written
THETA = 500000.0
SCALED = dict(factor=8.0, low=1.0, high=4.0, original=8192.0)


def to_bf16(x):
    """fp32 -> bf16 bits, round to nearest even; NaN stays one."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Kind:
    """f32 or bf16 values: how they lie in memory, and half a step of theirs."""

    def __init__(self, bf16):
        self.bf16, self.suffix, self.size = bf16, "_bf16" if bf16 else "", 2 if bf16 else 4
        self.memory, self.step = (np.uint16, UB16) if bf16 else (np.float32, 0.0)

    def held(self, x):
        """The values that memory holds of x."""
        return from_bf16(to_bf16(x)) if self.bf16 else np.ascontiguousarray(x, np.float32)

    def raw(self, x):
        return to_bf16(x) if self.bf16 else np.ascontiguousarray(x, np.float32)

    def values(self, raw):
        return from_bf16(raw) if self.bf16 else raw


KINDS = [Kind(False), Kind(True)]
both = pytest.mark.parametrize("kind", KINDS, ids=["f32", "bf16"])


def strided(kind, x, ld, lead):
    """Rows of x, ld elements apart, behind `lead` elements, the mark between and behind them."""
    out = np.zeros(lead + len(x) * ld + 3, kind.memory)
    out.view(np.uint8)[:] = MARK
    for r in range(len(x)):
        out[lead + r * ld:lead + r * ld + x.shape[1]] = kind.raw(x[r])
    return out


def rows_of(kind, buf, n, width, ld, lead, written=None):
    """The rows' values; everything outside them (and the rows that are not written) still holds the mark."""
    raw = buf.read(kind.memory).copy()
    out = np.stack([raw[lead + r * ld:lead + r * ld + width] for r in range(n)]) if n else np.zeros((0, width), kind.memory)
    for r in range(n):
        if written is None or written[r]:
            raw[lead + r * ld:lead + r * ld + width].view(np.uint8)[:] = MARK
    assert (raw.view(np.uint8) == MARK).all()
    return kind.values(out)


def marked(be, nbytes):
    return be.upload(np.full((nbytes + 3) // 4 * 4, MARK, np.uint8))


def floats(be, *v):
    return be.upload(np.float32(v))


# ---------------------------------------------------------------- the rotation

def turn_table(rot, scaling):
    return bmhip.rope_turns(rot, THETA, scaling, **SCALED)


def turned(x, pos, rot, layout, table, mscale):
    """x [n][heads][HD] in 64 bits, turned, and what the fp32 steps may be off: the angle of the table's turns is exact
    in integers.  cos and sin are off by 3 units of 2^-24 (the angle's two roundings at up to pi/4, their own one, the
    series' end), mscale, product and sum round once each: 6 (|x0| + |x1|) mscale."""
    x = x.astype(np.float64)
    y, off = x.copy(), np.zeros_like(x)
    h = rot // 2
    a = np.array([[(int(p) * int(t) % (1 << 64)) / 2.0 ** 64 for t in table[:h]] for p in pos]).reshape(len(pos), 1, h) * 2 * np.pi
    c, s = np.cos(a) * mscale, np.sin(a) * mscale
    i0, i1 = (np.arange(h), np.arange(h) + h) if layout == 0 else (2 * np.arange(h), 2 * np.arange(h) + 1)
    x0, x1 = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    off[..., i0] = off[..., i1] = 6 * U32 * (np.abs(x0) + np.abs(x1)) * abs(mscale)
    return y, off


def normed(x, gain, eps):
    """RMSNorm of heads in 64 bits.  The kernels round the factor 1 / sqrt, its product with the element and that with the gain
    to fp32: three roundings, beside the sum's and the root's far smaller ones (64 bits)."""
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)


def check(kind, got, want, off):
    """Within off (of the fp32 steps) and the result's rounding."""
    bad = ~(np.abs(got - want) <= off * 1.001 + kind.step * (np.abs(want) + off) + 1e-37)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


def positions(rng, n, far):
    p = rng.integers(-far, far, n).astype(np.int32)
    p[:1] = 0
    p[1:3] = [(1 << 31) - 1, -(1 << 31)][:max(0, n - 1)]
    return p


ROPE = [  # rows, heads, head size, rot
    (1, 1, 2, 2), (2, 3, 6, 4), (1, 12, 64, 64), (5, 2, 64, 0), (3, 5, 64, 32), (7, 3, 80, 40), (4, 2, 96, 96), (9, 4, 80, 20),
    (6, 3, 128, 64), (2, 40, 128, 128), (33, 2, 256, 256), (5, 1, 256, 64), (3, 2, 254, 252), (130, 9, 16, 8), (1, 1, 256, 2),
    (4, 3, 72, 24), (4, 3, 88, 88)]


@both
@pytest.mark.parametrize("layout", [0, 1], ids=["halves", "pairs"])
@pytest.mark.parametrize("N,NH,HD,rot", ROPE)
def test_rope_rows(be, N, NH, HD, rot, layout, kind):
    rng = np.random.default_rng(N * 1009 + NH * 101 + HD + rot)
    W = NH * HD
    x = kind.held(rng.standard_normal((N, W)) * np.exp(rng.uniform(-3, 3, (N, 1))))
    pos = positions(rng, N, 1 << 20)
    for scaling, ldx, ldo, lead in (("none", W, W, 0), ("yarn", W + 1, W + 3, 1), ("llama3", W + 8, W + 16, 8),
                                    ("linear", W + 4, W + 2, 4)):
        table, m = turn_table(rot, scaling)
        want, off = turned(x.reshape(N, NH, HD), pos, rot, layout, table, m)
        src, out = be.upload(strided(kind, x, ldx, lead)), marked(be, (lead + N * ldo + 3) * kind.size)
        shift = [lead * kind.size, lead * kind.size, 0, 0, 0, 0]
        assert be.dispatch("rope_forward_rows" + kind.suffix, [
            src, out, be.upload(pos), be.upload(table), be.params(N, NH, HD, rot, layout, ldx, ldo), floats(be, m)], (N,),
            (256,), offsets=shift) == 0
        got = rows_of(kind, out, N, W, ldo, lead)
        check(kind, got, want.reshape(N, W), off.reshape(N, W))
        # in place: the same bits
        assert be.dispatch("rope_forward_rows" + kind.suffix, [
            src, src, be.upload(pos), be.upload(table), be.params(N, NH, HD, rot, layout, ldx, ldx), floats(be, m)], (N,),
            (256,), offsets=shift) == 0
        assert np.array_equal(rows_of(kind, src, N, W, ldx, lead).view(np.uint32), got.view(np.uint32))


@both
@pytest.mark.parametrize("layout", [0, 1], ids=["halves", "pairs"])
@pytest.mark.parametrize("N,NH,HD,rot", [(3, 5000, 2, 2), (2, 3000, 64, 32)])
def test_rope_rows_of_many_heads(be, N, NH, HD, rot, layout, kind):
    """Rows that several workgroups share."""
    test_rope_rows(be, N, NH, HD, rot, layout, kind)


@both
@pytest.mark.parametrize("layout", [0, 1], ids=["halves", "pairs"])
def test_rows_past_the_cache_have_the_same_bits(be, layout, kind):
    """A call of more than 128 MB, which reads past the caches, against its rows in calls of fewer; in place as well."""
    NH, NKV, HD, rot = 4, 2, 128, 128
    N = (150 << 20) // ((NH + NKV) * HD * kind.size)
    rng = np.random.default_rng(8)
    block = kind.raw(rng.standard_normal((1 << 16) + 7).astype(np.float32))
    q, k = np.resize(block, (N, NH * HD)), np.resize(block[::-1], (N, NKV * HD))
    pos = (np.arange(N) % 50000).astype(np.int32)
    table, m = turn_table(rot, "none")
    gain = rng.standard_normal((2, HD)).astype(np.float32)
    src, out = [be.upload(q), be.upload(k)], [marked(be, q.nbytes), marked(be, k.nbytes)]
    rest = [be.upload(pos), be.upload(table), be.upload(gain)]

    def run(src, out, first, n):
        shift = [first * NH * HD * kind.size, first * NKV * HD * kind.size] * 2 + [first * 4, 0, 0, 0, 0]
        assert be.dispatch("qk_norm_rope_forward" + kind.suffix, src + out + rest + [
            be.params(n, NH, NKV, HD, rot, layout, NH * HD, NKV * HD, NH * HD, NKV * HD), floats(be, m, 1e-5)], (n,), (256,),
            offsets=shift) == 0

    for first in range(0, N, 30000):
        run(src, out, first, min(30000, N - first))
    want = [x.read(np.uint8) for x in out]
    out = [marked(be, q.nbytes), marked(be, k.nbytes)]
    run(src, out, 0, N)
    run(src, src, 0, N)
    for x in (out, src):
        assert all(np.array_equal(a.read(np.uint8), w) for a, w in zip(x, want))


@both
def test_rope_leaves_the_rest_of_a_head(be, kind):
    """Elements from rot on come through bit for bit, infinities and NaN too, and do not touch the turned ones."""
    N, NH, HD, rot = 3, 4, 64, 32
    rng = np.random.default_rng(1)
    x = kind.held(rng.standard_normal((N, NH, HD)))
    x[..., rot:] = np.float32([np.inf, np.nan, -np.inf, -0.0])[rng.integers(0, 4, (N, NH, HD - rot))]
    table, m = turn_table(rot, "none")
    for layout in (0, 1):
        out = marked(be, N * NH * HD * kind.size)
        assert be.dispatch("rope_forward_rows" + kind.suffix, [
            be.upload(kind.raw(x)), out, be.upload(np.int32([0, 5, 1 << 20])), be.upload(table),
            be.params(N, NH, HD, rot, layout, NH * HD, NH * HD), floats(be, m)], (N,), (256,)) == 0
        got = kind.values(out.read(kind.memory, N * NH * HD)).reshape(N, NH, HD)
        assert np.array_equal(got[..., rot:], x[..., rot:], equal_nan=True) and np.isfinite(got[..., :rot]).all()
        assert np.array_equal(got[0], x[0], equal_nan=True)  # position 0: no turn


def test_cos_and_sin_of_any_turn(be):
    """A million fractions of a turn, the quarters' borders among them: x = (1, 0) comes out as (cos, sin), within 2 units of 2^-24 and
    the 2^-32 of a turn that the fraction is kept to."""
    N, HD = 8192, 256
    rng = np.random.default_rng(52)
    table = rng.integers(0, 1 << 64, HD // 2, dtype=np.uint64)
    table[:16] = [(k << 61) + d & ((1 << 64) - 1) for k in range(8) for d in (0, -1)]
    pos = rng.integers(-(1 << 31), 1 << 31, N).astype(np.int32)
    pos[:4] = [0, 1, -1, 3]
    x = np.zeros((N, HD), np.float32)
    x[:, :HD // 2] = 1
    out = marked(be, x.nbytes)
    assert be.dispatch("rope_forward_rows", [be.upload(x), out, be.upload(pos), be.upload(table), be.params(N, 1, HD, HD, 0, HD, HD),
                                             floats(be, 1.0)], (N,), (256,)) == 0
    got = out.read(np.float32).reshape(N, 2, HD // 2).astype(np.float64)
    with np.errstate(over="ignore"):
        turn = pos.astype(np.int64).view(np.uint64)[:, None] * table
    a = turn.astype(np.float64) * (2 * np.pi / 2.0 ** 64)
    off = 2 * U32 + 2 * np.pi * 2.0 ** -32 + 1e-15
    assert np.abs(got[:, 0] - np.cos(a)).max() <= off and np.abs(got[:, 1] - np.sin(a)).max() <= off


def test_rope_of_more_work_items_than_an_axis_takes(be):
    """Heads of 256 at odd strides take 64 lanes each: 2^26 heads and more are over 2^32 work-items.  34 GB, in place, zeros but
    for a few rows, which the kernel itself (rot 0) puts there and takes back."""
    kind, NH, HD, rot = KINDS[1], 1024, 256, 64
    W = NH * HD
    ld, N = W + 1, (1 << 16) + 9  # heads of row 2^16 on lie past the axis
    rng = np.random.default_rng(44)
    rows = [0, 1, 40000, (1 << 16) - 1, 1 << 16, (1 << 16) + 1, N - 1]
    x = kind.held(rng.standard_normal((len(rows), W)))
    pos = positions(rng, N, 1 << 20)
    table, m = turn_table(rot, "yarn")
    big, turns, one, factor = be.alloc(N * ld * kind.size), be.upload(table), be.upload(np.int32([0])), floats(be, m)
    try:
        for r, v in zip(rows, x):
            assert be.dispatch("rope_forward_rows_bf16", [be.upload(kind.raw(v)), big, one, turns, be.params(1, NH, HD, 0, 0, W, W),
                                                          factor], (1,), (256,), offsets=[0, r * ld * kind.size, 0, 0, 0, 0]) == 0
        assert be.dispatch("rope_forward_rows_bf16", [big, big, be.upload(pos), turns, be.params(N, NH, HD, rot, 0, ld, ld),
                                                      factor], (N,), (256,)) == 0
        want, off = turned(x.reshape(len(rows), NH, HD), pos[rows], rot, 0, table, m)
        for r, w, o in zip(rows + [2, 50000, (1 << 16) + 5], list(want) + [np.zeros((NH, HD))] * 3, list(off) + [0.0] * 3):
            out = marked(be, W * kind.size)
            assert be.dispatch("rope_forward_rows_bf16", [big, out, one, turns, be.params(1, NH, HD, 0, 0, W, W), factor], (1,),
                               (256,), offsets=[r * ld * kind.size, 0, 0, 0, 0, 0]) == 0
            check(kind, kind.values(out.read(kind.memory)).reshape(NH, HD), w, o)
    finally:
        big.free()


def test_rope_keeps_lengths_and_distances(be):
    """Closed forms: a turn keeps a pair's length, and a dot product depends on the positions' difference alone."""
    NH, HD = 2, 64
    rng = np.random.default_rng(2)
    x = rng.standard_normal((1, NH * HD)).astype(np.float32)
    pos = np.int32([0, 7, 1000, 1007, 1 << 20, (1 << 20) + 7, (1 << 30), (1 << 30) + 7])
    rows = np.repeat(x, len(pos), 0)
    table, m = turn_table(HD, "none")
    out = marked(be, rows.nbytes)
    assert be.dispatch("rope_forward_rows", [be.upload(rows), out, be.upload(pos), be.upload(table),
                                             be.params(len(pos), NH, HD, HD, 0, NH * HD, NH * HD), floats(be, m)],
                       (8,), (256,)) == 0
    y = out.read(np.float32).reshape(len(pos), NH, HD).astype(np.float64)
    length = np.hypot(y[..., :HD // 2], y[..., HD // 2:])
    x = x.reshape(NH, HD).astype(np.float64)
    assert np.abs(length - np.hypot(x[:, :HD // 2], x[:, HD // 2:])).max() <= 12 * U32 * np.abs(x).max() * 2
    dots = np.einsum("phd,phd->ph", y[0::2], y[1::2])
    # each product of two elements is off by 12 U32 of the pair's magnitudes
    assert np.abs(dots - dots[0]).max() <= 2 * 12 * U32 * 2 * (x * x).sum(-1).max() * 2


@both
@pytest.mark.parametrize("layout", [0, 1], ids=["halves", "pairs"])
@pytest.mark.parametrize("N,NH,NKV,HD,rot", [(1, 1, 1, 2, 2), (1, 9, 3, 64, 64), (5, 4, 1, 64, 32), (3, 15, 5, 64, 64),
                                             (7, 3, 3, 80, 40), (2, 32, 8, 128, 128), (4, 2, 1, 256, 128), (66, 2, 1, 96, 0),
                                             (3, 2, 2, 254, 250), (2, 2, 5, 72, 72)])
def test_qk_norm_rope(be, N, NH, NKV, HD, rot, layout, kind):
    rng = np.random.default_rng(N * 1009 + NH * 101 + HD + rot)
    Q, K, eps = NH * HD, NKV * HD, 1e-5
    q, k = (kind.held(rng.standard_normal((N, w)) * np.exp(rng.uniform(-3, 3, (N, 1)))) for w in (Q, K))
    gain = (1 + 0.3 * rng.standard_normal((2, HD))).astype(np.float32)
    pos = positions(rng, N, 1 << 17)
    table, m = turn_table(rot, "yarn")
    for ldq, ldk, ldqo, ldko, lead in ((Q, K, Q, K, 0), (Q + 1, K + 2, Q + 3, K + 1, 1), (Q + K, Q + K, Q + 8, K + 8, 8)):
        bq, bk = be.upload(strided(kind, q, ldq, lead)), be.upload(strided(kind, k, ldk, lead))
        oq, ok = marked(be, (lead + N * ldqo + 3) * kind.size), marked(be, (lead + N * ldko + 3) * kind.size)
        sh = lead * kind.size

        def call(a, b, c, d, lc, ld):
            return be.dispatch("qk_norm_rope_forward" + kind.suffix, [
                a, b, c, d, be.upload(pos), be.upload(table), be.upload(gain),
                be.params(N, NH, NKV, HD, rot, layout, ldq, ldk, lc, ld), floats(be, m, eps)], (N,), (256,),
                offsets=[sh] * 4 + [0] * 5)

        assert call(bq, bk, oq, ok, ldqo, ldko) == 0
        first = []
        for x, buf, ld, g in ((q, oq, ldqo, gain[0]), (k, ok, ldko, gain[1])):
            y = normed(x.reshape(N, -1, HD), g, np.float64(np.float32(eps)))
            want, off = turned(y, pos, rot, layout, table, m)
            # the norm's three roundings of each element, carried through the turn
            carried = turned_sum(np.abs(y), rot, layout, abs(m)) * 3 * U32
            got = rows_of(kind, buf, N, x.shape[1], ld, lead)
            check(kind, got, want.reshape(got.shape), (off + carried).reshape(got.shape))
            first.append(got)
        assert call(bq, bk, bq, bk, ldq, ldk) == 0  # in place: the same bits
        for x, buf, ld, got in ((q, bq, ldq, first[0]), (k, bk, ldk, first[1])):
            assert np.array_equal(rows_of(kind, buf, N, x.shape[1], ld, lead).view(np.uint32), got.view(np.uint32))


def turned_sum(y, rot, layout, m):
    """|x0| + |x1| of each element's pair, times m; the element itself where nothing turns."""
    out, h = y.copy(), rot // 2
    i0, i1 = (np.arange(h), np.arange(h) + h) if layout == 0 else (2 * np.arange(h), 2 * np.arange(h) + 1)
    out[..., i0] = out[..., i1] = (y[..., i0] + y[..., i1]) * m
    return out


def test_qk_norm_of_extreme_heads(be):
    """Heads of zeros, of values whose squares leave fp32 on either side, and NaN or infinities in one head alone."""
    HD, NH = 64, 6
    rng = np.random.default_rng(3)
    x = rng.standard_normal((NH, HD)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e30)
    x[2] *= np.float32(1e-30)
    x[3, 5], x[4, 60] = np.nan, np.inf
    x[5] *= np.float32(1e38 / np.abs(x[5]).max())  # a factor below fp32's normal numbers
    gain, one = np.ones((2, HD), np.float32), be.upload(np.int32([0]))
    for eps in (1e-5, 0.0):
        oq, ok = marked(be, x.nbytes), marked(be, x.nbytes)
        assert be.dispatch("qk_norm_rope_forward", [
            be.upload(x), be.upload(x), oq, ok, one, one, be.upload(gain),
            be.params(1, NH, NH, HD, 0, 0, NH * HD, NH * HD, NH * HD, NH * HD), floats(be, 1.0, eps)], (1,), (256,)) == 0
        got = oq.read(np.float32).reshape(NH, HD)
        assert np.array_equal(got, ok.read(np.float32).reshape(NH, HD), equal_nan=True)
        rows = [1, 5] + ([2] if eps == 0 else [])
        want = normed(x[rows], gain[0], np.float64(np.float32(eps)))
        assert (np.abs(got[rows] - want) <= 3.01 * U32 * np.abs(want)).all()
        assert (got[0] == 0).all() if eps else np.isnan(got[0]).all()  # 0 / sqrt(0)
        assert np.isnan(got[3]).all() and np.isnan(got[4, 60]) and (got[4, :60] == 0).all()


@both
@pytest.mark.parametrize("HD,off0", [(64, 0), (6, 0), (64, 1)], ids=["wide", "narrow", "odd"])
def test_qk_norm_of_the_smallest_heads(be, HD, off0, kind):
    """Heads under 2^-128, down to the type's least number, whose factor 1 / sqrt(mean x^2) is past fp32: with eps 0 (or one as
    small) they come out like any others, beside heads that are ordinary."""
    size = [1.0, 2.0 ** -100, 2.0 ** -126, 2.0 ** -128, 2.0 ** -131, 2.0 ** -140, 0.0, 2.0 ** 40]
    NH = len(size)
    rng = np.random.default_rng(41)
    x = kind.held(rng.standard_normal((NH, HD)) * np.array(size)[:, None])
    x[6, 1] = 2.0 ** (-133 if kind.bf16 else -149)  # the least number alone
    x[5, 0] = x[6, 1]  # no head of zeros, which has no norm
    gain = (1 + 0.3 * rng.standard_normal((2, HD))).astype(np.float32)
    one = be.upload(np.int32([0]))
    for eps in (0.0, 2.0 ** -149):
        src = be.upload(strided(kind, x.reshape(1, -1), NH * HD, off0))
        out = [marked(be, (off0 + NH * HD + 3) * kind.size) for _ in range(2)]
        assert be.dispatch("qk_norm_rope_forward" + kind.suffix, [
            src, src] + out + [one, one, be.upload(gain), be.params(1, NH, NH, HD, 0, 0, *[NH * HD] * 4),
                               floats(be, 1.0, eps)], (1,), (256,), offsets=[off0 * kind.size] * 4 + [0] * 5) == 0
        for buf, g in zip(out, gain):
            want = normed(x, g, np.float64(np.float32(eps)))
            got = rows_of(kind, buf, 1, NH * HD, NH * HD, off0).reshape(NH, HD)
            check(kind, got, want, 3 * U32 * np.abs(want))


# ---------------------------------------------------------------- the cache

class Batch:
    """Sequences of `new` tokens behind cached ones, total keys each, in pages dealt out at random; `lead` rows before
    the first sequence and `tail` behind the last are no one's."""

    def __init__(self, be, rng, kind, new, total, page, NKV, HD, lead=0, tail=0, spare=2, fill=np.nan):
        self.new, self.total, self.page, self.NKV, self.HD, self.kind = list(new), list(total), page, NKV, HD, kind
        self.S = len(new)
        need = [(t + page - 1) // page for t in total]
        self.width, self.count = max(max(need), 1) + 1, sum(need) + spare
        order = rng.permutation(self.count).astype(np.int32)
        self.pages = rng.choice(np.int32([-1, self.count, 1 << 30, -(1 << 31)]), (self.S, self.width)).astype(np.int32)
        at = 0
        for s in range(self.S):  # entries past a sequence's keys are never read: they hold anything
            self.pages[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
        self.start = np.int32([lead + sum(self.new[:s]) for s in range(self.S + 1)])
        self.len = np.int32(total)
        self.N = int(self.start[-1]) + tail
        self.seq = np.full(self.N, -1)
        self.pos = np.zeros(self.N, np.int64)
        for s in range(self.S):
            for i in range(self.new[s]):
                self.seq[self.start[s] + i], self.pos[self.start[s] + i] = s, total[s] - self.new[s] + i
        self.cache = np.full((self.count, 2, NKV, page, HD), fill, np.float32)

    def place(self, s, j):
        return self.pages[s, j // self.page], j % self.page

    def fill(self, rng, sharp=1.0):
        """Keys and values of every sequence; returned as [S] lists of [NKV][total][HD]."""
        self.K, self.V = [], []
        for s in range(self.S):
            k, v = (self.kind.held(rng.standard_normal((self.NKV, self.total[s], self.HD)) * g) for g in (sharp, 1.0))
            self.set(s, k, v)
            self.K.append(k)
            self.V.append(v)

    def set(self, s, k, v):
        for j in range(k.shape[1]):
            pg, at = self.place(s, j)
            self.cache[pg, 0, :, at], self.cache[pg, 1, :, at] = k[:, j], v[:, j]

    def tables(self, be):
        return [be.upload(self.start), be.upload(self.len), be.upload(self.pages)]


BATCHES = [  # new tokens, total keys, page, lead, tail
    ([1], [1], 16, 0, 0),
    ([1], [17], 16, 0, 1),
    ([3], [3], 8, 0, 0),
    ([1, 1, 1], [5, 16, 33], 16, 0, 0),
    ([5, 0, 1, 9], [5, 7, 40, 20], 8, 2, 3),
    ([0, 0, 4, 0], [0, 3, 4, 0], 8, 1, 0),
    ([40, 1], [70, 1], 32, 0, 5),
]


@both
@pytest.mark.parametrize("norm", [0, 1], ids=["plain", "norm"])
@pytest.mark.parametrize("NH,NKV,HD,rot,layout", [(3, 1, 64, 64, 0), (15, 5, 64, 64, 0), (4, 2, 128, 64, 1), (2, 2, 80, 40, 0),
                                                  (0, 3, 64, 64, 0), (6, 3, 8, 0, 0), (2, 1, 256, 256, 1), (4, 4, 72, 24, 0)])
@pytest.mark.parametrize("new,total,page,lead,tail", BATCHES)
def test_kv_append(be, new, total, page, lead, tail, NH, NKV, HD, rot, layout, norm, kind):
    rng = np.random.default_rng(sum(total) * 31 + HD + NH)
    b = Batch(be, rng, kind, new, total, page, NKV, HD, lead, tail)
    Q, K, N = NH * HD, NKV * HD, b.N
    q, k, v = (kind.held(rng.standard_normal((N, w))) for w in (max(Q, 1), K, K))
    v.reshape(-1)[:4] = [np.inf, np.nan, -0.0, -np.inf]  # values go in as they are
    gain = (1 + 0.3 * rng.standard_normal((2, HD))).astype(np.float32)
    table, m = turn_table(rot, "llama3")
    eps = np.float64(np.float32(1e-5))
    cache0 = rng.integers(0, 1 << 16, (b.count, 2, NKV, page, HD * kind.size // 2)).astype(np.uint16)
    at = b.seq >= 0
    for ldq, ldk, ldv, ldqo, off0 in ((Q, K, K, Q, 0), (Q + 2 * K, Q + 2 * K, Q + 2 * K, Q, 0), (Q + 1, K + 3, K + 1, Q + 5, 3)):
        ldq, ldqo = max(ldq, 1), max(ldqo, 1)
        cache = be.upload(cache0)
        out = marked(be, (off0 + N * ldqo + 3) * kind.size)
        bufs = [be.upload(strided(kind, x, ld, off0)) for x, ld in ((q, ldq), (k, ldk), (v, ldv))]
        sh = off0 * kind.size
        assert be.dispatch("kv_append_paged" + kind.suffix, bufs + [out, cache] + b.tables(be) + [
            be.upload(table), be.upload(gain),
            be.params(N, b.S, NH, NKV, HD, rot, layout, ldq, ldk, ldv, ldqo, page, b.count, b.width, norm),
            floats(be, m, 1e-5)], (N,), (256,), offsets=[sh, sh, sh, sh] + [0] * 8) == 0
        if NH:
            y = q.reshape(N, NH, HD).astype(np.float64)
            y = normed(y, gain[0], eps) if norm else y
            want, off = turned(y, b.pos, rot, layout, table, m)
            off = off + turned_sum(np.abs(y), rot, layout, abs(m)) * 3 * U32 * norm
            got = rows_of(kind, out, N, Q, ldqo, off0, at)
            check(kind, got[at], want.reshape(N, Q)[at], off.reshape(N, Q)[at])
        else:
            assert (out.read(np.uint8) == MARK).all()
        y = k.reshape(N, NKV, HD).astype(np.float64)
        y = normed(y, gain[1], eps) if norm else y
        want, off = turned(y, b.pos, rot, layout, table, m)
        off = off + turned_sum(np.abs(y), rot, layout, abs(m)) * 3 * U32 * norm
        raw = cache.read(np.uint16)[:cache0.size].reshape(cache0.shape)
        held = kind.values(raw.view(kind.memory)).reshape(b.count, 2, NKV, page, HD)
        rest = raw.copy()
        for n in np.flatnonzero(at):
            pg, j = b.place(b.seq[n], int(b.pos[n]))
            check(kind, held[pg, 0, :, j], want[n], off[n])
            assert np.array_equal(held[pg, 1, :, j].reshape(-1), v[n], equal_nan=True)
            rest[pg, :, :, j] = cache0[pg, :, :, j]
        assert np.array_equal(rest, cache0)  # nothing else was written


@both
def test_kv_append_skips_what_has_no_place(be, kind):
    """Rows before position 0, on pages that are none and past the table: the cache keeps its bits there, q is turned all
    the same."""
    NH, NKV, HD, page = 2, 1, 64, 8
    # sequence 0: five rows over three keys (positions -2 .. 2); 1: pages 9 (none) and 0; 2: past the table; 3: page -1
    start, length = np.int32([0, 5, 11, 13, 14]), np.int32([3, 10, 25, 1])
    pages = np.int32([[2, -1, -1], [9, 0, -1], [3, 1, 4], [-1, -1, -1]])
    N, count = 14, 6
    pos = np.concatenate([np.arange(length[s] - (start[s + 1] - start[s]), length[s]) for s in range(4)])
    rng = np.random.default_rng(9)
    q, k, v = (kind.held(rng.standard_normal((N, w * HD))) for w in (NH, NKV, NKV))
    table, m = turn_table(HD, "none")
    cache = marked(be, count * 2 * NKV * page * HD * kind.size)
    out = marked(be, N * NH * HD * kind.size)
    assert be.dispatch("kv_append_paged" + kind.suffix, [be.upload(kind.raw(x)) for x in (q, k, v)] + [
        out, cache, be.upload(start), be.upload(length), be.upload(pages), be.upload(table), be.upload(table),
        be.params(N, 4, NH, NKV, HD, HD, 0, NH * HD, HD, HD, NH * HD, page, count, 3, 0), floats(be, m, 0.0)], (N,),
        (256,)) == 0
    want, off = turned(q.reshape(N, NH, HD), pos, HD, 0, table, m)
    check(kind, kind.values(out.read(kind.memory)).reshape(N, NH, HD), want, off)
    raw = cache.read(kind.memory).reshape(count, 2, page, HD)
    written = {(2, j): 2 + j for j in range(3)}  # sequence 0's positions 0 .. 2
    written.update({(0, j): 9 + j for j in range(2)})  # sequence 1's positions 8 and 9
    # sequence 2's positions 23 and 24: the first is in page 4, the second past the table's 24
    written[(4, 7)] = 11
    for pg in range(count):
        for j in range(page):
            if (pg, j) in written:
                assert np.array_equal(kind.values(raw[pg, 1, j]), v[written[pg, j]])
            else:
                assert (raw[pg, :, j].copy().view(np.uint8) == MARK).all(), (pg, j)


@both
@pytest.mark.parametrize("norm", [0, 1], ids=["plain", "norm"])
@pytest.mark.parametrize("HD,rot,layout,ld", [(64, 32, 0, 64), (64, 32, 1, 64), (8, 0, 0, 8), (40, 8, 0, 41), (256, 64, 1, 258)])
def test_what_passes_unturned_keeps_every_bit(be, HD, rot, layout, ld, norm, kind):
    """v, and without the norm q's and k's elements from rot on, of every pattern of bits that bf16 has (and as many of fp32),
    NaNs that signal among them."""
    rng = np.random.default_rng(HD)
    n, page = 65536 // HD + 5, 64
    turn = np.arange(HD) < rot
    bits = np.resize(rng.permutation(1 << 16).astype(np.uint16), n * HD).reshape(n, HD)
    if not kind.bf16:
        bits = bits.astype(np.uint32) << 16 | rng.integers(0, 1 << 16, (n, HD)).astype(np.uint32)
    x = np.where(turn, kind.raw(rng.standard_normal((n, HD))).view(bits.dtype), bits)
    table, m = turn_table(rot, "none")
    src = np.zeros((n, ld), bits.dtype)
    src[:, :HD] = x
    vsrc = np.zeros((n, ld), bits.dtype)
    vsrc[:, :HD] = bits
    width = -(-n // page)
    cache, out = be.alloc(width * 2 * page * HD * kind.size), be.alloc(n * ld * kind.size)
    assert be.dispatch("kv_append_paged" + kind.suffix, [
        be.upload(src), be.upload(src), be.upload(vsrc), out, cache, be.upload(np.int32([0, n])), be.upload(np.int32([n])),
        be.upload(np.arange(width, dtype=np.int32)), be.upload(table), be.upload(np.ones((2, HD), np.float32)),
        be.params(n, 1, 1, 1, HD, rot, layout, ld, ld, ld, ld, page, width, width, norm), floats(be, m, 1e-5)], (n,), (256,)) == 0
    raw = cache.read(bits.dtype).reshape(width, 2, page, HD)
    assert np.array_equal(raw[:, 1].reshape(-1, HD)[:n], bits)
    if not norm:
        assert np.array_equal(raw[:, 0].reshape(-1, HD)[:n, ~turn], bits[:, ~turn])
        assert np.array_equal(out.read(bits.dtype).reshape(n, ld)[:, :HD][:, ~turn], bits[:, ~turn])


@both
@pytest.mark.parametrize("S", [65, 1000, 4096])
def test_kv_append_of_many_sequences(be, S, kind):
    """As many sequences as a batch takes, some without tokens, in a call of more rows than a workgroup has: every row is in its place."""
    rng = np.random.default_rng(S)
    new = [int(x) for x in rng.choice([0, 0, 1, 1, 2, 3], S)]
    total = [n + int(rng.integers(0, 30)) for n in new]
    NH, NKV, HD, page = 2, 1, 16, 8
    b = Batch(be, rng, kind, new, total, page, NKV, HD, 1, 2)
    q, k, v = (kind.held(rng.standard_normal((b.N, w * HD))) for w in (NH, NKV, NKV))
    table, m = turn_table(HD, "none")
    cache = marked(be, b.cache.size * kind.size)
    out = marked(be, b.N * NH * HD * kind.size)
    assert be.dispatch("kv_append_paged" + kind.suffix, [be.upload(kind.raw(x)) for x in (q, k, v)] + [out, cache] + b.tables(be) + [
        be.upload(table), be.upload(table), be.params(b.N, S, NH, NKV, HD, HD, 0, NH * HD, HD, HD, NH * HD, page, b.count, b.width, 0),
        floats(be, m, 0.0)], (b.N,), (256,)) == 0
    at = np.flatnonzero(b.seq >= 0)
    want, off = turned(q.reshape(b.N, NH, HD), b.pos, HD, 0, table, m)
    got = rows_of(kind, out, b.N, NH * HD, NH * HD, 0, b.seq >= 0).reshape(b.N, NH, HD)
    check(kind, got[at], want[at], off[at])
    raw = cache.read(kind.memory, b.cache.size).reshape(b.cache.shape)
    want, off = turned(k.reshape(b.N, NKV, HD), b.pos, HD, 0, table, m)
    pg, j = b.pages[b.seq[at], b.pos[at] // page], b.pos[at] % page
    check(kind, kind.values(raw[pg, 0, :, j]), want[at], off[at])
    assert np.array_equal(kind.values(raw[pg, 1, :, j]).reshape(-1, HD), v[at])
    raw[pg, :, :, j] = np.full(1, MARK, np.uint8).repeat(kind.size).view(kind.memory)[0]
    assert (raw.view(np.uint8) == MARK).all()  # nothing else was written


@both
@pytest.mark.parametrize("norm", [0, 1], ids=["plain", "norm"])
def test_kv_append_past_the_cache_has_the_same_bits(be, norm, kind):
    """A call of more than 128 MB, which reads past the caches, against its rows in calls of fewer, each behind what is there."""
    NH, NKV, HD, page, S = 4, 2, 128, 64, 3
    W = (NH + 2 * NKV) * HD
    N = (150 << 20) // (W * kind.size) // S * S
    n = N // S
    rng = np.random.default_rng(51)
    block = kind.raw(rng.standard_normal((1 << 16) + 7).astype(np.float32))
    width = -(-n // page)
    qkv = be.upload(np.resize(block, (N, W)))
    pages = be.upload(rng.permutation(S * width).astype(np.int32).reshape(S, width))
    table, m = turn_table(HD, "none")
    rest = [be.upload(table), be.upload(rng.standard_normal((2, HD)).astype(np.float32))]

    def run(cache, out, start, length, first, rows):
        shift = first * W * kind.size
        assert be.dispatch("kv_append_paged" + kind.suffix, [
            qkv, qkv, qkv, out, cache, be.upload(np.int32(start)), be.upload(np.int32(length)), pages] + rest + [
            be.params(rows, S, NH, NKV, HD, HD, 0, W, W, W, NH * HD, page, S * width, width, norm), floats(be, m, 1e-5)], (rows,),
            (256,), offsets=[shift, shift + NH * HD * kind.size, shift + (NH + NKV) * HD * kind.size,
                             first * NH * HD * kind.size] + [0] * 8) == 0

    def buffers():
        return be.alloc(S * width * 2 * NKV * page * HD * kind.size), marked(be, N * NH * HD * kind.size)

    whole, parts = buffers(), buffers()
    run(*whole, [0, n, 2 * n, N], [n] * S, 0, N)
    for s in range(S):
        for a in range(0, n, 5000):
            c = min(5000, n - a)
            run(*parts, [0] * (s + 1) + [c] * (S - s), [a + c if x == s else 0 for x in range(S)], s * n + a, c)
    for x, y in zip(whole, parts):
        assert np.array_equal(x.read(np.uint8), y.read(np.uint8))


# ---------------------------------------------------------------- attention

def attend(b, q, NH, scale, causal=1, window=0):
    """The formula in 64 bits, and per element how far fp32 steps (and bf16's weights) may be off.

    A score: HD products and sums in any order, the scale and the exponent's argument: (HD + 12) U32 of scale * sum |q| |k|
    (the fp32 form's split operands leave three products of 2^-24 out: 4 more), and its own few roundings.  A weight: e^that, the exponential's 2 units, and for
    bf16 the rounding of the weights (not of their sum).  The sums over the keys: one rounding a key at most, and 64 for
    the partial sums that are joined.  The quotient: numerator and denominator."""
    out = np.zeros((b.N, NH, b.HD))
    off = np.zeros_like(out)
    R = NH // b.NKV
    for n in range(b.N):
        s = b.seq[n]
        if s < 0:
            continue
        last = b.pos[n] if causal else b.total[s] - 1
        first = max(0, last - window + 1) if window else 0
        if last < first:
            continue
        for h in range(NH):
            k, v = (x[s][h // R, first:last + 1].astype(np.float64) for x in (b.K, b.V))
            x = q[n, h].astype(np.float64)
            sc = k @ x * scale
            p = np.exp(sc - sc.max())
            p /= p.sum()
            out[n, h] = p @ v
            span = (np.abs(k) @ np.abs(x)).max() * abs(scale)
            e = (b.HD + 16) * U32 * span + 6 * U32 * np.abs(sc).max() + 4 * U32 + (len(p) + 64) * U32
            e = np.expm1(e)
            off[n, h] = (2 * e + b.kind.step) * (p @ np.abs(v))
    return out, off


def attend_values(b, NH, q, scale, window=0):
    """softmax(..) |V|, which the weights' rounding in `attend` is relative to."""
    c = Batch.__new__(Batch)
    c.__dict__.update(b.__dict__, V=[np.abs(v) for v in b.V])
    return attend(c, q, NH, scale, 1, window)[0]


def attention(be, b, q, NH, scale, causal=1, window=0, ldq=None, ldo=None, lead=0, cache=None, tables=None, out=None):
    """One call; the rows of out, checked to hold the mark wherever no sequence has a row."""
    kind, W = b.kind, NH * b.HD
    ldq, ldo = ldq or W, ldo or W
    out = out or marked(be, (lead + b.N * ldo + 3) * kind.size)
    cache = cache or be.upload(kind.raw(b.cache))
    assert be.dispatch("attention_forward_paged" + kind.suffix, [
        be.upload(strided(kind, q.reshape(b.N, W), ldq, lead)), cache, out] + (tables or b.tables(be)) + [
        be.params(b.N, b.S, NH, b.NKV, b.HD, ldq, ldo, b.page, b.count, b.width, causal, window), floats(be, scale)],
        (b.N,), (256,), offsets=[lead * kind.size, 0, lead * kind.size] + [0] * 5) == 0
    return rows_of(kind, out, b.N, W, ldo, lead, b.seq >= 0).reshape(b.N, NH, b.HD)


def compare(b, got, want, off):
    at = b.seq >= 0
    check(b.kind, got[at], want[at], off[at])


HEADS = [(1, 1, 64), (3, 1, 64), (15, 5, 64), (9, 3, 64), (8, 1, 128), (4, 4, 128), (16, 2, 80), (6, 2, 96), (7, 1, 8),
         (2, 1, 256), (20, 1, 64), (33, 1, 64), (12, 2, 40), (5, 5, 192), (40, 1, 128)]
ATTEND = BATCHES + [
    ([1, 1, 1, 1], [300, 64, 65, 129], 16, 0, 0),
    ([17], [60], 16, 0, 0),
    ([1, 130, 2], [200, 131, 2], 64, 0, 2),
    ([64, 33], [64, 97], 128, 0, 0),
    ([1], [1100], 16, 0, 0),
    ([2, 1], [515, 1030], 8, 1, 0),
    ([200], [333], 32, 0, 0),
]


@both
@pytest.mark.parametrize("NH,NKV,HD", HEADS)
@pytest.mark.parametrize("new,total,page,lead,tail", ATTEND)
def test_attention(be, new, total, page, lead, tail, NH, NKV, HD, kind):
    """Every batch by every head layout; pages' ends and pages of no one hold NaN."""
    rng = np.random.default_rng(sum(total) * 31 + sum(new) + HD + NH)
    b = Batch(be, rng, kind, new, total, page, NKV, HD, lead, tail)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, NH, HD)) * rng.uniform(0.5, 3, (NH, 1)))
    scale = float(np.float32(HD ** -0.5))
    want, off = attend(b, q, NH, scale)
    compare(b, attention(be, b, q, NH, scale), want, off)


@both
@pytest.mark.parametrize("window", [1, 2, 16, 31, 64, 100, 1000])
@pytest.mark.parametrize("new,total,page", [([1, 1], [300, 90], 16), ([70], [150], 32), ([130, 1, 5], [130, 400, 64], 64)])
def test_attention_window(be, new, total, page, window, kind):
    rng = np.random.default_rng(window + sum(total))
    b = Batch(be, rng, kind, new, total, page, 2, 64)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 6, 64)))
    want, off = attend(b, q, 6, 0.125, 1, window)
    compare(b, attention(be, b, q, 6, 0.125, 1, window), want, off)


@both
@pytest.mark.parametrize("NH,NKV,HD", [(4, 2, 64), (3, 1, 128)])
@pytest.mark.parametrize("new,total,page", [([1, 3], [40, 7], 16), ([70, 1, 0, 9], [50, 200, 8, 0], 32)])
def test_attention_without_order(be, new, total, page, NH, NKV, HD, kind):
    """causal 0: every row sees all of its sequence's keys (more new tokens than keys among them, and none)."""
    rng = np.random.default_rng(HD + sum(total))
    b = Batch(be, rng, kind, new, total, page, NKV, HD)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, NH, HD)))
    want, off = attend(b, q, NH, HD ** -0.5, 0)
    got = attention(be, b, q, NH, HD ** -0.5, 0)
    compare(b, got, want, off)
    assert (got[b.seq == 3] == 0).all()


@both
@pytest.mark.parametrize("new", [1, 3, 40, 140])
def test_attention_rows_that_see_nothing(be, new, kind):
    """More new tokens than keys: the rows before position 0 get zeros, whatever q holds there."""
    rng = np.random.default_rng(new)
    b = Batch(be, rng, kind, [new, new + 2], [0, new], 16, 2, 64)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 4, 64)))
    q[:new] = np.nan
    q[new:new + 2] = np.inf
    got = attention(be, b, q, 4, 0.125)
    assert (got[:new + 2] == 0).all()
    want, off = attend(b, np.where(np.isfinite(q), q, 0), 4, 0.125)
    check(kind, got[new + 2:], want[new + 2:], off[new + 2:])


@both
@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("new,total,window", [([1, 1], [64, 40], 0), ([64], [64], 0), ([50, 3], [61, 64], 0), ([64], [64], 7),
                                              ([33, 1], [64, 64], 20)])
def test_attention_weights(be, new, total, window, HD, kind):
    """V as the identity shows the weights: zeros exactly where a key is masked, and the softmax where it is not."""
    rng = np.random.default_rng(HD + sum(total))
    b = Batch(be, rng, kind, new, total, 16, 1, HD, fill=0.0)
    b.fill(rng)
    for s in range(b.S):
        b.V[s] = np.eye(total[s], HD, dtype=np.float32)[None]
        b.set(s, b.K[s], b.V[s])
    q = kind.held(rng.standard_normal((b.N, 3, HD)))
    want, off = attend(b, q, 3, HD ** -0.5, 1, window)
    got = attention(be, b, q, 3, HD ** -0.5, 1, window)
    assert np.array_equal(got == 0, want == 0)
    compare(b, got, want, off)
    assert (got[want > 0] > 0).all()


@both
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("NH,NKV,HD", [(3, 1, 64), (4, 2, 128), (2, 1, 96), (2, 1, 256)])
@pytest.mark.parametrize("new,total,window", [([64], [100], 0), ([5, 1], [33, 70], 0), ([40], [90], 16), ([150], [150], 50)])
def test_attention_masked_keys_hold_anything(be, new, total, window, NH, NKV, HD, what, kind):
    """A key or a value that is no number, at a place that only later rows (or with a window only earlier ones) see: the
    rows that do not see it are as ever, bit for bit; of those that do, a value's element, and for a key the row, is no
    finite number (a key's weight may also be 0, where its score is -infinity)."""
    rng = np.random.default_rng(HD + sum(total) + window)
    b = Batch(be, rng, kind, new, total, 16, NKV, HD)
    b.fill(rng)
    q = kind.held(np.abs(rng.standard_normal((b.N, NH, HD))) + 0.1)
    scale = HD ** -0.5
    want, off = attend(b, q, NH, scale, 1, window)
    clean = attention(be, b, q, NH, scale, 1, window)
    compare(b, clean, want, off)
    for part in (0, 1):
        for s in range(b.S):
            for j in sorted({total[s] - 1, max(0, total[s] - new[s]), total[s] - (new[s] + 1) // 2, max(0, total[s] - new[s] - 1)}):
                pg, at = b.place(s, j)
                kept = b.cache[pg, part, :, at].copy()
                b.cache[pg, part, 0, at, 5] = what
                got = attention(be, b, q, NH, scale, 1, window)
                b.cache[pg, part, :, at] = kept
                sees = (b.seq == s) & (b.pos >= j) & ((b.pos < j + window) if window else True)
                R = NH // NKV
                assert np.array_equal(got[~sees], clean[~sees]), (part, s, j)
                assert np.array_equal(got[:, R:], clean[:, R:])
                if part:
                    assert not np.isfinite(got[sees][:, :R, 5]).any()
                    rest = np.arange(HD) != 5
                    assert np.array_equal(got[:, :, rest], clean[:, :, rest])
                elif what != -np.inf:
                    assert not np.isfinite(got[sees][:, :R]).any()


@both
@pytest.mark.parametrize("HD", [64, 104, 200])
def test_attention_missing_pages(be, HD, kind):
    """Rows that see a key whose page is none, or lies past the table, get NaN; the others are as ever."""
    rng = np.random.default_rng(4)
    b = Batch(be, rng, kind, [40, 1, 2], [60, 70, 33], 16, 2, HD)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 4, HD)))
    want, off = attend(b, q, 4, 0.125)
    for bad in (-1, b.count, -(1 << 31), (1 << 31) - 1):
        t = b.tables(be)
        pages = b.pages.copy()
        pages[0, 2] = bad  # keys 32 .. 47 of sequence 0
        pages[2, 2] = bad  # key 32 of sequence 2, which its second row alone sees
        got = attention(be, b, q, 4, 0.125, tables=t[:2] + [be.upload(pages)])
        gone = ((b.seq == 0) & (b.pos >= 32)) | ((b.seq == 2) & (b.pos >= 32))
        assert np.isnan(got[gone]).all()
        check(kind, got[~gone], want[~gone], off[~gone])
        # a window that has passed them
        got = attention(be, b, q, 4, 0.125, 1, 4, tables=t[:2] + [be.upload(pages)])
        gone = ((b.seq == 0) & (b.pos >= 32) & (b.pos < 51)) | ((b.seq == 2) & (b.pos >= 32))
        assert np.isnan(got[gone]).all() and np.isfinite(got[~gone]).all()
    # keys past the table's room
    length = b.len.copy()
    length[1] = b.width * 16 + 1
    pages = np.where(b.pages < 0, 0, b.pages % b.count).astype(np.int32)
    t = b.tables(be)
    got = attention(be, b, q, 4, 0.125, tables=[t[0], be.upload(length), be.upload(pages)])
    assert np.isnan(got[b.seq == 1]).all()
    check(kind, got[b.seq == 0], want[b.seq == 0], off[b.seq == 0])


@both
@pytest.mark.parametrize("new,total", [([1, 1], [200, 3]), ([90], [120])])
def test_attention_strides(be, new, total, kind):
    rng = np.random.default_rng(8)
    b = Batch(be, rng, kind, new, total, 32, 2, 64, 1, 2)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 6, 64)))
    want, off = attend(b, q, 6, 0.125)
    W = 6 * 64
    for ldq, ldo, lead in ((W + 1, W + 3, 1), (W + 2, W + 2, 2), (W + 8, W + 24, 8), (3 * W, 2 * W, 4)):
        compare(b, attention(be, b, q, 6, 0.125, 1, 0, ldq, ldo, lead), want, off)


@both
def test_attention_scores_far_apart(be, kind):
    """Scores of +-1000s: the largest takes all; equal ones give the mean; a scale of 0 and a negative one."""
    rng = np.random.default_rng(11)
    for new, total in (([1], [500]), ([100], [130])):
        b = Batch(be, rng, kind, new, total, 16, 1, 64)
        b.fill(rng, 8.0)
        q = kind.held(rng.standard_normal((b.N, 4, 64)) * 8)
        for scale in (1.0, -1.0, 0.0):
            want, off = attend(b, q, 4, scale)
            compare(b, attention(be, b, q, 4, scale), want, off)


@both
@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("new,total", [([1, 2], [1500, 40]), ([40], [900]), ([130, 1], [333, 20])])
@pytest.mark.parametrize("at", [25, 29, 30, 31, 40, 100, "mixed"])
def test_attention_scores_past_what_tells_them_apart(be, at, new, total, HD, kind):
    """Scores of 2^at and a few steps of the type more, to 2^100, or of both signs from 1 to 2^34: q and K have one dimension, so a
    score is exact, and the answer is the softmax of those numbers: the largest takes all, or its equals share, or the steps are small
    enough for weights between.

    The exponent is one rounding of its own size and one of the row's base, which is a step of the score, up to 2^9 where that
    still lets a second weight live; the scale's rounding, the exponential, a rounding a key in the sums."""
    mixed, at = at == "mixed", 34 if at == "mixed" else at
    rng = np.random.default_rng(at * 1000 + HD + sum(new))
    step = 2.0 ** (-7 if kind.bf16 else -23)
    for sign, scale in ((1, 1.0), (-1, 1.0), (1, 0.7), (1, -1.0)):
        scale = float(np.float32(scale))
        b = Batch(be, rng, kind, new, total, 16, 1, HD, fill=0.0)
        b.fill(rng)
        d = int(rng.integers(0, HD))
        for s in range(b.S):
            k = np.zeros((1, total[s], HD), np.float32)
            k[0, :, d] = 2.0 ** (at // 2) * (1 + step * rng.integers(0, 5, total[s]))
            if mixed:  # rising from far below 0 to far above in the order of the keys, here and there the other way
                k[0, :, d] *= np.exp2(-rng.integers(0, 35, total[s])) * np.where(rng.random(total[s]) < 0.99, -1, 1)
                k[0, :total[s] // 2, d] = -np.abs(k[0, :total[s] // 2, d])
            b.K[s] = k
            b.set(s, k, b.V[s])
        q = np.zeros((b.N, 3, HD), np.float32)
        q[..., d] = sign * 2.0 ** (at - at // 2)
        got = attention(be, b, q, 3, scale)
        for n in range(b.N):
            s, seen = b.seq[n], b.pos[n] + 1
            k, v = (x[s][0, :seen].astype(np.float64) for x in (b.K, b.V))
            away = k[:, d] * q[n, 0, d] * scale
            away -= away.max()
            p = np.exp(away)
            p /= p.sum()
            e = (3 * np.abs(away) + min(2.0 ** (at - 22), 512.0) + 32 + seen + 64) * U32
            off = 2 * (p * e) @ np.abs(v)
            check(kind, got[n], np.broadcast_to(p @ v, (3, HD)), off + kind.step * (p @ np.abs(v)))


@both
def test_attention_many_sequences(be, kind):
    """More sequences than lanes, some without tokens, some without keys."""
    rng = np.random.default_rng(12)
    S = 300
    new = [int(x) for x in rng.choice([0, 1, 1, 1, 2, 5], S)]
    total = [n + int(rng.integers(0, 60)) if n else int(rng.integers(0, 5)) for n in new]
    b = Batch(be, rng, kind, new, total, 16, 1, 64, 0, 3)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 2, 64)))
    want, off = attend(b, q, 2, 0.125)
    compare(b, attention(be, b, q, 2, 0.125), want, off)


@both
@pytest.mark.parametrize("S,long", [(63, 0), (64, 0), (65, 0), (128, 900), (129, 4000), (1000, 2500), (4096, 0)])
def test_attention_of_as_many_sequences_as_a_batch_takes(be, S, long, kind):
    """Up to a wave's lanes and more than them, in 64s that are whole, empty and not; with some long sequences, among them the
    first and the last, whose keys are split."""
    rng = np.random.default_rng(S)
    new = [int(x) for x in rng.choice([0, 1, 1, 1, 2], S)]
    if S >= 1000:
        new[128:192] = [0] * 64
    total = [n + int(rng.integers(0, 40)) if n else 0 for n in new]
    if long:
        for s in (0, S // 2, S - 1):
            new[s], total[s] = 1 + s % 3, long + s
    b = Batch(be, rng, kind, new, total, 16, 1, 32, 0, 3)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 2, 32)))
    want, off = attend(b, q, 2, 0.2)
    first = attention(be, b, q, 2, 0.2)
    compare(b, first, want, off)
    assert np.array_equal(attention(be, b, q, 2, 0.2), first)


@pytest.mark.parametrize("S", [3, 200])
@pytest.mark.parametrize("how", ["falling", "overlapping", "negative", "past", "huge", "far"])
def test_attention_tables_that_are_no_batch(be, S, how):
    """Whatever start and len hold, rows outside N are not written and the call ends; the next call has its own results."""
    kind, rng = KINDS[1], np.random.default_rng(5)
    b = Batch(be, rng, kind, [2] * S, [40] * S, 16, 1, 64)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 2, 64)))
    want, off = attend(b, q, 2, 0.125)
    start, length = b.start.copy(), b.len.copy()
    if how == "falling":
        start = start[::-1].copy()
    elif how == "overlapping":
        start[:-1] = 0
        start[1::2] = b.N
    elif how == "negative":
        start -= b.N // 2
        length[::2] = -7
    elif how == "past":
        start += b.N // 2
    elif how == "huge":
        start[1:] = 2 ** 31 - 1
        length[:] = 2 ** 31 - 1
    else:
        length[:] = 2 ** 31 - 1
    room, past = b.N * 128 * kind.size, 1 << 16
    out = marked(be, room + past)
    tables = [be.upload(start), be.upload(length), be.upload(b.pages)]
    assert be.dispatch("attention_forward_paged_bf16", [be.upload(kind.raw(q)), be.upload(kind.raw(b.cache)), out] + tables + [
        be.params(b.N, b.S, 2, 1, 64, 128, 128, 16, b.count, b.width, 1, 0), floats(be, 0.125)], (b.N,), (256,)) == 0
    be.synchronize()
    mark = marked(be, past).read(np.uint8)
    assert np.array_equal(out.read(np.uint8)[room:], mark)
    compare(b, attention(be, b, q, 2, 0.125), want, off)


@both
@pytest.mark.parametrize("NH,NKV,HD", [(6, 2, 64), (4, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("new,total,causal,window", [([1], [3000], 0, 0), ([50], [2500], 0, 0), ([140, 1, 9], [2100, 1800, 40], 0, 0),
                                                     ([1, 2], [3000, 1700], 1, 700), ([50, 3], [2500, 900], 1, 33),
                                                     ([140, 1, 9], [2100, 1800, 40], 1, 700), ([70], [1500], 1, (1 << 31) - 1)])
def test_attention_masks_over_keys_in_parts(be, causal, window, new, total, NH, NKV, HD, kind):
    """Every mask where the keys that rows see are many enough to be split, and where a window leaves few of many."""
    rng = np.random.default_rng(sum(new) + HD)
    b = Batch(be, rng, kind, new, total, 16, NKV, HD)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, NH, HD)))
    scale = float(np.float32(HD ** -0.5))
    want, off = attend(b, q, NH, scale, causal, window)
    compare(b, attention(be, b, q, NH, scale, causal, window), want, off)


@both
@pytest.mark.parametrize("NH,NKV,HD", [(129, 1, 64), (300, 1, 8), (1100, 1, 128), (1200, 300, 8), (4096, 4096, 8)])
@pytest.mark.parametrize("new,total,window", [([1], [40], 0), ([3, 1], [130, 20], 0), ([2, 2], [700, 9], 60)])
def test_attention_of_many_heads(be, new, total, window, NH, NKV, HD, kind):
    """Groups of more heads than a unit has rows, so that a token's lie in several of them, and as many KV heads as there may be."""
    rng = np.random.default_rng(NH + sum(total))
    if NKV > 1000:
        new, total = new[:1], [min(total[0], 60)]
    b = Batch(be, rng, kind, new, total, 16, NKV, HD)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, NH, HD)))
    scale = float(np.float32(HD ** -0.5))
    want, off = attend(b, q, NH, scale, 1, window)
    compare(b, attention(be, b, q, NH, scale, 1, window), want, off)


@both
@pytest.mark.parametrize("causal,window", [(0, 0), (1, 300)])
def test_attention_masks_of_many_sequences(be, causal, window, kind):
    """The same for more sequences than lanes, a few of them long."""
    rng = np.random.default_rng(50)
    new = [int(x) for x in rng.choice([0, 1, 1, 2], 150)]
    total = [n + int(rng.integers(0, 50)) for n in new]
    for s, n, t in ((0, 1, 2500), (70, 40, 1500), (149, 3, 900)):
        new[s], total[s] = n, t
    b = Batch(be, rng, kind, new, total, 16, 1, 64, 2, 3)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 3, 64)))
    want, off = attend(b, q, 3, 0.125, causal, window)
    compare(b, attention(be, b, q, 3, 0.125, causal, window), want, off)


@both
def test_attention_long_context_beside_short_ones(be, kind):
    """One long sequence (joined from parts where the work is split) among short ones; the same bits every time."""
    rng = np.random.default_rng(13)
    b = Batch(be, rng, kind, [1, 1, 3, 1], [5000, 3, 700, 90], 16, 2, 64)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 6, 64)))
    want, off = attend(b, q, 6, 0.125)
    cache = be.upload(kind.raw(b.cache))
    first = attention(be, b, q, 6, 0.125, cache=cache)
    compare(b, first, want, off)
    for _ in range(5):
        assert np.array_equal(attention(be, b, q, 6, 0.125, cache=cache), first)


@both
@pytest.mark.parametrize("NH,NKV,HD", [(3, 1, 64), (5, 1, 72), (4, 2, 128), (2, 1, 200)])
@pytest.mark.parametrize("new,total", [([11], [1500]), ([22, 9], [1300, 2000]), ([43], [1900]), ([100, 1], [1111, 1])])
def test_attention_rows_in_parts(be, new, total, NH, NKV, HD, kind):
    """More rows than one wave's over keys that are split: every number of rows a unit's records may lie in, at heads whose
    outputs do and do not go round evenly in its lanes."""
    rng = np.random.default_rng(sum(new) + HD)
    b = Batch(be, rng, kind, new, total, 16, NKV, HD)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, NH, HD)))
    scale = float(np.float32(HD ** -0.5))
    want, off = attend(b, q, NH, scale)
    compare(b, attention(be, b, q, NH, scale), want, off)


@both
def test_attention_a_cache_past_32_bits(be, kind):
    """Pages whose elements lie past 2^32 bytes and past 2^31 elements of the cache's start."""
    NKV, HD, page = 1, 64, 65536
    count = (1 << 31) // (2 * NKV * page * HD) + 1  # the last page begins at element 2^31
    cache = be.alloc(count * 2 * NKV * page * HD * kind.size)
    table, m = turn_table(0, "none")
    rng = np.random.default_rng(14)
    n, start, length, pages = 70, np.int32([0, 70]), np.int32([70]), np.int32([[count - 1]])
    k, v, q = (kind.held(rng.standard_normal((n, HD))) for _ in range(3))
    tables = [be.upload(start), be.upload(length), be.upload(pages)]
    out = marked(be, n * HD * kind.size)
    assert be.dispatch("kv_append_paged" + kind.suffix, [
        out, be.upload(kind.raw(k)), be.upload(kind.raw(v)), out, cache] + tables + [be.upload(table), be.upload(table), be.params(
            n, 1, 0, NKV, HD, 0, 0, HD, HD, HD, HD, page, count, 1, 0), floats(be, 1.0, 0.0)], (n,), (256,)) == 0
    assert be.dispatch("attention_forward_paged" + kind.suffix, [be.upload(kind.raw(q)), cache, out] + tables + [be.params(
        n, 1, 1, NKV, HD, HD, HD, page, count, 1, 1, 0), floats(be, 0.125)], (n,), (256,)) == 0
    b = Batch.__new__(Batch)
    b.N, b.NKV, b.HD, b.kind, b.total = n, 1, HD, kind, [n]
    b.seq, b.pos, b.K, b.V = np.zeros(n, int), np.arange(n), [k[None]], [v[None]]
    want, off = attend(b, q[:, None], 1, 0.125)
    got = kind.values(out.read(kind.memory)).reshape(n, 1, HD)
    cache.free()
    check(kind, got, want, off)


def test_attention_of_more_work_items_than_an_axis_takes(be):
    """4096 sequences over 4096 KV heads, a workgroup each: over 2^32 work-items.  All have one page; a row that sees one key
    has that key's value bit for bit, and one that sees eight alike keys the mean of the values."""
    kind, S, NKV, HD, page = KINDS[1], 4096, 4096, 8, 8
    W = NKV * HD
    rng = np.random.default_rng(45)
    q = np.resize(kind.raw(rng.standard_normal(1 << 16)), (S, W))
    cache = kind.raw(rng.standard_normal((2, 2, NKV, page, HD)))
    cache[:, 0] = cache[:, 0, :, :1]  # the keys of a head are alike
    length = np.where(rng.random(S) < 0.5, 1, 8).astype(np.int32)
    length[[0, -1]] = 8, 1
    pages = rng.integers(0, 2, (S, 1)).astype(np.int32)
    out = marked(be, S * W * kind.size)
    assert be.dispatch("attention_forward_paged_bf16", [
        be.upload(q), be.upload(cache), out, be.upload(np.arange(S + 1, dtype=np.int32)), be.upload(length), be.upload(pages),
        be.params(S, S, NKV, NKV, HD, W, W, page, 2, 1, 1, 0), floats(be, HD ** -0.5)], (S,), (256,)) == 0
    got = out.read(kind.memory).reshape(S, NKV, HD)
    mean = kind.values(cache[:, 1]).astype(np.float64).mean(2)
    most = np.abs(kind.values(cache[:, 1])).astype(np.float64).mean(2)  # a sum of eight in fp32, its quotient
    for p in (0, 1):
        one, all_ = (pages[:, 0] == p) & (length == 1), (pages[:, 0] == p) & (length == 8)
        assert (got[one] == cache[p, 1, :, 0]).all()
        check(kind, kind.values(got[all_]), mean[p], 12 * U32 * most[p])


# ---------------------------------------------------------------- the operators together

@both
@pytest.mark.parametrize("norm", [0, 1], ids=["plain", "norm"])
def test_prompts_in_chunks_then_tokens(be, norm, kind):
    """Three sequences served as a program would: prompts in chunks of different sizes beside the others' single tokens,
    positions and pages growing, every step append and attention in one encoder over the same cache.  Each row against
    the formula over all that its sequence holds by then."""
    NH, NKV, HD, page, S = 6, 2, 64, 16, 3
    rng = np.random.default_rng(20 + norm)
    table, m = turn_table(HD, "none")
    gain = (1 + 0.3 * rng.standard_normal((2, HD))).astype(np.float32)
    steps = [[37, 5, 0], [40, 1, 1], [1, 1, 30], [0, 70, 1], [1, 1, 1], [1, 1, 1]]
    count, width, eps = 40, 12, np.float64(np.float32(1e-5))
    pages = rng.permutation(count)[:S * width].astype(np.int32).reshape(S, width)
    cache = be.alloc(count * 2 * NKV * page * HD * kind.size)
    held = [0] * S
    K, V, Koff = ([np.zeros((NKV, 0, HD)) for _ in range(S)] for _ in range(3))
    kern = [be.kernel(n + kind.suffix) for n in ("kv_append_paged", "attention_forward_paged")]
    for new in steps:
        N = sum(new)
        held = [a + n for a, n in zip(held, new)]
        start, length = np.int32([sum(new[:s]) for s in range(S + 1)]), np.int32(held)
        W = (NH + 2 * NKV) * HD
        qkv = kind.held(rng.standard_normal((N, W)))  # one stacked product's rows
        src, qo, out = be.upload(kind.raw(qkv)), marked(be, N * NH * HD * kind.size), marked(be, N * NH * HD * kind.size)
        tables = [be.upload(start), be.upload(length), be.upload(pages)]
        e = be.encoder()
        assert e.dispatch(kern[0], [src, src, src, qo, cache] + tables + [be.upload(table), be.upload(gain), be.params(
            N, S, NH, NKV, HD, HD, 0, W, W, W, NH * HD, page, count, width, norm), floats(be, m, 1e-5)], (N,), (256,),
            offsets=[0, NH * HD * kind.size, (NH + NKV) * HD * kind.size] + [0] * 9) == 0
        assert e.dispatch(kern[1], [qo, cache, out] + tables + [be.params(
            N, S, NH, NKV, HD, NH * HD, NH * HD, page, count, width, 1, 0), floats(be, 0.125)], (N,), (256,)) == 0
        e.commit()
        e.wait_timed()
        b = Batch.__new__(Batch)
        b.N, b.NKV, b.HD, b.kind, b.total = N, NKV, HD, kind, held
        b.seq = np.repeat(np.arange(S), new)
        b.pos = np.concatenate([np.arange(h - n, h) for h, n in zip(held, new)])
        q, k, v = (qkv[:, a:c].reshape(N, -1, HD).astype(np.float64) for a, c in (
            (0, NH * HD), (NH * HD, (NH + NKV) * HD), ((NH + NKV) * HD, W)))
        if norm:
            q, k = normed(q, gain[0], eps), normed(k, gain[1], eps)
        qt, _ = turned(q, b.pos, HD, 0, table, m)
        kt, _ = turned(k, b.pos, HD, 0, table, m)
        got_q = kind.values(qo.read(kind.memory)).reshape(N, NH, HD)
        raw = kind.values(cache.read(kind.memory)).reshape(count, 2, NKV, page, HD)
        # the operators are checked alone above: here each works on what the one before gave, and the whole stays near the formula
        assert np.abs(got_q - qt).max() <= (1e-5 if not kind.bf16 else 2 * UB16) * np.abs(qt).max()
        for s in range(S):
            at = b.seq == s
            K[s] = np.concatenate([K[s], kt[at].transpose(1, 0, 2)], 1)
            V[s] = np.concatenate([V[s], v[at].transpose(1, 0, 2)], 1)
        b.K = [np.stack([raw[pages[s, j // page], 0, :, j % page] for j in range(held[s])], 1) if held[s] else K[s] for s in range(S)]
        b.V = V
        for s in range(S):
            assert held[s] == 0 or np.abs(b.K[s] - K[s]).max() <= (1e-5 if not kind.bf16 else 2 * UB16) * np.abs(K[s]).max()
        want, off = attend(b, got_q, NH, 0.125)
        check(kind, kind.values(out.read(kind.memory)).reshape(N, NH, HD), want, off)


def test_agrees_with_the_one_sequence_kernels(be):
    """One sequence, fp32, a page for the whole context: kv_store and attention_forward over the same keys."""
    NH, NKV, HD, S = 15, 5, 64, 200
    rng = np.random.default_rng(30)
    k, v = (rng.standard_normal((S, NKV * HD)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((1, NH * HD)).astype(np.float32)
    flat, out1 = be.upload(np.stack([k, v])), marked(be, q.nbytes)
    assert be.dispatch("attention_forward", [be.upload(q), flat, out1, be.params(NH, HD, NKV, NKV * HD, S, 3, 0, S),
                                             floats(be, 0.125)], (NH,), (64,)) == 0
    b = Batch(be, rng, KINDS[0], [1], [S], 256, NKV, HD)
    b.K, b.V = ([x.reshape(S, NKV, HD).transpose(1, 0, 2)] for x in (k, v))
    b.set(0, b.K[0], b.V[0])
    got = attention(be, b, q.reshape(1, NH, HD), NH, 0.125)
    want, off = attend(b, q.reshape(1, NH, HD), NH, 0.125)
    check(KINDS[0], got, want, off)
    check(KINDS[0], out1.read(np.float32).reshape(1, NH, HD), want, off)


@both
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.3, 1e-30, 3.0])
@pytest.mark.parametrize("new,total,window", [([1, 3], [70, 20], 0), ([40], [90], 16), ([5, 1], [33, 1500], 0)])
def test_attention_scales(be, new, total, window, scale, kind):
    """No order among the keys (scale 0: the mean of the values a row sees), the smallest one first, one that takes all."""
    rng = np.random.default_rng(len(new) + window)
    b = Batch(be, rng, kind, new, total, 16, 2, 64)
    b.fill(rng)
    q = kind.held(rng.standard_normal((b.N, 4, 64)))
    scale = float(np.float32(scale))
    want, off = attend(b, q, 4, scale, window=window)
    compare(b, attention(be, b, q, 4, scale, window=window), want, off)


def test_attention_fp32_scores_lean_to_neither_side(be):
    """Scores of about 500, all of one sign, of keys with 24 bits beside ones with 8, whose products are whole: 65536 pairs'
    difference, in units of 2^-24 of a score, through the weights.  Roundings to nearest of bits without a pattern, under 2 units
    each, leave a mean within 6 * 2 / sqrt(65536) = 0.05; 0.3 has room for what the exponential and the quotient add (2^-22
    of a weight, 0.01 units).  Terms cut off towards zero leave -0.69."""
    kind, S, NH, HD, page = KINDS[0], 1024, 64, 16, 8
    rng = np.random.default_rng(46)
    q, ka = (rng.uniform(1, 2, (S, NH, HD)).astype(np.float32) for _ in range(2))
    kb = from_bf16(to_bf16(ka))
    cache = np.zeros((S, 2, NH, page, HD), np.float32)
    cache[:, 0, :, 0], cache[:, 0, :, 1], cache[:, 1, :, 0] = ka, kb, 1
    out, scale = marked(be, q.nbytes), 14.0
    assert be.dispatch("attention_forward_paged", [
        be.upload(q), be.upload(cache), out, be.upload(np.arange(S + 1, dtype=np.int32)), be.upload(np.full(S, 2, np.int32)),
        be.upload(np.arange(S, dtype=np.int32)), be.params(S, S, NH, NH, HD, NH * HD, NH * HD, page, S, 1, 1, 0),
        floats(be, scale)], (S,), (256,)) == 0
    p = out.read(np.float32).reshape(S, NH, HD)[..., 0].astype(np.float64)
    q, ka, kb = (x.astype(np.float64) for x in (q, ka, kb))
    a, b = scale * (q * ka).sum(-1), scale * (q * kb).sum(-1)
    mean = ((np.log(p / (1 - p)) - (a - b)) / (a * U32)).mean()
    assert abs(mean) < 0.3, mean


@pytest.mark.parametrize("NH,NKV,HD", [(3, 1, 8), (4, 2, 40), (15, 5, 64), (6, 2, 96), (8, 2, 128), (2, 1, 200), (4, 1, 256)])
@pytest.mark.parametrize("new,total,page,window", [
    ([1] * 6, [2, 40, 300, 300, 150, 77], 16, 0), ([1, 1], [1500, 1100], 64, 0), ([130], [333], 32, 0), ([70], [1300], 16, 0),
    ([40, 1], [200, 90], 8, 33)])
def test_attention_is_fp32_on_average(be, new, total, page, window, NH, NKV, HD):
    """The root of the mean square error over all elements within twice that of the roundings (tests/paged_exactness.py): the
    same arithmetic with a term of q, K, the weights or V missing is past four times."""
    rng = np.random.default_rng(sum(total) * 31 + HD)
    b = Batch(be, rng, KINDS[0], new, total, page, NKV, HD)
    b.fill(rng)
    q = rng.standard_normal((b.N, NH, HD)).astype(np.float32)
    scale = float(np.float32(HD ** -0.5))
    want, _ = attend(b, q, NH, scale, 1, window)
    err = want - attention(be, b, q, NH, scale, 1, window)
    allowed = np.zeros_like(want)
    for n in range(b.N):
        s, last = b.seq[n], b.pos[n]
        first = max(0, last - window + 1) if window else 0
        for h in range(NH):
            allowed[n, h] = deviation(q[n, h], *(x[s][h // (NH // NKV), first:last + 1] for x in (b.K, b.V)), scale)
    assert np.sqrt((err ** 2).mean() / (allowed ** 2).mean()) < 2


@pytest.mark.parametrize("NH,NKV,HD", [(3, 1, 8), (15, 5, 64), (32, 1, 64), (8, 2, 128), (4, 1, 200), (4, 1, 256)])
@pytest.mark.parametrize("new,total,window", [([1] * 5, [2, 40, 300, 150, 77], 0), ([1, 1], [1500, 1100], 0), ([1, 1], [600, 90], 33),
                                              ([1] * 70, [30] * 69 + [900], 0)])
def test_attention_of_few_rows_rounds_once_in_bf16(be, new, total, window, NH, NKV, HD):
    """Up to 32 rows of a KV head (single tokens): the weights go into the second product as two terms of bf16, 2^-17 of each, so
    that the result is off by its own rounding and fp32 steps alone."""
    rng = np.random.default_rng(sum(total) * 31 + HD)
    b = Batch(be, rng, KINDS[1], new, total, 16, NKV, HD)
    b.fill(rng)
    q = b.kind.held(rng.standard_normal((b.N, NH, HD)))
    scale = float(np.float32(HD ** -0.5))
    want, off = attend(b, q, NH, scale, 1, window)
    most = attend_values(b, NH, q, scale, window)
    check(b.kind, attention(be, b, q, NH, scale, 1, window), want, off + (2.0 ** -17 - b.kind.step) * most)


@pytest.mark.parametrize("NH,HD", [(1, 8), (3, 64), (2, 96), (1, 128), (2, 200), (1, 256)])
@pytest.mark.parametrize("new,ahead", [(1, 0), (5, 0), (8, 40), (8, 1200), (128, 30)])
def test_attention_gives_a_value_back_bit_for_bit(be, new, ahead, NH, HD):
    """fp32: a row whose weights are 1 for one key and 0 for all others has that key's value, all 24 bits of it: the three terms'
    sum, smallest first, is exact."""
    rng = np.random.default_rng(HD + new + ahead)
    total = ahead + new
    b = Batch(be, rng, KINDS[0], [new], [total], 16, 1, HD)
    b.K = [np.zeros((1, total, HD), np.float32)]
    b.V = [(rng.standard_normal((1, total, HD)) * np.exp2(rng.integers(-40, 100, (1, total, 1)))).astype(np.float32)]
    b.V[0][0, ::3] = 1 + rng.integers(0, 1 << 23, b.V[0][0, ::3].shape).astype(np.float32) * np.float32(2.0 ** -23)
    # keys are unit vectors, which repeat after HD; a row's q is one of the last HD keys that it sees: a score of 512, whose exponent
    # is exact, the others 0, and one of -512 for the earlier keys of the same direction
    q = np.zeros((new, NH, HD), np.float32)
    own = np.zeros((new, NH), int)
    for j in range(total):
        b.K[0][0, j, j % HD] = -16 if j < total - min(HD, total) else 16
    for i in range(new):
        for h in range(NH):
            lo = max(0, total - HD)
            own[i, h] = j = int(rng.integers(lo, ahead + i + 1)) if ahead + i >= lo else -1
            q[i, h, j % HD] = 32
    b.set(0, b.K[0], b.V[0])
    got = attention(be, b, q, NH, 1.0)
    for i in range(new):
        for h in range(NH):
            if own[i, h] >= 0:
                assert np.array_equal(got[i, h], b.V[0][0, own[i, h]]), (i, h)


@pytest.mark.parametrize("in_key", [0, 1], ids=["q", "key"])
@pytest.mark.parametrize("HD", [8, 64, 128, 256])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_scores_have_all_their_bits(be, new, HD, in_key):
    """fp32 scores that are a number's last 8 bits, what a form without some third terms has nothing of."""
    rng = np.random.default_rng(HD + new)
    q, k, v = last_bits(rng, new, 2 * new, HD, in_key)
    b = Batch(be, rng, KINDS[0], [new], [2 * new], 16, 1, HD, fill=0.0)
    b.K, b.V = [k[None]], [v[None]]
    b.set(0, b.K[0], b.V[0])
    got = attention(be, b, q[:, None], 1, 1.0)
    for i in range(new):
        assert last_bits_off(q[i], k[:new + i + 1], v[:new + i + 1], got[i, 0]) <= 1, i


@both
def test_attention_of_a_shared_prefix(be, kind):
    """Sequences whose first pages are the same ones, as after a common prompt, and one that is the same altogether."""
    rng = np.random.default_rng(21)
    new, total, page = [1, 2, 1, 1, 30], [100, 90, 100, 64, 94], 16
    b = Batch(be, rng, kind, new, total, page, 2, 64)
    b.fill(rng)
    for s in range(1, 5):
        n = 6 if s == 2 else 4
        b.pages[s, :n] = b.pages[0, :n]
        for x in (b.K, b.V):
            x[s][:, :min(n * page, total[s])] = x[0][:, :min(n * page, total[s])]
    b.pages[2], b.K[2], b.V[2] = b.pages[0], b.K[0], b.V[0]
    q = kind.held(rng.standard_normal((b.N, 6, 64)))
    want, off = attend(b, q, 6, 0.125)
    compare(b, attention(be, b, q, 6, 0.125), want, off)


class Context(ctypes.Structure):
    """backend_ctx_t up to its scratch memory (include/backend_hip_device.h)."""
    _fields_ = [("device", ctypes.c_void_p), ("queue", ctypes.c_void_p), ("library", ctypes.c_void_p),
                ("supports_bf16", ctypes.c_int), ("allocated", ctypes.c_size_t), ("peak", ctypes.c_size_t),
                ("threads", ctypes.c_int), ("memory", ctypes.c_size_t), ("most", ctypes.c_size_t), ("working", ctypes.c_size_t),
                ("unified", ctypes.c_int), ("cus", ctypes.c_int), ("clock", ctypes.c_int), ("name", ctypes.c_char * 64),
                ("busy", ctypes.c_double), ("buffers", ctypes.c_uint64), ("submitted", ctypes.c_uint64),
                ("done", ctypes.c_uint64), ("events", ctypes.c_void_p * 32), ("n_events", ctypes.c_int),
                ("last_stop", ctypes.c_void_p), ("last_stop_epoch", ctypes.c_uint64), ("scratch", ctypes.c_void_p),
                ("scratch_bytes", ctypes.c_size_t)]


@both
@pytest.mark.parametrize("keep", [0, 1 << 17, (1 << 17) + 1024 + 40000], ids=["none", "counters", "little"])
@pytest.mark.parametrize("S", [5, 150])
def test_attention_without_memory_for_parts(S, keep, kind):
    """A context that got no scratch memory, or next to none: the same rows, in fewer parts or unsplit."""
    other = bmhip.Backend()
    try:
        c = Context.from_address(other.ctx)
        assert c.scratch_bytes == 64 << 20 and c.scratch
        c.scratch_bytes = keep
        rng = np.random.default_rng(S)
        new = [1 + s % 3 for s in range(S)]
        total = [n + (3000 if s in (1, S - 1) else 20) for s, n in enumerate(new)]
        new[2], total[2] = 60, 1000
        b = Batch(other, rng, kind, new, total, 16, 2, 64)
        b.fill(rng)
        q = kind.held(rng.standard_normal((b.N, 6, 64)))
        want, off = attend(b, q, 6, 0.125)
        compare(b, attention(other, b, q, 6, 0.125), want, off)
    finally:
        other.close()


def test_two_contexts_at_once(be):
    """Passes of two contexts, each on its own stream and scratch memory, in flight together."""
    kind = KINDS[1]
    other = bmhip.Backend()
    try:
        rng = np.random.default_rng(31)
        jobs = []
        for c in (be, other):
            b = Batch(c, rng, kind, [1, 1], [3000, 2500], 16, 1, 64)
            b.fill(rng)
            q = kind.held(rng.standard_normal((b.N, 4, 64)))
            want, off = attend(b, q, 4, 0.125)
            out = marked(c, q.size * 2)
            bufs = [c.upload(kind.raw(q)), c.upload(kind.raw(b.cache)), out] + b.tables(c) + [c.params(
                2, 2, 4, 1, 64, 256, 256, 16, b.count, b.width, 1, 0), floats(c, 0.125)]
            c.synchronize()
            jobs.append((c, b, bufs, out, want, off))
        flying = []
        for _ in range(8):
            for c, b, bufs, out, want, off in jobs:
                e = c.encoder()
                for _ in range(4):
                    assert e.dispatch(c.kernel("attention_forward_paged_bf16"), bufs, (2,), (256,)) == 0
                e.commit()
                flying.append(e)
        for e in flying:
            e.wait_timed()
        for c, b, bufs, out, want, off in jobs:
            check(kind, kind.values(out.read(np.uint16)).reshape(want.shape), want, off)
        del jobs, bufs, out, flying
    finally:
        other.close()


def test_scratch_is_left_for_the_next_kernel(be):
    """Kernels that split their work share a context's scratch memory in stream order: attention_forward between passes
    over pages, both the same every time."""
    rng = np.random.default_rng(32)
    NH, NKV, HD, S = 15, 5, 64, 2048
    kv = rng.standard_normal((2, S, NKV * HD)).astype(np.float32)
    q = rng.standard_normal((1, NH * HD)).astype(np.float32)
    flat = [be.upload(q), be.upload(kv), marked(be, q.nbytes), be.params(NH, HD, NKV, NKV * HD, S, 3, 0, S), floats(be, 0.125)]
    b = Batch(be, rng, KINDS[0], [1, 1], [2048, 700], 16, NKV, HD)
    b.fill(rng)
    q2 = rng.standard_normal((2, NH, HD)).astype(np.float32)
    paged = [be.upload(q2), be.upload(b.cache), marked(be, q2.nbytes)] + b.tables(be) + [be.params(
        2, 2, NH, NKV, HD, NH * HD, NH * HD, 16, b.count, b.width, 1, 0), floats(be, 0.125)]
    seen = []
    for _ in range(4):
        e = be.encoder()
        for _ in range(3):
            assert e.dispatch(be.kernel("attention_forward"), flat, (NH,), (64,)) == 0
            assert e.dispatch(be.kernel("attention_forward_paged"), paged, (2,), (256,)) == 0
        e.commit()
        e.wait_timed()
        seen.append((flat[2].read(np.float32), paged[2].read(np.float32)))
    for x, y in seen[1:]:
        assert np.array_equal(x, seen[0][0]) and np.array_equal(y, seen[0][1])
    want, off = attend(b, q2, NH, 0.125)
    check(KINDS[0], seen[0][1].reshape(2, NH, HD), want, off)


@pytest.mark.parametrize("size", [64 << 20, 8 << 20])
def test_scratch_memory_holds_anything_but_counters(be, size):
    """What lies in a context's scratch memory behind its counters does not matter, and attention_forward cuts its work alike in one of
    8 MiB: its results have the same bits."""
    rng = np.random.default_rng(47)
    NH, NKV, HD, S = 15, 5, 64, 2048
    kv = rng.standard_normal((2, S, NKV * HD)).astype(np.float32)
    q = rng.standard_normal((1, NH * HD)).astype(np.float32)

    def flat(c):
        out = marked(c, q.nbytes)
        assert c.dispatch("attention_forward", [c.upload(q), c.upload(kv), out, c.params(NH, HD, NKV, NKV * HD, S, 3, 0, S),
                                                floats(c, 0.125)], (NH,), (64,)) == 0
        return out.read(np.float32)

    other = bmhip.Backend()
    try:
        c = Context.from_address(other.ctx)
        c.scratch_bytes = size
        hip = ctypes.CDLL("libamdhip64.so")
        hip.hipMemset.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t]
        other.synchronize()
        assert hip.hipMemset(c.scratch + (128 << 10), 0xFF, size - (128 << 10)) == 0 and hip.hipDeviceSynchronize() == 0
        for S_ in (3, 200):
            new = [1 + s % 2 for s in range(S_)]
            total = [n + (3000 if s in (0, S_ - 1) else 20) for s, n in enumerate(new)]
            for kind in KINDS:
                b = Batch(other, rng, kind, new, total, 16, 2, 64)
                b.fill(rng)
                x = kind.held(rng.standard_normal((b.N, 6, 64)))
                want, off = attend(b, x, 6, 0.125)
                compare(b, attention(other, b, x, 6, 0.125), want, off)
        assert np.array_equal(flat(other), flat(be))
    finally:
        other.close()
