# SPDX-License-Identifier: MPL-2.0
"""The 8-bit integer path (include/bm_q8.h) through the backend's C ABI against restatements in numpy.

Codes are compared for equality where their definition is made of single fp32 operations (quantize_rows_i8,
rmsnorm_forward_i8), scales and products with tolerances that count the roundings of 2^-24 (fp32) and 2^-8 (bf16)."""
import numpy as np
import pytest

import bmhip

pytestmark = pytest.mark.gpu
U32, UB16 = 2.0 ** -24, 2.0 ** -8  # half a step, relative
MARK = 0x5A  # what lies in buffers where nothing may be written


def to_bf16(x):
    """fp32 -> bf16 bits, round to nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def ld16(c):
    return (c + 15) // 16 * 16


def marked(be, nbytes):
    return be.upload(np.full((nbytes + 3) // 4 * 4, MARK, np.uint8))


def grid(p):
    """Codes and the largest magnitude of fp32 rows, each step in fp32 (see include/bm_q8.h); rows without a grid: 0."""
    with np.errstate(all="ignore"):
        top = np.abs(p).max(axis=1)
        inv = np.float32(127) * (np.float32(1) / top)
        fine = np.isfinite(inv) & np.isfinite(top)
        q = np.where(fine[:, None], np.rint(p * np.where(fine, inv, 0).astype(np.float32)[:, None]), 0)
    return q.astype(np.int8), top, fine


def strided(x, ld, esz_dtype, lead=0):
    """Rows of x, ld elements apart, behind `lead` elements, the gaps holding the mark."""
    out = np.full(lead + (x.shape[0] - 1) * ld + x.shape[1] if x.shape[0] else lead + 1, 0, esz_dtype)
    out.view(np.uint8)[:] = MARK
    for r in range(x.shape[0]):
        out[lead + r * ld:lead + r * ld + x.shape[1]] = x[r]
    return out


def check_codes(buf, want, ldq, C, lead=0):
    """The codes, zeros up to the 16-byte group's end, and the mark everywhere else."""
    M = want.shape[0]
    raw = buf.read(np.uint8)
    exp = np.full(raw.size, MARK, np.uint8)
    for r in range(M):
        at = lead + r * ldq
        exp[at:at + ld16(C)] = 0
        exp[at:at + C] = want[r].view(np.uint8)
    bad = np.flatnonzero(raw != exp)
    assert bad.size == 0, (bad[:8], raw[bad[:8]].view(np.int8), exp[bad[:8]].view(np.int8))


SHAPES = [(1, 1), (2, 3), (5, 12), (3, 15), (2, 16), (5, 17), (1, 64), (7, 100), (5, 150), (3, 200), (4, 255), (3, 256),
          (3, 300), (2, 500), (2, 576), (3, 960), (9, 1001), (2, 1024), (2, 1028), (2, 2047), (3, 2560), (2, 4096), (3, 4100),
          (1, 8192), (2, 10007), (2, 13000), (2, 16384), (2, 20011), (2, 32768), (1, 49152), (3, 40001), (333, 33), (1025, 8)]


def rows(rng, M, C):
    """Rows of different sizes, among them one of zeros, ties and a tiny one where there is room."""
    x = rng.standard_normal((M, C)).astype(np.float32) * np.exp(rng.uniform(-3, 3, (M, 1))).astype(np.float32)
    if M > 2:
        x[1] = 0
        x[1, ::2] = -0.0
        x[2] = np.float32(0.5) * rng.integers(-253, 254, C)  # halves of the grid of 127: ties to even
        x[2, 0] = 127
    if M > 4:
        x[3] *= np.float32(1e-38)
        x[4] *= np.float32(1e-42)
    return x


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,C", SHAPES)
def test_quantize_rows(be, M, C, bf16):
    rng = np.random.default_rng(M * 100003 + C)
    x = rows(rng, M, C)
    if bf16:
        x = from_bf16(to_bf16(x))
    q, top, fine = grid(x)
    s = np.where(fine, top / np.float32(127), np.float32(0))
    name = "quantize_rows_i8" + ("_bf16" if bf16 else "")
    # packed, and with strides and offsets that no wide access suits
    for lds, ldq, lead, qlead in ((C, ld16(C), 0, 0), (C + 4, ld16(C) + 16, 4, 32), (C + 3, ld16(C) + 64, 1, 16)):
        src = be.upload(strided(to_bf16(x) if bf16 else x, lds, np.uint16 if bf16 else np.float32, lead))
        bq, bs = marked(be, qlead + (M - 1) * ldq + ld16(C) + 48), marked(be, 4 * M + 16)
        assert be.dispatch(name, [src, bq, bs, be.params(M, C, lds, ldq)], (M,), (256,),
                           offsets=[lead * (2 if bf16 else 4), qlead, 8, 0]) == 0
        check_codes(bq, q, ldq, C, qlead)
        got = bs.read(np.float32)
        assert np.array_equal(got[2:2 + M], s) and (bs.read(np.uint8)[4 * M + 8:] == MARK).all()


@pytest.mark.parametrize("C", [5, 64, 960, 4097])
def test_rows_without_a_grid(be, C):
    """NaN and infinities anywhere in a row: zero codes and the scale NaN; their neighbours are as ever."""
    rng = np.random.default_rng(C)
    x = rng.standard_normal((7, C)).astype(np.float32)
    x[1, C - 1], x[2, 0], x[4, C // 2], x[5, 1] = np.nan, np.inf, -np.inf, np.nan
    x[5, 0] = np.inf
    q, top, _ = grid(x)
    bad = np.array([1, 2, 4, 5])
    src, bq, bs = be.upload(x), marked(be, 7 * ld16(C)), marked(be, 28)
    assert be.dispatch("quantize_rows_i8", [src, bq, bs, be.params(7, C, C, ld16(C))], (7,), (256,)) == 0
    check_codes(bq, q, ld16(C), C)
    s = bs.read(np.float32)
    assert np.isnan(s[bad]).all() and np.array_equal(np.delete(s, bad), np.delete(top, bad) / np.float32(127))
    # what is computed from them shows it
    back, out = marked(be, 7 * C * 4), marked(be, 7 * 3 * 4)
    assert be.dispatch("dequantize_rows_i8", [bq, bs, back, be.params(7, C, ld16(C), C)], (7,), (256,)) == 0
    v = back.read(np.float32).reshape(7, C)
    assert np.isnan(v[bad]).all() and np.isfinite(np.delete(v, bad, 0)).all()
    w, sw = be.upload(np.ones((3, ld16(C)), np.int8)), be.upload(np.ones(3, np.float32))
    assert be.dispatch("matmul_forward_i8", [bq, bs, w, sw, sw, out, be.params(7, C, 3, 0, ld16(C), ld16(C), 3)], (3, 7),
                       (256,)) == 0
    y = out.read(np.float32).reshape(7, 3)
    assert np.isnan(y[bad]).all() and np.isfinite(np.delete(y, bad, 0)).all()


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,C", SHAPES)
def test_dequantize_rows(be, M, C, bf16):
    rng = np.random.default_rng(M * 7 + C)
    q = rng.integers(-128, 128, (M, C)).astype(np.int8)
    s = np.exp(rng.uniform(-9, 3, M)).astype(np.float32)
    want = q.astype(np.float32) * s[:, None]
    want = to_bf16(want) if bf16 else want
    for ldq, ldd, lead in ((ld16(C), C, 0), (ld16(C) + 32, C + 5, 3)):
        bq = be.upload(strided(q, ldq, np.int8))
        bq = be.upload(np.concatenate([bq.read(np.int8), np.full(16, 77, np.int8)]))  # the last row's whole groups
        dst = marked(be, (lead + M * ldd) * (2 if bf16 else 4))
        assert be.dispatch("dequantize_rows_i8" + ("_bf16" if bf16 else ""),
                           [bq, be.upload(s), dst, be.params(M, C, ldq, ldd)], (M,), (256,),
                           offsets=[0, 0, lead * (2 if bf16 else 4), 0]) == 0
        got = dst.read(want.dtype)
        exp = np.full(got.size, 0, want.dtype)
        exp.view(np.uint8)[:] = MARK
        for r in range(M):
            exp[lead + r * ldd:lead + r * ldd + C] = want[r]
        assert np.array_equal(got.view(np.uint8), exp.view(np.uint8))


def norm_ref(x, r, w, eps):
    """Sum (fp32), codes, and the scale in 64 bits."""
    h = x if r is None else x + r
    q, top, fine = grid(h * w)
    rstd = 1 / np.sqrt((h.astype(np.float64) ** 2).mean(axis=1) + eps)
    with np.errstate(all="ignore"):
        return h, q, np.where(fine, top.astype(np.float64) * rstd / 127, 0)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,C", SHAPES)
def test_rmsnorm(be, M, C, bf16):
    rng = np.random.default_rng(M * 31 + C)
    x, r = rows(rng, M, C), rng.standard_normal((M, C)).astype(np.float32)
    w = rng.uniform(-1.5, 1.5, C).astype(np.float32)
    if M > 2:
        r[1:3] = 0  # a sum of zeros among the rows
    if bf16:
        x = from_bf16(to_bf16(x))
    eps = np.float32(1e-5)
    name = "rmsnorm_forward_i8" + ("_bf16" if bf16 else "")
    for res, shift, ldq in ((True, 0, ld16(C)), (True, 1, ld16(C) + 16), (False, 0, ld16(C)), (False, 1, ld16(C))):
        h, q, s = norm_ref(x, r if res else None, w, float(eps))
        bx = be.upload(np.concatenate([np.zeros(shift, np.uint16 if bf16 else np.float32),
                                       (to_bf16(x) if bf16 else x).ravel()]))
        br, bw = (be.upload(np.concatenate([np.zeros(shift, np.float32), v.ravel()])) for v in (r, w))
        bh, bq, bs = marked(be, (M * C + shift) * 4 + 16), marked(be, M * ldq + 16), marked(be, 4 * M + 16)
        assert be.dispatch(name, [bx, br, bw, bh, bq, bs, be.params(M, C, ldq, int(res)), be.upload(np.float32([eps]))],
                           (M,), (256,),
                           offsets=[shift * (2 if bf16 else 4), 4 * shift, 4 * shift, 4 * shift, 0, 0, 0, 0]) == 0
        raw = bh.read(np.uint8)
        if res:
            assert np.array_equal(raw[4 * shift:4 * (M * C + shift)].view(np.float32), h.ravel())
            assert (raw[:4 * shift] == MARK).all() and (raw[4 * (M * C + shift):] == MARK).all()
        else:
            assert (raw == MARK).all()
        check_codes(bq, q, ldq, C)
        # a fused kernel may round rstd, its product with the maximum, the 127th and the stored scale: four
        assert (np.abs(bs.read(np.float32, M) - s) <= 4 * U32 * s).all()
        assert (bs.read(np.uint8)[4 * M:] == MARK).all()


@pytest.mark.parametrize("C", [48, 960, 5000])
@pytest.mark.parametrize("where", ["residual", "x"])
def test_rmsnorm_in_place(be, C, where):
    """The sum in the residual's own buffer, or in an f32 branch's."""
    rng = np.random.default_rng(C)
    x, r, w = (rng.standard_normal(n).astype(np.float32) for n in ((3, C), (3, C), C))
    h, q, s = norm_ref(x, r, w, 1e-6)
    bx, br, bw, bq, bs = be.upload(x), be.upload(r), be.upload(w), marked(be, 3 * ld16(C)), marked(be, 12)
    assert be.dispatch("rmsnorm_forward_i8", [bx, br, bw, br if where == "residual" else bx, bq, bs,
                                              be.params(3, C, ld16(C), 1), be.upload(np.float32([1e-6]))], (3,), (256,)) == 0
    assert np.array_equal((br if where == "residual" else bx).read(np.float32).reshape(3, C), h)
    assert np.array_equal((bx if where == "residual" else br).read(np.float32).reshape(3, C),
                          x if where == "residual" else r)
    check_codes(bq, q, ld16(C), C)
    assert (np.abs(bs.read(np.float32) - s) <= 4 * U32 * s).all()


def test_rmsnorm_of_large_and_small_rows(be):
    """Rows whose squares pass fp32's range on either side, and one with a NaN and an infinity each."""
    rng = np.random.default_rng(3)
    C = 1000
    x = rng.standard_normal((6, C)).astype(np.float32)
    x[1] *= np.float32(1e25)
    x[2] *= np.float32(1e-25)
    x[3, 7], x[4, 999] = np.nan, -np.inf
    w = rng.uniform(0.5, 1.5, C).astype(np.float32)
    h, q, s = norm_ref(x, None, w, 1e-5)
    bq, bs = marked(be, 6 * ld16(C)), marked(be, 24)
    assert be.dispatch("rmsnorm_forward_i8", [be.upload(x), bq, be.upload(w), bq, bq, bs, be.params(6, C, ld16(C), 0),
                                              be.upload(np.float32([1e-5]))], (6,), (256,)) == 0
    check_codes(bq, q, ld16(C), C)
    got, ok = bs.read(np.float32), [0, 1, 2, 5]
    assert np.isnan(got[3:5]).all() and (np.abs(got[ok] - s[ok]) <= 4 * U32 * s[ok]).all()


# silu's exponential is taken of -g, whose product with log2(e) is rounded: |g| log2(e) half steps of the exponential, g
# up to 40 here; its own error, the sum, the quotient and the products are within 8 more
def SILU2(g):
    return (g * 1.4427 + 8) * U32


SILU = SILU2(40)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,C", SHAPES)
def test_swiglu(be, M, C, bf16):
    rng = np.random.default_rng(M * 13 + C)
    g, u = (np.clip(rows(rng, M, C), -40, 40) for _ in range(2))
    if bf16:
        g, u = from_bf16(to_bf16(g)), from_bf16(to_bf16(u))
    p = g.astype(np.float64) / (1 + np.exp(-g.astype(np.float64))) * u
    top = np.abs(p).max(axis=1)
    inv = np.where(top > 1e-35, 127 / np.where(top > 0, top, 1), 0)
    name = "swiglu_forward_i8" + ("_bf16" if bf16 else "")
    esz = 2 if bf16 else 4
    stacked = np.concatenate([g, u], axis=1)
    for ld, lead in ((2 * C, 0), (2 * C + 3, 1)):
        src = be.upload(strided(to_bf16(stacked) if bf16 else stacked, ld, np.uint16 if bf16 else np.float32, lead))
        bq, bs = marked(be, M * ld16(C) + 16), marked(be, 4 * M + 16)
        assert be.dispatch(name, [src, src, bq, bs, be.params(M, C, ld, ld16(C))], (M,), (256,),
                           offsets=[lead * esz, (lead + C) * esz, 0, 0, 0]) == 0
        raw = bq.read(np.int8)
        q = raw[:M * ld16(C)].reshape(M, ld16(C))
        assert not q[:, C:].any() and (raw[M * ld16(C):] == MARK).all()
        # a rounding to the nearest code of a value that is off by both p's and the maximum's error, of at most 127 each
        assert (np.abs(q[:, :C] - p * inv[:, None]) <= 0.5 + 127 * (2 * SILU + 4 * U32)).all()
        s = bs.read(np.float32, M)
        assert (np.abs(s - np.where(inv > 0, top / 127, 0)) <= (SILU + 2 * U32) * top / 127).all()
        assert (bs.read(np.uint8)[4 * M:] == MARK).all()


def test_swiglu_accuracy(be):
    """Rows of one value: their scale is silu(g) / 127.  The exponential is good to a unit (two half steps), its
    correction, the sum, the quotient and the scale round once each: six half steps, from g of -64 on."""
    rng = np.random.default_rng(8)
    g = np.concatenate([rng.uniform(-64, 90, 200000), rng.standard_normal(200000) * 3, 10.0 ** rng.uniform(-6, 30, 1000),
                        -(10.0 ** rng.uniform(-6, 1.8, 1000))]).astype(np.float32)
    n = g.size
    bq, bs = be.alloc(n * 16), be.alloc(n * 4)
    assert be.dispatch("swiglu_forward_i8", [be.upload(g), be.upload(np.ones(n, np.float32)), bq, bs,
                                             be.params(n, 1, 1, 16)], (n,), (256,)) == 0
    g64 = g.astype(np.float64)
    want = np.abs(g64 / (1 + np.exp(-g64))) / 127
    err = np.abs(bs.read(np.float32) - want) / want
    print("largest error in half steps: %.2f at %g" % (err.max() / U32, g[err.argmax()]))
    assert err.max() <= 6 * U32


def test_swiglu_limits(be):
    """Gates far out on both sides, and NaN and infinities."""
    g = np.array([[-200, -1e30, 1e30, 90], [np.nan, 1, 1, 1], [-np.inf, 1, 1, 1], [1, 1, 1, 1], [-104, -104, -90, -88]],
                 np.float32)
    u = np.array([[3, 4, 1e-30, -2], [1, 1, 1, 1], [1, 1, 1, 1], [1, np.inf, 1, 1], [1, -1, 2, 3]], np.float32)
    bq, bs = marked(be, 5 * 16), marked(be, 20)
    assert be.dispatch("swiglu_forward_i8", [be.upload(g), be.upload(u), bq, bs, be.params(5, 4, 4, 16)], (5,), (256,)) == 0
    q, s = bq.read(np.int8).reshape(5, 16)[:, :4], bs.read(np.float32)
    assert q[0].tolist() == [0, 0, 1, -127] and abs(s[0] - 180 / 127) < 1e-5  # 1 of 180 / 127 rounds to 1
    assert np.isnan(s[1:4]).all() and not q[1:4].any()
    # 264 exp(-88) = 1.6e-36 still has a grid (from 3.8e-37 on), and 180 exp(-90) is a tenth of it
    assert abs(s[4] - 264 * np.exp(-88.0) / 127) <= SILU2(90) * s[4] + 2.0 ** -149
    assert q[4].tolist() == [0, 0, -12, -127]


MATMULS = [(1, 1, 1), (1, 16, 3), (1, 960, 200), (1, 2560, 960), (2, 17, 16), (3, 576, 1536), (5, 1001, 77), (8, 960, 333),
           (15, 100, 31), (16, 64, 64), (17, 63, 65), (31, 65, 130), (32, 128, 128), (33, 127, 129), (48, 2000, 50),
           (63, 960, 960), (64, 2560, 64), (65, 576, 250), (100, 1000, 515), (128, 256, 256), (130, 4095, 200),
           (200, 1536, 576), (256, 512, 256), (257, 513, 259), (300, 33, 1000), (511, 960, 513), (600, 2048, 1024),
           (1024, 640, 1100)]


def product_ref(a, sa, w, sw, bias):
    y = a.astype(np.float64) @ w.astype(np.float64).T * sa.astype(np.float64)[:, None] * sw
    return y, y if bias is None else y + bias


def check_product(got, y, want, bf16, bias):
    """fp32 roundings: the sum's conversion, two products, the bias; then bf16."""
    tol = 3 * U32 * 1.01 * np.abs(y) + (U32 * 1.01 * np.abs(want) if bias else 0)
    if bf16:
        tol = tol + (np.abs(want) + tol) * UB16
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,C,OC", MATMULS)
def test_matmul(be, M, C, OC, bf16):
    """Every code (-128 too), garbage behind the codes of a row, packed rows and odd strides, with and without a bias."""
    rng = np.random.default_rng(M + 1009 * C + OC)
    sa, sw = np.exp(rng.uniform(-8, 1, M)).astype(np.float32), np.exp(rng.uniform(-8, 1, OC)).astype(np.float32)
    b = rng.standard_normal(OC).astype(np.float32)
    bsa, bsw, bb = be.upload(sa), be.upload(sw), be.upload(b)
    dt = np.uint16 if bf16 else np.float32
    for bias, pad, opad, lead in ((False, 0, 0, 0), (True, 16, 3, 1), (True, 48, 8, 4)):
        lda, ldw, ldo = ld16(C) + pad, ld16(C) + 2 * pad, OC + opad
        a, w = (rng.integers(-128, 128, (n, ld)).astype(np.int8) for n, ld in ((M, lda), (OC, ldw)))
        out = marked(be, (lead + M * ldo) * dt(0).itemsize)
        assert be.dispatch("matmul_forward_i8" + ("_bf16" if bf16 else ""), [
            be.upload(a), bsa, be.upload(w), bsw, bb, out, be.params(M, C, OC, int(bias), lda, ldw, ldo)], (OC, M), (256,),
            offsets=[0, 0, 0, 0, 0, lead * dt(0).itemsize, 0]) == 0
        raw = out.read(dt)
        got = raw[lead:lead + M * ldo].reshape(M, ldo)
        assert (raw[:lead].view(np.uint8) == MARK).all()
        assert (np.ascontiguousarray(got[:, OC:]).view(np.uint8) == MARK).all()
        y, want = product_ref(a[:, :C], sa, w[:, :C], sw, b if bias else None)
        check_product(from_bf16(got[:, :OC]) if bf16 else got[:, :OC], y, want, bf16, bias)


# rows, outputs, and sums of every count of stages up to a full turn of the rings and past it: few rows or outputs, tiles of
# 32 x 32, 32 x 64, 64 x 64, 128 x 64, 128 x 128 (stages of 64 columns, of 128) and 256 x 256, ragged on both sides
FORMS = [(9, 700), (13, 16399), (70, 1000), (200, 600), (395, 800), (700, 1000), (1000, 1300), (1601, 1590), (3300, 3290)]
SUMS = [1, 15, 64, 65, 100, 128, 129, 200, 257, 300, 384, 400, 450, 513, 576, 640, 700, 770, 832, 900, 1001, 1024, 1100, 1300,
        1500, 2050, 3001]


@pytest.mark.parametrize("M,OC", FORMS)
def test_matmul_every_form(be, M, OC):
    """Whole sums (scales of one), for equality: random codes' sums are whole fp32 numbers, in numpy's products too."""
    rng = np.random.default_rng(M)
    ld = ld16(max(SUMS))
    a, w = rng.integers(-128, 128, (M, ld)).astype(np.int8), rng.integers(-128, 128, (OC, ld)).astype(np.int8)
    ba, bw, one = be.upload(a), be.upload(w), be.upload(np.ones(max(M, OC), np.float32))
    fa, fw = a.astype(np.float32), w.astype(np.float32)
    out = marked(be, M * OC * 4)
    for C in SUMS:
        if M * OC > 10 ** 7 and C > 1024 and C != 1500:  # the largest of them: a product in numpy takes half a second
            continue
        assert be.dispatch("matmul_forward_i8", [ba, one, bw, one, one, out, be.params(M, C, OC, 0, ld, ld, OC)], (OC, M),
                           (256,)) == 0
        got = out.read(np.float32).reshape(M, OC)
        want = fa[:, :C] @ fw[:, :C].T
        assert np.abs(want).max() < 2 ** 24
        assert np.array_equal(got, want), (C, np.argwhere(got != want)[:4])


@pytest.mark.parametrize("M,OC", [(9, 700), (200, 600), (1000, 1300)])
def test_matmul_rounds_each_step(be, M, OC):
    """The sum, its product with the row's scale, that with the channel's, and the bias: four fp32 values, equal to
    numpy's, whatever the form."""
    rng = np.random.default_rng(M)
    C = 300
    a, w = rng.integers(-128, 128, (M, ld16(C))).astype(np.int8), rng.integers(-128, 128, (OC, ld16(C))).astype(np.int8)
    sa, sw = np.exp(rng.uniform(-3, 1, M)).astype(np.float32), np.exp(rng.uniform(-3, 1, OC)).astype(np.float32)
    b = (rng.standard_normal(OC) * 1e4).astype(np.float32)
    out = marked(be, M * OC * 4)
    assert be.dispatch("matmul_forward_i8", [be.upload(a), be.upload(sa), be.upload(w), be.upload(sw), be.upload(b), out,
                                             be.params(M, C, OC, 1, ld16(C), ld16(C), OC)], (OC, M), (256,)) == 0
    want = (a[:, :C].astype(np.float32) @ w[:, :C].astype(np.float32).T) * sa[:, None] * sw + b  # sums below 2^24: exact
    assert want.dtype == np.float32 and np.array_equal(out.read(np.float32).reshape(M, OC), want)


# one round of tiles on 256 CUs, ragged on both sides, where every sum takes that form: 32 x 32, 32 x 64, 64 x 64, 128 x 64,
# 128 x 128, 256 x 256
@pytest.mark.parametrize("M,OC", [(500, 500), (500, 1020), (1000, 1020), (2000, 1020), (2000, 2040), (4000, 4090)])
def test_matmul_one_round_of_tiles(be, M, OC):
    test_matmul_every_form(be, M, OC)


@pytest.mark.parametrize("M,C,OC", [(1, 4096, 1000), (16, 8000, 2000), (33, 4660, 446), (17, 3499, 2000), (9, 3500, 770),
                                    (67, 6978, 1216), (40, 2801, 2003), (38, 2405, 1432), (173, 1374, 704), (42, 2047, 2630),
                                    (42, 2048, 2630), (3, 1100, 20000), (16, 300, 14300), (4, 800, 14337), (15, 2100, 16399)])
def test_matmul_few_outputs(be, M, C, OC):
    """Both sides of every border of the forms for few rows or outputs, for equality."""
    rng = np.random.default_rng(M + OC)
    ld = ld16(C) + 16
    a, w = rng.integers(-100, 101, (M, ld)).astype(np.int8), rng.integers(-100, 101, (OC, ld)).astype(np.int8)
    one, out = be.upload(np.ones(max(M, OC), np.float32)), marked(be, M * OC * 4 + 64)
    assert be.dispatch("matmul_forward_i8", [be.upload(a), one, be.upload(w), one, one, out,
                                             be.params(M, C, OC, 0, ld, ld, OC)], (OC, M), (256,)) == 0
    want = (a[:, :C].astype(np.float64) @ w[:, :C].astype(np.float64).T).astype(np.float32)
    raw = out.read(np.float32)
    assert np.array_equal(raw[:M * OC].reshape(M, OC), want) and (raw[M * OC:].view(np.uint8) == MARK).all()


@pytest.mark.parametrize("M,OC", [(1000, 5100), (2000, 4000), (2000, 4400), (193, 48003), (33001, 250)])
def test_matmul_one_round_of_wide_tiles(be, M, OC):
    """The same for 128 x 192, 256 x 128 and 192 x 192, which take sums from 512 on."""
    test_matmul_every_form(be, M, OC)


@pytest.mark.parametrize("M,OC", [(500, 500), (500, 1020), (1000, 1020), (2000, 1020)])
def test_matmul_wide_stages(be, M, OC):
    """Long sums of one tile a CU, stages of 256 columns: 5 to 13 of them, whole and ragged."""
    rng = np.random.default_rng(OC)
    sums = [1280, 1281, 1536, 1599, 1792, 1793, 2047, 2048, 2049, 2305, 2560, 2561, 2830, 3080]
    ld = ld16(max(sums)) + 48
    a, w = rng.integers(-100, 101, (M, ld)).astype(np.int8), rng.integers(-100, 101, (OC, ld)).astype(np.int8)
    ba, bw, one, out = be.upload(a), be.upload(w), be.upload(np.ones(max(M, OC), np.float32)), marked(be, M * OC * 4)
    fa, fw = a.astype(np.float32), w.astype(np.float32)
    for C in sums:
        assert be.dispatch("matmul_forward_i8", [ba, one, bw, one, one, out, be.params(M, C, OC, 0, ld, ld, OC)], (OC, M),
                           (256,)) == 0
        want = fa[:, :C] @ fw[:, :C].T  # magnitudes of at most 100: sums of 3080 products below 2^25, these below 2^24
        assert np.abs(want).max() < 2 ** 24
        got = out.read(np.float32).reshape(M, OC)
        assert np.array_equal(got, want), (C, np.argwhere(got != want)[:4])


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,OC", [(4100, 5123), (5123, 4100), (2000, 9001), (4096, 4353), (257 * 256, 300)])
def test_matmul_in_two_parts(be, M, OC, bf16):
    """More 256 x 256 tiles than CUs and the rest beside them or below: scales, bias and outputs are each part's own."""
    rng = np.random.default_rng(M)
    C, ldo = 330, OC + 3
    a, w = rng.integers(-128, 128, (M, ld16(C))).astype(np.int8), rng.integers(-128, 128, (OC, ld16(C))).astype(np.int8)
    sa, sw = np.exp(rng.uniform(-3, 1, M)).astype(np.float32), np.exp(rng.uniform(-3, 1, OC)).astype(np.float32)
    b = (rng.standard_normal(OC) * 1e4).astype(np.float32)
    out = marked(be, M * ldo * (2 if bf16 else 4))
    assert be.dispatch("matmul_forward_i8" + ("_bf16" if bf16 else ""), [
        be.upload(a), be.upload(sa), be.upload(w), be.upload(sw), be.upload(b), out,
        be.params(M, C, OC, 1, ld16(C), ld16(C), ldo)], (OC, M), (256,)) == 0
    want = (a[:, :C].astype(np.float32) @ w[:, :C].astype(np.float32).T) * sa[:, None] * sw + b  # sums below 2^24: exact
    got = out.read(np.uint16 if bf16 else np.float32)[:M * ldo].reshape(M, ldo)
    assert np.array_equal(got[:, :OC], to_bf16(want) if bf16 else want)
    assert (np.ascontiguousarray(got[:, OC:]).view(np.uint8) == MARK).all()


@pytest.mark.parametrize("far", [1 << 23, (1 << 23) + 16])
def test_matmul_largest_tiles_over_far_rows(be, far):
    test_matmul_tiles_over_far_rows(be, 3900, 3850, far)


@pytest.mark.parametrize("M,OC", [(20, 16390), (33, 10250), (64, 16384), (65, 20010), (128, 49152), (129, 40000), (16400, 16),
                                  (16384, 33), (33000, 64), (33000, 65), (40000, 128), (40000, 130)])
def test_matmul_narrow_outputs(be, M, OC):
    """Few rows by many outputs and few outputs of many rows: tiles no wider than there are, for equality."""
    rng = np.random.default_rng(M + OC)
    C, ld = 333, 336
    a, w = rng.integers(-128, 128, (M, ld)).astype(np.int8), rng.integers(-128, 128, (OC, ld)).astype(np.int8)
    one, out = be.upload(np.ones(max(M, OC), np.float32)), marked(be, M * OC * 4 + 64)
    assert be.dispatch("matmul_forward_i8", [be.upload(a), one, be.upload(w), one, one, out,
                                             be.params(M, C, OC, 0, ld, ld, OC)], (OC, M), (256,)) == 0
    want = a[:, :C].astype(np.float32) @ w[:, :C].astype(np.float32).T
    raw = out.read(np.float32)
    assert np.array_equal(raw[:M * OC].reshape(M, OC), want) and (raw[M * OC:].view(np.uint8) == MARK).all()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_matmul_longest_sums(be, M):
    """The longest row of the lowest codes stays inside 32 bits, and its sum is exact."""
    C, OC = 131071, 40
    a, w = np.full((M, 131072), -128, np.int8), np.full((OC, 131072), -128, np.int8)
    w[1::2] = 127
    one = be.upload(np.ones(max(M, OC), np.float32))
    out = marked(be, M * OC * 4)
    assert be.dispatch("matmul_forward_i8", [be.upload(a), one, be.upload(w), one, one, out,
                                             be.params(M, C, OC, 0, 131072, 131072, OC)], (OC, M), (256,)) == 0
    got = out.read(np.float32).reshape(M, OC)
    assert (got[:, 0::2] == np.float32(128 * 128 * C)).all() and (got[:, 1::2] == np.float32(-128 * 127 * C)).all()


@pytest.mark.parametrize("M", [1, 3])
def test_matmul_rows_past_32_bits(be, M):
    """Rows of tokens, weights and outputs whose offsets pass 2^31 and 2^32 bytes."""
    C, OC, far = 100, 3, 1 << 30
    rng = np.random.default_rng(5)
    a, w = rng.integers(-128, 128, (M, 112)).astype(np.int8), rng.integers(-128, 128, (OC, 112)).astype(np.int8)
    one = be.upload(np.ones(4, np.float32))

    def spread(x):
        big, src = be.alloc((x.shape[0] - 1) * far + 112), be.upload(x)
        for r in range(x.shape[0]):
            assert be.dispatch("copy_buffer", [src, big, be.params(112, dtype=np.int64)], (112,), (256,),
                               offsets=[r * 112, r * far, 0]) == 0
        return big

    out = be.alloc(((M - 1) * far + OC) * 4)
    assert be.dispatch("matmul_forward_i8", [spread(a), one, spread(w), one, one, out, be.params(M, C, OC, 0, far, far, far)],
                       (OC, M), (256,)) == 0
    small = be.alloc(M * 12)
    for r in range(M):
        assert be.dispatch("copy_buffer", [out, small, be.params(12, dtype=np.int64)], (12,), (256,),
                           offsets=[4 * r * far, 12 * r, 0]) == 0
    assert np.array_equal(small.read(np.float32).reshape(M, OC), (a[:, :C].astype(np.int64) @ w[:, :C].astype(np.int64).T))


@pytest.mark.parametrize("M,OC,far", [(20, 2100, 1 << 29), (3300, 3290, 1 << 23), (3300, 3290, (1 << 23) + 16)])
def test_matmul_tiles_over_far_rows(be, M, OC, far):
    """Tiles whose tokens' rows lie far apart: past 2^32 bytes from the first, at the widest stride of the largest tiles
    and just past it."""
    C = 100
    rng = np.random.default_rng(far)
    a, w = rng.integers(-128, 128, (M, 112)).astype(np.int8), rng.integers(-128, 128, (OC, 112)).astype(np.int8)
    big, src, one = be.alloc((M - 1) * far + 112), be.upload(a), be.upload(np.ones(max(M, OC), np.float32))
    k, p, enc = be.kernel("copy_buffer"), be.params(112, dtype=np.int64), be.encoder()
    for r in range(M):
        assert enc.dispatch(k, [src, big, p], (112,), (256,), [r * 112, r * far, 0]) == 0
    enc.commit()
    enc.wait_timed()
    out = be.alloc(M * OC * 4)
    assert be.dispatch("matmul_forward_i8", [big, one, be.upload(w), one, one, out, be.params(M, C, OC, 0, far, 112, OC)],
                       (OC, M), (256,)) == 0
    want = a[:, :C].astype(np.float32) @ w[:, :C].astype(np.float32).T
    assert np.array_equal(out.read(np.float32).reshape(M, OC), want)
    big.free()


def test_quantize_rows_past_32_bits(be):
    """Rows of the source 2^31 bytes apart and of the codes 2^30."""
    M, C, far = 3, 50, 1 << 29
    x = np.random.default_rng(6).standard_normal((M, C)).astype(np.float32)
    q, top, _ = grid(x)
    big, codes, src, bs = be.alloc(((M - 1) * far + C) * 4), be.alloc((M - 1) * 2 * far + 64), be.upload(x), marked(be, 12)
    back, small = be.alloc(((M - 1) * far + C) * 4), be.alloc(M * 200)
    for r in range(M):
        assert be.dispatch("copy_buffer", [src, big, be.params(200, dtype=np.int64)], (200,), (256,),
                           offsets=[r * 200, 4 * r * far, 0]) == 0
    assert be.dispatch("quantize_rows_i8", [big, codes, bs, be.params(M, C, far, 2 * far)], (M,), (256,)) == 0
    assert be.dispatch("dequantize_rows_i8", [codes, bs, back, be.params(M, C, 2 * far, far)], (M,), (256,)) == 0
    for r in range(M):
        assert be.dispatch("copy_buffer", [back, small, be.params(200, dtype=np.int64)], (200,), (256,),
                           offsets=[4 * r * far, r * 200, 0]) == 0
    s = top / np.float32(127)
    assert np.array_equal(bs.read(np.float32), s)
    assert np.array_equal(small.read(np.float32).reshape(M, C), q.astype(np.float32) * s[:, None])


def test_more_rows_than_workgroups(be):
    """More rows than a launch has workgroups: every one is taken."""
    M, C = (1 << 20) + 777, 4
    x = (np.arange(M * C, dtype=np.int64) % 1013 - 500).astype(np.float32).reshape(M, C)
    q, top, fine = grid(x)
    bq, bs, back = be.alloc(M * 16), be.alloc(M * 4), be.alloc(M * C * 4)
    assert be.dispatch("quantize_rows_i8", [be.upload(x), bq, bs, be.params(M, C, C, 16)], (M,), (256,)) == 0
    assert np.array_equal(bq.read(np.int8).reshape(M, 16)[:, :C], q)
    s = np.where(fine, top / np.float32(127), 0).astype(np.float32)
    assert np.array_equal(bs.read(np.float32), s)
    assert be.dispatch("dequantize_rows_i8", [bq, bs, back, be.params(M, C, 16, C)], (M,), (256,)) == 0
    assert np.array_equal(back.read(np.float32).reshape(M, C), q.astype(np.float32) * s[:, None])


@pytest.mark.parametrize("name,M,C", [("quantize_rows_i8", 700, 9000), ("quantize_rows_i8", 600, 13000),
                                      ("quantize_rows_i8_bf16", 530, 17000), ("quantize_rows_i8", 40001, 150),
                                      ("quantize_rows_i8_bf16", 33000, 500)])
def test_quantize_rows_in_turns(be, name, M, C):
    """More rows than the CUs hold, in the forms whose workgroups take several in turn."""
    x = np.random.default_rng(C).standard_normal((M, C)).astype(np.float32)
    bf16 = name.endswith("bf16")
    if bf16:
        x = from_bf16(to_bf16(x))
    q, top, _ = grid(x)
    bq, bs = marked(be, M * ld16(C) + 16), marked(be, 4 * M)
    assert be.dispatch(name, [be.upload(to_bf16(x) if bf16 else x), bq, bs, be.params(M, C, C, ld16(C))], (M,), (256,)) == 0
    assert np.array_equal(bs.read(np.float32), top / np.float32(127))
    got = bq.read(np.int8)
    assert (got[M * ld16(C):] == MARK).all()
    got = got[:M * ld16(C)].reshape(M, ld16(C))
    assert np.array_equal(got[:, :C], q) and not got[:, C:].any()


@pytest.mark.parametrize("M,C", [(33333, 60), (40001, 150), (600, 8200)])
def test_rmsnorm_in_turns(be, M, C):
    rng = np.random.default_rng(C)
    x, r = rng.standard_normal((M, C)).astype(np.float32), rng.standard_normal((M, C)).astype(np.float32)
    w = rng.uniform(-1.5, 1.5, C).astype(np.float32)
    h, q, s = norm_ref(x, r, w, float(np.float32(1e-5)))
    bh, bq, bs = be.upload(r), marked(be, M * ld16(C)), marked(be, 4 * M)
    assert be.dispatch("rmsnorm_forward_i8", [be.upload(x), bh, be.upload(w), bh, bq, bs, be.params(M, C, ld16(C), 1),
                                              be.upload(np.float32([1e-5]))], (M,), (256,)) == 0
    assert np.array_equal(bh.read(np.float32).reshape(M, C), h)
    got = bq.read(np.int8).reshape(M, ld16(C))
    assert np.array_equal(got[:, :C], q) and not got[:, C:].any()
    assert (np.abs(bs.read(np.float32) - s) <= 4 * U32 * s).all()


@pytest.mark.parametrize("name,C", [("quantize_rows_i8", 300), ("quantize_rows_i8_bf16", 2049), ("rmsnorm_forward_i8", 270),
                                    ("rmsnorm_forward_i8_bf16", 600), ("swiglu_forward_i8_bf16", 1030)])
def test_rows_past_the_largest_launch(be, name, C):
    """2^20 rows are a launch's most workgroups where a wave or more takes a row: the first and last rows of more than that
    (those between are zeros)."""
    extra = 130
    M, ldq, esz = (1 << 20) + extra, ld16(C), 2 if name.endswith("bf16") else 4
    rng = np.random.default_rng(C)
    x, w = rng.standard_normal((2 * extra, C)).astype(np.float32), rng.uniform(0.5, 1.5, C).astype(np.float32)
    if esz == 2:
        x = from_bf16(to_bf16(x))
    src, few = be.alloc(M * C * esz), be.upload(to_bf16(x) if esz == 2 else x)
    half = extra * C * esz
    for at, to in ((0, 0), (half, (M - extra) * C * esz)):
        assert be.dispatch("copy_buffer", [few, src, be.params(half, dtype=np.int64)], (half,), (256,), offsets=[at, to, 0]) == 0
    codes, bs, back = be.alloc(M * ldq), be.alloc(4 * M), be.alloc(2 * extra * ldq)
    if name.startswith("quantize"):
        bufs, p = [src, codes, bs, be.params(M, C, C, ldq)], x
    elif name.startswith("rmsnorm"):
        bufs, p = [src, src, be.upload(w), src, codes, bs, be.params(M, C, ldq, 0), be.upload(np.float32([1e-5]))], x * w
    else:
        bufs = [src, src, codes, bs, be.params(M, C, C, ldq)]
        x64 = x.astype(np.float64)
        p = x64 / (1 + np.exp(-x64)) * x64
    assert be.dispatch(name, bufs, (M,), (256,)) == 0
    half = extra * ldq
    for at, to in ((0, 0), ((M - extra) * ldq, half)):
        assert be.dispatch("copy_buffer", [codes, back, be.params(half, dtype=np.int64)], (half,), (256,),
                           offsets=[at, to, 0]) == 0
    got, s = back.read(np.int8).reshape(2 * extra, ldq), bs.read(np.float32)
    assert not got[:, C:].any() and not s[extra:-extra].any()
    s = np.concatenate([s[:extra], s[-extra:]])
    if name.startswith("swiglu"):
        top = np.abs(p).max(axis=1)
        assert (np.abs(got[:, :C] - p * (127 / top)[:, None]) <= 0.5 + 127 * (2 * SILU + 4 * U32)).all()
        assert (np.abs(s - top / 127) <= (SILU + 2 * U32) * top / 127).all()
        return
    q, top, _ = grid(p)
    assert np.array_equal(got[:, :C], q)
    if name.startswith("rmsnorm"):
        want = top / (127 * np.sqrt((x.astype(np.float64) ** 2).mean(axis=1) + float(np.float32(1e-5))))
        assert (np.abs(s - want) <= 4 * U32 * want).all()
    else:
        assert np.array_equal(s, top / np.float32(127))


def mlp_buffers(be, rng, N, D, H):
    """A layer's MLP: its inputs, weights quantized on the device, and the dispatches in order."""
    x, r = to_bf16(rng.standard_normal((N, D))), rng.standard_normal((N, D)).astype(np.float32)
    g = rng.uniform(0.5, 1.5, D).astype(np.float32)
    w1, w2 = (rng.standard_normal(n).astype(np.float32) * 0.05 for n in ((2 * H, D), (D, H)))
    c = {}
    calls = []
    for k, w in (("1", w1), ("2", w2)):
        c["w" + k], c["s" + k] = be.alloc(w.shape[0] * ld16(w.shape[1])), be.alloc(4 * w.shape[0])
        calls.append(("quantize_rows_i8", [be.upload(w), c["w" + k], c["s" + k],
                                           be.params(*w.shape, w.shape[1], ld16(w.shape[1]))], None))
    h, q1, c1, gu = be.upload(r), be.alloc(N * ld16(D)), be.alloc(4 * N), be.alloc(N * 4 * H)
    q2, c2, y = be.alloc(N * ld16(H)), be.alloc(4 * N), be.alloc(N * D * 4)
    calls += [
        ("rmsnorm_forward_i8_bf16", [be.upload(x), h, be.upload(g), h, q1, c1, be.params(N, D, ld16(D), 1),
                                     be.upload(np.float32([1e-5]))], None),
        ("matmul_forward_i8_bf16", [q1, c1, c["w1"], c["s1"], c["s1"], gu,
                                    be.params(N, D, 2 * H, 0, ld16(D), ld16(D), 2 * H)], None),
        ("swiglu_forward_i8_bf16", [gu, gu, q2, c2, be.params(N, H, 2 * H, ld16(H))], [0, 2 * H, 0, 0, 0]),
        ("matmul_forward_i8", [q2, c2, c["w2"], c["s2"], c["s2"], y, be.params(N, H, D, 0, ld16(H), ld16(H), D)], None),
    ]
    return x, r, g, w1, w2, h, y, calls


@pytest.mark.parametrize("N,D,H", [(1, 576, 1536), (7, 100, 270), (64, 960, 2560), (130, 576, 1536)])
def test_mlp_run_together(be, N, D, H):
    """A decoder layer's MLP in one encoder, its weights quantized by the same path: every kernel's outputs against 64
    bits of what the kernel before it left (a value at a border of bf16 or of a grid may go to either side, and with a
    row's largest value all its codes, so the ends alone say little)."""
    rng = np.random.default_rng(N + D)
    x, r, g, w1, w2, h, y, calls = mlp_buffers(be, rng, N, D, H)
    enc = be.encoder()
    for name, bufs, off in calls:
        assert enc.dispatch(be.kernel(name), bufs, (N,), (256,), off) == 0
    enc.commit()
    enc.wait_timed()

    def codes(buf, n, c):
        return buf.read(np.int8).reshape(n, ld16(c))[:, :c]

    wq = []
    for (_, (_, q, s, _), _), w in zip(calls[:2], (w1, w2)):
        want, top, _ = grid(w)
        assert np.array_equal(codes(q, *w.shape), want) and np.array_equal(s.read(np.float32), top / np.float32(127))
        wq.append((want, top / np.float32(127)))
    (_, norm, _), (_, up, _), (_, act, _), (_, down, _) = calls[2:]
    hs, q1, s1 = norm_ref(from_bf16(x).reshape(N, D), r, g, float(np.float32(1e-5)))
    assert np.array_equal(h.read(np.float32).reshape(N, D), hs) and np.array_equal(codes(norm[4], N, D), q1)
    c1 = norm[5].read(np.float32)
    assert (np.abs(c1 - s1) <= 4 * U32 * s1).all()
    gu = from_bf16(up[5].read(np.uint16)).reshape(N, 2 * H)
    check_product(gu, *product_ref(q1, c1, *wq[0], None), True, False)
    g64 = gu.astype(np.float64)
    p = g64[:, :H] / (1 + np.exp(-g64[:, :H])) * g64[:, H:]
    top = np.abs(p).max(axis=1)
    q2, c2 = codes(act[2], N, H), act[3].read(np.float32)
    assert (np.abs(q2 - p * (127 / top)[:, None]) <= 0.5 + 127 * (2 * SILU + 4 * U32)).all()
    assert (np.abs(c2 - top / 127) <= (SILU + 2 * U32) * top / 127).all()
    check_product(y.read(np.float32).reshape(N, D), *product_ref(q2, c2, *wq[1], None), False, False)


def test_runs_kept_in_flight_and_two_contexts(be):
    """Passes over the same buffers committed behind one another, and the same work on another context's stream at the
    same time, give what one pass alone gives."""
    rng = np.random.default_rng(11)
    N, D, H = 70, 192, 500
    *_, y, calls = mlp_buffers(be, rng, N, D, H)
    other = bmhip.Backend()
    try:
        *_, y2, calls2 = mlp_buffers(other, np.random.default_rng(11), N, D, H)

        def commit(b, cs):
            enc = b.encoder()
            for name, bufs, off in cs:
                assert enc.dispatch(b.kernel(name), bufs, (N,), (256,), off) == 0
            enc.commit()
            return enc

        commit(be, calls).wait_timed()
        want = y.read(np.uint8)
        # (the residual was summed in place: from here on the norm's sum and what follows from it is another)
        prod, prod2 = calls[-1:], calls2[-1:]
        commit(other, calls2).wait_timed()
        assert np.array_equal(y2.read(np.uint8), want)
        encs = [commit(b, cs) for _ in range(20) for b, cs in ((be, prod), (other, prod2))]
        for e in encs:
            e.wait_timed()
        assert np.array_equal(y.read(np.uint8), want) and np.array_equal(y2.read(np.uint8), want)
        del calls2, prod2, y2
    finally:
        other.close()


@pytest.mark.parametrize("lo,hi", [(64, 80), (80, 87), (87, 92), (92, 112)])
def test_swiglu_accuracy_of_far_gates(be, lo, hi):
    """silu under -64, down to where it is nothing, in rows of one value times 2^40 (exact), which keeps their scales off the
    border of rows without a grid.  The exponential is good to a unit (two half steps), its correction, the product with g and
    the scale round once each: five, and one for what the correction leaves out.  Under fp32's normal range silu is rounded to
    a multiple of 2^-149."""
    n = 100000
    g = -np.random.default_rng(lo).uniform(lo, hi, n).astype(np.float32)
    bq, bs = be.alloc(n * 16), be.alloc(n * 4)
    assert be.dispatch("swiglu_forward_i8", [be.upload(g), be.upload(np.full(n, 2.0 ** 40, np.float32)), bq, bs,
                                             be.params(n, 1, 1, 16)], (n,), (256,)) == 0
    g64 = g.astype(np.float64)
    want = np.abs(g64 / (1 + np.exp(-g64))) * 2.0 ** 40 / 127
    err = np.abs(bs.read(np.float32) - want)
    print("largest error in half steps: %.2f" % (err / (U32 * want + 2.0 ** (40 - 150) / 127)).max())
    assert (err <= 6 * U32 * want + 2.0 ** (40 - 150) / 127).all()


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
def test_swiglu_codes_of_far_gates(be, bf16):
    """Rows of far gates alone: codes off the nearest by the errors of the value and of the row's largest, of 127 at most."""
    rng = np.random.default_rng(5)
    M, C = 300, 500
    g, u = -rng.uniform(64, 80, (M, C)).astype(np.float32), rng.uniform(-1e3, 1e3, (M, C)).astype(np.float32)
    g[:, 7] = g.max(axis=1)  # neighbours of the largest gate, so that a row has more than one code but 0
    for k in range(1, C, 3):
        g[:, k] = g[:, 7] - rng.uniform(0, 1, M).astype(np.float32)
    if bf16:
        g, u = from_bf16(to_bf16(g)), from_bf16(to_bf16(u))
    p = g.astype(np.float64) / (1 + np.exp(-g.astype(np.float64))) * u
    top = np.abs(p).max(axis=1)
    cast = to_bf16 if bf16 else np.copy
    bq, bs = be.alloc(M * ld16(C)), be.alloc(M * 4)
    assert be.dispatch("swiglu_forward_i8" + ("_bf16" if bf16 else ""), [be.upload(cast(g)), be.upload(cast(u)), bq, bs,
                                                                         be.params(M, C, C, ld16(C))], (M,), (256,)) == 0
    q = bq.read(np.int8).reshape(M, ld16(C))[:, :C]
    # silu 5 half steps, its product with up 1; twice (value, largest); the grid's factor 2, its product 1
    assert (np.abs(q - p * (127 / top)[:, None]) <= 0.5 + 127 * 16 * U32).all()

@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("C", [5, 300, 20011, 40001])
def test_quantize_rows_up_to_the_largest_number(be, C, bf16):
    """Rows whose largest value lies over 2^126, so that its reciprocal is subnormal, up to the type's largest."""
    rng = np.random.default_rng(C)
    tops = np.array([2.0 ** 126, 2.0 ** 126 * 1.01, 1e38, 1.7e38, 2.0 ** 127, 3e38, 3.3895314e38, 3.4028235e38], np.float32)
    x = (rng.uniform(-1, 1, (8, C)).astype(np.float32) * tops[:, None]).astype(np.float32)
    x[:, C // 2] = -tops
    if bf16:
        x[7, C // 2] = 3.3895314e38  # bf16's largest
        x = from_bf16(to_bf16(np.clip(x, -3.3895314e38, 3.3895314e38)))
    q, top, fine = grid(x)
    assert fine.all() and (np.abs(q).max(axis=1) == 127).all()
    bq, bs = marked(be, 8 * ld16(C)), marked(be, 32)
    assert be.dispatch("quantize_rows_i8" + ("_bf16" if bf16 else ""), [be.upload(to_bf16(x) if bf16 else x), bq, bs,
                                                                        be.params(8, C, C, ld16(C))], (8,), (256,)) == 0
    check_codes(bq, q, ld16(C), C)
    assert np.array_equal(bs.read(np.float32), top / np.float32(127))
