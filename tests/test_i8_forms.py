# SPDX-License-Identifier: MPL-2.0
"""Every kernel of the product of 8-bit codes (matmul_forward_i8, _bf16), each at shapes for which the rules are asserted to
choose it, so that a change of the rules shows here.  On the GPU: random scales of tokens and channels, a bias, ragged sides,
strides of their own, both output types, for equality with the same fp32 steps in numpy (the sums stay below 2^24, where fp32
products and sums of whole numbers are exact)."""
import ctypes

import numpy as np
import pytest

import bmhip

MARK = 0x5A


def ld16(c):
    return (c + 15) // 16 * 16


def to_bf16(x):
    """fp32 -> bf16 bits, round to nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + np.uint32(0x7FFF) + ((u >> 16) & np.uint32(1))) >> 16).astype(np.uint16)


def kernels(M, C, OC, lda, ldw):
    """(kernel, rows, columns) of a product's launches."""
    q = bmhip.lib().bmk_matmul_i8_kernel
    q.restype, q.argtypes = ctypes.c_char_p, [ctypes.c_int] * 6 + [ctypes.POINTER(ctypes.c_int)] * 2
    out = []
    while True:
        r, c = ctypes.c_int(), ctypes.c_int()
        name = q(M, C, OC, lda, ldw, len(out), ctypes.byref(r), ctypes.byref(c))
        if name is None:
            return out
        out.append((name.decode(), r.value, c.value))


def sums(stage, first, last):
    """Sums of `first` to `last` stages, the last of them holding one column, all, or something between."""
    tails = (1, stage, 17, stage - 1, 16, stage // 2 + 3, 15, stage - 16)
    return [(n - 1) * stage + tails[(n - first) % len(tails)] for n in range(first, last + 1)]


# kernel, rows, outputs, sums, row strides a multiple of 128 bytes
ONE = [
    ("few 4", 37, 1203, sums(64, 1, 20), False),  # up to a 16 x 16 tile for each CU
    ("few 4", 3, 20005, sums(64, 1, 10), False),  # up to three rows
    ("few 4", 15, 7001, sums(64, 1, 10), False),  # up to sixteen
    ("few 4", 131, 503, sums(64, 1, 10), False),  # short sums
    ("few 8", 37, 1203, sums(64, 56, 73), False),
    ("32x32 128", 499, 501, sums(128, 1, 9), False),  # one round
    ("32x32 128", 4446, 68, sums(128, 1, 8), False),  # more
    ("32x32 256", 499, 501, sums(256, 6, 12), False),
    ("32x64 128", 141, 5597, sums(128, 1, 8), False),
    ("32x64 256", 34, 4247, sums(256, 6, 12), False),
    ("64x64 128", 129, 4902, sums(128, 1, 8), False),
    ("64x64 256", 103, 4147, sums(256, 9, 14), False),
    ("128x64 128", 5273, 322, sums(128, 1, 8), False),
    ("128x64 256", 582, 1709, sums(256, 7, 13), False),
    ("128x64 128", 582, 1709, sums(128, 13, 20), True),
    ("128x64 256", 582, 1709, sums(256, 17, 19), True),
    ("128x128 64", 4567, 839, sums(64, 1, 8), False),
    ("128x128 128", 5725, 324, sums(128, 5, 11), False),
    ("128x192", 5381, 659, sums(128, 5, 11), False),
    ("256x128", 3675, 1544, sums(128, 5, 11), False),
    ("192x192", 1634, 4741, sums(128, 5, 11), False),
    ("256x256", 3999, 4090, [320], False),  # five stages
    # six to fourteen: every count left behind the loop of ten, none among them; and none behind two loops
    ("256x256", 1753, 5007, sums(64, 6, 14) + sums(64, 22, 22), False),
]
# the full rounds of 256 x 256 tiles and the rest of the rows, or of the columns: rows, sum, outputs, the rest's kernel
TWO = [
    (9001, 330, 2000, "rows", "128x64 128"), (577, 1294, 25071, "rows", "128x128 128"), (35389, 1154, 513, "rows", "192x192"),
    (49569, 896, 321, "rows", "256x128"), (41301, 1078, 385, "rows", "128x192"), (32893, 1309, 326, "rows", "32x32 256"),
    (388, 1202, 37483, "columns", "128x128 128"), (385, 715, 41350, "columns", "128x192"),
    (292, 1127, 50027, "columns", "192x192"), (388, 718, 45059, "columns", "256x128"),
    (258, 502, 35247, "columns", "64x64 128"), (260, 1293, 34050, "columns", "32x64 256"),
]
NAMES = {"few 4", "few 8", "32x32 128", "32x32 256", "32x64 128", "32x64 256", "64x64 128", "64x64 256", "128x64 128",
         "128x64 256", "128x128 64", "128x128 128", "128x192", "256x128", "192x192", "256x256"}


def stride(longest, lines):
    """A row stride for sums up to `longest`, a multiple of 128 bytes or not."""
    ld = (longest + 127) // 128 * 128
    return ld if lines else ld + 48


@pytest.mark.parametrize("kernel,M,OC,Cs,lines", ONE)
def test_a_shape_takes_the_kernel_it_stands_for(kernel, M, OC, Cs, lines):
    ld = stride(max(Cs), lines)
    for C in Cs:
        assert kernels(M, C, OC, ld, ld) == [(kernel, M, OC)], C


@pytest.mark.parametrize("M,C,OC,cut,rest", TWO)
def test_a_shape_is_cut_as_it_stands_for(M, C, OC, cut, rest):
    (first, m, n), (second, m2, n2) = kernels(M, C, OC, stride(C, False), stride(C, False))
    assert (first, second) == ("256x256", rest)
    assert (m + m2, n, n2) == (M, OC, OC) if cut == "rows" else (m, m2, n + n2) == (M, M, OC)


def test_every_kernel_has_a_shape():
    """And no other is chosen for any shape."""
    assert {k for k, *_ in ONE} == NAMES
    rng = np.random.default_rng(0)
    for M, C, OC in np.exp(rng.uniform(0, np.log([70000, 131071, 70000]), (20000, 3))).astype(int).tolist():
        got = kernels(M, C, OC, ld16(C), ld16(C))
        assert {k for k, *_ in got} <= NAMES and sum(m * n for _, m, n in got) == M * OC
        assert len(got) == 1 or (len(got) == 2 and got[0][0] == "256x256")


class Inputs:
    """Codes, scales and a bias on the device, and products of them."""

    def __init__(self, be, M, OC, longest, lines):
        rng = np.random.default_rng(M * 7919 + OC)
        self.be, self.M, self.OC, self.ld, self.ldo, self.lead = be, M, OC, stride(longest, lines), OC + 3, 5
        a, w = (rng.integers(-128, 128, (n, self.ld)).astype(np.int8) for n in (M, OC))
        self.sa, self.sw = (np.exp(rng.uniform(-3, 1, n)).astype(np.float32) for n in (M, OC))
        self.b = (rng.standard_normal(OC) * 1e4).astype(np.float32)
        self.bufs = [be.upload(v) for v in (a, self.sa, w, self.sw, self.b)]
        self.fa, self.fw = a.astype(np.float32), w.astype(np.float32)

    def check(self, C, bf16, bias):
        be, M, OC, esz = self.be, self.M, self.OC, 2 if bf16 else 4
        n = (self.lead + M * self.ldo) * esz
        out = be.upload(np.full(ld16(n), MARK, np.uint8))
        assert be.dispatch("matmul_forward_i8" + ("_bf16" if bf16 else ""), self.bufs + [
            out, be.params(M, C, OC, int(bias), self.ld, self.ld, self.ldo)], (OC, M), (256,),
            offsets=[0, 0, 0, 0, 0, self.lead * esz, 0]) == 0
        want = self.fa[:, :C] @ self.fw[:, :C].T
        assert np.abs(want).max() < 2 ** 24
        want *= self.sa[:, None]
        want *= self.sw
        if bias:
            want += self.b
        raw = out.read(np.uint8)
        got = raw[self.lead * esz:n].view(np.uint16 if bf16 else np.float32).reshape(M, self.ldo)
        want = to_bf16(want) if bf16 else want
        assert np.array_equal(got[:, :OC], want), (C, np.argwhere(got[:, :OC] != want)[:4])
        assert (np.ascontiguousarray(got[:, OC:]).view(np.uint8) == MARK).all()
        assert (raw[:self.lead * esz] == MARK).all() and (raw[n:] == MARK).all()
        out.free()

    def free(self):
        for b in self.bufs:
            b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("kernel,M,OC,Cs,lines", ONE)
def test_kernel(be, kernel, M, OC, Cs, lines, bf16):
    i = Inputs(be, M, OC, max(Cs), lines)
    for k, C in enumerate(Cs):
        i.check(C, bf16, k % 3 != 2)
    i.free()


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,C,OC,cut,rest", TWO)
def test_two_launches(be, M, C, OC, cut, rest, bf16):
    i = Inputs(be, M, OC, C, False)
    i.check(C, bf16, True)
    i.free()


@pytest.mark.gpu
@pytest.mark.parametrize("far", ["tokens", "weights"])
def test_largest_tiles_over_the_farthest_rows(be, far):
    """256 x 256 tiles over rows at the widest stride they take, whose offsets inside a tile pass 2^31 bytes, and the stride
    past it, which other tiles take."""
    M, OC, C, at = 1753, 5007, 330, 1 << 23
    if far == "weights":
        M, OC = OC, M
    rng = np.random.default_rng(7)
    a, w = (rng.integers(-128, 128, (n, 336)).astype(np.int8) for n in (M, OC))
    want = a[:, :C].astype(np.float32) @ w[:, :C].astype(np.float32).T
    k, p, one = be.kernel("copy_buffer"), be.params(336, dtype=np.int64), be.upload(np.ones(5007, np.float32))
    near, src = be.upload(w if far == "tokens" else a), be.upload(a if far == "tokens" else w)
    for ld, pair in ((at, True), (at + 16, False)):
        n = M if far == "tokens" else OC
        big, enc, out = be.alloc((n - 1) * ld + 336), be.encoder(), be.alloc(M * OC * 4)
        for r in range(n):
            assert enc.dispatch(k, [src, big, p], (336,), (256,), [r * 336, r * ld, 0]) == 0
        enc.commit()
        enc.wait_timed()
        ops, lds = ([big, one, near, one], (ld, 336)) if far == "tokens" else ([near, one, big, one], (336, ld))
        assert [name == "256x256" for name, *_ in kernels(M, C, OC, *lds)] == [pair]
        assert be.dispatch("matmul_forward_i8", ops + [one, out, be.params(M, C, OC, 0, *lds, OC)], (OC, M), (256,)) == 0
        assert np.array_equal(out.read(np.float32).reshape(M, OC), want)
        big.free()
        out.free()
