# SPDX-License-Identifier: MPL-2.0
"""Serving from a paged cache (include/bm_paged.h) on the CPU: the rotary table against its formulas, the launchers'
refusals (made before they touch the GPU, so addresses that nothing reads do), and the tables' lookups, bad ones among
them, inside arrays of their own."""
import ctypes
import math
import random
from fractions import Fraction

import numpy as np
import pytest

import bmhip
from paged_exactness import SIX, deviation, emulated, last_bits, last_bits_off

MAX_BUFFERS = 12
BASE = 1 << 20  # an address on a 16-byte boundary


class Launch(ctypes.Structure):
    """bmk_launch_t (csrc/bmk.h)."""
    _fields_ = [("stream", ctypes.c_void_p), ("n", ctypes.c_int), ("dev", ctypes.c_void_p * MAX_BUFFERS),
                ("val", ctypes.c_void_p * MAX_BUFFERS), ("bytes", ctypes.c_size_t * MAX_BUFFERS),
                ("grid", ctypes.c_int * 3), ("tg", ctypes.c_int * 3), ("scratch", ctypes.c_void_p),
                ("scratch_bytes", ctypes.c_size_t)]


def launch(name, sizes, params, floats, shift=()):
    """The launcher's answer for buffers of the given sizes, the params and floats in the last two; shift: {buffer:
    bytes} added to its address."""
    fn = getattr(bmhip.lib(), "bmk_launch_" + name)
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_void_p]
    a = Launch()
    a.n = len(sizes) + 2
    keep, keep_f = np.array(params, np.int32), np.array(floats, np.float32)
    for i, n in enumerate(sizes):
        a.dev[i] = BASE + (1 << 44) * i + dict(shift).get(i, 0)
        a.bytes[i] = n
    at = len(sizes)
    a.val[at], a.bytes[at] = keep.ctypes.data, keep.nbytes
    a.val[at + 1], a.bytes[at + 1] = keep_f.ctypes.data, keep_f.nbytes
    return fn(ctypes.byref(a))


def refused(capfd, *args, **kw):
    """Refused for its arguments: -1 and a message, and no launch was tried."""
    capfd.readouterr()
    rc = launch(*args, **kw)
    said = capfd.readouterr().err
    assert rc == -1 and "ERROR" in said and "launch failed" not in said, (rc, said)


# each operator: launcher, buffer sizes of one call, its params, its floats
N, S, NH, NKV, HD, ROT, PAGE, COUNT, WIDTH = 5, 2, 6, 3, 16, 8, 8, 7, 3
Q, K = NH * HD, NKV * HD


def calls(e):
    cache, tables = COUNT * 2 * NKV * PAGE * HD * e, [4 * (S + 1), 4 * S, 4 * S * WIDTH]
    return {
        "rope_rows": ([N * Q * e, N * Q * e, 4 * N, 4 * ROT], [N, NH, HD, ROT, 0, Q, Q], [1.0]),
        "qk_norm_rope": ([N * Q * e, N * K * e, N * Q * e, N * K * e, 4 * N, 4 * ROT, 8 * HD],
                         [N, NH, NKV, HD, ROT, 0, Q, K, Q, K], [1.0, 1e-5]),
        "kv_append": ([N * Q * e, N * K * e, N * K * e, N * Q * e, cache] + tables + [4 * ROT, 8 * HD],
                      [N, S, NH, NKV, HD, ROT, 0, Q, K, K, Q, PAGE, COUNT, WIDTH, 1], [1.0, 1e-5]),
        "attn_paged": ([N * Q * e, cache, N * Q * e] + tables,
                       [N, S, NH, NKV, HD, Q, Q, PAGE, COUNT, WIDTH, 1, 0], [0.25]),
    }


CALLS = {k + s: (k + s,) + v for s, e in (("", 4), ("_bf16", 2)) for k, v in calls(e).items()}
IDS = list(CALLS)


def kind(op):
    return op.replace("_bf16", "")


@pytest.mark.parametrize("op", IDS)
def test_a_short_buffer_is_refused(op, capfd):
    name, sizes, params, floats = CALLS[op]
    for i in range(len(sizes)):
        refused(capfd, name, [n - (j == i) for j, n in enumerate(sizes)], params, floats)
    refused(capfd, name, sizes, params[:-1], floats)
    refused(capfd, name, sizes, params, floats[:-1])


@pytest.mark.parametrize("op", IDS)
def test_a_misaligned_offset_is_refused(op, capfd):
    """The cache off a 16-byte boundary, the turns off an 8-byte one, everything else off its element's."""
    name, sizes, params, floats = CALLS[op]
    cache = {"kv_append": 4, "attn_paged": 1}.get(kind(op))
    turns = {"rope_rows": 3, "qk_norm_rope": 5, "kv_append": 8}.get(kind(op))
    for i in range(len(sizes)):
        for by in {cache: (1, 2, 4, 8), turns: (1, 2, 4)}.get(i, (1,)):
            refused(capfd, name, [n + 64 for n in sizes], params, floats, {i: by})


# names of the params by operator
NAMES = {
    "rope_rows": "N NH HD rot layout ldx ldo".split(),
    "qk_norm_rope": "N NH NKV HD rot layout ldq ldk ldqo ldko".split(),
    "kv_append": "N S NH NKV HD rot layout ldq ldk ldv ldqo page n_pages max_pages norm".split(),
    "attn_paged": "N S NH NKV HD ldq ldo page n_pages max_pages causal window".split(),
}
BAD = {
    "N": [-1, (1 << 30) + 1], "S": [-1, 4097, (1 << 30) + 1], "NH": [-1, (1 << 30) + 1], "NKV": [0, -1, 4097],
    "HD": [0, -8, 258, 264, 7], "rot": [-2, 3, 18], "layout": [-1, 2], "page": [0, -8, 1, 4, 12, 131072],
    "n_pages": [0, -1, (1 << 31) - 1], "max_pages": [0, -1, (1 << 30)], "norm": [-1, 2], "causal": [-1, 2], "window": [-1],
}


@pytest.mark.parametrize("op", IDS)
def test_bad_shapes_are_refused(op, capfd):
    name, sizes, params, floats = CALLS[op]
    roomy = [1 << 43] * len(sizes)
    names = NAMES[kind(op)]
    for i, n in enumerate(names):
        values = list(BAD.get(n, []))
        if n == "NKV" and kind(op) == "qk_norm_rope":
            values = [0, -1, (1 << 30) + 1]
        if n == "NH" and kind(op) != "kv_append":  # no q is allowed there
            values.append(0)
        if n == "HD" and kind(op) in ("kv_append", "attn_paged"):
            values.append(20)  # even, no multiple of 8
        if n == "n_pages":
            values = [0, -1]
        if n.startswith("ld"):
            values = [params[i] - 1, -params[i], 0, (1 << 30) + 1]
        for v in values:
            p = list(params)
            p[i] = v
            refused(capfd, name, roomy, p, floats)
    if kind(op) == "attn_paged":
        for changes in ({"NH": 7}, {"causal": 0, "window": 4}):  # heads that no KV head serves evenly; a window without order
            p = list(params)
            for k, v in changes.items():
                p[names.index(k)] = v
            refused(capfd, name, roomy, p, floats)
    if kind(op) in ("qk_norm_rope", "kv_append"):
        for eps in (-1e-5, math.nan):
            refused(capfd, name, sizes, params, [1.0, eps])


@pytest.mark.parametrize("op", IDS)
def test_sizes_past_32_bits_do_not_wrap(op, capfd):
    """Byte counts past 32 bits are compared as such, and more heads in all than an index holds are refused."""
    name, sizes, params, floats = CALLS[op]
    names = NAMES[kind(op)]
    p = list(params)
    p[0] = 1 << 26
    refused(capfd, name, [1 << 31] * len(sizes), p, floats)
    p[names.index("NH")] = 48
    for i, n in enumerate(names):
        if n in ("ldq", "ldqo", "ldx", "ldo"):
            p[i] = 48 * HD
    refused(capfd, name, [1 << 43] * len(sizes), p, floats)
    if "n_pages" in names:  # a cache of 2^38 tokens
        p = list(params)
        p[names.index("n_pages")], p[names.index("page")] = 1 << 22, 65536
        p[names.index("max_pages")] = 1
        refused(capfd, name, [1 << 43] * len(sizes), p, floats)


@pytest.mark.parametrize("op", IDS)
def test_no_rows_are_nothing_to_do(op):
    name, sizes, params, floats = CALLS[op]
    assert launch(name, [0] * len(sizes), [0] + params[1:], floats) == 0
    if "S" in NAMES[kind(op)]:
        assert launch(name, [0] * len(sizes), [params[0], 0] + params[2:], floats) == 0


def test_operators_are_in_the_kernel_table():
    lib = bmhip.lib()
    lib.bmk_find.restype, lib.bmk_find.argtypes = ctypes.c_void_p, [ctypes.c_char_p]
    for n in ("rope_forward_rows", "qk_norm_rope_forward", "kv_append_paged", "attention_forward_paged"):
        assert lib.bmk_find(n.encode()) and lib.bmk_find((n + "_bf16").encode())


# ---------------------------------------------------------------- the rotary table

def frequency(i, rot, theta, scaling, factor, low, high, original):
    """Radians a position, by the formulas in floats."""
    f = theta ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor
    if scaling == "llama3":
        length = 2 * math.pi / f
        if length > original / low:
            return f / factor
        if length < original / high:
            return f
        t = (original / length - low) / (high - low)
        return (1 - t) * f / factor + t * f
    if scaling == "yarn":
        def pair(x):
            return rot * math.log(original / (2 * math.pi * x)) / (2 * math.log(theta))
        a, b = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rot - 1)
        t = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
        return (1 - t) * f + t * f / factor
    return f


@pytest.mark.parametrize("scaling", ["none", "linear", "llama3", "yarn"])
@pytest.mark.parametrize("rot,theta", [(0, 10000.0), (2, 10000.0), (20, 1.5), (64, 10000.0), (128, 500000.0), (256, 1e6)])
def test_rope_turns(rot, theta, scaling):
    how = dict(factor=8.0, low=1.0, high=4.0, original=8192.0)
    table, mscale = bmhip.rope_turns(rot, theta, scaling, **how)
    assert mscale == (np.float32(0.1 * math.log(8.0) + 1) if scaling == "yarn" else 1)
    for i in range(rot // 2):
        want = frequency(i, rot, theta, scaling, **how) / (2 * math.pi)
        got = Fraction(int(table[i]), 1 << 64)
        # a float power and a few float operations: within 2^-46 of the value
        assert abs(got - Fraction(want)) <= Fraction(want) / (1 << 46) + Fraction(1, 1 << 63), (i, float(got), want)


def test_rope_turns_whole_turns_drop_out():
    """Pair 0 turns by one radian a position: 1 / 2 pi of a turn, of 2^64."""
    table, _ = bmhip.rope_turns(64, 10000.0)
    assert abs(int(table[0]) - 0x28BE60DB9391054A) <= 2  # 2^64 / 2 pi = 2935890503282001226.4


def test_rope_turns_refusals():
    for bad in ((3, 1e4), (-2, 1e4), (64, 1.0), (64, 0.0), (64, math.nan), (64, math.inf), (64, 1e4, "linear", 0.5),
                (64, 1e4, "linear", math.inf), (64, 1e4, "llama3", 8.0, 4.0, 1.0, 8192.0),
                (64, 1e4, "llama3", 8.0, 0.0, 4.0, 8192.0), (64, 1e4, "yarn", 8.0, 1.0, 4.0, 0.0),
                (64, 1e4, "yarn", math.nan, 1.0, 4.0, 8192.0)):
        with pytest.raises(ValueError):
            bmhip.rope_turns(*bad)
    out = np.zeros(32, np.uint64)
    m = ctypes.c_float()
    f = bmhip.lib().bm_rope_turns
    assert f(64, 4, 1e4, 1, 1, 2, 1, out.ctypes.data, ctypes.byref(m)) == -1  # no such scaling
    assert f(64, -1, 1e4, 1, 1, 2, 1, out.ctypes.data, ctypes.byref(m)) == -1
    assert f(64, 0, 1e4, 1, 1, 2, 1, None, ctypes.byref(m)) == -1 and f(64, 0, 1e4, 1, 1, 2, 1, out.ctypes.data, None) == -1


# ---------------------------------------------------------------- the tables' lookups

def lookup(start, length, pages, page, n_pages, n, j):
    """Sequence, position and page, the tables in arrays with guards that no lookup may take for numbers of theirs."""
    out = np.zeros(3, np.int32)
    fn = bmhip.lib().bmk_paged_lookup
    fn.restype = None
    fn.argtypes = [ctypes.c_void_p] * 3 + [ctypes.c_int] * 6 + [ctypes.c_void_p]
    t = [np.ascontiguousarray(x, np.int32) for x in (start, length, pages)]
    fn(*[x.ctypes.data for x in t], len(length), page, n_pages, t[2].shape[1], n, j, out.ctypes.data)
    return tuple(int(v) for v in out)


def test_rows_find_their_sequence():
    rng = random.Random(5)
    for _ in range(200):
        counts = [rng.choice([0, 0, 1, 1, 2, 7]) for _ in range(rng.randint(1, 9))]
        lead = rng.choice([0, 0, 3])
        start = [lead + sum(counts[:s]) for s in range(len(counts) + 1)]
        length = [c + rng.randint(0, 9) for c in counts]
        pages = np.arange(len(counts) * 4, dtype=np.int32).reshape(-1, 4)
        for n in range(-1, start[-1] + 3):
            s, p, _ = lookup(start, length, pages, 4, 1000, n, 0)
            if lead <= n < start[-1]:
                assert start[s] <= n < start[s + 1] and p == length[s] - counts[s] + n - start[s]
            else:
                assert s == -1


def test_keys_find_their_page():
    pages = [[3, 0, 6], [9, -1, 7]]
    for s in (0, 1):
        for j in range(-5, 20):
            want = pages[s][j // 4] if 0 <= j < 12 else -1
            want = want if 0 <= want < 7 else -1  # 7 pages: 7 and 9 are none, nor is -1
            assert lookup([0, 1, 2], [12, 12], pages, 4, 7, s, j)[2] == want
    for j in (-(1 << 31), (1 << 31) - 1, 12, -1):
        assert lookup([0, 1, 2], [12, 12], pages, 4, 7, 0, j)[2] == -1
    for p in (-(1 << 31), (1 << 31) - 1):
        assert lookup([0, 1], [12], [[p]], 4, 7, 0, 0)[2] == -1


def test_lookups_stay_inside_any_table():
    """Tables of anything: a sequence inside the batch or none, a page inside the cache or none, no endless search."""
    rng = np.random.default_rng(3)
    for _ in range(2000):
        S, width, page = int(rng.integers(1, 9)), int(rng.integers(1, 5)), 1 << int(rng.integers(0, 6))
        wild = [np.iinfo(np.int32).min, np.iinfo(np.int32).max, -1, 0, 1, 5]
        start, length = rng.choice(wild, S + 1), rng.choice(wild, S)
        pages = rng.choice(wild, (S, width))
        n, j = int(rng.integers(0, 12)), int(rng.choice(wild))
        s, _, pg = lookup(start, length, pages, page, 5, n, j)
        assert -1 <= s < S and -1 <= pg < 5


# ---------------------------------------------------------------- launches

@pytest.mark.parametrize("lanes", [256, 512])
def test_a_launch_stays_under_the_work_items_of_an_axis(lanes):
    """HIP refuses 2^32 work-items or more along an axis: up to there one row of workgroups, then as few rows as take them,
    all workgroups among them and fewer over than there are rows."""
    fn = bmhip.lib().bmk_paged_grid
    fn.restype, fn.argtypes = None, [ctypes.c_longlong, ctypes.c_int, ctypes.c_void_p]
    most = ((1 << 32) - 1) // lanes
    # 2^30 heads by 64 lanes each; 4096 KV heads of 4096 sequences, with a part of a unit for each
    sizes = [1, 2, 255, most - 1, most, most + 1, 2 * most, 2 * most + 1, (1 << 30) * 64 // lanes, 4096 * (4096 + 32) + 3080]
    for groups in sizes + [random.Random(lanes).randrange(1, 1 << 28) for _ in range(200)]:
        xy = np.zeros(2, np.uint32)
        fn(groups, lanes, xy.ctypes.data)
        x, y = (int(v) for v in xy)
        assert x * lanes < 1 << 32 and groups <= x * y < groups + y and y == -(-groups // most) <= 65535, (groups, x, y)
    for log in range(7):  # the rotation: 2^30 heads by 1 << log lanes each; the first head of any workgroup stays inside an int
        slots = 512 >> log
        xy = np.zeros(2, np.uint32)
        fn((1 << 30) // slots, 512, xy.ctypes.data)
        assert int(xy[0]) * int(xy[1]) * slots < 1 << 31


@pytest.mark.parametrize("room,want,tries", [(1 << 40, 64, 1), (64, 64, 1), (63, 8, 2), (8, 8, 2), (7, 0, 2), (0, 0, 2)])
def test_scratch_memory_of_a_full_device(room, want, tries):
    """64 MiB, or where there is not that much the 8 that attention_forward cuts its work for, or none."""
    asked = []
    hook = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t)

    def alloc(p, n):
        asked.append(n)
        if n > room << 20:
            return 2  # out of memory
        p[0] = 4096
        return 0

    fn = bmhip.lib().bmk_scratch_alloc
    fn.restype, fn.argtypes = ctypes.c_size_t, [ctypes.c_void_p, hook]
    p = ctypes.c_void_p(7)
    assert fn(ctypes.byref(p), hook(alloc)) == want << 20 and len(asked) == tries
    assert p.value == (4096 if want else None)


# ---------------------------------------------------------------- what the fp32 attention's bound tells apart

FOUR = [(1, 1), (1, 0), (0, 1), (0, 0)]
THREE = [(1, 0), (0, 1), (0, 0)]


@pytest.mark.parametrize("HD", [8, 40, 64, 128, 256])
@pytest.mark.parametrize("keys", [2, 40, 300, 1500])
def test_the_bound_on_average_error_wants_all_six_products(HD, keys):
    """The kernel's arithmetic with all products of terms is within it; without the third terms' products, of the scores or of the
    values, or with three products alone, the error is past four times the mean that the roundings leave."""
    rng = np.random.default_rng(HD * 10000 + keys)
    rows = [tuple(rng.standard_normal(s).astype(np.float32) for s in (HD, (keys, HD), (keys, HD))) for _ in range(12)]
    scale = float(np.float32(HD ** -0.5))

    def ratio(*products):
        err = want = 0.0
        for q, k, v in rows:
            sc = k.astype(np.float64) @ q.astype(np.float64) * scale
            p = np.exp(sc - sc.max())
            err += (((p / p.sum()) @ v.astype(np.float64) - emulated(q, k, v, scale, *products)) ** 2).sum()
            want += (deviation(q, k, v, scale) ** 2).sum()
        return math.sqrt(err / want)

    assert ratio() < 1
    for left in (FOUR, THREE):
        assert min(ratio(left, SIX), ratio(SIX, left)) > 4, (ratio(left, SIX), ratio(SIX, left))


@pytest.mark.parametrize("HD", [8, 64, 256])
def test_scores_of_last_bits_want_their_third_terms(HD):
    rng = np.random.default_rng(HD)
    for in_key in (0, 1):
        worst = {0: 0.0, 1: 0.0, 2: 0.0}
        for _ in range(40):
            q, k, v = last_bits(rng, 1, 2 + int(rng.integers(0, 30)), HD, in_key)
            for n, products in enumerate((SIX, FOUR, THREE)):
                worst[n] = max(worst[n], last_bits_off(q[0], k, v, emulated(q[0], k, v, 1.0, products)))
        assert worst[0] < 1 and worst[1] > 1000 and worst[2] > 1000, worst
