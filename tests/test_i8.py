# SPDX-License-Identifier: MPL-2.0
"""The 8-bit integer path's refusals (include/bm_q8.h), on the CPU: the launchers check shapes, strides, alignment and
buffer sizes before they touch the GPU, so addresses that nothing reads do for them here."""
import ctypes

import numpy as np
import pytest

import bmhip

MAX_BUFFERS = 12
BASE = 1 << 20  # an address on a 16-byte boundary


class Launch(ctypes.Structure):
    """bmk_launch_t (csrc/bmk.h)."""
    _fields_ = [("stream", ctypes.c_void_p), ("n", ctypes.c_int), ("dev", ctypes.c_void_p * MAX_BUFFERS),
                ("val", ctypes.c_void_p * MAX_BUFFERS), ("bytes", ctypes.c_size_t * MAX_BUFFERS),
                ("grid", ctypes.c_int * 3), ("tg", ctypes.c_int * 3), ("scratch", ctypes.c_void_p),
                ("scratch_bytes", ctypes.c_size_t)]


def launch(name, sizes, params, par, eps=None, shift=()):
    """The launcher's answer for buffers of the given sizes (index par: the params, par + 1: eps); shift: {buffer:
    bytes} added to its address."""
    fn = getattr(bmhip.lib(), "bmk_launch_" + name)
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_void_p]
    a = Launch()
    a.n = len(sizes)
    keep = np.array(params, np.int32)
    keep_eps = np.array([eps or 0], np.float32)
    for i, n in enumerate(sizes):
        a.dev[i] = BASE + (1 << 36) * i + dict(shift).get(i, 0)
        a.bytes[i] = n
    a.val[par], a.bytes[par] = keep.ctypes.data, keep.nbytes
    if eps is not None:
        a.val[par + 1], a.bytes[par + 1] = keep_eps.ctypes.data, 4
    return fn(ctypes.byref(a))


def refused(capfd, *args, **kw):
    """Refused for its arguments: -1 and a message, and no launch was tried."""
    capfd.readouterr()
    rc = launch(*args, **kw)
    said = capfd.readouterr().err
    assert rc == -1 and "ERROR" in said and "launch failed" not in said, (rc, said)


# each operator: launcher, buffer sizes of one call, its params, their index, eps, what each buffer needs
M, C, LD = 5, 40, 48
CALLS = {
    "quantize": ("quantize_rows_i8", [4 * M * C, LD * M, 4 * M, 0], (M, C, C, LD), 3, None),
    "quantize_bf16": ("quantize_rows_i8_bf16", [2 * M * C, LD * M, 4 * M, 0], (M, C, C, LD), 3, None),
    "back": ("dequantize_rows_i8", [LD * M, 4 * M, 4 * M * C, 0], (M, C, LD, C), 3, None),
    "back_bf16": ("dequantize_rows_i8_bf16", [LD * M, 4 * M, 2 * M * C, 0], (M, C, LD, C), 3, None),
    "norm": ("rmsnorm_i8", [4 * M * C, 4 * M * C, 4 * C, 4 * M * C, LD * M, 4 * M, 0, 0], (M, C, LD, 1), 6, 1e-5),
    "norm_bf16": ("rmsnorm_i8_bf16", [2 * M * C, 4 * M * C, 4 * C, 4 * M * C, LD * M, 4 * M, 0, 0], (M, C, LD, 1), 6,
                  1e-5),
    "swiglu": ("swiglu_i8", [4 * M * C, 4 * M * C, LD * M, 4 * M, 0], (M, C, C, LD), 4, None),
    "swiglu_bf16": ("swiglu_i8_bf16", [2 * M * C, 2 * M * C, LD * M, 4 * M, 0], (M, C, C, LD), 4, None),
    "matmul": ("matmul_i8", [LD * M, 4 * M, LD * 7, 4 * 7, 4 * 7, 4 * M * 7, 0], (M, C, 7, 1, LD, LD, 7), 6, None),
    "matmul_bf16": ("matmul_i8_bf16", [LD * M, 4 * M, LD * 7, 4 * 7, 4 * 7, 2 * M * 7, 0], (M, C, 7, 1, LD, LD, 7), 6,
                    None),
}


@pytest.mark.parametrize("op", CALLS)
def test_a_short_buffer_is_refused(op, capfd):
    name, sizes, params, par, eps = CALLS[op]
    for i in range(par):
        refused(capfd, name, [n - (j == i) for j, n in enumerate(sizes)], params, par, eps)
    refused(capfd, name, sizes, params[:-1], par, eps)  # a params buffer of too few numbers


@pytest.mark.parametrize("op", CALLS)
def test_a_misaligned_offset_is_refused(op, capfd):
    """Codes off a 16-byte boundary, everything else off its element's."""
    name, sizes, params, par, eps = CALLS[op]
    roomy = [n + 64 for n in sizes]
    for i in range(par):
        if i in ({"quantize": [1], "back": [0], "norm": [4], "swiglu": [2], "matmul": [0, 2]}[op.split("_")[0]]):
            for by in (1, 4, 8):
                refused(capfd, name, roomy, params, par, eps, {i: by})
        else:
            refused(capfd, name, roomy, params, par, eps, {i: 1})


@pytest.mark.parametrize("op", CALLS)
def test_bad_shapes_are_refused(op, capfd):
    name, sizes, params, par, eps = CALLS[op]
    roomy = [1 << 40] * len(sizes)
    at = {"rows": 0, "columns": 1}
    bad = [(at["rows"], -1), (at["columns"], 0), (at["columns"], -3), (at["rows"], (1 << 30) + 1),
           (at["columns"], (1 << 30) + 1)]
    kind = op.split("_")[0]
    codes = {"quantize": [3], "back": [2], "norm": [2], "swiglu": [3], "matmul": [4, 5]}[kind]
    for k in codes:  # strides of codes: too short, no multiple of 16, negative
        bad += [(k, 32), (k, 40), (k, 56), (k, -48), (k, 0)]
    for k in {"quantize": [2], "back": [3], "swiglu": [2], "matmul": [6]}.get(kind, []):  # element strides under a row
        bad += [(k, params[k] - 1), (k, -params[k])]
    if kind == "matmul":
        bad += [(2, 0), (2, -1), (1, 131072), (2, (1 << 30) + 1)]
    for k, v in bad:
        p = list(params)
        p[k] = v
        refused(capfd, name, roomy, p, par, eps)


def test_int32_sizes_do_not_wrap(capfd):
    """Byte counts past 32 bits are compared as such."""
    for op, p in (("quantize", (1 << 20, 1 << 13, 1 << 13, 1 << 13)), ("back", (1 << 20, 1 << 13, 1 << 13, 1 << 13)),
                  ("matmul", (1 << 20, 1 << 12, 1 << 12, 0, 1 << 12, 1 << 12, 1 << 12))):
        name, sizes, _, par, eps = CALLS[op]
        refused(capfd, name, [1 << 31] * len(sizes), p, par, eps)


@pytest.mark.parametrize("op", CALLS)
def test_no_rows_are_nothing_to_do(op):
    name, sizes, params, par, eps = CALLS[op]
    assert launch(name, [0] * len(sizes), (0,) + tuple(params[1:]), par, eps) == 0


def test_operators_are_in_the_kernel_table():
    lib = bmhip.lib()
    lib.bmk_find.restype, lib.bmk_find.argtypes = ctypes.c_void_p, [ctypes.c_char_p]
    for n in ("quantize_rows_i8", "dequantize_rows_i8", "rmsnorm_forward_i8", "swiglu_forward_i8", "matmul_forward_i8"):
        assert lib.bmk_find(n.encode()) and lib.bmk_find((n + "_bf16").encode())
