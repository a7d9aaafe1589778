# SPDX-License-Identifier: MPL-2.0
"""Whole passes of an MLP on the 8-bit integer path, committed behind one another and on two contexts at once.  In a file of its
own behind test_zz_no_alloc.py, which reads the device's free memory: the runtime serves small allocations from blocks of 2 MiB
and keeps freed ones, so what this test frees before it would hide the allocation that it looks for."""
import numpy as np
import pytest

import bmhip
from test_i8_gpu import MARK, mlp_buffers, to_bf16

pytestmark = pytest.mark.gpu


def test_whole_passes_in_flight_on_two_contexts(be):
    """Twenty passes of the MLP committed behind one another on each of two contexts at the same time, over the same
    intermediate buffers, which every pass overwrites with values of its own: three inputs in turn, others on the other
    context.  Each pass's output and sum, kept apart, are what the same pass gives alone."""
    N, D, H, passes = 70, 192, 500, 20
    other = bmhip.Backend()
    try:
        runs = []
        for b, seed in ((be, 12), (other, 13)):
            rng = np.random.default_rng(seed)
            *_, res, _, calls = mlp_buffers(b, rng, N, D, H)
            xs = [b.upload(to_bf16(rng.standard_normal((N, D)))) for _ in range(3)]
            ys, hs = (b.upload(np.full(passes * N * D * 4, MARK, np.uint8)) for _ in range(2))
            runs.append((b, calls, xs, res, ys, hs))

        def commit(run, x, at):
            """One pass over input x, its output and sum at the given place; weights are quantized anew as well."""
            b, calls, xs, res, ys, hs = run
            enc = b.encoder()
            for name, bufs, off in calls:
                if name.startswith("rmsnorm"):
                    bufs, off = [xs[x], res, bufs[2], hs] + bufs[4:], [0, 0, 0, at, 0, 0, 0, 0]
                if name == "matmul_forward_i8":
                    bufs, off = bufs[:5] + [ys] + bufs[6:], [0, 0, 0, 0, 0, at, 0]
                assert enc.dispatch(b.kernel(name), bufs, (N,), (256,), off) == 0
            enc.commit()
            return enc

        size, want = N * D * 4, []
        for run in runs:
            alone = []
            for x in range(3):
                commit(run, x, 0).wait_timed()
                alone.append((run[4].read(np.uint8)[:size], run[5].read(np.uint8)[:size]))
                run[4].write(np.full(size, MARK, np.uint8))
                run[5].write(np.full(size, MARK, np.uint8))
            want.append(alone)
        every = [y for alone in want for pair in alone for y in pair]
        assert len({y.tobytes() for y in every}) == 12 and all((y != MARK).any() for y in every)
        encs = [commit(run, p % 3, p * size) for p in range(passes) for run in runs]
        for e in encs:
            e.wait_timed()
        for run, alone in zip(runs, want):
            for buf, which in ((run[4], 0), (run[5], 1)):
                got = buf.read(np.uint8).reshape(passes, size)
                for p in range(passes):
                    assert np.array_equal(got[p], alone[p % 3][which]), (which, p)
        del runs, run, calls, xs, ys, hs, res, b
    finally:
        other.close()
