# SPDX-License-Identifier: MPL-2.0
"""Registers of the kernels over paged caches, as the compiler reports them (no GPU).  Nothing is spilled: a spill costs time
in the loop over the keys, and the compiler has put one between the ends of a branch that some lanes do not take, which lost
the other lanes' values."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"


def kernels(name, path):
    """{mangled name: (waves per SIMD, spilled registers, scratch bytes a lane)}"""
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Wall", "-Wno-unused-function", "-Xclang",
                        "-target-feature", "-Xclang", "-packed-fp32-ops", "-I", os.path.join(ROOT, "include"),
                        "-Rpass-analysis=kernel-resource-usage", "--offload-device-only", "-c",
                        os.path.join(ROOT, "bare.metal_amd", "csrc", name), "-o", path], capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0 and "warning:" not in r.stderr, r.stderr[-2000:]
    return {p.split()[0]: (int(re.search(r"Occupancy \[waves/SIMD\]: (\d+)", p).group(1)),
                           int(re.search(r"VGPRs Spill: (\d+)", p).group(1)),
                           int(re.search(r"ScratchSize \[bytes/lane\]: (\d+)", p).group(1)))
            for p in r.stderr.split("Function Name: ")[1:]}


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_attention_keeps_everything_in_registers(tmp_path):
    forms = {}
    for n, u in kernels("attn_paged.hip", str(tmp_path / "a.o")).items():
        if "k_attn_paged_plan" in n:
            assert u[1:] == (0, 0)
            continue
        m = re.match(r"\S*k_attn_pagedILb(\d)ELi(\d+)E", n)
        forms[bool(int(m.group(1))), int(m.group(2))] = u
    assert {f: u[0] for f, u in forms.items()} == {(True, 64): 3, (True, 128): 2, (True, 256): 1, (False, 64): 2,
                                                   (False, 128): 1, (False, 256): 1}
    assert all(u[1:] == (0, 0) for u in forms.values()), forms


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_rotations_keep_everything_in_registers(tmp_path):
    forms = kernels("rope_rows.hip", str(tmp_path / "r.o"))
    assert forms and all("k_rope_rows" in n and u[1:] == (0, 0) for n, u in forms.items()), forms
