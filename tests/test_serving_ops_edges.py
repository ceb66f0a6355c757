"""Calls of the operators on the caller's device buffers that lie at the edge of what include/hip_decode.h allows, as far as no GPU
is needed: the kernels' own source on the CPU under ASan (tests/kernel_emu/*_edges.cpp), one check per test."""
import os
import re
import subprocess

import pytest

from test_kernel_emulation import EMU, ROOT, host_clang


@pytest.fixture(scope="module")
def emulated(tmp_path_factory):
    cxx = host_clang()
    if cxx is None:
        pytest.skip("no clang++ for the host (the kernel text uses clang's vector types)")
    build = tmp_path_factory.mktemp("serving_ops_edges")
    for name in ("paged", "verify", "wave64"):
        text = open(os.path.join(ROOT, "rustane_amd", "csrc", "hipdec_%s.h" % name)).read()
        (build / ("kernel_%s.inc" % name)).write_text(re.sub(r"^#(pragma once|include .*)$", "", text, flags=re.M))
    built = {}

    def check(program, name):
        if program not in built:
            cmd = [cxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                   "-fno-omit-frame-pointer", "-pthread", "-Wno-psabi", "-I", str(build), "-I", EMU,
                   os.path.join(EMU, program + ".cpp"), "-o", str(build / program)]
            r = subprocess.run(cmd, capture_output=True, text=True)
            assert r.returncode == 0, r.stderr[-4000:]
            built[program] = str(build / program)
        r = subprocess.run([built[program], name], capture_output=True, text=True, timeout=900)
        assert r.returncode == 0 and "%s: 0 wrong" % name in r.stdout, (r.stdout[-4000:], r.stderr[-3000:])
    return check


# ---------------------------------------------------------------- verification of drafts
def test_negative_probabilities_and_random_numbers_count_as_zero(emulated):
    emulated("verify_edges", "negative_numbers")
