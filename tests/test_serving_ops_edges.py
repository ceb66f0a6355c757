"""Calls of the operators on the caller's device buffers that lie at the edge of what include/hip_decode.h allows, as far as no GPU
is needed: the kernels' own source on the CPU under ASan (tests/kernel_emu/*_edges.cpp), one check per test."""
import ctypes as C
import os
import re
import subprocess
import threading

import pytest

from rustane_amd import hipdec
from rustane_amd.hipdec import KvDtype, PagedCache, RowDtype
from test_kernel_emulation import EMU, ROOT, host_clang
from test_serving_ops import FAKE, attention, refused, verify


@pytest.fixture(scope="module")
def emulated(tmp_path_factory):
    cxx = host_clang()
    if cxx is None:
        pytest.skip("no clang++ for the host (the kernel text uses clang's vector types)")
    build = tmp_path_factory.mktemp("serving_ops_edges")
    for name in ("paged", "verify", "wave64"):
        text = open(os.path.join(ROOT, "rustane_amd", "csrc", "hipdec_%s.h" % name)).read()
        (build / ("kernel_%s.inc" % name)).write_text(re.sub(r"^#(pragma once|include .*)$", "", text, flags=re.M))
    pool = open(os.path.join(EMU, "paged_cache.cpp")).read()
    (build / "paged_pool.inc").write_text(pool[:pool.index("template <int HD")])
    built = {}
    # products and sums fused where the GPU's compiler fuses them, if this machine can
    fused = ["-mfma", "-ffp-contract=fast-honor-pragmas"] if re.search(r"^flags.* fma ", open("/proc/cpuinfo").read(), re.M) else []

    def check(program, name):
        if program not in built:
            cmd = [cxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                   "-fno-omit-frame-pointer", "-pthread", "-Wno-psabi", *fused, "-I", str(build), "-I", EMU,
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


def test_tiny_temperatures_with_a_saturated_soft_cap(emulated):
    emulated("verify_edges", "tiny_temperatures")


def test_soft_cap_and_exponential_are_right_to_64_bits(emulated):
    emulated("verify_edges", "elementary_accuracy")


def test_an_infinite_logit_is_the_largest_at_temperature_zero(emulated):
    emulated("verify_edges", "greedy_infinities")


def test_what_lies_too_far_below_the_maximum_has_no_probability(emulated):
    emulated("verify_edges", "far_below_the_maximum")


def test_verification_with_eight_logits_a_lane(emulated):
    emulated("verify_edges", "eight_logits_a_lane")


# ---------------------------------------------------------------- sizes at the launches' limits (no GPU: the host decides)
HUGE = 1 << 62                # workspace bytes


@pytest.mark.parametrize("kw,text", [
    # a launch counts its threads in 32 bits, and every launch of a call is looked at before the first
    (dict(n_seqs=9_000_000, max_drafts=0, vocab=256), "out of range"),       # the decision's workgroups of 512
    (dict(n_seqs=8_388_607, max_drafts=0, vocab=256), "device"),
    (dict(n_seqs=9_000_000, max_drafts=0, vocab=256, temperature=0.0), "out of range"),
    (dict(n_seqs=(1 << 24) - 1, max_drafts=1, vocab=1024), "out of range"),  # the statistics' of 256
    (dict(n_seqs=1 << 17, max_drafts=0, vocab=131071, dtype=RowDtype.BF16), "device"),   # 2^17 rows of 128 chunks, four to a workgroup
    (dict(n_seqs=1 << 19, max_drafts=0, vocab=131071, dtype=RowDtype.BF16), "out of range"),
])
def test_verification_counts_its_launches_as_they_are(kw, text):
    refused(lambda: verify(workspace_bytes=HUGE, **kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(n_rows=8192, heads=32, max_len=131072), "device"),                 # 8192 x 8 x 128 workgroups of 256
    (dict(n_rows=16384, heads=32, max_len=131072), "out of range"),
    (dict(n_rows=1 << 20, heads=8, max_len=250), "out of range"),            # one launch: 2^20 x 8 workgroups of 512 are one too many,
    (dict(n_rows=(1 << 20) - 1, heads=8, max_len=250), "device"),
    (dict(n_rows=1 << 20, heads=8, max_len=250, hd=256, kv_dtype=KvDtype.F32), "device"),    # ... of 256 are not
    (dict(n_rows=1 << 24, heads=8, max_len=1), "out of range"),
])
def test_attention_counts_its_launches_as_they_are(kw, text):
    kw = dict(kw)
    hd, dt = kw.pop("hd", 128), kw.pop("kv_dtype", KvDtype.BF16)
    c = PagedCache.make(FAKE, FAKE, dt, n_pages=4, page_size=16, kv_heads=8, hd=hd, page_table=FAKE, n_seqs=2, max_pages=2)
    refused(lambda: attention(cache=c, workspace=FAKE, workspace_bytes=HUGE, **kw), text)


# ---------------------------------------------------------------- rotary positions
def test_rotated_rows_are_off_by_their_roundings_only(emulated):
    emulated("paged_edges", "rotation_roundings")


# ---------------------------------------------------------------- texts of failed calls
def on_a_thread_of_its_own(call):
    out = []
    t = threading.Thread(target=lambda: out.append(call()))
    t.start()
    t.join()
    return out[0]


def test_any_thread_is_told_why_a_model_was_not_created():
    lib = hipdec.load_library()
    cfg, out = hipdec.Config.make(dim=64, hidden=64, heads=1, hd=64, seq=8, nlayers=2, vocab=8), C.c_void_p()
    text = lambda: lib.hipdec_last_error(None)  # noqa: E731

    def create(n_layers):
        one = (C.c_float * 1)()
        head = hipdec._Head(C.cast(one, C.POINTER(C.c_float)), C.cast(one, C.POINTER(C.c_float)))
        layers = (hipdec._Layer * 1)()
        return lib.hipdec_create(C.byref(cfg), layers, n_layers, C.byref(head), None, C.byref(out)), text()

    # the creating thread, and one that has not failed in anything itself
    rc, told = on_a_thread_of_its_own(lambda: create(7))
    assert rc == hipdec.ERR_ARG and b"layer count" in told
    assert b"layer count" in on_a_thread_of_its_own(text)
    # an operator's failure is the failing thread's own: it hides neither the other's text nor, later, its own creation's
    def operator_then_create():
        refused(lambda: attention(scale=0.0), "scale")
        mine, other = text(), on_a_thread_of_its_own(text)
        on_a_thread_of_its_own(lambda: create(9))
        return mine, other, text(), create(8)[1], on_a_thread_of_its_own(text)
    mine, other, still, later, told = on_a_thread_of_its_own(operator_then_create)
    assert b"scale" in mine and b"scale" in still and b"layer count" in other and b"layer count" in later and b"layer count" in told
    assert not out.value


# ---------------------------------------------------------------- one buffer for two things
def test_attention_in_place_needs_one_stride():
    wide = 8 * 128
    refused(lambda: attention(q_stride=wide, out_stride=wide + 8), "in place")
    refused(lambda: attention(q_stride=wide + 8, out_stride=wide), "in place")
    refused(lambda: attention(q_stride=wide + 8, out_stride=wide + 8), "device")                  # (allowed; the address is no device memory)
    refused(lambda: attention(n_rows=1, q_stride=wide + 8, out_stride=wide), "device")            # one row: no stride is used


def test_a_workspace_past_64_bits_is_refused_not_wrapped():
    sizes = []
    for n_rows, heads, kv_heads, hd, max_len in ((1 << 24, 65536, 1, 512, 1 << 30), (1 << 24, 65536, 65536, 512, 1 << 30), (1 << 24, 65536, 1, 510, 1 << 29)):
        refused(lambda: hipdec.attention_paged_workspace(n_rows, heads, kv_heads, hd, max_len), "out of range")
    for shift in range(0, 25):                               # up to there it grows with the rows
        try:
            sizes.append(hipdec.attention_paged_workspace(1 << shift, 65536, 8, 256, 1 << 26))
        except hipdec.HipDecodeError:
            sizes.append(1 << 64)
    assert sizes == sorted(sizes) and sizes[12] < 1 << 64
