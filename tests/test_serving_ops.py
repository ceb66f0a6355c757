"""The operators on the caller's device buffers (include/hip_decode.h: rotary positions with the append to a paged cache,
attention over it, verification of drafted tokens), as far as no GPU is needed: the kernels' own source run on the CPU
under ASan against fp64 restatements (bad page tables and odd inputs among them), every refusal of the entry points, the
frequencies against their formulas, and the workspace sizes."""
import ctypes as C
import concurrent.futures
import math
import os
import re
import subprocess

import numpy as np
import pytest

from rustane_amd import hipdec
from rustane_amd.hipdec import HipDecodeError, KvDtype, PagedCache, Rope, RopeScaling, RowDtype
from test_kernel_emulation import EMU, ROOT, host_clang


@pytest.fixture(scope="module")
def emulated(tmp_path_factory):
    cxx = host_clang()
    if cxx is None:
        pytest.skip("no clang++ for the host (the kernel text uses clang's vector types)")
    build = tmp_path_factory.mktemp("serving_ops_emu")
    for name in ("paged", "verify"):
        text = open(os.path.join(ROOT, "rustane_amd", "csrc", "hipdec_%s.h" % name)).read()
        (build / ("kernel_%s.inc" % name)).write_text(re.sub(r"^#(pragma once|include .*)$", "", text, flags=re.M))

    def compile_one(name):
        cmd = [cxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
               "-fno-omit-frame-pointer", "-pthread", "-Wno-psabi", "-I", str(build), "-I", EMU, os.path.join(EMU, name + ".cpp"),
               "-o", str(build / name)]
        return name, subprocess.run(cmd, capture_output=True, text=True)

    out = {}
    with concurrent.futures.ThreadPoolExecutor(2) as pool:
        for name, r in pool.map(compile_one, ("paged_cache", "verify_drafts")):
            assert r.returncode == 0, (name, r.stderr[-4000:])
            out[name] = str(build / name)
    return out


def test_paged_cache_kernels_source_on_the_cpu(emulated):
    r = subprocess.run([emulated["paged_cache"]], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and "0 checks failed" in r.stdout, (r.stdout[-4000:], r.stderr[-3000:])
    assert r.stdout.count("k_rope_append") == 5 and r.stdout.count("k_attn_paged<") >= 7


def test_draft_verification_kernels_source_on_the_cpu(emulated):
    r = subprocess.run([emulated["verify_drafts"]], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and "0 checks failed" in r.stdout, (r.stdout[-4000:], r.stderr[-3000:])
    assert r.stdout.count(" 0 mismatches") == 6


# ---------------------------------------------------------------- frequencies
@pytest.mark.parametrize("rot", [2, 64, 62, 128])
def test_frequencies_follow_their_formulas(rot):
    i = np.arange(rot // 2)
    plain = 10000.0 ** (-2.0 * i / rot)
    f, m = hipdec.rope_frequencies(rot)
    assert m == 1.0 and np.allclose(f, plain, rtol=1e-14)
    f, m = hipdec.rope_frequencies(rot, theta=500000.0, scaling=RopeScaling.LINEAR, factor=4.0)
    assert m == 1.0 and np.allclose(f, 500000.0 ** (-2.0 * i / rot) / 4.0, rtol=1e-14)
    if rot > 2:
        f, m = hipdec.rope_frequencies(rot, scaling=RopeScaling.BASE, factor=8.0)
        assert m == 1.0 and f[0] == 1.0                                    # the fastest pair stays,
        assert math.isclose(f[-1], plain[-1] / 8.0, rel_tol=1e-12)         # the slowest is divided by the factor
        assert np.all(np.diff(f) < 0)
    f, m = hipdec.rope_frequencies(rot, scaling=RopeScaling.PARTS, factor=8.0, trained=4096, slow_turns=1.0, fast_turns=32.0)
    turns = 4096 * plain / (2 * np.pi)
    keep = np.clip((turns - 1.0) / 31.0, 0, 1)
    assert np.allclose(f, plain * keep + plain / 8.0 * (1 - keep), rtol=1e-13)
    assert math.isclose(m, 0.1 * math.log(8.0) + 1.0, rel_tol=2.0 ** -24)
    # outside the mixed range: the library's own plain frequencies, bit for bit (numpy's powers differ from them by an ulp)
    own = hipdec.rope_frequencies(rot)[0]
    assert np.all(f[turns >= 32] == own[turns >= 32]) and np.all(f[turns <= 1] == own[turns <= 1] / 8)


def test_the_models_own_positions_are_the_plain_interleaved_form():
    # angle of pair i at position p: p * 10000^(-2 i / hd) (the oracle's table, built in fp32)
    f, _ = hipdec.rope_frequencies(128)
    p = np.arange(0, 2048, 37)[:, None]
    want = p.astype(np.float32) / np.power(np.float32(10000.0), (2 * np.arange(64) / np.float32(128)).astype(np.float32))
    assert np.max(np.abs(np.cos(p * f) - np.cos(want.astype(np.float64)))) < 2048 * 2.0 ** -22


# ---------------------------------------------------------------- refusals (no GPU: everything is refused on the host)
FAKE = 1 << 20                # stands for a device address: no call gets as far as using it


def cache(**kw):
    c = PagedCache.make(FAKE, FAKE, KvDtype.BF16, n_pages=4, page_size=16, kv_heads=2, hd=128, page_table=FAKE, n_seqs=2, max_pages=2)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def refused(call, text, status=hipdec.ERR_ARG):
    with pytest.raises(HipDecodeError) as e:
        call()
    assert e.value.status == status and text in str(e.value), str(e.value)


BAD_CACHES = [(dict(k=None), "null"), (dict(v=None), "null"), (dict(page_table=None), "null"), (dict(kv_dtype=2), "kv_dtype"),
              (dict(n_pages=0), "zero-sized"), (dict(kv_heads=0), "zero-sized"), (dict(hd=0), "zero-sized"), (dict(n_seqs=0), "zero-sized"),
              (dict(max_pages=0), "zero-sized"), (dict(n_pages=1 << 31), "too large"), (dict(page_size=0), "power of two"),
              (dict(page_size=12), "power of two"), (dict(page_size=1 << 17), "power of two"), (dict(stride_slot=-1), "negative")]


@pytest.mark.parametrize("change,text", BAD_CACHES)
def test_bad_caches_are_refused_by_both_operators(change, text):
    refused(lambda: attention(cache=cache(**change)), text)
    refused(lambda: append(cache=cache(**change)), text)


def attention(cache=cache(), q=FAKE, out=FAKE, lens=FAKE, n_rows=3, heads=8, max_len=20, **kw):
    hipdec.attention_paged(cache, q, out, lens, n_rows, heads, max_len, **kw)


def append(cache=cache(), rope=Rope.make(FAKE, 128), q=FAKE, k=FAKE, v=FAKE, q_out=FAKE, positions=FAKE, n_rows=3, heads=8, **kw):
    hipdec.rope_append_paged(rope, cache, q, k, v, q_out, positions, n_rows, heads, **kw)


def verify(logits=FAKE, drafts=FAKE, uniforms=FAKE, tokens=FAKE, accepted=FAKE, n_seqs=2, max_drafts=3, vocab=1000, workspace=FAKE,
           workspace_bytes=1 << 30, **kw):
    hipdec.verify_drafts(logits, drafts, uniforms, tokens, accepted, n_seqs, max_drafts, vocab, workspace=workspace,
                         workspace_bytes=workspace_bytes, **kw)


@pytest.mark.parametrize("kw,text,status", [
    (dict(q=None), "null", 1), (dict(out=None), "null", 1), (dict(lens=None), "null", 1), (dict(dtype=2), "dtype", 1),
    (dict(heads=0), "multiple", 1), (dict(heads=9), "multiple", 1), (dict(n_rows=1 << 40), "out of range", 1),
    (dict(max_len=1 << 40), "out of range", 1), (dict(scale=0.0), "scale", 1), (dict(scale=-1.0), "scale", 1),
    (dict(scale=math.nan), "scale", 1), (dict(scale=math.inf), "scale", 1), (dict(q_stride=8 * 128 - 4), "overlap", 1),
    (dict(out_stride=4), "overlap", 1), (dict(q=FAKE + 4), "aligned", 1), (dict(out=FAKE + 8), "aligned", 1),
    (dict(q_stride=8 * 128 + 2), "aligned", 1), (dict(dtype=RowDtype.BF16, out_stride=8 * 128 + 4), "aligned", 1),
    (dict(cache=cache(k=FAKE + 2)), "aligned", 1), (dict(cache=cache(stride_slot=132)), "aligned", 1),
    (dict(cache=cache(hd=96)), "head dim", 4), (dict(cache=cache(hd=80)), "head dim", 4), (dict(max_len=2000), "workspace", 1),
    (dict(max_len=2000, workspace=FAKE, workspace_bytes=16), "workspace", 1),
    (dict(max_len=2000, workspace=FAKE + 4, workspace_bytes=1 << 30), "workspace", 1),
    (dict(), "device", 1),                                                   # a plain address is no device memory
])
def test_attention_refuses(kw, text, status):
    refused(lambda: attention(**kw), text, status)


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(q_out=None), "null"), (dict(positions=None), "null"),
    (dict(rope=Rope.make(None, 128)), "null"), (dict(dtype=7), "dtype"), (dict(heads=0), "heads"), (dict(n_rows=1 << 40), "n_rows"),
    (dict(cache=cache(hd=127)), "hd"), (dict(cache=cache(hd=1024)), "hd"), (dict(rope=Rope.make(FAKE, 130)), "rot_dim"),
    (dict(rope=Rope.make(FAKE, 7)), "rot_dim"), (dict(rope=Rope.make(FAKE, 128, magnitude=math.nan)), "magnitude"),
    (dict(q_stride=100), "overlap"), (dict(k_stride=100), "overlap"), (dict(v_stride=255), "overlap"), (dict(q_out_stride=1000), "overlap"),
    (dict(q_stride=2048, q_out_stride=1024), "in place"), (dict(), "device"),
])
def test_append_refuses(kw, text):
    refused(lambda: append(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(logits=None), "null"), (dict(drafts=None), "null"), (dict(uniforms=None), "null"), (dict(tokens=None), "null"),
    (dict(accepted=None), "null"), (dict(dtype=2), "dtype"), (dict(temperature=-1.0), "temperature"), (dict(temperature=math.nan), "temperature"),
    (dict(temperature=math.inf), "temperature"), (dict(softcap=math.inf), "softcap"), (dict(softcap=math.nan), "softcap"),
    (dict(vocab=0, row_stride=1, prob_stride=1), "out of range"), (dict(vocab=262145), "out of range"), (dict(max_drafts=256), "out of range"),
    (dict(n_seqs=1 << 30), "out of range"), (dict(row_stride=999), "overlap"), (dict(draft_probs=FAKE, prob_stride=10), "overlap"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=100), "workspace"), (dict(workspace=FAKE + 8), "workspace"), (dict(), "device"),
])
def test_verification_refuses(kw, text):
    refused(lambda: verify(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=3), "rot_dim"), (dict(rot_dim=1024), "rot_dim"), (dict(theta=1.0), "theta"),
    (dict(theta=math.inf), "theta"), (dict(scaling=4), "scaling"), (dict(scaling=1, factor=0.5), "factor"), (dict(scaling=2, factor=math.nan), "factor"),
    (dict(rot_dim=2, scaling=2, factor=2.0), "base"), (dict(scaling=3, factor=2.0, trained=0.0), "trained"),
    (dict(scaling=3, factor=2.0, slow_turns=-1.0), "slow_turns"), (dict(scaling=3, factor=2.0, slow_turns=8.0, fast_turns=8.0), "fast_turns"),
])
def test_frequencies_refuse(kw, text):
    refused(lambda: hipdec.rope_frequencies(**dict(dict(rot_dim=64), **kw)), text)


def test_null_structs_and_size_queries():
    lib = hipdec.load_library()
    out = C.c_uint64()
    assert lib.hipdec_attention_paged(None, None, None, 0, None) == hipdec.ERR_ARG
    assert lib.hipdec_rope_append_paged(None, None, None, None) == hipdec.ERR_ARG
    assert lib.hipdec_verify_drafts(None, None, 0, None) == hipdec.ERR_ARG
    assert lib.hipdec_attention_paged_workspace(1, 8, 3, 128, 100, C.byref(out)) == hipdec.ERR_ARG
    assert lib.hipdec_attention_paged_workspace(1, 8, 2, 128, 100, None) == hipdec.ERR_ARG
    assert lib.hipdec_verify_drafts_workspace(1, 300, 100, C.byref(out)) == hipdec.ERR_ARG
    # no rows: nothing to do, whatever the pointers
    attention(n_rows=0, q=None)
    append(n_rows=0, q=None)
    verify(n_seqs=0, logits=None)
    # a short cache needs no workspace, a long one needs it for every row and head
    assert hipdec.attention_paged_workspace(1, 8, 2, 128, 256) == 0
    one = hipdec.attention_paged_workspace(1, 8, 2, 128, 50000)
    assert one > 0 and one % (8 * 130 * 4) == 0
    assert hipdec.verify_drafts_workspace(2, 3, 32768) >= 2 * 4 * 8 * 16


def test_a_workspace_serves_every_smaller_call():
    rng = np.random.default_rng(1)
    for _ in range(60):
        kvh, g = int(rng.choice([1, 2, 3, 8, 12, 32])), int(rng.choice([1, 2, 4, 7, 18]))
        n, length = int(rng.integers(1, 80)), int(2 ** rng.uniform(0, 17))
        c = cache(kv_heads=kvh, hd=64, stride_page=16 * kvh * 64, stride_slot=kvh * 64, stride_head=64)
        size = hipdec.attention_paged_workspace(n, kvh * g, kvh, 64, length)
        for _ in range(20):
            # (the workspace is looked at before the pointers, which are no device memory)
            refused(lambda: attention(cache=c, n_rows=int(rng.integers(1, n + 1)), heads=kvh * g, max_len=int(rng.integers(0, length + 1)),
                                      workspace=FAKE if size else None, workspace_bytes=size), "device")
        s, k, v = int(rng.integers(1, 70)), int(rng.integers(0, 9)), int(2 ** rng.uniform(0, 18))
        size = hipdec.verify_drafts_workspace(s, k, v)
        for _ in range(20):
            refused(lambda: verify(n_seqs=int(rng.integers(1, s + 1)), max_drafts=int(rng.integers(0, k + 1)), vocab=int(rng.integers(1, v + 1)),
                                   workspace_bytes=size), "device")


def test_errors_are_each_thread_s_own():
    import threading
    refused(lambda: attention(scale=0.0), "scale")
    seen = []
    t = threading.Thread(target=lambda: (refused(lambda: verify(temperature=-1.0), "temperature"),
                                         seen.append(hipdec.load_library().hipdec_last_error(None))))
    t.start()
    t.join()
    assert b"temperature" in seen[0] and b"scale" in hipdec.load_library().hipdec_last_error(None)
