"""Requests stepped together (hipdec_requests_*) at the edge of what include/hip_decode.h allows."""
import ctypes as C

import numpy as np
import pytest

from rustane_amd import hipdec
from rustane_amd.hipdec import HipDecodeError, KvDtype, NO_TOKEN
from test_gpu_requests import admit, alone, close, model
from test_zz_no_alloc import Hip

pytestmark = pytest.mark.gpu


def test_rejected_drafts_give_their_pages_back():
    m = model(kd=KvDtype.BF16)
    rng = np.random.default_rng(8)
    prompt = rng.integers(0, 700, 4)
    m.requests_open(4, 9, 3)
    for s in (0, 1):
        admit(m, s, prompt)                                  # a page each, full
    assert m.requests_len(0) == (4, 7)
    first = int(m.requests_step([1], [3])[0][0, 0])          # what follows, without drafts
    assert m.requests_len(1) == (5, 6)
    # twelve drafts of which the first is wrong: positions 4 .. 16 are written, one stays
    drafts = [[(first + 1) % 700] + [7] * 11]
    out, acc = m.requests_step([0], [3], drafts=drafts)
    assert acc[0] == 0 and out[0, 0] == first and np.all(out[0, 1:] == NO_TOKEN)
    assert m.requests_len(0) == (5, 5)                       # two pages each; five are left
    # the rest of the pool serves a third request of the length that just fits, and the first one goes on as if alone
    admit(m, 2, rng.integers(0, 700, 19))
    assert m.requests_len(2) == (19, 0)
    got = [m.requests_step([0], [t], logits=True)[2][0, 0] for t in (first, 9, 11)]
    close(np.stack(got), alone(m, prompt, [3, first, 9, 11])[1:], 2e-2)
    assert m.requests_len(0) == (8, 0)
    with pytest.raises(HipDecodeError) as e:
        m.requests_step([0], [1])
    assert e.value.status == hipdec.ERR_FULL and m.requests_len(0) == (8, 0)
    # partly kept drafts: what is kept stays, what lies behind it goes back
    for s in (0, 1, 2):
        m.requests_release(s)
    admit(m, 1, prompt)
    stream, tok = [], 3
    for _ in range(4):
        tok = int(m.requests_step([1], [tok])[0][0, 0])
        stream.append(tok)
    m.requests_release(1)
    admit(m, 0, prompt)
    out, acc = m.requests_step([0], [3], drafts=[stream[:2] + [(stream[2] + 1) % 700] + [5] * 10])
    assert acc[0] == 2 and out[0, :3].tolist() == stream[:3]
    assert m.requests_len(0) == (7, 7)


@pytest.mark.parametrize("seq,n", [(16, 20), (8, 32)])
def test_more_rows_than_the_window_has_positions(seq, n):
    m = model(seq=seq)
    rng = np.random.default_rng(9)
    prompts = [rng.integers(0, 700, i % (seq - 2)) for i in range(n)]
    m.requests_open(4, n * seq // 4, n)
    for s, p in enumerate(prompts):
        admit(m, s, p)
    fed = rng.integers(0, 700, (n, 2))
    seen = [m.requests_step(np.arange(n), fed[:, t], logits=True)[2][:, 0] for t in range(2)]
    for s in range(n):
        close(np.stack([x[s] for x in seen]), alone(m, prompts[s], fed[s]), 2e-3)


def test_more_samples_than_the_window_has_positions():
    m = model(seq=16)
    rng = np.random.default_rng(10)
    prompt, fed = rng.integers(0, 700, 5), rng.integers(0, 700, 24)
    want = np.concatenate([alone(m, prompt, [t]) for t in fed])
    m.set_len(0)
    m.prefill(np.asarray(prompt, np.uint32))
    m.batch_begin(24)
    got = m.decode_logits_from_ids_batch(np.asarray(fed, np.uint32))
    m.batch_end()
    close(np.asarray(got).reshape(24, -1), want, 2e-3)


def test_lengths_of_no_sequence_say_so():
    m = model()
    with pytest.raises(HipDecodeError) as e:
        m.requests_len(0)
    assert "no pages are open" in str(e.value)
    m.requests_open(8, 4, 2)
    for s in (0, 5):
        with pytest.raises(HipDecodeError) as e:
            m.requests_len(s)
        assert "no such sequence" in str(e.value)


def test_an_error_that_the_program_left_is_not_a_step_s():
    m, hip = model(), Hip()
    m.requests_open(8, 8, 2)
    m.set_len(0)
    m.prefill(np.arange(9, dtype=np.uint32))
    too_much = lambda: hip.rt.hipMalloc(C.byref(C.c_void_p()), 1 << 60)  # noqa: E731  (refused, and noted as the thread's last error)
    assert too_much() != 0
    m.requests_admit(1)
    assert m.requests_len(1)[0] == 9
    assert too_much() != 0
    lg = m.requests_step([1], [3], logits=True)[2]
    assert m.requests_len(1)[0] == 10
    close(lg[0], alone(m, np.arange(9), [3]), 2e-3)
