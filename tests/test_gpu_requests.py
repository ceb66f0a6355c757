"""Requests of their own prompts stepped together over a paged cache (hipdec_requests_*), against the model's own
single-row path: the logits of every row of a step are those the model gives when it decodes that request alone
(2e-3 of the largest logit with fp32 caches, as for the other multi-row paths: activations travel as pairs of bf16
numbers; 2e-2 with bf16 caches, the bound of that format), tokens follow from the returned logits exactly, rejected
drafts leave no trace, and pages are given and taken back."""
import numpy as np
import pytest

from rustane_amd import hipdec, synth
from rustane_amd.hipdec import Config, HipDecodeError, HipDecodeModel, KvDtype, NO_TOKEN, WeightDtype
from test_gpu_serving_ops import verified

CFG = dict(dim=256, hidden=640, heads=4, hd=64, seq=96, nlayers=2, vocab=700)


def model(wd=WeightDtype.BF16, kd=KvDtype.F32, kv_heads=None, **kw):
    cfg = Config.make(kv_heads=kv_heads, **dict(CFG, **kw))
    return HipDecodeModel(cfg, synth.make_weights(cfg, seed=5, std=0.08, round_bf16=True), weight_dtype=wd, kv_dtype=kd)


def alone(m, prompt, tokens):
    """Logits after each of `tokens` fed behind the prompt, by the model's own steps."""
    m.set_len(0)
    if len(prompt):
        m.prefill(np.asarray(prompt, np.uint32))
    return np.stack([m.decode_logits_from_id(int(t)) for t in tokens])


def admit(m, seq, prompt):
    m.set_len(0)
    if len(prompt):
        m.prefill(np.asarray(prompt, np.uint32))
    m.requests_admit(seq)


def close(got, want, tol):
    assert np.abs(got - want).max() <= tol * np.abs(want).max(), np.abs(got - want).max() / np.abs(want).max()


@pytest.mark.gpu
@pytest.mark.parametrize("wd,kd,kv_heads,hd,tol", [
    (WeightDtype.BF16, KvDtype.F32, 4, 64, 2e-3), (WeightDtype.BF16, KvDtype.BF16, 2, 64, 2e-2), (WeightDtype.F32, KvDtype.F32, 1, 64, 2e-3),
    (WeightDtype.FP8_E4M3, KvDtype.BF16, 4, 64, 2e-2), (WeightDtype.INT4_G128, KvDtype.F32, 2, 64, 2e-3), (WeightDtype.BF16, KvDtype.F32, 4, 128, 2e-3)])
def test_rows_of_a_step_equal_each_request_alone(wd, kd, kv_heads, hd, tol):
    m = model(wd, kd, kv_heads, hd=hd)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 700, n) for n in (1, 37, 16, 0)]
    m.requests_open(8, 60, 8)
    for s, p in zip((5, 0, 7, 2), prompts):
        admit(m, s, p)
        assert m.requests_len(s)[0] == len(p)
    fed = rng.integers(0, 700, (4, 6))
    # plain steps, some of the sequences in another order each time; then a step with two drafts each
    seen = {i: [] for i in range(4)}
    for t in range(3):
        order = rng.permutation(4)
        out, acc, lg = m.requests_step([(5, 0, 7, 2)[i] for i in order], [fed[i, t] for i in order], logits=True)
        assert np.all(acc == 0) and np.array_equal(out[:, 0], lg[:, 0].argmax(-1))
        for k, i in enumerate(order):
            seen[i].append(lg[k, 0])
    out, acc, lg = m.requests_step([5, 0, 7, 2], fed[:, 3], drafts=fed[:, 4:6], logits=True)
    for i in range(4):
        want = alone(m, prompts[i], fed[i])
        close(np.concatenate([np.stack(seen[i]), lg[i]]), want, tol)


@pytest.mark.gpu
def test_drafts_are_kept_or_leave_no_trace():
    m = model()
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 700, n) for n in (20, 7)]
    m.requests_open(4, 64, 2)
    for s, p in enumerate(prompts):
        admit(m, s, p)
    # what greedy steps without drafts give
    streams, tok = [[], []], np.array([3, 9])
    for _ in range(7):
        tok = m.requests_step([0, 1], tok)[0][:, 0]
        for s in range(2):
            streams[s].append(int(tok[s]))
    for s, p in enumerate(prompts):
        m.requests_release(s)
        admit(m, s, p)
    # the same with drafts: one sequence's are right, the other's second is wrong
    a, b = streams
    wrong = (b[1] + 1) % 700
    out, acc = m.requests_step([0, 1], [3, 9], drafts=[a[:3], [b[0], wrong, b[2]]])
    assert acc.tolist() == [3, 1]
    assert out[0].tolist() == a[:4] and out[1].tolist() == [b[0], b[1], NO_TOKEN, NO_TOKEN]
    assert [m.requests_len(s)[0] for s in (0, 1)] == [24, 9]
    # the rejected drafts' positions are written again; unequal numbers of drafts
    out, acc = m.requests_step([1, 0], [b[1], a[3]], drafts=[[b[2], b[3]], [a[4], 0]], n_drafts=[2, 1])
    assert acc.tolist() == [2, 1] and out[0].tolist() == b[2:5] and out[1].tolist() == [a[4], a[5], NO_TOKEN]


@pytest.mark.gpu
@pytest.mark.parametrize("with_probs", [False, True])
def test_sampled_steps_follow_the_returned_logits(with_probs):
    m = model(kd=KvDtype.BF16)
    rng = np.random.default_rng(6)
    m.requests_open(16, 40, 6)
    for s in range(5):
        admit(m, s, rng.integers(0, 700, 3 + s))
    K, T, cap = 4, 0.7, 5.0
    kept = 0
    for step in range(4):
        tokens, drafts = rng.integers(0, 700, 5), rng.integers(0, 700, (5, K))
        n, u = rng.integers(0, K + 1, 5), rng.random((5, K + 1), dtype=np.float32)
        probs = None
        if with_probs:                                       # a draft that is certain enough of little: many are kept
            probs = np.full((5, K, 700), 1e-4, np.float32)
        out, acc, lg = m.requests_step(np.arange(5), tokens, drafts=drafts, n_drafts=n, draft_probs=probs, uniforms=u, temperature=T, softcap=cap, logits=True)
        want, want_acc = verified(lg, drafts.astype(np.int64), n, u, T, cap, probs)
        assert np.array_equal(acc, want_acc) and np.array_equal(out, want)
        kept += int(acc.sum())
    assert kept > 0 or not with_probs


@pytest.mark.gpu
def test_pages_run_out_and_come_back():
    m = model()
    with pytest.raises(HipDecodeError):
        m.requests_step([0], [1])                            # nothing open
    m.requests_open(8, 5, 3)
    admit(m, 0, np.arange(16))                               # two pages, full
    admit(m, 1, np.arange(9))                                # two
    assert m.requests_len(0) == (16, 1)
    m.set_len(0)
    m.prefill(np.arange(17, dtype=np.uint32))
    with pytest.raises(HipDecodeError) as e:
        m.requests_admit(2)                                  # three
    assert e.value.status == hipdec.ERR_FULL and m.requests_len(0) == (16, 1)
    m.requests_step([0, 1], [1, 2])                          # the last page goes to sequence 0
    assert m.requests_len(0) == (17, 0)
    for _ in range(6):
        m.requests_step([1], [2])
    assert m.requests_len(1)[0] == 16
    with pytest.raises(HipDecodeError) as e:
        m.requests_step([0, 1], [1, 2])
    assert e.value.status == hipdec.ERR_FULL and m.requests_len(0)[0] == 17 and m.requests_len(1)[0] == 16
    m.requests_release(0)
    assert m.requests_len(1) == (16, 3)
    before = m.requests_step([1], [2], logits=True)[2]
    assert m.requests_len(1) == (17, 2)                      # (sequence 1's seventeenth position took one of the three)
    admit(m, 0, np.arange(100, 115))                         # 15 positions: both pages, which hold old keys behind them
    out, _, lg = m.requests_step([0], [5], logits=True)
    close(lg[0], alone(m, np.arange(100, 115), [5]), 2e-3)
    close(before[0], alone(m, np.arange(9), [2] * 8)[-1:], 2e-3)


@pytest.mark.gpu
def test_window_ends_and_refusals():
    m = model(seq=32)
    m.requests_open(8, 12, 4)
    admit(m, 0, np.arange(30))
    for call, status in (
            (lambda: m.requests_open(8, 12, 4), 1), (lambda: m.requests_admit(0), 1), (lambda: m.requests_admit(4), 1), (lambda: m.requests_release(1), 1),
            (lambda: m.requests_step([0, 0], [1, 1]), 1), (lambda: m.requests_step([1], [1]), 1), (lambda: m.requests_step([0], [700]), 1),
            (lambda: m.requests_step([0], [1], drafts=[[700]]), 1), (lambda: m.requests_step([0], [1], drafts=[[1]], n_drafts=[2]), 1),
            (lambda: m.requests_step([0], [1], temperature=0.5), 1), (lambda: m.requests_step([0], [1], temperature=-1.0, uniforms=[[0.5]]), 1),
            (lambda: m.requests_step([0], [1], drafts=[[1] * 32]), 1), (lambda: m.requests_step([0], [1], drafts=[[1, 2]]), 2)):
        with pytest.raises(HipDecodeError) as e:
            call()
        assert e.value.status == status, str(e.value)
    assert m.requests_len(0)[0] == 30
    # the last two positions, then the window is full
    out, acc = m.requests_step([0], [1], drafts=[[3]])
    assert m.requests_len(0)[0] == 31 + int(acc[0])
    m.requests_release(0)
    admit(m, 0, np.arange(32))
    with pytest.raises(HipDecodeError) as e:
        m.requests_step([0], [1])
    assert e.value.status == hipdec.ERR_FULL
    # the model's own steps go on as before, and a batch closes the requests' steps
    m.set_len(0)
    m.prefill(np.arange(4, dtype=np.uint32))
    m.batch_begin(2)
    with pytest.raises(HipDecodeError):
        m.requests_step([0], [1])
    m.decode_token_argmax_from_ids_batch([1, 2])
    m.batch_end()


@pytest.mark.gpu
def test_a_pool_that_does_not_fit_can_be_opened_smaller():
    m = model()
    with pytest.raises(HipDecodeError):
        m.requests_open(65536, 1 << 24, 2)                   # half a petabyte
    m.requests_open(16, 8, 2)
    admit(m, 1, np.arange(5))
    assert m.requests_step([1], [3])[0].shape == (1, 1)


def test_null_model_is_refused_without_a_gpu():
    lib = hipdec.load_library()
    assert lib.hipdec_requests_open(None, 16, 4, 1) == hipdec.ERR_ARG
    assert lib.hipdec_requests_admit(None, 0) == hipdec.ERR_ARG
    assert lib.hipdec_requests_release(None, 0) == hipdec.ERR_ARG
    assert lib.hipdec_requests_len(None, 0, None, None) == hipdec.ERR_ARG
    assert lib.hipdec_requests_step(None, 1, None, None, 0, None, None, None, None, 0.0, 0.0, None, None, None) == hipdec.ERR_ARG
