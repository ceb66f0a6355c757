"""Calls of the operators on the caller's device buffers at the edge of what include/hip_decode.h allows, on the GPU, against plain
fp64 restatements (those of test_gpu_serving_ops.py, whose head derives the tolerances of attention)."""
import numpy as np
import pytest

from rustane_amd import hipdec
from rustane_amd.hipdec import Rope, RopeScaling
from test_gpu_serving_ops import EPS, Cache, Rows, attend, attended, draft_case, fetch, hip, turned, verified, verify  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("hd,rot,interleaved,rows", [(128, 128, True, 3), (64, 64, False, 70), (64, 62, False, 9), (256, 128, True, 300), (512, 512, False, 2)])
def test_rotated_rows_are_off_by_their_roundings_only(hip, hd, rot, interleaved, rows):  # noqa: F811
    """Sine and cosine, with the magnitude, rounded to fp32 once, two products and a sum: 2 * 2^-24 (|x c| + |y s|) + 2^-24 of
    the result, and the angle's own rounding (2^-53 of it; the fp64 restatement has the same).  A far position's angle of
    2^24 rounded to fp32 as a fraction of a turn would be off by 1.9e-7 (|x| + |y|), wherever sine or cosine is small far more."""
    rng = np.random.default_rng(hd + rows)
    heads, kvh = 3, 1
    cache = Cache(hip, rng, [4] * rows, 4, kvh, hd, False, True, fill=False)
    x = rng.standard_normal((rows, heads + 2 * kvh, hd)).astype(np.float32)
    pos = rng.integers(0, 1 << 24, rows).astype(np.int32)
    pos[:2] = 0, -(1 << 24)
    freq, mag = hipdec.rope_frequencies(rot, scaling=RopeScaling.PARTS, factor=8.0)
    wide, d = (heads + 2 * kvh) * hd, hip.put(x)
    d_out = hip.put(np.zeros((rows, heads, hd), np.float32))
    hipdec.rope_append_paged(Rope.make(hip.put(freq), rot, interleaved=interleaved, magnitude=mag), cache.c, d, d + 4 * heads * hd,
                             d + 4 * (heads + kvh) * hd, d_out, hip.put(pos), rows, heads, slots=hip.put(np.ones(rows, np.int32)), row_stride=wide)
    hip.sync()
    got = np.concatenate([fetch(hip, d_out, (rows, heads, hd), False), cache.down()[0][cache.table[:, 0], 1]], axis=1)
    x = x[:, :heads + kvh]
    want = turned(x, pos, freq, mag, rot, interleaved)
    an = pos.astype(np.float64)[:, None, None] * freq
    e, o = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    ax, ay = np.abs(x[..., e].astype(np.float64)), np.abs(x[..., o].astype(np.float64))
    c, s = np.abs(np.cos(an)) * mag, np.abs(np.sin(an)) * mag
    tol = EPS * np.abs(want)
    tol[..., rot:] = 0.0
    for part, big in ((e, ax * c + ay * s), (o, ay * c + ax * s)):
        tol[..., part] += 2.01 * EPS * big + (ax + ay) * mag * (np.abs(an) + 1) * 2.0 ** -52
    assert np.all(np.abs(got - want) <= tol), (np.abs(got - want) / np.maximum(tol, 1e-30)).max()


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("b16", [False, True])
@pytest.mark.parametrize("max_len", [250, 1100])             # one launch; several splits and their join
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 64), (18, 1, 128)])
def test_attention_in_place(hip, b16, max_len, heads, kvh, hd):  # noqa: F811
    rng = np.random.default_rng(max_len + hd)
    lens = [250, 1, 0, 129, 249]
    cache = Cache(hip, rng, lens, 16, kvh, hd, True, False)
    q = Rows(rng.standard_normal((len(lens), heads, hd)).astype(np.float32), b16)
    stride = heads * hd + 16
    wide = np.full((len(lens), stride), 0x4240 if b16 else 48.0, q.raw.dtype)
    wide[:, :heads * hd] = q.raw.reshape(len(lens), -1)
    size = hipdec.attention_paged_workspace(len(lens), heads, kvh, hd, max_len)
    d = hip.put(wide)
    hipdec.attention_paged(cache.c, d, d, hip.put(np.asarray(lens, np.int32)), len(lens), heads, max_len, dtype=q.dtype, q_stride=stride,
                           out_stride=stride, workspace=hip.put(np.zeros(size // 4 + 4, np.float32)) if size else None, workspace_bytes=size)
    hip.sync()
    got = fetch(hip, d, (len(lens), stride), b16)
    assert np.all(got[:, heads * hd:] == 48.0)
    want, tol = attended(cache, q.x, range(len(lens)), lens, hd ** -0.5)
    got = got[:, :heads * hd].reshape(want.shape)
    assert np.all(np.abs(got - want) <= tol + (2.0 ** -8 * np.abs(want) if b16 else 0.0))


@pytest.mark.parametrize("max_len", [250, 3000])
def test_a_row_s_bits_are_its_own(hip, max_len):  # noqa: F811
    """With as many rows and the same max_len (which decide the splits) the other rows' queries, lengths and sequences make no difference."""
    rng = np.random.default_rng(max_len)
    lens = [200, 250, 17, 3] if max_len == 250 else [2999, 1500, 64, 700]
    cache = Cache(hip, rng, lens, 32, 2, 128, True, False)
    q = rng.standard_normal((4, 12, 128)).astype(np.float32)
    first = attend(hip, cache, Rows(q, False), [0, 1, 2, 3], lens, max_len=max_len)
    for seqs, others in (([0, 3, 3, 1], [1, 3, 0]), ([0, 0, -1, 2], [lens[0], 40, 5])):
        other = rng.standard_normal(q.shape).astype(np.float32) * 7.0
        other[0] = q[0]
        got = attend(hip, cache, Rows(other, False), seqs, [lens[0]] + others, max_len=max_len)
        assert np.array_equal(got[0], first[0])
        again = attend(hip, cache, Rows(other[[1, 0, 2, 3]], False), [seqs[1], 0, seqs[2], seqs[3]], [others[0], lens[0]] + others[1:], max_len=max_len)
        assert np.array_equal(again[1], first[0])            # ... nor does its place among them


# ---------------------------------------------------------------- verification
@pytest.mark.parametrize("S,K,V,b16,T,cap,with_probs,pad", [
    (32, 7, 32768, False, 0.8, 0.0, True, 0), (16, 4, 65000, True, 1.0, 20.0, False, 3),     # 4 to 12 million logits
    (3, 2, 100003, True, 0.7, 30.0, True, 1), (4, 1, 65537, False, 1.0, 0.0, False, 0), (2, 3, 131072, False, 0.0, 0.0, True, 0),
])
def test_verification_with_eight_logits_a_lane(hip, S, K, V, b16, T, cap, with_probs, pad):  # noqa: F811
    rng = np.random.default_rng(S * 3 + V)
    case = draft_case(rng, S, K, V, b16, T, with_probs)
    tokens, accepted = verify(hip, *case[:4], T, cap, case[4], row_pad=pad)
    want, want_acc = verified(case[0].x, *case[1:4], T, cap, case[4])
    assert np.array_equal(accepted, want_acc) and np.array_equal(tokens, want)


def test_negative_probabilities_and_random_numbers_count_as_zero(hip):  # noqa: F811
    rng = np.random.default_rng(14)
    S, K, V, T = 8, 3, 2051, 0.9
    lg, drafts, n, u, probs = draft_case(rng, S, K, V, False, T, True)
    n[:] = K
    x = lg.x
    probs[0, :, -1], u[0, :K] = -0.7, 0.99999                # the last token of a vocabulary that ends inside a chunk
    x[1, :, 5::7], probs[1, :, 5::7], u[1, :K] = -np.inf, -0.5, 0.99999
    probs[2] *= -1.0
    for s in (3, 4):                                         # drafts that the target cannot give
        x[s, np.arange(K), drafts[s]] = -np.inf
    u[3, :K], probs[4, np.arange(K), drafts[4]] = -0.25, -0.3
    u[5, K], u[6, K] = -3.0, -np.inf
    for p in (probs, None):
        tokens, accepted = verify(hip, Rows(x, False), drafts, n, u, T, 0.0, p)
        want, want_acc = verified(x, drafts, n, np.maximum(u, 0.0), T, 0.0, None if p is None else np.maximum(p, 0.0))
        assert np.array_equal(accepted, want_acc) and np.array_equal(tokens, want)


@pytest.mark.parametrize("T", [1e-12, 1e-18, 1e-20, 1e-30, 1.2e-38])
def test_tiny_temperatures_with_a_saturated_soft_cap(hip, T):  # noqa: F811
    """Logits of twenty caps and more are within the last bits of each other: only one of them may be kept or drawn."""
    rng = np.random.default_rng(15)
    S, K, V = 16, 3, 3000
    x = rng.standard_normal((S, K + 1, V)).astype(np.float32)
    x[..., 1::2] = 40.0 + 30.0 * rng.random((S, K + 1, V // 2), dtype=np.float32)
    drafts, n = rng.integers(0, V, (S, K)).astype(np.int32), np.full(S, K, np.int32)
    probs = np.full((S, K, V), 1.0 / V, np.float32)
    for p in (probs, None):
        tokens, accepted = verify(hip, Rows(x, False), drafts, n, rng.random((S, K + 1), dtype=np.float32), T, 2.0, p)
        for s in range(S):
            kept = tokens[s, :accepted[s] + 1]
            assert np.all(kept < V) and np.all(kept % 2 == 1) and np.all(tokens[s, accepted[s] + 1:] == hipdec.NO_TOKEN), (tokens[s], accepted[s])


@pytest.mark.parametrize("cap", [0.0, 4.0])
def test_an_infinite_logit_is_the_largest_at_temperature_zero(hip, cap):  # noqa: F811
    rng = np.random.default_rng(16)
    x = rng.standard_normal((4, 2, 1500)).astype(np.float32)
    x[..., 3] = np.finfo(np.float32).max
    x[1:, :, 500] = x[1:, :, 1400] = np.inf
    x[2, :, 40] = np.inf
    drafts = np.array([[3], [500], [40], [3]], np.int32)
    tokens, accepted = verify(hip, Rows(x, False), drafts, np.ones(4, np.int32), np.zeros((4, 2), np.float32), 0.0, cap)
    assert accepted.tolist() == [1, 1, 1, 0] and tokens.tolist() == [[3, 3], [500, 500], [40, 40], [500, hipdec.NO_TOKEN]]
