"""The operators on the caller's device buffers against plain fp64 restatements: rotary positions with the append to a
paged cache, attention over it, verification of drafted tokens; alone, together as a server would use them, captured
into a graph, on two streams at once, and with offsets past 32 bits.  (The HIP runtime, through ctypes, supplies the
buffers and streams.)

Tolerances.  A rounding to bf16 is off by at most 2^-8 of the value.  A rotation: the reduced angle is rounded to
fp32 (2^-25 of a turn, 1.9e-7 rad), sine and cosine are within 2 ulp (1.2e-7 each), two products, a sum and the
magnitude round (4 * 6e-8): 6e-7 of (|x| + |y|) * magnitude.  Attention: a score is a sum of hd products in fp32 (its
error at most hd * 2^-24 of sum |q k|, with three bf16 parts of q another 2^-24), the exponent adds 2 * 2^-24 of the largest
score and the exponential 2^-23, the weighted sum of n terms n * 2^-24: with d the largest score error, the output is
off by at most (2 d + 2 n * 2^-24 + 2^-22) * max |v|.  Tokens are whole numbers: equal."""
import ctypes as C

import numpy as np
import pytest

from rustane_amd import hipdec
from rustane_amd.hipdec import KvDtype, NO_TOKEN, PagedCache, Rope, RopeScaling, RowDtype
from test_zz_no_alloc import Hip

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def to_bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where((u & 0x7F800000) == 0x7F800000, (u >> 16).astype(np.uint16), r)


def of_bf16(u):
    return (np.asarray(u, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Rows:
    """Numbers of one of the two formats: what is stored, and the values it stands for."""

    def __init__(self, x, b16):
        self.b16, self.dtype = b16, RowDtype.BF16 if b16 else RowDtype.F32
        self.raw = to_bf16(x) if b16 else np.ascontiguousarray(x, np.float32)
        self.x = of_bf16(self.raw) if b16 else self.raw
        self.size = 2 if b16 else 4


@pytest.fixture
def hip():
    h = Hip()
    yield h
    h.free_all()


def fetch(hip, ptr, shape, b16):
    raw = hip.get(ptr, np.uint16 if b16 else np.float32, int(np.prod(shape))).reshape(shape)
    return of_bf16(raw) if b16 else raw


class Cache:
    """A pool on the device and its copy on the host, [page][slot][head][hd] whatever the layout."""

    def __init__(self, hip, rng, lens, page, kv_heads, hd, b16, token_major, n_seqs=None, spare=2, fill=True, max_pages=None):
        self.hip, self.page, self.b16, self.token_major, self.kvh, self.hd = hip, page, b16, token_major, kv_heads, hd
        n_seqs = len(lens) if n_seqs is None else n_seqs
        per = max(-(-max(max(lens), 1) // page), 1) if max_pages is None else max_pages
        self.n_pages = n_seqs * per + spare
        self.table = rng.permutation(self.n_pages)[:n_seqs * per].reshape(n_seqs, per).astype(np.int32)
        shape = (self.n_pages, page, kv_heads, hd)
        self.k, self.v = (np.full(shape, np.nan, np.float32) for _ in range(2))
        if fill:                                             # slots that no length covers stay NaN
            for s, n in enumerate(lens):
                for i in range(0, n, page):
                    p, m = self.table[s, i // page], min(page, n - i)
                    self.k[p, :m] = rng.standard_normal((m, kv_heads, hd)) * 1.2
                    self.v[p, :m] = rng.standard_normal((m, kv_heads, hd))
        if b16:
            self.k, self.v = of_bf16(to_bf16(self.k)), of_bf16(to_bf16(self.v))
        self.d_k, self.d_v, self.d_table = self._up(self.k), self._up(self.v), hip.put(self.table)
        self.c = PagedCache.make(self.d_k, self.d_v, KvDtype.BF16 if b16 else KvDtype.F32, n_pages=self.n_pages, page_size=page,
                                 kv_heads=kv_heads, hd=hd, page_table=self.d_table, n_seqs=n_seqs, max_pages=per, token_major=token_major)

    def _up(self, x):
        x = x if self.token_major else x.transpose(0, 2, 1, 3)
        return self.hip.put(to_bf16(x) if self.b16 else x)

    def down(self):
        shape = (self.n_pages, self.page, self.kvh, self.hd) if self.token_major else (self.n_pages, self.kvh, self.page, self.hd)
        return [x if self.token_major else x.transpose(0, 2, 1, 3) for x in (fetch(self.hip, p, shape, self.b16) for p in (self.d_k, self.d_v))]

    def rows(self, seq, n):
        """(keys, values) of the slots 0 .. n - 1 that have a page, fp64."""
        at = np.arange(n)
        pages = self.table[seq, at // self.page]
        ok = (pages >= 0) & (pages < self.n_pages)
        at, pages = at[ok] % self.page, pages[ok]
        return self.k[pages, at].astype(np.float64), self.v[pages, at].astype(np.float64)


# ---------------------------------------------------------------- rotary positions and the append
def turned(x, pos, freq, mag, rot, interleaved):
    """x[rows][heads][hd] in fp64, turned."""
    y, a = x.astype(np.float64).copy(), pos.astype(np.float64)[:, None, None] * freq
    c, s = np.cos(a) * mag, np.sin(a) * mag
    e, o = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., e], y[..., o] = x[..., e] * c - x[..., o] * s, x[..., o] * c + x[..., e] * s
    return y


def off_limits(x, rot, interleaved, mag):
    """|x| + |y| of each element's pair, times the magnitude."""
    a = np.abs(x.astype(np.float64))
    b = np.zeros_like(a)
    e, o = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    b[..., e] = b[..., o] = (a[..., e] + a[..., o]) * mag
    return b


@pytest.mark.parametrize("rows,heads,kvh,hd,rot,interleaved,b16,c16,page,token_major,pad", [
    (1, 12, 12, 128, 128, True, False, True, 16, True, 0),
    (7, 8, 2, 64, 64, False, True, True, 8, False, 0),
    (33, 32, 8, 128, 64, False, True, True, 64, False, 8),
    (5, 5, 1, 256, 256, True, False, False, 1, False, 4),
    (9, 4, 4, 192, 48, False, False, True, 4, True, 16),
    (6, 3, 3, 64, 62, False, True, False, 2, True, 0),       # 31 pairs: pair by pair
    (6, 3, 1, 10, 6, True, False, True, 4, False, 2),
    (4, 2, 2, 128, 128, False, True, True, 16, True, 3),     # rows that start unaligned
    (600, 4, 2, 64, 64, True, True, True, 32, False, 0),     # more rows than workgroups that run at once
    (3, 2, 1, 512, 0, True, False, True, 16, False, 0),      # nothing turned
])
def test_rope_append(hip, rows, heads, kvh, hd, rot, interleaved, b16, c16, page, token_major, pad):
    rng = np.random.default_rng(rows * 100 + hd)
    n_seqs = min(rows, 4)
    cache = Cache(hip, rng, [3 * page + 1] * n_seqs, page, kvh, hd, c16, token_major, max_pages=-(-rows // n_seqs) // page + 4)
    wide = (heads + 2 * kvh) * hd + pad
    x = Rows(rng.standard_normal((rows, wide)).astype(np.float32) * 2.0, b16)
    pos = rng.integers(0, 1 << 20, rows).astype(np.int32)
    pos[-1] = -3
    seqs = (np.arange(rows) % n_seqs).astype(np.int32)
    slots = (np.arange(rows) // n_seqs + 2).astype(np.int32)
    if rows > 3:
        slots[1], seqs[2], slots[3] = -1, n_seqs, cache.c.max_pages * page        # padding, no such sequence, no such slot
    freq, mag = hipdec.rope_frequencies(rot, scaling=RopeScaling.PARTS, factor=4.0) if rot else (np.zeros(1), 1.0)
    rope = Rope.make(hip.put(freq), rot, interleaved=interleaved, magnitude=mag)
    d_x, d_out = hip.put(x.raw), hip.put(np.zeros((rows, heads * hd + 8), x.raw.dtype))
    d_pos, d_slots, d_seqs = hip.put(pos), hip.put(slots), hip.put(seqs)
    hipdec.rope_append_paged(rope, cache.c, d_x, d_x + heads * hd * x.size, d_x + (heads + kvh) * hd * x.size, d_out, d_pos, rows, heads,
                             dtype=x.dtype, slots=d_slots, seqs=d_seqs, row_stride=wide, q_out_stride=heads * hd + 8)
    hip.sync()
    q, k, v = (x.x[:, a * hd:b * hd].reshape(rows, b - a, hd) for a, b in ((0, heads), (heads, heads + kvh), (heads + kvh, heads + 2 * kvh)))

    def check(got, x, b16):
        want = turned(x, pos_of, freq, mag, rot, interleaved) if rot else x.astype(np.float64)
        assert np.all(np.abs(got - want) <= 6e-7 * off_limits(x, rot, interleaved, mag) + (2.0 ** -8 * np.abs(want) if b16 else 0.0))

    out = fetch(hip, d_out, (rows, heads * hd + 8), b16)
    pos_of = pos
    check(out[:, :heads * hd].reshape(rows, heads, hd), q, b16)
    assert np.all(out[:, heads * hd:] == 0.0)
    got_k, got_v = cache.down()
    for t in range(rows):
        if slots[t] < 0 or seqs[t] >= n_seqs or slots[t] >= cache.c.max_pages * page:
            continue
        p, s = cache.table[seqs[t], slots[t] // page], slots[t] % page
        pos_of = pos[t:t + 1]
        check(got_k[p, s][None], k[t:t + 1], c16)
        assert np.array_equal(got_v[p, s], of_bf16(to_bf16(v[t])) if c16 else v[t])
        got_k[p, s], got_v[p, s] = cache.k[p, s], cache.v[p, s]
    assert np.array_equal(got_k, cache.k, equal_nan=True) and np.array_equal(got_v, cache.v, equal_nan=True)   # nothing else was touched


def test_rope_append_without_slots_and_sequences_and_in_place(hip):
    rng = np.random.default_rng(2)
    rows, heads, hd = 3, 4, 64
    cache = Cache(hip, rng, [40] * rows, 16, heads, hd, True, False)
    x = [rng.standard_normal((rows, heads, hd)).astype(np.float32) for _ in range(3)]
    pos = np.array([39, 0, 17], np.int32)
    freq, _ = hipdec.rope_frequencies(hd)
    d = [hip.put(a) for a in x]
    hipdec.rope_append_paged(Rope.make(hip.put(freq), hd), cache.c, d[0], d[1], d[2], d[0], hip.put(pos), rows, heads)
    hip.sync()
    want = turned(x[0], pos, freq, 1.0, hd, True)
    assert np.all(np.abs(fetch(hip, d[0], x[0].shape, False) - want) <= 6e-7 * off_limits(x[0], hd, True, 1.0))
    got_v = cache.down()[1]
    for t in range(rows):
        assert np.array_equal(got_v[cache.table[t, pos[t] // 16], pos[t] % 16], of_bf16(to_bf16(x[2][t])))


# ---------------------------------------------------------------- attention
def attended(cache, q, seqs, lens, scale):
    """(output, its tolerance without the rounding to the rows' format), fp64: q[rows][heads][hd]."""
    rows, heads, hd = q.shape
    g = heads // cache.kvh
    out, tol = np.zeros(q.shape), np.zeros((rows, heads, 1))
    for r in range(rows):
        if not 0 <= seqs[r] < len(cache.table) or lens[r] <= 0:
            continue
        k, v = cache.rows(seqs[r], lens[r])
        if not len(k):
            continue
        for h in range(heads):
            a, b = q[r, h].astype(np.float64), k[:, h // g]
            s = b @ a * scale
            w = np.exp(s - s.max())
            out[r, h] = w @ v[:, h // g] / w.sum()
            d = scale * (np.abs(b) @ np.abs(a)).max() * (hd + 2) * EPS + 2 * EPS * np.abs(s).max()
            tol[r, h] = (2 * d + 2 * len(k) * EPS + 2.0 ** -22) * np.abs(v[:, h // g]).max()
    return out, tol


def attend(hip, cache, q, seqs, lens, max_len=None, pad=0, scale=None, stream=None):
    rows, heads, hd = q.x.shape
    stride = heads * hd + pad
    wide = np.zeros((rows, stride), q.raw.dtype)
    wide[:, :heads * hd] = q.raw.reshape(rows, -1)
    max_len = max(lens) if max_len is None else max_len
    size = hipdec.attention_paged_workspace(rows, heads, cache.kvh, hd, max_len)
    ws = hip.put(np.full(size // 4 + 4, np.nan, np.float32)) if size else None
    d_q, d_out = hip.put(wide), hip.put(np.full((rows, stride), 0x4240 if q.b16 else 48.0, q.raw.dtype))
    hipdec.attention_paged(cache.c, d_q, d_out, hip.put(np.asarray(lens, np.int32)), rows, heads, max_len, dtype=q.dtype,
                           seqs=None if seqs is None else hip.put(np.asarray(seqs, np.int32)), q_stride=stride, out_stride=stride,
                           scale=scale, workspace=ws, workspace_bytes=size, stream=stream)
    hip.sync()
    out = fetch(hip, d_out, (rows, stride), q.b16)
    assert np.all(out[:, heads * hd:] == 48.0)               # between the rows: left as it was
    return out[:, :heads * hd].reshape(rows, heads, hd)


def check_attention(hip, cache, q, seqs, lens, **kw):
    got = attend(hip, cache, q, seqs, lens, **kw)
    bound = kw.get("max_len") or max(lens)
    seqs = list(range(len(lens))) if seqs is None else seqs
    want, tol = attended(cache, q.x, seqs, [min(n, bound, cache.c.max_pages * cache.page) for n in lens],
                         kw.get("scale") or q.x.shape[2] ** -0.5)
    assert np.all(np.abs(got - want) <= tol + (2.0 ** -8 * np.abs(want) if q.b16 else 0.0)), np.abs(got - want).max()
    for r, n in enumerate(lens):
        if n <= 0:
            assert np.all(got[r] == 0.0)
    return got


@pytest.mark.parametrize("b16,c16", [(False, True), (True, True), (False, False), (True, False)])
@pytest.mark.parametrize("hd", [64, 128, 192, 256])
@pytest.mark.parametrize("heads,kvh", [(4, 4), (8, 2), (7, 1), (18, 1)])
def test_attention_forms(hip, b16, c16, hd, heads, kvh):
    rng = np.random.default_rng(hd + heads + b16 + 2 * c16)
    lens = [1, 17, 300, 0, 129]                              # one split, and (max_len below) several
    cache = Cache(hip, rng, lens, 16, kvh, hd, c16, bool(heads % 2))
    q = Rows(rng.standard_normal((len(lens), heads, hd)).astype(np.float32) * 1.5, b16)
    check_attention(hip, cache, q, None, lens, max_len=250, pad=16)
    check_attention(hip, cache, q, None, lens, max_len=1100, pad=0)


@pytest.mark.parametrize("page", [1, 2, 8, 32, 256, 1024])
@pytest.mark.parametrize("token_major", [False, True])
def test_attention_pages(hip, page, token_major):
    rng = np.random.default_rng(page)
    lens = [513, 1, 255, 256, 257, 1023, 31, 33]
    cache = Cache(hip, rng, lens, page, 2, 128, True, token_major)
    check_attention(hip, cache, Rows(rng.standard_normal((8, 8, 128)).astype(np.float32), True), None, lens)


def test_attention_of_a_draft_s_rows(hip):
    # five rows of each of three sequences, each one entry longer: the rows of a draft, in an order of their own
    rng = np.random.default_rng(4)
    cache = Cache(hip, rng, [705, 70, 1505], 16, 2, 64, False, False)
    seqs = [2, 0, 1] * 5
    lens = [(1500, 700, 65)[i % 3] + i // 3 for i in range(15)]
    check_attention(hip, cache, Rows(rng.standard_normal((15, 8, 64)).astype(np.float32), False), seqs, lens)


def test_attention_many_rows_and_long_rows(hip):
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(0, 1500, 70)]
    cache = Cache(hip, rng, lens, 64, 4, 128, True, False)
    check_attention(hip, cache, Rows(rng.standard_normal((70, 16, 128)).astype(np.float32), True), None, lens)
    lens = [40001]
    cache = Cache(hip, rng, lens, 64, 2, 128, True, False)
    check_attention(hip, cache, Rows(rng.standard_normal((1, 8, 128)).astype(np.float32), False), None, lens)


def test_attention_sharp_and_flat_scores(hip):
    # scores of several hundred (one key takes everything, whichever split it lies in) and scores that are all equal
    rng = np.random.default_rng(6)
    lens = [900, 900]
    cache = Cache(hip, rng, lens, 16, 1, 128, True, False)
    q = rng.standard_normal((2, 4, 128)).astype(np.float32) * 40.0
    check_attention(hip, cache, Rows(q, True), None, lens)
    check_attention(hip, cache, Rows(np.zeros_like(q), False), None, lens)
    check_attention(hip, cache, Rows(q, False), None, lens, scale=0.01)


def test_attention_lengths_pages_and_sequences_out_of_range(hip):
    rng = np.random.default_rng(7)
    lens = [320, 320, 320, 320]
    cache = Cache(hip, rng, lens, 16, 2, 64, True, False)
    q = Rows(rng.standard_normal((4, 4, 64)).astype(np.float32), True)
    check_attention(hip, cache, q, None, [100000, -5, 320, 7], max_len=100000)          # the page table ends at 320
    check_attention(hip, cache, q, [0, 9, -1, 3], [320, 320, 320, 320])                 # sequences that do not exist: zeros
    table = cache.table.copy()
    table[0, :3], table[1, :], table[2, 5] = -1, cache.n_pages, 2 ** 31 - 1             # pages that do not exist are left out
    cache.table = table
    cache.c.page_table = hip.put(table)
    got = check_attention(hip, cache, q, None, [320, 320, 320, 40])
    assert np.all(got[1] == 0.0)                             # not a single slot left


def test_attention_ignores_what_lies_behind_the_length(hip):
    # the last page's other slots hold NaN (the fixture leaves them so) and infinities
    rng = np.random.default_rng(8)
    lens = [5, 130, 400]
    cache = Cache(hip, rng, lens, 64, 1, 128, False, True)
    cache.v[np.isnan(cache.v)] = np.inf
    cache.d_v = cache._up(cache.v)
    cache.c.v = cache.d_v
    got = check_attention(hip, cache, Rows(rng.standard_normal((3, 2, 128)).astype(np.float32), False), None, lens)
    assert np.all(np.isfinite(got))


def test_attention_with_offsets_past_32_bits(hip):
    # a pool of 5.4 GB each for keys and values; the sequence lives in its last pages
    page, kvh, hd, n_pages = 64, 8, 128, 40960
    bytes_each = n_pages * page * kvh * hd * 2
    rng = np.random.default_rng(9)
    base = []
    for _ in range(2):
        p = C.c_void_p()
        hip.ok(hip.rt.hipMalloc(C.byref(p), bytes_each))
        hip.bufs.append(p)
        base.append(p.value)
    used = np.array([n_pages - 1, 3, n_pages - 2, 32768], np.int32)
    n, heads = 4 * page - 5, 8
    cache = Cache(hip, rng, [n], page, kvh, hd, True, False, spare=0)
    for i, p in enumerate(used):
        for src, dst in ((cache.d_k, base[0]), (cache.d_v, base[1])):
            one = page * kvh * hd * 2
            hip.ok(hip.rt.hipMemcpy(C.c_void_p(dst + int(p) * one), C.c_void_p(src + int(cache.table[0, i]) * one), C.c_size_t(one), 3))
    cache.c.k, cache.c.v, cache.c.n_pages, cache.c.page_table = base[0], base[1], n_pages, hip.put(used)
    q = Rows(rng.standard_normal((1, heads, hd)).astype(np.float32), True)
    check_attention(hip, cache, q, None, [n])
    # and a key appended there
    freq, _ = hipdec.rope_frequencies(hd)
    x = Rows(rng.standard_normal((1, (heads + 2 * kvh) * hd)).astype(np.float32), True)
    d = hip.put(x.raw)
    hipdec.rope_append_paged(Rope.make(hip.put(freq), hd), cache.c, d, d + heads * hd * 2, d + (heads + kvh) * hd * 2, d, hip.put(np.array([4 * page - 1], np.int32)),
                             1, heads, dtype=RowDtype.BF16, row_stride=x.raw.shape[1], q_out_stride=x.raw.shape[1])
    hip.sync()
    got = hip.get(base[1] + (32768 * kvh * page + page - 1) * hd * 2, np.uint16, hd)      # head 0 of the last slot
    assert np.array_equal(got, x.raw[0, (heads + kvh) * hd:(heads + kvh + 1) * hd])


# ---------------------------------------------------------------- verification
def verified(lg, drafts, n, u, T, cap, probs):
    """(tokens, accepted) by the definition, fp64."""
    S, K = drafts.shape
    V = lg.shape[2]
    tokens, accepted = np.full((S, K + 1), NO_TOKEN, np.uint32), np.zeros(S, np.int32)
    for s in range(S):
        i, m = 0, int(np.clip(n[s], 0, K))
        while True:
            z = np.where(np.isnan(lg[s, i]), -np.inf, lg[s, i]).astype(np.float64)
            z = cap * np.tanh(z / cap) if cap > 0 else z
            best = int(np.argmax(z))
            if z[best] == -np.inf:
                p = np.zeros(V)
            elif T > 0:
                p = np.exp((z - z[best]) / T)
                p /= p.sum()
            else:
                p = (np.arange(V) == best).astype(np.float64)
            if i == m:
                break
            d = int(drafts[s, i])
            q = probs[s, i].astype(np.float64) if probs is not None and T > 0 else (np.arange(V) == d).astype(np.float64)
            if not (0 <= d < V and (float(u[s, i]) * q[d] < p[d] if T > 0 else d == best and p[d] > 0)):
                r = np.maximum(p - q, 0.0)
                p = r if r.sum() > 0 and T > 0 else p
                break
            tokens[s, i] = d
            i += 1
        if p.sum() > 0:
            run = np.cumsum(p)
            tokens[s, i] = min(int(np.searchsorted(run, float(u[s, K]) * run[-1], side="right")), int(np.flatnonzero(p)[-1])) if T > 0 else best
        accepted[s] = i
    return tokens, accepted


def verify(hip, lg, drafts, n, u, T, cap=0.0, probs=None, row_pad=0, stream=None):
    S, K = drafts.shape
    V = lg.x.shape[2]
    raw = np.full((S * (K + 1), V + row_pad), np.nan if not lg.b16 else 0x7FC0, lg.raw.dtype)
    raw[:, :V] = lg.raw.reshape(-1, V)
    size = hipdec.verify_drafts_workspace(S, K, V)
    ws = hip.put(np.full(size // 8 + 2, np.nan))
    d_tok, d_acc = hip.put(np.full((S, K + 1), 7, np.uint32)), hip.put(np.full(S, 7, np.int32))
    hipdec.verify_drafts(hip.put(raw), hip.put(drafts) if K else None, hip.put(u) if T > 0 else None, d_tok, d_acc, S, K, V, dtype=lg.dtype,
                         temperature=T, softcap=cap, n_drafts=hip.put(n), draft_probs=hip.put(probs) if probs is not None else None,
                         row_stride=V + row_pad, workspace=ws, workspace_bytes=size, stream=stream)
    hip.sync()
    return hip.get(d_tok, np.uint32, S * (K + 1)).reshape(S, K + 1), hip.get(d_acc, np.int32, S)


def draft_case(rng, S, K, V, b16, T, with_probs):
    lg = Rows(rng.standard_normal((S, K + 1, V)).astype(np.float32) * 3.0, b16)
    guess = lg.x[:, :K] + rng.standard_normal((S, K, V)).astype(np.float32) * 0.5
    e = np.exp((guess - guess.max(-1, keepdims=True)) / (T or 1.0))
    probs = (e / e.sum(-1, keepdims=True)).astype(np.float32)
    cum = probs.astype(np.float64).cumsum(-1)
    drafts = np.minimum((cum < rng.random((S, K, 1)) * cum[..., -1:]).sum(-1), V - 1).astype(np.int32)
    hit = rng.random((S, K)) < 0.5
    drafts = np.where(hit, lg.x[:, :K].argmax(-1), drafts).astype(np.int32) if K else drafts.reshape(S, 0)
    n = rng.integers(0, K + 1, S).astype(np.int32)
    n[0] = K + 9
    return lg, drafts, n, rng.random((S, K + 1), dtype=np.float32), probs if with_probs else None


@pytest.mark.parametrize("S,K,V,b16,T,cap,with_probs,pad", [
    (1, 4, 32768, False, 1.0, 0.0, False, 0), (6, 3, 1000, False, 0.8, 0.0, True, 1), (5, 7, 8191, True, 1.2, 0.0, True, 0),
    (40, 5, 100001, True, 0.7, 30.0, True, 0),               # chunks of 4096
    (3, 2, 262144, False, 1.0, 0.0, True, 0), (9, 1, 1, False, 1.0, 0.0, True, 0), (4, 0, 777, True, 0.9, 0.0, False, 5),
    (8, 4, 5000, False, 0.0, 0.0, True, 0), (8, 3, 257, True, 0.0, 10.0, False, 0), (2, 255, 300, False, 1.0, 0.0, True, 0),
    (16, 4, 4096, False, 0.01, 0.0, True, 0), (16, 4, 4097, False, 20.0, 2.0, False, 0),
])
def test_verify_drafts(hip, S, K, V, b16, T, cap, with_probs, pad):
    rng = np.random.default_rng(S * 7 + V)
    case = draft_case(rng, S, K, V, b16, T, with_probs)
    tokens, accepted = verify(hip, *case[:4], T, cap, case[4], row_pad=pad)
    want, want_acc = verified(case[0].x, *case[1:4], T, cap, case[4])
    assert np.array_equal(accepted, want_acc) and np.array_equal(tokens, want)


def test_verify_drafts_out_of_the_ordinary(hip):
    rng = np.random.default_rng(3)
    S, K, V, T = 9, 3, 3000, 0.9
    lg, drafts, n, u, probs = draft_case(rng, S, K, V, False, T, True)
    n[:] = K
    x = lg.x
    x[0, 0] = -np.inf                                        # a row without a possible token
    x[1, :, ::2] = np.nan                                    # impossible tokens
    x[2, :, 5], drafts[2] = np.inf, 5                        # one that takes everything
    probs[3] = 1.0                                           # the draft covers the target everywhere
    drafts[4] = [-1, V, 5]                                   # no such tokens
    u[5] = 0.0                                               # the first possible token
    x[5, :, :100] = -np.inf
    u[6, K] = 1.0                                            # the last possible token
    probs[7, :, 1::2] = np.nan
    x[8] = np.floor(x[8])                                    # ties
    for T in (0.9, 0.0):
        tokens, accepted = verify(hip, Rows(x, False), drafts, n, u, T, 0.0, probs)
        with np.errstate(invalid="ignore"):
            ref = np.where(np.isposinf(x), np.float32(3.4028235e38), x)
            p_ref = np.where(np.isnan(probs), np.float32(np.inf), probs)      # p - NaN leaves nothing, and so does p - inf
            want, want_acc = verified(ref, drafts, n, u, T, 0.0, p_ref)
        assert np.array_equal(accepted, want_acc) and np.array_equal(tokens, want), T
    assert tokens[0, 0] == NO_TOKEN


def test_verified_tokens_follow_the_target_s_distribution(hip):
    # 20000 sequences of one draft each: kept and redrawn tokens together are distributed as the target's softmax
    rng = np.random.default_rng(12)
    S, V = 20000, 5
    z = np.array([0.3, -1.0, 1.2, 0.0, 0.7], np.float32)
    q = np.array([0.4, 0.3, 0.1, 0.15, 0.05], np.float32)
    drafts = rng.choice(V, S, p=(q / q.sum()).astype(np.float64) / (q / q.sum()).astype(np.float64).sum()).astype(np.int32)[:, None]
    tokens, _ = verify(hip, Rows(np.broadcast_to(z, (S, 2, V)).copy(), False), drafts, np.ones(S, np.int32), rng.random((S, 2), dtype=np.float32), 1.0,
                       probs=np.broadcast_to(q, (S, 1, V)).copy())
    p = np.exp(z.astype(np.float64))
    p /= p.sum()
    share = np.bincount(tokens[:, 0], minlength=V) / S
    assert np.all(np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / S))          # five standard deviations


# ---------------------------------------------------------------- together
class Server:
    """Three requests of one attention layer whose output is projected to logits on the host side of the test: prompts
    appended at once, then steps of a draft's rows (append, attention, verification), all state on the device."""

    def __init__(self, hip, seed, stream=None):
        rng = np.random.default_rng(seed)
        self.hip, self.stream, self.S, self.K, self.V = hip, stream, 3, 2, 500
        self.heads, self.kvh, self.hd, self.page = 8, 2, 64, 8
        self.rows = self.S * (self.K + 1)
        self.cache = Cache(hip, rng, [120] * self.S, self.page, self.kvh, self.hd, True, False, fill=False)
        self.freq, self.mag = hipdec.rope_frequencies(self.hd, scaling=RopeScaling.LINEAR, factor=2.0)
        self.rope = Rope.make(hip.put(self.freq), self.hd, interleaved=False, magnitude=self.mag)
        self.wide = (self.heads + 2 * self.kvh) * self.hd
        size = hipdec.attention_paged_workspace(self.rows, self.heads, self.kvh, self.hd, 120 * 8)
        self.ws, self.ws_size = (hip.put(np.zeros(size // 4 + 4, np.float32)) if size else None), size
        vsize = hipdec.verify_drafts_workspace(self.S, self.K, self.V)
        self.vws, self.vws_size = hip.put(np.zeros(vsize // 8 + 2)), vsize
        self.d = {k: hip.put(np.zeros(n, t)) for k, n, t in (
            ("x", self.rows * self.wide, np.float32), ("q", self.rows * self.heads * self.hd, np.float32),
            ("out", self.rows * self.heads * self.hd, np.float32), ("pos", self.rows, np.int32), ("seqs", self.rows, np.int32),
            ("lens", self.rows, np.int32), ("logits", self.rows * self.V, np.float32), ("drafts", self.S * self.K, np.int32),
            ("u", self.rows, np.float32), ("tokens", self.rows, np.uint32), ("accepted", self.S, np.int32))}

    def put(self, name, a):
        a = np.ascontiguousarray(a)
        self.hip.ok(self.hip.rt.hipMemcpy(C.c_void_p(self.d[name]), a.ctypes.data_as(C.c_void_p), C.c_size_t(a.nbytes), 1))

    def step(self):
        """Enqueues one step of all rows."""
        q, kv, d = self.heads * self.hd, self.kvh * self.hd, self.d
        hipdec.rope_append_paged(self.rope, self.cache.c, d["x"], d["x"] + 4 * q, d["x"] + 4 * (q + kv), d["q"], d["pos"], self.rows, self.heads,
                                 seqs=d["seqs"], row_stride=self.wide, stream=self.stream)
        hipdec.attention_paged(self.cache.c, d["q"], d["out"], d["lens"], self.rows, self.heads, 120 * 8, seqs=d["seqs"], workspace=self.ws,
                               workspace_bytes=self.ws_size, stream=self.stream)
        hipdec.verify_drafts(d["logits"], d["drafts"], d["u"], d["tokens"], d["accepted"], self.S, self.K, self.V, temperature=0.8,
                             workspace=self.vws, workspace_bytes=self.vws_size, stream=self.stream)

    def inputs(self, rng, lens):
        """Random inputs for rows at the sequences' present lengths; returns what the step has to give, fp64."""
        K = self.K
        pos = np.array([lens[s] + i for s in range(self.S) for i in range(K + 1)], np.int32)
        seqs = np.repeat(np.arange(self.S), K + 1).astype(np.int32)
        x = rng.standard_normal((self.rows, self.wide)).astype(np.float32)
        lg, drafts, _, u, _ = draft_case(rng, self.S, K, self.V, False, 0.8, False)
        for name, a in (("x", x), ("pos", pos), ("seqs", seqs), ("lens", pos + 1), ("logits", lg.raw), ("drafts", drafts), ("u", u)):
            self.put(name, a)
        h, kv, hd = self.heads, self.kvh, self.hd
        q, k, v = (x[:, a * hd:b * hd].reshape(self.rows, -1, hd) for a, b in ((0, h), (h, h + kv), (h + kv, h + 2 * kv)))
        q, k = (turned(a, pos, self.freq, self.mag, hd, False).astype(np.float32) for a in (q, k))
        c = self.cache
        for t in range(self.rows):
            p, s = c.table[seqs[t], pos[t] // c.page], pos[t] % c.page
            c.k[p, s], c.v[p, s] = of_bf16(to_bf16(k[t])), of_bf16(to_bf16(v[t]))
        out, tol = attended(c, q, seqs, pos + 1, hd ** -0.5)
        # (keys on the border of a bf16 rounding, and queries, may differ by that or an fp32 rounding of the turn: each key by
        # 2^-8 of itself, hardly ever; a score by 2^-8 |q||k| scale of one key)
        return out, tol, verified(lg.x, drafts, np.full(self.S, K), u, 0.8, 0.0, None)

    def check(self, want):
        out, tol, (tokens, accepted) = want
        got = fetch(self.hip, self.d["out"], out.shape, False)
        assert np.abs(got - out).max() < 2.0 ** -8 * 4 and np.mean(np.abs(got - out) <= tol + 4e-6) > 0.9
        assert np.array_equal(self.hip.get(self.d["tokens"], np.uint32, self.rows).reshape(self.S, -1), tokens)
        assert np.array_equal(self.hip.get(self.d["accepted"], np.int32, self.S), accepted)
        return got, accepted


def test_the_operators_together_eager_and_captured(hip):
    """Steps whose lengths follow the accepted drafts, once eagerly and once replayed from a graph (with the program's own
    copies and waits between the replays): the same results bit for bit, and the fp64 restatement's."""
    runs = []
    for captured in (False, True):
        stream = hip.stream()
        srv = Server(hip, 1, stream.value)
        rng = np.random.default_rng(77)
        lens, got, exe = [0, 5, 60], [], C.c_void_p()
        for s, n in enumerate(lens):                         # what the earlier positions hold
            for i in range(n):
                p, a = srv.cache.table[s, i // 8], i % 8
                srv.cache.k[p, a], srv.cache.v[p, a] = (of_bf16(to_bf16(rng.standard_normal((2, 64)))) for _ in range(2))
        srv.cache.c.k, srv.cache.c.v = srv.cache._up(srv.cache.k), srv.cache._up(srv.cache.v)
        if captured:
            g = C.c_void_p()
            hip.ok(hip.rt.hipStreamBeginCapture(stream, 0))
            srv.step()
            hip.ok(hip.rt.hipStreamEndCapture(stream, C.byref(g)))
            hip.ok(hip.rt.hipGraphInstantiate(C.byref(exe), g, None, None, 0))
            hip.ok(hip.rt.hipGraphDestroy(g))
        for step in range(6):
            want = srv.inputs(rng, lens)
            hip.sync()
            if captured:
                hip.ok(hip.rt.hipGraphLaunch(exe, stream))
            else:
                srv.step()
            hip.ok(hip.rt.hipStreamSynchronize(stream))
            out, accepted = srv.check(want)
            got.append(out)
            lens = [n + int(a) + 1 for n, a in zip(lens, accepted)]
        runs.append(got)
        if captured:
            hip.ok(hip.rt.hipGraphExecDestroy(exe))
        hip.ok(hip.rt.hipStreamDestroy(stream))
    for a, b in zip(*runs):
        assert np.array_equal(a, b)


def test_two_streams_at_once_with_workspaces_of_their_own(hip):
    streams = [hip.stream(), hip.stream()]
    rng = np.random.default_rng(21)
    jobs = []
    for i, s in enumerate(streams):
        lens = [700 + 31 * i, 900, 33]
        cache = Cache(hip, rng, lens, 16, 2, 128, True, bool(i))
        q = Rows(rng.standard_normal((3, 8, 128)).astype(np.float32), True)
        size = hipdec.attention_paged_workspace(3, 8, 2, 128, 4000)
        case = draft_case(rng, 6, 3, 20000, False, 0.9, True)
        vsize = hipdec.verify_drafts_workspace(6, 3, 20000)
        jobs.append(dict(s=s, lens=lens, cache=cache, q=q, size=size, vsize=vsize, case=case, d_q=hip.put(q.raw), d_out=hip.put(np.zeros_like(q.raw)),
                         d_lens=hip.put(np.asarray(lens, np.int32)), ws=hip.put(np.zeros(size // 4 + 4, np.float32)), vws=hip.put(np.zeros(vsize // 8 + 2)),
                         lg=hip.put(case[0].raw), dr=hip.put(case[1]), n=hip.put(case[2]), u=hip.put(case[3]), p=hip.put(case[4]),
                         tok=hip.put(np.zeros((6, 4), np.uint32)), acc=hip.put(np.zeros(6, np.int32))))
    hip.sync()
    for _ in range(5):
        for j in jobs:
            hipdec.attention_paged(j["cache"].c, j["d_q"], j["d_out"], j["d_lens"], 3, 8, 4000, dtype=RowDtype.BF16, workspace=j["ws"],
                                   workspace_bytes=j["size"], stream=j["s"].value)
            hipdec.verify_drafts(j["lg"], j["dr"], j["u"], j["tok"], j["acc"], 6, 3, 20000, temperature=0.9, n_drafts=j["n"], draft_probs=j["p"],
                                 workspace=j["vws"], workspace_bytes=j["vsize"], stream=j["s"].value)
    hip.sync()
    for j in jobs:
        want, tol = attended(j["cache"], j["q"].x, [0, 1, 2], j["lens"], 128 ** -0.5)
        assert np.all(np.abs(fetch(hip, j["d_out"], want.shape, True) - want) <= tol + 2.0 ** -8 * np.abs(want))
        tokens, accepted = verified(j["case"][0].x, *j["case"][1:4], 0.9, 0.0, j["case"][4])
        assert np.array_equal(hip.get(j["tok"], np.uint32, 24).reshape(6, 4), tokens) and np.array_equal(hip.get(j["acc"], np.int32, 6), accepted)
    for s in streams:
        hip.ok(hip.rt.hipStreamDestroy(s))


@pytest.mark.parametrize("cap", [1e8, 1e14, 1e30, 3.4e38])
def test_a_cap_far_above_the_logits_changes_nothing(hip, cap):
    """|softcap(x) - x| < |x|^3 / (3 cap^2): below 2e-12 for |x| <= 40, as small as the draws' own rounding."""
    rng = np.random.default_rng(43)
    case = draft_case(rng, 6, 4, 2000, False, 0.8, True)
    plain, plain_acc = verify(hip, *case[:4], 0.8, 0.0, case[4])
    tokens, accepted = verify(hip, *case[:4], 0.8, cap, case[4])
    assert np.array_equal(accepted, plain_acc) and np.array_equal(tokens, plain)


@pytest.mark.parametrize("handle", [None, 1, 2])             # the default stream, its other handle, the thread's own
def test_the_streams_that_are_no_objects(hip, handle):
    rng = np.random.default_rng(41)
    lens = [40, 700]
    cache = Cache(hip, rng, lens, 16, 2, 64, True, False)
    check_attention(hip, cache, Rows(rng.standard_normal((2, 4, 64)).astype(np.float32), True), None, lens, stream=handle)
    case = draft_case(rng, 2, 3, 900, False, 0.9, True)
    tokens, accepted = verify(hip, *case[:4], 0.9, 0.0, case[4], stream=handle)
    want, want_acc = verified(case[0].x, *case[1:4], 0.9, 0.0, case[4])
    assert np.array_equal(accepted, want_acc) and np.array_equal(tokens, want)


def test_repeated_calls_give_the_same_bits(hip):
    rng = np.random.default_rng(31)
    lens = [5000, 64, 1999, 2000]
    cache = Cache(hip, rng, lens, 32, 2, 128, True, False)
    q = Rows(rng.standard_normal((4, 12, 128)).astype(np.float32), False)
    first = attend(hip, cache, q, None, lens)
    for _ in range(4):
        assert np.array_equal(attend(hip, cache, q, None, lens), first)
    # a row's result does not depend on the rows beside it (the same split)
    alone = attend(hip, cache, q, None, lens, max_len=5000)
    assert np.array_equal(alone, first)


def test_host_memory_is_refused(hip):
    rng = np.random.default_rng(1)
    cache = Cache(hip, rng, [20], 16, 2, 64, True, False)
    host = np.zeros(4096, np.float32)
    here = hip.put(np.zeros(4096, np.float32))
    for kw in (dict(q=host.ctypes.data & ~15, out=here), dict(q=here, out=host.ctypes.data & ~15)):
        with pytest.raises(hipdec.HipDecodeError) as e:
            hipdec.attention_paged(cache.c, kw["q"], kw["out"], hip.put(np.array([20], np.int32)), 1, 4, 20)
        assert e.value.status == hipdec.ERR_ARG and "device" in str(e.value)
