"""The serving operators on device buffers, as they are measured: rotary positions with the append to a paged
key-value cache, attention of new tokens over that cache, and the verification of drafted tokens.

`own` chooses between the elementary torch form of each operator and the library's entry points
(rustane_amd.hipdec); both take what prepare() made.  A pass is one call of one operator.
"""
import math

import torch

own = False

GOLDEN = 0.6180339887498949
F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"f32": F32, "bf16": BF16}
NO_TOKEN = -1            # what stands behind the last token of a sequence (0xffffffff as an unsigned number)


# ---------------------------------------------------------------- the cases
def _rope(name, tokens, heads, kv_heads, hd, rot, interleaved, scaling, far, rows, cache, page, token_major, prompt):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "hd": hd, "rot": rot,
            "interleaved": interleaved, "scaling": scaling, "far": far, "rows": rows, "cache": cache, "page": page,
            "token_major": token_major, "prompt": prompt}


def _attn(name, seqs, per_seq, low, high, heads, kv_heads, hd, rows, cache, page, token_major, empty=False):
    return {"name": name, "op": "attention", "seqs": seqs, "per_seq": per_seq, "low": low, "high": high, "heads": heads,
            "kv_heads": kv_heads, "hd": hd, "rows": rows, "cache": cache, "page": page, "token_major": token_major,
            "empty": empty}


def _verify(name, seqs, drafts, vocab, logits, probs, temperature, softcap, ragged):
    return {"name": name, "op": "verify", "seqs": seqs, "drafts": drafts, "vocab": vocab, "logits": logits, "probs": probs,
            "temperature": temperature, "softcap": softcap, "ragged": ragged}


def listed():
    return [
        # one decoded token of the 600M model (12 heads of 128, interleaved pairs): the smallest call, all latency
        _rope("rope_token_600m", 1, 12, 12, 128, 128, True, "plain", 2048, "f32", "bf16", 16, True, False),
        # 32 requests stepped together, grouped heads, half of each head rotated, positions far past the trained window
        _rope("rope_32_requests_far", 32, 32, 8, 128, 64, False, "parts", 131072, "bf16", "bf16", 64, False, False),
        # one prompt chunk of the 5B model
        _rope("rope_prompt_5b", 1024, 32, 32, 128, 128, True, "plain", 4096, "f32", "bf16", 16, True, True),
        # a long prompt at once, grouped heads, an odd number of rows: bandwidth
        _rope("rope_long_prompt", 8191, 32, 8, 128, 128, False, "ntk", 32768, "bf16", "bf16", 64, False, True),
        # one request of the 600M model after its 128-token prompt and 256 steps
        _attn("attn_token_600m", 1, 1, 385, 385, 12, 12, 128, "f32", "bf16", 16, True),
        # eight requests of the 600M model with prompts around 512 tokens
        _attn("attn_8_requests_600m", 8, 1, 513, 767, 12, 12, 128, "f32", "bf16", 16, True),
        # one request with a long context: few rows, so the cache's length is what can be split
        _attn("attn_long_context", 1, 1, 65536, 65536, 32, 8, 128, "bf16", "bf16", 64, False),
        # a full server: 64 requests of very different lengths, grouped heads
        _attn("attn_64_ragged", 64, 1, 1, 8192, 32, 8, 128, "bf16", "bf16", 64, False),
        # the rows of four drafts with four tokens each (a draft's rows read the same cache), fp32 cache, small pages
        _attn("attn_drafts_f32", 4, 5, 300, 1500, 8, 2, 64, "f32", "f32", 8, False, True),
        # four tokens looked up in the prompt, one request: no draft probabilities
        _verify("verify_lookup", 1, 4, 32768, "f32", False, 1.0, 0.0, False),
        # 32 requests with seven tokens each from a draft model, unequal draft lengths
        _verify("verify_32_requests", 32, 7, 32768, "f32", True, 0.8, 0.0, True),
        # a large vocabulary of odd size, logits in bf16
        _verify("verify_large_vocab", 64, 5, 131071, "bf16", True, 0.7, 30.0, True),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    largest = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("rope", "attention", "verify")}
    op = rng.choice(("rope", "attention", "attention", "verify"))
    while True:
        heads, kv_heads = rng.choice(((10, 10), (8, 8), (32, 32), (32, 8), (8, 2), (14, 2), (40, 8), (18, 1), (32, 1), (5, 1), (1, 1)))
        hd = rng.choice((64, 128, 192, 256))
        rows, cache = rng.choice((("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")))
        page, token_major = rng.choice((1, 4, 8, 16, 32, 64, 256)), rng.random() < 0.5
        if op == "rope":
            rot = rng.choice((hd, hd, hd // 2, hd // 4, hd - 2))
            prompt = rng.random() < 0.5
            case = _rope("", _spread(rng, 1, 8191 if prompt else 128), heads, kv_heads, hd, rot, rng.random() < 0.5,
                         rng.choice(("plain", "linear", "ntk", "parts")), _spread(rng, 8192, 1 << 20), rows, cache,
                         min(page, 64), token_major, prompt)
        elif op == "attention":
            high = _spread(rng, 1, 65536)
            low = high if rng.random() < 0.3 else rng.randint(1, high)
            case = _attn("", _spread(rng, 1, 128), rng.choice((1, 1, 1, 3, 8)), low, high, heads, kv_heads, hd, rows, cache,
                         page, token_major, rng.random() < 0.3)
        else:
            case = _verify("", _spread(rng, 1, 64), rng.choice((1, 2, 3, 4, 5, 7, 8)), _spread(rng, 500, 200000),
                           rng.choice(("f32", "bf16")), rng.random() < 0.6, rng.choice((0.0, 0.6, 0.8, 1.0, 1.5)),
                           rng.choice((0.0, 0.0, 30.0)), rng.random() < 0.5)
        if _cost(case) <= largest[op]:
            del case["name"]
            return case


def _cost(case):
    """What bounds the memory and time of either form: elements touched, padding included."""
    if case["op"] == "rope":
        return case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["hd"]
    if case["op"] == "attention":
        return case["seqs"] * case["per_seq"] * (case["high"] + 64) * (case["kv_heads"] + 8) * case["hd"]
    return case["seqs"] * (case["drafts"] + 1) * case["vocab"]


def _lengths(case):
    """Cache length of each row: sequence s has a length of [low, high], and its rows (a draft's) one entry more each."""
    out = [case["low"] + int(((s + 1) * GOLDEN) % 1.0 * (case["high"] - case["low"] + 1)) + i
           for s in range(case["seqs"]) for i in range(case["per_seq"])]
    return out[:-1] + [0] if case["empty"] and len(out) > 1 else out


def _draft_lengths(case):
    return [(case["drafts"] - int(((s + 1) * GOLDEN) % 1.0 * (case["drafts"] + 1)) if case["ragged"] else case["drafts"])
            for s in range(case["seqs"])]


def work(case):
    size = {"f32": 4, "bf16": 2}
    if case["op"] == "rope":
        q, k = case["tokens"] * case["heads"] * case["hd"], case["tokens"] * case["kv_heads"] * case["hd"]
        rows, cache = size[case["rows"]], size[case["cache"]]
        turned = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"]
        return {"bytes": 2 * q * rows + 2 * k * rows + 2 * k * cache + 12 * case["tokens"], "flops": 3 * turned}
    if case["op"] == "attention":
        lens = _lengths(case)
        kept = sum(max(lens[s * case["per_seq"]:(s + 1) * case["per_seq"]]) for s in range(case["seqs"]))
        row = case["heads"] * case["hd"]
        return {"bytes": 2 * kept * case["kv_heads"] * case["hd"] * size[case["cache"]] + 2 * len(lens) * row * size[case["rows"]],
                "flops": 4 * sum(lens) * row}
    drafts = _draft_lengths(case)
    rows = sum(drafts) + case["seqs"]
    return {"bytes": rows * case["vocab"] * size[case["logits"]] + (case["seqs"] * case["vocab"] * 4 if case["probs"] else 0),
            "flops": 4 * rows * case["vocab"]}


# ---------------------------------------------------------------- what a program has in hand
def _frequencies(rot, scaling):
    """Angle per position of each rotated pair, and the factor on the rotated numbers, for contexts eight times as
    long as the 4096 positions trained on."""
    base, trained, scale = 10000.0, 4096, 8.0
    p = torch.arange(rot // 2, dtype=torch.float64) * (2.0 / rot)
    if scaling == "ntk":
        return (base * scale ** (rot / max(rot - 2, 1))) ** -p, 1.0
    f = base ** -p
    if scaling == "linear":
        return f / scale, 1.0
    if scaling == "parts":
        turns = trained * f / (2.0 * math.pi)                # full turns within the trained window
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * keep + f / scale * (1.0 - keep), 0.1 * math.log(scale) + 1.0
    return f, 1.0


def _pool(pages, case, gen, filled):
    shape = ((pages, case["page"], case["kv_heads"], case["hd"]) if case["token_major"]
             else (pages, case["kv_heads"], case["page"], case["hd"]))
    if not filled:
        return torch.zeros(shape, device="cuda", dtype=TYPES[case["cache"]])
    return torch.randn(shape, device="cuda", dtype=F32, generator=gen).to(TYPES[case["cache"]])


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = case
    if c["op"] == "rope":
        t, width = c["tokens"], (c["heads"] + 2 * c["kv_heads"]) * c["hd"]
        qkv = torch.randn((t, width), device="cuda", dtype=F32, generator=gen).to(TYPES[c["rows"]])
        offset = torch.randint(0, c["far"], (1,), device="cuda", generator=gen)
        if c["prompt"]:                                      # one request: neighbouring positions
            seqs, slots = [0] * t, list(range(5, 5 + t))
            pos = (offset + torch.arange(t, device="cuda")).to(torch.int32)
        else:                                                # every row a request of its own
            seqs, slots = list(range(t)), [int((i + 1) * GOLDEN % 1.0 * 100) for i in range(t)]
            pos = torch.randint(0, c["far"], (t,), device="cuda", generator=gen).to(torch.int32)
        n_seqs = 1 if c["prompt"] else t
        per = -(-(max(slots) + 1) // c["page"])
        pages = n_seqs * per + 3
        table = torch.randperm(pages, device="cuda", generator=gen)[:n_seqs * per].reshape(n_seqs, per).to(torch.int32)
        freq, magnitude = _frequencies(c["rot"], c["scaling"])
        return {"qkv": qkv, "pos": pos, "slots": _int(slots), "seqs": _int(seqs), "table": table, "freq": freq.cuda(),
                "magnitude": magnitude, "k": _pool(pages, c, gen, False), "v": _pool(pages, c, gen, False)}
    if c["op"] == "attention":
        lens = _lengths(c)
        per = -(-max(max(lens), 1) // c["page"])
        pages = c["seqs"] * per + 3
        table = torch.randperm(pages, device="cuda", generator=gen)[:c["seqs"] * per].reshape(c["seqs"], per).to(torch.int32)
        q = torch.randn((len(lens), c["heads"], c["hd"]), device="cuda", dtype=F32, generator=gen)
        q *= 0.5 + 2.0 * torch.rand((1, c["heads"], 1), device="cuda", generator=gen)       # heads of unequal sharpness
        return {"q": q.to(TYPES[c["rows"]]), "lens": _int(lens), "table": table, "max_len": max(lens),
                "seqs": _int([s for s in range(c["seqs"]) for _ in range(c["per_seq"])]),
                "k": _pool(pages, c, gen, True), "v": _pool(pages, c, gen, True)}
    s, d, v = c["seqs"], c["drafts"], c["vocab"]
    logits = (3.0 * torch.randn((s, d + 1, v), device="cuda", dtype=F32, generator=gen)).to(TYPES[c["logits"]])
    guess = logits[:, :d].float() + 0.7 * torch.randn((s, d, v), device="cuda", dtype=F32, generator=gen)
    probs = torch.softmax(guess / (c["temperature"] or 1.0), dim=-1)
    u = torch.rand((s, d, 1), device="cuda", dtype=torch.float64, generator=gen) * 0.999999
    drafts = (probs.double().cumsum(-1) <= u).sum(-1).clamp(max=v - 1).to(torch.int32)
    if not c["probs"]:                                       # a looked-up draft: right more often than not
        hit = torch.rand((s, d), device="cuda", generator=gen) < 0.6
        drafts = torch.where(hit, logits[:, :d].float().argmax(-1).to(torch.int32), drafts)
    return {"logits": logits, "drafts": drafts.contiguous(), "n_drafts": _int(_draft_lengths(c)),
            "probs": probs.contiguous() if c["probs"] else None,
            "uniforms": torch.rand((s, d + 1), device="cuda", dtype=F32, generator=gen)}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:                                                  # the handles, outputs and workspace that a server keeps
        from rustane_amd import hipdec
        c, device = case, {"device": "cuda"}
        if c["op"] == "verify":
            state["tokens"] = torch.empty((c["seqs"], c["drafts"] + 1), dtype=torch.int32, **device)
            state["accepted"] = torch.empty(c["seqs"], dtype=torch.int32, **device)
            size = hipdec.verify_drafts_workspace(c["seqs"], c["drafts"], c["vocab"])
        else:
            state["cache"] = hipdec.PagedCache.make(
                state["k"].data_ptr(), state["v"].data_ptr(), hipdec.KvDtype[c["cache"].upper()], n_pages=state["k"].shape[0],
                page_size=c["page"], kv_heads=c["kv_heads"], hd=c["hd"], page_table=state["table"].data_ptr(),
                n_seqs=state["table"].shape[0], max_pages=state["table"].shape[1], token_major=c["token_major"])
        if c["op"] == "rope":
            state["rope"] = hipdec.Rope.make(state["freq"].data_ptr(), c["rot"], interleaved=c["interleaved"],
                                             magnitude=state["magnitude"])
            state["q_out"] = torch.empty((c["tokens"], c["heads"], c["hd"]), dtype=TYPES[c["rows"]], **device)
        else:
            if c["op"] == "attention":
                state["out"] = torch.empty_like(state["q"])
                size = hipdec.attention_paged_workspace(len(state["lens"]), c["heads"], c["kv_heads"], c["hd"], state["max_len"])
            state["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, **device)
    return state


# ---------------------------------------------------------------- the plain forms
def _by_position(pool, case):
    """The pool as [page][slot][kv head][hd] whatever its layout."""
    return pool if case["token_major"] else pool.permute(0, 2, 1, 3)


def _rotated(x, angle, magnitude, case):
    rot = case["rot"]
    cos = (angle.cos() * magnitude).float()[:, None]
    sin = (angle.sin() * magnitude).float()[:, None]
    x = x.float()
    turn = x[..., :rot]
    if case["interleaved"]:
        a, b = turn[..., 0::2], turn[..., 1::2]
        done = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turn[..., :rot // 2], turn[..., rot // 2:]
        done = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((done, x[..., rot:]), dim=-1)


def _plain_rope(st):
    c = st["case"]
    t, hd = c["tokens"], c["hd"]
    q, k, v = st["qkv"].split((c["heads"] * hd, c["kv_heads"] * hd, c["kv_heads"] * hd), dim=1)
    angle = st["pos"].double()[:, None] * st["freq"]          # far positions: the angle needs 64 bits
    q = _rotated(q.reshape(t, -1, hd), angle, st["magnitude"], c).to(TYPES[c["rows"]])
    k = _rotated(k.reshape(t, -1, hd), angle, st["magnitude"], c)
    slot = st["slots"].long()
    page = st["table"].long()[st["seqs"].long(), slot // c["page"]]
    _by_position(st["k"], c)[page, slot % c["page"]] = k.to(TYPES[c["cache"]])
    _by_position(st["v"], c)[page, slot % c["page"]] = v.reshape(t, -1, hd).to(TYPES[c["cache"]])
    return {"q": q, "k": st["k"], "v": st["v"]}


def _plain_attention(st):
    c = st["case"]
    r, n = len(st["lens"]), st["max_len"]
    g = c["heads"] // c["kv_heads"]
    slot = torch.arange(n, device="cuda")
    page = st["table"].long()[st["seqs"].long()][:, slot // c["page"]]                     # [row][slot]
    k = _by_position(st["k"], c)[page, slot % c["page"]].float().permute(0, 2, 3, 1).contiguous()
    q = st["q"].float().reshape(r, c["kv_heads"], g, c["hd"]) * (1.0 / math.sqrt(c["hd"]))
    score = torch.matmul(q, k)                                                             # [row][kv head][g][slot]
    del k
    seen = (slot < st["lens"][:, None])[:, None, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    weight = weight / torch.where(total > 0, total, 1.0)
    v = _by_position(st["v"], c)[page, slot % c["page"]].float().permute(0, 2, 1, 3).contiguous()
    return torch.matmul(weight, v).reshape(r, c["heads"], c["hd"]).to(TYPES[c["rows"]])


def _plain_verify(st):
    c = st["case"]
    s, d, v = c["seqs"], c["drafts"], c["vocab"]
    z = st["logits"].double()                                 # whole numbers come out: 64 bits near the borders
    if c["softcap"] > 0:
        z = c["softcap"] * torch.tanh(z / c["softcap"])
    best = z.argmax(-1)
    if c["temperature"] > 0:
        w = torch.exp((z - z.amax(-1, keepdim=True)) / c["temperature"])
        p = w / w.sum(-1, keepdim=True)
    else:
        p = torch.zeros_like(z).scatter_(-1, best[..., None], 1.0)
    step = torch.arange(d, device="cuda")
    drafted = step < st["n_drafts"][:, None]
    token = st["drafts"].long()
    target = p[:, :d].gather(-1, token[..., None])[..., 0]
    if st["probs"] is None or c["temperature"] == 0:
        guess = torch.zeros_like(p[:, :d]).scatter_(-1, token[..., None], 1.0)
    else:
        guess = st["probs"].double()
    u = st["uniforms"].double()
    agreed = drafted & (u[:, :d] * guess.gather(-1, token[..., None])[..., 0] < target)
    accepted = agreed.long().cumprod(-1).sum(-1)
    at = accepted[:, None, None].expand(s, 1, v)
    row = p.gather(1, at)[:, 0]
    rejected = accepted < st["n_drafts"]
    other = guess.gather(1, at.clamp(max=d - 1))[:, 0]
    rest = (row - other).clamp(min=0)
    row = torch.where(rejected[:, None] & (rest.sum(-1, keepdim=True) > 0), rest, row)
    run = row.cumsum(-1)
    drawn = (run <= u[:, d:] * run[:, -1:]).sum(-1)
    drawn = torch.minimum(drawn, v - 1 - (row.flip(-1) > 0).long().argmax(-1))             # never past the last possible token
    if c["temperature"] == 0:
        drawn = best.gather(1, accepted[:, None])[:, 0]
    step = torch.arange(d + 1, device="cuda")
    tokens = torch.cat((token, token[:, :1]), dim=1)
    tokens = torch.where(step < accepted[:, None], tokens, torch.where(step == accepted[:, None], drawn[:, None], NO_TOKEN))
    return {"tokens": tokens.to(torch.int32), "accepted": accepted.to(torch.int32)}


# ---------------------------------------------------------------- the library's calls
def _own(st):
    from rustane_amd import hipdec
    c, stream = st["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "rope":
        rows, size = st["qkv"].data_ptr(), st["qkv"].element_size()
        width, wide = c["heads"] * c["hd"], c["kv_heads"] * c["hd"]
        hipdec.rope_append_paged(st["rope"], st["cache"], rows, rows + width * size, rows + (width + wide) * size,
                                 st["q_out"].data_ptr(), st["pos"].data_ptr(), n_rows=c["tokens"], heads=c["heads"],
                                 dtype=hipdec.RowDtype[c["rows"].upper()], slots=st["slots"].data_ptr(),
                                 seqs=st["seqs"].data_ptr(), row_stride=width + 2 * wide, stream=stream)
        return {"q": st["q_out"], "k": st["k"], "v": st["v"]}
    if c["op"] == "attention":
        hipdec.attention_paged(st["cache"], st["q"].data_ptr(), st["out"].data_ptr(), st["lens"].data_ptr(),
                               n_rows=len(st["lens"]), heads=c["heads"], max_len=st["max_len"],
                               dtype=hipdec.RowDtype[c["rows"].upper()], seqs=st["seqs"].data_ptr(),
                               workspace=st["workspace"].data_ptr(), workspace_bytes=st["workspace"].numel(), stream=stream)
        return st["out"]
    hipdec.verify_drafts(st["logits"].data_ptr(), st["drafts"].data_ptr(), st["uniforms"].data_ptr(),
                         st["tokens"].data_ptr(), st["accepted"].data_ptr(), n_seqs=c["seqs"], max_drafts=c["drafts"],
                         vocab=c["vocab"], dtype=hipdec.RowDtype[c["logits"].upper()], temperature=c["temperature"],
                         softcap=c["softcap"], n_drafts=st["n_drafts"].data_ptr(),
                         draft_probs=None if st["probs"] is None else st["probs"].data_ptr(),
                         workspace=st["workspace"].data_ptr(), workspace_bytes=st["workspace"].numel(), stream=stream)
    return {"tokens": st["tokens"], "accepted": st["accepted"]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_rope(state) if op == "rope" else _plain_attention(state) if op == "attention" else _plain_verify(state)


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    c, st = case, _inputs(case, seed)
    if c["op"] == "rope":
        hd, rot, half = c["hd"], c["rot"], c["rot"] // 2
        x = st["qkv"].double().reshape(c["tokens"], -1, hd)
        turned = x[:, :c["heads"] + c["kv_heads"]]
        even = torch.arange(half, device="cuda") * (2 if c["interleaved"] else 1)
        odd = even + (1 if c["interleaved"] else half)
        phase = torch.polar(torch.full((c["tokens"], 1, half), st["magnitude"], dtype=torch.float64, device="cuda"),
                            (st["pos"].double()[:, None] * st["freq"])[:, None])
        z = torch.complex(turned[..., even], turned[..., odd]) * phase
        done = turned.clone()
        done[..., even], done[..., odd] = z.real, z.imag
        k, v = st["k"].double(), st["v"].double()
        slots, seqs, table = st["slots"].tolist(), st["seqs"].tolist(), st["table"].tolist()
        at = torch.tensor([table[s][p // c["page"]] * c["page"] + p % c["page"] for s, p in zip(seqs, slots)], device="cuda")
        for pool, rows in ((k, done[:, c["heads"]:]), (v, x[:, c["heads"] + c["kv_heads"]:])):
            flat = (pool if c["token_major"] else pool.transpose(1, 2)).reshape(-1, c["kv_heads"], hd).clone()
            flat[at] = rows
            flat = flat.reshape(-1, c["page"], c["kv_heads"], hd)
            pool.copy_(flat if c["token_major"] else flat.transpose(1, 2))
        return {"q": done[:, :c["heads"]], "k": k, "v": v}
    if c["op"] == "attention":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        g = c["heads"] // c["kv_heads"]
        for r, (n, s) in enumerate(zip(st["lens"].tolist(), st["seqs"].tolist())):
            pages = st["table"][s, :-(-n // c["page"])].long()
            order = (0, 1, 2, 3) if c["token_major"] else (0, 2, 1, 3)
            k, v = ((st[x][pages].permute(order).reshape(-1, c["kv_heads"], c["hd"])[:n]).double() for x in ("k", "v"))
            for h in range(c["kv_heads"] if n else 0):
                a = st["q"][r, h * g:(h + 1) * g].double() @ k[:, h].T.contiguous() / math.sqrt(c["hd"])
                out[r, h * g:(h + 1) * g] = torch.softmax(a, dim=-1) @ v[:, h].contiguous()
        return out
    s, d, v = c["seqs"], c["drafts"], c["vocab"]
    tokens = torch.full((s, d + 1), NO_TOKEN, dtype=torch.int32)
    accepted = torch.zeros(s, dtype=torch.int32)
    drafts, u, lengths = st["drafts"].tolist(), st["uniforms"].double().tolist(), st["n_drafts"].tolist()
    for i in range(s):
        n = 0
        while True:
            z = st["logits"][i, n].double()
            if c["softcap"] > 0:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            p = torch.softmax(z / c["temperature"], dim=-1) if c["temperature"] > 0 else (torch.arange(v, device="cuda") == z.argmax()).double()
            if n == lengths[i]:
                break
            q = (st["probs"][i, n].double() if st["probs"] is not None and c["temperature"] > 0
                 else (torch.arange(v, device="cuda") == drafts[i][n]).double())
            if not u[i][n] * float(q[drafts[i][n]]) < float(p[drafts[i][n]]):
                rest = torch.relu(p - q)
                p = rest if float(rest.sum()) > 0 else p
                break
            tokens[i, n] = drafts[i][n]
            n += 1
        if c["temperature"] > 0:
            run = torch.cumsum(p, dim=0)
            last = int(p.nonzero()[-1])
            tokens[i, n] = min(int(torch.searchsorted(run, run[-1:] * u[i][d], right=True)), last)
        else:
            tokens[i, n] = int(p.argmax()) if n == lengths[i] else int(z.argmax())
        accepted[i] = n
    return {"tokens": tokens, "accepted": accepted}
