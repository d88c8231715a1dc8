"""Speculative decoding on a block-scaled 8-bit cache: the operators, as they are called and as plain torch.

Three operators of one serving step of the 7B decoder (32 query heads over 8 kv heads of 128, vocabulary
128256; tensor-parallel shards of it have 16/4, 8/2 and 4/1 heads):

* append: rotary positions on q and k, and k and v into an fp8 e4m3 paged cache that has one power-of-two
  scale for each page and kv head;
* attention: causal attention over that cache, from one query token a sequence to a whole prompt, with an
  optional sliding window and first tokens that stay visible (sinks);
* verify: drafted tokens accepted or replaced against the target's probabilities, from given random numbers.

`own` selects the framework's kernels; otherwise `run` is elementary torch operations in 32 bits.
"""
import math
import sys

import torch

own = False

DEV = "cuda"
D = 128
THETA = 1e6
E4M3_MAX = 448.0
EXP_MIN, EXP_MAX = -64, 100      # exponents of the scales that append writes


def _framework(name):
    import importlib
    import os
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gfx1201-tuning-log_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    return importlib.import_module(name)


# ---- cases ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding sequence of the 7B model at a 4096-token context: the smallest call, where latency counts
        _attn("attend one sequence", ctx=(4095, 4095)),
        # the decode half of a busy serving step: 60 sequences at 2k..32k tokens in one call
        _attn("attend 60 ragged", seqs=60, ctx=(2048, 32767)),
        # a verification step: 8 sequences, the last token and four or five drafts each
        _attn("attend drafts", seqs=8, new=(5, 6), ctx=(3000, 4500)),
        # long chats on a model with a sliding window and four sink tokens, a 2-way tensor-parallel shard
        _attn("attend window", seqs=32, heads=16, kv_heads=4, ctx=(6001, 32001), window=4096, sinks=4),
        # four prompts of 512 to 2048 tokens in one varlen call
        _attn("attend prompts", seqs=4, new=(512, 2048), ctx=(0, 0)),
        # a chunk of a long prompt behind 14k tokens already cached, odd sizes, windowed, wide pages
        _attn("attend chunk window", seqs=2, new=(1777, 2011), ctx=(9001, 14003), block=64, window=3001, sinks=5),
        # the new tokens of eight decoding sequences
        _append("append 8 tokens", seqs=8, ctx=(100, 4000)),
        # a verification step's ragged drafts, wide pages, grouped 8 to 1
        _append("append drafts", seqs=33, new=(1, 8), ctx=(0, 3000), heads=32, kv_heads=4, block=32),
        # a serving step of 60 decodes and four 2048-token prompts (8252 tokens)
        _append("append serving step", seqs=60, ctx=(500, 3000), prompts=4, prompt=2048),
        # one sequence with four drafts
        _verify("verify one", seqs=1, drafts=(4, 4)),
        # a full batch with one to seven drafts each, every fourth sequence greedy
        _verify("verify 64", seqs=64, drafts=(1, 7), greedy_every=4),
        # drafts looked up in the prompt (no draft probabilities), bf16 logits of an odd smaller vocabulary
        _verify("verify lookup", seqs=17, drafts=(0, 5), vocab=32003, probs=False, half=True, greedy_every=3),
    ]


def _attn(name, seqs=1, new=(1, 1), ctx=(0, 0), heads=32, kv_heads=8, block=16, window=0, sinks=0):
    return {"name": name, "op": "attention", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "heads": heads, "kv_heads": kv_heads, "block": block, "window": window, "sinks": sinks,
            "prompts": 0, "prompt": 0}


def _append(name, seqs=1, new=(1, 1), ctx=(0, 0), heads=32, kv_heads=8, block=16, prompts=0, prompt=0):
    return {"name": name, "op": "append", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "heads": heads, "kv_heads": kv_heads, "block": block, "prompts": prompts,
            "prompt": prompt}


def _verify(name, seqs=1, drafts=(4, 4), vocab=128256, probs=True, half=False, greedy_every=0):
    return {"name": name, "op": "verify", "seqs": seqs, "new_lo": drafts[0] + 1, "new_hi": drafts[1] + 1,
            "vocab": vocab, "probs": probs, "half": half, "greedy_every": greedy_every, "prompts": 0, "prompt": 0}


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads, kv = rng.choice([(32, 8), (16, 4), (8, 2), (4, 1), (32, 4), (8, 1), (16, 8), (8, 8)])
    block = rng.choice([16, 16, 32, 64, 128])
    window, sinks = rng.choice([(0, 0), (0, 0), (log(64, 5000), rng.randint(0, 8))])
    what = rng.choice(["decode", "decode", "drafts", "prompts", "chunk", "append", "prompt append", "verify", "verify"])
    if what in ("decode", "drafts"):
        new = (1, 1) if what == "decode" else (1, rng.randint(2, 8))
        seqs = log(1, 64)
        hi = log(40, min(32000, 8_000_000 // (seqs * kv)))  # the largest listed call's tokens and fewer
        new = (rng.randint(0, 1), new[1])
        case = _attn("", seqs, new, (rng.randint(0, hi), hi), heads, kv, block, window, sinks)
    elif what == "prompts":
        seqs = rng.randint(1, 6)
        hi = log(20, 2048)
        case = _attn("", seqs, (rng.randint(1, hi), hi), (0, 0), heads, kv, block, window, sinks)
    elif what == "chunk":
        seqs, hi = rng.randint(1, 2), log(60, 2000)
        ctx = log(100, min(14000, 300_000_000 // (seqs * hi * heads)) + 100)
        case = _attn("", seqs, (rng.randint(33, hi), hi), (ctx // 2, ctx), heads, kv, block, window, sinks)
    elif what == "append":
        seqs, hi = log(1, 128), log(10, 3000)
        case = _append("", seqs, (rng.randint(0, 1), rng.randint(1, 8)), (rng.randint(0, hi), hi), heads, kv, block)
    elif what == "prompt append":
        hi = log(20, 1900)
        case = _append("", rng.randint(1, 60), (1, 1), (0, hi), heads, kv, block, rng.randint(1, 4), hi)
    else:
        lo = rng.randint(0, 4)
        case = _verify("", log(1, 64), (lo, lo + rng.randint(0, 3)), rng.choice([128256, 32003, log(1000, 128000)]),
                       rng.random() < 0.7, rng.random() < 0.4, rng.choice([0, 2, 5]))
    del case["name"]
    return case


def _between(lo, hi, n, step):
    """n whole numbers spread over [lo, hi], the same for every seed."""
    return [lo + int((hi - lo + 1) * ((i + 1) * step % 1.0)) if hi > lo else lo for i in range(n)]


def _lengths(c):
    """New tokens and total length (new ones included) of each sequence."""
    new = _between(c["new_lo"], c["new_hi"], c["seqs"], 0.7548776662) + [c["prompt"]] * c["prompts"]
    ctx = _between(c.get("ctx_lo", 0), c.get("ctx_hi", 0), c["seqs"], 0.6180339887) + [0] * c["prompts"]
    return new, [a + b for a, b in zip(new, ctx)]


# ---- inputs --------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"attention": _prepare_attention, "append": _prepare_append, "verify": _prepare_verify}[case["op"]](case, g)


def _index(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(case, total, g):
    """A block table of scattered pages (page 0 is nobody's) and the number of pages."""
    need = [-(-n // case["block"]) for n in total]
    perm = (torch.randperm(sum(need), device=DEV, generator=g) + 1).to(torch.int32)
    table = torch.zeros(len(total), max(need + [1]), dtype=torch.int32, device=DEV)
    rows = torch.arange(table.shape[1], device=DEV)[None, :] < torch.tensor(need, device=DEV)[:, None]
    table[rows] = perm
    return table, sum(need) + 1


def _codes(shape, g):
    """e4m3 codes of N(0, 64^2) values: pages whose scale makes them about N(0, 1)."""
    return (torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16) * 64).to(torch.float8_e4m3fn)


def _scales(nb, hkv, g):
    return torch.exp2(torch.randint(-7, -4, (nb, hkv), device=DEV, generator=g).float())


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return _index(out)


def _prepare_attention(c, g):
    new, total = _lengths(c)
    table, nb = _pages(c, total, g)
    shape = (nb, c["block"], c["kv_heads"], D)
    s = {"op": "attention", "cu": _starts(new), "lens": _index(total), "table": table, "max_new": max(new),
         "max_len": max(total), "window": c["window"], "sinks": c["sinks"], "scale": D ** -0.5,
         "q": torch.randn(sum(new), c["heads"], D, device=DEV, generator=g).to(torch.bfloat16),
         "k": _codes(shape, g), "v": _codes(shape, g), "ks": _scales(nb, c["kv_heads"], g),
         "vs": _scales(nb, c["kv_heads"], g)}
    s["out"] = torch.empty_like(s["q"])
    if own:
        s["workspace"] = _framework("block_cache").Workspace(DEV, c["seqs"], c["kv_heads"])
    return s


def _rope(positions):
    inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    ang = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv[None, :]
    return torch.cat([torch.cos(ang), torch.sin(ang)], 1).float()


def _prepare_append(c, g):
    new, total = _lengths(c)
    table, nb = _pages(c, total, g)
    shape = (nb, c["block"], c["kv_heads"], D)
    width = (c["heads"] + 2 * c["kv_heads"]) * D
    # a projection's output: its size drifts from token to token, so that pages outgrow their first scale
    size = torch.exp2(2 * torch.rand(sum(new), 1, device=DEV, generator=g) - 1)
    qkv = (torch.randn(sum(new), width, device=DEV, generator=g) * size).to(torch.bfloat16)
    return {"op": "append", "cu": _starts(new), "lens": _index(total), "table": table, "qkv": qkv,
            "rope": _rope(max(total)), "k": _codes(shape, g), "v": _codes(shape, g),
            "ks": _scales(nb, c["kv_heads"], g), "vs": _scales(nb, c["kv_heads"], g),
            "q": torch.empty(sum(new), c["heads"], D, dtype=torch.bfloat16, device=DEV)}


def _prepare_verify(c, g):
    new, _ = _lengths(c)
    rows, vocab, seqs = sum(new), c["vocab"], c["seqs"]
    logits = torch.randn(rows, vocab, device=DEV, generator=g) * 2
    favoured = torch.randint(0, vocab, (rows, 8), device=DEV, generator=g)
    logits.scatter_add_(1, favoured, 6 + 4 * torch.rand(rows, 8, device=DEV, generator=g))
    # the draft model: the target's logits, disturbed
    draft = torch.softmax(logits + 0.7 * torch.randn(rows, vocab, device=DEV, generator=g), 1)
    race = torch.empty(rows, vocab, device=DEV).exponential_(generator=g)
    picked = (draft / race).argmax(1)
    tokens = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    starts = _starts(new)
    first = torch.zeros(rows + 1, dtype=torch.bool, device=DEV)
    first[starts.long()] = True
    # row r's draft is the token fed to row r + 1
    tokens[1:] = torch.where(first[1:rows], tokens[1:], picked[:-1])
    temperature = 0.6 + 0.8 * torch.rand(seqs, device=DEV, generator=g)
    if c["greedy_every"]:
        temperature[::c["greedy_every"]] = 0
    noise = torch.empty(seqs, vocab, device=DEV).exponential_(generator=g)
    return {"op": "verify", "logits": logits.to(torch.bfloat16) if c["half"] else logits, "tokens": tokens,
            "cu": starts, "uniforms": torch.rand(rows, device=DEV, generator=g), "noise": noise.clamp_min_(1e-30),
            "temperature": temperature, "draft": draft if c["probs"] else None, "max_new": max(new)}


# ---- one pass ------------------------------------------------------------------------------------------
def run(s):
    if s["op"] == "attention":
        if own:
            return _framework("block_cache").attention(
                s["q"], s["k"], s["v"], s["ks"], s["vs"], s["out"], s["cu"], s["lens"], s["table"], s["scale"],
                max_qlen=s["max_new"], max_seq_len=s["max_len"], window=s["window"], sinks=s["sinks"],
                workspace=s["workspace"])
        return _attention(s)
    if s["op"] == "append":
        if own:
            _framework("block_cache").append(s["qkv"], s["rope"], s["k"], s["v"], s["ks"], s["vs"], s["cu"], s["lens"],
                                             s["table"], q_out=s["q"])
            return {"q": s["q"], "k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}
        return _append_plain(s)
    if own:
        out, accepted = _framework("speculative").verify(s["logits"], s["tokens"], s["cu"], s["uniforms"], s["noise"],
                                                         temperature=s["temperature"], draft_probs=s["draft"])
        return {"tokens": out, "accepted": accepted}
    return _verify_plain(s)


def _attention(s):
    """softmax(q k^T) v over the pages of each sequence, all sequences padded to the longest."""
    q, k, lens, table = s["q"], s["k"], s["lens"].long(), s["table"].long()
    heads, hkv, bs = q.shape[1], k.shape[2], k.shape[1]
    seqs, new = table.shape[0], s["max_new"]
    start = s["cu"].long()[:-1]
    count = s["cu"].long()[1:] - start
    at = torch.arange(new, device=q.device)
    real = at[None, :] < count[:, None]                                # [seqs, new]
    rows = torch.where(real, start[:, None] + at[None, :], 0)
    qs = q[rows].float().view(seqs, new, hkv, heads // hkv, D)
    keys = (k[table].float() * s["ks"][table][:, :, None, :, None]).view(seqs, -1, hkv, D)
    score = torch.einsum("bihgd,bjhd->bhgij", qs, keys) * s["scale"]
    del keys
    here = (lens - count)[:, None] + at[None, :]                       # position of each query
    j = torch.arange(table.shape[1] * bs, device=q.device)
    sees = (j <= here[..., None]) & real[..., None]
    if s["window"]:
        sees &= (j > here[..., None] - s["window"]) | (j < s["sinks"])
    sees = sees[:, None, None]                                         # [seqs, 1, 1, new, keys]
    score = score.masked_fill_(~sees, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp_(score.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    values = (s["v"][table].float() * s["vs"][table][:, :, None, :, None]).view(seqs, -1, hkv, D)
    values = torch.where(j[None, :, None, None] < lens[:, None, None, None], values, 0.0)
    o = torch.einsum("bhgij,bjhd->bihgd", p, values).reshape(seqs * new, heads, D)
    # back to the packed rows: row r is token r - start of its sequence
    r = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(s["cu"].long()[1:], r, right=True)
    return o[seq * new + r - start[seq]].to(torch.bfloat16)


def _rotate(x, cos, sin):
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _power(amax):
    """The smallest power of two s with amax <= 448 s."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(EXP_MIN, EXP_MAX)
    return torch.exp2(torch.where(amax == 0, EXP_MIN, e).float())


def _append_plain(s):
    qkv, lens, cu, table = s["qkv"].float(), s["lens"].long(), s["cu"].long(), s["table"].long()
    hkv, bs = s["k"].shape[2], s["k"].shape[1]
    tokens, heads = s["q"].shape[:2]
    r = torch.arange(tokens, device=qkv.device)
    seq = torch.searchsorted(cu[1:], r, right=True)
    pos = lens[seq] - cu[seq + 1] + r
    cos, sin = s["rope"][pos][:, None, :].split(D // 2, -1)
    x = qkv.view(tokens, heads + 2 * hkv, D)
    s["q"].copy_(_rotate(x[:, :heads], cos, sin))
    page, slot = table[seq, pos // bs], pos % bs
    # each sequence's first page may hold earlier tokens (page 0 stands in where it does not)
    count = cu[1:] - cu[:-1]
    begin = lens - count
    kept = torch.where(count > 0, begin % bs, 0)
    first = table.gather(1, (begin // bs).clamp(0, table.shape[1] - 1)[:, None])[:, 0]
    first = torch.where(kept > 0, first, 0)
    keep = torch.arange(bs, device=qkv.device)[None, :] < kept[:, None]
    for new, cache, scales in ((_rotate(x[:, heads:heads + hkv], cos, sin), s["k"], s["ks"]),
                               (x[:, heads + hkv:], s["v"], s["vs"])):
        amax = torch.zeros_like(scales).index_reduce_(0, page, new.abs().amax(-1), "amax")
        fresh = torch.zeros(scales.shape[0], dtype=torch.bool, device=qkv.device).index_fill_(0, page, True)
        held = torch.zeros_like(fresh).index_fill_(0, first, True)
        held[0] = fresh[0] = False
        old = scales.clone()
        grown = torch.where(held[:, None], torch.maximum(old, _power(amax)), _power(amax))
        scales.copy_(torch.where(fresh[:, None], grown, old))
        ratio = (old / scales)[first][:, None, :, None]
        was = cache[first]
        again = (was.float() * ratio).to(torch.float8_e4m3fn)
        mixed = torch.where(keep[:, :, None, None], again.view(torch.uint8), was.view(torch.uint8))
        cache.view(torch.uint8)[first] = mixed
        codes = (new / scales[page][..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        cache.view(torch.uint8)[page, slot] = codes.view(torch.uint8)
    return {"q": s["q"], "k": s["k"], "v": s["v"], "ks": s["ks"], "vs": s["vs"]}


def _verify_plain(s):
    logits, cu = s["logits"].float(), s["cu"].long()
    rows, vocab = logits.shape
    r = torch.arange(rows, device=logits.device)
    seq = torch.searchsorted(cu[1:], r, right=True)
    last = r == cu[seq + 1] - 1
    heat = s["temperature"][seq][:, None]
    top, best = logits.max(1, keepdim=True)
    p = torch.exp((logits - top) / torch.where(heat > 0, heat, 1.0))
    p = p / p.sum(1, keepdim=True)
    ids = torch.arange(vocab, device=logits.device)
    p = torch.where(heat > 0, p, (ids == best).float())
    draft = torch.where(last, 0, torch.roll(s["tokens"], -1))[:, None]
    q = s["draft"] if s["draft"] is not None else (ids == draft).float()
    yes = (s["uniforms"] * q.gather(1, draft)[:, 0] < p.gather(1, draft)[:, 0]) & ~last
    # the first row of each sequence whose draft is not taken (its last row at the latest)
    stop = torch.full((len(cu) - 1,), rows, device=logits.device)
    stop = stop.scatter_reduce_(0, seq, torch.where(yes, rows, r), "amin")
    left = torch.where(last[stop][:, None], p[stop], (p[stop] - q[stop]).clamp_min(0))
    left = torch.where(left.amax(1, keepdim=True) > 0, left, p[stop])
    token = (left / s["noise"]).argmax(1)
    out = torch.where(r < stop[seq], draft[:, 0], torch.where(r == stop[seq], token[seq], -1))
    return {"tokens": out, "accepted": (stop - cu[:-1]).to(torch.int32)}


# ---- what a pass cannot do without ------------------------------------------------------------------------
def _visible(n, total, window, sinks):
    """Keys that any query of a sequence sees, and (query, key) pairs."""
    begin = total - n
    if not window:
        return total, n * begin + n * (n + 1) // 2
    low = max(0, begin - window + 1)
    keys = total - low + min(sinks, low)
    pairs = sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(begin, total))
    return keys, pairs


def work(c):
    new, total = _lengths(c)
    tokens = sum(new)
    if c["op"] == "attention":
        seen = [_visible(n, t, c["window"], c["sinks"]) for n, t in zip(new, total)]
        keys, pairs = sum(k for k, _ in seen), sum(p for _, p in seen)
        pages = sum(-(-k // c["block"]) for k, _ in seen)
        return {"bytes": keys * 2 * c["kv_heads"] * D + pages * (2 * c["kv_heads"] * 4 + 4) + 2 * tokens * c["heads"] * D * 2,
                "flops": 4 * D * c["heads"] * pairs}
    if c["op"] == "append":
        width = c["heads"] + 2 * c["kv_heads"]
        bs, hkv = c["block"], c["kv_heads"]
        kept = sum((t - n) % bs for n, t in zip(new, total) if n)
        pages = sum(-(-t // bs) - (t - n) // bs for n, t in zip(new, total) if n)
        return {"bytes": tokens * D * (2 * width + 2 * c["heads"] + 2 * hkv) + tokens * 4 * D  # qkv in, q and codes out, angles
                + kept * 2 * hkv * D + pages * 2 * hkv * 8,
                "flops": tokens * D * (3 * (c["heads"] + hkv) + 4 * hkv)}
    size = 2 if c["half"] else 4
    return {"bytes": tokens * c["vocab"] * size + c["seqs"] * c["vocab"] * (8 if c["probs"] else 4),
            "flops": 4 * tokens * c["vocab"]}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "append":
        return _exact_append(s)
    return None


def _exact_attention(s):
    cu, lens, group = s["cu"].tolist(), s["lens"].tolist(), s["q"].shape[1] // s["k"].shape[2]
    bs = s["k"].shape[1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, total in enumerate(lens):
        lo, hi = cu[b], cu[b + 1]
        if hi == lo or total == 0:
            continue
        pages = s["table"][b, :-(-total // bs)].long()
        for h in range(s["k"].shape[2]):
            kd = (s["k"][pages][:, :, h].double() * s["ks"][pages, h].double()[:, None, None]).reshape(-1, D)[:total]
            vd = (s["v"][pages][:, :, h].double() * s["vs"][pages, h].double()[:, None, None]).reshape(-1, D)[:total]
            pos = torch.arange(total - (hi - lo), total, device=DEV)[:, None]
            key = torch.arange(total, device=DEV)[None, :]
            hidden = key > pos
            if s["window"]:
                hidden |= (key <= pos - s["window"]) & (key >= s["sinks"])
            for h1 in range(h * group, (h + 1) * group):
                x = s["q"][lo:hi, h1].double() @ kd.T * s["scale"]
                w = torch.softmax(x.masked_fill_(hidden, -math.inf), 1)
                out[lo:hi, h1] = w @ vd
    return out


def _e4m3(x):
    """The nearest e4m3 value, ties to even."""
    e = torch.frexp(x)[1].double() - 1
    step = torch.exp2(e.clamp_min(-6) - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append(s):
    hkv, bs, heads = s["k"].shape[2], s["k"].shape[1], s["q"].shape[1]
    cu, lens, table = s["cu"].tolist(), s["lens"].tolist(), s["table"].tolist()
    x = s["qkv"].double().view(-1, heads + 2 * hkv, D)
    pos = torch.cat([torch.arange(n - (b - a), n, device=DEV) for a, b, n in zip(cu, cu[1:], lens)])
    turn = torch.complex(s["rope"][pos, :D // 2].double(), s["rope"][pos, D // 2:].double())[:, None]
    z = torch.complex(x[:, :heads + hkv, :D // 2], x[:, :heads + hkv, D // 2:]) * turn
    qk = torch.cat([z.real, z.imag], -1)
    result = {"q": qk[:, :heads]}
    for name, rows, cache, scales in (("k", qk[:, heads:], s["k"].double(), s["ks"].double()),
                                      ("v", x[:, heads + hkv:], s["v"].double(), s["vs"].double())):
        where, what, held = [], [], []
        for b, total in enumerate(lens):
            begin, at = total - (cu[b + 1] - cu[b]), cu[b]
            while begin < total:
                end = min(total, (begin // bs + 1) * bs)
                where.append(table[b][begin // bs])
                what.append((at, at + end - begin, begin % bs))
                at, begin = at + end - begin, end
        sizes = rows.abs().amax(-1)
        tops = torch.stack([sizes[a:b].amax(0) for a, b, _ in what])
        m, e = torch.frexp(tops)
        grown = torch.exp2(torch.where(m <= 0.875, e - 9, e - 8).clamp(EXP_MIN, EXP_MAX).double())
        where = torch.tensor(where, device=DEV)
        held = torch.tensor([k for _, _, k in what], device=DEV)
        before = scales[where]
        after = torch.where(held[:, None] > 0, torch.maximum(before, grown), grown)
        scales[where] = after
        inside = torch.arange(bs, device=DEV)[None, :] < held[:, None]
        cache[where] = torch.where(inside[:, :, None, None], _e4m3(cache[where] * (before / after)[:, None, :, None]),
                                   cache[where])
        of = torch.cat([torch.full((b - a,), i, device=DEV) for i, (a, b, _) in enumerate(what)])
        slot = torch.cat([torch.arange(k, k + b - a, device=DEV) for a, b, k in what])
        cache[where[of], slot] = _e4m3(rows / after[of][..., None])
        result[name] = cache
        result[name + "s"] = scales
    return result
