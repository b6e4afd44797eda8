"""Timed cases of the serving operators: the 8-bit paged key/value cache (write, read back, attention) and
token log-probabilities, each with a plain torch form and its values in 64 bits.

    cache      new rows of K and V are quantised into their pages and read back as floats
    attention  the queries of new rows over their sequences' cached keys, for single tokens and for prompts
    score      log-probabilities of given tokens, entropy and the top alternatives; `train`: the gradient too

A cache holds codes c (8 bits, -127..127) and one power-of-two scale for each page (a block of `page` tokens)
and head; a stored value is c * scale.
"""

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
HEAD_DIMS = (16, 32, 64, 80, 96, 128)
PAGES = (16, 32, 64, 128)


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one generated token for each of 64 running sequences of a d_model 512 model
        {"name": "append-token", "op": "cache", "dtype": "bfloat16", "batch": 64, "kv_heads": 8, "head_dim": 64,
         "page": 16, "before": 1000, "new": 1},
        # prompts of unequal lengths that continue half-filled pages, odd head width
        {"name": "store-prompts", "op": "cache", "dtype": "bfloat16", "batch": 16, "kv_heads": 8, "head_dim": 96,
         "page": 64, "before": 77, "new": 2011},
        # reading whole sequences back, as before a full-precision recomputation
        {"name": "restore", "op": "cache", "dtype": "float32", "batch": 8, "kv_heads": 8, "head_dim": 64,
         "page": 32, "before": 4096, "new": 0},
        # the smallest call: one token of one sequence, 4 heads of 64, context 256
        {"name": "token-short", "op": "attention", "dtype": "float32", "batch": 1, "q_heads": 4, "kv_heads": 4,
         "head_dim": 64, "page": 16, "length": 256, "new": 1, "left": False},
        # one token for each of 64 sequences, 8 heads of 64, up to context 1024, left padding and an empty row
        {"name": "token-batch", "op": "attention", "dtype": "float32", "batch": 64, "q_heads": 8, "kv_heads": 8,
         "head_dim": 64, "page": 32, "length": 1024, "new": 1, "left": True},
        # few long sequences with shared key heads: the cache is the whole cost
        {"name": "token-long", "op": "attention", "dtype": "bfloat16", "batch": 4, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "length": 131071, "new": 1, "left": False},
        # 32 prompts of a full context, 8 heads of 64, context 1024, single precision
        {"name": "prompt", "op": "attention", "dtype": "float32", "batch": 32, "q_heads": 8, "kv_heads": 8,
         "head_dim": 64, "page": 32, "length": 1024, "new": 1024, "left": False},
        # a second part of two long prompts, behind what the cache holds already; lengths that end inside a page
        {"name": "prompt-continued", "op": "attention", "dtype": "bfloat16", "batch": 2, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "length": 8189, "new": 2043, "left": True},
        # the answers of a full batch of modular equations (4656 rows, 97 residues)
        {"name": "score-answers", "op": "score", "dtype": "float32", "rows": 4656, "vocab": 97, "top": 5,
         "masked": False, "train": False},
        # the next token of 8 sequences over a large vocabulary, part of it masked out
        {"name": "score-token", "op": "score", "dtype": "bfloat16", "rows": 8, "vocab": 131071, "top": 20,
         "masked": True, "train": False},
        # a training batch of 32 sequences of 1024 characters, vocabulary 64
        {"name": "train-characters", "op": "score", "dtype": "float32", "rows": 32768, "vocab": 64, "top": 0,
         "masked": False, "train": True},
        # a training batch over a large odd vocabulary
        {"name": "train-wide", "op": "score", "dtype": "bfloat16", "rows": 4096, "vocab": 32003, "top": 1,
         "masked": False, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("cache", "attention", "attention", "score"))
    dtype = rng.choice(tuple(DTYPES))
    if op == "score":
        rows, vocab = _log(rng, 1, 32768), _log(rng, 2, 131072)
        while rows * vocab > 4096 * 32003:
            rows, vocab = max(1, rows // 2), max(2, vocab * 3 // 4)
        return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "top": min(vocab, rng.choice((0, 1, 5, 20, 32))),
                "masked": rng.random() < 0.5, "train": rng.random() < 0.4}
    kv_heads, head_dim, page = rng.choice((1, 2, 3, 4, 8, 16)), rng.choice(HEAD_DIMS), rng.choice(PAGES)
    batch = _log(rng, 1, 128)
    if op == "cache":
        before, new = rng.choice((0, _log(rng, 1, 8192))), rng.choice((1, _log(rng, 2, 4096)))
        if before and rng.random() < 0.25:
            new = 0
        while (batch * (new if new else before) * kv_heads * head_dim > 16 * 2011 * 8 * 96
               or batch * (before + new) * kv_heads * head_dim > 4 * 8 * 131071 * 128):
            batch, before, new = max(1, batch // 2), before * 3 // 4, (max(1, new * 3 // 4) if new else 0)
        return {"op": op, "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
                "before": before, "new": new}
    group = rng.choice((1, 1, 2, 4, 8))
    new = rng.choice((1, 1, _log(rng, 2, 4096)))
    length = new + rng.choice((0, _log(rng, 1, 131072)))
    while (batch * kv_heads * length * head_dim > 4 * 8 * 131071 * 128
           or batch * kv_heads * group * new * length > 2 * 32 * 2043 * 8189):
        batch, length = max(1, batch // 2), max(1, length * 3 // 4)
        new = min(new, length)
    return {"op": op, "dtype": dtype, "batch": batch, "q_heads": kv_heads * group, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "length": length, "new": new, "left": rng.random() < 0.3}


def _sizes(case):
    """Per sequence: tokens in the cache with the new ones, new tokens, and the first visible position.  Sequences
    are of unequal lengths, the first of the longest; in prompts one of many may bring nothing new."""
    batch, new = case["batch"], case["new"]
    longest = case["before"] + new if case["op"] == "cache" else case["length"]
    lengths, news, firsts = [], [], []
    for b in range(batch):
        n = new
        if b and new > 1:
            n = 0 if b % 11 == 5 else new - b * 7919 % (new // 2 + 1)
        old = longest - new
        old -= b * 6007 % (old // 2 + 1) if b else 0
        lengths.append(old + n)
        news.append(n)
        first = 0
        if case.get("left"):
            first = lengths[b] if b % 16 == 7 else lengths[b] // 4 if b % 2 else 0
        firsts.append(first)
    return lengths, news, firsts


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] == "score":
        n, r = case["rows"] * case["vocab"], case["rows"]
        out = r * (3 * 4 + 8 * case["top"] + 4)
        if case["train"]:
            return {"bytes": 2 * n * size + out + 8 * r, "flops": 12 * n}
        return {"bytes": n * size + out, "flops": 5 * n}
    lengths, news, firsts = _sizes(case)
    heads, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "cache":
        new = 2 * sum(news) * heads * hd
        read = sum(n - f for n, f in zip(lengths, _read_from(case, lengths, news)))
        read = 2 * read * heads * hd
        return {"bytes": new * size + read * (1 + size) + new, "flops": 4 * new + 2 * read}
    seen = pairs = 0
    for n, m, f in zip(lengths, news, firsts):
        seen += max(0, n - f) if m else 0
        pairs += sum(max(0, n - m + i + 1 - f) for i in range(m))
    cache = 2 * seen * heads * (hd + 4 / page)
    return {"bytes": cache + sum(news) * case["q_heads"] * (2 * hd * size + 4),
            "flops": 4 * pairs * case["q_heads"] * hd}


# ------------------------------------------------------------------ inputs
def _read_from(case, lengths, news):
    """Where the cache case reads from: the start of the page that the first new token falls in, or everything."""
    page = case["page"]
    return [(n - m) // page * page if case["new"] else 0 for n, m in zip(lengths, news)]


def _padded(head_dim):
    return -(-head_dim // 32) * 32


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, dtype = "cuda", DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["op"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        logits = (normal(rows, vocab) * 3).to(dtype)
        tokens = torch.randint(0, vocab, (rows,), generator=g, device=dev, dtype=torch.int32)
        if case["masked"]:  # a grammar's mask; one row of many has no token left
            logits.masked_fill_(torch.rand(rows, vocab, generator=g, device=dev) < 0.3, float("-inf"))
            if rows > 4:
                logits[3].fill_(float("-inf"))
        if case["train"]:  # rows whose token is not supervised
            tokens[torch.rand(rows, generator=g, device=dev) < 0.1] = -1
        return {"case": case, "logits": logits, "tokens": tokens, "top": case["top"],
                "dlogprob": normal(rows), "dentropy": normal(rows) * 0.1}

    lengths, news, firsts = _sizes(case)
    batch, heads, hd, page = case["batch"], case["kv_heads"], case["head_dim"], case["page"]
    per = [-(-n // page) for n in lengths]
    used, wide = sum(per), max(1, max(per))
    order = torch.randperm(used + 2, generator=g, device=dev).to(torch.int32).cpu()
    order = order[order != used + 1]  # the pool's last page stays free
    table = torch.full((batch, wide), -1, dtype=torch.int32)  # entries past a sequence's pages name no page
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    pool = (used + 2, heads, page, _padded(hd))
    kv = []
    for _ in range(2):
        codes = (torch.randn(pool, generator=g, device=dev, dtype=torch.float16) * 31).round_().clamp_(-127, 127)
        codes[..., hd:] = 0
        kv.append(codes.to(torch.int8))
        scale = _power(torch.randint(-6, -3, pool[:2], generator=g, device=dev))
        free = torch.ones(used + 2, dtype=torch.bool)
        free[order[:used].long()] = False
        scale[free.to(dev)] = float("nan")  # pages that nothing has been written to
        kv.append(scale)
    offsets = [0]
    for n in news:
        offsets.append(offsets[-1] + n)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    state = {"case": case, "k": kv[0], "k_scale": kv[1], "v": kv[2], "v_scale": kv[3], "table": table.to(dev),
             "lengths": ints(lengths), "offsets": ints(offsets), "most": max(max(lengths), 1),
             "new": max(max(news), 0)}
    rows = offsets[-1]
    if case["op"] == "cache":
        gain = torch.exp2(torch.rand(1, heads, hd, generator=g, device=dev) * 4 - 2)  # channels of unequal size
        state["k_rows"] = (normal(rows, heads, hd) * gain).to(dtype)
        state["v_rows"] = normal(rows, heads, hd).to(dtype)
        state["from"] = ints(_read_from(case, lengths, news))
        state["tokens"] = max(max(n - f for n, f in zip(lengths, _read_from(case, lengths, news))), 1)
        state["spare"] = used + 1
    else:  # unit-RMS rows as QK normalisation leaves them, some heads sharper than others
        q = normal(rows, case["q_heads"], hd)
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-5)
        q = q * torch.exp2(torch.rand(1, case["q_heads"], 1, generator=g, device=dev) * 2)
        state["q"] = q.to(dtype)
        state["first"] = ints(firsts) if case["left"] else None
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["op"] == "cache":
        return _cache_own(state) if own else _cache_plain(state)
    if case["op"] == "attention":
        return _attention_own(state) if own else _attention_plain(state)
    return _score_own(state) if own else _score_plain(state)


def _own_cache(state):
    from grokking_abmod_b200 import ops
    return ops, ops.KvCache(state["k"], state["v"], state["k_scale"], state["v_scale"])


def _cache_own(state):
    ops, cache = _own_cache(state)
    if state["new"]:
        ops.cache_write(cache, state["k_rows"], state["v_rows"], state["table"], state["lengths"], state["offsets"],
                        max_new=state["new"])
    case = state["case"]
    return ops.cache_read(cache, state["table"], state["lengths"], state["tokens"], first=state["from"],
                          head_dim=case["head_dim"], dtype=DTYPES[case["dtype"]])


def _attention_own(state):
    ops, cache = _own_cache(state)
    return ops.cache_attention(state["q"], cache, state["table"], state["lengths"], state["offsets"],
                               first=state["first"], max_tokens=state["most"], max_new=state["new"])


def _score_own(state):
    from grokking_abmod_b200 import ops
    r = ops.token_logprobs(state["logits"], state["tokens"], state["top"])
    if not state["case"]["train"]:
        return r
    d = ops.token_logprobs_backward(state["logits"], state["tokens"], r.lse, r.entropy, state["dlogprob"],
                                    state["dentropy"])
    return (*r, d)


def _power(e):
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


# The smallest power of two s with amax <= 127 s, no smaller than 2^-126.
def _scale_of(amax):
    m, e = torch.frexp(amax)  # amax = m 2^e, 0.5 <= m < 1; 127 2^(e-7) = 0.9921875 2^e
    e = torch.where(m > 0.9921875, e - 6, e - 7).clamp(min=-126)
    return torch.where(amax > 0, _power(e), 2.0 ** -126)


def _cache_plain(state):
    case = state["case"]
    page, hd = case["page"], case["head_dim"]
    lengths, table = state["lengths"].long(), state["table"].long()
    dev = table.device
    if state["new"]:
        offsets = state["offsets"].long()
        old = lengths - (offsets[1:] - offsets[:-1])  # tokens before the new ones
        count = -(-state["new"] // page) + 1  # pages that new rows can fall in
        index = (old // page)[:, None] + torch.arange(count, device=dev)
        pos = (index * page)[..., None] + torch.arange(page, device=dev)  # [batch][count][page]
        fresh = (pos >= old[:, None, None]) & (pos < lengths[:, None, None])
        kept = pos < old[:, None, None]
        row = (offsets[:-1, None, None] + pos - old[:, None, None]).clamp(0, max(0, state["k_rows"].shape[0] - 1))
        pages = table.gather(1, index.clamp(max=table.shape[1] - 1))
        touched = fresh.any(-1)
        pages = torch.where(touched, pages, state["spare"])
        for rows, codes, scales in ((state["k_rows"], state["k"], state["k_scale"]),
                                    (state["v_rows"], state["v"], state["v_scale"])):
            x = rows[row].float().transpose(2, 3)  # [batch][count][heads][page][hd]
            new_slot, old_slot = fresh[:, :, None, :, None], kept[:, :, None, :, None]
            scale = _scale_of(torch.where(new_slot, x.abs(), 0).amax((-2, -1)))
            before = scales[pages]
            scale = torch.where(kept.any(-1)[..., None], torch.maximum(before, scale), scale)
            was = codes[pages]
            wide, ratio = scale[..., None, None], (before / scale)[..., None, None]
            out = torch.where(old_slot, (was.float() * ratio).round(), was.float())
            out[..., :hd] = torch.where(new_slot, (x / wide).round(), out[..., :hd])
            out = torch.where(touched[:, :, None, None, None], out, was.float())
            codes[pages] = out.to(torch.int8)
            scales[pages] = torch.where(touched[..., None], scale, before)
    pos = state["from"].long()[:, None] + torch.arange(state["tokens"], device=dev)
    there = pos < lengths[:, None]
    pages = table.gather(1, (pos // page).clamp(max=table.shape[1] - 1)).clamp(min=0)
    out = []
    for codes, scales in ((state["k"], state["k_scale"]), (state["v"], state["v_scale"])):
        x = codes[pages, :, pos % page][..., :hd].float() * scales[pages][..., None]
        out.append(torch.where(there[..., None, None], x, 0).to(DTYPES[case["dtype"]]))
    return tuple(out)


def _attention_plain(state):
    case = state["case"]
    heads, hd, page, group = case["kv_heads"], case["head_dim"], case["page"], case["q_heads"] // case["kv_heads"]
    batch, new, q = case["batch"], state["new"], state["q"]
    lengths, offsets = state["lengths"].long(), state["offsets"].long()
    dev = q.device
    pages = state["table"].long().clamp(min=0)
    pos = torch.arange(pages.shape[1] * page, device=dev)
    held = pos < lengths[:, None]

    def values(codes, scales):
        x = codes[pages][..., :hd].float() * scales[pages][..., None, None]
        x = x.transpose(1, 2).reshape(batch, heads, -1, hd)
        return torch.where(held[:, None, :, None], x, 0)

    news = offsets[1:] - offsets[:-1]
    i = torch.arange(new, device=dev)
    row = (offsets[:-1, None] + i).clamp(max=max(0, q.shape[0] - 1))
    x = q[row].float().reshape(batch, new, heads, group, hd).permute(0, 2, 3, 1, 4).reshape(batch, heads, -1, hd)
    x = x * (1.0 / math.sqrt(hd))
    s = x @ values(state["k"], state["k_scale"]).transpose(2, 3)
    at = (lengths - news)[:, None] + i  # each new row's own position
    seen = held[:, None, :] & (pos <= at[..., None])
    if state["first"] is not None:
        seen = seen & (pos >= state["first"].long()[:, None, None])
    s = s.view(batch, heads, group, new, -1)
    s = torch.where(seen[:, None, None], s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0, m)
    s = torch.exp(s - m)
    total = s.sum(-1, keepdim=True)
    o = s.view(batch, heads, group * new, -1) @ values(state["v"], state["v_scale"])
    o = o.view(batch, heads, group, new, hd) / torch.where(total == 0, 1, total)
    lse = ((m + torch.log(total)) * math.log2(math.e)).squeeze(-1)
    # back to packed rows
    r = torch.arange(q.shape[0], device=dev)
    b = torch.bucketize(r, offsets, right=True) - 1
    i = r - offsets[b]
    out = o.permute(0, 3, 1, 2, 4)[b, i].reshape(-1, case["q_heads"], hd).to(q.dtype)
    return out, lse.permute(0, 3, 1, 2)[b, i].reshape(-1, case["q_heads"]).t().contiguous()


def _score_plain(state):
    logits, tokens, top = state["logits"], state["tokens"].long(), state["top"]
    x = logits.float()
    m = x.amax(1, keepdim=True)
    m = torch.where(m == float("-inf"), 0, m)
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    empty, ignored = (s == 0).squeeze(1), tokens < 0
    log_s = torch.log(s)
    lse = (m + log_s).squeeze(1)
    entropy = (log_s + torch.where(e > 0, e * (m - x), 0).sum(1, keepdim=True) / s).squeeze(1)
    entropy = torch.where(empty, 0, entropy)
    logprob = x.gather(1, tokens.clamp(min=0)[:, None]).squeeze(1) - lse
    logprob = torch.where(empty, float("-inf"), logprob)
    logprob = torch.where(ignored, 0, logprob)
    # ties go to the lowest index: order-preserving bits of the value above the complemented index
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = bits * 2 ** 32 + (2 ** 32 - 1 - torch.arange(x.shape[1], device=x.device))
    index = 2 ** 32 - 1 - (torch.topk(key, top, dim=1).values & 0xFFFFFFFF)
    best = x.gather(1, index)
    best = torch.where(best == float("-inf"), best, best - lse[:, None])
    out = (logprob, entropy, lse, best, index.int())
    if not state["case"]["train"]:
        return out
    p = torch.where(empty[:, None], 0, torch.exp(x - torch.where(empty, 0, lse)[:, None]))
    dl = torch.where(ignored | empty, 0, state["dlogprob"])[:, None]
    hit = torch.arange(x.shape[1], device=x.device) == tokens[:, None]
    log_p = torch.where(p > 0, x - lse[:, None], 0)
    d = dl * (hit.float() - p) - state["dentropy"][:, None] * p * (log_p + entropy[:, None])
    return (*out, d.to(logits.dtype))


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "score":
        return _exact_score(state)
    if case["op"] == "cache":
        return _exact_cache(state)
    return _exact_attention(state)


def _exact_score(state):
    x = state["logits"].double()
    tokens = state["tokens"].long()
    lse = torch.logsumexp(x, 1)
    logp = torch.log_softmax(x, 1)
    empty = lse == float("-inf")
    p = torch.exp(logp)
    p[empty] = 0
    plogp = torch.where(p > 0, p * logp, 0)
    entropy = -plogp.sum(1)
    logprob = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    logprob[empty] = float("-inf")
    logprob[tokens < 0] = 0
    best, index = torch.sort(x, dim=1, descending=True, stable=True)
    best, index = best[:, :state["top"]], index[:, :state["top"]].int()
    best = torch.where(best == float("-inf"), best, best - lse[:, None])
    out = (logprob, entropy, lse, best, index)
    if not state["case"]["train"]:
        return out
    dl = state["dlogprob"].double() * ((tokens >= 0) & ~empty)
    d = -p * dl[:, None]
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], dl[:, None])
    d -= state["dentropy"].double()[:, None] * (plogp + p * entropy[:, None])
    return (*out, d)


def _power_at_least(a):
    m, e = math.frexp(a)  # a = m 2^e, 0.5 <= m < 1 or a = 0
    return math.ldexp(1.0, e - 1 if m == 0.5 else e) if a else 0.0


def _exact_cache(state):
    case = state["case"]
    page, hd, heads = case["page"], case["head_dim"], case["kv_heads"]
    lengths, offsets, start = state["lengths"].tolist(), state["offsets"].tolist(), state["from"].tolist()
    table = state["table"].tolist()
    out = []
    for name in ("k", "v"):
        codes, scales, rows = state[name].double(), state[name + "_scale"].double(), state[name + "_rows"].double()
        got = torch.zeros(case["batch"], state["tokens"], heads, hd, dtype=torch.float64, device=codes.device)
        for b, n in enumerate(lengths):
            old = n - (offsets[b + 1] - offsets[b])
            for j in range(start[b] // page, -(-n // page)):
                lo, hi = j * page, min(n, (j + 1) * page)
                c, s = codes[table[b][j]], scales[table[b][j]][:, None, None]
                value = c[:, :hi - lo, :hd] * s
                if hi > old:
                    begin = max(lo, old)
                    x = rows[offsets[b] + begin - old:offsets[b] + hi - old].transpose(0, 1)
                    need = [max(_power_at_least(a / 127), 2.0 ** -126) for a in x.abs().amax((1, 2)).tolist()]
                    need = torch.tensor(need, dtype=torch.float64, device=x.device)[:, None, None]
                    need = torch.maximum(need, s) if begin > lo else need
                    value = torch.cat((torch.round(value[:, :begin - lo] / need), torch.round(x / need)), 1) * need
                got[b, lo - start[b]:hi - start[b]] = value.transpose(0, 1)
        out.append(got)
    return tuple(out)


def _exact_attention(state):
    case = state["case"]
    hd, heads, group = case["head_dim"], case["kv_heads"], case["q_heads"] // case["kv_heads"]
    lengths, offsets, table = state["lengths"].tolist(), state["offsets"].tolist(), state["table"].long()
    first = state["first"].tolist() if state["first"] is not None else [0] * len(lengths)
    q = state["q"].double()
    out = torch.zeros_like(q)
    lse = torch.full((case["q_heads"], q.shape[0]), float("-inf"), dtype=torch.float64, device=q.device)
    for b, n in enumerate(lengths):
        lo, hi = offsets[b], offsets[b + 1]
        if hi == lo or first[b] >= n:
            continue
        pages = table[b, :-(-n // case["page"])]
        pos = torch.arange(n, device=q.device)
        at = torch.arange(n - (hi - lo), n, device=q.device)
        seen = ((pos[None] <= at[:, None]) & (pos[None] >= first[b])).repeat(group, 1)
        some = seen.any(1)
        for h in range(heads):
            k, v = ((state[c][pages, h].double() * state[c + "_scale"][pages, h].double()[:, None, None])
                    .reshape(-1, state[c].shape[-1])[:n, :hd] for c in ("k", "v"))
            x = q[lo:hi, h * group:(h + 1) * group].transpose(0, 1).reshape(-1, hd)
            s = (x @ k.t()) / math.sqrt(hd)
            s.masked_fill_(~seen, float("-inf"))
            total = torch.logsumexp(s, 1)
            w = torch.exp(s - torch.where(some, total, 0)[:, None])
            o = (w @ v).view(group, hi - lo, hd).transpose(0, 1)
            out[lo:hi, h * group:(h + 1) * group] = o
            lse[h * group:(h + 1) * group, lo:hi] = total.view(group, hi - lo) * math.log2(math.e)
    return out, lse
