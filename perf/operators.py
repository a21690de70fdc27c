"""The serving operators and the cases they are measured on: queries and keys normalised, rotated and stored into a paged
key/value cache (qk_rope), attention of chunks of new tokens over that cache (attention), and the choice of a token from
the logits (sample).

`run` computes a case in plain torch operations, or, with `own` set, through clutor_b200.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NORM_NONE, NORM_ROW, NORM_HEAD = 0, 1, 2
EPS = 1e-6


# ---- cases -----------------------------------------------------------------------------------------------------------------

def _qk(name, n_seq, q_max, kv_max, heads, kv_heads, hd, norm, pairs, page, src, cache, lens=1):
    return {"name": name, "op": "qk", "n_seq": n_seq, "q_max": q_max, "kv_max": kv_max, "heads": heads, "kv_heads": kv_heads,
            "hd": hd, "norm": norm, "pairs": pairs, "page": page, "src": src, "cache": cache, "lens": lens}


def _attn(name, n_seq, q_max, kv_max, heads, kv_heads, hd, page, cache, window=0, sinks=0, lens=1):
    return {"name": name, "op": "attn", "n_seq": n_seq, "q_max": q_max, "kv_max": kv_max, "heads": heads,
            "kv_heads": kv_heads, "hd": hd, "page": page, "cache": cache, "window": window, "sinks": sinks, "lens": lens}


def _sample(name, rows, vocab, mode, src="f32"):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "mode": mode, "src": src}


def listed():
    return [
        # one sequence decoding: the smallest call, one per layer of every token
        _qk("qk one token", 1, 1, 500, 32, 4, 128, NORM_HEAD, False, 64, "f32", "f16"),
        # 64 sequences decoding together, the norm over the whole row (olmoe)
        _qk("qk 64 sequences", 64, 1, 4000, 16, 16, 128, NORM_ROW, False, 16, "f32", "bf16"),
        # a ragged batch of prompt chunks at the widest attention of the configurations, half-precision projections
        _qk("qk prompts", 5, 2048, 5000, 64, 4, 128, NORM_HEAD, False, 64, "bf16", "bf16"),
        # one short sequence decoding: latency
        _attn("attn one token", 1, 1, 500, 32, 4, 128, 64, "f16"),
        # continuous batching: 64 sequences of very different lengths, one new token each
        _attn("attn 64 sequences", 64, 1, 8000, 32, 4, 128, 64, "bf16"),
        # one sequence with a long cache: the work has to be split over the length
        _attn("attn long cache", 1, 1, 100000, 64, 4, 128, 128, "f16"),
        # chunks behind cached prefixes under a sliding window with sinks, small heads
        _attn("attn window chunks", 6, 700, 9001, 32, 8, 64, 32, "bf16", window=1024, sinks=4),
        # a whole prompt at once: the largest product
        _attn("attn prompt", 1, 8192, 8192, 32, 4, 128, 64, "bf16"),
        # one row with every filter, the full vocabulary
        _sample("sample one row", 1, 151936, "mixed"),
        # a batch in which every request has its own settings
        _sample("sample 64 requests", 64, 151936, "mixed"),
        # a large batch from the whole distribution cut by top-p alone, a smaller vocabulary
        _sample("sample nucleus", 256, 50304, "nucleus"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk", "attn", "sample"])
    if op == "sample":
        vocab = _log(rng, 500, 200000)
        return _strip(_sample("", max(1, min(_log(rng, 1, 300), 30_000_000 // vocab)), vocab,
                              rng.choice(["mixed", "nucleus", "plain", "topk"]), rng.choice(["f32", "f32", "bf16", "f16"])))
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 16) if g * kv_heads <= 64])
    hd, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 48, 64, 128, 256])
    cache = rng.choice(["f16", "bf16"])
    if op == "qk":
        kv_max = _log(rng, 8, 20000)
        n_seq = _log(rng, 1, 128)
        q_max = min(kv_max, _log(rng, 1, max(1, 60_000_000 // (n_seq * (heads + 2 * kv_heads) * hd))))
        n_seq = max(1, min(n_seq, 300_000_000 // (kv_max * kv_heads * hd)))
        return _strip(_qk("", n_seq, q_max, kv_max, heads, kv_heads, hd, rng.choice([NORM_NONE, NORM_ROW, NORM_HEAD, NORM_HEAD]),
                          rng.random() < 0.3, page, rng.choice(["f32", "f32", cache]), cache, rng.randrange(1 << 20)))
    while True:
        n_seq, kv_max = _log(rng, 1, 128), _log(rng, 1, 60000)
        q_max = 1 if rng.random() < 0.4 else min(kv_max, _log(rng, 1, 4000))
        # the plain form's padded scores and gathered cache, and the product, stay below the largest listed case's
        if n_seq * kv_max * kv_heads * hd <= 150_000_000 and n_seq * heads * q_max * kv_max <= 1_000_000_000:
            break
    window, sinks = 0, 0
    if rng.random() < 0.35:
        window, sinks = _log(rng, 1, 4096), rng.choice([0, 0, 1, 4, 130])
    return _strip(_attn("", n_seq, q_max, kv_max, heads, kv_heads, hd, page, cache, window, sinks, rng.randrange(1 << 20)))


def _strip(case):
    del case["name"]
    return case


def _lengths(case):
    """The sequences' lengths, new tokens included, and how many of them are new: the first sequence the longest."""
    rng = random.Random(case["lens"])
    kv, q = [case["kv_max"]], [min(case["q_max"], case["kv_max"])]
    for _ in range(case["n_seq"] - 1):
        kv.append(rng.randint(max(1, case["kv_max"] // 8), case["kv_max"]))
        q.append(min(kv[-1], rng.randint(1, case["q_max"])))
    return kv, q


def _visible(kv, q, window, sinks):
    """(keys that any of the q new tokens sees, pairs of a new token and a key that it sees)."""
    pairs = 0
    for p in range(kv - q, kv):
        n = p + 1
        pairs += n if not window or n <= window else window + min(sinks, n - window)
    if not window:
        return kv, pairs
    first = max(0, kv - q - window + 1)
    return kv - first + min(sinks, first), pairs


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["src"] == "f32" else 2) + 28 * case["rows"], "flops": 2 * n}
    kv, q = _lengths(case)
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["hd"]
    t = sum(q)
    if case["op"] == "qk":
        size = 4 if case["src"] == "f32" else 2
        return {"bytes": t * ((heads + 2 * kv_heads) * hd * (size + 2) + hd * 4), "flops": t * (heads + kv_heads) * hd * 7}
    seen = [_visible(a, b, case["window"], case["sinks"]) for a, b in zip(kv, q)]
    return {"bytes": 2 * t * heads * hd * 2 + sum(s[0] for s in seen) * kv_heads * hd * 4,
            "flops": 4 * hd * heads * sum(s[1] for s in seen)}


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    s = dict(case)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = 2.2 * normal(rows, vocab)
        # a model's logits: a broad floor and a few candidates well above it
        at = torch.randint(vocab, (rows, 24), generator=g, device="cuda")
        x.scatter_add_(1, at, 4 + 9 * torch.rand(rows, 24, generator=g, device="cuda"))
        s["logits"] = x.to(TYPES[case["src"]])
        s["u"] = torch.rand(rows, generator=g, device="cuda")

        def pick(*values, dtype=torch.float32):
            i = torch.randint(len(values), (rows,), generator=g, device="cuda")
            return torch.tensor(values, dtype=dtype, device="cuda")[i]

        mode = case["mode"]
        ones, zeros = torch.ones(rows, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["temperature"] = pick(0.6, 0.7, 0.8, 1.0, 1.3, *([0.0] if mode == "mixed" and rows > 1 else []))
        s["top_k"] = pick(20, 40, 50, 200, 0 if rows > 1 else 64, dtype=torch.int32) if mode in ("mixed", "topk") else zeros
        s["top_p"] = pick(0.8, 0.9, 0.95, 1.0 if mode == "mixed" else 0.97) if mode in ("mixed", "nucleus") else ones
        s["min_p"] = pick(0.0, 0.02, 0.05) if mode == "mixed" else torch.zeros(rows, device="cuda")
        return s
    kv, q = _lengths(case)
    heads, kv_heads, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    cache = TYPES[case["cache"]]
    per_seq = -(-case["kv_max"] // page)
    need = sum(-(-n // page) for n in kv)
    pages = need + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)   # a cache that has been in use: pages anywhere
    table = torch.zeros(len(kv), per_seq, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(kv):
        c = -(-n // page)
        table[i, :c] = order[at:at + c]
        at += c
    s["k_pages"], s["v_pages"] = normal(pages, page, kv_heads, hd, dtype=cache), normal(pages, page, kv_heads, hd, dtype=cache)
    s["table"] = table
    s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["q_start"] = torch.tensor([0] + [sum(q[:i + 1]) for i in range(len(q))], dtype=torch.int32, device="cuda")
    s["max_q"], s["tokens"] = max(q), sum(q)
    if case["op"] == "attn":
        s["q"] = normal(sum(q), heads, hd, dtype=cache)
        s["scale"] = 1.0 / math.sqrt(hd)
        return s
    src = TYPES[case["src"]]
    # the projections as one product leaves them: a row holds the queries, the keys and the values
    qkv = (1.5 * normal(sum(q), heads + 2 * kv_heads, hd)).to(src)
    s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    if case["norm"] != NORM_NONE:
        whole = case["norm"] == NORM_ROW
        s["q_norm"] = 1 + 0.2 * normal(heads * hd if whole else hd)
        s["k_norm"] = 1 + 0.2 * normal(kv_heads * hd if whole else hd)
    else:
        s["q_norm"] = s["k_norm"] = None
    angle = torch.arange(case["kv_max"], dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(hd // 2, dtype=torch.float64) * 2 / hd)
    s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
    return s


# ---- the calls -------------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    return {"qk": _plain_qk, "attn": _plain_attn, "sample": _plain_sample}[state["op"]](state)


_context = None


def _own(s):
    global _context
    import clutor_b200 as cb
    if _context is None:
        _context = cb.Context(torch.cuda.current_device())
    if s["op"] == "sample":
        token, prob = _context.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        return {"token": token, "prob": prob}
    pages = cb.KvPages(s["k_pages"], s["v_pages"], s["table"])
    if s["op"] == "attn":
        return {"out": _context.attention(s["q"], pages, s["q_start"], s["kv_len"], max_q=s["max_q"], scale=s["scale"],
                                          window=s["window"], sinks=s["sinks"])}
    out = _context.qk_rope(s["q"], s["k"], s["v"], pages, s["q_start"], s["kv_len"], s["rope"], q_norm=s["q_norm"],
                           k_norm=s["k_norm"], norm=s["norm"], pairs=s["pairs"], eps=EPS)
    return {"q": out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


# ---- plain forms -----------------------------------------------------------------------------------------------------------

def _rows(s):
    """Each row's sequence, and its place among that sequence's new tokens."""
    row = torch.arange(s["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["q_start"][1:].contiguous(), row, right=True)
    return seq, row - s["q_start"][seq]


def _slots(s, seq, pos):
    """The cache rows (page * page size + slot) of positions of sequences."""
    pos = pos.long()
    return s["table"][seq, pos // s["page"]].long() * s["page"] + pos % s["page"]


def _plain_qk(s):
    hd, half = s["hd"], s["hd"] // 2
    seq, i = _rows(s)
    pos = (s["kv_len"] - (s["q_start"][1:] - s["q_start"][:-1]))[seq] + i

    def normed(x, w):
        if s["norm"] == NORM_NONE:
            return x
        if s["norm"] == NORM_HEAD:
            return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        return x * torch.rsqrt(x.square().mean((-1, -2), keepdim=True) + EPS) * w.view(x.shape[1:])

    cs = s["rope"][pos.long()][:, None]
    c, n = cs[..., :half], cs[..., half:]

    def turned(x):
        if s["pairs"]:
            a, b = x[..., 0::2], x[..., 1::2]
            return torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * c - b * n, a * n + b * c], -1)

    cache = s["k_pages"].dtype
    q, k = turned(normed(s["q"].float(), s["q_norm"])), turned(normed(s["k"].float(), s["k_norm"]))
    at = _slots(s, seq, pos)
    s["k_pages"].view(-1, s["kv_heads"], hd)[at] = k.to(cache)
    s["v_pages"].view(-1, s["kv_heads"], hd)[at] = s["v"].float().to(cache)
    return {"q": q.to(cache), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attn(s):
    heads, kv_heads, hd, n_seq, lq = s["heads"], s["kv_heads"], s["hd"], s["n_seq"], s["max_q"]
    lk, group = s["kv_max"], heads // kv_heads
    seq, i = _rows(s)
    q = torch.zeros(n_seq, lq, heads, hd, device="cuda")   # the sequences side by side, padded to the longest
    q[seq, i.long()] = s["q"].float()
    q = q.view(n_seq, lq, kv_heads, group, hd).permute(0, 2, 1, 3, 4).reshape(n_seq, kv_heads, lq * group, hd)
    j = torch.arange(lk, device="cuda", dtype=torch.int32)
    alive = j < s["kv_len"][:, None]
    at = torch.where(alive, _slots(s, torch.arange(n_seq, device="cuda")[:, None], j.expand(n_seq, lk)), 0)
    blank = ~alive[:, :, None, None]
    k = s["k_pages"].view(-1, kv_heads, hd)[at].float().masked_fill(blank, 0.0).permute(0, 2, 1, 3)
    v = s["v_pages"].view(-1, kv_heads, hd)[at].float().masked_fill(blank, 0.0).permute(0, 2, 1, 3)
    new = s["q_start"][1:] - s["q_start"][:-1]
    pos = (s["kv_len"] - new)[:, None] + torch.arange(lq, device="cuda", dtype=torch.int32)
    hidden = (j > pos[..., None]) | ~alive[:, None]
    if s["window"]:
        hidden |= (j <= pos[..., None] - s["window"]) & (j >= s["sinks"])
    hidden = hidden[:, None].repeat_interleave(group, 2)
    x = (q @ k.transpose(-1, -2)).mul_(s["scale"]).masked_fill_(hidden, -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min(-3e38)
    x = x.sub_(top).exp_()
    o = (x @ v) / x.sum(-1, keepdim=True).clamp_min(1e-37)
    o = o.view(n_seq, kv_heads, lq, group, hd).permute(0, 2, 1, 3, 4).reshape(n_seq, lq, heads, hd)
    return {"out": o[seq, i.long()].to(s["k_pages"].dtype)}


def _plain_sample(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"]).double()
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = ((x.double() - x[:, :1].double()) / t[:, None]).exp()   # in 64 bits: a sum decides which token's border u falls behind
    rank = torch.arange(vocab, device="cuda")
    k = torch.where(s["top_k"] <= 0, vocab, s["top_k"]).clamp_max(vocab)
    k = torch.where(greedy, 1, k)
    kept = rank < k[:, None]
    w = w * kept
    total = w.cumsum(1)
    want = s["top_p"].double()[:, None] * total[:, -1:]
    kept &= (total - w < want) | (s["top_p"] >= 1)[:, None]     # the shortest prefix that reaches the share, one token at least
    kept &= w >= s["min_p"].double()[:, None]
    kept[:, 0] = True
    w = torch.zeros(rows, vocab, dtype=torch.float64, device="cuda").scatter_(1, order, w * kept)
    total = w.cumsum(1)
    want = s["u"].double()[:, None] * total[:, -1:]
    token = (total <= want).sum(1).clamp_max(vocab - 1)
    return {"token": token.int(), "prob": (w.gather(1, token[:, None])[:, 0] / total[:, -1]).float()}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    q_start, kv_len = s["q_start"].tolist(), s["kv_len"].tolist()
    hd, heads, kv_heads, page = case["hd"], case["heads"], case["kv_heads"], case["page"]
    if case["op"] == "qk":
        out = torch.zeros(s["tokens"], heads, hd, dtype=torch.float64, device="cuda")
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        for b in range(case["n_seq"]):
            a, z = q_start[b], q_start[b + 1]
            first = kv_len[b] - (z - a)
            pos = torch.arange(first, kv_len[b], device="cuda")
            pg, slot = s["table"][b].long()[pos.div(page, rounding_mode="floor")], pos.remainder(page)
            cos, sin = s["rope"][first:kv_len[b]].double().unsqueeze(1).chunk(2, -1)
            for src, w, put in ((s["q"], s["q_norm"], None), (s["k"], s["k_norm"], kp)):
                x = src[a:z].double()
                if case["norm"] == NORM_HEAD:
                    x = x / (x.pow(2).sum(2, keepdim=True) / hd + EPS).sqrt() * w.double()
                elif case["norm"] == NORM_ROW:
                    x = x / (x.pow(2).sum((1, 2), keepdim=True) / x[0].numel() + EPS).sqrt() * w.double().reshape(1, -1, hd)
                even, odd = (x.unflatten(2, (hd // 2, 2)).unbind(3)) if case["pairs"] else x.unflatten(2, (2, hd // 2)).unbind(2)
                re, im = even * cos - odd * sin, odd * cos + even * sin
                y = torch.stack((re, im), 3).flatten(2) if case["pairs"] else torch.stack((re, im), 2).flatten(2)
                if put is None:
                    out[a:z] = y
                else:
                    put[pg, slot] = y
            vp[pg, slot] = s["v"][a:z].double()
        return {"q": out, "k_pages": kp, "v_pages": vp}
    out = torch.zeros(s["tokens"], heads, hd, dtype=torch.float64, device="cuda")
    for b in range(case["n_seq"]):
        n, a, z = kv_len[b], q_start[b], q_start[b + 1]
        pg = s["table"][b, :-(-n // page)].long()
        k, v = (t[pg].flatten(0, 1)[:n].double() for t in (s["k_pages"], s["v_pages"]))
        at = torch.arange(n, device="cuda")
        for r in range(a, z, 512):
            e = min(z, r + 512)
            pos = torch.arange(n - (z - r), n - (z - e), device="cuda").unsqueeze(1)
            see = at <= pos
            if case["window"]:
                see &= (pos - at < case["window"]) | (at < case["sinks"])
            for h in range(kv_heads):
                g = heads // kv_heads
                qs = s["q"][r:e, h * g:(h + 1) * g].double().transpose(0, 1)
                p = torch.softmax((qs @ k[:, h].T * s["scale"]).masked_fill(~see, float("-inf")), -1)
                out[r:e, h * g:(h + 1) * g] = (p @ v[:, h]).transpose(0, 1)
    return {"out": out}


def _exact_sample(s):
    tokens, probs = [], []
    for r in range(s["rows"]):
        x = s["logits"][r].double().cpu().numpy()
        t, k, p, m, u = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        order = (-x).argsort(kind="stable")
        if t <= 0:
            tokens.append(int(order[0]))
            probs.append(1.0)
            continue
        order = order[:int(k)] if 0 < k < len(x) else order
        e = (x[order] - x[order[0]]) / t
        w = torch.from_numpy(e).exp().numpy()
        if p < 1:
            n = int(w.cumsum().searchsorted(p * w.sum())) + 1
            order, w = order[:n], w[:n]
        order, w = order[w >= min(m, 1.0)], w[w >= min(m, 1.0)]
        by = order.argsort()
        order, w = order[by], w[by]
        at = min(int(w.cumsum().searchsorted(u * w.sum(), side="right")), len(w) - 1)
        tokens.append(int(order[at]))
        probs.append(float(w[at] / w.sum()))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}
