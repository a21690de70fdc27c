"""The serving operators on a B200 (clb200_qk_rope, clb200_attention, clb200_sample) against plain 64-bit forms.

Bars, each a bound by arithmetic on the operator's own roundings:
  qk_rope: the result is rounded once to the cache's type (half a step of it); before that every value went through at most
    ~40 fp32 roundings (squares, their tree of sums, root, quotient, two products, the rotation), each 2^-24 of a term.
  attention: scores are fp32 sums of hd products; an error d of a score changes a probability by at most 2 d relative; the
    probabilities are rounded to the cache's type (half a step each, and in fp16 at least 2^-25 absolute), their sums and the
    value sums are fp32 (n + 64 roundings at worst), the exponentials are good to 2^-21, the result is rounded once.
  sample: token equal; prob a quotient of two values good to 2^-40, rounded once.
"""
import copy

import numpy as np
import pytest

from tests import serving_ref as ref

pytestmark = pytest.mark.gpu
NP_TYPE = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


@pytest.fixture(scope="module")
def ctx():
    import clutor_b200 as cb
    c = cb.Context(0)
    yield c
    c.status()
    c.close()


def dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Batch:
    """A paged cache with `kv` positions per sequence, `q` of them new, in the given layout; unused slots hold NaN."""

    def __init__(self, kv, q, kv_heads, hd, page, cache, seed, layout="slots", spare=2):
        import torch

        import clutor_b200 as cb
        rng = np.random.default_rng(seed)
        self.kv, self.q, self.page, self.KV, self.D = list(kv), list(q), page, kv_heads, hd
        need = [-(-n // page) for n in kv]
        P = sum(need) + spare
        ids = rng.permutation(P).astype(np.int32)
        width = max(need + [1])
        table = np.full((len(kv), width), 7 * 10 ** 8, np.int32)   # ids past a sequence's pages are never read
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = ids[at:at + n]
            at += n
        dt = dtype(cache)
        if layout == "slots":
            pool = torch.full((2, P, page, kv_heads, hd), float("nan"), dtype=dt, device="cuda")
            k, v = pool[0], pool[1]
        elif layout == "heads":   # a page's heads one after another
            pool = torch.full((2, P, kv_heads, page, hd), float("nan"), dtype=dt, device="cuda")
            k, v = pool[0].transpose(1, 2), pool[1].transpose(1, 2)
        else:                     # keys and values of a page side by side, in rows wider than they need
            pool = torch.full((P, 2, page, kv_heads, hd + 16), float("nan"), dtype=dt, device="cuda")
            k, v = pool[:, 0, ..., :hd], pool[:, 1, ..., :hd]
        self.pool, self.k, self.v, self.np_table = pool, k, v, table
        self.pages = cb.KvPages(k, v, torch.from_numpy(table).cuda())
        self.q_start = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
        self.q_start_d, self.kv_len_d = torch.from_numpy(self.q_start).cuda(), torch.tensor(self.kv, dtype=torch.int32, device="cuda")
        self.T = int(self.q_start[-1])

    def fill(self, seed):
        """Random keys and values in every position's slot."""
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        for s, n in enumerate(self.kv):
            if n:
                p, i = self.where(s, np.arange(n))
                for t in (self.k, self.v):
                    t[p, i] = torch.randn(n, self.KV, self.D, generator=g, device="cuda").to(t.dtype)

    def where(self, s, pos):
        import torch
        return (torch.from_numpy(self.np_table[s][pos // self.page].astype(np.int64)).cuda(),
                torch.from_numpy((pos % self.page).astype(np.int64)).cuda())

    def cache_of(self, s):
        p, i = self.where(s, np.arange(self.kv[s]))
        return self.k[p, i].double().cpu().numpy(), self.v[p, i].double().cpu().numpy()


# ---- qk_rope ---------------------------------------------------------------------------------------------------------------

QK = [  # kv, q, heads, kv_heads, hd, page, src, cache, norm, pairs, layout, fused
    ([1], [1], 4, 2, 64, 16, "f32", "f16", 2, False, "slots", False),
    ([70, 1, 33], [70, 1, 3], 8, 2, 128, 32, "f32", "bf16", 2, False, "heads", True),
    ([70, 0, 40], [5, 0, 17], 16, 16, 128, 16, "f32", "f16", 1, False, "wide", True),
    ([50, 20], [50, 2], 3, 1, 256, 48, "bf16", "bf16", 2, True, "slots", True),
    ([17, 300], [17, 9], 5, 5, 64, 128, "f16", "f16", 0, True, "heads", False),
    ([129] * 40, [1] * 40, 32, 4, 128, 64, "f32", "f16", 2, False, "slots", True),
    ([33], [33], 7, 1, 64, 16, "f32", "bf16", 1, True, "wide", False),
]


@pytest.mark.parametrize("kv,q,H,KV,D,page,src,cache,norm,pairs,layout,fused", QK)
def test_qk_rope(ctx, kv, q, H, KV, D, page, src, cache, norm, pairs, layout, fused):
    import torch
    b = Batch(kv, q, KV, D, page, cache, seed=len(kv) + D, layout=layout)
    g = torch.Generator(device="cuda").manual_seed(11)
    pad = 3   # rows behind the last sequence
    T = b.T + pad
    if fused:
        qkv = (1.5 * torch.randn(T, H + 2 * KV, D, generator=g, device="cuda")).to(dtype(src))
        x, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    else:
        x, k, v = ((1.5 * torch.randn(T, n, D, generator=g, device="cuda")).to(dtype(src)) for n in (H, KV, KV))
    whole = norm == 1
    qn, kn = (1 + 0.3 * torch.randn(n * D if whole else D, generator=g, device="cuda") for n in (H, KV))
    angle = np.arange(max(kv))[:, None] * 1e4 ** (-np.arange(D // 2) * 2 / D)
    rope = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)).cuda()
    out = torch.full((T, H, D), 77.0, dtype=dtype(cache), device="cuda")
    before = b.pool.clone()
    got = ctx.qk_rope(x, k, v, b.pages, b.q_start_d, b.kv_len_d, rope, q_norm=qn if norm else None, k_norm=kn if norm else None,
                      norm=norm, pairs=pairs, eps=1e-5, out=out)
    ctx.status()
    assert got is out
    half, tiny = ref.HALF[NP_TYPE[cache]], 2.0 ** -25 if cache == "f16" else 0.0
    xs, ks, vs = (t.double().cpu().numpy() for t in (x, k, v))
    qw, kw, cs = qn.double().cpu().numpy(), kn.double().cpu().numpy(), rope.double().cpu().numpy()
    res = out.double().cpu().numpy()
    want_k, want_v = b.k.clone(), b.v.clone()
    for r, s, pos in ref.positions(b.q_start, kv):
        y, mag = ref.qk_rope(xs[r], qw, cs[pos], norm, pairs, 1e-5)
        assert (np.abs(res[r] - y) <= half * np.abs(y) + 40 * 2.0 ** -24 * mag + tiny).all()
        p, i = b.where(s, np.array([pos]))
        y, mag = ref.qk_rope(ks[r], kw, cs[pos], norm, pairs, 1e-5)
        gk = b.k[p, i][0].double().cpu().numpy()
        assert (np.abs(gk - y) <= half * np.abs(y) + 40 * 2.0 ** -24 * mag + tiny).all()
        assert torch.equal(b.v[p, i][0], v[r].to(dtype(cache)))
        want_k[p, i], want_v[p, i] = b.k[p, i], b.v[p, i]
    assert (res[b.T:] == 77.0).all()
    # nothing but the new tokens' slots was written
    after = b.pool.clone()
    b.pool.copy_(before)
    for r, s, pos in ref.positions(b.q_start, kv):
        p, i = b.where(s, np.array([pos]))
        b.k[p, i], b.v[p, i] = want_k[p, i], want_v[p, i]
    assert torch.equal(b.pool.view(torch.int16), after.view(torch.int16))


# ---- attention -------------------------------------------------------------------------------------------------------------

ATTN = [  # kv, q, heads, kv_heads, hd, page, cache, window, sinks, layout
    ([1], [1], 1, 1, 64, 16, "f16", 0, 0, "slots"),
    ([7, 1, 16, 17], [1, 1, 1, 1], 8, 2, 128, 16, "f16", 0, 0, "slots"),
    ([1000, 130, 0, 64, 65], [1, 1, 0, 1, 1], 32, 4, 128, 64, "bf16", 0, 0, "heads"),
    ([513, 100], [2, 4], 16, 1, 64, 32, "bf16", 0, 0, "wide"),
    ([3000], [1], 16, 2, 128, 48, "f16", 0, 0, "slots"),
    ([300, 40], [1, 1], 6, 2, 256, 16, "bf16", 0, 0, "heads"),
    ([200, 3, 150], [200, 3, 20], 8, 2, 128, 16, "bf16", 0, 0, "slots"),
    ([129], [129], 4, 4, 64, 64, "f16", 0, 0, "wide"),
    ([300, 128, 257], [255, 1, 257], 14, 2, 64, 32, "f16", 0, 0, "heads"),
    ([140, 70], [33, 70], 5, 1, 256, 16, "bf16", 0, 0, "slots"),
    ([600], [130], 32, 2, 128, 128, "bf16", 0, 0, "slots"),
    ([600, 90], [130, 90], 8, 4, 64, 16, "bf16", 37, 0, "slots"),
    ([600, 90], [130, 90], 8, 4, 128, 48, "f16", 100, 5, "heads"),
    ([900, 20], [1, 1], 8, 1, 128, 16, "f16", 1, 0, "slots"),
    ([900, 20, 400], [1, 1, 1], 8, 1, 64, 16, "bf16", 64, 130, "slots"),
    ([300], [3], 9, 3, 128, 16, "f16", 50, 2, "slots"),
    ([5, 9], [7, 9], 4, 2, 128, 16, "f16", 0, 0, "slots"),       # the first sequence's first rows have no position: they see nothing
    ([2, 2], [5, 0], 2, 2, 64, 16, "bf16", 1, 0, "slots"),
]


def attn_check(b, x, out, H, cache, window, sinks, scale, out_type=None):
    out_half, half = ref.HALF[NP_TYPE[out_type or cache]], ref.HALF[NP_TYPE[cache]]
    res, xs = out.double().cpu().numpy(), x.double().cpu().numpy()
    caches = [b.cache_of(s) if n else (np.zeros((0, b.KV, b.D)),) * 2 for s, n in enumerate(b.kv)]
    for r, s, pos in ref.positions(b.q_start, b.kv):
        k, v = caches[s]
        y, mag, flat, big = ref.attention(xs[r], k, v, pos, scale, window, sinks)
        rel = half + 2 * (b.D + 2) * 2.0 ** -24 * big + 2.0 ** -21 + (min(len(k), pos + 1) + 64) * 2.0 ** -23
        bar = out_half * np.abs(y) + mag * rel * 1.01 + (2.0 ** -25 * flat if cache == "f16" else 0) + (2.0 ** -25 if out_half == 2.0 ** -11 else 0)
        assert np.isfinite(res[r]).all(), (r, s, pos)
        worst = (np.abs(res[r] - y) - bar).max()
        assert worst <= 0, (r, s, pos, worst, np.abs(res[r] - y).max())


@pytest.mark.parametrize("kv,q,H,KV,D,page,cache,window,sinks,layout", ATTN)
def test_attention(ctx, kv, q, H, KV, D, page, cache, window, sinks, layout):
    import torch
    b = Batch(kv, q, KV, D, page, cache, seed=len(kv) + D + H, layout=layout)
    b.fill(5)
    g = torch.Generator(device="cuda").manual_seed(3)
    T = b.T + 2
    x = (2 * torch.randn(T, H, D, generator=g, device="cuda")).to(dtype(cache))
    out = torch.full((T, H, D), 77.0, dtype=dtype(cache), device="cuda")
    ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=max(q), window=window, sinks=sinks, out=out)
    ctx.status()
    attn_check(b, x, out, H, cache, window, sinks, D ** -0.5)
    assert (out[b.T:] == 77.0).all()
    again = ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=max(q), window=window, sinks=sinks)
    assert torch.equal(again[:b.T], out[:b.T])   # the same call gives the same bits
    loose = ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, window=window, sinks=sinks, scale=0.3, out_dtype=torch.float32)
    ctx.status()
    attn_check(b, x, loose, H, cache, window, sinks, float(np.float32(0.3)), out_type="f32")


# ---- sample ----------------------------------------------------------------------------------------------------------------

def sample_check(ctx, lg, u, t=None, k=None, p=None, m=None):
    import torch

    def dev(a, d):
        return None if a is None else torch.tensor(a, dtype=d, device="cuda")

    tok, prob = ctx.sample(lg, dev(u, torch.float32), dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32),
                           dev(m, torch.float32))
    ctx.status()
    tok, prob, xs = tok.cpu().numpy(), prob.cpu().numpy(), lg.double().cpu().numpy()

    def at(a, r, d):
        return d if a is None else a[r] if isinstance(a[r], int) else float(np.float32(a[r]))

    for r in range(len(xs)):
        want, wp = ref.sample(xs[r], at(u, r, 0), at(t, r, 1.0), at(k, r, 0), at(p, r, 1.0), at(m, r, 0.0))
        assert tok[r] == want, (r, tok[r], want)
        assert abs(prob[r] - wp) <= 2.0 ** -23 * wp + 1e-45, (r, prob[r], wp)


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 50304, 151936, 262144])
@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_sample_random(ctx, vocab, src):
    import torch
    rng = np.random.default_rng(vocab)
    R = 24
    g = torch.Generator(device="cuda").manual_seed(vocab)
    lg = (2.5 * torch.randn(R, vocab + 3, generator=g, device="cuda")).to(dtype(src))[:, :vocab]   # odd strides and starts
    u = [float(v) for v in rng.random(R).astype(np.float32)]
    u[0], u[1] = 0.0, float(np.float32(1 - 2.0 ** -24))
    t = [float(v) for v in rng.choice([0.0, 0.5, 0.8, 1.0, 1.7], R)]
    k = [int(v) for v in rng.choice([0, 1, 2, 40, 1000, vocab, 10 ** 6], R)]
    p = [float(v) for v in rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0], R)]
    m = [float(v) for v in rng.choice([0.0, 0.01, 0.2, 1.0, 2.0], R)]
    sample_check(ctx, lg, u, t, k, p, m)
    sample_check(ctx, lg, u)
    sample_check(ctx, lg, u, t)
    sample_check(ctx, lg, u, k=k)
    sample_check(ctx, lg, u, t, p=p)
    sample_check(ctx, lg, u, m=m)


def test_sample_ties_and_infinities(ctx):
    import torch
    inf, nan = float("inf"), float("nan")
    V = 5000
    lg = torch.zeros(12, V, device="cuda")           # all equal: ties go to the lowest ids
    lg[1, ::2] = -inf
    lg[2] = -inf
    lg[2, 4321] = -3.0
    lg[3] = -inf                                      # nothing
    lg[4] = nan
    lg[5, 17] = inf
    lg[5, 4000] = inf                                 # two at +infinity share everything
    lg[6] = nan
    lg[6, 9] = 1.0
    lg[7, 2500:] = -0.0                               # equal to 0
    lg[8, 1000:1100] = 1.0
    lg[9] = torch.linspace(-200, 200, V)
    lg[10] = -3e38
    lg[10, 3] = 3e38
    lg[11, 0] = 1e-30
    u = [0.999, 0.5, 0.3, 0.4, 0.2, 0.6, 0.1, 0.7, 0.5, 0.999, 0.5, 0.25]
    for kw in ({}, {"k": [7] * 12}, {"p": [0.5] * 12}, {"k": [100] * 12, "p": [0.25] * 12}, {"m": [0.5] * 12}, {"t": [0.0] * 12},
               {"t": [inf] * 12}, {"t": [1e-40] * 12}, {"k": [1] * 12}, {"k": [4999] * 12, "p": [0.9999] * 12, "t": [3.0] * 12}):
        sample_check(ctx, lg, u, **kw)


@pytest.mark.parametrize("v", [900, 20011, 100000])
def test_sample_logits_around_zero(ctx, v):
    """Both zeros and the smallest numbers of either sign, many times each, so that borders fall on zero and between the keys of its
    neighbours; and sets in one bin of the first histogram, which finer ones have to divide."""
    import torch
    rng = np.random.default_rng(v)
    R = 12
    tiny = np.array([0.0, -0.0, 1e-45, -1e-45, 3e-42, -3e-42, 1.2e-38, -1.2e-38, 1e-30, -1e-30], np.float32)
    lg = rng.choice(tiny, (R, v)).astype(np.float32)
    lg[4:8] += rng.normal(0, 1e-3, (4, v)).astype(np.float32) * (rng.random((4, v)) < 0.5)
    lg[8:] = -np.abs(lg[8:])
    lg[10:, ::7] = 2.0
    u = [float(x) for x in rng.random(R).astype(np.float32)]
    k = [int(x) for x in rng.integers(1, v, R)]
    for kw in ({"k": k}, {"p": [0.3] * R}, {"k": k, "p": [0.6] * R}, {"p": [0.5] * R, "t": [1e-3] * R}, {"k": k, "t": [1e-30] * R},
               {"k": [min(40, v // 2)] * R, "t": [1e-4] * R}):
        sample_check(ctx, torch.from_numpy(lg).cuda(), u, **kw)


def test_sample_distribution_of_many_rows(ctx):
    """700 rows of the same logits with u on a grid: the tokens come in the order of the cumulative distribution."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    lg = (3 * torch.randn(1, 2000, generator=g, device="cuda")).expand(700, 2000).contiguous()
    sample_check(ctx, lg, [float(np.float32((i + 0.5) / 700)) for i in range(700)], p=[0.95] * 700)


# ---- together --------------------------------------------------------------------------------------------------------------

def test_steps_together_captured(ctx):
    """Two sequences: a prompt chunk, then single tokens, through qk_rope -> attention -> a product -> sample, captured in one
    graph with its lengths in device memory and replayed for each step; the same steps one call at a time give the same bits."""
    import torch
    H, KV, D, V, page = 8, 2, 128, 999, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    angle = np.arange(64)[:, None] * 1e4 ** (-np.arange(D // 2) * 2 / D)
    rope = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)).cuda()
    qn, kn = (1 + 0.1 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    head = 0.05 * torch.randn(H * D, V, generator=g, device="cuda")
    data = torch.randn(8, 2, H + 2 * KV, D, generator=g, device="cuda")
    us = torch.rand(8, 2, generator=g, device="cuda")

    def make():
        b = Batch([30, 50], [1, 1], KV, D, page, "bf16", seed=4)
        b.pages.table.copy_(torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)[:, :b.pages.table.shape[1]])
        b.np_table = b.pages.table.cpu().numpy()
        b.kv = [30, 50]
        b.fill(9)
        b.kv_len_d.copy_(torch.tensor([30, 50], device="cuda"))
        return b

    def step(b, qkv, u):
        q = ctx.qk_rope(qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:], b.pages, b.q_start_d, b.kv_len_d, rope, q_norm=qn, k_norm=kn)
        o = ctx.attention(q, b.pages, b.q_start_d, b.kv_len_d, max_q=1)
        return ctx.sample(o.float().view(2, -1) @ head, u, top_p=torch.full((2,), 0.9, device="cuda"))

    b = make()
    eager = []
    for i in range(8):
        b.kv_len_d += 1
        tok, prob = step(b, data[i], us[i])
        eager.append((tok.tolist(), prob.tolist()))
    want_k = b.k.clone()
    c = make()
    qkv, u = data[0].clone(), us[0].clone()
    with torch.cuda.stream(torch.cuda.Stream()):
        step(c, qkv, u)   # warm-up writes position 29 / 49 again
    c2 = make()
    c.pool.copy_(c2.pool)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.kv_len_d += 1
        tok, prob = step(c, qkv, u)
    for i in range(8):
        qkv.copy_(data[i])
        u.copy_(us[i])
        graph.replay()
        torch.cuda.synchronize()
        assert (tok.tolist(), prob.tolist()) == eager[i]
    assert torch.equal(c.k.contiguous().view(torch.int16), want_k.contiguous().view(torch.int16))
    ctx.status()


def test_attention_many_sequences(ctx):
    """More sequences than one launch takes (512), and sequences without rows between others; few and many rows a head."""
    import torch
    rng = np.random.default_rng(8)
    for q_max, KV, H, D in ((1, 2, 6, 64), (9, 1, 8, 128)):
        n = 1100
        q = [int(v) for v in rng.integers(0, q_max + 1, n)]
        kv = [int(v) for v in np.maximum(rng.integers(0, 60, n), q)]
        b = Batch(kv, q, KV, D, 16, "bf16", seed=D)
        b.fill(1)
        x = torch.randn(b.T, H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(torch.bfloat16)
        out = ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=q_max)
        ctx.status()
        attn_check(b, x, out, H, "bf16", 0, 0, D ** -0.5)


def test_attention_large_offsets(ctx):
    """A cache whose elements lie beyond 2^31 elements and 2^32 bytes from its start."""
    import torch

    import clutor_b200 as cb
    KV, D, page, stride = 2, 64, 16, (1 << 31) // 3 // 8 * 8
    pool = torch.empty(2, 3 * stride + page * KV * D, dtype=torch.float16, device="cuda")
    k, v = (pool[i].as_strided((4, page, KV, D), (stride, KV * D, D, 1), pool[i].storage_offset()) for i in (0, 1))
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.tensor([[3, 0, 2], [1, 3, 2]], dtype=torch.int32, device="cuda")
    for p in range(4):
        k[p], v[p] = (torch.randn(page, KV, D, generator=g, device="cuda").half() for _ in range(2))
    pages = cb.KvPages(k, v, table)
    kv = torch.tensor([45, 33], dtype=torch.int32, device="cuda")
    for q in ([1, 1], [40, 33]):
        qs = torch.tensor([0, q[0], sum(q)], dtype=torch.int32, device="cuda")
        x = torch.randn(sum(q), 8, D, generator=g, device="cuda").half()
        out = ctx.attention(x, pages, qs, kv, max_q=max(q)).double().cpu().numpy()
        ctx.status()
        for s, (n, t) in enumerate(((45, [3, 0, 2]), (33, [1, 3, 2]))):
            kk, vv = (c[torch.tensor(t, device="cuda")].flatten(0, 1)[:n].double().cpu().numpy() for c in (k, v))
            for i in range(q[s]):
                r = int(qs[s]) + i
                y, mag, flat, big = ref.attention(x[r].double().cpu().numpy(), kk, vv, n - q[s] + i, D ** -0.5, 0, 0)
                assert (np.abs(out[r] - y) <= 2.0 ** -11 * np.abs(y) + mag * (2.0 ** -11 + 132 * 2.0 ** -24 * big + 2.0 ** -20) * 1.01 + 2.0 ** -25 * (flat + 1)).all()
    # and the store
    x = torch.randn(2, 8 + 2 * KV, D, generator=g, device="cuda")
    rope = torch.cat([torch.ones(64, D // 2), torch.zeros(64, D // 2)], 1).cuda()
    ctx.qk_rope(x[:, :8], x[:, 8:8 + KV], x[:, 8 + KV:], pages, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), kv, rope, norm=0)
    ctx.status()
    assert torch.equal(v[2, 44 % 16], x[0, 8 + KV:].half()) and torch.equal(k[2, 32 % 16], x[1, 8:8 + KV].half())


def test_streams_and_two_graphs_at_once(ctx):
    """Calls on a stream of their own, and two captured graphs of the same calls replayed at the same time: each has its own
    workspace, so neither disturbs the other. The lengths in device memory change between replays."""
    import torch
    H, KV, D = 16, 2, 128
    made = []
    for i, (kv, q) in enumerate((([900, 400], [1, 1]), ([500, 260], [130, 70]))):
        b = Batch(kv, q, KV, D, 32, "bf16", seed=i)
        b.fill(i)
        g = torch.Generator(device="cuda").manual_seed(i)
        x = torch.randn(b.T, H, D, generator=g, device="cuda").to(torch.bfloat16)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        first = ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=max(q), stream=stream)
        torch.cuda.synchronize()
        attn_check(b, x, first, H, "bf16", 0, 0, D ** -0.5)
        with torch.cuda.graph(graph):
            out = ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=max(q))
        made.append((b, x, stream, graph, out))
    for less in (0, 7, 100):
        for b, x, stream, graph, out in made:
            b.kv = [n - less for n in b.kv]
            b.kv_len_d.copy_(torch.tensor(b.kv, device="cuda"))
        torch.cuda.synchronize()
        for _ in range(10):
            for b, x, stream, graph, out in made:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for b, x, stream, graph, out in made:
            attn_check(b, x, out, H, "bf16", 0, 0, D ** -0.5)
    ctx.status()


@pytest.mark.parametrize("rows,vocab", [(80, 50304), (160, 1000), (80, 60001), (40, 100003), (3, 151936), (1, 8191),
                                        (300, 10000), (150, 20011), (30, 30000), (60, 40000)])
def test_sample_row_splits(ctx, rows, vocab):
    """Every number of CTAs a row (1, 2, 4, 8), and of threads."""
    import torch
    rng = np.random.default_rng(rows + vocab)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    lg = 2 * torch.randn(rows, vocab, generator=g, device="cuda")
    lg.scatter_add_(1, torch.randint(vocab, (rows, 8), generator=g, device="cuda"), 9 * torch.rand(rows, 8, generator=g, device="cuda"))
    sample_check(ctx, lg, [float(v) for v in rng.random(rows).astype(np.float32)], [float(v) for v in rng.choice([0.0, 0.6, 1.0, 1.4], rows)],
                 [int(v) for v in rng.choice([0, 1, 30, 200, 256, 257, 3000], rows)], [float(v) for v in rng.choice([0.2, 0.9, 0.99, 1.0], rows)],
                 [float(v) for v in rng.choice([0.0, 0.03], rows)])


# ---- what only the device can see ------------------------------------------------------------------------------------------

def status_says(ctx, text):
    import clutor_b200 as cb
    with pytest.raises(cb.ClutorError, match=text):
        ctx.status()
    ctx.status()   # reported once


@pytest.mark.parametrize("q", [1, 40])
def test_bad_pages_and_rows_are_reported(ctx, q):
    """Page ids out of range, a table too short and more rows than max_q: skipped on the device and reported; the other sequence's
    rows are right, and the next call is."""
    import torch
    H, KV, D = 8, 1, 128
    b = Batch([70, 90], [q, q], KV, D, 16, "f16", seed=3)
    b.fill(2)
    x = torch.randn(b.T, H, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    good = ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=q)
    ctx.status()
    for bad in (-1, b.pages.n_pages, 2 ** 31 - 1):
        keep = b.pages.table[0, 2].clone()
        b.pages.table[0, 2] = bad
        out = ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=q)
        status_says(ctx, "page")
        assert torch.equal(out[q:], good[q:])
        b.pages.table[0, 2] = keep
    b.kv_len_d[0] = 16 * b.pages.table.shape[1] + 1
    out = torch.full_like(good, 5.0)
    ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=q, out=out)
    status_says(ctx, "page")
    assert torch.equal(out[q:], good[q:]) and (out[:q] == 5.0).all()
    b.kv_len_d[0] = 70
    starts = torch.tensor([0, q, 2 * q + 9], dtype=torch.int32, device="cuda")   # past the rows there are
    ctx.attention(x, b.pages, starts, b.kv_len_d, max_q=q + 9, out=out)
    status_says(ctx, "rows")
    first = copy.copy(b)   # another max_q may choose another kernel: the same values within the bar, not the same bits
    first.kv, first.q_start = [70], b.q_start[:2]
    attn_check(first, x, out, H, "f16", 0, 0, D ** -0.5)
    out.fill_(5.0)
    if q > 1:
        ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=q - 1, out=out)
        status_says(ctx, "rows")
        assert (out == 5.0).all()
    assert torch.equal(ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=q), good)
    ctx.status()


def test_bad_positions_in_the_rotation_are_reported(ctx):
    import torch
    H, KV, D = 4, 2, 64
    b = Batch([20, 30], [2, 3], KV, D, 16, "bf16", seed=3)
    x = torch.randn(b.T, H + 2 * KV, D, device="cuda")
    rope = torch.ones(25, D, device="cuda")           # positions 27..29 of the second sequence are past it
    before = b.pool.clone()
    out = torch.full((b.T, H, D), 9.0, dtype=torch.bfloat16, device="cuda")
    ctx.qk_rope(x[:, :H], x[:, H:H + KV], x[:, H + KV:], b.pages, b.q_start_d, b.kv_len_d, rope, norm=0, out=out)
    status_says(ctx, "rows")
    assert (out[2:] == 9.0).all() and (out[:2] != 9.0).any()
    p, i = b.where(0, np.arange(18, 20))
    changed = b.pool.view(torch.int16) != before.view(torch.int16)
    b.pool.copy_(before)
    b.k[p, i] = 1.0
    b.v[p, i] = 1.0
    assert not (changed & ~(b.pool.view(torch.int16) != before.view(torch.int16))).any()   # only those two slots
    b.pages.table[0, 1] = 10 ** 6
    ctx.qk_rope(x[:, :H], x[:, H:H + KV], x[:, H + KV:], b.pages, b.q_start_d, b.kv_len_d, torch.ones(64, D, device="cuda"), norm=0, out=out)
    status_says(ctx, "page")


def test_python_refusals(ctx):
    import torch

    import clutor_b200 as cb
    H, KV, D = 4, 2, 64
    b = Batch([20], [2], KV, D, 16, "bf16", seed=3)
    b.fill(1)
    x = torch.randn(2, H, D, device="cuda").to(torch.bfloat16)
    good = (x, b.pages, b.q_start_d, b.kv_len_d)
    cases = [lambda: ctx.attention(x.cpu(), *good[1:]), lambda: ctx.attention(x.half(), *good[1:]), lambda: ctx.attention(x[..., :32], *good[1:]),
             lambda: ctx.attention(x, b.pages, b.q_start_d.long(), b.kv_len_d), lambda: ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d.cpu()),
             lambda: ctx.attention(*good, out=x[:1]), lambda: ctx.attention(*good, out=x), lambda: ctx.attention(*good, scale=-1.0),
             lambda: ctx.attention(x.transpose(1, 2).contiguous().transpose(1, 2), *good[1:]), lambda: ctx.attention(x[:, :3], *good[1:]),
             lambda: cb.KvPages(b.k, b.v.half(), b.pages.table), lambda: cb.KvPages(b.k.float(), b.v.float(), b.pages.table),
             lambda: cb.KvPages(b.k, b.v, b.pages.table.long()), lambda: cb.KvPages(b.k, b.v, b.pages.table.cpu()),
             lambda: ctx.sample(x[0], torch.rand(3, device="cuda")), lambda: ctx.sample(x[0].float(), torch.rand(H, device="cuda"), top_k=torch.ones(H, device="cuda")),
             lambda: ctx.sample(x[0].float().t(), torch.rand(D, device="cuda")), lambda: ctx.sample(torch.zeros(1, (1 << 18) + 1, device="cuda"), torch.rand(1, device="cuda"))]
    for f in cases:
        with pytest.raises(cb.ClutorError):
            f()
    assert ctx.attention(*good).shape == x.shape
    empty = x[:0]
    assert ctx.attention(empty, b.pages, torch.zeros(2, dtype=torch.int32, device="cuda"), b.kv_len_d).shape == (0, H, D)
    assert ctx.sample(torch.zeros(0, 9, device="cuda"), torch.zeros(0, device="cuda"))[0].shape == (0,)
    ctx.status()


@pytest.mark.parametrize("H,KV,D", [(14, 2, 64), (12, 4, 128), (5, 1, 256), (8, 1, 128)])
def test_attention_padding_has_no_say(ctx, H, KV, D):
    """What stands in the rows of a padded batch, NaN included, changes no bit of the others (a group that does not divide the
    kernel's 128 rows leaves rows that belong to nobody too)."""
    import torch
    b = Batch([300, 128, 57], [255, 1, 57], KV, D, 32, "f16", seed=D)
    b.fill(5)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (2 * torch.randn(b.T + 40, H, D, generator=g, device="cuda")).half()
    outs = []
    for pad in (0.0, float("nan"), 300.0, float("inf")):
        x[b.T:] = pad
        for _ in range(3):
            outs.append(ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=255)[:b.T].clone())
    ctx.status()
    for o in outs:
        assert torch.equal(o, outs[0])
