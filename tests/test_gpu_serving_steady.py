"""clb200_attention where its kernels run as they do in use: many tiles of one item in a CTA, one after another, so that rings wrap,
maxima move from tile to tile, the score buffers take turns many times, and windows jump inside a run. (The work is dealt to the CTAs
in equal runs; inputs of a few thousand positions in all give each a tile or two.) And clb200_sample on half-precision logits.

The bars are those of test_gpu_serving.py, each derived there from the operator's roundings; the 64-bit form is computed here on the
device, a block of rows at a time."""
import numpy as np
import pytest

from tests import serving_ref as ref
from tests.test_gpu_serving import NP_TYPE, Batch, dtype, sample_check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import clutor_b200 as cb
    c = cb.Context(0)
    yield c
    c.status()
    c.close()


def longest_stretch(kv, q, H, KV, D, max_q, window, sinks, sms):
    """(the most tiles of one item that follow one another in a CTA, the stages of that kernel's ring), from the rules in
    clutor_b200/csrc/attn.cuh and attn.cu."""
    group = H // KV
    need = max_q * group
    few = need <= 16 or (need <= 32 and D <= 128)
    tile = 64 if few or D == 256 else 128
    tokens = (16 if need <= 16 else 32) // group if few else (1 if D == 256 else 2) * (128 // group)
    ctas, lead, least = sms * (2 if few and D <= 128 else 1), 3 if few else 2, 1 if few else 2
    items = []
    for n, new in zip(kv, q):
        for t0 in range(0, new, tokens):
            lo, hi = n - new + t0, n - new + min(t0 + tokens, new) - 1
            end = hi // tile + 1 if hi >= 0 else 1
            first = max(lo - window + 1, 0) // tile if window else 0
            items.append(end - first + min(-(-sinks // tile), first))
    items = [n for n in items for _ in range(KV)]
    run = max(-(-sum(n + lead for n in items) // ctas), least)
    best = at = 0
    for n in items:
        a, z = at + lead, at + lead + n
        for c in range(a // run, (z - 1) // run + 1):
            best = max(best, min(z, (c + 1) * run) - max(a, c * run))
        at = z
    return best, (6 if D == 64 else 3) if few else (8 if D == 64 else 4)


NEEDLES = 24


def fill(b, slope, seed):
    """Keys and values of every position. Keys have a part along (1, .., 1), as the queries do: scores rise by `slope` over the
    sequence. Where that is little, 24 positions a key/value head, anywhere, hold four fifths of the weight between them, so that
    none can be left out or taken twice without a difference far above the bar."""
    import torch
    g, rng = torch.Generator(device="cuda").manual_seed(seed), np.random.default_rng(seed)
    for s, n in enumerate(b.kv):
        p, i = b.where(s, np.arange(n))
        score = np.repeat(np.linspace(0, slope, n)[:, None], b.KV, 1)
        if slope < 60:
            for h in range(b.KV):
                score[rng.choice(n, NEEDLES, replace=False), h] = slope + np.log(n / max(slope, 1) / NEEDLES) + 1.5
        along = torch.from_numpy((score / (2 * b.D ** 0.5)).astype(np.float32)).cuda()[..., None]
        b.k[p, i] = (torch.randn(n, b.KV, b.D, generator=g, device="cuda") + along).to(b.k.dtype)
        b.v[p, i] = torch.randn(n, b.KV, b.D, generator=g, device="cuda").to(b.v.dtype)


def check_rows(b, x, out, H, cache, window, sinks, out_type=None, rows=96):
    """Up to `rows` rows of each sequence, the first and last among them, against the 64-bit form."""
    import torch
    half, out_half = ref.HALF[NP_TYPE[cache]], ref.HALF[NP_TYPE[out_type or cache]]
    G, scale = H // b.KV, b.D ** -0.5
    for s, (n, new) in enumerate(zip(b.kv, b.q)):
        if not new:
            continue
        at = np.unique(np.linspace(0, new - 1, min(new, rows)).round().astype(int))
        p, i = b.where(s, np.arange(n))
        k, v = b.k[p, i].double(), b.v[p, i].double()
        for part in np.array_split(at, -(-len(at) // 16)):
            r = torch.from_numpy(part + int(b.q_start[s])).cuda()
            pos = torch.from_numpy(n - new + part).cuda()[:, None]
            j = torch.arange(n, device="cuda")
            see = j <= pos
            if window:
                see &= (j > pos - window) | (j < sinks)
            q = x[r].double().view(len(part), b.KV, G, b.D)
            hidden = ~see[:, None, None]
            score = (torch.einsum("rhgd,jhd->rhgj", q, k) * scale).masked_fill(hidden, -float("inf"))
            big = (torch.einsum("rhgd,jhd->rhgj", q.abs(), k.abs()) * scale).masked_fill(hidden, 0).amax(-1, keepdim=True)
            w = score.sub(score.amax(-1, keepdim=True)).exp()
            w /= w.sum(-1, keepdim=True)
            want, mag = torch.einsum("rhgj,jhd->rhgd", w, v), torch.einsum("rhgj,jhd->rhgd", w, v.abs())
            flat = torch.einsum("rj,jhd->rhd", see.double(), v.abs())[:, :, None]
            rel = half + 2 * (b.D + 2) * 2.0 ** -24 * big + 2.0 ** -21 + (see.sum(1)[:, None, None, None] + 64) * 2.0 ** -23
            bar = out_half * want.abs() + mag * rel * 1.01 + (2.0 ** -25 * flat if cache == "f16" else 0) + (2.0 ** -25 if out_half == 2.0 ** -11 else 0)
            over = ((out[r].double().view_as(want) - want).abs() - bar).amax().item()
            assert over <= 0, (s, part, over)   # NaN fails too


STEADY = [  # sequences' lengths, new tokens, heads, kv_heads, hd, page, cache, window, sinks, layout, slope
    # few rows
    ([2000] * 64, [1] * 64, 32, 4, 128, 64, "bf16", 0, 0, "slots", 12),
    ([2000 - 13 * i for i in range(64)], [1] * 64, 32, 4, 64, 32, "f16", 0, 0, "heads", 60),
    ([20000, 19937, 17001], [1, 1, 1], 16, 4, 128, 48, "f16", 0, 0, "wide", 60),
    ([20000, 18003, 20001], [1, 2, 1], 8, 8, 64, 16, "bf16", 0, 0, "slots", 0),
    ([2111 - 31 * i for i in range(40)], [1] * 40, 16, 2, 256, 16, "bf16", 0, 0, "heads", 60),
    ([20000, 20000], [2, 1], 12, 2, 256, 64, "f16", 0, 0, "slots", 12),
    ([2000 - 7 * i for i in range(48)], [1 + i % 4 for i in range(48)], 32, 4, 128, 16, "f16", 0, 0, "slots", 60),   # 32 rows
    ([2000 - 7 * i for i in range(48)], [1 + i % 3 for i in range(48)], 40, 8, 64, 16, "bf16", 0, 0, "wide", 12),
    ([2500 - 11 * i for i in range(64)], [1] * 64, 32, 4, 128, 16, "bf16", 1500, 100, "heads", 60),
    ([2500 - 11 * i for i in range(64)], [1 + i % 2 for i in range(64)], 16, 4, 64, 48, "f16", 1501, 70, "slots", 0),
    ([20000, 20000], [1, 1], 16, 4, 256, 128, "bf16", 9000, 300, "slots", 12),
    # many rows
    ([2000, 1900, 2047, 1333], [300, 280, 300, 120], 32, 4, 128, 64, "bf16", 0, 0, "slots", 60),
    ([2000, 1900, 2047, 1333], [300, 1, 300, 120], 32, 4, 128, 16, "f16", 0, 0, "heads", 12),
    ([20000, 19001], [130, 70], 16, 2, 128, 48, "bf16", 0, 0, "slots", 60),
    ([2000, 1900, 2049, 1333], [400, 380, 300, 120], 32, 8, 64, 32, "f16", 0, 0, "wide", 60),
    ([20000], [500], 14, 2, 64, 64, "bf16", 0, 0, "slots", 12),
    ([2000, 1500, 2001], [200, 180, 120], 16, 4, 256, 16, "bf16", 0, 0, "heads", 60),
    ([20000], [150], 4, 1, 256, 128, "f16", 0, 0, "slots", 60),
    ([2500, 2300], [700, 650], 32, 4, 128, 32, "bf16", 1300, 200, "slots", 12),
    ([4000, 3900], [900, 800], 16, 4, 64, 16, "f16", 2000, 5, "heads", 60),
    ([3000, 2900], [300, 290], 8, 2, 256, 48, "f16", 1100, 130, "wide", 60),
    ([5000] + [1500] * 40, [400] + [1] * 40, 32, 4, 128, 64, "bf16", 0, 0, "slots", 60),   # a chunk beside single tokens
    ([5000] + [1500] * 40, [400] + [1] * 40, 16, 4, 64, 16, "f16", 0, 0, "slots", 12),
    ([4000] + [1500] * 20, [200] + [1] * 20, 8, 2, 256, 16, "bf16", 0, 0, "heads", 12),
]


@pytest.mark.parametrize("kv,q,H,KV,D,page,cache,window,sinks,layout,slope", STEADY)
def test_attention_long_runs(ctx, kv, q, H, KV, D, page, cache, window, sinks, layout, slope):
    import torch
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    tiles, stages = longest_stretch(kv, q, H, KV, D, max(q), window, sinks, sms)
    assert tiles > stages + 2, (tiles, stages)
    b = Batch(kv, q, KV, D, page, cache, seed=D + H, layout=layout)
    fill(b, slope, seed=D)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(b.T + 2, H, D, generator=g, device="cuda") + 2).to(dtype(cache))
    out = torch.full((b.T + 2, H, D), 77.0, dtype=dtype(cache), device="cuda")
    ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=max(q), window=window, sinks=sinks, out=out)
    ctx.status()
    check_rows(b, x, out, H, cache, window, sinks)
    assert (out[b.T:] == 77.0).all()
    for _ in range(3):
        assert torch.equal(ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=max(q), window=window, sinks=sinks)[:b.T], out[:b.T])
    wide = ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=max(q), window=window, sinks=sinks, out_dtype=torch.float32)
    ctx.status()
    check_rows(b, x, wide, H, cache, window, sinks, out_type="f32", rows=24)


@pytest.mark.parametrize("rows,vocab", [(24, 1000), (24, 4097), (24, 50304), (5, 151936), (1, 151936), (70, 20011)])
def test_sample_half_logits(ctx, rows, vocab):
    """fp16 logits: many ties, infinities of both signs where values overflow, NaN, odd strides and starts."""
    import torch
    rng = np.random.default_rng(vocab + rows)
    g = torch.Generator(device="cuda").manual_seed(vocab)
    lg = (2.5 * torch.randn(rows, vocab + 3, generator=g, device="cuda")).half()[:, 1:vocab + 1]
    lg[0, ::7] = float("nan")
    lg[0, 3::11] = -float("inf")
    if rows > 2:
        lg[1] = (lg[1].float() * 1e5).half()   # most overflow: those at +infinity share everything
        lg[2] *= 2.0 ** -14                    # subnormal
    u = [float(v) for v in rng.random(rows).astype(np.float32)]
    t = [float(v) for v in rng.choice([0.0, 0.5, 0.8, 1.0, 1.7], rows)]
    k = [int(v) for v in rng.choice([0, 1, 2, 40, 1000, vocab], rows)]
    p = [float(v) for v in rng.choice([0.1, 0.5, 0.9, 1.0], rows)]
    m = [float(v) for v in rng.choice([0.0, 0.01, 0.2], rows)]
    for kw in ({}, {"t": t}, {"k": k}, {"p": p}, {"m": m}, {"t": t, "k": k, "p": p, "m": m}):
        sample_check(ctx, lg, u, **kw)
