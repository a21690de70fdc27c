"""clb200_qk_rope where a warp takes a token (many tokens) and where a token's heads take several rounds of loads (wide rows), against
the 64-bit form on the device.

The bar is test_gpu_serving.py's: half a step of the cache's type, and 40 fp32 roundings (2^-24 each) of a term. A norm over the whole row
adds the squares of a lane's share one after another: n = heads * head_dim / lanes additions, each off by 2^-24 of a sum that only grows,
so n 2^-24 of the mean of squares and half of that of its root."""
import numpy as np
import pytest

from tests import serving_ref as ref
from tests.test_gpu_serving import NP_TYPE, Batch, dtype

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import clutor_b200 as cb
    c = cb.Context(0)
    yield c
    c.status()
    c.close()


def turned(x, w, cs, norm, pairs, eps):
    """x [T, heads, hd] and cs [T, hd] in 64 bits -> (y, a bound on |terms of y|)."""
    import torch
    D = x.shape[-1]
    if norm == 2:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    elif norm == 1:
        x = x / (x.square().mean((-1, -2), keepdim=True) + eps).sqrt() * w.view(x.shape[1:])
    c, s = cs[:, None, :D // 2], cs[:, None, D // 2:]
    a, b = (x[..., 0::2], x[..., 1::2]) if pairs else (x[..., :D // 2], x[..., D // 2:])
    re, im, mag = a * c - b * s, a * s + b * c, a.abs() + b.abs()
    if pairs:
        return torch.stack([re, im], -1).flatten(-2), mag.repeat_interleave(2, -1)
    return torch.cat([re, im], -1), torch.cat([mag, mag], -1)


MANY = [700, 0, 1, 900, 37, 400]       # 2038 new tokens: a warp a token
FEW = [3, 1, 0, 5]
CASES = [  # new tokens, heads, kv_heads, hd, page, src, cache, norm, pairs, layout
    (MANY, 64, 4, 128, 64, "bf16", "bf16", 2, False, "slots"),
    (MANY, 32, 4, 128, 16, "f32", "f16", 2, True, "heads"),
    (MANY, 16, 16, 128, 32, "f32", "bf16", 1, False, "slots"),
    (MANY, 33, 11, 64, 48, "f16", "f16", 1, True, "wide"),
    (MANY, 24, 8, 64, 16, "f32", "f16", 0, False, "slots"),
    (MANY, 9, 3, 256, 128, "bf16", "bf16", 2, False, "wide"),
    (MANY, 5, 5, 256, 16, "f16", "f16", 1, False, "heads"),
    (MANY, 1, 1, 64, 64, "f32", "bf16", 2, True, "slots"),
    (FEW, 40, 20, 256, 16, "f32", "f16", 1, False, "slots"),     # a CTA a token: two rounds of loads and more
    (FEW, 200, 100, 64, 32, "bf16", "bf16", 2, True, "heads"),
    (FEW, 72, 36, 256, 16, "f16", "f16", 1, True, "wide"),
    (FEW, 120, 60, 128, 16, "f32", "bf16", 0, False, "slots"),
    (FEW, 120, 60, 128, 64, "f32", "bf16", 1, False, "heads"),
]


@pytest.mark.parametrize("new,H,KV,D,page,src,cache,norm,pairs,layout", CASES)
def test_qk_rope_many(ctx, new, H, KV, D, page, src, cache, norm, pairs, layout):
    import torch
    kv = [n + 13 * i for i, n in enumerate(new)]
    b = Batch(kv, new, KV, D, page, cache, seed=H + D, layout=layout)
    g = torch.Generator(device="cuda").manual_seed(11)
    T, pad = b.T, 9   # rows behind the last sequence
    qkv = (1.5 * torch.randn(T + pad, H + 2 * KV, D, generator=g, device="cuda")).to(dtype(src))
    qkv[T:] = float("nan")
    x, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    qn, kn = (1 + 0.3 * torch.randn(n * D if norm == 1 else D, generator=g, device="cuda") for n in (H, KV))
    angle = np.arange(max(kv))[:, None] * 1e4 ** (-np.arange(D // 2) * 2 / D)
    rope = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)).cuda()
    out = torch.full((T + pad, H, D), 77.0, dtype=dtype(cache), device="cuda")
    before = b.pool.clone()
    ctx.qk_rope(x, k, v, b.pages, b.q_start_d, b.kv_len_d, rope, q_norm=qn if norm else None, k_norm=kn if norm else None, norm=norm,
                pairs=pairs, eps=1e-5, out=out)
    ctx.status()
    where = ref.positions(b.q_start, kv)
    pos = torch.tensor([p for _, _, p in where], device="cuda")
    page_at = torch.tensor([int(b.np_table[s][p // page]) for _, s, p in where], device="cuda")
    cs = rope[pos].double()
    half, tiny = ref.HALF[NP_TYPE[cache]], 2.0 ** -25 if cache == "f16" else 0.0

    def check(got, src, w, heads):
        y, mag = turned(src[:T].double(), w.double(), cs, norm, pairs, 1e-5)
        roundings = 40 + (heads * D / 64 if norm == 1 else 0)
        assert ((got.double() - y).abs() <= half * y.abs() + roundings * 2.0 ** -24 * mag + tiny).all()

    check(out[:T], x, qn, H)
    gk = b.k[page_at, pos % page]
    check(gk, k, kn, KV)
    assert torch.equal(b.v[page_at, pos % page], v[:T].to(dtype(cache)))
    assert (out[T:] == 77.0).all()
    # nothing but the new tokens' slots was written
    after = b.pool.clone()
    b.pool.copy_(before)
    b.k[page_at, pos % page], b.v[page_at, pos % page] = gk, v[:T].to(dtype(cache))
    assert torch.equal(b.pool.view(torch.int16), after.view(torch.int16))


def test_bad_positions_where_a_warp_takes_a_token(ctx):
    """Positions past the rotary table and pages out of range: those tokens are skipped and reported, the others are as ever."""
    import torch

    import clutor_b200 as cb
    H, KV, D = 6, 2, 128
    b = Batch([1000, 1000], [1000, 1000], KV, D, 16, "bf16", seed=3)
    x = torch.randn(b.T, H + 2 * KV, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    args = (x[:, :H], x[:, H:H + KV], x[:, H + KV:], b.pages, b.q_start_d, b.kv_len_d)
    rope = torch.randn(1000, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    good = ctx.qk_rope(*args, rope, norm=0)
    ctx.status()
    stored = b.pool.clone()
    out = torch.full_like(good, 9.0)
    b.pool.fill_(5.0)
    ctx.qk_rope(*args, rope[:990], norm=0, out=out)
    with pytest.raises(cb.ClutorError, match="rows"):
        ctx.status()
    late = torch.arange(b.T, device="cuda") % 1000 >= 990
    assert torch.equal(out[~late], good[~late]) and (out[late] == 9.0).all()
    keep = b.pages.table[1, 7].clone()
    b.pages.table[1, 7] = b.pages.n_pages
    b.pool.fill_(5.0)
    ctx.qk_rope(*args, rope, norm=0, out=out)
    with pytest.raises(cb.ClutorError, match="page"):
        ctx.status()
    assert torch.equal(out, good)   # the queries do not hang on the page
    lost = int(keep)
    assert (b.k[lost] == 5.0).all() and (b.v[lost] == 5.0).all()
    b.k[lost], b.v[lost] = stored[0][lost], stored[1][lost]
    used = torch.from_numpy(np.unique(b.np_table[b.np_table < b.pages.n_pages])).long().cuda()
    rows = stored[:, used] == stored[:, used]   # slots that hold a token (the others were NaN)
    assert torch.equal(b.pool[:, used][rows], stored[:, used][rows])
    ctx.status()
