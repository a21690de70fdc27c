"""A sliding window's cache: pages that no new token sees any more have been given back, so their ids name nothing and what they held is
another's. And a program whose first serving calls are captured."""
import os
import subprocess
import sys

import numpy as np
import pytest

from tests.test_gpu_serving import Batch, attn_check, dtype

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ctx():
    import clutor_b200 as cb
    c = cb.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("gone", [-1, 10 ** 9, None])
@pytest.mark.parametrize("kv,q,H,KV,D,page,cache,window,sinks", [
    ([900, 333, 20], [1, 1, 1], 16, 2, 128, 16, "bf16", 64, 0),
    ([900, 333, 70], [1, 2, 1], 8, 2, 64, 48, "f16", 37, 5),
    ([901, 340], [1, 1], 8, 1, 256, 16, "bf16", 100, 17),
    ([900, 333, 70], [130, 33, 70], 16, 2, 128, 16, "bf16", 64, 0),
    ([905, 500], [40, 1], 16, 4, 64, 32, "f16", 33, 40),
    ([700, 333], [20, 90], 8, 1, 256, 16, "bf16", 50, 3),
    ([3000], [5], 16, 1, 128, 16, "f16", 200, 100),
])
def test_pages_outside_the_window_are_not_looked_at(ctx, kv, q, H, KV, D, page, cache, window, sinks, gone):
    import torch
    b = Batch(kv, q, KV, D, page, cache, seed=D + page)
    b.fill(5)
    whole = [b.cache_of(s) for s in range(len(kv))]
    for s, (n, new) in enumerate(zip(kv, q)):
        first = n - new - window + 1          # the lowest position that the first new token sees
        for p in range(-(-sinks // page), max(first, 0) // page):
            at = int(b.np_table[s, p])
            b.k[at], b.v[at] = float("nan"), float("nan")
            if gone is not None:
                b.pages.table[s, p] = gone
    x = (2 * torch.randn(b.T, H, D, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")).to(dtype(cache))
    out = ctx.attention(x, b.pages, b.q_start_d, b.kv_len_d, max_q=max(q), window=window, sinks=sinks)
    ctx.status()
    b.cache_of = lambda s: whole[s]
    attn_check(b, x, out, H, cache, window, sinks, D ** -0.5)


FIRST = """
import torch, clutor_b200 as cb
ctx = cb.Context(0)
H, KV, D, q = 8, 2, 128, {q}
pool = torch.randn(2, 9, 16, KV, D, device="cuda").half()
pages = cb.KvPages(pool[0], pool[1], torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8))
qkv = torch.randn(q, H + 2 * KV, D, device="cuda")
ends, kv = torch.tensor([0, q], dtype=torch.int32, device="cuda"), torch.tensor([100], dtype=torch.int32, device="cuda")
rope, u = torch.randn(128, D, device="cuda"), torch.rand(q, device="cuda")
def step():
    t = ctx.qk_rope(qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:], pages, ends, kv, rope, norm=0)
    o = ctx.attention(t, pages, ends, kv, max_q=q, out_dtype=torch.float32)
    return (t, o, *ctx.sample(o.view(q, -1), u, top_k=torch.full((q,), 9, dtype=torch.int32, device="cuda")))
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
ctx.status()
for a, b in zip(got, step()):
    assert torch.equal(a, b)
ctx.status()
print("equal")
"""


@pytest.mark.parametrize("q", [1, 40])
def test_first_calls_of_a_program_captured(q):
    r = subprocess.run([sys.executable, "-c", FIRST.format(q=q)], cwd=ROOT, capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and "equal" in r.stdout, r.stderr[-2000:]
