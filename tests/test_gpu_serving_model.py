"""The serving operators on a whole model's own path (a B200): the prompt's attention through clb200_qk_rope and
clb200_attention (CLB200_OPT_PROMPT_ATTENTION), and sampled generation (clb200_model_generate_sampled).

Bars. Prompt attention: against the same model's default attention on the integer path. Queries and probabilities are rounded to
half precision (2^-11 each); that alone is small, but every product after it takes its activations in 8 bits, where any
difference can move a value by one step, 1 / 127 of its block's largest. For normal values of 256 the largest is about 3 times
the root mean square (below 3.5), so one quantization can turn a small difference into at most 3.5 / 127 = 2.8e-2 relative L2,
and a layer has four (attention output, normed x, the experts' hidden values, the next norm): 0.11 a layer. The operators
themselves are held to their own bars in test_gpu_serving.py; this one tells a path that is wired up right (measured: up to
2.9e-2 over two or three layers) from one that is not (a mask or a page off gives differences of the logits' own size).
Sampled generation: the tokens are those of the plain 64-bit sampler on the logits of the same steps, exactly.
"""
import numpy as np
import pytest

from clutor_b200 import synth_model as sm
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

SHAPES = {
    "qwen3moe": sm.tiny(),
    "qwen3moe_gqa8": sm.tiny(n_layer=3, E=512, n_head=8, n_kv=1, hd=128, FF=512, NE=16, K=4, down_type=sm.T_Q4_K),
    "qwen3moe_hd64_gqa16": sm.tiny(E=512, n_head=16, n_kv=1, hd=64, FF=256, NE=32, K=8),
    "olmoe": sm.tiny(arch="olmoe", n_head=2, n_kv=2, hd=128),
    "granitemoe": sm.tiny(arch="granitemoe", n_head=2, n_kv=1, hd=128),
}


@pytest.fixture(scope="module")
def ctx():
    import clutor_b200 as cb
    c = cb.Context(0)
    yield c
    c.close()


def rel_l2(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


@pytest.mark.parametrize("name", sorted(SHAPES))
@pytest.mark.parametrize("n,batch", [(2, 64), (100, 16), (130, 64), (333, 512)])
def test_prompt_attention(ctx, name, n, batch):
    from clutor_b200.model import Model
    spec = SHAPES[name]
    m = Model(ctx, sm.image(spec, seed=5), 400)   # 400: the cache's last page is not a whole one
    prompt = np.random.default_rng(n).integers(0, m.n_vocab, n).astype(np.int32)
    ctx.set_exact(True)
    try:
        m.set_batch(batch)
        want = m.prefill(prompt)
        after_want = [m.step(int(t))[0] for t in prompt[:3]]
        m.reset()
        ctx.set_option(ctx.OPT_PROMPT_ATTENTION, 1)
        got = m.prefill(prompt)
        again = [m.step(int(t))[0] for t in prompt[:3]]
        m.reset()
        assert np.array_equal(m.prefill(prompt), got)   # the same bits again
        ctx.set_option(ctx.OPT_PROMPT_ATTENTION, 0)
        m.reset()
        assert np.array_equal(m.prefill(prompt), want)  # the default is untouched
        bar = 0.11 * m.n_layer
        assert rel_l2(got, want) <= bar
        for a, b in zip(again, after_want):
            assert rel_l2(a, b) <= bar
    finally:
        ctx.set_option(ctx.OPT_PROMPT_ATTENTION, 0)
        ctx.set_exact(False)
        m.close()


def test_prompt_attention_option_values(ctx):
    import clutor_b200 as cb
    for v in (-1, 2):
        with pytest.raises(cb.ClutorError):
            ctx.set_option(ctx.OPT_PROMPT_ATTENTION, v)


@pytest.mark.parametrize("how", [dict(temperature=0.0), dict(top_k=1), dict(temperature=0.7, top_k=40, top_p=0.9, min_p=0.02),
                                 dict(temperature=1.5), dict(top_p=0.5)])
def test_generate_sampled(ctx, how):
    from clutor_b200.model import Model
    m = Model(ctx, sm.image(SHAPES["qwen3moe"], seed=5), 64)
    try:
        n = 12
        u = np.random.default_rng(3).random(n).astype(np.float32)
        tokens, probs = m.generate_sampled(7, n, u, **how)
        assert m.pos == n and m.tokens(0, n) == tokens
        m.reset()
        cur = 7
        for i in range(n):
            lg, greedy, _ = m.step(cur)
            want, p = ref.sample(lg, u[i], **{k: float(np.float32(v)) if k != "top_k" else v for k, v in how.items()})
            assert tokens[i] == want and abs(probs[i] - p) <= 2.0 ** -23 * p
            if how in (dict(temperature=0.0), dict(top_k=1)):
                assert want == greedy
            cur = want
        if how == dict(temperature=0.0):
            m.reset()
            assert m.generate(7, n) == tokens
    finally:
        m.close()


def test_generate_sampled_refusals(ctx):
    import clutor_b200 as cb
    from clutor_b200.model import Model
    m = Model(ctx, sm.image(SHAPES["qwen3moe"], seed=5), 16)
    try:
        for token, n in ((-1, 2), (m.n_vocab, 2), (3, 17)):
            with pytest.raises(cb.ClutorError):
                m.generate_sampled(token, n, np.zeros(n, np.float32))
        with pytest.raises(cb.ClutorError):
            m.generate_sampled(3, 2, np.zeros(3, np.float32))
        assert m.pos == 0 and m.generate_sampled(3, 0, np.zeros(0, np.float32)) == ([], [])
        assert len(m.generate_sampled(3, 16, np.full(16, 0.5, np.float32))[0]) == 16
    finally:
        m.close()
