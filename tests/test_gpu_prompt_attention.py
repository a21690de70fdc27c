"""CLB200_OPT_PROMPT_ATTENTION seen through one layer whose output is its attention: the experts' down matrices are zero, and every
matrix is Q6_K, whose values are even about zero, so that no common part hides what the positions contribute. The logits are then the
output matrix times the normed sum of the embedding and the O product of the attention.

Bar. The attention itself differs by the rounding of queries and probabilities to fp16: scores of a standard deviation of a few move by
2^-12 of it each, so the output by about d = 7e-4 of its root mean square. Two products take that in 8 bits (the O product and the output
matrix). A value that differs by d falls into another step of s with probability d / s, and then differs by s, so the squares' mean is
s d; s is 1 / 127 of the largest of 256 normal values, 4 root mean squares at most: 0.0315. The two together: sqrt(2 s d) = 6.6e-3.
BAR is three times that.

What one position contributes is then checked by itself: the change of the logits when its token is replaced, of those tokens that change
the default path's logits by 6e-2 at least. Each of the two runs is off by BAR at most, so the change by sqrt(2) BAR / 6e-2 = 0.47 of it;
a position that is not seen, or seen in another's place, gives a difference of about 1."""
import numpy as np
import pytest

from clutor_b200 import gguf
from clutor_b200 import synth_model as sm

pytestmark = pytest.mark.gpu

BAR, LEAST = 2e-2, 6e-2
Q6 = dict(n_layer=1, embd_type=sm.T_Q6_K, q_type=sm.T_Q6_K, k_type=sm.T_Q6_K, o_type=sm.T_Q6_K)
SHAPES = {
    "qwen3moe": sm.tiny(**Q6),
    "qwen3moe_gqa8": sm.tiny(E=512, n_head=8, n_kv=1, hd=128, FF=512, NE=16, K=4, **Q6),
    "qwen3moe_hd64_gqa16": sm.tiny(E=512, n_head=16, n_kv=1, hd=64, FF=256, NE=32, K=8, **Q6),
    "olmoe": sm.tiny(arch="olmoe", n_head=2, n_kv=2, hd=128, **Q6),
    "granitemoe": sm.tiny(arch="granitemoe", n_head=2, n_kv=1, hd=128, **Q6),
}


def image(spec):
    w = sm.writer(spec, seed=5)
    if spec.arch == "granitemoe":   # no norm of queries and keys: the scores' standard deviation by the scale
        w.add("granitemoe.attention.scale", gguf.F32, 1e-5)
    for t in w.tensors:
        if t.name.endswith("ffn_down_exps.weight"):
            raw = np.asarray(t.data()).copy()
            raw.reshape(-1, 210)[:, 208:] = 0
            t.data = raw
    return w.image()


@pytest.fixture(scope="module")
def ctx():
    import clutor_b200 as cb
    c = cb.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("name", sorted(SHAPES))
@pytest.mark.parametrize("n,batch", [(2, 64), (66, 64), (130, 64), (200, 100), (333, 512)])
def test_every_position_contributes_what_it_should(ctx, name, n, batch):
    from clutor_b200.model import Model
    m = Model(ctx, image(SHAPES[name]), 400)   # 400: the cache's last page is not a whole one
    prompt = np.random.default_rng(n).integers(0, m.n_vocab, n).astype(np.int32)

    def run(tokens, option):
        ctx.set_option(ctx.OPT_PROMPT_ATTENTION, option)
        m.reset()
        return m.prefill(tokens).astype(np.float64)

    ctx.set_exact(True)
    try:
        m.set_batch(batch)
        want, got = run(prompt, 0), run(prompt, 1)
        size = np.linalg.norm(want)
        assert np.linalg.norm(got - want) <= BAR * size
        tried = 0
        for j in sorted({0, min(63, n - 2), min(64, n - 2), n // 2 - 1, n - 2}):
            most, other = 0.0, prompt
            for t in range(0, m.n_vocab, 8):   # the token that changes the default path's logits most
                p = prompt.copy()
                p[j] = t
                d = np.linalg.norm(run(p, 0) - want)
                if d > most:
                    most, other = d, p
            if most < LEAST * size:
                continue
            tried += 1
            change, seen = run(other, 0) - want, run(other, 1) - got
            assert np.linalg.norm(seen - change) <= 0.5 * np.linalg.norm(change), j
        assert tried >= 1
    finally:
        ctx.set_option(ctx.OPT_PROMPT_ATTENTION, 0)
        ctx.set_exact(False)
        m.close()
