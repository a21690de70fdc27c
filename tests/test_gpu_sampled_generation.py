"""Sampled generation on a model whose logits leave nothing to draw from, and on one with more tokens than the sampling takes."""
import numpy as np
import pytest

from clutor_b200 import synth_model as sm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import clutor_b200 as cb
    c = cb.Context(0)
    yield c
    c.status()
    c.close()


def blocks_scaled_by(monkeypatch, spec, half):
    """The output matrix's fp16 block scales (the last two bytes of a Q6_K block) become `half`."""
    quant = sm._quant

    def scaled(type_, rows, cols, *rest):
        raw = quant(type_, rows, cols, *rest).copy()
        if rows == spec.vocab and type_ == spec.out_type:
            raw.reshape(-1, 210)[:, 208:] = np.array([half], np.float16).view(np.uint8)
        return raw

    monkeypatch.setattr(sm, "_quant", scaled)


@pytest.mark.parametrize("n", [1, 2, 7])
@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_nothing_to_draw_from_is_an_error(ctx, monkeypatch, n, temperature):
    """Every logit NaN: whichever step it is, the last one too, the call says so and the position stays."""
    import clutor_b200 as cb
    from clutor_b200.model import Model
    spec = sm.tiny()
    blocks_scaled_by(monkeypatch, spec, np.nan)
    m = Model(ctx, sm.image(spec, seed=5), 32)
    try:
        assert np.isnan(m.step(3)[0]).all() and m.pos == 1
        for _ in range(2):
            with pytest.raises(cb.ClutorError, match="step 0 .* no logit above -infinity"):
                m.generate_sampled(3, n, np.full(n, 0.5, np.float32), temperature=temperature)
            assert m.pos == 1
    finally:
        m.close()


def test_too_many_tokens_are_refused_before_a_step(ctx):
    import clutor_b200 as cb
    from clutor_b200.model import Model
    m = Model(ctx, sm.image(sm.tiny(vocab=(1 << 18) + 256), seed=5, fast=True), 16)
    try:
        want = m.step(7)[0]
        m.reset()
        for _ in range(3):
            with pytest.raises(cb.ClutorError, match="logits a row"):
                m.generate_sampled(9, 2, np.full(2, 0.5, np.float32))
            assert m.pos == 0
        # no step of the refused calls is on its way: the device's state is the next step's own
        assert np.array_equal(m.step(7)[0], want) and m.tokens(0, 1) == [int(want.argmax())]
    finally:
        m.close()
