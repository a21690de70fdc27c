"""The refusals of the serving operators, without a GPU: the C entry points check their arguments before they look at the
context, so every refusal is reached with no context, and a call that they would take ends at "no context". The pointers are
never read. Also the plain 64-bit forms the GPU tests compare against, on known answers."""
import ctypes as C

import numpy as np
import pytest

import clutor_b200 as cb
from tests import serving_ref as ref

P = 1 << 20   # a 16-byte aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    from clutor_b200 import build
    build.build()
    return cb.lib()


def call(fn, *structs):
    err = C.create_string_buffer(512)
    rc = fn(None, *[C.byref(s) if s is not None else None for s in structs], None, err, 512)
    assert rc == 1
    return err.value.decode()


def kv(**kw):
    s = cb.KvStruct(P, P, cb.T_F16, 10, 64, 4, 128, 64 * 512, 512, 128, P, 8, 8, 2, P, P)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def qk(**kw):
    s = cb.QkStruct(5, 32, cb.T_F32, 3 * P, 4 * P, 5 * P, 4096, 512, 512, 2, P, P, 1e-6, P, 100, 0, 9 * P, 4096)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def attn(**kw):
    s = cb.AttnStruct(5, 32, 5, 3 * P, 4096, 9 * P, cb.T_F16, 4096, 0.1, 0, 0, 20 * P, 1 << 30)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def sampling(**kw):
    s = cb.SamplingStruct(3, 1000, cb.T_F32, P, 1000, P, None, None, None, None, P, None)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_good_calls_reach_the_context(L):
    assert call(L.clb200_qk_rope, kv(), qk()) == "no context"
    assert call(L.clb200_qk_rope, kv(type=cb.T_BF16), qk(src_type=cb.T_BF16, norm=0, q_norm=None, k_norm=None)) == "no context"
    assert call(L.clb200_attention, kv(), attn()) == "no context"
    assert call(L.clb200_attention, kv(page_size=48), attn(out_type=cb.T_F32, window=3, sinks=9)) == "no context"
    assert call(L.clb200_sample, sampling()) == "no context"
    assert call(L.clb200_sample, sampling(rows=0)) == "no context"


@pytest.mark.parametrize("bad,says", [
    ({"type": cb.T_F32}, "cache is F32"), ({"type": 77}, "unsupported"), ({"head_dim": 96}, "head_dim 96"),
    ({"page_size": 8}, "page_size 8"), ({"page_size": 40}, "page_size 40"), ({"page_size": 0}, "page_size 0"), ({"n_kv": 0}, "out of range"),
    ({"n_pages": 0}, "out of range"), ({"n_seq": -1}, "out of range"), ({"n_seq": 1 << 17}, "out of range"),
    ({"table_width": -1}, "out of range"), ({"table_stride": 7}, "out of range"), ({"table_width": (1 << 24) + 1, "table_stride": 1 << 25}, "2^30 positions"),
    ({"slot_stride": 100}, "strides"), ({"slot_stride": 516}, "strides"), ({"head_stride": 64}, "strides"), ({"page_stride": -8}, "strides"),
    ({"page_stride": 0}, "strides"), ({"k": None}, "missing"), ({"v": None}, "missing"), ({"q_start": None}, "missing"),
    ({"kv_len": None}, "missing"), ({"table": None}, "missing"), ({"k": P + 8}, "16-byte"), ({"v": P + 2}, "16-byte")])
def test_cache_refusals(L, bad, says):
    assert says in call(L.clb200_qk_rope, kv(**bad), qk())
    assert says in call(L.clb200_attention, kv(**bad), attn())


@pytest.mark.parametrize("bad,says", [
    ({"T": -1}, "out of range"), ({"n_head": 0}, "out of range"), ({"src_type": cb.T_BF16}, "cache's type"), ({"src_type": cb.T_Q8_0}, "cache's type"),
    ({"q": None}, "missing"), ({"out": None}, "missing"), ({"rope": None}, "missing"), ({"norm": 3}, "norm 3"), ({"norm": -1}, "norm -1"),
    ({"q_norm": None}, "weights"), ({"k_norm": None, "norm": 1}, "weights"), ({"pairs": 2}, "pairs 2"), ({"n_pos": 0}, "0 positions"),
    ({"q_stride": 4088}, "strides"), ({"k_stride": 516}, "strides"), ({"out_stride": 4100}, "strides"), ({"q": 3 * P + 4}, "16-byte"),
    ({"rope": P + 4}, "16-byte"), ({"out": 3 * P}, "overlaps"), ({"out": 3 * P + 16}, "overlaps"), ({"out": 4 * P - 4096}, "overlaps")])
def test_qk_rope_refusals(L, bad, says):
    assert says in call(L.clb200_qk_rope, kv(), qk(**bad))


@pytest.mark.parametrize("bad,says", [
    ({"T": -1}, "query heads"), ({"n_head": 30}, "query heads"), ({"n_head": 0}, "query heads"), ({"n_head": 68, "q_stride": 1 << 14, "out_stride": 1 << 14}, "query heads"),
    ({"max_q": -1}, "max_q"), ({"out_type": cb.T_BF16}, "out is BF16"), ({"q": None}, "missing"), ({"out": None}, "missing"),
    ({"scale": 0.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"scale": -1.0}, "scale"),
    ({"window": -1}, "window"), ({"sinks": -1}, "sinks"), ({"q_stride": 4088}, "strides"), ({"out_stride": 4097}, "strides"),
    ({"q": 3 * P + 8}, "16-byte"), ({"out": 3 * P + 4096 * 8}, "overlaps")])
def test_attention_refusals(L, bad, says):
    assert says in call(L.clb200_attention, kv(), attn(**bad))


@pytest.mark.parametrize("bad,says", [
    ({"rows": -1}, "-1 rows"), ({"vocab": 0}, "0 logits"), ({"vocab": (1 << 18) + 1, "stride": 1 << 19}, "logits"), ({"type": cb.T_Q4_K}, "F32, F16 or BF16"),
    ({"logits": None}, "missing"), ({"u": None}, "missing"), ({"token": None}, "missing"), ({"stride": 999}, "999 elements"),
    ({"logits": P + 2}, "boundary"), ({"logits": P + 1, "type": cb.T_F16}, "boundary")])
def test_sample_refusals(L, bad, says):
    assert says in call(L.clb200_sample, sampling(**bad))


def test_missing_structs(L):
    assert "no cache" in call(L.clb200_qk_rope, None, qk())
    assert "no cache" in call(L.clb200_attention, kv(), None)
    assert "no arguments" in call(L.clb200_sample, None)


def test_plain_sample_known_answers():
    x = np.log([0.1, 0.4, 0.2, 0.3])
    assert [ref.sample(x, u)[0] for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert ref.sample(x, 0.5, top_k=2) == (1, pytest.approx(4 / 7))
    assert ref.sample(x, 0.6, top_k=2)[0] == 3
    assert ref.sample(x, 0.99, top_p=0.65) == (3, pytest.approx(3 / 7))     # 0.4 + 0.3 reaches 0.65
    assert ref.sample(x, 0.99, top_p=0.75)[0] == 3 and ref.sample(x, 0.6, top_p=0.75) == (2, pytest.approx(2 / 9))
    assert ref.sample(x, 0.99, min_p=0.6)[0] == 3                           # 0.3 / 0.4 stays, 0.2 / 0.4 goes
    assert ref.sample(x, 0.3, temperature=0.0) == (1, 1.0)
    assert ref.sample([0.0, 0.0, 0.0, 0.0], 0.6, top_k=2) == (1, 0.5)       # ties: the lowest ids
    assert ref.sample([np.nan, -np.inf], 0.5) == (-1, 0.0)
    assert ref.sample([0.0, np.inf, np.nan, np.inf], 0.5) == (3, 0.5)


def test_plain_attention_known_answers():
    k = np.eye(3)[:, None, :] * 0
    v = np.array([[1.0, 0, 0], [0, 2.0, 0], [0, 0, 4.0]])[:, None, :]
    q = np.ones((2, 3))
    assert np.allclose(ref.attention(q, k, v, 2, 1.0, 0, 0)[0], [[1 / 3, 2 / 3, 4 / 3]] * 2)
    assert np.allclose(ref.attention(q, k, v, 1, 1.0, 0, 0)[0], [[0.5, 1, 0]] * 2)
    assert np.allclose(ref.attention(q, k, v, 2, 1.0, 1, 1)[0], [[0.5, 0, 2]] * 2)
    assert np.allclose(ref.attention(q, k, v, -1, 1.0, 0, 0)[0], 0)


def test_plain_rotation_known_answers():
    x = np.array([[3.0, 4.0, 0.0, 0.0]])
    y, _ = ref.qk_rope(x, None, np.array([0.0, 1.0, 1.0, 0.0]), 0, False, 0)
    assert np.allclose(y, [[0, 4, 3, 0]])            # the pair (0, 2) by a right angle, (1, 3) not
    y, _ = ref.qk_rope(x, None, np.array([0.0, 1.0, 1.0, 0.0]), 0, True, 0)
    assert np.allclose(y, [[-4, 3, 0, 0]])           # the pair (0, 1)
    y, _ = ref.qk_rope(x, np.full(4, 2.0), np.array([1.0, 1.0, 0.0, 0.0]), 2, False, 0)
    assert np.allclose(y, np.array([[3, 4, 0, 0]]) / 2.5 * 2)


def test_packed_layouts_equal_the_structs():
    """The byte layouts that the Python calls pack are those of the C structs, field for field."""
    for S, layout in ((cb.KvStruct, cb._KV), (cb.QkStruct, cb._QK), (cb.AttnStruct, cb._ATTN), (cb.SamplingStruct, cb._SAMPLING)):
        assert C.sizeof(S) == layout.size
        values = [float(i + 1) if t is C.c_float else i + 1 for i, (_, t) in enumerate(S._fields_)]
        buf = C.create_string_buffer(layout.size)
        layout.pack_into(buf, 0, *values)
        assert [getattr(S.from_buffer_copy(buf), f) for f, _ in S._fields_] == values
