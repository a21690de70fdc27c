"""The Python side of the serving calls without a GPU: what it packs for the C entry points and what it refuses. The tensors are
stand-ins that have a layout and an address on a device, and no memory; nothing reads the addresses."""
import ctypes as C

import pytest
import torch

import clutor_b200 as cb

P = 1 << 20   # a 16-byte aligned address


class Laid:
    """A tensor's layout: that of `like`, a CPU or meta tensor, said to lie on cuda:`at`."""

    def __init__(self, like, at=0):
        self.like, self.at, self.dtype, self.shape, self.device = like, at, like.dtype, like.shape, torch.device("cuda", max(at, 0))

    def __getattr__(self, name):   # stride, dim, numel, is_contiguous
        return getattr(self.like, name)

    def get_device(self):
        return self.at

    def data_ptr(self):
        return P


def ids(*shape):
    return torch.zeros(shape, dtype=torch.int32, device="meta")


def pages(table, n_pages=9, page=16, KV=2, D=64, dt=torch.float16):
    kv = Laid(torch.empty(n_pages, page, KV, D, dtype=dt, device="meta"))
    return cb.KvPages(kv, kv, Laid(table))


class Library:
    """Stands in for the library under a Context on device `at`: keeps the structs that the serving calls pass."""

    def __init__(self, at=0):
        self.at, self.calls, self.opened = at, [], []

    def context(self, device=0):
        self.opened.append(cb.Context(device))
        return self.opened[-1]

    def clb200_open(self, device, err, n):
        return device + 10 if device >= 0 else 5   # the handle: 5 for the current device

    def clb200_device(self, handle):
        return self.at if handle == 5 else handle - 10

    def clb200_close(self, handle):
        pass

    def clb200_attention_work(self, handle, kv, a):
        return 0

    def _take(self, what, *at):
        self.calls.append([S.from_buffer_copy(C.string_at(p, C.sizeof(S))) for S, p in zip(what, at)])
        return 0

    def clb200_qk_rope(self, handle, kv, a, stream, err, n):
        return self._take((cb.KvStruct, cb.QkStruct), kv, a)

    def clb200_attention(self, handle, kv, a, stream, err, n):
        return self._take((cb.KvStruct, cb.AttnStruct), kv, a)

    def clb200_sample(self, handle, a, stream, err, n):
        return self._take((cb.SamplingStruct,), a)


class Stream:
    cuda_stream = 7


@pytest.fixture
def library(monkeypatch):
    """A stand-in for the library, under every Context that the test opens."""
    made = Library()
    monkeypatch.setattr(cb, "lib", lambda: made)
    yield made
    for c in made.opened:
        c.handle = None   # nothing for the real library to close


def passed(library, p):
    """The clb200_kv that a call on the pages p passes."""
    n = p.table.shape[0]
    q = Laid(torch.empty(3, 4, p.head_dim, dtype=p.dtype, device="meta"))
    library.context().attention(q, p, Laid(ids(n + 1)), Laid(ids(n)), out=q, stream=Stream)
    return library.calls[-1][0]


@pytest.mark.parametrize("table,stride", [(ids(8, 5), 5), (ids(8, 7)[:, :5], 7), (ids(1, 5), 5), (ids(1, 7)[:, :5], 7), (ids(1, 5).expand(1, 5), 5),
                                          (ids(5).as_strided((1, 5), (2, 1)), 5), (ids(4, 1), 1), (ids(3, 0), 1), (ids(0, 4), 4)])
def test_table_rows_apart(library, table, stride):
    s = passed(library, pages(table))
    assert (s.n_seq, s.table_width, s.table_stride) == (*table.shape, stride)


@pytest.mark.parametrize("table", [ids(1, 5).expand(8, 5), ids(1, 1).expand(3, 1), ids(20).as_strided((4, 5), (3, 1)),
                                   ids(20).as_strided((2, 5), (4, 1)), ids(5).as_strided((2, 5), (0, 1))])
def test_table_rows_that_share_memory_are_refused(table):
    """A row of the table is read table_width ids from table_stride ids behind the row before: rows nearer to one another would be
    read where the table does not reach."""
    with pytest.raises(cb.ClutorError, match="rows of table"):
        pages(table)


def sample_tensors(R, V):
    f = Laid(torch.empty(R, device="meta"))
    return Laid(torch.empty(R, V, device="meta")), f, Laid(ids(R)), f


def test_calls_of_two_threads_keep_their_own_arguments(library, monkeypatch):
    """The library runs without Python's lock, so a second call may be prepared while it does: a call's arguments stay as they are
    until it returns. The second call is made here from inside the first one's."""
    ctx = library.context()
    kv = pages(ids(2, 5))
    q = Laid(torch.empty(3, 4, 64, dtype=torch.float16, device="meta"))
    kw = dict(out=q, stream=Stream)
    ends = Laid(ids(3)), Laid(ids(2))
    rope = Laid(torch.empty(30, 64, device="meta"))
    k = Laid(torch.empty(3, 2, 64, dtype=torch.float16, device="meta"))
    calls = [lambda: ctx.attention(q, kv, *ends, scale=0.5, window=9, **kw), lambda: ctx.attention(q, pages(ids(2, 3)), *ends, max_q=2, **kw),
             lambda: ctx.qk_rope(q, k, k, kv, *ends, rope, norm=0, pairs=True, **kw),
             lambda: ctx.qk_rope(q, k, k, pages(ids(2, 8)), *ends, rope, norm=0, eps=0.5, **kw),
             *(lambda R=R: ctx.sample(*sample_tensors(R, 100)[:2], token=sample_tensors(R, 100)[2], prob=sample_tensors(R, 100)[3], stream=Stream)
               for R in (3, 5))]
    alone = []
    for call in calls:
        call()
        alone.append([bytes(s) for s in library.calls[-1]])
    for i, outer in enumerate(calls):
        for inner in calls:
            take, depth = Library._take, [0]

            def nested(self, what, *at):
                depth[0] += 1
                if depth[0] == 1:
                    inner()
                return take(self, what, *at)   # the outer call's arguments, read after the inner call

            monkeypatch.setattr(Library, "_take", nested)
            outer()
            monkeypatch.setattr(Library, "_take", take)
            assert [bytes(s) for s in library.calls[-1]] == alone[i]


def test_refusals_are_the_frameworks_own(library):
    """Tensors of another rank and numbers that no C argument holds raise what every other refusal raises."""
    ctx, kv = library.context(), pages(ids(2, 5))
    q, k, rope = (Laid(torch.empty(*s, dtype=d, device="meta")) for s, d in
                  (((3, 4, 64), torch.float16), ((3, 2, 64), torch.float16), ((30, 64), torch.float32)))
    flat, ends = Laid(torch.empty(3, 256, dtype=torch.float16, device="meta")), (Laid(ids(3)), Laid(ids(2)))
    kw = dict(out=q, stream=Stream)
    x, u, token, prob = sample_tensors(3, 100)
    cases = [lambda: ctx.attention(flat, kv, *ends, **kw), lambda: ctx.attention(q, kv, *ends, out=flat, stream=Stream),
             lambda: ctx.attention(q, kv, *ends, window=1 << 31, **kw), lambda: ctx.attention(q, kv, *ends, sinks=1 << 40, **kw),
             lambda: ctx.attention(q, kv, *ends, max_q=1 << 31, **kw),
             lambda: ctx.qk_rope(flat, k, k, kv, *ends, rope, norm=0, **kw), lambda: ctx.qk_rope(q, flat, k, kv, *ends, rope, norm=0, **kw),
             lambda: ctx.qk_rope(q, k, k, kv, *ends, u, norm=0, **kw),
             lambda: ctx.sample(u, u, token=token, prob=prob, stream=Stream), lambda: ctx.sample(rope, u, token=x, prob=prob, stream=Stream),
             lambda: ctx.sample(Laid(torch.empty(1, 3, 100, device="meta")), u, token=token, prob=prob, stream=Stream)]
    for f in cases:
        with pytest.raises(cb.ClutorError):
            f()
    assert not library.calls
    ctx.attention(q, kv, *ends, window=(1 << 31) - 1, **kw)
    assert library.calls[-1][1].window == (1 << 31) - 1


def test_context_on_the_current_device(library):
    """Context(-1) is on the device that was current, and takes the tensors there."""
    library.at = 3
    ctx = library.context(-1)
    assert ctx.device == 3
    x, u, token, prob = (Laid(t.like, 3) for t in sample_tensors(3, 100))
    ctx.sample(x, u, token=token, prob=prob, stream=Stream)
    assert len(library.calls) == 1
    with pytest.raises(cb.ClutorError, match="cuda:3"):
        ctx.sample(Laid(x.like, 0), u, token=token, prob=prob, stream=Stream)
    assert library.context(2).device == 2
