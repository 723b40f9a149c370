"""A Context's calls go to its stream -- its own, or torch's current one --
whatever stream was set on the library's context through the C call since."""
import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from molten_b200 import _lib, lfm


class FakeLibrary:
    """The context calls of the library, on a stream word in host memory."""

    def __init__(self):
        self.word, self.sets = C.c_void_p(), 0

    def mc_create(self, device, stream, out):
        out._obj.value, self.word.value = 0x1000, stream
        return 0

    def mc_set_stream(self, h, stream):
        if not h:
            return _lib.MC_EINVAL
        self.word.value = stream
        self.sets += 1
        return 0

    def mc_stream_slot(self, h):
        return C.addressof(self.word)

    def mc_destroy(self, h):
        return 0

    def mc_last_error(self):
        return b"mc_set_stream: null context"


@pytest.fixture
def fake(monkeypatch):
    lib = FakeLibrary()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    lib.current = 0x700
    monkeypatch.setattr(lfm, "_raw_stream", lambda index: lib.current)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: SimpleNamespace(cuda_stream=lib.current))
    made = []
    lib.context = lambda own: made.append(lfm.Context(0, own and SimpleNamespace(cuda_stream=own))) or made[-1]
    yield lib
    for ctx in made:
        ctx.h = None  # nothing of it is the library's


@pytest.mark.parametrize("own", [None, 0x500])
def test_a_stream_set_behind_the_context_is_put_back(fake, own):
    ctx = fake.context(own)
    for current, behind in [(0x700, None), (0x700, 0x900), (0x800, None), (0x800, 0x700), (0, 0x900), (0x700, 0)]:
        fake.current = current
        if behind is not None:
            fake.mc_set_stream(0x1000, behind)
        assert ctx.handle.value == 0x1000
        assert (fake.word.value or 0) == (own or current), (current, behind)
    sets = fake.sets
    for _ in range(3):  # nothing to put back: no call
        assert ctx.handle.value == 0x1000
    assert fake.sets == sets


@pytest.mark.parametrize("own", [None, 0x500])
def test_a_closed_context_is_refused(fake, own):
    ctx = fake.context(own)
    ctx.close()
    with pytest.raises(_lib.McError, match="null context"):
        ctx.handle
    ctx.close()


def test_contexts_on_one_stream(fake):
    a, b, c, d = (fake.context(s) for s in (None, None, 0x500, 0x600))
    assert a.same_stream(b) and a.same_stream(a) and c.same_stream(fake.context(0x500))
    assert not a.same_stream(c) and not c.same_stream(a) and not c.same_stream(d)
    b.index = 1
    assert not a.same_stream(b)


def test_the_stream_word_of_no_context():
    from molten_b200 import build
    build.build()
    assert _lib.lib().mc_stream_slot(None) is None


@pytest.mark.gpu
@pytest.mark.parametrize("own", [False, True])
def test_calls_follow_torch_after_a_stream_was_set_behind(own):
    """The call's launch lies in the graph that its stream captures."""
    mine, other = torch.cuda.Stream(), torch.cuda.Stream()
    ctx = lfm.Context(0, mine if own else None)
    try:
        x = torch.randn(256, device="cuda").to(torch.bfloat16)
        y, want = torch.zeros_like(x), torch.zeros_like(x)
        torch.cuda.synchronize()
        lfm.silu_mul_bf16(ctx, x, x, want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(mine):
            _lib.check(_lib.lib().mc_set_stream(ctx.h, other.cuda_stream))
            with torch.cuda.graph(graph, stream=mine):
                lfm.silu_mul_bf16(ctx, x, x, y)
        torch.cuda.synchronize()
        assert not y.any(), "captured, not run"
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and bool(want.any())
    finally:
        ctx.close()
