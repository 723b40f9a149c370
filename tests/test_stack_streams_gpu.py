"""The decode stack on a context with a stream of its own: the same tokens as
on torch's current stream, whatever that one is busy with."""
import pytest
import torch

from molten_b200 import kv, lfm, sample
from molten_b200.stack import DecodeStack
from tests.test_stack_serving_gpu import BS, E, make_layers, make_rules

pytestmark = pytest.mark.gpu

BUSY = 100_000_000  # cycles: 50 ms


def tokens_of(ctx, layers, head, embed, B, path, with_rules, sampled, steps, busy):
    """The tokens of each step as read_tokens gives them; `busy` streams have work ahead of every call."""
    def hold():
        for s in busy:
            with torch.cuda.stream(s):
                torch.cuda._sleep(BUSY)

    hold()
    st = DecodeStack(ctx, layers, head, embed, B, n_experts=E, moe_path=path,
                     kv=kv.PagedBatch(ctx, B, 4 * B, BS, 4), rules=make_rules(B, 2) if with_rules else None,
                     sampling=sample.Sampling(temperature=2.0, seed=7) if sampled else None)
    torch.cuda.synchronize()  # the rules' tensors are the caller's
    hold()
    st.start(torch.arange(B, dtype=torch.int32, device="cuda") * 91 + 5, pos=1)
    got = []
    for _ in range(steps):
        hold()
        st.step()
        got.append(st.read_tokens().tolist())
    return got


@pytest.mark.parametrize("B,path,with_rules,sampled", [(1, "fused", True, False), (1, "fused", False, True), (3, "gemv", True, False),
                                                       (4, "grouped", False, False)])
def test_a_stack_on_a_stream_of_its_own(cuda_ctx, B, path, with_rules, sampled):
    layers, head, embed = make_layers(400 + B, 2, (0,), 4 * B, torch.bfloat16)
    torch.cuda.synchronize()
    want = tokens_of(cuda_ctx, layers, head, embed, B, path, with_rules, sampled, 4, [])
    stream = torch.cuda.Stream()
    ctx = lfm.Context(0, stream)
    try:
        for busy in ([torch.cuda.current_stream()], [stream]):
            for L in layers:
                if "attn" in L:
                    for t in (L["attn"]["cache"].k, L["attn"]["cache"].v):
                        t.view(torch.uint8).fill_(0x7f)
            torch.cuda.synchronize()
            assert tokens_of(ctx, layers, head, embed, B, path, with_rules, sampled, 4, busy) == want
    finally:
        torch.cuda.synchronize()
        ctx.close()


def test_a_cache_with_fewer_pages_than_the_batch_is_refused(cuda_ctx):
    """Any one of the layers; a cache with more pages is fine."""
    layers, head, embed = make_layers(420, 2, (0, 1), 5, torch.bfloat16)
    build = lambda pages: DecodeStack(cuda_ctx, layers, head, embed, 1, n_experts=E,  # noqa: E731
                                      kv=kv.PagedBatch(cuda_ctx, 1, pages, BS, 5))
    with pytest.raises(ValueError, match="fewer pages"):
        build(6)
    build(5)
    layers[1]["attn"]["cache"] = kv.KvCache.empty(4, 8, BS)
    with pytest.raises(ValueError, match="fewer pages"):
        build(5)
    build(4)


def test_a_batch_of_another_stream_is_refused(cuda_ctx):
    """Its plan would run beside the steps; another context on the same stream is fine."""
    layers, head, embed = make_layers(421, 1, (0,), 5, torch.bfloat16)
    stream = torch.cuda.Stream()
    own, same, plain = lfm.Context(0, stream), lfm.Context(0, stream), lfm.Context(0)
    try:
        build = lambda a, b: DecodeStack(a, layers, head, embed, 1, n_experts=E, kv=kv.PagedBatch(b, 1, 5, BS, 5))  # noqa: E731
        for a, b in ((cuda_ctx, own), (own, cuda_ctx)):
            with pytest.raises(ValueError, match="another stream"):
                build(a, b)
        build(cuda_ctx, plain)
        build(own, same)
    finally:
        torch.cuda.synchronize()
        for c in (own, same, plain):
            c.close()
