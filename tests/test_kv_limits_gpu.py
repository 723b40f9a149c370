"""The paged attention at its limits: a wait that only a part of a warp runs
out of, weights far below the largest one."""
import pytest
import torch

from molten_b200 import _lib, kv
from tests import serving_ref as ref
from tests.test_kv_gpu import attention_case, check_attention, gen, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,H,K,fp8", [(64, 8, 2, False), (128, 8, 2, False), (64, 32, 2, True), (128, 8, 2, True)])
def test_a_wait_that_one_lane_runs_out_of(cuda_ctx, D, H, K, fp8):
    """One lane gives up just before the copies are reported, the other 31 find
    them: the warp gives up as one. The status says so, what it was working on
    is NaN, everything else is right, and the next call is whole again."""
    lens = [6000, 3, 9000, 0, 700]
    q, cache, table, keys = attention_case(14, lens, H, K, D, 16, fp8)
    ws, st = kv.paged_attention_workspace(D), torch.zeros(1, dtype=torch.int32, device="cuda")
    out, n = torch.empty_like(q), i32(lens)
    kv.paged_attention(cuda_ctx, q, cache, table, n, out, ws, status=st)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    cuda_ctx.set_test_flags(_lib.TEST_LATE_KV_ARRIVE)
    try:
        begin.record()
        kv.paged_attention(cuda_ctx, q, cache, table, n, out, ws, status=st)
        end.record()
        torch.cuda.synchronize()
    finally:
        cuda_ctx.set_test_flags(0)
    assert begin.elapsed_time(end) < 500, "the other lanes' waits (1 s at most) found the copies"
    assert st.item() == _lib.KV_WAIT
    for r in range(len(lens)):
        k, v = keys[r]
        want, _, e, _ = ref.attention(q[r], k, v, D ** -0.5)
        right = (out[r].double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * e
        assert bool((right | torch.isnan(out[r])).all())
        assert bool(torch.isnan(out[r]).any()) == (r == 0)
    st.zero_()
    kv.paged_attention(cuda_ctx, q, cache, table, n, out, ws, status=st)
    check_attention(out, None, q, keys, lens)
    assert st.item() == 0 and not ws[:4096].any()


def sink_case(seed, n, H, K, D, bs, gap, scaled):
    """One request of n keys in an e4m3 cache: key 0 scores highest and has V = 0, the others score
    some `gap` (natural logs) below it and carry the result. Returns q, the cache, its table, the
    keys' values and the scale that makes the gap."""
    g = gen(seed)
    pm = lambda *s: torch.randint(0, 2, s, generator=g, device="cuda") * 2.0 - 1  # noqa: E731
    u = pm(K, D)  # a direction for each KV head
    k = u * (6 + 0.5 * torch.randint(-1, 2, (n, K, D), generator=g, device="cuda"))
    k[0] = 8 * u
    v = torch.randn(n, K, D, generator=g, device="cuda") * 2
    v[0] = 0
    kind = torch.float8_e4m3fn
    k, v = k.to(kind), v.to(kind)
    heads = 1 + torch.arange(H // K, device="cuda") / 64
    q = (u[:, None] * heads[:, None]).reshape(1, H, D).to(torch.bfloat16)
    pages = -(-n // bs)
    table = torch.randperm(pages, generator=g, device="cuda")[None].int()
    c = kv.KvCache.empty(pages, K, bs, D, kind)
    at = torch.arange(n, device="cuda")
    page, off = table[0].long()[at // bs], at % bs
    for cache, rows in ((c.k, k), (c.v, v)):
        cache.view(torch.uint8).fill_(0x7f)
        cache.view(torch.uint8)[page, :, off] = rows.view(torch.uint8)
    k, v = k.double(), v.double()
    if scaled:
        s = [0.5 + torch.rand(K, generator=g, device="cuda") for _ in range(2)]
        c = kv.KvCache(c.k, c.v, *s)
        k, v = k * s[0].double()[:, None], v * s[1].double()[:, None]
    return q, c, table, k, v, gap / (2 * D)


@pytest.mark.parametrize("gap", [4.0, 10.0, 16.0, 17.5, 20.0])
@pytest.mark.parametrize("n,H,K,D,scaled", [(100, 8, 2, 64, False), (384, 32, 8, 64, False), (384, 16, 1, 128, False),
                                            (300, 8, 1, 128, True), (7000, 32, 8, 64, True), (5000, 16, 1, 64, False)])
def test_a_sink_above_a_flat_tail_in_an_8_bit_cache(cuda_ctx, n, H, K, D, scaled, gap):
    """Weights e^-4 to e^-20 of the largest one, whose V is zero, make up the whole result. The kernel
    holds a weight as two f16 parts of 2^15 times it (11 bits each, relative): what the bound of
    ref.attention says, and no less than half of f16's last step, 2^-25 / 2^15 = 2^-40 of the largest."""
    q, c, table, k, v, scale = sink_case(n + D, n, H, K, D, 16, gap, scaled)
    out, lse = torch.empty_like(q), torch.empty(1, H, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv.paged_attention(cuda_ctx, q, c, table, i32([n]), out, kv.paged_attention_workspace(D), scale=scale, lse=lse, status=st)
    want, wl, e, el = ref.attention(q[0], k, v, scale)
    floor = 2.0 ** -40 * v.abs().sum(0).repeat_interleave(H // K, 0)  # the largest weight is 1 at most
    off = (out[0].double() - want).abs()
    assert bool((off <= ref.BF16_HALF * want.abs() + 1.01 * (e + floor)).all()), (off / want.abs().mean()).max().item()
    assert bool(((lse[0].double() - wl).abs() <= el).all()) and st.item() == 0
