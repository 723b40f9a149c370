"""logits_process and logits_mark against a 64-bit statement of their rules."""
import math

import pytest
import torch

from molten_b200 import lfm, sample
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

INF = math.inf


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def bitmap(flags):
    """bool [rows, V] -> int32 [rows, ceil(V / 32)]."""
    rows, V = flags.shape
    f = torch.zeros(rows, -(-V // 32) * 32, dtype=torch.int64, device=flags.device)
    f[:, :V] = flags.long()
    w = (f.view(rows, -1, 32) << torch.arange(32, device=f.device)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


def case(seed, B, V, f32, rep=True, counts=True, biased=0, mask=None):
    g = gen(seed)
    x = torch.randn(B, V, generator=g, device="cuda") * 4
    x = x if f32 else x.to(torch.bfloat16)
    r, d = sample.LogitsRules(), dict(seen=None, n=None, bias=None, allow=None)
    u = lambda: torch.rand(B, generator=g, device="cuda")  # noqa: E731
    if rep:
        d["seen"] = torch.rand(B, V, generator=g, device="cuda") < 0.2
        r.seen, r.repetition = bitmap(d["seen"]), 0.7 + u()
    if counts:
        n = torch.randint(0, 70000, (B, V), generator=g, device="cuda").clamp(max=65535)
        n = torch.where(torch.rand(B, V, generator=g, device="cuda") < 0.3, n.clamp(max=9), torch.where(n > 65000, n, 0))
        d["n"] = n
        r.counts = torch.where(n >= 32768, n - 65536, n).short()
        r.frequency, r.presence = (u() - 0.3) * 0.01, u()
    if biased:
        ids, vals, start = [], [], [0]
        for b in range(B):
            k = biased if b % 3 else 0
            i = torch.randint(0, V, (k,), generator=g, device="cuda").sort().values  # repeats among them
            ids.append(i)
            vals.append(torch.randn(k, generator=g, device="cuda") * 5)
            start.append(start[-1] + k)
        r.bias_start = torch.tensor(start, dtype=torch.int32, device="cuda")
        r.bias_ids, r.bias_values = torch.cat(ids).int(), torch.cat(vals)
        d["bias"] = list(zip(ids, vals))
    if mask:
        rows = {"own": B, "shared": 2, "nothing": B}[mask]
        d["allow"] = torch.rand(rows, V, generator=g, device="cuda") < 0.5
        if mask == "nothing":
            d["allow"][0] = False
        r.allowed = bitmap(d["allow"])
        d["row"] = list(range(B))
        if mask == "shared":
            d["row"] = [(0, -1, 1, 7)[b % 4] for b in range(B)]
            r.allowed_row = torch.tensor(d["row"], dtype=torch.int32, device="cuda")
    return x, r, d


def want_of(x, r, d):
    """The rules in 64 bits, and what the fp32 roundings are relative to (six at most)."""
    v = x.double()
    size = v.abs()
    if d["seen"] is not None:
        p = r.repetition.double()[:, None]
        v = torch.where(d["seen"], torch.where(v > 0, v / p, v * p), v)
        size = torch.maximum(size, v.abs())
    if d["n"] is not None:
        n, f, q = d["n"].double(), r.frequency.double()[:, None], r.presence.double()[:, None]
        v = v - f * n - q * (n > 0)
        size = size + 2 * (f * n).abs() + q.abs()
    if d["bias"] is not None:
        v, size = v.clone(), size.clone()
        for b, (ids, vals) in enumerate(d["bias"]):
            v[b].index_add_(0, ids, vals.double())
            size[b].index_add_(0, ids, 4 * vals.double().abs())
    if d["allow"] is not None:
        for b, row in enumerate(d["row"]):
            if 0 <= row < d["allow"].shape[0]:
                v[b] = torch.where(d["allow"][row], v[b], -INF)
    return v, 6 * ref.U32 * size


def check(out, x, r, d, best, ctx):
    want, err = want_of(x, r, d)
    dead = want == -INF
    assert torch.equal(out == -INF, dead)
    half = ref.U32 if out.dtype == torch.float32 else ref.BF16_HALF
    off = (out.double() - want).abs()[~dead]
    assert bool((off <= half * want[~dead].abs() + 1.01 * err[~dead]).all()), off.max().item()
    if best is not None:
        tok = torch.zeros(out.shape[0], dtype=torch.int32, device="cuda")
        lfm.token_tail(ctx, best, tok)
        top = out.amax(1, keepdim=True)
        first = torch.where(out == top, torch.arange(out.shape[1], device="cuda"), out.shape[1]).amin(1)
        assert torch.equal(tok.long(), first)
        assert not best.any()


@pytest.mark.parametrize("B,V,f32,rep,counts,biased,mask", [
    (1, 65536, False, True, True, 20, "own"), (3, 65536, False, True, True, 300, "shared"), (2, 1, False, True, True, 2, "own"),
    (5, 7, True, True, True, 3, "own"), (4, 2047, False, True, True, 50, "nothing"), (4, 2049, True, True, True, 50, "shared"),
    (2, 128000, False, False, False, 0, "own"), (2, 32000, True, False, True, 0, None), (3, 50257, False, True, False, 5000, None),
    (1, 50257, False, True, True, 7, "own"), (9, 4096, False, False, False, 4000, None), (6, 33, False, False, False, 0, "nothing"),
    (4, 1000, True, False, False, 0, None), (300, 512, False, True, True, 10, "shared")])
def test_rules(cuda_ctx, B, V, f32, rep, counts, biased, mask):
    x, r, d = case(B + V, B, V, f32, rep, counts, biased, mask)
    x0 = x.clone()
    out, best = torch.full_like(x, math.nan), torch.zeros(B, dtype=torch.int64, device="cuda")
    sample.logits_process(cuda_ctx, x, out, r, best)
    check(out, x0, r, d, best, cuda_ctx)
    assert torch.equal(x, x0)
    sample.logits_process(cuda_ctx, x, x, r)  # in place
    assert torch.equal(x, out)


@pytest.mark.parametrize("f32", [False, True])
def test_strided_rows(cuda_ctx, f32):
    B, V = 3, 3001
    x, r, d = case(5, B, V, f32, biased=9, mask="own")
    wide = torch.zeros(B, V + 13, dtype=x.dtype, device="cuda")
    wide[:, 5:5 + V] = x
    back = torch.full((B, V + 3), 9.0, dtype=x.dtype, device="cuda")
    best = torch.zeros(B, dtype=torch.int64, device="cuda")
    sample.logits_process(cuda_ctx, wide[:, 5:5 + V], back[:, 1:1 + V], r, best)
    check(back[:, 1:1 + V].contiguous(), x, r, d, best, cuda_ctx)
    assert bool((back[:, 0] == 9).all()) and bool((back[:, 1 + V:] == 9).all())


def test_nan_and_infinities(cuda_ctx):
    V = 64
    x = torch.zeros(3, V, dtype=torch.bfloat16, device="cuda")
    x[0, 3], x[0, 9], x[0, 10] = math.nan, 2.0, math.nan
    x[1, 5], x[1, 6] = INF, -INF
    x[2] = math.nan
    allow = torch.ones(3, V, dtype=torch.bool, device="cuda")
    allow[0, 10] = allow[1, 5] = False
    out, best = torch.empty_like(x), torch.zeros(3, dtype=torch.int64, device="cuda")
    sample.logits_process(cuda_ctx, x, out, sample.LogitsRules(allowed=bitmap(allow)), best)
    assert math.isnan(out[0, 3]) and out[0, 10] == -INF and out[1, 5] == -INF and out[1, 6] == -INF
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    lfm.token_tail(cuda_ctx, best, tok)
    assert tok.tolist() == [9, 0, -1], "NaN never wins; a row of NaN has no token"


def test_mark(cuda_ctx):
    B, V = 6, 1000
    r = sample.LogitsRules(seen=torch.zeros(B, 32, dtype=torch.int32, device="cuda"),
                           counts=torch.zeros(B, V, dtype=torch.int16, device="cuda"))
    r.counts[0, 31] = -1  # 65535
    toks = torch.tensor([31, 0, 999, 1000, -1, 32], dtype=torch.int32, device="cuda")
    for _ in range(3):
        sample.logits_mark(cuda_ctx, toks, r, V)
    flags = torch.zeros(B, V, dtype=torch.bool, device="cuda")
    want = torch.zeros(B, V, dtype=torch.int16, device="cuda")
    for b, t in ((0, 31), (1, 0), (2, 999), (5, 32)):
        flags[b, t], want[b, t] = True, 3
    want[0, 31] = -1
    assert torch.equal(r.seen, bitmap(flags)) and torch.equal(r.counts, want)


def test_penalties_follow_the_draws(cuda_ctx):
    """Greedy steps with marking: a token's penalty grows until another wins."""
    V = 128
    logits = torch.zeros(1, V, dtype=torch.bfloat16, device="cuda")
    logits[0, 7], logits[0, 90] = 4.0, 3.0
    one = lambda v: torch.full((1,), v, device="cuda")  # noqa: E731
    r = sample.LogitsRules(seen=torch.zeros(1, 4, dtype=torch.int32, device="cuda"), repetition=one(1.0),
                           counts=torch.zeros(1, V, dtype=torch.int16, device="cuda"), frequency=one(0.75), presence=one(0.5))
    out, best = torch.empty_like(logits), torch.zeros(1, dtype=torch.int64, device="cuda")
    tok = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = []
    for _ in range(4):
        sample.logits_process(cuda_ctx, logits, out, r, best)
        lfm.token_tail(cuda_ctx, best, tok)
        sample.logits_mark(cuda_ctx, tok, r, V)
        got.append(tok.item())
    # 7: 4, then 2.75, 2.0; 90: 3, then 1.75
    assert got == [7, 90, 7, 7]
