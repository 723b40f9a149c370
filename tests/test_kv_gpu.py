"""The paged cache and its attention on the GPU: kv_plan / kv_release against a
loop over the requests, qk_norm_rope and paged_attention against 64-bit
statements of their formulas (tests/serving_ref.py), at the lengths, layouts
and masks where they can go wrong; the calls together, captured and replayed."""
import math
import random

import pytest
import torch

from molten_b200 import _lib, kv
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

NAN = float("nan")
I32 = torch.int32


def i32(v):
    return torch.tensor(v, dtype=I32, device="cuda")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def bf16(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


# ------------------------------------------------------------------ bookkeeping

class Plan:
    """The buffers of one kv_plan."""

    def __init__(self, lens, table, free, n_free, max_tokens):
        R = len(lens)
        self.lens, self.table, self.free, self.n_free = i32(lens), i32(table), i32(free), i32([n_free])
        z = lambda n: torch.full((n,), 77, dtype=I32, device="cuda")  # noqa: E731
        self.seq, self.n_free_out, self.row_start = z(R), z(1), z(R + 1)
        self.positions, self.token_req, self.kv_lens = z(max_tokens), z(max_tokens), z(max_tokens)
        self.slots = torch.full((max_tokens,), 77, dtype=torch.int64, device="cuda")
        self.status = torch.zeros(1, dtype=I32, device="cuda")

    def run(self, ctx, new, bs, in_place=False):
        seq, nf = (self.lens, self.n_free) if in_place else (self.seq, self.n_free_out)
        kv.kv_plan(ctx, self.lens, None if new is None else i32(new), bs, self.table, self.free, self.n_free, seq, nf,
                   self.row_start, self.positions, self.token_req, self.kv_lens, self.slots, self.status)
        return dict(seq=seq.tolist(), n_free=nf.item(), row_start=self.row_start.tolist(), positions=self.positions.tolist(),
                    token_req=self.token_req.tolist(), kv_lens=self.kv_lens.tolist(), slots=self.slots.tolist())


def random_batch(rnd, R, bs, width, most_new, spare):
    lens = [rnd.choice((0, 0, 1, bs - 1, bs, rnd.randrange(width * bs + 1))) for _ in range(R)]
    lens = [min(n, width * bs) for n in lens]
    pages = list(range(R * width + 5))
    rnd.shuffle(pages)
    table, at = [], 0
    for n in lens:
        held = -(-n // bs)
        table.append(pages[at:at + held] + [-9] * (width - held))
        at += held
    free = pages[at:] + [-5] * at
    new = [rnd.choice((0, 1, 1, rnd.randrange(most_new + 1))) for _ in range(R)]
    return lens, new, table, free, max(0, min(len(pages) - at, spare))


@pytest.mark.parametrize("R,bs,width,most_new,spare,max_tokens", [
    (1, 16, 4, 1, 10, 1), (1, 1, 7, 5, 100, 9), (5, 4, 3, 6, 100, 40), (33, 16, 4, 40, 40, 700), (100, 3, 5, 4, 20, 150),
    (1024, 8, 4, 3, 4000, 2100), (2500, 16, 3, 9, 3000, 9000), (7, 128, 2, 200, 100, 1400), (64, 20, 30, 300, 2000, 12000),
    (40, 16, 4, 10, 0, 300), (9, 1000000, 1, 3, 9, 20)])
def test_plan_matches_the_loop(cuda_ctx, R, bs, width, most_new, spare, max_tokens):
    rnd = random.Random(R * 1000 + bs)
    lens, new, table, free, n_free = random_batch(rnd, R, bs, min(width, 30), most_new, spare)
    P = Plan(lens, table, free, n_free, max_tokens)
    for _ in range(2):  # with other buffers for the results a call may be repeated
        got = P.run(cuda_ctx, new, bs)
    rows = [list(t) for t in table]
    want, status = ref.plan(lens, new, bs, rows, free, n_free, max_tokens)
    assert got == want
    assert P.table.tolist() == rows
    assert P.status.item() == status
    assert P.lens.tolist() == lens and P.n_free.item() == n_free


def test_plan_one_token_each_by_default_and_in_place(cuda_ctx):
    rnd = random.Random(3)
    lens, _, table, free, n_free = random_batch(rnd, 20, 4, 6, 1, 100)
    lens = [min(n, 4 * 6 - 3) for n in lens]
    P = Plan(lens, table, free, n_free, 20)
    rows = [list(t) for t in table]
    for _ in range(3):  # the lengths and the free list advance by themselves
        got = P.run(cuda_ctx, None, 4, in_place=True)
        want, status = ref.plan(lens, [1] * 20, 4, rows, free, n_free, 20)
        assert got == want and status == 0 and P.table.tolist() == rows
        lens, n_free = want["seq"], want["n_free"]


def test_plan_refuses_bad_lengths_and_keeps_the_rest(cuda_ctx):
    table = [[0, -1], [1, -1], [2, -1], [-1, -1], [3, -1]]
    free = [9, 8, 7, 6, 5]
    lens, new = [4, -3, 2, 0, 3], [1, 2, -1, 9, 1]
    P = Plan(lens, table, free, 5, 8)
    got = P.run(cuda_ctx, new, 4)
    rows = [list(t) for t in table]
    want, status = ref.plan(lens, new, 4, rows, free, 5, 8)
    assert got == want and P.status.item() == status == 8 | 2 | 4
    assert P.table.tolist() == rows


@pytest.mark.parametrize("in_place", [False, True])
def test_release_returns_the_pages(cuda_ctx, in_place):
    rnd = random.Random(5)
    R, bs, width = 1500, 8, 6
    lens, _, table, free, n_free = random_batch(rnd, R, bs, width, 1, 10 ** 6)
    done = [int(rnd.random() < 0.3) * rnd.choice((1, 7, -1)) for _ in range(R)]
    L, F, N = i32(lens), i32(free), i32([n_free])
    lo, no = (L, N) if in_place else (torch.full_like(L, 5), torch.full_like(N, 5))
    st = torch.zeros(1, dtype=I32, device="cuda")
    kv.kv_release(cuda_ctx, i32(done), L, bs, i32(table), F, N, lo, no, st)
    for r in range(R):
        if done[r]:
            held = -(-lens[r] // bs)
            free[n_free:n_free + held] = table[r][:held]
            n_free += held
    assert lo.tolist() == [0 if d else n for d, n in zip(done, lens)]
    assert no.item() == n_free and F.tolist() == free and st.item() == 0


def test_release_beyond_the_free_list(cuda_ctx):
    F = i32([4, 5, 6])
    L, N = i32([9, 9]), i32([2])
    st = torch.zeros(1, dtype=I32, device="cuda")
    kv.kv_release(cuda_ctx, i32([1, 1]), L, 4, i32([[1, 2, 3], [7, 8, 9]]), F, N, L, N, st)
    assert F.tolist() == [4, 5, 1] and N.item() == 3 and L.tolist() == [0, 0]
    assert st.item() == _lib.KV_LIST_FULL
    with pytest.raises(_lib.McError, match="free list"):
        kv.raise_on_status(st, "kv_release")


# ------------------------------------------------------------------ norm, rotation, cache write

def rope_case(seed, T, H, K, D, fp8, blocks=None, bs=16, fused=True):
    g = gen(seed)
    rows = bf16(g, T, (H + 2 * K) * D + (8 if fused else 0), scale=2.0)
    q = rows[:, :H * D].view(T, H, D)
    k = rows[:, H * D:(H + K) * D].view(T, K, D)
    v = rows[:, (H + K) * D:(H + 2 * K) * D].view(T, K, D)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
    blocks = blocks or -(-T // bs) + 2
    c = kv.KvCache.empty(blocks, K, bs, D, kind)
    for t in (c.k, c.v):
        t.view(torch.uint8).fill_(0x35)
    norm = lambda: (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)  # noqa: E731
    return g, q, k, v, norm(), norm(), c


def check_store(cache, slots, rows, err, scale, bs, untouched):
    """The cache rows at slots hold `rows` (64 bits, fp32 error err), the others the fill."""
    K, D = rows.shape[1], rows.shape[2]
    flat = cache.transpose(1, 2).reshape(-1, K, D)
    used = torch.tensor([s for s in slots if s >= 0], device="cuda")
    at = torch.tensor([i for i, s in enumerate(slots) if s >= 0], device="cuda")
    if used.numel():
        got, want, e = flat.view(torch.uint8 if cache.dtype != torch.bfloat16 else cache.dtype)[used], rows[at], err[at]
        if cache.dtype == torch.bfloat16:
            assert bool(((got.double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * e).all())
        else:
            got = got.view(torch.float8_e4m3fn).double()
            if scale is not None:
                want, e = want / scale.double()[:, None], e / scale.double()[:, None] + ref.U32 * (want / scale.double()[:, None]).abs()
            want = want.clamp(-448, 448)
            assert bool(((got - want).abs() <= ref.E4M3_HALF * want.abs() + 2.0 ** -10 + 1.1 * e).all())
    rest = torch.ones(flat.shape[0], dtype=torch.bool, device="cuda")
    rest[used] = False
    assert bool((flat[rest].contiguous().view(torch.uint8) == untouched).all()), "slots not named stay as they were"


@pytest.mark.parametrize("T,H,K,D,rot,inter,fp8,far", [
    (1, 32, 8, 64, 64, False, False, 5000), (3, 32, 8, 64, 64, True, False, 200000), (17, 4, 1, 64, 32, False, False, 2 ** 31 - 1),
    (5, 1, 1, 64, 16, True, False, 100), (9, 6, 2, 128, 128, False, False, 1000000), (2, 40, 8, 128, 64, True, False, 50),
    (33, 8, 8, 128, 112, False, True, 131072), (4, 32, 8, 64, 64, False, True, 4096), (7, 3, 3, 64, 48, True, True, 9000),
    (11, 16, 2, 128, 0, False, False, 10), (200, 64, 8, 128, 128, False, True, 70000)])
def test_norm_rope_and_store(cuda_ctx, T, H, K, D, rot, inter, fp8, far):
    bs = 16
    g, q, k, v, qw, kw, c = rope_case(T + D + rot, T, H, K, D, fp8, bs=bs)
    ks = vs = None
    if fp8:
        ks, vs = (0.02 * torch.rand(K, generator=g, device="cuda") + 0.002 for _ in range(2))
        c = kv.KvCache(c.k, c.v, ks, vs)
    pos = torch.randint(0, far, (T,), generator=g, device="cuda", dtype=I32)
    pos[0] = far - 1
    slots = torch.randperm(c.k.shape[0] * bs, generator=g, device="cuda")[:T]
    if T > 2:
        slots[1] = -1
    turns = kv.rope_turns(rot, 1e6).cuda() if rot else None
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    out = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda")
    st = torch.zeros(1, dtype=I32, device="cuda")
    kv.qk_norm_rope(cuda_ctx, q, k, v, qw, kw, pos, turns, out, c, slots, interleaved=inter, status=st)
    freqs = [1e6 ** (-2 * i / rot) for i in range(rot // 2)] if rot else []
    want, size = ref.norm_rope(q0, qw, pos, freqs, rot, inter, 1e-5)
    assert bool(((out.double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * ref.norm_rope_error(D) * size).all())
    want, size = ref.norm_rope(k0, kw, pos, freqs, rot, inter, 1e-5)
    check_store(c.k, slots.tolist(), want, ref.norm_rope_error(D) * size, ks, bs, 0x35)
    check_store(c.v, slots.tolist(), v0.double(), torch.zeros_like(v0, dtype=torch.float64), vs, bs, 0x35)
    assert st.item() == 0 and torch.equal(q, q0) and torch.equal(k, k0)


@pytest.mark.parametrize("H", [7000, 8000, 16384])
def test_norm_rope_more_heads_than_a_wave(cuda_ctx, H):
    """Above 24 heads of 128 for each of a wave's CTAs (7104 and more on 148 SMs) one row of CTAs takes every token."""
    T, K, D = 3, 1, 128
    g, q, k, v, qw, kw, c = rope_case(H, T, H, K, D, False, bs=4, fused=False)
    pos, slots = i32([5, 0, 70000]), torch.tensor([2, 0, 1], device="cuda")
    out = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda")
    kv.qk_norm_rope(cuda_ctx, q, k, v, qw, kw, pos, kv.rope_turns(D).cuda(), out, c, slots)
    want, size = ref.norm_rope(q, qw, pos, [1e6 ** (-2 * i / D) for i in range(D // 2)], D, False, 1e-5)
    assert bool(((out.double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * ref.norm_rope_error(D) * size).all())
    check_store(c.v, [2, 0, 1], v.double(), torch.zeros_like(v, dtype=torch.float64), None, 4, 0x35)


def test_norm_rope_in_place_in_a_fused_row_and_of_one_token(cuda_ctx):
    for T in (5, 1):
        g, q, k, v, qw, kw, c = rope_case(9, T, 4, 2, 64, False, bs=4)
        pos = torch.arange(T, device="cuda", dtype=I32) + 9
        turns = kv.rope_turns(64).cuda()
        out = torch.empty(T, 4, 64, dtype=torch.bfloat16, device="cuda")
        kv.qk_norm_rope(cuda_ctx, q, k, v, qw, kw, pos, turns, out, c)
        first = c.k.clone()
        k0 = k.clone()
        if T == 1:  # a row whose stride to the next, which is not there, is odd
            q = q.as_strided(q.shape, (q.stride(0) + 1, 64, 1))
        kv.qk_norm_rope(cuda_ctx, q, k, v, qw, kw, pos, turns, q, c)
        assert torch.equal(q, out) and torch.equal(k, k0)
        assert torch.equal(c.k.view(torch.uint8), first.view(torch.uint8))


def test_norm_rope_in_place_without_v_norm_or_slots(cuda_ctx):
    T, H, K, D = 6, 4, 2, 64
    g, q, k, v, qw, kw, c = rope_case(1, T, H, K, D, False, blocks=1, bs=8, fused=False)
    pos = torch.arange(T, device="cuda", dtype=I32) * 1000
    q0 = q.clone()
    kv.qk_norm_rope(cuda_ctx, q, k, None, None, None, pos, kv.rope_turns(D, 10000.0).cuda(), q, c)
    freqs = [1e4 ** (-2 * i / D) for i in range(D // 2)]
    want, size = ref.norm_rope(q0, None, pos, freqs, D, False, 0)
    assert bool(((q.double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * ref.norm_rope_error(D) * size).all())
    want, size = ref.norm_rope(k, None, pos, freqs, D, False, 0)
    check_store(c.k, list(range(T)), want, ref.norm_rope_error(D) * size, None, 8, 0x35)
    assert bool((c.v.view(torch.uint8) == 0x35).all())


def test_norm_rope_zero_rows_and_saturation(cuda_ctx):
    g, q, k, v, qw, kw, c = rope_case(2, 3, 2, 1, 64, True, bs=4)
    q.zero_()
    v[0, 0, :4] = torch.tensor([3e4, -3e4, NAN, float("inf")], dtype=torch.bfloat16)
    out = torch.empty(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    pos = i32([0, 1, 2])
    kv.qk_norm_rope(cuda_ctx, q, k, v, qw, kw, pos, kv.rope_turns(64).cuda(), out, c)
    assert bool((out == 0).all())
    got = c.v[0, 0, 0, :4].float().tolist()
    assert got[0] == 448 and got[1] == -448 and math.isnan(got[2]) and got[3] == 448


def test_norm_rope_slot_outside_the_cache(cuda_ctx):
    g, q, k, v, qw, kw, c = rope_case(3, 4, 2, 1, 64, False, blocks=2, bs=4)
    slots = torch.tensor([8, 3, -2, 2 ** 62], device="cuda")
    out = torch.empty(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    st = torch.zeros(1, dtype=I32, device="cuda")
    pos = i32([1, 2, 3, 4])
    kv.qk_norm_rope(cuda_ctx, q, k, v, qw, kw, pos, kv.rope_turns(64).cuda(), out, c, slots, status=st)
    want, size = ref.norm_rope(k, kw, pos, [1e6 ** (-2 * i / 64) for i in range(32)], 64, False, 1e-5)
    check_store(c.k, [-1, 3, -1, -1], want, ref.norm_rope_error(64) * size, None, 4, 0x35)
    assert st.item() == _lib.KV_BAD_SLOT


# ------------------------------------------------------------------ attention

def attention_case(seed, lens, H, K, D, bs, fp8=False, halves=False, width=None, req=None, scale=1.0):
    """A cache whose rows that nothing may read hold NaN, a table whose unused entries are out of range."""
    g = gen(seed)
    n_req = len(lens) if req is None else max(req) + 1
    need = [0] * n_req
    for r, n in enumerate(lens):
        at = r if req is None else req[r]
        need[at] = max(need[at], n)
    width = width or max(1, max(-(-n // bs) for n in need) + 1)
    pages = [-(-n // bs) for n in need]
    blocks = sum(pages) + 2
    order = torch.randperm(blocks, generator=g, device="cuda").tolist()
    kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
    nan = 0x7f if fp8 else 0xff
    if halves:
        both = torch.empty(blocks, 2, K, bs, D, dtype=kind, device="cuda")
        ck, cv = both[:, 0], both[:, 1]
        both.view(torch.uint8).fill_(nan)
    else:
        ck, cv = (torch.empty(blocks, K, bs, D, dtype=kind, device="cuda") for _ in range(2))
        for t in (ck, cv):
            t.view(torch.uint8).fill_(nan)
    table = torch.full((n_req, width), -1, dtype=I32, device="cuda")
    table[:, 1::2] = 10 ** 9
    keys, at = [], 0
    big = 16.0 if fp8 else 1.0
    for r in range(n_req):
        n = need[r]
        kr, vr = ((torch.randn(n, K, D, generator=g, device="cuda") * big * scale).to(kind) for _ in range(2))
        for j in range(pages[r]):
            p = order[at]
            at += 1
            table[r, j] = p
            part = slice(j * bs, min(n, (j + 1) * bs))
            m = part.stop - part.start
            for cache, rows in ((ck, kr), (cv, vr)):
                cache.view(torch.uint8)[p, :, :m] = rows.view(torch.uint8)[part].transpose(0, 1)
        keys.append((kr, vr))
    s = None
    if fp8:
        s = [(0.5 + torch.rand(K, generator=g, device="cuda")) / big for _ in range(2)]
        keys = [(a.double() * s[0].double()[:, None], b.double() * s[1].double()[:, None]) for a, b in keys]
    cache = kv.KvCache(ck, cv, *(s or (None, None)))
    q = bf16(g, len(lens), H, D, scale=1.5)
    return q, cache, table, keys


def check_attention(got, lse, q, keys, lens, req=None, scale=None, window=0):
    scale = scale or 1 / math.sqrt(q.shape[2])
    for r, n in enumerate(lens):
        k, v = keys[r if req is None else req[r]]
        want, wl, e, el = ref.attention(q[r], k[:n], v[:n], scale, window)
        off = (got[r].double() - want).abs()
        assert bool((off <= ref.BF16_HALF * want.abs() + 1.01 * e).all()), (r, n, off.max().item())
        if lse is not None:
            assert bool(((lse[r].double() - wl).abs() <= el).all() if n else (lse[r] == wl).all()), (r, n)


EDGES = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("lens,H,K,D,bs,fp8,window", [
    (EDGES, 32, 8, 64, 16, False, 0), (EDGES, 32, 8, 64, 16, True, 0), (EDGES, 16, 2, 128, 16, False, 0),
    (EDGES, 16, 2, 128, 32, True, 0), (EDGES, 8, 8, 64, 1, False, 0), (EDGES, 6, 2, 64, 20, False, 0),
    (EDGES, 12, 1, 64, 7, True, 0), (EDGES, 32, 1, 128, 300, False, 0), (EDGES, 9, 1, 64, 64, False, 0),
    (EDGES, 32, 8, 64, 16, False, 1), (EDGES, 32, 8, 64, 16, False, 64), (EDGES, 4, 4, 128, 8, True, 100),
    ([0], 4, 1, 64, 16, False, 0), ([1], 4, 1, 64, 16, True, 0), ([0, 0, 0], 4, 4, 128, 16, False, 0),
    ([5000, 0, 1, 12345, 64], 8, 2, 64, 16, False, 0), ([5000, 0, 1, 9001, 64], 8, 2, 128, 24, True, 0),
    ([40000], 2, 1, 64, 128, False, 0), ([40000], 3, 1, 128, 16, True, 0), ([40000, 300], 4, 2, 64, 16, False, 30001),
    (EDGES, 16, 1, 64, 16, False, 0), (EDGES, 32, 2, 128, 16, True, 0), (EDGES, 24, 1, 128, 16, False, 33),
    ([5000, 0, 1, 9001, 64], 48, 2, 64, 16, False, 0), ([5000, 0, 1, 9001, 64], 20, 2, 128, 16, True, 0),
    ([20000], 16, 1, 128, 16, False, 0), ([20000, 7], 31, 1, 64, 16, True, 0), ([3] * 700, 4, 1, 64, 4, False, 0), (list(range(300)), 4, 2, 64, 16, False, 17)])
def test_attention(cuda_ctx, lens, H, K, D, bs, fp8, window):
    q, cache, table, keys = attention_case(len(lens) + H + D + bs, lens, H, K, D, bs, fp8)
    out = torch.full_like(q, NAN)
    lse = torch.full((len(lens), H), NAN, device="cuda")
    ws = kv.paged_attention_workspace(D)
    st = torch.zeros(1, dtype=I32, device="cuda")
    for _ in range(2):
        kv.paged_attention(cuda_ctx, q, cache, table, i32(lens), out, ws, window=window, lse=lse, status=st)
    check_attention(out, lse, q, keys, lens, window=window)
    assert st.item() == 0
    assert not ws[:2048].any(), "the joining counters are zero again"


@pytest.mark.parametrize("lens,H,K,D,bs,fp8,window", [
    ([20000] + 200 * [0], 8, 2, 64, 16, False, 0),            # one long row among empty ones
    (90 * [1, 130, 0, 700], 4, 2, 64, 16, True, 0),           # many short pieces in a CTA
    ([3000, 17, 2500, 1, 900, 6000, 0, 40] * 6, 8, 4, 128, 24, False, 0),
    ([3000, 17, 2500, 1, 900, 6000, 0, 40] * 9, 16, 8, 64, 16, True, 1000),
    ([129 * i % 5000 for i in range(40)], 32, 2, 64, 32, False, 0),  # 16 heads a tile
])
def test_attention_pieces_of_unlike_rows(cuda_ctx, lens, H, K, D, bs, fp8, window):
    """Batches whose split counts the starts of the pieces."""
    q, c, table, keys = attention_case(len(lens) + D, lens, H, K, D, bs, fp8)
    out = torch.full_like(q, NAN)
    lse = torch.full((len(lens), H), NAN, device="cuda")
    st = torch.zeros(1, dtype=I32, device="cuda")
    ws = kv.paged_attention_workspace(D)
    for _ in range(2):  # the second finds the counters as the first left them
        kv.paged_attention(cuda_ctx, q, c, table, i32(lens), out, ws, window=window, lse=lse, status=st)
    assert st.item() == 0
    check_attention(out, lse, q, keys, lens, window=window)


def test_attention_strided_rows_and_halves(cuda_ctx):
    lens, H, K, D, bs = [100, 3, 777, 0], 8, 2, 64, 16
    q, cache, table, keys = attention_case(1, lens, H, K, D, bs, halves=True)
    row = torch.zeros(4, (H + 4) * D, dtype=torch.bfloat16, device="cuda")
    row[:, 2 * D:(2 + H) * D] = q.view(4, -1)
    qs = row[:, 2 * D:(2 + H) * D].view(4, H, D)
    back = torch.full((4, H * D + 16), 7.0, dtype=torch.bfloat16, device="cuda")
    out = back[:, 8:8 + H * D].view(4, H, D)
    kv.paged_attention(cuda_ctx, qs, cache, table, i32(lens), out, kv.paged_attention_workspace(D))
    check_attention(out, None, q, keys, lens)
    assert bool((back[:, :8] == 7).all()) and bool((back[:, 8 + H * D:] == 7).all())


def test_attention_rows_of_one_request(cuda_ctx):
    """Draft tokens: several rows read prefixes of one request; -1 is a row of none."""
    lens, req = [50, 51, 52, 0, 300, 9, 0], [0, 0, 0, 0, 2, 1, 0]
    q, cache, table, keys = attention_case(2, lens, 8, 2, 64, 16, req=req)
    out, lse = torch.empty_like(q), torch.empty(7, 8, device="cuda")
    st = torch.zeros(1, dtype=I32, device="cuda")
    rows = i32([0, 0, 0, 0, 2, 1, -1])
    kv.paged_attention(cuda_ctx, q, cache, table, i32(lens[:6] + [5]), out, kv.paged_attention_workspace(64), row_req=rows, lse=lse,
                       status=st)
    check_attention(out, lse, q, keys, lens, req)
    assert st.item() == 0


def test_attention_over_the_scatter_cache(cuda_ctx):
    """A contiguous [KV heads, max_seq, 64] cache is one page."""
    g = gen(9)
    K, S, n = 8, 640, 577
    kc, vc = bf16(g, K, S, 64), bf16(g, K, S, 64)
    q = bf16(g, 1, 32, 64)
    out = torch.empty_like(q)
    kv.paged_attention(cuda_ctx, q, kv.KvCache(kc[None], vc[None]), i32([[0]]), i32([n]), out, kv.paged_attention_workspace(64))
    check_attention(out, None, q, [(kc.transpose(0, 1), vc.transpose(0, 1))], [n])


def test_attention_extreme_scores(cuda_ctx):
    """Scores from -4000 to 4000: the running maximum keeps every exponential in range."""
    lens = [1, 300, 4097]
    q, cache, table, keys = attention_case(4, lens, 4, 1, 64, 16, scale=40.0)
    out, lse = torch.empty_like(q), torch.empty(3, 4, device="cuda")
    kv.paged_attention(cuda_ctx, q * 8, cache, table, i32(lens), out, kv.paged_attention_workspace(64), lse=lse)
    assert bool(torch.isfinite(out.float()).all())
    check_attention(out, lse, q * 8, keys, lens)


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_query_range(cuda_ctx, fp8):
    """Query rows from 2^-100 to 2^100, one all zero."""
    lens = [200] * 5
    q, cache, table, keys = attention_case(5, lens, 4, 2, 64, 16, fp8)
    q = q.clone()
    for r, e in enumerate((-100, -14, 0, 30, None)):
        q[r] = 0 if e is None else q[r] * 2.0 ** e
    scales = [2.0 ** 97, 2.0 ** 11, 0.125, 2.0 ** -33, 1.0]
    for r, s in enumerate(scales):
        out, lse = torch.empty_like(q[r:r + 1]), torch.empty(1, 4, device="cuda")
        kv.paged_attention(cuda_ctx, q[r:r + 1], cache, table[r:r + 1], i32([200]), out, kv.paged_attention_workspace(64), scale=s,
                           lse=lse)
        check_attention(out, lse, q[r:r + 1], keys[r:r + 1], [200], scale=s)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30, 3.0])
def test_attention_scales(cuda_ctx, scale, fp8):
    """Zero weighs every key alike, a negative one turns the order around."""
    lens = [1, 77, 500]
    q, cache, table, keys = attention_case(12, lens, 8, 2, 64, 16, fp8)
    out, lse = torch.empty_like(q), torch.empty(3, 8, device="cuda")
    kv.paged_attention(cuda_ctx, q, cache, table, i32(lens), out, kv.paged_attention_workspace(64), scale=scale, lse=lse)
    for r, n in enumerate(lens):
        k, v = keys[r]
        want, wl, e, el = ref.attention(q[r], k[:n], v[:n], scale)
        assert bool(((out[r].double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * e.abs()).all()), (r, n)
        assert bool(((lse[r].double() - wl).abs() <= el.abs()).all())


def test_attention_a_wait_that_runs_out(cuda_ctx):
    """Copies that are never reported: the wait gives up at its limit, the status
    says so, what they were needed for is NaN, nothing else changes, and the
    next call is whole again."""
    lens = [6000, 3, 9000, 0, 700]
    q, cache, table, keys = attention_case(13, lens, 8, 2, 128, 16)
    ws, st = kv.paged_attention_workspace(128), torch.zeros(1, dtype=I32, device="cuda")
    out = torch.empty_like(q)
    n = i32(lens)
    cuda_ctx.set_wait_limit(1_000_000)
    cuda_ctx.set_test_flags(_lib.TEST_SKIP_KV_ARRIVE)
    try:
        kv.paged_attention(cuda_ctx, q, cache, table, n, out, ws, status=st)
        torch.cuda.synchronize()
    finally:
        cuda_ctx.set_wait_limit(0)
        cuda_ctx.set_test_flags(0)
    assert st.item() == _lib.KV_WAIT
    for r in range(len(lens)):
        k, v = keys[r]
        want, _, e, _ = ref.attention(q[r], k, v, 128 ** -0.5)
        right = (out[r].double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * e
        assert bool((right | torch.isnan(out[r])).all())
        assert bool(torch.isnan(out[r]).any()) == (r == 0)
    with pytest.raises(_lib.McError, match="in time"):
        kv.raise_on_status(st, "paged_attention")
    st.zero_()
    kv.paged_attention(cuda_ctx, q, cache, table, n, out, ws, status=st)
    check_attention(out, None, q, keys, lens)
    assert st.item() == 0 and not ws[:4096].any()


def test_attention_status_of_bad_pages_rows_and_lengths(cuda_ctx):
    lens = [40, 40, 40, 1000]
    q, cache, table, keys = attention_case(6, [40, 40, 40, 40], 4, 2, 64, 16, width=3)
    table = table.clone()
    table[0, 1] = 10 ** 9   # keys 16 to 31 are left out
    table[1, 0] = -7
    out, lse = torch.empty_like(q), torch.empty(4, 4, device="cuda")
    ws, st = kv.paged_attention_workspace(64), torch.zeros(1, dtype=I32, device="cuda")
    kv.paged_attention(cuda_ctx, q[:2], cache, table[:2], i32(lens[:2]), out[:2], ws, lse=lse[:2], status=st)
    k0, v0 = (torch.cat((t[:16], t[32:])) for t in keys[0])
    k1, v1 = (t[16:] for t in keys[1])
    check_attention(out[:2], lse[:2], q[:2], [(k0, v0), (k1, v1)], [24, 24])
    assert st.item() == _lib.KV_BAD_PAGE
    st.zero_()
    kv.paged_attention(cuda_ctx, q, cache, table, i32([3, -4, 40, 5]), out, ws, row_req=i32([4, 2, 2, -2]), lse=lse, status=st)
    assert st.item() == _lib.KV_BAD_ROW | _lib.KV_BAD_LENGTH
    for r in (0, 1, 3):
        assert bool((out[r] == 0).all()) and bool((lse[r] == -math.inf).all())
    check_attention(out[2:3], lse[2:3], q[2:3], [keys[2]], [40])
    st.zero_()  # longer than the block table: as many keys as it has pages for
    kv.paged_attention(cuda_ctx, q[2:3], cache, table[2:3, :2].contiguous(), i32([40]), out[2:3], ws, status=st)
    assert st.item() == _lib.KV_BAD_LENGTH
    check_attention(out[2:3], None, q[2:3], [keys[2]], [32])
    st.fill_(_lib.KV_BAD_ROW)
    with pytest.raises(_lib.McError, match="no request"):
        kv.raise_on_status(st, "paged_attention")


def test_attention_repeats_bit_for_bit(cuda_ctx):
    lens = [9000, 17, 4000, 0, 333]
    q, cache, table, _ = attention_case(7, lens, 32, 8, 64, 16)
    ws = kv.paged_attention_workspace(64)
    first = None
    for _ in range(20):
        out = torch.empty_like(q)
        kv.paged_attention(cuda_ctx, q, cache, table, i32(lens), out, ws)
        first = out if first is None else first
        assert torch.equal(out.view(torch.int16), first.view(torch.int16))


def test_two_streams_with_a_workspace_each(cuda_ctx):
    from molten_b200 import lfm
    lens = [7000, 300, 64]
    q, cache, table, keys = attention_case(8, lens, 16, 4, 64, 16)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [lfm.Context(0, stream=s) for s in streams]
    outs = [[torch.empty_like(q) for _ in range(10)] for _ in range(2)]
    wss = [kv.paged_attention_workspace(64) for _ in range(2)]
    n = i32(lens)
    torch.cuda.synchronize()
    for i in range(10):
        for s in range(2):
            kv.paged_attention(ctxs[s], q, cache, table, n, outs[s][i], wss[s])
    torch.cuda.synchronize()
    check_attention(outs[0][0], None, q, keys, lens)
    for s in range(2):
        for o in outs[s]:
            assert torch.equal(o.view(torch.int16), outs[0][0].view(torch.int16))


def test_offsets_past_32_bits(cuda_ctx):
    """A cache of more than 2^32 elements: rows written to and read from its last pages."""
    K, bs, D, H = 8, 16, 64, 16
    blocks = 2 ** 32 // (K * bs * D) + 6
    c = kv.KvCache.empty(blocks, K, bs, D)
    T = 40
    g, q, k, v, qw, kw, _ = rope_case(11, T, H, K, D, False)
    pages = [blocks - 1, 0, blocks - 3]
    slots = torch.tensor([pages[t // bs] * bs + t % bs for t in range(T)], device="cuda")
    pos = torch.arange(T, device="cuda", dtype=I32)
    out = torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda")
    kv.qk_norm_rope(cuda_ctx, q, k, v, qw, kw, pos, kv.rope_turns(D).cuda(), out, c, slots)
    rows = [torch.cat([t[p] for p in pages], 1).transpose(0, 1)[:T] for t in (c.k, c.v)]
    want, size = ref.norm_rope(k, kw, pos, [1e6 ** (-2 * i / D) for i in range(D // 2)], D, False, 1e-5)
    assert bool(((rows[0].double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * ref.norm_rope_error(D) * size).all())
    assert torch.equal(rows[1], v)
    got = torch.empty(1, H, D, dtype=torch.bfloat16, device="cuda")
    kv.paged_attention(cuda_ctx, out[-1:], c, i32([pages]), i32([T]), got, kv.paged_attention_workspace(D))
    check_attention(got, None, out[-1:], [tuple(rows)], [T])


# ------------------------------------------------------------------ together

def test_a_batch_on_the_stream_of_its_context():
    """The bookkeeping's own tensors are made, cleared and read on the context's stream, whatever stream is current."""
    from molten_b200 import lfm
    ctx = lfm.Context(0, torch.cuda.Stream())
    try:
        for _ in range(20):
            batch = kv.PagedBatch(ctx, 3, 6, 4, 2)
            batch.plan()
            batch.check()
            assert batch.lens.tolist() == [1, 1, 1] and batch.slots.tolist() == [0, 4, 8]
            batch.clear()
            batch.plan()
            batch.check()
            assert batch.lens.tolist() == [1, 1, 1] and batch.block_table[:, 0].tolist() == [0, 1, 2]
            batch.plan(i32([8, 0, 0]))  # outgrows its table
            with pytest.raises(_lib.McError, match="outgrew"):
                batch.check()
    finally:
        ctx.close()


@pytest.mark.parametrize("fp8,captured", [(False, False), (True, False), (False, True)])
def test_a_served_batch(cuda_ctx, fp8, captured):
    """Prompts of uneven lengths, decode steps with a finished and a new
    request: plan, norm + rotation + store, attention, against a dense 64-bit
    attention over each request's whole history. Captured: one decode step,
    replayed while the lengths advance on the device."""
    H, K, D, bs, width, R = 8, 2, 64, 8, 12, 4
    g = gen(40)
    blocks = 40
    kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
    cache = kv.KvCache.empty(blocks, K, bs, D, kind)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x7f if fp8 else 0xff)
    table = torch.full((R, width), -1, dtype=I32, device="cuda")
    free = torch.randperm(blocks, generator=g, device="cuda").int()
    n_free, lens = i32([blocks]), i32([0] * R)
    turns = kv.rope_turns(D, 1e4).cuda()
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16) for _ in range(2))
    ws = kv.paged_attention_workspace(D)
    st = torch.zeros(1, dtype=I32, device="cuda")
    freqs = [1e4 ** (-2 * i / D) for i in range(D // 2)]
    history = [[] for _ in range(R)]  # each request's K and V as the cache holds them

    class Step:
        def __init__(self, T):
            self.x = torch.empty(T, (H + 2 * K) * D, dtype=torch.bfloat16, device="cuda")
            z = lambda n: torch.empty(n, dtype=I32, device="cuda")  # noqa: E731
            self.new, self.row_start, self.pos, self.req, self.kvl = z(R), z(R + 1), z(T), z(T), z(T)
            self.slots = torch.empty(T, dtype=torch.int64, device="cuda")
            self.q, self.out = (torch.empty(T, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))

        def run(self):
            T = self.x.shape[0]
            part = lambda a, n: self.x[:, a * D:(a + n) * D].view(T, n, D)  # noqa: E731
            kv.kv_plan(cuda_ctx, lens, self.new, bs, table, free, n_free, lens, n_free, self.row_start, self.pos, self.req,
                       self.kvl, self.slots, st)
            kv.qk_norm_rope(cuda_ctx, part(0, H), part(H, K), part(H + K, K), qw, kw, self.pos, turns, self.q, cache, self.slots,
                            status=st)
            kv.paged_attention(cuda_ctx, self.q, cache, table, self.kvl, self.out, ws, row_req=self.req, status=st)

    def check(s, new):
        t = 0
        for r in range(R):
            for _ in range(new[r]):
                row = s.x[t:t + 1]
                k, _ = ref.norm_rope(row[:, H * D:(H + K) * D].view(1, K, D), kw, i32([len(history[r])]), freqs, D, False, 1e-5)
                slot = s.slots[t].item()
                held = [c[slot // bs, :, slot % bs].double() for c in (cache.k, cache.v)]
                half = ref.E4M3_HALF if fp8 else ref.BF16_HALF
                assert bool(((held[0] - k[0]).abs() <= half * k[0].abs() + (2.0 ** -10 if fp8 else 0) + 1e-4).all())
                history[r].append(held)
                ks, vs = (torch.stack([h[i] for h in history[r]]) for i in range(2))
                want, _, e, _ = ref.attention(s.q[t], ks, vs, D ** -0.5)
                assert bool(((s.out[t].double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * e).all()), (r, t)
                t += 1
        for u in range(t, s.x.shape[0]):
            assert s.slots[u].item() == -1 and bool((s.out[u] == 0).all())

    prompt = Step(40)
    new = [13, 0, 8, 1]
    prompt.new.copy_(i32(new))
    prompt.x.normal_(generator=g)
    prompt.run()
    check(prompt, new)
    step, graph = Step(R), None
    for i in range(12):
        new = [1, 0, 1, 1]
        if i == 5:  # request 2 is done; request 1 starts in its pages
            kv.kv_release(cuda_ctx, i32([0, 0, 1, 0]), lens, bs, table, free, n_free, lens, n_free, st)
            history[2] = []
        if i >= 5:
            new = [1, 1, 0, 1]
        step.new.copy_(i32(new))
        step.x.normal_(generator=g)
        if captured and i == 2:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
                step.run()
            torch.cuda.current_stream().wait_stream(side)
        graph.replay() if graph else step.run()
        check(step, new)
    assert st.item() == 0
    assert lens.tolist() == [len(h) for h in history]
    held = [p for r in range(R) for p in table[r, :-(-lens[r].item() // bs)].tolist()]
    assert sorted(held + free[:n_free.item()].tolist()) == list(range(blocks)), "every page is held once or free"
