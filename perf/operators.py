"""Timed cases of the serving operators: the cache's bookkeeping (kv_plan, kv_release), the norm
and rotation of queries and keys with the cache write (qk_norm_rope), attention of new tokens over
the paged cache (paged_attention) and the rules on logits (logits_process).

``run`` computes a case in plain torch operations, or, where ``own`` is true, with the calls of
molten_b200. Head layouts and vocabularies are those of this repository's tests (32 query and 8
KV heads of 64, vocabularies of 65536 and 128000) and generic ones next to them.
"""
import math

import torch

own = False

DEV = "cuda"


def listed():
    plan, rope, attn, rules = "kv_plan", "qk_norm_rope", "paged_attention", "logits_process"
    return [
        # one token for each of eight requests: the bookkeeping of an interactive decode step
        dict(name="plan_step_8", op=plan, reqs=8, block=16, longest=2048, prompt=0, release=False),
        # a full server's step: 256 requests, some of them finished since the last step
        dict(name="plan_step_256", op=plan, reqs=256, block=16, longest=8192, prompt=0, release=True),
        # admission of a batch of prompts of uneven lengths
        dict(name="plan_prompts_48", op=plan, reqs=48, block=32, longest=64, prompt=1500, release=False),
        # the decode step of one sequence
        dict(name="rope_1", op=rope, tokens=1, heads=32, kv_heads=8, dim=64, rot=64, inter=False, fp8=False, far=2000),
        # a batched step with an 8-bit cache, far into long contexts
        dict(name="rope_61_fp8", op=rope, tokens=61, heads=32, kv_heads=8, dim=128, rot=128, inter=True, fp8=True, far=120000),
        # a prompt's rows
        dict(name="rope_4096", op=rope, tokens=4096, heads=32, kv_heads=8, dim=64, rot=64, inter=False, fp8=False, far=8192),
        # the first answer token after a short prompt: latency
        dict(name="attn_1_short", op=attn, rows=1, per=1, shortest=100, longest=100, heads=32, kv_heads=8, dim=64, block=16, fp8=False, window=0),
        # one sequence at the far end of a long context
        dict(name="attn_1_long", op=attn, rows=1, per=1, shortest=131071, longest=131071, heads=32, kv_heads=8, dim=64, block=16, fp8=False, window=0),
        # a batch of uneven contexts
        dict(name="attn_32_ragged", op=attn, rows=32, per=1, shortest=17, longest=6000, heads=32, kv_heads=8, dim=64, block=16, fp8=False, window=0),
        # a full server with an 8-bit cache and wider heads
        dict(name="attn_64_fp8", op=attn, rows=64, per=1, shortest=4000, longest=8200, heads=64, kv_heads=8, dim=128, block=32, fp8=True, window=0),
        # one sequence's logits with penalties, a few biased tokens and a grammar
        dict(name="rules_1", op=rules, rows=1, vocab=65536, f32=False, penalties=True, biased=20, grammar=True),
        # a batch of requests over a wide vocabulary
        dict(name="rules_48", op=rules, rows=48, vocab=128000, f32=False, penalties=True, biased=300, grammar=True),
    ]


def _log(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(("kv_plan", "qk_norm_rope", "paged_attention", "paged_attention", "logits_process"))
    if op == "kv_plan":
        prompt = rng.choice((0, 0, 1)) and _log(rng, 2, 2000)
        return dict(op=op, reqs=_log(rng, 1, 512 if not prompt else 64), block=rng.choice((8, 16, 24, 32, 64, 128)),
                    longest=_log(rng, 16, 16384), prompt=prompt, release=rng.random() < 0.5)
    if op == "qk_norm_rope":
        dim = rng.choice((64, 64, 128))
        kv = rng.choice((1, 2, 4, 8))
        return dict(op=op, tokens=_log(rng, 1, 4096), heads=kv * rng.choice((1, 2, 4)), kv_heads=kv, dim=dim,
                    rot=rng.choice((dim, dim, dim // 2)), inter=rng.random() < 0.4, fp8=rng.random() < 0.4, far=_log(rng, 5, 1000000))
    if op == "paged_attention":
        dim, kv = rng.choice((64, 64, 128)), rng.choice((1, 2, 4, 8))
        rows = _log(rng, 1, 128)
        fp8 = rng.random() < 0.4
        most = min(131072, (1 << 29) // (rows * kv * dim))
        longest = _log(rng, min(32, most), most)
        return dict(op=op, rows=rows, per=rng.choice((1, 1, 1, 2, 4)), shortest=rng.choice((0, longest // 3, longest)), longest=longest,
                    heads=kv * rng.choice((1, 2, 4, 6, 8)), kv_heads=kv, dim=dim, block=rng.choice((1, 8, 16, 16, 20, 32, 64, 256)), fp8=fp8,
                    window=rng.choice((0, 0, 0, 4096, 500)))
    return dict(op=op, rows=_log(rng, 1, 48), vocab=_log(rng, 1000, 128000), f32=rng.random() < 0.3, penalties=rng.random() < 0.7,
                biased=rng.choice((0, 3, 300)), grammar=rng.random() < 0.6)


# ------------------------------------------------------------------ inputs

_held = {}


def _context():
    """The library context that a program makes once."""
    if "ctx" not in _held:
        from molten_b200 import lfm
        _held["ctx"] = lfm.Context(0)
    return _held["ctx"]


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32, device=DEV)


def _ceil(a, b):
    return (a + b - 1) // b


def _lens(g, n, low, high):
    if low >= high:
        return torch.full((n,), high, dtype=torch.int32, device=DEV)
    return torch.randint(low, high + 1, (n,), generator=g, device=DEV, dtype=torch.int32)


def _prepare_plan(c, g):
    R, bs = c["reqs"], c["block"]
    most_new = max(1, c["prompt"])
    width = _ceil(c["longest"] + most_new, bs)
    blocks = R * width + 7
    lens = _lens(g, R, 0, c["longest"])
    new = _lens(g, R, 1, most_new)
    order = torch.randperm(blocks, generator=g, device=DEV).int()
    have = _ceil(lens.long(), bs)
    column = torch.arange(width, device=DEV)
    held = column[None, :] < have[:, None]
    at = torch.cumsum(have, 0)[:, None] - have[:, None] + column[None, :]
    table = torch.where(held, order[at.clamp(max=blocks - 1)], torch.full_like(at, -1, dtype=torch.int32))
    n_free = (blocks - have.sum()).int().reshape(1)
    # the free list is a stack: its first n_free entries are free
    free = order.flip(0).contiguous()
    total = R * most_new
    s = dict(lens=lens, new=new, table=table.contiguous(), free=free, n_free=n_free, blocks=blocks, seq=_i32(R), n_free_out=_i32(1),
             row_start=_i32(R + 1), positions=_i32(total), token_req=_i32(total), kv_lens=_i32(total),
             slots=torch.zeros(total, dtype=torch.int64, device=DEV), done=None, lens_mid=_i32(R), n_free_mid=_i32(1))
    # the program's table: a pass finds it as the last one left it, the plan writes the same entries again
    s["table_out"] = s["table"].clone()
    if c["release"]:
        s["done"] = (torch.rand(R, generator=g, device=DEV) < 0.1).int()
    return s


def _rows_bf16(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(torch.bfloat16)


def _prepare_rope(c, g):
    T, H, K, D, bs = c["tokens"], c["heads"], c["kv_heads"], c["dim"], 16
    qkv = _rows_bf16(g, T, (H + 2 * K) * D)  # one row of the fused projection for each token
    blocks = _ceil(T, bs) + 1
    kind = torch.float8_e4m3fn if c["fp8"] else torch.bfloat16
    slots = torch.randperm(blocks * bs, generator=g, device=DEV)[:T]
    norm = lambda: (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(torch.bfloat16)  # noqa: E731
    s = dict(q=qkv[:, :H * D].view(T, H, D), k=qkv[:, H * D:(H + K) * D].view(T, K, D), v=qkv[:, (H + K) * D:].view(T, K, D),
             qw=norm(), kw=norm(), positions=torch.randint(0, c["far"], (T,), generator=g, device=DEV, dtype=torch.int32), theta=1e6,
             slots=slots, q_out=torch.empty(T, H, D, dtype=torch.bfloat16, device=DEV),
             kc=_rows_bf16(g, blocks, K, bs, D).to(kind), vc=_rows_bf16(g, blocks, K, bs, D).to(kind), ks=None, vs=None)
    if c["fp8"]:
        s["ks"] = 0.01 + 0.02 * torch.rand(K, generator=g, device=DEV)
        s["vs"] = 0.01 + 0.02 * torch.rand(K, generator=g, device=DEV)
    if own:
        from molten_b200 import kv
        s["ctx"] = _context()
        s["turns"] = kv.rope_turns(c["rot"], s["theta"]).to(DEV)
        s["cache"] = kv.KvCache(s["kc"], s["vc"], s["ks"], s["vs"])
    return s


def _prepare_attn(c, g):
    per, bs, H, K, D = c["per"], c["block"], c["heads"], c["kv_heads"], c["dim"]
    R = _ceil(c["rows"], per)  # requests; `per` query rows each (draft tokens)
    width = _ceil(c["longest"], bs)
    blocks = R * width + 1
    q = _rows_bf16(g, c["rows"], H, D, scale=1.5)
    kind = torch.float8_e4m3fn if c["fp8"] else torch.bfloat16
    big = 8.0 if c["fp8"] else 1.0
    kc = torch.empty(blocks, K, bs, D, dtype=torch.bfloat16, device=DEV).normal_(0, big, generator=g).to(kind)
    vc = torch.empty(blocks, K, bs, D, dtype=torch.bfloat16, device=DEV).normal_(0, big, generator=g).to(kind)
    table = torch.randperm(blocks, generator=g, device=DEV)[:R * width].int().view(R, width).contiguous()
    lens = _lens(g, R, c["shortest"], c["longest"])
    req = torch.arange(c["rows"], device=DEV, dtype=torch.int32) // per
    back = per - 1 - torch.arange(c["rows"], device=DEV, dtype=torch.int32) % per
    rows = (lens[req.long()] - back).clamp(min=0).int()
    s = dict(q=q, kc=kc, vc=vc, table=table, lens=rows, req=req if per > 1 else None, scale=1 / math.sqrt(D), ks=None, vs=None,
             out=torch.empty_like(q), lse=torch.empty(c["rows"], H, device=DEV))
    if c["fp8"]:
        s["ks"] = (0.5 + torch.rand(K, generator=g, device=DEV)) / big
        s["vs"] = (0.5 + torch.rand(K, generator=g, device=DEV)) / big
    if own:
        from molten_b200 import kv
        s["ctx"] = _context()
        s["cache"] = kv.KvCache(kc, vc, s["ks"], s["vs"])
        s["ws"] = kv.paged_attention_workspace(D, DEV)
    return s


def _prepare_rules(c, g):
    B, V = c["rows"], c["vocab"]
    words = _ceil(V, 32)
    logits = torch.randn(B, V, generator=g, device=DEV) * 3
    s = dict(logits=logits if c["f32"] else logits.to(torch.bfloat16), seen=None, counts=None, rep=None, freq=None, pres=None, start=None,
             ids=None, vals=None, allowed=None)
    s["out"] = torch.empty_like(s["logits"])
    s["token"] = _i32(B)
    u32 = lambda *shape: torch.randint(-2 ** 31, 2 ** 31, shape, generator=g, device=DEV, dtype=torch.int64).int()  # noqa: E731
    if c["penalties"]:
        s["seen"] = u32(B, words) & u32(B, words) & u32(B, words) & u32(B, words)
        s["counts"] = torch.where(torch.rand(B, V, generator=g, device=DEV) < 0.01, 1 + torch.randint(0, 5, (B, V), generator=g, device=DEV), 0).short()
        s["rep"] = 1 + 0.3 * torch.rand(B, generator=g, device=DEV)
        s["freq"], s["pres"] = (torch.rand(B, generator=g, device=DEV) for _ in range(2))
    if c["biased"]:
        n = c["biased"]
        s["start"] = (torch.arange(B + 1, device=DEV) * n).int()
        s["ids"] = torch.rand(B, V, generator=g, device=DEV).argsort(1)[:, :n].sort(1).values.int().reshape(-1).contiguous()
        s["vals"] = torch.randn(B * n, generator=g, device=DEV) * 4
    if c["grammar"]:
        s["allowed"] = u32(B, words) | u32(B, words)
        s["allowed"][:, 0] |= 1
    if own:
        from molten_b200 import sample
        s["ctx"] = _context()
        s["rules"] = sample.LogitsRules(seen=s["seen"], counts=s["counts"], repetition=s["rep"], frequency=s["freq"], presence=s["pres"],
                                        bias_start=s["start"], bias_ids=s["ids"], bias_values=s["vals"], allowed=s["allowed"])
        s["best"] = torch.zeros(B, dtype=torch.int64, device=DEV)
    return s


_PREPARE = {"kv_plan": _prepare_plan, "qk_norm_rope": _prepare_rope, "paged_attention": _prepare_attn, "logits_process": _prepare_rules}


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = _PREPARE[case["op"]](case, g)
    s["case"] = case
    if own:
        s["ctx"] = _context()
    return s


# ------------------------------------------------------------------ plain forms

def _plain_release(s):
    bs, R = s["case"]["block"], s["lens"].numel()
    done = s["done"] != 0
    have = torch.where(done, _ceil(s["lens"].long(), bs), 0)
    first = torch.cumsum(have, 0) - have
    column = torch.arange(s["table"].shape[1], device=DEV)
    held = column[None, :] < have[:, None]
    at = torch.where(held, s["n_free"].long() + first[:, None] + column[None, :], s["blocks"])
    room = torch.cat((s["free"], s["free"][:1]))
    free = room.scatter(0, at.reshape(-1), s["table"].reshape(-1))[:-1]
    return torch.where(done, 0, s["lens"]), (s["n_free"] + have.sum()).int(), free


def _plain_plan(s):
    bs = s["case"]["block"]
    lens, n_free, free = s["lens"], s["n_free"], s["free"]
    if s["done"] is not None:
        lens, n_free, free = _plain_release(s)
    lens, new, table = lens.long(), s["new"].long(), s["table"]
    R, width = table.shape
    total = s["slots"].numel()
    ends = torch.cumsum(new, 0)
    have, want = _ceil(lens, bs), _ceil(lens + new, bs)
    fits = (want <= width) & (ends <= total)
    need = torch.where(fits, want - have, 0)
    taken = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (taken <= n_free))
    seq = torch.where(ok, lens + new, lens)
    used = torch.where(ok & (need > 0), taken, 0).max()
    column = torch.arange(width, device=DEV)[None, :]
    fresh = ok[:, None] & (column >= have[:, None]) & (column < want[:, None])
    at = n_free.long() - 1 - (taken - need)[:, None] - (column - have[:, None])
    table = torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table)
    t = torch.arange(total, device=DEV)
    req = torch.searchsorted(ends, t, right=True)
    live = req < R
    r = req.clamp(max=R - 1)
    pos = lens[r] + t - (ends - new)[r]
    page = table.reshape(-1)[(r * width + (pos // bs).clamp(max=width - 1))].long()
    written = live & ok[r]
    return dict(seq=seq.int(), n_free=(n_free - used).int(), table=table, free=free, row_start=torch.cat((torch.zeros_like(ends[:1]), ends)).int(),
                positions=torch.where(live, pos, 0).int(), token_req=torch.where(live, req, -1).int(),
                kv_lens=torch.where(written, pos + 1, 0).int(), slots=torch.where(written, page * bs + pos % bs, -1))


def _plain_turn(x, w, positions, theta, rot, inter, eps=1e-5):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.float()
    f = theta ** (torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / -rot)
    angle = positions.double()[:, None] * f[None, :]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    part = x[..., :rot]
    a, b = (part[..., 0::2], part[..., 1::2]) if inter else (part[..., :rot // 2], part[..., rot // 2:])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((c, d), -1).flatten(-2) if inter else torch.cat((c, d), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_store(cache, slots, rows, scale):
    bs = cache.shape[2]
    if scale is not None:
        rows = (rows / scale[None, :, None]).clamp(-448, 448)
    rows = rows.to(cache.dtype)
    page, off = slots // bs, slots % bs
    if cache.dtype == torch.bfloat16:
        cache[page, :, off] = rows
    else:
        cache.view(torch.uint8)[page, :, off] = rows.view(torch.uint8)


def _plain_rope(s):
    c = s["case"]
    q = _plain_turn(s["q"], s["qw"], s["positions"], s["theta"], c["rot"], c["inter"]).to(torch.bfloat16)
    k = _plain_turn(s["k"], s["kw"], s["positions"], s["theta"], c["rot"], c["inter"])
    _plain_store(s["kc"], s["slots"], k, s["ks"])
    _plain_store(s["vc"], s["slots"], s["v"].float(), s["vs"])
    return dict(q=q, k=s["kc"], v=s["vc"])


def _plain_attn(s):
    c = s["case"]
    rows, H, D = s["q"].shape
    K, bs = c["kv_heads"], c["block"]
    table = s["table"] if s["req"] is None else s["table"][s["req"].long()]
    long = table.shape[1] * bs
    k = s["kc"][table.long()].float().permute(0, 2, 1, 3, 4).reshape(rows, K, long, D)
    v = s["vc"][table.long()].float().permute(0, 2, 1, 3, 4).reshape(rows, K, long, D)
    q = s["q"].float().view(rows, K, H // K, D)
    score = (q @ k.transpose(-1, -2)) * s["scale"]
    if s["ks"] is not None:
        score = score * s["ks"][None, :, None, None]
    j = torch.arange(long, device=DEV)[None, :]
    n = s["lens"].long()[:, None]
    seen = j < n
    if c["window"]:
        seen &= j >= n - c["window"]
    score = torch.where(seen[:, None, None, :], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, 1.0, total)
    if s["vs"] is not None:
        out = out * s["vs"][None, :, None, None]
    lse = torch.log(total) + top
    return dict(out=out.view(rows, H, D).to(torch.bfloat16), lse=lse.view(rows, H))


def _bits(words, vocab):
    j = torch.arange(vocab, device=DEV)
    return (words[:, j // 32] >> (j % 32).int()) & 1 != 0


def _plain_rules(s):
    v = s["logits"].float()
    V = v.shape[1]
    if s["rep"] is not None:
        rep = s["rep"][:, None]
        v = torch.where(_bits(s["seen"], V), torch.where(v > 0, v / rep, v * rep), v)
        n = s["counts"].float()
        v = v - s["freq"][:, None] * n - torch.where(n > 0, s["pres"][:, None], 0.0)
    if s["ids"] is not None:
        at = s["ids"].long().view(v.shape[0], -1)
        v = v.scatter_add(1, at, s["vals"].view(v.shape[0], -1))
    if s["allowed"] is not None:
        v = torch.where(_bits(s["allowed"], V), v, float("-inf"))
    out = v.to(s["logits"].dtype)
    j = torch.arange(V, device=DEV)[None, :]
    token = torch.where(out == out.amax(-1, keepdim=True), j, V).amin(-1)  # ties to the lowest index
    return dict(out=out, token=token.int())


# ------------------------------------------------------------------ the framework's calls

def _own_plan(s):
    from molten_b200 import kv
    bs, lens, n_free = s["case"]["block"], s["lens"], s["n_free"]
    if s["done"] is not None:
        kv.kv_release(s["ctx"], s["done"], lens, bs, s["table"], s["free"], n_free, s["lens_mid"], s["n_free_mid"])
        lens, n_free = s["lens_mid"], s["n_free_mid"]
    kv.kv_plan(s["ctx"], lens, s["new"], bs, s["table_out"], s["free"], n_free, s["seq"], s["n_free_out"], s["row_start"], s["positions"],
               s["token_req"], s["kv_lens"], s["slots"])
    return dict(seq=s["seq"], n_free=s["n_free_out"], table=s["table_out"], free=s["free"], row_start=s["row_start"], positions=s["positions"],
                token_req=s["token_req"], kv_lens=s["kv_lens"], slots=s["slots"])


def _own_rope(s):
    from molten_b200 import kv
    kv.qk_norm_rope(s["ctx"], s["q"], s["k"], s["v"], s["qw"], s["kw"], s["positions"], s["turns"], s["q_out"], s["cache"], s["slots"],
                    interleaved=s["case"]["inter"])
    return dict(q=s["q_out"], k=s["kc"], v=s["vc"])


def _own_attn(s):
    from molten_b200 import kv
    kv.paged_attention(s["ctx"], s["q"], s["cache"], s["table"], s["lens"], s["out"], s["ws"], scale=s["scale"], row_req=s["req"],
                       window=s["case"]["window"], lse=s["lse"])
    return dict(out=s["out"], lse=s["lse"])


def _own_rules(s):
    from molten_b200 import lfm, sample
    sample.logits_process(s["ctx"], s["logits"], s["out"], s["rules"], s["best"])
    lfm.token_tail(s["ctx"], s["best"], s["token"])
    return dict(out=s["out"], token=s["token"])


_PLAIN = {"kv_plan": _plain_plan, "qk_norm_rope": _plain_rope, "paged_attention": _plain_attn, "logits_process": _plain_rules}
_OWN = {"kv_plan": _own_plan, "qk_norm_rope": _own_rope, "paged_attention": _own_attn, "logits_process": _own_rules}


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ work and exact values

def work(case):
    c = case
    if c["op"] == "kv_plan":
        R = c["reqs"]
        most = max(1, c["prompt"])
        width = _ceil(c["longest"] + most, c["block"])
        mean = R * (most + 1) / 2
        # lengths, counts and sums of the requests, the fresh table entries, 20 bytes of maps a token
        return dict(bytes=R * 16 + 8 * (mean / c["block"] + R) + 4 * mean + 20 * R * most + (4 * R * width * 0.1 if c["release"] else 0),
                    flops=0)
    if c["op"] == "qk_norm_rope":
        n = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        out = c["heads"] * c["dim"] * 2 + 2 * c["kv_heads"] * c["dim"] * (1 if c["fp8"] else 2)
        return dict(bytes=c["tokens"] * (2 * n + out + 12), flops=c["tokens"] * n * 8)
    if c["op"] == "paged_attention":
        R = _ceil(c["rows"], c["per"])
        mean = (c["shortest"] + c["longest"]) / 2
        if c["window"]:
            mean = min(mean, c["window"] + c["per"])
        page = 2 * c["kv_heads"] * c["dim"] * (1 if c["fp8"] else 2)
        return dict(bytes=R * mean * page + R * _ceil(int(mean), c["block"]) * 4 + c["rows"] * c["heads"] * (c["dim"] * 4 + 4),
                    flops=c["rows"] * mean * 4 * c["heads"] * c["dim"])
    V = c["vocab"]
    each = (8 if c["f32"] else 4) + (2.125 if c["penalties"] else 0) + (0.125 if c["grammar"] else 0)
    return dict(bytes=c["rows"] * (V * each + 8 * c["biased"]), flops=c["rows"] * V * 6)


def exact(case, seed):
    """The operators' definitions in 64 bits, request by request and head by head."""
    if case["op"] == "kv_plan":
        return None
    s = prepare(case, seed)
    return {"qk_norm_rope": _exact_rope, "paged_attention": _exact_attn, "logits_process": _exact_rules}[case["op"]](case, s)


def _exact_rope(c, s):
    rot, D, bs = c["rot"], c["dim"], s["kc"].shape[2]
    half = rot // 2
    pairs = [(2 * i, 2 * i + 1) if c["inter"] else (i, i + half) for i in range(half)]
    first, second = [a for a, _ in pairs], [b for _, b in pairs]
    freq = torch.tensor([math.exp(-2 * i / rot * math.log(s["theta"])) for i in range(half)], dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.ones_like(freq)[None, :], s["positions"].double()[:, None] * freq)[:, None, :]

    def normed_and_turned(x, w):
        x = x.double()
        y = w.double() * x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + 1e-5)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    def stored(cache, rows, scale):
        flat = cache.double().transpose(1, 2).reshape(-1, c["kv_heads"], D)  # [slot][head][dim]
        flat[s["slots"]] = rows if scale is None else torch.clamp(rows / scale.double()[:, None], -448.0, 448.0)
        return flat.view(-1, bs, c["kv_heads"], D).transpose(1, 2)

    return dict(q=normed_and_turned(s["q"], s["qw"]), k=stored(s["kc"], normed_and_turned(s["k"], s["kw"]), s["ks"]),
                v=stored(s["vc"], s["v"].double(), s["vs"]))


def _exact_attn(c, s):
    rows, H, D = s["q"].shape
    group = H // c["kv_heads"]
    out = torch.zeros(rows, H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((rows, H), float("-inf"), dtype=torch.float64, device=DEV)
    lens, req = s["lens"].tolist(), list(range(rows)) if s["req"] is None else s["req"].tolist()
    for r in range(rows):
        n = lens[r]
        low = max(0, n - c["window"]) if c["window"] else 0
        if n <= low:
            continue
        at = torch.arange(low, n, device=DEV)
        page, off = s["table"][req[r]].long()[at // c["block"]], at % c["block"]
        k, v = s["kc"][page, :, off].double(), s["vc"][page, :, off].double()  # [token][head][dim]
        if s["ks"] is not None:
            k, v = k * s["ks"].double()[:, None], v * s["vs"].double()[:, None]
        q = s["q"][r].double().view(-1, group, D)
        score = torch.einsum("hgd,thd->hgt", q, k) * s["scale"]
        lse[r] = torch.logsumexp(score, -1).reshape(-1)
        out[r] = torch.einsum("hgt,thd->hgd", torch.softmax(score, -1), v).reshape(H, D)
    return dict(out=out, lse=lse)


def _exact_rules(c, s):
    out = s["logits"].double().clone()
    for b in range(c["rows"]):
        row = out[b]
        if s["rep"] is not None:
            there = _bits(s["seen"][b:b + 1], c["vocab"])[0]
            rep = s["rep"][b].double()
            row[there] = torch.where(row[there] > 0, row[there] / rep, row[there] * rep)
            n = s["counts"][b].double()
            row -= s["freq"][b].double() * n + s["pres"][b].double() * (n > 0)
        if s["ids"] is not None:
            low, high = s["start"][b].item(), s["start"][b + 1].item()
            row[s["ids"][low:high].long()] += s["vals"][low:high].double()
        if s["allowed"] is not None:
            row[~_bits(s["allowed"][b:b + 1], c["vocab"])[0]] = float("-inf")
    return dict(out=out, token=None)
