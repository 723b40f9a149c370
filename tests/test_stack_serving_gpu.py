"""The decode stack with attention layers and rules on logits
(molten_b200.stack): every step equals the same public calls made one by one,
bit for bit, eagerly and captured in a CUDA graph; the attention inside agrees
with a 64-bit statement over the request's history."""
import numpy as np
import pytest
import torch

from molten_b200 import _lib, kv, lfm, sample, synth
from molten_b200.stack import DecodeStack
from tests import serving_ref as ref
from tests.gpu_util import dev_bf16, dev_qw

pytestmark = pytest.mark.gpu

H, D, HEADS, KV_HEADS, E, I, V, BS = 2048, 64, 32, 8, 8, 512, 4096, 8


def make_layers(seed, n, attn_in, blocks, dtype):
    g = synth.rng(seed)
    layers = []
    for i in range(n):
        L = dict(proj=dev_qw(*synth.quant_weights_np(g, H, H)), norm_w=dev_bf16(synth.norm_weight_np(g)),
                 router=dev_bf16(synth.router_np(g, E)), gate=dev_qw(*synth.quant_weights_np(g, E * I, H)),
                 up=dev_qw(*synth.quant_weights_np(g, E * I, H)), down=dev_qw(*synth.quant_weights_np(g, E * H, I)))
        if i in attn_in:
            c = kv.KvCache.empty(blocks, KV_HEADS, BS, D, dtype)
            for t in (c.k, c.v):
                t.view(torch.uint8).fill_(0x7f)
            gain = lambda: dev_bf16(synth.f32_to_bf16_bits(g.normal(1, 0.1, D).astype(np.float32)))  # noqa: E731
            L["attn"] = dict(norm_w=dev_bf16(synth.norm_weight_np(g)),
                             qkv=dev_qw(*synth.quant_weights_np(g, (HEADS + 2 * KV_HEADS) * D, H)), q_norm=gain(), k_norm=gain(),
                             cache=c)
        layers.append(L)
    return layers, dev_qw(*synth.quant_weights_np(g, V, H, 6), bits=6), dev_bf16(synth.activations_np(g, V, H))


def make_rules(B, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    one = lambda v: torch.full((B,), v, device="cuda")  # noqa: E731
    r = sample.LogitsRules(seen=torch.zeros(B, V // 32, dtype=torch.int32, device="cuda"), repetition=one(1.3),
                           counts=torch.zeros(B, V, dtype=torch.int16, device="cuda"), frequency=one(0.5), presence=one(0.25))
    r.allowed = torch.randint(-2 ** 31, 2 ** 31, (1, V // 32), generator=g, device="cuda", dtype=torch.int64).int()
    r.allowed_row = torch.tensor([0] + [-1] * (B - 1), dtype=torch.int32, device="cuda")
    return r


class ByHand:
    """The stack's step in public calls, on buffers of its own."""

    def __init__(self, ctx, layers, head, embed, B, width, blocks, rules):
        self.ctx, self.layers, self.head, self.embed, self.B, self.rules = ctx, layers, head, embed, B, rules
        self.kv = kv.PagedBatch(ctx, B, blocks, BS, width)
        self.caches = [kv.KvCache(L["attn"]["cache"].k.clone(), L["attn"]["cache"].v.clone()) if "attn" in L else None
                       for L in layers]
        self.seen_q = {}

    def step(self, tokens):
        ctx, B = self.ctx, self.B
        bf = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        x = self.embed[tokens.long()]
        self.kv.plan()
        for n, L in enumerate(self.layers):
            p, mix = bf(B, H), x
            if "attn" in L:
                A = L["attn"]
                normed, rows = bf(B, H), bf(B, (HEADS + 2 * KV_HEADS) * D)
                lfm.add_rmsnorm(ctx, x, None, A["norm_w"], None, normed)
                lfm.gemv_quant(ctx, A["qkv"], normed, rows)
                q, k, v = (t.reshape(B, -1, D) for t in rows.split([HEADS * D, KV_HEADS * D, KV_HEADS * D], 1))
                kv.qk_norm_rope(ctx, q, k, v, A["q_norm"], A["k_norm"], self.kv.positions, kv.rope_turns(D, 1e6).cuda(), q,
                                self.caches[n], self.kv.slots)
                out = bf(B, HEADS, D)
                kv.paged_attention(ctx, q, self.caches[n], self.kv.block_table, self.kv.kv_lens, out,
                                   kv.paged_attention_workspace(D))
                self.seen_q[n] = (q, out)
                mix = out.view(B, H)
            lfm.gemv_quant(ctx, L["proj"], mix, p)
            hout, normed, logits, ids, wts = bf(B, H), bf(B, H), torch.empty(B, E, device="cuda"), i32(B, 4), bf(B, 4)
            lfm.router_addnorm_route(ctx, x, p, L["norm_w"], hout, normed, L["router"], logits, None, ids, wts, i32(B))
            act, nxt = bf(B, 4, I), bf(B, H)
            lfm.gemv_gather_act(ctx, L["gate"], L["up"], normed, ids, act, n_experts=E)
            lfm.gemv_gather_down_combine4(ctx, L["down"], act, ids, wts, nxt, n_experts=E)
            x = nxt
        y = bf(B, V)
        lfm.gemv_quant(ctx, self.head, x, y)
        best, tok = torch.zeros(B, dtype=torch.int64, device="cuda"), i32(B)
        if self.rules is not None:
            sample.logits_process(ctx, y, y, self.rules, best)
            lfm.token_tail(ctx, best, tok)
            sample.logits_mark(ctx, tok, self.rules, V)
        else:
            lfm.argmax_bf16(ctx, y, tok)
        return tok


@pytest.mark.parametrize("B,fused,dtype,with_rules", [(1, True, torch.bfloat16, False), (1, False, torch.bfloat16, True),
                                                      (3, False, torch.bfloat16, True), (4, False, torch.float8_e4m3fn, False)])
def test_stack_with_attention_and_rules(cuda_ctx, B, fused, dtype, with_rules):
    blocks, width, steps = 4 * B + 1, 4, 13
    layers, head, embed = make_layers(200 + B, 3, (0, 2), blocks, dtype)
    start = torch.arange(B, dtype=torch.int32, device="cuda") * 91 + 5
    hand = ByHand(cuda_ctx, layers, head, embed, B, width, blocks, make_rules(B, 1) if with_rules else None)
    batch = kv.PagedBatch(cuda_ctx, B, blocks, BS, width)
    st = DecodeStack(cuda_ctx, layers, head, embed, B, n_experts=E, moe_path="fused" if B == 1 else "gemv", fuse_proj=fused,
                     kv=batch, rules=make_rules(B, 1) if with_rules else None)
    assert st.launches_per_step() == 3 * {(1, True): 1, (1, False): 2}.get((B, fused), 4) + 2 + 1 + 2 * (4 + fused) + 2 * with_rules
    st.start(start)
    toks, graph = start, None
    for s in range(steps):
        toks = hand.step(toks)
        if s == 4:
            graph = torch.cuda.CUDAGraph()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
                st.step()
            torch.cuda.current_stream().wait_stream(side)
        graph.replay() if graph else st.step()
        assert torch.equal(st.read_tokens(), toks.cpu()), f"step {s}"
        assert batch.lens.tolist() == [s + 1] * B
    for n in (0, 2):
        q, out = hand.seen_q[n]
        c = hand.caches[n]
        for b in range(B):
            at = torch.arange(steps, device="cuda")
            page = batch.block_table[b].long()[at // BS]
            k, v = c.k[page, :, at % BS], c.v[page, :, at % BS]
            want, _, e, _ = ref.attention(q[b], k, v, D ** -0.5)
            assert bool(((out[b].double() - want).abs() <= ref.BF16_HALF * want.abs() + 1.01 * e).all())
    # a request outgrows its block table: refused, and the stack says so
    for s in range(steps, width * BS):
        graph.replay()
    st.check()
    graph.replay()
    with pytest.raises(_lib.McError, match="outgrew"):
        st.check()
    assert batch.lens.tolist() == [width * BS] * B
    batch.clear()
    st.start(start)
    st.step()
    st.check()
    assert batch.lens.tolist() == [1] * B


def test_sampled_stack_under_a_grammar(cuda_ctx):
    """temperature > 0: the draw only meets tokens that the mask allows."""
    layers, head, embed = make_layers(300, 1, (0,), 5, torch.bfloat16)
    allow = torch.zeros(V, dtype=torch.bool)
    allow[[3, 700, 4095, 64, 65]] = True
    words = torch.zeros(1, V // 32, dtype=torch.int64)
    for t in torch.nonzero(allow)[:, 0].tolist():
        words[0, t // 32] |= 1 << (t % 32)
    rules = sample.LogitsRules(allowed=torch.where(words >= 2 ** 31, words - 2 ** 32, words).int().cuda())
    st = DecodeStack(cuda_ctx, layers, head, embed, 1, n_experts=E, sampling=sample.Sampling(temperature=50.0, seed=3),
                     kv=kv.PagedBatch(cuda_ctx, 1, 5, BS, 5), rules=rules)
    st.start(torch.tensor([9], dtype=torch.int32, device="cuda"))
    got = set()
    for _ in range(30):
        st.step()
        got.add(st.read_tokens().item())
    assert got <= {3, 64, 65, 700, 4095} and len(got) > 1


def test_stack_refusals(cuda_ctx):
    layers, head, embed = make_layers(301, 1, (0,), 5, torch.bfloat16)
    with pytest.raises(ValueError, match="PagedBatch"):
        DecodeStack(cuda_ctx, layers, head, embed, 1, n_experts=E)
    with pytest.raises(ValueError, match="one token row"):
        DecodeStack(cuda_ctx, layers, head, embed, 2, n_experts=E, kv=kv.PagedBatch(cuda_ctx, 3, 5, BS, 5))
    with pytest.raises(ValueError, match="shapes"):
        DecodeStack(cuda_ctx, layers, head, embed, 1, n_experts=E, kv=kv.PagedBatch(cuda_ctx, 1, 5, BS + 1, 5))
