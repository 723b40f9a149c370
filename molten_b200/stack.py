"""The stacked decode loop of BASELINE cfg4 on the decode kernels.

One decode step for a batch of B tokens (rows x [B, 2048], each the
embedding row of the token being decoded):

    for each of the L layers:
        p   = proj_l(x)                             Q4 2048x2048 GEMV (gemv_quant)
        out = MoE_l(h = x, b = p)                   add + RMSNorm + router + top-4 +
                                                    SwiGLU experts + weighted combine
        x   = out
    key   = argmax over the Q6 LM head of x         gemv_head_argmax
    token = key's index; x = embed[token]           token_tail (reads and clears key)

The MoE layer normalises its input (RMSNorm of h + b) before the router and
the experts, so activations stay bounded over the stack without a separate
residual stream. The expert part runs one of three ways (``moe_path``):

  "fused"    B = 1: the one-launch fused layer, the default at batch 1;
             with ``fuse_proj`` (the default) the layer's projection runs
             inside the same launch (moe_decode_layer_proj: one launch per
             layer, bit-identical to gemv_quant + moe_decode_layer);
  "grouped"  B > 1: router_addnorm_route for the B rows, then the prefill
             MoE FFN (moe_prefill: route, sort, gather, tensor-core grouped
             GEMMs, combine), so each routed expert's rows are read and
             dequantised once per step for all of its tokens -- the default
             above B = 16 (measured on B200: 2439 vs 1987 tokens/s for "gemv"
             vs "grouped" at B = 16, 2473 vs 3123 at B = 32); activations match the oracle within the prefill
             tolerance, the ids given the same logits bit for bit;
  "gemv"     any B: router_addnorm_route, gemv_gather_act and
             gemv_gather_down_combine4, per-token GEMVs bit-identical to the
             oracle -- the default for 1 < B <= 16.

The token feeds back on the device, so a step can be captured once in a CUDA
graph and replayed.

A layer with an ``attn`` entry (a dict: norm_w [2048], qkv the Q4 projection of
the (heads + 2 KV heads) x head_dim rows, q_norm and k_norm [head_dim], cache a
``kv.KvCache``) mixes tokens before its projection: p = proj_l(attention(x)),
with RMSNorm, qkv GEMV, qk_norm_rope and paged_attention over that cache. The
batch's pages are kept by ``kv`` (a ``kv.PagedBatch``), planned once a step for
all layers; every row of the batch adds its token to its own request.

``rules`` (a ``sample.LogitsRules``): the requests' penalties, biases and grammar
masks, applied to the head's logits before the greedy token or the draw; the
tokens then count towards the penalties.

With ``sampling`` (batch 1, the reference's temperature > 0 path,
lfm/sample.rs), the head stores its bf16 logits (gemv_quant) and the draw
(mc_sample_draw) folds the sampled token into the same key the greedy head
writes; the token tail then runs unchanged and mc_sample_mark adds the token
to the seen set and advances the device position, so the sampled step is
graph-capturable too.
"""
from __future__ import annotations

import torch

from molten_b200 import kv as paged
from molten_b200 import lfm
from molten_b200.sample import logits_mark, logits_process


class DecodeStack:
    def __init__(self, ctx: lfm.Context, layers: list[dict], head, embed: torch.Tensor,
                 batch: int, n_experts: int = 64, moe_path: str | None = None, sampling=None,
                 fuse_proj: bool = True, kv: paged.PagedBatch | None = None, rules=None,
                 rope_theta: float = 1e6):
        self.ctx, self.layers, self.head, self.embed = ctx, layers, head, embed
        self.sampling = sampling
        lfm.ensure(sampling is None or batch == 1, "sampling decodes one sequence")
        self.B, self.E = batch, n_experts
        # measured on B200 (40 layers): batch 8 runs faster on the per-token
        # GEMVs, batch 32 on the grouped expert GEMMs
        self.path = moe_path or ("fused" if batch == 1 else "gemv" if batch <= 16 else "grouped")
        lfm.ensure(self.path in ("fused", "grouped", "gemv"), f"moe_path {self.path!r}")
        lfm.ensure(self.path != "fused" or batch == 1, "the fused layer is batch 1")
        self.fuse_proj = fuse_proj and self.path == "fused"
        # the buffers are zeroed on the stream that the steps run on
        with torch.cuda.stream(ctx.stream):
            self._allocate(kv, rules, rope_theta)

    def _allocate(self, kv: paged.PagedBatch | None, rules, rope_theta: float) -> None:
        ctx, layers, head, embed, batch, n_experts, sampling = (
            self.ctx, self.layers, self.head, self.embed, self.B, self.E, self.sampling)
        H = embed.shape[1]
        I = layers[0]["gate"].out_features // n_experts
        dev = embed.device
        bf = lambda *s: torch.empty(s, dtype=torch.bfloat16, device=dev)
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
        self.x = bf(batch, H)                    # step input: embedding rows
        self.p, self.hout, self.normed = bf(batch, H), bf(batch, H), bf(batch, H)
        self.outs = (bf(batch, H), bf(batch, H))
        self.logits = torch.empty((batch, n_experts), dtype=torch.float32, device=dev)
        self.ids = [i32(batch, 4) for _ in layers]
        self.wts = [bf(batch, 4) for _ in layers]
        self.counter = i32(batch)
        self.act = bf(batch, 4, I)
        self.keys = torch.zeros(batch, dtype=torch.int64, device=dev)
        self.tokens = i32(batch)
        self.tail_norm_w = torch.ones(H, dtype=torch.bfloat16, device=dev)
        self.tail_normed = bf(batch, H)
        self.ws = None
        if self.path == "fused":
            words = (lfm.moe_decode_proj_workspace_words(I) if self.fuse_proj
                     else lfm.moe_decode_workspace_words(I))
            self.ws = torch.zeros(words, dtype=torch.int32, device=dev)
        self.pws = None
        if self.path == "grouped":
            nb = lfm.moe_prefill_workspace_size(batch, n_experts, H, I)
            self.pws = torch.zeros(nb, dtype=torch.uint8, device=dev)
        self.kv, self.rules = kv, rules
        self.attn = None
        with_attn = [L["attn"] for L in layers if "attn" in L]
        lfm.ensure(not with_attn or kv is not None, "attention layers need a PagedBatch")
        if with_attn:
            lfm.ensure(kv.lens.numel() == batch and kv.slots.numel() == batch,
                       "the PagedBatch has one token row for each row of the batch")
            lfm.ensure(kv.ctx.same_stream(ctx), "the PagedBatch's context enqueues on another stream")
            c = with_attn[0]["cache"]
            D, K = c.head_dim, c.n_kv_heads
            heads = with_attn[0]["qkv"].out_features // D - 2 * K
            for A in with_attn:
                lfm.ensure(A["cache"].head_dim == D and A["cache"].n_kv_heads == K and
                           A["qkv"].out_features == (heads + 2 * K) * D and heads * D == H and
                           A["cache"].block_size == kv.block_size, "attention layer shapes")
                lfm.ensure(A["cache"].k.shape[0] >= kv.free_list.numel(),
                           "an attention layer's cache has fewer pages than the PagedBatch")
            rows = bf(batch, (heads + 2 * K) * D)
            part = lambda a, n: rows[:, a * D:(a + n) * D].view(batch, n, D)  # noqa: E731
            self.attn = dict(normed=bf(batch, H), rows=rows, q=part(0, heads), k=part(heads, K),
                             v=part(heads + K, K), q_out=bf(batch, heads, D),
                             out=bf(batch, heads, D),
                             turns=paged.rope_turns(D, rope_theta).to(dev),
                             ws=paged.paged_attention_workspace(D, dev))
        self.head_logits = None
        if sampling is not None or rules is not None:
            self.head_logits = bf(batch, head.out_features)
        self.sample = None
        if sampling is not None:
            from molten_b200.sample import SampleScratch
            self.sample = SampleScratch(ctx, head.out_features)
            self.pos = torch.zeros(1, dtype=torch.int32, device=dev)

    def start(self, tokens: torch.Tensor, pos: int = 0, seen=()) -> None:
        """Loads the embedding rows of the first tokens (int32 [B]); with
        sampling, ``pos`` is the absolute position of the token the next step
        draws and ``seen`` the sequence's token ids so far. A context with a
        stream of its own waits for the current one, where ``tokens`` were made."""
        stream, current = self.ctx.stream, torch.cuda.current_stream(self.ctx.device)
        if stream != current:
            stream.wait_stream(current)
            if tokens.is_cuda:
                tokens.record_stream(stream)
        with torch.cuda.stream(stream):
            self.x.copy_(self.embed[tokens.long()])
            if self.sample is not None:
                self.pos.fill_(pos)
                self.sample.upload_seen(list(seen) + [int(t) for t in tokens.cpu()])

    def _attend(self, A: dict, cur: torch.Tensor) -> torch.Tensor:
        """The attention of one layer on the rows ``cur``: [B, 2048]."""
        ctx, b, batch = self.ctx, self.attn, self.kv
        lfm.add_rmsnorm(ctx, cur, None, A["norm_w"], None, b["normed"])
        lfm.gemv_quant(ctx, A["qkv"], b["normed"], b["rows"])
        paged.qk_norm_rope(ctx, b["q"], b["k"], b["v"], A["q_norm"], A["k_norm"], batch.positions,
                           b["turns"], b["q_out"], A["cache"], batch.slots, status=batch.status)
        paged.paged_attention(ctx, b["q_out"], A["cache"], batch.block_table, batch.kv_lens,
                              b["out"], b["ws"], row_req=batch.token_req, status=batch.status)
        return b["out"].view(cur.shape)

    def step(self) -> None:
        ctx, cur = self.ctx, self.x
        if self.attn is not None:
            self.kv.plan()
        for l, L in enumerate(self.layers):
            nxt = self.outs[l % 2]
            attn = L.get("attn")
            if self.fuse_proj and attn is None:
                # the next layer's router rows and projection codes into L2
                # while this layer exchanges its act rows (its norm weights
                # are read before the launch's dependency wait anyway)
                following = self.layers[(l + 1) % len(self.layers)]
                ctx.prefetch_next(following["router"], following["proj"].codes)
                lfm.moe_decode_layer_proj(ctx, cur, L["proj"], L["norm_w"], self.hout, self.normed,
                                          L["router"], self.logits, None, self.ids[l],
                                          self.wts[l], L["gate"], L["up"], L["down"], nxt,
                                          self.ws, n_experts=self.E)
                cur = nxt
                continue
            lfm.gemv_quant(ctx, L["proj"], cur if attn is None else self._attend(attn, cur), self.p)
            if self.path == "fused":
                following = self.layers[(l + 1) % len(self.layers)]
                ctx.prefetch_next(following["router"], following["norm_w"])
                lfm.moe_decode_layer(ctx, cur, self.p, L["norm_w"], self.hout, self.normed,
                                     L["router"], self.logits, None, self.ids[l], self.wts[l],
                                     L["gate"], L["up"], L["down"], nxt, self.ws,
                                     n_experts=self.E)
            else:
                lfm.router_addnorm_route(ctx, cur, self.p, L["norm_w"], self.hout, self.normed,
                                         L["router"], self.logits, None, self.ids[l],
                                         self.wts[l], self.counter)
                if self.path == "grouped":
                    lfm.moe_prefill(ctx, self.normed, self.logits, L["gate"], L["up"], L["down"],
                                    self.pws, nxt, n_experts=self.E)
                else:
                    lfm.gemv_gather_act(ctx, L["gate"], L["up"], self.normed, self.ids[l],
                                        self.act, n_experts=self.E)
                    lfm.gemv_gather_down_combine4(ctx, L["down"], self.act, self.ids[l],
                                                  self.wts[l], nxt, n_experts=self.E)
            cur = nxt
        if self.head_logits is None:
            lfm.gemv_head_argmax(ctx, self.head, cur, self.keys)
        else:
            lfm.gemv_quant(ctx, self.head, cur, self.head_logits)
        if self.rules is not None:
            logits_process(ctx, self.head_logits, self.head_logits, self.rules,
                           self.keys if self.sample is None else None)
        if self.sample is not None:
            self.sample.encode_draw(self.head_logits[0], self.keys, self.sampling, self.pos)
        lfm.token_tail(ctx, self.keys, self.tokens,
                       (self.embed, self.tail_norm_w, self.x, self.tail_normed))
        if self.rules is not None:
            logits_mark(ctx, self.tokens, self.rules, self.head.out_features)
        if self.sample is not None:
            self.sample.encode_mark(self.tokens, self.pos)

    def status_words(self) -> list[torch.Tensor]:
        """The device status words this stack's kernels report into (the
        fused layer's sticky workspace word, the grouped GEMMs' word)."""
        words = []
        if self.ws is not None:
            words.append(self.ws[2:3])
        if self.pws is not None:
            I = self.layers[0]["gate"].out_features // self.E
            words.append(lfm.prefill_workspace_view(self.pws, self.B, self.E, self.x.shape[1],
                                                    I)["status"])
        return words

    def check(self) -> None:
        """Waits for the stream and raises McError if any kernel of the steps
        run so far reported a wait that ran out (the tokens are then invalid)."""
        with torch.cuda.stream(self.ctx.stream):
            for w in self.status_words():
                lfm.raise_on_status(w, f"decode stack ({self.path})")
        if self.attn is not None:
            self.kv.check()

    def read_tokens(self) -> torch.Tensor:
        """The last step's tokens on the host, after check()."""
        self.check()
        with torch.cuda.stream(self.ctx.stream):
            return self.tokens.cpu()

    def launches_per_step(self) -> int:
        per_layer = {"fused": 1 if self.fuse_proj else 2, "gemv": 4,
                     "grouped": 2 + lfm.MOE_PREFILL_LAUNCHES}[self.path]
        n = len(self.layers) * per_layer + 2
        if self.attn is not None:
            # norm, qkv, norm + rotation, attention, and the projection the fused layer leaves out
            n_attn = sum("attn" in L for L in self.layers)
            n += 1 + n_attn * (4 + self.fuse_proj)
        if self.rules is not None:
            n += 1 + (self.rules.seen is not None or self.rules.counts is not None)
        if self.sampling is not None:
            s = self.sampling
            full = (s.top_k == 0 or s.top_k >= self.head.out_features) and s.top_p >= 1.0
            n += 1 + (1 if full else 2 + 3 * ((s.top_k > 0) + (s.top_p < 1.0)))
        return n
