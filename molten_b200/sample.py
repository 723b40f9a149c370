"""Random sampling of the decode step (lfm/sample.rs mirrored over the C ABI).

``Sampling`` holds one request's validated parameters
(lfm/sample.rs:87-170: temperature 0 or >= 1e-6, top_k >= 0 with k >= vocab
meaning off, top_p in (0, 1], repetition_penalty in [1e-6, 1e6], a 64-bit
seed; absent / null / temperature 0 means greedy). ``SampleScratch`` owns the
device buffers of the draw -- the workspace (zeroed once, left zero by every
call) and the sequence's seen-token bitmap -- and encodes the draw of one
token into the zeroed 64-bit argmax key that ``lfm.token_tail`` reads, as
``SampleScratch::encode_draw`` does (lfm/sample.rs:248-338). Tokens never
leave the device between steps.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib
from .kv import _on, _ptr
from .lfm import Context, _p, ensure

MIN_TEMPERATURE = 1e-6
PENALTY_RANGE = (1e-6, 1e6)
_FIELDS = {"temperature", "top_k", "top_p", "repetition_penalty", "seed"}


@dataclass(frozen=True)
class Sampling:
    temperature: float = 1.0
    top_k: int = 0            # 0 = off (values >= the vocabulary are off too)
    top_p: float = 1.0        # 1 = off
    repetition_penalty: float = 1.0
    seed: int = 0

    @staticmethod
    def from_request(value, vocab: int) -> "Sampling | None":
        """Parses a request's ``sampling`` object; None means greedy decoding."""
        if value is None:
            return None
        ensure(isinstance(value, dict), "generate.sampling must be an object")
        for k in value:
            ensure(k in _FIELDS, f"unknown sampling field {k!r}")

        def number(key, default):
            x = value.get(key, default)
            ensure(isinstance(x, (int, float)) and not isinstance(x, bool),
                   f"sampling.{key} must be a number")
            ensure(math.isfinite(x), f"sampling.{key} must be finite")
            return float(x)

        temperature = number("temperature", 1.0)
        ensure(temperature >= 0.0, "sampling.temperature must be >= 0")
        top_p = number("top_p", 1.0)
        ensure(0.0 < top_p <= 1.0, "sampling.top_p must be in (0, 1]")
        pen = number("repetition_penalty", 1.0)
        ensure(PENALTY_RANGE[0] <= pen <= PENALTY_RANGE[1],
               f"sampling.repetition_penalty must be in [{PENALTY_RANGE[0]}, {PENALTY_RANGE[1]}]")
        top_k = value.get("top_k", 0)
        ensure(isinstance(top_k, int) and not isinstance(top_k, bool) and top_k >= 0,
               "sampling.top_k must be a non-negative integer")
        seed = value.get("seed", 0)
        ensure(isinstance(seed, int) and not isinstance(seed, bool) and 0 <= seed < 2 ** 64,
               "sampling.seed must be an integer in [0, 2^64)")
        if temperature == 0.0:
            return None
        ensure(temperature >= MIN_TEMPERATURE,
               f"sampling.temperature must be 0 (greedy) or at least {MIN_TEMPERATURE}")
        return Sampling(temperature, 0 if top_k >= vocab else top_k, top_p, pen, seed)

    def uses_penalty(self) -> bool:
        return self.repetition_penalty != 1.0

    def c(self) -> _lib.Sampling:
        return _lib.Sampling(self.temperature, self.top_k, self.top_p, self.repetition_penalty,
                             self.seed)


class SampleScratch:
    """Device buffers of the sampled step for one sequence."""

    def __init__(self, ctx: Context, vocab: int, device=None):
        ensure(vocab % 4 == 0 and vocab >= 4, "vocab must be a multiple of 4")
        dev = device or ctx.device
        self.ctx, self.vocab = ctx, vocab
        n = int(_lib.lib().mc_sample_workspace_bytes(vocab))
        self.ws = torch.zeros(n, dtype=torch.uint8, device=dev)
        self.seen = torch.zeros((vocab + 31) // 32, dtype=torch.int32, device=dev)

    def upload_seen(self, tokens) -> None:
        """Sets the seen set to the given token ids (the sequence so far)."""
        import numpy as np
        bits = np.zeros(self.seen.numel(), np.uint32)
        for t in tokens:
            t = int(t)
            if 0 <= t < self.vocab:
                bits[t // 32] |= np.uint32(1 << (t % 32))
        self.seen.copy_(torch.from_numpy(bits.view(np.int32)))

    def encode_draw(self, logits: torch.Tensor, best: torch.Tensor, s: Sampling,
                    pos: int | torch.Tensor) -> None:
        """Draws the token at absolute position ``pos`` from bf16 ``logits``
        [vocab] into ``best`` (int64 [1], zero on entry). ``pos`` may be a
        device int32 [1] tensor (read on the device: a captured step draws at
        the position ``encode_mark`` advanced)."""
        ensure(logits.numel() == self.vocab and logits.dtype == torch.bfloat16,
               "sampling logits row")
        ensure(best.dtype == torch.int64 and best.numel() >= 1, "sampling key")
        dev_pos = isinstance(pos, torch.Tensor)
        ensure(dev_pos or 0 <= pos < 2 ** 32, "position exceeds u32")
        sp = s.c()
        _lib.call("mc_sample_draw", self.ctx.handle, _p(logits), self.vocab,
                  _p(self.seen) if s.uses_penalty() else None, _lib.C.byref(sp),
                  0 if dev_pos else pos, _p(pos) if dev_pos else None, _p(best),
                  _p(self.ws), self.ws.numel())

    def encode_mark(self, tok: torch.Tensor, pos: torch.Tensor | None = None) -> None:
        """After the token tail wrote ``tok`` (int32 [1]): adds it to the seen
        set, and advances the device position ``pos`` (int32 [1]) when given."""
        ensure(tok.numel() == 1 and tok.dtype == torch.int32, "sampled token slot")
        _lib.call("mc_sample_mark", self.ctx.handle, _p(tok), _p(self.seen), self.vocab, _p(pos))


@dataclass
class LogitsRules:
    """The rules of a batch of requests on their logits rows [batch, vocab];
    None leaves a rule out.

    ``seen``: u32 bitmap (int32 [batch, ceil(vocab / 32)]) of the tokens that
    ``repetition`` (f32 [batch]) divides (positive logits) or multiplies;
    ``counts``: u16 counts (int16 [batch, vocab]) for ``frequency`` and
    ``presence`` (f32 [batch]); ``bias_start`` (int32 [batch + 1]),
    ``bias_ids`` (int32, ascending within a row) and ``bias_values`` (f32): the
    biases of row b are the entries bias_start[b] .. bias_start[b + 1];
    ``allowed``: u32 bitmap (int32 [masks, ceil(vocab / 32)]), 0 bits become
    -inf; ``allowed_row`` (int32 [batch]): the mask of each row (-1: none;
    None: mask b for row b)."""
    seen: torch.Tensor | None = None
    counts: torch.Tensor | None = None
    repetition: torch.Tensor | None = None
    frequency: torch.Tensor | None = None
    presence: torch.Tensor | None = None
    bias_start: torch.Tensor | None = None
    bias_ids: torch.Tensor | None = None
    bias_values: torch.Tensor | None = None
    allowed: torch.Tensor | None = None
    allowed_row: torch.Tensor | None = None


def _vocab_rows(ctx: Context, t: torch.Tensor, what: str) -> tuple[int, int]:
    row, one = t.stride()
    if one != 1 or not _on(ctx, t):
        ensure(one == 1 or t.shape[1] == 1, f"{what}: rows [batch, vocab], each contiguous")
        ensure(_on(ctx, t), f"{what} must be on {ctx.device}")
    return t.data_ptr(), row


def logits_process(ctx: Context, logits: torch.Tensor, out: torch.Tensor, rules: LogitsRules,
                   best: torch.Tensor | None = None) -> None:
    """Applies ``rules`` to ``logits`` [batch, vocab] (bf16 or f32) into
    ``out`` (logits itself, or apart from it): repetition, frequency and
    presence, biases, then the grammar mask. ``best`` (int64 [batch], zero on
    entry): takes the greedy keys that lfm.token_tail reads."""
    shape, dtype = logits.shape, logits.dtype
    ensure(len(shape) == 2 and dtype in (torch.bfloat16, torch.float32) and out.dtype is dtype
           and out.shape == shape, "logits_process: logits and out [batch, vocab], BF16 or F32")
    B, V = shape
    lp, ls = _vocab_rows(ctx, logits, "logits")
    op, os = _vocab_rows(ctx, out, "out")
    W = (V + 31) // 32
    i32, f32 = torch.int32, torch.float32
    r = rules
    n_bias = 0 if r.bias_ids is None else r.bias_ids.numel()
    ensure(r.allowed is None or (r.allowed.dim() == 2 and r.allowed.shape[1] == W),
           "allowed shape")
    _lib.call("mc_logits_process", ctx.handle, lp, ls,
              _lib.DTYPE_BF16 if dtype is torch.bfloat16 else _lib.DTYPE_F32, V, B,
              _ptr(ctx, r.seen, i32, "seen", B * W),
              _ptr(ctx, r.counts, torch.int16, "counts", B * V),
              _ptr(ctx, r.repetition, f32, "repetition", B),
              _ptr(ctx, r.frequency, f32, "frequency", B),
              _ptr(ctx, r.presence, f32, "presence", B),
              _ptr(ctx, r.bias_start, i32, "bias_start", B + 1),
              _ptr(ctx, r.bias_ids, i32, "bias_ids"),
              _ptr(ctx, r.bias_values, f32, "bias_values", n_bias), n_bias,
              _ptr(ctx, r.allowed, i32, "allowed"),
              _ptr(ctx, r.allowed_row, i32, "allowed_row", B),
              0 if r.allowed is None else r.allowed.shape[0], op, os,
              _ptr(ctx, best, torch.int64, "best", B))


def logits_mark(ctx: Context, tokens: torch.Tensor, rules: LogitsRules, vocab: int) -> None:
    """Adds the drawn ``tokens`` (int32 [batch]) to the rules' seen bitmap and
    counts (a no-op for rules that go by neither)."""
    if rules.seen is None and rules.counts is None:
        return
    B = tokens.numel()
    _lib.call("mc_logits_mark", ctx.handle, _ptr(ctx, tokens, torch.int32, "tokens"), B,
              _ptr(ctx, rules.seen, torch.int32, "seen", B * ((vocab + 31) // 32)),
              _ptr(ctx, rules.counts, torch.int16, "counts", B * vocab), vocab)
