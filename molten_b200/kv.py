"""The paged key-value cache and the attention of new tokens over it.

Between the Q/K/V projections and the output projection of a batched decode
step: ``kv_plan`` finds each new token's page, position and slot from the
requests' lengths on the device, ``qk_norm_rope`` norms and rotates queries
and keys and writes K and V to their slots, ``paged_attention`` attends, and
``kv_release`` gives a finished request's pages back. Like the functions of
``lfm``, each checks its arguments (ValueError, nothing enqueued), then
enqueues on the context's stream; tensors are CUDA tensors owned by the
caller. The reference's decode attention does norm, rotation and attention
over one contiguous cache in one dispatch; that cache ([KV heads, max_seq, 64],
as ``lfm.proj3_gemv_scatter`` writes V) is a ``KvCache`` of one page.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib
from .lfm import Context, ensure

#: Status bits of the calls below (``status``: int32 [1], OR-ed into).
STATUS_BITS = {
    _lib.KV_NO_PAGES: "the free list ran out", _lib.KV_TABLE_FULL: "a request outgrew its block table",
    _lib.KV_ROWS_FULL: "more token rows than the maps hold", _lib.KV_BAD_LENGTH: "a bad length",
    _lib.KV_LIST_FULL: "more pages than the free list holds", _lib.KV_BAD_SLOT: "a slot outside the cache",
    _lib.KV_BAD_PAGE: "a page outside the cache", _lib.KV_BAD_ROW: "a row of no request",
    _lib.KV_WAIT: "a copy did not arrive in time"}


def raise_on_status(status: torch.Tensor, what: str) -> None:
    """Reads a status word (waits for the stream) and raises McError if any
    bit is set."""
    v = int(status.reshape(-1)[0].item()) & 0xffffffff
    if v:
        why = ", ".join(m for b, m in STATUS_BITS.items() if v & b) or "unknown bits"
        raise _lib.McError(_lib.MC_EINVAL, f"{what}: status 0x{v:x} ({why})")


def _on(ctx: Context, t: torch.Tensor) -> bool:
    return t.get_device() == ctx.index


def _ptr(ctx: Context, t: torch.Tensor | None, dtype: torch.dtype, what: str,
         numel: int | None = None) -> int | None:
    """Address of a contiguous tensor of ``dtype`` (and ``numel``) on the
    context's device."""
    if t is None:
        return None
    if (t.dtype is not dtype or t.get_device() != ctx.index or not t.is_contiguous()
            or (numel is not None and t.numel() != numel)):
        ensure(t.dtype == dtype, f"{what} expects {dtype}")
        ensure(_on(ctx, t), f"{what} must be on {ctx.device}")
        ensure(t.is_contiguous(), f"{what} must be contiguous")
        ensure(False, f"{what} shape")
    return t.data_ptr()


def _rows(ctx: Context, t: torch.Tensor, shape: torch.Size, what: str) -> tuple[int, int]:
    """Address and token stride of bf16 rows [tokens, heads, dim] whose heads
    are contiguous (a part of a fused projection row is fine)."""
    if t.shape != shape or t.dtype is not torch.bfloat16 or t.get_device() != ctx.index:
        ensure(t.dtype == torch.bfloat16 and t.dim() == 3, f"{what} expects BF16 [rows, heads, dim]")
        ensure(_on(ctx, t), f"{what} must be on {ctx.device}")
        ensure(False, f"{what} shape")
    token, head, one = t.stride()
    if shape[0] <= 1:
        token = shape[1] * shape[2]  # a single row's distance to the next says nothing
    if one != 1 or head != shape[2]:
        ensure((one == 1 or shape[2] == 1) and (head == shape[2] or shape[1] == 1),
               f"{what}: a row's heads must be contiguous")
    return t.data_ptr(), token


@dataclass(frozen=True, eq=False)
class KvCache:
    """Pages of K and V: [num_blocks, KV heads, block_size, head_dim] in bf16
    or float8_e4m3fn, contiguous but for the distance between pages (the same
    for both, so K and V may be the halves of one [num_blocks, 2, ...]
    tensor); ``k_scale`` / ``v_scale``: optional f32 [KV heads] of an 8-bit
    cache (stored = value / scale). The tensors stay the same ones: their
    addresses are taken here."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None

    def __post_init__(self):
        k, v = self.k, self.v
        ensure(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.device == v.device,
               "KV cache: k and v are alike, [blocks, KV heads, block size, head dim]")
        ensure(k.dtype in (torch.bfloat16, torch.float8_e4m3fn), "KV cache: BF16 or float8_e4m3fn")
        _, heads, size, dim = k.shape
        ensure(k.numel() > 0, "KV cache: empty")
        for t in (k, v):
            ensure(t[0].is_contiguous() and (t.shape[0] == 1 or t.stride(0) == k.stride(0)),
                   "KV cache: pages must be contiguous, K's and V's equally far apart")
        for s in (self.k_scale, self.v_scale):
            ensure(s is None or (s.dtype == torch.float32 and s.numel() == heads and
                                 s.is_contiguous() and s.device == k.device), "KV cache scales")
        dt = _lib.DTYPE_BF16 if k.dtype == torch.bfloat16 else _lib.DTYPE_E4M3
        p = lambda s: None if s is None else s.data_ptr()  # noqa: E731
        stride = k.stride(0) if k.shape[0] > 1 else heads * size * dim
        self.__dict__.update(
            n_kv_heads=heads, head_dim=dim, _index=k.get_device(),
            _where=(k.data_ptr(), v.data_ptr(), dt, k.shape[0], size, stride),
            _scales=(p(self.k_scale), p(self.v_scale)))

    @property
    def block_size(self) -> int:
        return self.k.shape[2]

    @staticmethod
    def empty(num_blocks: int, n_kv_heads: int, block_size: int, head_dim: int = 64,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> "KvCache":
        shape = (num_blocks, n_kv_heads, block_size, head_dim)
        return KvCache(torch.empty(shape, dtype=dtype, device=device),
                       torch.empty(shape, dtype=dtype, device=device))


def kv_plan(ctx: Context, lens: torch.Tensor, new_lens: torch.Tensor | None, block_size: int,
            block_table: torch.Tensor, free_list: torch.Tensor, n_free: torch.Tensor,
            seq_lens: torch.Tensor, n_free_out: torch.Tensor, row_start: torch.Tensor,
            positions: torch.Tensor, token_req: torch.Tensor, kv_lens: torch.Tensor,
            slots: torch.Tensor, status: torch.Tensor | None = None) -> None:
    """One step's bookkeeping: request r holding lens[r] tokens adds
    new_lens[r] (None: one each); takes the pages they need from the free list
    (a stack of n_free entries) into ``block_table`` [requests, width] and
    fills the maps of the token rows (packed in request order): positions,
    request, kv_lens (position + 1), slots (int64, -1: none); rows behind the
    last get 0, -1, 0, -1. A request that does not fit is refused whole (its
    length stays, its rows get kv_len 0 and slot -1, ``status`` says why).
    All int32 but slots. seq_lens may be lens, n_free_out may be n_free."""
    i32 = torch.int32
    n = lens.numel()
    ensure(block_table.dim() == 2 and block_table.shape[0] == n, "block table [requests, width]")
    rows = slots.numel()
    _lib.call("mc_kv_plan", ctx.handle, _ptr(ctx, lens, i32, "lens"),
              _ptr(ctx, new_lens, i32, "new_lens", n), n, block_size,
              _ptr(ctx, block_table, i32, "block_table"), block_table.shape[1],
              _ptr(ctx, free_list, i32, "free_list"), _ptr(ctx, n_free, i32, "n_free", 1),
              free_list.numel(), _ptr(ctx, seq_lens, i32, "seq_lens", n),
              _ptr(ctx, n_free_out, i32, "n_free_out", 1),
              _ptr(ctx, row_start, i32, "row_start", n + 1),
              _ptr(ctx, positions, i32, "positions", rows),
              _ptr(ctx, token_req, i32, "token_req", rows),
              _ptr(ctx, kv_lens, i32, "kv_lens", rows), _ptr(ctx, slots, torch.int64, "slots"),
              rows, _ptr(ctx, status, i32, "status", 1))


def kv_release(ctx: Context, done: torch.Tensor, lens: torch.Tensor, block_size: int,
               block_table: torch.Tensor, free_list: torch.Tensor, n_free: torch.Tensor,
               lens_out: torch.Tensor, n_free_out: torch.Tensor,
               status: torch.Tensor | None = None) -> None:
    """Gives the pages of the requests with done[r] != 0 back to the free list
    and sets their length to 0. lens_out may be lens, n_free_out n_free."""
    i32 = torch.int32
    n = lens.numel()
    ensure(block_table.dim() == 2 and block_table.shape[0] == n, "block table [requests, width]")
    _lib.call("mc_kv_release", ctx.handle, _ptr(ctx, done, i32, "done", n),
              _ptr(ctx, lens, i32, "lens"), n, block_size,
              _ptr(ctx, block_table, i32, "block_table"), block_table.shape[1],
              _ptr(ctx, free_list, i32, "free_list"), _ptr(ctx, n_free, i32, "n_free", 1),
              free_list.numel(), _ptr(ctx, lens_out, i32, "lens_out", n),
              _ptr(ctx, n_free_out, i32, "n_free_out", 1), _ptr(ctx, status, i32, "status", 1))


def rope_turns(rot_dim: int, theta: float = 1e6, position_scale: float = 1.0) -> torch.Tensor:
    """The rotation frequencies position_scale * theta^(-2i / rot_dim) as
    fractions of a turn per position in 64-bit fixed point: int64 [rot_dim / 2]
    on the host, to be uploaded once."""
    ensure(rot_dim >= 2, f"rope_turns: rot_dim {rot_dim}")
    out = torch.empty(rot_dim // 2, dtype=torch.int64)
    _lib.call("mc_rope_turns", theta, position_scale, rot_dim, out.data_ptr())
    return out


def qk_norm_rope(ctx: Context, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None,
                 q_norm_w: torch.Tensor | None, k_norm_w: torch.Tensor | None,
                 positions: torch.Tensor | None, turns: torch.Tensor | None,
                 q_out: torch.Tensor, cache: KvCache, slots: torch.Tensor | None = None,
                 interleaved: bool = False, eps: float = 1e-5,
                 status: torch.Tensor | None = None) -> None:
    """Per-head RMSNorm (gains [head_dim]; None: no norm) and rotation of the
    query rows q [T, heads, dim] into q_out and of the key rows k [T, KV heads,
    dim] into the cache at slots [T] (int64, -1: not written; None: slot t),
    with v's rows beside them (None: V is there already). ``turns``: rope_turns
    of the rotated dimensions on the device (None: no rotation)."""
    shape = q.shape
    ensure(len(shape) == 3, "qk_norm_rope: q expects [rows, heads, dim]")
    T, H, D = shape
    heads = cache.n_kv_heads
    ensure(cache.head_dim == D and tuple(k.shape) == (T, heads, D),
           "qk_norm_rope: k rows match the cache")
    qp, qs = _rows(ctx, q, shape, "q")
    kp, ks = _rows(ctx, k, k.shape, "k")
    vp, vs = (None, 0) if v is None else _rows(ctx, v, k.shape, "v")
    op, os = _rows(ctx, q_out, shape, "q_out")
    ensure(cache._index == ctx.index, f"the cache must be on {ctx.device}")
    rot = 0 if turns is None else 2 * turns.numel()
    ensure(rot == 0 or positions is not None, "qk_norm_rope: rotation needs positions")
    b16 = torch.bfloat16
    _lib.call("mc_qk_norm_rope", ctx.handle, qp, qs, kp, ks, vp, vs, T, H, heads, D,
              _ptr(ctx, q_norm_w, b16, "q_norm_w", D), _ptr(ctx, k_norm_w, b16, "k_norm_w", D),
              eps, _ptr(ctx, positions, torch.int32, "positions", T),
              _ptr(ctx, turns, torch.int64, "turns"), rot, int(interleaved), op, os,
              _ptr(ctx, slots, torch.int64, "slots", T), *cache._where, *cache._scales,
              _ptr(ctx, status, torch.int32, "status", 1))


def paged_attention_workspace(head_dim: int, device="cuda") -> torch.Tensor:
    """A workspace of paged_attention, for one chain of ordered calls, zeroed on
    the current stream. Zero it again if lengths or rows changed while a call ran."""
    n = int(_lib.lib().mc_paged_attention_workspace_bytes(head_dim))
    ensure(n > 0, f"paged_attention: head_dim {head_dim} (64 and 128 are built)")
    return torch.zeros(n, dtype=torch.uint8, device=device)


def paged_attention(ctx: Context, q: torch.Tensor, cache: KvCache, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, out: torch.Tensor, workspace: torch.Tensor,
                    scale: float | None = None, row_req: torch.Tensor | None = None,
                    window: int = 0, lse: torch.Tensor | None = None,
                    status: torch.Tensor | None = None) -> None:
    """Attention of the query rows q [rows, heads, dim] over the first
    kv_lens[row] keys of block_table[row_req[row]] (None: row), the last
    ``window`` of them if positive; out like q, lse f32 [rows, heads] optional.
    ``scale``: 1 / sqrt(dim) if None. A row without keys gives zeros and -inf."""
    shape = q.shape
    ensure(len(shape) == 3, "paged_attention: q expects [rows, heads, dim]")
    rows, H, D = shape
    heads = cache.n_kv_heads
    ensure(cache.head_dim == D and H % heads == 0, "paged_attention: query heads match the cache")
    ensure(block_table.dim() == 2, "block table [requests, width]")
    ensure(cache._index == ctx.index, f"the cache must be on {ctx.device}")
    qp, qs = _rows(ctx, q, shape, "q")
    op, os = _rows(ctx, out, shape, "out")
    i32 = torch.int32
    n_req, width = block_table.shape
    _lib.call("mc_paged_attention", ctx.handle, qp, qs, rows, H, *cache._where, heads, D,
              *cache._scales, _ptr(ctx, block_table, i32, "block_table"), n_req, width, _ptr(ctx, kv_lens, i32, "kv_lens", rows),
              _ptr(ctx, row_req, i32, "row_req", rows), window,
              1.0 / math.sqrt(D) if scale is None else scale, op, os,
              _ptr(ctx, lse, torch.float32, "lse", rows * H),
              _ptr(ctx, workspace, torch.uint8, "workspace"), workspace.numel(),
              _ptr(ctx, status, i32, "status", 1))


class PagedBatch:
    """The bookkeeping of one batch of requests over paged caches: lengths, block
    tables and the free list on the device, and the token maps of a step.
    Every layer's ``KvCache`` has ``num_blocks`` pages of ``block_size``; a
    request's pages have the same numbers in each of them. ``max_tokens``: token
    rows of a step (one for each request by default)."""

    def __init__(self, ctx: Context, n_req: int, num_blocks: int, block_size: int,
                 table_width: int, max_tokens: int | None = None):
        dev = ctx.device
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)  # noqa: E731
        T = n_req if max_tokens is None else max_tokens
        self.ctx, self.block_size = ctx, block_size
        with torch.cuda.stream(ctx.stream):
            self.lens, self.n_free = i32(n_req), i32(1)
            self.block_table = torch.full((n_req, table_width), -1, dtype=torch.int32, device=dev)
            self.free_list = i32(num_blocks)
            self.row_start, self.status = i32(n_req + 1), i32(1)
            self.positions, self.token_req, self.kv_lens = i32(T), i32(T), i32(T)
            self.slots = torch.zeros(T, dtype=torch.int64, device=dev)
        self.clear()

    def clear(self) -> None:
        """Every request empty, every page free (on the context's stream, as all calls)."""
        n = self.free_list.numel()
        with torch.cuda.stream(self.ctx.stream):
            self.lens.zero_()
            self.status.zero_()
            self.n_free.fill_(n)
            torch.arange(n - 1, -1, -1, out=self.free_list)

    def plan(self, new_lens: torch.Tensor | None = None) -> None:
        """The next step: new_lens tokens (None: one each) for the requests."""
        kv_plan(self.ctx, self.lens, new_lens, self.block_size, self.block_table, self.free_list,
                self.n_free, self.lens, self.n_free, self.row_start, self.positions,
                self.token_req, self.kv_lens, self.slots, self.status)

    def release(self, done: torch.Tensor) -> None:
        """Frees the pages of the requests with done[r] != 0 and empties them."""
        kv_release(self.ctx, done, self.lens, self.block_size, self.block_table, self.free_list,
                   self.n_free, self.lens, self.n_free, self.status)

    def check(self) -> None:
        """Waits for the stream and raises McError if a request was refused or
        an index was out of range since the last clear()."""
        with torch.cuda.stream(self.ctx.stream):
            raise_on_status(self.status, "paged batch")
