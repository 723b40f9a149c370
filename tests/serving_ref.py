"""Plain 64-bit statements of the serving operators for their GPU tests, and
the tolerances that follow from their arithmetic."""
import torch

BF16_HALF = 2.0 ** -8      # half a bf16 step, relative
E4M3_HALF = 2.0 ** -4      # half an e4m3 step, relative; subnormals: 2^-10 absolute
U32 = 2.0 ** -24           # half an fp32 step, relative


def plan(lens, new, bs, table, free, n_free, max_tokens):
    """kv_plan, request by request, on lists (table: list of lists, changed in
    place). Returns a dict of lists and the status bits."""
    R, width = len(lens), len(table[0])
    rows, counted, used, status = 0, 0, 0, 0
    out = dict(seq=[], row_start=[0], positions=[0] * max_tokens, token_req=[-1] * max_tokens,
               kv_lens=[0] * max_tokens, slots=[-1] * max_tokens)
    nf = min(max(n_free, 0), len(free))
    for r in range(R):
        n, add = lens[r], new[r]
        ok = True
        if n < 0 or add < 0:
            n, add, ok = max(n, 0), 0, False
            status |= 8
        have, want = -(-n // bs), -(-(n + add) // bs)
        if ok and want > width:
            ok = False
            status |= 2
        if ok and rows + add > max_tokens:
            ok = False
            status |= 4
        if ok:
            first = counted
            counted += want - have
            if want > have and counted > nf:
                ok = False
                status |= 1
            elif want > have:
                used = counted
                for j in range(have, want):
                    table[r][j] = free[nf - 1 - (first + j - have)]
        for j in range(add):
            t = rows + j
            if t < max_tokens:
                out["positions"][t], out["token_req"][t] = n + j, r
                if ok:
                    out["kv_lens"][t] = n + j + 1
                    out["slots"][t] = table[r][(n + j) // bs] * bs + (n + j) % bs
        rows += add
        out["row_start"].append(rows)
        out["seq"].append(n + add if ok else n)
    out["n_free"] = nf - used
    return out, status


def norm_rope(x, w, positions, freqs, rot, interleaved, eps):
    """[T, heads, D] in 64 bits -> the rows, and the size of what each element is made of."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    size = x.abs().clone()
    y = x.clone()
    half = rot // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = positions.double() * freqs[i]
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def norm_rope_error(D):
    """fp32 error relative to `size`: the squares' sum is off by D + 2 steps
    and enters by half, root, quotient and two products 2 steps each at most,
    the angle (24 bits of half a turn) and sincos 16 steps, the rotation 4."""
    return ((D + 2) / 2 + 8 + 16 + 4) * U32


def attention(q, k, v, scale, window=0):
    """One row: q [H, D], k, v [n, K, D] in 64 bits -> out [H, D], lse [H] and
    their fp32 error bounds."""
    H, D = q.shape
    n, K = k.shape[0], k.shape[1]
    if window and n > window:
        k, v, n = k[-window:], v[-window:], window
    if n == 0:
        z = torch.zeros(H, D, dtype=torch.float64, device=q.device)
        return z, torch.full((H,), float("-inf"), dtype=torch.float64, device=q.device), z, z[:, 0]
    q, k, v = q.double().view(K, H // K, D), k.double(), v.double()
    s = torch.einsum("kgd,nkd->kgn", q, k) * scale
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    out = torch.einsum("kgn,nkd->kgd", p, v)
    # a score: D products and sums of q and k (q in 24 bits of its largest element), two
    # scalings; a weight: its score's error, exp2 and its argument, P in 16 bits; a sum of n
    # weights and of n products, rescaled at most once a step of 16 keys and joined
    terms = (q.abs().amax(-1, keepdim=True) * k.abs().amax((0, 2))[:, None, None]).squeeze(-1) * D * scale
    ds = (D + 8) * U32 * terms + 4 * U32 * s.abs().amax(-1)
    dw = 2 * ds + 2.0 ** -16 + 8 * U32 * (1 + s.abs().amax(-1)) + (2 * n + 64) * U32
    weight = torch.einsum("kgn,nkd->kgd", p, v.abs())
    return (out.reshape(H, D), lse.reshape(H), (dw[..., None] * weight).reshape(H, D),
            (dw + 4 * U32 * lse.abs()).reshape(H))
