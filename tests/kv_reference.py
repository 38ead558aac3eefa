"""Plain 64-bit forms of the paged KV cache operators, and how far a 16- or 32-bit kernel may be from them."""
import math

import torch


def rotary(x, positions, inv_freq, interleaved=False, magnitude=1.0, inverse=False):
    """x [..., heads, dim], positions [...]: the rotated heads in 64 bits, and the sum of each pair's magnitudes."""
    x = x.double()
    n = inv_freq.numel()
    angle = positions.double().unsqueeze(-1) * inv_freq.double() * (-1.0 if inverse else 1.0)
    cos, sin = torch.cos(angle).unsqueeze(-2), torch.sin(angle).unsqueeze(-2)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), torch.zeros_like(x)
    y[..., first] = magnitude * (a * cos - b * sin)
    y[..., second] = magnitude * (b * cos + a * sin)
    size[..., first] = size[..., second] = magnitude * (a.abs() + b.abs())
    return y, size


def rotary_tolerance(y, size, dtype):
    """The kernel's angle, in turns, is rounded once to 32 bits (2^-24 of half a turn: 2^-22.3 radians at most), sine
    and cosine are off by at most 2^-22, the products and the sum by three roundings of 2^-24: below 2^-20 of
    |a| + |b| together. Then one rounding to the type."""
    return size * 2.0 ** -20 + y.abs() * (torch.finfo(dtype).eps / 2) * 1.01 + 1e-30


def sequence_keys(pool, table_row, length):
    """Keys, values [length, kv_heads, dim] of a sequence and which of its tokens have a page, in 64 bits."""
    pages, _, heads, page_tokens, dim = pool.shape
    p = torch.arange(length, device=pool.device)
    column = p // page_tokens
    page = torch.full_like(p, -1)
    inside = column < table_row.numel()
    page[inside] = table_row.long()[column[inside]]
    good = (page >= 0) & (page < pages)
    page = torch.where(good, page, 0)
    kv = pool[page, :, :, p % page_tokens].double()  # [length, 2, heads, dim]
    return kv[:, 0], kv[:, 1], good


def attention(q, pool, table, lens, starts, scale=None, causal=True, window=0):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits; rows of no sequence are NaN.

    The tolerance: with u half a step of the type, each weight is rounded to the type for the second product (u of
    sum w |v|), the output once (u of |out|). A score is a sum of dim products in 32 bits, off by at most
    (dim + 2) 2^-24 of scale * sum |q k|; its weight by that and 2^-20 (exp), relative. The sums over n keys add n
    2^-24 each, and the rescaling of a running sum as much again."""
    rows, q_heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    group = q_heads // pool.shape[2]
    u = torch.finfo(q.dtype).eps / 2
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    lse, tol, ltol = out[..., 0].clone(), out.clone(), out[..., 0].clone()
    starts, lens = starts.tolist(), lens.tolist()
    for b, length in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        if hi == lo:
            continue
        k, v, good = sequence_keys(pool, table[b], length)
        at = torch.arange(length - (hi - lo), length, device=q.device)[:, None]
        key = torch.arange(length, device=q.device)
        seen = good.expand(hi - lo, length)
        if causal:
            seen = seen & (key <= at)
        if window:
            seen = seen & (key > at - window)
        some = seen.any(0)
        k = torch.where(some[:, None, None], k, 0.0).repeat_interleave(group, 1)
        v = torch.where(some[:, None, None], v, 0.0).repeat_interleave(group, 1)
        x = q[lo:hi].double()
        s = torch.einsum("nhd,lhd->hnl", x, k) * scale
        s = s.masked_fill(~seen, -math.inf)
        m = s.amax(-1, keepdim=True) if length else torch.full(s.shape[:-1] + (1,), -math.inf, device=q.device, dtype=s.dtype)
        m = torch.where(m == -math.inf, 0.0, m)
        w = torch.exp(s - m)
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
        out[lo:hi] = torch.einsum("hnl,lhd->nhd", w, v)
        lse[lo:hi] = (m + total.log())[..., 0].transpose(0, 1)
        big = torch.einsum("nhd,lhd->hnl", x.abs(), k.abs()).masked_fill(~seen, 0.0) * abs(scale)
        off = (big.amax(-1) if length else total[..., 0]) * (dim + 2) * 2.0 ** -24 + 2.0 ** -20
        n = length * 2.0 ** -23
        size = torch.einsum("hnl,lhd->nhd", w, v.abs())
        tol[lo:hi] = 1.02 * (u * out[lo:hi].abs() + (u + 2 * off.transpose(0, 1)[..., None] + 2 * n) * size) + 1e-30
        ltol[lo:hi] = off.transpose(0, 1) + n + lse[lo:hi].abs().nan_to_num(posinf=0.0) * 2.0 ** -22
    return out, lse, tol, ltol


def batch(news, lens, page_tokens, pages=None, width=None, seed=0, index=torch.int32, device="cpu"):
    """Tables of a ragged batch: (page_table, seq_lens, query_starts, pages). Pages are shuffled."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page_tokens) for n in lens]
    pages = sum(held) + 2 if pages is None else pages
    width = max(held + [0]) + 1 if width is None else width
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), width), pages - 1, dtype=torch.int64)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    make = lambda v: torch.as_tensor(v, dtype=index).to(device)  # noqa: E731
    return make(table), make(lens), make(starts), pages
