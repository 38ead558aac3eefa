"""Operators on paged KV caches: rotary positions, appending, attention.

A cache is a tensor ``[pages, 2, kv_heads, page_tokens, head_dim]`` (keys at
index 0 of the second axis, values at 1) with any strides but the last, so a
pool whose pages hold ``[2, page_tokens, kv_heads, head_dim]`` is passed as
``pool.transpose(2, 3)``. ``mpcomm.models.KVPoolSpec.as_cache`` gives this
view of a pool of byte pages, the pages that ``paged_gather`` and
``paged_scatter`` move.

A batch is ragged. Rows ``query_starts[b] .. query_starts[b + 1]`` of a
tensor of new tokens are the newest tokens of sequence b, and
``seq_lens[b]`` counts all its tokens, those rows among them. Token p lies
in slot ``p % page_tokens`` of page ``page_table[b, p // page_tokens]``. Rows
behind the last sequence are padding. The three tables are int32 or int64
device tensors, read by the kernels only: nothing here waits for the GPU, and
a captured CUDA graph follows what they hold when it is replayed.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _native

__all__ = ["rotary_frequencies", "rotary", "paged_append", "paged_attention"]

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_INDEX = {torch.int32: 0, torch.int64: 1}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: int = 0, low: float = 1.0, high: float = 4.0,
                       device: Optional[torch.device] = None) -> torch.Tensor:
    """Angles in radians a position of the ``rotary_dim // 2`` pairs, in 64 bits: ``base ** (-2 i / rotary_dim)``.

    ``scaling`` stretches them for contexts ``factor`` times longer:

    * ``"linear"``: every frequency divided by ``factor`` (positions interpolated);
    * ``"base"``: a larger base, which leaves the fastest pair as it is and divides the slowest by ``factor``;
    * ``"bands"``: pairs that turn fewer than ``low`` times within ``original_length`` positions are divided, those
      that turn more than ``high`` times stay, blended linearly in the number of turns between;
    * ``"ramp"``: the same with the blend linear in the pair's index, between the (whole) indices where the turns
      pass ``high`` and ``low``.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be positive and even")
    if not base > 1.0 or not factor > 0.0:
        raise ValueError("base must be over 1 and factor positive")
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("scaling 'base' needs at least two pairs")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = base ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling in ("bands", "ramp"):
        if original_length <= 0 or not high > low > 0.0:
            raise ValueError(f"scaling '{scaling}' needs original_length and high > low > 0")
        if scaling == "bands":
            keep = ((original_length * freq / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        else:
            def index(turns):
                return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

            first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), rotary_dim - 1)
            keep = 1.0 - ((i - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
    elif scaling not in ("none", "base"):
        raise ValueError(f"unknown scaling '{scaling}'")
    return freq.to(device) if device is not None else freq


def _check(err: int, what: str) -> None:
    if err != 0:
        raise RuntimeError(f"mpcomm {what} failed with CUDA error {err}")


def _stream(stream: Optional[torch.cuda.Stream], device: torch.device) -> int:
    if stream is None:
        return torch.cuda.current_stream(device).cuda_stream
    if stream.device != device:
        raise ValueError(f"stream is on {stream.device}, the tensors on {device}")
    return stream.cuda_stream


def _empty(like: torch.Tensor, shape, dtype, stream: Optional[torch.cuda.Stream]) -> torch.Tensor:
    """A new tensor that belongs to the stream it is written on."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=like.device)


def _on_gpu(what: str, device: torch.device) -> None:
    if device.type != "cuda":
        raise ValueError(f"mpcomm {what} runs on CUDA tensors, not on {device}")


def _index(t: torch.Tensor, what: str, device: torch.device) -> int:
    kind = _INDEX.get(t.dtype)
    if kind is None or t.device != device:
        raise ValueError(f"{what} must be an int32 or int64 tensor on {device}")
    return kind


def _frequencies(inv_freq: torch.Tensor, dim: int, device: torch.device) -> None:
    if inv_freq.dtype not in (torch.float64, torch.float32) or inv_freq.dim() != 1 or inv_freq.device != device \
            or not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq must be a contiguous float64 or float32 vector on {device}")
    if not 0 < 2 * inv_freq.numel() <= dim:
        raise ValueError(f"inv_freq has {inv_freq.numel()} pairs, a head of {dim} has room for 1 to {dim // 2}")


def _no_gradient(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"mpcomm {what} has no gradient: call it under torch.no_grad()")


def _own_memory(t: torch.Tensor, what: str) -> None:
    """Refuses a destination two of whose elements share a place."""
    reach = 0
    for stride, size in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        if stride <= reach:
            raise ValueError(f"{what} overlaps itself")
        reach += (size - 1) * stride


def _turn(x, positions, inv_freq, interleaved, magnitude, sign, out, stream):
    four = x.dim() == 4
    heads, dim = x.shape[-2:]
    batch, tokens = (x.shape[0], x.shape[1]) if four else (1, x.shape[0])
    xs, os = x.stride(), out.stride()
    ps = positions.stride()
    group = (x.data_ptr(), out.data_ptr(), xs[0] if four else 0, *xs[-3:], os[0] if four else 0, *os[-3:], heads, 1, -1)
    _check(_native.kv_rows([group], dim, inv_freq.numel(), interleaved, batch * tokens, tokens, inv_freq.data_ptr(),
                           inv_freq.dtype == torch.float64, magnitude, sign, positions.data_ptr(),
                           _INDEX[positions.dtype], ps[0] if positions.dim() == 2 else 0, ps[-1], None,
                           _TYPES[x.dtype], x.device.index, _stream(stream, x.device), 0), "rotary")
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, inv_freq, interleaved, magnitude, sign):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (interleaved, magnitude, sign)
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        return _turn(x, positions, inv_freq, interleaved, magnitude, sign, out, None) if x.numel() else out

    @staticmethod
    def backward(ctx, grad):
        positions, inv_freq = ctx.saved_tensors
        interleaved, magnitude, sign = ctx.how
        # the rotation is linear and its transpose is the rotation back, so a gradient of the gradient is one more
        return _Rotary.apply(grad, positions, inv_freq, interleaved, magnitude, -sign), None, None, None, None, None


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False,
           magnitude: float = 1.0, out: Optional[torch.Tensor] = None,
           stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Turns each pair of a head by ``position * inv_freq`` radians and scales it by ``magnitude``.

    ``x`` is ``[tokens, heads, head_dim]`` or ``[batch, tokens, heads, head_dim]`` (bf16, fp16 or fp32, any strides);
    ``positions`` has the shape of its token axes, or ``[tokens]`` for all of a batch (int32 or int64, negative ones
    turn back). Of each head the first ``2 * len(inv_freq)`` elements are turned, the pairs being elements ``i`` and
    ``i + len(inv_freq)``, or ``2 i`` and ``2 i + 1`` with ``interleaved``; the rest is copied unscaled. Angles are
    reduced in 64 bits, so positions may be as far as they like.

    ``out`` may be ``x`` itself, or memory apart from it. Differentiable in ``x`` (any number of times) without
    ``out`` and ``stream``. As with any autograd graph that is captured into a CUDA graph, capture the forward and
    the backward pass together, and let no eager graph of the same leaves live meanwhile.
    """
    if x.dim() not in (3, 4) or x.dtype not in _TYPES:
        raise ValueError("x must be a [(batch,) tokens, heads, head_dim] bf16, fp16 or fp32 tensor")
    device = x.device
    _index(positions, "positions", device)
    if positions.shape != x.shape[:-2] and not (x.dim() == 4 and positions.shape == x.shape[1:2]):
        raise ValueError(f"positions {tuple(positions.shape)} do not fit x {tuple(x.shape)}")
    _frequencies(inv_freq, x.shape[-1], device)
    if torch.is_grad_enabled() and x.requires_grad:
        if out is not None or stream is not None:
            raise ValueError("rotary has a gradient only without out and stream")
        _on_gpu("rotary", device)
        return _Rotary.apply(x, positions, inv_freq, bool(interleaved), float(magnitude), 1.0)
    if out is None:
        _on_gpu("rotary", device)
        out = _empty(x, x.shape, x.dtype, stream)
    else:
        if out.shape != x.shape or out.dtype != x.dtype or out.device != device:
            raise ValueError("out must have the shape, type and device of x")
        _no_gradient("rotary", out)
        _own_memory(out, "out")
    _on_gpu("rotary", device)
    if x.numel() == 0:
        return out
    return _turn(x, positions, inv_freq, bool(interleaved), float(magnitude), 1.0, out, stream)


def _batch(pool, page_table, seq_lens, query_starts, device):
    if pool.dim() != 5 or pool.shape[1] != 2 or pool.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("the cache must be a [pages, 2, kv_heads, page_tokens, head_dim] bf16 or fp16 tensor")
    kinds = (_index(page_table, "page_table", device), _index(seq_lens, "seq_lens", device),
             _index(query_starts, "query_starts", device))
    if page_table.dim() != 2 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table must be [seqs, width] with unit stride in a row")
    seqs, width = page_table.shape
    if seq_lens.shape != (seqs,) or query_starts.shape != (seqs + 1,):
        raise ValueError(f"a page_table of {seqs} sequences needs seq_lens [{seqs}] and query_starts [{seqs + 1}]")
    if not seq_lens.is_contiguous() or not query_starts.is_contiguous():
        raise ValueError("seq_lens and query_starts must be contiguous")
    if 0 in pool.shape[2:]:
        raise ValueError("the cache has no heads, no tokens in a page or no elements in a head")
    return (page_table.data_ptr(), kinds[0], page_table.stride(0), width, seq_lens.data_ptr(), kinds[1],
            query_starts.data_ptr(), kinds[2], seqs, pool.shape[3], pool.shape[0])


def _strides(t: torch.Tensor):
    """Strides, with those of axes of one element (which are not used) aligned."""
    return tuple(st if n > 1 else 8 for n, st in zip(t.shape[:-1], t.stride())) + (t.stride(-1),)


def _rows(t: torch.Tensor, what: str, pool: torch.Tensor, device: torch.device) -> None:
    if t.dim() != 3 or t.dtype != pool.dtype or t.device != device or t.shape[2] != pool.shape[4]:
        raise ValueError(f"{what} must be a [tokens, heads, {pool.shape[4]}] {pool.dtype} tensor on {device}")


def paged_append(k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, query_starts: torch.Tensor, *, inv_freq: Optional[torch.Tensor] = None,
                 interleaved: bool = False, magnitude: float = 1.0, positions: Optional[torch.Tensor] = None,
                 q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                 stream: Optional[torch.cuda.Stream] = None, status_ptr: int = 0):
    """Stores the new tokens' keys and values ``[tokens, kv_heads, head_dim]`` (any strides) in their slots of the
    cache, in one launch, and returns ``pool``.

    With ``inv_freq`` the keys are rotated on the way as :func:`rotary` does, by their places in their sequences or
    by ``positions`` ``[tokens]``. With ``q`` ``[tokens, q_heads, head_dim]`` the same launch rotates the queries too,
    into ``q_out`` (``q`` itself, memory apart from ``q``, ``k``, ``v``, or by default a new tensor), and
    ``(pool, q_out)`` is returned; padding rows of ``q_out`` stay as they were, in a new tensor undefined.

    ``pool`` is device memory or pinned host memory. A token whose column is behind the page table's width, whose
    page is outside the pool, or that lies before its sequence (``seq_lens[b]`` below its new tokens) stores nothing
    and sets bit 2 of the uint32 device word at ``status_ptr``. Slots that two tokens of one call share get one of
    them. bf16 and fp16.
    """
    device = k.device
    batch = _batch(pool, page_table, seq_lens, query_starts, device)
    if pool.device != device and not (pool.device.type == "cpu" and pool.is_pinned()):
        raise ValueError(f"the cache must lie on {device} or in pinned host memory")
    _rows(k, "k", pool, device)
    _rows(v, "v", pool, device)
    kv_heads, dim = pool.shape[2], pool.shape[4]
    if k.shape[1] != kv_heads or v.shape != k.shape:
        raise ValueError(f"k and v must have {kv_heads} heads and the same tokens")
    _no_gradient("paged_append", k, v, q, pool, q_out)
    _own_memory(pool, "the cache")
    rows = k.shape[0]
    pairs = freq = wide = 0
    if inv_freq is not None:
        _frequencies(inv_freq, dim, device)
        pairs, freq, wide = inv_freq.numel(), inv_freq.data_ptr(), inv_freq.dtype == torch.float64
    elif q is not None or positions is not None:
        raise ValueError("q and positions need inv_freq")
    pos = pos64 = pos_stride = 0
    if positions is not None:
        pos64 = _index(positions, "positions", device)
        if positions.shape != (rows,):
            raise ValueError(f"positions must be [{rows}]")
        pos, pos_stride = positions.data_ptr(), positions.stride(0)
    ps, size = pool.stride(), pool.element_size()
    slot = (ps[0], ps[3], ps[2], ps[4], kv_heads)
    at = pool.data_ptr()
    groups = [(k.data_ptr(), at, 0, *k.stride(), *slot, pairs > 0, 0),
              (v.data_ptr(), at + ps[1] * size, 0, *v.stride(), *slot, 0, 1)]
    if q is not None:
        _rows(q, "q", pool, device)
        if q.shape[0] != rows:
            raise ValueError("q must have the tokens of k")
        if q_out is None:
            _on_gpu("paged_append", device)
            q_out = _empty(q, q.shape, q.dtype, stream)
        else:
            _rows(q_out, "q_out", pool, device)
            if q_out.shape != q.shape:
                raise ValueError("q_out must have the shape of q")
            _own_memory(q_out, "q_out")
        groups.append((q.data_ptr(), q_out.data_ptr(), 0, *q.stride(), 0, *q_out.stride(), q.shape[1], 1, -1))
    elif q_out is not None:
        raise ValueError("q_out needs q")
    _on_gpu("paged_append", device)
    if rows and batch[8]:
        _check(_native.kv_rows(groups, dim, pairs, bool(interleaved), rows, rows, freq, wide, float(magnitude), 1.0,
                               pos, pos64, 0, pos_stride, batch, _TYPES[pool.dtype], device.index,
                               _stream(stream, device), status_ptr), "paged_append")
    return pool if q is None else (pool, q_out)


def paged_attention(q: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                    query_starts: torch.Tensor, *, scale: Optional[float] = None, causal: bool = True,
                    window: int = 0, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    stream: Optional[torch.cuda.Stream] = None, status_ptr: int = 0):
    """Attention of the new tokens' queries ``[tokens, q_heads, head_dim]`` over their sequences' cached tokens.

    The new tokens' own keys and values are in the cache already (:func:`paged_append`). Query head h reads key head
    ``h // (q_heads // kv_heads)``. ``scale`` is ``head_dim ** -0.5`` by default. A causal row sees the keys up to its
    own place, with ``window`` the last ``window`` of them; without ``causal`` a row sees all ``seq_lens[b]``. Single
    tokens, whole prompts and chunks may stand in one batch.

    Returns the output in ``out`` (its padding rows stay as they were) or in a new tensor (zeros there), with
    ``return_lse`` also the rows' log-sum-exp of the scaled scores, fp32 ``[tokens, q_heads]``, by which results over
    parts of a context can be joined. A row that sees no key gives zeros and -inf. Keys on pages that the table or
    the pool does not have are not seen, and set bit 2 of the uint32 device word at ``status_ptr``. Slots behind a
    sequence's end or before its window may hold anything, NaN included; a NaN or infinity in a value that some new
    token sees may reach the other new tokens of its sequence.

    bf16 and fp16, ``head_dim`` a multiple of 8 up to 128, ``page_tokens`` a multiple of 8, all strides of ``q``,
    ``out`` and ``pool`` multiples of 16 bytes but the last, which is one element. The cache is in device memory.
    """
    device = q.device
    batch = _batch(pool, page_table, seq_lens, query_starts, device)
    if pool.device != device:
        raise ValueError(f"the cache must lie on {device}")
    _rows(q, "q", pool, device)
    _no_gradient("paged_attention", q, pool, out)
    kv_heads, page_tokens, dim = pool.shape[2:]
    rows, q_heads = q.shape[0], q.shape[1]
    if q_heads == 0 or q_heads % kv_heads:
        raise ValueError(f"{q_heads} query heads cannot share {kv_heads} key heads")
    if dim % 8 or dim > 128 or page_tokens % 8:
        raise ValueError("head_dim must be a multiple of 8 up to 128, page_tokens a multiple of 8")
    if window < 0 or (window and not causal):
        raise ValueError("window must be positive, and needs causal")
    ps, qs = _strides(pool), _strides(q)
    if ps[4] != 1 or (ps[0] | ps[1] | ps[2] | ps[3]) % 8 or pool.data_ptr() % 16 or min(ps) < 1:
        raise ValueError("the cache must have unit stride in a head and 16-byte aligned strides otherwise")
    if qs[2] != 1 or (qs[0] | qs[1]) % 8 or q.data_ptr() % 16 or min(qs) < 1:
        raise ValueError("q must have unit stride in a head and 16-byte aligned strides otherwise")
    fresh = out is None
    if fresh:
        _on_gpu("paged_attention", device)
        out = _empty(q, q.shape, q.dtype, stream)
    else:
        _rows(out, "out", pool, device)
        if out.shape != q.shape:
            raise ValueError("out must have the shape of q")
        _own_memory(out, "out")
    os = _strides(out)
    if os[2] != 1 or (os[0] | os[1]) % 8 or out.data_ptr() % 16:
        raise ValueError("out must have unit stride in a head and 16-byte aligned strides otherwise")
    _on_gpu("paged_attention", device)
    lse = _empty(q, (rows, q_heads), torch.float32, stream) if return_lse else None
    if rows:
        need = _native.paged_attention_workspace(rows, q_heads, kv_heads, dim, batch[8], device.index)
        space = _empty(q, (need,), torch.uint8, stream) if need else None
        _check(_native.paged_attention(
            q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1], lse.data_ptr() if return_lse else 0,
            pool.data_ptr(), ps[0], ps[1], ps[2], ps[3], rows, q_heads, kv_heads, dim,
            dim ** -0.5 if scale is None else float(scale), bool(causal), int(window), fresh, batch,
            space.data_ptr() if need else 0, need, _TYPES[pool.dtype], device.index, _stream(stream, device),
            status_ptr), "paged_attention")
    return (out, lse) if return_lse else out
