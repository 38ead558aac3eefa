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

Tensors that a call writes and the caller gave (``out``, ``q_out``, the cache) count as changed in place: autograd
refuses a backward pass that had saved what they held, as after any such operator of torch.
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .. import _native

__all__ = ["rotary_frequencies", "rotary", "paged_append", "paged_attention"]

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_CACHE_TYPES = (torch.bfloat16, torch.float16)
_WAIT_RAN_OUT = -1  # of a native call
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


# A call of a few tokens is over on the GPU in microseconds, so the checks below read each tensor's shape, strides and
# device once, and compare plain integers.

# Of a device's number: the raw handle, without a Stream object. A torch without CUDA has no such function.
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _check(err: int, what: str) -> None:
    if err != 0:
        raise RuntimeError(f"mpcomm {what} failed with CUDA error {err}")


def _stream(stream: Optional[torch.cuda.Stream], device: int) -> int:
    if stream is None:
        return _current_stream(device)
    if stream.device.index != device:
        raise ValueError(f"stream is on {stream.device}, the tensors on cuda:{device}")
    return stream.cuda_stream


def _empty(like: torch.Tensor, shape, dtype, stream: Optional[torch.cuda.Stream]) -> torch.Tensor:
    """A new tensor that belongs to the stream it is written on."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _empty_like(like: torch.Tensor, stream: Optional[torch.cuda.Stream]) -> torch.Tensor:
    """The same of the shape and type of another, whatever its strides. 1.5 us; torch.empty, given all by name, 3.3."""
    if stream is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    with torch.cuda.stream(stream):
        return torch.empty_like(like, memory_format=torch.contiguous_format)


def _on_gpu(what: str, device: int) -> None:
    if device < 0:
        raise ValueError(f"mpcomm {what} runs on CUDA tensors")


def _index(t: torch.Tensor, what: str, device: int) -> int:
    kind = _INDEX.get(t.dtype)
    if kind is None or t.get_device() != device:
        raise ValueError(f"{what} must be an int32 or int64 tensor on the other tensors' device")
    return kind


def _frequencies(inv_freq: torch.Tensor, dim: int, device: int) -> int:
    """The number of pairs."""
    if inv_freq.dtype not in (torch.float64, torch.float32) or inv_freq.dim() != 1 or inv_freq.get_device() != device \
            or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float64 or float32 vector on the other tensors' device")
    pairs = inv_freq.shape[0]
    if not 0 < 2 * pairs <= min(dim, 8192):
        raise ValueError(f"inv_freq has {pairs} pairs, a head of {dim} has room for 1 to {min(dim, 8192) // 2}")
    return pairs


def _no_gradient(what: str) -> None:
    raise RuntimeError(f"mpcomm {what} has no gradient: call it under torch.no_grad()")


def _no_tangents(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses forward-mode differentiation, which the kernels would lose. Outside of a dual level (a number of 0 or
    more, where torch says it) no tensor has a tangent, and looking at none of them saves half a microsecond each."""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"mpcomm {what} has no forward-mode gradient")


def _own_memory(t: torch.Tensor, what: str) -> None:
    """Refuses a destination two of whose elements share a place."""
    if t.is_contiguous():
        return
    reach = 0
    for stride, size in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        if stride <= reach:
            raise ValueError(f"{what} overlaps itself")
        reach += (size - 1) * stride


def _turn(x, positions, inv_freq, interleaved, magnitude, sign, out, stream):
    shape, xs, os, ps, device = x.shape, x.stride(), out.stride(), positions.stride(), x.get_device()
    if len(shape) == 4:
        batch, tokens, heads, dim = shape
        group = (x.data_ptr(), out.data_ptr(), *xs, *os, heads, 1, -1)
    else:
        tokens, heads, dim = shape
        batch = 1
        group = (x.data_ptr(), out.data_ptr(), 0, *xs, 0, *os, heads, 1, -1)
    err = _native.kv_rows((group,), dim, inv_freq.shape[0], interleaved, batch * tokens, tokens, inv_freq.data_ptr(),
                          inv_freq.dtype is torch.float64, magnitude, sign, positions.data_ptr(),
                          _INDEX[positions.dtype], ps[0] if len(ps) == 2 else 0, ps[-1], None, _TYPES[x.dtype], device,
                          _stream(stream, device), 0)
    if err:
        _check(err, "rotary")
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, inv_freq, how):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = how
        out = _empty_like(x, None)
        return out if 0 in x.shape else _turn(x, positions, inv_freq, *how, out, None)

    @staticmethod
    def backward(ctx, grad):
        # the rotation is linear and its transpose is the rotation back, so a gradient of the gradient is one more
        positions, inv_freq = ctx.saved_tensors
        interleaved, magnitude, sign = ctx.how
        _no_tangents("rotary's gradient", grad)
        if grad.requires_grad and torch.is_grad_enabled():
            return _Rotary.apply(grad, positions, inv_freq, (interleaved, magnitude, -sign)), None, None, None
        out = _empty_like(grad, None)
        if 0 not in grad.shape:
            _turn(grad, positions, inv_freq, interleaved, magnitude, -sign, out, None)
        return out, None, None, None


def rotary(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *, interleaved: bool = False,
           magnitude: float = 1.0, out: Optional[torch.Tensor] = None,
           stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Turns each pair of a head by ``position * inv_freq`` radians and scales it by ``magnitude``.

    ``x`` is ``[tokens, heads, head_dim]`` or ``[batch, tokens, heads, head_dim]`` (bf16, fp16 or fp32, any strides);
    ``positions`` has the shape of its token axes, or ``[tokens]`` for all of a batch (int32 or int64, negative ones
    turn back). Of each head the first ``2 * len(inv_freq)`` elements are turned, the pairs being elements ``i`` and
    ``i + len(inv_freq)``, or ``2 i`` and ``2 i + 1`` with ``interleaved``; the rest is copied unscaled. Angles are
    reduced in 64 bits, off by at most 2^-51 of themselves: by 2^-20 radians at a position of 2^31 and a radian each.

    ``out`` may be ``x`` itself, or memory apart from it. Differentiable in ``x`` (any number of times) without
    ``out`` and ``stream``, not in ``inv_freq``: frequencies that require a gradient are refused, and so is
    forward mode. As with any autograd graph that is captured into a CUDA graph, capture the forward and
    the backward pass together, and let no eager graph of the same leaves live meanwhile.
    """
    shape, device = x.shape, x.get_device()
    if len(shape) not in (3, 4) or x.dtype not in _TYPES:
        raise ValueError("x must be a [(batch,) tokens, heads, head_dim] bf16, fp16 or fp32 tensor")
    _index(positions, "positions", device)
    if positions.shape != shape[:-2] and not (len(shape) == 4 and positions.shape == shape[1:2]):
        raise ValueError(f"positions {tuple(positions.shape)} do not fit x {tuple(shape)}")
    _frequencies(inv_freq, shape[-1], device)
    _no_tangents("rotary", x, inv_freq, out)
    if inv_freq.requires_grad and torch.is_grad_enabled():
        _no_gradient("rotary in inv_freq")
    if x.requires_grad and torch.is_grad_enabled():
        if out is not None or stream is not None:
            raise ValueError("rotary has a gradient only without out and stream")
        _on_gpu("rotary", device)
        return _Rotary.apply(x, positions, inv_freq, (bool(interleaved), float(magnitude), 1.0))
    given = out
    if out is None:
        _on_gpu("rotary", device)
        out = _empty_like(x, stream)
    else:
        if out.shape != shape or out.dtype != x.dtype or out.get_device() != device:
            raise ValueError("out must have the shape, type and device of x")
        if out.requires_grad and torch.is_grad_enabled():
            _no_gradient("rotary into out")
        _own_memory(out, "out")
        _on_gpu("rotary", device)
    if 0 not in shape:
        _turn(x, positions, inv_freq, bool(interleaved), float(magnitude), 1.0, out, stream)
        if given is not None:
            increment_version(given)
    return out


def _batch(pool, page_table, seq_lens, query_starts, device):
    """The cache's shape and the batch as the native calls take it."""
    shape = pool.shape
    if len(shape) != 5 or shape[1] != 2 or pool.dtype not in _CACHE_TYPES:
        raise ValueError("the cache must be a [pages, 2, kv_heads, page_tokens, head_dim] bf16 or fp16 tensor")
    if 0 in shape[2:]:
        raise ValueError("the cache has no heads, no tokens in a page or no elements in a head")
    if page_table.dim() != 2:
        raise ValueError("page_table must be [seqs, width]")
    seqs, width = page_table.shape
    row, one = page_table.stride()
    if one != 1 and width > 1:
        raise ValueError("page_table must have unit stride in a row")
    if seq_lens.shape != (seqs,) or query_starts.shape != (seqs + 1,):
        raise ValueError(f"a page_table of {seqs} sequences needs seq_lens [{seqs}] and query_starts [{seqs + 1}]")
    if not (seq_lens.is_contiguous() and query_starts.is_contiguous()):
        raise ValueError("seq_lens and query_starts must be contiguous")
    return shape, (page_table.data_ptr(), _index(page_table, "page_table", device), row, width,
                   seq_lens.data_ptr(), _index(seq_lens, "seq_lens", device),
                   query_starts.data_ptr(), _index(query_starts, "query_starts", device), seqs, shape[3], shape[0])


def _rows(t: torch.Tensor, what: str, pool: torch.Tensor, dim: int, device: int):
    """The shape of a tensor of new tokens."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or t.dtype != pool.dtype or t.get_device() != device:
        raise ValueError(f"{what} must be a [tokens, heads, {dim}] {pool.dtype} tensor on the other tensors' device")
    return shape


def _aligned(t: torch.Tensor, shape, what: str):
    """Strides that wide accesses can take. Those of axes of one element are not used; they are given as 8."""
    strides = t.stride()
    if 1 in shape:
        strides = tuple(st if n > 1 else 8 for n, st in zip(shape[:-1], strides)) + strides[-1:]
    bits = 0
    for st in strides[:-1]:
        bits |= st if st > 0 else 1
    if strides[-1] != 1 or bits % 8 or t.data_ptr() % 16:
        raise ValueError(f"{what} must have unit stride in a head, other strides of 16 bytes or multiples, aligned to 16 bytes")
    return strides


def paged_append(k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, query_starts: torch.Tensor, *, inv_freq: Optional[torch.Tensor] = None,
                 interleaved: bool = False, magnitude: float = 1.0, positions: Optional[torch.Tensor] = None,
                 q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                 stream: Optional[torch.cuda.Stream] = None, status_ptr: int = 0):
    """Stores the new tokens' keys and values ``[tokens, kv_heads, head_dim]`` (any strides) in their slots of the
    cache, in one launch, and returns ``pool``.

    With ``inv_freq`` the keys are rotated on the way as :func:`rotary` does, by their places in their sequences or
    by ``positions`` ``[tokens]``. With ``q`` ``[tokens, q_heads, head_dim]`` the same launch rotates the queries too,
    into ``q_out`` (``q`` itself, memory apart from ``q``, or by default a new tensor; apart from ``k``, ``v`` and the
    cache), and ``(pool, q_out)`` is returned; padding rows of ``q_out`` stay as they were, in a new tensor undefined.

    ``pool`` is device memory or pinned host memory. A token whose column is behind the page table's width, whose
    page is outside the pool, or that lies before its sequence (``seq_lens[b]`` below its new tokens) stores nothing
    and sets bit 2 of the uint32 device word at ``status_ptr``. Slots that two tokens of one call share get one of
    them. bf16 and fp16.
    """
    device = k.get_device()
    cache, batch = _batch(pool, page_table, seq_lens, query_starts, device)
    kv_heads, dim = cache[2], cache[4]
    if pool.get_device() != device and not (pool.device.type == "cpu" and pool.is_pinned()):
        raise ValueError("the cache must lie on the other tensors' device or in pinned host memory")
    shape = _rows(k, "k", pool, dim, device)
    if shape[1] != kv_heads or _rows(v, "v", pool, dim, device) != shape:
        raise ValueError(f"k and v must have {kv_heads} heads and the same tokens")
    if (k.requires_grad or v.requires_grad or pool.requires_grad or (q is not None and q.requires_grad)
            or (q_out is not None and q_out.requires_grad)
            or (inv_freq is not None and inv_freq.requires_grad)) and torch.is_grad_enabled():
        _no_gradient("paged_append")
    _no_tangents("paged_append", k, v, pool, q, q_out, inv_freq)
    _own_memory(pool, "the cache")
    rows = shape[0]
    pairs = freq = wide = 0
    if inv_freq is not None:
        pairs, freq, wide = _frequencies(inv_freq, dim, device), inv_freq.data_ptr(), inv_freq.dtype is torch.float64
    elif q is not None or positions is not None:
        raise ValueError("q and positions need inv_freq")
    pos = pos64 = pos_stride = 0
    if positions is not None:
        pos64 = _index(positions, "positions", device)
        if positions.shape != (rows,):
            raise ValueError(f"positions must be [{rows}]")
        pos, pos_stride = positions.data_ptr(), positions.stride(0)
    page, plane, head, token, element = pool.stride()
    at, turn = pool.data_ptr(), pairs > 0
    groups = ((k.data_ptr(), at, 0, *k.stride(), page, token, head, element, kv_heads, turn, 0),
              (v.data_ptr(), at + plane * 2, 0, *v.stride(), page, token, head, element, kv_heads, 0, 1))
    written = [pool]
    if q is not None:
        q_shape = _rows(q, "q", pool, dim, device)
        if q_shape[0] != rows:
            raise ValueError("q must have the tokens of k")
        if q_out is None:
            _on_gpu("paged_append", device)
            q_out = _empty_like(q, stream)
        else:
            if _rows(q_out, "q_out", pool, dim, device) != q_shape:
                raise ValueError("q_out must have the shape of q")
            _own_memory(q_out, "q_out")
            written.append(q_out)
        groups += ((q.data_ptr(), q_out.data_ptr(), 0, *q.stride(), 0, *q_out.stride(), q_shape[1], 1, -1),)
    elif q_out is not None:
        raise ValueError("q_out needs q")
    _on_gpu("paged_append", device)
    if rows and batch[8]:
        err = _native.kv_rows(groups, dim, pairs, bool(interleaved), rows, rows, freq, wide, float(magnitude), 1.0, pos,
                              pos64, 0, pos_stride, batch, _TYPES[pool.dtype], device, _stream(stream, device), status_ptr)
        if err:
            _check(err, "paged_append")
        increment_version(written)
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
    parts of a context can be joined. A row that sees no key gives zeros and -inf, a padding row -inf.
    Keys on pages that the table or the pool does not have (a table too narrow for ``seq_lens`` among them) are not
    seen, and set bit 2 of the uint32 device word at ``status_ptr``. Slots behind a sequence's end or before its
    window may hold anything, NaN included; a NaN or infinity in a value that some new token sees may reach the other
    new tokens of its sequence.

    The kernel's waits are bounded. One that ran out (a GPU that does not work as it should) leaves outputs that mean
    nothing: it sets bit 0 of the word at ``status_ptr``, and without one the next call raises a ``RuntimeError``.

    bf16 and fp16, ``head_dim`` a multiple of 8 up to 128, ``page_tokens`` a multiple of 8, all strides of ``q``,
    ``out`` and ``pool`` multiples of 16 bytes but the last, which is one element. The cache is in device memory.
    A call takes a workspace of its own, 39 MB on 148 SMs for heads over 64 and 20 MB up to 64, whatever its sizes.
    """
    device = q.get_device()
    cache, batch = _batch(pool, page_table, seq_lens, query_starts, device)
    _, _, kv_heads, page_tokens, dim = cache
    if pool.get_device() != device:
        raise ValueError("the cache must lie on the other tensors' device")
    shape = _rows(q, "q", pool, dim, device)
    rows, q_heads, _ = shape
    if (q.requires_grad or pool.requires_grad or (out is not None and out.requires_grad)) and torch.is_grad_enabled():
        _no_gradient("paged_attention")
    _no_tangents("paged_attention", q, pool, out)
    if q_heads == 0 or q_heads % kv_heads:
        raise ValueError(f"{q_heads} query heads cannot share {kv_heads} key heads")
    if dim % 8 or dim > 128 or page_tokens % 8:
        raise ValueError("head_dim must be a multiple of 8 up to 128, page_tokens a multiple of 8")
    if window < 0 or (window and not causal):
        raise ValueError("window must be positive, and needs causal")
    page, plane, head, token, _ = _aligned(pool, cache, "the cache")
    q_token, q_head, _ = _aligned(q, shape, "q")
    fresh = out is None
    if fresh:
        _on_gpu("paged_attention", device)
        out = _empty_like(q, stream)
    else:
        if _rows(out, "out", pool, dim, device) != shape:
            raise ValueError("out must have the shape of q")
        _own_memory(out, "out")
    o_token, o_head, _ = _aligned(out, shape, "out")
    _on_gpu("paged_attention", device)
    lse = _empty(q, (rows, q_heads), torch.float32, stream) if return_lse else None
    if rows:
        need = _workspace(dim > 64, device)
        space = _empty(q, need, torch.uint8, stream)
        err = _native.paged_attention(
            q.data_ptr(), q_token, q_head, out.data_ptr(), o_token, o_head, lse.data_ptr() if return_lse else 0,
            pool.data_ptr(), page, plane, head, token, rows, q_heads, kv_heads, dim,
            dim ** -0.5 if scale is None else float(scale), bool(causal), window, fresh, batch, space.data_ptr(), need,
            _TYPES[pool.dtype], device, _stream(stream, device), status_ptr)
        if err:
            if err == _WAIT_RAN_OUT:
                raise RuntimeError("mpcomm paged_attention: a wait in an earlier call's kernel ran out, what that call "
                                   "returned is not to be used; this call did nothing")
            _check(err, "paged_attention")
        if not fresh:
            increment_version(out)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=None)
def _workspace(wide: bool, device: int) -> int:
    """Bytes that a call needs on a device, whatever its sizes but for heads of over 64 elements."""
    return _native.paged_attention_workspace(128 if wide else 64, device)
