"""GPU tests of rotary positions, appending to a paged KV cache and attention over it, against 64-bit forms."""
import math
import os
import subprocess
import sys

import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu

from mpcomm import ops  # noqa: E402
from mpcomm.models import KVPoolSpec  # noqa: E402
from mpcomm import _native  # noqa: E402

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _randn(*shape, dtype=BF16, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(dtype).cuda()


def _near(got, want, tolerance, what=""):
    bad = ~((got.double() - want).abs() <= tolerance)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: " \
        f"{got[bad][0].item()} for {want[bad][0].item()}, tolerance {tolerance[bad][0].item()}"


# ---- rotary --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,part", [(1, 1, 2, 2), (1, 40, 128, 128), (37, 3, 96, 48), (130, 5, 80, 80),
                                                   (5, 7, 10, 6), (3, 2, 256, 256), (700, 33, 64, 32),
                                                   (2, 3, 1030, 514), (9000, 5, 128, 128)])
def test_rotary_matches_the_formula(dtype, interleaved, tokens, heads, dim, part):
    x = _randn(tokens, heads, dim, dtype=dtype, seed=tokens)
    freq = ops.rotary_frequencies(part, 500000.0, "linear", 4.0, device="cuda")
    pos = torch.randint(-4, 1 << 20, (tokens,), generator=torch.Generator().manual_seed(1)).cuda()
    got = ops.rotary(x, pos, freq, interleaved=interleaved, magnitude=1.25)
    want, size = ref.rotary(x, pos, freq, interleaved, 1.25)
    _near(got, want, ref.rotary_tolerance(want, size, dtype))
    assert torch.equal(got[..., part:], x[..., part:])


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_rotary_strides_batches_and_in_place(index):
    qkv = _randn(2, 19, 12, 64, seed=3)
    freq = ops.rotary_frequencies(64, device="cuda").float()
    pos = torch.arange(19, dtype=index, device="cuda") * 1001
    for x in (qkv[:, :, 2:7], qkv.transpose(1, 2)[:, :12], qkv[:, :, :, ::2].expand(2, 19, 12, 32), qkv[..., 1:33],
              qkv[:, :, :1].expand(2, 19, 4, 64)):
        p = torch.arange(x.shape[1], dtype=index, device="cuda") * 1001
        f = freq[:x.shape[-1] // 2]
        want, size = ref.rotary(x, p.expand(x.shape[:2]), f)
        _near(ops.rotary(x, p, f), want, ref.rotary_tolerance(want, size, BF16))
        _near(ops.rotary(x, p.expand(x.shape[:2]), f), want, ref.rotary_tolerance(want, size, BF16))
    before = qkv.clone()
    part = qkv[:, :, 2:7]
    want, size = ref.rotary(part, pos.expand(2, 19), freq)
    assert ops.rotary(part, pos, freq, out=part) is part
    _near(part, want, ref.rotary_tolerance(want, size, BF16))
    assert torch.equal(qkv[:, :, :2], before[:, :, :2]) and torch.equal(qkv[:, :, 7:], before[:, :, 7:])
    wide = torch.zeros(2, 19, 9, 64, dtype=BF16, device="cuda")
    ops.rotary(before[:, :, 2:7], pos, freq, out=wide[:, :, 1:6])
    assert torch.equal(wide[:, :, 1:6], part) and not wide[:, :, 0].any() and not wide[:, :, 6:].any()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(interleaved):
    x = _randn(2, 9, 3, 16, dtype=FP32, seed=5).requires_grad_()
    freq = ops.rotary_frequencies(8, device="cuda")
    pos = torch.arange(9, device="cuda") * 77
    gy = _randn(2, 9, 3, 16, dtype=FP32, seed=6)
    y = ops.rotary(x, pos, freq, interleaved=interleaved, magnitude=0.5)
    gx, = torch.autograd.grad(y, x, gy)
    want, size = ref.rotary(gy, pos.expand(2, 9), freq, interleaved, 0.5, inverse=True)
    _near(gx, want, ref.rotary_tolerance(want, size, FP32))
    # against differences: the map is linear, so a difference over any step is its derivative, off by the roundings
    step = _randn(2, 9, 3, 16, dtype=FP32, seed=7)
    with torch.no_grad():
        d = ops.rotary(x + step, pos, freq, interleaved=interleaved, magnitude=0.5).double() - y.detach().double()
    left, right = (d * gy).sum(), (gx.double() * step).sum()
    assert abs(left - right) <= 2.0 ** -18 * (gy.abs().double() * (x.detach().abs() + step.abs()).double()).sum() * 2
    # a gradient that comes with zero strides
    ops.rotary(x, pos, freq, interleaved=interleaved).sum().backward()
    want, size = ref.rotary(torch.ones_like(x), pos.expand(2, 9), freq, interleaved, inverse=True)
    _near(x.grad, want, ref.rotary_tolerance(want, size, FP32))


def test_rotary_gradient_of_a_broadcast_head_and_double_backward():
    x = _randn(6, 1, 32, dtype=FP32).requires_grad_()
    gy = _randn(6, 4, 32, dtype=FP32, seed=1).requires_grad_()
    freq, pos = ops.rotary_frequencies(32, device="cuda"), torch.arange(6, device="cuda")
    y = ops.rotary(x.expand(6, 4, 32), pos, freq)
    gx, = torch.autograd.grad(y, x, gy, create_graph=True)
    want, size = ref.rotary(gy.detach(), pos, freq, inverse=True)
    _near(gx.detach(), want.sum(1, keepdim=True), 4 * ref.rotary_tolerance(want, size, FP32).sum(1, keepdim=True))
    back, = torch.autograd.grad(gx, gy, torch.ones_like(gx))  # the rotation of ones: the forward map again
    want, size = ref.rotary(torch.ones(6, 4, 32, device="cuda"), pos, freq)
    _near(back, want, ref.rotary_tolerance(want, size, FP32))


def test_rotary_training_step_captured_and_replayed():
    freq, pos = ops.rotary_frequencies(64, device="cuda"), torch.arange(40, device="cuda")
    x, gy = _randn(40, 4, 64).requires_grad_(), _randn(40, 4, 64, seed=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.rotary(x, pos, freq), x, gy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.rotary(x, pos, freq)
        gx, = torch.autograd.grad(y, x, gy)
    for seed in (3, 4):
        with torch.no_grad():
            x.copy_(_randn(40, 4, 64, seed=seed))
            gy.copy_(_randn(40, 4, 64, seed=seed + 10))
        graph.replay()
        for got, of, inverse in ((y, x, False), (gx, gy, True)):
            want, size = ref.rotary(of.detach(), pos, freq, inverse=inverse)
            _near(got.detach(), want, ref.rotary_tolerance(want, size, BF16))


def test_rotary_of_nothing_and_on_a_stream():
    freq = ops.rotary_frequencies(64, device="cuda")
    x = torch.empty(0, 4, 64, dtype=BF16, device="cuda")
    assert ops.rotary(x, torch.empty(0, dtype=torch.int64, device="cuda"), freq).shape == (0, 4, 64)
    z = x.clone().requires_grad_()
    ops.rotary(z, torch.empty(0, dtype=torch.int64, device="cuda"), freq).sum().backward()
    assert z.grad.shape == z.shape
    x, pos = _randn(512, 8, 64), torch.arange(512, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ops.rotary(x, pos, freq, stream=side)
    side.synchronize()
    assert torch.equal(got, ops.rotary(x, pos, freq))


# ---- append --------------------------------------------------------------------------------------------------

def _pool(pages, heads, page_tokens, dim, dtype=BF16, token_major=False, seed=9):
    if token_major:
        return _randn(pages, 2, page_tokens, heads, dim, dtype=dtype, seed=seed).transpose(2, 3)
    return _randn(pages, 2, heads, page_tokens, dim, dtype=dtype, seed=seed)


def _expect_append(pool, k, v, table, lens, starts, rotate=None):
    """The cache in 64 bits and what its elements may be off by (zero: equal)."""
    want, tol = pool.double(), torch.zeros(pool.shape, dtype=torch.float64, device=pool.device)
    for b in range(lens.numel()):
        lo, hi = int(starts[b]), int(starts[b + 1])
        for t in range(lo, hi):
            p = int(lens[b]) - (hi - t)
            if p < 0 or p // pool.shape[3] >= table.shape[1]:
                continue
            page = int(table[b, p // pool.shape[3]])
            if not 0 <= page < pool.shape[0]:
                continue
            slot = p % pool.shape[3]
            want[page, 1, :, slot] = v[t].double()
            if rotate is None:
                want[page, 0, :, slot] = k[t].double()
            else:
                y, size = ref.rotary(k[t], torch.tensor(rotate[2][t] if len(rotate) > 2 else p, device="cuda"), *rotate[:2])
                want[page, 0, :, slot] = y
                tol[page, 0, :, slot] = ref.rotary_tolerance(y, size, pool.dtype)
    return want, tol


@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("dtype,heads,dim,page_tokens,news,lens", [
    (BF16, 8, 128, 16, [1, 1, 1, 1], [1, 16, 17, 200]),
    (FP16, 2, 64, 32, [5, 0, 33, 1], [5, 70, 40, 1]),
    (BF16, 3, 80, 24, [50], [90]),
    (FP16, 1, 10, 5, [7, 3], [7, 6]),
    (BF16, 4, 128, 1, [3, 2], [3, 9]),
    (BF16, 1, 16, 8, [b % 3 for b in range(1100)], [b % 3 + b % 40 for b in range(1100)]),
])
def test_append_stores_every_token_in_its_slot(token_major, dtype, heads, dim, page_tokens, news, lens):
    table, lens, starts, pages = ref.batch(news, lens, page_tokens, device="cuda")
    rows = sum(news)
    qkv = _randn(rows, 4 * heads, dim, dtype=dtype, seed=2)
    q, k, v = qkv[:, :2 * heads], qkv[:, 2 * heads:3 * heads], qkv[:, 3 * heads:]
    pool = _pool(pages, heads, page_tokens, dim, dtype, token_major)
    want, tol = _expect_append(pool, k, v, table, lens, starts)
    assert ops.paged_append(k, v, pool, table, lens, starts) is pool
    assert torch.equal(pool.double(), want)
    # rotated, queries too
    freq = ops.rotary_frequencies(dim, device="cuda")
    pool = _pool(pages, heads, page_tokens, dim, dtype, token_major)
    want, tol = _expect_append(pool, k, v, table, lens, starts, (freq, True))
    got, turned = ops.paged_append(k, v, pool, table, lens, starts, inv_freq=freq, interleaved=True, q=q)
    assert got is pool
    _near(pool, want, tol, "cache")
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(news, lens.tolist())]).cuda()
    want, size = ref.rotary(q, pos, freq, True)
    _near(turned, want, ref.rotary_tolerance(want, size, dtype), "queries")


def test_append_in_place_padding_positions_and_int64_tables():
    news, lens = [3, 4], [20, 4]
    table, lens, starts, pages = ref.batch(news, lens, 8, index=torch.int64, device="cuda")
    wide = torch.full((2, 11), -5, dtype=torch.int64, device="cuda")
    wide[:, :table.shape[1]] = table
    table = wide[:, :table.shape[1]]  # rows further apart than they are long
    qkv = _randn(9, 8, 32, seed=2)  # two padding rows
    before = qkv.clone()
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    freq = ops.rotary_frequencies(16, device="cuda")
    places = torch.tensor([5, 4, 3, 100, 50, 2, 1, 0, 0], dtype=torch.int32, device="cuda")
    pool = _pool(pages, 2, 8, 32)
    want, tol = _expect_append(pool, k, v, table, lens, starts, (freq, False, places.tolist()))
    _, out = ops.paged_append(k, v, pool, table, lens, starts, inv_freq=freq, positions=places, q=q, q_out=q)
    assert out is q
    _near(pool, want, tol)
    turned, size = ref.rotary(before[:7, :4], places[:7], freq)
    _near(q[:7], turned, ref.rotary_tolerance(turned, size, BF16))
    assert torch.equal(q[7:], before[7:, :4]) and torch.equal(qkv[:, 4:], before[:, 4:])


def test_append_skips_tokens_without_a_slot_and_says_so():
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 99], [-1, 2], [3, 4]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([9, 3, 17], dtype=torch.int32, device="cuda")  # a bad page, a bad page, one column too many
    starts = torch.tensor([0, 9, 14, 16], dtype=torch.int32, device="cuda")  # and a sequence shorter than its tokens
    k, v = _randn(16, 1, 16), _randn(16, 1, 16, seed=1)
    pool = _pool(5, 1, 8, 16)
    want, _ = _expect_append(pool, k, v, table, lens, starts)
    ops.paged_append(k, v, pool, table, lens, starts, status_ptr=status.data_ptr())
    assert torch.equal(pool.double(), want) and status.item() == 4


def test_append_to_a_pinned_pool():
    spec = KVPoolSpec(kv_heads=2, head_dim=64, page_tokens=16)
    host = spec.make_pool(6, seed=1)
    table, lens, starts, _ = ref.batch([5, 1], [30, 17], 16, pages=6, device="cuda")
    k, v = _randn(6, 2, 64), _randn(6, 2, 64, seed=1)
    cache = spec.as_cache(host)
    want, _ = _expect_append(cache.cuda(), k, v, table, lens, starts)
    ops.paged_append(k, v, cache, table, lens, starts)
    torch.cuda.synchronize()
    assert torch.equal(cache.double(), want.cpu())


def test_append_of_nothing():
    pool = _pool(2, 1, 8, 16)
    before = pool.clone()
    none = torch.empty(0, 1, 16, dtype=BF16, device="cuda")
    zero = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.paged_append(none, none, pool, zero(1, 1), zero(1), zero(2))
    k = _randn(3, 1, 16)
    ops.paged_append(k, k, pool, zero(0, 1), zero(0), zero(1))  # all padding
    ops.paged_append(k, k, pool, zero(2, 0), zero(2) + 3, torch.tensor([0, 3, 3], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool, before)


# ---- attention -----------------------------------------------------------------------------------------------

def _attention_case(news, lens, q_heads=8, kv_heads=2, dim=128, page_tokens=16, dtype=BF16, token_major=False, pad=0,
                    index=torch.int32, causal=True, window=0, scale=None, spread=1.0, spoil=False, seed=0):
    table, lens, starts, pages = ref.batch(news, lens, page_tokens, seed=seed, index=index, device="cuda")
    pool = _pool(pages, kv_heads, page_tokens, dim, dtype, token_major, seed=seed + 1)
    if spoil:  # what no sequence holds may hold anything
        held = torch.zeros(pages, page_tokens, dtype=torch.bool)
        for b, n in enumerate(lens.tolist()):
            for p in range(n):
                held[int(table[b, p // page_tokens]), p % page_tokens] = True
        pool.permute(0, 3, 1, 2, 4)[~held.cuda()] = math.nan
    q = _randn(sum(news) + pad, q_heads, dim, dtype=dtype, seed=seed + 2, spread=spread)
    how = {"causal": causal, "window": window, "scale": scale}
    return (q, pool, table, lens, starts), how


def _check_attention(args, how, news, pad=0):
    q = args[0]
    rows = sum(news)
    want, lse, tol, ltol = ref.attention(*args, **how)
    got, got_lse = ops.paged_attention(*args, **how, return_lse=True)
    _near(got[:rows], want[:rows], tol[:rows], "out")
    empty = lse[:rows] == -math.inf
    assert torch.equal(got_lse[:rows] == -math.inf, empty) and not got[:rows][empty].any()
    _near(got_lse[:rows][~empty], lse[:rows][~empty], ltol[:rows][~empty], "lse")
    assert not got[rows:].any() and (got_lse[rows:] == -math.inf).all()
    out = _randn(*q.shape, dtype=q.dtype, seed=99)
    before = out.clone()
    assert ops.paged_attention(*args, **how, out=out) is out
    assert torch.equal(out[:rows], got[:rows]) and torch.equal(out[rows:], before[rows:])


ONE = [1]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [8, 64, 72, 128])
@pytest.mark.parametrize("news,lens", [
    (ONE, [1]), (ONE, [127]), (ONE, [128]), (ONE, [129]), (ONE, [1000]), (ONE, [4097]),
    ([1] * 9, [1, 5, 16, 17, 700, 128, 0, 256, 2000]),
    ([3, 0, 1, 200, 17], [3, 9, 1, 300, 500]),
    ([129], [129]), ([64], [1111]), ([65], [1111]), ([513], [513]),
])
def test_attention_over_lengths(dtype, dim, news, lens):
    args, how = _attention_case(news, lens, dim=dim, dtype=dtype, spoil=True)
    _check_attention(args, how, news)


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (4, 4), (8, 1), (5, 1), (14, 2), (64, 8), (48, 3), (71, 1), (300, 1)])
@pytest.mark.parametrize("news,lens", [([1, 1, 1], [300, 40, 1]), ([70, 2], [333, 2])])
def test_attention_over_head_layouts(q_heads, kv_heads, news, lens):
    args, how = _attention_case(news, lens, q_heads, kv_heads, dim=64, spoil=True, seed=3)
    _check_attention(args, how, news)


@pytest.mark.parametrize("page_tokens", [8, 16, 24, 48, 128, 200, 256])
@pytest.mark.parametrize("token_major", [False, True])
def test_attention_over_pages(page_tokens, token_major):
    news = [1, 40, 5, 1]
    args, how = _attention_case(news, [700, 300, 5, 129], page_tokens=page_tokens, token_major=token_major, spoil=True,
                                pad=4, index=torch.int64, seed=4)
    _check_attention(args, how, news, pad=4)


@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 2), (True, 100), (True, 128), (True, 5000)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_over_masks(causal, window, dim):
    news = [1, 300, 64, 1, 2]
    args, how = _attention_case(news, [1200, 700, 64, 30, 1], causal=causal, window=window, dim=dim, seed=5)
    _check_attention(args, how, news)  # the last sequence is shorter than its new tokens


@pytest.mark.parametrize("spread,scale", [(40.0, None), (0.0, None), (1.0, 0.0), (1.0, -0.3), (3.0, 1.0)])
@pytest.mark.parametrize("news", [[1, 1], [150, 3]])
def test_attention_over_scores(spread, scale, news):
    args, how = _attention_case(news, [900, 200], spread=spread, scale=scale, seed=6)
    _check_attention(args, how, news)


def test_attention_with_rising_scores_and_lowest_values():
    """Scores that grow along the context move the running maximum at every step; the lowest value of the type, as a
    mask adds it, and infinities in scores that are seen."""
    args, how = _attention_case([2], [1500], q_heads=2, kv_heads=1, dim=64, dtype=BF16, seed=7)
    q, pool, table, lens, starts = args
    q.fill_(0.125)
    for p in range(1500):
        pool[int(table[0, p // 16]), 0, 0, p % 16] = p / 8.0
    _check_attention(args, how, [2])
    q.zero_()
    q[..., 0] = 1.0
    pool[:, 0, ..., 0] = torch.finfo(BF16).min
    pool[int(table[0, 3]), 0, 0, 5, 0] = 1.0
    want, lse, tol, ltol = ref.attention(*args, **how)
    got, got_lse = ops.paged_attention(*args, **how, return_lse=True)
    _near(got, want, tol)
    pool[:, 0, ..., 0] = -math.inf
    pool[int(table[0, 3]), 0, 0, 5, 0] = 1.0
    got = ops.paged_attention(*args, **how)
    want = pool[int(table[0, 3]), 1, 0, 5].expand(2, 2, 64)
    assert torch.equal(got, want)


def test_attention_skips_bad_pages_and_says_so():
    news = [1, 5, 2]
    args, how = _attention_case(news, [200, 300, 16], dim=64, seed=8)
    q, pool, table, lens, starts = args
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.paged_attention(*args, status_ptr=status.data_ptr())
    assert status.item() == 0
    table[0, 3], table[1, 0], table[1, 18] = -1, pool.shape[0], 1 << 30
    table[2, 0] = -7  # every page of a sequence
    want, lse, tol, ltol = ref.attention(*args, **how)
    got, got_lse = ops.paged_attention(*args, return_lse=True, status_ptr=status.data_ptr())
    _near(got, want, tol)
    assert (got_lse[6:] == -math.inf).all() and not got[6:].any() and status.item() == 4
    # lengths behind the table's width
    lens[0] = 5000
    want, lse, tol, ltol = ref.attention(*args, **how)
    _near(ops.paged_attention(*args), want, tol)


def test_attention_with_values_that_the_window_has_left():
    """Pages before the window may be given to others: NaN there, and page numbers that are none."""
    args, how = _attention_case([1, 40], [500, 400], dim=128, window=70, seed=9)
    q, pool, table, lens, starts = args
    want, lse, tol, ltol = ref.attention(*args, **how)
    for b, first in ((0, 500 - 70), (1, 400 - 40 - 70 + 1)):
        for p in range(first):
            page = int(table[b, p // 16])
            if page >= 0:
                pool[page, :, :, p % 16] = math.nan
        table[b, :first // 16] = -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _near(ops.paged_attention(*args, **how, status_ptr=status.data_ptr()), want, tol)
    assert status.item() == 0


def test_attention_of_strided_queries_and_outputs():
    args, how = _attention_case([9, 1], [50, 333], q_heads=4, kv_heads=2, dim=64, seed=10)
    plain = ops.paged_attention(*args)
    qkv = torch.zeros(10, 8, 64, dtype=BF16, device="cuda")
    qkv[:, 1:5] = args[0]
    out = torch.zeros(4, 10, 64, dtype=BF16, device="cuda").transpose(0, 1)  # head-major
    ops.paged_attention(qkv[:, 1:5], *args[1:], out=out)
    assert torch.equal(out, plain)
    ops.paged_attention(qkv[:, 1:5], *args[1:], out=qkv[:, 1:5])  # in place
    assert torch.equal(qkv[:, 1:5], plain) and not qkv[:, 5:].any()


def test_attention_of_nothing():
    args, how = _attention_case([2], [20], dim=64)
    q, pool, table, lens, starts = args
    assert ops.paged_attention(q[:0], *args[1:]).shape == (0, 8, 64)
    zero = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    for tables in ((zero(0, 3), zero(0), zero(1)), (zero(1, 0), lens, starts), (table, lens * 0, starts),
                   (table, lens, starts * 0)):
        out, lse = ops.paged_attention(q, pool, *tables, return_lse=True)
        assert not out.any() and (lse == -math.inf).all()
    out, lse = ops.paged_attention(q, pool[:0], table, lens, starts, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()


def test_attention_is_the_same_every_time():
    args, how = _attention_case([1] * 5 + [300], [3000, 1, 777, 128, 129, 2000], q_heads=8, kv_heads=2, seed=11)
    first = ops.paged_attention(*args, return_lse=True)
    for _ in range(5):
        again = ops.paged_attention(*args, return_lse=True)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


def test_attention_on_two_streams_at_once():
    cases = [_attention_case([1] * 20, [2000 + 37 * i for i in range(20)], seed=s) for s in (12, 13)]
    want = [ops.paged_attention(*args) for args, _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            got[i].append(ops.paged_attention(*cases[i][0], stream=s))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_attention_captured_and_replayed_over_a_growing_context():
    args, how = _attention_case([1, 1, 4], [40, 1, 100], dim=64, seed=14)
    q, pool, table, lens, starts = args
    table = torch.randint(0, pool.shape[0], (3, 64), dtype=torch.int32, device="cuda")
    args = (q, pool, table, lens, starts)
    ops.paged_attention(*args)
    graphs = []
    for _ in range(2):  # two graphs of the same call
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_attention(*args)
        graphs.append((graph, out))
    for grow in (0, 1, 200, 700):
        lens.copy_(torch.tensor([40 + grow, 1 + grow, 100 + grow]))
        want, _, tol, _ = ref.attention(*args)
        for graph, out in graphs:
            graph.replay()
        for graph, out in graphs:
            _near(out, want, tol)


def test_attention_over_a_long_cache():
    """Offsets into the pool pass 2^32 bytes (and 2^31 elements): a pool of 4.5 GiB, most of it untouched."""
    pages = 70000
    pool = torch.empty(pages, 2, 8, 16, 128, dtype=BF16, device="cuda")
    table = torch.arange(pages - 40, pages, dtype=torch.int32, device="cuda").view(2, 20)
    lens = torch.tensor([320, 300], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    pool[-40:] = _randn(40, 2, 8, 16, 128, seed=15)
    k, v = _randn(3, 8, 128, seed=16), _randn(3, 8, 128, seed=17)
    ops.paged_append(k, v, pool, table, lens, starts)
    last = pool[int(table[1, 18]), :, :, 11]
    assert torch.equal(last[0], k[2]) and torch.equal(last[1], v[2])
    q = _randn(3, 32, 128, seed=18)
    want, _, tol, _ = ref.attention(q, pool, table, lens, starts)
    _near(ops.paged_attention(q, pool, table, lens, starts), want, tol)


# ---- together ------------------------------------------------------------------------------------------------

def test_a_prompt_in_chunks_then_tokens_through_a_host_pool():
    """What a server does: a prompt appended and attended in chunks, its pages moved to a pinned host pool and back
    into other pages, decoding going on there; against attention over all of it at once."""
    spec = KVPoolSpec(kv_heads=2, head_dim=64, page_tokens=16)
    total, chunk, heads = 150, 47, 8
    qkv = _randn(total, heads + 4, 64, seed=20)
    freq = ops.rotary_frequencies(64, 500000.0, device="cuda")
    device = torch.randint(0, 256, (24, spec.page_bytes), dtype=torch.uint8, device="cuda")
    cache = spec.as_cache(device)
    order = torch.randperm(24, generator=torch.Generator().manual_seed(1))
    table = order[:10].to(torch.int32).cuda().view(1, 10)
    got = []

    def step(lo, hi):
        x = qkv[lo:hi]
        lens = torch.tensor([hi], dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda")
        _, q = ops.paged_append(x[:, heads:heads + 2], x[:, heads + 2:], cache, table, lens, starts, inv_freq=freq, q=x[:, :heads])
        got.append(ops.paged_attention(q, cache, table, lens, starts))

    at = 0
    while at < 141:
        step(at, min(141, at + chunk))
        at = min(141, at + chunk)
    host = torch.empty(9, spec.page_bytes, dtype=torch.uint8).pin_memory()
    ops.paged_scatter(ops.paged_gather(device, table[0, :9].long()), torch.arange(9, device="cuda"), host)
    device.fill_(255)  # NaN everywhere
    table = order[12:22].to(torch.int32).cuda().view(1, 10)
    ops.paged_scatter(ops.paged_gather(host, torch.arange(9, device="cuda")), table[0, :9].long(), device)
    for t in range(141, total):
        step(t, t + 1)

    pos = torch.arange(total, device="cuda")
    q, k = ops.rotary(qkv[:, :heads], pos, freq), ops.rotary(qkv[:, heads:heads + 2], pos, freq)
    pool = torch.stack((k, qkv[:, heads + 2:])).transpose(1, 2).unsqueeze(0).contiguous()  # one page of `total` tokens
    one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    want, _, tol, _ = ref.attention(q, pool, one, one[0] + total, torch.tensor([0, total], device="cuda"))
    _near(torch.cat(got), want, tol)


def test_parts_of_a_context_join_by_their_log_sum_exp():
    args, how = _attention_case([1, 1], [640, 200], q_heads=4, kv_heads=4, dim=64, seed=21)
    q, pool, table, lens, starts = args
    want, _, tol, _ = ref.attention(*args)
    split = torch.tensor([320, 96], dtype=torch.int32, device="cuda")
    head = ops.paged_attention(q, pool, table, split, starts, causal=False, return_lse=True)
    rest = torch.stack([torch.cat([table[b, s // 16:], table[b, :s // 16]]) for b, s in enumerate((320, 96))])
    tail = ops.paged_attention(q, pool, rest, lens - split, starts, causal=False, return_lse=True)
    w = torch.softmax(torch.stack((head[1], tail[1])).double(), 0)[..., None]
    joined = w[0] * head[0].double() + w[1] * tail[0].double()
    # each part is rounded to the type once more, and its own weights: twice the tolerance of one
    size = torch.maximum(head[0].abs(), tail[0].abs()).double()
    _near(joined, want, 2 * tol + size * 2.0 ** -8)


@pytest.mark.parametrize("news,lens", [
    ([512] * 8, [512] * 8),  # many short runs of two full streams
    ([1, 300] * 10, [40, 300] * 10),  # single tokens and chunks in turn
    ([1] * 64, [130 + 61 * i for i in range(64)]),  # more sequences than a warp, odd numbers of blocks
    ([1] * 70 + [200], list(range(1, 141, 2)) + [900]),
])
def test_attention_over_many_runs_back_to_back(news, lens):
    """Runs of one and of two streams in one CTA, call after call: every call the same, and right."""
    args, how = _attention_case(news, lens, q_heads=32, kv_heads=8, spoil=True, seed=30)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _check_attention(args, how, news)
    first = ops.paged_attention(*args)
    for _ in range(200):
        again = ops.paged_attention(*args, status_ptr=status.data_ptr())
    assert torch.equal(again, first) and status.item() == 0


def test_attention_workspaces_of_any_contents():
    """Memory that was marked by other calls, and a captured call replayed with others between."""
    args, how = _attention_case([1] * 3 + [90], [5000, 900, 20, 3000], q_heads=16, kv_heads=4, seed=31)
    other, _ = _attention_case([1] * 6, [4000] * 6, q_heads=8, kv_heads=1, dim=64, seed=32)
    want, want_other = ops.paged_attention(*args), ops.paged_attention(*other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(*args)
    for n in range(30):
        junk = torch.randint(0, 256, (48 << 20,), dtype=torch.uint8, device="cuda")  # what the next call's workspace is made of
        del junk
        assert torch.equal(ops.paged_attention(*args), want)
        out.zero_()
        graph.replay()
        assert torch.equal(ops.paged_attention(*other), want_other)
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("news", [[1, 1], [70, 3]])
def test_attention_passes_on_what_is_not_a_number(news):
    """NaN in a query or in a seen key, and a score of infinity, make their rows NaN, as the formula does, and no other
    rows of their sequence's earlier tokens or of other sequences."""
    args, how = _attention_case(news, [300, 200], q_heads=4, kv_heads=2, dim=64, seed=33)
    q, pool, table, lens, starts = args
    want, _, tol, _ = ref.attention(*args)
    q[0, 1, 5] = math.nan
    got, lse = ops.paged_attention(*args, return_lse=True)
    assert got[0, 1].isnan().all() and lse[0, 1].isnan()
    rest = torch.ones(got.shape[:2], dtype=torch.bool, device="cuda")
    rest[0, 1] = False
    _near(got[rest], want[rest], tol[rest])
    q[0, 1, 5] = math.inf
    assert ops.paged_attention(*args)[0, 1].isnan().all()  # infinite scores of both signs
    q[0, 1] = 0.0
    pool[int(table[1, 0]), 0, 1, 3, 0] = math.nan  # a key of the second sequence, seen by all its tokens through heads 2, 3
    got = ops.paged_attention(*args)
    assert got[news[0]:, 2:].isnan().all() and not got[:, :2].isnan().any() and not got[:news[0]].isnan().any()


def test_append_and_attention_between_the_rows_of_one_buffer():
    """Queries, keys, values, rotated queries and outputs side by side in one buffer."""
    args, how = _attention_case([6, 1], [40, 300], q_heads=4, kv_heads=2, dim=64, seed=34)
    q, pool, table, lens, starts = args
    freq = ops.rotary_frequencies(64, device="cuda")
    k, v = _randn(7, 2, 64, seed=35), _randn(7, 2, 64, seed=36)
    other = pool.clone()
    _, turned = ops.paged_append(k, v, other, table, lens, starts, inv_freq=freq, q=q)
    want = ops.paged_attention(turned, other, table, lens, starts)
    wide = torch.cat((q, k, v, torch.zeros(7, 8, 64, dtype=BF16, device="cuda")), 1)
    ops.paged_append(wide[:, 4:6], wide[:, 6:8], pool, table, lens, starts, inv_freq=freq, q=wide[:, :4], q_out=wide[:, 8:12])
    ops.paged_attention(wide[:, 8:12], pool, table, lens, starts, out=wide[:, 12:])
    assert torch.equal(wide[:, 8:12], turned) and torch.equal(wide[:, 12:], want) and torch.equal(wide[:, :4], q)
    for bad in (wide[:, 9:13], wide[:, 7:11]):
        with pytest.raises(ValueError):
            ops.paged_attention(wide[:, 8:12], pool, table, lens, starts, out=bad)
    with pytest.raises(ValueError):
        ops.rotary(wide[:, :4], torch.arange(7, device="cuda"), freq, out=wide[:, 1:5])


@pytest.mark.parametrize("hot", [0, 4000, 8191])
@pytest.mark.parametrize("seqs,new", [(160, 1), (80, 256)])
def test_attention_in_fp16_keeps_many_small_weights(hot, seqs, new):
    """8,191 keys 25.2 powers of two below one other: their values are all that most of the output has. Enough
    sequences that a CTA reads a long run of keys against one reference.

    The weights are rounded with a step of 2^-24, off by 2^-25 each, where the largest is at least 2^7: n 2^-32 of the
    largest value for n keys. The output's own step below 2^-14 is 2^-24."""
    dim, length, page = 64, 8192, 128
    pool = torch.zeros(length // page, 2, 1, page, dim, dtype=FP16, device="cuda")
    pool[:, 1, :, :, 1:] = 1.0
    at = pool[hot // page, :, 0, hot % page]
    at[0, 0], at[1, 1:], at[1, 0] = 1.0, 0.0, 1.0
    q = torch.zeros(seqs * new, 1, dim, dtype=FP16, device="cuda")
    q[..., 0] = 17.5
    table = torch.arange(length // page, dtype=torch.int32, device="cuda").expand(seqs, -1).contiguous()
    lens = torch.full((seqs,), length, dtype=torch.int32, device="cuda")
    starts = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * new
    one, one_lse, tol, ltol = ref.attention(q[:1], pool, table[:1], lens[:1], starts[:2].clamp(max=1), scale=1.0, causal=False)
    got, lse = ops.paged_attention(q, pool, table, lens, starts, scale=1.0, causal=False, return_lse=True)
    off = length * 2.0 ** -32 + 2.0 ** -25
    _near(got, one.expand_as(got), (tol + off).expand_as(got), "out")
    _near(lse, one_lse.expand_as(lse), ltol.expand_as(lse), "lse")


@pytest.mark.parametrize("causal", [True, False])
def test_attention_says_when_a_table_is_too_narrow_or_the_pool_empty(causal):
    """Keys behind the table's last column, and those of a pool without pages, are not seen: bit 2, as of a bad page."""
    args, _ = _attention_case([1, 3], [200, 40], dim=64, seed=40)
    q, pool, table, lens, starts = args
    status, room = torch.zeros(1, dtype=torch.int32, device="cuda"), table.shape[1] * 16

    def run(*call):
        status.zero_()
        got = ops.paged_attention(*call, causal=causal, status_ptr=status.data_ptr())
        return got, status.item()

    for length, want_status in ((room, 0), (room + 1, 4), (5000, 4), (1 << 30, 4)):
        lens[0] = length
        want, _, tol, _ = ref.attention(q, pool, table, lens.clamp(max=5000), starts, causal=causal)
        got, bits = run(*args)
        _near(got, want, tol)
        assert bits == want_status, length
    wide = lens.long()
    wide[0] = 1 << 40
    assert run(q, pool, table, wide, starts)[1] == 4
    none = torch.tensor([0, 0, 4], dtype=torch.int32, device="cuda")  # nothing new in the sequence that is too long
    assert run(q, pool, table, lens, none)[1] == 0
    got, bits = run(q, pool[:0], table, lens, none)
    assert bits == 4 and not got.any()
    assert run(q, pool[:0], table, lens * 0, none)[1] == 0


def test_writes_are_seen_by_autograd():
    """A tensor that some operator saved for its backward pass is written by ours: the backward pass says so."""
    args, _ = _attention_case([1, 3], [20, 40], q_heads=4, kv_heads=2, dim=64, seed=42)
    q, pool, table, lens, starts = args
    k, v = _randn(4, 2, 64, seed=1), _randn(4, 2, 64, seed=2)
    freq, pos = ops.rotary_frequencies(64, device="cuda"), torch.arange(4, device="cuda")
    batch = (pool, table, lens, starts)
    out = torch.empty_like(q)
    for to, call in ((q, lambda: ops.rotary(q, pos, freq, out=q)), (out, lambda: ops.rotary(q, pos, freq, out=out)),
                     (pool, lambda: ops.paged_append(k, v, *batch)),
                     (q, lambda: ops.paged_append(k, v, *batch, inv_freq=freq, q=q, q_out=q)),
                     (out, lambda: ops.paged_append(k, v, *batch, inv_freq=freq, q=q, q_out=out)),
                     (out, lambda: ops.paged_attention(q, *batch, out=out)), (q, lambda: ops.paged_attention(q, *batch, out=q))):
        w = torch.ones((), dtype=BF16, device="cuda", requires_grad=True)
        y = (to * w).sum()  # saves `to`
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    read = (q, k, v, table, lens, starts, pos, freq)
    was = [t._version for t in read]
    ops.rotary(q, pos, freq), ops.paged_append(k, v, *batch, inv_freq=freq, q=q), ops.paged_attention(q, *batch)
    assert [t._version for t in read] == was
    with torch.inference_mode():
        x = torch.zeros(4, 2, 64, dtype=BF16, device="cuda")
        ops.rotary(x, pos, freq, out=x)


def test_attention_fills_the_log_sum_exp_of_padding_rows():
    """-inf whether the output is new or given."""
    args, _ = _attention_case([1, 3], [200, 40], dim=64, pad=70, seed=41)
    q, pool, table, lens, starts = args
    starts = starts + 2  # padding in front, too
    for out in (None, torch.empty_like(q)):
        junk = torch.full(q.shape[:2], 5.0, device="cuda")
        del junk
        lse = ops.paged_attention(q, pool, table, lens, starts, out=out, return_lse=True)[1]
        assert (lse[:2] == -math.inf).all() and (lse[6:] == -math.inf).all() and lse[2:6].isfinite().all()


@pytest.mark.parametrize("dim,q_heads", [(8, 1), (24, 5), (64, 40), (72, 3), (96, 7), (128, 32)])
@pytest.mark.parametrize("front,behind", [(0, 700), (300, 0), (5, 1), (700, 300)])
def test_attention_of_batches_that_are_mostly_padding(dim, q_heads, front, behind):
    """Rows of no sequence before and behind the batch's: zeros and -inf, and nothing else is touched."""
    args, _ = _attention_case([1, 3], [200, 40], q_heads, 1, dim, pad=front + behind, dtype=FP16, seed=43)
    q, pool, table, lens, starts = args
    starts = starts + front
    want, want_lse, tol, ltol = ref.attention(q, pool, table, lens, starts)
    live = slice(front, front + 4)
    junk = torch.full(q.shape, 5.0, dtype=FP16, device="cuda")
    del junk
    got, lse = ops.paged_attention(q, pool, table, lens, starts, return_lse=True)
    _near(got[live], want[live], tol[live])
    _near(lse[live], want_lse[live], ltol[live])
    for rows in (slice(0, front), slice(front + 4, None)):
        assert not got[rows].any() and (lse[rows] == -math.inf).all()
    out = torch.full((q.shape[0], q_heads + 1, dim), 7.0, dtype=FP16, device="cuda")
    ops.paged_attention(q, pool, table, lens, starts, out=out[:, :q_heads])
    assert torch.equal(out[live, :q_heads], got[live]) and (out[:, q_heads] == 7.0).all()
    assert (out[:front] == 7.0).all() and (out[front + 4:] == 7.0).all()


def test_attention_says_that_a_wait_of_an_earlier_call_ran_out():
    """The word that such a kernel writes is written from the host here: the next call raises, the one after works."""
    args, _ = _attention_case([1, 3], [200, 40], dim=64, seed=44)
    want = ops.paged_attention(*args)
    for out in (None, torch.zeros_like(args[0])):
        assert _native._paged_attention_give_up()
        with pytest.raises(RuntimeError, match="a wait in an earlier call's kernel ran out"):
            ops.paged_attention(*args, out=out)
        assert out is None or not out.any()
        assert torch.equal(ops.paged_attention(*args, out=out), want)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.paged_attention(*args, status_ptr=status.data_ptr())
    assert status.item() == 0


def test_attention_whose_first_call_is_captured():
    """In a process of its own: what the first call sets up is set up while a stream is being captured."""
    code = """
import torch
import kv_reference as ref
from mpcomm import ops
table, lens, starts, pages = ref.batch([1, 3], [200, 40], 16, device="cuda")
pool, q = (torch.randn(s, device="cuda").bfloat16() for s in ((pages, 2, 2, 16, 64), (4, 8, 64)))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = ops.paged_attention(q, pool, table, lens, starts)
graph.replay()
want, _, tol, _ = ref.attention(q, pool, table, lens, starts)
assert ((out.double() - want).abs() <= tol).all()
assert torch.equal(ops.paged_attention(q, pool, table, lens, starts), out)
"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join((here, os.path.dirname(here))))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0, r.stderr[-2000:]


def test_attention_counts_tiles_of_long_prompts():
    """Sequences of 15 to 33 tiles of 64 tokens, whose tiles a lane or a warp counts, among single tokens."""
    news = [960, 1, 1024, 1025, 1, 2117]
    args, how = _attention_case(news, [960, 300, 1500, 1025, 1, 2200], q_heads=4, kv_heads=1, dim=64, spoil=True, seed=45)
    _check_attention(args, how, news)
