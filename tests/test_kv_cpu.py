"""Paged KV cache operators without a GPU: frequencies, cache views and every refusal."""
import math
import os
import re
import shutil
import subprocess
import sys
import types

import pytest
import torch

import kv_reference as ref
from mpcomm import ops
from mpcomm.models import LLAMA3_8B_KV, KVPoolSpec
from mpcomm.ops import kv

BF16 = torch.bfloat16


def _refused(call, for_the_device=False):
    with pytest.raises(ValueError) as e:
        call()
    assert ("runs on CUDA tensors" in str(e.value)) == for_the_device, str(e.value)


def test_frequencies():
    plain = ops.rotary_frequencies(8, 10000.0)
    assert plain.dtype == torch.float64
    assert torch.allclose(plain, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert torch.equal(ops.rotary_frequencies(8, scaling="linear", factor=4.0), plain / 4.0)
    wide = ops.rotary_frequencies(8, scaling="base", factor=3.0)
    assert wide[0] == 1.0 and math.isclose(wide[-1], plain[-1] / 3.0, rel_tol=1e-13)
    n = 128
    f = ops.rotary_frequencies(n, 500000.0)
    bands = ops.rotary_frequencies(n, 500000.0, "bands", 8.0, 8192, low=1.0, high=4.0)
    ramp = ops.rotary_frequencies(n, 500000.0, "ramp", 8.0, 8192, low=1.0, high=32.0)
    index = lambda turns: n * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(500000.0))  # noqa: E731
    first, last = math.floor(index(32.0)), math.ceil(index(1.0))
    for i in range(n // 2):
        turns = 8192 * f[i].item() / (2 * math.pi)
        keep = 1.0 if turns > 4.0 else 0.0 if turns < 1.0 else (turns - 1.0) / 3.0
        assert math.isclose(bands[i], f[i] * (keep + (1 - keep) / 8.0), rel_tol=1e-12)
        keep = 1.0 - min(1.0, max(0.0, (i - first) / (last - first)))
        assert math.isclose(ramp[i], f[i] * (keep + (1 - keep) / 8.0), rel_tol=1e-12)


@pytest.mark.parametrize("args", [(7,), (0,), (8, 0.5), (8, 1e4, "spline"), (8, 1e4, "linear", 0.0), (2, 1e4, "base", 2.0),
                                  (8, 1e4, "bands", 2.0), (8, 1e4, "ramp", 2.0, 100, 4.0, 4.0)])
def test_frequencies_refuse(args):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(*args)


def test_cache_view_of_a_byte_pool():
    spec = KVPoolSpec(kv_heads=2, head_dim=8, page_tokens=4)
    pool = torch.arange(3 * spec.page_bytes, dtype=torch.int64).to(torch.uint8).view(3, spec.page_bytes)
    cache = spec.as_cache(pool)
    assert cache.shape == (3, 2, 2, 4, 8) and cache.data_ptr() == pool.data_ptr()
    cache[1, 1, 0, 2] = 1.0
    at = spec.page_bytes // 2 + 2 * 8 * 2  # the values' half of the page, third token of the first head
    assert torch.equal(pool[1, at:at + 16].view(BF16), torch.ones(8, dtype=BF16))
    assert LLAMA3_8B_KV.as_cache(torch.zeros(1, 65536, dtype=torch.uint8)).shape == (1, 2, 8, 16, 128)
    for bad, dtype in ((pool[0], BF16), (pool[:, :-2], BF16), (pool.view(torch.int8), BF16), (pool, torch.float32)):
        with pytest.raises(ValueError):
            spec.as_cache(bad, dtype)


def test_rotary_refuses():
    x, pos, freq = torch.zeros(4, 2, 16, dtype=BF16), torch.arange(4), ops.rotary_frequencies(16)
    for bad in (lambda: ops.rotary(x[0], pos, freq), lambda: ops.rotary(x.double(), pos, freq),
                lambda: ops.rotary(x, pos[:3], freq), lambda: ops.rotary(x, pos.float(), freq),
                lambda: ops.rotary(x, pos, ops.rotary_frequencies(18)), lambda: ops.rotary(x, pos, freq[:0]),
                lambda: ops.rotary(x, pos, freq.half()), lambda: ops.rotary(x, pos, freq[::2]),
                lambda: ops.rotary(x, pos, freq, out=x[:, :1]), lambda: ops.rotary(x, pos, freq, out=x.float()),
                lambda: ops.rotary(x, pos, freq, out=x[:1].expand(4, 2, 16)),
                lambda: ops.rotary(x.float().requires_grad_(), pos, freq, out=x.float())):
        _refused(bad)
    for plain in (lambda: ops.rotary(x, pos, freq, out=torch.zeros_like(x)), lambda: ops.rotary(x, pos, freq),
                  lambda: ops.rotary(x.clone().requires_grad_(), pos, freq)):
        _refused(plain, for_the_device=True)
    with pytest.raises(RuntimeError):
        ops.rotary(x, pos, freq, out=torch.zeros_like(x).requires_grad_())


def _call(op, **change):
    table, lens, starts, pages = ref.batch([3, 1], [20, 9], 8)
    a = {"q": torch.zeros(4, 4, 16, dtype=BF16), "k": torch.zeros(4, 2, 16, dtype=BF16), "v": torch.zeros(4, 2, 16, dtype=BF16),
         "pool": torch.zeros(pages, 2, 2, 8, 16, dtype=BF16), "table": table, "lens": lens, "starts": starts}
    how = {n: v for n, v in change.items() if n not in a}
    a.update({n: v(a[n]) if callable(v) else v for n, v in change.items() if n in a})
    batch = (a["pool"], a["table"], a["lens"], a["starts"])
    if op == "append":
        return ops.paged_append(a["k"], a["v"], *batch, **how)
    return ops.paged_attention(a["q"], *batch, **how)


BATCH = [
    {"pool": lambda t: t[:, 0]}, {"pool": lambda t: t[:, :1]}, {"pool": lambda t: t.float()}, {"pool": lambda t: t[..., :0]},
    {"table": lambda t: t[0]}, {"table": lambda t: t.float()}, {"table": lambda t: t.t().contiguous().t()},
    {"lens": lambda t: t[:1]}, {"lens": lambda t: t.to(torch.int16)}, {"lens": lambda t: t[:1].expand(2)},
    {"starts": lambda t: t[:2]}, {"starts": lambda t: t.double()},
]


@pytest.mark.parametrize("change", BATCH + [
    {}, {"k": lambda t: t[:, :1]}, {"k": lambda t: t.half()}, {"k": lambda t: t[..., :8]}, {"v": lambda t: t[:3]},
    {"v": lambda t: t[0]}, {"pool": lambda t: t[:1].expand(9, 2, 2, 8, 16)}, {"inv_freq": torch.ones(9)},
    {"inv_freq": torch.ones(8, dtype=torch.int64)}, {"q": None}, {"positions": torch.arange(4)},
    {"inv_freq": torch.ones(8), "positions": torch.arange(3)}, {"inv_freq": torch.ones(8), "positions": torch.ones(4)},
    {"inv_freq": torch.ones(8), "q_out": torch.zeros(4, 4, 16, dtype=BF16)},
])
def test_append_refuses(change):
    if "q" in change:  # queries without frequencies
        kv = torch.zeros(1, 2, 16, dtype=BF16)
        _refused(lambda: ops.paged_append(kv, kv, torch.zeros(1, 2, 2, 8, 16, dtype=BF16), *ref.batch([1], [1], 8)[:3], q=kv))
        return
    _refused(lambda: _call("append", **change), for_the_device=not change)


@pytest.mark.parametrize("change", BATCH + [
    {}, {"q": lambda t: t[:, :3]}, {"q": lambda t: t[:, :0]}, {"q": lambda t: t.half()}, {"q": lambda t: t[..., :8]},
    {"q": lambda t: t[0]}, {"window": -1}, {"window": 4, "causal": False}, {"out": torch.zeros(4, 4, 16)},
    {"out": torch.zeros(3, 4, 16, dtype=BF16)}, {"out": torch.zeros(1, 4, 16, dtype=BF16).expand(4, 4, 16)},
    {"out": torch.zeros(4, 4, 32, dtype=BF16)[..., ::2]}, {"out": torch.zeros(4, 4, 20, dtype=BF16)[..., :16]},
    {"q": lambda t: torch.zeros(4, 4, 20, dtype=BF16)[..., :16]}, {"q": lambda t: torch.zeros(4, 4, 17, dtype=BF16)[..., 1:]},
    {"q": lambda t: torch.zeros(16, 4, 4, dtype=BF16).permute(1, 2, 0)},
    {"pool": lambda t: torch.zeros(8, 2, 2, 8, 20, dtype=BF16)[..., :16]}, {"pool": lambda t: t[..., :12]},
    {"pool": lambda t: t[:, :, :, :4]}, {"pool": lambda t: torch.zeros(8, 2, 2, 8, 136, dtype=BF16)},
    {"pool": lambda t: torch.zeros(8, 2, 2, 16, 8, dtype=BF16).transpose(3, 4)},
])
def test_attention_refuses(change):
    _refused(lambda: _call("attention", **change), for_the_device=not change)


def test_no_silent_loss_of_gradients():
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    for op, name in (("append", "k"), ("append", "v"), ("append", "pool"), ("attention", "q"), ("attention", "pool")):
        with pytest.raises(RuntimeError, match="no gradient"):
            _call(op, **{name: grad})


def test_overlapping_destinations_are_refused():
    """The binding compares the memory that sources and destinations span before anything is launched."""
    import mpcomm

    rows, heads, dim = 4, 2, 8
    strides = (0, heads * dim, dim, 1)
    call = lambda src, dst: mpcomm._native.kv_rows(  # noqa: E731
        [(src, dst, *strides, *strides, heads, 1, -1)], dim, 0, False, 0, rows, 0, False, 1.0, 1.0, 0, 0, 0, 0, None, 0, 0, 0)
    assert call(4096, 4096) == 0  # no rows: nothing is launched
    call = lambda src, dst: mpcomm._native.kv_rows(  # noqa: E731
        [(src, dst, *strides, *strides, heads, 1, -1)], dim, 0, False, rows, rows, 0, False, 1.0, 1.0, 0, 0, 0, 0, None, 7, 0, 0)
    for shift in (2, 64, 126, -126):
        with pytest.raises(ValueError):
            call(4096, 4096 + shift)
    # rows between rows of one buffer, 6 heads wide: heads 0-1 to 2-3 and 4-5 to 0-1 share nothing, 0-1 to 1-2 do
    wide = (0, 6 * dim, dim, 1)
    call = lambda src, dst, d=-1: mpcomm._native.kv_rows(  # noqa: E731
        [(4096 + src * 16, 4096 + dst * 16, *wide, *wide, heads, 1, -1)], dim, 0, False, rows, rows, 0, False, 1.0, 1.0, 0, 0, 0,
        0, None, 7, d, 0)
    for src, dst in ((0, 2), (4, 0), (2, 4)):
        assert call(src, dst) != 0  # goes on to the launch, which has no such type or device here
    for src, dst in ((0, 1), (1, 0), (4, 5), (5, 0)):
        with pytest.raises(ValueError):
            call(src, dst)


def test_overlapping_outputs_of_attention_are_refused():
    import mpcomm

    def call(out, out_strides=(64, 16), q_strides=(64, 16), q=1 << 20, pool=1 << 30):
        batch = (0, 0, 1, 1, 0, 0, 0, 0, 1, 8, 4)
        return mpcomm._native.paged_attention(q, *q_strides, out, *out_strides, 0, pool, 512, 256, 128, 16, 4, 4, 2, 16, 1.0,
                                              True, 0, False, batch, 0, 0, 7, -1, 0)

    q = 1 << 20
    for fine in (q, q + 512, q - 512, (1 << 30) - 512):
        assert call(fine) != 0  # on to the launch
    assert call(q + 128, (128, 16), (128, 16)) != 0  # between the queries' rows
    for bad in (q + 2, q + 128, q - 128, (1 << 30) - 2, (1 << 30) + 100):
        with pytest.raises(ValueError):
            call(bad)
    with pytest.raises(ValueError):
        call(q, (64, 16), (128, 16))


def test_native_plan():
    """Index arithmetic of the paged cache and the split of attention's work over CTAs, on the host."""
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native", "bin", "test_kv")
    assert os.path.exists(exe), "native tests not built (run __graft_entry__.build())"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


def test_overlap_of_interleaved_and_degenerate_strides():
    """Axes of one element, and strides of zero, say nothing about memory; heads and elements may lie between others."""
    import mpcomm

    def call(dst, to, src=4096, of=None, rows=4, tokens=4, heads=2, dim=8):
        group = (src, src + dst * 2, *(of or to), *to, heads, 1, -1)
        return mpcomm._native.kv_rows([group], dim, 0, False, rows, tokens, 0, False, 1.0, 1.0, 0, 0, 0, 0, None, 7, -1, 0)

    for fine in (  # on to the launch, which has no such type or device here
        {"dst": 0, "to": (0, 16, 8, 1)}, {"dst": 0, "to": (0, 16, 99, 1), "of": (0, 16, 5, 1), "heads": 1},
        {"dst": 0, "to": (7, 16, 8, 1), "of": (5, 16, 8, 1)},
        {"dst": 8, "to": (0, 48, 24, 1)}, {"dst": -16, "to": (0, 48, 24, 1)},  # [tokens, heads, 3, dim]
        {"dst": 32, "to": (0, 8, 64, 1)},  # [heads, 2, tokens, dim]
        {"dst": 1, "to": (0, 32, 16, 2)},  # every second element
    ):
        assert call(**fine) != 0
    assert call(16, (32, 0, 8, 1), rows=4, tokens=1) != 0  # a batch of single tokens, between each other
    for tokens in (1, 2, 4):
        with pytest.raises(ValueError):
            call(2, (0, 0, 8, 1), tokens=tokens)  # no stride in rows at all
    for dst, to in ((4, (0, 48, 24, 1)), (24, (0, 48, 24, 1)), (28, (0, 8, 64, 1)), (8, (0, 8, 64, 1)), (2, (0, 32, 16, 2))):
        with pytest.raises(ValueError):
            call(dst, to)


def test_queries_in_place_that_are_keys_too_are_refused():
    """Turned in place while they are read as keys or values: what the cache would hold hangs on the order."""
    import mpcomm

    rows, heads, dim = 4, 2, 8
    wide = (0, 6 * dim, dim, 1)  # rows of six heads

    def call(k, v, q, q_out):
        batch = (0, 0, 1, 1, 0, 0, 0, 0, 1, 8, 4)
        plane = (2 * heads * 8 * dim, dim, 8 * dim, 1)
        group = lambda src, dst, *how: (4096 + src * dim * 2, dst, *wide, *how)  # noqa: E731
        groups = [group(k, 1 << 30, *plane, heads, 1, 0), group(v, (1 << 30) + heads * 8 * dim * 2, *plane, heads, 0, 1),
                  group(q, 4096 + q_out * dim * 2, *wide, heads, 1, -1)]
        return mpcomm._native.kv_rows(groups, dim, 0, False, rows, rows, 0, False, 1.0, 1.0, 0, 0, 0, 0, batch, 7, -1, 0)

    assert call(2, 4, 0, 0) != 0 and call(2, 4, 4 * 6, 0) != 0  # apart: on to the launch, which has no such type here
    for k, v, q in ((0, 4, 0), (1, 4, 0), (2, 1, 2), (4, 0, 0)):
        with pytest.raises(ValueError):
            call(k, v, q, q)


def test_rotated_queries_in_the_cache_are_refused():
    """Both are written by one launch, in no order."""
    import mpcomm

    rows, heads, dim, pages, cache = 4, 2, 8, 4, 1 << 30
    row, plane = (0, heads * dim, dim, 1), (2 * heads * 8 * dim * 2, dim, 8 * dim, 1)  # pages twice as far apart as they are long

    def call(q_out):
        batch = (0, 0, 1, 1, 0, 0, 0, 0, 1, 8, pages)
        groups = [(4096, cache, *row, *plane, heads, 1, 0), (8192, cache + heads * 8 * dim * 2, *row, *plane, heads, 0, 1),
                  (1 << 20, q_out, *row, *row, heads, 1, -1)]
        return mpcomm._native.kv_rows(groups, dim, 0, False, rows, rows, 0, False, 1.0, 1.0, 0, 0, 0, 0, batch, 7, -1, 0)

    page = plane[0] * 2
    for fine in (1 << 20, cache - rows * heads * dim * 2, cache + page // 2, cache + page * pages):
        assert call(fine) != 0  # on to the launch, which has no such type or device here
    for bad in (cache, cache - 2, cache + page // 2 - 2, cache + page - 2):
        with pytest.raises(ValueError):
            call(bad)


def test_more_heads_than_can_be_counted_are_refused():
    import mpcomm

    def call(*heads):
        groups = [(4096, 1 << 50, 0, 4, 2, 1, 0, 4, 2, 1, h, 1, -1) for h in heads]
        return mpcomm._native.kv_rows(groups, 2, 0, False, 1, 1, 0, False, 1.0, 1.0, 0, 0, 0, 0, None, 7, -1, 0)

    assert call(1 << 30) != 0  # on to the launch, which has no such type or device here
    for bad in ((1 << 31,), ((1 << 30) + 1,), (1 << 32,), (-1,), (1 << 29, 1 << 29, 1), (1 << 62, 1 << 62)):
        with pytest.raises(ValueError):
            call(*bad)


def test_import_on_a_torch_without_cuda():
    """What runs on the host loads and runs there; the operators refuse."""
    code = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda")]:
    delattr(torch._C, name)
from mpcomm import ops
assert ops.crc32_host(b"123456789") == 0xCBF43926
try:
    ops.rotary(torch.zeros(1, 1, 2), torch.zeros(1, dtype=torch.int64), ops.rotary_frequencies(2))
except ValueError as e:
    assert "runs on CUDA tensors" in str(e)
else:
    raise AssertionError("taken")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0, r.stderr[-2000:]


def test_no_silent_loss_of_the_gradients_of_frequencies_and_outputs():
    x, pos, freq = torch.zeros(4, 2, 16), torch.arange(4), ops.rotary_frequencies(16)
    learned = freq.clone().requires_grad_()
    q = torch.zeros(4, 4, 16, dtype=BF16)
    for call in (lambda: ops.rotary(x, pos, learned), lambda: ops.rotary(x.clone().requires_grad_(), pos, learned),
                 lambda: ops.rotary(x, pos, learned, out=torch.zeros_like(x)), lambda: _call("append", inv_freq=learned),
                 lambda: _append_q(q, learned), lambda: _append_q(q.clone().requires_grad_(), freq),
                 lambda: _append_q(q, freq, q_out=q.clone().requires_grad_()),
                 lambda: _call("attention", out=q.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            _refused(call, for_the_device=True)


def _append_q(q, inv_freq, **how):
    table, lens, starts, pages = ref.batch([3, 1], [20, 9], 8)
    kv = torch.zeros(4, 2, 16, dtype=BF16)
    return ops.paged_append(kv, kv, torch.zeros(pages, 2, 2, 8, 16, dtype=BF16), table, lens, starts, inv_freq=inv_freq, q=q, **how)


def test_no_silent_loss_of_tangents():
    x, pos, freq = torch.zeros(4, 2, 16), torch.arange(4), ops.rotary_frequencies(16)
    q = torch.zeros(4, 4, 16, dtype=BF16)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.rotary(dual(x), pos, freq), lambda: ops.rotary(x, pos, dual(freq)),
                     lambda: ops.rotary(dual(x.clone().requires_grad_()), pos, freq), lambda: ops.rotary(x, pos, freq, out=dual(x)),
                     lambda: _call("append", k=dual), lambda: _call("append", v=dual), lambda: _call("append", pool=dual),
                     lambda: _call("append", inv_freq=dual(freq)), lambda: _append_q(dual(q), freq),
                     lambda: _append_q(q, freq, q_out=dual(q)), lambda: _call("attention", q=dual),
                     lambda: _call("attention", pool=dual), lambda: _call("attention", out=dual(q))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no forward-mode gradient"):
                    call()
        saved = types.SimpleNamespace(saved_tensors=(pos, freq), how=(False, 1.0, 1.0))
        with pytest.raises(RuntimeError, match="no forward-mode gradient"):
            kv._Rotary.backward(saved, dual(x))
        _refused(lambda: ops.rotary(x, pos, freq), for_the_device=True)  # plain tensors are taken
        _refused(lambda: _call("attention"), for_the_device=True)


def test_attention_kernels_have_the_registers_that_their_warps_divide(tmp_path):
    """The warps take and give registers of what a CTA is launched with, which is what the compiler chose: as many as
    the source counts on, or every launch is refused. Nothing may be spilled either."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no CUDA compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    source = os.path.join(root, "csrc", "kernels", "paged_attention.cu")
    want = re.search(r"kRegsLaunch = (\d+)", open(source).read()).group(1)
    r = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-DNDEBUG", "--expt-relaxed-constexpr",
                        "-std=c++17", "-I" + os.path.join(root, "csrc"), "-I" + os.path.join(root, "include"), "-Xptxas", "-v",
                        "-cubin", "-o", str(tmp_path / "kernels.cubin"), source], capture_output=True, text=True, timeout=500)
    assert r.returncode == 0, r.stderr[-2000:]
    found = re.findall(r"Compiling entry function '\S*?(paged_attention_kernel|join_kernel)(?:.*\n)*?.*?(\d+) bytes spill stores"
                       r"(?:.*\n)*?.*?Used (\d+) registers", r.stderr)
    assert sorted(name for name, _, _ in found) == ["join_kernel"] * 4 + ["paged_attention_kernel"] * 4, r.stderr[-2000:]
    for name, spilled, registers in found:
        assert spilled == "0"
        assert name == "join_kernel" or registers == want
