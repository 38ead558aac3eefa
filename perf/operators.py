"""The operators of a paged KV cache, as cases to measure: rotary positions, appending keys and values to the
cache with the rotation applied on the way, and attention of new tokens over the cached pages.

A case is a dict of plain values. ``prepare`` makes what a serving or training program holds before the call,
``run`` is one pass of the operator: in elementary torch operations, or (``own``) through ``mpcomm.ops``.
``exact`` is the operator's definition in 64 bits.

A batch is ragged: the rows of sequence b are ``starts[b] .. starts[b + 1]``, they are its newest tokens, and
``lens[b]`` counts all its tokens, those rows among them. Token p of a sequence lies in slot ``p % page_tokens``
of page ``table[b, p // page_tokens]``. Rows behind the last sequence are padding and stay as they were.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_SCORES = 4096 * 16384 * 32  # scores of the largest listed chunk, padding included
MOST_GATHER = 64 * 8192 * 8 * 128  # keys of the largest listed decode batch, padding included


# ---- cases -----------------------------------------------------------------------------------------------

def _rotary(name, dtype, batch, tokens, heads, dim, part, interleaved, far, train, scaling="none"):
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "tokens": tokens, "heads": heads, "dim": dim,
            "part": part, "interleaved": interleaved, "far": far, "train": train, "scaling": scaling}


def _cache(name, op, dtype, seqs, new, kv, q_heads, kv_heads, dim, page_tokens, ragged, chunks, **more):
    c = {"name": name, "op": op, "dtype": dtype, "seqs": seqs, "new": new, "kv": kv, "q_heads": q_heads, "kv_heads": kv_heads,
         "dim": dim, "page_tokens": page_tokens, "ragged": ragged, "chunks": chunks, "token_major": False, "pad": 0}
    if op == "append":
        c.update({"part": dim, "interleaved": False, "rotate": True, "scaling": "none"})
    else:
        c.update({"causal": True, "window": 0, "lse": False})
    c.update(more)
    return c


def listed():
    return [
        # queries and keys of one decoding step of a few requests: 8 rows of a fused projection; launch latency counts
        _rotary("rotary_step", "bf16", 1, 8, 40, 128, 128, False, 8192, False),
        # a training step's queries: two sequences of 4,096 tokens, forward and gradient
        _rotary("rotary_train", "bf16", 2, 4096, 32, 128, 128, False, 4096, True),
        # a long-context variant: interleaved pairs, half of each head, scaled frequencies, far positions, odd count
        _rotary("rotary_far", "fp16", 1, 4099, 24, 96, 48, True, 1 << 20, True, "bands"),
        # one decoding step of 64 requests: a token each into the 64 KiB pages of the 8-head, 128-wide cache
        _cache("append_step", "append", "bf16", 64, 1, 8192, 32, 8, 128, 16, True, 64),
        # prompts being read: four ragged chunks of up to 4,096 tokens
        _cache("append_chunk", "append", "bf16", 4, 4096, 8192, 32, 8, 128, 16, True, 4),
        # another model's layout: token-major pages, 64-wide heads, interleaved pairs, padded rows
        _cache("append_odd", "append", "fp16", 7, 301, 1999, 12, 4, 64, 32, True, 7, token_major=True, interleaved=True, part=32,
               pad=5, scaling="linear"),
        # one request decoding alone: the smallest call
        _cache("decode_one", "attention", "bf16", 1, 1, 1000, 32, 8, 128, 16, False, 1),
        # a serving batch decoding: 64 requests of up to 8,192 tokens
        _cache("decode_batch", "attention", "bf16", 64, 1, 8192, 32, 8, 128, 16, True, 64),
        # two very long contexts decoding
        _cache("decode_long", "attention", "bf16", 2, 1, 131072, 32, 8, 128, 16, False, 2, lse=True),
        # prompts in chunks next to decoding requests, as a serving step mixes them
        _cache("mixed_step", "attention", "bf16", 34, 512, 4096, 32, 8, 128, 16, True, 2, pad=3),
        # a sliding window, 64-wide heads, six queries to a key head, token-major pages of 32
        _cache("chunk_window", "attention", "fp16", 8, 777, 2500, 24, 4, 64, 32, True, 8, window=512, token_major=True, lse=True),
        # a large chunk of one long prompt
        _cache("chunk_large", "attention", "bf16", 1, 4096, 16384, 32, 8, 128, 16, False, 1),
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention"])
    scaling = rng.choice(["none", "linear", "bands"])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        heads, batch = _log(rng, 1, 64), rng.choice([1, 1, 2, 3])
        tokens = _log(rng, 1, max(1, min(16384, 8192 * 32 * 128 // (dim * heads * batch))))
        return {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "batch": batch, "tokens": tokens, "heads": heads, "dim": dim,
                "part": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.4, "far": _log(rng, 2048, 1 << 20),
                "train": rng.random() < 0.5, "scaling": scaling}
    dim, kv_heads, group = rng.choice([64, 80, 96, 128, 128]), rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([1, 2, 4, 4, 5, 8])
    q_heads = kv_heads * group
    seqs = _log(rng, 1, 128)
    c = {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "seqs": seqs, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
         "page_tokens": rng.choice([8, 16, 16, 32, 64, 128, 48]), "ragged": rng.random() < 0.7, "token_major": rng.random() < 0.4,
         "pad": rng.choice([0, 0, 1, 6])}
    if op == "append":
        c["new"] = rng.choice([1, _log(rng, 1, max(1, min(4096, 4 * 4096 * 48 * 128 // (seqs * (q_heads + 2 * kv_heads) * dim))))])
        c["kv"] = c["new"] + _log(rng, 1, 8192)
        c.update({"chunks": seqs, "part": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.4, "rotate": rng.random() < 0.8,
                  "scaling": scaling})
        return c
    c["kv"] = _log(rng, 1, max(1, min(131072, MOST_GATHER // (seqs * kv_heads * dim))))
    c["new"] = rng.choice([1, _log(rng, 1, max(1, min(4096, c["kv"], MOST_SCORES // (seqs * q_heads * c["kv"]))))])
    c["chunks"] = rng.choice([seqs, seqs, max(1, seqs // 16)])
    c["causal"] = rng.random() < 0.85
    c["window"] = _log(rng, 16, 8192) if c["causal"] and rng.random() < 0.3 else 0
    c["lse"] = rng.random() < 0.4
    return c


def _lengths(case):
    """New and all tokens of each sequence: of the case alone, the first sequence with the most of both."""
    rng = random.Random("%(seqs)d %(new)d %(kv)d %(chunks)d" % case)
    new, lens = [], []
    for b in range(case["seqs"]):
        n = case["new"] if b < case["chunks"] else 1
        if case["ragged"] and b:
            n = rng.randint(max(1, n // 4), n)
            if b % 7 == 6 and case["new"] > 1:
                n = 0  # a request that has nothing in this step
        new.append(n)
        lens.append(rng.randint(max(n, case["kv"] // 4), case["kv"]) if case["ragged"] and b else case["kv"])
    return new, lens


def _frequencies(part, scaling):
    """Radians a position for each pair, as a model's configuration gives them: plain, divided by a factor, or divided
    for the long wavelengths only, with a smooth band between."""
    f = torch.arange(0, part, 2, dtype=torch.float64) / part
    f = 500000.0 ** -f
    if scaling == "linear":
        f = f / 4.0
    if scaling == "bands":
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / 8.0 * (1 - keep)
    return f


def _magnitude(scaling):
    return 1.0 if scaling == "none" else 1.1


# ---- inputs ----------------------------------------------------------------------------------------------

def _randn(shape, dtype, g, spread=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(spread).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "rotary":
        shape = (case["batch"], case["tokens"], case["heads"], case["dim"])
        s["x"] = _randn(shape, dtype, g).requires_grad_(case["train"])
        s["positions"] = torch.randint(0, case["far"], shape[:2], generator=g, device="cuda", dtype=torch.int64)
        s["inv_freq"] = _frequencies(case["part"], case["scaling"]).cuda()
        if case["train"]:
            s["gy"] = _randn(shape, dtype, g)
        return s
    new, lens = _lengths(case)
    rows, hq, hk, d, p = sum(new) + case["pad"], case["q_heads"], case["kv_heads"], case["dim"], case["page_tokens"]
    held = [-(-n // p) for n in lens]
    pages = sum(held) + 3
    s["rows"], s["new"], s["lens_host"] = sum(new), max(new), max(lens)
    s["starts"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    width = max(held) + 2  # columns behind a sequence's own pages are not looked at
    at = torch.tensor([sum(held[:b]) for b in range(len(held))], device="cuda")[:, None] + torch.arange(width, device="cuda")
    s["table"] = order[at.clamp(max=pages - 1)].contiguous()
    shape = (pages, 2, p, hk, d) if case["token_major"] else (pages, 2, hk, p, d)
    pool = torch.empty(shape, dtype=dtype, device="cuda")
    step = max(1, (1 << 28) // (2 * hk * p * d))
    for i in range(0, pages, step):
        pool[i:i + step] = _randn((min(step, pages - i),) + shape[1:], dtype, g)
    s["pool"] = pool.transpose(2, 3) if case["token_major"] else pool  # [pages, 2, kv heads, page tokens, dim]
    # queries, keys and values are parts of one fused projection's rows
    s["qkv"] = _randn((rows, hq + 2 * hk, d), dtype, g, 1.5)
    s["q"], s["k"], s["v"] = s["qkv"][:, :hq], s["qkv"][:, hq:hq + hk], s["qkv"][:, hq + hk:]
    s["out"] = _randn((rows, hq, d), dtype, g)  # a step's own buffer, with the last step's rows in it
    if case["op"] == "append":
        s["inv_freq"] = _frequencies(case["part"], case["scaling"]).cuda() if case["rotate"] else None
    return s


# ---- the plain forms -------------------------------------------------------------------------------------

def _rotate(x, angle, interleaved, magnitude, sign):
    """x [..., heads, dim] in 32 bits, angle [..., pairs] in 64."""
    half = angle.shape[-1]
    cos = (torch.cos(angle) * magnitude).float().unsqueeze(-2)
    sin = (torch.sin(angle) * magnitude * sign).float().unsqueeze(-2)
    part, rest = x[..., :2 * half].float(), x[..., 2 * half:].float()
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _places(s):
    """Sequence and position of each row that is not padding."""
    row = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"][1:].contiguous(), row, right=True)
    first = s["starts"][:-1]
    position = (s["lens"] - (s["starts"][1:] - first))[seq] + row - first[seq]
    return seq, position.long(), (row - first[seq]).long()


def _plain_rotary(s):
    c, x = s["case"], s["x"].detach()
    angle = s["positions"].double().unsqueeze(-1) * s["inv_freq"]
    m = _magnitude(c["scaling"])
    y = _rotate(x, angle, c["interleaved"], m, 1.0)
    return (y, _rotate(s["gy"], angle, c["interleaved"], m, -1.0)) if c["train"] else (y,)


def _plain_append(s):
    c, n, p = s["case"], s["rows"], s["case"]["page_tokens"]
    seq, position, _ = _places(s)
    k, v, q = s["k"][:n], s["v"][:n], s["q"][:n]
    if c["rotate"]:
        angle = position.double().unsqueeze(-1) * s["inv_freq"]
        m = _magnitude(c["scaling"])
        k, q = _rotate(k, angle, c["interleaved"], m, 1.0), _rotate(q, angle, c["interleaved"], m, 1.0)
        s["out"][:n] = q
    page = s["table"][seq, position // p].long()
    s["pool"][page, 0, :, position % p] = k
    s["pool"][page, 1, :, position % p] = v
    return (s["pool"], s["out"]) if c["rotate"] else (s["pool"],)


def _plain_attention(s):
    c, n = s["case"], s["rows"]
    b, hk, d, p = c["seqs"], c["kv_heads"], c["dim"], c["page_tokens"]
    group = c["q_heads"] // hk
    used = s["table"][:, :-(-s["lens_host"] // p)].long()
    kv = s["pool"][used].permute(2, 0, 3, 1, 4, 5).reshape(2, b, hk, -1, d).float()  # [2, seqs, kv heads, tokens, dim]
    new = s["starts"][1:] - s["starts"][:-1]
    step = torch.arange(s["new"], device="cuda")
    rows = (s["starts"][:-1, None] + step).clamp(max=n - 1).long()
    q = s["q"][rows].float().reshape(b, -1, hk, group, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    scores = torch.matmul(q, kv[0].transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(b, hk, -1, group, kv.shape[3])
    key = torch.arange(kv.shape[3], device="cuda")
    position = ((s["lens"] - new)[:, None] + step)[:, :, None]
    seen = (key < s["lens"][:, None, None]).expand(b, s["new"], -1)
    if c["causal"]:
        seen = seen & (key <= position)
    if c["window"]:
        seen = seen & (key > position - c["window"])
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    weight = scores.sub_(most).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(b, hk, -1, kv.shape[3]), kv[1]).view(b, hk, -1, group, d)
    out = torch.where(total > 0, out / total, 0.0)
    seq, _, at = _places(s)
    s["out"][:n] = out[seq, :, at].reshape(n, -1, d).to(s["out"].dtype)
    if not c["lse"]:
        return (s["out"],)
    lse = (most + total.log()).squeeze(-1)
    return s["out"], lse[seq, :, at].reshape(n, -1)


# ---- the framework's calls -------------------------------------------------------------------------------

def _own(s):
    from mpcomm import ops

    c = s["case"]
    if c["op"] == "rotary":
        y = ops.rotary(s["x"], s["positions"], s["inv_freq"], interleaved=c["interleaved"], magnitude=_magnitude(c["scaling"]))
        return (y.detach(), *torch.autograd.grad(y, s["x"], s["gy"])) if c["train"] else (y,)
    batch = (s["pool"], s["table"], s["lens"], s["starts"])
    if c["op"] == "append":
        if not c["rotate"]:
            return (ops.paged_append(s["k"], s["v"], *batch),)
        return ops.paged_append(s["k"], s["v"], *batch, inv_freq=s["inv_freq"], interleaved=c["interleaved"],
                                magnitude=_magnitude(c["scaling"]), q=s["q"], q_out=s["out"])
    got = ops.paged_attention(s["q"], *batch, causal=c["causal"], window=c["window"], out=s["out"], return_lse=c["lse"])
    return (got[0], got[1][:s["rows"]]) if c["lse"] else (got,)


def run(state):
    if own:
        return _own(state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention}[state["case"]["op"]](state)


# ---- what a pass has to move and compute -------------------------------------------------------------------

def _seen_keys(case, new, length):
    """(keys that some new token sees, pairs of a new token and a key that it sees) of one sequence."""
    if not new:
        return 0, 0
    if not case["causal"]:
        return length, new * length
    window = case["window"] or length
    first, last = length - new + 1, length  # keys up to and with the token itself
    pairs = sum(min(n, window) for n in range(first, last + 1))
    return last - max(0, first - window), pairs


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotary":
        n = case["batch"] * case["tokens"]
        both = 2 if case["train"] else 1
        turned = n * case["heads"] * case["part"]
        return {"bytes": both * 2 * n * case["heads"] * case["dim"] * size + n * 8 + case["part"] * 4, "flops": both * 3 * turned}
    new, lens = _lengths(case)
    rows, hq, hk, d = sum(new), case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        heads = 2 * hk + (hq if case["rotate"] else 0)
        return {"bytes": 2 * rows * heads * d * size + rows * 4, "flops": 3 * rows * (hq + hk) * case["part"] if case["rotate"] else 0}
    keys, pairs = (sum(x) for x in zip(*(_seen_keys(case, n, m) for n, m in zip(new, lens))))
    pages = sum(-(-m // case["page_tokens"]) for m in lens)
    return {"bytes": 2 * rows * hq * d * size + 2 * keys * hk * d * size + 4 * pages + (4 * rows * hq if case["lse"] else 0),
            "flops": 4 * pairs * hq * d}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------

def _turn(x, position, freq, interleaved, magnitude, inverse=False):
    """Each pair of x [tokens, heads, dim], as a complex number, times magnitude * exp(i * position * frequency)."""
    x = x.double().clone()
    n = freq.numel()
    turn = torch.polar(torch.full((), float(magnitude), dtype=torch.float64, device=x.device).expand(position.numel(), n),
                       position.double().reshape(-1, 1) * freq)[:, None]
    if inverse:
        turn = turn.conj()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        m, shape = _magnitude(case["scaling"]), s["x"].shape
        args = (s["positions"], s["inv_freq"], case["interleaved"], m)
        y = _turn(s["x"].detach().flatten(0, 1), *args).view(shape)
        return (y, _turn(s["gy"].flatten(0, 1), *args, inverse=True).view(shape)) if case["train"] else (y,)
    new, lens = _lengths(case)
    p, hk, d = case["page_tokens"], case["kv_heads"], case["dim"]
    out, lse, row = s["out"].double(), [], 0
    pool = s["pool"].double() if case["op"] == "append" else None
    for b, (n, length) in enumerate(zip(new, lens)):
        position = torch.arange(length - n, length, device="cuda")
        here = slice(row, row + n)
        row += n
        if n == 0:
            continue
        if case["op"] == "append":
            k = s["k"][here].double()
            if case["rotate"]:
                how = (position, s["inv_freq"], case["interleaved"], _magnitude(case["scaling"]))
                k, out[here] = _turn(s["k"][here], *how), _turn(s["q"][here], *how)
            page, slot = s["table"][b][position // p].long(), position % p
            pool[page, 0, :, slot], pool[page, 1, :, slot] = k, s["v"][here].double()
            continue
        pages = s["table"][b, :-(-length // p)].long()
        key = torch.arange(length, device="cuda")
        hidden = torch.zeros((n, length), dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= key > position[:, None]
        if case["window"]:
            hidden |= key <= position[:, None] - case["window"]
        group, sums = case["q_heads"] // hk, []
        for h in range(hk):
            kv = s["pool"][pages, :, h].double().transpose(0, 1).reshape(2, -1, d)[:, :length]
            q = s["q"][here, h * group:(h + 1) * group].double()
            t = torch.einsum("ngd,ld->gnl", q, kv[0]).div_(math.sqrt(d)).masked_fill_(hidden, -math.inf)
            sums.append(torch.logsumexp(t, -1))  # [group, n]
            t = torch.softmax(t, -1)
            out[here, h * group:(h + 1) * group] = torch.einsum("gnl,ld->ngd", t, kv[1])
        lse.append(torch.cat(sums).transpose(0, 1))
    if case["op"] == "append":
        return (pool, out) if case["rotate"] else (pool,)
    return (out, torch.cat(lse)) if case["lse"] else (out,)
