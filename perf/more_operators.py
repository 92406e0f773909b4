"""Rotary positions with several axes, a paged cache of keys and values, and the attention of single tokens over it, as measurable cases.

`listed()` are fixed cases, `draw()` gives others of the same ranges; a case is a dict of plain values whose "kind" says
which public entry points it calls:

  rotary    lact_b200.layer_ops.rotary_axes            queries and keys by their positions, forward (and gradients, with train)
  write     lact_b200.layer_ops.paged_cache_write      new keys and values into a cache of bf16
  store     paged_cache_write, paged_cache_read        ... into a cache of 8 bits, and back as the values that these stand for
  read      lact_b200.layer_ops.paged_cache_read       the last tokens of every sequence out of the cache
  step      lact_b200.layer_ops.paged_attention_step   attention of one new token of every sequence over its pages
  generate  rotary_axes, paged_cache_write, paged_attention_step   a layer's attention in one step of generation

With `own` false, `run` is the same mathematics in elementary operations in 32 bits (angles in 64); `exact()` is the definition in 64.

  pair j of axis a:  (x, y) -> (x cos t - y sin t, y cos t + x sin t),  t = positions[.., a] frequencies[j]
  row j of n_i of sequence i has position lengths[i] - n_i + j; it lies in page page_table[i, position // page_size]
  8 bits: a power of two 2^(b - 127) for every row of a head, the smallest with max |x| / 2^(b - 127) <= 448; x / 2^(b - 127) in e4m3
  o = softmax(d^-0.5 q K^T) V over the last `window` of a sequence's `length` tokens

Inputs: q, k, v ~ N(0, 1) in bf16, keys with a scale of its own for every channel (0.5 to 2); pages in a random order.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
TYPES = {"bf16": BF16, "f32": F32}


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the new tokens of a few dozen users, before their keys go to the cache: launch latency
        dict(name="rotary_tokens", kind="rotary", batch=32, tokens=0, heads=12, kv_heads=12, dim=128, sections="64", halves=True,
             dtype="bf16", train=False),
        # a language model's layer in training at its usual length
        dict(name="rotary_text_train", kind="rotary", batch=2, tokens=32768, heads=12, kv_heads=12, dim=128, sections="64", halves=True,
             dtype="bf16", train=True),
        # a video layer in training: 21 frames of 1560 tokens, time, height and width
        dict(name="rotary_video_train", kind="rotary", batch=1, tokens=32760, heads=12, kv_heads=12, dim=128, sections="22,21,21",
             halves=False, dtype="bf16", train=True),
        # an image encoder in full precision, odd rows of patches, a part of every head turned
        dict(name="rotary_image_f32", kind="rotary", batch=3, tokens=4081, heads=6, kv_heads=2, dim=64, sections="11,13", halves=False,
             dtype="f32", train=False),
        # prefill of several users' prompts packed back to back: their keys and values into the pages
        dict(name="write_prompts", kind="write", batch=9, tokens=20011, heads=8, kv_heads=8, dim=128, page=64, packed=True, bits=16),
        # frames of a video kept in 8 bits for those that follow, and read back for them
        dict(name="store_frames", kind="store", batch=2, tokens=14040, heads=12, kv_heads=12, dim=128, page=128, packed=False, bits=8),
        # windows of several users' caches read back for the next pieces of their prompts
        dict(name="read_windows", kind="read", batch=24, tokens=2048, heads=4, kv_heads=4, dim=128, page=16, packed=False, bits=8),
        # generation for one user after a short question: launch latency
        dict(name="step_one", kind="step", batch=1, tokens=777, heads=12, kv_heads=12, dim=128, page=64, window=0, bits=16),
        # generation for a few users over very long documents, shared key / value heads
        dict(name="step_long", kind="step", batch=4, tokens=131072, heads=16, kv_heads=4, dim=128, page=64, window=0, bits=16),
        # generation for many users, each with a length of its own, a cache of 8 bits, shared heads
        dict(name="step_many", kind="step", batch=64, tokens=16384, heads=32, kv_heads=8, dim=128, page=32, window=0, bits=8),
        # generation in a layer with a sliding window
        dict(name="step_window", kind="step", batch=192, tokens=5000, heads=12, kv_heads=12, dim=64, page=16, window=2048, bits=16),
        # a layer's attention in one step of generation for a few dozen users: turn, write, attend
        dict(name="generate", kind="generate", batch=48, tokens=4099, heads=12, kv_heads=4, dim=128, page=64, window=0, bits=16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    kind = rng.choice(("rotary", "rotary", "write", "store", "read", "step", "step", "step", "generate"))
    kv = rng.choice((1, 2, 3, 4, 6, 8, 12))
    c = dict(kind=kind, batch=1, tokens=1, heads=kv * rng.choice((1, 1, 2, 3, 4, 8)), kv_heads=kv, dim=rng.choice((64, 128, 128)))
    if kind == "rotary":
        axes = rng.choice((1, 1, 2, 3))
        pairs = c["dim"] // 2 if rng.random() < 0.7 else 8 * rng.randint(1, c["dim"] // 16)
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        c.update(sections=",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs])), halves=rng.random() < 0.5,
                 dtype=rng.choice(("bf16", "bf16", "f32")), train=rng.random() < 0.5)
        c["tokens"] = 0 if axes == 1 and rng.random() < 0.2 else _log(rng, 1, 40000)
        c["batch"] = _log(rng, 1, 512) if c["tokens"] == 0 else rng.choice((1, 1, 2, 3, 8))
    else:
        c.update(page=rng.choice((16, 32, 64, 128, 256)), bits={"write": 16, "store": 8, "generate": 16}.get(kind, rng.choice((8, 16))))
        if kind in ("write", "store", "read"):
            c["packed"] = rng.random() < 0.5
            c["batch"] = rng.choice((1, 2, 5, 9, 24))
            c["tokens"] = _log(rng, 1, 32768)
        else:
            c["batch"] = _log(rng, 1, 256)
            c["window"] = 0 if kind == "generate" or rng.random() < 0.6 else _log(rng, 1, 8192)
            c["tokens"] = _log(rng, 1, 131072)
    while work(c)["bytes"] > most or c["batch"] * c["tokens"] * c["kv_heads"] * c["dim"] > 300000000:
        c["tokens" if c["tokens"] > 64 else "batch"] //= 2
    return c


def _lengths(c):
    """How many tokens each sequence of a batch has: of a batch that generates, uneven; one that is not used in larger ones."""
    n, top = c["batch"], c["tokens"]
    if c["kind"] in ("step", "generate"):
        return [0 if n > 8 and i == 5 else max(1, top * (11 - (7 * i) % 11) // 11) for i in range(n)]
    if c["packed"]:   # `tokens` rows in all; earlier tokens in front of them
        return [rows + (13 * i) % 29 for i, rows in enumerate(_rows(c))]
    # `tokens` rows of each entry; some sequences are shorter (their first rows pad the batch), others have earlier tokens
    return [max(1, top - 7) if i % 3 == 1 else top + (13 * i) % 29 for i in range(n)]


def _rows(c):
    """Rows of each sequence in a packed batch of `tokens` rows; the second of more than two has none."""
    n = c["batch"]
    share = [0 if i == 1 and n > 2 else 1 + (7 * i + 3) % 5 for i in range(n)]
    ends = [c["tokens"] * sum(share[:i + 1]) // sum(share) for i in range(n)]
    return [e - b for b, e in zip([0] + ends, ends)]


def _sections(c):
    return [int(x) for x in c["sections"].split(",")]


# ---------------------------------------------------------------------------------------------------------- inputs
def _rows_8bit(x):
    """Rows (last axis) in 8 bits: e4m3 values and the byte of their power of two."""
    top = x.float().abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    byte = (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-126) + 127
    return torch.ldexp(x.float(), 127 - byte).to(E4M3), byte[..., 0].to(torch.uint8)


def _frequencies(sections, base=10000.0):
    return torch.cat([base ** (-torch.arange(n, dtype=F64) / n) for n in sections]).cuda()


def _grid(c, axes):
    """Positions of the tokens: one after the other; rows and columns; frames, rows and columns."""
    i = torch.arange(c["tokens"])
    if axes == 1:
        return i[:, None].int().cuda()
    if axes == 2:
        return torch.stack([i // 77, i % 77], 1).int().cuda()
    return torch.stack([i // 1560, i % 1560 // 52, i % 52], 1).int().cuda()


def _cache(c, gen, seqs, lengths):
    """Pages in a random order, with random keys and values of all their rows."""
    pages_of = [-(-n // c["page"]) for n in lengths]
    n = max(1, sum(pages_of) + 3)
    order = torch.randperm(n, generator=gen, device="cuda").int()
    wide = max(1, max(pages_of))
    starts = torch.tensor([sum(pages_of[:i]) for i in range(seqs)], device="cuda")
    at = torch.arange(wide, device="cuda")
    table = torch.where(at < torch.tensor(pages_of, device="cuda")[:, None], order[(starts[:, None] + at).clamp(max=n - 1)], -1).int()
    shape, bits = (n, c["kv_heads"], c["page"], c["dim"]), c["bits"]
    spread = torch.rand(c["kv_heads"], 1, c["dim"], device="cuda", generator=gen) * 1.5 + 0.5
    s = dict(table=table, lengths=torch.tensor(lengths, dtype=torch.int32).cuda())
    step = max(1, (1 << 26) // (c["kv_heads"] * c["page"] * c["dim"]))
    for name in "kv":
        data = torch.empty(shape, dtype=BF16 if bits == 16 else E4M3, device="cuda")
        byte = None if bits == 16 else torch.empty(shape[:3], dtype=torch.uint8, device="cuda")
        for b in range(0, n, step):
            x = torch.randn((min(step, n - b), *shape[1:]), device="cuda", generator=gen)
            x = (x * spread if name == "k" else x).to(BF16)
            if bits == 16:
                data[b:b + step] = x
            else:
                data[b:b + step], byte[b:b + step] = _rows_8bit(x)
        s["c" + name], s["b" + name] = data, byte
    return s


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    b, h, hk, d, kind = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["kind"]
    if kind == "rotary":
        dt, sec = TYPES[c["dtype"]], _sections(c)
        s = dict(case=c, freq=_frequencies(sec), sections=sec)
        if c["tokens"] == 0:
            s.update(q=randn(b, h, d).to(dt), k=randn(b, hk, d).to(dt),
                     pos=torch.randint(0, 131072, (b, 1), device="cuda", generator=gen).int())
        else:
            s.update(q=randn(b, c["tokens"], h, d).to(dt), k=randn(b, c["tokens"], hk, d).to(dt), pos=_grid(c, len(sec)))
        if c["train"]:
            s.update(dq=randn(*s["q"].shape).to(dt), dk=randn(*s["k"].shape).to(dt))
            s["q"].requires_grad_(), s["k"].requires_grad_()
        return s
    lengths = _lengths(c)
    s = dict(case=c, **_cache(c, gen, b, lengths))
    if kind in ("step", "generate"):
        s["q"] = randn(b, h, d).to(BF16)
        if kind == "generate":
            s.update(k=randn(b, hk, d).to(BF16), v=randn(b, hk, d).to(BF16), freq=_frequencies([d // 2]), sections=[d // 2],
                     pos=(s["lengths"] - 1).clamp(min=0)[:, None])
        return s
    s["cu"] = None
    if c["packed"]:
        s["cu"] = torch.tensor([0] + _rows(c), dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    if kind != "read":   # keys and values as they leave a fused projection
        kv = randn(*((1, c["tokens"]) if c["packed"] else (b, c["tokens"])), 2 * hk, d).to(BF16)
        s.update(k=kv[:, :, :hk], v=kv[:, :, hk:])
    return s


# ---------------------------------------------------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "rotary":
        if own:
            from lact_b200 import layer_ops as lo
            q, k = lo.rotary_axes(s["q"], s["k"], s["pos"], s["freq"], s["sections"], interleaved=not c["halves"])
        else:
            cos, sin = _plain_angles(s)
            q, k = _plain_turn(s["q"], cos, sin, c["halves"]), _plain_turn(s["k"], cos, sin, c["halves"])
        if not c["train"]:
            return q, k
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    if own:
        from lact_b200 import layer_ops as lo
        cache = lo.PagedCache(s["ck"], s["cv"], s["bk"], s["bv"])
        if kind == "write":
            lo.paged_cache_write(cache, s["k"], s["v"], s["table"], s["lengths"], cu_seqlens=s["cu"])
            return s["ck"], s["cv"]
        if kind == "store":
            lo.paged_cache_write(cache, s["k"], s["v"], s["table"], s["lengths"], cu_seqlens=s["cu"])
        if kind in ("store", "read"):
            return lo.paged_cache_read(cache, s["table"], s["lengths"], c["tokens"], cu_seqlens=s["cu"])
        if kind == "step":
            return lo.paged_attention_step(s["q"], cache, s["table"], s["lengths"], window_size=c["window"] or None)
        q, k = lo.rotary_axes(s["q"], s["k"], s["pos"], s["freq"], s["sections"])
        lo.paged_cache_write(cache, k[:, None], s["v"][:, None], s["table"], s["lengths"])
        return lo.paged_attention_step(q, cache, s["table"], s["lengths"]), s["ck"], s["cv"]
    if kind == "write":
        _plain_write(s, s["k"], s["v"])
        return s["ck"], s["cv"]
    if kind == "store":
        _plain_write(s, s["k"], s["v"])
    if kind in ("store", "read"):
        return _plain_read(s)
    if kind == "step":
        return _plain_step(s, s["q"])
    cos, sin = _plain_angles(s)
    _plain_write(s, _plain_turn(s["k"], cos, sin, True)[:, None], s["v"][:, None])
    return _plain_step(s, _plain_turn(s["q"], cos, sin, True)), s["ck"], s["cv"]


def _plain_angles(s):
    sec = torch.tensor(s["sections"], device="cuda")
    of_pair = torch.repeat_interleave(torch.arange(len(sec), device="cuda"), sec, output_size=s["freq"].numel())
    t = (s["pos"][..., of_pair].double() * s["freq"])[..., None, :]   # [.., 1 (heads), pairs]
    return torch.cos(t).float(), torch.sin(t).float()


def _plain_turn(x, cos, sin, halves):
    p = cos.shape[-1]
    f = x.float()
    a, b = (f[..., :p], f[..., p:2 * p]) if halves else (f[..., 0:2 * p:2], f[..., 1:2 * p:2])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([u, w], -1) if halves else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([turned, f[..., 2 * p:]], -1).to(x.dtype)


def _plain_places(s):
    """Page and row of every row of the batch, and which rows have one."""
    c = s["case"]
    n = 1 if c["kind"] == "generate" else c["tokens"]
    at = torch.arange(n, device="cuda")
    if s.get("cu") is not None:
        seq = torch.searchsorted(s["cu"], at, right=True, out_int32=True).long() - 1
        pos = s["lengths"][seq] - (s["cu"][seq + 1] - at)
    else:
        seq = torch.arange(c["batch"], device="cuda")[:, None].expand(-1, n).reshape(-1)
        pos = s["lengths"][seq] - n + at.repeat(c["batch"])
    there = pos >= 0
    pos = pos.clamp(min=0)
    return s["table"][seq, pos // c["page"]].long(), pos % c["page"], there


def _plain_write(s, k, v):
    page, row, there = _plain_places(s)
    page, row = page[there], row[there]
    for name, x in (("k", k), ("v", v)):
        x = x.reshape(-1, *x.shape[2:])[there]
        if s["case"]["bits"] == 16:
            s["c" + name][page, :, row] = x
        else:
            x, byte = _rows_8bit(x)
            s["c" + name].view(torch.uint8)[page, :, row] = x.view(torch.uint8)
            s["b" + name][page, :, row] = byte


def _plain_rows(s, name, page, row):
    """Rows of the cache, [.., heads, dim], in 32 bits."""
    if s["case"]["bits"] == 16:
        return s["c" + name][page, :, row].float()
    x = s["c" + name].view(torch.uint8)[page, :, row].view(E4M3).float()
    return torch.ldexp(x, s["b" + name][page, :, row].int()[..., None] - 127)


def _plain_read(s):
    c = s["case"]
    page, row, there = _plain_places(s)
    page = page.clamp(min=0)
    both = torch.stack([_plain_rows(s, n, page, row) for n in "kv"]) * there[:, None, None]
    return both.reshape(-1, c["tokens"], c["kv_heads"], c["dim"]).to(BF16)


def _plain_step(s, q):
    c = s["case"]
    b, h, d = q.shape
    hk = c["kv_heads"]
    first = (s["lengths"] - c["window"]).clamp(min=0) if c["window"] else torch.zeros_like(s["lengths"])
    span = min(c["tokens"], c["window"] or c["tokens"])
    pos = first[:, None] + torch.arange(span, device="cuda")
    seen = pos < s["lengths"][:, None]
    pos = torch.where(seen, pos, 0)
    page = s["table"].gather(1, (pos // c["page"]).long()).clamp(min=0).long()
    k = _plain_rows(s, "k", page, pos % c["page"])   # [b, span, hk, d]
    p = (q.float() * d ** -0.5).reshape(b, hk, h // hk, d) @ k.permute(0, 2, 3, 1)
    del k
    p = p.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-1e30))
    v = _plain_rows(s, "v", page, pos % c["page"])
    v = torch.where(seen[..., None, None], v, 0.0)
    o = p @ v.transpose(1, 2)
    return (o / p.sum(-1, keepdim=True).clamp(min=1e-30)).reshape(b, h, d).to(q.dtype)


# ---------------------------------------------------------------------------------------------------------- 64 bits
@torch.no_grad()
def exact(case, seed):
    s, c = prepare(case, seed), case
    kind = c["kind"]
    if kind == "rotary":
        outs = [_exact_turn(s, s[n], 1.0, c["halves"]) for n in "qk"]
        return outs + ([_exact_turn(s, s["d" + n], -1.0, c["halves"]) for n in "qk"] if c["train"] else [])
    if kind == "write":
        return [_exact_written(s, n, s[n]) for n in "kv"]
    if kind == "store":
        hold = {n: _exact_8bit(s[n].double()) for n in "kv"}
        return _exact_window(s, lambda n, i, j0, rows, t0: hold[n][i, j0 + rows])
    if kind == "read":
        return _exact_window(s, lambda n, i, j0, rows, t0: _exact_rows(s, n, t0, rows))
    if kind == "step":
        return _exact_step(s, s["q"].double(), None)
    q, k = (_exact_turn(s, s[n], 1.0, True) for n in "qk")
    s.update(k=k[:, None], v=s["v"][:, None].double(), cu=None)
    q, k = q.to(BF16).double(), k.to(BF16).double()   # the turned ones are handed on in the activations' type
    return [_exact_step(s, q, {"k": k, "v": s["v"][:, 0]})] + [_exact_written(s, n, s[n]) for n in "kv"]


def _exact_turn(s, x, sign, halves):
    x = x.detach().double()
    y, j = x.clone(), 0
    pairs = sum(s["sections"])
    for axis, n in enumerate(s["sections"]):
        for _ in range(n):
            t = s["pos"][..., axis].double()[..., None] * s["freq"][j]
            a, b = (j, j + pairs) if halves else (2 * j, 2 * j + 1)
            y[..., a] = x[..., a] * torch.cos(t) - sign * x[..., b] * torch.sin(t)
            y[..., b] = x[..., b] * torch.cos(t) + sign * x[..., a] * torch.sin(t)
            j += 1
    return y


def _exact_8bit(x):
    """What a row in 8 bits stands for: multiples of the spacing of 4-bit significands, at least 2^-9 of the row's power of two."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -140))) - 8
    e = torch.where(top > 448 * torch.exp2(e), e + 1, e).clamp(min=-126)
    u = x * torch.exp2(-e)
    space = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(u / space) * space * torch.exp2(e)   # (ties to even)


def _exact_spans(s):
    """(sequence, first row, rows, entry) of the batch."""
    c = s["case"]
    if s["cu"] is None:
        return [(i, 0, 1 if c["kind"] == "generate" else c["tokens"], i) for i in range(c["batch"])]
    rows = _rows(c)
    return [(i, sum(rows[:i]), n, 0) for i, n in enumerate(rows)]


def _exact_written(s, name, x):
    c, out = s["case"], s["c" + name].double()
    for i, j0, n, entry in _exact_spans(s):
        length = int(s["lengths"][i])
        pos = torch.arange(max(0, length - n), length, device="cuda")
        page = s["table"][i].long()[pos // c["page"]]
        out[page, :, pos % c["page"]] = x[entry, j0 + n - len(pos):j0 + n].double()
    return out


def _exact_rows(s, name, seq, pos):
    """Rows [positions, heads, dim] of one sequence in the cache."""
    c = s["case"]
    page = s["table"][seq].long()[pos // c["page"]]
    if c["bits"] == 16:
        return s["c" + name][page, :, pos % c["page"]].double()
    x = s["c" + name].view(torch.uint8)[page, :, pos % c["page"]].view(E4M3).double()
    return x * torch.exp2(s["b" + name][page, :, pos % c["page"]].double() - 127)[..., None]


def _exact_window(s, rows_of):
    c = s["case"]
    entries = 1 if s["cu"] is not None else c["batch"]
    out = torch.zeros(2, entries, c["tokens"], c["kv_heads"], c["dim"], dtype=F64, device="cuda")
    for i, j0, n, entry in _exact_spans(s):
        length = int(s["lengths"][i])
        m = min(n, length)
        for side, name in enumerate("kv"):
            if c["kind"] == "store":
                rows = rows_of(name, entry, j0, torch.arange(n - m, n, device="cuda"), i)
            else:
                rows = rows_of(name, entry, j0, torch.arange(length - m, length, device="cuda"), i)
            out[side, entry, j0 + n - m:j0 + n] = rows
    return out.reshape(2 * entries, c["tokens"], c["kv_heads"], c["dim"])


def _exact_step(s, q, last):
    c = s["case"]
    b, h, d = q.shape
    hk, out = c["kv_heads"], torch.zeros(b, h, d, dtype=F64, device="cuda")
    for i in range(b):
        length = int(s["lengths"][i])
        if length <= 0:
            continue
        pos = torch.arange(max(0, length - c["window"]) if c["window"] else 0, length, device="cuda")
        k, v = (_exact_rows(s, n, i, pos) for n in "kv")
        if last is not None:
            k[-1], v[-1] = last["k"][i], last["v"][i]
        x = torch.einsum("jgd,ljd->jgl", q[i].reshape(hk, -1, d), k) * d ** -0.5
        out[i] = torch.einsum("jgl,ljd->jgd", torch.softmax(x, -1), v).reshape(h, d)
    return out


# ---------------------------------------------------------------------------------------------------------- least work
def work(case):
    c = case
    b, h, hk, d, kind = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["kind"]
    if kind == "rotary":
        e = b * max(1, c["tokens"]) * (h + hk) * d
        passes = 4 if c["train"] else 2     # q, k and their turned ones; then the gradients of both
        return {"bytes": passes * e * TYPES[c["dtype"]].itemsize, "flops": passes // 2 * 3 * e}
    row = d * 2 if c["bits"] == 16 else d + 1
    if kind in ("write", "store", "read"):
        rows = (1 if c["packed"] else b) * c["tokens"] * hk * 2
        return {"bytes": rows * {"write": 4 * d, "store": 4 * d + 2 * row, "read": 2 * d + row}[kind], "flops": rows * d}
    seen = sum(min(n, c["window"] or n) for n in _lengths(c))
    step = {"bytes": 2 * seen * hk * row + 4 * b * h * d, "flops": 4 * seen * h * d}
    if kind == "generate":
        step["bytes"] += 4 * b * h * d + 4 * b * hk * d + 4 * b * hk * d + 4 * b * hk * d   # q, k turned; k, v to the cache
    return step
