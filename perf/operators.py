"""Linear attention with a decay per head, and group norm with an activation, as measurable cases.

`listed()` are fixed cases, `draw()` gives others of the same ranges; a case is a dict of plain values whose "kind" says
which public entry point it calls:

  step    lact_b200.layer_ops.linear_attention_step   one new token of every sequence, recurrent form
  prompt  lact_b200.layer_ops.linear_attention        chunked form, forward
  train   the same, forward and the gradients of q, k, v (and of the initial state)
  norm    lact_b200.layer_ops.group_norm              channels last, forward (and gradients, with train)

With `own` false, `run` is the same mathematics in elementary operations in 32 bits; `exact()` is the definition in 64.

  S_t = exp(g_h) S_(t-1) + k_t v_t^T,   o_t = scale q_t^T S_t                       (per head, S in dk x dv)
  y = act((x - mean) / sqrt(var + eps) * weight + bias), mean and var over a sample's tokens and a group's channels

Inputs: q, k, v ~ N(0, 1) in bf16, g_h between -0.7 and -0.001, spread over its logarithm (a horizon of 1.4 to 1000
tokens), states ~ N(0, 1) in fp32, scale dk^-0.5; x ~ N(m, s) with m and s of its own for every channel.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": BF16, "f32": F32}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # generation for one user: a token of one sequence, where launch latency counts
        dict(name="decode_one", kind="step", batch=1, heads=12, kv_heads=12, dk=128, dv=128),
        # generation for many users at once: every sequence's state is read and written
        dict(name="decode_batch", kind="step", batch=192, heads=12, kv_heads=12, dk=128, dv=128),
        # one short question: a prompt of a length no tile divides, few heads
        dict(name="prompt_short", kind="prompt", batch=1, tokens=203, heads=8, kv_heads=8, dk=64, dv=64, sequences=0,
             state_in=False, state_out=True),
        # prefill of one long document at a language model's usual length; the state goes on to generation
        dict(name="prompt_long", kind="prompt", batch=1, tokens=32768, heads=12, kv_heads=12, dk=128, dv=128, sequences=0,
             state_in=False, state_out=True),
        # prefill of several users' prompts packed back to back, shared key / value heads, each with its state so far
        dict(name="prompt_packed", kind="prompt", batch=1, tokens=20011, heads=16, kv_heads=4, dk=64, dv=128, sequences=9,
             state_in=True, state_out=True),
        # a layer's training step at a language model's usual length
        dict(name="linear_train", kind="train", batch=2, tokens=32768, heads=12, kv_heads=12, dk=128, dv=128, sequences=0,
             state_in=False, state_out=False),
        # training on packed documents, shared key / value heads
        dict(name="linear_train_packed", kind="train", batch=1, tokens=7003, heads=12, kv_heads=4, dk=64, dv=64, sequences=5,
             state_in=False, state_out=False),
        # the norm of every head of every token behind the attention of a generation step
        dict(name="norm_few_tokens", kind="norm", samples=24, spots=1, channels=1536, groups=12, dtype="bf16", silu=True, train=False),
        # ... and of a training step
        dict(name="norm_tokens_train", kind="norm", samples=65536, spots=1, channels=1536, groups=12, dtype="bf16", silu=True, train=True),
        # a picture encoder's block in training: 8 maps of 64 x 64, 512 channels in 32 groups
        dict(name="norm_maps_train", kind="norm", samples=8, spots=4096, channels=512, groups=32, dtype="bf16", silu=True, train=True),
        # a video decoder's last block: two frames of 480 x 832, three channels to a group
        dict(name="norm_frames", kind="norm", samples=2, spots=399360, channels=96, groups=32, dtype="bf16", silu=True, train=False),
        # the same kind of block in full precision, an odd number of spots
        dict(name="norm_f32_train", kind="norm", samples=4, spots=6235, channels=384, groups=24, dtype="f32", silu=False, train=True),
    ]


MOST = 2 * 32768 * 12 * 128   # elements of the largest listed inputs


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _linear_heads(rng):
    kv = rng.choice((1, 2, 3, 4, 6, 8, 12, 16))
    return kv * rng.choice((1, 1, 1, 2, 3, 4)), kv, rng.choice((64, 128, 128)), rng.choice((64, 128, 128))


def draw(rng):
    kind = rng.choice(("step", "prompt", "prompt", "train", "train", "norm", "norm", "norm"))
    if kind == "norm":
        groups = rng.choice((1, 4, 8, 12, 16, 24, 32))
        channels = groups * rng.choice((1, 3, 4, 5, 8, 16, 20, 24, 40, 64, 128))
        samples, spots = (_log(rng, 1, 65536), 1) if rng.random() < 0.4 else (rng.choice((1, 2, 3, 4, 8, 16)), _log(rng, 2, 400000))
        while samples * spots * channels > MOST * 3 // 4:
            if spots > 1:
                spots = max(1, spots // 2)
            else:
                samples = max(1, samples // 2)
        return dict(kind=kind, samples=samples, spots=spots, channels=channels, groups=groups,
                    dtype=rng.choice(("bf16", "bf16", "f32")), silu=rng.random() < 0.6, train=rng.random() < 0.5)
    heads, kv, dk, dv = _linear_heads(rng)
    if kind == "step":
        most = max(1, 40000000 // (heads * dk * dv))
        return dict(kind=kind, batch=_log(rng, 1, min(512, most)), heads=heads, kv_heads=kv, dk=dk, dv=dv)
    sequences = rng.choice((0, 0, 1, 3, 8, 17))
    batch = 1 if sequences else rng.choice((1, 1, 2, 3, 8))
    most = min(32768, MOST // (batch * heads * max(dk, dv)))
    tokens = _log(rng, 1, most)
    if rng.random() < 0.3 and tokens >= 128:
        tokens -= tokens % 128
    train = kind == "train"
    return dict(kind=kind, batch=batch, tokens=tokens, heads=heads, kv_heads=kv, dk=dk, dv=dv, sequences=sequences,
                state_in=rng.random() < 0.4, state_out=rng.random() < (0.3 if train else 0.7))


def _lengths(c):
    """Lengths of a packed batch's sequences: uneven, and the second of more than two is empty."""
    n, total = c["sequences"], c["tokens"]
    share = [0.0 if i == 1 and n > 2 else 1.0 + (7 * i + 3) % 5 for i in range(n)]
    ends, at = [], 0.0
    for x in share:
        at += x
        ends.append(int(round(total * at / sum(share))))
    return [e - b for b, e in zip([0] + ends, ends)]


# ---------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    if c["kind"] == "norm":
        dt, C = TYPES[c["dtype"]], c["channels"]
        shape = (c["samples"], c["spots"], C) if c["spots"] > 1 else (c["samples"], C)
        x = randn(*shape).mul_(0.5 + randn(C).abs_()).add_(randn(C)).to(dt)
        s = dict(case=c, x=x, weight=1.0 + 0.2 * randn(C), bias=0.2 * randn(C))
        if c["train"]:
            s["dy"] = randn(*shape).to(dt)
            for n in ("x", "weight", "bias"):
                s[n].requires_grad_()
        return s
    b, h, hk, dk, dv = c["batch"], c["heads"], c["kv_heads"], c["dk"], c["dv"]
    spread = torch.rand(h, device="cuda", generator=gen)
    s = dict(case=c, log_decay=-(0.7 * torch.exp(spread * math.log(0.001 / 0.7))))
    if c["kind"] == "step":
        s.update(q=randn(b, h, dk).to(BF16), k=randn(b, hk, dk).to(BF16), v=randn(b, hk, dv).to(BF16),
                 state=randn(b, h, dk, dv), new=torch.empty(b, h, dk, dv, device="cuda"))
        return s
    l, n = c["tokens"], c["sequences"] or b
    s.update(q=randn(b, l, h, dk).to(BF16), k=randn(b, l, hk, dk).to(BF16), v=randn(b, l, hk, dv).to(BF16),
             state=randn(n, h, dk, dv) if c["state_in"] else None, cu=None)
    if c["sequences"]:
        s["cu"] = torch.tensor([0] + _lengths(c), dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    if c["kind"] == "train":
        s["do"] = randn(b, l, h, dv).to(BF16)
        s["dstate"] = randn(n, h, dk, dv) if c["state_out"] else None
        for name in ("q", "k", "v", "state"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


# ---------------------------------------------------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    if c["kind"] == "step":
        if own:
            from lact_b200 import layer_ops as lo
            return lo.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], new_state=s["new"]), s["new"]
        return _plain_step(s)
    if c["kind"] == "norm":
        act = "silu" if c["silu"] else None
        if own:
            from lact_b200 import layer_ops as lo
            y = lo.group_norm(s["x"], c["groups"], s["weight"], s["bias"], EPS, activation=act)
        else:
            y = _plain_norm(s)
        if not c["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"]))
    if own:
        from lact_b200 import layer_ops as lo
        o, last = lo.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], initial_state=s["state"],
                                      output_final_state=c["state_out"], cu_seqlens=s["cu"])
    else:
        o, last = _plain_linear(s)
    outs = [o] + ([last] if c["state_out"] else [])
    if c["kind"] == "prompt":
        return outs
    leaves = [s[n] for n in ("q", "k", "v", "state") if s[n] is not None]
    grads = torch.autograd.grad(outs, leaves, [s["do"]] + ([s["dstate"]] if c["state_out"] else []))
    return [t.detach() for t in outs] + list(grads)


def _heads(x, h):
    """Shared heads (axis -2) repeated, in 32 bits."""
    return x.float().repeat_interleave(h // x.shape[-2], dim=-2)


def _plain_step(s):
    h, scale = s["q"].shape[1], s["q"].shape[2] ** -0.5
    q, k, v = s["q"].float(), _heads(s["k"], h), _heads(s["v"], h)
    new = s["state"] * torch.exp(s["log_decay"])[:, None, None] + k[..., :, None] * v[..., None, :]
    return (scale * (q[..., None, :] @ new)[..., 0, :]).to(s["q"].dtype), new


def _plain_linear(s):
    """Chunks of 128 tokens, one after the other; sequences of a packed batch likewise."""
    c, g = s["case"], s["log_decay"]
    h, dk, dv = c["heads"], c["dk"], c["dv"]
    q, k, v = (x.transpose(1, 2) for x in (s["q"].float() * dk ** -0.5, _heads(s["k"], h), _heads(s["v"], h)))  # [b, h, l, d]
    lengths = _lengths(c) if c["sequences"] else [c["tokens"]]
    outs, states, at = [], [], 0
    for n, length in enumerate(lengths):
        S = q.new_zeros(q.shape[0], h, dk, dv)
        if s["state"] is not None:
            S = s["state"][n:n + 1] if c["sequences"] else s["state"]
        for begin in range(at, at + length, 128):
            end = min(begin + 128, at + length)
            qc, kc, vc = q[:, :, begin:end], k[:, :, begin:end], v[:, :, begin:end]
            i = torch.arange(end - begin, device=q.device)
            gap = i[:, None] - i[None, :]
            D = torch.exp(g[:, None, None] * gap.clamp(min=0)) * (gap >= 0)
            since = torch.exp(g[:, None] * (i + 1))[..., None]
            left = torch.exp(g[:, None] * (len(i) - 1 - i))[..., None]
            outs.append(((qc @ kc.transpose(-1, -2)) * D) @ vc + since * (qc @ S))
            S = torch.exp(g * len(i))[:, None, None] * S + (kc * left).transpose(-1, -2) @ vc
        states.append(S)
        at += length
    return torch.cat(outs, dim=2).transpose(1, 2).contiguous().to(BF16), torch.cat(states)


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float().reshape(c["samples"], c["spots"], c["groups"], -1)
    centred = x - x.mean(dim=(1, 3), keepdim=True)
    xhat = centred * torch.rsqrt((centred * centred).mean(dim=(1, 3), keepdim=True) + EPS)
    y = xhat.reshape(s["x"].shape) * s["weight"] + s["bias"]
    if c["silu"]:
        y = y * torch.sigmoid(y)
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------------------------------------------------- 64 bits
@torch.no_grad()
def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "norm":
        return _exact_norm(s)
    h = c["heads"]
    lam = torch.exp(s["log_decay"].double())
    q, k, v = (s[n].double() for n in "qkv")
    share = h // c["kv_heads"]
    if c["kind"] == "step":
        kh, vh = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
        new = s["state"].double() * lam[:, None, None] + torch.einsum("bhk,bhv->bhkv", kh, vh)
        return torch.einsum("bhk,bhkv->bhv", q, new) * c["dk"] ** -0.5, new
    # token by token: rows are (batch, head), states [rows, dk, dv]
    b, l, dk, dv = c["batch"], c["tokens"], c["dk"], c["dv"]
    rows = lambda x: x.repeat_interleave(h // x.shape[2], 2).permute(1, 0, 2, 3).reshape(l, b * h, x.shape[3])
    q, k, v = rows(q) * dk ** -0.5, rows(k), rows(v)
    lam = lam.repeat(b)[:, None, None]
    n_seq = c["sequences"] or 1
    spans, at = [], 0
    for length in (_lengths(c) if c["sequences"] else [l]):
        spans.append((at, at + length))
        at += length
    start = lambda t, n: (torch.zeros(b * h, dk, dv, dtype=F64, device="cuda") if t is None else
                          t.double().reshape(n_seq, -1, dk, dv)[n].clone())
    train = c["kind"] == "train"
    o, dq = torch.empty_like(v), torch.empty_like(q)
    do = rows(s["do"].double()) if train else None
    last, dfirst = [], []
    for n, (t0, t1) in enumerate(spans):
        S = start(s["state"], n)
        for t in range(t0, t1):
            S.mul_(lam).baddbmm_(k[t][:, :, None], v[t][:, None, :])
            torch.bmm(q[t][:, None, :], S, out=o[t][:, None, :])
            if train:
                torch.bmm(S, do[t][:, :, None], out=dq[t][:, :, None])
        last.append(S)
    back = lambda x: x.reshape(l, b, h, -1).permute(1, 0, 2, 3)
    outs = [back(o)] + ([torch.cat(last).reshape(-1, h, dk, dv)] if c["state_out"] else [])
    if not train:
        return outs
    dk_, dv_ = torch.empty_like(k), torch.empty_like(v)
    for n, (t0, t1) in enumerate(spans):
        R = start(s["dstate"], n)   # gradient of the state behind token t
        for t in range(t1 - 1, t0 - 1, -1):
            R.baddbmm_(q[t][:, :, None], do[t][:, None, :])
            torch.bmm(R, v[t][:, :, None], out=dk_[t][:, :, None])
            torch.bmm(k[t][:, None, :], R, out=dv_[t][:, None, :])
            R.mul_(lam)
        dfirst.append(R)
    shared = lambda x: back(x).reshape(b, l, c["kv_heads"], share, -1).sum(3)
    outs += [back(dq) * dk ** -0.5, shared(dk_), shared(dv_)]
    return outs + ([torch.cat(dfirst).reshape(-1, h, dk, dv)] if c["state_in"] else [])


def _exact_norm(s):
    c = s["case"]
    n, G, C = c["samples"], c["groups"], c["channels"]
    x = s["x"].double().reshape(n, c["spots"], G, C // G)
    var, mean = torch.var_mean(x, dim=(1, 3), keepdim=True, correction=0)
    inv = 1.0 / torch.sqrt(var + EPS)
    xhat = (x - mean) * inv
    w, bias = s["weight"].double().reshape(G, C // G), s["bias"].double().reshape(G, C // G)
    z = xhat * w + bias
    gate = 1.0 / (1.0 + torch.exp(-z))
    y = z * gate if c["silu"] else z
    if not c["train"]:
        return y.reshape(s["x"].shape)
    dz = s["dy"].double().reshape(z.shape)
    if c["silu"]:
        dz = dz * (gate * (1.0 + z * (1.0 - gate)))
    dw, db = (dz * xhat).sum((0, 1)).reshape(C), dz.sum((0, 1)).reshape(C)
    t = dz * w
    dx = inv * (t - t.mean((1, 3), keepdim=True) - xhat * (t * xhat).mean((1, 3), keepdim=True))
    return y.reshape(s["x"].shape), dx.reshape(s["x"].shape), dw, db


# ---------------------------------------------------------------------------------------------------------- least work
def work(case):
    c = case
    if c["kind"] == "norm":
        e, size = c["samples"] * c["spots"] * c["channels"], TYPES[c["dtype"]].itemsize
        passes = 5 if c["train"] else 2      # x, y; then x, dy, dx
        return {"bytes": passes * e * size, "flops": (30 if c["train"] else 10) * e}
    h, hk, dk, dv = c["heads"], c["kv_heads"], c["dk"], c["dv"]
    if c["kind"] == "step":
        rows = c["batch"] * h
        return {"bytes": 8 * rows * dk * dv + 2 * c["batch"] * (h * (dk + dv) + hk * (dk + dv)), "flops": 5 * rows * dk * dv}
    tokens, n = c["batch"] * c["tokens"], c["sequences"] or c["batch"]
    states = 4 * n * h * dk * dv * (int(c["state_in"]) + int(c["state_out"]))
    inputs, out = 2 * tokens * (h * dk + hk * (dk + dv)), 2 * tokens * h * dv
    least = 4 * tokens * h * dk * dv         # the state's update and its product with a row, token by token
    if c["kind"] == "prompt":
        return {"bytes": inputs + out + states, "flops": least}
    return {"bytes": (inputs + out + states) + (2 * inputs + out + states), "flops": least * 7 // 2}
