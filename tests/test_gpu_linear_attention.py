"""Linear attention with a decay per head against the recurrence in 64 bits (oracle.linear_attention): outputs, states, gradients.

Tolerances.  Half a step of bf16 is 2^-8 of a value.  An output is a sum of terms (q_i . k_j) lambda^(i-j) v_j within a tile, whose
weights are rounded to bf16 once, and of q S with the incoming state rounded once; the sum is rounded once more at the end.  With A
the same operator on absolute values, |error| <= 2^-8 |o| + 2^-8 A + fp32 roundings (2^-24 for each of the at most few hundred
additions in a row, exponentials good to 2^-20: 2^-14 A covers them).  States are sums of k v^T with k scaled in two bf16 pieces, which
leave 2^-16, in fp32: |error| <= (2^-16 + 2^-20 * tiles + 2^-20) A.  Norm by norm the roundings have random signs: a relative error
of 2^-7 (one half step inside, one at the end, each at its worst) for outputs and gradients, 2^-16 for states."""
import pytest
import torch

from oracle import lact_oracle as orc

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def lo():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lact_b200 import build
    build.build()
    from lact_b200 import layer_ops
    return layer_ops


def _inputs(b, l, h, hk, dk, dv, n=None, seed=0, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * l + dk)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    decay = -0.7 * torch.exp(-7.0 * torch.rand(h, device="cuda", generator=g))
    n = b if n is None else n
    return dict(q=rn(b, l, h, dk).to(dtype), k=rn(b, l, hk, dk).to(dtype), v=rn(b, l, hk, dv).to(dtype), g=decay, S=rn(n, h, dk, dv),
                do=rn(b, l, h, dv).to(dtype), dS=rn(n, h, dk, dv))


def _near(got, want, size, half, norm, what):
    """|got - want| <= half * (|want| + size) element by element, and `norm` as a whole."""
    got = got.double()
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got).all()), what
    err = (got - want).abs()
    over = (err - half * (want.abs() + size)).max()
    assert float(over) <= 0.0, (what, float(over))
    scale = float(want.norm())
    assert float(err.norm()) <= norm * scale + 1e-30, (what, float(err.norm()) / max(scale, 1e-30))


OUT = dict(half=2.0 ** -8 + 2.0 ** -14, norm=2.0 ** -7)
STATE = dict(half=2.0 ** -15, norm=2.0 ** -16)


def _check(lo, x, cu=None, state=True, dstate=True, scale=None, grads=True):
    from lact_b200 import synchronize_and_check
    leaves = {n: x[n].clone().requires_grad_() for n in ("q", "k", "v")}
    S = x["S"].clone().requires_grad_() if state else None
    cu_dev = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    o, last = lo.linear_attention(leaves["q"], leaves["k"], leaves["v"], x["g"], scale, S, True, cu_dev)
    ins = list(leaves.values()) + ([S] if state else [])
    got = torch.autograd.grad([o, last] if dstate else [o], ins, [x["do"], x["dS"]] if dstate else [x["do"]]) if grads else ()
    synchronize_and_check()
    ref = [x[n].double().requires_grad_() for n in ("q", "k", "v")] + ([x["S"].double().requires_grad_()] if state else [])
    ro, rlast = orc.linear_attention(*ref[:3], x["g"], scale, ref[3] if state else None, cu)
    size = [t.detach().abs().requires_grad_() for t in ref]
    so, slast = orc.linear_attention(*size[:3], x["g"], None if scale is None else abs(scale), size[3] if state else None, cu)
    _near(o.detach(), ro.detach(), so.detach(), **OUT, what="o")
    _near(last.detach(), rlast.detach(), slast.detach(), **STATE, what="last state")
    if not grads:
        return
    do, dS = x["do"].double(), x["dS"].double()
    ro, so = (t + 0.0 * sum(i.sum() for i in ins_) for t, ins_ in ((ro, ref), (so, size)))   # (no tokens: a graph all the same)
    want = torch.autograd.grad([ro, rlast], ref, [do, dS if dstate else torch.zeros_like(dS)])
    bound = torch.autograd.grad([so, slast], size, [do.abs(), dS.abs() if dstate else torch.zeros_like(dS)])
    for name, a, w, s in zip(("dq", "dk", "dv", "dS"), got, want, bound):
        assert a.dtype == (F32 if name == "dS" else BF16)
        _near(a, w, s, **(STATE if name == "dS" else OUT), what=name)


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (64, 128), (128, 64)])
@pytest.mark.parametrize("l", [1, 2, 9, 127, 128, 129, 300, 513])
def test_lengths_and_head_sizes(lo, l, dk, dv):
    _check(lo, _inputs(2, l, 3, 3, dk, dv))


@pytest.mark.parametrize("h,hk", [(4, 2), (6, 1), (5, 5), (12, 4)])
def test_shared_heads(lo, h, hk):
    _check(lo, _inputs(2, 200, h, hk, 64, 128))


@pytest.mark.parametrize("state,dstate", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("l", [5, 260])
def test_without_states(lo, l, state, dstate):
    _check(lo, _inputs(1, l, 2, 2, 128, 128), state=state, dstate=dstate)


@pytest.mark.parametrize("scale", [1.0, 0.3, -2.0])
def test_scales(lo, scale):
    _check(lo, _inputs(1, 190, 2, 1, 64, 64), scale=scale)


@pytest.mark.parametrize("cu", [[0, 300], [0, 0, 300], [0, 1, 2, 130, 130, 300], [0, 128, 256, 300], [0, 77, 205, 300, 300],
                                [5, 40, 41, 290], [0, 0], [300, 300, 300], [0] + [i * 3 for i in range(1, 101)]])
@pytest.mark.parametrize("h,hk", [(3, 3), (4, 2)])
def test_packed_sequences(lo, cu, h, hk):
    """Empty sequences, sequences of one token, tokens before the first and behind the last one (outputs and gradients of zero)."""
    _check(lo, _inputs(1, 300, h, hk, 64, 128, n=len(cu) - 1), cu=cu)


def test_many_entries(lo):
    _check(lo, _inputs(40, 140, 6, 6, 64, 64))


def test_a_long_sequence_of_few_heads(lo):
    _check(lo, _inputs(1, 5000, 2, 2, 64, 64), grads=False)


def _tiles(q, k, v, decay, S, size=100):
    """The same in 64 bits by tiles of `size` tokens (differentiable; the oracle goes token by token)."""
    b, l, h, dk = q.shape
    share = h // k.shape[2]
    q, k, v = (t.double().transpose(1, 2) for t in (q * dk ** -0.5, k.repeat_interleave(share, 2), v.repeat_interleave(share, 2)))
    g, outs = decay.double(), []
    for a in range(0, l, size):
        qc, kc, vc = q[:, :, a:a + size], k[:, :, a:a + size], v[:, :, a:a + size]
        i = torch.arange(qc.shape[2], device=q.device, dtype=torch.float64)
        gap = i[:, None] - i
        W = torch.exp(g[:, None, None] * gap.clamp(min=0)) * (gap >= 0)
        outs.append((qc @ kc.transpose(2, 3) * W) @ vc + torch.exp(g[:, None] * (i + 1))[..., None] * (qc @ S))
        S = torch.exp(g * len(i))[:, None, None] * S + (kc * torch.exp(g[:, None] * (len(i) - 1 - i))[..., None]).transpose(2, 3) @ vc
    return torch.cat(outs, 2).transpose(1, 2), S


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (64, 128), (128, 64)])
@pytest.mark.parametrize("b,l,h,hk", [(10, 1411, 16, 8), (2, 9001, 10, 10)])
def test_many_tiles_a_block(lo, b, l, h, hk, dk, dv):
    """Runs of ten tiles a block, over whole sequences and over cut ones (20 sequences and heads of 71 tiles)."""
    from lact_b200 import synchronize_and_check
    x = _inputs(b, l, h, hk, dk, dv)
    leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "S")]
    o, last = lo.linear_attention(*leaves[:3], x["g"], None, leaves[3], True)
    got = torch.autograd.grad([o, last], leaves, [x["do"], x["dS"]])
    short = lo.linear_attention(*leaves[:3], x["g"], None, leaves[3])[0]     # (without the last state: two pieces of the keys)
    ref = [x[n].double().requires_grad_() for n in ("q", "k", "v", "S")]
    ro, rlast = _tiles(*ref[:3], x["g"], ref[3])
    want = torch.autograd.grad([ro, rlast], ref, [x["do"].double(), x["dS"].double()])
    synchronize_and_check()
    for name, a, w in zip(("o", "o2", "dq", "dk", "dv"), (o, short, *got[:3]), (ro, ro, *want[:3])):
        a, w = a.detach(), w.detach()
        assert float((a.double() - w).norm()) <= OUT["norm"] * float(w.norm()), name
    for name, a, w in (("last", last.detach(), rlast.detach()), ("dS", got[3], want[3])):
        assert float((a.double() - w).norm()) <= STATE["norm"] * float(w.norm()), name


def test_decays_at_the_ends(lo):
    """No decay, no memory (-inf), and decays that underflow within a tile."""
    x = _inputs(1, 400, 6, 6, 64, 64)
    x["g"] = torch.tensor([0.0, float("-inf"), -1e-6, -3.0, -60.0, -1e30], device="cuda")
    _check(lo, x)


def test_views_and_foreign_strides(lo):
    """Slices of a fused projection, a batch expanded from one entry, tokens ahead of the batch, an odd offset."""
    b, l, h, d = 2, 150, 4, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g).to(BF16)
    decay = torch.full((h,), -0.1, device="cuda")
    fused = rn(b, l, 3 * h * d).chunk(3, dim=-1)
    forms = [[t.reshape(b, l, h, d) for t in fused], [rn(1, l, h, d).expand(b, l, h, d) for _ in range(3)],
             [rn(l, b, h, d).transpose(0, 1) for _ in range(3)], [rn(b, h, l, d).transpose(1, 2) for _ in range(3)],
             [rn(b * l * h * d + 1)[1:].reshape(b, l, h, d) for _ in range(3)]]
    for q, k, v in forms:
        o, last = lo.linear_attention(q, k, v, decay, output_final_state=True)
        want, wlast = lo.linear_attention(q.clone(), k.clone(), v.clone(), decay, output_final_state=True)
        assert torch.equal(o, want) and torch.equal(last, wlast)
        leaf = q.detach().requires_grad_()
        lo.linear_attention(leaf, k, v, decay)[0].backward(v)      # (the gradient of the output is a view, too)
        plain = q.clone().requires_grad_()
        lo.linear_attention(plain, k.clone(), v.clone(), decay)[0].backward(v.clone())
        assert torch.equal(leaf.grad, plain.grad)


def test_no_tokens(lo):
    x = _inputs(2, 0, 3, 3, 64, 64)
    o, last = lo.linear_attention(x["q"], x["k"], x["v"], x["g"], initial_state=x["S"], output_final_state=True)
    assert o.shape == (2, 0, 3, 64) and torch.equal(last, x["S"]) and last.data_ptr() != x["S"].data_ptr()
    S = x["S"].clone().requires_grad_()
    q = x["q"].clone().requires_grad_()
    lo.linear_attention(q, x["k"], x["v"], x["g"], initial_state=S, output_final_state=True)[1].backward(x["dS"])
    assert torch.equal(S.grad, x["dS"]) and q.grad.shape == q.shape


@pytest.mark.parametrize("b,h,hk,dk,dv", [(1, 1, 1, 64, 64), (3, 4, 2, 64, 128), (17, 12, 12, 128, 128), (2, 6, 1, 128, 64)])
def test_step(lo, b, h, hk, dk, dv):
    """In place and into another array; the same as a prompt of one token behind the state."""
    x = _inputs(b, 1, h, hk, dk, dv)
    q, k, v = (x[n][:, 0] for n in "qkv")
    want, wlast = orc.linear_attention(x["q"], x["k"], x["v"], x["g"], None, x["S"])
    size, slast = orc.linear_attention(x["q"].abs(), x["k"].abs(), x["v"].abs(), x["g"], None, x["S"].abs())
    before, new = x["S"].clone(), torch.full_like(x["S"], float("nan"))
    o = lo.linear_attention_step(q, k, v, x["g"], x["S"], new_state=new)
    assert torch.equal(x["S"], before)
    _near(o, want[:, 0], size[:, 0], **OUT, what="o")
    _near(new, wlast, slast, **STATE, what="state")
    o2 = lo.linear_attention_step(q, k, v, x["g"], x["S"])
    assert torch.equal(o, o2) and torch.equal(x["S"], new)
    with pytest.raises(ValueError):
        lo.linear_attention_step(q, k, v, x["g"], x["S"][..., ::2].repeat_interleave(2, -1)[:, :, :, :dv].transpose(2, 3).contiguous().transpose(2, 3))
    if b > 1:
        flat = torch.zeros(x["S"].numel() + 64, device="cuda")
        with pytest.raises(ValueError):   # overlapping, not the same
            lo.linear_attention_step(q, k, v, x["g"], flat[:-64].view_as(x["S"]), new_state=flat[64:].view_as(x["S"]))
    with pytest.raises(NotImplementedError):
        lo.linear_attention_step(q.clone().requires_grad_(), k, v, x["g"], x["S"])


def test_prompt_then_steps(lo):
    """A prompt, then tokens one by one, is the whole sequence at once; pieces of a prompt likewise."""
    x = _inputs(2, 333, 4, 2, 64, 128)
    whole, last = lo.linear_attention(x["q"], x["k"], x["v"], x["g"], output_final_state=True)
    part = lambda a, b: tuple(x[n][:, a:b] for n in "qkv")
    o1, S = lo.linear_attention(*part(0, 200), x["g"], output_final_state=True)
    o2, S = lo.linear_attention(*part(200, 329), x["g"], initial_state=S, output_final_state=True)
    rows = [lo.linear_attention_step(*(t[:, 0] for t in part(i, i + 1)), x["g"], S) for i in range(329, 333)]
    want, wlast = orc.linear_attention(x["q"], x["k"], x["v"], x["g"])
    size, slast = orc.linear_attention(x["q"].abs(), x["k"].abs(), x["v"].abs(), x["g"])
    for o, s in ((whole, last), (torch.cat([o1, o2, torch.stack(rows, 1)], 1), S)):
        _near(o, want, size, **OUT, what="o")
        _near(s, wlast, slast, **STATE, what="state")


def test_refusals(lo):
    x = _inputs(2, 20, 4, 2, 64, 64)
    q, k, v, g, S = (x[n] for n in ("q", "k", "v", "g", "S"))
    cu = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    for kind, call in [(ValueError, lambda: lo.linear_attention(q, k, v, g, cu_seqlens=cu)),
                       (ValueError, lambda: lo.linear_attention(q, k, v, g, initial_state=S[:1])),
                       (ValueError, lambda: lo.linear_attention(q, k, v, g, initial_state=S.to(BF16))),
                       (ValueError, lambda: lo.linear_attention(q[:1], k[:1], v[:1], g, cu_seqlens=cu[:1])),
                       (ValueError, lambda: lo.linear_attention(q[:1], k[:1], v[:1], g, cu_seqlens=cu.float())),
                       (ValueError, lambda: lo.linear_attention(q, k, v, g.cpu())), (ValueError, lambda: lo.linear_attention(q, k, v, g, 0.0)),
                       (ValueError, lambda: lo.linear_attention(q, k, v, g, float("inf"))),
                       (ValueError, lambda: lo.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, S[:1])),
                       (ValueError, lambda: lo.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, S, new_state=S.double())),
                       (NotImplementedError, lambda: lo.linear_attention(q, k, v, g.clone().requires_grad_()))]:
        with pytest.raises(kind):
            call()


def test_bounds_that_are_wrong_stay_inside(lo):
    """cu_seqlens past the end, falling or negative: nothing outside is read or written (the numbers are then unspecified)."""
    x = _inputs(1, 200, 2, 2, 64, 64, n=3)
    for cu in ([0, 150, 900, 1200], [0, 150, 90, 200], [-50, 20, 100, 200]):
        o, last = lo.linear_attention(x["q"], x["k"], x["v"], x["g"], None, x["S"], True, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert o.shape == (1, 200, 2, 64) and last.shape == x["S"].shape


def test_sequences_keep_their_nan(lo):
    """A sequence that has diverged does not touch its neighbours, whose tiles begin and end between its tokens; of a sequence, the
    tiles before the bad token stay."""
    x = _inputs(1, 500, 2, 2, 64, 64, n=3)
    cu = torch.tensor([0, 130, 331, 500], dtype=torch.int32, device="cuda")
    args = lambda y: (y["q"], y["k"], y["v"], x["g"], None, x["S"], True, cu)
    o, last = lo.linear_attention(*args(x))
    for name in ("q", "k", "v"):
        y = {n: x[n].clone() for n in ("q", "k", "v")}
        y[name][:, 130:331] = float("nan")
        oy, ly = lo.linear_attention(*args(y))
        assert torch.equal(oy[:, :130], o[:, :130]) and torch.equal(oy[:, 331:], o[:, 331:])
        assert torch.equal(ly[0], last[0]) and torch.equal(ly[2], last[2])
        assert bool(oy[:, 130:331].isnan().all())
        y = {n: x[n].clone() for n in ("q", "k", "v")}
        y[name][0, 130 + 140, :, 3] = float("inf")
        oy, ly = lo.linear_attention(*args(y))
        assert torch.equal(oy[:, 130:130 + 128], o[:, 130:130 + 128]) and not bool(oy[0, 130 + 140].isfinite().all())
        leaves = [y[n].clone().requires_grad_() for n in ("q", "k", "v")]
        ref = [x[n].clone().requires_grad_() for n in ("q", "k", "v")]
        for t in (leaves, ref):
            lo.linear_attention(*t, x["g"], None, x["S"], False, cu)[0].backward(x["do"])
        for a, r in zip(leaves, ref):
            assert torch.equal(a.grad[:, :130], r.grad[:, :130]) and torch.equal(a.grad[:, 331:], r.grad[:, 331:])


def test_same_bits_every_time_and_on_other_streams(lo):
    x = _inputs(2, 700, 4, 2, 128, 64)

    def go():
        leaves = [x[n].clone().requires_grad_() for n in ("q", "k", "v", "S")]
        o, last = lo.linear_attention(*leaves[:3], x["g"], None, leaves[3], True)
        return [o, last, *torch.autograd.grad([o, last], leaves, [x["do"], x["dS"]])]
    first = go()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    runs = []
    for s in streams * 2:     # two calls at once
        with torch.cuda.stream(s):
            runs.append(go())
    torch.cuda.synchronize()
    for r in runs:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_captured_and_replayed(lo):
    """Forward, backward and a step in one graph; a second graph beside it, replayed in turn; new inputs at every replay."""
    xs = [_inputs(1, 400, 4, 4, 64, 64, seed=s) for s in range(3)]

    def go(q, k, v, S, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, S)]
        o, last = lo.linear_attention(*leaves[:3], xs[0]["g"], None, leaves[3], True)
        grads = torch.autograd.grad([o], leaves, [do])
        with torch.no_grad():
            token = lo.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], xs[0]["g"], last.detach())
        return [o.detach(), token, *grads]
    static = [[xs[0][n].clone() for n in ("q", "k", "v", "S", "do")] for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in static:
            go(*s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(go(*s))
        graphs.append(gr)
    for i, j in ((1, 2), (2, 0)):
        for s, n in zip(static, (i, j)):
            for t, name in zip(s, ("q", "k", "v", "S", "do")):
                t.copy_(xs[n][name])
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for got, n in zip(outs, (i, j)):
            want = go(*(xs[n][name] for name in ("q", "k", "v", "S", "do")))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    from lact_b200 import synchronize_and_check
    synchronize_and_check()


def test_compiled_caller(lo):
    """One operator for a compiled caller, without a graph break."""
    x = _inputs(1, 140, 2, 2, 64, 64)

    def f(q, k, v, g, S):
        o, last = lo.linear_attention(q * 1.0, k, v, g, None, S, True)
        return o.float().sum() + last.sum()
    leaf = x["q"].clone().requires_grad_()
    want = f(leaf, x["k"], x["v"], x["g"], x["S"])
    want.backward()
    other = x["q"].clone().requires_grad_()
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(other, x["k"], x["v"], x["g"], x["S"])
    got.backward()
    assert torch.equal(got, want) and torch.equal(other.grad, leaf.grad)
    step = lambda q, k, v, g, S, new: lo.linear_attention_step(q * 1.0, k, v, g, S, new_state=new)
    token = tuple(x[n][:, 0] for n in "qkv")
    news = [torch.zeros_like(x["S"]) for _ in range(2)]
    with torch.no_grad():
        plain = step(*token, x["g"], x["S"], news[0])
        traced = torch.compile(step, fullgraph=True, backend="aot_eager")(*token, x["g"], x["S"], news[1])
    assert torch.equal(plain, traced) and torch.equal(news[0], news[1])
