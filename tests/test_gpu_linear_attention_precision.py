"""Linear attention: its errors are those of the roundings that the kernels name, and no more.

The tiles round twice on the way to an output: the weights of a tile's tokens and the copy of the incoming state to bf16, and the sum
to bf16.  Both are done here in 64 bits: with `inner` the error that the first leaves and `last` that of rounding the exact output, which
are independent of one another, the kernel's error is sqrt(inner^2 + last^2) of the norm.  What it computes in 32 bits (2^-24 an addition,
2^-22 an exponential, at most some tens of them in a row) is a thousandth of that; with random signs over the 10^5 and more values of a
case the norm is within 1 % of its expectation, and 5 % are allowed.  A weight or a copy with one bit less would be 60 % above.
Few tokens and single ones are in 32 bits inside: `last` alone.

States: decayed rows of the keys are three bf16 pieces, 2^-25 of each.  What is left: a tile's sum D is added up by the tensor core,
which cuts off, in 24 steps (8 of 16 tokens, three pieces): half a step of 2^-23 each and all to the same side, of partial sums that grow to D
over the first eight, is at most 21.5 * 2^-24; two exponentials and their exponents' roundings 2^-21; the additions in fp32, 2^-24 a
tile, of at most eight tiles that have not decayed: 1.3e-6 + 0.5e-6 + 0.1e-6 (these with random signs), below 2^-19.  (Two pieces leave
2.7e-6.)"""
import pytest
import torch

from oracle import lact_oracle as orc

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module")
def lo():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lact_b200 import build
    build.build()
    from lact_b200 import layer_ops
    return layer_ops


def _bf16(t):
    return t.to(BF16).double()


def _operator(x, y, z, S, g, reverse, rounded):
    """out_t = x_t^T S_t over heads ahead of tokens, [b, h, l, .] in 64 bits, by the kernel's tiles: 128 tokens from the sequence's start.
    Backwards in time the state before the last token is not decayed by it."""
    if reverse:
        x, y, z = (t.flip(2) for t in (x, y, z))
    l, at, outs = x.shape[2], 0, []
    sizes = [128] * (l // 128) + ([l % 128] if l % 128 else [])
    for c, n in enumerate(reversed(sizes) if reverse else sizes):
        xc, yc, zc = x[:, :, at:at + n], y[:, :, at:at + n], z[:, :, at:at + n]
        first = 0 if reverse and c == 0 else 1
        i = torch.arange(n, device=x.device, dtype=F64)
        gap = i[:, None] - i
        P = (xc @ yc.transpose(2, 3)) * torch.exp(g[:, None, None] * gap.clamp(min=0)) * (gap >= 0)
        copy = S
        if rounded:
            P, copy = _bf16(P), _bf16(S)
        outs.append(P @ zc + torch.exp(g[:, None] * (i + first))[..., None] * (xc @ copy))
        S = (torch.exp(g * (n - 1 + first))[:, None, None] * S +
             (yc * torch.exp(g[:, None] * (n - 1 - i))[..., None]).transpose(2, 3) @ zc)
        at += n
    o = torch.cat(outs, 2)
    return (o.flip(2) if reverse else o), S


def _expected(q, k, v, do, S, dS, g, scale):
    """name -> (exact, with the tiles' inner rounding)."""
    heads = lambda t: t.double().transpose(1, 2)
    q, k, v, do = (heads(t) for t in (q, k, v, do))
    T = lambda t: t.transpose(2, 3)
    out = {}
    for rounded in (False, True):
        o, last = _operator(q, k, v, S, g, False, rounded)
        dq, _ = _operator(do, v, k, T(S), g, False, rounded)
        R = dS / scale
        dv, _ = _operator(k, q, do, R, g, True, rounded)
        dk, dfirst = _operator(v, do, q, T(R), g, True, rounded)
        for name, t in (("o", o), ("dq", dq), ("dv", dv), ("dk", dk)):
            out.setdefault(name, []).append((t * scale).transpose(1, 2))
        if not rounded:
            out["last"], out["dS"] = last, T(dfirst) * torch.exp(g)[:, None, None] * scale
    return out


def _inputs(b, l, h, dk, dv):
    gen = torch.Generator(device="cuda").manual_seed(b + l + h + dk)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    g = -0.7 * torch.exp(-6.5 * torch.rand(h, device="cuda", generator=gen))
    return rn(b, l, h, dk).to(BF16), rn(b, l, h, dk).to(BF16), rn(b, l, h, dv).to(BF16), rn(b, l, h, dv).to(BF16), rn(b, h, dk, dv), rn(
        b, h, dk, dv), g


def _relative(a, want):
    return float((a.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (64, 128), (128, 64)])
@pytest.mark.parametrize("b,l,h", [(1, 6001, 3), (4, 1280, 16), (2, 300, 40), (8, 40, 30)])
def test_tiles(lo, b, l, h, dk, dv):
    """Cut sequences and whole ones, one tile and many, a broken last tile."""
    q, k, v, do, S, dS, g = _inputs(b, l, h, dk, dv)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, S)]
    o, last = lo.linear_attention(*leaves[:3], g, None, leaves[3], True)
    dq, dk_, dv_, dfirst = torch.autograd.grad([o, last], leaves, [do, dS])
    ref = _expected(q, k, v, do, S.double(), dS.double(), g.double(), dk ** -0.5)
    for name, got in (("o", o.detach()), ("dq", dq), ("dk", dk_), ("dv", dv_)):
        exact, inner = ref[name]
        allowed = 1.05 * (_relative(inner, exact) ** 2 + _relative(_bf16(exact), exact) ** 2) ** 0.5
        assert _relative(got, exact) <= allowed, (name, _relative(got, exact), allowed)
    for name, got in (("last", last.detach()), ("dS", dfirst)):
        assert _relative(got, ref[name]) <= 2.0 ** -19, (name, _relative(got, ref[name]))


@pytest.mark.parametrize("b,l,h", [(20, 1, 30), (5, 9, 20), (100, 3, 12)])
def test_few_tokens_and_steps(lo, b, l, h):
    q, k, v, do, S, dS, g = _inputs(b, l, h, 128, 64)
    o, last = lo.linear_attention(q, k, v, g, None, S, True)
    exact, elast = orc.linear_attention(q, k, v, g, None, S)
    allowed = 1.01 * _relative(_bf16(exact), exact) + 2.0 ** -19
    assert _relative(o, exact) <= allowed and _relative(last, elast) <= 2.0 ** -19
    if l == 1:
        o = lo.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, S)
        assert _relative(o[:, None], exact) <= allowed and _relative(S, elast) <= 2.0 ** -19
