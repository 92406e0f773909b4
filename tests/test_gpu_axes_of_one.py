"""Layouts that axes of one entry leave open: PyTorch calls them contiguous, the kernels read strides.  The same values in plain copies
give the same bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def lo():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lact_b200 import build
    build.build()
    from lact_b200 import layer_ops
    return layer_ops


def _rn(*s, seed=0):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + sum(s))).to(BF16)


def _copy(t):
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t.detach())


def _heads(b, l, h, d, seed):
    x = _rn(b, l, h, d, seed=seed)
    yield x.transpose(1, 2).contiguous().transpose(1, 2)                  # heads ahead of tokens
    yield torch.empty(x.numel() + 1, dtype=BF16, device="cuda")[1:].view(x.shape).copy_(x)     # off a 16-byte boundary
    if b == 1:
        yield x.as_strided((b, l, h, d), (l * h * d + 3, h * d, d, 1))
    if h == 1:
        yield x.as_strided((b, l, h, d), (l * d, d, 5, 1))
    if l == 1:
        yield x.as_strided((b, l, h, d), (h * d, 3, d, 1))


@pytest.mark.parametrize("b,l,lk,h", [(1, 1, 40, 4), (3, 1, 300, 4), (2, 1, 1, 1), (1, 40, 40, 2), (2, 60, 1, 4)])
def test_attention(lo, b, l, lk, h):
    for q, k, v, do in zip(*(_heads(b, n, h, 64, i) for i, n in enumerate((l, lk, lk, l)))):
        for call in (lo.block_attention, lo.sliding_window_attention) if l == lk else (lo.block_attention,):
            got, want = [], []
            for out, ts in ((got, (q, k, v, do)), (want, [_copy(t) for t in (q, k, v, do)])):
                leaves = [t.detach().requires_grad_() for t in ts[:3]]
                o = call(*leaves)
                out += [o, *torch.autograd.grad(o, leaves, ts[3])]
            assert all(torch.equal(a, w) for a, w in zip(got, want))


def test_attention_over_a_cache(lo):
    q, kc, vc, k, v = (next(_heads(1, n, 4, 64, i)) for i, n in enumerate((1, 40, 40, 1, 1)))
    op = torch.ops.lact_b200.swa_fwd_cache
    assert torch.equal(op(q, kc, vc, k, v, 0.125), op(*(_copy(t) for t in (q, kc, vc, k, v)), 0.125))


def _rows(b, s, n, seed):
    x = _rn(b, s, n, seed=seed)
    yield torch.empty(x.numel() + 1, dtype=BF16, device="cuda")[1:].view(x.shape).copy_(x)
    if b == 1:
        yield x.as_strided((b, s, n), (s * n + 3, n, 1))
    if s == 1:
        yield x.as_strided((b, s, n), (n, 3, 1))
        yield x.transpose(1, 2).contiguous().transpose(1, 2)


@pytest.mark.parametrize("b,s", [(1, 1), (3, 1), (1, 7)])
def test_layer_passes(lo, b, s):
    w = torch.ones(64, device="cuda")
    x = _rn(b * 2, s, 64, seed=9)
    for a, c, d in zip(*(_rows(b, s, 128, i) for i in range(3))):
        for call in (lambda p, q, r: lo.qkv_prologue(p, q, r, 2), lambda p, q, r: (lo.out_epilogue(x, w, 2, p, q),)):
            got, want = [], []
            for out, ts in ((got, (a, c, d)), (want, [_copy(t) for t in (a, c, d)])):
                leaves = [t.detach().requires_grad_() for t in ts]
                o = call(*leaves)
                out += [*o, *torch.autograd.grad(sum(t.float().square().sum() for t in o), leaves, allow_unused=True)]
            assert all(torch.equal(g, w_) for g, w_ in zip(got, want) if w_ is not None)
