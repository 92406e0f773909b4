"""Linear attention, its steps and group norm on arrays of more than 2^31 elements: every batch entry holds the same values, and has to give
the same bits as the first."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
FAR = 2 ** 31 + 2 ** 26


@pytest.fixture(scope="module")
def lo():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    if torch.cuda.get_device_properties(0).total_memory < 100e9:
        pytest.skip("needs 100 GB")
    from lact_b200 import build
    build.build()
    from lact_b200 import layer_ops
    yield layer_ops
    torch.cuda.empty_cache()


def _same(t, step=1):
    """Entry by entry (the first against each: no second copy of the whole)."""
    return all(torch.equal(t[i], t[0]) for i in range(step, t.shape[0], step))


def _copies(t, n):
    return t.expand(n, *t.shape[1:]).contiguous()


def _rn(*s, seed=0):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def test_prompts(lo):
    """As many heads as SMs: every CTA takes whole sequences, so that entries do not differ by where their runs begin."""
    b, h, d = 16, torch.cuda.get_device_properties(0).multi_processor_count, 128
    l = FAR // (b * h * d) + 1
    one = [_rn(1, l, h, d, seed=i).to(BF16) for i in range(4)]
    g = -0.1 * torch.rand(h, device="cuda")
    q, k, v, do = (_copies(t, b) for t in one)
    assert q.numel() > 2 ** 31
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o, _ = lo.linear_attention(*leaves, g)
    assert _same(o.detach())
    grads = torch.autograd.grad(o, leaves, do)
    assert all(_same(t) for t in grads)
    small = [t[:, -300:].clone() for t in one]     # the first entry itself against a call of a size that other tests check
    want, S = lo.linear_attention(one[0][:, :-300], one[1][:, :-300], one[2][:, :-300], g, output_final_state=True)
    tail = lo.linear_attention(*small[:3], g, initial_state=S)[0]
    got = o.detach()[-1:, -300:].double()
    assert float((got - tail.double()).norm()) <= 2.0 ** -7 * float(got.norm())


def test_a_packed_prompt(lo):
    h, d = 2 * torch.cuda.get_device_properties(0).multi_processor_count, 64
    n = 32
    l = FAR // (n * h * d) + 1
    one = [_rn(1, l, h, d, seed=i).to(BF16) for i in range(3)]
    g = -0.1 * torch.rand(h, device="cuda")
    q, k, v = (_copies(t, n).view(1, n * l, h, d) for t in one)
    cu = torch.arange(n + 1, device="cuda", dtype=torch.int32) * l
    o = lo.linear_attention(q, k, v, g, cu_seqlens=cu)[0].view(n, l, h, d)
    want = lo.linear_attention(*one, g)[0].double()
    for i in (0, n // 2, n - 1):    # (the runs begin elsewhere in each: the same numbers within their roundings)
        assert float((o[i:i + 1].double() - want).norm()) <= 2.0 ** -7 * float(want.norm())


def test_steps(lo):
    h, d = 96, 128
    b = FAR // (h * d * d) + 1
    one = [_rn(1, h, d, seed=i).to(BF16) for i in range(3)]
    S1, g = _rn(1, h, d, d), -0.1 * torch.rand(h, device="cuda")
    S = _copies(S1, b)
    assert S.numel() > 2 ** 31
    o = lo.linear_attention_step(*(_copies(t, b) for t in one), g, S)
    want = lo.linear_attention_step(*one, g, S1)
    assert _same(o) and _same(S) and torch.equal(o[:1], want) and torch.equal(S[:1], S1)


@pytest.mark.parametrize("shape,groups", [((1, 1536), 12), ((1, 3001, 96), 32), ((1, 1, 5000), 8)])
def test_group_norm(lo, shape, groups):
    n = FAR // (shape[-1] * (shape[1] if len(shape) == 3 else 1)) + 1
    one, dy1 = (_rn(*shape, seed=i).to(BF16) for i in range(2))
    w, b = _rn(shape[-1], seed=3), _rn(shape[-1], seed=4)
    x, dy = _copies(one, n), _copies(dy1, n)
    assert x.numel() > 2 ** 31
    x.requires_grad_()
    y = lo.group_norm(x, groups, w, b, activation="silu")
    dx, = torch.autograd.grad(y, x, dy)
    x1 = one.clone().requires_grad_()
    y1 = lo.group_norm(x1, groups, w, b, activation="silu")
    d1, = torch.autograd.grad(y1, x1, dy1)
    for got, want in ((y.detach(), y1.detach()), (dx, d1)):
        far = got.reshape(n, -1)
        if shape[1:] != (3001, 96):     # (chunks of spots differ with the number of samples, and with them the order of the sums)
            assert torch.equal(far[:1], want.reshape(1, -1))
        else:
            assert float((far[:1].double() - want.reshape(1, -1).double()).norm()) <= 2.0 ** -8 * float(want.double().norm())
        for a in range(0, n, 4096):
            part = far[a:a + 4096]
            assert torch.equal(part, far[:1].expand_as(part)), a
