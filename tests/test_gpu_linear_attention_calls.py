"""Linear attention: calls around the operator itself - states that a backward still needs, layouts that axes of one leave open."""
import pytest
import torch

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


def _rn(*s, seed=0):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + sum(s)))


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("l", [4, 200])
def test_a_state_that_a_backward_needs_may_not_be_stepped_on(lo, l, mode):
    q, k, v = (_rn(2, l, 4, 64, seed=i).to(BF16) for i in range(3))
    g, S = torch.full((4,), -0.1, device="cuda"), _rn(2, 4, 64, 64)
    leaf = q.clone().requires_grad_()
    o = lo.linear_attention(leaf, k, v, g, initial_state=S)[0]
    version = S._version
    with mode():
        lo.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, S)
    assert S._version == version + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(v)
    # into another array, the backward has its state
    o = lo.linear_attention(leaf, k, v, g, initial_state=S)[0]
    new = torch.empty_like(S)
    with torch.no_grad():
        lo.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, S, new_state=new)
    o.backward(v)
    assert new._version == 1 and bool(leaf.grad.isfinite().all())


def _forms(b, l, h, d, seed):
    """[b, l, h, d] values laid out in ways that PyTorch counts as contiguous where an axis has one entry."""
    x = _rn(b, l, h, d, seed=seed).to(BF16)
    yield x.transpose(1, 2).contiguous().transpose(1, 2)                  # heads ahead of tokens
    if b == 1:                                                            # a batch stride that nothing aligns
        yield x.as_strided((b, l, h, d), (l * h * d + 3, h * d, d, 1))
    if h == 1:
        yield x.as_strided((b, l, h, d), (l * d, d, 5, 1))
    if l == 1:
        yield x.as_strided((b, l, h, d), (h * d, 3, d, 1))


@pytest.mark.parametrize("b,l,h,hk", [(1, 1, 4, 2), (3, 1, 4, 4), (1, 1, 1, 1), (1, 40, 4, 2), (2, 40, 1, 1), (1, 300, 4, 2), (1, 150, 1, 1)])
@pytest.mark.parametrize("packed", [False, True])
def test_axes_of_one_entry(lo, b, l, h, hk, packed):
    if packed and b > 1:
        pytest.skip("packed sequences are a batch of one")
    cu = torch.tensor([0, l], dtype=torch.int32, device="cuda") if packed else None
    g = torch.full((h,), -0.1, device="cuda")
    for q, k, v, do in zip(*(_forms(b, l, n, 64, i) for i, n in enumerate((h, hk, hk, h)))):
        got, want = [], []
        for out, operands in ((got, (q, k, v, do)), (want, [t.clone(memory_format=torch.contiguous_format) for t in (q, k, v, do)])):
            leaves = [t.detach().requires_grad_() for t in operands[:3]]
            o, last = lo.linear_attention(*leaves, g, output_final_state=True, cu_seqlens=cu)
            out += [o, last, *torch.autograd.grad(o, leaves, operands[3])]
        assert all(torch.equal(a, w) for a, w in zip(got, want))


@pytest.mark.parametrize("b,h,hk", [(1, 4, 2), (3, 4, 4), (1, 1, 1), (3, 1, 1)])
def test_axes_of_one_entry_of_a_step(lo, b, h, hk):
    g, S = torch.full((h,), -0.1, device="cuda"), _rn(b, h, 64, 64)
    for forms in zip(*(_forms(b, 1, n, 64, i) for i, n in enumerate((h, hk, hk)))):
        news = [torch.zeros_like(S) for _ in range(2)]
        o = lo.linear_attention_step(*(t[:, 0] for t in forms), g, S, new_state=news[0])
        want = lo.linear_attention_step(*(t[:, 0].clone(memory_format=torch.contiguous_format) for t in forms), g, S, new_state=news[1])
        assert torch.equal(o, want) and torch.equal(*news)
