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
