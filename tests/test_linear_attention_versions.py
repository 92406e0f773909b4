"""linear_attention_step writes a state in place: autograd has to learn of it, on every way there (shape-only tensors: no GPU)."""
import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def op():
    from lact_b200 import build
    build.build()
    from lact_b200 import _lib
    _lib.load_ops()
    return torch.ops.lact_b200.linear_attention_step


def _token(b=2, h=4, d=64):
    return (*(torch.empty(b, h, d, dtype=BF16, device="meta") for _ in range(3)), torch.empty(h, device="meta"), 0.1)


def _state(b=2, h=4, d=64):
    return torch.empty(b, h, d, d, device="meta")


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
def test_a_step_gives_the_written_state_a_new_version(op, mode):
    state, new, token = _state(), _state(), _token()
    with mode():
        op(*token, state, state)
        assert state._version == 1
        op(*token, state, new)
    assert state._version == 1 and new._version == 1      # what is read alone keeps its own


def test_states_of_inference_mode_have_no_version(op):
    token = _token()
    with torch.inference_mode():
        state = _state()
        op(*token, state, state)
    with torch.no_grad():
        op(*token, state, state)                          # (outside of the mode as well: a serving loop may leave it)
    assert state.is_inference()


def test_a_backward_that_has_saved_the_state_raises(op):
    state, x = _state(), _state().requires_grad_()
    loss = (x * state).sum()
    with torch.no_grad():
        op(*_token(), state, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
