"""Forward-mode derivatives: no operator has a formula for them, and each says so (shape-only tensors: no GPU)."""
import pytest
import torch
import torch.autograd.forward_ad as fw

BF16, F32 = torch.bfloat16, torch.float32


def _t(*s, dtype=BF16):
    return torch.empty(*s, dtype=dtype, device="meta")


@pytest.fixture(scope="module")
def ops():
    from lact_b200 import build
    build.build()
    from lact_b200 import _lib
    _lib.load_ops()
    return torch.ops.lact_b200


def _linear():
    return [_t(1, 8, 4, 64), _t(1, 8, 4, 64), _t(1, 8, 4, 64), _t(4, dtype=F32), 0.1, _t(1, 4, 64, 64, dtype=F32), None, True]


def _step():
    return [_t(2, 4, 64), _t(2, 4, 64), _t(2, 4, 64), _t(4, dtype=F32), 0.1, _t(2, 4, 64, 64, dtype=F32), _t(2, 4, 64, 64, dtype=F32)]


def _norm():
    return [_t(3, 8, 64), _t(64, dtype=F32), _t(64, dtype=F32), 4, 1e-5, True]


def _swa():
    return [_t(1, 8, 4, 64), _t(1, 8, 4, 64), _t(1, 8, 4, 64), 0, 0.1]


def _swa_cache():
    return [_t(1, 8, 4, 64), _t(1, 9, 4, 64), _t(1, 9, 4, 64), _t(1, 8, 4, 64), _t(1, 8, 4, 64), 0.1]


def _qkv():
    return [_t(1, 8, 64), _t(1, 8, 64), _t(1, 8, 64), 1, True, True, None, None, 64, 0, None]


def _lr():
    return [_t(1, 8, 3, dtype=F32), _t(1, 8, 1), 1, 0.1]


def _out():
    return [_t(2, 8, 64), _t(64, dtype=F32), _t(1, 8, 128), _t(1, 8, 128), 2, 1e-5]


def _ffn():
    return [_t(1, 128, 64), _t(1, 64, 64), _t(1, 8, 64)]


def _fw_grads():
    return _ffn() + [_t(1, 8, 64)] + [_t(1, 8, 1, dtype=F32) for _ in range(3)]


def _l2():
    return [_t(1, 8, 64, dtype=F32), _t(1, 8, 64), _t(1, 8, 1, dtype=F32), 1e-5, True]


def _scan():
    from lact_b200 import program as P
    w = [_t(1, 64, 64, dtype=F32) for _ in range(3)]
    steps, cfg = [P.UPDATE, 0, 8, 0, P.APPLY, 0, 8, 0], [0] * 10 + [-1, 0, 0, 0]
    return w + [_t(1, 8, 64) for _ in range(3)] + [_t(1, 8, 1, dtype=F32) for _ in range(4)] + [None, None, None, steps, cfg, 0.0]


CASES = [("swa_fwd", _swa), ("swa_fwd_cache", _swa_cache), ("qkv_prologue", _qkv), ("lr_prologue", _lr), ("out_epilogue", _out),
         ("swiglu_ffn_fwd", _ffn), ("fw_grads_fwd", _fw_grads), ("l2_norm_add_fwd", _l2), ("scan_fwd", _scan),
         ("linear_attention_fwd", _linear), ("linear_attention_step", _step), ("group_norm_fwd", _norm)]


@pytest.mark.parametrize("name,make", CASES)
@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
def test_a_tangent_is_refused(ops, name, make, mode):
    """Of every argument by itself, with and without gradients."""
    op = getattr(ops, name)
    for i, a in enumerate(make()):
        if not isinstance(a, torch.Tensor):
            continue
        for grad in (False, True):
            args = make()
            with mode(), fw.dual_level():
                args[i] = fw.make_dual(args[i].requires_grad_() if grad else args[i], torch.empty_like(args[i]))
                with pytest.raises(NotImplementedError):
                    op(*args)


@pytest.mark.parametrize("name,make", CASES)
def test_calls_without_tangents_are_as_they_were(ops, name, make):
    op = getattr(ops, name)
    with fw.dual_level():
        op(*make())
        dual = fw.make_dual(_t(3), _t(3))    # (of another computation)
        assert fw.unpack_dual(dual).tangent is not None
    args = make()
    with fw.dual_level():
        args[0] = fw.make_dual(args[0], torch.empty_like(args[0]))
        args[0] = fw.unpack_dual(args[0]).primal
        op(*args)
