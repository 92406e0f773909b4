"""Group norm: what the entry points refuse, checked on the host, and the oracle against differences and PyTorch's own."""
import ctypes as C

import pytest
import torch

from oracle import lact_oracle as orc

BF16 = torch.bfloat16


class _Config(C.Structure):
    _fields_ = [(n, C.c_int64) for n in ("n", "s", "channels", "groups", "x_ns", "x_ss", "dy_ns", "dy_ss")] + [
        ("dtype", C.c_int32), ("silu", C.c_int32), ("eps", C.c_float)]


def _config(**over):
    c = dict(n=2, s=50, channels=96, groups=8, x_ns=4800, x_ss=96, dy_ns=4800, dy_ss=96, dtype=1, silu=1, eps=1e-5)
    c.update(over)
    return _Config(**c)


@pytest.fixture(scope="module")
def lib():
    from lact_b200 import build
    build.build()
    from lact_b200 import _lib
    return _lib.lib()


@pytest.mark.parametrize("over,code", [(dict(n=0), -2), (dict(s=0), -2), (dict(channels=0), -2), (dict(groups=0), -2), (dict(groups=7), -2),
                                       (dict(dtype=2), -3), (dict(eps=-1.0), -5), (dict(eps=float("nan")), -5), (dict(eps=float("inf")), -5),
                                       (dict(channels=1 << 21), -2), (dict(s=(1 << 30) + 1), -2)])
def test_bad_configurations_are_refused(lib, over, code):
    n, c, p = C.c_size_t(0), _config(**over), C.c_void_p(4096)
    assert lib.lact_group_norm_workspace_bytes(C.byref(c), 0, C.byref(n)) == code
    assert lib.lact_group_norm_fwd(C.byref(c), p, p, p, p, p, None, C.c_size_t(0), None) == code
    assert lib.lact_group_norm_bwd(C.byref(c), p, p, p, p, p, p, p, p, None, C.c_size_t(0), None) == code


def test_missing_and_crooked_pointers_are_refused(lib):
    c, p, z = _config(), C.c_void_p(4096), C.c_size_t(0)
    assert lib.lact_group_norm_fwd(C.byref(c), None, p, p, p, p, None, z, None) == -1
    assert lib.lact_group_norm_fwd(C.byref(c), p, None, None, None, p, None, z, None) == -1
    assert lib.lact_group_norm_fwd(C.byref(c), p, p, p, C.c_void_p(4098), p, None, z, None) == -2
    assert lib.lact_group_norm_bwd(C.byref(c), p, p, p, p, None, p, p, p, None, z, None) == -1
    assert lib.lact_group_norm_workspace_bytes(None, 0, C.byref(z)) == -1


@pytest.mark.parametrize("over,back", [(dict(x_ns=4801), 0), (dict(x_ss=100), 0), (dict(dy_ss=97), 1), (dict(dy_ns=4804), 1)])
def test_strides_that_break_an_access_are_refused(lib, over, back):
    c, p, z = _config(**over), C.c_void_p(4096), C.c_size_t(0)
    if back:
        assert lib.lact_group_norm_bwd(C.byref(c), p, p, p, p, p, p, p, p, None, z, None) in (-2, -7, -8)
    else:
        assert lib.lact_group_norm_fwd(C.byref(c), p, p, p, p, p, None, z, None) in (-2, -7, -8)   # (-7, -8: no device here)


def test_python_checks():
    from lact_b200 import layer_ops as lo
    x, w = torch.zeros(2, 5, 24), torch.zeros(24)
    for kind, call in [(ValueError, lambda: lo.group_norm(x, 5)), (ValueError, lambda: lo.group_norm(x, 0)),
                       (ValueError, lambda: lo.group_norm(x[0, 0], 4)), (TypeError, lambda: lo.group_norm(x.double(), 4)),
                       (TypeError, lambda: lo.group_norm(x.half(), 4)), (ValueError, lambda: lo.group_norm(x, 4, w[:12])),
                       (ValueError, lambda: lo.group_norm(x, 4, w, w[:3])), (TypeError, lambda: lo.group_norm(x, 4, w.double())),
                       (ValueError, lambda: lo.group_norm(x, 4, activation="relu")), (ValueError, lambda: lo.group_norm(x, 4, eps=-1.0)),
                       (ValueError, lambda: lo.group_norm(x, 4, eps=float("nan"))), (ValueError, lambda: lo.group_norm(x[..., :0], 4)),
                       (ValueError, lambda: lo.group_norm(x, 4, w, w))]:   # (the last: no CUDA)
        with pytest.raises(kind):
            call()


def test_oracle_against_pytorch_and_differences():
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 3, 4, 12), (12,), (12,)))
    want = torch.nn.functional.group_norm(x.movedim(-1, 1), 4, w, b, 1e-3).movedim(1, -1)
    assert torch.allclose(orc.group_norm(x, 4, w, b, 1e-3), want, rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda *a: orc.group_norm(a[0], 4, a[1], a[2], 1e-3, True), [t.requires_grad_() for t in (x, w, b)])
