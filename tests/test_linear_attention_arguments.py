"""Linear attention: what the entry points refuse, checked on the host, and the oracle against differences and a second form."""
import ctypes as C

import pytest
import torch

from oracle import lact_oracle as orc

BF16 = torch.bfloat16


class _Config(C.Structure):
    _fields_ = [(n, C.c_int64) for n in ("batch", "tokens", "heads", "kv_heads", "dk", "dv", "sequences", "q_ts", "q_bs", "k_ts", "k_bs",
                                         "v_ts", "v_bs", "do_ts", "do_bs")] + [("scale", C.c_float)]


def _config(**over):
    c = dict(batch=2, tokens=300, heads=4, kv_heads=2, dk=64, dv=128, sequences=0, q_ts=256, q_bs=256 * 300, k_ts=128, k_bs=128 * 300,
             v_ts=256, v_bs=256 * 300, do_ts=512, do_bs=512 * 300, scale=0.125)
    c.update(over)
    return _Config(**c)


@pytest.fixture(scope="module")
def lib():
    from lact_b200 import build
    build.build()
    from lact_b200 import _lib
    return _lib.lib()


@pytest.mark.parametrize("over,code", [(dict(dk=96), -2), (dict(dv=32), -2), (dict(kv_heads=3), -2), (dict(kv_heads=0), -2),
                                       (dict(heads=0), -2), (dict(tokens=0), -2), (dict(batch=0), -2), (dict(batch=70000), -2),
                                       (dict(tokens=(1 << 30) + 1), -2), (dict(sequences=-1), -2), (dict(sequences=3), -5),
                                       (dict(scale=0.0), -5), (dict(scale=float("nan")), -5), (dict(scale=float("inf")), -5)])
def test_bad_configurations_are_refused(lib, over, code):
    n = C.c_size_t(0)
    c = _config(**over)
    assert lib.lact_linear_attention_workspace_bytes(C.byref(c), 0, C.byref(n)) == code
    p = C.c_void_p(4096)   # (never looked at)
    one = C.c_void_p(4096)
    assert lib.lact_linear_attention_fwd(C.byref(c), p, p, p, p, None, None, None, p, None, C.c_size_t(0), one, None) == code
    assert lib.lact_linear_attention_bwd(C.byref(c), p, p, p, p, None, None, None, C.c_size_t(0), p, None, p, p, p, None, None, C.c_size_t(0),
                                         one, None) == code


@pytest.mark.parametrize("over", [dict(q_ts=255), dict(q_ts=248), dict(k_bs=9), dict(v_ts=128)])
def test_bad_strides_are_refused(lib, over):
    c, p = _config(**over), C.c_void_p(4096)
    assert lib.lact_linear_attention_fwd(C.byref(c), p, p, p, p, None, None, None, p, None, C.c_size_t(0), p, None) == -2


def test_missing_and_crooked_pointers_are_refused(lib):
    c, p, z = _config(), C.c_void_p(4096), C.c_size_t(0)
    call = lambda q, g, o, st: lib.lact_linear_attention_fwd(C.byref(c), q, p, p, g, None, None, None, o, None, z, st, None)
    assert call(None, p, p, p) == -1 and call(p, None, p, p) == -1 and call(p, p, None, p) == -1 and call(p, p, p, None) == -1
    assert call(C.c_void_p(4098), p, p, p) == -2 and call(p, p, C.c_void_p(4104), p) == -2
    assert lib.lact_linear_attention_step(C.byref(c), p, p, p, p, p, p, p, None) == -2            # more than one token
    c = _config(tokens=1)
    assert lib.lact_linear_attention_step(C.byref(c), p, p, p, p, None, p, p, None) == -1


def test_crooked_states_are_refused(lib):
    c, p, bad, z = _config(), C.c_void_p(4096), C.c_void_p(4104), C.c_size_t(0)
    for s_in, s_out in ((bad, None), (None, bad)):
        assert lib.lact_linear_attention_fwd(C.byref(c), p, p, p, p, None, s_in, s_out, p, None, z, p, None) == -2
    for s_in, d_out, d_in in ((bad, None, None), (None, bad, None), (None, None, bad)):
        assert lib.lact_linear_attention_bwd(C.byref(c), p, p, p, p, None, s_in, None, z, p, d_out, p, p, p, d_in, None, z, p, None) == -2
    c = _config(tokens=1)
    for s_in, s_out in ((bad, p), (p, bad)):
        assert lib.lact_linear_attention_step(C.byref(c), p, p, p, p, s_in, s_out, p, None) == -2


def _args(h=4, hk=2, dk=64, dv=128, l=5, b=2):
    return (torch.zeros(b, l, h, dk, dtype=BF16), torch.zeros(b, l, hk, dk, dtype=BF16), torch.zeros(b, l, hk, dv, dtype=BF16),
            torch.zeros(h))


def test_python_checks():
    from lact_b200 import layer_ops as lo
    q, k, v, g = _args()
    bad = [((q.float(), k, v, g), TypeError), ((q[:, :, :3], k, v, g[:3]), ValueError), ((q, k, v[..., :96], g), ValueError),
           ((q, k[:, :4], v, g), ValueError), ((q, k, v, g[:2]), ValueError), ((q, k, v, g.double()), ValueError),
           ((q[0], k, v, g), ValueError), ((q, k[:, :, :0], v[:, :, :0], g), ValueError), ((q, k, v, g), ValueError)]  # (the last: no CUDA)
    for args, kind in bad:
        with pytest.raises(kind):
            lo.linear_attention(*args)
        if args[0].dim() == 4:
            with pytest.raises(kind):
                lo.linear_attention_step(*(t[:, 0] for t in args[:3]), args[3], torch.zeros(2, 4, 64, 128))


def test_oracle_against_the_quadratic_form_and_differences():
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    q, k, v, S0 = rn(2, 9, 4, 3), rn(2, 9, 2, 3), rn(2, 9, 2, 5), rn(2, 4, 3, 5)
    decay = -torch.rand(4, generator=g, dtype=torch.float64)
    o, last = orc.linear_attention(q, k, v, decay, 0.7, S0)
    i = torch.arange(9.0, dtype=torch.float64)
    W = torch.exp(decay[:, None, None] * (i[:, None] - i)) * (i[:, None] >= i)
    kk, vv = k.repeat_interleave(2, 2), v.repeat_interleave(2, 2)
    want = torch.einsum("bihd,bjhd,hij,bjhe->bihe", q, kk, W, vv)
    want += torch.einsum("bihd,hi,bhde->bihe", q, torch.exp(decay[:, None] * (i + 1)), S0)
    assert torch.allclose(o, 0.7 * want, rtol=1e-12, atol=1e-12)
    assert torch.autograd.gradcheck(lambda *a: orc.linear_attention(*a[:3], decay, 0.7, a[3]),
                                    [t.requires_grad_() for t in (q, k, v, S0)])
