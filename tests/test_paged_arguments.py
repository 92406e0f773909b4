"""Rotary positions and the paged cache: what the entry points refuse, on the host; versions of what is written; the oracles against
other ways to the same numbers."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as fw

from oracle import lact_oracle as orc

BF16, F32, E4M3, I32 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int32


class _Rotary(C.Structure):
    _fields_ = [(n, C.c_int64) for n in ("batch", "tokens", "q_heads", "k_heads", "head_dim", "q_bs", "q_ts", "q_hs", "k_bs", "k_ts", "k_hs",
                                         "position_bs", "position_ts", "position_as")] + [("sections", C.c_int64 * 8)] + [
        (n, C.c_int32) for n in ("axes", "position_bytes", "dtype", "interleaved", "backwards")]


class _Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "k_exponent", "v_exponent")] + [
        (n, C.c_int64) for n in ("pages", "kv_heads", "page_size", "head_dim", "k_page_stride", "v_page_stride", "ke_page_stride", "ve_page_stride")] + [
        ("page_table", C.c_void_p), ("table_cols", C.c_int64), ("table_stride", C.c_int64), ("lengths", C.c_void_p), ("sequences", C.c_int64)]


def _rotary(**over):
    c = dict(batch=2, tokens=5, q_heads=4, k_heads=2, head_dim=64, q_bs=1280, q_ts=256, q_hs=64, k_bs=640, k_ts=128, k_hs=64, position_bs=0, position_ts=2,
             position_as=1, sections=(20, 12), axes=2, position_bytes=4, dtype=1, interleaved=0, backwards=0)
    c.update(over)
    c["sections"] = (C.c_int64 * 8)(*c["sections"])
    return _Rotary(**c)


def _cache(**over):
    page = 2 * 16 * 64
    c = dict(k=4096, v=8192, k_exponent=None, v_exponent=None, pages=3, kv_heads=2, page_size=16, head_dim=64, k_page_stride=page, v_page_stride=page,
             ke_page_stride=32, ve_page_stride=32, page_table=4096, table_cols=4, table_stride=4, lengths=4096, sequences=2)
    c.update(over)
    return _Cache(**c)


@pytest.fixture(scope="module")
def lib():
    from lact_b200 import build
    build.build()
    from lact_b200 import _lib
    return _lib.lib()


P = C.c_void_p(4096)


@pytest.mark.parametrize("over,code", [
    (dict(batch=0), -2), (dict(tokens=0), -2), (dict(q_heads=0), -2), (dict(k_heads=-1), -2), (dict(head_dim=63), -2), (dict(head_dim=514), -2), (dict(dtype=2), -3),
    (dict(position_bytes=2), -3), (dict(axes=0), -2), (dict(axes=9), -2), (dict(sections=(20, 13)), -2), (dict(sections=(0, 0)), -2), (dict(sections=(-1, 3)), -2),
    (dict(sections=(1 << 62, 1 << 62)), -2), (dict(tokens=1 << 31), -2)])
def test_bad_rotary_configurations_are_refused(lib, over, code):
    assert lib.lact_rotary_axes(C.byref(_rotary(**over)), P, P, P, P, P, P, None) == code


def test_missing_rotary_pointers_are_refused(lib):
    for hole in range(6):
        args = [None if i == hole else P for i in range(6)]
        assert lib.lact_rotary_axes(C.byref(_rotary()), *args, None) == -1
    assert lib.lact_rotary_axes(C.byref(_rotary(k_heads=0)), P, None, P, P, P, None, None) in (-7, -8)   # (no device here)
    assert lib.lact_rotary_axes(None, P, P, P, P, P, P, None) == -1


def _step(lib, c, q=P, q_bs=256, q_hs=64, heads=4, window=0, scale=0.1, o=P, room=P, nbytes=1 << 30, status=P):
    return lib.lact_paged_attention_step(C.byref(c), q, C.c_int64(q_bs), C.c_int64(q_hs), C.c_int64(heads), C.c_int64(window), C.c_float(scale), o, room,
                                         C.c_size_t(nbytes), status, None)


def _write(lib, c, k=P, v=P, strides=(128, 640, 64, 128, 640, 64), batch=2, tokens=5, cu=None):
    s = [C.c_int64(x) for x in strides]
    return lib.lact_paged_cache_write(C.byref(c), k, *s[:3], v, *s[3:], C.c_int64(batch), C.c_int64(tokens), cu, None)


def _read(lib, c, out=P, batch=2, tokens=5, cu=None):
    return lib.lact_paged_cache_read(C.byref(c), out, C.c_int64(batch), C.c_int64(tokens), cu, None)


@pytest.mark.parametrize("over,code", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(page_table=None), -1), (dict(lengths=None), -1), (dict(k_exponent=4096), -5), (dict(head_dim=96), -2),
    (dict(page_size=8), -2), (dict(page_size=24), -2), (dict(page_size=512), -2), (dict(pages=0), -2), (dict(pages=1 << 31), -2), (dict(kv_heads=0), -2),
    (dict(sequences=0), -2), (dict(table_cols=0), -2), (dict(table_cols=(1 << 26) + 1), -2), (dict(k=4112), -2), (dict(k_page_stride=2047), -2),
    (dict(v_page_stride=2056), -2), (dict(k_exponent=4096, v_exponent=4096, ke_page_stride=31), -2),
    (dict(k_exponent=4096, v_exponent=4100), -2), (dict(k_exponent=4096, v_exponent=4096, ve_page_stride=40), -2)])
def test_bad_caches_are_refused(lib, over, code):
    c = _cache(**over)
    n = C.c_size_t(0)
    assert lib.lact_paged_attention_step_bytes(C.byref(c), C.c_int64(4), C.c_int64(0), C.byref(n)) == code
    assert _step(lib, c) == code and _write(lib, c) == code and _read(lib, c) == code


def test_bad_calls_on_a_cache_are_refused(lib):
    c = _cache()
    n = C.c_size_t(0)
    size = lambda heads=4, window=0, c=c: (lib.lact_paged_attention_step_bytes(C.byref(c), C.c_int64(heads), C.c_int64(window), C.byref(n)), n.value)
    assert size() == (0, 0)                                     # 64 positions: a CTA a unit, no pieces
    rc, nbytes = size(c=_cache(table_cols=4096))
    assert rc == 0 and nbytes > 0
    assert size(window=2 ** 63 - 1, c=_cache(table_cols=4096)) == (0, nbytes)   # (as no window)
    assert size(heads=3)[0] == -2 and size(heads=0)[0] == -2 and size(window=-1)[0] == -2
    for over, code in [(dict(q=None), -1), (dict(o=None), -1), (dict(status=None), -1), (dict(o=C.c_void_p(4104)), -2), (dict(q=C.c_void_p(4104)), -2), (dict(q_bs=257), -2), (dict(q_hs=68), -2), (dict(heads=5), -2),
                       (dict(scale=float("nan")), -5), (dict(scale=float("inf")), -5)]:
        assert _step(lib, c, **over) == code
    for over in (dict(room=None), dict(nbytes=nbytes - 1), dict(room=C.c_void_p(4100))):
        assert _step(lib, _cache(table_cols=4096), **over) == -4
    for over, code in [(dict(k=None), -1), (dict(v=None), -1), (dict(v=C.c_void_p(4104)), -2), (dict(strides=(128, 640, 63, 128, 640, 64)), -2),
                       (dict(strides=(128, 640, 64, 129, 640, 64)), -2), (dict(batch=3), -5), (dict(batch=2, cu=P), -5), (dict(tokens=0), -2)]:
        assert _write(lib, c, **over) == code
    for over, code in [(dict(out=None), -1), (dict(out=C.c_void_p(4112)), -2), (dict(batch=1), -5), (dict(tokens=0), -2)]:
        assert _read(lib, c, **over) == code


def test_python_checks_of_rotary_axes():
    from lact_b200 import layer_ops as lo
    q, k, p, f = torch.zeros(2, 5, 4, 64), torch.zeros(2, 5, 2, 64), torch.zeros(5, 2, dtype=I32), lo.rotary_frequencies([20, 12])
    call = lambda q=q, k=k, p=p, f=f, s=(20, 12): lo.rotary_axes(q, k, p, f, s)
    for kind, over in [(ValueError, dict(q=q[0, 0])), (TypeError, dict(q=q.double())), (TypeError, dict(q=q.half())), (TypeError, dict(k=k.to(BF16))),
                       (ValueError, dict(k=k[:, :4])), (ValueError, dict(k=k[..., :32])), (ValueError, dict(k=k[0])), (ValueError, dict(k=k[:, :, :0])),
                       (ValueError, dict(q=q[..., :63], k=None)), (TypeError, dict(p=p.float())), (ValueError, dict(p=p[:4])), (ValueError, dict(p=p[:, :1])),
                       (ValueError, dict(p=p.expand(3, 5, 2))), (TypeError, dict(f=f.float())), (ValueError, dict(f=f[:-1])), (ValueError, dict(s=(20, 13))),
                       (ValueError, dict(s=())), (ValueError, dict(s=[4] * 9)), (ValueError, dict(s=(33, -1))), (ValueError, {})]:   # (the last: no CUDA)
        with pytest.raises(kind):
            call(**over)


def test_python_checks_of_the_cache():
    from lact_b200 import layer_ops as lo
    c, c8 = lo.paged_cache(3, 16, 2, 64), lo.paged_cache(3, 16, 2, 64, E4M3)
    assert c.k_exponent is None and c8.k.dtype == E4M3 and c8.v_exponent.shape == (3, 2, 16)
    with pytest.raises(TypeError):
        lo.paged_cache(3, 16, 2, 64, torch.float16)
    t, n = torch.zeros(2, 4, dtype=I32), torch.zeros(2, dtype=I32)
    q, x = torch.zeros(2, 4, 64, dtype=BF16), torch.zeros(2, 5, 2, 64, dtype=BF16)
    step = lambda c=c, q=q, t=t, n=n, **kw: lo.paged_attention_step(q, c, t, n, **kw)
    write = lambda c=c, k=x, v=x, t=t, n=n, cu=None: lo.paged_cache_write(c, k, v, t, n, cu)
    read = lambda c=c, t=t, n=n, tokens=5, cu=None: lo.paged_cache_read(c, t, n, tokens, cu)
    wide = lo.paged_cache(3, 16, 4, 64)
    bad_caches = [(TypeError, c._replace(k=c.k.float(), v=c.v.float())), (TypeError, c8._replace(k=c.k, v=c.v)), (TypeError, c8._replace(k_exponent=None, v_exponent=None)),
                  (ValueError, c8._replace(k_exponent=None)), (TypeError, c8._replace(k_exponent=c8.k_exponent.int())), (ValueError, c8._replace(v_exponent=c8.v_exponent[:2])),
                  (ValueError, c._replace(v=c.v[:2])), (ValueError, c._replace(k=c.k[..., :32], v=c.v[..., :32])), (ValueError, c._replace(k=c.k[:, :, :8], v=c.v[:, :, :8])),
                  (ValueError, c._replace(k=c.k.transpose(1, 2).contiguous().transpose(1, 2))), (ValueError, c._replace(v=wide.v[:, ::2])),
                  (ValueError, lo.PagedCache(c.k[:0], c.v[:0]))]
    for kind, bad in bad_caches:
        for call in (step, write, read):
            with pytest.raises(kind):
                call(c=bad)
    for kind, over in [(TypeError, dict(t=t.float())), (TypeError, dict(n=n.float())), (ValueError, dict(t=t[0])), (ValueError, dict(n=n[:1])), (ValueError, dict(t=t[:, :0])),
                       (ValueError, {})]:   # (the last: no CUDA)
        for call in (step, write, read):
            with pytest.raises(kind):
                call(**over)
    for kind, over in [(ValueError, dict(q=q[0])), (TypeError, dict(q=q.float())), (ValueError, dict(q=q[:1])), (ValueError, dict(q=q[:, :3])), (ValueError, dict(q=q[..., :32])),
                       (ValueError, dict(window_size=-3)), (ValueError, dict(softmax_scale=float("nan"))), (ValueError, dict(softmax_scale=float("inf")))]:
        with pytest.raises(kind):
            step(**over)
    cu = torch.tensor([0, 2, 5], dtype=I32)
    for kind, over in [(ValueError, dict(k=x[0], v=x[0])), (TypeError, dict(k=x.float(), v=x.float())), (ValueError, dict(v=x[:, :4])), (ValueError, dict(k=x[:, :, :1], v=x[:, :, :1])),
                       (ValueError, dict(k=x[:1], v=x[:1])), (ValueError, dict(cu=cu)), (ValueError, dict(k=x[:1], v=x[:1], cu=cu[:2])), (TypeError, dict(k=x[:1], v=x[:1], cu=cu.float()))]:
        with pytest.raises(kind):
            write(**over)
    for kind, over in [(ValueError, dict(tokens=-1)), (ValueError, dict(cu=cu[:2])), (TypeError, dict(cu=cu.float()))]:
        with pytest.raises(kind):
            read(**over)


def _meta(*s, dtype=BF16):
    return torch.empty(*s, dtype=dtype, device="meta")


def _meta_args():
    cache = [_meta(3, 2, 16, 64, dtype=E4M3), _meta(3, 2, 16, 64, dtype=E4M3), _meta(3, 2, 16, dtype=torch.uint8), _meta(3, 2, 16, dtype=torch.uint8)]
    table, lengths = _meta(2, 4, dtype=I32), _meta(2, dtype=I32)
    return {"paged_cache_write": cache + [_meta(2, 5, 2, 64), _meta(2, 5, 2, 64), table, lengths, None], "paged_cache_read": cache + [table, lengths, 5, None],
            "paged_attention_step": [_meta(2, 4, 64)] + cache + [table, lengths, 0, 0.1],
            "rotary_axes": [_meta(2, 5, 4, 64), _meta(2, 5, 2, 64), _meta(5, 1, dtype=I32), _meta(32, dtype=torch.float64), [32], False]}


@pytest.fixture(scope="module")
def ops(lib):
    from lact_b200 import _lib
    _lib.load_ops()
    return torch.ops.lact_b200


@pytest.mark.parametrize("name", sorted(_meta_args()))
def test_shapes_tangents_and_gradients(ops, name):
    op = getattr(ops, name)
    out = op(*_meta_args()[name])
    shapes = {"paged_cache_write": None, "paged_cache_read": (4, 5, 2, 64), "paged_attention_step": (2, 4, 64)}
    assert out is None if name == "paged_cache_write" else name == "rotary_axes" or out.shape == shapes[name]
    for i, a in enumerate(_meta_args()[name]):
        if not isinstance(a, torch.Tensor) or a.dtype not in (BF16, torch.float64):
            continue
        for mode in (torch.enable_grad, torch.no_grad):
            args = _meta_args()[name]
            with mode(), fw.dual_level():
                args[i] = fw.make_dual(args[i], torch.empty_like(args[i]))
                with pytest.raises(NotImplementedError):
                    op(*args)
        args = _meta_args()[name]
        args[i].requires_grad_()
        if name == "rotary_axes" and a.dtype == BF16:
            assert any(t.requires_grad for t in op(*args))
            continue
        with pytest.raises(NotImplementedError):
            op(*args)
        with torch.no_grad():
            op(*args)


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
def test_what_is_written_gets_a_new_version(ops, mode):
    args = _meta_args()["paged_cache_write"]
    with mode():
        ops.paged_cache_write(*args)
        ops.paged_cache_read(*args[:4], *args[6:8], 5, None)
    assert [t._version for t in args[:8]] == [1, 1, 1, 1, 0, 0, 0, 0]


def test_a_backward_that_has_saved_the_cache_raises(ops):
    cache = [_meta(3, 2, 16, 64), _meta(3, 2, 16, 64), None, None]
    x = _meta(3, 2, 16, 64).requires_grad_()
    loss = (x * cache[0]).sum()
    ops.paged_cache_write(*cache, *_meta_args()["paged_cache_write"][4:])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---------------------------------------------------------------------------------------------- the oracles
def test_frequencies():
    from lact_b200 import layer_ops as lo
    f = lo.rotary_frequencies([22, 21, 21])
    assert f.dtype == torch.float64 and f.shape == (64,) and f[0] == f[22] == f[43] == 1.0
    assert torch.allclose(f[:22], 10000.0 ** (-torch.arange(0, 44, 2).double() / 44))
    assert torch.allclose(lo.rotary_frequencies([16, 24, 24], 5e5, shared=True), 5e5 ** (-torch.arange(0, 128, 2).double() / 128))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_oracle(interleaved):
    g = torch.Generator().manual_seed(0)
    x, f = torch.randn(2, 3, 2, 12, generator=g, dtype=torch.float64), torch.rand(5, generator=g, dtype=torch.float64)
    p = torch.randint(-9, 9, (2, 3, 2), generator=g)
    y = orc.rotary_axes(x, p, f, [2, 3], interleaved)
    for j in range(5):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + 5)
        t = (p[..., int(j >= 2)] * f[j])[..., None]
        assert torch.allclose(y[..., a], x[..., a] * torch.cos(t) - x[..., b] * torch.sin(t), rtol=1e-13, atol=1e-13)
        assert torch.allclose(y[..., b], x[..., b] * torch.cos(t) + x[..., a] * torch.sin(t), rtol=1e-13, atol=1e-13)
    assert torch.equal(y[..., 10:], x[..., 10:])
    assert torch.autograd.gradcheck(lambda x: orc.rotary_axes(x, p, f, [2, 3], interleaved), x.requires_grad_())


def test_8_bit_oracle_against_the_types_own_rounding():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(300, 64, generator=g) * torch.exp2(torch.randint(-140, 120, (300, 1), generator=g).float())).to(BF16)
    x[0] = 0
    x[1, 3], x[2, 5] = float("nan"), float("-inf")
    x[3, 0], x[4] = 2.0 ** 127 * 1.9, 2.0 ** -133
    values, byte = orc.rows_in_8_bits(x)
    fine = torch.isfinite(x.float()).all(-1)
    assert bool((byte[~fine] == 255).all()) and bool(values[~fine].isnan().all()) and int((~fine).sum()) == 2
    scaled = x[fine].double() * torch.exp2(127 - byte[fine].double())[:, None]
    top = scaled.abs().amax(-1)
    assert bool((top <= 448)[byte[fine] < 246].all()) and bool((top > 224)[(byte[fine] > 1) & (byte[fine] < 246)].all())
    own = scaled.clamp(-448, 448).float().to(E4M3).double() * torch.exp2(byte[fine].double() - 127)[:, None]
    assert torch.equal(own, values[fine])
    back = values[fine].to(BF16).double()
    assert torch.equal(back[(byte[fine] > 3)], values[fine][byte[fine] > 3])   # (exact in bf16 down to its smallest numbers)


def test_attention_oracle_against_dense():
    g = torch.Generator().manual_seed(2)
    q, k, v = torch.randn(2, 4, 8, generator=g), torch.randn(5, 2, 4, 8, generator=g), torch.randn(5, 2, 4, 8, generator=g)
    table, lengths = torch.tensor([[3, 1, -1], [4, 0, 2]]), torch.tensor([6, 11])
    o, size, score = orc.paged_attention_step(q, k, v, table, lengths, window=5)
    for i, pages in enumerate(([3, 1], [4, 0, 2])):
        kk = torch.cat([k[p] for p in pages], 1)[:, int(lengths[i]) - 5:int(lengths[i])].double().repeat_interleave(2, 0)
        vv = torch.cat([v[p] for p in pages], 1)[:, int(lengths[i]) - 5:int(lengths[i])].double().repeat_interleave(2, 0)
        want = torch.nn.functional.scaled_dot_product_attention(q[i].double()[:, None], kk, vv)[:, 0]
        assert torch.allclose(o[i], want, rtol=1e-12, atol=1e-12)
    assert bool((size >= o.abs() - 1e-12).all()) and bool((score > 0).all())
