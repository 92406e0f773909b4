"""Rotary positions with several axes against the formula in 64 bits (oracle.rotary_axes): outputs and gradients.

Tolerances.  h is half a step of the result's type (bf16 2^-8, fp32 2^-24).  An angle in turns is good to half a step of fp32 at a size
of 1/2 (2^-26 turns, 2^-23.3 radians) and 2^-52 of the turns themselves (positions below 2^31: 2^-21 turns, 2^-18.3; below 2^20: nothing);
cosine and sine to 2^-20.9 with the approximations that bf16 results take (their argument, too, rounded: 2^-23 at pi), to 2^-23 with the
functions of fp32.  Each result is two products and a sum: |error| <= h |y| + e (|x| + |y|) of its pair, with e = 2^-20 (bf16) and
2^-21.5 (fp32, the three roundings' 2^-24 included); far positions add 2^-18."""
import pytest
import torch

from oracle import lact_oracle as orc

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
HALF, ANGLE = {BF16: 2.0 ** -8, F32: 2.0 ** -24}, {BF16: 2.0 ** -20, F32: 2.0 ** -21.5}


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


def _near(got, want, x, P, interleaved, dtype, far=0.0):
    """`x`: what was turned; a pair's size bounds the error of both its values."""
    v = x.double().abs()
    size = v.clone()
    a, b = (v[..., 0:2 * P:2], v[..., 1:2 * P:2]) if interleaved else (v[..., :P], v[..., P:2 * P])
    both = a + b
    if interleaved:
        size[..., 0:2 * P:2], size[..., 1:2 * P:2] = both, both
    else:
        size[..., :P], size[..., P:2 * P] = both, both
    size[..., 2 * P:] = 0
    err = (got.double() - want).abs()
    over = err - HALF[dtype] * want.abs() - (ANGLE[dtype] + far) * size
    over[..., 2 * P:] = err[..., 2 * P:]
    assert got.dtype == dtype and got.is_contiguous() and float(over.max()) <= 0.0, float(over.max())


def _check(lo, q, k, pos, sections, interleaved, far=0.0, base=10000.0):
    f = lo.rotary_frequencies(sections, base, device="cuda")
    P = sum(sections)
    leaves = [t.detach().requires_grad_() for t in (q, k) if t is not None]
    outs = lo.rotary_axes(leaves[0], leaves[1] if k is not None else None, pos, f, sections, interleaved)
    assert (outs[1] is None) == (k is None)
    outs = [t for t in outs if t is not None]
    dys = [_rn(*t.shape, seed=7).to(t.dtype) for t in outs]
    grads = torch.autograd.grad(outs, leaves, dys)
    for x, y, dy, dx in zip(leaves, outs, dys, grads):
        want = orc.rotary_axes(x.detach(), pos, f, sections, interleaved)
        _near(y.detach(), want, x.detach(), P, interleaved, x.dtype, far)
        ref = x.detach().double().requires_grad_()
        rd = torch.autograd.grad(orc.rotary_axes(ref, pos, f, sections, interleaved), ref, dy.double())[0]
        _near(dx, rd, dy, P, interleaved, x.dtype, far)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,sections", [(64, (32,)), (128, (22, 21, 21)), (64, (11, 13)), (128, (8,)), (6, (1, 2)), (2, (1,)), (10, (3,)), (96, (0, 20, 0, 4)), (512, (100, 100, 56)),
                                        (36, (5, 1, 1, 1, 1, 1, 1, 1))])
def test_sections(lo, dtype, interleaved, d, sections):
    q, k = _rn(2, 37, 5, d).to(dtype), _rn(2, 37, 3, d, seed=1).to(dtype)
    pos = torch.randint(-50, 4000, (37, len(sections)), device="cuda", dtype=torch.int32)
    _check(lo, q, k, pos, list(sections), interleaved)


@pytest.mark.parametrize("b,l,h,hk", [(1, 1, 1, 1), (1, 1, 64, 1), (3, 1, 7, 7), (1, 2049, 1, 0), (2, 700, 12, 12), (1, 5000, 3, 2), (40, 9, 16, 2)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sizes(lo, b, l, h, hk, dtype):
    q, k = _rn(b, l, h, 64).to(dtype), _rn(b, l, hk, 64, seed=1).to(dtype) if hk else None
    pos = torch.arange(l, device="cuda")[:, None]
    _check(lo, q, k, pos, [32], False)
    own = torch.randint(0, 9999, (b, l, 1), device="cuda")      # positions of each entry, int64
    _check(lo, q, k, own, [32], True)
    _check(lo, q, k, own[:1].int(), [16], True)


@pytest.mark.parametrize("n", [1, 33, 4000])
def test_new_tokens(lo, n):
    q, k = _rn(n, 12, 128).to(BF16), _rn(n, 4, 128, seed=1).to(BF16)
    pos = torch.randint(0, 131072, (n, 2), device="cuda", dtype=torch.int32)
    _check(lo, q, k, pos, [40, 24], False)
    wide = pos.long().repeat(1, 3)[:, ::3]                      # positions with strides of their own
    assert torch.equal(wide[:, 0], pos[:, 0].long())
    _check(lo, q, k, wide, [40, 24], False)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_far_positions(lo, dtype):
    q = _rn(1, 64, 4, 64).to(dtype)
    pos = torch.randint(0, 1 << 20, (64, 1), device="cuda", dtype=torch.int32)
    _check(lo, q, None, pos, [32], False)
    ends = torch.tensor([0, -1, 2 ** 31 - 1, -2 ** 31], device="cuda").repeat(16)[:, None]
    _check(lo, q, None, ends.int(), [32], False, far=2.0 ** -18)


def _layouts(x):
    b, l, h, d = x.shape
    yield x.transpose(1, 2).contiguous().transpose(1, 2)
    fused = torch.zeros(b, l, h * d + 8, device="cuda", dtype=x.dtype)
    fused[..., 8:] = x.reshape(b, l, h * d)
    yield fused[..., 8:].reshape(b, l, h, d)
    odd = torch.zeros(b, l, h, d + 1, device="cuda", dtype=x.dtype)
    odd[..., 1:] = x
    yield odd[..., 1:]                                          # rows off every boundary
    yield x.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)   # features apart
    yield x[:, :1].expand(b, l, h, d)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts(lo, dtype, interleaved):
    f, pos = lo.rotary_frequencies([20, 12], device="cuda"), torch.randint(0, 999, (2, 19, 2), device="cuda")
    for q, k in zip(_layouts(_rn(2, 19, 4, 64).to(dtype)), _layouts(_rn(2, 19, 2, 64, seed=1).to(dtype))):
        got = lo.rotary_axes(q, k, pos, f, [20, 12], interleaved)
        want = lo.rotary_axes(q.clone(memory_format=torch.contiguous_format), k.clone(memory_format=torch.contiguous_format), pos, f, [20, 12], interleaved)
        assert all(torch.equal(a, w) for a, w in zip(got, want))


def test_what_is_not_turned_is_copied_and_stays_apart(lo):
    x = _rn(1, 9, 3, 64).to(BF16)
    x[..., 40], x[0, 2, 1, 63], x[0, 4, 0, 3] = float("nan"), float("inf"), float("-inf")
    f, pos = lo.rotary_frequencies([16], device="cuda"), torch.arange(9, device="cuda")[:, None]
    y, _ = lo.rotary_axes(x, None, pos, f, [16])
    assert bool(y[..., 40].isnan().all()) and torch.equal(y[..., 41:], x[..., 41:]) and torch.equal(y[..., 32:40], x[..., 32:40])
    spoiled = torch.zeros_like(x, dtype=torch.bool)
    spoiled[..., 40] = spoiled[0, 2, 1, 63] = True
    spoiled[0, 4, 0, 3] = spoiled[0, 4, 0, 19] = True
    assert bool(y.isfinite()[~spoiled].all()) and not bool(y.isfinite()[spoiled].any())


def test_frequencies_of_every_size(lo):
    """Several turns a position, backwards, none; what is not finite makes its own pairs NaN."""
    f = torch.tensor([0.0, -0.3, 7.0, -100.25, 1e6, 3.141592653589793, 1e-12, 2.5e9], device="cuda", dtype=torch.float64)
    x, pos = _rn(1, 30, 2, 16), torch.randint(-9, 9, (30, 1), device="cuda")
    for interleaved in (False, True):
        y, _ = lo.rotary_axes(x, None, pos, f, [8], interleaved)
        # (the formula's own angle, in 64 bits, is off by half a step of 2.25e10: 2^-19)
        _near(y, orc.rotary_axes(x, pos, f, [8], interleaved), x, 8, interleaved, torch.float32, far=2.0 ** -18)
    bad = f.clone()
    bad[2], bad[5] = float("inf"), float("nan")
    y, _ = lo.rotary_axes(x, None, pos, bad, [8])
    lost = torch.zeros(16, dtype=torch.bool, device="cuda")
    lost[[2, 5, 10, 13]] = True
    assert torch.equal(y.isnan(), lost.expand_as(y))


@pytest.mark.parametrize("h,hk,d", [(96, 12, 128), (40, 0, 96), (24, 24, 512), (7, 1, 6)])
def test_many_heads(lo, h, hk, d):
    q, k = _rn(2, 33, h, d).to(BF16), _rn(2, 33, hk, d, seed=1).to(BF16) if hk else None
    _check(lo, q, k, torch.randint(0, 999, (33, 1), device="cuda"), [d // 2], True)
    _check(lo, q, k, torch.randint(0, 999, (33, 1), device="cuda"), [d // 2 - 1], False)


def test_shared_keys_get_the_sum_of_their_gradients(lo):
    """Keys broadcast over heads and entries: the gradient of the one they come from."""
    f, pos = lo.rotary_frequencies([32], device="cuda"), torch.arange(7, device="cuda")[:, None]
    k, dy = _rn(1, 7, 1, 64).requires_grad_(), _rn(3, 7, 4, 64, seed=2)
    y, _ = lo.rotary_axes(k.expand(3, 7, 4, 64), None, pos, f, [32])
    dk, = torch.autograd.grad(y, k, dy)
    ref = k.detach().double().requires_grad_()
    want, = torch.autograd.grad(orc.rotary_axes(ref.expand(3, 7, 4, 64), pos, f, [32]), ref, dy.double())
    # (twelve terms, each off by 2^-21.5 of its pair's size and rounded, and eleven sums in fp32)
    size = (dy.abs().sum((0, 2), keepdim=True).double() * 2).reshape(1, 7, 1, 64)
    size = size + size.roll(32, -1)
    assert bool(((dk.double() - want).abs() <= 2.0 ** -20 * size).all())


def test_more_than_2_to_31_elements(lo):
    """Every batch entry holds the same values and has to give the same bits as the first."""
    if torch.cuda.get_device_properties(0).total_memory < 100e9:
        pytest.skip("needs 100 GB")
    b, l, h, hk, d = 9, 30001, 64, 2, 128
    one = [_rn(1, l, n, d, seed=i).to(BF16) for i, n in enumerate((h, hk))]
    f, pos = lo.rotary_frequencies([64], device="cuda"), torch.arange(l, device="cuda")[:, None]
    q, k = (t.expand(b, -1, -1, -1).contiguous() for t in one)
    assert q.numel() > 2 ** 31
    y, z = lo.rotary_axes(q, k, pos, f, [64])
    want = lo.rotary_axes(*one, pos, f, [64])
    assert all(torch.equal(y[i], want[0][0]) and torch.equal(z[i], want[1][0]) for i in range(b))
    del y, z
    y, _ = lo.rotary_axes(q.view(1, b * l, h, d), None, pos.repeat(b, 1), f, [64])
    assert all(torch.equal(y[0, i * l:(i + 1) * l], want[0][0]) for i in range(b))


def test_gradients_against_differences(lo):
    """Linear: a difference over a step of any size is the derivative, up to the roundings of its two outputs (2^-24 of each, over the step)."""
    q, f = _rn(1, 5, 2, 16), lo.rotary_frequencies([5, 3], device="cuda")
    pos, dy = torch.randint(0, 50, (5, 2), device="cuda"), _rn(1, 5, 2, 16, seed=3)
    leaf = q.clone().requires_grad_()
    dq = torch.autograd.grad(lo.rotary_axes(leaf, None, pos, f, [5, 3])[0], leaf, dy)[0]
    for i in range(0, q.numel(), 7):
        e = torch.zeros_like(q)
        e.view(-1)[i] = 1.0
        up, down = (lo.rotary_axes(q + s * e, None, pos, f, [5, 3])[0] for s in (1.0, -1.0))
        diff = float(((up.double() - down.double()) / 2 * dy.double()).sum())
        size = float(((up.abs() + down.abs()) * dy.abs()).double().sum())
        assert abs(diff - float(dq.view(-1)[i])) <= 2.0 ** -21 * size


def test_one_gradient_and_the_gradient_of_a_gradient(lo):
    q, k = _rn(1, 6, 2, 64).to(BF16).requires_grad_(), _rn(1, 6, 1, 64).to(BF16)
    f, pos = lo.rotary_frequencies([32], device="cuda"), torch.arange(6, device="cuda")[:, None]
    yq, yk = lo.rotary_axes(q, k, pos, f, [32])
    w = _rn(1, 6, 2, 64, seed=2).to(BF16).requires_grad_()
    dq, = torch.autograd.grad(yq, q, w, create_graph=True)
    ddw, = torch.autograd.grad(dq, w, q.detach())               # the gradient by w of <dq, q> is the turned q
    assert torch.equal(ddw, yq.detach())
    k2 = k.detach().requires_grad_()
    yq, yk = lo.rotary_axes(q.detach(), k2, pos, f, [32])
    dk, = torch.autograd.grad(yk.float().sum(), k2)
    assert dk.shape == k2.shape and bool(dk.isfinite().all())
    q1, k1 = q.detach().requires_grad_(), k.detach().requires_grad_()
    yq, yk = lo.rotary_axes(q1, k1, pos, f, [32])
    dq1, dk1 = torch.autograd.grad(yk.float().sum(), (q1, k1), allow_unused=True)
    assert dq1 is None and torch.equal(dk1, dk)


def test_empty_and_changed(lo):
    f = lo.rotary_frequencies([32], device="cuda")
    y, z = lo.rotary_axes(torch.zeros(0, 4, 64, device="cuda"), torch.zeros(0, 2, 64, device="cuda"), torch.zeros(0, 1, device="cuda", dtype=torch.int32), f, [32])
    assert y.shape == (0, 4, 64) and z.shape == (0, 2, 64)
    q, pos = _rn(1, 6, 2, 64).requires_grad_(), torch.arange(6, device="cuda")[:, None]
    y = lo.rotary_axes(q, None, pos, f, [32])[0]
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_captured_training_step(lo):
    f, pos = lo.rotary_frequencies([22, 21, 21], device="cuda"), torch.randint(0, 99, (300, 3), device="cuda")
    data = [_rn(1, 300, 6, 128, seed=s).to(BF16) for s in range(4)]
    q, k, dy = (t.clone() for t in data[:3])

    def step():
        a, b = q.detach().requires_grad_(), k.detach().requires_grad_()
        y, z = lo.rotary_axes(a, b, pos, f, [22, 21, 21], True)
        return [y.detach(), z.detach(), *torch.autograd.grad((y, z), (a, b), (dy, dy))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for s in (1, 2, 3):
        q.copy_(data[s])
        pos.add_(17)
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_a_compiled_call(lo):
    f, pos = lo.rotary_frequencies([32], device="cuda"), torch.arange(40, device="cuda")[:, None]
    q, k = _rn(2, 40, 4, 64).to(BF16), _rn(2, 40, 2, 64).to(BF16)

    @torch.compile(fullgraph=True, backend="aot_eager")
    def call(q, k):
        a, b = lo.rotary_axes(q, k, pos, f, [32])
        return (a * 2).float().sum() + b.float().sum()
    a, b = (t.clone().requires_grad_() for t in (q, k))
    got = torch.autograd.grad(call(a, b), (a, b))
    y, z = lo.rotary_axes(a, b, pos, f, [32])
    want = torch.autograd.grad((y * 2).float().sum() + z.float().sum(), (a, b))
    assert all(torch.equal(g, w) for g, w in zip(got, want))
