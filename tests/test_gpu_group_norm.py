"""Group norm with an activation against the formula in 64 bits (oracle.group_norm): outputs and gradients.

Tolerances.  h is half a step of the result's type (bf16 2^-8, fp32 2^-24).  xhat = (x - mean) / std: mean and squares are sums in fp32 of
at most a few hundred values one after the other and then of such sums, good to 2^-17 of the values' size, so that z = xhat w + b is
good to 2^-16 (|w| (|xhat| + |mean| / std) + |b|); the activation has a slope of at most 1.1 and adds 2^-19.  The gradient's terms are
dz = dy act'(z) with |act''| <= 1/2 and two such sums; with a = 1.1 |dy w| (1 + |mean| / std + |xhat|):
|error of dx| <= h |dx| + 2^-15 (a + mean(a) + |xhat| mean(a |xhat|)) / std.  Weights' gradients: 2^-14 of the sum of absolute terms.
As a whole: h (the end's rounding) + 2^-16 relative to the norm, and 2^-14 for the weights' gradients."""
import pytest
import torch

from oracle import lact_oracle as orc

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


@pytest.fixture(scope="module")
def lo():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lact_b200 import build
    build.build()
    from lact_b200 import layer_ops
    return layer_ops


def _inputs(shape, dtype, seed=0, far=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    C = shape[-1]
    x = (rn(*shape) * (0.5 + rn(C).abs()) + far * rn(C)).to(dtype)
    return x, 1.0 + 0.2 * rn(C), 0.2 * rn(C), rn(*shape).to(dtype)


def _near(got, want, tol, norm, what):
    got = got.double()
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), what
    err = (got - want).abs()
    over = (err - tol).max()
    assert float(over) <= 0.0, (what, float(over))
    assert float(err.norm()) <= norm * float(want.norm()) + 1e-30, (what, float(err.norm() / want.norm()))


def _check(lo, x, w, b, dy, groups, silu, eps=1e-5, grads=True):
    act = "silu" if silu else None
    leaves = [t.detach().clone().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = lo.group_norm(leaves[0], groups, leaves[1], leaves[2], eps, act)
    assert y.dtype == x.dtype and y.is_contiguous()
    h = HALF[x.dtype]
    ref = [t.detach().double().requires_grad_() if t is not None else None for t in (x, w, b)]
    ry = orc.group_norm(ref[0], groups, ref[1], ref[2], eps, silu)
    n, C = x.shape[0], x.shape[-1]
    grouped = lambda t: t.reshape(n, -1, groups, C // groups)
    v = grouped(x.double())
    var, mean = torch.var_mean(v, dim=(1, 3), keepdim=True, correction=0)
    std = torch.sqrt(var + eps)
    one = torch.ones(C, device="cuda", dtype=torch.float64)
    aw = (one if w is None else w.double().abs()).reshape(groups, -1)
    ab = (0 * one if b is None else b.double().abs()).reshape(groups, -1)
    xh, far = ((v - mean) / std).abs(), mean.abs() / std
    tol = h * ry.detach().abs() + (2.0 ** -16 * (aw * (xh + far) + ab)).reshape(x.shape) + 1e-30
    _near(y.detach(), ry.detach(), tol, h + 2.0 ** -16, "y")
    if not grads:
        return
    ins = [t for t in leaves if t is not None]
    got = torch.autograd.grad(y, ins, dy)
    want = torch.autograd.grad(ry, [t for t in ref if t is not None], dy.double())
    a = 1.1 * grouped(dy.double()).abs() * (1 + far + xh)
    aw_ = a * aw
    m = (aw_ + aw_.mean((1, 3), keepdim=True) + xh * (aw_ * xh).mean((1, 3), keepdim=True)) / std
    assert got[0].dtype == x.dtype
    _near(got[0], want[0], h * want[0].abs() + (2.0 ** -15 * m).reshape(x.shape) + 1e-30, h + 2.0 ** -15, "dx")
    rest = [n_ for n_, t in (("dw", w), ("db", b)) if t is not None]
    for name, g_, w_ in zip(rest, got[1:], want[1:]):
        size = (a * (xh if name == "dw" else 1.0)).sum((0, 1)).reshape(C)
        half = HALF[g_.dtype]
        _near(g_, w_, half * w_.abs() + 2.0 ** -14 * size, half + 2.0 ** -14, name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape,groups", [((1, 128), 1), ((7, 1536), 12), ((700, 96), 32), ((65, 60), 12), ((3000, 8), 8), ((33, 40), 8),
                                          ((5, 1536), 1), ((129, 384), 4), ((9, 1000), 5), ((3, 4096), 32), ((4, 5120), 16), ((2, 9000), 3),
                                          ((300, 3), 3), ((20, 1), 1), ((50, 2500), 2)])
def test_one_spot(lo, shape, groups, dtype):
    """Norms per token: groups of whole and of broken vectors, of 2^n and other numbers of them, rows up to more than a block holds."""
    _check(lo, *_inputs(shape, dtype), groups, True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape,groups", [((2, 50, 96), 32), ((1, 2, 8), 2), ((3, 7, 9, 64), 4), ((1, 4099, 20), 4), ((16, 33, 512), 32),
                                          ((2, 5, 3, 8, 24), 24), ((1, 700, 3), 1), ((1, 65, 2500), 5), ((2, 1000, 4096), 1), ((200, 3, 16), 2)])
@pytest.mark.parametrize("silu", [False, True])
def test_many_spots(lo, shape, groups, dtype, silu):
    _check(lo, *_inputs(shape, dtype), groups, silu)


@pytest.mark.parametrize("w,b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("shape", [(40, 64), (2, 40, 64)])
def test_without_weights(lo, shape, w, b):
    x, weight, bias, dy = _inputs(shape, F32)
    _check(lo, x, weight if w else None, bias if b else None, dy, 8, True)


@pytest.mark.parametrize("shape", [(40, 64), (2, 40, 64)])
def test_weights_of_16_bits(lo, shape):
    x, w, b, dy = _inputs(shape, BF16)
    _check(lo, x, w.to(BF16), b.to(BF16), dy, 8, True)


@pytest.mark.parametrize("shape", [(64, 96), (2, 3001, 48)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_means_far_from_zero(lo, shape, dtype):
    """Channel means of hundreds of standard deviations, and a first spot far from all others."""
    x, w, b, dy = _inputs(shape, dtype, far=300.0)
    _check(lo, x, w, b, dy, 8, False)
    x, w, b, dy = _inputs(shape, dtype)
    x[:, :1] = x[:, :1] + 2000.0
    _check(lo, x, w, b, dy, 8, False)


@pytest.mark.parametrize("shape", [(5, 64), (2, 600, 64)])
def test_constant_groups(lo, shape):
    """No variance: the output is the activated bias, gradients are finite; with eps = 0 the division by zero shows as NaN."""
    x, w, b, dy = _inputs(shape, F32)
    x[:] = 3.0
    y = lo.group_norm(x, 8, w, b, 1e-5)
    assert torch.equal(y, b.expand_as(y))
    leaf = x.clone().requires_grad_()
    lo.group_norm(leaf, 8, w, b, 1e-5, "silu").backward(dy)
    assert bool(leaf.grad.isfinite().all())
    assert bool(lo.group_norm(x, 8, w, b, 0.0).isnan().all())


@pytest.mark.parametrize("shape", [(50, 96), (3, 500, 96)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_in_its_group(lo, shape, bad):
    x, w, b, dy = _inputs(shape, BF16)
    want = lo.group_norm(x, 8, w, b, activation="silu")
    y_in = x.clone()
    y_in[1, ..., 40] = bad            # channel 40: group 3 (36 to 47)
    got = lo.group_norm(y_in, 8, w, b, activation="silu")
    keep = torch.ones_like(x, dtype=torch.bool)
    keep[1, ..., 36:48] = False
    assert torch.equal(got[keep], want[keep]) and bool((~got[~keep].isfinite()).any())
    assert bool(got[1, ..., 41].isnan().all())


def test_views_and_foreign_strides(lo):
    g = torch.Generator(device="cuda").manual_seed(3)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    wide = rn(4, 30, 200).to(BF16)
    for x in (wide[..., 8:104], wide[..., 3:99], wide[:, ::2, :96], wide.transpose(0, 1)[..., :96], rn(4 * 30 * 96 + 1)[1:].view(4, 30, 96),
              rn(1, 30, 96).expand(4, 30, 96), rn(4, 96, 30).transpose(1, 2), wide[:, 0, 5:101], rn(4, 6, 5, 96)[:, :, 1:4]):
        want = lo.group_norm(x.contiguous().clone(), 8, activation="silu")
        assert bool(torch.equal(lo.group_norm(x, 8, activation="silu"), want))
        leaf, plain = x.detach().requires_grad_(), x.contiguous().clone().requires_grad_()
        lo.group_norm(leaf, 8, activation="silu").backward(x.detach())
        lo.group_norm(plain, 8, activation="silu").backward(x.contiguous().clone())
        same = torch.equal(leaf.grad, plain.grad)
        assert same


def test_empty(lo):
    w = torch.ones(16, device="cuda", requires_grad=True)
    for shape in ((0, 16), (0, 4, 16), (3, 0, 16)):
        x = torch.zeros(*shape, device="cuda", requires_grad=True)
        y = lo.group_norm(x, 4, w)
        assert y.shape == shape
        w.grad = None
        y.sum().backward()
        assert x.grad.shape == shape and torch.equal(w.grad, torch.zeros_like(w))


def test_more_samples_than_a_grid_axis(lo):
    x, w, b, dy = _inputs((70000, 2, 8), BF16)
    _check(lo, x, w, b, dy, 2, True)


def test_captured_on_a_side_stream_and_again(lo):
    data = [_inputs(s, BF16, seed=i) for i, s in enumerate(((200, 512), (2, 3000, 64)))]
    side = torch.cuda.Stream()

    def go():
        out = []
        for x, w, b, dy in data:
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            y = lo.group_norm(leaves[0], 8, leaves[1], leaves[2], activation="silu")
            out += [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        return out
    want = [t.clone() for t in go()]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(go(), want))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go()
    for _ in range(3):
        for x, w, b, dy in data:
            x.neg_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, go()))


def test_compiled_caller(lo):
    x, w, b, dy = _inputs((2, 40, 64), BF16)
    f = lambda t, w_: lo.group_norm(t * 1.0, 8, w_, b, activation="silu").float().sum()
    grads = []
    for fn in (f, torch.compile(f, fullgraph=True, backend="aot_eager")):
        leaf, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        fn(leaf, wl).backward()
        grads.append((leaf.grad, wl.grad))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


def test_a_layer_of_both(lo):
    """Linear attention and the norm of its heads with the activation, as a layer runs them: forward and gradients against the
    oracle's chain on the same bf16 values between the two."""
    b, l, h, d = 2, 300, 4, 64
    g = torch.Generator(device="cuda").manual_seed(9)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    q, k, v, dy = (rn(b, l, h, d).to(BF16) for _ in range(4))
    decay, w = -0.1 * torch.rand(h, device="cuda", generator=g), 1.0 + 0.1 * rn(h * d)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, w)]
    o, _ = lo.linear_attention(*leaves[:3], decay)
    y = lo.group_norm(o.reshape(b * l, h * d), h, leaves[3], activation="silu")
    got = torch.autograd.grad(y, leaves, dy.reshape(b * l, h * d))
    ref = [t.double().requires_grad_() for t in (q, k, v, w)]
    ro, _ = orc.linear_attention(*ref[:3], decay)
    ry = orc.group_norm(ro.reshape(b * l, h * d), h, ref[3], silu=True)
    want = torch.autograd.grad(ry, ref, dy.reshape(b * l, h * d).double())
    # three roundings of half a step one after the other (weights, o, y), four for the gradients (dy's way back through o)
    assert float((y.detach().double() - ry.detach()).norm()) <= 3 * 2.0 ** -8 * float(ry.detach().norm())
    for a, r in zip(got, want):
        assert float((a.double() - r).norm()) <= 4 * 2.0 ** -8 * float(r.norm())
