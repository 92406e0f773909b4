"""Attention of single tokens over a paged cache against the formula in 64 bits (oracle.paged_attention_step), and with the calls around it.

Tolerances.  With A = sum of w |v| for an output and S the largest scale sum |q k| of its row: a score is a sum of d products in fp32,
each addition good to 2^-23 (tensor cores cut where they do not round), and d / 16 + 4 of them follow one another within one and across
products; with its scaling and the exponential's 2^-22 a weight is off by s = (d / 8 + 16) 2^-23 S + 2^-22 |x| <= (d / 8 + 32) 2^-23 S +
2^-21 of itself, in the numerator and the denominator.  Weights are rounded to two bf16 pieces (2^-16), or to fp16 (2^-11, and 2^-25 of
the largest w 2^e for what is smaller: times the values over their power of two, at most 448, of all n tokens).  Sums over n tokens
are n / 16 products one after the other at most, plus 64 pieces: (n / 16 + 64) 2^-23.  So
  |error| <= 2^-8 |o| + A (2 s + 2^-16 or 2^-11 + (n / 16 + 64) 2^-22) + (8 bits) n 448 2^-25 max(w 2^e)."""
import pytest
import torch

from oracle import lact_oracle as orc

pytestmark = pytest.mark.gpu
BF16, E4M3, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


@pytest.fixture(scope="module")
def lo():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lact_b200 import build
    build.build()
    from lact_b200 import layer_ops
    return layer_ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rn(*s, seed=0):
    return torch.randn(*s, device="cuda", generator=_gen(seed + sum(s)))


def _cache(lo, lengths, size, heads, d, bits, seed=0, spread=0.0):
    """Random keys and values; NaN (8 bits: NaN codes and bytes) in every row that no sequence has."""
    need = [-(-max(n, 0) // size) for n in lengths]
    pages = sum(need) + 4
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:sum(need)].tolist()
    table = torch.full((len(lengths), max(need + [0]) + 1), -1)
    used = torch.zeros(pages, size, dtype=torch.bool)
    for i, n in enumerate(need):
        for j in range(n):
            table[i, j] = order.pop()
            used[table[i, j], :min(size, lengths[i] - j * size)] = True
    used = used.cuda()[:, None, :, None].expand(pages, heads, size, 1)
    rows = [_rn(pages, heads, size, d, seed=seed + 1 + i) * torch.exp2(spread * _rn(pages, heads, size, 1, seed=seed + 3 + i)) for i in range(2)]
    rows = [r.to(BF16) for r in rows]
    if bits == 16:
        c = lo.PagedCache(*(torch.where(used, r, torch.full_like(r, float("nan"))) for r in rows))
        stands = [r.double() for r in rows]
        exps = None
    else:
        stands, exps, codes = [], [], []
        for r in rows:
            top = r.float().abs().amax(-1, keepdim=True)
            m, e = torch.frexp(top)
            byte = (e - 9 + (m > 0.875).int()).clamp(min=-126) + 127
            code = torch.ldexp(r.float(), 127 - byte).to(E4M3)
            stands.append(code.double() * torch.exp2(byte.double() - 127))
            codes.append(torch.where(used, code.view(torch.uint8), torch.full_like(code.view(torch.uint8), 0x7F)).view(E4M3))
            exps.append(torch.where(used[..., 0], byte[..., 0], 255).to(torch.uint8))
        c = lo.PagedCache(*codes, *exps)
    return c, table.to(I32).cuda(), torch.tensor(lengths, dtype=I32, device="cuda"), stands


def _tolerance(q, o, size, score, lengths, window, stands, table, c, scale):
    d = q.shape[-1]
    n = torch.tensor([min(max(x, 0), window or x) for x in lengths], device="cuda", dtype=torch.float64).clamp(min=0)[:, None, None]
    s = (d / 8 + 32) * 2.0 ** -23 * score + 2.0 ** -21
    tol = 2.0 ** -8 * o.abs() + size * (2 * s + (2.0 ** -16 if c.k_exponent is None else 2.0 ** -11) + (n / 16 + 64) * 2.0 ** -22) + 1e-30
    if c.k_exponent is not None:
        # max(w 2^e) is at most max |v| / 224 of the weights' largest product, itself at most the largest of sum w |v| over the head's features
        tol = tol + n * 448 * 2.0 ** -25 * (size.amax(-1, keepdim=True) / 224)
    return tol


def _check(lo, lengths, heads, share, d, size, bits, window=None, scale=None, seed=0, spread=0.0, q=None):
    c, table, n, stands = _cache(lo, lengths, size, heads, d, bits, seed, spread)
    q = _rn(len(lengths), heads * share, d, seed=seed + 9).to(BF16) if q is None else q
    o = lo.paged_attention_step(q, c, table, n, window, scale)
    lo.L.synchronize_and_check()
    want, size_, score = orc.paged_attention_step(q, *stands, table, lengths, window, scale)
    tol = _tolerance(q, want, size_, score, lengths, window, stands, table, c, scale)
    assert o.dtype == BF16 and o.is_contiguous() and bool(o.isfinite().all())
    over = ((o.double() - want).abs() - tol).amax()
    assert float(over) <= 0.0, float(over)
    return o


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 95, 96, 97, 192, 193, 384, 385, 500, 1000, 1537]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,share", [(1, 1), (2, 3), (3, 8), (2, 9), (1, 16), (2, 17), (1, 40), (12, 1)])
def test_heads(lo, bits, d, heads, share):
    _check(lo, LENGTHS, heads, share, d, 16, bits)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("size", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window", [None, 1, 15, 16, 17, 100, 383, 1024, 100000, 2 ** 63 - 1])
def test_windows_and_pages(lo, bits, size, window):
    _check(lo, LENGTHS, 2, 4, 64 if size == 32 else 128, size, bits, window)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("lengths", [[1], [16], [90], [5000], [40000], [0], [-5, 0], [131072], [3, 70000, 1, 0, 20000, 64], [257] * 300, list(range(0, 700)),
                                     [96 * 4 + 1] * 3, [20000] + [1] * 1500])
def test_lengths(lo, bits, lengths):
    _check(lo, lengths, 2, 2, 64, 64, bits)


@pytest.mark.parametrize("bits", [16, 8])
def test_every_cut(lo, bits):
    """Units of many lengths next to one another: runs begin and end at all places within them, hold whole units, or lie within one."""
    for i, n in enumerate((385, 700, 1111, 3000, 9999, 30000)):
        _check(lo, [n, n // 3, n + 95, 7, n // 2 + 1], 1 + i % 3, 5, 128, 16, bits, seed=i)
        _check(lo, [n] * 40, 3, 1, 64, 32, bits, seed=i)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,share", [(1, 12), (3, 16), (1, 40)])
def test_cut_units_of_many_heads(lo, bits, d, heads, share):
    _check(lo, [9999, 30, 0, 14000, 5000], heads, share, d, 32, bits)
    _check(lo, [4000] * 20, heads, share, d, 16, bits, window=1500)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 5.0])
def test_scales(lo, bits, scale):
    """Sharp weights, too: maxima that rise many times, weights that vanish."""
    _check(lo, [1, 40, 1000, 5000], 2, 4, 64, 16, bits, scale=scale)


@pytest.mark.parametrize("bits", [16, 8])
def test_rising_scores(lo, bits):
    """Every later key scores higher than all before, or lower."""
    c, table, n, stands = _cache(lo, [3000, 3000], 64, 1, 64, bits)
    ramp = torch.linspace(0, 3, 3000, device="cuda")
    k = torch.zeros(2, 3000, 1, 64, device="cuda")
    k[0, :, 0, 0], k[1, :, 0, 0] = ramp, -ramp
    v = _rn(2, 3000, 1, 64).to(BF16)
    lo.paged_cache_write(c, k.to(BF16), v, table, n)
    back = lo.paged_cache_read(c, table, n, 3000).reshape(2, 2, 3000, 64)
    q = torch.zeros(2, 2, 64, device="cuda", dtype=BF16)
    q[..., 0] = 100.0
    o = lo.paged_attention_step(q, c, table, n, softmax_scale=1.0)
    w = torch.softmax(100.0 * back[0, ..., 0].double(), -1)
    want = torch.einsum("bl,bld->bd", w, back[1].double())[:, None].expand(2, 2, 64)
    size = torch.einsum("bl,bld->bd", w, back[1].double().abs())[:, None]
    s = 40 * 2.0 ** -23 * 300 + 2.0 ** -21
    tol = 2.0 ** -8 * want.abs() + size * (2 * s + 2.0 ** -11 + 252 * 2.0 ** -22) + 3000 * 2.0 ** -24 * size.amax(-1, keepdim=True)
    assert bool(((o.double() - want).abs() <= tol).all())


def test_values_of_every_size(lo):
    """8 bits: rows whose powers of two are far apart; queries over the whole range of bf16."""
    _check(lo, [40, 700, 5000], 2, 4, 128, 16, 8, spread=3.0)
    _check(lo, [40, 700, 5000], 2, 4, 128, 16, 16, spread=3.0)
    for e in (-120, -50, 50, 110):     # (scales up to 1e18 are taken)
        q = (_rn(3, 8, 128, seed=e + 200) * 2.0 ** e).to(BF16)
        for bits in (8, 16):
            _check(lo, [40, 700, 5000], 2, 4, 128, 16, bits, q=q, scale=min(2.0 ** -e / 11, 1e18))
    q = _rn(3, 8, 128, seed=3).to(BF16)
    q[0, 0], q[1, 3, 1:] = 0, 0
    q[2, 5] *= torch.exp2(torch.linspace(-30, 5, 128, device="cuda")).to(BF16)
    _check(lo, [40, 700, 5000], 2, 4, 128, 16, 8, q=q)


@pytest.mark.parametrize("bits", [16, 8])
def test_nan_and_infinity(lo, bits):
    """Within the window they reach their own sequence and head alone; outside of it they are not looked at."""
    lengths, window = [700, 700, 700, 700], 300
    c, table, n, stands = _cache(lo, lengths, 64, 3, 64, bits)
    want = lo.paged_attention_step(_q := _rn(4, 6, 64).to(BF16), c, table, n, window)

    def spoil(t, e, i, head, p, value):
        page, row = int(table[i, p // 64]), p % 64
        if bits == 16:
            t[page, head, row, 5] = value
        else:
            e[page, head, row] = 255
    spoil(c.k, c.k_exponent, 0, 1, 650, float("nan"))
    spoil(c.v, c.v_exponent, 1, 2, 450, float("nan"))
    spoil(c.v, c.v_exponent, 2, 0, 699, float("inf"))
    for p in (0, 399):
        spoil(c.k, c.k_exponent, 3, 0, p, float("inf"))
        spoil(c.v, c.v_exponent, 3, 1, p, float("nan"))
    q = _q.clone()
    q[3, 5, 7] = float("nan")
    got = lo.paged_attention_step(q, c, table, n, window)
    bad = torch.zeros(4, 6, dtype=torch.bool, device="cuda")
    bad[0, 2:4] = bad[1, 4:6] = bad[2, 0:2] = bad[3, 5] = True
    spoiled = ~got.isfinite()
    assert torch.equal(got[~bad], want[~bad]) and not bool(spoiled[~bad].any()) and bool(spoiled[bad].any(-1).all())
    assert bool(got[0, 2:4].isnan().all()) and bool(got[3, 5].isnan().all())
    # an infinite score: the softmax of infinities is NaN, as in plain arithmetic
    q = _q.clone()
    q[0, 0, 0] = float("inf")
    assert bool(lo.paged_attention_step(q, c, table, n, window)[0, 0].isnan().all())


@pytest.mark.parametrize("bits", [16, 8])
def test_pages_that_are_not_there(lo, bits):
    """Left out and told; others' results do not change."""
    lengths = [3000, 3000, 3000]
    c, table, n, stands = _cache(lo, lengths, 64, 2, 64, bits)
    q = _rn(3, 4, 64).to(BF16)
    want = lo.paged_attention_step(q, c, table, n)
    bad = table.clone()
    bad[1, 7], bad[1, 9] = -1, 1 << 29
    lo.L.synchronize_and_check()
    got = lo.paged_attention_step(q, c, bad, n)
    with pytest.raises(lo.L.LactError, match="page number or a length"):
        lo.L.synchronize_and_check()
    seen = torch.ones(3000, dtype=torch.bool, device="cuda")
    seen[7 * 64:8 * 64] = seen[9 * 64:10 * 64] = False
    rows = lambda t: t[table[1].long()[:47]].permute(0, 2, 1, 3).reshape(-1, 2, 64)[:3000]
    x = torch.einsum("jgd,ljd->jgl", q[1].double().reshape(2, 2, 64), rows(stands[0])) / 8
    w = torch.softmax(x.masked_fill(~seen, float("-inf")), -1)
    plain = torch.einsum("jgl,ljd->jgd", w, rows(stands[1])).reshape(4, 64)
    size = torch.einsum("jgl,ljd->jgd", w, rows(stands[1]).abs()).reshape(4, 64)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert bool(((got[1].double() - plain).abs() <= 2.0 ** -8 * plain.abs() + size * 2.0 ** -10 + 2.0 ** -13 * size.amax(-1, keepdim=True)).all())
    long = n.clone()
    long[0] = 1 << 30                                  # past the table's end
    lo.paged_attention_step(q, c, table.clamp(min=0), long)
    with pytest.raises(lo.L.LactError):
        lo.L.synchronize_and_check()
    lo.L.synchronize_and_check()


@pytest.mark.parametrize("lengths", [[90, 100], [90, 20000], [100] * 200])   # a cluster; cut units; one CTA a unit
def test_a_window_without_a_page(lo, lengths):
    c, table, n, _ = _cache(lo, lengths, 64, 2, 64, 16)
    q = _rn(len(lengths), 4, 64).to(BF16)
    want = lo.paged_attention_step(q, c, table, n)
    bad = table.clone()
    bad[1] = -1
    lo.L.synchronize_and_check()
    got = lo.paged_attention_step(q, c, bad, n)
    with pytest.raises(lo.L.LactError, match="page number or a length"):
        lo.L.synchronize_and_check()
    assert bool(got[1].isnan().all()) and torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:])


def test_layouts(lo):
    for bits in (16, 8):
        c, table, n, _ = _cache(lo, [600, 70, 0], 32, 2, 64, bits)
        q = _rn(3, 8, 64).to(BF16)
        want = lo.paged_attention_step(q, c, table, n)
        fused = torch.zeros(3, 16, 64, device="cuda", dtype=BF16)
        fused[:, 8:] = q
        odd = torch.zeros(3, 8, 65, device="cuda", dtype=BF16)
        odd[..., 1:] = q
        for x in (fused[:, 8:], q.transpose(0, 1).contiguous().transpose(0, 1), odd[..., 1:], q.transpose(1, 2).contiguous().transpose(1, 2)):
            assert torch.equal(lo.paged_attention_step(x, c, table, n), want)
        assert torch.equal(lo.paged_attention_step(q, c, table.long().t().contiguous().t(), n.long()), want)
        two = [None if t is None else torch.stack([t.view(torch.uint8), torch.zeros_like(t.view(torch.uint8))], 1).view(t.dtype)[:, 0] for t in c]   # pages apart
        assert torch.equal(lo.paged_attention_step(q, lo.PagedCache(*two), table, n), want)
        one, t1, n1, _ = _cache(lo, [50], 64, 1, 64, bits)
        x = _rn(1, 1, 64).to(BF16)
        assert torch.equal(lo.paged_attention_step(x.as_strided((1, 1, 64), (3, 5, 1)), one, t1, n1), lo.paged_attention_step(x, one, t1, n1))


def test_the_same_bits_again_and_beside_others(lo):
    """Runs follow lengths alone, so that a call repeats itself; another stream's call at the same time changes nothing."""
    c, table, n, _ = _cache(lo, [9000, 4000, 20000, 1], 64, 2, 128, 8)
    q = _rn(4, 16, 128).to(BF16)
    want = lo.paged_attention_step(q, c, table, n)
    side = [torch.cuda.Stream() for _ in range(3)]
    got = []
    torch.cuda.synchronize()
    for i in range(30):
        with torch.cuda.stream(side[i % 3]):
            got.append(lo.paged_attention_step(q, c, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("bits", [16, 8])
def test_captured_calls_follow_the_lengths(lo, bits):
    """Two graphs in turn, with an eager call between them: each has its own counters."""
    top = [3000, 40, 700]
    c, table, n, _ = _cache(lo, top, 64, 2, 64, bits)
    q = _rn(3, 4, 64).to(BF16)
    lo.paged_attention_step(q, c, table, n)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(lo.paged_attention_step(q, c, table, n))
        graphs.append(g)
    for lengths in ([3000, 40, 700], [1, 1, 1], [0, 0, 0], [2999, 3, 650], [400, 39, 5], [1537, 0, 384]):
        n.copy_(torch.tensor(lengths, dtype=I32))
        for i in (0, 1, 1, 0):
            outs[i].fill_(7)
            graphs[i].replay()
            assert torch.equal(outs[i], lo.paged_attention_step(q, c, table, n))


def test_a_compiled_layer(lo):
    c, table, n, _ = _cache(lo, [70, 20], 16, 2, 64, 8)
    x = [_rn(2, 1, h, 64).to(BF16) for h in (4, 2, 2)]
    f, pos = lo.rotary_frequencies([32], device="cuda"), (n - 1)[:, None]

    def call(q, k, v):
        q, k = lo.rotary_axes(q[:, 0], k[:, 0], pos, f, [32])
        lo.paged_cache_write(c, k[:, None], v, table, n)
        return lo.paged_attention_step(q, c, table, n, 50)
    want = call(*x)
    for t in (c.k, c.v):
        t.view(torch.uint8)[table.long()[0, 4], :, 5].fill_(1)
    assert torch.equal(torch.compile(call, fullgraph=True, backend="aot_eager")(*x), want)


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_gradients_are_refused_and_modes_taken(lo, mode):
    c, table, n, _ = _cache(lo, [70, 20], 16, 2, 64, 16)
    q = _rn(2, 4, 64).to(BF16)
    want = lo.paged_attention_step(q, c, table, n)
    with pytest.raises(NotImplementedError):
        lo.paged_attention_step(q.clone().requires_grad_(), c, table, n)
    with mode():
        assert torch.equal(lo.paged_attention_step(q.clone().requires_grad_(), c, table, n), want)


def test_empty_calls(lo):
    c = lo.paged_cache(4, 16, 2, 64, device="cuda")
    o = lo.paged_attention_step(torch.zeros(0, 4, 64, device="cuda", dtype=BF16), c, torch.zeros(0, 3, dtype=I32, device="cuda"), torch.zeros(0, dtype=I32, device="cuda"))
    assert o.shape == (0, 4, 64)
    o = lo.paged_attention_step(_rn(2, 4, 64).to(BF16), c, torch.full((2, 500), -1, dtype=I32, device="cuda"), torch.zeros(2, dtype=I32, device="cuda"))
    assert bool((o == 0).all())


def test_a_cache_of_more_than_2_to_31_elements(lo):
    if torch.cuda.get_device_properties(0).total_memory < 100e9:
        pytest.skip("needs 100 GB")
    for bits, pages in ((16, 262400), (8, 524800)):
        c = lo.paged_cache(pages, 64, 1, 128, BF16 if bits == 16 else E4M3, "cuda")
        table = (pages - 1 - torch.arange(32, dtype=I32, device="cuda")).reshape(2, -1)
        n = torch.tensor([1024, 700], dtype=I32, device="cuda")
        x = _rn(2, 1024, 1, 128).to(BF16)
        lo.paged_cache_write(c, x, -x, table, n)
        small = lo.PagedCache(*(None if t is None else t[-32:].clone() for t in c))
        q = _rn(2, 8, 128).to(BF16)
        assert torch.equal(lo.paged_attention_step(q, c, table, n), lo.paged_attention_step(q, small, table - (pages - 32), n))
        del c
        torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------------------- as they are used together
@pytest.mark.parametrize("window", [None, 48])
@pytest.mark.parametrize("share", [1, 4])
def test_generation_gives_what_the_whole_sequence_gives(lo, window, share):
    """A prompt turned and written, then token after token turned, written and attended: the outputs of sliding_window_attention over the
    whole (which rounds its weights to bf16: 2^-8 of sum w |v| on its side, and its own rounding)."""
    b, l, first, hk, d = 2, 150, 100, 2, 64
    h = hk * share
    q, k, v = (_rn(b, l, n, d, seed=i).to(BF16) for i, n in enumerate((h, hk, hk)))
    f, pos = lo.rotary_frequencies([d // 2], device="cuda"), torch.arange(l, device="cuda", dtype=I32)[:, None]
    q, k = lo.rotary_axes(q, k, pos, f, [d // 2])
    whole = lo.sliding_window_attention(q, *(t.repeat_interleave(share, 2) for t in (k, v)), window)
    c = lo.paged_cache(24, 16, hk, d, device="cuda")
    table = torch.randperm(24, generator=torch.Generator().manual_seed(0))[:20].reshape(2, 10).to(I32).cuda()
    n = torch.full((b,), first, dtype=I32, device="cuda")
    lo.paged_cache_write(c, k[:, :first], v[:, :first], table, n)
    for t in range(first, l):
        n.add_(1)
        lo.paged_cache_write(c, k[:, t:t + 1], v[:, t:t + 1], table, n)
        o = lo.paged_attention_step(q[:, t], c, table, n, window)
        _, size, _ = orc.paged_attention_step(q[:, t], c.k, c.v, table, [t + 1] * b, window)
        err = (o.double() - whole[:, t].double()).abs()
        assert bool((err <= 2 * 2.0 ** -8 * whole[:, t].double().abs() + size * (2.0 ** -8 + 2.0 ** -12)).all())


@pytest.mark.parametrize("bits", [16, 8])
def test_frames_read_back_for_the_next(lo, bits):
    """The video layer's generation step on a cache in pages: the keys and values it reads back are those of a contiguous cache."""
    b, frame, h, d = 2, 60, 3, 64
    f = lo.rotary_frequencies([12, 10, 10], device="cuda")
    place = lambda t: torch.tensor([[t, y, x] for y in range(6) for x in range(10)], device="cuda", dtype=I32)
    c = lo.paged_cache(16, 32, h, d, BF16 if bits == 16 else E4M3, "cuda")
    table, n = torch.arange(16, dtype=I32, device="cuda").reshape(2, 8), torch.zeros(b, dtype=I32, device="cuda")
    held = []
    for t in range(4):
        q, k, v = (_rn(b, frame, h, d, seed=10 * t + i).to(BF16) for i in range(3))
        q, k = lo.rotary_axes(q, k, place(t), f, [12, 10, 10], interleaved=True)
        if t:
            kv = lo.paged_cache_read(c, table, n, min(t, 2) * frame)
            want = torch.cat([torch.cat([x[i] for x in held[-2:]], 1) for i in range(2)])
            assert torch.equal(kv, want)
            o = lo.sliding_window_attention_inference(q, k, v, frame, kv_cache=kv)
            assert torch.equal(o, lo.sliding_window_attention_inference(q, k, v, frame, kv_cache=want))
        n.add_(frame)
        lo.paged_cache_write(c, k, v, table, n)
        held.append([x if bits == 16 else orc.rows_in_8_bits(x)[0].to(BF16) for x in (k, v)])
