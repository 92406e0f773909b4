"""Attention of single tokens where queries are very large and keys very small: scores of an ordinary size, whatever the factors that a kernel
takes apart.  Tolerances: those of test_gpu_paged_attention (its docstring)."""
import pytest
import torch

from oracle import lact_oracle as orc
from test_gpu_paged_attention import BF16, E4M3, I32, _cache, _rn, _tolerance, lo  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
LENGTHS = [1, 40, 700, 5000]


def _check(lo, c, table, n, stands, q, scale):  # noqa: F811
    o = lo.paged_attention_step(q, c, table, n, None, scale)
    lo.L.synchronize_and_check()
    want, size, score = orc.paged_attention_step(q, *stands, table, LENGTHS, None, scale)
    assert 0.5 < float(score.max()) < 1000.0                # (the softmax has something to do)
    tol = _tolerance(q, want, size, score, LENGTHS, None, stands, table, c, scale)
    assert bool(o.isfinite().all()) and bool(((o.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("share", [2, 12])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [16, 8])
def test_large_queries_on_small_keys(lo, bits, d, share):  # noqa: F811
    c, table, n, stands = _cache(lo, LENGTHS, 32, 2, d, bits)
    small = 2.0 ** -118
    if bits == 16:
        c.k.mul_(small)
    else:
        c.k_exponent.copy_(torch.where(c.k_exponent == 255, c.k_exponent.int(), c.k_exponent.int() - 118))   # (bytes of 1 and 2)
        assert int(c.k_exponent[c.k_exponent < 255].max()) < 4 and int(c.k_exponent.min()) > 0
    k = stands[0] * small if bits == 8 else (stands[0].to(BF16) * small).double()
    q = (_rn(len(LENGTHS), 2 * share, d) * 2.0 ** 118).to(BF16)
    _check(lo, c, table, n, [k, stands[1]], q, d ** -0.5)


@pytest.mark.parametrize("share", [2, 12])
@pytest.mark.parametrize("d", [64, 128])
def test_the_smallest_power_of_two(lo, d, share):  # noqa: F811
    """A byte of 0 stands for 2^-127 (the write has 1 at least; a cache may be filled by others)."""
    c, table, n, stands = _cache(lo, LENGTHS, 32, 2, d, 8)
    pages, heads, size, _ = c.k.shape
    rows = (_rn(pages, heads, size, d, seed=5) * 16).clamp(-448, 448).to(E4M3)
    c.k.view(torch.uint8).copy_(rows.view(torch.uint8))
    c.k_exponent.zero_()
    q = (_rn(len(LENGTHS), 2 * share, d) * 2.0 ** 118).to(BF16)
    _check(lo, c, table, n, [rows.double() * 2.0 ** -127, stands[1]], q, 32 * d ** -0.5)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("length", [40, 700, 30000])           # one CTA or a cluster; cut units
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_value_that_is_not_finite_spoils_its_feature_alone(lo, d, length, value):  # noqa: F811
    """The outputs of that feature, of the heads that share the row; all others keep their bits.  A weight w meets an infinity in two pieces, hi =
    bf16(w) > 0 and lo = bf16(w - hi): hi inf + lo inf is infinite for lo > 0 and NaN for lo <= 0, so that either is right."""
    lengths = [length, length + 3, 17]
    c, table, n, _ = _cache(lo, lengths, 64, 3, d, 16)
    q = _rn(3, 6, d).to(BF16)
    want = lo.paged_attention_step(q, c, table, n)
    for p in (0, length // 2, length - 1):
        held = c.v.clone()
        c.v[int(table[0, p // 64]), 1, p % 64, 5] = value
        got = lo.paged_attention_step(q, c, table, n)
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[0, 2:4, 5] = True
        wrong = got[bad].isnan() if value != value else got[bad].isnan() | (got[bad] == value)
        assert bool(wrong.all()) and torch.equal(got[~bad], want[~bad])
        c.v.copy_(held)


def test_every_value_of_8_bits_read_back(lo):  # noqa: F811
    """All codes under all bytes, as bf16 rounds what they stand for: exact from byte 3 to 246 (2^-9 2^-124 is bf16's smallest number, 448 2^119 below its largest)."""
    c = lo.paged_cache(16, 256, 1, 64, E4M3, "cuda")
    code = torch.arange(256, device="cuda", dtype=torch.uint8)
    c.k.view(torch.uint8).copy_(code.reshape(4, 1, 1, 64).repeat(4, 1, 256, 1))       # page p: codes 64 (p % 4) on; row r: byte r
    c.v.view(torch.uint8).copy_(code.flip(0).reshape(4, 1, 1, 64).repeat(4, 1, 256, 1))
    for e in c[2:]:
        e.copy_(code.expand(16, 1, 256))
    table, n = torch.arange(16, device="cuda", dtype=I32)[None], torch.tensor([4096], dtype=I32, device="cuda")
    got = lo.paged_cache_read(c, table, n, 4096).reshape(2, 16, 256, 64)
    power = torch.exp2(code.double() - 127)
    power[255] = float("nan")
    for x, y in zip(got, (c.k, c.v)):
        stands = y.double()[:, 0] * power[:, None]
        want = stands.to(BF16)
        assert torch.equal(x.isnan(), want.isnan()) and torch.equal(x.nan_to_num(0.0, 1e38, -1e38), want.nan_to_num(0.0, 1e38, -1e38))
        fine = stands[:, 3:247].nan_to_num()
        assert torch.equal(x[:, 3:247].double().nan_to_num(), fine)
