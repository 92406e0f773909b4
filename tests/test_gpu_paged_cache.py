"""The paged cache: what is written, what is read back, and what is left alone (exact: the oracle's rounding to 8 bits has no tolerance)."""
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


def _rn(*s, seed=0):
    return torch.randn(*s, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + sum(s)))


def _bytes(t):
    return None if t is None else t.view(torch.uint8).clone()


def _filled(lo, pages, size, heads, d, bits):
    """A cache whose every byte is told from a written one."""
    c = lo.paged_cache(pages, size, heads, d, BF16 if bits == 16 else E4M3, "cuda")
    for i, t in enumerate(c):
        if t is not None:
            t.view(torch.uint8).fill_(0x31 + i)
    return c


def _table(lengths, size, pages, extra=2, seed=0):
    """Pages in random order; -1 and numbers far out of range behind a sequence's last."""
    need = [-(-max(n, 0) // size) for n in lengths]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:sum(need)].tolist()
    table = torch.full((len(lengths), max(need + [0]) + extra), -1)
    table[:, -1] = 1 << 30
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.long)
    return table.to(I32).cuda()


def _check(lo, size, heads, d, bits, lengths, rows, packed, k=None, v=None, cache=None, table=None):
    pages = sum(-(-max(n, 0) // size) for n in lengths) + 5
    cache = _filled(lo, pages, size, heads, d, bits) if cache is None else cache
    table = _table(lengths, size, cache.k.shape[0]) if table is None else table
    total = sum(rows)
    shape = (1, total, heads, d) if packed else (len(rows), rows[0], heads, d)
    k = _rn(*shape, seed=1).to(BF16) if k is None else k
    v = _rn(*shape, seed=2).to(BF16) * 3 if v is None else v
    cu = torch.tensor([0] + rows).cumsum(0).to(I32).cuda() if packed else None
    n = torch.tensor(lengths, dtype=I32).cuda()
    before = [None if t is None else t.clone() for t in cache]
    lo.paged_cache_write(cache, k, v, table, n, cu)
    places = orc.paged_places(lengths, rows, table.cpu(), size)
    want = [None if t is None else t.view(torch.uint8).clone() for t in before]
    back = torch.zeros(2, total, heads, d, dtype=BF16, device="cuda")
    if places:
        r, page, row = (torch.tensor(x).cuda() for x in zip(*places))
        for side, x in enumerate((k, v)):
            x = x.reshape(total, heads, d)[r]
            if bits == 16:
                want[side].view(BF16)[page, :, row] = x
                back[side, r] = x
            else:
                values, byte = orc.rows_in_8_bits(x)
                fine = byte < 255
                coded = (values * torch.exp2(127 - byte.double())[..., None]).float().to(E4M3).view(torch.uint8)
                want[side][page, :, row] = torch.where(fine[..., None], coded, torch.full_like(coded, 0x7F))
                want[2 + side][page, :, row] = byte
                back[side, r] = values.to(BF16)
    for got, w in zip(cache, want):
        assert got is None or torch.equal(got.view(torch.uint8), w)
    got = lo.paged_cache_read(cache, table, n, total if packed else rows[0], cu)
    assert got.dtype == BF16 and got.shape == ((2, total, heads, d) if packed else (2 * len(rows), rows[0], heads, d))
    got = got.reshape(2, total, heads, d)
    assert torch.equal(got.isnan(), back.isnan()) and torch.equal(got.nan_to_num(), back.nan_to_num())
    lo.L.synchronize_and_check()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("size,heads,d", [(16, 1, 64), (16, 3, 128), (32, 12, 64), (64, 8, 128), (128, 4, 64), (256, 2, 128), (64, 40, 64)])
def test_sizes(lo, bits, size, heads, d):
    _check(lo, size, heads, d, bits, [37, 5, 300, 16, 15], [9] * 5, False)
    _check(lo, size, heads, d, bits, [37, 0, 300, 256, 15], [37, 0, 41, 256, 1], True)


@pytest.mark.parametrize("bits", [16, 8])
def test_lengths(lo, bits):
    """New tokens alone, more rows than tokens (padded in front), sequences that are not in use, lengths below zero."""
    _check(lo, 16, 2, 64, bits, [1, 17, 16, 0, -3, 1000], [1] * 6, False)
    _check(lo, 16, 2, 64, bits, [1, 33, 0, 20, 64, -9], [33] * 6, False)
    _check(lo, 16, 2, 64, bits, [0, 0], [4] * 2, False)
    _check(lo, 32, 2, 128, bits, [5], [5], True)
    _check(lo, 32, 2, 128, bits, [3, 0, 0, 70], [8, 0, 4, 2], True)
    _check(lo, 64, 4, 128, bits, [9000, 2048], [4500, 2048], True)
    _check(lo, 64, 4, 128, bits, [3000, 2500, 10], [2500] * 3, False)


def test_rows_of_every_size(lo):
    """8 bits: rows over the whole range of bf16, ties, zeros, NaN and infinities."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(1, 400, 2, 64, device="cuda", generator=g) * torch.exp2(torch.randint(-140, 120, (1, 400, 2, 1), device="cuda", generator=g).float())
    k = x.to(BF16)
    k[0, 0], k[0, 1, 0], k[0, 2] = 0, 448.0, 2.0 ** -133
    k[0, 3, 0, 5], k[0, 4, 1, 63], k[0, 5, 0, 0] = float("nan"), float("inf"), float("-inf")
    k[0, 6] = torch.arange(-64, 64, device="cuda").reshape(2, 64).to(BF16) * 1.0625      # on and between the grid's points
    k[0, 7], k[0, 7, :, 3] = 1.0, 1.75 * 2 ** 9
    k[0, 8], k[0, 8, :, 3] = 1.0, 1.7578125 * 2 ** 9
    k[0, 9], k[0, 10] = 2.0 ** 127 * 1.9921875, -2.0 ** 127 * 1.5
    _check(lo, 16, 2, 64, 8, [400], [400], False, k=k, v=k.flip(1).contiguous())
    ties = torch.arange(0, 256, device="cuda").float().reshape(1, 4, 1, 64) + 0.5
    _check(lo, 16, 1, 64, 8, [4], [4], False, k=ties.to(BF16), v=-ties.to(BF16))


@pytest.mark.parametrize("bits", [16, 8])
def test_layouts(lo, bits):
    b, l, h, d = 2, 21, 3, 64
    x = _rn(b, l, h, d, seed=5).to(BF16)
    fused = torch.zeros(b, l, 2 * h * d + 8, device="cuda", dtype=BF16)
    fused[..., :h * d] = x.reshape(b, l, h * d)
    odd = torch.zeros(b, l, h, d + 1, device="cuda", dtype=BF16)
    odd[..., 1:] = x
    for k in (fused[..., :h * d].reshape(b, l, h, d), x.transpose(1, 2).contiguous().transpose(1, 2), odd[..., 1:],
              x.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)):
        _check(lo, 16, h, d, bits, [40, 21], [l] * b, False, k=k, v=k)
    one = x[:1, :1].as_strided((1, 1, h, d), (3, 5, d, 1))                               # axes of one entry with foreign strides
    _check(lo, 16, h, d, bits, [7], [1], False, k=one, v=one)
    # pages of keys and values side by side in one array, and of several layers; an int64 table that is a view
    whole = torch.zeros(12, 2, h, 16, d, device="cuda", dtype=BF16 if bits == 16 else torch.uint8)
    exps = torch.zeros(12, 2, h, 16, device="cuda", dtype=torch.uint8)
    data = whole if bits == 16 else whole.view(E4M3)
    c = lo.PagedCache(data[:, 0], data[:, 1], *((exps[:, 0], exps[:, 1]) if bits == 8 else ()))
    table = _table([40, 21], 16, 12).long().repeat(1, 2)[:, ::2]
    table = torch.stack([_table([40, 21], 16, 12).long(), torch.zeros(2, 5, device="cuda", dtype=torch.long) - 7], 2)[:, :, 0]
    _check(lo, 16, h, d, bits, [40, 21], [l] * b, False, cache=c, table=table)


def test_a_page_that_is_not_there_is_left_out_and_told(lo):
    for bits in (16, 8):
        c = _filled(lo, 6, 16, 2, 64, bits)
        table = torch.tensor([[0, -1, 2], [3, 6, 4], [5, 1, 1]], dtype=I32, device="cuda")
        lengths = torch.tensor([40, 40, 70], dtype=I32, device="cuda")     # (the third: past its row of the table)
        x = _rn(3, 30, 2, 64).to(BF16)
        lo.L.synchronize_and_check()
        lo.paged_cache_write(c, x, x, table, lengths)
        with pytest.raises(lo.L.LactError, match="page number or a length"):
            lo.L.synchronize_and_check()
        lo.L.synchronize_and_check()                                       # (told once)
        good = torch.tensor([[0, 1, 2], [3, 1, 4], [5, 1, 1]], dtype=I32, device="cuda")
        # (positions 40 to 47 of the third are there: rows 8 to 15 of page 1)
        assert bool((_bytes(c.k)[1, :, :8] == 0x31).all()) and bool((_bytes(c.v)[5] == 0x32).all()) and not bool((_bytes(c.k)[1, :, 8:] == 0x31).all())
        got = lo.paged_cache_read(c, table, lengths, 30).reshape(2, 3, 30, 2, 64)
        with pytest.raises(lo.L.LactError):
            lo.L.synchronize_and_check()
        full = lo.paged_cache_read(c, good, lengths.clamp(max=40), 30).reshape(2, 3, 30, 2, 64)
        lost = torch.zeros(3, 30, dtype=torch.bool, device="cuda")
        pos = torch.arange(10, 40, device="cuda")
        lost[:2] = (pos >= 16) & (pos < 32)
        assert bool((got[:, :2][:, lost[:2]] == 0).all()) and torch.equal(got[:, :2][:, ~lost[:2]], full[:, :2][:, ~lost[:2]])
        lo.L.synchronize_and_check()


def test_numbers_of_64_bits_stay_out_of_range(lo):
    """A page number or a length that 32 bits would make a valid one is left out and told."""
    c = _filled(lo, 6, 16, 1, 64, 16)
    x = _rn(2, 1, 1, 64).to(BF16)
    table = torch.tensor([[(1 << 32) + 1], [2]], device="cuda")
    lo.L.synchronize_and_check()
    lo.paged_cache_write(c, x, x, table, torch.tensor([1, 1], device="cuda"))
    with pytest.raises(lo.L.LactError):
        lo.L.synchronize_and_check()
    assert bool((_bytes(c.k)[1] == 0x31).all()) and torch.equal(c.k[2, 0, 0], x[1, 0, 0])
    lo.paged_cache_write(c, x, x, table.clamp(max=3), torch.tensor([(1 << 32) + 1, 0], device="cuda"))
    with pytest.raises(lo.L.LactError):
        lo.L.synchronize_and_check()
    assert bool((_bytes(c.k)[3] == 0x31).all())
    lo.paged_cache_write(c, x, x, table.clamp(max=3), torch.tensor([-(1 << 40), 0], device="cuda"))
    lo.L.synchronize_and_check()
    assert bool((_bytes(c.k)[3] == 0x31).all())


def test_bounds_that_fall_or_pass_the_end_stay_inside(lo):
    c = _filled(lo, 8, 16, 1, 64, 16)
    lengths = torch.tensor([16, 16, 16], dtype=I32, device="cuda")
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=I32, device="cuda")
    x = _rn(1, 20, 1, 64).to(BF16)
    for cu in ([0, 9, 4, 20], [5, 8, 8, 400], [-7, 3, 3, 12], [25, 30, 31, 32]):
        lo.paged_cache_write(c, x, x, table, lengths, torch.tensor(cu, dtype=I32, device="cuda"))
        lo.paged_cache_read(c, table, lengths, 20, torch.tensor(cu, dtype=I32, device="cuda"))
    lo.L.synchronize_and_check()
    assert bool((_bytes(c.k)[6:] == 0x31).all())
    c = _filled(lo, 8, 16, 1, 64, 16)      # rows ahead of the first sequence and behind the last are not of any
    lo.paged_cache_write(c, x, x, table, lengths, torch.tensor([3, 8, 8, 12], dtype=I32, device="cuda"))
    got = lo.paged_cache_read(c, table, lengths, 20, torch.tensor([3, 8, 8, 12], dtype=I32, device="cuda"))
    want = torch.zeros_like(x)
    want[:, 3:12] = x[:, 3:12]
    assert torch.equal(got, torch.cat([want, want]))


def test_refusals_on_the_device(lo):
    c = lo.paged_cache(4, 16, 2, 64, device="cuda")
    t, n, x = torch.zeros(1, 2, dtype=I32, device="cuda"), torch.ones(1, dtype=I32, device="cuda"), torch.zeros(1, 1, 2, 64, dtype=BF16, device="cuda")
    for bad in (lambda: lo.paged_cache_write(c, c.k[:1, :, :1].transpose(1, 2), x, t, n), lambda: lo.paged_cache_write(lo.PagedCache(c.k, c.k), x, x, t, n),
                lambda: lo.paged_cache_write(c, x.cpu(), x, t, n), lambda: lo.paged_cache_read(c, t.cpu(), n, 4)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        lo.paged_cache_write(c, x.clone().requires_grad_(), x, t, n)
    off = torch.zeros(4 * 2 * 16 * 64 + 8, dtype=BF16, device="cuda")[8:].reshape(4, 2, 16, 64)   # 16 bytes past a boundary of 32
    with pytest.raises(ValueError):
        lo.paged_cache_read(lo.PagedCache(off, off), t, n, 4)


def test_empty_calls(lo):
    c = lo.paged_cache(4, 16, 2, 64, device="cuda")
    t, n = torch.zeros(0, 2, dtype=I32, device="cuda"), torch.zeros(0, dtype=I32, device="cuda")
    x = torch.zeros(0, 5, 2, 64, dtype=BF16, device="cuda")
    lo.paged_cache_write(c, x, x, t, n)
    assert lo.paged_cache_read(c, t, n, 5).shape == (0, 5, 2, 64)
    t, n = torch.zeros(3, 2, dtype=I32, device="cuda"), torch.ones(3, dtype=I32, device="cuda")
    x = torch.zeros(3, 0, 2, 64, dtype=BF16, device="cuda")
    lo.paged_cache_write(c, x, x, t, n)
    assert lo.paged_cache_read(c, t, n, 0).shape == (6, 0, 2, 64)


@pytest.mark.parametrize("bits", [16, 8])
def test_captured_calls_follow_the_lengths(lo, bits):
    c, eager = (_filled(lo, 20, 16, 2, 64, bits) for _ in range(2))
    n = torch.tensor([3, 17], dtype=I32, device="cuda")
    table = _table([60, 60], 16, 20)
    x = _rn(2, 1, 2, 64).to(BF16)
    call = lambda c: (lo.paged_cache_write(c, x, x, table, n), lo.paged_cache_read(c, table, n, 8))[1]
    call(c), call(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(c)
    for i in range(40):
        n.add_(1)
        x.copy_(_rn(2, 1, 2, 64, seed=i))
        graph.replay()
        assert torch.equal(out, call(eager))
    assert all(torch.equal(_bytes(a), _bytes(b)) for a, b in zip(c, eager) if a is not None)


def test_a_cache_of_more_than_2_to_31_elements(lo):
    if torch.cuda.get_device_properties(0).total_memory < 100e9:
        pytest.skip("needs 100 GB")
    for bits, pages in ((16, 262400), (8, 524800)):
        c = lo.paged_cache(pages, 64, 1, 128, BF16 if bits == 16 else E4M3, "cuda")
        assert c.k.numel() > 2 ** 31
        table = torch.arange(pages, dtype=I32, device="cuda").reshape(2, -1).flip(0)
        n = torch.tensor([pages * 32, pages * 32 - 5], dtype=I32, device="cuda")
        x = _rn(2, 300, 1, 128).to(BF16)
        lo.paged_cache_write(c, x, -x, table, n)
        got = lo.paged_cache_read(c, table, n, 300)
        want = x if bits == 16 else orc.rows_in_8_bits(x)[0].to(BF16)
        assert torch.equal(got[:2], want) and torch.equal(got[2:], -want)
        del c, got
        torch.cuda.empty_cache()
