"""Attention of single tokens with a window: pages that hold none of it may have been given back (their entries of the page table say
nothing), whatever the page's size, the type and where in a page or a step of the kernel the window begins."""
import pytest
import torch

from test_gpu_paged_attention import BF16, I32, _cache, _rn, lo  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def _given_back(table, lengths, size, window, entry):
    """The table without the pages in front of every sequence's window."""
    first = torch.tensor([max(n - window, 0) // size for n in lengths], device="cuda")[:, None]
    return torch.where(torch.arange(table.shape[1], device="cuda") < first, torch.full_like(table, entry), table)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("window", [1, 16, 17, 40, 64, 130])
def test_pages_in_front_of_a_window_are_not_asked_for(lo, bits, d, size, window):  # noqa: F811
    lengths = list(range(250, 315)) + [window, window + 1, 5, 0]          # (windows that begin at all places modulo 64)
    c, table, n, _ = _cache(lo, lengths, size, 2, d, bits)
    q = _rn(len(lengths), 6, d).to(BF16)
    want = lo.paged_attention_step(q, c, table, n, window)
    lo.L.synchronize_and_check()
    for entry in (-1, 1 << 30):
        got = lo.paged_attention_step(q, c, _given_back(table, lengths, size, window, entry), n, window)
        lo.L.synchronize_and_check()                                       # (nothing is told)
        assert torch.equal(got, want)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [16, 32])
@pytest.mark.parametrize("sequences,window", [(1, 300), (3, 5000), (150, 3000)])   # a cluster; cut units
def test_pages_in_front_of_a_long_window_are_not_asked_for(lo, bits, d, size, sequences, window):  # noqa: F811
    for shift in (0, 7, 16, 33, 48, 63):
        lengths = [6400 + shift + 16 * i for i in range(sequences)]
        c, table, n, _ = _cache(lo, lengths, size, 1, d, bits, seed=shift)
        q = _rn(len(lengths), 2, d).to(BF16)
        want = lo.paged_attention_step(q, c, table, n, window)
        lo.L.synchronize_and_check()
        got = lo.paged_attention_step(q, c, _given_back(table, lengths, size, window, -1), n, window)
        lo.L.synchronize_and_check()
        assert torch.equal(got, want)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("size", [16, 32, 64])
def test_a_page_within_the_window_is_still_asked_for(lo, bits, size):  # noqa: F811
    """Its first page, of which one row is seen, and its last."""
    length = 20 * size
    for window, entry in ((size + 1, 18), (1, 19)):
        c, table, n, _ = _cache(lo, [length, length], size, 1, 64, bits)
        q = _rn(2, 2, 64).to(BF16)
        want = lo.paged_attention_step(q, c, table, n, window)
        lo.L.synchronize_and_check()
        table = table.clone()
        table[1, entry] = -1
        got = lo.paged_attention_step(q, c, table, n, window)
        with pytest.raises(lo.L.LactError, match="page number or a length"):
            lo.L.synchronize_and_check()
        assert torch.equal(got[0], want[0])
