"""What the calls on a paged cache tell the host: a page that is not there, but not in the place of a wait that ran out."""
import ctypes as C

import pytest
import torch

from test_gpu_paged_attention import BF16, I32, _rn, lo  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def _word():
    from lact_b200 import _lib as L
    word = C.POINTER(C.c_int32)()
    L.check(L.lib().lact_status_host_word(C.byref(word)), "word")
    return word


@pytest.mark.parametrize("call", ["write", "read", "step"])
def test_a_missing_page_does_not_replace_a_wait_that_ran_out(lo, call):  # noqa: F811
    """The word is written by the host here; a replay does not look at it before its kernels run."""
    c = lo.paged_cache(4, 16, 2, 64, device="cuda")
    table, n = torch.full((1, 2), -1, dtype=I32, device="cuda"), torch.tensor([20], dtype=I32, device="cuda")
    x = _rn(1, 20, 2, 64).to(BF16)
    run = {"write": lambda: lo.paged_cache_write(c, x, x, table, n), "read": lambda: lo.paged_cache_read(c, table, n, 20),
           "step": lambda: lo.paged_attention_step(x[:, 0], c, table, n)}[call]
    run()
    with pytest.raises(lo.L.LactError, match="102"):
        lo.L.synchronize_and_check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for before, after in ((101, 101), (0, 102), (101, 101)):
        word = _word()
        word[0] = before
        graph.replay()
        torch.cuda.synchronize()
        assert word[0] == (before | 102 << 8)             # (a byte for each)
        text = lo.L.lib().lact_error_string(word[0])
        assert text == lo.L.lib().lact_error_string(after) and b"unknown" not in text
        with pytest.raises(lo.L.LactError, match=str(after)):
            lo.L.synchronize_and_check()
        assert word[0] == 0
    lo.L.synchronize_and_check()


def test_many_missing_pages_are_told_quickly(lo):  # noqa: F811
    """80000 rows without a page (80 us where a store tells it, 2.4 s where every one is an atomic operation on the host's memory)."""
    c = lo.paged_cache(2, 64, 8, 128, device="cuda")
    table, n = torch.full((8, 157), -1, dtype=I32, device="cuda"), torch.full((8,), 10000, dtype=I32, device="cuda")
    lo.paged_cache_read(c, table, n, 10)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(lo.L.LactError, match="102"):
        lo.L.synchronize_and_check()
    with torch.cuda.graph(graph):
        lo.paged_cache_read(c, table, n, 10000)
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    graph.replay()
    b.record()
    torch.cuda.synchronize()
    with pytest.raises(lo.L.LactError, match="102"):
        lo.L.synchronize_and_check()
    assert a.elapsed_time(b) < 100
