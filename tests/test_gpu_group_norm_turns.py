"""Group norm of many tokens (one spot a sample): the launch has as many blocks as are resident, and each goes through its rows in turns -
the next rows are fetched while these are worked on, the last turn ends anywhere, weights' gradients add up over the turns, and the
forward takes two rows a turn of a thread once there are enough.  The row counts come from the device's SMs, so that every case has the
turns that its name says; tolerances as in test_gpu_group_norm.py (they do not depend on the number of turns: a thread adds one value a
turn to its weights' gradients, at most six here)."""
import pytest
import torch

from launched_kernels import kernels
from test_gpu_group_norm import BF16, F32, _check, _inputs, lo  # noqa: F401  (lo: the fixture)

pytestmark = pytest.mark.gpu


def _rows_of_one_turn(C, groups, dtype):
    """Rows that all resident blocks hold together, and the vectors of a thread: 768 threads an SM."""
    width = 8 if dtype == BF16 else 4
    while C // groups % width:
        width //= 2
    vectors = C // width
    assert vectors <= 1024
    a_thread = 1 if vectors <= 256 else 2 if vectors <= 512 else 4
    rows = 1 if a_thread > 1 else 256 // vectors
    threads = 256 if a_thread > 1 else (rows * vectors + 31) // 32 * 32
    return torch.cuda.get_device_properties(0).multi_processor_count * (768 // threads) * rows, a_thread


# groups of 2^n vectors (sums among lanes) and of others (through shared memory), whole and broken vectors, one to four of them a thread
SHAPES = [(1536, 12, BF16), (1536, 32, BF16), (96, 32, BF16), (60, 60, BF16), (64, 4, BF16), (384, 4, F32), (1000, 5, F32), (1536, 12, F32),
          (4096, 32, BF16), (2560, 5, BF16), (4096, 32, F32)]


@pytest.mark.parametrize("turns", [1.0, 1.4, 2.6, 4.03, 5.7])
@pytest.mark.parametrize("C,groups,dtype", SHAPES)
def test_turns(lo, C, groups, dtype, turns):
    whole, a_thread = _rows_of_one_turn(C, groups, dtype)
    n = int(whole * turns) + (1 if turns > 1.0 else 0)
    if n % 2 == 0 and turns > 1.0:
        n += 1
    x, w, b, dy = _inputs((n, C), dtype)
    _check(lo, x, w, b, dy, groups, True)
    two = turns >= 4.0 and a_thread == 1
    assert kernels(lambda: lo.group_norm(x, groups, w, b, activation="silu"), {f"Li{a_thread}ELi1ELb0E": 1, f"Li{a_thread}ELi2ELb0E": 2}) == [
        2 if two else 1]


def test_no_activation_and_no_weights_in_turns(lo):
    for groups in (12, 32):
        n = int(_rows_of_one_turn(1536, groups, BF16)[0] * 4.6) | 1
        x, w, b, dy = _inputs((n, 1536), BF16)
        _check(lo, x, None, None, dy, groups, False)
        _check(lo, x, w.to(BF16), b.to(BF16), dy, groups, False)


def test_a_row_does_not_depend_on_its_turn(lo):
    """Rows by themselves (a turn each) give the bits that they have in the middle of a long call, views of wider rows included."""
    for C, groups, dtype in SHAPES:
        whole, _ = _rows_of_one_turn(C, groups, dtype)
        n = int(whole * 4.5) | 1
        wide = _inputs((n, C + 16), dtype)[0]
        x = wide[:, 8:8 + C]
        y = lo.group_norm(x, groups, activation="silu")
        for at in (0, whole - 1, whole, 2 * whole + 3, n - 1):
            assert torch.equal(y[at:at + 1], lo.group_norm(x[at:at + 1], groups, activation="silu")), (C, groups, at)
