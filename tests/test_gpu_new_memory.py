"""What the operators allocate is PyTorch's own new memory: filled where PyTorch is asked to fill it, and seen where it is asked what it runs."""
import os
import subprocess
import sys

import pytest
import torch

from launched_kernels import kernels
from test_gpu_paged_attention import BF16, I32, _rn, lo  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def _calls(lo):  # noqa: F811
    x, p, f = _rn(2, 40, 3, 64).to(BF16), torch.zeros(40, 1, dtype=I32, device="cuda"), lo.rotary_frequencies([32], device="cuda")
    c, table = lo.paged_cache(8, 16, 3, 64, device="cuda"), torch.arange(8, dtype=I32, device="cuda").reshape(2, 4)
    n = torch.tensor([40, 30], dtype=I32, device="cuda")
    y = _rn(2, 40, 64)
    return {"rotary_axes": (2, lambda: lo.rotary_axes(x, x, p, f, [32])), "paged_cache_read": (1, lambda: lo.paged_cache_read(c, table, n, 20)),
            "paged_attention_step": (1, lambda: lo.paged_attention_step(x[:, 0], c, table, n)),
            "group_norm": (1, lambda: lo.group_norm(y, 4, torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")))}


@pytest.mark.parametrize("name", ["rotary_axes", "paged_cache_read", "paged_attention_step", "group_norm"])
def test_new_memory_is_filled_where_that_is_asked_for(lo, name):  # noqa: F811
    arrays, call = _calls(lo)[name]
    fills = lambda: len(kernels(call, {"FillFunctor": "fill"}))
    plain, want = fills(), call()
    before = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    try:
        torch.use_deterministic_algorithms(True)
        torch.utils.deterministic.fill_uninitialized_memory = True
        assert fills() >= plain + arrays
        got = call()
        torch.utils.deterministic.fill_uninitialized_memory = False
        assert fills() == plain
    finally:
        torch.use_deterministic_algorithms(before[0])
        torch.utils.deterministic.fill_uninitialized_memory = before[1]
    for a, b in zip(*((t if isinstance(t, (tuple, list)) else (t,)) for t in (got, want))):
        assert torch.equal(a, b)


def test_new_memory_is_seen_by_the_profiler():
    """In a process of its own: one that has used the profiler and captures graphs after that finds nothing when it uses it again."""
    code = """
import torch
from lact_b200 import layer_ops
from test_gpu_new_memory import _calls
for name, (arrays, call) in _calls(layer_ops).items():
    call()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        call()
    assert sum(e.name == "aten::empty" for e in prof.events()) >= arrays, name
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.pathsep.join([root, os.path.join(root, "tests")])
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300, env={**os.environ, "PYTHONPATH": path})
    assert r.returncode == 0, r.stdout + r.stderr
