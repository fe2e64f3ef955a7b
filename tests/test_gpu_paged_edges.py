"""Paged-cache operators on the GPU at the edges of their ranges: counts,
variants and orders of calls that the sizes of an ordinary batch do not reach.
Oracles and tolerances are those of test_gpu_paged.py."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------- assign_pages --
def test_assign_pages_of_any_count_in_a_new_process():
    """Counts around the shared memory that needs no opting in, where no larger call has opted in before."""
    script = """
import sys, torch
import numa_allreduce_b200 as nab
i32 = dict(dtype=torch.int32, device="cuda")
for b in [int(x) for x in sys.argv[1:]]:
    starts = torch.arange(b + 1, **i32)
    r = nab.assign_pages(torch.full((b,), 16, **i32), torch.zeros(b, 2, **i32), torch.arange(b, **i32),
                         torch.zeros(1, **i32), 16, query_start=starts, num_tokens=b)
    assert r.slots.tolist() == [16 * i for i in range(b)] and r.lengths.eq(17).all(), b
    r = nab.assign_pages(torch.full((b,), 16, **i32), torch.zeros(b, 2, **i32), torch.arange(b, **i32),
                         torch.zeros(1, **i32), 16)
    assert r.slots.tolist() == [16 * i for i in range(b)], b
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for counts in (["6135", "6136"], ["6140"], ["6143", "6144", "6145"], ["8192"]):
        p = subprocess.run([sys.executable, "-c", script, *counts], cwd=root, capture_output=True, text=True, timeout=300)
        assert p.returncode == 0, p.stderr[-2000:]
