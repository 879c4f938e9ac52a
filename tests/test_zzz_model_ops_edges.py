# SPDX-License-Identifier: Apache-2.0
"""The operators of a decode step over the 4-bit paged cache where they can go
wrong: sizes next to a limit, starts that no program should pass, values far
apart, scratch that is used again at once."""

import subprocess
import sys

import pytest
import torch

from conftest import ROOT, gpu_count

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if gpu_count() == 0:
        pytest.skip("no GPU")


# ---- plan ---------------------------------------------------------------------

PLAN_FIRST = """
import sys
import torch
from vkccl_b200.ops.paging import plan_pages
n = int(sys.argv[1])
i = lambda x: x.to(torch.int32)
ones = torch.ones(n, dtype=torch.int32, device="cuda")
table = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
free = i(torch.arange(n, device="cuda"))
p = plan_pages(torch.zeros_like(ones), ones, table, free, i(torch.tensor([n], device="cuda")), 16, n)
k = torch.arange(n, device="cuda")
assert torch.equal(table[:, 0], i(k)) and (table[:, 1] == -1).all() and torch.equal(p.slots, i(16 * k))
assert torch.equal(p.requests, i(k)) and torch.equal(p.q_starts, i(torch.arange(n + 1, device="cuda")))
assert (p.lens == 1).all() and (p.kv_lens == 1).all() and p.free_count.tolist() == [0]
"""


@pytest.mark.parametrize("batch", [6078, 6079, 6144, 6145])
def test_plan_first_of_a_process_takes_every_batch(batch):
    """Shared memory next to 48 KiB (8 bytes a request and the kernel's own 528): the limit is raised by the first call,
    whichever batch it has."""
    done = subprocess.run([sys.executable, "-c", PLAN_FIRST, str(batch)], capture_output=True, text=True, timeout=200, cwd=ROOT)
    assert done.returncode == 0, done.stderr[-2000:]
