"""Edges of the paged cache on the GPU, at sizes and values where a rounding, a
limit or an address goes wrong. Worlds and 64-bit forms are those of
test_paged_gpu.py and paged_ref.py."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tests.test_paged_gpu import ints

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


# ---------------------------------------------------------------- select: tables next to the 48 KB default
SELECT_TABLES = """
import sys
sys.path.insert(0, {root!r})
import torch
import __graft_entry__ as ge
from tests.test_paged_gpu import World, check_select
pkg, cuda = ge.load_package(), torch.device("cuda", 0)
d, batch = {d}, {batch}
for pages in (9200, 9700, 10240, 11200, 11700, 12000, 12288):  # ascending: no call is covered by a larger one before it
    w = World([900, 16, 333, 0] + [40] * (batch - 4), 2, d, 8, "fp16")
    w.table = [row[:w.width] + [-7] * (pages - w.width) for row in w.table]
    w.width = pages
    check_select(pkg, cuda, w, 4, 2, d, "fp16", 7)
print("all tables done")
"""


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("batch", [4, 80])
def test_select_from_tables_near_the_default_shared_memory(pkg, cuda, d, batch):
    """Ranks that fit 48 KB by themselves but not beside the block's own variables, each width the largest of its
    process so far; few pairs run in blocks of 512 threads, many in blocks of 256."""
    r = subprocess.run([sys.executable, "-c", SELECT_TABLES.format(root=str(ROOT), d=d, batch=batch)], cwd=ROOT,
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "all tables done" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


# ---------------------------------------------------------------- errors
def test_a_failed_call_leaves_no_error_for_the_next(pkg, cuda):
    """A refused allocation is reported by its own call and not by a later launch."""
    small = pkg.CUDAAttention(None, 160, 2, 16, {"headDim": 80, "ropeTheta": 1e4})
    qkv, pos = torch.ones(1, 480, dtype=torch.float16, device=cuda), ints([0], cuda)
    exp = small.decode(qkv, pos)
    with pytest.raises(pkg.TlaError, match="OUT_OF_MEMORY"):
        pkg.CUDAAttention(None, 64 * 256, 64, (1 << 31) - 1, {"headDim": 256, "maxBatch": 1024})
    assert torch.equal(small.decode(qkv, pos), exp)
