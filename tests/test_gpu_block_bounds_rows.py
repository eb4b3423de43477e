"""block_bounds of listed rows, where the list is empty."""
import pytest
import torch

from heterocache_b200 import ops
from paged_reference import D, Cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("last", [0, 1])
def test_an_empty_list_is_no_row(cuda_device, last):
    c = Cache([500, 70], torch.bfloat16, cuda_device)
    lim = torch.full((c.kp.shape[0], 4, 2, D), 7.0, dtype=torch.bfloat16, device=cuda_device)
    none = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    got = ops.block_bounds(c.kp, c.table, c.lens, lim, c.err, rows=none, last=last)
    assert got is lim and bool((lim == 7.0).all()) and int(c.err) == 0
