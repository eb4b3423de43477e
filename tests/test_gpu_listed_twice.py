"""ops.flash_decode_blocks over lists that name a block more than once: its tokens count as often."""
import pytest
import torch

from heterocache_b200 import ops
from paged_reference import BLOCK, D, DT, Cache, attention_tolerance, softmax_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_a_block_listed_twice_counts_twice(cuda_device, dt):
    dev, dtype, KV, H = cuda_device, DT[dt], 3, 6
    c = Cache([700, 130, 64], dtype, dev)
    lists = [[2, 2, 5, 10, 10, 10], [0, 2, 2], [0, 0]]
    blocks = torch.full((KV, 6), -1, dtype=torch.int32, device=dev)
    for r, x in enumerate(lists):
        blocks[r, :len(x)] = torch.tensor(x, dtype=torch.int32)
    counts = torch.tensor([len(x) for x in lists], dtype=torch.int32, device=dev)
    q = torch.randn(1, H, 1, D, generator=torch.Generator().manual_seed(3)).to(dtype).to(dev)
    out = ops.flash_decode_blocks(q, c.kp, c.vp, c.table, c.lens, blocks, counts, num_kv_heads=KV,
                                  workspace=ops.Workspace(dev), err=c.err)
    assert int(c.err) == 0
    for r, x in enumerate(lists):
        n = int(c.lens[r])
        k, v = c.rows(r)
        t = torch.tensor([i for j in x for i in range(j * BLOCK, min(n, (j + 1) * BLOCK))], device=dev)
        y = q[0, 2 * r:2 * r + 2, 0].double()
        tol = attention_tolerance(dtype, [y], [k[t]], [v[t]], D ** -0.5, len(t))
        assert float((out[0, 2 * r:2 * r + 2].double() - softmax_rows(y, k[t], v[t], D ** -0.5)).abs().max()) <= tol
