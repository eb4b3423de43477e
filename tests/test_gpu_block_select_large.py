"""ops.block_select at sizes that take its other forms: four blocks a lane, several turns of a CTA over a row's blocks,
and rows of more blocks than shared memory holds keys.  Page tables name a few hundred pages again and again, so that
many scores are equal and the lowest block has to win."""
import pytest
import torch

from heterocache_b200 import ops
from paged_reference import BLOCK, D, DT, block_scores

pytestmark = pytest.mark.gpu


def _rows(rows, blocks, pages, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    width = (max(blocks) + 3) // 4
    table = torch.randint(0, pages, (rows, width), generator=g, dtype=torch.int32).to(dev)
    a, b = torch.randn(pages, 4, 1, D, generator=g), torch.randn(pages, 4, 1, D, generator=g)
    lim = torch.cat([torch.minimum(a, b), torch.maximum(a, b)], 2).to(dtype).to(dev)
    lens = [n * BLOCK - (r * 13) % BLOCK for r, n in zip(range(rows), blocks)]
    return table, lim, torch.tensor(lens, dtype=torch.int32, device=dev)


def _expected(q, lim, table, blocks, KV, n_select, sink, recent):
    """Ascending lists of each row: the stable order of the scores, highest first."""
    G, lists = q.shape[1] // KV, []
    flat = lim.view(-1, 2, D)
    for r, m in enumerate(blocks):
        j = torch.arange(m, device=q.device)
        x = q[r // KV, r % KV * G:(r % KV + 1) * G, 0]
        score = block_scores(x, flat[:, 0], flat[:, 1])[table[r].long()[j // 4] * 4 + j % 4]
        must = (j < sink) | (j >= m - recent)  # in, whatever the others' scores are
        rest = j[~must][torch.sort(score[~must], descending=True, stable=True).indices]
        lists.append(torch.cat([j[must], rest])[:n_select].sort().values.tolist())
    return lists


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("bsz,KV,G,least,most,n_select,sink,recent", [
    (16, 8, 4, 700, 1000, 64, 1, 2),       # four blocks a lane, for four heads,
    (16, 8, 3, 990, 1000, 33, 0, 0),
    (16, 8, 2, 990, 1001, 64, 0, 1),       # two
    (16, 8, 1, 1, 1000, 7, 1, 1),          # and one
    (64, 8, 4, 995, 1003, 40, 1, 2),       # 512 rows: a CTA has more than one turn
    (64, 8, 7, 995, 1003, 40, 1, 2),
    (1, 8, 4, 4090, 4099, 64, 1, 2),       # around what shared memory holds
    (1, 3, 8, 9000, 9003, 100, 2, 3),      # beyond it
    (1, 3, 1, 9000, 9003, 4200, 2, 3),
])
def test_selection(cuda_device, bsz, KV, G, least, most, n_select, sink, recent, dt):
    dev, dtype, rows = cuda_device, DT[dt], bsz * KV
    blocks = [least + (r * 7) % (most - least + 1) for r in range(rows)]
    table, lim, lens = _rows(rows, blocks, 300, dtype, dev, seed=rows + G)
    q = torch.randn(bsz, KV * G, 1, D, generator=torch.Generator().manual_seed(G)).to(dtype).to(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    got, counts = ops.block_select(q, lim, table, lens, num_kv_heads=KV, n_select=n_select, sink=sink, recent=recent,
                                   workspace=ops.Workspace(dev), err=err)
    want = _expected(q, lim, table, blocks, KV, n_select, sink, recent)
    assert int(err) == 0 and counts.tolist() == [len(x) for x in want]
    assert got.tolist() == [x + [-1] * (n_select - len(x)) for x in want]


def test_nan_and_infinite_scores_of_long_rows(cuda_device):
    """Keys read from global memory: the highest (NaN) and the lowest order as in shared memory."""
    dev, KV = cuda_device, 2
    blocks = [5000, 9001]
    table, lim, lens = _rows(2, blocks, 300, torch.bfloat16, dev, seed=5)
    lim[7, 2, 0, 3], lim[8, 1, 1, 4], lim[9, 0] = float("nan"), float("inf"), -float("inf")
    q = torch.randn(1, 4, 1, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    for n in (3, 30, 3000):
        got, _ = ops.block_select(q, lim, table, lens, num_kv_heads=KV, n_select=n, sink=0, recent=1,
                                  workspace=ops.Workspace(dev), err=err)
        assert got.tolist() == _expected(q, lim, table, blocks, KV, n, 0, 1)
    assert int(err) == 0
