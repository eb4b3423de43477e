"""Tokens appended as drafts (lengths kept apart) and dropped: the block bounds follow what the rows hold."""
import pytest
import torch

from heterocache_b200 import ops
from paged_reference import BLOCK, D, DT, Cache, rng_lens

pytestmark = pytest.mark.gpu


def _tokens(bsz, KV, T, dtype, dev, seed, big=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (big * torch.randn(bsz, n, T, D, generator=g).to(dtype).to(dev) for n in (2 * KV, KV, KV))
    one, zero = torch.ones(1, T, D, dtype=dtype, device=dev), torch.zeros(1, T, D, dtype=dtype, device=dev)
    return q, k, v, one, zero  # (no rotation: keys go to the pages as they are)


def _check_bounds(c, lim):
    for r in range(len(c.lens)):
        keys, _ = c.rows(r)
        for j in range((keys.shape[0] + BLOCK - 1) // BLOCK):
            part = keys[j * BLOCK:(j + 1) * BLOCK]
            at = lim[int(c.table[r, j // 4]), j % 4].double()
            assert torch.equal(at[0], part.amin(0)) and torch.equal(at[1], part.amax(0)), (r, j)


def _start(lens, dtype, dev, T):
    c = Cache(lens, dtype, dev, width=(max(lens) + 2 * T) // 256 + 2, spare=2 * len(lens) + 3)
    lim = torch.zeros(c.kp.shape[0], 4, 2, D, dtype=dtype, device=dev)
    ops.block_bounds(c.kp, c.table, c.lens, lim, c.err)
    return c, lim


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,then", [(1, 1), (5, 1), (5, 5), (1, 5), (70, 1), (3, 100)])
def test_an_append_after_dropped_drafts(cuda_device, dt, T, then):
    """Drafts far outside the other keys are dropped, other tokens appended in their place."""
    dev, dtype, bsz, KV = cuda_device, DT[dt], 3, 4
    c, lim = _start([0, 1, 62, 63, 64, 65, 100, 191, 192, 255, 256, 300], dtype, dev, max(T, then))
    ws, drafted = ops.Workspace(dev), torch.zeros_like(c.lens)
    for i in range(2):  # drafted, dropped, drafted again
        q, k, v, cos, sin = _tokens(bsz, KV, T, dtype, dev, 7 + i, big=100.0)
        ops.rope_append(q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err, workspace=ws,
                        heads_len_out=drafted, bounds=lim)
        kept, c.lens = c.lens, drafted
        _check_bounds(c, lim)  # with the drafts
        c.lens = kept
    q, k, v, cos, sin = _tokens(bsz, KV, then, dtype, dev, 9)
    ops.rope_append(q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err, workspace=ws,
                    bounds=lim)
    assert int(c.err) == 0
    _check_bounds(c, lim)


@pytest.mark.parametrize("T", [1, 4])
def test_a_dropped_nan_is_gone(cuda_device, T):
    """A NaN key among the drafts keeps its block selected only while the row holds it."""
    dev, dtype, bsz, KV = cuda_device, torch.bfloat16, 1, 2
    c, lim = _start([1000, 700], dtype, dev, T)
    ws, drafted = ops.Workspace(dev), torch.zeros_like(c.lens)
    q, k, v, cos, sin = _tokens(bsz, KV, T, dtype, dev, 1)
    k[0, 1, T - 1] = float("nan")
    args = (cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err)
    ops.rope_append(q, k, v, *args, workspace=ws, heads_len_out=drafted, bounds=lim)
    assert lim[int(c.table[1, 2]), 2].isnan().all()  # token 700 lies in block 10
    q, k, v, _, _ = _tokens(bsz, KV, T, dtype, dev, 2)
    ops.rope_append(q, k, v, *args, workspace=ws, bounds=lim)
    _check_bounds(c, lim)
    assert int(c.err) == 0


def test_bounds_of_the_last_block_after_a_drop(cuda_device):
    """Where nothing is appended after the drop, block_bounds over the last token's block is enough."""
    dev, dtype, bsz, KV, T = cuda_device, torch.bfloat16, 2, 4, 90
    c, lim = _start(rng_lens(8, 1, 600, 5), dtype, dev, T)
    drafted = torch.zeros_like(c.lens)
    q, k, v, cos, sin = _tokens(bsz, KV, T, dtype, dev, 1, big=50.0)
    ops.rope_append(q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err,
                    workspace=ops.Workspace(dev), heads_len_out=drafted, bounds=lim)
    ops.block_bounds(c.kp, c.table, c.lens, lim, c.err, last=1)
    assert int(c.err) == 0
    _check_bounds(c, lim)


@pytest.mark.parametrize("T", [1, 2])
@pytest.mark.parametrize("dt,bsz", [("bf16", 140), ("bf16", 513), ("fp32", 70), ("fp32", 300)])
def test_many_rows(cuda_device, T, dt, bsz):
    """Up to four thousand rows and a few, each with bounds to follow."""
    dev, dtype, KV = cuda_device, DT[dt], 8
    lens = rng_lens(bsz * KV, 0, 300, 3)
    c, lim = _start(lens, dtype, dev, T)
    used = sum((n + T + 255) // 256 - (n + 255) // 256 for n in lens)
    q, k, v, cos, sin = _tokens(bsz, KV, T, dtype, dev, 4)
    ops.rope_append(q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err,
                    workspace=ops.Workspace(dev), bounds=lim)
    assert int(c.err) == 0 and int(c.free_ptr) == used and c.lens.tolist() == [n + T for n in lens]
    fresh = lim.clone()
    ops.block_bounds(c.kp, c.table, c.lens, fresh, c.err)
    assert torch.equal(fresh, lim) and int(c.err) == 0
    pos = c.lens.long() - 1
    row = torch.arange(bsz * KV, device=dev)
    assert torch.equal(c.vp[c.table[row, pos // 256].long(), pos % 256, 0], v[:, :, -1].reshape(-1, D))
