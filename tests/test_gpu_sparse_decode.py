"""Block bounds, block selection and the decode attention over listed blocks, against plain 64-bit forms."""
import math

import pytest
import torch

from heterocache_b200 import ops
from paged_reference import (BLOCK, D, DT, Cache, attention_tolerance, block_scores, pick, rng_lens, softmax_rows)

pytestmark = pytest.mark.gpu


def _bounds(c, dev):
    lim = torch.full((c.kp.shape[0], 4, 2, D), float("nan"), dtype=c.kp.dtype, device=dev)
    ops.block_bounds(c.kp, c.table, c.lens, lim, c.err)
    return lim


def _expected(c, q, lim, KV, n_select, sink, recent):
    bsz, H = q.shape[:2]
    G, lists = H // KV, []
    for r in range(bsz * KV):
        m = (int(c.lens[r]) + BLOCK - 1) // BLOCK
        j = torch.arange(m, device=q.device)
        at = lim[c.table[r].long()[j // 4], j % 4]
        x = q[r // KV, r % KV * G:(r % KV + 1) * G, 0]
        u = block_scores(x, at[:, 0], at[:, 1]).tolist() if m else []
        lists.append(pick(u, n_select, sink, recent))
    return lists


def _attend(c, q, lists, KV, scale=D ** -0.5):
    bsz, H = q.shape[:2]
    G = H // KV
    out = torch.zeros(bsz, H, D, dtype=torch.float64, device=q.device)
    ks, vs, qs = [], [], []
    for r, blocks in enumerate(lists):
        n = int(c.lens[r])
        k, v = c.rows(r)
        t = [x for j in blocks for x in range(j * BLOCK, min(n, (j + 1) * BLOCK))]
        t = torch.tensor(t, dtype=torch.long, device=q.device)
        x = q[r // KV, r % KV * G:(r % KV + 1) * G, 0].double()
        out[r // KV, r % KV * G:(r % KV + 1) * G] = softmax_rows(x, k[t], v[t], scale)
        ks.append(k[t]), vs.append(v[t]), qs.append(x)
    n = max(len(x) for x in lists) * BLOCK
    return out, attention_tolerance(q.dtype, qs, ks, vs, scale, n)


def _query(bsz, H, dtype, dev, seed=3):
    return torch.randn(bsz, H, 1, D, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_bounds(cuda_device, dt):
    lens = [0, 1, 63, 64, 65, 256, 257, 700]
    c = Cache(lens, DT[dt], cuda_device)
    lim = _bounds(c, cuda_device)
    for r, n in enumerate(lens):
        k, _ = c.rows(r)
        for j in range((n + BLOCK - 1) // BLOCK):
            part = k[j * BLOCK:(j + 1) * BLOCK]
            at = lim[int(c.table[r, j // 4]), j % 4].double()
            assert torch.equal(at[0], part.amin(0)) and torch.equal(at[1], part.amax(0)), (r, j)
    # blocks of nobody stay as they were
    n_blocks = sum((n + BLOCK - 1) // BLOCK for n in lens)
    assert int((~lim.isnan()).all(-1).all(-1).sum()) == n_blocks and int(c.err) == 0


def test_bounds_of_some_rows_and_the_last_tokens(cuda_device):
    lens = [500, 70, 300, 0]
    c = Cache(lens, torch.bfloat16, cuda_device)
    full = _bounds(c, cuda_device)
    lim = torch.full_like(full, float("nan"))
    ops.block_bounds(c.kp, c.table, c.lens, lim, c.err, rows=torch.tensor([2, 0, 3, 0], dtype=torch.int32,
                                                                        device=cuda_device), last=100)
    want = {(0, 6), (0, 7), (2, 3), (2, 4)}  # tokens 400.. of 500, 200.. of 300
    for r, n in enumerate(lens):
        for j in range((n + BLOCK - 1) // BLOCK):
            p = int(c.table[r, j // 4])
            if (r, j) in want:
                assert torch.equal(lim[p, j % 4], full[p, j % 4])
            else:
                assert lim[p, j % 4].isnan().all(), (r, j)
    assert int(c.err) == 0
    ops.block_bounds(c.kp, c.table, c.lens, lim, c.err, rows=torch.tensor([4], dtype=torch.int32, device=cuda_device))
    assert int(c.err) == 1 << 4


def test_bounds_keep_nan_and_infinities(cuda_device):
    c = Cache([130], torch.float16, cuda_device)
    c.kp[int(c.table[0, 0]), 3, 0, 5] = float("nan")
    c.kp[int(c.table[0, 0]), 70, 0, 6] = float("inf")
    c.kp[int(c.table[0, 0]), 129, 0, 7] = -float("inf")
    lim = _bounds(c, cuda_device)[int(c.table[0, 0])]
    assert lim[0, :, 5].isnan().all() and lim[1, 1, 6] == math.inf and lim[2, 0, 7] == -math.inf
    assert int(lim[:3].isnan().sum()) == 2


CASES = [
    # bsz, H, KV, least and greatest length, n_select, sink, recent
    (1, 4, 1, 0, 0, 4, 1, 1),
    (1, 8, 8, 1, 70, 1, 0, 1),
    (1, 32, 8, 200, 900, 5, 1, 2),
    (2, 28, 4, 0, 3000, 9, 0, 0),
    (3, 64, 8, 1000, 5000, 16, 2, 3),
    (1, 8, 8, 9000, 40000, 64, 1, 2),
    (4, 8, 4, 500, 600, 10, 5, 5),
    (2, 4, 4, 4096, 4096, 63, 1, 1),
    (30, 32, 8, 64, 1500, 7, 1, 1),
]


@pytest.mark.parametrize("bsz,H,KV,lo,hi,n_select,sink,recent", CASES)
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_selection_and_attention(cuda_device, bsz, H, KV, lo, hi, n_select, sink, recent, dt):
    dev, dtype = cuda_device, DT[dt]
    c = Cache(rng_lens(bsz * KV, lo, hi, n_select), dtype, dev, seed=lo)
    q = _query(bsz, H, dtype, dev)
    lim = _bounds(c, dev)
    lists = _expected(c, q, lim, KV, n_select, sink, recent)
    ref, tol = _attend(c, q, lists, KV)
    out, blocks, counts = ops.flash_decode_sparse(q, c.kp, c.vp, c.table, c.lens, lim, num_kv_heads=KV,
                                                  n_select=n_select, sink=sink, recent=recent,
                                                  workspace=ops.Workspace(dev), err=c.err)
    assert int(c.err) == 0
    assert counts.tolist() == [len(x) for x in lists]
    assert blocks.tolist() == [x + [-1] * (n_select - len(x)) for x in lists]
    assert float((out.double() - ref).abs().max()) <= tol


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_equal_scores_go_to_the_lowest_block(cuda_device, dt):
    """All scores equal (a zero query), and runs of equal blocks."""
    dev, dtype, KV, H = cuda_device, DT[dt], 2, 4
    c = Cache([5000, 3000], dtype, dev)
    lim = _bounds(c, dev)
    q = torch.zeros(1, H, 1, D, dtype=dtype, device=dev)
    ws = ops.Workspace(dev)
    sel = lambda **k: ops.block_select(q, lim, c.table, c.lens, num_kv_heads=KV, workspace=ws, err=c.err, **k)[0]  # noqa: E731
    assert sel(n_select=6, sink=0, recent=0).tolist() == [[0, 1, 2, 3, 4, 5]] * 2
    assert sel(n_select=6, sink=1, recent=2).tolist() == [[0, 1, 2, 3, 77, 78], [0, 1, 2, 3, 45, 46]]
    q = _query(1, H, dtype, dev)
    lim.copy_(lim[int(c.table[0, 0]), 0].expand_as(lim))  # every block alike
    assert sel(n_select=4, sink=0, recent=1).tolist() == [[0, 1, 2, 78], [0, 1, 2, 46]]
    # two kinds of block in turn: the better kind's lowest
    j = torch.arange(79, device=dev)
    odd = (j % 2 == 1)[:, None, None]
    at = (c.table[0].long()[j // 4], j % 4)
    lim[at] = torch.where(odd, lim[at] + 1 * q[0, :2, 0].sum(0).sign().to(dtype), lim[at])
    want = _expected(c, q, lim, KV, 10, 0, 0)
    assert sel(n_select=10, sink=0, recent=0).tolist() == want
    assert int(c.err) == 0


def test_close_scores(cuda_device):
    """Scores that differ by less than a 32-bit sum's error, which 64 bits tell apart."""
    dev, KV = cuda_device, 1
    c = Cache([64 * 200], torch.float32, dev)
    lim = _bounds(c, dev)
    q = _query(1, 2, torch.float32, dev)
    base = lim[int(c.table[0, 0]), 0].clone()
    g = torch.Generator().manual_seed(0)
    for j in range(200):
        x = base.clone()
        x[:, 3] += float(torch.rand(1, generator=g)) * 3e-6
        lim[int(c.table[0, j // 4]), j % 4] = x
    want = _expected(c, q, lim, KV, 50, 1, 1)
    got, _ = ops.block_select(q, lim, c.table, c.lens, num_kv_heads=KV, n_select=50, workspace=ops.Workspace(dev),
                              err=c.err)
    assert got.tolist() == want


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_infinite_and_nan_bounds(cuda_device, dt):
    dev, dtype, KV, H = cuda_device, DT[dt], 2, 8
    c = Cache([6400, 6400], dtype, dev)
    lim = _bounds(c, dev)
    page = c.table[0].long()
    for j, (side, value) in {7: (1, math.inf), 20: (0, -math.inf), 33: (0, math.nan), 41: (1, -math.inf)}.items():
        lim[page[j // 4], j % 4, side, 11] = value
    lim[page[12], 2] = torch.tensor([-math.inf, math.inf], dtype=dtype, device=dev)[:, None]
    q = _query(1, H, dtype, dev)
    for n in (3, 8, 30):
        want = _expected(c, q, lim, KV, n, 1, 1)
        got, _ = ops.block_select(q, lim, c.table, c.lens, num_kv_heads=KV, n_select=n,
                                  workspace=ops.Workspace(dev), err=c.err)
        assert got.tolist() == want
    assert int(c.err) == 0


def test_a_length_beyond_the_table_and_a_bad_page(cuda_device):
    dev, KV = cuda_device, 1
    c = Cache([3000], torch.bfloat16, dev, width=12)
    lim, q, ws = _bounds(c, dev), _query(1, 2, torch.bfloat16, dev), ops.Workspace(dev)
    c.lens[0] = 12 * 256 + 1
    got, n = ops.block_select(q, lim, c.table, c.lens, num_kv_heads=KV, n_select=4, workspace=ws, err=c.err)
    assert int(c.err) == 1 << 4 and int(n) == 4 and int(got.max()) < 48
    c.err.zero_()
    c.lens[0] = 3000
    c.table[0, 5] = c.kp.shape[0]
    got, n = ops.block_select(q, lim, c.table, c.lens, num_kv_heads=KV, n_select=4, workspace=ws, err=c.err)
    assert int(c.err) == 1 << 4 and not set(got[0].tolist()) & {20, 21, 22, 23}


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_listed_blocks_given_by_the_caller(cuda_device, dt):
    """Any ascending lists: none, the last block alone, all; a block that is not the row's is reported."""
    dev, dtype, KV, H = cuda_device, DT[dt], 4, 8
    c = Cache([700, 700, 130, 0], dtype, dev)
    q, ws = _query(1, H, dtype, dev), ops.Workspace(dev)
    lists = [[10], list(range(11)), [], []]
    blocks = torch.full((4, 11), -1, dtype=torch.int32, device=dev)
    for r, x in enumerate(lists):
        blocks[r, :len(x)] = torch.tensor(x, dtype=torch.int32)
    counts = torch.tensor([len(x) for x in lists], dtype=torch.int32, device=dev)
    ref, tol = _attend(c, q, lists, KV)
    out = ops.flash_decode_blocks(q, c.kp, c.vp, c.table, c.lens, blocks, counts, num_kv_heads=KV, workspace=ws,
                                  err=c.err)
    assert int(c.err) == 0 and float((out.double() - ref).abs().max()) <= tol
    assert (out[0, 4:] == 0).all()
    blocks[0, 0], counts[2] = 10 ** 6, 1
    blocks[2, 0] = 0
    ref, tol = _attend(c, q, [[], lists[1], [0], []], KV)
    out = ops.flash_decode_blocks(q, c.kp, c.vp, c.table, c.lens, blocks, counts, num_kv_heads=KV, workspace=ws,
                                  err=c.err)
    assert int(c.err) == 1 << 4 and float((out.double() - ref).abs().max()) <= tol


def test_all_blocks_equal_plain_decode(cuda_device):
    dev, KV, H, dtype = cuda_device, 8, 32, torch.bfloat16
    c = Cache(rng_lens(KV, 100, 4000, 1), dtype, dev, fill=0.0)
    q, ws = _query(1, H, dtype, dev), ops.Workspace(dev)
    a = ops.flash_decode(q, c.kp, c.vp, c.table, c.lens, num_kv_heads=KV, workspace=ws, err=c.err)
    b, blocks, counts = ops.flash_decode_sparse(q, c.kp, c.vp, c.table, c.lens, _bounds(c, dev), num_kv_heads=KV,
                                                n_select=63, workspace=ws, err=c.err)
    assert counts.tolist() == ((c.lens + 63) // 64).tolist()
    assert torch.equal(a, b)
