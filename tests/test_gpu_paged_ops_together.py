"""The paged operators one after another, on two streams at once, from graphs, and in pools past 2^31 elements."""
import pytest
import torch

from heterocache_b200 import ops
from paged_reference import D, PAGE, Cache, rng_lens

pytestmark = pytest.mark.gpu
H, KV = 16, 4


class _Decoder:
    """A batch whose sequences share their first tokens: a step appends one
    token a row, then attends both ways."""

    def __init__(self, dev, bsz, seed, dtype=torch.bfloat16, offset=0, pool=None):
        shared = [512, 300, 0, 64]
        lens = [shared[h] + n for b in range(bsz) for h, n in enumerate(rng_lens(KV, 1, 700, seed * 100 + b))]
        c = Cache(lens, dtype, dev, seed=seed, spare=bsz * KV + 3)
        self.c, self.dev, self.dtype, self.seed = c, dev, dtype, seed
        n = c.kp.shape[0]
        if pool:  # the same pages at the end of pools of `pool` pages
            self.kp, self.vp = (torch.zeros(pool, PAGE, 1, D, dtype=dtype, device=dev) for _ in range(2))
            self.kp[pool - n:], self.vp[pool - n:] = c.kp, c.vp
            c.table += (c.table >= 0).int() * (pool - n)
            c.free += pool - n
        else:
            self.kp, self.vp = c.kp, c.vp
        self.n = n
        self.shared = torch.tensor(shared, dtype=torch.int32, device=dev)
        self.ws = ops.Workspace(dev)
        self.bounds = torch.zeros(self.kp.shape[0], 4, 2, D, dtype=dtype, device=dev)
        ops.block_bounds(self.kp, c.table, c.lens, self.bounds, c.err)
        self.q, self.k, self.v = (torch.zeros(bsz, h, 1, D, dtype=dtype, device=dev) for h in (H, KV, KV))
        self.cos, self.sin = (torch.zeros(bsz, 1, D, dtype=dtype, device=dev) for _ in range(2))

    def inputs(self, step):
        g = torch.Generator().manual_seed(1000 * self.seed + step)
        for x in (self.q, self.k, self.v, self.cos, self.sin):
            x.copy_(torch.randn(x.shape, generator=g))

    def step(self):
        c = self.c
        q = ops.rope_append(self.q, self.k, self.v, self.cos, self.sin, self.kp, self.vp, c.table, c.lens, c.free,
                            c.free_ptr, c.err, workspace=self.ws, bounds=self.bounds)
        a = ops.flash_decode_shared(q, self.kp, self.vp, c.table, c.lens, self.shared, num_kv_heads=KV,
                                    workspace=self.ws, err=c.err)
        b, blocks, counts = ops.flash_decode_sparse(q, self.kp, self.vp, c.table, c.lens, self.bounds,
                                                    num_kv_heads=KV, n_select=6, sink=1, recent=2,
                                                    workspace=self.ws, err=c.err)
        return q, a, b, blocks, counts

    def state(self):
        c, n = self.c, self.n
        return [c.lens, c.free_ptr, c.err, self.kp[-n:].nan_to_num(), self.vp[-n:].nan_to_num(),
                self.bounds[-n:]]


def _run(decoder, steps):
    outs = []
    for i in range(steps):
        decoder.inputs(i)
        outs.append([x.clone() for x in decoder.step()])
    return outs


def _same(got, want):
    return all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


STEPS = 12


def test_two_streams_at_once(cuda_device):
    """Two batches with a workspace each, their steps interleaved on two streams: what each gives alone."""
    alone = [_Decoder(cuda_device, bsz, seed) for seed, bsz in ((1, 3), (2, 9))]
    want = [_run(d, STEPS) for d in alone]
    both = [_Decoder(cuda_device, bsz, seed) for seed, bsz in ((1, 3), (2, 9))]
    streams = [torch.cuda.Stream(cuda_device) for _ in both]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(STEPS):
        for d, s, o in zip(both, streams, got):
            with torch.cuda.stream(s):
                d.inputs(i)
                o.append([x.clone() for x in d.step()])
    torch.cuda.synchronize()
    for a, b, x, y in zip(alone, both, want, got):
        assert int(a.c.err) == 0 and _same(y, x) and _same([b.state()], [a.state()])


def test_two_graphs_at_once(cuda_device):
    """A step of each batch in a graph, both replayed at the same time, against eager steps."""
    alone = [_Decoder(cuda_device, bsz, seed) for seed, bsz in ((3, 2), (4, 17))]
    want = [_run(d, STEPS) for d in alone]
    both = [_Decoder(cuda_device, bsz, seed) for seed, bsz in ((3, 2), (4, 17))]
    streams, graphs, outs = [torch.cuda.Stream(cuda_device) for _ in both], [], []
    for d in both:  # the workspaces grow before a capture
        d.inputs(0)
        lens, table, ptr, err = d.c.lens.clone(), d.c.table.clone(), d.c.free_ptr.clone(), d.c.err.clone()
        kp, vp, lim = d.kp.clone(), d.vp.clone(), d.bounds.clone()
        d.step()
        for dst, src in ((d.c.lens, lens), (d.c.table, table), (d.c.free_ptr, ptr), (d.c.err, err), (d.kp, kp),
                         (d.vp, vp), (d.bounds, lim)):
            dst.copy_(src)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(d.step())
        graphs.append(g)
    got = [[], []]
    for i in range(STEPS):
        for d, s, g, o, out in zip(both, streams, graphs, got, outs):
            with torch.cuda.stream(s):
                d.inputs(i)
                g.replay()
                o.append([x.clone() for x in out])
    torch.cuda.synchronize()
    for a, b, x, y in zip(alone, both, want, got):
        assert int(b.c.err) == 0 and _same(y, x) and _same([b.state()], [a.state()])


def test_pools_past_two_to_the_31_elements(cuda_device):
    """Pages whose elements start beyond 2^31 in a 4.6 GB pool, against the same pages in a small one."""
    small, large = _Decoder(cuda_device, 3, 5), _Decoder(cuda_device, 3, 5, pool=70000)
    want, got = _run(small, 6), _run(large, 6)
    assert int(small.c.err) == 0 and _same(got, want) and _same([large.state()], [small.state()])


@pytest.mark.parametrize("last", [2 ** 31 - 1, 2 ** 31 - 62, 100000, 65, 64, 1])
def test_bounds_of_any_number_of_last_tokens(cuda_device, last):
    """``last`` may be any count; blocks before the last tokens' keep what they held, rows listed twice count once."""
    lens = [0, 1, 64, 65, 300, 513]
    c = Cache(lens, torch.bfloat16, cuda_device)
    whole, part = (torch.full((c.kp.shape[0], 4, 2, D), 7.0, dtype=torch.bfloat16, device=cuda_device)
                   for _ in range(2))
    ops.block_bounds(c.kp, c.table, c.lens, whole, c.err)
    rows = torch.tensor([5, 0, 1, 2, 3, 4, 5, 5], dtype=torch.int32, device=cuda_device)
    ops.block_bounds(c.kp, c.table, c.lens, part, c.err, rows=rows, last=last)
    assert int(c.err) == 0
    for r, n in enumerate(lens):
        for j in range((n + 63) // 64):
            page = int(c.table[r, j // 4])
            want = whole[page, j % 4] if j >= max(0, n - last) // 64 else torch.full_like(whole[0, 0], 7.0)
            assert torch.equal(part[page, j % 4], want), (r, j)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("own", [1, 2, 3, 63, 66])
def test_an_infinite_value_of_the_last_token(cuda_device, dt, own):
    """Infinity times a probability that is not zero is infinity, in its dim alone; what is behind it adds nothing."""
    lens = [64 + own] * KV
    c = Cache(lens, dt, cuda_device)
    for r in range(KV):
        c.vp[c.table[r, 0], lens[r] - 1, 0, 5] = float("inf")
    q = torch.randn(1, H, 1, D, generator=torch.Generator().manual_seed(1)).to(dt).to(cuda_device)
    shared = torch.full((KV,), 64, dtype=torch.int32, device=cuda_device)
    bounds = torch.zeros(c.kp.shape[0], 4, 2, D, dtype=dt, device=cuda_device)
    ops.block_bounds(c.kp, c.table, c.lens, bounds, c.err)
    ws = ops.Workspace(cuda_device)
    a = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, shared, num_kv_heads=KV, workspace=ws, err=c.err)
    b = ops.flash_decode_sparse(q, c.kp, c.vp, c.table, c.lens, bounds, num_kv_heads=KV, n_select=4, workspace=ws,
                                err=c.err)[0]
    for out in (a, b):
        assert int(c.err) == 0 and (out[..., 5] == float("inf")).all()
        assert out[..., :5].isfinite().all() and out[..., 6:].isfinite().all()
