"""ops.flash_decode_shared where a CTA of the prefix part walks many tiles: accumulation and rescaling over tiles,
reuse of its buffers, pages beyond the first 32, several segments; and more KV heads than a warp has lanes.

How far an output may be off, relative to its row's norm: the output's rounding and the probabilities' are half a step
each (16-bit types), a logit is a 32-bit sum of 128 products in the row and in its maximum, the exponential is 2^-22
off, and the 32-bit sums over n terms round n times: at random, sqrt(n) half steps of 2^-24 (four times that here)."""
import math

import pytest
import torch

from heterocache_b200 import ops
from paged_reference import D, DT, PAGE, half_step

pytestmark = pytest.mark.gpu


class _Prefix:
    """Sequences that share their first tokens, in shuffled pages; tails of a few tokens.  Keys grow in one
    direction by ``grow`` (in logits of a query of that direction) over each 1000 tokens, then fall back: a tile of 128
    raises the maximum of the rows that grow by more than the factor 2^8 up to which it is let be."""

    def __init__(self, bsz, H, KV, shared, tail, dtype, dev, seed=0, grow=0.0):
        g = torch.Generator(dev).manual_seed(seed)
        self.bsz, self.H, self.KV, self.G = bsz, H, KV, H // KV
        self.shared, self.lens = shared, [shared[r % KV] + (r * 7) % (tail + 1) for r in range(bsz * KV)]
        pages = lambda n: (n + PAGE - 1) // PAGE  # noqa: E731
        first = [pages(n) for n in shared]
        own = [pages(n) - shared[r % KV] // PAGE for r, n in enumerate(self.lens)]
        total = sum(first) + sum(own[KV:]) + sum(pages(n) - first[r] for r, n in enumerate(self.lens[:KV]))
        ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((bsz * KV, max(pages(n) for n in self.lens) + 1), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(self.lens):
            start = 0 if r < KV else shared[r % KV] // PAGE
            m = pages(max(n, shared[r] if r < KV else n)) - start
            table[r, start:start + m] = torch.tensor(ids[at:at + m], dtype=torch.int32)
            at += m
        assert at == total
        rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
        kp, vp = rnd(total, PAGE, 1, D), rnd(total, PAGE, 1, D).to(dtype)
        self.q = rnd(bsz, H, 1, D)
        if grow:
            u = torch.nn.functional.normalize(rnd(D), dim=0)
            for h in range(KV):
                t = torch.arange(shared[h], device=dev)
                kp[table[h].to(dev)[t // PAGE].long(), t % PAGE, 0] += (t % 1000 / 1000)[:, None] * grow * u
            # rows that grow, rows that shrink, rows that do neither, in every warp
            self.q += (torch.arange(bsz * H, device=dev) % 3 - 1).view(bsz, H, 1, 1) * math.sqrt(D) * u
        self.kp, self.vp, self.q = kp.to(dtype), vp, self.q.to(dtype)
        self.table = table.to(dev)
        i32 = dict(dtype=torch.int32, device=dev)
        self.s, self.hl, self.err = torch.tensor(shared, **i32), torch.tensor(self.lens, **i32), torch.zeros(1, **i32)

    def span(self, group, tile, ctas):
        """Tiles of a CTA, by the launch's plan: tiles of all heads and row groups over the CTAs."""
        tiles = sum((n + tile - 1) // tile for n in self.shared) * ((self.bsz * self.G + group - 1) // group)
        return (tiles + ctas - 1) // ctas

    def call(self, ws, out=None):
        return ops.flash_decode_shared(self.q, self.kp, self.vp, self.table, self.hl, self.s, num_kv_heads=self.KV,
                                       workspace=ws, err=self.err, out=out)

    def check(self, out, seqs=None):
        dev, worst = out.device, 0.0
        for h in range(self.KV):
            n = int(self.s[h])
            t = torch.arange(n, device=dev)
            page = self.table[h].long()[t // PAGE]
            k0, v0 = self.kp[page, t % PAGE, 0].double(), self.vp[page, t % PAGE, 0].double()
            for b in seqs or range(self.bsz):
                r = b * self.KV + h
                t = torch.arange(n, max(n, int(self.hl[r])), device=dev)
                page = self.table[r].long()[t // PAGE]
                k = torch.cat([k0, self.kp[page, t % PAGE, 0].double()])
                v = torch.cat([v0, self.vp[page, t % PAGE, 0].double()])
                x = self.q[b, h * self.G:(h + 1) * self.G, 0].double()
                got = out[b, h * self.G:(h + 1) * self.G].double()
                if k.shape[0] == 0:
                    assert (got == 0).all()
                    continue
                want = torch.softmax(x @ k.T * D ** -0.5, -1) @ v
                logit = 130 * 2.0 ** -24 * float((x.abs() @ k.abs().T).max()) * D ** -0.5 + 2.0 ** -22
                tol = 2 * logit + 8 * math.sqrt(k.shape[0]) * 2.0 ** -24
                if out.dtype != torch.float32:
                    tol += 2 * half_step(out.dtype)
                off = (got - want).norm(dim=-1) / want.norm(dim=-1)
                assert bool((off <= tol).all()), (b, h, float(off.max()), tol)


def _sms(dev):
    return torch.cuda.get_device_properties(dev).multi_processor_count


@pytest.mark.parametrize("grow", [0.0, 60.0])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("bsz,H,KV,shared,group,least", [
    (4, 16, 4, [40000] * 4, 128, 9),                      # 16 rows: both streams have them
    (4, 16, 4, [40000, 33, 25001, 60000], 128, 7),        # CTAs that cross segments after several tiles
    (31, 16, 4, [30000, 5000, 30001, 29999], 128, 5),     # 124 rows
    (80, 16, 4, [30000] * 4, 256, 13),                    # 320 rows: in the last group stream 1 has none
    (100, 16, 4, [30000, 1000, 20000, 128], 256, 5),      # 400 rows: in the last group stream 1 has 16
])
def test_many_tiles(cuda_device, bsz, H, KV, shared, group, least, dt, grow):
    p = _Prefix(bsz, H, KV, shared, 5, DT[dt], cuda_device, seed=bsz, grow=grow)
    assert p.span(group, 128, _sms(cuda_device)) >= least
    ws = ops.Workspace(cuda_device)
    out = p.call(ws)
    assert int(p.err) == 0
    p.check(out, range(0, bsz, max(1, bsz // 9)))
    assert torch.equal(out, p.call(ws))  # the same bits again


def test_a_span_of_more_than_32_pages(cuda_device):
    """The page ids of a CTA's span come 32 at a time."""
    p = _Prefix(340, 16, 2, [60000, 59990], 3, torch.bfloat16, cuda_device, seed=1, grow=30.0)
    assert p.span(256, 128, _sms(cuda_device)) > 66
    out = p.call(ops.Workspace(cuda_device))
    assert int(p.err) == 0
    p.check(out, [0, 1, 31, 32, 100, 255, 256, 338, 339])


@pytest.mark.parametrize("grow", [0.0, 60.0])
@pytest.mark.parametrize("bsz,H,KV,shared", [(2, 16, 4, [20000, 100, 30001, 9000]), (5, 16, 4, [20000] * 4),
                                             (20, 16, 4, [12000] * 4), (40, 16, 4, [9000, 64, 8999, 33])])
def test_many_tiles_fp32(cuda_device, bsz, H, KV, shared, grow):
    """16, 32 and 64 rows a CTA, one or more groups."""
    p = _Prefix(bsz, H, KV, shared, 5, torch.float32, cuda_device, seed=bsz, grow=grow)
    rows = bsz * H // KV
    group = 16 if rows <= 16 else 32 if rows <= 32 else 64
    assert p.span(group, 32, 2 * _sms(cuda_device)) >= 4
    out = p.call(ops.Workspace(cuda_device))
    assert int(p.err) == 0
    p.check(out, range(0, bsz, max(1, bsz // 9)))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("KV", [33, 70])
def test_more_kv_heads_than_lanes(cuda_device, KV, dt):
    shared = [(137 * h * h) % 900 for h in range(KV)]
    p = _Prefix(3, 2 * KV, KV, shared, 40, DT[dt], cuda_device, seed=KV)
    out = p.call(ops.Workspace(cuda_device))
    assert int(p.err) == 0
    p.check(out)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_a_graph_reads_lengths_and_tables_at_its_replay(cuda_device, dt):
    """Lengths, shared lengths (0 among them) and page tables change between replays; each replay's output is theirs."""
    dev, bsz, H, KV = cuda_device, 4, 8, 2
    p = _Prefix(bsz, H, KV, [3000, 1024], 200, DT[dt], dev, seed=3)
    for r in range(KV, bsz * KV):  # every row's table complete
        n = p.shared[r % KV] // PAGE
        p.table[r, :n] = p.table[r % KV, :n]
    ws, out = ops.Workspace(dev), torch.empty(bsz, H, D, dtype=p.q.dtype, device=dev)
    p.call(ws, out)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        p.call(ws, out)
    lens, table = p.hl.clone(), p.table.clone()
    for shared, cut, turn in (([3000, 1024], 0, 0), ([2560, 0], 40, 0), ([0, 0], 0, 1), ([256, 1024], 900, 1),
                              ([2999, 1023], 1, 0), ([3000, 1024], 0, 0)):
        p.s.copy_(torch.tensor(shared, dtype=torch.int32))
        p.hl.copy_((lens - cut).clamp_min(0))
        p.table.copy_(table)
        if turn:  # the rows' first two pages change places
            p.table[:, 0], p.table[:, 1] = table[:, 1], table[:, 0]
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert int(p.err) == 0
        p.check(out)
