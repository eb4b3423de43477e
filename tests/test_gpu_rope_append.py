"""ops.rope_append against a plain 64-bit rotation and page bookkeeping on the host."""
import pytest
import torch

from heterocache_b200 import ops
from paged_reference import BLOCK, D, DT, PAGE, Cache, half_step, rng_lens, rotate

pytestmark = pytest.mark.gpu


def _inputs(bsz, H, KV, T, dtype, dev, seed, trig=None, layout="proj"):
    g = torch.Generator().manual_seed(seed)

    def heads(n):
        x = torch.randn(bsz, T, n, D, generator=g).to(dtype).to(dev)
        return x.transpose(1, 2) if layout == "proj" else x.transpose(1, 2).contiguous()
    ang = torch.rand(bsz, T, D, generator=g, dtype=torch.float64) * 6.3
    cos, sin = ang.cos().to(trig or dtype).to(dev), ang.sin().to(trig or dtype).to(dev)
    return heads(H), heads(KV), heads(KV), cos, sin


def _tables_after(table, lens, counts, KV, free):
    """Page table, lengths and free pages used after the append."""
    table, at, ends = [list(t) for t in table], 0, []
    for r, n in enumerate(lens):
        end = n + counts[r // KV]
        for p in range(n // PAGE, (end + PAGE - 1) // PAGE if end > n else n // PAGE):
            if table[r][p] == -1:
                table[r][p] = free[at]
                at += 1
        ends.append(end)
    return table, ends, at


def _check_rotated(got, x, cos, sin):
    """One rounding to the type, and two half steps of 2^-24 of each product."""
    ref = rotate(x, cos, sin)
    a, z = x.double()[..., :64].abs(), x.double()[..., 64:].abs()
    c, s = cos.double().abs(), sin.double().abs()
    size = torch.cat([a * c[..., :64] + z * s[..., :64], z * c[..., 64:] + a * s[..., 64:]], -1)
    r = 0.0 if got.dtype == torch.float32 else half_step(got.dtype)
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # a subnormal's step
    tol = r * ref.abs() + (1 + r) * 2 * 2.0 ** -24 * size + tiny
    assert ((got.double() - ref).abs() <= tol).all()


CASES = [
    # bsz, H, KV, T, least and greatest past length, type, type of cos and sin
    (1, 32, 8, 1, 0, 0, "bf16", None),
    (1, 32, 8, 1, 255, 257, "bf16", "fp32"),
    (3, 28, 4, 1, 60, 70, "fp16", None),
    (5, 8, 8, 1, 250, 520, "fp32", None),
    (2, 7, 1, 3, 0, 130, "bf16", None),
    (3, 32, 8, 63, 100, 300, "fp16", "fp32"),
    (2, 32, 8, 64, 0, 64, "bf16", None),
    (2, 16, 2, 65, 190, 260, "fp32", None),
    (2, 28, 4, 700, 1, 600, "bf16", "fp32"),
    (70, 8, 8, 1, 200, 300, "bf16", None),
    (40, 8, 8, 5, 250, 256, "fp16", None),
]


@pytest.mark.parametrize("bsz,H,KV,T,lo,hi,dt,trig", CASES)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("bounds", [False, True])
def test_append_matches_plain(cuda_device, bsz, H, KV, T, lo, hi, dt, trig, ragged, bounds):
    dev, dtype = cuda_device, DT[dt]
    lens = rng_lens(bsz * KV, lo, hi, T + lo)
    counts = rng_lens(bsz, 0, T, 7) if ragged else [T] * bsz
    total = sum((counts[r // KV] + PAGE - 1) // PAGE + 1 for r in range(bsz * KV))
    c = Cache(lens, dtype, dev, seed=T, width=(hi + T + PAGE - 1) // PAGE + 1, spare=total)
    q, k, v, cos, sin = _inputs(bsz, H, KV, T, dtype, dev, 5, DT[trig] if trig else None)
    table, ends, used = _tables_after(c.table.tolist(), lens, counts, KV, c.free.tolist())
    before = {n: getattr(c, n).clone() for n in ("kp", "vp")}
    lim = None
    if bounds:
        lim = torch.full((c.kp.shape[0], 4, 2, D), 7.0, dtype=dtype, device=dev)
        ops.block_bounds(c.kp, c.table, c.lens, lim, c.err)
    q_out = torch.full(q.shape, 3.0, dtype=dtype, device=dev)
    ws = ops.Workspace(dev)
    got = ops.rope_append(q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err, workspace=ws,
                          counts=torch.tensor(counts, dtype=torch.int32, device=dev) if ragged else None, q_out=q_out,
                          bounds=lim)
    torch.cuda.synchronize()
    assert got is q_out and int(c.err) == 0 and int(ws.counter.abs().sum()) == 0
    assert c.table.tolist() == table and c.lens.tolist() == ends and int(c.free_ptr) == used
    written = torch.zeros(c.kp.shape[:2], dtype=torch.bool)
    for b in range(bsz):
        n = counts[b]
        _check_rotated(got[b, :, :n], q[b, :, :n], cos[b, :n], sin[b, :n])
        assert (got[b, :, n:] == 3.0).all()
        for h in range(KV):
            r = b * KV + h
            t = torch.arange(lens[r], ends[r])
            page = torch.tensor(table[r])[t // PAGE]
            written[page, t % PAGE] = True
            _check_rotated(c.kp[page, t % PAGE, 0], k[b, h, :n], cos[b, :n], sin[b, :n])
            assert torch.equal(c.vp[page, t % PAGE, 0], v[b, h, :n])
    same = ~written.to(dev)
    for n in ("kp", "vp"):  # nothing else is written (NaN compares as bits)
        kind = torch.int32 if dtype == torch.float32 else torch.int16
        assert torch.equal(getattr(c, n)[same].view(kind), before[n][same].view(kind))
    if bounds:
        for r in range(bsz * KV):
            keys, _ = c.rows(r)
            for j in range((ends[r] + BLOCK - 1) // BLOCK):
                part = keys[j * BLOCK:(j + 1) * BLOCK]
                at = lim[table[r][j // 4], j % 4].double()
                assert torch.equal(at[0], part.amin(0)) and torch.equal(at[1], part.amax(0)), (r, j)


def test_steps_then_a_chunk(cuda_device):
    """Single tokens, a chunk, single tokens: the rows hold all of them in order, and the bounds are those of the pages."""
    dev, dtype, KV, H, bsz = cuda_device, torch.bfloat16, 4, 8, 2
    c = Cache([0] * (bsz * KV), dtype, dev, width=4, spare=8 * 4)
    lim = torch.zeros(c.kp.shape[0], 4, 2, D, dtype=dtype, device=dev)
    ws, seen = ops.Workspace(dev), []
    for i, T in enumerate([1, 1, 300, 1, 63, 1]):
        q, k, v, cos, sin = _inputs(bsz, H, KV, T, dtype, dev, 50 + i)
        ops.rope_append(q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err, workspace=ws,
                        bounds=lim)
        seen.append(v)
    v = torch.cat(seen, 2)
    assert int(c.err) == 0 and c.lens.tolist() == [v.shape[2]] * (bsz * KV)
    fresh = lim.clone()
    ops.block_bounds(c.kp, c.table, c.lens, fresh, c.err)
    for r in range(bsz * KV):
        assert torch.equal(c.rows(r)[1], v[r // KV, r % KV].double())
        for j in range((v.shape[2] + BLOCK - 1) // BLOCK):
            p = int(c.table[r, j // 4])
            assert torch.equal(fresh[p, j % 4], lim[p, j % 4]), (r, j)


def test_in_place_query_shared_angles_and_other_lengths(cuda_device):
    """q_out is q; cos and sin of one sequence for all; new lengths elsewhere, so that the append can be done again."""
    dev, dtype, KV, H, bsz, T = cuda_device, torch.float16, 2, 6, 3, 4
    lens = [254, 10, 300, 0, 63, 64]
    c = Cache(lens, dtype, dev, width=3, spare=9)
    q, k, v, cos, sin = _inputs(bsz, H, KV, T, dtype, dev, 9, layout="dense")
    cos, sin, q0 = cos[:1], sin[0], q.clone()
    new = torch.zeros(6, dtype=torch.int32, device=dev)
    ws = ops.Workspace(dev)
    out = ops.rope_append(q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err, workspace=ws,
                          q_out=q, heads_len_out=new)
    assert out is q
    _check_rotated(q, q0, cos[0], sin)
    assert c.lens.tolist() == lens and new.tolist() == [n + T for n in lens]
    first = (c.table.clone(), c.free_ptr.clone(), c.kp.clone())
    ops.rope_append(q0, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err, workspace=ws,
                    heads_len_out=new)
    for a, b in zip(first, (c.table, c.free_ptr, c.kp)):
        assert torch.equal(a.nan_to_num(), b.nan_to_num())
    assert int(c.err) == 0


@pytest.mark.parametrize("what", ["oom", "count", "length", "page", "table"])
def test_what_cannot_be_appended_leaves_the_cache(cuda_device, what):
    dev, dtype, KV, H, bsz, T = cuda_device, torch.bfloat16, 2, 4, 2, 3
    lens = [255, 256, 10, 511]
    c = Cache(lens, dtype, dev, width=3, spare=3)
    counts = torch.tensor([T, T], dtype=torch.int32, device=dev)
    code = 4
    if what == "oom":
        c.free, code = c.free[:2], 3  # rows 0, 1 and 3 need a page each
    elif what == "count":
        counts[1] = T + 1
    elif what == "length":
        c.lens[2] = -1
    elif what == "page":
        c.table[0, 0] = c.kp.shape[0]
    else:
        c.table, counts = c.table[:, :2].contiguous(), counts  # row 3 reaches a third page
    q, k, v, cos, sin = _inputs(bsz, H, KV, T, dtype, dev, 3)
    names = ("kp", "vp", "table", "lens", "free_ptr")
    before = [getattr(c, n).clone() for n in names]
    ws = ops.Workspace(dev)
    ops.rope_append(q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err, workspace=ws,
                    counts=counts)
    torch.cuda.synchronize()
    assert int(c.err) == 1 << code and int(ws.counter.abs().sum()) == 0
    for n, b in zip(names, before):
        assert torch.equal(getattr(c, n).nan_to_num(), b.nan_to_num()), n


def test_no_tokens(cuda_device):
    c = Cache([5, 6], torch.bfloat16, cuda_device)
    q, k, v, cos, sin = _inputs(1, 4, 2, 0, torch.bfloat16, cuda_device, 1)
    out = ops.rope_append(q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err,
                          workspace=ops.Workspace(cuda_device))
    assert out.shape == (1, 4, 0, D) and c.lens.tolist() == [5, 6] and int(c.err) == 0


def test_captured_and_replayed(cuda_device):
    """A decode step in a graph: each replay appends one token, a page is taken where one is needed."""
    dev, dtype, KV, H = cuda_device, torch.bfloat16, 2, 4
    c = Cache([254, 3], dtype, dev, width=2, spare=3)
    ws = ops.Workspace(dev)
    q, k, v, cos, sin = _inputs(1, H, KV, 1, dtype, dev, 1)
    q_out = torch.empty_like(q)
    args = (q, k, v, cos, sin, c.kp, c.vp, c.table, c.lens, c.free, c.free_ptr, c.err)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        ops.rope_append(*args, workspace=ws, q_out=q_out)
    vs = []
    for i in range(5):
        new = _inputs(1, H, KV, 1, dtype, dev, 100 + i)
        for dst, src in zip((q, k, v, cos, sin), new):
            dst.copy_(src)
        g.replay()
        vs.append(new[2])
        _check_rotated(q_out, new[0], new[3][:, None], new[4][:, None])
    assert int(c.err) == 0 and c.lens.tolist() == [259, 8] and int(c.free_ptr) == 1
    for r in range(KV):
        assert torch.equal(c.rows(r)[1][-5:], torch.cat(vs, 2)[0, r].double())
