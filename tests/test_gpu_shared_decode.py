"""ops.flash_decode_shared against plain 64-bit attention over the shared tokens and each row's own."""
import pytest
import torch

from heterocache_b200 import ops
from paged_reference import D, DT, PAGE, Cache, attention_tolerance, softmax_rows

pytestmark = pytest.mark.gpu


def _setup(bsz, H, KV, shared, tails, dtype, dev, seed=0, own_pages=True):
    """Sequence 0's rows hold the shared tokens; the other rows' first pages
    are theirs only from the page in which the shared tokens end (-1 before)."""
    lens = [shared[h] + tails[b][h] for b in range(bsz) for h in range(KV)]
    c = Cache(lens, dtype, dev, seed=seed)
    for r in range(KV, bsz * KV):
        c.table[r, :shared[r % KV] // PAGE] = -1
    q = torch.randn(bsz, H, 1, D, generator=torch.Generator().manual_seed(seed + 1)).to(dtype).to(dev)
    return c, q, torch.tensor(shared, dtype=torch.int32, device=dev)


def _reference(c, q, shared, bsz, H, KV, scale=D ** -0.5, new=None):
    G = H // KV
    out = torch.zeros(bsz, H, D, dtype=torch.float64, device=q.device)
    ks, vs, qs = [], [], []
    for h in range(KV):
        n = int(shared[h])
        t = torch.arange(n, device=q.device)
        page = c.table[h].long()[t // PAGE]
        k0, v0 = c.kp[page, t % PAGE, 0].double(), c.vp[page, t % PAGE, 0].double()
        for b in range(bsz):
            r = b * KV + h
            m = int(c.lens[r])
            t = torch.arange(n, max(n, m), device=q.device)
            page = c.table[r].long()[t // PAGE]
            k = torch.cat([k0, c.kp[page, t % PAGE, 0].double()])
            v = torch.cat([v0, c.vp[page, t % PAGE, 0].double()])
            if new is not None:
                k, v = torch.cat([k, new[0][b, h].double()]), torch.cat([v, new[1][b, h].double()])
            x = q[b, h * G:(h + 1) * G, 0].double()
            out[b, h * G:(h + 1) * G] = softmax_rows(x, k, v, scale)
            ks.append(k), vs.append(v), qs.append(x)
    n = max(k.shape[0] for k in ks)
    return out, attention_tolerance(q.dtype, qs, ks, vs, scale, n)


CASES = [
    # bsz, H, KV, shared, longest tail
    (1, 4, 1, [1], 0),
    (1, 8, 8, [0, 1, 63, 64, 65, 127, 128, 300], 5),
    (2, 32, 8, [256, 0, 1000, 31, 32, 33, 255, 257], 70),
    (4, 28, 4, [600, 511, 129, 1], 300),
    (5, 32, 4, [700, 128, 0, 64], 20),
    (9, 16, 2, [2000, 3], 100),
    (17, 32, 4, [513, 700, 1, 130], 40),   # 136 query rows: over 128
    (33, 64, 8, [300, 200, 100, 50, 25, 12, 6, 3], 10),  # 264: over 256
    (70, 8, 2, [900, 40], 3),
]


@pytest.mark.parametrize("bsz,H,KV,shared,tail", CASES)
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_matches_plain(cuda_device, bsz, H, KV, shared, tail, dt):
    g = torch.Generator().manual_seed(bsz)
    tails = torch.randint(0, tail + 1, (bsz, KV), generator=g).tolist()
    c, q, s = _setup(bsz, H, KV, shared, tails, DT[dt], cuda_device, seed=bsz)
    ref, tol = _reference(c, q, s, bsz, H, KV)
    out = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV,
                                  workspace=ops.Workspace(cuda_device), err=c.err)
    assert out.dtype == q.dtype and int(c.err) == 0
    assert float((out.double() - ref).abs().max()) <= tol


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_long_prefix(cuda_device, dt):
    """Splits of the prefix over all SMs, joined; one head far longer than the others."""
    bsz, H, KV, shared = 6, 32, 4, [20000, 100, 0, 4097]
    tails = [[7, 0, 300, 1]] * bsz
    c, q, s = _setup(bsz, H, KV, shared, tails, DT[dt], cuda_device, seed=2)
    ref, tol = _reference(c, q, s, bsz, H, KV)
    out = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV,
                                  workspace=ops.Workspace(cuda_device), err=c.err)
    assert int(c.err) == 0 and float((out.double() - ref).abs().max()) <= tol
    # a reference rounded once is as far off as the kernel, to a factor: no split went missing
    rel = float((out.double() - ref).norm() / ref.norm())
    assert rel <= {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -16}[dt]


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_new_token_strides_scale_and_out(cuda_device, dt):
    bsz, H, KV, shared = 3, 8, 2, [130, 0]
    dtype = DT[dt]
    c, q, s = _setup(bsz, H, KV, shared, [[0, 0], [5, 0], [64, 1]], dtype, cuda_device)
    wide = torch.zeros(bsz, H, 3, 2 * D, dtype=dtype, device=cuda_device)
    wide[:, :, 1:2, :D] = q
    q = wide[:, :, 1:2, :D]
    kn = torch.randn(bsz, 2 * KV, 1, D, device=cuda_device).to(dtype)[:, ::2]
    vn = torch.randn(bsz, KV, 2, D, device=cuda_device).to(dtype)[:, :, 1:]
    ref, tol = _reference(c, q, s, bsz, H, KV, scale=0.3, new=(kn, vn))
    out = torch.full((bsz, H, D), 9.0, dtype=dtype, device=cuda_device)
    got = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV, scale=0.3, out=out,
                                  workspace=ops.Workspace(cuda_device), err=c.err, k_new=kn, v_new=vn)
    assert got is out and int(c.err) == 0 and float((out.double() - ref).abs().max()) <= tol


def test_rows_shorter_than_the_prefix_and_empty(cuda_device):
    """A row that is no longer than the prefix attends to the prefix alone; nothing at all gives zeros."""
    bsz, H, KV, shared = 3, 4, 2, [100, 0]
    c, q, s = _setup(bsz, H, KV, shared, [[9, 0]] * 3, torch.bfloat16, cuda_device)
    c.lens[2], c.lens[4] = 0, 60
    ref, tol = _reference(c, q, s, bsz, H, KV)
    out = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV,
                                  workspace=ops.Workspace(cuda_device), err=c.err)
    assert int(c.err) == 0 and float((out.double() - ref).abs().max()) <= tol
    assert (out[:, 2:] == 0).all()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_a_bad_page_is_reported(cuda_device, dt):
    bsz, H, KV, shared = 2, 4, 1, [600]
    c, q, s = _setup(bsz, H, KV, shared, [[3], [4]], DT[dt], cuda_device)
    c.table[0, 1] = c.kp.shape[0] + 5
    ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV, workspace=ops.Workspace(cuda_device),
                            err=c.err)
    assert int(c.err) == 1 << 4
    c.err.zero_()
    c.table[0, 1] = -1
    ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV, workspace=ops.Workspace(cuda_device),
                            err=c.err)
    assert int(c.err) == 1 << 4


def test_large_logits(cuda_device):
    """Logits of some thousands: the running maximum carries every split."""
    bsz, H, KV, shared = 3, 8, 2, [700, 300]
    c, q, s = _setup(bsz, H, KV, shared, [[40, 3]] * 3, torch.bfloat16, cuda_device)
    q = q * 100
    ref, tol = _reference(c, q, s, bsz, H, KV)
    out = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV,
                                  workspace=ops.Workspace(cuda_device), err=c.err)
    assert float((out.double() - ref).abs().max()) <= tol


def test_captured_lengths_change(cuda_device):
    """A graph reads lengths, shared lengths and tables when it is replayed."""
    dev, bsz, H, KV = cuda_device, 4, 8, 2
    c, q, s = _setup(bsz, H, KV, [400, 256], [[60, 30]] * bsz, torch.bfloat16, dev)
    ws = ops.Workspace(dev)
    out = torch.empty(bsz, H, D, dtype=q.dtype, device=dev)
    call = lambda: ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV, workspace=ws,  # noqa: E731
                                           err=c.err, out=out)
    call()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        call()
    for cut in ((0, 0), (30, 1)):
        c.lens -= cut[0]
        s -= cut[1]
        if cut[1]:
            s[0] = 256  # a shorter prefix: the rows' own pages start earlier (page 1 on)
        ref, tol = _reference(c, q, s, bsz, H, KV) if not cut[1] else (None, None)
        g.replay()
        torch.cuda.synchronize()
        if ref is not None:
            assert float((out.double() - ref).abs().max()) <= tol
    assert int(c.err) in (0, 1 << 4)


def test_many_rows_of_one_prompt_equal_plain_decode(cuda_device):
    """With every row's table complete, flash_decode over whole rows gives the same."""
    dev, bsz, H, KV, dtype = cuda_device, 16, 32, 8, torch.bfloat16
    shared = [512 * (1 + h % 3) for h in range(KV)]
    tails = [[(b * 7 + h) % 50 for h in range(KV)] for b in range(bsz)]
    c, q, s = _setup(bsz, H, KV, shared, tails, dtype, dev, seed=4)
    for b in range(1, bsz):
        for h in range(KV):
            n = shared[h] // PAGE
            c.table[b * KV + h, :n] = c.table[h, :n]
    kp, vp = c.kp.nan_to_num(), c.vp.nan_to_num()
    a = ops.flash_decode(q, kp, vp, c.table, c.lens, num_kv_heads=KV, workspace=ops.Workspace(dev), err=c.err)
    b = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV, workspace=ops.Workspace(dev),
                                err=c.err)
    assert int(c.err) == 0
    # both are half a step and a probability's half step from the exact value
    assert float((a.double() - b.double()).abs().max()) <= 4 * 2.0 ** -8 * float(vp.double().abs().max())


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_what_rows_hold_before_their_own_tokens_is_not_read(cuda_device, dt):
    """The page in which the shared tokens end: in the other sequences' copies of it, NaN before their own tokens."""
    bsz, H, KV, shared = 3, 8, 2, [300, 70]
    c, q, s = _setup(bsz, H, KV, shared, [[9, 1], [33, 0], [64, 100]], DT[dt], cuda_device)
    ref, tol = _reference(c, q, s, bsz, H, KV)
    for r in range(KV, bsz * KV):
        n, page = shared[r % KV] % PAGE, int(c.table[r, shared[r % KV] // PAGE])
        c.kp[page, :n], c.vp[page, :n] = float("nan"), float("nan")
    out = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV,
                                  workspace=ops.Workspace(cuda_device), err=c.err)
    assert int(c.err) == 0 and float((out.double() - ref).abs().max()) <= tol


def test_on_another_stream(cuda_device):
    """Append and both attentions on a side stream, ordered by it alone."""
    dev, bsz, H, KV, dtype = cuda_device, 4, 8, 2, torch.bfloat16
    c, q, s = _setup(bsz, H, KV, [700, 400], [[60, 30]] * bsz, dtype, dev)
    ref, tol = _reference(c, q, s, bsz, H, KV)
    ws, side = ops.Workspace(dev), torch.cuda.Stream(dev)
    later = torch.zeros_like(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        later.copy_(q)  # the query is there only when the stream gets to it
        out = ops.flash_decode_shared(later, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV, workspace=ws, err=c.err)
    side.synchronize()
    assert int(c.err) == 0 and float((out.double() - ref).abs().max()) <= tol


def test_a_stalled_prefix_gives_up(cuda_device):
    """No key tile is loaded (injected): every wait runs out, the flag says so, and the next call is right."""
    dev, bsz, H, KV = cuda_device, 5, 8, 2
    c, q, s = _setup(bsz, H, KV, [2000, 300], [[60, 30]] * bsz, torch.bfloat16, dev)
    ref, tol = _reference(c, q, s, bsz, H, KV)
    ws = ops.Workspace(dev)
    call = lambda: ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV, workspace=ws,  # noqa: E731
                                           err=c.err)
    ops.set_wait_limits(5_000_000, inject_stall=True)  # 5 ms
    try:
        call()
        torch.cuda.synchronize()
        assert int(c.err) & (1 << 7)
    finally:
        ops.set_wait_limits(0, inject_stall=False)
    c.err.zero_()
    out = call()
    assert int(c.err) == 0 and float((out.double() - ref).abs().max()) <= tol
