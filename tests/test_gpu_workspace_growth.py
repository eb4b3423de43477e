"""A workspace that grows after a call on it was captured: the graph's replays stay right and write no one else's memory."""
import pytest
import torch

from heterocache_b200 import ops
from paged_reference import D, DT, Cache, attention_tolerance, softmax_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_replay_after_growth(cuda_device, dt):
    dev, dtype, H, KV, G = cuda_device, DT[dt], 8, 2, 4
    c = Cache([900, 700], dtype, dev)
    q = torch.randn(1, H, 1, D, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
    s = torch.tensor([600, 300], dtype=torch.int32, device=dev)
    ws, out = ops.Workspace(dev), torch.empty(1, H, D, dtype=dtype, device=dev)
    call = lambda: ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV, workspace=ws,  # noqa: E731
                                           err=c.err, out=out)
    call()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        call()
    size = ws.buf.numel()
    many = Cache([300] * (64 * KV), dtype, dev)
    ops.flash_decode_shared(torch.zeros(64, H, 1, D, dtype=dtype, device=dev), many.kp, many.vp, many.table, many.lens,
                            torch.zeros(KV, dtype=torch.int32, device=dev), num_kv_heads=KV, workspace=ws, err=c.err)
    assert ws.buf.numel() > size
    others = [torch.full((size // 4,), i, dtype=torch.int32, device=dev) for i in range(8)]
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert int(c.err) == 0 and all(bool((x == i).all()) for i, x in enumerate(others))
    want = torch.zeros(1, H, D, dtype=torch.float64, device=dev)
    ks, vs, qs = [], [], []
    for r in range(KV):
        k, v = c.rows(r)
        x = q[0, r * G:(r + 1) * G, 0].double()
        want[0, r * G:(r + 1) * G] = softmax_rows(x, k, v, D ** -0.5)
        ks.append(k), vs.append(v), qs.append(x)
    tol = attention_tolerance(dtype, qs, ks, vs, D ** -0.5, 900)
    assert float((out.double() - want).abs().max()) <= tol
