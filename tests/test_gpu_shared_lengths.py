"""ops.flash_decode_shared with lengths that no row can have: reported, and the other rows' outputs stay right.

(Unclamped, the padded length of such a row, (2^31 - 1 + 63) in 32 bits, is negative, and with it the sums over the
rows by which the launch splits its work.)"""
import pytest
import torch

from heterocache_b200 import ops
from paged_reference import D, DT, PAGE, Cache, attention_tolerance, softmax_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [2 ** 31 - 1, 2 ** 30, None])
@pytest.mark.parametrize("full", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_a_length_beyond_the_table(cuda_device, dt, bad, full):
    """``full``: every entry of the row's table is a page, so that no page is missing either."""
    dev, dtype, bsz, KV, H, G = cuda_device, DT[dt], 4, 2, 8, 4
    shared = [300, 100]
    c = Cache([shared[r % KV] + 20 + 7 * r for r in range(bsz * KV)], dtype, dev, width=3, fill=0.0)
    s = torch.tensor(shared, dtype=torch.int32, device=dev)
    q = torch.randn(bsz, H, 1, D, generator=torch.Generator().manual_seed(2)).to(dtype).to(dev)
    lens, wrong = c.lens.tolist(), 5
    c.lens[wrong] = 3 * PAGE + 1 if bad is None else bad
    if full:
        c.table[wrong, 1:] = c.table[wrong, 0]
    out = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV, workspace=ops.Workspace(dev),
                                  err=c.err)
    torch.cuda.synchronize()
    assert int(c.err) == 1 << 4
    for r, n in enumerate(lens):
        if r == wrong:
            continue
        h = r % KV
        (k0, v0), (k1, v1) = c.rows(h, shared[h]), c.rows(r, n)
        k, v = torch.cat([k0, k1[shared[h]:]]), torch.cat([v0, v1[shared[h]:]])
        x = q[r // KV, h * G:(h + 1) * G, 0].double()
        tol = attention_tolerance(dtype, [x], [k], [v], D ** -0.5, k.shape[0])
        off = out[r // KV, h * G:(h + 1) * G].double() - softmax_rows(x, k, v, D ** -0.5)
        assert float(off.abs().max()) <= tol, r
    # the next call, with the lengths mended, is right for every row
    c.err.zero_()
    c.lens[wrong] = lens[wrong]
    if not full:
        again = ops.flash_decode_shared(q, c.kp, c.vp, c.table, c.lens, s, num_kv_heads=KV,
                                        workspace=ops.Workspace(dev), err=c.err)
        assert int(c.err) == 0 and bool(again.isfinite().all())
