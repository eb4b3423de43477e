"""Forks of several layers, eager and from a graph, and update_rope of several sequences."""
import pytest
import torch

from heterocache_b200.cache import HeteroCache, HeteroCacheConfig, attention_together
from heterocache_b200.roles import derive_runtime_data, synthetic_roles
from heterocache_b200.synthetic import LLAMA_8B, DriftingDecode, prefill_inputs
from paged_reference import D, PAGE, attention_tolerance, half_step, rotate, softmax_rows

pytestmark = pytest.mark.gpu
GEO = LLAMA_8B
H, KV, G = GEO.num_heads, GEO.num_kv_heads, GEO.groups


def _cache(layers, **other):
    data = derive_runtime_data(synthetic_roles(layers, KV, seed=13), layers, KV)
    args = dict(stable_threshold=0.9, real_offload=False, max_gen_len=64, decode_step=50, num_attn_heads=H,
                num_kv_heads=KV, num_layers=layers)
    args.update(other)
    return HeteroCache(HeteroCacheConfig(data, **args))


def _prefill(c, L, seed, dev, layer):
    q, k, v = (t.to(dev) for t in prefill_inputs(GEO, L, seed=seed, dtype=torch.bfloat16, q_positions=32))
    c.update(k, v, layer)
    c.init_coefficient(q, k, layer)
    c.prefill_select(q, k, v, layer)
    return q[:, :, -1:, :].cpu()


def _row(c, r, layer):
    t = torch.arange(int(c.heads_len[layer][r]), device=c.key_pools[layer].device)
    page = c.block_tables[layer][r].long()[t // PAGE]
    return c.key_pools[layer][page, t % PAGE, 0].double(), c.value_pools[layer][page, t % PAGE, 0].double()


def _attend(c, q, layer, bsz=1):
    out = torch.zeros(bsz, H, D, dtype=torch.float64, device=q.device)
    ks, vs, qs = [], [], []
    for r in range(bsz * KV):
        k, v = _row(c, r, layer)
        b, h = r // KV, r % KV
        x = q[b, h * G:(h + 1) * G, 0].double()
        out[b, h * G:(h + 1) * G] = softmax_rows(x, k, v, D ** -0.5)
        ks.append(k), vs.append(v), qs.append(x)
    return out, attention_tolerance(q.dtype, qs, ks, vs, D ** -0.5, max(k.shape[0] for k in ks))


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("defer", [False, True])
def test_steps_of_a_fork_of_two_layers(cuda_device, graph, defer):
    """Each member's outputs are the attention over its own rows, layer by layer, whether the step is launched or
    replayed; a step that is captured advances the host's mirrors once, and is replayed once."""
    dev, L, n, layers = cuda_device, 1500, 3, 2
    prompt = _cache(layers)
    for layer in range(layers):
        q0 = _prefill(prompt, L, 60 + layer, dev, layer)
    group = prompt.fork(n)
    gens = [[DriftingDecode(GEO, seed=10 * layer + i, q0=q0, dtype=torch.bfloat16) for i in range(n)]
            for layer in range(layers)]
    q, k, v = (torch.zeros(layers, n, m, 1, D, dtype=torch.bfloat16, device=dev) for m in (H, KV, KV))
    out = torch.zeros(layers, n, H, D, dtype=torch.bfloat16, device=dev)
    for c in group.members:
        c.prepare_decode(list(range(layers)), q[0, :1])

    def step():
        for layer in range(layers):
            for i, c in enumerate(group.members):
                c.update(k[layer, i:i + 1], v[layer, i:i + 1], layer, {"query_states": q[layer, i:i + 1],
                                                                      "defer_append": defer})
            attention_together(group, q[layer], layer, out=out[layer])
            for i, c in enumerate(group.members):
                c.decode_select(q[layer, i:i + 1], layer)
        for c in group.members:
            c.join_retrievals()

    for t in range(6):
        for layer in range(layers):
            for i in range(n):
                for dst, src in zip((q, k, v), gens[layer][i].step()):
                    dst[layer, i:i + 1].copy_(src)
        if graph and t > 0:  # (the first step makes the workspace)
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g):
                step()
            g.replay()
        else:
            step()
        torch.cuda.synchronize()
        for i, c in enumerate(group.members):
            for layer in range(layers):
                assert c.heads_len[layer].tolist() == c._hlen[layer].tolist()
                want, tol = _attend(c, q[layer, i:i + 1], layer)
                assert float((out[layer, i:i + 1].double() - want).abs().max()) <= tol, (t, i, layer)
                for r in range(KV):  # the step's token is the member's own
                    pk, pv = _row(c, r, layer)
                    assert torch.equal(pk[-1], k[layer, i, r, 0].double()) and torch.equal(pv[-1], v[layer, i, r, 0].double())
    for c in group.members:
        c.check_errors()


@pytest.mark.parametrize("sparse", [0, 40])
def test_update_rope_of_two_sequences(cuda_device, sparse):
    """Two sequences of one length: each one's own angles, pages and attention.  (Blocks enough for every row: the
    block-sparse form attends to all of them.)"""
    dev, L, bsz = cuda_device, 900, 2
    c = _cache(1, sparse_blocks=sparse, max_gen_len=2000)  # (the pool is sized for one: room to decode holds the other)
    q, k, v = (torch.cat([x, y], 0).to(dev) for x, y in zip(*(prefill_inputs(
        GEO, L, seed=70 + i, dtype=torch.bfloat16, q_positions=32) for i in range(bsz))))
    c.update(k, v, 0)
    c.init_coefficient(q, k, 0)
    c.prefill_select(q, k, v, 0)
    g = torch.Generator().manual_seed(1)
    for step in range(5):
        q, k, v = (torch.randn(bsz, n, 1, D, generator=g).to(dev, torch.bfloat16) for n in (H, KV, KV))
        ang = torch.rand(bsz, 1, D, generator=g, dtype=torch.float64) * 6.3
        cos, sin = ang.cos().to(dev, torch.bfloat16), ang.sin().to(dev, torch.bfloat16)
        lens = c.heads_len[0].tolist()
        rq = c.update_rope(q, k, v, cos, sin, 0)
        half = half_step(torch.bfloat16)  # the one rounding; two 32-bit roundings of products below 2^3 beside it
        want = rotate(q, cos[:, None], sin[:, None])
        assert ((rq.double() - want).abs() <= half * want.abs() + 2.0 ** -20).all()
        assert c.heads_len[0].tolist() == [n + 1 for n in lens] == c._hlen[0].tolist()
        want = rotate(k, cos[:, None], sin[:, None])
        for r in range(bsz * KV):
            pk, pv = _row(c, r, 0)
            assert ((pk[-1] - want[r // KV, r % KV, 0]).abs() <= half * want[r // KV, r % KV, 0].abs() + 2.0 ** -20).all()
            assert torch.equal(pv[-1], v[r // KV, r % KV, 0].double())
        want, tol = _attend(c, rq, 0, bsz)
        assert float((c.attention(rq, 0).double() - want).abs().max()) <= tol
    c.check_errors()
