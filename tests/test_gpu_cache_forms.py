"""The cache's ways to the paged operators: rotation inside the append, block-sparse decode attention, and
continuations of one prompt that share its pages -- each over whole decode steps with drift checks and retrievals."""
import pytest
import torch

from heterocache_b200 import ops
from heterocache_b200.attention import LlamaAttention, Qwen2Attention
from heterocache_b200.cache import (HeteroCache, HeteroCacheConfig, attention_together, flush_checks_together)
from heterocache_b200.graph import DecodeStepGraph
from heterocache_b200.roles import derive_runtime_data, synthetic_roles
from heterocache_b200.synthetic import LLAMA_8B, DriftingDecode, prefill_inputs
from paged_reference import BLOCK, D, PAGE, attention_tolerance, block_scores, half_step, pick, rotate, softmax_rows

pytestmark = pytest.mark.gpu
GEO = LLAMA_8B
H, KV, G = GEO.num_heads, GEO.num_kv_heads, GEO.groups


def _cache(layers=1, **other):
    data = derive_runtime_data(synthetic_roles(layers, KV, seed=13), layers, KV)
    args = dict(compression_ratio=0.5, stable_threshold=0.9, real_offload=False, max_gen_len=64, decode_step=4,
                num_attn_heads=H, num_kv_heads=KV, num_layers=layers)
    args.update(other)
    return HeteroCache(HeteroCacheConfig(data, **args))


def _prefill(c, L, seed, dev, layer=0):
    q, k, v = prefill_inputs(GEO, L, seed=seed, dtype=torch.bfloat16, q_positions=32)
    qd, kd, vd = q.to(dev), k.to(dev), v.to(dev)
    c.update(kd, vd, layer)
    c.init_coefficient(qd, kd, layer)
    c.prefill_select(qd, kd, vd, layer)
    return q[:, :, -1:, :]


def _row(c, r, layer=0):
    t = torch.arange(int(c.heads_len[layer][r]), device=c.key_pools[layer].device)
    page = c.block_tables[layer][r].long()[t // PAGE]
    return c.key_pools[layer][page, t % PAGE, 0].double(), c.value_pools[layer][page, t % PAGE, 0].double()


def _attend(c, q, layer=0):
    """Attention of one sequence over its cache's rows, and the tolerance."""
    out = torch.zeros(1, H, D, dtype=torch.float64, device=q.device)
    ks, vs, qs = [], [], []
    for r in range(KV):
        k, v = _row(c, r, layer)
        x = q[0, r * G:(r + 1) * G, 0].double()
        out[0, r * G:(r + 1) * G] = softmax_rows(x, k, v, D ** -0.5)
        ks.append(k), vs.append(v), qs.append(x)
    return out, attention_tolerance(q.dtype, qs, ks, vs, D ** -0.5, max(k.shape[0] for k in ks))


def _angles(pos, dev, dtype=torch.bfloat16):
    f = pos * 500000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    f = torch.cat([f, f])[None, None]
    return f.cos().to(dev, dtype), f.sin().to(dev, dtype)


def test_update_rope_steps(cuda_device):
    """Steps through update_rope: rotated query back (and in the drift check's buffer), rotated key in the pages."""
    dev, L = cuda_device, 900
    c = _cache()
    _prefill(c, L, 3, dev)
    g = torch.Generator().manual_seed(5)
    for step in range(9):
        q, k, v = (torch.randn(1, n, 1, D, generator=g).to(dev, torch.bfloat16) for n in (H, KV, KV))
        cos, sin = _angles(L + step, dev)
        lens = c.heads_len[0].tolist()
        slot = c._qcount[0]
        rq = c.update_rope(q, k, v, cos, sin, 0)
        want = rotate(q, cos[:, None], sin[:, None])
        size = half_step(torch.bfloat16) * want.abs() + 2.0 ** -21 * q.double().abs().amax()
        assert ((rq.double() - want).abs() <= size).all()
        assert torch.equal(c._qbuf[0][slot], rq[0, :, 0])
        assert c.heads_len[0].tolist() == [n + 1 for n in lens] == c._hlen[0].tolist()
        want = rotate(k, cos[:, None], sin[:, None])
        for r in range(KV):
            pk, pv = _row(c, r)
            assert ((pk[-1] - want[0, r, 0]).abs() <= half_step(torch.bfloat16) * want[0, r, 0].abs()
                    + 2.0 ** -21 * k.double().abs().amax()).all()
            assert torch.equal(pv[-1], v[0, r, 0].double())
        ref, tol = _attend(c, rq)
        out = c.attention(rq, 0)
        assert float((out.double() - ref).abs().max()) <= tol
        c.decode_select(rq, 0)
    c.join_retrievals()
    c.check_errors()
    assert c._seen_tokens == L + 9


def test_update_rope_refuses(cuda_device):
    c = _cache()
    x = torch.zeros(1, KV, 2, D, dtype=torch.bfloat16, device=cuda_device)
    q = torch.zeros(1, H, 2, D, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError, match="one token"):
        c.update_rope(q, x, x, x[:, 0], x[:, 0], 0)
    with pytest.raises(RuntimeError, match="prefill first"):
        c.update_rope(q[:, :, :1], x[:, :, :1], x[:, :, :1], x[:, 0, :1], x[:, 0, :1], 0)


@pytest.mark.parametrize("cls", [LlamaAttention, Qwen2Attention])
def test_attention_class_with_fused_rope(cuda_device, cls):
    """The patched classes with and without fused_rope: the same step to the rounding of the rotation."""
    from transformers import LlamaConfig
    cfg = LlamaConfig(hidden_size=512, num_attention_heads=8, num_key_value_heads=4, head_dim=128)
    dev, L = cuda_device, 600
    torch.manual_seed(0)
    attn = cls(cfg, layer_idx=0).to(dev, torch.bfloat16).eval()
    data = derive_runtime_data(synthetic_roles(1, 4, seed=3, star_size=3), 1, 4)
    make = lambda fused: HeteroCache(HeteroCacheConfig(  # noqa: E731
        data, real_offload=False, max_gen_len=32, decode_step=5, num_attn_heads=8, num_kv_heads=4, num_layers=1,
        stable_threshold=0.999, fused_rope=fused))
    plain, fused = make(False), make(True)
    h = torch.randn(1, L, 512, device=dev, dtype=torch.bfloat16)
    cos = torch.cat([_angles(t, dev)[0] for t in range(L)], 1)
    sin = torch.cat([_angles(t, dev)[1] for t in range(L)], 1)
    with torch.no_grad():
        for c in (plain, fused):
            attn(h, position_embeddings=(cos, sin), past_key_values=c)
        for step in range(7):
            x = torch.randn(1, 1, 512, device=dev, dtype=torch.bfloat16)
            emb = _angles(L + step, dev)
            a = attn(x, position_embeddings=emb, past_key_values=plain)[0]
            b = attn(x, position_embeddings=emb, past_key_values=fused)[0]
            # the rotation's roundings (three against one) and the outputs': a few half steps of the largest values
            assert float((a.float() - b.float()).abs().max()) <= 8 * half_step(torch.bfloat16) * max(
                1.0, float(a.float().abs().max()))
    for c in (plain, fused):
        c.join_retrievals()
        c.check_errors()
    assert plain.heads_len[0].tolist() == fused.heads_len[0].tolist()
    assert torch.equal(plain.block_tables[0], fused.block_tables[0])


@pytest.mark.parametrize("offload", [False, True])
@pytest.mark.parametrize("rope", [False, True])
def test_sparse_cache_steps(cuda_device, offload, rope):
    """Block-sparse steps through page boundaries, drift checks and retrievals: the bounds stay those of the pages,
    and the output is the attention over the blocks that they select."""
    dev, L, n_sel, sink, recent = cuda_device, 3000, 9, 1, 2
    c = _cache(real_offload=offload, sparse_blocks=n_sel, sparse_sink=sink, sparse_recent=recent)
    q0 = _prefill(c, L, 21, dev)
    gen = DriftingDecode(GEO, seed=8, q0=q0, dtype=torch.bfloat16)
    fired = 0
    for step in range(24):
        q, k, v = (t.to(dev) for t in gen.step())
        if rope:
            q = c.update_rope(q, k, v, *_angles(step, dev), 0)
        else:
            c.update(k, v, 0, {"query_states": q, "defer_append": step % 2 == 0})
        out = c.attention(q, 0)
        torch.cuda.synchronize()
        lim, fresh = c._bounds[0], torch.zeros_like(c._bounds[0])
        ops.block_bounds(c.key_pools[0], c.block_tables[0], c.heads_len[0], fresh, c._err)
        ks, vs, qs, want = [], [], [], torch.zeros(1, H, D, dtype=torch.float64, device=dev)
        for r in range(KV):
            m = (int(c.heads_len[0][r]) + BLOCK - 1) // BLOCK
            j = torch.arange(m, device=dev)
            at = (c.block_tables[0][r].long()[j // 4], j % 4)
            assert torch.equal(lim[at], fresh[at]), (step, r)
            x = q[0, r * G:(r + 1) * G, 0]
            blocks = pick(block_scores(x, lim[at][:, 0], lim[at][:, 1]).tolist(), n_sel, sink, recent)
            key, val = _row(c, r)
            t = torch.tensor([i for b in blocks for i in range(b * BLOCK, min(key.shape[0], (b + 1) * BLOCK))], device=dev)
            want[0, r * G:(r + 1) * G] = softmax_rows(x.double(), key[t], val[t], D ** -0.5)
            ks.append(key[t]), vs.append(val[t]), qs.append(x.double())
        tol = attention_tolerance(q.dtype, qs, ks, vs, D ** -0.5, n_sel * BLOCK)
        assert float((out.double() - want).abs().max()) <= tol, step
        c.decode_select(q, 0, defer=True)
        c.join_retrievals()
        if step % 4 == 3:
            fired += int(c._jobs[0].trigger[:c._jobs[0].n_jobs].sum())
    c.check_errors()
    assert fired > 0


def test_sparse_steps_from_a_graph(cuda_device):
    """DecodeStepGraph over a sparse cache: the replayed steps are the eager ones."""
    dev, L = cuda_device, 1500
    pair = [_cache(layers=2, sparse_blocks=8) for _ in range(2)]
    for c in pair:
        for layer in range(2):
            q0 = _prefill(c, L, 30 + layer, dev, layer)
    eager, graphed = pair
    g = DecodeStepGraph(graphed, [0, 1])
    gens = [DriftingDecode(GEO, seed=50 + i, q0=q0, dtype=torch.bfloat16) for i in range(2)]
    for step in range(9):
        qkv = [tuple(t.to(dev) for t in x.step()) for x in gens]
        for layer, (q, k, v) in enumerate(qkv):
            g.q[layer].copy_(q), g.k[layer].copy_(k), g.v[layer].copy_(v)
        outs = []
        for layer, (q, k, v) in enumerate(qkv):
            eager.update(k, v, layer, {"query_states": q, "defer_append": True})
            outs.append(eager.attention(q, layer))
            eager.decode_select(q, layer, defer=True)
        eager.join_retrievals()
        got = g.step()
        torch.cuda.synchronize()
        for layer in range(2):
            assert torch.equal(got[layer], outs[layer]), (step, layer)
            assert torch.equal(eager.heads_len[layer], graphed.heads_len[layer])
    for c in pair:
        c.check_errors()


def test_sparse_refusals(cuda_device):
    with pytest.raises(ValueError, match="sparse_blocks"):
        _cache(sparse_blocks=3, sparse_sink=2, sparse_recent=2)
    c = _cache(sparse_blocks=4)
    _prefill(c, 600, 1, cuda_device)
    q = torch.zeros(1, H, 1, D, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(NotImplementedError, match="mirrors"):
        c.attention(q, 0, mirrors=[16])
    with pytest.raises(NotImplementedError, match="fork"):
        c.fork(2)


@pytest.mark.parametrize("offload", [False, True])
def test_fork_matches_caches_of_their_own(cuda_device, offload):
    """Three continuations of one prompt against three caches that each prefilled it: the same triggers, lengths and
    pages at every step, outputs to the rounding of the split."""
    dev, L, n = cuda_device, 3000, 3
    prompt = _cache(real_offload=offload)
    q0 = _prefill(prompt, L, 77, dev)
    own = [_cache(real_offload=offload) for _ in range(n)]
    for c in own:
        _prefill(c, L, 77, dev)
    group = prompt.fork(n)
    shared = group.shared_len[0].tolist()
    sat = {h for m in prompt.data["leader_member_relations"][0].values() for h in m}
    lens = prompt.heads_len[0].tolist()
    assert shared == [0 if h in sat else lens[h] // PAGE * PAGE for h in range(KV)] and max(shared) == 2816
    gens = [DriftingDecode(GEO, seed=900 + i, q0=q0, dtype=torch.bfloat16) for i in range(n)]
    fired = 0
    for step in range(13):
        qkv = [tuple(t.to(dev) for t in g.step()) for g in gens]
        defer = step % 3 != 2
        for c, (q, k, v) in zip(own, qkv):
            c.update(k, v, 0, {"query_states": q, "defer_append": defer})
        for c, (q, k, v) in zip(group.members, qkv):
            c.update(k, v, 0, {"query_states": q, "defer_append": defer})
        a = torch.cat([c.attention(q, 0) for c, (q, _, _) in zip(own, qkv)], 0)
        b = attention_together(group, torch.cat([q for q, _, _ in qkv], 0), 0)
        for cs in (own, group.members):
            for c, (q, _, _) in zip(cs, qkv):
                c.decode_select(q, 0, defer=True)
            if offload:
                for c in cs:
                    c.join_retrievals()
            else:
                flush_checks_together(cs)
        torch.cuda.synchronize()
        biggest = max(float(c.value_pools[0].float().abs().max()) for c in own)
        assert float((a.double() - b.double()).abs().max()) <= 4 * half_step(torch.bfloat16) * biggest, step
        for x, y in zip(own, group.members):
            for z in (x, y):
                z._wait_append(0)
                z._wait_retrieval(0)
            torch.cuda.synchronize()
            assert torch.equal(x._jobs[0].trigger, y._jobs[0].trigger), step
            assert torch.equal(x.heads_len[0], y.heads_len[0])
            fired += int(y._jobs[0].trigger[:y._jobs[0].n_jobs].sum())
            for r in range(KV):
                for s, t in zip(_row(x, r), _row(y, r)):
                    assert torch.equal(s, t), (step, r)
    for c in own + group.members:
        c.join_retrievals()
        c.check_errors()
    assert fired > 0
    # the prompt's own cache is as it was: its first step is an own cache's first step
    q, k, v = (t.to(dev) for t in DriftingDecode(GEO, seed=900, q0=q0, dtype=torch.bfloat16).step())
    fresh = _cache(real_offload=offload)
    _prefill(fresh, L, 77, dev)
    outs = []
    for c in (prompt, fresh):
        c.update(k, v, 0, {"query_states": q})
        outs.append(c.attention(q, 0))
    assert torch.equal(*outs)


def test_fork_refuses_a_cache_in_the_middle_of_decoding(cuda_device):
    c = _cache()
    q0 = _prefill(c, 700, 5, cuda_device)
    with pytest.raises(ValueError, match="at least one"):
        c.fork(0)
    with pytest.raises(ValueError, match="4096 rows"):
        c.fork(513)
    q, k, v = (t.to(cuda_device) for t in DriftingDecode(GEO, seed=1, q0=q0, dtype=torch.bfloat16).step())
    c.update(k, v, 0, {"query_states": q})
    c.attention(q, 0)
    c.decode_select(q, 0)
    with pytest.raises(RuntimeError, match="right after its prefill"):
        c.fork(2)


@pytest.mark.parametrize("kind", ["llama", "qwen"])
@pytest.mark.parametrize("sparse", [0, 6])
def test_model_graph_with_fused_rope(cuda_device, kind, sparse):
    """A whole model's decode, eager and from graphs, with the rotation in the append and block-sparse attention:
    the same tokens and pages."""
    import transformers
    from heterocache_b200.attention import patch_transformers
    from heterocache_b200.graph import ModelDecodeGraph
    patch_transformers()
    torch.manual_seed(1)
    args = dict(hidden_size=1024, num_attention_heads=8, num_key_value_heads=4, intermediate_size=2048,
                num_hidden_layers=2, vocab_size=512, max_position_embeddings=4096)
    cfg = transformers.LlamaConfig(head_dim=128, **args) if kind == "llama" else transformers.Qwen2Config(**args)
    cfg._attn_implementation = "sdpa"
    cls = transformers.LlamaForCausalLM if kind == "llama" else transformers.Qwen2ForCausalLM
    model = cls(cfg).to(cuda_device, torch.bfloat16).eval()
    data = derive_runtime_data(synthetic_roles(2, 4, seed=5, star_size=3), 2, 4)
    ids = torch.randint(0, 512, (1, 800), device=cuda_device)

    def prefilled():
        c = HeteroCache(HeteroCacheConfig(data, stable_threshold=0.9, real_offload=False, max_gen_len=32,
                                          decode_step=5, num_attn_heads=8, num_kv_heads=4, num_layers=2,
                                          fused_rope=True, sparse_blocks=sparse))
        with torch.no_grad():
            out = model(input_ids=ids, past_key_values=c, use_cache=True, logits_to_keep=1)
        return c, out.logits[:, -1:].argmax(-1)

    eager, tok = prefilled()
    tokens = []
    with torch.no_grad():
        for t in range(12):
            pos = torch.tensor([[800 + t]], device=cuda_device)
            out = model(input_ids=tok, past_key_values=eager, use_cache=True, position_ids=pos, cache_position=pos[0],
                        logits_to_keep=1)
            tok = out.logits[:, -1:].argmax(-1)
            tokens.append(int(tok))
    eager.join_retrievals()
    graphed, tok = prefilled()
    runner = ModelDecodeGraph(model, graphed, tok.clone(), torch.tensor([[800]], device=cuda_device))
    assert [int(runner.step()) for _ in range(12)] == tokens
    for c in (eager, graphed):
        c.check_errors()
    for layer in range(2):
        assert torch.equal(graphed.heads_len[layer], eager.heads_len[layer])
        assert torch.equal(graphed.block_tables[layer], eager.block_tables[layer])
        assert (graphed.key_pools[layer].float() - eager.key_pools[layer].float()).abs().max().item() <= 2e-2
