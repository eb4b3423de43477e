"""A cache that takes a second prompt: block-sparse attention selects by the second prompt's keys."""
import pytest
import torch

from heterocache_b200 import ops
from heterocache_b200.cache import HeteroCache, HeteroCacheConfig
from heterocache_b200.roles import derive_runtime_data, synthetic_roles
from heterocache_b200.synthetic import LLAMA_8B, prefill_inputs

pytestmark = pytest.mark.gpu
GEO = LLAMA_8B


@pytest.mark.parametrize("rope", [False, True])
def test_bounds_of_a_second_prompt(cuda_device, rope):
    dev, L, KV, H, D = cuda_device, 900, GEO.num_kv_heads, GEO.num_heads, 128
    data = derive_runtime_data(synthetic_roles(1, KV, seed=13), 1, KV)
    c = HeteroCache(HeteroCacheConfig(data, real_offload=False, max_gen_len=64, decode_step=50, num_attn_heads=H,
                                      num_kv_heads=KV, num_layers=1, sparse_blocks=6))
    buf = None
    for prompt in range(2):
        q, k, v = (t.to(dev) for t in prefill_inputs(GEO, L, seed=40 + prompt, dtype=torch.bfloat16, q_positions=32))
        c.update(k, v, 0)
        c.init_coefficient(q, k, 0)
        c.prefill_select(q, k, v, 0)
        g = torch.Generator().manual_seed(prompt)
        for step in range(2):
            q, k, v = (torch.randn(1, n, 1, D, generator=g).to(dev, torch.bfloat16) for n in (H, KV, KV))
            if rope:
                one = torch.ones(1, 1, D, dtype=torch.bfloat16, device=dev)
                q = c.update_rope(q, k, v, one, torch.zeros_like(one), 0)
            else:
                c.update(k, v, 0, {"query_states": q})
            c.attention(q, 0)
            lim, fresh = c._bounds[0], c._bounds[0].clone()
            ops.block_bounds(c.key_pools[0], c.block_tables[0], c.heads_len[0], fresh, c._err)
            assert torch.equal(lim, fresh), (prompt, step)
        assert buf is None or c._bounds[0].data_ptr() == buf  # (a captured graph holds the address)
        buf = c._bounds[0].data_ptr()
    c.check_errors()
