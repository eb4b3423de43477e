"""An update_rope that is refused leaves the cache's host mirrors where they were (on the CPU: nothing is launched)."""
import numpy as np
import pytest
import torch

from heterocache_b200.cache import HeteroCache, HeteroCacheConfig
from heterocache_b200.roles import derive_runtime_data, synthetic_roles

H, KV, D, L = 32, 8, 128, 512


def _cache(gen=64, **other):
    """A cache as its prefill leaves it, without the kernels: pages of every row mapped, lengths set."""
    data = derive_runtime_data(synthetic_roles(1, KV, seed=13), 1, KV)
    c = HeteroCache(HeteroCacheConfig(data, real_offload=False, max_gen_len=gen, decode_step=4, num_attn_heads=H,
                                      num_kv_heads=KV, num_layers=1, **other))
    dev = torch.device("cpu")
    c._ensure_device(dev)
    c.bsz, c.head_dim, c.prefill_len, c.base_compress_len, c._seen_tokens = 1, D, L, L // 2, L
    c._init_layer_storage(0, dev, torch.bfloat16)
    c._hlen[0][:] = c._mapped[0] * 256 - 3
    c.heads_len[0].copy_(torch.from_numpy(c._hlen[0].astype(np.int32)))
    return c


def _state(c):
    return (c._hlen[0].tolist(), c._mapped[0].tolist(), c.free_block_pointers[0], c._seen_tokens, c._qcount[0],
            c._q_staged[0])


def _args(**other):
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    a = dict(query_states=z(1, H, 1, D), key_states=z(1, KV, 1, D), value_states=z(1, KV, 1, D), cos=z(1, 1, D),
             sin=z(1, 1, D))
    a.update(other)
    return a


@pytest.mark.parametrize("name,value", [
    ("cos", torch.zeros(1, 1, D, dtype=torch.float64)),
    ("sin", torch.zeros(1, 2, D, dtype=torch.bfloat16)),
    ("value_states", torch.zeros(1, KV, 1, D)),
    ("query_states", torch.zeros(1, H, 1, D)),
    (None, None),  # all as they should be, but not on a GPU
])
def test_mirrors_stay(name, value):
    c = _cache()
    for _ in range(5):  # across a page border of every row
        before = _state(c)
        with pytest.raises((ValueError, TypeError)):
            c.update_rope(layer_idx=0, **_args(**({name: value} if name else {})))
        assert _state(c) == before


@pytest.mark.parametrize("bad", [torch.zeros(1, H, 1, D), torch.zeros(1, H - 8, 1, D, dtype=torch.bfloat16),
                                 torch.zeros(1, H, 1, D, dtype=torch.bfloat16, device="meta")])
def test_a_refused_query_makes_no_buffer(bad, monkeypatch):
    """The drift check's query buffer is made from a query that fits the pages."""
    from heterocache_b200 import ops
    c = _cache()
    with pytest.raises(ValueError, match="the query must be"):
        c.update_rope(layer_idx=0, **_args(query_states=bad))
    assert c._qbuf[0] is None
    monkeypatch.setattr(ops, "rope_append", lambda q, *a, q_out=None, **k: q_out.copy_(q))
    c.update_rope(layer_idx=0, **_args())
    assert c._qbuf[0].dtype == torch.bfloat16 and tuple(c._qbuf[0].shape) == (4, H, D)


def test_mirrors_advance_with_the_append(monkeypatch):
    from heterocache_b200 import ops
    c = _cache(gen=300)
    monkeypatch.setattr(ops, "rope_append", lambda q, *a, **k: q)
    rows, free = c._hlen[0].copy(), c.free_block_pointers[0]
    for step in range(1, 6):
        c.update_rope(layer_idx=0, **_args())
        assert c._hlen[0].tolist() == (rows + step).tolist() and c._seen_tokens == L + step
        assert c.free_block_pointers[0] == free + (KV if step > 3 else 0)


def test_out_of_pages_is_raised_before_the_launch(monkeypatch):
    from heterocache_b200 import ops
    c = _cache(gen=300)
    c.free_blocks[0] = c.free_blocks[0][:KV - 1]

    def launch(q, *a, **k):
        launch.n += 1
        return q
    launch.n = 0
    monkeypatch.setattr(ops, "rope_append", launch)
    for _ in range(3):
        c.update_rope(layer_idx=0, **_args())
    before = _state(c)
    with pytest.raises(RuntimeError, match="OOM"):
        c.update_rope(layer_idx=0, **_args())
    assert launch.n == 3 and _state(c) == before
