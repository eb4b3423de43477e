"""ops.Workspace: what it has handed out stays allocated when it grows (captured graphs, and kernels that
another stream still runs, hold the address)."""
import torch

from heterocache_b200.ops import Workspace


def test_buffers_outlive_growth():
    ws = Workspace("cpu")
    first = ws.get(1000)
    at, n = first.data_ptr(), first.numel()
    store = first.untyped_storage()
    refs = store._weak_ref()
    first.fill_(7)
    del first, store
    second = ws.get(10 * n)
    assert second.numel() >= 10 * n and second.data_ptr() != at
    kept = torch.UntypedStorage._new_with_weak_ptr(refs)
    assert kept is not None and kept.data_ptr() == at  # still allocated
    del kept
    torch.UntypedStorage._free_weak_ref(refs)


def test_growth_is_geometric():
    """A workspace that grows a little each time holds no more than a few times its size."""
    ws, seen = Workspace("cpu"), {}
    for n in range(1 << 20, 40 << 20, 1 << 18):
        b = ws.get(n)
        seen[b.data_ptr()] = b.numel()
    assert sum(seen.values()) <= 4 * max(seen.values())


def test_reset_clears_every_buffer():
    ws = Workspace("cpu")
    a = ws.get(100)
    a.fill_(3)
    b = ws.get(10 * a.numel())
    b.fill_(4)
    ws.counter.fill_(5)
    ws.reset()
    assert not a.any() and not b.any() and not ws.counter.any()
    assert ws.get(100) is b or ws.get(100).data_ptr() == b.data_ptr()
