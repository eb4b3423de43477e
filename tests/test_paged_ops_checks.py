"""What rope_append, flash_decode_shared and flash_decode_sparse refuse, on the host and before any launch."""
import pytest
import torch

from heterocache_b200 import ops

D = 128
i32 = torch.int32


class _Scratch:
    counter = torch.zeros(4, dtype=i32)

    def get(self, nbytes):
        raise AssertionError("refusals come before the workspace is used")


def _append_args(**other):
    bf = torch.bfloat16
    a = dict(q=torch.zeros(2, 4, 3, D, dtype=bf), k=torch.zeros(2, 2, 3, D, dtype=bf),
             v=torch.zeros(2, 2, 3, D, dtype=bf), cos=torch.zeros(2, 3, D, dtype=bf), sin=torch.zeros(2, 3, D, dtype=bf),
             k_pool=torch.zeros(5, 256, 1, D, dtype=bf), v_pool=torch.zeros(5, 256, 1, D, dtype=bf),
             block_table=torch.zeros(4, 2, dtype=i32), heads_len=torch.zeros(4, dtype=i32),
             free_blocks=torch.zeros(2, dtype=i32), free_ptr=torch.zeros(1, dtype=i32), err=torch.zeros(1, dtype=i32),
             workspace=_Scratch())
    a.update(other)
    return a


@pytest.mark.parametrize("name,value,what", [
    ("q", torch.zeros(2, 4, 2, D, dtype=torch.bfloat16), "share batch"),
    ("q", torch.zeros(2, 4, 3, D), "share batch"),
    ("q", torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16), "contiguous last dim"),
    ("q", torch.zeros(2, 4, 3, D, dtype=torch.float64), "unsupported dtype"),
    ("v", torch.zeros(2, 1, 3, D, dtype=torch.bfloat16), "same shape"),
    ("cos", torch.zeros(2, 2, D, dtype=torch.bfloat16), "cos needs"),
    ("cos", torch.zeros(3, 3, D, dtype=torch.bfloat16), "cos needs"),
    ("sin", torch.zeros(2, 3, D), "share a dtype"),
    ("cos", torch.zeros(2, 3, D, dtype=torch.float16), "share a dtype"),
    ("cos", torch.zeros(2, 3, 2 * D, dtype=torch.bfloat16)[..., ::2], "contiguous last dim"),
    ("k_pool", torch.zeros(5, 128, 1, D, dtype=torch.bfloat16), "k_pool"),
    ("k_pool", torch.zeros(5, 256, 1, D), "k_pool"),
    ("v_pool", torch.zeros(4, 256, 1, D, dtype=torch.bfloat16), "same shape"),
    ("v_pool", torch.zeros(10, 256, 1, D, dtype=torch.bfloat16)[::2], "v_pool"),
    ("block_table", torch.zeros(3, 2, dtype=i32), "row per"),
    ("block_table", torch.zeros(4, 2, dtype=torch.int64), "int32"),
    ("heads_len", torch.zeros(3, dtype=i32), "row per"),
    ("free_ptr", torch.zeros(0, dtype=i32), "need an entry"),
    ("free_blocks", torch.zeros(4, dtype=i32)[::2], "int32"),
    ("counts", torch.zeros(1, dtype=i32), "entry per sequence"),
    ("counts", torch.zeros(2, dtype=torch.int64), "int32"),
    ("q_out", torch.zeros(2, 4, 2, D, dtype=torch.bfloat16), "q_out"),
    ("q_out", torch.zeros(2, 4, 3, D), "q_out"),
    ("heads_len_out", torch.zeros(3, dtype=i32), "heads_len_out"),
    ("bounds", torch.zeros(4, 4, 2, D, dtype=torch.bfloat16), "bounds"),
    ("bounds", torch.zeros(5, 4, 2, D), "bounds"),
])
def test_rope_append_refuses(name, value, what):
    err = TypeError if what == "unsupported dtype" else ValueError
    with pytest.raises(err, match=what):
        ops.rope_append(**_append_args(**{name: value}))


def test_rope_append_refuses_host_tensors_and_several_devices():
    with pytest.raises(ValueError, match="CUDA device"):
        ops.rope_append(**_append_args())
    with pytest.raises(ValueError, match="different devices"):
        ops.rope_append(**_append_args(free_ptr=torch.zeros(1, dtype=i32, device="meta")))


def _decode_args(**other):
    bf = torch.bfloat16
    a = dict(q=torch.zeros(2, 4, 1, D, dtype=bf), k_pool=torch.zeros(5, 256, 1, D, dtype=bf),
             v_pool=torch.zeros(5, 256, 1, D, dtype=bf), block_table=torch.zeros(4, 2, dtype=i32),
             heads_len=torch.zeros(4, dtype=i32), num_kv_heads=2, workspace=_Scratch(), err=torch.zeros(1, dtype=i32))
    a.update(other)
    return a


BOTH = [
    ("q", torch.zeros(2, 4, 2, D, dtype=torch.bfloat16), "one query position"),
    ("q", torch.zeros(2, 5, 1, D, dtype=torch.bfloat16), "split evenly"),
    ("q", torch.zeros(2, 4, 1, D), "dtype"),
    ("num_kv_heads", 3, "split evenly"),
    ("num_kv_heads", 0, "split evenly"),
    ("block_table", torch.zeros(3, 2, dtype=i32), "row per"),
    ("heads_len", torch.zeros(4, dtype=torch.int64), "int32"),
]


@pytest.mark.parametrize("name,value,what", BOTH + [
    ("k_pool", torch.zeros(5, 256, 1, D, dtype=torch.float16), "k_pool"),
    ("v_pool", torch.zeros(6, 256, 1, D, dtype=torch.bfloat16), "same shape"),
    ("out", torch.zeros(2, 4, D), "out must"),
    ("out", torch.zeros(2, 4, 2 * D, dtype=torch.bfloat16)[..., :D], "out must"),
    ("shared_len", torch.zeros(1, dtype=i32), "shared_len"),
    ("shared_len", torch.zeros(2), "int32"),
    ("k_new", torch.zeros(2, 2, 1, D, dtype=torch.bfloat16), "come together"),
])
def test_flash_decode_shared_refuses(name, value, what):
    with pytest.raises(ValueError, match=what):
        ops.flash_decode_shared(**_decode_args(**{"shared_len": torch.zeros(2, dtype=i32), name: value}))


def test_flash_decode_shared_refuses_a_new_token_of_another_shape():
    new = torch.zeros(2, 4, 1, D, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="k_new/v_new"):
        ops.flash_decode_shared(**_decode_args(shared_len=torch.zeros(2, dtype=i32), k_new=new, v_new=new))


@pytest.mark.parametrize("name,value,what", BOTH + [
    ("bounds", torch.zeros(5, 4, 2, D), "bounds"),
    ("bounds", torch.zeros(5, 2, 2, D, dtype=torch.bfloat16), "bounds"),
    ("n_select", 0, "n_select"),
    ("n_select", 2, "n_select"),
    ("sink", -1, "n_select"),
    ("recent", 9, "n_select"),
    ("blocks", torch.zeros(4, 3, dtype=i32), "blocks needs"),
    ("counts", torch.zeros(3, dtype=i32), "blocks needs"),
    ("blocks", torch.zeros(4, 4), "int32"),
])
def test_flash_decode_sparse_refuses(name, value, what):
    a = _decode_args(bounds=torch.zeros(5, 4, 2, D, dtype=torch.bfloat16), n_select=4, sink=1, recent=2)
    a[name] = value
    with pytest.raises(ValueError, match=what):
        ops.flash_decode_sparse(**a)


@pytest.mark.parametrize("name,value,what", [
    ("blocks", torch.zeros(3, 4, dtype=i32), "blocks needs"),
    ("blocks", torch.zeros(4, 0, dtype=i32), "blocks needs"),
    ("counts", torch.zeros(3, dtype=i32), "blocks needs"),
])
def test_flash_decode_blocks_refuses(name, value, what):
    a = _decode_args(blocks=torch.zeros(4, 4, dtype=i32), counts=torch.zeros(4, dtype=i32))
    a[name] = value
    with pytest.raises(ValueError, match=what):
        ops.flash_decode_blocks(**a)


@pytest.mark.parametrize("name,value,what", [
    ("bounds", torch.zeros(5, 4, 2, D), "bounds"),
    ("heads_len", torch.zeros(3, dtype=i32), "row per"),
    ("rows", torch.zeros(3, dtype=torch.int64), "int32"),
    ("last", -1, "negative"),
])
def test_block_bounds_refuses(name, value, what):
    bf = torch.bfloat16
    a = dict(k_pool=torch.zeros(5, 256, 1, D, dtype=bf), block_table=torch.zeros(4, 2, dtype=i32),
             heads_len=torch.zeros(4, dtype=i32), bounds=torch.zeros(5, 4, 2, D, dtype=bf), err=torch.zeros(1, dtype=i32))
    a[name] = value
    with pytest.raises(ValueError, match=what):
        ops.block_bounds(**a)


def test_the_library_refuses_bad_arguments():
    """Status codes of the C entries, without a GPU: 1 invalid, 2 type, 6 workspace, 8 unsupported."""
    import __graft_entry__
    from heterocache_b200 import _lib
    __graft_entry__.build()
    lib = _lib.lib()
    P = 64  # an aligned address that is never read: every call is refused on the host

    def append(dt=1, tr=1, bsz=2, H=4, KV=2, T=3, d=D, q=P, qst=D, cos=P, cst=D, table=P, mb=2, lens=P, free=P, nf=3,
               counter=P):
        return lib.hc_rope_append(dt, tr, bsz, H, KV, T, d, q, 3 * 4 * D, D, qst, P, 3 * D, D, D, P, 3 * D, D, D, cos,
                                  3 * D, cst, P, 3 * D, D, P, D, D, D, None, P, P, 5, table, mb, lens, P, free, nf, P,
                                  None, counter, None, None)
    assert append(dt=7) == 2 and append(tr=2) == 2
    for bad in (dict(bsz=0), dict(KV=0), dict(T=-1), dict(d=64), dict(mb=0), dict(q=P + 8), dict(qst=D + 1),
                dict(cos=P + 2), dict(cst=D + 2), dict(table=None), dict(lens=None), dict(free=None),
                dict(counter=None)):
        assert append(**bad) == 1, bad
    assert append(mb=1 << 24) == 8

    def select(dt=1, bsz=1, G=4, d=D, q=P, n=4, sink=1, recent=1, ws=None, nbytes=0, mb=4):
        return lib.hc_block_select(dt, bsz, 2, G, d, q, 2 * G * D, D, P, 5, P, mb, P, n, sink, recent, P, P, ws, nbytes,
                                   None, None)
    assert select(dt=9) == 2 and select(d=96) == 1 and select(q=P + 4) == 1
    assert select(n=0) == 1 and select(sink=-1) == 1 and select(sink=3, recent=2) == 1
    assert select(G=9) == 8 and select(bsz=3000) == 8
    assert select() == 6 and select(ws=P, nbytes=16) == 6
    assert lib.hc_block_bounds(1, 0, D, P, 5, P, 2, P, None, 0, 0, P, None, None) == 1
    assert lib.hc_block_bounds(1, 2, D, P, 5, P, 2, P, None, 0, -1, P, None, None) == 1
    assert lib.hc_block_bounds(1, 2, D, P, 5, P, 2, P, P, 0, 0, P, None, None) == 0  # no rows

    def blocks(G=4, lists=P, n=4, ws=None):
        return lib.hc_flash_decode_blocks(1, 1, 2, G, D, P, 2 * G * D, D, P, P, 5, P, 2, P, lists, P, n, 0.0, P, ws, 0,
                                          None, None)
    assert blocks(lists=None) == 1 and blocks(n=0) == 1 and blocks(G=9) == 8
    assert blocks(n=1 << 26) == 8

    def shared(G=4, lens=P, kn=None, vn=None, ws=None, nbytes=0, bsz=2):
        return lib.hc_flash_decode_shared(1, bsz, 2, G, D, P, 2 * G * D, D, P, P, 5, P, 2, P, lens, kn, vn, D, D, D, D,
                                          0.0, P, ws, nbytes, None, None)
    assert shared(lens=None) == 1 and shared(kn=P) == 1 and shared(G=9) == 8 and shared(bsz=3000) == 8
    assert shared() == 6 and shared(ws=P, nbytes=1 << 10) == 6
    assert lib.hc_flash_decode_shared_workspace_size(1, 4, 8, 4, D) > 0
    assert lib.hc_flash_decode_shared_workspace_size(5, 4, 8, 4, D) == 0
    assert lib.hc_block_select_workspace_size(1, 8, 100) >= 8 * 400 * 8


def test_fork_pages():
    """The page tables of a fork: whole pages shared, the last one and private heads copied, spare pages apart."""
    import numpy as np
    from heterocache_b200.cache import fork_pages
    bt = np.full((3, 6), -1, dtype=np.int32)
    bt[0, :3], bt[1, :2], bt[2, :2] = [0, 1, 2], [3, 4], [5, 6]
    tables, shared, copies, free, total = fork_pages(bt, [600, 512, 300], 300, 6, {2}, 3)
    assert shared.tolist() == [512, 512, 0]
    assert tables[0, 0].tolist() == [0, 1, 2, -1, -1, -1] and tables[0, 2].tolist() == [5, 6, -1, -1, -1, -1]
    for i in (1, 2):
        assert tables[i, 0, :2].tolist() == [0, 1] and tables[i, 1, :2].tolist() == [3, 4]
        own = [tables[i, 0, 2], *tables[i, 2, :2]]
        assert tables[i, 2, 1] == tables[i, 2, 0] + 1  # retrievals write a private head's pages as one piece
        assert len(set(own)) == 3 and min(own) >= 7
        assert [c for c in copies if c[1] in own] == [(2, own[0]), (5, own[1]), (6, own[2])]
    # 600, 512 and 300 tokens grow by 300: 1, 2 and 1 pages more
    assert [len(f) for f in free] == [4, 4, 4]
    ids = sorted(sum(free, []) + [int(c[1]) for c in copies])
    assert ids == list(range(7, total))


def test_config_checks_sparse_blocks():
    from heterocache_b200.cache import HeteroCacheConfig
    with pytest.raises(ValueError, match="sparse_blocks"):
        HeteroCacheConfig({}, sparse_blocks=2, sparse_sink=1, sparse_recent=2)
    assert HeteroCacheConfig({}).sparse_blocks == 0 and not HeteroCacheConfig({}).fused_rope
