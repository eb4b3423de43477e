"""The C entries of the paged operators: missing buffers and workspaces off their alignment are refused on the host."""
import pytest

from heterocache_b200 import _lib

D, P = 128, 64  # P: an aligned address that is never read, every call here being refused


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    return _lib.lib()


def _append(lib, **o):
    a = dict(q=P, k=P, v=P, cos=P, sin=P, q_out=P, kp=P, vp=P, n=5, T=3)
    a.update(o)
    return lib.hc_rope_append(1, 1, 2, 4, 2, a["T"], D, a["q"], 12 * D, D, D, a["k"], 6 * D, D, D, a["v"], 6 * D, D, D,
                              a["cos"], 3 * D, D, a["sin"], 3 * D, D, a["q_out"], 12 * D, D, D, None, a["kp"], a["vp"],
                              a["n"], P, 2, P, P, P, 3, P, None, P, None, None)


@pytest.mark.parametrize("name", ["q", "k", "v", "cos", "sin", "q_out", "kp", "vp"])
def test_append_wants_its_buffers(lib, name):
    assert _append(lib, **{name: None}) == 1


@pytest.mark.parametrize("name", ["kp", "bounds"])
def test_bounds_want_their_buffers(lib, name):
    a = dict(kp=P, bounds=P)
    a[name] = None
    assert lib.hc_block_bounds(1, 2, D, a["kp"], 5, P, 2, P, None, 0, 0, a["bounds"], None, None) == 1


@pytest.mark.parametrize("name", ["q", "bounds"])
def test_select_wants_its_buffers(lib, name):
    a = dict(q=P, bounds=P)
    a[name] = None
    assert lib.hc_block_select(1, 1, 2, 4, D, a["q"], 8 * D, D, a["bounds"], 5, P, 4, P, 4, 1, 1, P, P, P, 1 << 20,
                               None, None) == 1


ATTEND = ["q", "kp", "vp", "table", "lens", "out"]


@pytest.mark.parametrize("name", ATTEND)
def test_attention_over_blocks_wants_its_buffers(lib, name):
    a = {n: P for n in ATTEND}
    a[name] = None
    assert lib.hc_flash_decode_blocks(1, 1, 2, 4, D, a["q"], 8 * D, D, a["kp"], a["vp"], 5, a["table"], 2, a["lens"], P,
                                      P, 4, 0.0, a["out"], P, 1 << 30, None, None) == 1


@pytest.mark.parametrize("name", ATTEND + ["bounds", "blocks", "counts"])
def test_sparse_wants_its_buffers(lib, name):
    a = {n: P for n in ATTEND + ["bounds", "blocks", "counts"]}
    a[name] = None
    assert lib.hc_flash_decode_sparse(1, 1, 2, 4, D, a["q"], 8 * D, D, a["kp"], a["vp"], 5, a["table"], 2, a["lens"],
                                      a["bounds"], 4, 1, 1, 0.0, a["out"], a["blocks"], a["counts"], P, 1 << 30, None,
                                      None) == 1


@pytest.mark.parametrize("name", ATTEND)
def test_shared_wants_its_buffers(lib, name):
    a = {n: P for n in ATTEND}
    a[name] = None
    assert lib.hc_flash_decode_shared(1, 2, 2, 4, D, a["q"], 8 * D, D, a["kp"], a["vp"], 5, a["table"], 2, a["lens"], P,
                                      None, None, 0, 0, 0, 0, 0.0, a["out"], P, 1 << 30, None, None) == 1


def test_a_workspace_off_its_alignment(lib):
    big = 1 << 30
    assert lib.hc_block_select(1, 1, 2, 4, D, P, 8 * D, D, P, 5, P, 4, P, 4, 1, 1, P, P, P + 4, big, None, None) == 6
    assert lib.hc_flash_decode_blocks(1, 1, 2, 4, D, P, 8 * D, D, P, P, 5, P, 2, P, P, P, 4, 0.0, P, P + 4, big, None,
                                      None) == 6
    assert lib.hc_flash_decode_sparse(1, 1, 2, 4, D, P, 8 * D, D, P, P, 5, P, 2, P, P, 4, 1, 1, 0.0, P, P, P, P + 8,
                                      big, None, None) == 6
