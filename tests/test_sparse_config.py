"""HeteroCacheConfig's block-sparse options: what no decode step could use is refused when it is given."""
import pytest

from heterocache_b200.cache import HeteroCacheConfig


@pytest.mark.parametrize("blocks,sink,recent", [(4, -1, 2), (4, 3, -1), (-1, 0, 0), (-4, -3, -2), (2, 1, 2)])
def test_refused(blocks, sink, recent):
    with pytest.raises(ValueError, match="sparse_"):
        HeteroCacheConfig({}, sparse_blocks=blocks, sparse_sink=sink, sparse_recent=recent)


@pytest.mark.parametrize("blocks,sink,recent", [(0, 1, 2), (1, 0, 0), (3, 1, 2), (64, 0, 64)])
def test_taken(blocks, sink, recent):
    c = HeteroCacheConfig({}, sparse_blocks=blocks, sparse_sink=sink, sparse_recent=recent)
    assert (c.sparse_blocks, c.sparse_sink, c.sparse_recent) == (blocks, sink, recent)
