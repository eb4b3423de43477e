"""rope_append: a q_out that overlaps itself is refused, one of any other order is not, on the host."""
import pytest
import torch

from heterocache_b200 import ops
from test_paged_ops_checks import _append_args, i32

D = 128
bf = torch.bfloat16


@pytest.mark.parametrize("name,value", [
    ("q_out", torch.zeros(2, 1, 3, D, dtype=bf).expand(2, 4, 3, D)),            # one head's rows for all
    ("q_out", torch.zeros(2, 4, 1, D, dtype=bf).expand(2, 4, 3, D)),            # one token's
    ("q_out", torch.zeros(1, 4, 3, D, dtype=bf).expand(2, 4, 3, D)),            # one sequence's
    ("q_out", torch.zeros(4096, dtype=bf).as_strided((2, 4, 3, D), (1024, 256, 64, 1))),  # rows that overlap
])
def test_an_output_that_overlaps_itself(name, value):
    with pytest.raises(ValueError, match="overlap"):
        ops.rope_append(**_append_args(**{name: value}))


def test_outputs_of_any_order_are_taken():
    """Dense in another order, with gaps, or of extent 1 with any stride: refused only for not being on a GPU."""
    for q_out in (torch.zeros(3, 2, 4, D, dtype=bf).permute(1, 2, 0, 3), torch.zeros(2, 8, 6, 2 * D, dtype=bf)[:, ::2, ::2, :D],
                  torch.zeros(2, 3, 4, D, dtype=bf).transpose(1, 2)):
        with pytest.raises(ValueError, match="CUDA device"):
            ops.rope_append(**_append_args(q_out=q_out))
    one = _append_args(q=torch.zeros(1, 4, 1, D, dtype=bf), k=torch.zeros(1, 2, 1, D, dtype=bf),
                       v=torch.zeros(1, 2, 1, D, dtype=bf), cos=torch.zeros(1, 1, D, dtype=bf),
                       sin=torch.zeros(1, 1, D, dtype=bf), block_table=torch.zeros(2, 2, dtype=i32),
                       heads_len=torch.zeros(2, dtype=i32),
                       q_out=torch.zeros(4 * D, dtype=bf).as_strided((1, 4, 1, D), (0, D, 0, 1)))
    with pytest.raises(ValueError, match="CUDA device"):
        ops.rope_append(**one)


def test_a_query_that_overlaps_itself_is_no_output():
    """q may be expanded where it is read alone, not where it is q_out too."""
    q = torch.zeros(2, 1, 3, D, dtype=bf).expand(2, 4, 3, D)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.rope_append(**_append_args(q=q))
    with pytest.raises(ValueError, match="overlap"):
        ops.rope_append(**_append_args(q=q, q_out=q))
