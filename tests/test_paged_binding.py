"""The native calls of the paged operators: arguments of another kind are refused as Python errors."""
import pytest
import torch

from heterocache_b200 import _lib, ops
from test_paged_ops_checks import _append_args, _decode_args, i32

D = 128


@pytest.fixture(scope="module", autouse=True)
def _built():
    import __graft_entry__
    __graft_entry__.build()


@pytest.mark.parametrize("name", ["q", "cos", "k_pool", "block_table", "err"])
@pytest.mark.parametrize("value", [None, 3, "x", [1.0]])
def test_what_is_no_tensor(name, value):
    with pytest.raises(TypeError, match=f"{name} must be a tensor"):
        ops.rope_append(**_append_args(**{name: value}))


@pytest.mark.parametrize("name", ["counts", "q_out", "heads_len_out", "bounds"])
def test_optional_operands_are_tensors_or_none(name):
    with pytest.raises(TypeError, match=f"{name} must be a tensor"):
        ops.rope_append(**_append_args(**{name: 7}))
    with pytest.raises(ValueError, match="CUDA device"):
        ops.rope_append(**_append_args(**{name: None}))


@pytest.mark.parametrize("name,value,error", [
    ("n_select", 2 ** 32 + 4, ValueError), ("sink", -2 ** 40, ValueError), ("n_select", 2 ** 70, OverflowError),
    ("n_select", "4", TypeError), ("num_kv_heads", 2.0, TypeError), ("scale", "x", TypeError), ("scale", None, TypeError),
])
def test_numbers(name, value, error):
    a = _decode_args(bounds=torch.zeros(5, 4, 2, D, dtype=torch.bfloat16), n_select=4, sink=1, recent=2)
    a[name] = value
    with pytest.raises(error):
        ops.flash_decode_sparse(**a)


def test_tensors_without_dimensions():
    with pytest.raises(ValueError, match="contiguous last dim"):
        ops.rope_append(**_append_args(q=torch.zeros((), dtype=torch.bfloat16)))
    with pytest.raises(ValueError, match="row per"):
        ops.rope_append(**_append_args(block_table=torch.zeros((), dtype=i32)))
    with pytest.raises(ValueError, match="bounds must"):
        ops.block_select(**{k: v for k, v in _decode_args(bounds=torch.zeros(()), n_select=4).items()
                            if k not in ("k_pool", "v_pool")})


def test_the_number_of_arguments():
    for name in ("rope_append", "flash_decode_shared", "block_bounds", "block_select", "flash_decode_blocks",
                 "flash_decode_sparse"):
        with pytest.raises(TypeError, match="arguments in place of"):
            getattr(_lib.paged(), name)(torch.zeros(1))
