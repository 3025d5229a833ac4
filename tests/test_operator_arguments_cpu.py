"""Arguments that the rotary operators and the shared-prefix decode refuse: one
tensor as two inputs of a call in place, pools without heads.  Refusals come
before any launch."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from test_rope_cpu import _Cuda


@pytest.mark.parametrize("which", ["q", "k"])
def test_one_tensor_as_q_and_k_is_not_rotated_in_place(which):
    """q's rows would be written while k's, the same, are still to be read."""
    from b200attn import qk_norm_rope_b200, rope_table

    x = torch.zeros(3, 4, 32)
    pos, table = torch.zeros(3, dtype=torch.int64), rope_table(8, 32)
    q, k = (_Cuda(x), x)
    out = {"q_out": x} if which == "q" else {"k_out": x}
    with pytest.raises(ValueError, match="not overlap the inputs"):
        qk_norm_rope_b200(q, k, pos, table, **out)
    with pytest.raises(ValueError, match="not overlap the inputs"):
        same = _Cuda(x)
        qk_norm_rope_b200(same, same, pos, table, **out)


def test_one_tensor_as_k_and_v_of_an_append_in_place():
    from b200attn import rope_kv_append_b200, rope_table

    x = torch.zeros(3, 2, 32)
    pool = SimpleNamespace(k=torch.zeros(1, 4, 4, 2, 32), v=torch.zeros(1, 4, 4, 2, 32), block_size=4)
    with pytest.raises(ValueError, match="not overlap the inputs"):
        rope_kv_append_b200(_Cuda(x), torch.zeros(3, 2, 32), x, pool, torch.arange(3),
                            torch.zeros(3, dtype=torch.int64), rope_table(8, 32), 0, q_out=x)


def test_a_pool_without_heads():
    from b200attn import shared_prefix_decode_b200

    pool = SimpleNamespace(k=torch.zeros(1, 2, 16, 0, 32), v=torch.zeros(1, 2, 16, 0, 32), block_size=16)
    tables = torch.zeros(3, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="head dimension"):
        shared_prefix_decode_b200(_Cuda(torch.zeros(3, 8, 32)), pool, tables[0], 16, tables,
                                  torch.full((3,), 17), 0)
