"""Shared-prefix decode with block tables wider than the sequences need, as a
serving loop keeps them, and with views of the columns that they do need."""
from __future__ import annotations

import pytest
import torch

from shared_prefix_common import assert_close, case, to_device

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("size", [(2, 8, 2, 64, 16, 100, [5, 700]),
                                  (260, 8, 8, 64, 16, 80, [i % 9 for i in range(259)] + [3000]),
                                  (260, 32, 8, 128, 16, 400, [i % 9 for i in range(259)] + [5000])],
                         ids=lambda s: str(s[:6]))
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_wide_tables_and_views_of_their_first_columns(size, dtype):
    from b200attn import _lib, shared_prefix_decode_b200

    cpu = case(*size, dtype, seed=91)
    rows = size[0] * size[1] // size[2]
    pieces = False if dtype == F32 else "split" if rows <= 128 else True
    c = to_device(cpu)
    need = c.tables.shape[1]
    wide = torch.full((size[0], 2048), -1, dtype=torch.int64, device="cuda")
    wide[:, :need] = c.tables
    for tables in (c.tables, wide, wide[:, :need], wide[:, : need + 40]):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = shared_prefix_decode_b200(c.q, c.pool, c.table, c.prefix, tables, c.lens, c.layer,
                                        status=status)
        assert int(status) == 0
        assert_close(cpu, out, tensor_cores=pieces)
    # A row that the view cuts off is told, and zero; the others are whole.
    cut = wide[:, : need - 2]
    out = shared_prefix_decode_b200(c.q, c.pool, c.table, c.prefix, cut, c.lens, c.layer,
                                    status=status)
    assert int(status) == _lib.DEV_BAD_LENGTH
    cpu.lens[-1] = 0
    assert not out[-1].any()
    assert_close(cpu, out, tensor_cores=pieces)
