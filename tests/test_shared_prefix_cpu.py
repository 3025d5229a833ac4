"""Host side of the shared-prefix decode, without a GPU."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from shared_prefix_common import assert_close, case, plain
from test_rope_cpu import _Cuda


def test_plain_form_equals_the_oracle_of_the_paged_decode():
    import oracle

    cpu = case(3, 4, 4, 32, 16, 48, [5, 0, 33], torch.float32, seed=3)
    cpu.tables[:, :3] = cpu.table
    want = oracle.paged_decode_dense(cpu.q, cpu.pool.k, cpu.pool.v, cpu.tables, cpu.lens, 0,
                                     compute_dtype=torch.float64)
    assert torch.allclose(plain(cpu)[0], want, rtol=0, atol=1e-12)
    assert_close(cpu, want.float(), tensor_cores=False)


def _args(**kw):
    from b200attn import _lib

    i64 = _lib.INDEX_I64
    v = dict(pool=_lib.KVPool(1 << 20, 2 << 20, 2, 8, 16, 2, 64, _lib.DTYPE_BF16), layer_idx=1,
             batch=3, num_q_heads=8, prefix_len=33, table_width=4, q=3 << 20, q_s0=512, q_s1=64,
             q_s2=1, out=4 << 20, out_s0=512, out_s1=64, out_s2=1, prefix_table=5 << 20,
             prefix_table_len=3, prefix_table_stride=1, block_tables=6 << 20, block_table_s0=4,
             block_table_s1=1, context_lengths=7 << 20, context_length_stride=1,
             q_dtype=_lib.DTYPE_BF16, out_dtype=_lib.DTYPE_BF16, prefix_table_dtype=i64,
             block_table_dtype=i64, context_length_dtype=i64)
    v.update(kw)
    return _lib.SharedPrefixArgs(**v)


BAD = {
    "layer": dict(layer_idx=2),
    "empty batch": dict(batch=0),
    "no query heads": dict(num_q_heads=0),
    "heads not a multiple": dict(num_q_heads=7),
    "too many rows": dict(batch=1 << 23, num_q_heads=64),
    "no columns": dict(table_width=0),
    "negative prefix": dict(prefix_len=-1),
    "prefix too long": dict(prefix_len=1 << 30, prefix_table_len=1 << 30),
    "short prefix table": dict(prefix_table_len=2),
    "null prefix table": dict(prefix_table=None),
    "null q": dict(q=None),
    "null out": dict(out=None),
    "null tables": dict(block_tables=None),
    "null lengths": dict(context_lengths=None),
    "q dtype": dict(q_dtype=5),
    "out dtype": dict(out_dtype=5),
    "prefix table dtype": dict(prefix_table_dtype=5),
    "tables dtype": dict(block_table_dtype=5),
    "lengths dtype": dict(context_length_dtype=5),
}


@pytest.mark.parametrize("why", BAD)
def test_c_entry_refuses(why):
    from b200attn import _lib

    lib = _lib.load()
    rc = lib.b200_shared_prefix_decode(ctypes.byref(_args(**BAD[why])), None)
    assert rc in (_lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED) and _lib.last_error(lib)


def test_c_entry_refuses_null_and_a_misaligned_workspace():
    from b200attn import _lib

    lib = _lib.load()
    assert ctypes.sizeof(_lib.SharedPrefixArgs) == 64 + 24 * 8 + 6 * 4
    assert lib.b200_shared_prefix_decode(None, None) == _lib.ERR_INVALID_ARGUMENT
    a = _args(workspace=(8 << 20) + 16, workspace_bytes=1 << 30)
    assert lib.b200_shared_prefix_decode(ctypes.byref(a), None) == _lib.ERR_WORKSPACE


def test_workspace_size_is_bounded_by_the_parts():
    from b200attn import _lib

    size = _lib.load().b200_shared_prefix_decode_workspace_size
    bf16 = _lib.DTYPE_BF16
    assert size(0, 8, 8, 128, 0, 4, 16, bf16, bf16) == 0
    assert size(4, 8, 16, 128, 0, 4, 16, bf16, bf16) == 0  # fewer query heads than heads
    assert size(4, 32, 8, 128, 2048, 132, 16, bf16, bf16) > 0
    # A row has at most 64 parts of the prefix and 32 of its own.
    for b, width in ((1, 1), (3, 4096), (64, 4096), (256, 65536), (3, 65536)):
        for prefix in (0, 1, 4096, width * 16):
            got = size(b, 32, 8, 128, prefix, width, 16, bf16, bf16)
            assert 0 < got <= b * 32 * 96 * (128 + 2) * 4 + b * 8 * 4 + 4 * 256


def test_python_entry_refuses():
    from b200attn import shared_prefix_decode_b200

    cpu = case(3, 8, 2, 32, 16, 33, [1, 2, 3], torch.float32, seed=1)
    with pytest.raises(ValueError, match="CUDA"):
        shared_prefix_decode_b200(cpu.q, cpu.pool, cpu.table, 33, cpu.tables, cpu.lens, 0)
    with pytest.raises(RuntimeError, match="inference"):
        shared_prefix_decode_b200(cpu.q.clone().requires_grad_(), cpu.pool, cpu.table, 33, cpu.tables,
                                  cpu.lens, 0)

    def refuse(match, q=cpu.q, pool=cpu.pool, table=cpu.table, prefix=33, tables=cpu.tables,
               lens=cpu.lens, layer=0, **kw):
        with pytest.raises(ValueError, match=match):
            shared_prefix_decode_b200(_Cuda(q), pool, table, prefix, tables, lens, layer, **kw)

    refuse("shape", q=cpu.q[0])
    refuse("nonzero", q=cpu.q[:0])
    refuse("float32", q=cpu.q.double())
    refuse("head dimension", q=cpu.q[..., :16])
    refuse("head dimension", q=cpu.q[:, :7])
    refuse("block_tables", tables=cpu.tables[:2])
    refuse("block_tables", tables=cpu.tables[:, :0])
    refuse("context_lengths", lens=cpu.lens[:2])
    refuse("integers", lens=cpu.lens.float())
    refuse("integers", tables=cpu.tables.float())
    refuse("layer_idx", layer=1)
    refuse("prefix_len", prefix=-1)
    refuse("incomplete", prefix=49)
    refuse("1-D", table=cpu.table[None])
    refuse("integer", table=cpu.table.float())
    refuse("status", status=torch.zeros(1))
    refuse("out must", out=torch.zeros(3, 8, 16))
    refuse("overlap itself", out=torch.zeros(1, 1, 32).expand(3, 8, 32))
    refuse("overlap the inputs", q=(both := torch.zeros(4, 8, 32))[:3], out=both[1:])
    half = torch.zeros(3, 8, 64, dtype=torch.bfloat16)
    refuse("overlap the inputs", q=half.view(torch.float32), out=half[..., :32])
    pool = SimpleNamespace(k=cpu.pool.k.half(), v=cpu.pool.v.half(), block_size=16)
    refuse("dtype", pool=pool)


def test_torch_op_has_a_fake_shape():
    import b200attn  # noqa: F401

    with FakeTensorMode():
        q = torch.empty(3, 8, 64, device="cuda")
        pool = torch.empty(1, 2, 16, 2, 64, device="cuda")
        t = torch.empty(3, dtype=torch.int64, device="cuda")
        out = torch.ops.b200attn.shared_prefix_decode(q, pool, pool, t, 16, t[:, None], t, 0)
        assert out.shape == q.shape
