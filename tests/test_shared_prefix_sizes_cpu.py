"""The workspace query of the shared-prefix decode over all sizes, without a GPU."""
from __future__ import annotations

import subprocess
import sys

import b200attn  # noqa: F401
from b200attn import _lib

BF16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F32
GOOD = (64, 32, 8, 128, 4096, 1024, 16, BF16, BF16)


def _with(**kw):
    names = ("batch", "hq", "hkv", "d", "prefix", "width", "block", "kv", "q")
    return tuple(kw.get(n, g) for n, g in zip(names, GOOD))


REFUSED = {
    "prefix of 2^39 - 768, whose 32-bit tile count is -6": _with(prefix=((1 << 32) - 6) * 128),
    "prefix of 2^30": _with(prefix=1 << 30),
    "prefix of 2^62": _with(prefix=1 << 62),
    "negative prefix": _with(prefix=-1),
    "too many rows": _with(batch=1 << 23),
    "rows past 64 bits": _with(batch=1 << 62, hq=1 << 15),
    "wide table": _with(width=1 << 30),
    "no columns": _with(width=0),
    "heads not a multiple": _with(hq=33),
    "no key heads": _with(hkv=0),
    "no query heads": _with(hq=0),
    "wide heads": _with(d=136),
    "no head": _with(d=0),
    "odd pages": _with(block=24),
    "long pages": _with(block=512),
    "no pages": _with(block=0),
}


def test_sizes_that_the_call_refuses_need_no_workspace():
    # In a process of its own: a division by zero in the library would end this one.
    code = (f"import sys; sys.path[:0] = {sys.path!r}\n"
            "from b200attn import _lib\n"
            "size = _lib.load().b200_shared_prefix_decode_workspace_size\n"
            f"for why, sizes in {REFUSED!r}.items():\n"
            "    assert size(*sizes) == 0, why\n")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr


def test_sizes_at_the_limits():
    size = _lib.load().b200_shared_prefix_decode_workspace_size
    for kv, q in ((BF16, BF16), (BF16, F32), (F32, F32)):
        for kw in (dict(prefix=(1 << 30) - 1, width=1 << 20), dict(batch=1 << 20, hq=32, hkv=1),
                   dict(batch=1, hq=1, hkv=1, prefix=0, width=1), dict(batch=1023, hq=65535, hkv=65535),
                   dict(width=(1 << 30) - 1)):
            assert size(*_with(kv=kv, q=q, **kw)) > 0


def test_wide_tables_do_not_multiply_the_parts_of_a_large_batch():
    """A row's own parts cost workspace, and CTAs, by the table's width: few in a
    large batch, all 32 in a small one."""
    size = _lib.load().b200_shared_prefix_decode_workspace_size
    part = lambda b: b * 32 * (128 + 2) * 4  # noqa: E731
    wide, tight = (size(*_with(batch=256, width=w)) for w in (8192, (4096 + 128) // 16))
    assert 0 < wide - tight <= 7 * part(256) + 1024
    wide, tight = (size(*_with(batch=16, width=w)) for w in (8192, (4096 + 128) // 16))
    assert wide - tight >= 28 * part(16)
