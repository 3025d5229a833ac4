"""Shared-prefix decode of pools that hold infinities where they are read: the
outputs are those of the definition, infinite or not numbers where it has them."""
from __future__ import annotations

import copy

import pytest
import torch

from shared_prefix_common import bound, case, plain, to_device

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")

# b, hq, hkv, d, block, prefix, own: few rows, one tile of rows, two, a second that is partly full.
SIZES = [(3, 8, 2, 64, 16, 600, [5, 130, 40]),
         (20, 16, 16, 64, 16, 3001, [3 + i % 7 for i in range(20)]),
         (5, 64, 16, 128, 16, 2801, [4, 64, 17, 33, 200]),
         (40, 32, 8, 128, 32, 2900, [2 + i for i in range(40)])]
TYPES = [(BF16, BF16), (F16, BF16), (F32, BF16), (F32, F32)]
ALL = [pytest.mark.parametrize("size", SIZES, ids=lambda s: str(s[:6])),
       pytest.mark.parametrize("types", TYPES, ids=str)]


def _all(f):
    for mark in ALL:
        f = mark(f)
    return f


def _run(cpu):
    from b200attn import shared_prefix_decode_b200

    c = to_device(cpu)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = shared_prefix_decode_b200(c.q, c.pool, c.table, c.prefix, c.tables, c.lens, c.layer,
                                    status=status)
    assert int(status) == 0
    return out.cpu()


def _row(cpu, i, n):
    """(page, row) of position n of sequence i."""
    page = cpu.table[n // cpu.block] if n < cpu.prefix else cpu.tables[i, n // cpu.block]
    return int(page), n % cpu.block


def _check(cpu, got, tensor_cores):
    want, spread, _ = plain(cpu)
    for what, test in (("NaN", torch.isnan), ("+inf", torch.isposinf), ("-inf", torch.isneginf)):
        other = int((test(got) != test(want)).sum())
        assert other == 0, f"{other} elements of {want.numel()} are {what} on one side alone"
    fine = want.isfinite()
    # Scores of -inf have no rounding; the bound goes by the finite ones.
    finite = copy.copy(cpu)
    finite.pool = copy.copy(cpu.pool)
    finite.pool.k = torch.where(cpu.pool.k.isinf(), 0.0, cpu.pool.k)
    big = plain(finite)[2]
    lim = bound(cpu, want, spread, big, tensor_cores)
    bad = int((~((got.double() - want).abs() <= lim) & fine).sum())
    assert bad == 0, f"{bad} elements beyond the bound"
    return want


def _weights(types, size):
    rows = size[0] * size[1] // size[2]
    if types[1] == F32 or types[0] == F32:
        return False
    return "split" if types[0] == F16 or rows <= 128 else True


@_all
def test_infinite_values_give_infinities(size, types):
    """Elements of V that are infinite, of prefix and own keys, with weights of
    every kind; the elements beside them keep their numbers."""
    cpu = case(*size, *types, seed=61)
    v = cpu.pool.v
    for n, d, x in ((0, 3, INF), (size[5] // 2, 9, -INF), (size[5] - 1, 17, INF)):
        v[0][_row(cpu, 0, n)][:, d] = x
    for i in range(size[0]):
        v[0][_row(cpu, i, size[5])][0, 21] = -INF
        v[0][_row(cpu, i, int(cpu.lens[i]) - 1)][-1, 30] = INF
    want = _check(cpu, _run(cpu), _weights(types, size))
    assert want.isinf().sum() >= 4 * size[0] and not want.isnan().any()


@_all
def test_infinities_of_both_signs_are_no_number(size, types):
    cpu = case(*size, *types, seed=62)
    cpu.pool.v[0][_row(cpu, 0, 1)][:, 5] = INF
    cpu.pool.v[0][_row(cpu, 0, size[5] - 2)][:, 5] = -INF
    want = _check(cpu, _run(cpu), _weights(types, size))
    assert want[..., 5].isnan().all()


@_all
def test_a_key_with_an_infinite_element(size, types):
    """Its score is -inf for about half of the rows, which it gives no weight,
    and +inf for the others, which have no softmax."""
    cpu = case(*size, *types, seed=63)
    cpu.pool.k[0][_row(cpu, 0, 7)][:, 11] = INF
    cpu.pool.k[0][_row(cpu, 0, size[5] - 1)][:, 40] = -INF
    cpu.q[..., 40] = -cpu.q[..., 11]  # every infinite score of a row has one sign
    for i in range(size[0]):
        cpu.pool.k[0][_row(cpu, i, size[5] + 1)][:, 11] = INF
    want = _check(cpu, _run(cpu), _weights(types, size))
    odd = want.isnan().any(-1)
    assert odd.any() and not odd.all()


@ALL[0]
@pytest.mark.parametrize("types", [(F32, BF16), (F32, F32)], ids=str)
def test_queries_next_to_the_largest_number(size, types):
    """Queries beyond bf16's largest number are finite in float32; keys small enough
    keep their scores of ordinary size."""
    cpu = case(*size, *types, seed=65)
    cpu.q[..., 4] = 3.4e38
    cpu.pool.k[..., 4] = (cpu.pool.k[..., 4].float().sign() * 2.0 ** -125).to(types[1])
    _check(cpu, _run(cpu), False)


@pytest.mark.parametrize("shift", [0.0, 6.0, -40.0])
@_all
def test_whole_key_tiles_without_weight(size, types, shift):
    """Scores of -inf over most of the prefix's key tiles, so that parts begin
    with them or hold nothing else; the others' scores are moved by ``shift``."""
    cpu = case(*size, *types, seed=64)
    d = size[3]
    cpu.q[..., 2] = 1.0
    k = cpu.pool.k[0]
    at = torch.arange(cpu.prefix)
    rows = cpu.table[at // cpu.block], at % cpu.block
    none = (at // 128 % 4 != 3) & (at != 5)
    k[rows[0], rows[1], :, 2] = torch.where(none, -INF, shift * d ** 0.5)[:, None].to(k.dtype)
    _check(cpu, _run(cpu), _weights(types, size))
