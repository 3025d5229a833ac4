"""Waits of the shared-prefix decode's tcgen05 kernel, read from its source: a
wait that runs out cannot be made to happen here, and what follows it must
hold for whole warps."""
from __future__ import annotations

import re
from pathlib import Path

import b200attn

SOURCE = Path(b200attn.__file__).parents[1] / "csrc" / "shared_prefix_tc.cu"


def _code() -> str:
    text = SOURCE.read_text()
    return re.sub(r"//[^\n]*", "", text)


def test_every_wait_is_a_vote_of_the_warp():
    """A lane that leaves a loop by its own poll of a barrier, or its own look at
    the abort flag, would leave the others at a full-mask vote without it."""
    code = _code()
    helpers = re.findall(r"__device__ __forceinline__ bool warp_wait\([^{]*\{[^}]*\}", code)
    assert len(helpers) == 2
    for h in helpers:
        assert re.search(r"return __all_sync\(0xffffffffu, mbar_wait\(bar, parity\)", h)
        code = code.replace(h, "")
    assert "mbar_wait(" not in code
    # Outside the helpers the flag is only set.
    uses = re.findall(r"\*abort_flag[^;]*;", code)
    assert sorted(u.replace(" ", "") for u in uses) == ["*abort_flag=0;", "*abort_flag=1;"]


def test_every_tmem_load_is_held_by_its_wait():
    """The registers of a load are operands of the wait behind it: a wait that
    names none lets the compiler move their use ahead of it."""
    code = _code()
    assert "tmem_wait_ld(" not in code
    waited = set(re.findall(r"\w+", " ".join(re.findall(r"\bwait_ld(?:4|32)\(([^;]*)\);", code))))
    loads = re.findall(r"\btmem_ld(2|32)\(([^;]*)\);", code)
    assert len(loads) >= 8
    for kind, args in loads:
        for name in [x.strip().split("[")[0] for x in args.split(",")][-2 if kind == "2" else -1:]:
            assert name in waited, args


def test_zero_rows_in_place_of_queries_wait_for_the_prefix():
    """The own-key kernels run beside the prefix's, which reads q; a row without a
    valid length is written without its parts, so that nothing else orders it
    behind those reads where out is q."""
    for name in ("shared_prefix.cu", "shared_prefix_own.cu"):
        code = re.sub(r"//[^\n]*", "", SOURCE.with_name(name).read_text())
        bad = code.split("B200_DEV_BAD_LENGTH);")
        assert len(bad) == 2
        wait, store = bad[1].find("if (p.out == p.q) wait_for_previous();"), bad[1].find("store_elem(")
        assert 0 <= wait < store


def test_waits_of_the_prefill_are_votes_too():
    """Single lanes wait for themselves only inside lane 0's branches."""
    code = re.sub(r"//[^\n]*", "", SOURCE.with_name("prefill_tc.cu").read_text())
    softmax = code[code.index("const int w = wg;"):]
    helper = "return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0;"
    assert softmax.count(helper) == 1 and "mbar_wait(" not in softmax.replace(helper, "")
    # Reads of the flag: lane 0's, for its warp, and a vote.
    reads = re.findall(r"[^;{}]*\*reinterpret_cast<volatile int32_t\*>\(abort_flag\)[^;]*;", code)
    assert len(reads) == 2
    assert "if (lane == 0)" in reads[0] and "__any_sync(0xffffffffu," in reads[1]


def test_no_kernel_waits_for_tmem_without_its_registers():
    for path in SOURCE.parent.glob("*.cu*"):
        code = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r'"tcgen05\.wait::ld[^"]*"([^;]*);', code):
            assert '"+f"(' in m[1] or '"+r"(' in m[1], (path.name, m[0])
        if "tmem_ld" in code and path.suffix == ".cu":
            assert re.search(r"\bwait_ld(?:2|4|32)\(", code), path.name
