"""CPU test of the kernels' source: LDS that asynchronous copies fill is read behind the wait for them.

The builtin that waits touches no memory as the compiler sees it, so nothing but what follows it (an empty asm that clobbers
memory, or a barrier with one) keeps the compiler from moving reads of the copied bytes before it."""

import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "tttj_2026_amd" / "csrc"
SOURCES = sorted(p for p in CSRC.iterdir() if p.suffix in (".hip", ".hpp") and "wait_vmcnt<" in p.read_text())
FENCE = re.compile(r"asm volatile|raw_barrier\(\)|__syncthreads\(\)")
PASSED = re.compile(r"wait_vmcnt<|^else|^\}|^#pragma")  # other branches, closing braces


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_reads_stay_behind_their_wait(source):
    lines = [re.sub(r"//.*", "", line).strip() for line in source.read_text().split("\n")]
    for at, line in enumerate(lines):
        if "wait_vmcnt<" not in line or "break;" in line:  # (a switch of waits: its callers have the barrier)
            continue
        after = next(x for x in lines[at + 1:] if x and not PASSED.search(x))
        if source.name == "gemm_tile.hpp" and after.startswith("constexpr int RL"):
            continue  # the last wait of a branch: the epilogue begins with a barrier
        assert FENCE.search(after), (source.name, at + 1, after)


def test_all_waits_are_looked_at():
    assert {"seq_attention.hpp", "gemm_tile.hpp", "gemm_narrow.hpp", "attention_block.hpp"} <= {p.name for p in SOURCES}
