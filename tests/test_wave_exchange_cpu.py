"""Where lanes of a wave hand results to each other through LDS without a barrier of the workgroup, the source says so to the
compiler: a fence or a statement that clobbers memory stands between the writes and the reads. Without it the order of the two
hangs on what the compiler knows of their addresses, which no test of results shows."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "bigsmall_amd" / "csrc"
ORDERS = re.compile(r'__builtin_amdgcn_fence\(__ATOMIC_ACQ_REL, "wavefront"\)|asm volatile\("" ::: "memory"\)')


def _body(file, function):
    text = re.sub(r"//[^\n]*", "", (CSRC / file).read_text())
    at = text.index("{", text.index(f" {function}("))
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at:i]
    raise AssertionError(f"{function} does not end")


@pytest.mark.parametrize("file,function,write,read", [
    ("fp8_linear.hip", "store_tile", "*(uint2*)(own", "*(const uint4*)(own"),
    ("fp8_linear.hip", "store_large", "*(uint2*)(own", "*(const uint4*)(own"),
    ("draft_verify.hip", "pick_kernel", "sums[piece] = sum", "pick(plain, W, sums")])
def test_writes_come_before_other_lanes_reads(file, function, write, read):
    body = _body(file, function)
    first, last = body.rindex(write), body.rindex(read)
    assert first < last and ORDERS.search(body, first, last), f"{function}: nothing orders its writes and reads"
