"""Which kernel the products of the GPU tests run on, by the dispatch's own table: a size that a changed table sends elsewhere is
noticed here."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

import test_gpu_fp8
import test_gpu_fp8_large

SOURCE = (Path(__file__).resolve().parents[1] / "bigsmall_amd" / "csrc" / "fp8_linear.hip").read_text()
CUS = 256


def _table():
    text = SOURCE[SOURCE.index("const Shape SHAPES[] = {"):]
    number = r"([\d.]+)f?, "
    rows = re.findall(r"\{" + number * 8 + r"(\w+)(?:<\w+<([\d, ]+)>>)?\}", text[:text.index("};")])
    return [tuple(map(float, r[:8])) + (r[8] + ("_" + r[9].replace(", ", "_") if r[9] else ""),) for r in rows]


def _pick(t, n, k):
    """The shape's name and its number of tiles."""
    blocks, best = -(-k // 128), None
    for rows_w, rows_x, waves, fixed, start, one, start2, two, name in _table():
        tiles = -(-n // int(rows_w)) * -(-t // int(rows_x))
        each, turns = -(-tiles // CUS), -(-blocks // int(waves))
        us = fixed + each // 2 * (start2 + turns * two) + each % 2 * (start + turns * one)
        if best is None or us < best[0]:
            best = us, name, tiles
    return best[1:]


def test_the_table_is_read_whole():
    names = [r[-1] for r in _table()]
    assert len(names) == len(set(names)) == 9 and names[-1] == "large_go" and SOURCE.count("_go<") + 1 == 9


@pytest.mark.parametrize("t,n,k", test_gpu_fp8_large.SEVERAL_TILES)
def test_several_large_tiles_to_a_workgroup(t, n, k):
    name, tiles = _pick(t, n, k)
    assert name == "large_go" and tiles > CUS


def test_every_shape_is_tested():
    sizes = [s for s in test_gpu_fp8.SHAPES + test_gpu_fp8.LARGE + test_gpu_fp8.MANY + test_gpu_fp8_large.SEVERAL_TILES]
    assert {_pick(*s)[0] for s in sizes} == {r[-1] for r in _table()}
