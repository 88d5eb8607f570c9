"""Where the cuts of the attention's line of work fall (csrc/attention_line.h, compiled for the host)."""
from __future__ import annotations

import pathlib
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "neuronmlp-on-tpu_b200" / "csrc"
COSTS, SNAPS, STEPS = (2, 4), (2, 4, 8, 16), range(1, 41)


@pytest.fixture(scope="module")
def places(tmp_path_factory):
    """{(cost, snap, steps): the step of the cut for every place in the unit}."""
    if shutil.which("g++") is None:
        pytest.skip("needs a C++ compiler")
    tmp = tmp_path_factory.mktemp("line")
    src = tmp / "line.cpp"
    src.write_text('#include <cstdio>\n#include <initializer_list>\n#include "attention_line.h"\nint main() {\n'
                   f'for (int cost : {{{", ".join(map(str, COSTS))}}}) for (int snap : {{{", ".join(map(str, SNAPS))}}})\n'
                   f'for (int steps = 1; steps <= {STEPS[-1]}; ++steps) {{\n'
                   'std::printf("%d %d %d", cost, snap, steps);\n'
                   'for (int in = 0; in < cost + steps; ++in) std::printf(" %d", svdmlp::cut_step(in, steps, cost, snap));\n'
                   'std::printf("\\n"); }\n}\n')
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(src), "-o", str(tmp / "line")], check=True)
    rows = subprocess.run([str(tmp / "line")], check=True, capture_output=True, text=True).stdout.splitlines()
    table = [tuple(map(int, r.split())) for r in rows]
    return {r[:3]: r[3:] for r in table}


def test_cuts_keep_their_order(places):
    """A cut behind another never falls before it: no step is done twice, none is left out."""
    assert len(places) == len(COSTS) * len(SNAPS) * len(STEPS)
    for key, row in places.items():
        assert list(row) == sorted(row), key
        assert row[0] == 0 and 0 <= row[-1] <= key[2], key


def test_short_units_are_whole_and_long_ones_are_cut_at_every_step(places):
    for (cost, snap, steps), row in places.items():
        if steps <= snap:
            assert set(row) <= {0, steps}
            assert all((j == steps) == (2 * i > steps + cost) for i, j in enumerate(row))
        else:
            assert row == (0,) * cost + tuple(range(steps))
