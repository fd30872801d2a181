"""The shapes that linear attention's passes take (tests/walk_plan.cpp compiles the launcher's rules for the host alone)."""
import math
import os
import shutil
import subprocess

import pytest

from tests import walk_cases

HERE = os.path.dirname(os.path.abspath(__file__))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    """[(type, packed, sequences, tokens, heads, dim, columns, passes together)] -> [(state rows, waves, late, chunk, segment, split, cost)]."""
    if shutil.which(HIPCC) is None:
        pytest.skip("no hipcc")
    tool = str(tmp_path_factory.mktemp("plan") / "walk_plan")
    subprocess.run([HIPCC, "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", os.path.join(HERE, "walk_plan.cpp"), "-o", tool], check=True)

    def ask(rows):
        text = "".join(" ".join(str(int(v)) for v in r) + "\n" for r in rows)
        out = subprocess.run([tool], input=text, capture_output=True, text=True, check=True).stdout.splitlines()
        assert len(out) == len(rows)
        return [(*map(int, line.split()[:6]), float(line.split()[6])) for line in out]

    return ask


def test_every_plan_has_a_cost(plans):
    rows = [(t, packed, count, n, h, d, c, together) for t in range(3) for packed in (0, 1) for count in (1, 7, 500) for n in (0, 1, 30, 64, 65, 128, 3000)
            for h in (1, 32) for d, c in ((16, 16), (64, 128), (128, 128), (256, 256)) for together in (1, 3)]
    for row, (dk, w, late, chunk, segment, split, cost) in zip(rows, plans(rows)):
        assert math.isfinite(cost) and 0 < cost < 1e12, row
        assert dk >= row[5] and segment % chunk == 0 and segment > 0 and split == (row[3] > segment), row


def test_sequences_of_one_chunk_form_their_scores_once(plans):
    """128 columns a workgroup of more than 64, whatever the estimate says of either."""
    rows = [(t, packed, 9, n, 8, d, c, 1) for t in range(3) for packed in (0, 1) for n in (1, 32) for d in (32, 64, 128, 256) for c in (65, 128, 200)]
    assert all(p[1] == 8 for p in plans(rows))
    assert all(p[1] == 4 for p in plans([(t, 0, 9, 32, 8, 64, 64, 1) for t in range(3)]))


def test_the_cases_reach_every_walk(plans):
    """tests/walk_cases.py, which the GPU's tests run: every shape of every type, split and not; those that two workgroups a CU take
    forwards and backwards."""
    reached = {}
    for c in walk_cases.CASES:
        for kind in c["types"]:
            for part, (dk, w, late, _, _, split, _) in zip(("forward", "backward", "backward"), plans(walk_cases.passes(c, kind))):
                reached.setdefault((kind, dk, w, split, late), set()).add(part)
    shapes = {(dk, w) for dk in (32, 64, 128, 256) for w in (4, 8)} | {(dk, w) for dk in (32, 64) for w in (1, 2)}
    assert {r[:4] for r in reached} == {(kind, *s, split) for kind in range(3) for s in shapes for split in (0, 1)}
    late = {r[:4] for r in reached if r[4]}
    assert late == {(kind, dk, 8, split) for kind, dks in ((0, (32, 64)), (2, (32, 64, 128))) for dk in dks for split in (0, 1)}
    assert all(reached[(*r, 1)] == {"forward", "backward"} for r in late)
