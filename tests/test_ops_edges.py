"""Index rules of the operators on device tensors at their edges (csrc/z2h_ops_rules.h), on the CPU."""
import itertools
import subprocess

import pytest

from ops_cut_cases import BLOCKS, CASES, group_tables


def test_ops_edges(root, tmp_path):
    exe = tmp_path / "ops_edges_kat"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", f"-I{root / 'include'}",
                    str(root / "tests" / "native" / "ops_edges_kat.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


@pytest.fixture(scope="module")
def cut_tool(root, tmp_path_factory):
    exe = tmp_path_factory.mktemp("ops_cut") / "ops_cut"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", f"-I{root / 'include'}", str(root / "tests" / "native" / "ops_cut.cpp"), "-o", str(exe)],
                   check=True)
    return exe


@pytest.mark.parametrize("name", list(CASES))
def test_cut_cases_reach_what_they_are_for(cut_tool, name):
    c = CASES[name]
    start, prefix = group_tables(c)
    rows = [0, *itertools.accumulate(c["rows"])]
    head = [BLOCKS, c["kvh"], c["heads"] // c["kvh"], len(c["lens"]), len(prefix)]
    text = " ".join(map(str, head + rows + c["lens"] + (start + prefix if prefix else [])))
    out = subprocess.run([str(cut_tool)], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
    keys = ("tiles", "strips", "shift", "share", "head", "longest", "several", "small")
    narrow, wide = (dict(zip(keys, map(int, line.split()))) for line in out[:2])
    assert c["reaches"](narrow, wide), (narrow, wide)
