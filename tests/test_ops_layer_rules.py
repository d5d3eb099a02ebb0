"""The refusals, sizes and index rules of the operators for whole prompts, experts and a cache's upkeep (csrc/z2h_ops_rules.h), on the CPU."""
import subprocess


def test_ops_layer_rules(root, tmp_path):
    exe = tmp_path / "ops_layer_kat"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", f"-I{root / 'include'}",
                    str(root / "tests" / "native" / "ops_layer_kat.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
