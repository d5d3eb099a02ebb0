"""The refusals, page look-ups, rotary frequencies and workspace rules of the operators on device tensors
(csrc/z2h_ops_rules.h), on the CPU."""
import subprocess


def test_ops_rules(root, tmp_path):
    exe = tmp_path / "ops_rules_kat"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", f"-I{root / 'include'}",
                    str(root / "tests" / "native" / "ops_rules_kat.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
