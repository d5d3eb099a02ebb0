"""The operators' entry points when a kernel cannot be launched, on the CPU: their host side alone, over a runtime that counts launches."""
import os
import subprocess


def test_no_launch_behind_one_that_failed(root, tmp_path):
    csrc = root / "zonos2.cpp_amd" / "csrc"
    inc = [f"-I{root / 'include'}", f"-I{csrc}", f"-I{root / 'zonos2.cpp_amd' / 'host'}"]
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    objs = []
    for src in (csrc / "z2h_moe.hip", csrc / "z2h_pages.hip", csrc / "z2h_prompt.hip", csrc / "z2h_ops.hip",
                root / "tests" / "native" / "ops_launch_kat.cpp"):
        objs.append(tmp_path / (src.stem + ".o"))
        subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "--offload-arch=gfx950", "-O0", "-std=c++17", "-w", *inc, "-c", str(src),
                        "-o", str(objs[-1])], check=True)
    exe = tmp_path / "ops_launch_kat"
    # (no device code is there to be registered)
    subprocess.run(["g++", *map(str, objs), "-Wl,--unresolved-symbols=ignore-all", "-no-pie", "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
