"""The tcgen05 attention operator's loading warp, compiled for the CPU behind
stand-ins for the barrier and copy operations (loader_on_host.cpp): when a wait
runs out, the CTA leaves only after its copies have landed."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "laya_zig_b200", "csrc")


def test_no_copy_outlives_its_cta(tmp_path):
    exe = str(tmp_path / "loader")
    subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", "-Wno-unknown-pragmas", "-I", CSRC,
                    os.path.join(HERE, "loader_on_host.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
