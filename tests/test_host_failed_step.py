"""A decode step that fails enqueues nothing, on every layout, eager and of a plan: tests/cpp/failed_step_test.cpp, with HIP calls of its own
in the library's place.  Host code only."""
import os
import subprocess

from breccia_amd import build

HERE = os.path.dirname(os.path.abspath(__file__))


def test_a_step_that_fails_launches_nothing(tmp_path):
    out = str(tmp_path / "failed_step_test")
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(build._hipcc())))
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(HERE, "..", "include"),
                    "-I", os.path.join(rocm, "include"), "-rdynamic", os.path.join(HERE, "cpp", "failed_step_test.cpp"), "-o", out,
                    "-L" + build.HERE, "-lbreccia_kv", "-Wl,-rpath," + os.path.abspath(build.HERE), "-Wl,--allow-shlib-undefined"], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr[-2000:]
