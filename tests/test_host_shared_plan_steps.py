"""What planning a batch whose entries share pages costs the host, in walks looked at (tests/cpp/shared_plan_steps_test.cpp)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_no_walk_is_cut_over_and_over(tmp_path):
    out = str(tmp_path / "shared_plan_steps_test")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover",
                    os.path.join(HERE, "cpp", "shared_plan_steps_test.cpp"), "-o", out], check=True)
    r = subprocess.run([out, "5", "30000"], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr[-2000:]
