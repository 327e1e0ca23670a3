"""The table changes that go along with a compaction (tests/cpp/compact_updates_test.cpp)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))


def test_changes_and_what_they_cost(tmp_path):
    out, src = str(tmp_path / "compact_updates_test"), os.path.join(HERE, "..", "breccia_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", os.path.join(HERE, "cpp", "compact_updates_test.cpp"), os.path.join(src, "allocator.cpp"),
                    "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.returncode, r.stdout, r.stderr[-2000:])
