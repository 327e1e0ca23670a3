"""Block tables of more than 2^31 entries, 11 GB of host memory (tests/cpp/table_offsets_test.cpp), and of more than any change can name."""
import os
import subprocess

import pytest

from breccia_amd import lib as L
from breccia_amd.kv import BkvError, Pool

HERE = os.path.dirname(os.path.abspath(__file__))


def free_gib():
    with open("/proc/meminfo") as f:
        return next(int(line.split()[1]) for line in f if line.startswith("MemAvailable:")) / 2 ** 20


def test_changes_behind_the_middle_of_a_large_arena(tmp_path):
    if free_gib() < 20:
        pytest.skip("takes 11 GB of memory")
    out, src = str(tmp_path / "table_offsets_test"), os.path.join(HERE, "..", "breccia_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", os.path.join(HERE, "cpp", "table_offsets_test.cpp"), os.path.join(src, "allocator.cpp"),
                    "-o", out], check=True)
    r = subprocess.run([out], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.returncode, r.stdout, r.stderr[-2000:])


def test_larger_arenas_are_refused():
    with pytest.raises(BkvError) as e:
        Pool(n_pages=16, max_seqs=1 << 12, max_pages_per_seq=1 << 20, host_only=True)
    assert e.value.status == L.ERR_INVALID and "block tables" in e.value.message
