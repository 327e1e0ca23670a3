"""Registers and memory instructions of the e4m3 kernels, as the compiler reports them.  No device is needed."""
import re

import pytest

from test_host_registers import compiled, scratch_of_kernels


@pytest.mark.parametrize("source, kernels", [("f8p_decode.hip", 8), ("f8p_move.hip", 33)])
def test_nothing_spills(source, kernels):
    scratch = {k: int(v) for k, v in scratch_of_kernels(source).items()}
    assert len(scratch) == kernels, sorted(scratch)
    assert not any(scratch.values()), scratch


def test_chunk_kernels_spill_nothing_that_a_page_fetches_back():
    # one tile of rows a wave: values of the prologue and the epilogue, under 80 bytes a lane; two tiles: none
    scratch = {k: int(v) for k, v in scratch_of_kernels("f8p_chunk.hip").items() if "chunk_attn_f8p_kernel" in k}
    assert len(scratch) == 4, sorted(scratch)
    for name, size in scratch.items():
        assert size <= (80 if re.search(r"kernelILi1E", name) else 0), scratch


@pytest.mark.parametrize("source", ["f8p_decode.hip", "f8p_move.hip", "f8p_chunk.hip"])
def test_addresses_are_known_to_be_global_or_lds(source):
    # a flat access waits for both counters
    assert not re.findall(r"^\s+flat_\w+", compiled(source)[1], re.M)
