"""Axes of pairs that no byte holds reach the library as an axis that no call has (it refuses those), not as the one that their low bits name."""
import ctypes as C

import numpy as np
import pytest

from breccia_amd import kv

ADDR = 0x1000  # never touched


def handed_over(monkeypatch, pair_axis):
    """The number of axes and the axis of each pair, as the library gets them."""
    got = []
    monkeypatch.setattr(kv.lib, "bkv_append_kprep_axes", lambda *a: got.append((a[13], list((C.c_uint8 * 4).from_address(C.addressof(a[14]))))) or 0)
    with kv.Pool(n_pages=8, max_seqs=1, host_only=True) as p:
        p.append_kprep_axes(0, [0], [0], [1], ADDR, ADDR, ADDR, 1e-6, ADDR, 8, 16, pair_axis, ADDR, 1)
    return got[0]


@pytest.mark.parametrize("kind", [list, tuple, lambda x: np.array(x, np.int64), lambda x: np.array(x + x, np.int32)[:4]])
def test_axes_of_pairs(monkeypatch, kind):
    assert handed_over(monkeypatch, kind([0, 3, 1, 2])) == (4, [0, 3, 1, 2])
    for bad in (255, 256, 257, 1 << 30, -1, -255):
        assert handed_over(monkeypatch, kind([0, 1, bad, 3])) == (256, [0, 1, 255, 3])
