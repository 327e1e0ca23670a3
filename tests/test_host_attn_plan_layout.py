"""The cut of decode batches into work-groups for each layout's kernels: what holds of every cut (test_host_abi.py) at the number of pages
that a layout's waves walk side by side.  No device is needed."""
import numpy as np
import pytest

from breccia_amd import kv, lib as L
from breccia_amd.kv import BkvError

LAYOUTS = {L.LAYOUT_F16: 4, L.LAYOUT_Q8V: 4, L.LAYOUT_I8H: 4, L.LAYOUT_F8P: 8}


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n_cu", [256, 64, 8])
def test_every_cut_covers_its_pages_and_fits(layout, n_cu):
    rng = np.random.Generator(np.random.PCG64(78))
    for n_kv in range(1, L.MAX_KV_HEAD + 1):
        for group in (1, 5, 8, 12, 16):
            cap = 4096 * 8 // group if group > 8 else 4096
            for n in (1, 2, 7, 33, 64):
                for sel_groups in (0, 1, 5, 129):
                    pos = rng.integers(0, 40000, size=n)
                    if n >= 33:
                        pos[: n // 2] = rng.integers(0, 64, size=n // 2)
                    splits, pps, total = kv.attn_plan(n_cu, n_kv, n_kv * group, pos, sel_groups, layout=layout)
                    pages = np.full(n, sel_groups) if sel_groups else pos // 16 + 1
                    assert total == int(splits.sum()) * n_kv <= cap
                    assert np.all(pps % LAYOUTS[layout] == 0) and np.all(splits >= 1)
                    assert np.all(splits * pps >= pages) and np.all((splits - 1) * pps < pages)     # none empty
                    assert total <= max(2 * n_cu, n * n_kv)
                    if layout != L.LAYOUT_F8P:
                        same = kv.attn_plan(n_cu, n_kv, n_kv * group, pos, sel_groups)
                        assert np.array_equal(splits, same[0]) and np.array_equal(pps, same[1]) and total == same[2]


def test_refusals():
    for bad in (-1, 4):
        with pytest.raises(BkvError) as e:
            kv.attn_plan(256, 2, 16, [5], layout=bad)
        assert e.value.status == L.ERR_INVALID
    with pytest.raises(BkvError) as e:
        kv.attn_plan(256, L.MAX_KV_HEAD + 1, 17, [5], layout=L.LAYOUT_F8P)
    assert e.value.status == L.ERR_INVALID
