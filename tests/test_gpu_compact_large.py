"""A compaction of more pages than all slots of the argument ring hold: it goes round, behind its own launches."""
import pytest

from breccia_amd import lib as L
from test_gpu_compact import make, run

pytestmark = pytest.mark.gpu


def test_more_pages_than_the_ring_holds():
    n = 34 * 16384 * 16 + 5
    p, seqs, rng = make(L.LAYOUT_F16, [n], n_layers=1, n_kv=1, hd=32, seed=31, spare=34 * 16384 + 9)
    with p:
        run(p, seqs, [n], [3], [n - 100], rng)
