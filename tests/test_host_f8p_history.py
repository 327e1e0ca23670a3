"""What a page of the e4m3 layout holds after a history of writes and rollbacks, against the bound that include/breccia_kv.h gives for it:
a finite value x of at most 448 * 2^31 is held to 2^-4 |x| + 2^-9 * 2^E, E the largest exponent that its page, head and side have had since
it was written.  (Coded, it is off by 2^-4 |x| or 2^-10 * 2^e at most.  Coded again under a scale that is larger than all before, it is off
by another 2^-10 * 2^e; under any other it is the same number.  These add up to less than 2^-9 * 2^E.)  No device is needed."""
import numpy as np
import pytest

import f8p_model as M
from test_gpu_f8p import rng_of, rows_of

PAGE = M.PAGE


class History:
    """A sequence in an image of one kv head, what its cells were given, and the largest exponents since."""

    def __init__(self, n_pages=4):
        self.img = M.F8Image(1, n_pages)
        self.table = np.arange(n_pages, dtype=np.int32)
        self.given = np.zeros((2, 0, 256))
        self.seen = np.zeros((2, 0), dtype=np.int64)       # E of every cell
        self.capacity = n_pages * PAGE

    def write(self, pos0, k, v):
        n = k.shape[0]
        self.given = np.concatenate([self.given[:, :pos0], np.stack([k, v])[:, :, 0]], axis=1)
        self.seen = np.concatenate([self.seen[:, :pos0], np.full((2, n), M.E_LO)], axis=1)
        assert self.img.append(self.table, pos0, k, v) == 0
        for lp in range(pos0 // PAGE, (pos0 + n - 1) // PAGE + 1):
            cells = slice(lp * PAGE, min((lp + 1) * PAGE, pos0 + n))
            for side in (0, 1):
                self.seen[side, cells] = np.maximum(self.seen[side, cells], self.img.exps(lp)[0, side])

    def held(self):
        return np.stack(self.img.gather(self.table, 0, self.given.shape[1]))[:, :, 0].astype(np.float64)

    def check(self):
        error = np.abs(self.held() - self.given)
        bound = 2.0 ** -4 * np.abs(self.given) + 2.0 ** (self.seen - 9.0)[:, :, None]
        assert np.all(error <= bound), float(np.max(error / bound))


@pytest.mark.parametrize("seed", range(12))
def test_held_values_stay_within_the_bound(seed):
    rng = rng_of(60, seed)
    h = History()
    for _ in range(40):
        at = h.given.shape[1]
        if at and rng.random() < 0.4:
            at = int(rng.integers(max(0, at - 20), at + 1))      # rolled back
        if at >= h.capacity - 1:
            at = int(rng.integers(0, 8))
        n = int(rng.integers(1, min(12, h.capacity - at) + 1))
        spread = 2.0 ** rng.uniform(-8, 12)
        h.write(at, rows_of(rng, n, 1, spread), rows_of(rng, n, 1, 1 / spread))
        h.check()


def test_kept_rows_depend_on_the_writes_before():
    # rows 100 times as large come and go: the exponent is back where it was, the rows below have lost what lay under the large steps
    rng = rng_of(61)
    rows, big, again = rows_of(rng, 9, 1), rows_of(rng, 3, 1, 100.0), rows_of(rng, 1, 1)
    straight, rolled = History(), History()
    straight.write(0, rows, rows)
    rolled.write(0, rows, rows)
    rolled.write(9, big, big)
    for h in (straight, rolled):
        h.write(9, again, again)
        h.check()
    assert np.array_equal(straight.img.exps(0), rolled.img.exps(0))
    a, b = straight.held()[:, :9], rolled.held()[:, :9]
    assert not np.array_equal(a, b)
    lost = np.abs(b - rows[None, :, 0].astype(np.float64))
    assert np.max(lost) > 2.0 ** -9 * 2.0 ** int(straight.img.exps(0).max())      # more than the page's exponent now accounts for
    # nor is a page of two writes that of one
    whole = History()
    whole.write(0, np.concatenate([rows, big]), np.concatenate([rows, big]))
    rolled = History()
    rolled.write(0, rows, rows)
    rolled.write(9, big, big)
    whole.check(), rolled.check()
    assert np.array_equal(whole.img.exps(0), rolled.img.exps(0)) and not np.array_equal(whole.held(), rolled.held())


def test_cells_that_were_never_written_count_below_the_first_written_one():
    rng = rng_of(62)
    h = History()
    old = rows_of(rng, 16, 1, 1e5)
    h.write(0, old, old)                                    # whoever had the page before
    x = rows_of(rng, 4, 1)
    h.img.append(h.table, 3, x, x)
    assert h.img.exps(0)[0, 0] == M.exponent(h.img.gather(h.table, 0, 3)[0]) > M.exponent(x)
    h.img.append(h.table, 0, x, x)                          # begun at the page's first cell, nothing of it counts
    assert h.img.exps(0)[0, 0] == M.exponent(x)
