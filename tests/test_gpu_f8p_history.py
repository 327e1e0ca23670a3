"""Rows that are taken back on pages of the e4m3 layout, on the device: the bound that the header gives for what stays (tested on its own
in test_host_f8p_history.py), and the way to keep them as they were."""
import numpy as np
import pytest

import f8p_model as M
from test_gpu_f8p import rng_of, rows_of

pytestmark = pytest.mark.gpu


def test_rows_below_a_rejected_one_stay_within_the_bound():
    rng = rng_of(63)
    with M.F8Twin(n_pages=8) as tw:
        s = tw.pool.seq_create()
        tw.pool.seq_reserve(s, 9)
        rows = [rows_of(rng, 9, 2), rows_of(rng, 9, 2)]
        tw.append(0, [s], [0], rows[:1], rows[1:])
        for spread in (1e2, 1e4, 3.0):                      # three drafts, none accepted
            big = rows_of(rng, 3, 2, spread)
            tw.pool.seq_reserve(s, 12)
            tw.append(0, [s], [9], [big], [big])
            tw.pool.seq_truncate(s, 9)
            page = tw.pool.block_table(s)[0]
            if spread == 1e4:
                most = tw.images[0].exps(page)[:2].copy()    # the largest exponents this page has had
        tw.pool.seq_reserve(s, 10)
        one = rows_of(rng, 1, 2)
        tw.append(0, [s], [9], [one], [one])
        tw.assert_pools_equal()
        assert np.all(tw.images[0].exps(page)[:2] < most)
        for side, got in enumerate(tw.pool.gather(0, s, 0, 9)):
            x = rows[side].astype(np.float64)
            error = np.abs(got - x)
            assert np.all(error <= 2.0 ** -4 * np.abs(x) + 2.0 ** (most[:, side] - 9.0)[None, :, None])
            assert np.max(error) > 2.0 ** -9 * 2.0 ** int(tw.images[0].exps(page)[:2].max())


def test_a_draft_in_a_fork_leaves_the_page_as_it_was():
    rng = rng_of(64)
    with M.F8Twin(n_pages=16) as tw:
        pool = tw.pool
        s = pool.seq_create()
        pool.seq_reserve(s, 40)
        rows = rows_of(rng, 25, 2)
        tw.append(0, [s], [0], [rows], [rows])
        pool.seq_truncate(s, 25)
        before = pool.gather(0, s, 0, 25)
        draft = pool.seq_fork(s, 25)
        for src, dst in pool.seq_reserve(draft, 30):
            pool.page_copy([(src, dst)])
            tw.images[0].page_copy([(src, dst)])
        big = rows_of(rng, 5, 2, 1e5)
        tw.append(0, [draft], [25], [big], [big])
        assert not np.array_equal(pool.gather(0, draft, 16, 9)[0], before[0][16:])
        pool.seq_free(draft)
        one = rows_of(rng, 1, 2, 0.1)
        assert not len(pool.seq_reserve(s, 26))
        tw.append(0, [s], [25], [one], [one])
        tw.assert_pools_equal()
        for got, was in zip(pool.gather(0, s, 0, 25), before):
            assert np.array_equal(got, was)                 # as large as they were, under the same scale
