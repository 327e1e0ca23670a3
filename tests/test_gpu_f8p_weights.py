"""Attention over e4m3 pages where most of what a row gets comes with small weights: one key far above all others that brings nothing (an
attention sink: V of zeros), or one loud value of V in a page.  Errors are measured against the output itself, element by element.

What they may be.  A weight w enters the products as two f16 numbers, hi to nearest and the rest to nearest: off by 2^-22 w at most, or
by 2^-25 where f16 has run out of exponents, in units of 2^(reference), and the largest term lies 2^9 above the reference or
higher.  So a row whose terms all lie `gap` bits below the largest is off by 2^-22 + 2^(gap - 34) of itself.  To that come the logit (at most
`gap` + 1 in base 2, 2^-21 relative: 22-bit q, and the products' sums) and f32 sums over the walk, a product for each 32 cells and
as many additions again in the fold and the merge as there are ranges (64 at most), 2^-24 each."""
import numpy as np
import pytest

import f8p_model as M
from breccia_amd import lib as L
from breccia_amd.kv import DeviceBuffer, Graph, Stream
from test_gpu_f8p import cells_at, chunk, lists, rng_of, rows_of
from test_gpu_f8p_long import attend

pytestmark = pytest.mark.gpu

GAPS = np.array([12.3, 17.4, 19.7, 21.6, 23.4, 24.7, 25.6, 26.8])     # bits that the heads' largest term is above the others


def bar(gap, n):
    return 2.0 ** -22 + 2.0 ** (gap - 34) + (gap + 1) * 2.0 ** -21 + (n / 32 + 64) * 2.0 ** -24


def rows_with_a_sink(rng, n, n_kv, at):
    """K, V and a direction u: cell `at` has K = u and V = 0, all others K = 0 and V of one sign."""
    u = rng.choice([-1.0, 1.0], 256).astype(np.float32)
    k = np.zeros((n, n_kv, 256), np.float32)
    k[at] = u
    v = 1 + np.abs(rows_of(rng, n, n_kv))
    v[at] = 0
    return k, v, u


def queries(u, n_rows, n_q, n_kv):
    """Heads of one kv head take the gaps in turn: q . u / 16 = gap * ln 2."""
    gaps = GAPS[np.arange(n_q) % (n_q // n_kv) % GAPS.size]
    q = np.broadcast_to((gaps * np.log(2.0) / 16.0)[:, None] * u, (n_rows, n_q, 256))
    return np.ascontiguousarray(q, dtype=np.float32), gaps


def held_rows(tw, seq, n, k, v):
    tw.pool.seq_reserve(seq, n)
    tw.append(0, [seq], [0], [k], [v])
    return cells_at(tw, 0, seq, n)


def check(got, want, gaps, n, what):
    error = np.max(np.abs(got.astype(np.float64) - want) / np.abs(want), axis=-1)
    assert np.all(error <= bar(gaps, n)), (what, np.round(np.log2(np.maximum(error, 1e-30)), 1), np.round(np.log2(bar(gaps, n)), 1))


def test_decode_behind_a_sink():
    # 64 entries at 8 kv heads: a work-group each, whose waves walk a quarter of the cells
    n, n_kv, n_q, b = 4210, 8, 64, 64
    rng = rng_of(50)
    with M.F8Twin(n_pages=400, n_kv=n_kv, max_seqs=b) as tw:
        a = tw.pool.seq_create()
        k, v, u = rows_with_a_sink(rng, n, n_kv, 0)
        hk, hv = held_rows(tw, a, n, k, v)
        seqs = [a] + [tw.pool.seq_fork(a, n) for _ in range(b - 1)]
        q, gaps = queries(u, b, n_q, n_kv)
        pos = [n - 1 - 5 * i for i in range(b)]
        got = attend(tw.pool, 0, seqs, pos, q, n_q)
        for i in (0, 1, 63):
            check(got[i], M.attend64(q[i:i + 1], hk, hv, [range(pos[i] + 1)], 1 / 16.0)[0], gaps, n, i)
        ids = np.stack([np.concatenate([[0], 1 + rng.permutation(n // 4)[:512]]) for _ in range(b)])
        got = lists(tw, seqs, pos, q, n_q, ids, [513] * b, 513)
        for i in (0, 1, 63):
            cells = (4 * ids[i, :, None] + np.arange(4)).reshape(-1)
            check(got[i], M.attend64(q[i:i + 1], hk, hv, [cells[cells <= pos[i]]], 1 / 16.0)[0], gaps, n, i)


@pytest.mark.parametrize("before, t, n_q, captured, cut", [(8000, 41, 16, False, 1), (8000, 41, 16, True, 0), (6600, 1500, 24, False, 0)])
@pytest.mark.parametrize("at", [0, 3000])
def test_chunks_behind_a_sink(before, t, n_q, captured, cut, at):
    # walks cut into ranges, whole ones (a captured call's) of one tile of rows a wave, and of two
    n = before + t
    rng = rng_of(51, before, captured, at)
    with M.F8Twin(n_pages=512) as tw:
        s = tw.pool.seq_create()
        k, v, u = rows_with_a_sink(rng, n, 2, at)
        hk, hv = held_rows(tw, s, n, k, v)
        q, gaps = queries(u, t, n_q, 2)
        if captured:
            st = Stream()
            qd, od = DeviceBuffer.from_numpy(q), DeviceBuffer(q.nbytes)
            tw.pool.prefill_attn(0, [s], [before], [t], n_q, qd, od, 1 / 16.0, stream=st)
            st.sync()
            graph = Graph(st)
            tw.pool.prefill_attn(0, [s], [before], [t], n_q, qd, od, 1 / 16.0, stream=st)
            graph.end()
            graph.launch()
            got = od.download(np.float32, stream=st).reshape(q.shape)
            graph.destroy()
        else:
            tw.pool.timing_enable(True)
            got = chunk(tw, 0, [s], [before], [q], n_q)[0]
            tw.pool.timing_enable(False)
            assert tw.pool.timing_read(L.STAGE_ATTN_MERGE)[0] == cut
        for i in (0, t // 2, t - 1):
            check(got[i], M.attend64(q[i:i + 1], hk, hv, [range(before + i + 1)], 1 / 16.0)[0], gaps, n, i)


@pytest.mark.parametrize("t", [1, 1500])
def test_a_loud_value_leaves_the_other_elements_alone(t):
    # one value of 2^20 in a page of V that holds nothing else: the page's scale is 18 bits above the others', and so is its weight
    n_q, n = 24, 3000
    rng = rng_of(52, t)
    with M.F8Twin(n_pages=200) as tw:
        s = tw.pool.seq_create()
        u = rng.choice([-1.0, 1.0], 256).astype(np.float32)
        k = np.broadcast_to(u, (n, 2, 256)).copy()
        v = 1 + np.abs(rows_of(rng, n, 2))
        k[:16], v[:16] = 0, 0
        v[3, :, 7] = 2.0 ** 20
        hk, hv = held_rows(tw, s, n, k, v)
        assert tw.images[0].exps(tw.pool.block_table(s)[0])[0, 1] - tw.images[0].exps(tw.pool.block_table(s)[1])[0, 1] == 18
        logits = -np.linspace(0.15, 4.45, n_q)          # of the other pages, in base 2
        q = np.ascontiguousarray(np.broadcast_to((logits * np.log(2.0) / 16.0)[:, None] * u, (t, n_q, 256)), dtype=np.float32)
        if t == 1:
            got = attend(tw.pool, 0, [s], [n - 1], q, n_q)
        else:
            got = chunk(tw, 0, [s], [n - t], [q], n_q)[0]
        for i in {0, t - 1}:
            want = M.attend64(q[i:i + 1], hk, hv, [range(n - t + i + 1)], 1 / 16.0)[0]
            check(got[i], want, 18 - logits, n, i)
