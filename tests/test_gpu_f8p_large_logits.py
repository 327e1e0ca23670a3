"""Attention over e4m3 pages with logits so large that a step of f32 at their size is up to 256: the largest wins alone, whatever such a step
does to the reference that weights are taken against.  K is a row of signs times 1, 1.125, 1.25, 1.5 or 1.75 (exact as codes) and q a
multiple of the signs, so two different logits are 1/16 of the largest apart or more, and what a row gets is the V of the cell that is
alone with its largest: off by the two f16 numbers of a weight and the sums, 2^-22 each."""
import numpy as np
import pytest

import f8p_model as M
from breccia_amd.kv import DeviceBuffer, Graph, Stream
from test_gpu_f8p import cells_at, chunk, rng_of, rows_of
from test_gpu_f8p_long import attend

pytestmark = pytest.mark.gpu


RECORDS = {1.0: (1.0, [(100, 1.125), (370, 1.25), (1100, 1.5), (1680, 1.75)]), -1.0: (1.75, [(100, 1.5), (370, 1.25), (1100, 1.125), (1680, 1.0)])}


def check(got, v, pos, n_q, what):
    cell = max(c for c in (100, 370, 1100, 1680) if c <= pos)       # the last record
    want = v[cell].astype(np.float64).repeat(n_q // 2, axis=0)
    assert np.max(np.abs(got - want) / np.max(np.abs(want))) <= 2.0 ** -21, what


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("power", range(20, 32))
def test_the_largest_logit_wins(power, sign):
    n, n_q = 1700, 16
    rng = rng_of(100, power)
    with M.F8Twin(n_pages=120) as tw:
        s = tw.pool.seq_create()
        # logits of one sign, from 2^power in base 2 up to 2.1 times that, with ever larger ones along the sequence
        u = rng.choice([-1.0, 1.0], 256).astype(np.float32)
        others, records = RECORDS[sign]
        size = np.full(n, others, np.float32)
        for cell, x in records:
            size[cell] = x
        k = np.ascontiguousarray(np.broadcast_to((size[:, None] * u)[:, None], (n, 2, 256)), dtype=np.float32)
        v = rows_of(rng, n, 2)
        tw.pool.seq_reserve(s, n)
        tw.append(0, [s], [0], [k], [v])
        hk, hv = cells_at(tw, 0, s, n)
        assert np.array_equal(hk, k)
        t = 1600
        q = sign * 2.0 ** power * np.log(2.0) / 16 * np.linspace(1, 1.2, t * n_q).reshape(t, n_q, 1) * u
        q = np.ascontiguousarray(q, dtype=np.float32)
        got = attend(tw.pool, 0, [s], [n - 1], q[:1], n_q)
        check(got[0], hv, n - 1, n_q, "decode")
        whole = chunk(tw, 0, [s], [n - t], [q], n_q)[0]         # two tiles of rows a wave
        for i in (0, 700, t - 1):
            check(whole[i], hv, n - t + i, n_q, "two tiles")
        cut = chunk(tw, 0, [s], [n - 41], [q[:41]], n_q)[0]
        st = Stream()
        qd, od = DeviceBuffer.from_numpy(q[:41]), DeviceBuffer(q[:41].nbytes)
        graph = Graph(st)
        tw.pool.prefill_attn(0, [s], [n - 41], [41], n_q, qd, od, 1 / 16.0, stream=st)
        graph.end()
        graph.launch()
        one = od.download(np.float32, stream=st).reshape(41, n_q, 256)
        graph.destroy()
        for i in (0, 40):
            check(cut[i], hv, n - 41 + i, n_q, "cut")
            check(one[i], hv, n - 41 + i, n_q, "one tile")
