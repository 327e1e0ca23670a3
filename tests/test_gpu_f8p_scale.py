"""Attention over e4m3 pages with a scale of the logits that is no number, or none that f32 holds in base 2: NaN everywhere, whatever the
signs of the logits, and never an average or zeros."""
import numpy as np
import pytest

import f8p_model as M
from breccia_amd.kv import DeviceBuffer
from test_gpu_f8p import rng_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("sign", [-1.0, 0.0, 1.0, None])
def test_a_scale_that_is_not_finite_gives_nan(scale, sign):
    rng = rng_of(80)
    n_q, n = 24, 2400
    with M.F8Twin(n_pages=160) as tw:
        pool = tw.pool
        s = pool.seq_create()
        pool.seq_reserve(s, n)
        x = np.abs(rng.standard_normal((n, 2, 256))).astype(np.float32)     # the logits' signs are q's
        tw.append(0, [s], [0], [x], [x])
        q = rng.standard_normal((1600, n_q, 256)).astype(np.float32)
        if sign is not None:
            q = np.abs(q) * np.float32(sign)
        qd, od = DeviceBuffer.from_numpy(q), DeviceBuffer.from_numpy(np.zeros_like(q))
        ids, counts = DeviceBuffer.from_numpy(np.arange(40, dtype=np.uint32)), DeviceBuffer.from_numpy(np.array([40], np.uint32))

        def all_nan(rows):
            got = od.download(np.float32, rows * n_q * 256)
            od.upload(np.zeros_like(got))
            return bool(np.isnan(got).all())

        pool.decode_attn(0, [s], [n - 1], n_q, qd, od, float(scale))
        assert all_nan(1)
        pool.decode_attn_select(0, [s], [n - 1], n_q, qd, od, float(scale), ids, 40, counts, 40)
        assert all_nan(1)
        for t in (41, 600, 1600):                           # cut, one tile of rows a wave, two
            pool.prefill_attn(0, [s], [n - t], [t], n_q, qd, od, float(scale))
            assert all_nan(t), t
        for b in (qd, od, ids, counts):
            b.free()
