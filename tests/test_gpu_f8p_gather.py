"""bkv_gather of an e4m3 pool asks nothing of its outputs' alignment that the other layouts don't: rows at every multiple of 4 bytes."""
import numpy as np
import pytest

import f8p_model as M
from breccia_amd.kv import DeviceBuffer
from breccia_amd.lib import check, lib
from test_gpu_f8p import cells_at, fill, rng_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [0, 4, 8, 12])
def test_gather_into_any_float(offset):
    rng = rng_of(90)
    n, n_kv = 37, 3
    with M.F8Twin(n_pages=8, n_kv=n_kv) as tw:
        s = tw.pool.seq_create()
        fill(tw, s, n, rng)
        size = n * n_kv * 256
        bufs = [DeviceBuffer.from_numpy(np.full(size + 8, 7.0, np.float32)) for _ in range(2)]
        check(lib.bkv_gather(tw.pool.handle, 0, s, 0, n, bufs[0].at(offset), bufs[1].at(offset), None))
        for b, want in zip(bufs, cells_at(tw, 0, s, n)):
            got = b.download(np.float32, size + 8)
            at = offset // 4
            assert np.array_equal(got[at:at + size].reshape(want.shape), want)
            assert np.all(got[:at] == 7.0) and np.all(got[at + size:] == 7.0)
            b.free()
