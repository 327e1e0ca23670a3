"""Scales of int8 rows where the last bit of the quotient decides: the rule's scale is the binary16 of the f32 quotient amax / 127.  A product with
the reciprocal of 127 is off by a bit of f32 for one amax in twenty, and for the ones below that bit is what lies between two binary16
numbers.  Every byte that rows leave in the pool, appended, compacted and behind the rotary's K preparation."""
import numpy as np
import pytest

from breccia_amd import lib as L
from breccia_amd.kv import DeviceBuffer, Pool, device_sync, rope_table

pytestmark = pytest.mark.gpu


def largest_values():
    """All f32 of [1, 2) whose quotient and product round to different binary16 numbers."""
    m = np.arange(1 << 23, 1 << 24, dtype=np.uint32).astype(np.float32) * np.float32(2.0 ** -23)
    d = np.float32(127.0)
    q, r = m / d, m * (np.float32(1.0) / d)
    assert 0.02 < np.mean(q != r) < 0.08
    return m[(q * 16).astype(np.float16) != (r * 16).astype(np.float16)]


def test_the_values_are_the_ones_that_matter():
    # and of these quotients, in 64 bits beyond the middle of two binary16 numbers, the f32 quotient is on the right side
    m = largest_values()
    assert m.size >= 4
    q = m.astype(np.float64) / 127 * 16
    near = (m / np.float32(127.0) * 16).astype(np.float16).astype(np.float64)
    assert np.all(np.abs(near - q) <= np.spacing((q).astype(np.float16)).astype(np.float64) / 2)


def rows_of(rng, n, n_kv):
    """Rows whose blocks of 32 have one of those values as their largest, over all powers of two that a scale can have."""
    m = largest_values()
    top = m[rng.integers(0, m.size, (n, n_kv, 8))] * np.exp2(rng.integers(-6, 16, (n, n_kv, 8))).astype(np.float32)
    x = rng.uniform(-1, 1, (n, n_kv, 8, 32)).astype(np.float32) * top[..., None]
    at = rng.integers(0, 32, top.shape)
    np.put_along_axis(x, at[..., None], (top * np.where(rng.random(top.shape) < 0.5, -1, 1).astype(np.float32))[..., None], -1)
    return x.reshape(n, n_kv, 256)


def image(x):
    """[n, n_kv, 256] -> bytes of the rows [n, n_kv, 272], by the rule."""
    b = x.reshape(*x.shape[:2], 8, 32)
    scale = (np.abs(b).max(-1) / np.float32(127.0)).astype(np.float16)
    t = (b / scale.astype(np.float32)[..., None]).clip(-127, 127).astype(np.float64)
    codes = np.trunc(t + np.copysign(0.5, t)).astype(np.int8)
    return np.concatenate([codes.reshape(*x.shape[:2], 256).view(np.uint8), scale.view(np.uint8).reshape(*x.shape[:2], 16)], -1)


def held(p, seq, n, which):
    n_kv = p.desc.n_kv_head
    pages = p.read_layer(0, which).reshape(p.desc.n_pages, n_kv, 16, 272)[p.block_table(seq)]
    return pages.transpose(0, 2, 1, 3).reshape(-1, n_kv, 272)[:n]


@pytest.mark.parametrize("n, n_kv", [(1, 1), (2, 2), (333, 4), (3000, 2)])
def test_rows_appended_and_compacted(n, n_kv):
    rng = np.random.Generator(np.random.PCG64(n))
    k, v = rows_of(rng, n, n_kv), rows_of(rng, n, n_kv)
    with Pool(n_layers=1, n_pages=2 * (-(-n // 16)) + 2, n_kv_head=n_kv, head_dim=256, layout=L.LAYOUT_I8H, max_seqs=2) as p:
        s = p.seq_create()
        p.seq_reserve(s, n)
        bufs = [DeviceBuffer.from_numpy(x) for x in (k, v)]
        p.append(0, [s], [0], [n], *bufs)
        device_sync()
        for which, x in ((0, k), (1, v)):
            assert np.array_equal(held(p, s, n, which), image(x))
        ids = np.sort(rng.permutation(n)[:max(1, n // 2)]).astype(np.uint32)
        bufs.append(DeviceBuffer.from_numpy(ids))
        p.seq_compact([s], [0], [ids.size], bufs[2])
        device_sync()
        for which, x in ((0, k), (1, v)):
            assert np.array_equal(held(p, s, ids.size, which), image(x[ids]))
        for b in bufs:
            b.free()


@pytest.mark.parametrize("n", [3, 700])
def test_values_behind_the_rotary_of_axes(n):
    # V goes as it is; K's norm and rotary are others' tests
    rng = np.random.Generator(np.random.PCG64(n))
    k, v = rows_of(rng, n, 2), rows_of(rng, n, 2)
    table = rope_table(1e7, 64, n + 1)
    with Pool(n_layers=1, n_pages=-(-n // 16) + 1, n_kv_head=2, head_dim=256, layout=L.LAYOUT_I8H, max_seqs=1) as p:
        s = p.seq_create()
        p.seq_reserve(s, n)
        bufs = [DeviceBuffer.from_numpy(x) for x in (k, v, np.ones(256, np.float32), table, np.arange(2 * n, dtype=np.int32))]
        p.append_kprep_axes(0, [s], [0], [n], *bufs[:3], 1e-6, bufs[3], 64, n + 1, [0, 1] * 16, bufs[4], n)
        device_sync()
        assert np.array_equal(held(p, s, n, 1), image(v))
        for b in bufs:
            b.free()
