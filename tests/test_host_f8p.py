"""The e4m3 layout without a device: its numpy restatement against the published value set, the page's bytes, and the refusals."""
import ctypes as C

import numpy as np
import pytest

import f8p_model as M
from breccia_amd import kv, lib as L
from breccia_amd.kv import BkvError, Pool


def expect(status, fn, *a, **k):
    with pytest.raises(BkvError) as ei:
        fn(*a, **k)
    assert ei.value.status == status and ei.value.message, ei.value
    return ei.value.message


def test_codes_are_e4m3_rounded_to_nearest_even():
    torch = pytest.importorskip("torch")
    rng = np.random.Generator(np.random.PCG64(1))
    borders = np.sort(np.concatenate([M.VALUES[np.isfinite(M.VALUES)], ]))
    mids = (borders[1:] + borders[:-1]) / 2
    x = np.concatenate([borders, mids, np.nextafter(mids, 1e9), np.nextafter(mids, -1e9), rng.standard_normal(20000) * 2.0 ** rng.integers(-14, 9, 20000)])
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(M.encode(x, 0), want)
    assert np.array_equal(M.encode(x * np.float32(2.0 ** 7), 7), want)


def test_exponent_is_the_smallest_that_holds_the_largest_value():
    for top, e in [(448.0, 0), (np.nextafter(np.float32(448), np.float32(1e9)), 1), (224.0, -1), (1.75, -8), (1.76, -7), (0.0, -32), (1e-30, -32),
                   (448 * 2.0 ** 31, 31), (3e38, 31), (np.inf, -32)]:
        assert M.exponent([top, np.nan]) == e, top


def test_every_byte_of_a_unit_has_one_value():
    for at in (M.K_AT, M.V_AT):
        assert np.array_equal(np.sort(at.reshape(-1)), np.arange(M.UNIT))
        for b in range(4):   # a selection block is one run of 1 KiB
            assert at[4 * b:4 * b + 4].min() == 1024 * b and at[4 * b:4 * b + 4].max() == 1024 * b + 1023


def pool(**kw):
    kw.setdefault("n_pages", 64)
    return Pool(layout=L.LAYOUT_F8P, host_only=True, **kw)


def test_geometry():
    with pool(n_layers=3, n_kv_head=4) as p:
        assert p.page_bytes(0) == 4 * 4096 + 128 and p.page_bytes(1) == 4 * 4096
        assert p.swap_page_bytes() == 3 * (8 * 4096 + 128)
    for hd in (32, 128):
        expect(L.ERR_INVALID, pool, head_dim=hd)


def test_entries_of_one_append_must_not_meet_in_a_page():
    z = C.c_void_p(0x1000)
    with pool() as p:
        a, b = p.seq_create(), p.seq_create()
        p.seq_reserve(a, 200)
        p.seq_reserve(b, 200)
        for pos0, n in [([0, 15], [15, 1]), ([32, 5], [3, 40]), ([7, 7], [1, 1])]:
            assert "same page" in expect(L.ERR_INVALID, p.append, 0, [a, a], pos0, n, z, z)
            assert "same page" in expect(L.ERR_INVALID, p.append, 0, [a, a], pos0, n, z, z, f16_rows=True)
            assert "same page" in expect(L.ERR_INVALID, p.append_kprep, 0, [a, a], pos0, n, z, z, z, 1e-6, z, 64, 512)
        # neighbouring pages, another sequence, nothing to write: past the check, to the missing device
        for seqs, pos0, n in [([a, a], [0, 16], [16, 1]), ([a, b], [3, 3], [4, 4]), ([a, a], [5, 5], [0, 1])]:
            expect(L.ERR_NO_DEVICE, p.append, 0, seqs, pos0, n, z, z)


@pytest.mark.parametrize("layout", [L.LAYOUT_F16, L.LAYOUT_Q8V, L.LAYOUT_I8H, L.LAYOUT_F8P])
@pytest.mark.parametrize("f16", [False, True])
def test_read_rows_refusals(layout, f16):
    z = C.c_void_p(0x1000)
    with Pool(layout=layout, n_pages=16, max_seqs=4, host_only=True) as p:
        s = p.seq_create()
        p.seq_reserve(s, 40)                            # 48 cells addressable
        expect(L.ERR_RANGE, p.read_rows, 1, [s], [0], [1], z, z, f16_rows=f16)
        expect(L.ERR_RANGE, p.read_rows, 0, [s + 1], [0], [1], z, z, f16_rows=f16)
        for c0, n in [(-1, 2), (0, -1), (0, 49), (48, 1), (2 ** 62, 1), (2 ** 63 - 1, 2 ** 31 - 1)]:
            expect(L.ERR_RANGE, p.read_rows, 0, [s], [c0], [n], z, z, f16_rows=f16)
        expect(L.ERR_INVALID, p.read_rows, 0, [s] * 65, [0] * 65, [1] * 65, z, z, f16_rows=f16)
        expect(L.ERR_NO_DEVICE, p.read_rows, 0, [s, s], [0, 3], [48, 5], z, z, f16_rows=f16)
        fn = L.lib.bkv_read_rows_f16 if f16 else L.lib.bkv_read_rows
        expect(L.ERR_INVALID, lambda: kv.check(fn(None, 0, 0, None, None, None, z, z, None)))
        expect(L.ERR_INVALID, lambda: kv.check(fn(p.handle, 0, 1, None, None, None, z, z, None)))
        expect(L.ERR_INVALID, lambda: kv.check(fn(p.handle, 0, -1, None, None, None, z, z, None)))


def test_attention_of_such_a_pool_keeps_its_checks():
    z = C.c_void_p(0x1000)
    with pool(n_pages=8, max_seqs=4) as p:
        s = p.seq_create()
        p.seq_reserve(s, 40)
        expect(L.ERR_RANGE, p.decode_attn, 0, [s], [48], 16, z, z, 0.0625)
        expect(L.ERR_INVALID, p.decode_attn, 0, [s], [5], 34, z, z, 0.0625)      # 17 heads a kv head
        expect(L.ERR_RANGE, p.prefill_attn, 0, [s], [40], [9], 16, z, z, 0.0625)
        expect(L.ERR_INVALID, p.decode_step, 0, [s, s], [5, 6], z, z, 16, z, z, 0.0625)
        expect(L.ERR_RANGE, p.decode_step, 0, [s], [40], z, z, 16, z, z, 0.0625)
        expect(L.ERR_NO_DEVICE, p.prefill_attn, 0, [s], [0], [40], 16, z, z, 0.0625)


@pytest.mark.parametrize("f16", [False, True])
def test_reading_back_takes_the_short_way(f16):
    one = np.array([1], np.int32)
    z = 0x1000
    with Pool(layout=L.LAYOUT_F8P, n_pages=16, max_seqs=2, host_only=True) as p:
        s = np.array([p.seq_create()], np.int32)
        p.seq_reserve(int(s[0]), 17)
        for cell, status in ((0, L.ERR_NO_DEVICE), (-1, L.ERR_RANGE)):
            at = np.array([cell], np.int64)
            assert kv._hot.read_rows(p.handle, 0, s, at, one, z, z, None, f16) == status
            fast = expect(status, p.read_rows, 0, s, at, one, z, z, f16_rows=f16)
            assert fast == expect(status, p.read_rows, 0, s.tolist(), at.tolist(), [1], z, z, f16_rows=f16)
        assert kv._hot.read_rows(p.handle, 0, s, at, np.array([1, 1], np.int32), z, z, None, f16) is NotImplemented


def test_what_no_launch_takes_is_refused():
    # 256 threads for each page, kv head and side; 2^32 threads an axis
    z = C.c_void_p(0x1000)
    with Pool(layout=L.LAYOUT_F8P, n_pages=600_000, n_kv_head=16, max_seqs=2, max_pages_per_seq=600_000, host_only=True) as p:
        s = p.seq_create()
        most = 16 * ((1 << 32) // (16 * 512) - 2)
        p.seq_reserve(s, most + 4096)
        assert "more than a launch takes" in expect(L.ERR_INVALID, p.append, 0, [s], [5], [most], z, z)
        assert "more than a launch takes" in expect(L.ERR_INVALID, p.append_kprep, 0, [s], [5], [most], z, z, z, 1e-6, z, 64, 16)
        expect(L.ERR_NO_DEVICE, p.append, 0, [s], [5], [most - 1], z, z)
    with Pool(layout=L.LAYOUT_F16, n_pages=600_000, n_kv_head=16, max_seqs=2, max_pages_per_seq=600_000, host_only=True) as p:
        s = p.seq_create()
        p.seq_reserve(s, 16 * 600_000)
        most = 16 * ((1 << 32) // (16 * 1024) - 2)
        assert "more than a launch takes" in expect(L.ERR_INVALID, p.read_rows, 0, [s], [5], [most], z, z)
        expect(L.ERR_NO_DEVICE, p.read_rows, 0, [s], [5], [most - 1], z, z)
