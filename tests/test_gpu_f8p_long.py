"""The e4m3 layout where sizes change what runs: walks that go past the caches, ranges of more pages than a wave keeps the ids of, lists
of more blocks than that, pools whose bytes lie past 2^32, prefixes that went through host memory and disk, calls on two streams."""
import numpy as np
import pytest

import f8p_model as M
import oracle
from breccia_amd import lib as L
from breccia_amd.kv import DeviceBuffer, Graph, Pool, StepPlan, Stream, device_sync, rope_table
from gpu_common import REF_BAR_MAX_REL, check_attn
from test_gpu_f8p import cells_at, chunk, fill, lists, rng_of, rows_of

pytestmark = pytest.mark.gpu


def attend(pool, layer, seqs, pos, q, n_q, call="decode_attn", stream=None):
    qd, od = DeviceBuffer.from_numpy(q), DeviceBuffer(q.nbytes)
    getattr(pool, call)(layer, seqs, pos, n_q, qd, od, 1 / 16.0, stream=stream)
    if stream is not None:
        stream.sync()
    out = od.download(np.float32).reshape(q.shape)
    qd.free(), od.free()
    return out


@pytest.mark.parametrize("n_seqs", [3, 20])     # few entries' arguments and many's
def test_loads_past_the_caches_change_nothing(n_seqs):
    # what decides is the bytes of all layers: the same cells in a pool of 1 layer (6 MiB of them) and of 64
    ctx = [int(n) for n in rng_of(30, n_seqs).integers(1, 2 * 6000 // n_seqs, n_seqs)]
    q = rng_of(31).standard_normal((n_seqs, 16, 256)).astype(np.float32)
    got = []
    for n_layers in (1, 64):
        with M.F8Twin(n_layers=n_layers, n_pages=sum(n // 16 + 1 for n in ctx), max_seqs=n_seqs) as tw:
            seqs = [tw.pool.seq_create() for _ in ctx]
            for s, n in zip(seqs, ctx):
                fill(tw, s, n, rng_of(32, s), layer=n_layers - 1, step=4096)
            got.append([attend(tw.pool, n_layers - 1, seqs, [n - 1 for n in ctx], q, 16, c) for c in ("decode_attn", "decode_attn_static")])
            k, v = cells_at(tw, n_layers - 1, seqs[0], ctx[0])
            want = M.attend64(q[:1], k, v, [range(ctx[0])], 1 / 16.0)[0]
            assert check_attn(got[-1][0][0], want)[1] <= REF_BAR_MAX_REL
        assert (sum(ctx) * 2 * 512 * n_layers >= 96 << 20) == (n_layers == 64)
    assert np.array_equal(got[0], got[1])


def test_ranges_longer_than_the_ids_a_wave_keeps():
    # 64 entries at 8 kv heads leave one work-group each: 264 pages of one, 66 a wave; 129 groups of listed blocks, 33 a wave
    n, n_kv, n_q, b = 4210, 8, 8, 64
    rng = rng_of(33)
    with M.F8Twin(n_pages=400, n_kv=n_kv, max_seqs=b) as tw:
        pool = tw.pool
        pool.fill(0xFF)
        for img in tw.images:
            img.kp[:], img.vp[:] = 0xFF, 0xFF
        pool.set_free_order(rng.permutation(400).astype(np.int32))
        a = pool.seq_create()
        fill(tw, a, n, rng)
        seqs = [a] + [pool.seq_fork(a, n) for _ in range(b - 1)]
        pos = [n - 1 - 3 * i for i in range(b)]
        q = rng.standard_normal((b, n_q, 256)).astype(np.float32)
        got = attend(pool, 0, seqs, pos, q, n_q)
        k, v = cells_at(tw, 0, a, n)
        for i in (0, 1, 31, 63):
            assert check_attn(got[i], M.attend64(q[i:i + 1], k, v, [range(pos[i] + 1)], 1 / 16.0)[0], str(i))[1] <= REF_BAR_MAX_REL
        ids = np.stack([rng.permutation(n // 4 + 1)[:513] for _ in range(b)])
        counts = [513 - 8 * i for i in range(b)]
        got = lists(tw, seqs, pos, q, n_q, ids, counts, 513)
        for i in (0, 1, 31, 63):
            cells = (4 * ids[i, :counts[i], None] + np.arange(4)).reshape(-1)
            cells = cells[cells <= pos[i]]
            assert check_attn(got[i], M.attend64(q[i:i + 1], k, v, [cells], 1 / 16.0)[0], str(i))[1] <= REF_BAR_MAX_REL


def test_a_list_is_not_read_past_its_length():
    # the last list's entries end with the buffer: eight lists of 7 in rows of 40, the last row cut off behind its seventh
    rng = rng_of(34)
    n_q = 16
    with M.F8Twin(n_pages=64, max_seqs=8) as tw:
        s = tw.pool.seq_create()
        fill(tw, s, 700, rng)
        q = rng.standard_normal((8, n_q, 256)).astype(np.float32)
        ids = rng.integers(0, 175, (8, 40)).astype(np.uint32)
        counts = np.full(8, 7, np.uint32)
        whole = lists(tw, [s] * 8, [699] * 8, q, n_q, ids, counts, 40)
        bufs = [DeviceBuffer.from_numpy(x) for x in (q, np.zeros_like(q), ids.reshape(-1)[:7 * 40 + 7].copy(), counts)]
        tw.pool.decode_attn_select(0, [s] * 8, [699] * 8, n_q, bufs[0], bufs[1], 1 / 16.0, bufs[2], 40, bufs[3], 40)
        assert np.array_equal(bufs[1].download(np.float32).reshape(q.shape), whole)
        for b in bufs:
            b.free()


def everything(pool, high):
    """Writes, reads and attends a sequence of the pool every way there is -> what came out, page order no part of it."""
    n_kv, n_q = 16, 32
    rng = rng_of(35)
    pool.set_free_order(np.arange(pool.desc.n_pages, dtype=np.int32)[::-1].copy() if high else rng_of(36).permutation(pool.desc.n_pages).astype(np.int32))
    out = []
    s = pool.seq_create()
    pool.seq_reserve(s, 360)
    if high:
        assert int(pool.block_table(s).min()) * n_kv * 4096 > 1 << 32
    host = [rows_of(rng, 200, n_kv), rows_of(rng, 200, n_kv), rows_of(rng, 150, n_kv), rows_of(rng, 150, n_kv),
            np.ones(256, np.float32), rope_table(1e6, 64, 512), rng.standard_normal((100, n_q, 256)).astype(np.float32),
            np.arange(0, 80, 3, dtype=np.uint32), np.array([27], np.uint32)]
    k, v, k2, v2, gamma, table, q, ids, counts = bufs = [DeviceBuffer.from_numpy(x) for x in host]
    o = DeviceBuffer(max(host[6].nbytes, 350 * n_kv * 1024))
    o2 = DeviceBuffer(350 * n_kv * 1024)
    pool.append(0, [s], [0], [200], k, v)
    pool.append_kprep(0, [s], [200], [150], k2, v2, gamma, 1e-6, table, 64, 512)
    pool.decode_step(0, [s], [350], k, v, n_q, q, o, 1 / 16.0)
    out.append(o.download(np.float32, n_q * 256))
    pool.decode_attn_select(0, [s], [350], n_q, q, o, 1 / 16.0, ids, 27, counts, 27)
    out.append(o.download(np.float32, n_q * 256))
    pool.prefill_attn(0, [s], [250], [100], n_q, q, o, 1 / 16.0)
    out.append(o.download(np.float32, 100 * n_q * 256))
    pool.read_rows(0, [s], [1], [350], o, o2)
    out += [x.download(np.float32, 350 * n_kv * 256) for x in (o, o2)]
    b = pool.seq_fork(s, 340)
    for pair in pool.seq_reserve(b, 342):
        pool.page_copy([pair])
    pool.decode_step(0, [b], [340], k, v, n_q, q, o, 1 / 16.0)
    out.append(o.download(np.float32, n_q * 256))
    for x in bufs + [o, o2]:
        x.free()
    return out


def test_pages_past_four_gigabytes():
    kw = dict(n_layers=1, n_kv_head=16, head_dim=256, layout=L.LAYOUT_F8P, max_seqs=4, max_pages_per_seq=64)
    with Pool(n_pages=64, **kw) as small:
        want = everything(small, False)
    with Pool(n_pages=66200, **kw) as large:
        got = everything(large, True)
    assert all(np.isfinite(w).all() for w in want)
    for i, (g, w) in enumerate(zip(got, want)):
        assert np.array_equal(g, w), i


def test_a_prefix_through_host_memory_and_disk(tmp_path):
    rng = rng_of(37)
    prompt = rng.integers(0, 32000, 16 * 12 + 5).astype(np.int32)
    with M.F8Twin(n_layers=2, n_pages=40, max_seqs=4, max_pages_per_seq=20) as tw:
        pool = tw.pool
        slab = pool.swap_page_bytes()
        pool.prefix_tiers(5 * slab, str(tmp_path / "tier.bin"), 10 * slab)
        a = pool.seq_create()
        for layer in range(2):
            fill(tw, a, prompt.size, rng, layer, 2.0 ** (5 * layer))
        rows = [cells_at(tw, layer, a, 192) for layer in range(2)]
        q = rng.standard_normal((1, 16, 256)).astype(np.float32)
        want = [attend(pool, layer, [a], [191], q, 16) for layer in range(2)]
        assert pool.prefix_insert(a, prompt) == 12
        pool.seq_free(a)
        assert pool.prefix_evict(40) == 12
        held = pool.seq_create()
        pool.seq_reserve(held, 16 * 16)                 # other rows in the pages that were given back
        for layer in range(2):
            x = rows_of(rng, 256, 2, 100.0)
            tw.append(layer, [held], [0], [x], [x])
        s, m = pool.seq_create_from_prefix(prompt)
        assert m == 192
        for layer in range(2):
            got = pool.gather(layer, s, 0, m)
            assert np.array_equal(got[0], rows[layer][0]) and np.array_equal(got[1], rows[layer][1])
            assert np.array_equal(attend(pool, layer, [s], [191], q, 16), want[layer])
        # the request's own rows behind the adopted ones
        pool.seq_reserve(s, 200)
        x = rows_of(rng, 5, 2)
        tw.append(0, [s], [192], [x], [x])
        assert np.array_equal(pool.gather(0, s, 0, m)[0], rows[0][0])


def test_two_pools_on_two_streams():
    rng = rng_of(38)
    n_q = 16
    with M.F8Twin(n_pages=200) as a, M.F8Twin(n_pages=200) as b:
        seqs, qs, want = [], [], []
        for tw in (a, b):
            s = tw.pool.seq_create()
            fill(tw, s, 1500, rng)
            seqs.append(s)
            qs.append(rng.standard_normal((300, n_q, 256)).astype(np.float32))
            want.append((chunk(tw, 0, [s], [1200], [qs[-1]], n_q)[0], attend(tw.pool, 0, [s], [1499], qs[-1][:1], n_q)))
        device_sync()
        streams = [Stream(), Stream()]
        bufs = [[DeviceBuffer.from_numpy(q), DeviceBuffer(q.nbytes), DeviceBuffer(n_q * 1024), DeviceBuffer(1500 * 2 * 512), DeviceBuffer(1500 * 2 * 512)]
                for q in qs]
        for _ in range(5):
            for tw, s, st, (qd, oc, od, ko, vo) in zip((a, b), seqs, streams, bufs):
                tw.pool.prefill_attn(0, [s], [1200], [300], n_q, qd, oc, 1 / 16.0, stream=st)
                tw.pool.decode_attn(0, [s], [1499], n_q, qd, od, 1 / 16.0, stream=st)
                tw.pool.read_rows(0, [s], [0], [1500], ko, vo, stream=st, f16_rows=True)
        for tw, s, st, (qd, oc, od, ko, vo), w in zip((a, b), seqs, streams, bufs, want):
            st.sync()
            assert np.array_equal(oc.download(np.float32).reshape(w[0].shape), w[0])
            assert np.array_equal(od.download(np.float32).reshape(w[1].shape), w[1])
            for got, rows in zip((ko, vo), cells_at(tw, 0, s, 1500)):
                assert np.array_equal(got.download(np.uint16).view(np.float16).reshape(rows.shape), rows.astype(np.float16))


def test_captured_writes_reads_and_attention_replay():
    # the same cells written again by every replay from buffers that change, eager calls of another sequence in between
    rng = rng_of(39)
    n_q, n = 16, 45
    gamma, table = np.ones(256, np.float32), rope_table(1e6, 64, 128)
    with M.F8Twin(n_pages=32) as tw:
        pool, st = tw.pool, Stream()
        a, other = pool.seq_create(), pool.seq_create()
        for s in (a, other):
            pool.seq_reserve(s, 100)
            fill(tw, s, 60, rng)
        kd, vd, hk, hv, qd = (DeviceBuffer(x) for x in (n * 2 * 1024, n * 2 * 1024, 7 * 2 * 512, 7 * 2 * 512, n_q * 1024))
        gd, td = DeviceBuffer.from_numpy(gamma), DeviceBuffer.from_numpy(table)
        od, ko, vo = DeviceBuffer(n_q * 1024), DeviceBuffer(100 * 2 * 1024), DeviceBuffer(100 * 2 * 1024)

        def calls(stream):
            pool.append(0, [a], [41], [7], hk, hv, stream=stream, f16_rows=True)
            pool.append_kprep(0, [a], [48], [n], kd, vd, gd, 1e-6, td, 64, 128, stream=stream)
            pool.decode_attn_static(0, [a], [92], n_q, qd, od, 1 / 16.0, stream=stream)
            pool.read_rows(0, [a], [0], [93], ko, vo, stream=stream)

        st.sync()
        graph = Graph(st)
        calls(st)
        graph.end()
        for turn in range(4):
            k, v, q = rows_of(rng, n, 2, 1.0 + turn), rows_of(rng, n, 2, 2.0 ** turn), rng.standard_normal((1, n_q, 256)).astype(np.float32)
            h = [rows_of(rng, 7, 2, 2.0 ** -turn).astype(np.float16) for _ in range(2)]
            for buf, x in ((kd, k), (vd, v), (qd, q), (hk, h[0].view(np.uint16)), (hv, h[1].view(np.uint16))):
                buf.upload(x, st)
            graph.launch()
            got = [b.download(np.float32, count, st) for b, count in ((od, n_q * 256), (ko, 93 * 512), (vo, 93 * 512))]
            x = rows_of(rng, 10, 2)
            tw.append(0, [other], [60], [x], [x])
            # the cache's load rule: codes of exponent field 0 read as signed zeros
            wide = [np.where(np.abs(x) < 2.0 ** -14, np.copysign(np.float32(0), x), x).astype(np.float32) for x in h]
            tw.images[0].append(pool.block_table(a), 41, *wide)
            tok = (48 + np.arange(n)).astype(np.int32)
            tw.images[0].append(pool.block_table(a), 48, oracle.k_prep(k, 2, 256, gamma, 1e-6, table, 64, tok), v)
            tw.assert_pools_equal()
            ck, cv = cells_at(tw, 0, a, 93)
            assert np.array_equal(got[1].reshape(ck.shape), ck) and np.array_equal(got[2].reshape(cv.shape), cv)
            assert check_attn(got[0].reshape(n_q, 256), M.attend64(q, ck, cv, [range(93)], 1 / 16.0)[0])[1] <= REF_BAR_MAX_REL
            calls(st)
            assert np.array_equal(od.download(np.float32, n_q * 256, st), got[0])
        graph.destroy()


@pytest.mark.parametrize("n, longest", [(9, 700), (9, 3001), (40, 700)])    # few entries and many, by the grid and by the search
def test_a_prompt_beside_single_tokens_and_empty_entries(n, longest):
    # entries of very different lengths, none at all among them, first, last and in the middle
    rng = rng_of(40, n)
    lens = [0, 1, 0, 0, longest, 1, 1, 0, 33] + [int(x) for x in rng.integers(0, 2, max(n - 11, 0))] + [19, 0][:max(n - 9, 0)]
    at = [int(x) for x in rng.integers(0, 40, n)]
    gamma, table = (1 + 0.1 * rng.standard_normal(256)).astype(np.float32), rope_table(1e7, 64, 8192)
    with M.F8Twin(n_pages=500, max_seqs=n) as tw:
        pool = tw.pool
        pool.set_free_order(rng.permutation(500).astype(np.int32))
        seqs = [pool.seq_create() for _ in lens]
        for s, p, m in zip(seqs, at, lens):
            pool.seq_reserve(s, p + 2 * m + 1)
            if p:
                fill(tw, s, p, rng)
        ks, vs = ([rows_of(rng, m, 2) for m in lens] for _ in range(2))
        tw.append(0, seqs, at, ks, vs)
        tw.assert_pools_equal()
        bufs = [DeviceBuffer.from_numpy(np.concatenate(x)) for x in (ks, vs)] + [DeviceBuffer.from_numpy(x) for x in (gamma, table)]
        behind = [p + m for p, m in zip(at, lens)]
        pool.append_kprep(0, seqs, behind, lens, bufs[0], bufs[1], bufs[2], 1e-6, bufs[3], 64, 8192)
        device_sync()
        for s, p, m, k, v in zip(seqs, behind, lens, ks, vs):
            if m:
                tok = (p + np.arange(m)).astype(np.int32)
                tw.images[0].append(pool.block_table(s), p, oracle.k_prep(k, 2, 256, gamma, 1e-6, table, 64, tok), v)
        tw.assert_pools_equal()
        total = sum(lens)
        ko, vo = DeviceBuffer(total * 2048), DeviceBuffer(total * 2048)
        pool.read_rows(0, seqs, behind, lens, ko, vo)
        want = [np.concatenate(w) for w in zip(*[tw.images[0].gather(pool.block_table(s), p, m) for s, p, m in zip(seqs, behind, lens)])]
        for got, w in zip((ko, vo), want):
            assert np.array_equal(got.download(np.float32).reshape(w.shape), w)
        for x in bufs + [ko, vo]:
            x.free()


@pytest.mark.parametrize("layout, hd, n_kv", [(L.LAYOUT_F16, 32, 1), (L.LAYOUT_F16, 256, 2), (L.LAYOUT_Q8V, 64, 3), (L.LAYOUT_I8H, 256, 1)])
@pytest.mark.parametrize("n", [9, 40])
def test_reading_back_very_different_lengths(layout, hd, n_kv, n):
    rng = rng_of(41, layout, hd, n)
    lens = [0, 1, 0, 0, 300, 1, 1, 0, 33] + [int(x) for x in rng.integers(0, 3, max(n - 11, 0))] + [19, 0][:max(n - 9, 0)]
    with Pool(n_pages=200, n_kv_head=n_kv, head_dim=hd, layout=layout, max_seqs=n) as pool:
        pool.set_free_order(rng.permutation(200).astype(np.int32))
        seqs = [pool.seq_create() for _ in lens]
        for s, m in zip(seqs, lens):
            pool.seq_reserve(s, m + 3)
        rows = [rng.standard_normal((sum(lens) + 3 * n, n_kv, hd)).astype(np.float32) for _ in range(2)]
        kd, vd = (DeviceBuffer.from_numpy(x) for x in rows)
        pool.append(0, seqs, [0] * n, [m + 3 for m in lens], kd, vd)
        total = sum(lens)
        ko, vo = DeviceBuffer(total * n_kv * hd * 4), DeviceBuffer(total * n_kv * hd * 4)
        pool.read_rows(0, seqs, [2] * n, lens, ko, vo)
        want = [np.concatenate(w) for w in zip(*[pool.gather(0, s, 2, m) for s, m in zip(seqs, lens) if m])]
        for got, w in zip((ko, vo), want):
            assert np.array_equal(got.download(np.float32).reshape(w.shape), w)
        for x in (kd, vd, ko, vo):
            x.free()


def test_a_captured_plan_of_long_walks_replays_eager_steps():
    # 64 layers: pages go past the caches in the plan's launches as in the eager ones
    lens, n_q, layer, n_tok = [1500, 700, 33], 16, 63, 6
    assert sum(lens) * 2 * 512 * 64 >= 96 << 20
    with M.F8Twin(n_layers=64, n_pages=160) as a, M.F8Twin(n_layers=64, n_pages=160) as b:
        for tw in (a, b):
            seqs = [tw.pool.seq_create() for _ in lens]
            for s, n in zip(seqs, lens):
                fill(tw, s, n, rng_of(42, s), layer)
                tw.pool.seq_reserve(s, n + n_tok)
        rng, st = rng_of(43), Stream()
        kd, vd, qd, od = DeviceBuffer(3 * 2048), DeviceBuffer(3 * 2048), DeviceBuffer(3 * n_q * 1024), DeviceBuffer(3 * n_q * 1024)
        plan = StepPlan(a.pool, seqs, lens, n_tok, n_q, st)
        st.sync()
        graph = Graph(st)
        plan.decode(layer, kd, vd, qd, od, 1 / 16.0, stream=st)
        plan.advance(st)
        graph.end()
        for t in range(n_tok):
            q = rng.standard_normal((3, n_q, 256)).astype(np.float32)
            kd.upload(rows_of(rng, 3, 2), st), vd.upload(rows_of(rng, 3, 2), st), qd.upload(q, st)
            graph.launch()
            got = od.download(np.float32, stream=st)
            b.pool.decode_step(layer, seqs, [n + t for n in lens], kd, vd, n_q, qd, od, 1 / 16.0, stream=st)
            assert np.array_equal(got, od.download(np.float32, stream=st)), t
        assert np.array_equal(a.pool.read_layer(layer, 0), b.pool.read_layer(layer, 0))
        graph.destroy()
        plan.destroy()
