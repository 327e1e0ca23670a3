"""The e4m3 layout on the device: pool bytes against the restatement in f8p_model.py, attention against 64 bits over what the pool
holds, at the bars of the other layouts (1e-5 of max(|w|, 1) on N(0, 1) rows: q and the weights enter as two f16 numbers, 2^-21
relative at most, sums in f32)."""
import numpy as np
import pytest

import f8p_model as M
import oracle
from breccia_amd import lib as L
from breccia_amd.kv import BkvError, DeviceBuffer, Graph, Pool, StepPlan, Stream, device_sync, rope_table
from gpu_common import REF_BAR_MAX_REL, Twin, check_attn
from helpers import max_rel

pytestmark = pytest.mark.gpu


def rng_of(*seed):
    return np.random.Generator(np.random.PCG64(list(seed)))


def rows_of(rng, n, n_kv, spread=1.0):
    return (rng.standard_normal((n, n_kv, 256)) * spread).astype(np.float32)


def fill(tw, seq, n, rng, layer=0, spread=1.0, step=1024):
    tw.pool.seq_reserve(seq, max(n, tw.pool.seq_len(seq)))
    for at in range(0, n, step):
        t = min(step, n - at)
        tw.append(layer, [seq], [at], [rows_of(rng, t, tw.g.n_kv, spread)], [rows_of(rng, t, tw.g.n_kv, spread)])


def cells_at(tw, layer, seq, n):
    return tw.images[layer].gather(tw.pool.block_table(seq), 0, n)


# ---- rows in and out ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n_kv", [1, 2, 3, 16])
@pytest.mark.parametrize("f16", [False, True])
def test_append_stores_the_layouts_bytes(n_kv, f16):
    rng = rng_of(1, n_kv, f16)
    with M.F8Twin(n_pages=128, n_kv=n_kv, max_seqs=24) as tw:
        tw.pool.set_free_order(rng.permutation(128).astype(np.int32))
        lens = [1, 15, 16, 17, 40, 97, 3] + [1] * 11          # more than 16 entries in one call too
        seqs = [tw.pool.seq_create() for _ in lens]
        for s, n in zip(seqs, lens):
            tw.pool.seq_reserve(s, n + 40)
        at = [0] * len(lens)
        for turn in range(4):                                   # chunks at odd places behind each other, growing scales
            size = lens if turn == 0 else [int(rng.integers(0, 14)) for _ in lens]
            spread = [float(2.0 ** rng.integers(-6, 7)) for _ in lens]
            ks, vs = ([rows_of(rng, n, n_kv, sp) for n, sp in zip(size, spread)] for _ in range(2))
            if f16:
                ks, vs = ([a.astype(np.float16).view(np.uint16) for a in x] for x in (ks, vs))
            tw.append(0, seqs, at, ks, vs, f16_rows=f16)
            at = [a + n for a, n in zip(at, size)]
            tw.assert_pools_equal()


def test_values_at_the_ends_of_the_rule():
    # largest, beyond it, subnormal codes, halfway cases, infinities and NaN, f32 subnormals, signed zeros, an all-zero page
    rng = rng_of(2)
    bits = rng.integers(0, 2 ** 32, 48 * 2 * 256, dtype=np.uint64).astype(np.uint32).view(np.float32).reshape(48, 2, 256).copy()
    bits[0:16] = rows_of(rng, 16, 2)
    bits[3, 0, :8] = [np.inf, -np.inf, np.nan, 448.0, -448.0, 0.0, -0.0, 1e-40]
    half = np.float32(2.0) ** rng.integers(-9, 8, (16, 2, 256)) * (1 + rng.integers(0, 64, (16, 2, 256)) / 64.0)   # ties among them
    bits[16:32] = half.astype(np.float32)
    zeros = np.zeros((16, 2, 256), np.float32)
    top = np.full((16, 2, 256), 3e38, np.float32)
    tiny = rows_of(rng, 16, 2, 1e-30)
    with M.F8Twin(n_pages=16) as tw:
        s = tw.pool.seq_create()
        tw.pool.seq_reserve(s, 96)
        k = np.concatenate([bits, zeros, top, tiny])
        tw.append(0, [s], [0], [k], [k[::-1].copy()])
        tw.assert_pools_equal()
        gk, gv = tw.pool.gather(0, s, 0, 96)
        wk, wv = cells_at(tw, 0, s, 96)
        assert np.array_equal(gk, wk, equal_nan=True) and np.array_equal(gv, wv, equal_nan=True)


def test_a_rewritten_page_depends_on_its_rows_alone():
    # rolled back and written again: what a larger row left behind is gone, rows behind the last written are cleared
    rng = rng_of(3)
    with M.F8Twin(n_pages=8) as tw:
        tw.pool.fill(0xFF)
        for img in tw.images:
            img.kp[:], img.vp[:] = 0xFF, 0xFF
        s = tw.pool.seq_create()
        tw.pool.seq_reserve(s, 16)
        first, big, again = rows_of(rng, 9, 2), rows_of(rng, 3, 2, 1e4), rows_of(rng, 1, 2)
        tw.append(0, [s], [0], [first], [first])
        tw.append(0, [s], [9], [big], [big])
        tw.assert_pools_equal()
        tw.pool.seq_truncate(s, 9)
        tw.pool.seq_reserve(s, 10)
        tw.append(0, [s], [9], [again], [again])
        tw.assert_pools_equal()
        page = tw.pool.block_table(s)[0]
        assert tw.images[0].exps(page)[:2].max() <= M.exponent([5.0])


@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("n_rot", [2, 64, 256])
def test_kprep_is_the_preparation_and_the_append(n_rot, positions):
    rng = rng_of(4, n_rot, positions)
    lens, at = [33, 1, 16, 50], [0, 5, 16, 7]
    gamma = (1 + 0.3 * rng.standard_normal(256)).astype(np.float32)
    table = rope_table(1e7, n_rot, 60)
    where = rng.integers(-3, 80, 128).astype(np.int32) if positions else None
    with M.F8Twin(n_pages=32, n_kv=2) as tw:
        seqs = [tw.pool.seq_create() for _ in lens]
        for s, n, p in zip(seqs, lens, at):
            tw.pool.seq_reserve(s, n + p)
            if p:
                x = rows_of(rng, p, 2)
                tw.append(0, [s], [0], [x], [x])
        ks, vs = ([rows_of(rng, n, 2, 3.0) for n in lens] for _ in range(2))
        bufs = [DeviceBuffer.from_numpy(a) for a in (np.concatenate(ks), np.concatenate(vs), gamma, table)]
        pd = DeviceBuffer.from_numpy(where) if positions else None
        tw.pool.append_kprep(0, seqs, at, lens, bufs[0], bufs[1], bufs[2], 1e-6, bufs[3], n_rot, 60, pd)
        device_sync()
        for s, n, p, k, v in zip(seqs, lens, at, ks, vs):
            cells = p + np.arange(n)
            tok = np.clip(cells if where is None else where[cells], 0, 59).astype(np.int32)
            assert tw.images[0].append(tw.pool.block_table(s), p, oracle.k_prep(k, 2, 256, gamma, 1e-6, table, n_rot, tok), v) == 0
        tw.assert_pools_equal()
        for b in bufs:
            b.free()


@pytest.mark.parametrize("layout, hd", [(L.LAYOUT_F16, 256), (L.LAYOUT_F16, 96), (L.LAYOUT_Q8V, 256), (L.LAYOUT_Q8V, 32), (L.LAYOUT_I8H, 256),
                                        (L.LAYOUT_F8P, 256)])
@pytest.mark.parametrize("n_kv", [1, 3])
def test_rows_come_back_as_the_cache_holds_them(layout, hd, n_kv):
    rng = rng_of(5, layout, hd, n_kv)
    lens = [1, 16, 100, 33, 7]
    with Pool(n_pages=40, n_kv_head=n_kv, head_dim=hd, layout=layout, max_seqs=20) as pool:
        pool.set_free_order(rng.permutation(40).astype(np.int32))
        seqs = [pool.seq_create() for _ in lens]
        for s, n in zip(seqs, lens):
            pool.seq_reserve(s, n)
            x = (rng.standard_normal((2, n, n_kv, hd)) * 0.02).astype(np.float32)
            kd, vd = DeviceBuffer.from_numpy(x[0]), DeviceBuffer.from_numpy(x[1])
            pool.append(0, [s], [0], [n], kd, vd)
            device_sync()
            kd.free(), vd.free()
        for pick, c0, n in [([0], [0], [1]), ([2, 3, 2, 1, 4], [5, 0, 0, 15, 0], [95, 33, 17, 1, 0]), (list(range(5)) * 4, [0] * 20, lens * 4)]:
            want = [np.concatenate(w) for w in zip(*[pool.gather(0, seqs[i], a, m) for i, a, m in zip(pick, c0, n) if m])]
            for f16 in (False, True):
                dt = np.float16 if f16 else np.float32
                size = want[0].size
                # a guard behind the rows: nothing is written past them
                ko, vo = (DeviceBuffer.from_numpy(np.full(size + 8, 7.0, dt)) for _ in range(2))
                pool.read_rows(0, [seqs[i] for i in pick], c0, n, ko, vo, f16_rows=f16)
                for o, w in zip((ko, vo), want):
                    got = o.download(dt, size + 8)
                    assert np.array_equal(got[:size].reshape(w.shape), w.astype(dt)) and np.all(got[size:] == 7.0)
                    o.free()


# ---- decode attention -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("n_q, n_kv, ctx", [
    (16, 2, [1]), (2, 2, [2, 15, 16, 17, 31, 32, 33]), (24, 2, [300, 64, 65, 128, 1000]), (16, 1, [129, 4097]), (15, 3, [257, 31]),
    (16, 16, [48, 700]), (5, 1, [2048]), (32, 4, [5, 511]), (16, 2, [7] * 40)])
def test_decode_matches_64_bits(n_q, n_kv, ctx):
    rng = rng_of(6, n_q, n_kv, len(ctx))
    with M.F8Twin(n_pages=400, n_kv=n_kv, max_seqs=len(ctx)) as tw:
        tw.pool.fill(0xFF)                                      # NaN wherever nothing was written
        for img in tw.images:
            img.kp[:], img.vp[:] = 0xFF, 0xFF
        tw.pool.set_free_order(rng.permutation(400).astype(np.int32))
        seqs = [tw.pool.seq_create() for _ in ctx]
        for s, n in zip(seqs, ctx):
            fill(tw, s, n, rng)
        q = rng.standard_normal((len(ctx), n_q, 256)).astype(np.float32)
        # the gate as a model leaves it, beside q in one row, and 4 bytes off a 16-byte boundary
        gate = rng.standard_normal((len(ctx), n_q, 512)).astype(np.float32)
        pos = [n - 1 for n in ctx]
        plain = tw.decode_attn(0, seqs, pos, q, n_q)
        gated = tw.decode_attn(0, seqs, pos, q, n_q, gate=gate, gate_strides=(n_q * 512, 512))
        again = tw.decode_attn(0, seqs, pos, q, n_q)
        assert np.array_equal(plain, again)
        for i, (s, n) in enumerate(zip(seqs, ctx)):
            k, v = cells_at(tw, 0, s, n)
            want = M.attend64(q[i:i + 1], k, v, [range(n)], 1 / 16.0)[0]
            assert check_attn(plain[i], want)[1] <= REF_BAR_MAX_REL
            assert check_attn(gated[i], want / (1 + np.exp(-gate[i, :, :256].astype(np.float64))))[1] <= REF_BAR_MAX_REL


def relative_to_values(got, want, v):
    """Errors in units of the largest value a row averages over."""
    return np.max(np.abs(got.astype(np.float64) - want)) / max(float(np.max(np.abs(v))), 1e-300)


@pytest.mark.parametrize("what", ["v scales far apart", "k scales far apart", "large q", "small q", "zero pages", "tiny rows", "huge rows"])
def test_decode_over_scales_far_apart(what):
    rng = rng_of(7, len(what))
    n, n_q = 777, 16
    with M.F8Twin(n_pages=64) as tw:
        s = tw.pool.seq_create()
        k, v = rows_of(rng, n, 2), rows_of(rng, n, 2)
        q = rng.standard_normal((1, n_q, 256)).astype(np.float32)
        page = np.arange(n) // 16
        if what == "v scales far apart":
            v *= (2.0 ** rng.integers(-30, 31, page.max() + 1))[page, None, None]
        elif what == "k scales far apart":
            k *= (2.0 ** -rng.integers(0, 20, page.max() + 1))[page, None, None]
        elif what == "large q":
            q *= 1e9
            k *= 1e-9
        elif what == "small q":
            q *= 1e-25
        elif what == "zero pages":
            v[page % 2 == 0] = 0.0
            k[page % 3 == 0] = 0.0
        elif what == "tiny rows":
            v *= 1e-8
            k *= 1e-8
        else:
            v *= 1e9
            k *= 1e9
            q *= 1e-9
        k, v = k.astype(np.float32), v.astype(np.float32)
        tw.pool.seq_reserve(s, n)
        tw.append(0, [s], [0], [k], [v])
        tw.assert_pools_equal()
        got = tw.decode_attn(0, [s], [n - 1], q, n_q)[0]
        hk, hv = cells_at(tw, 0, s, n)
        want = M.attend64(q, hk, hv, [range(n)], 1 / 16.0)[0]
        # Logits are sums of 256 products of size |q K| / 16: their f32 error is at most 2^-21 of the sum of magnitudes (22-bit
        # q, f32 sums over 8 products in a row and 32 side by side), and enters the output twice over.
        reach = np.max(np.abs(q[0].astype(np.float64)) @ np.abs(hk[:, 0].astype(np.float64)).T) / 16
        assert relative_to_values(got, want, hv) <= 2 * (2.0 ** -21 * max(reach, 1.0)) + 2.0 ** -20, what


def test_nan_reaches_whoever_attends_it_and_nobody_else():
    rng = rng_of(8)
    n, n_q = 70, 16
    with M.F8Twin(n_pages=32) as tw:
        s = tw.pool.seq_create()
        tw.pool.seq_reserve(s, n)
        k, v = rows_of(rng, n, 2), rows_of(rng, n, 2)
        k[50, 0, 3] = np.nan
        v[44, 1, 17] = np.inf
        tw.append(0, [s], [0], [k], [v])
        q = rng.standard_normal((1, n_q, 256)).astype(np.float32)
        for pos in (43, 44, 49, 50, 69):
            got = tw.decode_attn(0, [s], [pos], q, n_q)[0]
            nan = np.zeros((n_q, 256), bool)
            nan[:8] = pos >= 50
            nan[8:, 17] = pos >= 44
            assert np.array_equal(np.isnan(got), nan), pos
        t = 37                                                  # the same from inside a chunk: tokens 40 .. 69 and before
        for pos0, t in ((33, 37), (43, 1), (40, 12)):
            qc = rng.standard_normal((t, n_q, 256)).astype(np.float32)
            got = chunk(tw, 0, [s], [pos0], [qc], n_q)[0]
            nan = np.zeros((t, n_q, 256), bool)
            at = pos0 + np.arange(t)
            nan[at >= 50, :8] = True
            nan[at >= 44, 8:, 17] = True
            assert np.array_equal(np.isnan(got), nan), pos0
            hk, hv = cells_at(tw, 0, s, n)
            hk, hv = np.nan_to_num(hk), np.nan_to_num(hv)
            want = M.attend64(qc, hk, hv, [range(p + 1) for p in at], 1 / 16.0)
            assert max_rel(np.where(nan, 0, got), np.where(nan, 0, want)) <= REF_BAR_MAX_REL


def lists(tw, seqs, pos, q, n_q, ids, counts, max_ids, gate=None):
    bufs = [DeviceBuffer.from_numpy(a) for a in (q, np.zeros_like(q), ids.astype(np.uint32), np.asarray(counts, np.uint32))]
    gd = None if gate is None else DeviceBuffer.from_numpy(gate)
    tw.pool.decode_attn_select(0, seqs, pos, n_q, bufs[0], bufs[1], 1 / 16.0, bufs[2], ids.shape[1], bufs[3], max_ids, gate_dev=gd,
                               gate_seq_stride=n_q * 256, gate_head_stride=256)
    out = bufs[1].download(np.float32, q.size).reshape(q.shape)
    for b in bufs:
        b.free()
    return out


@pytest.mark.parametrize("n_q, n_kv, max_ids", [(24, 2, 40), (16, 2, 1), (3, 3, 513), (16, 1, 5)])
def test_lists_match_64_bits(n_q, n_kv, max_ids):
    rng = rng_of(9, n_q, max_ids)
    ctx = [1, 3000, 17, 500, 64, 900]
    with M.F8Twin(n_pages=400, n_kv=n_kv, max_seqs=8) as tw:
        tw.pool.fill(0xFF)
        for img in tw.images:
            img.kp[:], img.vp[:] = 0xFF, 0xFF
        tw.pool.set_free_order(rng.permutation(400).astype(np.int32))
        seqs = [tw.pool.seq_create() for _ in ctx]
        for s, n in zip(seqs, ctx):
            fill(tw, s, n, rng)
        ids = np.full((len(ctx), max_ids + 3), 0xDEADBEEF, np.uint32)
        counts, cells = [], []
        for i, n in enumerate(ctx):
            # unordered, some twice, some past the position or past any address; one list empty, one longer than its bound
            m = 0 if i == 3 else int(rng.integers(1, max_ids + 1))
            pick = rng.integers(0, (n - 1) // 4 + 3, m).astype(np.uint32)
            if m > 2:
                pick[1] = 0xFFFFFFFF
            ids[i, :m] = pick
            counts.append(m if m < max_ids else m + 2)
            some = np.concatenate([4 * int(b) + np.arange(4) for b in pick if b < 2 ** 29] + [np.zeros(0, np.int64)])
            cells.append(some[some < n])
        q = rng.standard_normal((len(ctx), n_q, 256)).astype(np.float32)
        gate = rng.standard_normal(q.shape).astype(np.float32)
        got = lists(tw, seqs, [n - 1 for n in ctx], q, n_q, ids, counts, max_ids, gate)
        for i, (s, n) in enumerate(zip(seqs, ctx)):
            k, v = cells_at(tw, 0, s, n)
            want = M.attend64(q[i:i + 1], k, v, [cells[i]], 1 / 16.0, gate[i:i + 1])[0]
            assert check_attn(got[i], want, str(i))[1] <= REF_BAR_MAX_REL
            if cells[i].size == 0:
                assert not got[i].any()


def test_step_is_append_and_attention():
    rng = rng_of(10)
    lens, n_q = [1, 15, 16, 300, 47], 24
    with M.F8Twin(n_pages=128) as a, M.F8Twin(n_pages=128) as b:
        for tw in (a, b):
            seqs = [tw.pool.seq_create() for _ in lens]
            for s, n in zip(seqs, lens):
                fill(tw, s, n, rng_of(11, s))
                tw.pool.seq_reserve(s, n + 20)
        q = rng.standard_normal((len(lens), n_q, 256)).astype(np.float32)
        qd, oa, ob = DeviceBuffer.from_numpy(q), DeviceBuffer(q.nbytes), DeviceBuffer(q.nbytes)
        for t in range(20):
            k, v = rows_of(rng, len(lens), 2, 1.0 + t), rows_of(rng, len(lens), 2, 1.0 + t)
            kd, vd = DeviceBuffer.from_numpy(k), DeviceBuffer.from_numpy(v)
            pos = [n + t for n in lens]
            a.pool.decode_step(0, seqs, pos, kd, vd, n_q, qd, oa, 1 / 16.0)
            b.append(0, seqs, pos, [r[None] for r in k], [r[None] for r in v])
            (b.pool.decode_attn_static if t % 2 else b.pool.decode_attn)(0, seqs, pos, n_q, qd, ob, 1 / 16.0)
            assert np.array_equal(oa.download(np.float32), ob.download(np.float32)), t
            kd.free(), vd.free()
        b.assert_pools_equal()
        for which in (0, 1):
            assert np.array_equal(a.pool.read_layer(0, which), b.pool.read_layer(0, which))


def test_captured_step_plan_replays_eager_steps():
    lens, n_q, n_layers, n_tok = [31, 200, 16], 16, 2, 24
    with M.F8Twin(n_layers=n_layers, n_pages=64) as a, M.F8Twin(n_layers=n_layers, n_pages=64) as b:
        for tw in (a, b):
            seqs = [tw.pool.seq_create() for _ in lens]
            for s, n in zip(seqs, lens):
                for layer in range(n_layers):
                    fill(tw, s, n, rng_of(12, s, layer), layer)
                tw.pool.seq_reserve(s, n + n_tok)
        rng, st = rng_of(13), Stream()
        shape, per = (n_layers, len(lens), 2, 256), len(lens) * n_q * 256 * 4
        kd, vd = (DeviceBuffer(int(np.prod(shape)) * 4) for _ in range(2))
        qd, od = DeviceBuffer(n_layers * per), DeviceBuffer(n_layers * per)
        row = len(lens) * 2 * 256 * 4
        plan = StepPlan(a.pool, seqs, lens, n_tok, n_q, st)
        st.sync()
        graph = Graph(st)
        for layer in range(n_layers):
            plan.decode(layer, kd.at(layer * row), vd.at(layer * row), qd.at(layer * per), od.at(layer * per), 1 / 16.0, stream=st)
        plan.advance(st)
        graph.end()
        for t in range(n_tok):
            k, v = (rng.standard_normal(shape).astype(np.float32) * (1 + t % 5) for _ in range(2))
            q = rng.standard_normal((n_layers, len(lens), n_q, 256)).astype(np.float32)
            kd.upload(k, st), vd.upload(v, st), qd.upload(q, st)
            graph.launch()
            got = od.download(np.float32, stream=st)
            for layer in range(n_layers):
                b.pool.decode_step(layer, seqs, [n + t for n in lens], kd.at(layer * row), vd.at(layer * row), n_q, qd.at(layer * per),
                                   od.at(layer * per), 1 / 16.0, stream=st)
            assert np.array_equal(got, od.download(np.float32, stream=st)), t
        for layer in range(n_layers):
            for which in (0, 1):
                assert np.array_equal(a.pool.read_layer(layer, which), b.pool.read_layer(layer, which))
        assert plan.state(st)[1:] == (n_tok, 1) or plan.state(st)[1] <= n_tok
        graph.destroy()
        plan.destroy()


# ---- chunks ---------------------------------------------------------------------------------------------------
def chunk(tw, layer, seqs, pos0, qs, n_q, gates=None, strides=None, stream=None):
    n_tok = [q.shape[0] for q in qs]
    q = np.concatenate([q.reshape(-1, n_q, 256) for q in qs])
    qd, od = DeviceBuffer.from_numpy(q), DeviceBuffer.from_numpy(np.full(q.size + 4, 3.0, np.float32))
    gd, ts, hs = None, 0, 0
    if gates is not None:
        gd = DeviceBuffer.from_numpy(gates)
        ts, hs = strides
    tw.pool.prefill_attn(layer, seqs, pos0, n_tok, n_q, qd, od, 1 / 16.0, gate_dev=gd, gate_tok_stride=ts, gate_head_stride=hs, stream=stream)
    if stream is not None:
        stream.sync()
    out = od.download(np.float32, q.size + 4)
    assert np.all(out[q.size:] == 3.0)
    for b in (qd, od, gd):
        if b is not None:
            b.free()
    return np.split(out[:q.size].reshape(q.shape), np.cumsum(n_tok)[:-1])


@pytest.mark.parametrize("n_q, n_kv, cases, cut", [
    (16, 2, [(0, 1)], False), (16, 2, [(0, 40), (15, 17), (16, 16), (31, 2), (100, 0)], None), (24, 2, [(517, 41)], True), (2, 2, [(0, 200)], None),
    (34, 2, [(60, 33)], None), (20, 1, [(5, 77), (1000, 3)], None), (15, 3, [(130, 70)], None), (16, 16, [(40, 20), (0, 33)], None),
    (16, 2, [(2999, 1)], True), (16, 2, [(700, 900), (3, 1300)], None), (24, 2, [(0, 1500)] * 4, False)])
def test_chunks_match_64_bits(n_q, n_kv, cases, cut):
    rng = rng_of(14, n_q, n_kv, len(cases), cases[0][1])
    with M.F8Twin(n_pages=512, n_kv=n_kv, max_seqs=8) as tw:
        tw.pool.fill(0xFF)
        for img in tw.images:
            img.kp[:], img.vp[:] = 0xFF, 0xFF
        tw.pool.set_free_order(rng.permutation(512).astype(np.int32))
        seqs = [tw.pool.seq_create() for _ in cases]
        for s, (before, t) in zip(seqs, cases):
            fill(tw, s, before + t, rng)
        qs = [rng.standard_normal((t, n_q, 256)).astype(np.float32) for _, t in cases]
        total = sum(t for _, t in cases)
        gate = rng.standard_normal((total, n_q, 512)).astype(np.float32)
        tw.pool.timing_enable(True)
        plain = chunk(tw, 0, seqs, [b for b, _ in cases], qs, n_q)
        tw.pool.timing_enable(False)
        if cut is not None:
            assert tw.pool.timing_read(L.STAGE_ATTN_MERGE)[0] == int(cut)
        gated = chunk(tw, 0, seqs, [b for b, _ in cases], qs, n_q, gate, (n_q * 512, 512))
        odd = np.concatenate([np.zeros(1, np.float32), gate[:, :, :256].reshape(-1)])      # a gate 4 bytes off alignment
        at = 0
        for s, (before, t), q, out, out_g in zip(seqs, cases, qs, plain, gated):
            k, v = cells_at(tw, 0, s, before + t)
            for i in sorted({0, 1, t // 3, t // 2, t - 2, t - 1} & set(range(t))):
                want = M.attend64(q[i:i + 1], k, v, [range(before + i + 1)], 1 / 16.0)[0]
                assert check_attn(out[i], want, "%d + %d" % (before, i))[1] <= REF_BAR_MAX_REL
                want = want / (1 + np.exp(-gate[at + i, :, :256].astype(np.float64)))
                assert check_attn(out_g[i], want)[1] <= REF_BAR_MAX_REL
            at += t
        gd = DeviceBuffer.from_numpy(odd)
        q = np.concatenate(qs)
        qd, od = DeviceBuffer.from_numpy(q), DeviceBuffer(max(q.nbytes, 16))
        tw.pool.prefill_attn(0, seqs, [b for b, _ in cases], [t for _, t in cases], n_q, qd, od, 1 / 16.0, gate_dev=gd.at(4),
                             gate_tok_stride=n_q * 256, gate_head_stride=256)
        assert np.array_equal(od.download(np.float32, q.size).reshape(q.shape), np.concatenate(gated))
        for b in (gd, qd, od):
            b.free()


@pytest.mark.parametrize("what", ["v scales far apart", "zero pages", "large q"])
@pytest.mark.parametrize("before, t", [(300, 50), (0, 700)])
def test_chunks_over_scales_far_apart(what, before, t):
    rng = rng_of(15, len(what), before)
    n, n_q = before + t, 16
    with M.F8Twin(n_pages=64) as tw:
        s = tw.pool.seq_create()
        k, v = rows_of(rng, n, 2), rows_of(rng, n, 2)
        q = rng.standard_normal((t, n_q, 256)).astype(np.float32)
        page = np.arange(n) // 16
        if what == "large q":
            q, k = (q * 1e9).astype(np.float32), (k * 1e-9).astype(np.float32)
        elif what == "zero pages":
            v[page % 2 == 0] = 0.0
        else:
            v = (v * (2.0 ** rng.integers(-30, 31, page.max() + 1))[page, None, None]).astype(np.float32)
        tw.pool.seq_reserve(s, n)
        tw.append(0, [s], [0], [k], [v])
        got = chunk(tw, 0, [s], [before], [q], n_q)[0]
        hk, hv = cells_at(tw, 0, s, n)
        for i in (0, 1, t // 2, t - 1):
            want = M.attend64(q[i:i + 1], hk, hv, [range(before + i + 1)], 1 / 16.0)[0]
            reach = np.max(np.abs(q[i].astype(np.float64)) @ np.abs(hk[:, 0].astype(np.float64)).T) / 16
            assert relative_to_values(got[i], want, hv[:before + i + 1]) <= 2 * (2.0 ** -21 * max(reach, 1.0)) + 2.0 ** -20, (what, i)


def test_captured_chunk_replays():
    rng = rng_of(16)
    n_q, before, t = 16, 500, 40
    with M.F8Twin(n_pages=64) as tw:
        s, st = tw.pool.seq_create(), Stream()
        fill(tw, s, before + t, rng)
        q = rng.standard_normal((t, n_q, 256)).astype(np.float32)
        qd, od = DeviceBuffer.from_numpy(q), DeviceBuffer(q.nbytes)
        tw.pool.prefill_attn(0, [s], [before], [t], n_q, qd, od, 1 / 16.0, stream=st)
        st.sync()
        g = Graph(st)
        tw.pool.prefill_attn(0, [s], [before], [t], n_q, qd, od, 1 / 16.0, stream=st)
        g.end()
        k, v = cells_at(tw, 0, s, before + t)
        for turn in range(3):
            q = rng.standard_normal((t, n_q, 256)).astype(np.float32)
            qd.upload(q, st)
            g.launch()
            got = od.download(np.float32, stream=st).reshape(q.shape)
            for i in (0, t - 1):
                assert check_attn(got[i], M.attend64(q[i:i + 1], k, v, [range(before + i + 1)], 1 / 16.0)[0])[1] <= REF_BAR_MAX_REL
        g.destroy()


# ---- together -------------------------------------------------------------------------------------------------
def test_a_conversation_forked_swapped_and_continued():
    """Prompt in chunks, decode steps, a fork with its copied page, pages out to the host and back, a rollback: every token's
    attention against 64 bits, and every byte of the pool against the model."""
    rng = rng_of(17)
    n_q, n_layers = 24, 2
    with M.F8Twin(n_layers=n_layers, n_pages=96, max_seqs=4) as tw:
        pool = tw.pool
        pool.set_free_order(rng.permutation(96).astype(np.int32))
        a = pool.seq_create()

        def prompt(seq, at, t):
            for src, dst in pool.seq_reserve(seq, at + t):
                pool.page_copy([(src, dst)])
                for img in tw.images:
                    img.page_copy([(src, dst)])
            for layer in range(n_layers):
                x = [rows_of(rng, t, 2, 2.0 ** layer) for _ in range(2)]
                tw.append(layer, [seq], [at], [x[0]], [x[1]])
                q = rng.standard_normal((t, n_q, 256)).astype(np.float32)
                got = chunk(tw, layer, [seq], [at], [q], n_q)[0]
                k, v = cells_at(tw, layer, seq, at + t)
                want = M.attend64(q[[0, -1]], k, v, [range(at + 1), range(at + t)], 1 / 16.0)
                assert check_attn(got[[0, -1]], want)[1] <= REF_BAR_MAX_REL

        def token(seqs, pos):
            for s, p in zip(seqs, pos):
                for src, dst in pool.seq_reserve(s, p + 1):
                    pool.page_copy([(src, dst)])
                    for img in tw.images:
                        img.page_copy([(src, dst)])
            for layer in range(n_layers):
                k, v = rows_of(rng, len(seqs), 2), rows_of(rng, len(seqs), 2)
                q = rng.standard_normal((len(seqs), n_q, 256)).astype(np.float32)
                bufs = [DeviceBuffer.from_numpy(x) for x in (k, v, q, np.zeros_like(q))]
                pool.decode_step(layer, seqs, pos, bufs[0], bufs[1], n_q, bufs[2], bufs[3], 1 / 16.0)
                got = bufs[3].download(np.float32).reshape(q.shape)
                for i, (s, p) in enumerate(zip(seqs, pos)):
                    assert tw.images[layer].append(pool.block_table(s), p, k[i], v[i]) == 0
                    hk, hv = cells_at(tw, layer, s, p + 1)
                    want = M.attend64(q[i:i + 1], hk, hv, [range(p + 1)], 1 / 16.0)[0]
                    assert check_attn(got[i], want)[1] <= REF_BAR_MAX_REL
                for b in bufs:
                    b.free()

        prompt(a, 0, 130)
        prompt(a, 130, 45)
        for p in range(175, 180):
            token([a], [p])
        b = pool.seq_fork(a, 178)                       # inside a page: the child's first token copies it
        for t in range(4):
            token([a, b], [180 + t, 178 + t])
        host = pool.host_alloc(3 * pool.swap_page_bytes())
        c = pool.seq_create()
        prompt(c, 0, 64)
        before = [tw.images[layer].gather(pool.block_table(c), 16, 48) for layer in range(n_layers)]
        pool.seq_evict(c, 1, 3, host)
        pool.swap_wait()
        prompt(b, 182, 40)                              # takes pages that c gave back
        pool.seq_restore(c, 1, 3, host)
        pool.swap_wait()
        for layer in range(n_layers):
            got = pool.gather(layer, c, 16, 48)
            assert np.array_equal(got[0], before[layer][0]) and np.array_equal(got[1], before[layer][1])
        pool.seq_truncate(b, 200)                       # rejected tokens
        for p in range(200, 204):
            token([b], [p])
        for layer in range(n_layers):
            for s, n in ((a, 184), (b, 204)):
                got, want = pool.gather(layer, s, 0, n), tw.images[layer].gather(pool.block_table(s), 0, n)
                assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        host.free()
        pool.check()
