"""The e4m3 layout restated in 64 bits with numpy, from its definition (include/breccia_kv.h, BKV_LAYOUT_F8P): the value rule, the
bytes of a page, and what a write does to a page.  The pools of the GPU tests are compared with it byte for byte."""
import numpy as np

import oracle
from breccia_amd import lib as L
from breccia_amd.kv import Pool
from gpu_common import Twin

E_LO, E_HI, TOP, HD, PAGE, UNIT = -32, 31, 448.0, 256, 16, 4096


def exponent(x):
    """The scale's exponent for values x (finite ones count)."""
    x = np.abs(np.asarray(x, dtype=np.float64))
    top = np.max(np.where(np.isfinite(x), x, 0.0), initial=0.0)
    for e in range(E_LO, E_HI):
        if top <= TOP * 2.0 ** e:
            return e
    return E_HI


def code_values():
    """The 256 values of e4m3, NaN at 0x7f and 0xff."""
    c = np.arange(256)
    ex, m = (c >> 3) & 15, c & 7
    v = np.where(ex == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (np.maximum(ex, 1) - 10.0))
    v = np.where(c & 0x80, -v, v)
    v[[0x7F, 0xFF]] = np.nan
    return v


VALUES = code_values()


def encode(x, e):
    """Codes of x under 2^e: nearest, ties to even, NaN where x is not finite."""
    x = np.asarray(x, dtype=np.float64)
    fin = np.isfinite(x)
    y = np.clip(np.where(fin, x, 0.0) / 2.0 ** e, -TOP, TOP)
    a = np.abs(y)
    ex = np.maximum(np.frexp(np.maximum(a, 2.0 ** -40))[1] - 1, -6)          # the binade, subnormals with the lowest
    n = np.rint(a / 2.0 ** (ex - 3.0)).astype(np.int64)                      # steps of an eighth of it
    code = np.where(n < 8, n, ((ex + 6) << 3) + n)                           # n == 16: the next binade's first code
    code = code | np.where(np.signbit(y), 0x80, 0)
    return np.where(fin, code, 0x7F).astype(np.uint8)


def k_offset(cell, d):
    h, u, s, k = d >> 7, (d >> 5) & 3, (d >> 2) & 7, d & 3
    return (cell >> 2) * 1024 + (8 * h + s) * 64 + (cell & 3) * 16 + 4 * u + k


def v_offset(cell, d):
    return (cell >> 2) * 1024 + 4 * d + (cell & 3)


_C, _D = np.meshgrid(np.arange(PAGE), np.arange(HD), indexing="ij")
K_AT, V_AT = k_offset(_C, _D), v_offset(_C, _D)


class F8Image:
    """One layer's pool bytes, written and read through block tables (the interface of oracle.PoolImage)."""

    def __init__(self, n_kv, n_pages):
        self.n_kv = n_kv
        self.kp = np.zeros((n_pages, n_kv * UNIT + 128), dtype=np.uint8)
        self.vp = np.zeros((n_pages, n_kv * UNIT), dtype=np.uint8)

    k = property(lambda self: self.kp.reshape(-1))
    v = property(lambda self: self.vp.reshape(-1))

    def exps(self, page):
        return self.kp[page, self.n_kv * UNIT:].view(np.int32).reshape(-1, 2)

    def units(self, page, h):
        return ((self.kp[page, h * UNIT:(h + 1) * UNIT], K_AT, 0), (self.vp[page, h * UNIT:(h + 1) * UNIT], V_AT, 1))

    def append(self, table, pos0, k, v, capacity_cells=None):
        rows = [np.asarray(a, dtype=np.float32).reshape(-1, self.n_kv, HD) for a in (k, v)]
        n = rows[0].shape[0]
        if capacity_cells is not None and pos0 + n > capacity_cells:
            return 1
        for lp in range(pos0 // PAGE, (pos0 + n - 1) // PAGE + 1):
            kept, end = max(pos0 - lp * PAGE, 0), min(pos0 + n - lp * PAGE, PAGE)
            page = int(table[lp])
            for h in range(self.n_kv):
                for unit, at, side in self.units(page, h):
                    x = np.zeros((PAGE, HD))
                    old = 2.0 ** int(np.clip(self.exps(page)[h, side], E_LO, E_HI))
                    x[:kept] = VALUES[unit[at]][:kept] * old
                    with np.errstate(invalid="ignore"):
                        x[kept:end] = rows[side][lp * PAGE + kept - pos0:lp * PAGE + end - pos0, h]
                    e = exponent(x)
                    unit[at] = encode(x, e)
                    self.exps(page)[h, side] = e
        return 0

    def gather(self, table, cell0, n):
        out = np.zeros((2, n, self.n_kv, HD))
        for i in range(n):
            page, c = int(table[(cell0 + i) // PAGE]), (cell0 + i) % PAGE
            for h in range(self.n_kv):
                for unit, at, side in self.units(page, h):
                    out[side, i, h] = VALUES[unit[at[c]]] * 2.0 ** int(np.clip(self.exps(page)[h, side], E_LO, E_HI))
        return out[0].astype(np.float32), out[1].astype(np.float32)

    def page_copy(self, pairs):
        for s, d in pairs:
            self.kp[d], self.vp[d] = self.kp[s], self.vp[s]


def same_codes(a, b):
    """Bytes equal, the two NaN codes taken for one."""
    return np.array_equal(np.where(a == 0xFF, 0x7F, a), np.where(b == 0xFF, 0x7F, b))


class F8Twin(Twin):
    """A device pool of this layout and its images."""

    def __init__(self, n_layers=1, n_pages=512, n_kv=2, max_seqs=16, max_pages_per_seq=None):
        self.pool = Pool(n_layers=n_layers, n_pages=n_pages, n_kv_head=n_kv, head_dim=HD, layout=L.LAYOUT_F8P, max_seqs=max_seqs,
                         max_pages_per_seq=max_pages_per_seq)
        self.g = oracle.Geom(n_kv, HD, PAGE)
        self.layout = L.LAYOUT_F8P
        self.images = [F8Image(n_kv, n_pages) for _ in range(n_layers)]

    def assert_pools_equal(self, layer=0):
        img = self.images[layer]
        got = self.pool.read_layer(layer, 0).reshape(img.kp.shape), self.pool.read_layer(layer, 1).reshape(img.vp.shape)
        split = img.n_kv * UNIT
        assert np.array_equal(got[0][:, split:], img.kp[:, split:]), "exponents"
        assert same_codes(got[0][:, :split], img.kp[:, :split]), "K codes"
        assert same_codes(got[1], img.vp), "V codes"


def attend64(q, k, v, cells_of_row, scale, gate=None):
    """Attention in 64 bits: q [T, n_q, HD], k / v [C, n_kv, HD] f32, row t over the listed cells (zeros where none)."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    group = q.shape[1] // k.shape[1]
    out = np.zeros(q.shape)
    for t, cells in enumerate(cells_of_row):
        cells = np.asarray(cells, dtype=np.int64)
        if cells.size == 0:
            continue
        for h in range(q.shape[1]):
            with np.errstate(invalid="ignore"):
                s = (k[cells, h // group] @ q[t, h]) * scale
                p = np.exp(s - np.max(s))
                out[t, h] = (p @ v[cells, h // group]) / p.sum()
    return out if gate is None else out / (1.0 + np.exp(-np.asarray(gate, dtype=np.float64)))
