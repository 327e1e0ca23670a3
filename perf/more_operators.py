"""Operators of conversations that branch, as they are measured: decode attention of a batch whose sequences share prefixes, a
sequence's cells compacted to those that a list keeps, and rows written with a rotary of several axes.

A case is a dict of plain values.  `kind`:

  shared   attention of one token of every entry.  "groups": of each its shared cells and, entry by entry, the cells that it has of
           its own behind them ("cells|own,own,...;cells|own,..."); q and the output [entries, n_q, 256]
  compact  of every sequence the cells from `first` on become the listed ones, in all layers, on a fork that leaves the sequence as it
           was.  "lists": the same for all ("one"), or of its own for each kv head of each layer ("own").  Then the new
           cells are read back as rows ("rows"), or a token attends what the sequence has now, layer by layer ("attend")
  axes     rows behind what their first pages hold, K through RMSNorm and a rotary whose pairs turn by the token's position on
           one of several axes ("pairs": axis of each pair), then read back

What a cache holds (`layout`): "f16" rows of binary16; "i8" codes with a binary16 scale for 32 values; "e4m3" codes with a power of two
as scale for each page of 16 cells and kv head, which is that of all rows in the page.

With `own` the calls are those of breccia_amd.kv.Pool, without it the same in elementary torch operations in 32 bits.
"""
import math
import random

import numpy as np
import torch

own = False

HD, PAGE = 256, 16                      # head dim, cells of a page
EPS, FREQ = 1e-6, 1e7                   # the K preparation of the model
SCALE = 1.0 / 16.0
E_LO, E_HI, TOP = -32, 31, 448.0        # e4m3: exponents of the scales, the largest code


def _ints(text):
    return [int(v) for v in text.split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _uniform(seed, n, lo, hi):
    r = random.Random(seed)
    return [r.randint(lo, hi) for _ in range(n)]


def _groups(case):
    return [(int(g.split("|")[0]), _ints(g.split("|")[1])) for g in case["groups"].split(";")]


def _shared(groups, n_q=16, n_kv=2, gate=False, layout="f16"):
    return dict(kind="shared", layout=layout, n_q=n_q, n_kv=n_kv, gate=gate, groups=";".join("%d|%s" % (c, _text(o)) for c, o in groups))


def _compact(length, first, keep, lists="one", then="rows", layers=4, n_kv=2, layout="f16"):
    return dict(kind="compact", layout=layout, n_kv=n_kv, layers=layers, lists=lists, then=then, length=_text(length), first=_text(first),
                keep=_text(keep))


def _pairs(sections, interleaved):
    """The axis of each pair: the axes one after the other, or in turns for as long as an axis has pairs left."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def _axes(pos0, tokens, sections=(11, 11, 10), interleaved=True, n_kv=2, layout="f16"):
    return dict(kind="axes", layout=layout, n_kv=n_kv, pos0=_text(pos0), tokens=_text(tokens), pairs=_text(_pairs(sections, interleaved)))


def listed():
    named = [
        # four samples of one short prompt, a few tokens in: launches and latency
        ("shared_samples_b4", _shared([(517, [38, 12, 25, 7])])),
        # 32 answers to one prompt
        ("shared_answers_b32", _shared([(8192, _uniform(21, 32, 1, 1024))])),
        # questions to one long document, the model's heads and output gate
        ("shared_document_b64", _shared([(65519, _uniform(22, 64, 50, 2000))], n_q=24, gate=True)),
        # several prompts with their samples in one batch, a compressed cache
        ("shared_prompts_b64_e4m3", _shared([(16384, _uniform(23, 16, 10, 700)), (2049, _uniform(24, 16, 10, 700)),
                                             (9001, _uniform(25, 24, 10, 700)), (0, _uniform(26, 8, 100, 4000))], layout="e4m3")),
        # an int8 cache, one odd prefix
        ("shared_answers_b24_i8", _shared([(12289, _uniform(27, 24, 1, 500))], layout="i8")),
        # the accepted path of a draft tree: five of sixteen cells stay, sixteen conversations
        ("compact_drafts_b16", _compact([n + 16 for n in _uniform(31, 16, 500, 2000)], _uniform(31, 16, 500, 2000), [5] * 16)),
        # a long conversation brought to a quarter, every head keeps its own cells; then the next token
        ("compact_long_attend", _compact([32768], [0], [8192], lists="own", then="attend")),
        # first cells and a window of the last ones, of eight conversations, in a compressed cache
        ("compact_windows_b8_e4m3", _compact(_uniform(32, 8, 3000, 9000), [4] * 8, _uniform(33, 8, 1000, 2000), lists="one", layout="e4m3")),
        # the same cells for all heads of an int8 cache, odd sizes
        ("compact_ragged_i8", _compact([1501, 4097, 333], [37, 1024, 0], [700, 2049, 1], layout="i8", n_kv=4)),
        # a new token of each of 32 conversations with pictures
        ("axes_tokens_b32", _axes(_uniform(41, 32, 0, 511), [1] * 32)),
        # two prompts with pictures
        ("axes_prompts", _axes([0, 0], [8191, 8191])),
        # ragged pieces of them into a compressed cache; the axes' pairs one after the other, 128 values turn
        ("axes_ragged_e4m3", _axes([1501, 37, 900, 16, 3], [333, 700, 1021, 17, 2], (16, 24, 24), False, 4, "e4m3")),
    ]
    return [dict(case, name=name) for name, case in named]


def _log(rng, lo, hi):
    """An integer of lo..hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "shared", "compact", "compact", "compact", "axes", "axes"])
    layout = rng.choice(["f16", "f16", "e4m3", "i8"])
    n_kv = rng.choice([2, 2, 2, 1, 4, 3])
    if kind == "shared":
        n_q = n_kv * rng.choice([8, 8, 12, 4, 16, 1] if n_kv < 3 else [8, 5, 4])
        groups, left, cost = [], _log(rng, 1, 64), 100_000_000
        while left > 0:
            n = rng.choice([1, left, _log(rng, 1, left)])
            cells, most = rng.choice([0, _log(rng, 1, 65536), _log(rng, 1, 65536)]), _log(rng, 1, 2000)
            members = [_log(rng, 1, most) for _ in range(n)]
            left -= n
            pairs = (cells * n + sum(members)) * n_q
            if groups and pairs > cost:
                break
            if pairs > cost:
                cells = cost // (n * n_q)
            groups.append((cells, members))
            cost -= min(cost, pairs)
        return _shared(groups, n_q, n_kv, rng.random() < 0.5, layout)
    if kind == "compact":
        n, layers = _log(rng, 1, 32), rng.choice([1, 2, 4])
        total = _log(rng, max(64, n), 65536 // (n_kv * layers) * 2)
        length = [max(1, _log(rng, max(1, total // n // 4), total // n + 1)) for _ in range(n)]
        first = [rng.choice([0, rng.randint(0, m)]) for m in length]
        keep = [rng.randint(min(1, m - f), _log(rng, 1, m - f) if m > f else 0) for m, f in zip(length, first)]
        keep = [m or int(f == 0) for m, f in zip(keep, first)]     # something is left of each
        if not any(keep):
            first[0], keep[0] = first[0] - 1, 1
        return _compact(length, first, keep, rng.choice(["one", "own"]), rng.choice(["rows", "attend"]), layers, n_kv, layout)
    n, total = _log(rng, 1, 64), _log(rng, 64, 32768 // n_kv)
    each = max(1, total // n)
    tokens = [max(1, each + rng.randint(-min(each // 2, 100), min(each // 2, 100))) for _ in range(n)]
    sections = rng.choice([(11, 11, 10), (16, 24, 24), (8, 12, 12), (32, 32), (20, 5, 4, 3)])
    return _axes([rng.choice([0, rng.randint(1, 2000)]) for _ in tokens], tokens, sections, rng.random() < 0.5, n_kv, layout)


class _State:
    pool = None

    def __del__(self):
        if self.pool is not None:
            self.pool.destroy()


# ---- what a cache holds of rows -----------------------------------------------------------------
def _pages(rows):
    """[cells, n_kv, 256] -> [pages, 16, n_kv, 256], the last page filled up with zeros."""
    n = rows.shape[0]
    full = (n + PAGE - 1) // PAGE * PAGE
    if full != n:
        rows = torch.cat([rows, rows.new_zeros(full - n, *rows.shape[1:])])
    return rows.reshape(-1, PAGE, *rows.shape[1:])


def _hold(layout, rows):
    """Rows [cells, n_kv, 256] (f32) from a page's first cell on -> what the cache keeps of them."""
    if layout == "f16":
        return (torch.where(rows.abs() < 2.0 ** -14, torch.zeros_like(rows), rows).half(),)   # it holds no subnormals
    if layout == "i8":
        b = rows.reshape(*rows.shape[:-1], HD // 32, 32)
        a = b.abs().amax(-1, keepdim=True)
        s = torch.where(a > 0, (a / 127.0).half().float(), torch.ones_like(a))
        s = torch.where(s < 2.0 ** -14, torch.full_like(s, 2.0 ** -14), s)
        t = (b / s).clamp(-127.0, 127.0).double()
        return (torch.where(t < 0, -torch.floor(0.5 - t), torch.floor(t + 0.5)).to(torch.int8), s.half())
    x = _pages(rows)
    a = x.abs().amax((1, 3), keepdim=True)
    m, e = torch.frexp(a)                        # a = m * 2^e, m of 1/2 .. 1
    e = torch.where(a > 0, e - 9 + (m > 0.875).to(e.dtype), E_LO).clamp(E_LO, E_HI)
    return ((x * torch.exp2(-e.float())).clamp(-TOP, TOP).to(torch.float8_e4m3fn), torch.exp2(e.float()))


def _value(held, cells):
    """The rows of the first `cells` cells, f32 [cells, n_kv, 256]."""
    if len(held) == 1:
        return held[0][:cells].float()
    codes, scales = held
    x = codes.float() * scales.float()
    return x.reshape(-1, x.shape[2], HD)[:cells] if codes.dtype == torch.float8_e4m3fn else x.reshape(*x.shape[:-2], HD)[:cells]


def _joined(layout, held, cells, rows):
    """What pages that hold `cells` cells hold once `rows` stand behind these."""
    if layout == "e4m3":                         # the scale is that of all rows in a page
        return _hold(layout, torch.cat([_value(held, cells), rows]))
    return tuple(torch.cat([a[:cells], b]) for a, b in zip(held, _hold(layout, rows)))


# ---- inputs -------------------------------------------------------------------------------------
def _draws(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    return randn


def _spread(randn, n_kv):
    """Channels of K differ in size, a few by far."""
    s = torch.exp(0.4 * randn(n_kv, HD))
    return torch.where(randn(n_kv, HD) > 2.0, 3.0 * s, s)


def _rows(randn, n, n_kv, spread):
    return randn(n, n_kv, HD) * spread, randn(n, n_kv, HD) * torch.exp(0.5 * randn(n, n_kv, 1))


def _table(n, pairs, device):
    """cos and sin of the rotary's angles [n, pairs, 2], worked out in 64 bits."""
    inv = torch.tensor([FREQ ** (-1.0 * i / pairs) for i in range(pairs)], dtype=torch.float64, device=device)
    angle = torch.arange(n, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack([torch.cos(angle), torch.sin(angle)], -1).float().contiguous()


def _positions(seed, n_axes, pos0, tokens):
    """Positions of a sequence's tokens on each axis: text goes on by one on all of them, a picture stands at one time, its rows
    and columns of patches on the axes behind (with two axes: those), and the text after it goes on behind the largest."""
    r = random.Random(seed)
    out, at = [], pos0
    while len(out) < tokens:
        for _ in range(r.randint(1, 60)):
            out.append([at] * n_axes)
            at += 1
        h, w = r.randint(4, 24), r.randint(4, 24)
        out += [([at] + [at + y, at + x] + [at + x // 2] * 4)[:n_axes] if n_axes > 2 else [at + y, at + x] for y in range(h) for x in range(w)]
        at += max(h, w)
    return out[:tokens]


def _inputs(case, seed):
    """Everything a pass is given, in plain form."""
    randn = _draws(seed)
    n_kv, kind = case["n_kv"], case["kind"]
    x = _State()
    if kind == "shared":
        spread = _spread(randn, n_kv)
        x.groups = _groups(case)
        x.prefix = [_rows(randn, cells, n_kv, spread) for cells, _ in x.groups]
        x.tails = [[_rows(randn, m, n_kv, spread) for m in members] for _, members in x.groups]
        n = sum(len(members) for _, members in x.groups)
        x.q = randn(n, case["n_q"], HD)
        x.gate = randn(n, case["n_q"], HD) if case["gate"] else None
        return x
    if kind == "compact":
        x.length, x.first, x.keep = _ints(case["length"]), _ints(case["first"]), _ints(case["keep"])
        layers = case["layers"]
        spread = [_spread(randn, n_kv) for _ in range(layers)]
        x.rows = [[_rows(randn, n, n_kv, s) for n in x.length] for s in spread]
        of = (layers, n_kv) if case["lists"] == "own" else (1, 1)
        x.lists = torch.empty(*of, sum(x.keep), dtype=torch.int32, device="cuda")
        at = 0
        for n, f, m in zip(x.length, x.first, x.keep):
            if m:
                score = randn(*of, n - f)
                x.lists[:, :, at:at + m] = (score.topk(m, -1).indices.sort(-1).values + f).int()
            at += m
        if case["then"] == "attend":
            x.q = randn(layers, len(x.length), 8 * n_kv, HD)
        return x
    x.pos0, x.tokens = _ints(case["pos0"]), _ints(case["tokens"])
    spread = _spread(randn, n_kv)
    x.before = [p // PAGE * PAGE for p in x.pos0]
    x.held = [_rows(randn, p - f, n_kv, spread) for p, f in zip(x.pos0, x.before)]
    x.k, x.v = _rows(randn, sum(x.tokens), n_kv, spread)
    x.gamma = 1.0 + 0.1 * randn(HD)
    pairs = _ints(case["pairs"])
    spots = [s for i, (p, t) in enumerate(zip(x.pos0, x.tokens)) for s in _positions(seed * 100 + i, max(pairs) + 1, p, t)]
    x.positions = torch.tensor(spots, dtype=torch.int32).t().contiguous().cuda()
    x.table = _table(int(x.positions.max()) + 1, len(pairs), "cuda")
    return x


def prepare(case, seed):
    s = _inputs(case, seed)
    s.case = case
    kind, n_kv, layout = case["kind"], case["n_kv"], case["layout"]
    if not own:
        if kind == "shared":
            # the prefix' pages, and each entry's own from the page in which it leaves them
            s.caches = []
            for (cells, members), prefix, tails in zip(s.groups, s.prefix, s.tails):
                base = cells // PAGE * PAGE
                whole = [_hold(layout, p[:base]) for p in prefix]
                rest = [_hold(layout, p[base:]) for p in prefix]
                s.caches.append((whole, [[_joined(layout, r, cells - base, t) for r, t in zip(rest, tail)] for tail in tails]))
            s.prefix = s.tails = None
        elif kind == "compact":
            s.caches = [[tuple(_hold(layout, r) for r in pair) for pair in layer] for layer in s.rows]
            s.rows = None
        else:
            s.caches = [tuple(_hold(layout, r) for r in pair) for pair in s.held]
            s.held = None
        torch.cuda.synchronize()
        return s
    from breccia_amd import lib as L
    from breccia_amd.kv import Pool

    def make(pages, layers, n_seqs):
        n = int(sum(pages) / 0.6) + 1
        pool = s.pool = Pool(n_layers=layers, n_pages=n, n_kv_head=n_kv, head_dim=HD, max_seqs=n_seqs, max_pages_per_seq=max(pages),
                             layout={"f16": L.LAYOUT_F16, "i8": L.LAYOUT_I8H, "e4m3": L.LAYOUT_F8P}[layout])
        pool.set_free_order(np.random.RandomState(seed).permutation(n).astype(np.int32))
        return pool

    def up(cells):
        return (cells + PAGE - 1) // PAGE

    def write(pool, layer, seq, first, pair):
        if pair[0].shape[0]:
            pool.append(layer, [seq], [first], [pair[0].shape[0]], pair[0].data_ptr(), pair[1].data_ptr())

    if kind == "shared":
        ends = [cells + m for cells, members in s.groups for m in members]
        pool = make([up(e) for e in ends], 1, len(ends) + len(s.groups))
        seqs, entries, cells_of = [], [], []
        for (cells, members), prefix, tails in zip(s.groups, s.prefix, s.tails):
            base = pool.seq_create()
            pool.seq_reserve(base, cells)
            write(pool, 0, base, 0, prefix)
            for m, tail in zip(members, tails):
                seq = pool.seq_fork(base, cells)
                copies = pool.seq_reserve(seq, cells + m)
                if copies:
                    pool.page_copy(copies)
                write(pool, 0, seq, cells, tail)
                seqs.append(seq)
            entries.append(len(members))
            cells_of.append(cells)
        s.seqs, s.pos = np.array(seqs, dtype=np.int32), np.array([e - 1 for e in ends], dtype=np.int64)
        s.entries, s.cells = np.array(entries, dtype=np.int32), np.array(cells_of, dtype=np.int64)
        s.out = torch.zeros_like(s.q)
    elif kind == "compact":
        pool = make([up(n) * 2 for n in s.length], case["layers"], 2 * len(s.length))
        s.seqs = [pool.seq_create() for _ in s.length]
        for seq, n in zip(s.seqs, s.length):
            pool.seq_reserve(seq, n)
        for layer, rows in enumerate(s.rows):
            for seq, pair in zip(s.seqs, rows):
                write(pool, layer, seq, 0, pair)
        if case["lists"] == "own":
            s.strides = (s.lists.stride(0), s.lists.stride(1))
        else:
            s.strides = (0, 0)
        s.first_a, s.keep_a = np.array(s.first, dtype=np.int64), np.array(s.keep, dtype=np.int32)
        if case["then"] == "attend":
            s.out = torch.zeros_like(s.q)
            s.last = s.first_a + s.keep_a - 1
        else:
            shape = (case["layers"], sum(s.keep), n_kv, HD)
            wanted = torch.float16 if layout == "f16" else torch.float32
            s.k_out, s.v_out = (torch.zeros(*shape, dtype=wanted, device="cuda") for _ in range(2))
    else:
        ends = [p + t for p, t in zip(s.pos0, s.tokens)]
        pool = make([up(e) for e in ends], 1, len(ends))
        s.seqs = np.array([pool.seq_create() for _ in ends], dtype=np.int32)
        for seq, end, first, pair in zip(s.seqs.tolist(), ends, s.before, s.held):
            pool.seq_reserve(seq, end)
            write(pool, 0, seq, first, pair)
        s.pos, s.n_tok = np.array(s.pos0, dtype=np.int64), np.array(s.tokens, dtype=np.int32)
        s.cell0 = np.array(s.before, dtype=np.int64)
        s.n_cells = np.array([e - f for e, f in zip(ends, s.before)], dtype=np.int32)
        s.pair_axis = np.array(_ints(case["pairs"]), dtype=np.uint8)
        wanted = torch.float16 if layout == "f16" else torch.float32
        s.k_out, s.v_out = (torch.zeros(int(s.n_cells.sum()), n_kv, HD, dtype=wanted, device="cuda") for _ in range(2))
    s.prefix = s.tails = s.rows = s.held = None
    torch.cuda.synchronize()
    return s


# ---- a pass ---------------------------------------------------------------------------------------
def _run_own(s):
    case, pool = s.case, s.pool
    if case["kind"] == "shared":
        n_q = case["n_q"]
        gate = {} if s.gate is None else {"gate_dev": s.gate.data_ptr(), "gate_seq_stride": n_q * HD, "gate_head_stride": HD}
        pool.decode_attn_shared(0, s.seqs, s.pos, s.entries, s.cells, n_q, s.q.data_ptr(), s.out.data_ptr(), SCALE, **gate)
        return s.out
    f16 = case["layout"] == "f16"
    if case["kind"] == "axes":
        pool.append_kprep_axes(0, s.seqs, s.pos, s.n_tok, s.k.data_ptr(), s.v.data_ptr(), s.gamma.data_ptr(), EPS, s.table.data_ptr(),
                               2 * s.pair_axis.size, s.table.shape[0], s.pair_axis, s.positions.data_ptr(), s.positions.shape[1])
        pool.read_rows(0, s.seqs, s.cell0, s.n_cells, s.k_out.data_ptr(), s.v_out.data_ptr(), f16_rows=f16)
        return s.k_out, s.v_out
    forks = [pool.seq_fork(seq, n) for seq, n in zip(s.seqs, s.length)]
    pool.seq_compact(forks, s.first_a, s.keep_a, s.lists.data_ptr(), *s.strides)
    if case["then"] == "attend":
        for layer in range(case["layers"]):
            pool.decode_attn(layer, forks, s.last, s.q.shape[2], s.q[layer].data_ptr(), s.out[layer].data_ptr(), SCALE)
        out = s.out
    else:
        for layer in range(case["layers"]):
            pool.read_rows(layer, forks, s.first_a, s.keep_a, s.k_out[layer].data_ptr(), s.v_out[layer].data_ptr(), f16_rows=f16)
        out = s.k_out, s.v_out
    for seq in forks:
        pool.seq_free(seq)
    return out


def _attend(q, k, v):
    """q [n_q, 256]; k, v [C, n_kv, 256] -> [n_q, 256]"""
    n_kv = k.shape[1]
    x = q.reshape(n_kv, -1, HD)
    out = []
    for h in range(n_kv):
        a = (x[h] @ k[:, h].t().contiguous()) * SCALE
        p = torch.exp(a - a.amax(-1, keepdim=True))
        out.append((p @ v[:, h].contiguous()) / p.sum(-1, keepdim=True))
    return torch.cat(out)


def _turned(x, gamma, table, positions, pairs):
    """RMSNorm and the rotary, in 64 bits with f32 between the two: what follows is a rounding to few bits, and values next to its
    borders must not cross them.  x [n, n_kv, 256], positions [axes, n]."""
    d = x.double()
    y = (d * (1.0 / torch.sqrt((d * d).sum(-1, keepdim=True) / HD + EPS)) * gamma.double()).float()
    half = len(pairs)
    a, b = y[..., :half].double(), y[..., half:2 * half].double()
    spots = positions.long()[torch.tensor(pairs, device=x.device)].t()                      # [n, half]
    turn = table[spots, torch.arange(half, device=x.device)].double()[:, None]              # [n, 1, half, 2]
    cos, sin = turn[..., 0], turn[..., 1]
    return torch.cat([(a * cos - b * sin).float(), (a * sin + b * cos).float(), y[..., 2 * half:]], -1)


def _picked(rows, lists, layer, at, m):
    """The listed cells of rows [cells, n_kv, 256], head by head."""
    n_kv = rows.shape[1]
    of = lists[min(layer, lists.shape[0] - 1), :, at:at + m].long()
    return torch.stack([rows[of[min(h, of.shape[0] - 1)], h] for h in range(n_kv)], 1)


def _run_plain(s):
    case = s.case
    layout = case["layout"]
    if case["kind"] == "shared":
        out, i = torch.empty_like(s.q), 0
        for (cells, members), (whole, tails) in zip(s.groups, s.caches):
            base = cells // PAGE * PAGE
            front = [_value(c, base) for c in whole]
            for m, tail in zip(members, tails):
                k, v = (torch.cat([f, _value(t, cells - base + m)]) for f, t in zip(front, tail))
                out[i] = _attend(s.q[i], k, v)
                i += 1
        return out if s.gate is None else out * (1.0 / (1.0 + torch.exp(-s.gate)))
    to = torch.float16 if layout == "f16" else torch.float32
    if case["kind"] == "axes":
        outs, at = ([], []), 0
        pairs = _ints(case["pairs"])
        for i, (p, t) in enumerate(zip(s.pos0, s.tokens)):
            kept = p - s.before[i]
            new = _turned(s.k[at:at + t], s.gamma, s.table, s.positions[:, at:at + t], pairs), s.v[at:at + t]
            at += t
            for rows, cache, out in zip(new, s.caches[i], outs):
                out.append(_value(_joined(layout, cache, kept, rows), kept + t))
        return tuple(torch.cat(o).to(to) for o in outs)
    rows_out = ([], [])
    attended = torch.empty_like(s.q) if case["then"] == "attend" else None
    for layer, caches in enumerate(s.caches):
        at = 0
        for i, (n, f, m) in enumerate(zip(s.length, s.first, s.keep)):
            pair = []
            for cache, out in zip(caches[i], rows_out):
                rows = _value(cache, n)
                page = f // PAGE * PAGE if layout == "e4m3" and m else f     # e4m3: the page it begins in is held anew
                new = torch.cat([rows[page:f], _picked(rows, s.lists, layer, at, m)])
                new = _value(_hold(layout, new), new.shape[0])
                out.append(new[f - page:])
                pair.append(torch.cat([rows[:page], new]))
            at += m
            if attended is not None:
                attended[layer, i] = _attend(s.q[layer, i], *pair)
    if attended is not None:
        return attended
    return tuple(torch.cat(o).reshape(case["layers"], -1, case["n_kv"], HD).to(to) for o in rows_out)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    n_kv, layout = case["n_kv"], case["layout"]
    row = 2 * n_kv * {"f16": 512, "i8": 272, "e4m3": 256}[layout]     # bytes of a cell in the cache, K and V
    plain = 2 * n_kv * HD * (2 if layout == "f16" else 4)              # of a cell as rows that are read back
    if case["kind"] == "shared":
        n_q, groups = case["n_q"], _groups(case)
        held = sum(c + sum(o) for c, o in groups)
        n = sum(len(o) for _, o in groups)
        pairs = sum(c * len(o) + sum(o) for c, o in groups)
        return {"bytes": held * row + n * (3 if case["gate"] else 2) * n_q * HD * 4, "flops": pairs * n_q * HD * 4}
    if case["kind"] == "axes":
        kept, new = sum(p % PAGE for p in _ints(case["pos0"])), sum(_ints(case["tokens"]))
        return {"bytes": new * 2 * n_kv * HD * 4 + ((2 if layout == "e4m3" else 1) * kept + 2 * new) * row + (kept + new) * plain, "flops": 0}
    first, keep, layers = _ints(case["first"]), _ints(case["keep"]), case["layers"]
    moved = sum(m + (f % PAGE if m else 0) for f, m in zip(first, keep))
    lists = 4 * sum(keep) * (layers * n_kv if case["lists"] == "own" else 1)
    if case["then"] == "rows":
        return {"bytes": layers * (2 * moved * row + sum(keep) * (row + plain)) + lists, "flops": 0}
    cells = sum(f + m for f, m in zip(first, keep))
    return {"bytes": layers * (2 * moved * row + cells * row + len(keep) * 2 * 8 * n_kv * HD * 4) + lists, "flops": layers * cells * 8 * n_kv * HD * 4}


# ---- the same in 64 bits ----------------------------------------------------------------------------
def _held64(layout, rows):
    """What a cache holds of rows [cells, n_kv, 256] from a page's first cell on, from the definitions."""
    x = rows.double()
    if layout == "f16":
        near = x.float().half().double()
        return torch.where(x.abs() < 2.0 ** -14, torch.zeros_like(near), near)
    if layout == "i8":
        blocks = x.unflatten(-1, (HD // 32, 32))
        largest = blocks.abs().max(-1, keepdim=True).values
        scale = (largest.float() / 127).half().double().clamp(min=2.0 ** -14)
        scale = torch.where(largest == 0, torch.ones_like(scale), scale)
        t = (blocks.float() / scale.float()).double().clamp(-127, 127)
        return (torch.trunc(t + torch.copysign(torch.full_like(t, 0.5), t)) * scale).flatten(-2)
    out = torch.empty_like(x)
    for at in range(0, x.shape[0], PAGE * 512):
        part = x[at:at + PAGE * 512]
        n = part.shape[0]
        pad = torch.zeros((n + PAGE - 1) // PAGE * PAGE, *part.shape[1:], dtype=x.dtype, device=x.device)
        pad[:n] = part
        page = pad.reshape(-1, PAGE, *part.shape[1:])
        largest = page.abs().amax(1).amax(-1)                     # [pages, n_kv]
        scale = torch.full_like(largest, 2.0 ** E_HI)
        for e in range(E_HI, E_LO - 1, -1):
            scale = torch.where(largest <= TOP * 2.0 ** e, torch.full_like(scale, 2.0 ** e), scale)
        y = (page / scale[:, None, :, None]).clamp(-TOP, TOP)
        step = torch.full_like(y, 2.0 ** -9)                      # below 2^-6, and in the lowest binade
        for b in range(-5, 9):
            step = torch.where(y.abs() >= 2.0 ** b, torch.full_like(step, 2.0 ** (b - 3)), step)
        y = torch.round(y / step) * step * scale[:, None, :, None]
        out[at:at + n] = y.reshape(pad.shape)[:n]
    return out


def _attend64(q, k, v):
    group = q.shape[0] // k.shape[1]
    out = torch.empty_like(q)
    for h in range(q.shape[0]):
        score = (k[:, h // group].contiguous() @ q[h]) / math.sqrt(HD)
        out[h] = torch.softmax(score, 0) @ v[:, h // group].contiguous()
    return out


def exact(case, seed):
    """The same in 64 bits over the same draws."""
    x = _inputs(case, seed)
    layout, n_kv = case["layout"], case["n_kv"]
    if case["kind"] == "shared":
        out, i = torch.empty(x.q.shape, dtype=torch.float64, device="cuda"), 0
        for (cells, members), prefix, tails in zip(x.groups, x.prefix, x.tails):
            base = cells - cells % PAGE
            once = [_held64(layout, r) for r in prefix]
            for m, tail in zip(members, tails):
                k, v = (torch.cat([c[:base], _held64(layout, torch.cat([c[base:], t.double()]))]) for c, t in zip(once, tail))
                out[i] = _attend64(x.q[i].double(), k, v)
                i += 1
        return out if x.gate is None else out * torch.sigmoid(x.gate.double())
    if case["kind"] == "axes":
        axis = torch.tensor(_ints(case["pairs"]), device="cuda")
        half, outs, at = axis.numel(), ([], []), 0
        for i, (p, t) in enumerate(zip(x.pos0, x.tokens)):
            k, v = x.k[at:at + t].double(), x.v[at:at + t].double()
            k = (k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * x.gamma.double()).float().double()   # the steps hand f32 on
            turn = torch.empty(t, half, dtype=torch.complex128, device="cuda")
            for j in range(half):
                turn[:, j] = torch.view_as_complex(x.table[x.positions[axis[j], at:at + t].long(), j].double())
            pair = torch.complex(k[..., :half], k[..., half:2 * half]) * turn[:, None]
            k = torch.cat([pair.real.float().double(), pair.imag.float().double(), k[..., 2 * half:]], -1)
            at += t
            for new, old, out in zip((k, v), x.held[i], outs):
                out.append(_held64(layout, torch.cat([_held64(layout, old), new])))
        return tuple(torch.cat(o) for o in outs)
    out_rows = ([], [])
    attended = torch.zeros(x.q.shape, dtype=torch.float64, device="cuda") if case["then"] == "attend" else None
    for layer in range(case["layers"]):
        at = 0
        for i, (f, m) in enumerate(zip(x.first, x.keep)):
            seen = []
            for side in range(2):
                had = _held64(layout, x.rows[layer][i][side])
                heads = []
                for h in range(n_kv):
                    ids = x.lists[layer if x.lists.shape[0] > 1 else 0, h if x.lists.shape[1] > 1 else 0, at:at + m].long()
                    heads.append(had[ids, h])
                now = torch.cat([had[:f], torch.stack(heads, 1)])
                if m and layout == "e4m3":
                    begin = f - f % PAGE
                    now = torch.cat([now[:begin], _held64(layout, now[begin:])])
                seen.append(now)
                out_rows[side].append(now[f:])
            at += m
            if attended is not None:
                attended[layer, i] = _attend64(x.q[layer, i].double(), *seen)
    if attended is not None:
        return attended
    return tuple(torch.cat(o).reshape(case["layers"], -1, n_kv, HD) for o in out_rows)
