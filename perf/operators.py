"""The operators of a cache held in e4m3 (BKV_LAYOUT_F8P), as they are measured: rows quantised on their way into the
cache, rows read back, attention of single tokens and of chunks over it.

Such a pool keeps one scale for every page of 16 cells, kv head and side (K or V), a power of two 2^e:

    e     the smallest of -32 .. 31 with which the page's largest finite value is at most 448 * 2^e (31 where none is)
    code  x * 2^-e, kept inside +-448, rounded to e4m3 (to nearest, ties to even)
    value code * 2^e

A row written into a page that holds rows already joins them: those below it are coded again under the scale of all.

A case is a dict of plain values.  `kind`:

  write   rows (f32 or f16; "kprep": K through RMSNorm and rotary first) behind what their first pages hold, then the
          pages written read back, in the rows' type
  read    whole sequences read back, as a step that hands a prefix to other code does
  decode  attention of one token of every sequence; with "blocks" over lists of 4-cell blocks
  chunk   causal attention of a chunk of every sequence, whose own rows are in the cache

With `own` the calls are those of breccia_amd.kv.Pool, without it the same in elementary torch operations in 32 bits.
"""
import math
import random

import numpy as np
import torch

own = False

HD, PAGE, BLOCK = 256, 16, 4            # head dim, cells of a page, cells of a selection block
EPS, N_ROT, FREQ = 1e-6, 64, 1e7        # the K preparation of the model
SCALE = 1.0 / 16.0
E_LO, E_HI, TOP = -32, 31, 448.0


def _text(values):
    return ",".join(str(int(v)) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")]


def _uniform(seed, n, lo, hi):
    r = random.Random(seed)
    return [r.randint(lo, hi) for _ in range(n)]


def _write(pos0, tokens, source="f32", n_kv=2):
    return dict(kind="write", source=source, n_kv=n_kv, pos0=_text(pos0), tokens=_text(tokens))


def _read(cells, rows="f16", n_kv=2):
    return dict(kind="read", rows=rows, n_kv=n_kv, cells=_text(cells))


def _decode(ctx, n_q=16, n_kv=2, gate=False, blocks=0):
    """ctx: cells each token sees, its own among them; blocks: length of its list, 0 for all cells."""
    return dict(kind="decode", n_q=n_q, n_kv=n_kv, gate=gate, blocks=blocks, ctx=_text(ctx))


def _chunk(prefix, tokens, n_q=16, n_kv=2, gate=False):
    return dict(kind="chunk", n_q=n_q, n_kv=n_kv, gate=gate, prefix=_text(prefix), tokens=_text(tokens))


def listed():
    named = [
        # the new rows of one decode step, one token of each of 32 conversations, anywhere in their pages
        ("write_tokens_b32", _write(_uniform(11, 32, 0, 511), [1] * 32)),
        # two prompts on their way into the cache with the model's K preparation
        ("write_prompts_kprep", _write([0, 0], [8191, 8191], "kprep")),
        # chunks of odd sizes at odd places from a producer that keeps f16
        ("write_ragged_f16", _write([1501, 37, 900, 16, 3], [333, 700, 1021, 17, 2], "f16", n_kv=4)),
        # three conversations handed to code that wants plain rows
        ("read_turns", _read([517, 41, 1333])),
        # a long document the same way
        ("read_long", _read([131072])),
        # four short conversations: launches and latency
        ("decode_short_b4", _decode([38, 513, 1001, 2049])),
        # eight sequences of 1k to 32k, the model's heads and output gate
        ("decode_mixed_b8", _decode(_uniform(3, 8, 1024, 32768), n_q=24, gate=True)),
        # long contexts, what a compressed cache is for
        ("decode_long_b16", _decode(_uniform(5, 16, 8192, 131072))),
        # the block selection's lists: 512 blocks and the token's own
        ("decode_lists_b8", _decode(_uniform(6, 8, 8192, 32768), n_q=24, gate=True, blocks=513)),
        # a short follow-up question in a conversation
        ("chunk_short", _chunk([517], [41])),
        # chunked prefill of four prompts
        ("chunk_4x1024", _chunk([1536] * 4, [1024] * 4)),
        # a whole prompt in one call, the model's heads and output gate
        ("chunk_prompt_4k", _chunk([0], [4096], n_q=24, gate=True)),
    ]
    return [dict(case, name=name) for name, case in named]


def _log(rng, lo, hi):
    """An integer of lo..hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["write", "write", "read", "decode", "decode", "decode", "lists", "chunk", "chunk", "chunk"])
    n_kv = rng.choice([2, 2, 2, 1, 4, 3])
    n_q = n_kv * rng.choice([8, 8, 12, 4, 16, 1] if n_kv < 3 else [8, 5, 4])
    gate = rng.random() < 0.5
    if kind == "write":
        n, total = _log(rng, 1, 64), _log(rng, 64, 32768 // n_kv)
        each = max(1, total // n)
        tokens = [max(1, each + rng.randint(-min(each // 2, 100), min(each // 2, 100))) for _ in range(n)]
        return _write([rng.choice([0, rng.randint(1, 2000)]) for _ in tokens], tokens, rng.choice(["f32", "f16", "kprep"]), n_kv)
    if kind == "read":
        n, total = _log(rng, 1, 64), _log(rng, 64, 131072 // n_kv)
        return _read([max(1, total // n + rng.randint(0, min(15, total // n))) for _ in range(n)], rng.choice(["f32", "f16"]), n_kv)
    if kind in ("decode", "lists"):
        lo = 2048 if kind == "lists" else 1
        hi = _log(rng, max(32, lo * 2), 131072)
        ctx = [_log(rng, max(lo, hi // 32), hi) for _ in range(_log(rng, 1, 64 if kind == "decode" else 16))]
        while sum(ctx) * n_kv > 1_600_000 and len(ctx) > 1:
            ctx.pop()
        return _decode(ctx, n_q, n_kv, gate, rng.choice([0, 0, 512, 513, 77])) if kind == "lists" else _decode(ctx, n_q, n_kv, gate)
    tokens = [_log(rng, 2, 4096) for _ in range(_log(rng, 1, 16))]
    prefix = [rng.choice([0, _log(rng, 1, 8192)]) for _ in tokens]
    pairs = [t * p + t * (t + 1) // 2 for t, p in zip(tokens, prefix)]
    while sum(pairs) * n_q > 180_000_000 and len(pairs) > 1:
        tokens.pop(), prefix.pop(), pairs.pop()
    if sum(pairs) * n_q > 180_000_000:
        tokens, prefix = [rng.randint(300, 1400)], [rng.randint(0, 2000)]
    return _chunk(prefix, tokens, n_q, n_kv, gate)


class _State:
    pool = None

    def __del__(self):
        if self.pool is not None:
            self.pool.destroy()


def _code(x):
    """Rows [pages, 16, n_kv, 256] (f32, 16 of a page) -> codes and the scales [pages, 1, n_kv, 1]."""
    a = x.abs().amax((1, 3), keepdim=True)
    m, e = torch.frexp(a)                        # a = m * 2^e, m of 1/2 .. 1
    e = torch.where(a > 0, e - 9 + (m > 0.875).to(e.dtype), E_LO).clamp(E_LO, E_HI)
    return (x * torch.exp2(-e.float())).clamp(-TOP, TOP).to(torch.float8_e4m3fn), torch.exp2(e.float())


def _pages(rows):
    """[cells, n_kv, 256] -> [pages, 16, n_kv, 256], the last page filled up with zeros."""
    n = rows.shape[0]
    full = (n + PAGE - 1) // PAGE * PAGE
    if full != n:
        rows = torch.cat([rows, rows.new_zeros(full - n, *rows.shape[1:])])
    return rows.reshape(-1, PAGE, *rows.shape[1:])


def _value(held, cells):
    codes, scales = held
    return (codes.float() * scales).reshape(-1, *codes.shape[2:])[:cells]


def _draws(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    return randn


def _rows(randn, n, n_kv, spread):
    """K and V of n cells.  Channels of K differ in size, a few by far; V's rows do, from token to token."""
    k = randn(n, n_kv, HD) * spread
    v = randn(n, n_kv, HD) * torch.exp(0.5 * randn(n, n_kv, 1))
    return k, v


def _spread(randn, n_kv):
    s = torch.exp(0.4 * randn(n_kv, HD))
    return torch.where(randn(n_kv, HD) > 2.0, 3.0 * s, s)


def _table(n, device):
    """cos and sin of the rotary's angles [n, N_ROT / 2, 2], worked out in 64 bits."""
    inv = torch.tensor([FREQ ** (-2.0 * i / N_ROT) for i in range(N_ROT // 2)], dtype=torch.float64, device=device)
    angle = torch.arange(n, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack([torch.cos(angle), torch.sin(angle)], -1).float().contiguous()


def _inputs(case, seed):
    """Everything a pass is given, in plain form: what the cache holds as f32 rows per sequence (`held`, from cell
    `first` on), and the inputs of the call."""
    randn = _draws(seed)
    kind, n_kv = case["kind"], case["n_kv"]
    x = _State()
    spread = _spread(randn, n_kv)
    if kind == "write":
        x.pos0, x.tokens = _ints(case["pos0"]), _ints(case["tokens"])
        x.first = [p // PAGE * PAGE for p in x.pos0]
        x.held = [_rows(randn, p - f, n_kv, spread) for p, f in zip(x.pos0, x.first)]
        x.k, x.v = _rows(randn, sum(x.tokens), n_kv, spread)
        if case["source"] == "f16":
            x.k, x.v = x.k.half(), x.v.half()
            x.k = torch.where(x.k.abs() < 2.0 ** -14, torch.zeros_like(x.k), x.k)   # a cache reads no f16 subnormals
            x.v = torch.where(x.v.abs() < 2.0 ** -14, torch.zeros_like(x.v), x.v)
        if case["source"] == "kprep":
            x.gamma = 1.0 + 0.1 * randn(HD)
            x.table = _table(max(p + t for p, t in zip(x.pos0, x.tokens)), "cuda")
        return x
    cells = _ints(case["cells"]) if kind == "read" else _ints(case["ctx"]) if kind == "decode" else \
        [p + t for p, t in zip(_ints(case["prefix"]), _ints(case["tokens"]))]
    x.cells, x.first = cells, [0] * len(cells)
    x.held = [_rows(randn, n, n_kv, spread) for n in cells]
    if kind == "read":
        return x
    x.tokens = [1] * len(cells) if kind == "decode" else _ints(case["tokens"])
    x.pos0 = [n - t for n, t in zip(cells, x.tokens)]
    total = sum(x.tokens)
    x.q = randn(total, case["n_q"], HD)
    x.gate = randn(total, case["n_q"], HD) if case["gate"] else None
    if kind == "decode" and case["blocks"]:
        most = case["blocks"]
        x.ids = torch.zeros(total, most, dtype=torch.int32, device="cuda")
        counts = []
        for i, n in enumerate(cells):
            last = (n - 1) // BLOCK
            pick = torch.randperm(last, generator=torch.Generator().manual_seed(seed * 1000 + i))[:most - 1]
            pick = torch.cat([pick.sort().values, torch.tensor([last])]).int()
            x.ids[i, :pick.numel()] = pick.cuda()
            counts.append(pick.numel())
        x.listed = counts
        x.counts = torch.tensor(counts, dtype=torch.int32, device="cuda")
    return x


def prepare(case, seed):
    s = _inputs(case, seed)
    s.case = case
    held, s.held = s.held, None
    n_kv = case["n_kv"]
    if not own:
        # the cache: codes and scales of every page
        s.cache = [tuple(_code(_pages(r)) for r in pair) for pair in held]
        torch.cuda.synchronize()
        return s
    from breccia_amd import lib as L
    from breccia_amd.kv import Pool

    # cells each sequence holds once the pass is over
    ends = [p + t for p, t in zip(s.pos0, s.tokens)] if case["kind"] == "write" else s.cells
    pages = [(e + PAGE - 1) // PAGE for e in ends]
    n_pages = int(sum(pages) / 0.6) + 1
    pool = s.pool = Pool(n_layers=1, n_pages=n_pages, n_kv_head=n_kv, head_dim=HD, layout=L.LAYOUT_F8P, max_seqs=len(ends),
                         max_pages_per_seq=max(pages))
    pool.set_free_order(np.random.RandomState(seed).permutation(n_pages).astype(np.int32))
    s.seqs = np.array([pool.seq_create() for _ in ends], dtype=np.int32)
    for seq, end, first, (k, v) in zip(s.seqs.tolist(), ends, s.first, held):
        pool.seq_reserve(seq, end)
        if k.shape[0]:
            pool.append(0, [seq], [first], [k.shape[0]], k.data_ptr(), v.data_ptr())
    if case["kind"] in ("write", "read"):
        s.cell0 = np.array(s.first, dtype=np.int64)
        s.n_cells = np.array([e - f for e, f in zip(ends, s.first)], dtype=np.int32)
        wanted = torch.float16 if case.get("rows", case.get("source")) == "f16" else torch.float32
        s.k_out, s.v_out = (torch.zeros(int(s.n_cells.sum()), n_kv, HD, dtype=wanted, device="cuda") for _ in range(2))
    else:
        s.out = torch.zeros_like(s.q)
    if case["kind"] != "read":
        s.pos = np.array(s.pos0, dtype=np.int64)
        s.n_tok = np.array(s.tokens, dtype=np.int32)
    torch.cuda.synchronize()
    return s


def _run_own(s):
    case, pool = s.case, s.pool
    kind = case["kind"]
    if kind in ("write", "read"):
        if kind == "write":
            k, v = s.k.data_ptr(), s.v.data_ptr()
            if case["source"] == "kprep":
                pool.append_kprep(0, s.seqs, s.pos, s.n_tok, k, v, s.gamma.data_ptr(), EPS, s.table.data_ptr(), N_ROT,
                                  s.table.shape[0])
            else:
                pool.append(0, s.seqs, s.pos, s.n_tok, k, v, f16_rows=case["source"] == "f16")
        pool.read_rows(0, s.seqs, s.cell0, s.n_cells, s.k_out.data_ptr(), s.v_out.data_ptr(),
                       f16_rows=s.k_out.dtype == torch.float16)
        return s.k_out, s.v_out
    n_q, q, out = case["n_q"], s.q.data_ptr(), s.out.data_ptr()
    gate = {}
    if s.gate is not None:
        gate = {"gate_dev": s.gate.data_ptr(), "gate_head_stride": HD,
                "gate_tok_stride" if kind == "chunk" else "gate_seq_stride": n_q * HD}
    if kind == "chunk":
        pool.prefill_attn(0, s.seqs, s.pos, s.n_tok, n_q, q, out, SCALE, **gate)
    elif case["blocks"]:
        pool.decode_attn_select(0, s.seqs, s.pos, n_q, q, out, SCALE, s.ids.data_ptr(), case["blocks"], s.counts.data_ptr(),
                                case["blocks"], **gate)
    else:
        pool.decode_attn(0, s.seqs, s.pos, n_q, q, out, SCALE, **gate)
    return s.out


def _prepared(x, gamma, table):
    """RMSNorm and the rotary of the first N_ROT values, in 64 bits with f32 between the two: what follows is a rounding
    to 4 bits, and values next to its borders must not cross them.  x [n, n_kv, 256], table [n, N_ROT / 2, 2]."""
    d = x.double()
    y = (d * (1.0 / torch.sqrt((d * d).sum(-1, keepdim=True) / HD + EPS)) * gamma.double()).float()
    half = N_ROT // 2
    a, b = y[..., :half].double(), y[..., half:N_ROT].double()
    cos, sin = table[:, None, :, 0].double(), table[:, None, :, 1].double()
    return torch.cat([(a * cos - b * sin).float(), (a * sin + b * cos).float(), y[..., N_ROT:]], -1)


def _attend(q, k, v, pos):
    """q [T, n_q, 256]; k, v [C, n_kv, 256]; row t sees cells 0 .. pos + t, or all (pos None)."""
    tokens, n_q = q.shape[:2]
    n_kv = k.shape[1]
    group = n_q // n_kv
    out = torch.empty_like(q)
    for h in range(n_kv):
        keys, values = k[:, h].t().contiguous(), v[:, h].contiguous()
        step = max(1, (1 << 28) // (keys.shape[1] * group))
        for t in range(0, tokens, step):
            rows = q[t:t + step, h * group:(h + 1) * group]
            n = rows.shape[0]
            s = (rows.reshape(-1, HD) @ keys) * SCALE
            if pos is not None:
                cell = torch.arange(keys.shape[1], device=q.device)
                last = torch.arange(pos + t, pos + t + n, device=q.device).repeat_interleave(group)
                s = s.masked_fill(cell[None, :] > last[:, None], float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = (p @ values) / p.sum(-1, keepdim=True)
            out[t:t + n, h * group:(h + 1) * group] = o.reshape(n, group, HD)
    return out


def _cells_of(ids, ctx):
    cells = (ids[:, None] * BLOCK + torch.arange(BLOCK, device=ids.device)).reshape(-1)
    return cells[cells < ctx]


def _run_plain(s):
    case = s.case
    kind = case["kind"]
    if kind == "write":
        outs, at = ([], []), 0
        for i, (p, t) in enumerate(zip(s.pos0, s.tokens)):
            kept = p - s.first[i]
            new = [s.k[at:at + t].float(), s.v[at:at + t].float()]
            if case["source"] == "kprep":
                new[0] = _prepared(new[0], s.gamma, s.table[p:p + t])
            at += t
            for rows, cache, out in zip(new, s.cache[i], outs):
                out.append(_value(_code(_pages(torch.cat([_value(cache, kept), rows]))), kept + t))
        return tuple(torch.cat(o).to(s.k.dtype) for o in outs)
    if kind == "read":
        to = torch.float16 if case["rows"] == "f16" else torch.float32
        return tuple(torch.cat([_value(c[j], n) for c, n in zip(s.cache, s.cells)]).to(to) for j in range(2))
    out, at = torch.empty_like(s.q), 0
    for i, (n, t) in enumerate(zip(s.cells, s.tokens)):
        k, v = (_value(c, n) for c in s.cache[i])
        if case.get("blocks"):
            cells = _cells_of(s.ids[i, :s.listed[i]].long(), n)
            k, v = k[cells], v[cells]
        out[at:at + t] = _attend(s.q[at:at + t], k, v, s.pos0[i] if kind == "chunk" else None)
        at += t
    return out if s.gate is None else out * (1.0 / (1.0 + torch.exp(-s.gate)))


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    kind, n_kv = case["kind"], case["n_kv"]
    row = 2 * n_kv * HD     # bytes of a cell in the cache, K and V
    if kind == "write":
        size = 2 if case["source"] == "f16" else 4
        kept, new = sum(p % PAGE for p in _ints(case["pos0"])), sum(_ints(case["tokens"]))
        return {"bytes": row * (kept + new * size + (kept + new) * (1 + size)), "flops": 0}
    if kind == "read":
        return {"bytes": sum(_ints(case["cells"])) * row * (3 if case["rows"] == "f16" else 5), "flops": 0}
    n_q = case["n_q"]
    token = (3 if case["gate"] else 2) * n_q * HD * 4   # q, out, gate
    if kind == "chunk":
        prefix, tokens = _ints(case["prefix"]), _ints(case["tokens"])
        pairs = sum(t * p + t * (t + 1) // 2 for t, p in zip(tokens, prefix))
        return {"bytes": sum(tokens) * token + sum(p + t for t, p in zip(tokens, prefix)) * row, "flops": pairs * n_q * HD * 4}
    cells = _ints(case["ctx"])
    n, lists = len(cells), 0
    if case["blocks"]:
        cells = [min(c, case["blocks"] * BLOCK) for c in cells]
        lists = sum((c + BLOCK - 1) // BLOCK * 4 for c in cells)
    return {"bytes": sum(cells) * row + n * token + lists, "flops": sum(cells) * n_q * HD * 4}


def _held64(rows):
    """What a cache holds of rows [cells, n_kv, 256], from the definition: the scale found by trying every e, the codes
    by rounding to a whole number of steps of the value's binade."""
    x = rows.double()
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


def exact(case, seed):
    """The same in 64 bits over the same draws."""
    x = _inputs(case, seed)
    kind, n_kv = case["kind"], case["n_kv"]
    if kind == "write":
        outs, at = ([], []), 0
        for i, (p, t) in enumerate(zip(x.pos0, x.tokens)):
            k, v = x.k[at:at + t].double(), x.v[at:at + t].double()
            at += t
            if case["source"] == "kprep":
                # the operator's steps hand f32 on
                k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * x.gamma.double()
                k = k.float().double()
                turn = torch.view_as_complex(x.table[p:p + t].double())[:, None, :]
                pair = torch.complex(k[..., :N_ROT // 2], k[..., N_ROT // 2:N_ROT]) * turn
                k = torch.cat([pair.real.float().double(), pair.imag.float().double(), k[..., N_ROT:]], -1)
            for new, old, out in zip((k, v), x.held[i], outs):
                out.append(_held64(torch.cat([_held64(old), new])))
        return tuple(torch.cat(o) for o in outs)
    if kind == "read":
        return tuple(torch.cat([_held64(pair[j]) for pair in x.held]) for j in range(2))
    out, at = torch.empty(x.q.shape, dtype=torch.float64, device="cuda"), 0
    for i, (n, t) in enumerate(zip(x.cells, x.tokens)):
        k, v = (_held64(r) for r in x.held[i])
        x.held[i] = None
        if case.get("blocks"):
            seen = _cells_of(x.ids[i, :x.listed[i]].long(), n)
            k, v = k[seen], v[seen]
        group = case["n_q"] // n_kv
        for r in range(0, t, 128):
            m = min(128, t - r)
            for h in range(case["n_q"]):
                score = (x.q[at + r:at + r + m, h].double() @ k[:, h // group].t().contiguous()) / math.sqrt(HD)
                if kind == "chunk":
                    dead = torch.arange(n, device="cuda")[None] > torch.arange(x.pos0[i] + r, x.pos0[i] + r + m, device="cuda")[:, None]
                    score[dead] = -math.inf
                out[at + r:at + r + m, h] = torch.softmax(score, -1) @ v[:, h // group].contiguous()
        at += t
    return out if x.gate is None else out * torch.sigmoid(x.gate.double())
