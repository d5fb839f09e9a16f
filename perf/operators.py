"""What is measured of the paged-cache operators: appending rows (query / key
norms, rotation, 16- or 4-bit storage), attention with a window and sinks over
a 16-bit cache, attention over a 4-bit cache, and forking / compacting pages.

`own` selects the framework's kernels (`fmd_b200.PagedCache`); otherwise the
operators are computed in plain torch operations in 32 bits.

Storage, as `PagedCache` documents it. A page holds 64 positions. 16 bits:
[layer][page][k|v][kv head][64][dim]. 4 bits: per (layer, page, k|v, kv head)
64 rows of dim / 2 code bytes, then 64 rows of dim / 32 f16 scales; a value is
(code - 8) * scale of its block of 32 dims. Code bytes of a key row: four
chunks c of dim / 8 bytes, in chunk c one little-endian 32-bit word per block
g holding dims 32 g + 8 c + e, e = 0..7, nibble (e >> 1) + 4 (e & 1). Code
bytes of a value row: 32-bit words w holding dims 8 w + e with nibble e.
"""

import importlib
import math
import random

import torch

own = False

PAGE = 64
EPS = 1e-6
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- cases -----------------------------------------------------------------------


def listed():
    dec = dict(heads=16, kv_heads=8, dim=128)
    return [
        # one live transcription: its next token's row goes into the cache
        dict(name="append_one", op="append", kind="bf16", dtype="bf16", seqs=1, rows=1, ctx=2311, rot=128,
             inter=False, **dec),
        # a decode step of a full batch, keys already normed and rotated, 4-bit cache
        dict(name="append_batch_q4", op="append", kind="q4", dtype="bf16", seqs=64, rows=64, ctx=4300, rot=0,
             inter=False, **dec),
        # prompts of three requests in one pass (odd lengths), norm and rotation fused
        dict(name="append_prompts", op="append", kind="bf16", dtype="bf16", seqs=3, rows=10007, ctx=0, rot=128,
             inter=False, **dec),
        # the same into a 4-bit cache, f16
        dict(name="append_prompts_q4", op="append", kind="q4", dtype="f16", seqs=4, rows=16384, ctx=100, rot=0,
             inter=False, **dec),
        # one stream far into a long recording: only the window and the sinks are read
        dict(name="window_one", op="attend", kind="bf16", dtype="bf16", seqs=1, chunk=1, lo=16001, hi=16001,
             window=4096, sinks=4, **dec),
        # a batch of streams, contexts 300 .. 16k, f16
        dict(name="window_batch", op="attend", kind="f16", dtype="f16", seqs=64, chunk=1, lo=300, hi=16384,
             window=2048, sinks=64, **dec),
        # two prompt chunks of 2,048 rows behind long histories
        dict(name="window_chunks", op="attend", kind="bf16", dtype="bf16", seqs=2, chunk=2048, lo=6000, hi=14336,
             window=4096, sinks=4, **dec),
        # one long recording decoded from a 4-bit cache
        dict(name="q4_one", op="attend", kind="q4", dtype="bf16", seqs=1, chunk=1, lo=16384, hi=16384, window=0,
             sinks=0, **dec),
        # the 64-sequence decode step over 4-bit caches, contexts 300 .. 16k
        dict(name="q4_batch", op="attend", kind="q4", dtype="bf16", seqs=64, chunk=1, lo=300, hi=16384, window=0,
             sinks=0, **dec),
        # a prompt chunk over a 4-bit cache (odd chunk and history), f16
        dict(name="q4_chunk", op="attend", kind="q4", dtype="f16", seqs=1, chunk=2001, lo=9001, hi=9001, window=0,
             sinks=0, **dec),
        # eight hypotheses forked from one prompt in the middle of a page, every layer of the model
        dict(name="fork", op="fork", kind="bf16", dtype="bf16", layers=28, kv_heads=8, dim=128, length=2311,
             children=8),
        # a fragmented 4-bit pool made dense again
        dict(name="compact", op="compact", kind="q4", dtype="bf16", layers=28, kv_heads=8, dim=128, pages=1500,
             slots=48, used=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "window", "window", "q4", "q4", "fork", "compact"])
    dim = rng.choice([128, 128, 64])
    kv_heads = rng.randint(1, 8)
    if op == "append":
        q4 = rng.random() < 0.5
        dtype = rng.choice(["bf16", "f16"])
        seqs = _log(rng, 1, 64)
        return dict(op="append", kind="q4" if q4 else dtype, dtype=dtype, heads=kv_heads * rng.choice([1, 2, 4]),
                    kv_heads=kv_heads, dim=dim, seqs=seqs, rows=seqs * _log(rng, 1, max(2, 8000 // seqs)),
                    ctx=rng.randint(0, 3000), rot=0 if q4 else rng.choice([dim, dim // 2]),
                    inter=not q4 and rng.random() < 0.5)
    if op in ("window", "q4"):
        dtype = rng.choice(["bf16", "f16"])
        chunk = 1 if rng.random() < 0.6 else _log(rng, 2, 1000)
        group = rng.choice([1, 2, 2, 4, 8]) if chunk == 1 else rng.choice([1, 2, 2, 4])
        seqs = _log(rng, 1, 64) if chunk == 1 else _log(rng, 1, max(2, min(8, 1000 // chunk)))
        lo = _log(rng, 1, 4000) + chunk - 1
        hi = lo + (_log(rng, 1, 12000) if chunk == 1 else _log(rng, 1, 5000))
        window = _log(rng, 1, 4096) if op == "window" or rng.random() < 0.3 else 0
        return dict(op="attend", kind="q4" if op == "q4" else dtype, dtype=dtype, heads=kv_heads * group,
                    kv_heads=kv_heads, dim=dim, seqs=seqs, chunk=chunk, lo=lo, hi=hi, window=window,
                    sinks=rng.choice([0, 1, 4, 64, 100]) if window else 0)
    kind = rng.choice(["bf16", "f16", "q4"])
    if op == "fork":
        return dict(op="fork", kind=kind, dtype="bf16", layers=rng.randint(1, 28), kv_heads=kv_heads, dim=dim,
                    length=_log(rng, 1, 6000), children=_log(rng, 1, 32))
    return dict(op="compact", kind=kind, dtype="bf16", layers=rng.randint(1, 16), kv_heads=kv_heads, dim=dim,
                pages=_log(rng, 20, 700), slots=_log(rng, 1, 64), used=rng.uniform(0.2, 0.95))


# ---- sizes of a case (from its own numbers, not from the seed) -------------------


def _shapes(case):
    """Rows of each sequence and the position of its first row."""
    r = random.Random("%(seqs)d %(kv_heads)d %(dim)d" % case)
    n = case["seqs"]
    if case["op"] == "append":
        cuts = sorted(r.sample(range(1, case["rows"]), n - 1)) if n > 1 else []
        if case["rows"] == n:
            cuts = list(range(1, n))
        counts = [b - a for a, b in zip([0] + cuts, cuts + [case["rows"]])]
        starts = [r.randint(0, 2 * case["ctx"]) if n > 1 else case["ctx"] for _ in range(n)]
        return counts, starts
    total = [_log(r, case["lo"], case["hi"]) for _ in range(n)]
    if n > 1:
        total[0], total[-1] = case["lo"], case["hi"]
    return [case["chunk"]] * n, [t - case["chunk"] for t in total]


def _block_bytes(case):
    """Bytes of one (layer, page, k|v, kv head) block."""
    return PAGE * case["dim"] * 2 if case["kind"] != "q4" else PAGE * (case["dim"] // 2 + case["dim"] // 16)


def _visible(case, pos):
    """Keys that a row at `pos` sees."""
    w, s = case["window"], case["sinks"]
    return pos + 1 if w == 0 else min(w, pos + 1) + min(s, max(0, pos + 1 - w))


def _union(case, start, count):
    """Keys that any row of a chunk sees."""
    w, s = case["window"], case["sinks"]
    end = start + count
    first = max(0, start - w + 1) if w else 0
    return end - first + min(s, first)


def work(case):
    if case["op"] == "append":
        rows, d, hq, hkv = case["rows"], case["dim"], case["heads"], case["kv_heads"]
        byts = 2 * rows * (hq + 2 * hkv) * d + rows * 2 * hkv * _block_bytes(case) // PAGE
        if case["rot"]:
            byts += 2 * rows * hq * d + 4 * rows * case["rot"]
        if case["kind"] == "q4":  # the rows read back
            byts += rows * 2 * hkv * (_block_bytes(case) // PAGE + 4 * d)
        return {"bytes": byts, "flops": rows * (hq + 2 * hkv) * d * 6}
    if case["op"] == "attend":
        counts, starts = _shapes(case)
        keys = sum(_union(case, a, n) for n, a in zip(counts, starts))
        pairs = sum(sum(_visible(case, a + i) for i in range(n)) for n, a in zip(counts, starts))
        d = case["dim"]
        byts = keys * 2 * case["kv_heads"] * _block_bytes(case) // PAGE + 2 * 2 * sum(counts) * case["heads"] * d
        return {"bytes": byts, "flops": 4 * d * case["heads"] * pairs}
    per_row = case["layers"] * 2 * case["kv_heads"] * _block_bytes(case) // PAGE
    if case["op"] == "fork":
        n = case["children"]
        full = case["length"] // PAGE
        return {"bytes": (n + 1) * (case["length"] % PAGE) * per_row + 4 * (n + 1) * (full + 1), "flops": 0}
    table, n_used = _fragmented(case)
    moved = len({p for row in table for p in row if p >= n_used})
    entries = sum(len(row) for row in table)
    return {"bytes": 2 * moved * PAGE * per_row + 8 * entries, "flops": 0}


def _fragmented(case):
    """Page tables of a pool after many requests came and went: scattered pages,
    some shared by two slots. Returns (pages of each slot, pages in use)."""
    r = random.Random("%(pages)d %(slots)d" % case)
    pages = r.sample(range(case["pages"]), max(1, int(case["pages"] * case["used"])))
    table = [[] for _ in range(case["slots"])]
    for p in pages:
        table[r.randrange(case["slots"])].append(p)
    for s in range(1, case["slots"], 7):  # forked slots: a shared prefix
        table[s] = table[s - 1][: len(table[s - 1]) // 2] + table[s]
    return table, len(pages)


# ---- plain storage ------------------------------------------------------------------


def _code_order(dim, value):
    """Dim of each nibble of a row, in byte order (low nibble first)."""
    dims = torch.empty(dim // 8, 8, dtype=torch.long)
    for w in range(dim // 8):
        for e in range(8):
            if value:
                dims[w, e] = 8 * w + e
            else:
                c, g = divmod(w, dim // 32)
                dims[w, (e >> 1) + 4 * (e & 1)] = 32 * g + 8 * c + e
    return dims.reshape(-1)


def _quantise(x):
    """f32 (..., dim) -> codes (..., dim), f16 scales (..., dim / 32)."""
    b = x.float().unflatten(-1, (-1, 32))
    i = b.abs().argmax(-1, keepdim=True)
    m = torch.gather(b, -1, i)
    code = torch.floor(-8 * b / torch.where(m == 0, 1.0, m) + 8.5).clamp(0, 15)
    return code.flatten(-2).to(torch.uint8), (m.squeeze(-1) / -8).half()


class _Plain:
    """The pool as torch tensors: the plain form's way to it."""

    def __init__(self, case, pool, layers, pages):
        self.q4 = case["kind"] == "q4"
        self.dim = case["dim"]
        d, h = case["dim"], case["kv_heads"]
        if not self.q4:
            self.rows16 = pool.view(DT[case["kind"]]).view(layers, pages, 2, h, PAGE, d)
        else:
            blk = pool.view(layers, pages, 2, h, _block_bytes(case))
            self.codes = blk[..., : PAGE * d // 2].unflatten(-1, (PAGE, d // 2))
            self.scales = blk[..., PAGE * d // 2:].view(torch.float16).unflatten(-1, (PAGE, d // 32))
            order = [_code_order(d, v).to(pool.device) for v in (False, True)]
            self.order = order
            self.inverse = [torch.argsort(o) for o in order]

    def write(self, layer, pages, offs, kv, x):
        if not self.q4:
            self.rows16[layer, pages, kv, :, offs] = x.to(self.rows16.dtype)
            return
        code, scale = _quantise(x)
        n = code[..., self.order[kv]].unflatten(-1, (-1, 2))
        self.codes[layer, pages, kv, :, offs] = n[..., 0] | (n[..., 1] << 4)
        self.scales[layer, pages, kv, :, offs] = scale

    def read(self, layer, pages, offs, kv, dtype=torch.float32):
        """(n, kv heads, dim) values of the given positions."""
        if not self.q4:
            return self.rows16[layer, pages, kv, :, offs].to(dtype)
        c = self.codes[layer, pages, kv, :, offs]
        n = torch.stack([c & 15, c >> 4], -1).flatten(-2)[..., self.inverse[kv]]
        s = self.scales[layer, pages, kv, :, offs].to(dtype)
        return ((n.to(dtype) - 8).unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


# ---- inputs --------------------------------------------------------------------------


def _cache(state):
    """The framework's cache over the state's pool and page table."""
    pkg = importlib.import_module("__graft_entry__").load_package()
    case = state["case"]
    return pkg.PagedCache(layers=state["layers"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                          n_pages=state["pages"], max_slots=state["table"].shape[0],
                          max_pages_per_slot=state["table"].shape[1], kind=case["kind"], pool=state["pool"],
                          page_table=state["table"], slots=state["slots"])


def _new_state(case, gen, tables, lengths, layers, n_pages, max_pages=None):
    dev = gen.device
    width = max_pages or max(len(t) for t in tables)
    host = torch.zeros(len(tables), width, dtype=torch.int32)
    for i, t in enumerate(tables):
        host[i, : len(t)] = torch.tensor(t, dtype=torch.int32)
    pool = torch.zeros(layers * n_pages * 2 * case["kv_heads"] * _block_bytes(case), dtype=torch.uint8, device=dev)
    state = dict(case=case, layers=layers, pages=n_pages, pool=pool, table=host.to(dev),
                 slots=[(i, list(t), n) for i, (t, n) in enumerate(zip(tables, lengths)) if t], tables=tables)
    state["plain"] = _Plain(case, pool, layers, n_pages)
    return state


def _fill(state, gen):
    """Random keys and values of every page: normed keys, plain values. Pages
    of a 4-bit pool that are only moved hold any bytes."""
    case, p = state["case"], state["plain"]
    if p.q4 and case["op"] != "attend":
        state["pool"].random_(0, 256, generator=gen)
        return
    for layer in range(state["layers"]):
        for a in range(0, state["pages"], 256):
            pages = torch.arange(a, min(a + 256, state["pages"]), device=gen.device).repeat_interleave(PAGE)
            offs = torch.arange(PAGE, device=gen.device).repeat(len(pages) // PAGE)
            for kv in range(2):
                x = torch.randn(len(pages), case["kv_heads"], case["dim"], generator=gen, device=gen.device)
                p.write(layer, pages, offs, kv, x.to(DT[case["dtype"]]))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    if case["op"] in ("append", "attend"):
        counts, starts = _shapes(case)
        need = [-(-(a + n) // PAGE) for n, a in zip(counts, starts)]
        n_pages = sum(need) + 3
        ids = torch.randperm(n_pages, generator=gen, device=dev).tolist()
        tables = [[ids.pop() for _ in range(k)] for k in need]
        state = _new_state(case, gen, tables, [a + n for n, a in zip(counts, starts)], 1, n_pages)
        rows = sum(counts)
        dt = DT[case["dtype"]]
        state["row0"] = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(dev)
        state["pos0"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        state["slot"] = torch.arange(len(counts), dtype=torch.int32, device=dev)
        state["max_rows"] = max(counts)
        seq = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)).to(dev)
        pos = torch.cat([torch.arange(a, a + n) for n, a in zip(counts, starts)]).to(dev)
        state["pos"] = pos
        state["page"] = state["table"][seq, pos // PAGE].long()
        state["off"] = pos % PAGE
        if case["op"] == "attend":
            _fill(state, gen)
            state["q"] = torch.randn(rows, case["heads"], case["dim"], generator=gen, device=dev).to(dt)
            state["out"] = torch.empty_like(state["q"])
        else:
            # one fused projection's output: q, k and v are strided views of it
            hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
            x = torch.randn(rows, hq + 2 * hkv, d, generator=gen, device=dev).to(dt)
            state["q"], state["k"], state["v"] = x[:, :hq], x[:, hq: hq + hkv], x[:, hq + hkv:]
            if case["rot"]:
                half = case["rot"] // 2
                inv = 1.0 / 1e6 ** (torch.arange(half, device=dev, dtype=torch.float64) / half)
                ang = torch.arange(int(pos.max()) + 1, device=dev, dtype=torch.float64)[:, None] * inv
                state["cos"], state["sin"] = ang.cos().float(), ang.sin().float()
                state["qw"], state["kw"] = (
                    (1 + 0.1 * torch.randn(d, generator=gen, device=dev)).to(dt) for _ in range(2))
                state["q_out"] = torch.empty(rows, hq, d, dtype=dt, device=dev)
            else:
                state["k_val"] = torch.empty(rows, hkv, d, dtype=torch.float32, device=dev)
                state["v_val"] = torch.empty_like(state["k_val"])
    elif case["op"] == "fork":
        n, full = case["children"], -(-case["length"] // PAGE)
        n_pages = full + n + 2
        ids = torch.randperm(full + 2, generator=gen, device=dev).tolist()[:full]
        state = _new_state(case, gen, [ids] + [[]] * n, [case["length"]] + [0] * n, case["layers"], n_pages,
                           max_pages=full + 4)
        _fill(state, gen)
        free = sorted(set(range(n_pages)) - set(ids))
        state["fresh"] = free[:n]  # the lowest free pages, in the children's order
    else:
        tables, n_used = _fragmented(case)
        state = _new_state(case, gen, tables, [len(t) * PAGE for t in tables], case["layers"], case["pages"])
        _fill(state, gen)
        state["before"] = state["table"].clone()
        state["counts"] = torch.tensor([len(t) for t in tables], dtype=torch.int32, device=dev)
        state["n_used"] = n_used
    state["own"] = _cache(state) if own else None
    return state


# ---- one pass ------------------------------------------------------------------------


def run(state):
    if own:
        if state["own"] is None:
            state["own"] = _cache(state)
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "fork": _plain_fork,
            "compact": _plain_compact}[state["case"]["op"]](state)


def _run_own(state):
    case, cache = state["case"], state["own"]
    if case["op"] == "compact":
        # the same fragmented tables every pass
        state["table"].copy_(state["before"])
        n = cache.compact_tables(state["table"], state["counts"])
        return {"table": state["table"], "pool": _values(state), "used": n}
    if case["op"] == "fork":
        children = list(range(1, case["children"] + 1))
        cache.fork(0, children)
        cache.release(*children)
        return {"table": state["table"], "pool": _values(state)}
    rows = state.get("rows")
    if rows is None:
        rows = state["rows"] = cache.rows(state["slot"], state["pos0"],
                                          state["row0"] if state["max_rows"] > 1 else None, state["max_rows"])
    if case["op"] == "attend":
        return cache.attend(0, rows, state["q"], window=case["window"], sinks=case["sinks"], out=state["out"])
    if case["rot"]:
        q = cache.append(0, rows, state["k"], state["v"], q=state["q"], q_norm=state["qw"], k_norm=state["kw"],
                         eps=EPS, cos=state["cos"], sin=state["sin"], interleaved=case["inter"],
                         q_out=state["q_out"])
        return {"q": q, "pool": _values(state)}
    cache.append(0, rows, state["k"], state["v"])
    if case["kind"] == "q4":
        k, v = cache.read(0, rows, k_out=state["k_val"], v_out=state["v_val"])
        return {"k": k, "v": v}
    return {"pool": _values(state)}


def _values(state):
    """The pool itself; a 4-bit pool is only moved about: its bytes."""
    return state["pool"] if state["case"]["kind"] == "q4" else state["plain"].rows16


def _plain_norm_rotate(x, w, cos, sin, inter):
    x = x.float()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    r, rest = x[..., : 2 * half], x[..., 2 * half:]
    if inter:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., :half], r[..., half:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, rest], -1)


def _plain_append(state):
    case, p = state["case"], state["plain"]
    q, k, v = state["q"], state["k"], state["v"]
    if case["rot"]:
        cos, sin = state["cos"][state["pos"]], state["sin"][state["pos"]]
        q = _plain_norm_rotate(q, state["qw"], cos, sin, case["inter"]).to(q.dtype)
        k = _plain_norm_rotate(k, state["kw"], cos, sin, case["inter"])
    p.write(0, state["page"], state["off"], 0, k)
    p.write(0, state["page"], state["off"], 1, v)
    if case["rot"]:
        return {"q": q, "pool": _values(state)}
    if case["kind"] == "q4":
        return {"k": p.read(0, state["page"], state["off"], 0), "v": p.read(0, state["page"], state["off"], 1)}
    return {"pool": _values(state)}


def _plain_attend(state):
    case, p = state["case"], state["plain"]
    q, out = state["q"], torch.empty_like(state["out"])
    group = case["heads"] // case["kv_heads"]
    scale = case["dim"] ** -0.5
    counts, starts = _shapes(case)
    w, s = case["window"], case["sinks"]
    r = 0
    for i, (n, a) in enumerate(zip(counts, starts)):
        key = torch.arange(a + n, device=q.device)
        if w:  # only keys that some row sees
            key = key[(key > a - w) | (key < s)]
        page, off = state["table"][i][key // PAGE].long(), key % PAGE
        k, v = p.read(0, page, off, 0), p.read(0, page, off, 1)
        row = torch.arange(a, a + n, device=q.device)[:, None]
        seen = key <= row
        if w:
            seen &= (key > row - w) | (key < s)
        for h in range(case["kv_heads"]):
            qh = q[r: r + n, h * group: (h + 1) * group].float().transpose(0, 1)
            x = (qh @ k[:, h].T * scale).masked_fill(~seen, -math.inf)
            x = torch.exp(x - x.amax(-1, keepdim=True))
            o = x @ v[:, h] / x.sum(-1, keepdim=True)
            out[r: r + n, h * group: (h + 1) * group] = o.transpose(0, 1).to(out.dtype)
        r += n
    return out


def _plain_fork(state):
    case = state["case"]
    full, part = divmod(case["length"], PAGE)
    table, src = state["table"], state["tables"][0]
    n = case["children"]
    table[1: n + 1, :full] = table[0, :full]
    if part:
        fresh = torch.tensor(state["fresh"], device=table.device)
        table[1: n + 1, full] = fresh.int()
        p = state["plain"]
        for t in ([p.codes, p.scales] if p.q4 else [p.rows16]):
            t[:, fresh, :, :, :part] = t[:, src[full]: src[full] + 1, :, :, :part]
    return {"table": table, "pool": _values(state)}


def _plain_compact(state):
    table = state["table"]
    table.copy_(state["before"])
    live = torch.arange(table.shape[1], device=table.device) < state["counts"][:, None]
    used = torch.zeros(state["pages"], dtype=torch.bool, device=table.device)
    used[table[live].long()] = True
    n = used.sum()
    ids = torch.arange(state["pages"], device=table.device)
    src, dst = ids[used & (ids >= n)], ids[~used & (ids < n)]
    pool = state["pool"].view(state["layers"], state["pages"], -1)
    pool[:, dst] = pool[:, src]
    ids[src] = dst
    table[live] = ids[table[live].long()].int()
    return {"table": table, "pool": _values(state), "used": n.to(torch.int32)}


# ---- the definition in 64 bits -----------------------------------------------------------


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # copies: there is nothing to compute
    state = prepare(case, seed)
    values = state["plain"]
    counts, starts = _shapes(case)
    if case["op"] == "attend":
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device=state["q"].device)
        q = state["q"].double()
        group = case["heads"] // case["kv_heads"]
        r = 0
        for i in range(len(counts)):
            last = starts[i] + counts[i] - 1
            key = torch.arange(last + 1, device=q.device)
            page = state["table"][i, key // PAGE].long()
            k = values.read(0, page, key % PAGE, 0, torch.float64)
            v = values.read(0, page, key % PAGE, 1, torch.float64)
            for j in range(0, counts[i], 256):
                n = min(256, counts[i] - j)
                row = starts[i] + j + torch.arange(n, device=q.device)
                hidden = key[None] > row[:, None]
                if case["window"]:
                    hidden |= (row[:, None] - key[None] >= case["window"]) & (key[None] >= case["sinks"])
                for h in range(case["heads"]):
                    x = q[r + j: r + j + n, h] @ k[:, h // group].T / math.sqrt(case["dim"])
                    x[hidden] = -math.inf
                    out[r + j: r + j + n, h] = torch.softmax(x, -1) @ v[:, h // group]
            r += counts[i]
        return out
    if case["rot"]:
        half = case["rot"] // 2
        pair = torch.arange(half, device=state["q"].device)
        first = 2 * pair if case["inter"] else pair
        second = first + 1 if case["inter"] else first + half
        turn = torch.complex(state["cos"].double(), state["sin"].double())[state["pos"]][:, None]

        def turned(x, w):
            x = x.double()
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            return x

        pool = values.rows16.double()
        pool[0, state["page"], 0, :, state["off"]] = turned(state["k"], state["kw"])
        pool[0, state["page"], 1, :, state["off"]] = state["v"].double()
        return {"q": turned(state["q"], state["qw"]), "pool": pool}
    if case["kind"] != "q4":
        return None

    def stored(x):
        b = x.double().unflatten(-1, (-1, 32))
        top = b.abs().argmax(-1, keepdim=True)
        m = torch.gather(b, -1, top)
        level = torch.where(m == 0, 0.0, torch.floor(-8 * b / m + 0.5).clamp(-8, 7))
        return (level * (m / -8).half().double()).flatten(-2)

    return {"k": stored(state["k"]), "v": stored(state["v"])}
