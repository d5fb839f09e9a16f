"""A paged key/value cache and its operators (`include/fmd_cache.h`).

`PagedCache` holds the keys and values of many sequences ("slots") in pages of
64 positions, in the activations' 16 bits or in 4 bits, and offers what a
decoder does with them: `append` rows (query / key norms and the rotation in
the same pass), `attend` over them with a sliding window and sinks, `fork` a
sequence, `evict` what a window no longer sees, `release` and `compact`. The
pages' bookkeeping is on the host; the operators run on the current CUDA
stream of the cache's device and never synchronise. Tensors are torch tensors
(torch is only the allocator here). No counterpart in the reference, whose
cache is one dense 16-bit tensor per layer (qwen3.rs:33-108).

A decode loop:

    rows = cache.step([0, 1], [1, 1])        # one new position each
    for layer in range(layers):
        q = cache.append(layer, rows, k, v, q=q, q_norm=..., cos=..., sin=...)
        out = cache.attend(layer, rows, q, window=4096, sinks=4)

A captured step keeps its rows and moves them on itself (`rows.advance()` in the
graph); `cache.advance(slots)` before each replay keeps the books.
"""

from __future__ import annotations

import ctypes as C
import heapq
from dataclasses import dataclass

from . import _lib

PAGE = 64
_FORMATS = {"f16": _lib.CACHE_F16, "bf16": _lib.CACHE_BF16, "q4": _lib.CACHE_Q4}


def _fail(message: str, status: int = _lib.FMD_EINVAL):
    raise _lib.FmdError(status, message)


@dataclass
class CacheRows:
    """The rows of a call (`fmd_cache_rows`): sequence i owns rows
    `row0[i]:row0[i + 1]` (row i when `row0` is None) at positions `pos0[i]`,
    `pos0[i] + 1`, ... of `slot[i]`; slot -1 is padding. All int32 device
    tensors, so a captured graph reads what they hold when it is replayed."""

    slot: object
    pos0: object
    row0: object
    n_rows: int
    max_rows: int

    def advance(self, n: int = 1) -> None:
        """Move every sequence on by `n` positions, on the device, for launches
        whose positions no `step` gave out (a captured graph's). The cache's books
        follow by `PagedCache.advance`, called before those launches."""
        self.pos0.add_(n)



class PagedCache:
    """A cache of `n_pages` pages for up to `max_slots` sequences of up to
    `64 * max_pages_per_slot` positions. `kind`: "f16" or "bf16" (rows of that
    dtype) or "q4" (rows of either). `pool` and `page_table` may be the caller's
    (uint8 of `pool_bytes`, int32 `[max_slots, max_pages_per_slot]`), with
    `slots` as `(slot, its pages, its length)` for what they hold already (a table
    that the cache makes gets their pages). One host
    thread at a time may change the bookkeeping (open, step, fork, evict, release,
    compact); the operators may run on several streams, as long as no call writes
    what another reads."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, n_pages: int, max_slots: int,
                 max_pages_per_slot: int, kind: str = "bf16", device="cuda", pool=None, page_table=None, slots=()):
        import torch

        self.lib = _lib.load()
        if kind not in _FORMATS:
            _fail(f"kind must be one of {sorted(_FORMATS)}, not {kind!r}")
        if min(layers, kv_heads, n_pages, max_slots, max_pages_per_slot) < 1:
            _fail("layers, kv_heads, n_pages, max_slots and max_pages_per_slot must be at least 1")
        if head_dim not in (64, 128):
            _fail(f"head_dim must be 64 or 128, not {head_dim}", _lib.FMD_ENOTSUP)
        if max_pages_per_slot * PAGE > 2**31 - 1:
            _fail("positions are 32-bit", _lib.FMD_ENOTSUP)
        self.layers, self.kv_heads, self.head_dim, self.kind = layers, kv_heads, head_dim, kind
        self.n_pages, self.max_slots, self.max_pages_per_slot = n_pages, max_slots, max_pages_per_slot
        self.format = _FORMATS[kind]
        self.pool_bytes = (layers * n_pages * 2 * kv_heads *
                           int(self.lib.fmd_cache_block_bytes(self.format, head_dim)))
        self.device = torch.device(device if pool is None else pool.device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if pool is None:
            pool = torch.zeros(self.pool_bytes, dtype=torch.uint8, device=self.device)
        own_table = page_table is None
        if own_table:
            page_table = torch.full((max_slots, max_pages_per_slot), -1, dtype=torch.int32, device=self.device)
        if pool.dtype != torch.uint8 or pool.numel() != self.pool_bytes or not pool.is_contiguous():
            _fail(f"pool must be a contiguous uint8 tensor of {self.pool_bytes} bytes")
        if (page_table.dtype != torch.int32 or tuple(page_table.shape) != (max_slots, max_pages_per_slot)
                or not page_table.is_contiguous()):
            _fail("page_table must be a contiguous int32 tensor [max_slots, max_pages_per_slot]")
        if page_table.device != self.device:
            _fail("pool and page_table must be on the same device")
        self.pool, self.page_table = pool, page_table
        self._c = _lib.Cache(pool.data_ptr(), page_table.data_ptr(), self.format, layers, n_pages, kv_heads, head_dim,
                             max_slots, max_pages_per_slot, 0)
        self._ref = C.byref(self._c)
        self._index = pool.get_device()
        self._cuda, self._f32 = torch.cuda, torch.float32
        self._dtypes = ({torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16} if kind == "q4" else
                        {{"f16": torch.float16, "bf16": torch.bfloat16}[kind]: self.format})
        self._status = torch.zeros(2, dtype=torch.int32, device=self.device)
        self._status_at = self._status.data_ptr()
        self._workspaces: dict = {}
        # bookkeeping: pages of each open slot (-1: evicted), its length, names of each page
        self._pages: list = [None] * max_slots
        self._length = [0] * max_slots
        self._names = [0] * n_pages
        for slot, pages, length in slots:
            if not 0 <= slot < max_slots or self._pages[slot] is not None:
                _fail(f"bad slot {slot}")
            if len(pages) > max_pages_per_slot or not 0 <= length <= PAGE * len(pages):
                _fail(f"slot {slot}: {length} positions do not fit its pages")
            if any(not -1 <= p < n_pages for p in pages):
                _fail(f"slot {slot}: page out of range")
            self._pages[slot], self._length[slot] = list(pages), length
            for p in pages:
                if p >= 0:
                    self._names[p] += 1
            if own_table:
                self._upload(slot, 0)
        self._free = [p for p in range(n_pages) if self._names[p] == 0]  # a heap: the lowest page goes first

    # -- bookkeeping ---------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, slot: int) -> int:
        self._open(slot)
        return self._length[slot]

    def pages(self, slot: int) -> list:
        """The slot's pages in order; -1 where `evict` freed one."""
        return list(self._open(slot))

    def _open(self, slot: int) -> list:
        if not 0 <= slot < self.max_slots or self._pages[slot] is None:
            _fail(f"slot {slot} is not open")
        return self._pages[slot]

    def open(self, slot: int, positions: int = 0) -> None:
        """Open an empty sequence, with pages for its first `positions`."""
        if not 0 <= slot < self.max_slots:
            _fail(f"slot {slot} is out of range")
        if self._pages[slot] is not None:
            _fail(f"slot {slot} is already open", _lib.FMD_EBUSY)
        self._pages[slot], self._length[slot] = [], 0
        try:
            self.reserve(slot, positions)
        except _lib.FmdError:
            self._pages[slot] = None
            raise

    def release(self, *slots: int) -> None:
        """Close sequences; pages that no other slot names are free again."""
        if len(set(slots)) != len(slots):
            _fail("a slot is listed twice")
        for s in slots:
            self._open(s)
        names, free, common, m = self._names, self._free, [], 0

        def drop(pages, n):
            for p in pages:
                if p >= 0:
                    names[p] -= n
                    if not names[p]:
                        heapq.heappush(free, p)

        for s in slots:
            # slots that differ from the one before in their last page only, as forks do, give
            # the others up together
            pages = self._pages[s]
            self._pages[s], self._length[s] = None, 0
            n = len(common)
            if not n or pages[:n] != common:
                drop(common, m)
                common, m = pages[:-1], 0
                n = len(common)
            m += 1
            drop(pages[n:], 1)
        drop(common, m)

    def _drop(self, page: int) -> None:
        if page >= 0:
            self._names[page] -= 1
            if self._names[page] == 0:
                heapq.heappush(self._free, page)

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._names[p] = 1
        return p

    def _upload(self, slot: int, first: int, pages=None) -> None:
        import torch

        row = (self._pages[slot] if pages is None else pages)[first:]
        if row:
            self.page_table[slot, first:first + len(row)].copy_(torch.tensor(row, dtype=torch.int32))

    def reserve(self, slot: int, positions: int) -> None:
        """Give the slot pages for its first `positions` positions."""
        pages = self._open(slot)
        need = -(-positions // PAGE)
        if need > self.max_pages_per_slot:
            _fail(f"slot {slot}: {positions} positions exceed {self.max_pages_per_slot} pages", _lib.FMD_EOVERFLOW)
        have = len(pages)
        if need - have > len(self._free):
            _fail("the cache has too few free pages", _lib.FMD_ENOMEM)
        if need > have:
            pages += [self._take() for _ in range(need - have)]
            self._upload(slot, have)

    def step(self, slots, counts) -> CacheRows:
        """Rows for `counts[i]` new positions of each slot, which become part of
        its length: pass them to every layer's `append`, then `attend`. A page
        that is shared with another slot and about to be written is copied
        first."""
        import torch

        slots, counts = list(slots), list(counts)
        pos0 = self._extend(slots, counts)
        row0 = None
        if any(n != 1 for n in counts):
            row0 = [0]
            for n in counts:
                row0.append(row0[-1] + n)
        dev = self.device
        return CacheRows(torch.tensor(slots, dtype=torch.int32).to(dev), torch.tensor(pos0, dtype=torch.int32).to(dev),
                         None if row0 is None else torch.tensor(row0, dtype=torch.int32).to(dev), sum(counts),
                         max(counts, default=0))

    def advance(self, slots, n: int = 1) -> None:
        """The books of `n` new positions of each slot, as `step` keeps them, for
        rows that move on by themselves (`CacheRows.advance`, a replayed graph): call
        it before the launches that write the positions, so that their pages are
        there and the slot's own, and `length`, `step`, `fork` and `evict` know of
        them."""
        slots = list(slots)
        self._extend(slots, [n] * len(slots))

    def _extend(self, slots, counts) -> list:
        """Make `counts[i]` new positions part of each slot, with pages of its own
        for them; returns the slots' lengths before."""
        if len(slots) != len(counts) or any(n < 0 for n in counts):
            _fail("one count >= 0 per slot")
        if len(set(slots)) != len(slots):
            _fail("a slot is listed twice")
        # entries that need a page of their own (shared with a slot that keeps it, or evicted)
        fresh, given, own = 0, {}, [[] for _ in slots]
        for s, n, mine in zip(slots, counts, own):
            pages, at = self._open(s), self._length[s]
            need = -(-(at + n) // PAGE)
            if need > self.max_pages_per_slot:
                _fail(f"slot {s}: {at + n} positions exceed {self.max_pages_per_slot} pages", _lib.FMD_EOVERFLOW)
            fresh += max(0, need - len(pages))
            for k in range(at // PAGE, min(need, len(pages)) if n else 0):  # the pages that are written
                p = pages[k]
                if p < 0:
                    mine.append(k)
                elif self._names[p] - given.get(p, 0) > 1:  # the last to write a page keeps it
                    given[p] = given.get(p, 0) + 1
                    mine.append(k)
            fresh += len(mine)
        if fresh > len(self._free):
            _fail("the cache has too few free pages", _lib.FMD_ENOMEM)
        taken = [heapq.heappop(self._free) for _ in range(fresh)]
        moves, changed, new = [], [], iter(taken)
        for s, n, mine in zip(slots, counts, own):
            more = -(-(self._length[s] + n) // PAGE) - len(self._pages[s])
            if mine or more > 0:
                pages = list(self._pages[s])
                for k in mine:
                    p, pages[k] = pages[k], next(new)
                    if p >= 0:
                        moves.append((p, pages[k]))
                first = mine[0] if mine else len(pages)
                pages += [next(new) for _ in range(more)]
                changed.append((s, pages, first))
        try:
            if moves:
                self.copy_pages([a for a, _ in moves], [b for _, b in moves])
            for s, pages, first in changed:
                self._upload(s, first, pages)
        except BaseException:
            self._free += taken  # nothing else has changed
            heapq.heapify(self._free)
            raise
        for p in taken:
            self._names[p] = 1
        for p, _ in moves:
            self._drop(p)
        for s, pages, _ in changed:
            self._pages[s] = pages
        pos0 = [self._length[s] for s in slots]
        for s, n in zip(slots, counts):
            self._length[s] += n
        return pos0

    def rows(self, slot, pos0, row0=None, max_rows: int = 1, n_rows: int | None = None) -> CacheRows:
        """Rows from device tensors of the caller (a device-side scheduler, a
        graph); `n_rows` defaults to the rows that `append` or `attend` is given."""
        import torch

        for name, t, n in (("slot", slot, None), ("pos0", pos0, 0), ("row0", row0, 1)):
            if t is None and name == "row0":
                continue
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
                _fail(f"{name} must be a contiguous 1-D int32 tensor")
            if t.device != self.device:
                _fail(f"{name} must be on {self.device}")
            if n is not None and t.shape[0] != slot.shape[0] + n:
                _fail(f"{name} must have {slot.shape[0] + n} entries")
        if max_rows < 0 or (row0 is None and max_rows != 1):
            _fail("max_rows must be the rows of the longest sequence")
        return CacheRows(slot, pos0, row0, -1 if n_rows is None else n_rows, max_rows)

    # -- operators -------------------------------------------------------------------------
    def _call(self, fn, *args) -> None:
        cuda, index = self._cuda, self._index
        if cuda.current_device() == index:
            st = fn(self._ref, *args, cuda.current_stream(index).cuda_stream)
        else:
            with cuda.device(index):
                st = fn(self._ref, *args, cuda.current_stream(index).cuda_stream)
        if st != _lib.FMD_OK:
            raise _lib.FmdError(st, f"{fn.__name__}: {self.lib.fmd_status_string(st).decode()}")

    def check(self) -> None:
        """Wait for the operators, on every stream of the device, and raise if a row
        or page was out of range."""
        if self.device.type == "cuda":
            self._cuda.synchronize(self.device)
        st = int(self._status[0].item())
        if st != 0:
            self._status.zero_()
            if st == _lib.FMD_ETIMEDOUT:
                self._workspaces.clear()  # their counters may be left in the middle
            raise _lib.FmdError(st, "a device-side wait gave up" if st == _lib.FMD_ETIMEDOUT else
                                "a slot, position or page was out of range")

    def _dtype(self, t, name: str) -> int:
        code = self._dtypes.get(t.dtype)
        if code is None:
            _fail(f"{name} must be {'float16 or bfloat16' if self.kind == 'q4' else self.kind}, not {t.dtype}")
        return code

    def _heads(self, t, name: str, heads: int, rows: int, dtype) -> tuple:
        """(address, row stride, head stride) of a [rows, heads, head_dim] tensor."""
        if t.dim() != 3:
            _fail(f"{name} must be [rows, {heads or 'heads'}, {self.head_dim}], not {tuple(t.shape)}")
        n, h, d = t.shape
        if d != self.head_dim or (heads and h != heads):
            _fail(f"{name} must be [rows, {heads or 'heads'}, {self.head_dim}], not {(n, h, d)}")
        if t.get_device() != self._index:
            _fail(f"{name} must be on {self.device}")
        if n != rows or t.dtype != dtype:
            _fail(f"{name} must have the rows and dtype of the others")
        row, head, dim = t.stride()
        if n <= 1:
            row = 0
        if h <= 1:
            head = 0
        at = t.data_ptr()
        if (dim != 1 or (row | head) & 7 or at & 15) and t.numel():
            _fail(f"{name}: heads must be contiguous, 16-byte aligned, with strides of multiples of 8 elements")
        return at, row, head

    def _rows_c(self, rows: CacheRows, n: int):
        slot, row0 = rows.slot, rows.row0
        if rows.n_rows > n:
            _fail(f"the rows need {rows.n_rows} rows of the tensors, not {n}")
        seqs = slot.shape[0]
        if row0 is None and n < seqs:
            _fail(f"{seqs} sequences need a row each, not {n}")
        return C.byref(_lib.CacheRows(slot.data_ptr(), rows.pos0.data_ptr(), None if row0 is None else row0.data_ptr(),
                                      seqs, n, rows.max_rows, 0))

    def append(self, layer: int, rows: CacheRows, k, v, q=None, q_norm=None, k_norm=None, eps: float = 1e-6, cos=None,
               sin=None, interleaved: bool = False, q_out=None):
        """Store the rows' keys and values `[rows, kv_heads, head_dim]` at their
        positions, with `q_norm` / `k_norm` (RMS norm weights of a head) and the
        rotation of the first `2 * cos.shape[1]` dims by `cos[position]`,
        `sin[position]` (f32 tables; pairs i and i + half, or neighbours if
        `interleaved`) applied to queries and keys in the same pass. Returns the
        normed and rotated queries (`q_out`, which may be `q`), or None without
        `q`; rows of padding and behind the last sequence are left as they were in
        `q_out`, and hold anything without it. f32 arithmetic, one rounding per value.
        No gradients: operators of the cache are for inference."""
        if not 0 <= layer < self.layers:
            _fail(f"layer {layer} is out of range")
        code, dtype, n = self._dtype(k, "k"), k.dtype, k.shape[0]
        k_at, k_row, k_head = self._heads(k, "k", self.kv_heads, n, dtype)
        v_at, v_row, v_head = self._heads(v, "v", self.kv_heads, n, dtype)
        q_at = o_at = qn_at = kn_at = cos_at = sin_at = None
        q_row = q_head = o_row = o_head = heads = rot = table = 0
        if q is not None:
            q_at, q_row, q_head = self._heads(q, "q", 0, n, dtype)
            heads = q.shape[1]
            if q_out is None:
                q_out = q.new_empty(q.shape)
            o_at, o_row, o_head = self._heads(q_out, "q_out", heads, n, dtype)
        elif q_out is not None or q_norm is not None:
            _fail("q_out and q_norm need q")
        if q_norm is not None:
            qn_at = self._weight(q_norm, "q_norm", dtype)
        if k_norm is not None:
            kn_at = self._weight(k_norm, "k_norm", dtype)
        if (cos is None) != (sin is None):
            _fail("cos and sin go together")
        if cos is not None:
            cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
            if (cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != self._f32 or sin.dtype != self._f32
                    or not cos.is_contiguous() or not sin.is_contiguous() or (cos_at | sin_at) & 15
                    or cos.get_device() != self._index or sin.get_device() != self._index):
                _fail("cos and sin must be aligned contiguous f32 tables [positions, pairs]")
            table, pairs = cos.shape
            rot = 2 * pairs
            if table < 1 or pairs % 4 or not 0 < rot <= self.head_dim:
                _fail("the rotated dims must be a multiple of 8, at most head_dim")
        args = _lib.CacheAppendArgs(k_at, v_at, q_at, o_at, k_row, k_head, v_row, v_head, q_row, q_head, o_row, o_head,
                                    qn_at, kn_at, cos_at, sin_at, eps, code, heads, rot, table, bool(interleaved))
        self._call(self.lib.fmd_cache_append, layer, self._rows_c(rows, n), C.byref(args), self._status_at)
        return q_out

    def _weight(self, w, name: str, dtype) -> int:
        at = w.data_ptr()
        if (w.dtype != dtype or w.dim() != 1 or w.numel() != self.head_dim or not w.is_contiguous()
                or w.get_device() != self._index or at & 15):
            _fail(f"{name} must be an aligned contiguous [{self.head_dim}] tensor of the rows' dtype")
        return at

    def read(self, layer: int, rows: CacheRows, k_out=None, v_out=None, n_rows: int | None = None):
        """The cached keys and values of the rows' positions, f32
        `[rows, kv_heads, head_dim]`."""
        import torch

        if not 0 <= layer < self.layers:
            _fail(f"layer {layer} is out of range")
        if n_rows is None:
            n_rows = k_out.shape[0] if k_out is not None else rows.n_rows
        shape = (n_rows, self.kv_heads, self.head_dim)
        if n_rows < 0:
            _fail("n_rows is needed")
        k_out = torch.zeros(shape, dtype=torch.float32, device=self.device) if k_out is None else k_out
        v_out = torch.zeros(shape, dtype=torch.float32, device=self.device) if v_out is None else v_out
        for t in (k_out, v_out):
            if (t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != self.device
                    or t.data_ptr() % 16):
                _fail(f"outputs must be aligned contiguous f32 tensors {shape}")
        self._call(self.lib.fmd_cache_read, layer, self._rows_c(rows, n_rows), k_out.data_ptr(), v_out.data_ptr(),
                   self._status_at)
        return k_out, v_out

    def workspace(self, n_heads: int, n_seqs: int, max_rows: int = 1):
        """A zeroed workspace for `attend` calls of up to `n_seqs` sequences of
        up to `max_rows` rows, for callers that keep their own (one for each graph
        or stream whose calls may run at the same time)."""
        import torch

        n = int(self.lib.fmd_cache_attend_workspace(C.byref(self._c), n_heads, n_seqs, max_rows))
        return self._fresh_workspace(n)

    def _fresh_workspace(self, n: int):
        import torch

        w = torch.empty(max(n, 16), dtype=torch.uint8, device=self.device)
        w[:_lib.CACHE_WORKSPACE_ZERO].zero_()
        return w

    def _workspace(self, n_heads: int, rows: CacheRows):
        cuda = self._cuda
        n = self.lib.fmd_cache_attend_workspace(self._ref, n_heads, rows.slot.shape[0], rows.max_rows)
        if n == 0:
            return None
        if cuda.current_device() == self._index:
            capturing = cuda.is_current_stream_capturing()
        else:
            with cuda.device(self._index):
                capturing = cuda.is_current_stream_capturing()
        if capturing:
            # a graph's own: graphs replayed at the same time must not share one
            return self._fresh_workspace(n)
        key = cuda.current_stream(self._index).cuda_stream
        w = self._workspaces.get(key)
        if w is None or w.numel() < n:
            w = self._workspaces[key] = self._fresh_workspace(n)
        return w

    def attend(self, layer: int, rows: CacheRows, q, window: int = 0, sinks: int = 0, scale: float | None = None,
               out=None, workspace=None):
        """Attention of queries `[rows, heads, head_dim]` over their slots' cached
        positions j <= p (p: the row's own, already appended): all of them, or
        with `window` > 0 those with j > p - window or j < sinks. `scale` defaults
        to head_dim ** -0.5. Returns `out` (not `q` itself; rows of padding and
        behind the last sequence are left as they were)."""
        if not 0 <= layer < self.layers:
            _fail(f"layer {layer} is out of range")
        if not 0 <= window < 2**31 or not 0 <= sinks < 2**31:
            _fail("window and sinks must be >= 0")
        code, n = self._dtype(q, "q"), q.shape[0]
        q_at, q_row, q_head = self._heads(q, "q", 0, n, q.dtype)
        heads = q.shape[1]
        if heads % self.kv_heads or heads // self.kv_heads not in (1, 2, 4, 8, 16):
            _fail(f"heads must be {self.kv_heads} x 1, 2, 4, 8 or 16, not {heads}", _lib.FMD_ENOTSUP)
        if out is None:
            out = q.new_zeros(q.shape)
        o_at, o_row, o_head = self._heads(out, "out", heads, n, q.dtype)
        rows_c = self._rows_c(rows, n)
        if workspace is None:
            workspace = self._workspace(heads, rows)
        elif workspace.dtype.itemsize != 1 or workspace.device != self.device or not workspace.is_contiguous():
            _fail("workspace must be a contiguous uint8 tensor of this device (PagedCache.workspace)")
        ws, nb = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
        args = _lib.CacheAttendArgs(q_at, o_at, q_row, q_head, o_row, o_head,
                                    self.head_dim ** -0.5 if scale is None else scale, code, heads, window, sinks)
        self._call(self.lib.fmd_cache_attend, layer, rows_c, C.byref(args), ws, nb, self._status_at)
        return out

    # -- pages ----------------------------------------------------------------------------
    def copy_pages(self, src, dst) -> None:
        """Copy pages `src[i]` to `dst[i]` in every layer (contents only)."""
        src, dst = list(src), list(dst)
        if len(src) != len(dst):
            _fail("src and dst must be as long")
        if src and not 0 <= min(min(src), min(dst)) <= max(max(src), max(dst)) < self.n_pages:
            _fail("page out of range")
        if len(set(dst)) != len(dst) or set(dst) & set(src):
            _fail("a page is written twice, or read and written")
        ia = C.c_int32 * len(src)
        self._call(self.lib.fmd_cache_copy_pages, len(src), ia(*src), ia(*dst))

    def fork(self, src: int, dsts) -> None:
        """Give each closed slot of `dsts` the sequence of `src`: full pages are
        shared, the rows behind them are copied to a page of its own."""
        dsts = list(dsts)
        pages, n = self._open(src), self._length[src]
        full, part = divmod(n, PAGE)
        for d in dsts:
            if not 0 <= d < self.max_slots:
                _fail(f"slot {d} is out of range")
            if self._pages[d] is not None:
                _fail(f"slot {d} is already open", _lib.FMD_EBUSY)
        if len(set(dsts)) != len(dsts):
            _fail("a slot is listed twice")
        if part and pages[full] < 0:
            _fail(f"slot {src}: its last page was evicted")
        if part and len(dsts) > len(self._free):
            _fail("the cache has too few free pages", _lib.FMD_ENOMEM)
        m, shared, names = len(dsts), pages[:full], self._names
        fresh = [heapq.heappop(self._free) for _ in dsts] if part else [-1] * m
        ia = C.c_int32 * m
        try:
            self._call(self.lib.fmd_cache_fork, m, ia(*[src] * m), ia(*dsts), ia(*[n] * m), ia(*fresh),
                       self._status_at)
        except BaseException:
            if part:
                self._free += fresh  # nothing else has changed
                heapq.heapify(self._free)
            raise
        for p in fresh if part else ():
            names[p] = 1
        for d, p in zip(dsts, fresh):
            self._pages[d] = shared + [p] if part else shared.copy()
            self._length[d] = n
        for p in shared:
            if p >= 0:
                names[p] += m

    def evict(self, slot: int, window: int, sinks: int = 0) -> int:
        """Free the slot's pages that no later row sees with this window and
        sinks; returns how many. `attend` must not be given more afterwards. Later
        rows are those behind the slot's length: call it after the launches of the
        rows that `step` or `advance` gave out."""
        if window < 1 or sinks < 0:
            _fail("window must be >= 1 and sinks >= 0")
        pages, n = self._open(slot), self._length[slot]
        first, last = -(-sinks // PAGE), (n - window + 1) // PAGE  # pages [first, last) lie between them
        gone = [k for k in range(first, min(last, len(pages))) if pages[k] >= 0]
        for k in gone:
            self._drop(pages[k])
            pages[k] = -1
        if gone:
            self._upload(slot, gone[0])
        return len(gone)

    def compact_tables(self, page_table, n_entries):
        """Make the pages named by the first `n_entries[slot]` entries of each row
        of `page_table` dense, in every layer (`fmd_cache_compact`), for callers
        whose tables live on the device: the i-th used page at or above the number
        in use moves into the i-th free page below it, and the entries follow.
        Returns the number in use as a device tensor."""
        import torch

        if (page_table.dtype != torch.int32 or tuple(page_table.shape) != (self.max_slots, self.max_pages_per_slot)
                or not page_table.is_contiguous() or page_table.device != self.device):
            _fail("page_table must be a contiguous int32 tensor [max_slots, max_pages_per_slot] of this device")
        if (n_entries.dtype != torch.int32 or tuple(n_entries.shape) != (self.max_slots,)
                or not n_entries.is_contiguous() or n_entries.device != self.device):
            _fail("n_entries must be a contiguous int32 tensor [max_slots] of this device")
        c = _lib.Cache.from_buffer_copy(self._c)
        c.page_table = page_table.data_ptr()
        nb = int(self.lib.fmd_cache_compact_workspace(C.byref(c)))
        ws = torch.empty(nb, dtype=torch.uint8, device=self.device)
        used = torch.empty((), dtype=torch.int32, device=self.device)
        with torch.cuda.device(self.device):
            st = self.lib.fmd_cache_compact(C.byref(c), C.c_void_p(n_entries.data_ptr()), C.c_void_p(ws.data_ptr()), nb,
                                            C.c_void_p(used.data_ptr()), C.c_void_p(self._status.data_ptr()),
                                            C.c_void_p(torch.cuda.current_stream().cuda_stream))
        if st != _lib.FMD_OK:
            raise _lib.FmdError(st, f"fmd_cache_compact: {self.lib.fmd_status_string(st).decode()}")
        return used

    def compact(self) -> int:
        """Move the pages in use to the front of the pool; returns how many are
        in use."""
        import torch

        counts = torch.tensor([len(p or ()) for p in self._pages], dtype=torch.int32).to(self.device)
        self.compact_tables(self.page_table, counts)
        used = [p for p in range(self.n_pages) if self._names[p]]
        n = len(used)
        holes = [p for p in range(n) if not self._names[p]]
        to = dict(zip([p for p in used if p >= n], holes))
        self._pages = [None if r is None else [to.get(p, p) for p in r] for r in self._pages]
        for a, b in to.items():
            self._names[b], self._names[a] = self._names[a], 0
        self._free = list(range(n, self.n_pages))
        return n
