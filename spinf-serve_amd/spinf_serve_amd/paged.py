"""A paged cache of keys and values: contents that stay after their pass, and the attention of new tokens over them.

  PagedCache     the pages of one layer's keys and values
  PagedBatch     one call's requests: lengths, page tables, trees of new tokens; the work lists, compiled once per head geometry
  paged_attn     attention of the new tokens (single tokens, chunks, trees of questions) over what is stored
  paged_weights  the attention weight that every stored key received, added to what it had
  cache_evict    the stored keys with the least weight dropped, the others moved together into other pages

The reference keeps no such cache: its contents are read anew with every request, and its decoder copies a pass's keys and values
(spinf_serve/decode.py:129-171).  All device work goes through libspinf_tree.so; there is no CPU or PyTorch path.
"""

from __future__ import annotations

import ctypes as C
import os
import threading
import weakref
from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from . import _lib
from .masks import _Shared, _staging

# which kernel the work lists are made for (spinf_paged_plan_args.variant): 0 = the library's choice, 1 = the one whose waves share rows and divide the
# keys, 2 = the one whose waves have rows of their own.  For tests and measurements: results differ in their last bits.
VARIANT = int(os.environ.get("SPINF_PAGED_VARIANT", "0"))


@dataclass(frozen=True)
class PagedCache:
    """k, v: [pages, page, hkv, d] bf16 in any memory order whose rows of d are contiguous; page a multiple of 16.  What unused entries hold does not
    matter."""

    k: torch.Tensor
    v: torch.Tensor

    def __post_init__(self):
        for name, t in (("k", self.k), ("v", self.v)):
            if t.dim() != 4 or t.dtype != torch.bfloat16 or t.stride(3) != 1:
                raise ValueError(f"{name} must be bf16 [pages, page, key / value heads, head dim] with contiguous head dims")
            if any(s % 8 for s in t.stride()[:3]) or t.data_ptr() % 16:
                raise ValueError(f"{name} must be 16-byte aligned with strides that are multiples of 8 elements")
        if self.k.shape != self.v.shape or self.k.device != self.v.device:
            raise ValueError(f"k {tuple(self.k.shape)} on {self.k.device} and v {tuple(self.v.shape)} on {self.v.device} differ")
        if self.page < 16 or self.page % 16:
            raise ValueError(f"pages of {self.page} keys: a multiple of 16 is needed")
        if self.k.shape[3] not in (64, 128, 256, 512):
            raise ValueError(f"head dim {self.k.shape[3]} not supported (64, 128, 256, 512)")

    @property
    def page(self) -> int:
        return self.k.shape[1]

    @classmethod
    def empty(cls, pages: int, page: int, hkv: int, d: int, device="cuda") -> "PagedCache":
        """unwritten pages, each head's rows of a page next to each other in memory"""
        k, v = (torch.empty((pages, hkv, page, d), dtype=torch.bfloat16, device=device).transpose(1, 2) for _ in range(2))
        return cls(k, v)


LONGEST = 1 << 30   # stored keys of a request


def _whole(x, what) -> int:
    try:
        n = int(x)
    except OverflowError:
        n = None
    if n is None or n != x:
        raise ValueError(f"{what} {x}: a whole number is needed")
    return n


def _wholes(x, what):
    """-> int64 array of these values, which have to be whole numbers"""
    a = np.asarray(x).reshape(-1)
    if a.dtype.kind not in "iub":
        f = np.asarray(a, np.float64)
        if not (np.abs(f) < 2.0**63).all() or (f != np.floor(f)).any():
            raise ValueError(f"{what} must be whole numbers")
    elif a.dtype == np.uint64 and (a >> np.uint64(63)).any():
        raise ValueError(f"{what} must be whole numbers of 64 bits")
    return np.ascontiguousarray(a, np.int64)


def _lengths(x, what):
    a = _wholes(x, what)
    if len(a) and (a.min() < 0 or a.max() > LONGEST):
        raise ValueError(f"{what} must lie in 0 .. 2^30")
    return a.astype(np.int32)


class PagedBatch:
    """The requests of a call, shared by its layers.  Request r has kv_lens[r] stored keys, the last q_lens[r] of them its new tokens; stored key s lies
    in entry s % page of page tables[r][s // page].  The rows of a call's tensors are the requests' new tokens back to back.

    The new tokens of a request follow each other, or (end, pos given) are trees: the branches in pre-order, end[t] = the exclusive end of row t's
    subtree in rows of the call, pos[t] = its position (at most its place among the stored keys).  A row sees all keys stored before the new tokens, and
    of these the ones whose subtree it lies in.

    A request that cache_evict has trimmed stores fewer keys than its text has tokens, rotated by the positions they had.  dropped[r] says how many are gone: its new tokens'
    positions are their places plus that (of a tree, what pos says: the same at most).  A window counts places, so a call over such a batch takes none.

    Host threads and streams may share a batch: what a first call makes is made once, and a call on another stream waits for the copies.  A recorded graph reads the batch's
    lists on the device, as it reads the call's tensors: both have to live as long as the graph is replayed."""

    def __init__(self, q_lens, kv_lens, table, need, page, device, end, pos, dropped=None):
        """pos: counted in places, without what was dropped"""
        self._lock = threading.RLock()
        self.q_lens, self.kv_lens, self.page, self.device = q_lens, kv_lens, page, device
        self._table, self._need = table, need       # the pages back to back, and how many each request has
        self._end, self._pos, self._dropped = end, pos, dropped
        self.tokens = int(q_lens.sum(dtype=np.int64))
        self.max_page = int(table.max()) if len(table) else -1
        self.longest = int(kv_lens.max(initial=0))
        self._plans, self._moves, self._dev, self._rows = {}, {}, None, None
        self._calls = {}    # argument blocks without their tensors' addresses, by the tensors' shapes and strides and the call's numbers

    @classmethod
    def build(cls, q_lens, kv_lens, tables, page, device="cuda", end=None, pos=None, dropped=None) -> "PagedBatch":
        """tables: per request its pages (a list or a row of an integer array; entries behind the stored keys are ignored).  Host data only."""
        q_lens, kv_lens = _lengths(q_lens, "q_lens"), _lengths(kv_lens, "kv_lens")
        page = _whole(page, "page")
        if page < 16 or page % 16 or page > 1 << 20:
            raise ValueError(f"pages of {page} keys: a multiple of 16 is needed, at most 2^20")
        if len(q_lens) != len(kv_lens) or len(tables) != len(kv_lens):
            raise ValueError(f"{len(q_lens)} q_lens, {len(kv_lens)} kv_lens and {len(tables)} tables")
        need = -(-kv_lens.astype(np.int64) // page)
        table = cls._pages(tables, need, kv_lens, page)
        if len(table) and (table.min() < 0 or table.max() >= 1 << 31):
            raise ValueError("page numbers must lie in 0 .. 2^31 - 1")
        if dropped is not None:
            dropped = _lengths(dropped, "dropped")
            if len(dropped) != len(kv_lens):
                raise ValueError(f"{len(dropped)} values of dropped for {len(kv_lens)} requests")
            dropped = dropped if dropped.any() else None
        if (end is None) != (pos is None):
            raise ValueError("a tree needs both end and pos")
        if end is not None:
            end, pos = _wholes(end, "end"), _wholes(pos, "pos")
            tokens = int(q_lens.sum(dtype=np.int64))
            if len(end) != tokens or len(pos) != tokens:
                raise ValueError(f"end and pos hold {len(end)} and {len(pos)} values for {tokens} new tokens")
            if (q_lens > kv_lens).any():
                raise ValueError("a tree's new tokens are among the stored keys: q_lens must not exceed kv_lens")
            if dropped is not None:
                pos = pos - np.repeat(dropped, q_lens)
            if tokens:
                at = np.arange(tokens) - np.repeat(np.cumsum(q_lens, dtype=np.int64) - kv_lens, q_lens)
                if end.min() < 0 or end.max() > tokens or pos.min() < 0 or (pos > at).any():
                    raise ValueError("end must lie in 0 .. tokens, pos (less what was dropped) in 0 .. the token's place among the stored keys")
            end, pos = end.astype(np.int32), pos.astype(np.int32)
        return cls(q_lens, kv_lens, table.astype(np.int32), need, page, torch.device(device), end, pos, dropped)

    @staticmethod
    def _pages(tables, need, kv_lens, page):
        """the requests' pages back to back"""
        if isinstance(tables, np.ndarray) and tables.ndim == 2 and tables.dtype.kind in "iu" and (not len(need) or need.max() <= tables.shape[1]):
            return tables[np.arange(tables.shape[1]) < need[:, None]].astype(np.int64)
        parts = []
        for r, n in enumerate(need.tolist()):
            t = tables[r]
            t = np.array(t[:n]) if type(t) is list else np.asarray(t)[:n]
            if t.shape != (n,) or (n and t.dtype.kind not in "iu"):
                raise ValueError(f"request {r}: {kv_lens[r]} stored keys need {n} pages of {page}, whole numbers; its table gives {t.shape} of {t.dtype}")
            parts.append(t)
        return np.concatenate(parts).astype(np.int64) if parts else np.zeros(0, np.int64)

    def __reduce__(self):
        """copied and saved as what it is built from"""
        tables = np.split(self._table, np.cumsum(self._need)[:-1]) if len(self._need) else []
        return PagedBatch.build, (self.q_lens, self.kv_lens, tables, self.page, str(self.device), self._end, self._positions() if self._pos is not None else None, self._dropped)

    def _reach(self, shared):
        if shared.device.type == "cuda":
            shared.reach(_lib.raw_stream(shared.device.index))

    def _not_recording(self):
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a batch's first call of a kind copies its lists to the device, which cannot be recorded: make that call before the capture")

    def _upload(self, *arrays):
        """int32 arrays back to back, each 16-byte aligned, in one copy -> device tensor, where each begins"""
        self._not_recording()
        at, n = [], 0
        for a in arrays:
            at.append(n)
            n += -(-max(len(a), 1) // 4) * 4   # (an empty one has a place of its own too: no entry of it is read, but its address is passed)
        buf = _staging(max(n, 4), self.device)
        host = buf.numpy()
        for a, i in zip(arrays, at):
            host[i : i + len(a)] = a
        dev = buf.to(self.device, non_blocking=True)
        return dev, at, _Shared(dev) if dev.is_cuda else None

    def _device(self):
        if self._dev is None:
            with self._lock:
                if self._dev is None:
                    tree = self._end is not None
                    cu, tab = (np.cumsum(x, dtype=np.int64) - x for x in (self.q_lens, self._need))
                    reqs = np.stack([cu, self.q_lens, self.kv_lens, tab], 1).astype(np.int32).reshape(-1)
                    arrays = (reqs, self._table, self._end, self._pos) if tree else (reqs, self._table)
                    dev, at, shared = self._upload(*arrays)
                    parts = [dev[i : i + max(len(a), 1)] for a, i in zip(arrays, at)]
                    self._dev = (*parts, *[None] * (4 - len(parts))), shared
        parts, shared = self._dev
        if shared is not None:
            self._reach(shared)
        return parts

    def device_data(self):
        """-> device tensors table, end, pos (the latter None without trees)"""
        return self._device()[1:]

    def device_requests(self):
        """-> device tensor [4 requests] int32: first row, new tokens, stored keys, first page in the table"""
        return self._device()[0]

    def check_move(self, into, keep: int):
        """raises unless the pages of `into` can take what stays of this batch's requests; settled once for a pair of batches"""
        got = self._moves.get(keep)
        if got is not None and got() is into:
            return
        if len(into.kv_lens) != len(self.kv_lens):
            raise ValueError(f"cache_evict: {len(self.kv_lens)} requests into {len(into.kv_lens)}")
        stay = np.minimum(self.kv_lens, keep)
        if (into.kv_lens < stay).any():
            raise ValueError("cache_evict: the trimmed requests have fewer stored keys than stay")
        need = -(-stay.astype(np.int64) // self.page)
        first = np.cumsum(into._need) - into._need
        pages = into._table[np.repeat(first - (np.cumsum(need) - need), need) + np.arange(need.sum())]
        if len(np.unique(pages)) < len(pages) or np.isin(pages, self._table).any():
            raise ValueError("cache_evict: a page to be written twice, or one that is read")
        self._moves[keep] = weakref.ref(into)

    def _positions(self):
        """of the new tokens, in their texts"""
        if self._pos is None:
            base = np.cumsum(self.q_lens, dtype=np.int64) - self.kv_lens
            pos = np.maximum(np.arange(self.tokens) - np.repeat(base, self.q_lens), 0).astype(np.int32)
        else:
            pos = self._pos
        return pos if self._dropped is None else pos + np.repeat(self._dropped, self.q_lens)

    def rows(self):
        """-> (slots, positions) of the new tokens, device tensors int64 and int32: where the rows' keys and values go in the cache (page * page size +
        entry; -1 where a request has fewer stored keys than new tokens), and the rows' positions in their texts (`dropped` counted)"""
        if self._rows is None:
            with self._lock:
                if self._rows is None:
                    base = np.cumsum(self.q_lens, dtype=np.int64) - self.kv_lens      # row - stored place, by request
                    at = np.arange(self.tokens) - np.repeat(base, self.q_lens)
                    page = np.repeat(np.cumsum(self._need) - self._need, self.q_lens) + np.maximum(at, 0) // self.page
                    inside = at >= 0
                    slots = np.full(self.tokens, -1, np.int64)
                    slots[inside] = self._table[page[inside]].astype(np.int64) * self.page + at[inside] % self.page
                    dev, i, shared = self._upload(slots.view(np.int32), self._positions())
                    self._rows = dev[: 2 * self.tokens].view(torch.int64), dev[i[1] : i[1] + self.tokens], shared
        slots, pos, shared = self._rows
        if shared is not None:
            self._reach(shared)
        return slots, pos

    def plan(self, hq: int, hkv: int, d: int, window: int):
        """the work lists for a head geometry and a window (0: none) -> (lists on the device, counts, where wave, block, runs, joins begin)"""
        key = (hq, hkv, d, window, VARIANT)
        got = self._plans.get(key)
        if got is None:
            with self._lock:
                got = self._plans.get(key)
                if got is None:
                    got = self._plans[key] = self._compile(*key)
        if got[3] is not None:
            self._reach(got[3])
        return got[:3]

    def keep(self, key, args, device, *geometry):
        """notes an argument block with what it points into: the plan of `geometry`, if any, and the batch's own data"""
        shared = [self._dev[1]] + ([self._plans[(*geometry, VARIANT)][3]] if geometry else [])
        if len(self._calls) > 256:
            self._calls.clear()
        self._calls[key] = bytes(args), device, tuple(x for x in shared if x is not None)

    def _compile(self, hq, hkv, d, window, variant):
        self._not_recording()
        lib = _lib.load_library()
        a = _lib.PagedPlanArgs()
        a.q_lens, a.kv_lens, a.reqs = self.q_lens.ctypes.data, self.kv_lens.ctypes.data, len(self.kv_lens)
        if self._end is not None:
            a.end, a.pos = self._end.ctypes.data, self._pos.ctypes.data
        a.hq, a.hkv, a.d, a.page, a.window, a.variant = hq, hkv, d, self.page, window, variant
        h = C.c_void_p()
        _lib.check(lib.spinf_paged_plan_build(C.byref(a), C.byref(h)), "paged_plan")
        try:
            counts = (C.c_int64 * 5)()
            _lib.check(lib.spinf_paged_plan_counts(h, counts), "paged_plan_counts")
            sizes = [12 * counts[0], 12 * counts[1], 4 * counts[2], 8 * counts[3]]
            at = [0, sizes[0], sizes[0] + sizes[1], sum(sizes[:3])]
            buf = _staging(max(sum(sizes), 4), self.device)
            p = buf.data_ptr()
            _lib.check(lib.spinf_paged_plan_export(h, *(p + 4 * i for i in at)), "paged_plan_export")
        finally:
            lib.spinf_paged_plan_free(h)
        dev = buf.to(self.device, non_blocking=True)
        return dev, list(counts), at, _Shared(dev) if dev.is_cuda else None


def _check_call(q, k, v, tokens, page, max_page, what):
    """raises on tensors the kernels do not take"""
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.stride(2) != 1:
        raise ValueError(f"{what}: q must be bf16 [new tokens, query heads, head dim] with contiguous head dims")
    if q.shape[0] != tokens:
        raise ValueError(f"{what}: the batch has {tokens} new tokens, q {q.shape[0]} rows")
    if q.shape[2] != k.shape[3]:
        raise ValueError(f"{what}: head dim {q.shape[2]} of q, {k.shape[3]} of the cache")
    if k.shape[2] <= 0 or q.shape[1] <= 0 or q.shape[1] % k.shape[2]:
        raise ValueError(f"{what}: {q.shape[1]} query heads do not group over {k.shape[2]} key / value heads")
    if k.shape[1] != page:
        raise ValueError(f"{what}: the batch counts pages of {page} keys, the cache has {k.shape[1]}")
    if max_page >= k.shape[0]:
        raise ValueError(f"{what}: page {max_page} in a table, the cache has {k.shape[0]}")
    if not q.is_cuda:
        raise RuntimeError(f"{what} runs on ROCm device tensors only (no CPU path)")
    if q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        raise ValueError(f"{what}: q must be 16-byte aligned with strides that are multiples of 8 elements")


def _window(window, batch=None) -> int:
    """(a window as wide as the longest request may be hides nothing: wider ones are that one, and any of them fits the library's 32 bits)"""
    w = _whole(window, "window") if window is not None else 0
    if w < 0:
        raise ValueError(f"window {w}")
    if w and batch is not None and batch._dropped is not None:
        raise ValueError(f"window {w}: of a trimmed request's keys the places tell no distances")
    return min(w, LONGEST)


def _fill(a, q, k, v, page, window, scale, softcap):
    a.q, a.q_tok, a.q_head = q.data_ptr(), q.stride(0), q.stride(1)
    a.k, a.v = k.data_ptr(), v.data_ptr()
    a.k_page, a.k_row, a.k_head = k.stride()[:3]
    a.v_page, a.v_row, a.v_head = v.stride()[:3]
    a.hq, a.hkv, a.d, a.page, a.window = q.shape[1], k.shape[2], q.shape[2], page, window
    a.scale, a.softcap = scale, softcap


def _paged_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, end: Optional[torch.Tensor], pos: Optional[torch.Tensor],
                lists: torch.Tensor, counts: list[int], at: list[int], page: int, max_page: int, tokens: int, scale: float, window: int, softcap: float,
                want_lse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    a = _attn_block(q, k, v, table, end, pos, lists, counts, at, page, max_page, tokens, scale, window, softcap)
    out, lse = _attn_run(a, q, k, v, want_lse)
    return out, torch.empty((0,), dtype=torch.float32, device=q.device) if lse is None else lse


def _attn_block(q, k, v, table, end, pos, lists, counts, at, page, max_page, tokens, scale, window, softcap):
    """the argument block of a call but for the memory of q, k, v, the outputs and the workspace; raises on tensors the kernels do not take"""
    _check_call(q, k, v, tokens, page, max_page, "paged_attn")
    _lib.same_device(q.device, k, v, table, end, pos, lists)
    a = _lib.PagedArgs()
    _fill(a, q, k, v, page, window, scale, softcap)
    a.o_tok, a.o_head = q.shape[1] * q.shape[2], q.shape[2]
    a.table = table.data_ptr()
    if end is not None:
        a.end, a.pos = end.data_ptr(), pos.data_ptr()
    base = lists.data_ptr()
    a.wave, a.block, a.runs, a.joins = (base + 4 * i for i in at)
    a.n_wave, a.n_block, _, a.n_joins, a.part_rows = counts
    return a


def _attn_run(a, q, k, v, want_lse, stream=None):
    device = q.device
    T, hq, d = q.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = None
    if want_lse:
        lse = torch.empty((T, hq), dtype=torch.float32, device=device)
        a.lse = lse.data_ptr()
    if T:
        a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        if a.part_rows:
            n = a.part_rows * (d + 2)
            work = torch.empty(n, dtype=torch.float32, device=device)
            a.workspace, a.workspace_bytes = work.data_ptr(), 4 * n
        _lib.launch(_lib.load_library().spinf_paged_attn_fwd, a, device, "paged_attn", stream)
    return out, lse


_paged_op = torch.library.custom_op("spinf::paged_attn", _paged_attn, mutates_args=())


@_paged_op.register_fake
def _(q, k, v, table, end, pos, lists, counts, at, page, max_page, tokens, scale, window, softcap, want_lse):
    return (torch.empty(q.shape, dtype=torch.bfloat16, device=q.device),
            torch.empty(q.shape[:2] if want_lse else (0,), dtype=torch.float32, device=q.device))


def paged_attn(q, cache: PagedCache, batch: PagedBatch, scale=None, window=None, softcap=None, return_lse=False):
    """q [new tokens, hq, d] bf16 -> [new tokens, hq, d] bf16: softmax over the stored keys that each row sees of scale q.k (with ``softcap``: of softcap
    tanh(scale q.k / softcap)), times the values.  Row i of a request, stored at place c + i, sees the keys up to its own place (of a tree's new tokens
    those whose subtree it lies in), with ``window`` those less than ``window`` positions behind it.  A row that sees nothing is zeros.
    return_lse: also the natural log of each row's sum of exponentials, [new tokens, hq] fp32 (-inf where a row sees nothing).
    fp32 throughout, but for the probabilities: each is rounded to bf16 once for the product with its value (their sum takes the unrounded ones), which with the output's own
    rounding leaves an error of up to 2^-8 of a value's size against 2^-9 with 32 bits.
    The new tokens' own keys and values have to be in the cache (qk_norm_rope_put).  A request's rows are the same bits whatever else is in the batch."""
    k, v = cache.k, cache.v
    eager = _lib.eager(q, k, v)
    if eager:   # a later layer or step of this batch: everything but the tensors' memory was settled by the first
        key = (q.shape, q.stride(), q.dtype, k.shape, k.stride(), v.stride(), scale, window, softcap, VARIANT)
        got = batch._calls.get(key)
        if got is not None and q.device == got[1] == k.device == v.device:
            stream = _lib.raw_stream(got[1].index)
            for shared in got[2]:
                if stream not in shared.streams:
                    shared.reach(stream)
            out, lse = _attn_run(_lib.PagedArgs.from_buffer_copy(got[0]), q, k, v, return_lse, stream)
            return (out, lse) if return_lse else out
    w = _window(window, batch)
    sc = float(scale) if scale is not None else q.shape[-1] ** -0.5
    cap = float(softcap) if softcap else 0.0
    _check_call(q, k, v, batch.tokens, batch.page, batch.max_page, "paged_attn")
    _lib.same_device(q.device, k, v)
    table, end, pos = batch.device_data()
    lists, counts, at = batch.plan(q.shape[1], k.shape[2], q.shape[2], w)
    args = (q, k, v, table, end, pos, lists, counts, at, batch.page, batch.max_page, batch.tokens, sc, w, cap)
    if eager:
        a = _attn_block(*args)
        batch.keep(key, a, q.device, q.shape[1], k.shape[2], q.shape[2], w)
        out, lse = _attn_run(a, q, k, v, return_lse)
    else:
        out, lse = _paged_op(*args, bool(return_lse))
    return (out, lse) if return_lse else out


def _paged_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, acc: Optional[torch.Tensor], table: torch.Tensor, reqs: torch.Tensor,
                   end: Optional[torch.Tensor], pos: Optional[torch.Tensor], page: int, max_page: int, tokens: int, max_q: int, longest: int, n_reqs: int, keys: int, scale: float,
                   window: int, softcap: float) -> torch.Tensor:
    return _weights_run(_weights_block(q, k, lse, acc, table, reqs, end, pos, page, max_page, tokens, max_q, longest, n_reqs, keys, scale, window, softcap), q, k, lse, acc)


def _weights_block(q, k, lse, acc, table, reqs, end, pos, page, max_page, tokens, max_q, longest, n_reqs, keys, scale, window, softcap):
    _check_call(q, k, k, tokens, page, max_page, "paged_weights")
    _lib.same_device(q.device, k, lse, acc, table, reqs, end, pos)
    if lse.dtype != torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous():
        raise ValueError(f"paged_weights: lse must be contiguous fp32 {tuple(q.shape[:2])}")
    if acc is not None and (acc.dtype != torch.float32 or acc.shape != (n_reqs, k.shape[2], keys) or not acc.is_contiguous()):
        raise ValueError(f"paged_weights: acc must be contiguous fp32 [{n_reqs}, {k.shape[2]}, keys]")
    if keys < longest:
        raise ValueError(f"paged_weights: acc holds {keys} keys, a request has {longest}")
    a = _lib.PagedWeightsArgs()
    a.q_tok, a.q_head, (a.k_page, a.k_row, a.k_head) = q.stride(0), q.stride(1), k.stride()[:3]
    a.table, a.reqs = table.data_ptr(), reqs.data_ptr()
    if end is not None:
        a.end, a.pos = end.data_ptr(), pos.data_ptr()
    a.n_reqs, a.tokens, a.max_q, a.keys = n_reqs, tokens, max_q, keys
    a.hq, a.hkv, a.d, a.page, a.window, a.scale, a.softcap = q.shape[1], k.shape[2], q.shape[2], page, window, scale, softcap
    return a


def _weights_run(a, q, k, lse, acc, stream=None):
    out = torch.empty((a.n_reqs, a.hkv, a.keys), dtype=torch.float32, device=q.device)
    a.q, a.k, a.lse, a.out = q.data_ptr(), k.data_ptr(), lse.data_ptr(), out.data_ptr()
    if acc is not None:
        a.acc = acc.data_ptr()
    _lib.launch(_lib.load_library().spinf_paged_weights, a, q.device, "paged_weights", stream)
    return out


_weights_op = torch.library.custom_op("spinf::paged_weights", _paged_weights, mutates_args=())


@_weights_op.register_fake
def _(q, k, lse, acc, table, reqs, end, pos, page, max_page, tokens, max_q, longest, n_reqs, keys, scale, window, softcap):
    return torch.empty((n_reqs, k.shape[2], keys), dtype=torch.float32, device=q.device)


def paged_weights(q, cache: PagedCache, batch: PagedBatch, lse, scale=None, window=None, softcap=None, acc=None):
    """-> [requests, hkv, keys] fp32: acc (None: zeros over the longest request's keys) plus, for every stored key and key / value head, the attention weight that
    the new tokens' query heads gave it in paged_attn(q, cache, batch, scale, window, softcap, return_lse=True), whose log-sums are ``lse``.  Entries
    behind a request's stored keys are acc's.  Sums in one fixed order, without atomics."""
    k = cache.k
    eager = _lib.eager(q, k, lse, acc)
    if eager:
        key = ("weights", q.shape, q.stride(), q.dtype, k.shape, k.stride(), lse.shape, lse.stride(), lse.dtype, acc if acc is None else (acc.shape, acc.stride(), acc.dtype), scale, window, softcap)
        got = batch._calls.get(key)
        if got is not None and q.device == got[1] == k.device == lse.device and (acc is None or acc.device == got[1]):
            stream = _lib.raw_stream(got[1].index)
            for shared in got[2]:
                if stream not in shared.streams:
                    shared.reach(stream)
            return _weights_run(_lib.PagedWeightsArgs.from_buffer_copy(got[0]), q, k, lse, acc, stream)
    w = _window(window, batch)
    sc = float(scale) if scale is not None else q.shape[-1] ** -0.5
    longest = batch.longest
    keys = longest if acc is None else acc.shape[-1]
    _check_call(q, k, k, batch.tokens, batch.page, batch.max_page, "paged_weights")
    table, end, pos = batch.device_data()
    args = (q, k, lse, acc, table, batch.device_requests(), end, pos, batch.page, batch.max_page, batch.tokens, int(batch.q_lens.max(initial=0)), longest, len(batch.kv_lens), int(keys), sc, w, float(softcap) if softcap else 0.0)
    if not eager:
        return _weights_op(*args)
    a = _weights_block(*args)
    batch.keep(key, a, q.device)
    return _weights_run(a, q, k, lse, acc)


def _cache_evict(k: torch.Tensor, v: torch.Tensor, acc: torch.Tensor, table: torch.Tensor, reqs: torch.Tensor, new_table: torch.Tensor, new_reqs: torch.Tensor,
                 page: int, keep: int, sink: int, recent: int) -> tuple[torch.Tensor, torch.Tensor]:
    _lib.same_device(acc.device, k, v, table, new_table, reqs, new_reqs)
    return _evict_run(_evict_block(k, v, acc, table, reqs, page, keep, sink, recent), k, v, acc, new_table, new_reqs)


def _evict_block(k, v, acc, table, reqs, page, keep, sink, recent):
    R, hkv, keys = acc.shape
    a = _lib.EvictArgs()
    a.keys, a.n_reqs, a.hkv, a.d, a.page, a.keep, a.sink, a.recent = keys, R, hkv, k.shape[3], page, keep, sink, recent
    a.reqs, a.table = reqs.data_ptr(), table.data_ptr()
    a.k_page, a.k_row, a.k_head = k.stride()[:3]
    a.v_page, a.v_row, a.v_head = v.stride()[:3]
    return a


def _evict_run(a, k, v, acc, new_table, new_reqs, stream=None):
    device, shape = acc.device, (a.n_reqs, a.hkv, a.keep)
    kept = torch.empty(shape, dtype=torch.int32, device=device)
    new_acc = torch.empty_like(kept, dtype=torch.float32)
    if not (a.n_reqs and a.keep and a.keys):   # no stored key at all
        return kept.fill_(-1), new_acc.zero_()
    a.acc, a.k, a.v, a.kept, a.new_acc = acc.data_ptr(), k.data_ptr(), v.data_ptr(), kept.data_ptr(), new_acc.data_ptr()
    a.new_table, a.new_reqs = new_table.data_ptr(), new_reqs.data_ptr()
    _lib.launch(_lib.load_library().spinf_cache_evict, a, device, "cache_evict", stream)
    return kept, new_acc


_evict_op = torch.library.custom_op("spinf::cache_evict", _cache_evict, mutates_args=("k", "v"))


@_evict_op.register_fake
def _(k, v, acc, table, reqs, new_table, new_reqs, page, keep, sink, recent):
    shape = (*acc.shape[:2], keep)
    return torch.empty(shape, dtype=torch.int32, device=acc.device), torch.empty(shape, dtype=torch.float32, device=acc.device)


def cache_evict(cache: PagedCache, batch: PagedBatch, into: PagedBatch, acc, keep: int, sink: int = 0, recent: int = 0):
    """Trims every request of ``batch`` to at most ``keep`` stored keys, per key / value head: all stay where there are no more, else the first ``sink``, the last
    ``recent``, and of the others those with the largest ``acc`` [requests, hkv, keys] fp32 (ties to the lowest index, NaN above everything).  Their keys
    and values are copied, in order, into the first entries of the pages that ``into`` (the batch of the trimmed requests) gives them: the old pages stay
    as they are, since other requests may share them; into's pages must be none of batch's.  Rotated keys keep their positions: later batches of these requests are built with
    ``dropped``, and a layer with a window, which goes by places, is not trimmed this way.
    -> kept [requests, hkv, keep] int32 (the places that stayed, ascending, -1 behind them) and their acc (0 behind them): the next paged_weights' acc"""
    k, v = cache.k, cache.v
    pages, page, hkv, _ = k.shape
    R = len(batch.kv_lens)
    eager = _lib.eager(acc, k, v)
    if eager:
        key = ("evict", acc.shape, acc.stride(), acc.dtype, k.shape, k.stride(), v.stride(), keep, sink, recent)
        got = batch._calls.get(key)
        if got is not None and acc.device == got[1] == k.device == v.device and into.page == page and into.max_page < pages:
            batch.check_move(into, keep)
            new = into._device()
            if new[0].device == got[1]:
                stream = _lib.raw_stream(got[1].index)
                for shared in got[2]:
                    if stream not in shared.streams:
                        shared.reach(stream)
                return _evict_run(_lib.EvictArgs.from_buffer_copy(got[0]), k, v, acc, new[1], new[0], stream)
    keep, sink, recent = (_whole(x, f"cache_evict: {name}") for x, name in ((keep, "keep"), (sink, "sink"), (recent, "recent")))
    if sink < 0 or recent < 0 or sink + recent > keep or keep > LONGEST:
        raise ValueError(f"cache_evict: keep {keep}, of these the first {sink} and the last {recent}")
    if acc.dtype != torch.float32 or acc.dim() != 3 or acc.shape[0] != R or acc.shape[1] != hkv or not acc.is_contiguous():
        raise ValueError(f"cache_evict: acc must be contiguous fp32 [{R}, {hkv}, keys]")
    if acc.shape[2] < batch.longest:
        raise ValueError(f"cache_evict: acc holds {acc.shape[2]} keys, a request has {batch.longest}")
    if batch.page != page or into.page != page:
        raise ValueError(f"cache_evict: the batches count pages of {batch.page} and {into.page} keys, the cache has {page}")
    if max(batch.max_page, into.max_page) >= pages:
        raise ValueError(f"cache_evict: page {max(batch.max_page, into.max_page)} in a table, the cache has {pages}")
    batch.check_move(into, keep)
    if not acc.is_cuda:
        raise RuntimeError("cache_evict runs on ROCm device tensors only (no CPU path)")
    old, new = batch._device(), into._device()
    if not eager:
        return _evict_op(k, v, acc, old[1], old[0], new[1], new[0], page, keep, sink, recent)
    _lib.same_device(acc.device, k, v, *old[:2], *new[:2])
    a = _evict_block(k, v, acc, old[1], old[0], page, keep, sink, recent)
    batch.keep(key, a, acc.device)
    return _evict_run(a, k, v, acc, new[1], new[0])
