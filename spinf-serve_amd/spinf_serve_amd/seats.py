"""Seats: requests that go on token by token below contents that they share, with lengths, pages and places on the GPU, so that a recorded step can be replayed for the next one.

  PagedSeats   the seats' books: keys, pages out of a common pool, what each content is; the work lists of the attention
  seats_attn   attention of a step's new tokens: a content's keys read once for all seats below it, a seat's own keys after them

A PagedBatch (paged.py) is the other way: any tree of new tokens, lengths and pages chosen on the host, new for every step.  The reference keeps no cache between requests
(spinf_serve/decode.py:129-171 copies a pass's keys and values).  All device work goes through libspinf_tree.so; there is no CPU or PyTorch path.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np
import torch

from . import _lib
from .masks import _Shared
from .paged import LONGEST, PagedCache, _lengths, _whole, _wholes

_MOST_KEYS = 1 << 28


def _up4(n: int) -> int:
    return -(-n // 4) * 4


class PagedSeats:
    """``seats`` places for requests that go on at a time, `rows` rows to a step's tensors.  Seat r has lens[r] keys of its own (at most ``keys``), in pages out of ``pool``, behind
    the stored keys of content content[r] (-1: of none); own key s lies in entry s % page of page table[r, s // page].

    Device tensors, int32, kept by `step` and to be read only, but for ``content``, which the program writes (before the step that brings the seat's first token):
      content [seats]    which content a seat's request goes on below; a number that is none of them is as -1 (written in place: the seats keep this tensor)
      lens [seats]       own keys, the last step's new ones with them
      took, first        [seats] and [seats + 1]: the new tokens the last step gave each seat, and the row its first one is; first[-1]: rows in use
      table [seats, ceil(keys / page)], free [pool], left [1]: the seats' pages (behind a seat's keys: anything), the stack of free ones (its first left[0] entries)
      slots [rows] int64, pos [rows]: the rows' places in the cache and positions, as qk_norm_rope_put takes them; -1 and 0 behind the last row of as many as the last step had (behind those: an older
                         step's; `step` returns its own)

    What `step` and `seats_attn` do is ordered as their streams are: calls that share seats follow each other.  A recorded graph reads and writes these tensors: they have to
    live as long as it is replayed."""

    def __init__(self, geo, state, work, slots, pos, content, max_page, heads, dropped):
        self._geo, self._state, self._work, self.slots, self.pos, self.content = geo, state, work, slots, pos, content
        self.max_page, self.heads, self._dropped = max_page, heads, dropped
        self.device = state.device
        lay = _layout(geo)
        R, rows, page, keys, pool = geo[:5]
        part = lambda name, n: state[lay[name] : lay[name] + n]  # noqa: E731
        self.lens, self.took, self.first, self.left, self.free = part("lens", R), part("took", R), part("first", R + 1), part("left", 1), part("free", pool)
        self.table = part("table", R * -(-keys // page)).view(R, -1)
        self.seats, self.rows, self.page, self.keys = R, rows, page, keys
        self._now = rows    # rows of the last step
        self._calls = {}
        self._shared = None
        if state.is_cuda:
            self._shared = _Shared(state, work, slots, pos, content)
            self._args = _step_args(state, work, slots, pos, content, geo)

    @classmethod
    def build(cls, seats, rows, page, keys, pool, contents=None, stored=None, heads=(), dropped=None, device="cuda") -> "PagedSeats":
        """pool: page numbers, handed out from the last to the first.  contents: (stored keys, page lists), as PagedBatch.build takes kv_lens and tables; dropped: of each content how many of its keys
        cache_evict took away (its text goes on behind them).  stored: own keys that the seats have at the start (their pages are the first to be taken, seat by seat).
        heads: the head geometries of the calls to come, (query heads, key / value heads, head dim) or, of a layer with a window, (.., window).  Host data only."""
        lib = _lib.load_library()
        R, rows, page, keys = (_whole(x, f"PagedSeats: {n}") for x, n in ((seats, "seats"), (rows, "rows"), (page, "page"), (keys, "keys")))
        if page < 16 or page % 16 or page > 1 << 20:
            raise ValueError(f"pages of {page} keys: a multiple of 16 is needed, at most 2^20")
        if not 1 <= keys <= _MOST_KEYS:
            raise ValueError(f"PagedSeats: {keys} keys of a seat (1 .. 2^28)")
        pool = _wholes(pool, "pool")
        c_lens = _lengths(contents[0] if contents is not None else [], "contents")
        tables = contents[1] if contents is not None else []
        if len(tables) != len(c_lens):
            raise ValueError(f"PagedSeats: {len(c_lens)} contents and {len(tables)} tables")
        if len(c_lens) and c_lens.max() > _MOST_KEYS:
            raise ValueError("PagedSeats: a content has at most 2^28 keys")
        gone = _lengths(dropped, "dropped") if dropped is not None else np.zeros(len(c_lens), np.int32)
        if len(gone) != len(c_lens):
            raise ValueError(f"PagedSeats: {len(gone)} values of dropped for {len(c_lens)} contents")
        if len(c_lens) and int(c_lens.astype(np.int64).max() + gone.max()) + keys > LONGEST:
            raise ValueError("PagedSeats: positions beyond 2^30")
        need = -(-c_lens.astype(np.int64) // page)
        from .paged import PagedBatch

        listed = PagedBatch._pages(tables, need, c_lens, page)
        own = _lengths(stored, "stored") if stored is not None else np.zeros(max(R, 0), np.int32)
        if len(own) != R or (len(own) and own.max() > keys):
            raise ValueError(f"PagedSeats: stored gives {len(own)} seats up to {own.max(initial=0)} keys; there are {R} of at most {keys}")
        every = np.concatenate([listed, pool])
        if len(every) and (every.min() < 0 or every.max() >= 1 << 31):
            raise ValueError("page numbers must lie in 0 .. 2^31 - 1")
        if len(np.unique(pool)) < len(pool) or np.isin(pool, listed).any():
            raise ValueError("PagedSeats: a page of the pool twice, or one that a content lies in")
        taken = -(-own.astype(np.int64) // page)
        if taken.sum() > len(pool):
            raise ValueError(f"PagedSeats: the seats' stored keys need {taken.sum()} pages, the pool has {len(pool)}")
        kinds = []
        for h in heads:
            hq, hkv, d, *w = (_whole(x if x is not None else 0, "PagedSeats: heads") for x in h)
            if len(w) > 1 or (w and w[0] < 0):
                raise ValueError(f"PagedSeats: heads {tuple(h)}: (query heads, key / value heads, head dim) or (.., window)")
            kinds.append((hq, hkv, d, min(w[0], LONGEST) if w else 0))
        if gone.any() and any(k[3] for k in kinds):
            raise ValueError("PagedSeats: of a trimmed content's keys the places tell no distances: no window")
        if len(kinds) > 8 or len(set(kinds)) < len(kinds):
            raise ValueError(f"PagedSeats: head geometries {kinds}: at most 8, each once")
        if len(pool) > 1 << 28 or max([*(x for k in kinds for x in k), R, rows]) > LONGEST or min([*(x for k in kinds for x in k), R, rows]) < 0:
            raise ValueError("PagedSeats: numbers out of range")
        geo = [R, rows, page, keys, len(pool), len(c_lens), int(c_lens.max(initial=0)), int(need.sum()), len(kinds), *(x for k in kinds for x in k)]
        a = _numbers(geo)
        rooms = (C.c_int64 * 5)()
        for i in range(len(kinds)):
            _lib.check(lib.spinf_seats_rooms(C.byref(a), i, rooms), "PagedSeats")
            geo += list(rooms)
        if not kinds:   # (the numbers are checked all the same)
            a.kinds, a.kind[0].hq, a.kind[0].hkv, a.kind[0].d = 1, 1, 1, 64
            _lib.check(lib.spinf_seats_rooms(C.byref(a), 0, rooms), "PagedSeats")
        lay = _layout(geo)
        host = np.zeros(lay["all"], np.int32)
        host[: len(listed)] = listed
        width = -(-keys // page)
        table = np.full((R, width), -1, np.int32)
        at = np.cumsum(taken) - taken
        order = pool[::-1].astype(np.int64)
        for r in np.flatnonzero(taken):
            table[r, : taken[r]] = order[at[r] : at[r] + taken[r]]
        host[lay["table"] : lay["table"] + R * width] = table.reshape(-1)
        host[lay["lens"] : lay["lens"] + R] = own
        host[lay["free"] : lay["free"] + len(pool)] = pool
        host[lay["left"]] = len(pool) - taken.sum()
        host[lay["shared"] : lay["shared"] + 3 * len(c_lens)] = np.stack([c_lens, c_lens + gone, np.cumsum(need) - need], 1).reshape(-1)
        device = torch.device(device)
        state = torch.from_numpy(host).to(device)   # (a copy that is done when it returns: calls on any stream may follow)
        work = torch.zeros(lay["work"], dtype=torch.int32, device=device)
        slots = torch.full((rows,), -1, dtype=torch.int64, device=device)
        pos = torch.zeros(rows, dtype=torch.int32, device=device)
        content = torch.full((R,), -1, dtype=torch.int32, device=device)
        return cls(geo, state, work, slots, pos, content, int(every.max(initial=-1)), tuple(kinds), bool(gone.any()))

    def _reach(self):
        on = _lib.raw_stream(self.device.index)
        if on not in self._shared.streams:
            self._shared.reach(on)
        return on

    def step(self, new, drop=None, rows=None):
        """First the last drop[r] own keys of every seat go (drop None: none; as many as there are at most: a large number empties the seat) and pages that hold none any more are free
        again; then new[r] tokens come to seat r (below 1: none), with the pages they need.  A seat gets all of its tokens or none: none where they would pass ``keys``, where what the seats up to it
        ask for is more than ``rows`` rows, or more pages than are free (`took` says).  new, drop: [seats] int32 on the device.  rows: of this step's tensors, at most the seats' (None: as many).
        -> slots, pos [rows] (of the seats' own tensors)"""
        n = self.rows if rows is None else _whole(rows, "PagedSeats.step: rows")
        if not 1 <= n <= self.rows:
            raise ValueError(f"PagedSeats.step: {n} rows, the seats were built for up to {self.rows}")
        self._check(new, "new")
        if drop is not None:
            self._check(drop, "drop")
        if self._shared is None:
            raise RuntimeError("PagedSeats.step runs on ROCm device tensors only (no CPU path)")
        if _lib.eager(self._state, new, drop):
            a = _lib.SeatsArgs.from_buffer_copy(self._args)
            a.come, a.drop, a.rows = new.data_ptr(), drop.data_ptr() if drop is not None else None, n
            _lib.launch(_lib.load_library().spinf_seats_step, a, self.device, "seats_step", self._reach())
        else:
            self._reach()
            _step_op(self._state, self._work, self.slots, self.pos, self.content, new, drop, self._geo, n)
        self._now = n
        return (self.slots, self.pos) if n == self.rows else (self.slots[:n], self.pos[:n])

    def _check(self, t, what):
        if t.dtype != torch.int32 or t.shape != (self.seats,) or not t.is_contiguous():
            raise ValueError(f"PagedSeats.step: {what} must hold {self.seats} contiguous int32 values")
        if t.device != self.device:
            raise ValueError(f"PagedSeats.step: {what} on {t.device}, the seats are on {self.device}")


# geo: seats, rows, page, keys, pool, contents, longest content, pages of contents, head geometries; of each hq, hkv, d, window; of each what spinf_seats_rooms says
def _kinds(geo):
    n = geo[8]
    return [geo[9 + 4 * i : 13 + 4 * i] for i in range(n)]


def _rooms(geo, i):
    at = 9 + 4 * geo[8] + 5 * i
    return geo[at : at + 5]


def _layout(geo):
    """where things begin in the state and in the work lists, in int32"""
    R, rows, page, keys, pool, contents, _, listed, n = geo[:9]
    lay, at = {"pages": 0}, _up4(listed)
    for name, size in (("table", R * -(-keys // page)), ("lens", R), ("free", pool), ("left", 1), ("first", R + 1), ("took", R), ("stay", R), ("shared", 3 * contents)):
        lay[name] = at
        at += _up4(max(size, 1))   # (an empty one has a place of its own too: its address is passed)
    lay["all"] = at
    at, lists = 0, []
    for i in range(n):
        wave, single, block, last, _ = _rooms(geo, i)
        begins = []
        for size in (24 * wave, 24 * single, 24 * block, 12 * last, 5, rows + 1, 2 * R + 1):
            begins.append(at)
            at += _up4(size)
        lists.append(begins)
    lay["lists"], lay["work"] = lists, max(at, 4)
    return lay


def _numbers(geo):
    a = _lib.SeatsArgs()
    a.seats, a.rows, a.page, a.keys, a.pool, a.contents, a.longest = geo[:7]
    a.table_at, a.kinds = _up4(geo[7]), geo[8]
    for i, k in enumerate(_kinds(geo)):
        a.kind[i].hq, a.kind[i].hkv, a.kind[i].d, a.kind[i].window = k
    return a


def _point(kind, work, begins):
    base = work.data_ptr()
    kind.wave, kind.single, kind.block, kind.last, kind.counts, kind.parts, kind.seat_parts = (base + 4 * i for i in begins)


def _step_args(state, work, slots, pos, content, geo):
    a, lay, base = _numbers(geo), _layout(geo), state.data_ptr()
    a.content, a.slots, a.pos, a.lists = content.data_ptr(), slots.data_ptr(), pos.data_ptr(), base
    a.lens, a.free, a.left, a.first, a.took, a.stay, a.shared = (base + 4 * lay[x] for x in ("lens", "free", "left", "first", "took", "stay", "shared"))
    for i, begins in enumerate(lay["lists"]):
        _point(a.kind[i], work, begins)
    return a


def _step(state: torch.Tensor, work: torch.Tensor, slots: torch.Tensor, pos: torch.Tensor, content: torch.Tensor, new: torch.Tensor, drop: Optional[torch.Tensor], geo: list[int],
          rows: int) -> None:
    _lib.same_device(state.device, work, slots, pos, content, new, drop)
    a = _step_args(state, work, slots, pos, content, geo)
    a.come, a.drop, a.rows = new.data_ptr(), drop.data_ptr() if drop is not None else None, rows
    _lib.launch(_lib.load_library().spinf_seats_step, a, state.device, "seats_step")


_step_op = torch.library.custom_op("spinf::seats_step", _step, mutates_args=("state", "work", "slots", "pos"))


@_step_op.register_fake
def _(state, work, slots, pos, content, new, drop, geo, rows):
    return None


def _attn_block(q, k, v, state, work, pos, geo, index, scale, softcap):
    """the argument block of a call but for the memory of q, k, v, the outputs and the workspace; raises on tensors the kernels do not take"""
    _lib.same_device(q.device, k, v, state, work, pos)
    lay, base = _layout(geo), state.data_ptr()
    a = _lib.SeatsAttnArgs()
    a.q_tok, a.q_head, a.o_tok, a.o_head = q.stride(0), q.stride(1), q.shape[1] * q.shape[2], q.shape[2]
    a.k_page, a.k_row, a.k_head = k.stride()[:3]
    a.v_page, a.v_row, a.v_head = v.stride()[:3]
    a.lists, a.first, a.pos = base, base + 4 * lay["first"], pos.data_ptr()
    a.kind.hq, a.kind.hkv, a.kind.d, a.kind.window = _kinds(geo)[index]
    _point(a.kind, work, lay["lists"][index])
    n = _numbers(geo)   # (room for as many rows as these: a step of few needs little of what the seats' most would)
    n.rows = q.shape[0]
    rooms = (C.c_int64 * 5)()
    _lib.check(_lib.load_library().spinf_seats_rooms(C.byref(n), index, rooms), "seats_attn")
    for i in range(5):
        a.rooms[i] = rooms[i]
    a.rows, a.seats, a.page, a.scale, a.softcap = q.shape[0], geo[0], geo[2], scale, softcap
    return a


def _attn_run(a, q, k, v, want_lse, stream=None):
    rows, hq, d = q.shape
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = None
    if want_lse:
        lse = torch.empty((rows, hq), dtype=torch.float32, device=q.device)
        a.lse = lse.data_ptr()
    n = a.rooms[4] * hq * (d + 2)
    work = torch.empty(n, dtype=torch.float32, device=q.device)
    a.workspace, a.workspace_bytes = work.data_ptr(), 4 * n
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    _lib.launch(_lib.load_library().spinf_seats_attn_fwd, a, q.device, "seats_attn", stream)
    return out, lse


def _seats_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, state: torch.Tensor, work: torch.Tensor, pos: torch.Tensor, geo: list[int], index: int, scale: float, softcap: float,
                want_lse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    out, lse = _attn_run(_attn_block(q, k, v, state, work, pos, geo, index, scale, softcap), q, k, v, want_lse)
    return out, torch.empty((0,), dtype=torch.float32, device=q.device) if lse is None else lse


_attn_op = torch.library.custom_op("spinf::seats_attn", _seats_attn, mutates_args=())


@_attn_op.register_fake
def _(q, k, v, state, work, pos, geo, index, scale, softcap, want_lse):
    return (torch.empty(q.shape, dtype=torch.bfloat16, device=q.device),
            torch.empty(q.shape[:2] if want_lse else (0,), dtype=torch.float32, device=q.device))


def seats_attn(q, cache: PagedCache, seats: PagedSeats, scale=None, window=None, softcap=None, return_lse=False):
    """q [rows, hq, d] bf16, the new tokens of the last `step` -> [rows, hq, d] bf16: softmax over the keys that each row sees of scale q.k (with ``softcap``: of softcap tanh(scale q.k /
    softcap)), times the values.  A row sees the stored keys of its seat's content and its seat's own keys up to its own, with ``window`` those less than ``window`` places behind it.  Rows behind
    the step's last (seats.first[-1] of them are in use) come out as zeros, with a log-sum of -inf.  return_lse: also the natural log of each row's sum of exponentials, [rows, hq] fp32.
    Seats one after the other below the same content share its reading: put them next to each other.  fp32 throughout, but for the probabilities, each rounded to bf16 once for the
    product with its value, as in paged_attn (one token on few keys of its own: not rounded).  How keys are cut into pieces goes by all lengths of the step: the same step gives the same bits, a
    row beside other seats differs in the rounding of its sums.  What a row does not see may be anything, NaN and infinities too.
    The rows are the last step's (its ``rows``); replayed behind a step of more tokens than q has rows, all of them are NaN, behind one of fewer rows those after its tokens are zeros.
    (hq, key / value heads, d) and the window have to be among the seats' ``heads``.  The new tokens' own keys and values have to be in the cache (qk_norm_rope_put)."""
    k, v = cache.k, cache.v
    eager = _lib.eager(q, k, v)
    if eager:   # a later layer or step: everything but the tensors' memory was settled by the first
        key = (q.shape, q.stride(), q.dtype, k.shape, k.stride(), v.stride(), scale, window, softcap)
        got = seats._calls.get(key)
        if got is not None and q.shape[0] == seats._now and q.device == seats.device == k.device and not q.data_ptr() % 16:
            out, lse = _attn_run(_lib.SeatsAttnArgs.from_buffer_copy(got), q, k, v, return_lse, seats._reach())
            return (out, lse) if return_lse else out
    w = _whole(window, "window") if window is not None else 0
    if w < 0:
        raise ValueError(f"window {w}")
    w = min(w, LONGEST)
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("seats_attn: q must be bf16 [rows, query heads, head dim] with contiguous head dims")
    if q.shape[0] != seats._now:
        raise ValueError(f"seats_attn: the last step has {seats._now} rows, q {q.shape[0]}")
    if (q.shape[1], k.shape[2], q.shape[2], w) not in seats.heads or q.shape[2] != k.shape[3]:
        raise ValueError(f"seats_attn: {q.shape[1]} query heads on {k.shape[2]} of {q.shape[2]} dims (the cache: {k.shape[3]}), window {w}: the seats were built for {seats.heads}")
    if k.shape[1] != seats.page:
        raise ValueError(f"seats_attn: the seats count pages of {seats.page} keys, the cache has {k.shape[1]}")
    if seats.max_page >= k.shape[0]:
        raise ValueError(f"seats_attn: page {seats.max_page} is the seats' or a content's, the cache has {k.shape[0]}")
    if not q.is_cuda:
        raise RuntimeError("seats_attn runs on ROCm device tensors only (no CPU path)")
    if q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        raise ValueError("seats_attn: q must be 16-byte aligned with strides that are multiples of 8 elements")
    _lib.same_device(q.device, k, v, seats._state)
    sc = float(scale) if scale is not None else q.shape[-1] ** -0.5
    cap = float(softcap) if softcap else 0.0
    index = seats.heads.index((q.shape[1], k.shape[2], q.shape[2], w))
    seats._reach()
    args = (q, k, v, seats._state, seats._work, seats.pos, seats._geo, index, sc, cap)
    if eager:
        a = _attn_block(*args)
        out, lse = _attn_run(a, q, k, v, return_lse)
        if _lib.lasting(key):
            if len(seats._calls) > 256:
                seats._calls.clear()
            for x in ("q", "k", "v", "out", "lse", "workspace"):
                setattr(a, x, None)
            seats._calls[key] = bytes(a)
    else:
        out, lse = _attn_op(*args, bool(return_lse))
    return (out, lse) if return_lse else out
