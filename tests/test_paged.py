"""The paged cache: work lists against the dense mask (CPU), refusals, and the kernels against the float64 oracle (gpu)."""

import copy
import ctypes as C
import pickle

import numpy as np
import pytest
import torch

import spinf_serve_amd as sa
from oracle import paged as op
from spinf_serve_amd import _lib, paged

BF16 = torch.bfloat16


# ------------------------------------------------------------------------------------------------ requests
def tree_rows(rng, base, stored, branches, lo, hi, depth=3):
    """end (rows of the call) and pos of a random forest of branches below `stored` keys, in pre-order"""
    end, pos, path = [], [], []
    for _ in range(branches):
        while len(path) > int(rng.integers(0, min(len(path), depth) + 1)):
            for i in path.pop():
                end[i] = base + len(end)
        start = pos[path[-1][-1]] + 1 if path else stored
        n = int(rng.integers(lo, hi + 1))
        path.append(list(range(len(end), len(end) + n)))
        end += [0] * n
        pos += range(start, start + n)
    while path:
        for i in path.pop():
            end[i] = base + len(end)
    return end, pos


def make_batch(q_lens, kv_lens, page, device="cpu", tree=None, seed=0, spare=3):
    """-> batch, pages in all; tree (lo, hi): every request's new tokens are a random forest of about q_lens[r] tokens"""
    rng = np.random.default_rng(seed)
    end = pos = None
    if tree:
        end, pos, lens, kv = [], [], [], []
        for q, L in zip(q_lens, kv_lens):
            c = L - q
            e, p = tree_rows(rng, len(end), c, max(1, 2 * q // (sum(tree))), *tree) if q else ([], [])
            lens.append(len(e))
            kv.append(c + len(e))
            end += e
            pos += p
        q_lens, kv_lens = lens, kv
    need = [-(-n // page) for n in kv_lens]
    ids = rng.permutation(sum(need) + spare)[: sum(need)]
    tables = [x.tolist() for x in np.split(ids, np.cumsum(need)[:-1])]
    return sa.PagedBatch.build(q_lens, kv_lens, tables, page, device, end=end, pos=pos), sum(need) + spare


def dense(b, window):
    """per request the oracle's visibility matrix"""
    out, base = [], 0
    for T, L in zip(b.q_lens, b.kv_lens):
        rows = slice(base, base + T)
        out.append(op.visible(T, L, None if b._end is None else b._end[rows], None if b._pos is None else b._pos[rows], base, window))
        base += T
    return out


PLANS = [  # q_lens, kv_lens, page, (hq, hkv, d), window, tree
    ([1], [1], 16, (4, 4, 64), 0, None),
    ([1, 1, 1], [0, 33, 700], 16, (8, 2, 128), 0, None),
    ([1, 3], [4097, 130], 48, (16, 1, 512), 0, None),
    ([5, 40, 0, 129], [2, 100, 7, 129], 32, (6, 2, 64), 0, None),          # more new tokens than stored ones: rows that see nothing
    ([200, 64], [457, 64], 80, (4, 2, 128), 0, None),
    ([200, 1, 33], [457, 900, 300], 64, (4, 2, 128), 100, None),
    ([70, 70], [70, 400], 16, (4, 4, 64), 1, None),
    ([60, 90], [361, 90], 64, (4, 2, 256), 0, (1, 9)),
    ([60, 90], [361, 151], 48, (10, 2, 64), 40, (4, 24)),
    ([700, 20], [1170, 31], 64, (16, 8, 256), 0, (8, 16)),
    ([2500], [3300], 64, (16, 8, 64), 0, None),
    ([1300], [3300], 64, (32, 8, 64), 700, None),
    ([1100, 2], [1400, 2], 64, (32, 16, 128), 0, (2, 30)),
]


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("q_lens,kv_lens,page,heads,window,tree", PLANS)
def test_work_lists_are_the_dense_mask(q_lens, kv_lens, page, heads, window, tree, variant, monkeypatch):
    monkeypatch.setattr(paged, "VARIANT", variant)
    b, _ = make_batch(q_lens, kv_lens, page, tree=tree)
    hq, hkv, d = heads
    group = hq // hkv
    lists, counts, at = b.plan(hq, hkv, d, window)
    lists = lists.numpy()
    nw, nb, nr, nj, parts = counts
    assert variant == 0 or not (nb, nw)[variant - 1]
    runs = lists[at[2] : at[2] + 4 * nr].reshape(-1, 4)
    see = [np.repeat(x, group, 0) for x in dense(b, window)]
    cu = np.cumsum(b.q_lens) - b.q_lens
    tab = np.cumsum(b._need) - b._need
    seen = [np.zeros((T * group, L), np.int8) for T, L in zip(b.q_lens, b.kv_lens)]
    of_head = {}
    pieces, used = {}, np.zeros(max(parts, 1), np.int32)
    for kind, n, off, groups in ((0, nw, at[0], 1), (1, nb, at[1], 4)):
        for it in lists[off : off + 12 * n].reshape(-1, 12):
            cu_, T, L, tab_, kvh, row0, first, n_runs, tiles, part, r, nsplit = (int(x) for x in it)
            assert (cu_, T, L, tab_) == (cu[r], b.q_lens[r], b.kv_lens[r], tab[r]) and 0 <= row0 < T * group and row0 % 32 == 0
            pieces.setdefault((r, kvh, row0, groups), []).append((part, nsplit))
            if part >= 0:
                rows = min(32 * groups, T * group - row0)
                used[part : part + rows] += 1
            of_head.setdefault((r, row0, groups, len(pieces[r, kvh, row0, groups])), set()).add((first, n_runs))
            count = 0
            for kt, cnt, bits, _ in runs[first : first + n_runs].tolist():
                assert cnt > 0
                count += cnt
                if kvh:   # (the same runs as head 0's)
                    continue
                for t in range(kt, kt + cnt):
                    assert 0 <= 32 * t < L
                    keys = slice(32 * t, min(32 * t + 32, L))
                    for g in range(groups):
                        rows = slice(row0 + 32 * g, min(row0 + 32 * g + 32, T * group))
                        if rows.start >= rows.stop:
                            continue
                        block = see[r][rows, keys]
                        if bits >> g & 1 and not bits >> (4 + g) & 1:   # unmasked: whole, 32 stored keys
                            assert block.all() and 32 * t + 32 <= L
                        if not bits >> g & 1:
                            assert not block.any()
                        seen[r][rows, keys] += 1
            assert count == tiles
    for r, s in enumerate(seen):   # every visible pair in exactly one piece, no pair in two
        assert (s <= 1).all() and (s >= see[r]).all()
    assert all(len(x) == 1 for x in of_head.values())
    for (r, kvh, row0, groups), ps in pieces.items():
        assert len(ps) == ps[0][1] and (len(ps) > 1) == (ps[0][0] >= 0)
    rows = sorted((int(r), h, x) for r, T in enumerate(b.q_lens) for h in range(hkv) for x in range(T * group))
    got = sorted((r, h, x) for (r, h, row0, g) in pieces for x in range(row0, min(row0 + 32 * g, int(b.q_lens[r]) * group)))
    assert got == rows and (used <= 1).all()
    joins = lists[at[3] : at[3] + 8 * nj].reshape(-1, 8)
    joined = {(int(j[0]), int(j[1]), int(j[2]) + x) for j in joins for x in range(j[3])}
    assert joined == {(int(cu[r]), h, x) for (r, h, row0, g), ps in pieces.items() if len(ps) > 1 for x in range(row0, min(row0 + 32 * g, int(b.q_lens[r]) * group))}


def branches(counts, stored, page, device="cpu"):
    """-> batch, pages in all; request r: branches of counts[r] tokens each below stored[r] keys"""
    end, pos = [], []
    for lens, c in zip(counts, stored):
        for n in lens:
            end += [len(end) + n] * n
            pos += range(c, c + n)
    q_lens = [sum(lens) for lens in counts]
    kv_lens = [c + n for c, n in zip(stored, q_lens)]
    need = [-(-n // page) for n in kv_lens]
    tables = np.split(np.arange(sum(need)), np.cumsum(need)[:-1])
    return sa.PagedBatch.build(q_lens, kv_lens, [t.tolist() for t in tables], page, device, end=end, pos=pos), sum(need)


def by_the_kernels_rule(b, window, it, kt, bits, g, groups, group, N):
    """[rows, 32] bool: what a kernel lets row group g of an item see of tile kt, from the tile's bits: whole where the group has no masked bit; else the tokens up
    to a row's own, and where some group is masked and the tile holds new tokens of a tree, of these the ones whose subtree the row lies in"""
    cu, T, L, row0 = int(it[0]), int(it[1]), int(it[2]), int(it[5])
    c = L - T
    tok = np.arange(row0 + 32 * g, min(row0 + 32 * g + 32, N))[:, None] // group
    s = 32 * kt + np.arange(32)[None]
    if groups == 1 and not bits & 16 or groups > 1 and (bits >> g) & 17 == 1:
        return np.ones((len(tok), 32), bool)
    u = s - c
    see = u <= tok
    fresh = np.zeros_like(u, bool)
    at = s
    if b._end is not None and bits & 0xf0 and 32 * kt + 32 > c:
        fresh = u >= 0
        new = np.clip(u, 0, T - 1)
        see = see & (~fresh | (cu + tok < b._end[cu + new]))
        at = np.where(fresh, b._pos[cu + new], s)
    if window:
        place = c + tok if b._pos is None else b._pos[cu + tok]
        see = see & (place - at < window)
    return see


# branches that end on a row group's boundary inside an item, with tiles that lie wholly in an earlier one
BOUNDARIES = [  # branches, stored, page, (hq, hkv, d), window
    ([[80, 48]], [64], 64, (16, 8, 256), 0),
    ([[80, 48] * 5], [64], 64, (16, 8, 256), 0),
    ([[96] * 3, [48, 80]], [470, 32], 48, (16, 8, 128), 0),
    ([[80] * 4], [512], 16, (12, 12, 64), 0),
    ([[96, 64, 96]], [64], 32, (4, 2, 128), 70),
    ([[40, 24, 40]], [96], 16, (4, 1, 512), 0),
]


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("q_lens,kv_lens,page,heads,window,tree", [x for x in PLANS if x[5]] + [(c, s, p, h, w, None) for c, s, p, h, w in BOUNDARIES] + [PLANS[5], PLANS[3]])
def test_what_the_bits_of_a_tile_let_rows_see_is_the_dense_mask(q_lens, kv_lens, page, heads, window, tree, variant, monkeypatch):
    """every row group of an item computes all of its tiles, those it sees nothing of among them"""
    monkeypatch.setattr(paged, "VARIANT", variant)
    b, _ = branches(q_lens, kv_lens, page) if isinstance(q_lens[0], list) else make_batch(q_lens, kv_lens, page, tree=tree)
    hq, hkv, d = heads
    group = hq // hkv
    lists, (nw, nb, nr, _, _), at = b.plan(hq, hkv, d, window)
    lists = lists.numpy()
    runs = lists[at[2] : at[2] + 4 * nr].reshape(-1, 4)
    see = [np.repeat(x, group, 0) for x in dense(b, window)]
    for n, off, groups in ((nw, at[0], 1), (nb, at[1], 4)):
        for it in lists[off : off + 12 * n].reshape(-1, 12):
            if it[4]:   # (the same runs as head 0's)
                continue
            r, L, N = int(it[10]), int(it[2]), int(it[1]) * group
            for kt, cnt, bits, _ in runs[it[6] : it[6] + it[7]].tolist():
                for t in range(kt, kt + cnt):
                    for g in range(groups):
                        rows = slice(int(it[5]) + 32 * g, min(int(it[5]) + 32 * g + 32, N))
                        if rows.start < rows.stop:
                            got = by_the_kernels_rule(b, window, it, t, bits, g, groups, group, N)
                            assert np.array_equal(got[:, : L - 32 * t], see[r][rows, 32 * t : min(32 * t + 32, L)]) and not got[:, L - 32 * t :].any(), (r, rows, t, bits)


def test_a_request_is_cut_the_same_way_whatever_shares_the_call():
    alone, _ = make_batch([1], [5000], 64)
    both, _ = make_batch([300, 1, 1], [2000, 5000, 17], 64)

    def cuts(b, L):
        lists, counts, at = b.plan(8, 2, 128, 0)
        items = lists.numpy()[: 12 * counts[0]].reshape(-1, 12)
        runs = lists.numpy()[at[2] :].reshape(-1)[: 4 * counts[2]].reshape(-1, 4)
        return sorted((int(i[4]), int(i[11]), *runs[i[6] : i[6] + i[7], :3].reshape(-1).tolist()) for i in items if i[2] == L)

    assert cuts(alone, 5000) == cuts(both, 5000) and len(cuts(alone, 5000)) > 2


@pytest.mark.parametrize("variant,size", [(1, 16), (2, 48)])
def test_pieces_hold_at_least_half_of_their_size(variant, size, monkeypatch):
    monkeypatch.setattr(paged, "VARIANT", variant)
    for tiles in (1, size - 1, size, size + 1, 2 * size - 1, 2 * size + 1, 5 * size + 3):
        b, _ = make_batch([1], [32 * tiles], 16)
        lists, counts, at = b.plan(4, 1, 128, 0)
        n = counts[variant - 1]
        pieces = lists.numpy()[at[variant - 1] :][: 12 * n].reshape(-1, 12)[:, 8]
        assert n == -(-tiles // size) and pieces.sum() == tiles and pieces.max() - pieces.min() <= 1 and (n == 1 or pieces.min() >= size // 2)


def test_rows_slots_and_positions():
    b = sa.PagedBatch.build([2, 3, 2], [18, 1, 16], [[5, 2], [7], [9]], 16, "cpu")
    slots, pos = b.rows()
    assert slots.tolist() == [2 * 16, 2 * 16 + 1, -1, -1, 7 * 16, 9 * 16 + 14, 9 * 16 + 15] and slots.dtype == torch.int64
    assert pos.tolist() == [16, 17, 0, 0, 0, 14, 15] and pos.dtype == torch.int32
    for c in (copy.deepcopy(b), pickle.loads(pickle.dumps(b))):
        assert c.rows()[0].tolist() == slots.tolist() and c.plan(4, 2, 64, 0)[1] == b.plan(4, 2, 64, 0)[1]
    empty = sa.PagedBatch.build([], [], [], 16, "cpu")
    assert empty.rows()[0].numel() == 0 and empty.plan(4, 2, 64, 0)[1] == [0] * 5


def test_positions_of_trimmed_requests():
    """new tokens go on from their text's position, not from their place among the keys that stayed"""
    b = sa.PagedBatch.build([2, 1, 3], [10, 40, 5], [[0], [1, 2, 3], [4]], 16, "cpu", dropped=[90, 0, 7])
    slots, pos = b.rows()
    assert slots.tolist() == [8, 9, 3 * 16 + 7, 4 * 16 + 2, 4 * 16 + 3, 4 * 16 + 4] and pos.tolist() == [98, 99, 39, 9, 10, 11]
    tree = dict(q_lens=[3, 2], kv_lens=[13, 6], tables=[[0], [1]], page=16, device="cpu", end=[3, 2, 3, 4, 5], pos=[110, 111, 111, 4, 4])
    t = sa.PagedBatch.build(**tree, dropped=[100, 0])
    assert t.rows()[1].tolist() == [110, 111, 111, 4, 4]
    plain = sa.PagedBatch.build(**{**tree, "pos": [10, 11, 11, 4, 4]})
    assert torch.equal(t.plan(4, 2, 64, 0)[0], plain.plan(4, 2, 64, 0)[0]) and all(torch.equal(x, y) for x, y in zip(t.device_data(), plain.device_data()))
    for x in (b, t, plain):
        for c in (copy.deepcopy(x), pickle.loads(pickle.dumps(x))):
            assert c.rows()[0].tolist() == x.rows()[0].tolist() and c.rows()[1].tolist() == x.rows()[1].tolist()
    for bad in (dict(dropped=[100]), dict(dropped=[100, -1]), dict(dropped=[100, 0.5]), dict(dropped=[99, 0]), dict(dropped=[111, 0]), dict()):
        with pytest.raises(ValueError):
            sa.PagedBatch.build(**{**tree, **bad})
    c = sa.PagedCache.empty(8, 16, 2, 64, "cpu")
    q = torch.zeros((6, 4, 64), dtype=BF16)
    with pytest.raises(ValueError, match="trimmed"):
        sa.paged_attn(q, c, b, window=8)
    with pytest.raises(ValueError, match="trimmed"):
        sa.paged_weights(q, c, b, torch.zeros((6, 4)), window=8)
    with pytest.raises(RuntimeError, match="ROCm"):
        sa.paged_attn(q, c, b, window=0)


@pytest.mark.parametrize("bad", [
    dict(page=24), dict(page=0), dict(q_lens=[-1, 1]), dict(kv_lens=[20]), dict(tables=[[0, 1]]), dict(tables=[[0], [1]]), dict(tables=[[0, -1], [1]]),
    dict(tables=[[0, 1 << 31], [1]]), dict(end=[1, 2]), dict(end=[1, 3], pos=[19, 5]), dict(end=[1, 2], pos=[20, 5]), dict(end=[1], pos=[19]),
    dict(end=[1, 2, 3], pos=[19, 5, 6], q_lens=[1, 40]), dict(tables=[[0.5, 1.5], [1.0]]),
])
def test_batches_that_make_no_sense_are_refused(bad):
    good = dict(q_lens=[1, 1], kv_lens=[20, 6], tables=[[0, 1], [2]], page=16)
    sa.PagedBatch.build(**good, device="cpu", end=[1, 2], pos=[19, 5])
    with pytest.raises(ValueError):
        sa.PagedBatch.build(**{**good, **bad}, device="cpu")


@pytest.mark.parametrize("bad", [
    dict(q_lens=[1.5, 1]), dict(kv_lens=[20, 6.9]), dict(kv_lens=[float("nan"), 6]), dict(kv_lens=[float("inf"), 6]), dict(kv_lens=[2**32 + 20, 6]), dict(q_lens=[2**64 - 1, 1]),
    dict(kv_lens=np.array([2**63 + 20, 6], np.uint64)), dict(end=[1, 1.5]), dict(pos=[18.5, 5]), dict(page=16.5), dict(page=2**32 + 16), dict(page=(1 << 20) + 16),
])
def test_numbers_that_would_be_cut_are_refused(bad):
    good = dict(q_lens=[1, 1], kv_lens=[20, 6], tables=[[0, 1], [2]], page=16, end=[1, 2], pos=[19, 5])
    a = sa.PagedBatch.build(**good, device="cpu")
    b = sa.PagedBatch.build(**{**good, "q_lens": torch.tensor([1, 1]), "kv_lens": np.array([20.0, 6.0]), "page": np.int64(16), "end": np.array([1, 2], np.uint8)}, device="cpu")
    assert a.rows()[0].tolist() == b.rows()[0].tolist() and b.kv_lens.tolist() == [20, 6]
    with pytest.raises(ValueError):
        sa.PagedBatch.build(**{**good, **bad}, device="cpu")


def test_caches_that_the_kernels_do_not_take_are_refused():
    k = torch.zeros((4, 16, 2, 64), dtype=BF16)
    sa.PagedCache(k, k)
    for bad in (k.float(), k[:, :, :, ::2], k.transpose(2, 3), k[:, :8], torch.zeros((4, 16, 2, 96), dtype=BF16), torch.zeros((4, 16, 2, 68), dtype=BF16)[..., :64], k[0]):
        with pytest.raises(ValueError):
            sa.PagedCache(bad, bad)
    with pytest.raises(ValueError):
        sa.PagedCache(k, k[:2])
    c = sa.PagedCache.empty(3, 32, 2, 64, "cpu")
    assert c.k.shape == (3, 32, 2, 64) and c.k[0, :, 0].is_contiguous() and c.page == 32


def test_plan_and_attention_refuse_bad_arguments_at_the_c_entry(lib):
    h = C.c_void_p()
    assert lib.spinf_paged_plan_build(None, C.byref(h)) == -1
    lens = np.array([1, 4], np.int32)
    a = _lib.PagedPlanArgs(lens.ctypes.data, lens.ctypes.data, 2, None, None, 4, 2, 64, 16, 0, 0)
    assert lib.spinf_paged_plan_build(C.byref(a), None) == -1
    for field, value in (("hq", 3), ("hkv", 0), ("d", 96), ("page", 24), ("window", -1), ("variant", 3), ("reqs", -1), ("end", lens.ctypes.data), ("kv_lens", None)):
        x = _lib.PagedPlanArgs.from_buffer_copy(a)
        setattr(x, field, value)
        assert lib.spinf_paged_plan_build(C.byref(x), C.byref(h)) == -1, field
    assert lib.spinf_paged_plan_build(C.byref(a), C.byref(h)) == 0
    assert lib.spinf_paged_plan_export(h, None, None, None, None) == -1 and lib.spinf_paged_plan_counts(h, None) == -1
    lib.spinf_paged_plan_free(h)
    lib.spinf_paged_plan_free(None)
    assert lib.spinf_paged_attn_fwd(None, None) == -1
    b = _lib.PagedArgs()
    assert lib.spinf_paged_attn_fwd(C.byref(b), None) == 0   # nothing to do
    b.n_wave = 1
    assert lib.spinf_paged_attn_fwd(C.byref(b), None) == -1
    sizes = (C.c_int64 * 5)()
    assert lib.spinf_paged_struct_sizes(sizes, 5) == 0 and lib.spinf_paged_struct_sizes(sizes, 4) == -1
    assert list(sizes) == [C.sizeof(x) for x in (_lib.PagedPlanArgs, _lib.PagedArgs, _lib.RopeArgs, _lib.PagedWeightsArgs, _lib.EvictArgs)]


def test_attention_refuses_tensors_before_any_launch():
    b, pages = make_batch([2], [20], 16)
    c = sa.PagedCache.empty(pages, 16, 2, 64, "cpu")
    q = torch.zeros((2, 4, 64), dtype=BF16)
    with pytest.raises(RuntimeError, match="ROCm"):
        sa.paged_attn(q, c, b)
    for bad in (q.float(), q[:1], q[:, :3], torch.zeros((2, 4, 128), dtype=BF16), q[..., ::2], q[0]):
        with pytest.raises(ValueError):
            sa.paged_attn(bad, c, b)
    with pytest.raises(ValueError, match="page"):
        sa.paged_attn(q, sa.PagedCache.empty(pages, 32, 2, 64, "cpu"), b)
    with pytest.raises(ValueError, match="in a table"):
        sa.paged_attn(q, sa.PagedCache.empty(b.max_page, 16, 2, 64, "cpu"), b)
    with pytest.raises(ValueError, match="window"):
        sa.paged_attn(q, c, b, window=-3)


def test_windows_of_any_width_are_taken_for_what_they_are():
    b, _ = make_batch([70, 2], [300, 130], 16)
    none = b.plan(4, 2, 128, paged._window(None))
    for window in (1 << 30, 2**31 - 1, 2**31, 2**32 + 5, 2**70, np.int64(2**40), float(2**40)):
        lists, counts, at = b.plan(4, 2, 128, paged._window(window))
        assert counts == none[1] and torch.equal(lists, none[0]), window
    assert paged._window(5) == paged._window(np.int32(5)) == paged._window(5.0) == 5 and paged._window(0) == 0
    for window in (-1, -(2**32) + 5, 2.5, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            paged._window(window)


# ------------------------------------------------------------------------------------------------ attention on the GPU
def fill(batch, pages, heads, seed, device, peaky=True, order="heads"):
    """cache and queries of unit scale; order of the cache's memory: a head's rows of a page together, or a row's heads"""
    hq, hkv, d = heads
    g = torch.Generator().manual_seed(seed)
    shape = (pages, hkv, batch.page, d) if order == "heads" else (pages, batch.page, hkv, d)
    k, v = (torch.randn(shape, generator=g).to(BF16).to(device) for _ in range(2))
    if order == "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    q = torch.randn((batch.tokens, hq, d), generator=g)
    if peaky:
        q *= 1 + 3 * (torch.rand(batch.tokens, hq, 1, generator=g) < 0.2)
    return sa.PagedCache(k, v), q.to(BF16).to(device)


def reference(q, cache, batch, scale, window=0, softcap=0.0):
    """out, lse, and what the kernel's results may be off by"""
    qn, kn, vn = (t.float().cpu().numpy() for t in (q, cache.k, cache.v))
    d = qn.shape[2]
    out, lse, tol, ltol = [], [], [], []
    base = 0
    for r, see in enumerate(dense(batch, window)):
        T, L = see.shape
        at = int(batch._need[:r].sum())
        table = batch._table[at : at + batch._need[r]]
        o, s, mag, size = op.attention(qn[base : base + T].astype(np.float64), op.stored(kn, table, L), op.stored(vn, table, L), see, scale, softcap)
        # scores: d products summed in fp32, then scaled (and capped: the cap's slope is at most 1, its own error 2^-22 of the cap)
        terr = size * (d + 4) * 2.0**-24 + softcap * 2.0**-21 + 2.0**-20
        # probabilities: exp of the score's error, rounded to bf16 (8 significant bits: 2^-8); sums in fp32; the output's own rounding to bf16
        out.append(o)
        lse.append(s)
        tol.append(1.02 * (2.0**-8 * (mag + np.abs(o)) + mag * (2 * terr[..., None] + (L + 64) * 2.0**-24)) + 1e-30)
        ltol.append(terr + (L + 64) * 2.0**-24 + np.where(np.isfinite(s), np.abs(s), 0) * 2.0**-22)
        base += T
    return tuple(np.concatenate(x) for x in (out, lse, tol, ltol))


def close(got, want, tol):
    got = got.float().cpu().numpy().astype(np.float64)
    assert got.shape == want.shape
    with np.errstate(invalid="ignore"):
        off = np.where(got == want, 0, np.abs(got - want))
    worst = float(np.nanmax(np.where(tol > 0, off / np.maximum(tol, 1e-300), 0), initial=0))
    ok = bool((off <= tol).all())
    assert ok, f"worst {worst} of the bound, {int((~(off <= tol)).sum())} values"


ATTN = [  # q_lens, kv_lens, page, (hq, hkv, d), window, softcap, tree
    ([1], [1], 16, (4, 4, 64), 0, 0.0, None),
    ([1, 1, 1, 1], [0, 33, 700, 32], 16, (8, 2, 128), 0, 0.0, None),
    ([1, 2], [2100, 130], 48, (16, 1, 512), 0, 0.0, None),
    ([1, 1], [1500, 64], 64, (24, 4, 256), 0, 30.0, None),
    ([1, 4], [3001, 257], 80, (12, 12, 64), 0, 0.0, None),
    ([1, 1], [3001, 40], 16, (10, 2, 128), 300, 20.0, None),
    ([5, 40, 0, 129], [2, 100, 7, 129], 32, (6, 2, 64), 0, 0.0, None),
    ([200, 64], [457, 64], 80, (4, 2, 128), 0, 0.0, None),
    ([200, 1, 33], [457, 900, 300], 48, (4, 2, 256), 100, 50.0, None),
    ([70, 70], [70, 400], 16, (4, 4, 64), 1, 0.0, None),
    ([60, 90], [361, 90], 64, (4, 2, 256), 0, 0.0, (1, 9)),
    ([60, 90], [361, 151], 48, (10, 2, 64), 40, 0.0, (4, 24)),
    ([10, 14], [70, 151], 16, (2, 1, 512), 0, 0.0, (2, 5)),
    ([3, 6], [470, 35], 16, (4, 2, 128), 30, 10.0, (1, 3)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("variant,order", [(1, "heads"), (2, "rows")])
@pytest.mark.parametrize("q_lens,kv_lens,page,heads,window,softcap,tree", ATTN)
def test_attention_against_the_oracle(dev, q_lens, kv_lens, page, heads, window, softcap, tree, variant, order, monkeypatch):
    """either kernel on every case, whichever the rule would take"""
    monkeypatch.setattr(paged, "VARIANT", variant)
    b, pages = make_batch(q_lens, kv_lens, page, dev, tree)
    cache, q = fill(b, pages, heads, 1, dev, order=order)
    scale = heads[2] ** -0.5
    out, lse = sa.paged_attn(q, cache, b, window=window or None, softcap=softcap or None, return_lse=True)
    want, wlse, tol, ltol = reference(q, cache, b, scale, window, softcap)
    close(out, want, tol)
    close(lse, wlse, ltol)
    assert torch.equal(out, sa.paged_attn(q, cache, b, scale, window, softcap))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("q_lens,kv_lens,page,heads,window,tree", [
    ([1, 3], [45, 130], 16, (4, 2, 128), 0, None),
    ([40, 70], [90, 70], 48, (4, 2, 64), 25, None),
    ([50, 20], [130, 33], 16, (4, 2, 256), 0, (1, 9)),
    ([9], [40], 32, (2, 1, 512), 0, (2, 5)),
])
def test_what_a_row_does_not_see_leaves_no_trace(dev, q_lens, kv_lens, page, heads, window, tree, variant, monkeypatch):
    """NaN and infinities behind the stored keys, in other requests' pages and in new tokens that some rows do not see: those rows' results stay what they are, and
    only rows that see such a key are not finite"""
    monkeypatch.setattr(paged, "VARIANT", variant)
    b, pages = make_batch(q_lens, kv_lens, page, dev, tree)
    cache, q = fill(b, pages, heads, 3, dev)
    clean = sa.paged_attn(q, cache, b, window=window or None)
    slots, _ = b.rows()
    stored = torch.zeros(pages * page, dtype=torch.bool, device=dev)
    at = 0
    for n, L in zip(b._need, b.kv_lens):
        s = np.arange(L)
        stored[torch.from_numpy(b._table[at : at + n][s // page].astype(np.int64) * page + s % page).to(dev)] = True
        at += n
    rubbish = ~stored.view(pages, page)
    for t, x in ((cache.k, float("nan")), (cache.v, float("inf"))):
        t[rubbish] = x
    assert torch.equal(sa.paged_attn(q, cache, b, window=window or None), clean)
    # one request's last-but-one new token turns into NaN / inf: the rows that do not see it keep their values (to rounding: they may be computed row by row)
    row = int(b.q_lens[0]) - 2 if b.q_lens[0] > 1 else int(b.tokens) - 2
    slot = int(slots[row])
    cache.k[slot // page, slot % page] = float("nan")
    cache.v[slot // page, slot % page] = float("-inf")
    out, lse = sa.paged_attn(q, cache, b, window=window or None, return_lse=True)
    base = np.cumsum(b.q_lens) - b.q_lens
    touched = np.zeros(b.tokens, bool)
    for r, see in enumerate(dense(b, window)):
        T, L = see.shape
        if base[r] <= row < base[r] + T:
            touched[base[r] : base[r] + T] = see[:, L - T + row - base[r]]
    touched = torch.from_numpy(touched).to(dev)
    assert touched.any() and not touched.all()
    assert out[touched].isnan().all() and lse[touched].isnan().all()
    keep = clean[~touched].float()
    # twice what rounding may cost: probabilities to bf16 in one computation and not in the other, values at most 5 (unit scale, these sizes)
    assert torch.isfinite(out[~touched]).all() and ((out[~touched].float() - keep).abs() <= 2.0**-8 * (5 + keep.abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("counts,stored,page,heads,window", BOUNDARIES)
def test_branches_that_end_inside_an_item_against_the_oracle(dev, counts, stored, page, heads, window, variant, monkeypatch):
    monkeypatch.setattr(paged, "VARIANT", variant)
    b, pages = branches(counts, stored, page, dev)
    cache, q = fill(b, pages, heads, 17, dev)
    out, lse = sa.paged_attn(q, cache, b, window=window or None, return_lse=True)
    want, wlse, tol, ltol = reference(q, cache, b, heads[2] ** -0.5, window)
    close(out, want, tol)
    close(lse, wlse, ltol)


@pytest.mark.gpu
def test_a_request_has_the_same_bits_whatever_shares_the_call(dev):
    heads = (8, 2, 128)
    b, pages = make_batch([1, 300, 37, 2], [4100, 700, 1500, 65], 64, dev)
    cache, q = fill(b, pages, heads, 5, dev)
    out = sa.paged_attn(q, cache, b)
    tables = np.split(b._table, np.cumsum(b._need)[:-1])
    base = 0
    for r, (T, L) in enumerate(zip(b.q_lens, b.kv_lens)):
        one = sa.PagedBatch.build([T], [L], [tables[r]], 64, dev)
        assert torch.equal(sa.paged_attn(q[base : base + T], cache, one), out[base : base + T])
        base += T


# many rows at 512 dims (halves that exchange their scores): chunks, a window with a cap, trees, keys cut into pieces, two key / value heads
HALVES = [
    ([33, 9], [700, 9], 48, (16, 1, 512), 200, 30.0, None),
    ([70, 1], [70, 40], 16, (4, 2, 512), 0, 0.0, None),
    ([30, 22], [130, 60], 16, (8, 1, 512), 40, 0.0, (2, 8)),
    ([40], [3300], 64, (4, 1, 512), 0, 0.0, None),
]
# pieces per row: a few up to more than four times the groups that a join's rows may have; few rows and many
PIECES = [
    ([3, 1], [1100, 2600], 16, (4, 1, 64), 0, 0.0, None),
    ([9], [3600], 48, (4, 1, 128), 0, 20.0, None),
    ([5, 2], [7000, 4400], 64, (3, 1, 64), 0, 0.0, None),
    ([1], [13000], 16, (6, 1, 64), 0, 0.0, None),
    ([2], [35000], 64, (1, 1, 64), 0, 0.0, None),
    ([150], [3300], 64, (2, 1, 128), 0, 0.0, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("q_lens,kv_lens,page,heads,window,softcap,tree", HALVES + PIECES)
def test_halves_and_pieces_against_the_oracle(dev, q_lens, kv_lens, page, heads, window, softcap, tree, variant, monkeypatch):
    test_attention_against_the_oracle(dev, q_lens, kv_lens, page, heads, window, softcap, tree, variant, "heads", monkeypatch)


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,kv_lens,window,tree", [([50, 20], [130, 33], 0, (1, 9)), ([40, 70], [90, 70], 25, None)])
def test_halves_leave_no_trace_of_unseen_keys(dev, q_lens, kv_lens, window, tree, monkeypatch):
    test_what_a_row_does_not_see_leaves_no_trace(dev, q_lens, kv_lens, 16, (4, 1, 512), window, tree, 2, monkeypatch)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("q_lens,kv_lens,page,hq,tree,variant", [
    ([3], [700], 16, 4, None, 1), ([9, 2], [1100, 40], 48, 4, None, 1), ([8], [900], 16, 16, (2, 4), 1), ([60, 2], [3400, 40], 64, 4, None, 2),
])
def test_halves_of_pieces_with_rubbish_in_one_of_them(dev, q_lens, kv_lens, page, hq, tree, variant, half, bad, monkeypatch):
    """keys cut into pieces, and a value that is not finite in one half of 512 dims alone: the rows that do not see it keep both halves"""
    monkeypatch.setattr(paged, "VARIANT", variant)
    b, pages = make_batch(q_lens, kv_lens, page, dev, tree)
    cache, q = fill(b, pages, (hq, 1, 512), 41, dev)
    assert b.plan(hq, 1, 512, 0)[1][3]
    clean = sa.paged_attn(q, cache, b)
    row = int(b.q_lens[0]) - 1
    slot = int(b.rows()[0][row])
    cache.v[slot // page, slot % page, 0, 256 * half : 256 * half + 256] = bad
    out = sa.paged_attn(q, cache, b)
    see = dense(b, 0)[0]
    touched = np.zeros(b.tokens, bool)
    touched[: see.shape[0]] = see[:, see.shape[1] - see.shape[0] + row]
    touched = torch.from_numpy(touched).to(dev)
    assert touched.any() and not touched.all()
    keep = clean[~touched].float()
    # as above: probabilities to bf16 in one computation and not in the other, values at most 5
    assert torch.isfinite(out[~touched]).all() and ((out[~touched].float() - keep).abs() <= 2.0**-8 * (5 + keep.abs())).all()
    halves = out[touched].unflatten(2, (2, 256))
    assert not torch.isfinite(halves[:, :, half]).any() and torch.isfinite(halves[:, :, 1 - half]).all()


def test_joins_cover_every_row_of_cut_keys():
    """share: groups of 16 lanes per row, a power of two, the fewest that ask for a row's pieces four at a time (16 at most)"""
    for n, hq, hkv, d in ((1100, 4, 1, 64), (3600, 8, 2, 128), (9000, 16, 1, 512), (40000, 3, 1, 64), (90000, 24, 4, 256)):
        b, _ = make_batch([3], [n], 16)
        lists, counts, at, _ = b._compile(hq, hkv, d, 0, 0)
        joins = lists[at[3] : at[3] + 8 * counts[3]].reshape(-1, 8)
        assert len(joins)
        rows = sorted((int(j[1]), int(j[2]) + x) for j in joins for x in range(j[3]))
        assert rows == [(h, r) for h in range(hkv) for r in range(3 * hq // hkv)]
        for _, _, _, count, part, pieces, stride, share in joins.tolist():
            assert share in (1, 2, 4, 8, 16) and 1 <= count <= 16 // share
            assert share == 16 or 4 * share >= pieces and (share == 1 or 2 * share < pieces)
            assert 0 <= part and part + count + (pieces - 1) * stride <= counts[4]


@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 512])
def test_strided_queries_and_a_single_key(dev, d):
    b, pages = make_batch([3, 40], [3, 61], 16, dev)
    heads = (4, 2, d)
    cache, q = fill(b, pages, heads, 6, dev)
    wide = torch.zeros((b.tokens, 9, d + 8), dtype=BF16, device=dev)
    wide[:, 3:7, :d] = q
    assert torch.equal(sa.paged_attn(wide[:, 3:7, :d], cache, b), sa.paged_attn(q, cache, b))
    one = sa.PagedBatch.build([1], [1], [[2]], 16, dev)   # a row that sees one key is that key's value
    assert torch.equal(sa.paged_attn(q[:1], cache, one)[0], cache.v[2, 0].repeat_interleave(2, 0))
    none = sa.PagedBatch.build([2], [0], [[]], 16, dev)
    out, lse = sa.paged_attn(q[:2], cache, none, return_lse=True)
    assert not out.any() and (lse == float("-inf")).all()
    empty = sa.PagedBatch.build([0, 0], [0, 5], [[], [1]], 16, dev)
    assert sa.paged_attn(q[:0], cache, empty).shape == (0, 4, d)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [1, 2])
def test_scores_that_range_widely(dev, variant, monkeypatch):
    """the running maximum rises late and by much, and stays finite where exp alone would not"""
    monkeypatch.setattr(paged, "VARIANT", variant)
    b, pages = make_batch([2, 33], [700, 500], 64, dev)
    cache, q = fill(b, pages, (4, 2, 128), 8, dev)
    cache.k.mul_(torch.linspace(0.1, 12, pages, device=dev).to(BF16)[:, None, None, None])
    q = q * 4
    out, lse = sa.paged_attn(q, cache, b, return_lse=True)
    want, wlse, tol, ltol = reference(q, cache, b, 128**-0.5)
    close(out, want, tol)
    close(lse, wlse, ltol)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [1, 2])
def test_a_window_wider_than_every_request_is_none(dev, variant, monkeypatch):
    monkeypatch.setattr(paged, "VARIANT", variant)
    b, pages = make_batch([70, 2], [300, 130], 16, dev)
    cache, q = fill(b, pages, (4, 2, 128), 46, dev)
    want, lse = sa.paged_attn(q, cache, b, return_lse=True)
    weight = sa.paged_weights(q, cache, b, lse)
    for window in (1 << 30, 2**31 - 30, 2**31 - 1, 2**31, 2**32 + 5):
        assert torch.equal(sa.paged_attn(q, cache, b, window=window), want), window
        got = sa.paged_weights(q, cache, b, lse, window=window)
        assert torch.equal(got, weight), window
    # the C entry by itself, with the widest window that its 32 bits hold
    lists, counts, at = b.plan(4, 2, 128, 1 << 30)
    a = paged._attn_block(q, cache.k, cache.v, *b.device_data(), lists, counts, at, 16, b.max_page, b.tokens, 128**-0.5, 2**31 - 1, 0.0)
    assert torch.equal(paged._attn_run(a, q, cache.k, cache.v, False)[0], want)


CAPS = [0.5, 3.0, 30.0, 50.0, 1e3, 1e4, 1e5, 1e6, 1e7, 1e30, 2e38]


def capped(q, cache, batch, scale, softcap):
    """as `reference`, with no more allowed than the scores' own digits: the cap's tanh is off by some 2^-22 of a score, taken as 2^-20"""
    qn, kn, vn = (t.float().cpu().numpy() for t in (q, cache.k, cache.v))
    out, lse, tol, ltol = [], [], [], []
    base = 0
    for r, see in enumerate(dense(batch, 0)):
        T, L = see.shape
        at = int(batch._need[:r].sum())
        table = batch._table[at : at + batch._need[r]]
        o, s, mag, size = op.attention(qn[base : base + T].astype(np.float64), op.stored(kn, table, L), op.stored(vn, table, L), see, scale, softcap)
        terr = size * ((qn.shape[2] + 4) * 2.0**-24 + 2.0**-20) + 2.0**-20
        out.append(o)
        lse.append(s)
        tol.append(1.02 * (2.0**-8 * (mag + np.abs(o)) + mag * (2 * terr[..., None] + (L + 64) * 2.0**-24)) + 1e-30)
        ltol.append(terr + (L + 64) * 2.0**-24 + np.where(np.isfinite(s), np.abs(s), 0) * 2.0**-22)
        base += T
    return tuple(np.concatenate(x) for x in (out, lse, tol, ltol))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("softcap", CAPS)
@pytest.mark.parametrize("heads", [(4, 2, 128), (4, 1, 512), (8, 2, 64), (4, 2, 256)])
def test_caps_of_every_size(dev, softcap, variant, heads, monkeypatch):
    monkeypatch.setattr(paged, "VARIANT", variant)
    b, pages = make_batch([1, 40], [900, 130], 64, dev)
    cache, q = fill(b, pages, heads, 43, dev)
    out, lse = sa.paged_attn(q, cache, b, softcap=softcap, return_lse=True)
    want, wlse, tol, ltol = capped(q, cache, b, heads[2] ** -0.5, softcap)
    close(lse, wlse, ltol)
    close(out, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", CAPS)
def test_weights_under_caps_of_every_size(dev, softcap):
    b, pages = make_batch([3, 40], [900, 130], 64, dev)
    heads = (4, 2, 128)
    cache, q = fill(b, pages, heads, 44, dev)
    scale = heads[2] ** -0.5
    lse = torch.from_numpy(capped(q, cache, b, scale, softcap)[1].astype(np.float32)).to(dev)
    got = sa.paged_weights(q, cache, b, lse, softcap=softcap)
    qn, kn, ln = q.double().cpu().numpy(), cache.k.float().cpu().numpy(), lse.double().cpu().numpy()
    base = 0
    for r, see in enumerate(dense(b, 0)):
        T, L = see.shape
        at = int(b._need[:r].sum())
        k = op.stored(kn, b._table[at : at + b._need[r]], L)
        rows = slice(base, base + T)
        want = op.weights(qn[rows], k, see, ln[rows], scale, softcap)
        size = max(float((np.abs(qn[rows, h]) @ np.abs(k[:, h // 2]).T).max()) for h in range(4)) * scale
        rel = size * ((heads[2] + 4) * 2.0**-24 + 2.0**-20) + (T * 2 + 40) * 2.0**-24 + 2.0**-20
        close(got[r, :, :L], want, rel * want + 1e-30)
        base += T


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("softcap", [0.5, 2.0])
def test_infinite_scores_weigh_what_the_cap_leaves_them(dev, softcap, variant, monkeypatch):
    """keys of -inf, a request's first page of them: scores of minus the cap, seen like others"""
    monkeypatch.setattr(paged, "VARIANT", variant)
    heads = (4, 2, 128)
    b, pages = make_batch([2, 40], [130, 90], 32, dev)
    cache, q = fill(b, pages, heads, 45, dev)
    q = q.abs() + 0.01
    for r in range(2):
        cache.k[int(b._table[int(b._need[:r].sum())])] = float("-inf")
    out, lse = sa.paged_attn(q, cache, b, softcap=softcap, return_lse=True)
    qn, kn, vn = (t.float().cpu().numpy().astype(np.float64) for t in (q, cache.k, cache.v))
    base = 0
    for r, see in enumerate(dense(b, 0)):
        T, L = see.shape
        at = int(b._need[:r].sum())
        table = b._table[at : at + b._need[r]]
        rows = slice(base, base + T)
        o, s, mag, _ = op.attention(qn[rows], op.stored(kn, table, L), op.stored(vn, table, L), see, 128**-0.5, softcap)
        # scores of at most 2: their errors are far below 2^-16
        close(out[rows], o, 1.02 * 2.0**-8 * (mag + np.abs(o)) + mag * 2.0**-14)
        close(lse[rows], s, 2.0**-15 + 0 * s)
        base += T


@pytest.mark.gpu
def test_scales_and_caps_outside_the_range_are_refused(dev):
    b, pages = make_batch([2], [20], 16, dev)
    cache, q = fill(b, pages, (4, 2, 64), 0, dev)
    for bad in (dict(scale=3e38), dict(softcap=1e-39, scale=1.0), dict(softcap=float("inf")), dict(softcap=float("nan"))):
        with pytest.raises(ValueError):
            sa.paged_attn(q, cache, b, **bad)
        with pytest.raises(ValueError):
            sa.paged_weights(q, cache, b, torch.zeros((2, 4), device=dev), **bad)


# ------------------------------------------------------------------------------------------------ weights
WEIGHTS = [  # q_lens, kv_lens, page, (hq, hkv, d), window, softcap, tree
    ([1, 1, 0, 1], [1, 700, 33, 32], 16, (8, 2, 128), 0, 0.0, None),
    ([1], [2100], 48, (16, 1, 512), 0, 0.0, None),
    ([64, 5, 40], [457, 5, 2], 80, (4, 2, 256), 0, 30.0, None),
    ([33, 70], [400, 300], 64, (12, 12, 64), 50, 0.0, None),
    ([60, 20], [361, 35], 48, (10, 2, 64), 0, 0.0, (1, 9)),
    ([60, 20], [100, 35], 32, (4, 2, 128), 12, 0.0, (4, 24)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("q_lens,kv_lens,page,heads,window,softcap,tree", WEIGHTS)
def test_weights_against_the_oracle(dev, q_lens, kv_lens, page, heads, window, softcap, tree):
    b, pages = make_batch(q_lens, kv_lens, page, dev, tree)
    cache, q = fill(b, pages, heads, 11, dev)
    scale = heads[2] ** -0.5
    _, lse = sa.paged_attn(q, cache, b, scale, window, softcap, return_lse=True)
    longest = int(b.kv_lens.max())
    acc = torch.rand((len(b.kv_lens), heads[1], longest + 5), device=dev)
    got = sa.paged_weights(q, cache, b, lse, scale, window, softcap, acc=acc)
    bare = sa.paged_weights(q, cache, b, lse, scale, window, softcap)
    assert got.shape == acc.shape and bare.shape == (len(b.kv_lens), heads[1], longest)
    qn, kn, ln = q.double().cpu().numpy(), cache.k.float().cpu().numpy(), lse.double().cpu().numpy()
    base = 0
    for r, see in enumerate(dense(b, window)):
        T, L = see.shape
        at = int(b._need[:r].sum())
        k = op.stored(kn, b._table[at : at + b._need[r]], L)
        rows = slice(base, base + T)
        want = op.weights(qn[rows], k, see, ln[rows], scale, softcap)
        # each weight: the score's error (d products in fp32) and exp2's, sums of T x group terms in fp32
        group = heads[0] // heads[1]
        size = max([float((np.abs(qn[rows, h]) @ np.abs(k[:, h // group]).T).max(initial=0)) for h in range(heads[0])], default=0) * scale
        rel = size * (heads[2] + 4) * 2.0**-24 + softcap * 2.0**-21 + (T * group + 40) * 2.0**-24 + 2.0**-20
        a = acc[r].double().cpu().numpy()
        close(bare[r, :, :L], want, rel * want + 1e-30)
        close(got[r, :, :L], a[:, :L] + want, rel * want + 2.0**-23 * (a[:, :L] + want))
        assert torch.equal(got[r, :, L:], acc[r, :, L:]) and not bare[r, :, L:].any()
        # what every row gave away sums to one
        seen = see.any(1)
        assert abs(float(bare[r].double().sum()) - seen.sum() * heads[0]) <= seen.sum() * heads[0] * (2 * rel + 1e-5)
        base += T


@pytest.mark.gpu
def test_weights_of_rubbish_that_nobody_sees(dev):
    b, pages = make_batch([2, 1], [20, 45], 16, dev)
    cache, q = fill(b, pages, (4, 2, 64), 12, dev)
    _, lse = sa.paged_attn(q, cache, b, return_lse=True)
    want = sa.paged_weights(q, cache, b, lse)
    slot = int(b.rows()[0][1])     # the request's last token: its first row does not see it
    other = torch.ones(pages, dtype=torch.bool)
    other[b._table.astype(np.int64)] = False
    cache.k[other.to(dev)] = float("nan")
    cache.k[int(b._table[1]), 4:] = float("nan")   # behind the first request's 20 keys
    assert torch.equal(sa.paged_weights(q, cache, b, lse), want)
    q0, lse0 = q.clone(), lse.clone()
    lse0[1] = float("-inf")                        # a row that counts as one that saw nothing
    cache.k[slot // 16, slot % 16] = float("nan")
    got = sa.paged_weights(q0, cache, b, lse0)
    assert torch.isfinite(got[0, :, :19]).all()


def test_weights_and_eviction_refuse_bad_arguments():
    b, pages = make_batch([2, 1], [40, 20], 16)
    c = sa.PagedCache.empty(pages, 16, 2, 64, "cpu")
    q, lse = torch.zeros((3, 4, 64), dtype=BF16), torch.zeros((3, 4))
    with pytest.raises(RuntimeError, match="ROCm"):
        sa.paged_weights(q, c, b, lse)
    with pytest.raises(ValueError):
        sa.paged_weights(q[:2], c, b, lse)
    free = sorted(set(range(pages)) - set(b._table.tolist()))
    into = sa.PagedBatch.build([0, 0], [16, 16], [free[:1], free[1:2]], 16, "cpu")
    acc = torch.zeros((2, 2, 40))
    with pytest.raises(RuntimeError, match="ROCm"):
        sa.cache_evict(c, b, into, acc, 16, 4, 4)
    bad = sa.PagedBatch.build([0, 0], [16, 16], [free[:1], b._table[:1]], 16, "cpu")
    twice = sa.PagedBatch.build([0, 0], [16, 16], [free[:1], free[:1]], 16, "cpu")
    short = sa.PagedBatch.build([0, 0], [16, 15], [free[:1], free[1:2]], 16, "cpu")
    one = sa.PagedBatch.build([0], [16], [free[:1]], 16, "cpu")
    for x in (bad, twice, short, one):
        with pytest.raises(ValueError):
            sa.cache_evict(c, b, x, acc, 16, 4, 4)
    for args in ((acc[:, :, :39], 16, 4, 4), (acc.double(), 16, 4, 4), (acc[:1], 16, 4, 4), (acc, 16, 14, 4), (acc, 16, -1, 4), (acc, -1, 0, 0)):
        with pytest.raises(ValueError):
            sa.cache_evict(c, b, into, *args)


def test_eviction_refuses_counts_that_32_bits_or_whole_numbers_do_not_hold():
    b, pages = make_batch([2, 1], [40, 20], 16)
    c = sa.PagedCache.empty(pages + 4, 16, 2, 64, "cpu")
    into = sa.PagedBatch.build([0, 0], [40, 16], [[pages, pages + 1, pages + 2], [pages + 3]], 16, "cpu")
    acc = torch.zeros((2, 2, 40))
    with pytest.raises(RuntimeError, match="ROCm"):   # (all is well but the device)
        sa.cache_evict(c, b, into, acc, 16.0, np.int64(4), 4)
    for args in ((2**32 + 16, 4, 4), (2**30 + 1, 4, 4), (16, 2**32 + 4, 4), (16, 4, 2**32), (2**40, 2**32, 2**32), (16.5, 4, 4), (16, 0.5, 4), (16, 4, 3.5), (float("inf"), 0, 0)):
        with pytest.raises(ValueError):
            sa.cache_evict(c, b, into, acc, *args)


# ------------------------------------------------------------------------------------------------ eviction
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "wild"])
@pytest.mark.parametrize("kv_lens,keep,sink,recent,page,hkv,d", [
    ([900, 40, 33], 40, 4, 7, 16, 2, 64), ([5000, 0, 1], 64, 0, 0, 48, 1, 128), ([130, 129], 128, 4, 64, 64, 3, 256), ([300], 90, 0, 90, 32, 2, 512), ([77, 500], 1, 0, 0, 16, 2, 64),
    ([20000], 7777, 1, 2, 80, 1, 64),
])
def test_eviction_against_the_oracle(dev, kv_lens, keep, sink, recent, page, hkv, d, kind):
    R, longest = len(kv_lens), max(kv_lens)
    rng = np.random.default_rng(4)
    need, new = [-(-n // page) for n in kv_lens], [-(-min(n, keep) // page) for n in kv_lens]
    pages = sum(need) + sum(new) + 2
    ids = rng.permutation(pages)
    cut = np.cumsum(need + new)
    parts = np.split(ids, cut)[: 2 * R]
    b = sa.PagedBatch.build([0] * R, kv_lens, parts[:R], page, dev)
    into = sa.PagedBatch.build([0] * R, [min(n, keep) for n in kv_lens], parts[R:], page, dev)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn((pages, page, hkv, d), generator=g).to(BF16).to(dev) for _ in range(2))
    cache = sa.PagedCache(k, v)
    acc = torch.rand((R, hkv, longest + 3), generator=g) ** 4
    if kind == "ties":
        acc = (acc * 6).floor() / 6
    elif kind == "equal":
        acc = torch.full_like(acc, 0.25)
    elif kind == "wild":   # both signs and zeros, infinities, NaN, subnormals
        acc = torch.randn(acc.shape, generator=g)
        pick = torch.randint(0, 12, acc.shape, generator=g)
        for i, x in enumerate((float("inf"), float("-inf"), float("nan"), 0.0, -0.0, 1e-42, -1e-42)):
            acc[pick == i] = x
    before = k.clone(), v.clone()
    accd = acc.to(dev)
    kept, new_acc = sa.cache_evict(cache, b, into, accd, keep, sink, recent)
    assert kept.shape == new_acc.shape == (R, hkv, keep)
    wk, wv = (t.clone() for t in before)
    for r, n in enumerate(kv_lens):
        m = min(n, keep)
        for h in range(hkv):
            places = op.keep_places(acc[r, h].numpy(), n, keep, sink, recent)
            assert kept[r, h].tolist() == places.tolist() + [-1] * (keep - m), (r, h)
            assert np.array_equal(new_acc[r, h].cpu().numpy(), np.concatenate([acc[r, h].numpy()[places], np.zeros(keep - m, np.float32)]), equal_nan=True)
            src, dst = parts[r][places // page], parts[R + r][np.arange(m) // page]
            src, dst, e, f = (torch.from_numpy(np.ascontiguousarray(x)).to(dev) for x in (src, dst, places % page, np.arange(m) % page))
            for t, old in ((wk, before[0]), (wv, before[1])):
                t[dst, f, h] = old[src, e, h]
    assert torch.equal(k, wk) and torch.equal(v, wv)   # the kept rows, in order, and nothing else


# ------------------------------------------------------------------------------------------------ norms and rotation
ROPE = [  # tokens, hq, hkv, d, rot, neighbours, plus_one, tables, weights, pos
    (1, 4, 2, 64, 64, False, False, torch.float32, BF16, torch.int32),
    (37, 24, 4, 256, 64, False, True, BF16, BF16, torch.int64),
    (1000, 16, 8, 256, 256, False, False, torch.float32, torch.float32, None),
    (130, 10, 2, 128, 32, True, True, torch.float32, BF16, torch.int32),
    (65, 16, 1, 512, 512, True, False, BF16, None, torch.int64),
    (9, 3, 3, 64, 16, False, False, torch.float32, BF16, None),
    (5, 5, 1, 128, 0, False, False, torch.float32, BF16, None),
]


def rope_case(dev, T, hq, hkv, d, rot, tables, weights, pos, seed=0):
    g = torch.Generator().manual_seed(seed)
    y = torch.randn((T, (hq + 2 * hkv) * d + 8), generator=g).mul_(torch.rand((T, 1), generator=g) * 4).to(BF16).to(dev)
    q, k, v = (t.unflatten(1, (-1, d)) for t in y[:, 8:].split([hq * d, hkv * d, hkv * d], 1))
    w = [None, None] if weights is None else [(1 + 0.3 * torch.randn(d, generator=g)).to(weights).to(dev) for _ in range(2)]
    n = 500 if pos is not None else T
    ang = torch.rand((n, rot // 2), generator=g) * 6.3
    full = torch.cat([ang, ang], 1)    # as models hand them over: both halves, of which the first is passed
    cos, sin = (f(full).to(tables).to(dev)[:, : rot // 2] for f in (torch.cos, torch.sin))
    p = None if pos is None else torch.randint(0, n, (T,), generator=g).to(pos).to(dev)
    return q, k, v, *w, cos, sin, p


def rope_want(x, w, cos, sin, p, eps, neighbours, plus_one):
    f = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    at = np.arange(x.shape[0]) if p is None else p.cpu().numpy()
    want = op.norm_rope(f(x), f(w), f(cos)[at], f(sin)[at], eps, neighbours, plus_one)
    # fp32 arithmetic (a sum of d squares, some ten roundings, of terms no larger than the pair's length), then one rounding to bf16
    size = np.abs(op.norm_rope(f(x), f(w), np.zeros_like(f(cos)[at]), np.ones_like(f(sin)[at]), eps, neighbours, plus_one)) + np.abs(
        op.norm_rope(f(x), f(w), np.ones_like(f(cos)[at]), np.zeros_like(f(sin)[at]), eps, neighbours, plus_one))
    return want, 2.0**-8 * np.abs(want) + (x.shape[2] / 2 + 24) * 2.0**-24 * 1.5 * size + 1e-30


@pytest.mark.gpu
@pytest.mark.parametrize("T,hq,hkv,d,rot,neighbours,plus_one,tables,weights,pos", ROPE)
def test_norm_and_rotation_against_the_oracle(dev, T, hq, hkv, d, rot, neighbours, plus_one, tables, weights, pos):
    q, k, v, wq, wk, cos, sin, p = rope_case(dev, T, hq, hkv, d, rot, tables, weights, pos)
    got = sa.qk_norm_rope(q, k, wq, wk, cos, sin, 1e-6, p, neighbours, plus_one)
    for x, w, y in zip((q, k), (wq, wk), got):
        assert y.is_contiguous() and y.dtype == BF16
        close(y, *rope_want(x, w, cos, sin, p, 1e-6, neighbours, plus_one))
    # with the cache: the same queries, the keys and values at their places, everything else as it was
    page = 16
    pages = -(-T // page) + 2
    g = torch.Generator().manual_seed(9)
    slots = torch.randperm(pages * page, generator=g)[:T].to(dev)
    if T > 3:
        slots[1] = -1
        slots[2] = pages * page
    for v_norm in (False, True):
        cache = sa.PagedCache.empty(pages, page, hkv, d, dev)
        cache.k.fill_(7)
        cache.v.fill_(5)
        q2 = sa.qk_norm_rope_put(q, k, v, wq, wk, cos, sin, 1e-6, cache, slots, p, neighbours, plus_one, v_norm)
        inside = (slots >= 0) & (slots < pages * page)
        wantk, wantv = torch.full_like(cache.k, 7), torch.full_like(cache.v, 5)
        s = slots[inside]
        wantk[s // page, s % page] = got[1][inside]
        wantv[s // page, s % page] = v[inside]
        assert torch.equal(cache.k, wantk)
        if not v_norm:
            assert torch.equal(cache.v, wantv)
        else:
            want, tol = rope_want(v, None, cos[:, :0], sin[:, :0], p, 1e-6, False, False)
            i = inside.cpu().numpy()
            close(cache.v[s // page, s % page], want[i], tol[i])
            rest = torch.ones(pages * page, dtype=torch.bool, device=dev)
            rest[s] = False
            assert (cache.v.flatten(0, 1)[rest] == 5).all()
        known = slots < pages * page
        assert torch.equal(q2[known], got[0][known]) and q2[~known].isnan().all()


@pytest.mark.gpu
def test_rows_that_say_so_themselves(dev):
    """a position outside the tables: a query and a key of NaN, the value as it is; a row of zeros, of infinities, of NaN"""
    q, k, v, wq, wk, cos, sin, _ = rope_case(dev, 5, 4, 2, 64, 32, torch.float32, BF16, torch.int32)
    pos = torch.tensor([0, -1, 500, 499, 3], device=dev)
    got = sa.qk_norm_rope(q, k, wq, wk, cos, sin, 1e-6, pos)
    for y in got:
        assert y[1:3].isnan().all() and torch.isfinite(y[[0, 3, 4]]).all()
    q = q.clone()
    q[0] = 0
    q[3, 1] = float("inf")
    q[4, 2, 5] = float("nan")
    a, b = sa.qk_norm_rope(q, k, wq, wk, cos, sin, 1e-6, pos)
    assert not a[0].any() and torch.equal(b[[0, 3, 4]], got[1][[0, 3, 4]])
    assert torch.equal(a[3, [0, 2, 3]], got[0][3, [0, 2, 3]]) and a[4, 2].isnan().all() and torch.equal(a[4, [0, 1, 3]], got[0][4, [0, 1, 3]])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 256])
def test_rows_whose_mean_square_is_subnormal(dev, d):
    q, k, v, wq, wk, cos, sin, p = rope_case(dev, 9, 4, 2, d, 32, torch.float32, BF16, torch.int32, seed=3)
    q, k = q.clone(), k.clone()
    for t in (q, k):
        t.mul_(2.0**-64)
    got = sa.qk_norm_rope(q, k, wq, wk, cos, sin, 0.0, p)
    for x, w, y in zip((q, k), (wq, wk), got):
        want, tol = rope_want(x, w, cos, sin, p, 0.0, False, False)
        # squares of up to 2^-124 in steps of 2^-149: their mean, of 2^-132 and more here, is off by 2^-17 at most
        assert float((x.double() ** 2).mean(-1).min()) > 2.0**-132
        close(y, want, tol + 2.0**-17 * np.abs(want) + 2.0**-17 * np.abs(want).max(-1, keepdims=True))


def test_norm_and_rotation_refuse_bad_arguments():
    q, k, w, c = torch.zeros((3, 4, 64), dtype=BF16), torch.zeros((3, 2, 64), dtype=BF16), torch.zeros(64), torch.zeros((3, 16))
    with pytest.raises(RuntimeError, match="ROCm"):
        sa.qk_norm_rope(q, k, w, w, c, c, 1e-6)


@pytest.mark.gpu
def test_norm_and_rotation_refuse_tensors_before_any_launch(dev):
    q, k, w, c = (t.to(dev) for t in (torch.zeros((3, 4, 64), dtype=BF16), torch.zeros((3, 2, 64), dtype=BF16), torch.zeros(64), torch.zeros((3, 16))))
    good = dict(q=q, k=k, wq=w, wk=w, cos=c, sin=c, eps=1e-6, pos=None)
    sa.qk_norm_rope(**good)
    with pytest.raises(RuntimeError, match="ROCm"):   # (the same call elsewhere is not a known one)
        sa.qk_norm_rope(**{n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in good.items()})
    for one in ("q", "k", "wq", "wk", "cos", "sin"):
        with pytest.raises((RuntimeError, ValueError)):
            sa.qk_norm_rope(**{**good, one: good[one].cpu()})
    for one in ("q", "k"):   # the same strides, another alignment
        t = torch.zeros(good[one].numel() + 8, dtype=BF16, device=dev)[1 : 1 + good[one].numel()].view(good[one].shape)
        with pytest.raises(ValueError, match="aligned"):
            sa.qk_norm_rope(**{**good, one: t})
    long = torch.zeros((3, 40), device=dev)
    for bad in (dict(q=q.float()), dict(q=q[:2]), dict(k=k[..., ::2]), dict(wq=w[:32]), dict(wq=w.half()), dict(wq=w.to(BF16)), dict(cos=c.double()), dict(sin=c[:, :8]),
                dict(cos=c[:2], sin=c[:2]), dict(cos=long, sin=long), dict(cos=c[:, :4], sin=c[:, :4]), dict(pos=torch.zeros(2, dtype=torch.int64, device=dev)),
                dict(pos=torch.zeros(3, device=dev)), dict(eps=-1.0), dict(eps=float("nan")), dict(wq=w.cpu()), dict(cos=torch.zeros((3, 17), device=dev)[:, 1:], sin=c),
                dict(q=torch.zeros((3, 4, 96), dtype=BF16, device=dev), k=torch.zeros((3, 2, 96), dtype=BF16, device=dev))):
        with pytest.raises(ValueError):
            sa.qk_norm_rope(**{**good, **bad})
    cache, slots = sa.PagedCache.empty(2, 16, 2, 64, dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for bad in (dict(slots=slots.int()), dict(slots=slots[:2]), dict(v=k[:2]), dict(cache=sa.PagedCache.empty(2, 16, 2, 128, dev)), dict(cache=sa.PagedCache.empty(2, 16, 1, 64, dev)),
                dict(cache=sa.PagedCache.empty(0, 16, 2, 64, dev))):
        with pytest.raises(ValueError):
            sa.qk_norm_rope_put(**{**good, "v": k, "cache": cache, "slots": slots, **bad})


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.gpu
def test_streams_compiled_programs_and_recorded_graphs(dev):
    heads = (8, 2, 128)
    b, pages = make_batch([1, 70], [900, 300], 64, dev)
    cache, q = fill(b, pages, heads, 21, dev)
    acc = torch.rand((2, 2, 900), device=dev)
    want, lse = sa.paged_attn(q, cache, b, return_lse=True)
    weight = sa.paged_weights(q, cache, b, lse, acc=acc)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    fresh = pickle.loads(pickle.dumps(b))      # its uploads are made on the default stream, then used on another
    fresh.device_data()
    with torch.cuda.stream(side):
        assert torch.equal(sa.paged_attn(q, cache, fresh), want)
        assert torch.equal(sa.paged_weights(q, cache, fresh, lse, acc=acc), weight)
    torch.cuda.synchronize()
    torch.library.opcheck(torch.ops.spinf.paged_weights.default, (q, cache.k, lse, acc, *[b.device_data()[0], b.device_requests(), None, None], 64, b.max_page, b.tokens, 70, 900, 2, 900, 0.1, 0, 0.0),
                          test_utils=("test_schema", "test_faketensor"))
    lists, counts, at = b.plan(8, 2, 128, 0)
    torch.library.opcheck(torch.ops.spinf.paged_attn.default, (q, cache.k, cache.v, b.device_data()[0], None, None, lists, counts, at, 64, b.max_page, b.tokens, 0.1, 0, 0.0, True),
                          test_utils=("test_schema", "test_faketensor"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, l2 = sa.paged_attn(q, cache, b, return_lse=True)
        w2 = sa.paged_weights(q, cache, b, l2, acc=acc)
    for seed in range(3):
        q.copy_(fill(b, pages, heads, 30 + seed, dev)[1])
        graph.replay()
        torch.cuda.synchronize()
        e, el = sa.paged_attn(q, cache, b, return_lse=True)
        assert torch.equal(out, e) and torch.equal(l2, el) and torch.equal(w2, sa.paged_weights(q, cache, b, el, acc=acc))
        torch.cuda.synchronize()


class Layer:
    """one pass through all of the operators, over a cache that `fresh` puts back"""

    def __init__(self, dev):
        g = torch.Generator().manual_seed(7)
        self.heads = (8, 2, 128)
        self.b, pages = make_batch([1, 70], [900, 300], 64, dev, spare=12)
        self.cache, self.q = fill(self.b, pages, self.heads, 21, dev)
        self.k, self.v = (torch.randn((71, 2, 128), generator=g).to(BF16).to(dev) for _ in range(2))
        self.w = torch.rand(128, generator=g).to(dev)
        ang = torch.rand((1000, 32), generator=g).to(dev)
        self.cos, self.sin = ang.cos(), ang.sin()
        self.slots, self.pos = self.b.rows()
        free = sorted(set(range(pages)) - set(self.b._table.tolist()))
        self.into = sa.PagedBatch.build([0, 0], [200, 200], [free[:4], free[4:8]], 64, dev)
        self.acc = torch.rand((2, 2, 900), generator=g).to(dev)
        self.kept = self.cache.k.clone(), self.cache.v.clone()
        self.want = self.run(self.q, self.k, self.v, self.acc)
        self.left = self.cache.k.clone(), self.cache.v.clone()
        self.fresh()

    def fresh(self):
        self.cache.k.copy_(self.kept[0])
        self.cache.v.copy_(self.kept[1])

    def run(self, q, k, v, acc):
        a, c = sa.qk_norm_rope(q, k, self.w, self.w, self.cos, self.sin, 1e-6, self.pos)
        y = sa.qk_norm_rope_put(q, k, v, self.w, self.w, self.cos, self.sin, 1e-6, self.cache, self.slots, self.pos)
        out, lse = sa.paged_attn(y, self.cache, self.b, return_lse=True)
        weight = sa.paged_weights(y, self.cache, self.b, lse, acc=acc)
        return (a, c, y, out, lse, weight, *sa.cache_evict(self.cache, self.b, self.into, weight, 200, 4, 8))

    def check(self, got):
        assert all(torch.equal(x, y) for x, y in zip((*got, self.cache.k, self.cache.v), (*self.want, *self.left)))


@pytest.mark.gpu
def test_the_registered_operators_of_the_cache(dev):
    """schemas (what they write among it) and shapes without memory"""
    x, tests, ops = Layer(dev), ("test_schema", "test_faketensor"), torch.ops.spinf
    table = (x.w, x.w, x.cos, x.sin, 1e-6)
    torch.library.opcheck(ops.qk_norm_rope.default, (x.q, x.k, *table, x.pos, False, False), test_utils=tests)
    torch.library.opcheck(ops.qk_norm_rope_put.default, (x.q, x.k, x.v, *table, x.cache.k, x.cache.v, x.slots, x.pos, False, False, False), test_utils=tests)
    old, new = x.b._device(), x.into._device()
    torch.library.opcheck(ops.cache_evict.default, (x.cache.k, x.cache.v, x.acc, old[1], old[0], new[1], new[0], 64, 200, 4, 8), test_utils=tests)


@pytest.mark.gpu
def test_a_compiled_pass_over_the_cache(dev):
    x = Layer(dev)
    torch._dynamo.reset()
    try:
        compiled = torch.compile(x.run, backend="aot_eager")
        for _ in range(2):
            x.check(compiled(x.q, x.k, x.v, x.acc))
            x.fresh()
    finally:
        torch._dynamo.reset()
    x.check(x.run(x.q, x.k, x.v, x.acc))


@pytest.mark.gpu
def test_a_recorded_pass_over_the_cache(dev):
    x = Layer(dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = x.run(x.q, x.k, x.v, x.acc)
    for seed in range(3):
        x.q.copy_(fill(x.b, x.cache.k.shape[0], x.heads, 50 + seed, dev)[1])
        x.fresh()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*out, x.cache.k, x.cache.v)]
        x.fresh()
        assert all(torch.equal(a, b) for a, b in zip(got, (*x.run(x.q, x.k, x.v, x.acc), x.cache.k, x.cache.v)))
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_host_threads_share_a_batch(dev):
    """first calls of four threads, each on a stream of its own"""
    import threading

    x = Layer(dev)
    want, lse = sa.paged_attn(x.q, x.cache, x.b, return_lse=True)
    weight = sa.paged_weights(x.q, x.cache, x.b, lse)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(10):
        b, start, got = pickle.loads(pickle.dumps(x.b)), threading.Barrier(4), [None] * 4

        def run(i):
            with torch.cuda.stream(streams[i]):
                start.wait(60)
                for _ in range(3):
                    out, l2 = sa.paged_attn(x.q, x.cache, b, return_lse=True)
                    w2 = sa.paged_weights(x.q, x.cache, b, l2)
                streams[i].synchronize()
            got[i] = out, l2, w2, b.rows()[0]

        threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for t in got for a, c in zip(t, (want, lse, weight, x.slots)))


@pytest.mark.gpu
def test_a_session_equals_reading_anew(dev):
    """examples/paged_session.py: documents, later questions and tokens over the cache against tree_attn over the whole stream"""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_session.py")
    spec = importlib.util.spec_from_file_location("paged_session", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    off = module.main(dev)
    # values of unit scale (at most about 5): two computations' probabilities and outputs, each rounded to bf16 once
    assert all(off[x] <= 4 * 2.0**-8 * 5 for x in ("documents", "questions", "steps")), off
    assert off["weights"] <= 1e-4, off


@pytest.mark.gpu
def test_questions_below_a_trimmed_content(dev):
    """examples/paged_session.py's last step: rotation goes on at the text's position; the keys that stayed and nothing else are seen"""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_session.py")
    spec = importlib.util.spec_from_file_location("paged_session", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    # values of unit scale (at most about 5); probabilities and outputs rounded to bf16 once, and the projections of two calls may round apart
    assert module.main(dev, steps=1, keep=100)["trimmed"] <= 4 * 2.0**-8 * 5


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """pages whose bytes begin beyond 2^32, read, written and moved"""
    page, hkv, d = 64, 8, 256
    pages = (5 << 30) // (page * hkv * d * 2)
    cache = sa.PagedCache.empty(pages, page, hkv, d, dev)
    small = sa.PagedCache.empty(12, page, hkv, d, dev)
    g = torch.Generator().manual_seed(3)
    for a, b in ((small.k, cache.k), (small.v, cache.v)):
        a.copy_(torch.randn(a.shape, generator=g).to(BF16))
        b[-12:] = a
    far = [pages - 12 + i for i in range(12)]
    q = torch.randn((70, 16, d), generator=g).to(BF16).to(dev)
    make = lambda ids: sa.PagedBatch.build([1, 69], [250, 130], [ids[:4], ids[4:7]], page, dev)  # noqa: E731
    near, there = make(list(range(12))), make(far)
    want, lse = sa.paged_attn(q, small, near, return_lse=True)
    assert torch.equal(sa.paged_attn(q, cache, there), want)
    w = sa.paged_weights(q, small, near, lse)
    assert torch.equal(sa.paged_weights(q, cache, there, lse), w)
    outs = []
    for c, b, ids in ((small, near, list(range(12))), (cache, there, far)):
        into = sa.PagedBatch.build([0, 0], [100, 100], [ids[7:9], ids[9:11]], page, dev)
        outs.append((sa.cache_evict(c, b, into, w, 100, 4, 8), c.k[ids].clone(), c.v[ids].clone()))
    assert all(torch.equal(x, y) for x, y in zip((*outs[0][0], *outs[0][1:]), (*outs[1][0], *outs[1][1:])))
    ang = torch.rand((3, 32), generator=g).to(dev)
    k, v = (torch.randn((3, hkv, d), generator=g).to(BF16).to(dev) for _ in range(2))
    for c, ids in ((small, list(range(12))), (cache, far)):
        slots = torch.tensor([ids[11] * page, ids[11] * page + 63, ids[0] * page + 5], device=dev)
        sa.qk_norm_rope_put(q[:3], k, v, None, None, ang.cos(), ang.sin(), 1e-6, c, slots)
    assert torch.equal(small.k, cache.k[-12:]) and torch.equal(small.v, cache.v[-12:])


@pytest.mark.gpu
def test_calls_refuse_what_the_kernels_do_not_take(dev):
    b, pages = make_batch([2], [20], 16, dev)
    cache, q = fill(b, pages, (4, 2, 64), 0, dev)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(softcap=-2.0), dict(window=-1)):
        with pytest.raises(ValueError):
            sa.paged_attn(q, cache, b, **bad)
        with pytest.raises(ValueError):
            sa.paged_weights(q, cache, b, torch.zeros((2, 4), device=dev), **bad)
    with pytest.raises(RuntimeError, match="ROCm"):
        sa.paged_attn(q.cpu(), cache, b)
    odd = torch.zeros((2, 4, 65), dtype=BF16, device=dev)[..., 1:]
    with pytest.raises(ValueError, match="aligned"):
        sa.paged_attn(odd, cache, b)
    for lse in (torch.zeros((2, 4), device=dev).double(), torch.zeros((2, 3), device=dev), torch.zeros((4, 2), device=dev).t(), torch.zeros((2, 4))):
        with pytest.raises(ValueError):
            sa.paged_weights(q, cache, b, lse)
    for acc in (torch.zeros((1, 2, 19), device=dev), torch.zeros((1, 4, 20), device=dev), torch.zeros((1, 2, 20), device=dev).double()):
        with pytest.raises(ValueError):
            sa.paged_weights(q, cache, b, torch.zeros((2, 4), device=dev), acc=acc)
    fresh = pickle.loads(pickle.dumps(b))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="recorded"):
        with torch.cuda.graph(graph):
            sa.paged_attn(q, cache, fresh)
    torch.cuda.synchronize()
    assert torch.equal(sa.paged_attn(q, cache, fresh), sa.paged_attn(q, cache, b))
