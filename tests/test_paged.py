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


def test_a_request_is_cut_the_same_way_whatever_shares_the_call():
    alone, _ = make_batch([1], [5000], 64)
    both, _ = make_batch([300, 1, 1], [2000, 5000, 17], 64)

    def cuts(b, L):
        lists, counts, at = b.plan(8, 2, 128, 0)
        items = lists.numpy()[: 12 * counts[0]].reshape(-1, 12)
        runs = lists.numpy()[at[2] :].reshape(-1)[: 4 * counts[2]].reshape(-1, 4)
        return sorted((int(i[4]), int(i[11]), *runs[i[6] : i[6] + i[7], :3].reshape(-1).tolist()) for i in items if i[2] == L)

    assert cuts(alone, 5000) == cuts(both, 5000) and len(cuts(alone, 5000)) > 2


def test_rows_slots_and_positions():
    b = sa.PagedBatch.build([2, 3, 2], [18, 1, 16], [[5, 2], [7], [9]], 16, "cpu")
    slots, pos = b.rows()
    assert slots.tolist() == [2 * 16, 2 * 16 + 1, -1, -1, 7 * 16, 9 * 16 + 14, 9 * 16 + 15] and slots.dtype == torch.int64
    assert pos.tolist() == [16, 17, 0, 0, 0, 14, 15] and pos.dtype == torch.int32
    for c in (copy.deepcopy(b), pickle.loads(pickle.dumps(b))):
        assert c.rows()[0].tolist() == slots.tolist() and c.plan(4, 2, 64, 0)[1] == b.plan(4, 2, 64, 0)[1]
    empty = sa.PagedBatch.build([], [], [], 16, "cpu")
    assert empty.rows()[0].numel() == 0 and empty.plan(4, 2, 64, 0)[1] == [0] * 5


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
    sizes = (C.c_int64 * 2)()
    assert lib.spinf_paged_struct_sizes(sizes, 2) == 0 and lib.spinf_paged_struct_sizes(sizes, 3) == -1
    assert list(sizes) == [C.sizeof(_lib.PagedPlanArgs), C.sizeof(_lib.PagedArgs)]


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
