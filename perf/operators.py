"""What is timed of the paged cache's operators: the calls a service makes that keeps the keys and values of contents it has read.

  rope     norms and rotation of a layer's queries and keys, the keys and values into their places in the cache
  attn     attention of new tokens over the cache: single tokens, chunks, and trees of questions below a stored content
  weights  the attention weight that stored keys received from new tokens, added to what they had before
  evict    the stored keys with the least weight dropped, the others moved together into other pages

A case is a dict of plain values.  ``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the public
calls of spinf_serve_amd.  Lengths, trees and page tables belong to the case; the seed draws the tensors.
"""

from __future__ import annotations

import os
import sys
import zlib

import numpy as np
import torch

own = False
DEV = "cuda"


def _package():
    at = os.path.join(os.getcwd(), "spinf-serve_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import spinf_serve_amd

    return spinf_serve_amd


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of 48 requests in a hybrid model: a quarter of 256 dims rotated, tables in bf16, weights about zero
        _rope("rope_step", tokens=48, hq=24, hkv=4, d=256, rot=64, put=True, page=64, plus_one=True, tables="bf16"),
        # the headline pass of the benchmark (27k tokens), 16 / 8 heads of 256, values normed too
        _rope("rope_pass", tokens=27452, hq=16, hkv=8, d=256, rot=256, put=True, page=64, v_norm=True, tables="fp32"),
        # one request's 24 questions below a stored content of 301 tokens: latency
        _attn("attn_request", reqs=1, stored=301, tree="star", branches=24, lo=4, hi=24, hq=16, hkv=8, d=256, page=64),
        # the benchmark's headline pass with its 24 contents stored before: 56 questions each
        _attn("attn_pass", reqs=24, stored=470, tree="star", branches=56, lo=8, hi=16, hq=16, hkv=8, d=256, page=64),
        # long documents read in chunks: the second 8k of two of them, 128-dim heads
        _attn("attn_chunk", reqs=2, stored=8192, new=8192, hq=32, hkv=16, d=128, page=128),
        # chunks of a sliding layer with capped scores, pages that end inside a tile, odd lengths
        _attn("attn_sliding", reqs=7, stored=4099, spread=0.3, new=517, hq=16, hkv=8, d=256, page=48, window=1024, softcap=50.0),
        # one decoding step of a busy server: 64 requests of very different lengths
        _attn("attn_step", reqs=64, stored=3000, spread=0.7, new=1, hq=24, hkv=4, d=256, page=64),
        # one decoding step of a single long document on a layer with one key / value head of 512 dims
        _attn("attn_long_step", reqs=1, stored=131071, new=1, hq=16, hkv=1, d=512, page=16),
        # the weights of a decoding step
        _weights("weights_step", reqs=16, stored=2500, spread=0.5, new=1, hq=16, hkv=8, d=256, page=64),
        # the weights that the last 64 tokens of long prompts gave to all of them
        _weights("weights_prompt", reqs=4, stored=16001, spread=0.2, new=64, hq=32, hkv=16, d=128, page=64),
        # one short request trimmed, and a server's long ones
        _evict("evict_request", reqs=1, stored=900, keep=512, sink=4, recent=64, hkv=8, d=256, page=64),
        _evict("evict_server", reqs=16, stored=12000, spread=0.4, keep=4096, sink=4, recent=256, hkv=8, d=128, page=64),
    ]


def _rope(name, tokens, hq, hkv, d, rot, put=False, page=64, neighbours=False, plus_one=False, v_norm=False, tables="fp32"):
    return dict(name=name, kind="rope", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, put=put, page=page, neighbours=neighbours, plus_one=plus_one, v_norm=v_norm, tables=tables)


def _attn(name, reqs, stored, hq, hkv, d, page, spread=0.0, new=0, tree="", branches=0, lo=0, hi=0, window=0, softcap=0.0):
    return dict(name=name, kind="attn", reqs=reqs, stored=stored, spread=spread, new=new, tree=tree, branches=branches, lo=lo, hi=hi,
                hq=hq, hkv=hkv, d=d, page=page, window=window, softcap=softcap)


def _weights(name, **kw):
    return dict(_attn(name, **kw), kind="weights")


def _evict(name, reqs, stored, keep, sink, recent, hkv, d, page, spread=0.0, ties=False):
    return dict(name=name, kind="evict", reqs=reqs, stored=stored, spread=spread, keep=keep, sink=sink, recent=recent, hkv=hkv, d=d, page=page, ties=ties)


HEADS = [(16, 8, 256), (16, 1, 512), (24, 4, 256), (32, 16, 128), (16, 4, 64), (12, 12, 64), (10, 2, 128)]


def _log(rng, a, b):
    """a whole number, spread over the logarithm of a .. b"""
    return min(b, max(a, int(round(a * (b / a) ** rng.random()))))


def draw(rng):
    """one more case of these ranges, costing no more than the largest listed one"""
    kind = rng.choice(["rope", "attn", "attn", "attn", "weights", "evict"])
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice([16, 32, 48, 64, 80, 128])
    if kind == "rope":
        rot = rng.choice([d, d, d // 2, d // 4])
        c = _rope("", tokens=_log(rng, 1, 24000), hq=hq, hkv=hkv, d=d, rot=rot, put=rng.random() < 0.6, page=page, neighbours=rng.random() < 0.3,
                  plus_one=rng.random() < 0.4, v_norm=rng.random() < 0.4, tables=rng.choice(["fp32", "bf16"]))
    elif kind == "evict":
        stored = _log(rng, 24, 40000)
        keep = max(8, int(stored * rng.uniform(0.1, 0.9)))
        c = _evict("", reqs=min(_log(rng, 1, 32), max(1, 100000 // stored)), stored=stored, spread=rng.choice([0.0, 0.5]), keep=keep, sink=rng.randint(0, 4),
                   recent=rng.randint(0, keep // 4), hkv=hkv, d=min(d, 256), page=page, ties=rng.random() < 0.4)
    else:
        form = rng.choice(["step", "chunk", "tree"]) if kind == "attn" else rng.choice(["step", "chunk"])
        window = rng.choice([0, 0, 256, 1024]) if d <= 256 else 0
        more = dict(hq=hq, hkv=hkv, d=d, page=page, spread=rng.choice([0.0, 0.6]), window=window, softcap=rng.choice([0.0, 0.0, 30.0]))
        if form == "step":
            stored = _log(rng, 1, 100000)
            c = _attn("", reqs=min(_log(rng, 1, 96), max(1, 150000 // stored)), stored=stored, new=rng.choice([1, 1, 1, 2, 4]), **more)
        elif form == "chunk":
            stored, new = _log(rng, 1, 12000), _log(rng, 5, 4096 if kind == "attn" else 96)
            c = _attn("", reqs=min(_log(rng, 1, 24), max(1, 16000 // (stored + new) * 4096 // max(new, 512))), stored=stored, new=new, **more)
        else:
            lo = rng.randint(1, 12)
            c = _attn("", reqs=_log(rng, 1, 24), stored=_log(rng, 16, 2048), tree=rng.choice(["star", "trie"]), branches=_log(rng, 2, 64), lo=lo, hi=lo + rng.randint(0, 12), **more)
        c["kind"] = kind
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ lengths, trees, pages: from the case alone
def _shape(case):
    """-> new tokens by request, stored keys by request (the new ones included), subtree ends and depths of the rows of trees (else None)"""
    g = np.random.default_rng(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    q_lens, kv_lens, end, pos = [], [], [], []
    for r in range(case["reqs"]):
        stored = int(np.clip(round(case["stored"] * (np.exp(case["spread"] * g.standard_normal()) if case["spread"] else 1.0)), 0, 2 * case["stored"]))
        new = case.get("new", 0)
        if case.get("tree"):
            lens = g.integers(case["lo"], case["hi"] + 1, case["branches"])
            open_rows, base, level = [], sum(q_lens), 0
            ends, depths = [], []
            for n in lens:   # a branch hangs on the content, or in tries also on a branch before it (pre-order)
                level = int(g.integers(0, min(level + 1, 5) + 1)) if case["tree"] == "trie" and ends else 0
                level = min(level, len(open_rows))
                while len(open_rows) > level:
                    for i in open_rows.pop():
                        ends[i] = base + len(ends)
                first, start = len(ends), (depths[open_rows[-1][-1]] + 1 if open_rows else stored)
                open_rows.append(list(range(first, first + int(n))))
                ends += [0] * int(n)
                depths += range(start, start + int(n))
            while open_rows:
                for i in open_rows.pop():
                    ends[i] = base + len(ends)
            new = len(ends)
            end += ends
            pos += depths
        q_lens.append(new)
        kv_lens.append(stored + new)
    return q_lens, kv_lens, (np.array(end, np.int64) if case.get("tree") else None), (np.array(pos, np.int64) if case.get("tree") else None)


def _tables(case, lens, first=0):
    """a page table per request: pages from `first` on, in an order as a busy allocator leaves them"""
    need = [-(-n // case["page"]) for n in lens]
    g = np.random.default_rng(7 + sum(need))
    ids = first + g.permutation(sum(need))
    cut = np.cumsum([0] + need)
    return [ids[a:b].tolist() for a, b in zip(cut[:-1], cut[1:])]


def _normal(gen, *shape, std=1.0):
    out = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
    flat = out.view(-1)
    for a in range(0, flat.numel(), 1 << 27):
        part = flat[a : a + (1 << 27)]
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV) * std)
    return out


def _pages(gen, pages, page, hkv, d):
    """keys and values as normed projections have them: unit scale, one key in fifty that draws more weight"""
    k, v = _normal(gen, pages, hkv, page, d), _normal(gen, pages, hkv, page, d)
    k *= (1 + 1.5 * (torch.rand((pages, hkv, page, 1), generator=gen, device=DEV) < 0.02)).to(torch.bfloat16)
    return k.transpose(1, 2), v.transpose(1, 2)   # [pages, page, hkv, d], a head's rows of a page next to each other


# ------------------------------------------------------------------------------------------------ what a program has before the call
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(case=case, scale=case["d"] ** -0.5)
    if case["kind"] == "rope":
        return _prepare_rope(state, case, gen)
    q_lens, kv_lens, end, pos = _shape(case)
    tables = _tables(case, kv_lens)
    pages = sum(map(len, tables))
    keep = case.get("keep", 0)
    into = _tables(case, [min(n, keep) for n in kv_lens], first=pages) if keep else []
    hkv, d, page = case["hkv"], case["d"], case["page"]
    k, v = _pages(gen, max(1, pages + sum(map(len, into))), page, hkv, d)
    state.update(q_lens=q_lens, kv_lens=kv_lens, end=end, pos=pos, tables=tables, into=into, k=k, v=v,
                 places=[torch.tensor(t, dtype=torch.int64, device=DEV) for t in tables], new_places=[torch.tensor(t, dtype=torch.int64, device=DEV) for t in into])
    if keep:
        n = max(kv_lens)
        acc = torch.rand((len(kv_lens), hkv, n), generator=gen, device=DEV) ** 4   # a few keys hold most of the weight
        if case["ties"]:
            acc = (acc * 8).floor() / 8
        state["acc"] = acc
    else:
        state["q"] = _normal(gen, sum(q_lens), case["hq"], d)
    if case["kind"] == "weights":
        state["acc"] = torch.rand((len(kv_lens), hkv, max(kv_lens)), generator=gen, device=DEV)
        state["lse"] = torch.cat([_softmax(*x)[1] for x in _scores(state, torch.float32)])
    if own:
        sa = _package()
        state["cache"] = sa.PagedCache(k, v)
        state["batch"] = sa.PagedBatch.build(q_lens, kv_lens, tables, page, DEV, end=end, pos=pos)
        if keep:
            state["into_batch"] = sa.PagedBatch.build([0] * len(kv_lens), [min(n, keep) for n in kv_lens], into, page, DEV)
    return state


def _prepare_rope(state, case, gen):
    T, hq, hkv, d, rot = (case[x] for x in ("tokens", "hq", "hkv", "d", "rot"))
    y = _normal(gen, T, (hq + 2 * hkv) * d)   # the projection's output: queries, keys and values side by side
    state["q"], state["k"], state["v"] = (t.unflatten(1, (-1, d)) for t in y.split([hq * d, hkv * d, hkv * d], 1))
    base = 0.0 if case["plus_one"] else 1.0
    state["wq"], state["wk"] = ((base + 0.2 * torch.randn(d, generator=gen, device=DEV)).to(torch.bfloat16) for _ in range(2))
    ang = torch.arange(4096, device=DEV)[:, None] * 10000.0 ** (-torch.arange(rot // 2, device=DEV) / (rot // 2))[None]
    dt = torch.float32 if case["tables"] == "fp32" else torch.bfloat16
    state["cos"], state["sin"] = ang.cos().to(dt), ang.sin().to(dt)
    state["pos"] = torch.randint(0, 4096, (T,), generator=gen, device=DEV, dtype=torch.int32)
    if case["put"]:
        page = case["page"]
        pages = -(-T // page) + 3
        state["slots"] = torch.randperm(pages * page, generator=gen, device=DEV)[:T].contiguous()
        state["ck"], state["cv"] = _pages(gen, pages, page, hkv, d)
        if own:
            state["cache"] = _package().PagedCache(state["ck"], state["cv"])
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else _run_plain)(s, s["case"])


def _run_own(s, c):
    sa = _package()
    if c["kind"] == "rope":
        how = dict(pos=s["pos"], neighbours=c["neighbours"], plus_one=c["plus_one"])
        if c["put"]:
            q = sa.qk_norm_rope_put(s["q"], s["k"], s["v"], s["wq"], s["wk"], s["cos"], s["sin"], 1e-6, s["cache"], s["slots"], v_norm=c["v_norm"], **how)
            return q, s["ck"], s["cv"]
        return sa.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], 1e-6, **how)
    if c["kind"] == "attn":
        return sa.paged_attn(s["q"], s["cache"], s["batch"], s["scale"], window=c["window"] or None, softcap=c["softcap"] or None)
    if c["kind"] == "weights":
        return sa.paged_weights(s["q"], s["cache"], s["batch"], s["lse"], s["scale"], window=c["window"] or None, softcap=c["softcap"] or None, acc=s["acc"])
    kept, acc = sa.cache_evict(s["cache"], s["batch"], s["into_batch"], s["acc"], c["keep"], sink=c["sink"], recent=c["recent"])
    return kept, acc, s["k"], s["v"]


def _run_plain(s, c):
    if c["kind"] == "rope":
        T, hq, hkv = c["tokens"], c["hq"], c["hkv"]
        q, k = (_norm_rope(s[x], s["w" + x], s, c) for x in "qk")
        if not c["put"]:
            return q.bfloat16(), k.bfloat16()
        v = s["v"].float()
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) if c["v_norm"] else v
        at = (s["slots"] // c["page"], s["slots"] % c["page"])
        s["ck"][at], s["cv"][at] = k.bfloat16(), v.bfloat16()
        return q.bfloat16(), s["ck"], s["cv"]
    if c["kind"] == "attn":
        return torch.cat([_softmax(*x)[0] for x in _scores(s, torch.float32, values=True)])
    if c["kind"] == "weights":
        return _add_weights(s, torch.float32)
    return _evict_plain(s, c)


def _norm_rope(x, w, s, c, dt=torch.float32):
    x = x.to(dt)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (w.to(dt) + (1 if c["plus_one"] else 0))
    at = s["pos"].long()
    cos, sin = s["cos"][at].to(dt)[:, None], s["sin"][at].to(dt)[:, None]
    rot, half = c["rot"], c["rot"] // 2
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["neighbours"] else (x[..., :half], x[..., half:rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if c["neighbours"] else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _gathered(pages, places, n):
    """a request's stored rows [n, hkv, d]"""
    return pages[places].flatten(0, 1)[:n]


def _scores(s, dt, values=False):
    """request by request and, where they are many, some rows at a time: (scores [hkv, rows, group, keys], -inf where a row does not see a
    key; the values [hkv, keys, d])"""
    c = s["case"]
    hkv, d, group = c["hkv"], c["d"], c["hq"] // c["hkv"]
    base = 0
    for r, (T, L) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        places = s["places"][r]
        k = _gathered(s["k"], places, L).to(dt).transpose(0, 1)
        v = _gathered(s["v"], places, L).to(dt).transpose(0, 1) if values else None
        q = s["q"][base : base + T].to(dt).view(T, hkv, group, d).transpose(0, 1)
        key = torch.arange(L, device=DEV)
        at = key.clone()                                # positions of the stored keys
        last = torch.full((L,), 1 << 40, device=DEV)    # the stored index behind a key's subtree
        if s["end"] is not None:
            at[L - T :] = torch.from_numpy(s["pos"][base : base + T]).to(DEV)
            last[L - T :] = torch.from_numpy(s["end"][base : base + T]).to(DEV) - base + (L - T)
        some = max(1, (1 << 28) // max(1, hkv * group * L))
        for a in range(0, T, some):
            rows = torch.arange(L - T + a, L - T + min(a + some, T), device=DEV)[:, None]
            see = (key <= rows) & (rows < last)
            if c["window"]:
                see &= at[rows] - at < c["window"]
            qs = q[:, a : a + some]
            t = (qs.reshape(hkv, -1, d) @ k.transpose(1, 2)).view(hkv, qs.shape[1], group, L) * s["scale"]
            if c["softcap"]:
                t = c["softcap"] * torch.tanh(t / c["softcap"])
            yield t.masked_fill_(~see[None, :, None], float("-inf")), v, (r, base + a)
        base += T


def _softmax(t, v, where):
    """-> out [rows, hq, d] in bf16 (None without values), log of the sum of exponentials [rows, hq] in 32 bits"""
    hkv, rows, group, L = t.shape
    top = t.amax(-1, keepdim=True) if L else t.new_full((hkv, rows, group, 1), float("-inf"))
    top = torch.where(top.isinf(), 0.0, top)
    p = (t - top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log())[..., 0].permute(1, 0, 2).reshape(rows, hkv * group)
    if v is None:
        return None, lse.float()
    out = (p.view(hkv, rows * group, L) @ v) / torch.where(total > 0, total, 1.0).view(hkv, rows * group, 1)
    out = out.view(hkv, rows, group, -1).permute(1, 0, 2, 3).reshape(rows, hkv * group, -1)
    return (out.to(torch.bfloat16) if t.dtype == torch.float32 else out), lse


def _add_weights(s, dt):
    out = s["acc"].to(dt, copy=True)
    for t, _, (r, row) in _scores(s, dt):
        hkv, rows, group, L = t.shape
        lse = s["lse"][row : row + rows].to(dt).view(rows, hkv, group).permute(1, 0, 2)
        lse = torch.where(lse.isinf(), 0.0, lse)
        out[r, :, :L] += (t - lse[..., None]).exp_().sum((1, 2))
    return out


def _evict_plain(s, c):
    R, hkv, page = len(s["kv_lens"]), c["hkv"], c["page"]
    kept = torch.full((R, hkv, c["keep"]), -1, dtype=torch.int32, device=DEV)
    acc = torch.zeros((R, hkv, c["keep"]), device=DEV)
    for r, n in enumerate(s["kv_lens"]):
        m = min(n, c["keep"])
        if n <= c["keep"]:
            at = torch.arange(n, device=DEV).expand(hkv, n)
        else:
            first, last = c["sink"], n - c["recent"]
            order = s["acc"][r, :, first:last].sort(dim=1, descending=True, stable=True)[1]
            some = order[:, : m - c["sink"] - c["recent"]] + first
            ends = [torch.arange(*x, device=DEV).expand(hkv, -1) for x in ((0, first), (last, n))]
            at = torch.cat([ends[0], some, ends[1]], 1).sort(1)[0]
        kept[r, :, :m] = at
        acc[r, :, :m] = s["acc"][r].gather(1, at)
        to = s["new_places"][r]
        slot = torch.arange(m, device=DEV)
        for pages in (s["k"], s["v"]):
            rows = _gathered(pages, s["places"][r], n)
            pages[to[slot // page], slot % page] = rows.gather(0, at.t()[..., None].expand(m, hkv, c["d"]))
    return kept, acc, s["k"], s["v"]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    d, hkv = case["d"], case["hkv"]
    if case["kind"] == "rope":
        T, heads = case["tokens"], case["hq"] + case["hkv"] + (case["hkv"] if case["put"] else 0)
        table = min(T, 4096) * case["rot"] * (4 if case["tables"] == "fp32" else 2)
        return {"bytes": T * heads * d * 4 + table + T * (12 if case["put"] else 4), "flops": T * heads * d * 6}
    q_lens, kv_lens, end, pos = _shape(case)
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in kv_lens)
        return {"bytes": hkv * (kept * d * 8 + sum(kv_lens) * 4 + len(kv_lens) * case["keep"] * 8), "flops": hkv * sum(kv_lens)}
    pairs = keys = 0
    base = 0
    W = case["window"] or 1 << 40
    for T, L in zip(q_lens, kv_lens):
        c = L - T
        if T:
            at = np.arange(c, L) if end is None else pos[base : base + T]
            before = np.minimum(c, np.maximum(0, W - 1 - (at - c)))   # stored keys that a row sees
            pairs += int(before.sum())
            if end is None:
                pairs += int(np.minimum(np.arange(1, T + 1), W).sum())
            else:
                pairs += int((np.minimum(end[base : base + T] - base, T) - np.arange(T)).sum())   # (no tree here is as deep as a window)
            keys += int(before.max()) + T
        base += T
    rows = sum(q_lens)
    if case["kind"] == "attn":
        return {"bytes": keys * hkv * d * 4 + rows * case["hq"] * d * 4, "flops": 4 * d * case["hq"] * pairs}
    return {"bytes": keys * hkv * d * 2 + rows * case["hq"] * (2 * d + 4) + len(kv_lens) * hkv * max(kv_lens) * 8, "flops": 2 * d * case["hq"] * pairs}


# ------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_rope(s, case)
    if kind == "evict":
        return _exact_evict(s, case)
    hkv, d, group = case["hkv"], case["d"], case["hq"] // case["hkv"]
    out = torch.zeros((sum(s["q_lens"]), case["hq"], d), dtype=torch.float64, device=DEV)
    weight = s["acc"].double() if kind == "weights" else None
    base = 0
    for r, (T, L) in enumerate(zip(s["q_lens"], s["kv_lens"])):
        token = np.arange(L)
        place = torch.tensor([s["tables"][r][t // case["page"]] for t in range(0, L, case["page"])], dtype=torch.int64, device=DEV)
        seen = torch.from_numpy(_visible(case, s, base, T, L)).to(DEV)
        for h in range(hkv):
            keys = s["k"][place, :, h].reshape(-1, d)[: len(token)].double()
            vals = s["v"][place, :, h].reshape(-1, d)[: len(token)].double()
            step = max(1, (1 << 27) // max(1, L))
            for head in range(h * group, (h + 1) * group):
                for a in range(0, T, step):
                    rows = slice(a, min(T, a + step))
                    logit = s["q"][base : base + T][rows, head].double() @ keys.mT * s["scale"]
                    if case["softcap"]:
                        logit = torch.tanh(logit / case["softcap"]) * case["softcap"]
                    logit = torch.where(seen[rows], logit, -torch.inf)
                    if kind == "attn":
                        prob = torch.nan_to_num(torch.softmax(logit, -1), nan=0.0)
                        out[base : base + T][rows, head] = prob @ vals
                    else:
                        prob = torch.where(seen[rows], torch.exp(logit - s["lse"][base : base + T][rows, head, None].double()), 0.0)
                        weight[r, h, :L] += prob.sum(0)
        base += T
    return out if kind == "attn" else weight


def _visible(case, s, base, T, L):
    """[T, L]: which stored keys a request's rows see, from the definition"""
    c = L - T
    row, key = np.arange(T)[:, None], np.arange(L)[None, :]
    see = key <= c + row
    at = np.arange(L)
    if s["end"] is not None:
        end = s["end"][base : base + T] - base
        at[c:] = s["pos"][base : base + T]
        see[:, c:] &= row < end[None, :]
    if case["window"]:
        see &= at[c:][:, None] - at[None, :] < case["window"]
    return see


def _exact_rope(s, case):
    def turn(x, w):
        x = x.double()
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (w.double() + float(case["plus_one"]))
        at = s["pos"].long()
        z = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        rot = case["rot"]
        if case["neighbours"]:
            pair = torch.view_as_complex(y[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * z
            y[..., :rot] = torch.view_as_real(pair).flatten(-2)
        else:
            pair = torch.complex(y[..., : rot // 2].contiguous(), y[..., rot // 2 : rot].contiguous()) * z
            y[..., : rot // 2], y[..., rot // 2 : rot] = pair.real, pair.imag
        return y

    q, k = turn(s["q"], s["wq"]), turn(s["k"], s["wk"])
    if not case["put"]:
        return q, k
    v = s["v"].double()
    if case["v_norm"]:
        v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6)
    ck, cv = s["ck"].double(), s["cv"].double()
    for t, rows in ((ck, k), (cv, v)):
        t[s["slots"] // case["page"], s["slots"] % case["page"]] = rows
    return q, ck, cv


def _exact_evict(s, case):
    R, hkv, keep, page = len(s["kv_lens"]), case["hkv"], case["keep"], case["page"]
    acc = s["acc"].cpu().numpy()
    kept, kept_acc = np.full((R, hkv, keep), -1, np.int32), np.zeros((R, hkv, keep))
    k, v = s["k"].clone(), s["v"].clone()
    for r, n in enumerate(s["kv_lens"]):
        m = min(n, keep)
        for h in range(hkv):
            rank = acc[r, h, :n].astype(np.float64).copy()
            rank[: case["sink"]] = np.inf
            rank[n - case["recent"] :] = np.inf
            at = np.sort(np.lexsort((np.arange(n), -rank))[:m])
            kept[r, h, :m], kept_acc[r, h, :m] = at, acc[r, h, at]
            src, dst = np.array(s["tables"][r])[at // page], np.array(s["into"][r])[np.arange(m) // page]
            src, at, dst, slot = (torch.from_numpy(np.asarray(x, np.int64)).to(DEV) for x in (src, at % page, dst, np.arange(m) % page))
            for t, old in ((k, s["k"]), (v, s["v"])):
                t[dst, slot, h] = old[src, at, h]
    return torch.from_numpy(kept), torch.from_numpy(kept_acc), k.double(), v.double()
