"""What is timed of a decoding step over stored contents whose lengths, pages and draws stay on the GPU: the calls that one recorded graph replays, token by token.

  step    the seats' bookkeeping: keys given up, pages returned and taken, the new tokens' places in the cache and their positions
  attn    attention of the seats' new tokens over the content they share with others and over the keys of their own
  sample  the next tokens, drawn from logits with temperature, top-k, top-p and min-p by given random numbers

A case is a dict of plain values.  ``own`` false: elementary torch operations, in 32 bits (running sums of probabilities in 64, where the place of a border decides about
a token) and rounded once at the end.  ``own`` true: the public calls of spinf_serve_amd.  Lengths and pages belong to the case and the seed; the seed draws the tensors.
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
        # one token for each of 64 requests of a server, four drafts of the step before given up first: the smallest call
        _step("step_drafts", seats=64, own=2900, spread=0.6, new=4, page=64, contents=6),
        # the headline pass's 24 x 56 branches, one token each, pages of 16
        _step("step_branches", seats=1344, own=9, spread=0.4, new=1, page=16, contents=24),
        # every seat is taken by a new request, whose prompt comes whole: a hundred thousand rows
        _step("step_prompts", seats=48, own=2100, spread=0.3, new=0, page=64, contents=0),
        # one content of 301 tokens, 24 questions' answers below it: latency
        _attn("attn_request", contents=1, stored=301, per=24, own=14, own_spread=0.4, new=1, hq=16, hkv=8, d=256, page=64),
        # the headline pass's 24 contents and 56 branches each, one token of every branch
        _attn("attn_branches", contents=24, stored=470, spread=0.2, per=56, own=9, own_spread=0.3, new=1, hq=16, hkv=8, d=256, page=16),
        # a long document that 48 requests go on below, each with a few hundred tokens of its own
        _attn("attn_document", contents=1, stored=65536, per=48, own=600, own_spread=0.6, new=1, hq=24, hkv=4, d=256, page=64),
        # the global layers of 512 dims: four long contents, drafts of four tokens, two seats below no content
        _attn("attn_global", contents=4, stored=12011, spread=0.4, per=11, own=777, own_spread=0.5, new=4, hq=16, hkv=1, d=512, page=32, alone=2),
        # a sliding layer with capped scores: questions of 150 tokens read below contents of odd lengths, pages that end inside a tile
        _attn("attn_sliding", contents=7, stored=4099, spread=0.3, per=5, own=211, new=150, hq=16, hkv=8, d=256, page=48, window=1024, softcap=50.0),
        # the next token of one request
        _sample("sample_one", rows=1, vocab=262144, dtype="fp32", temperature=0.8, top_k=40),
        # a server's step, each request with settings of its own, logits in bf16
        _sample("sample_step", rows=64, vocab=151936, dtype="bf16", mixed=True),
        # every branch of a pass draws from the whole vocabulary
        _sample("sample_plain", rows=320, vocab=262144, dtype="fp32", temperature=1.0),
        # nucleus of flat rows: thousands of tokens stay
        _sample("sample_nucleus", rows=96, vocab=262144, dtype="fp32", temperature=1.3, top_p=0.97, min_p=0.0005),
    ]


def _step(name, seats, own, new, page, contents, spread=0.0):
    """own: keys of a seat's own before the call, with what it drops; new 0: all of them go, and a prompt of about as many tokens comes"""
    return dict(name=name, kind="step", seats=seats, own=own, spread=spread, new=new, page=page, contents=contents)


def _attn(name, contents, stored, per, own, new, hq, hkv, d, page, spread=0.0, own_spread=0.0, alone=0, window=0, softcap=0.0):
    """own: keys of a seat's own, with the new ones; per: seats below each content; alone: seats below none"""
    return dict(name=name, kind="attn", contents=contents, stored=stored, spread=spread, per=per, own=own, own_spread=own_spread, new=new, hq=hq, hkv=hkv, d=d, page=page,
                alone=alone, window=window, softcap=softcap)


def _sample(name, rows, vocab, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False):
    return dict(name=name, kind="sample", rows=rows, vocab=vocab, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, mixed=mixed)


HEADS = [(16, 8, 256), (16, 1, 512), (24, 4, 256), (32, 16, 128), (16, 4, 64), (12, 12, 64), (10, 2, 128)]


def _log(rng, a, b):
    """a whole number, spread over the logarithm of a .. b"""
    return min(b, max(a, int(round(a * (b / a) ** rng.random()))))


def draw(rng):
    """one more case of these ranges, costing no more than the largest listed one"""
    kind = rng.choice(["step", "attn", "attn", "attn", "sample", "sample"])
    page = rng.choice([16, 32, 48, 64, 80, 128])
    if kind == "step":
        seats = _log(rng, 1, 1500)
        new = rng.choice([1, 1, 2, 4, 8, 0])
        own = _log(rng, 2 * max(new, 1), max(24, min(8000, 120000 // seats)))
        c = _step("", seats=seats, own=own, spread=rng.choice([0.0, 0.5]), new=new, page=page, contents=rng.choice([0, 1, 3, 24]))
    elif kind == "attn":
        hq, hkv, d = rng.choice(HEADS)
        new = rng.choice([1, 1, 1, 2, 4, _log(rng, 5, 200)])
        c = _attn("", contents=_log(rng, 1, 24), stored=_log(rng, 1, 60000), spread=rng.choice([0.0, 0.4]), per=_log(rng, 1, 64), own=new - 1 + _log(rng, 1, 3000),
                  own_spread=rng.choice([0.0, 0.5]), new=new, hq=hq, hkv=hkv, d=d, page=page, alone=rng.choice([0, 0, 1, 5]), window=rng.choice([0, 0, 256, 1024]) if d <= 256 else 0,
                  softcap=rng.choice([0.0, 0.0, 30.0]))
        while True:   # (the contents' pages, the seats' and the products, each within what the largest listed cases have)
            tokens = c["contents"] * c["per"] * c["new"]
            if c["contents"] * c["stored"] > 80000:
                c["contents"] = max(1, c["contents"] // 2)
            elif c["contents"] * c["per"] * c["own"] * hkv * d > 60_000_000 or tokens * (c["stored"] + c["own"]) * hq * d > 20_000_000_000:
                c["per"] = max(1, c["per"] // 2)
                if c["per"] == 1:
                    c["contents"], c["new"] = max(1, c["contents"] // 2), max(1, c["new"] // 2)
            else:
                break
    else:
        vocab = _log(rng, 1000, 262144)
        some = rng.choice(["plain", "k", "p", "min", "all", "mixed"])
        c = _sample("", rows=_log(rng, 1, min(512, 60_000_000 // vocab)), vocab=vocab, dtype=rng.choice(["fp32", "bf16"]), temperature=round(rng.uniform(0.3, 1.6), 2),
                    top_k=_log(rng, 1, 400) if some in ("k", "all") else 0, top_p=round(rng.uniform(0.3, 0.995), 3) if some in ("p", "all") else 1.0,
                    min_p=round(rng.uniform(0.001, 0.3), 4) if some in ("min", "all") else 0.0, mixed=some == "mixed")
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ lengths and pages: from the case and, of steps, the seed
def _rng(case, seed=0):
    return np.random.default_rng(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()) + seed)


def _around(g, mean, spread, n, least=1):
    x = np.round(mean * np.exp(spread * g.standard_normal(n))) if spread else np.full(n, mean)
    return np.clip(x, least, 2 * mean).astype(np.int64)


def _shape(case):
    """-> of attn: content lengths, the content of each seat (-1: none), its own keys with the new ones, the new ones"""
    g = _rng(case)
    stored = _around(g, case["stored"], case["spread"], case["contents"])
    content = np.concatenate([np.repeat(np.arange(case["contents"]), case["per"]), np.full(case["alone"], -1)])
    lens = _around(g, case["own"], case["own_spread"], len(content), least=case["new"])
    return stored, content, lens, np.full(len(content), case["new"])


def _pages_of(n, page):
    return -(-n // page)


def _shuffled(g, lens, page, first=0):
    """a page table per length: pages from `first` on, in an order as a busy allocator leaves them"""
    need = _pages_of(lens, page)
    ids = first + g.permutation(int(need.sum()))
    return np.split(ids, np.cumsum(need)[:-1])


def _normal(gen, *shape):
    out = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
    flat = out.view(-1)
    for a in range(0, flat.numel(), 1 << 27):
        part = flat[a : a + (1 << 27)]
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV))
    return out


# ------------------------------------------------------------------------------------------------ what a program has before the call
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"step": _prepare_step, "attn": _prepare_attn, "sample": _prepare_sample}[case["kind"]](dict(case=case), case, gen, seed)


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(DEV)


def _book(s, pool, tables, lens, keys, rows, page, content, stored):
    """the seats' books as the plain form keeps them: the pages in hand out of a stack whose last page goes first, seat by seat"""
    R = len(lens)
    table = np.full((R, _pages_of(keys, page)), -1, np.int64)
    left = len(pool)
    for r, n in enumerate(_pages_of(np.asarray(lens), page)):
        table[r, :n] = pool[left - n : left][::-1]
        left -= n
    s["book"] = dict(lens=_i32(lens), table=_i32(table), free=_i32(pool), left=_i32([left]), first=_i32(np.zeros(R + 1)), slots=torch.full((rows,), -1, dtype=torch.int64, device=DEV),
                     pos=torch.zeros(rows, dtype=torch.int32, device=DEV), content=_i32(content), text=_i32(np.append(stored, 0)))
    if own:
        seats = _package().PagedSeats.build(seats=R, rows=rows, page=page, keys=keys, pool=pool, contents=(stored, tables[: len(stored)]), stored=lens, heads=s.get("heads", ()), device=DEV)
        seats.content.copy_(s["book"]["content"])
        s["seats"] = seats


def _prepare_step(s, case, gen, seed):
    g = _rng(case)
    R, page = case["seats"], case["page"]
    new = np.full(R, case["new"]) if case["new"] else _around(g, case["own"], case["spread"], R)
    lens = _around(g, case["own"], case["spread"], R, least=2 * max(case["new"], 1))
    stored = _around(g, 470, 0.3, case["contents"])
    g = _rng(case, seed)   # (which seat has which length)
    new, lens = g.permutation(new), g.permutation(lens)
    tables = _shuffled(g, stored, page)
    shared = int(_pages_of(stored, page).sum())
    keys = 2 * case["own"] + 16
    pool = shared + g.permutation(int(_pages_of(lens, page).sum() + _pages_of(new, page).sum()) + 3)
    rows = int(new.sum()) + 5
    content = g.integers(-1, case["contents"], R) if case["contents"] else np.full(R, -1)
    _book(s, pool, tables, lens, keys, rows, page, content, stored)
    s["new"], s["drop"] = _i32(new), _i32(new if case["new"] else np.full(R, 1 << 30))
    s["rows"], s["keys"] = rows, keys
    run(s)   # (the pass before: its tokens are the ones that go)
    return s


def _prepare_attn(s, case, gen, seed):
    stored, content, lens, new = _shape(case)
    g = _rng(case)
    page, hkv, d = case["page"], case["hkv"], case["d"]
    tables = _shuffled(g, stored, page)
    shared = int(_pages_of(stored, page).sum())
    pool = shared + g.permutation(int(_pages_of(lens, page).sum()) + 1)
    pages = shared + len(pool)
    k, v = _normal(gen, pages, hkv, page, d), _normal(gen, pages, hkv, page, d)
    k *= (1 + 1.5 * (torch.rand((pages, hkv, page, 1), generator=gen, device=DEV) < 0.02)).to(torch.bfloat16)   # one key in fifty draws more weight
    s["k"], s["v"] = k.transpose(1, 2), v.transpose(1, 2)   # [pages, page, hkv, d], a head's rows of a page next to each other
    rows = int(new.sum()) + int(new.sum()) // 16
    s["rows"], s["keys"] = rows, int(lens.max())
    s["heads"] = [(case["hq"], hkv, d, case["window"])]
    s["q"] = _normal(gen, rows, case["hq"], d)
    _book(s, pool, tables, lens - new, s["keys"], rows, page, content, stored)
    s["new"], s["drop"] = _i32(new), None
    _step_plain(s, case)
    if own:
        s["seats"].step(s["new"])
        s["cache"] = _package().PagedCache(s["k"], s["v"])
    table = s["book"]["table"].cpu().numpy()
    s["stored"], s["content"], s["lens"], s["news"] = stored, content, lens, new
    s["shared"] = [torch.from_numpy(np.asarray(t, np.int64)).to(DEV) for t in tables]
    s["places"] = [torch.from_numpy(table[r, : _pages_of(n, page)].astype(np.int64)).to(DEV) for r, n in enumerate(lens)]
    return s


def _prepare_sample(s, case, gen, seed):
    rows, vocab = case["rows"], case["vocab"]
    # a bulk of unlikely tokens, and some that a context makes likely
    x = torch.randn((rows, vocab), generator=gen, device=DEV) * 2.2
    at = torch.randint(0, vocab, (rows, 200), generator=gen, device=DEV)
    x.scatter_reduce_(1, at, 4 + 9 * torch.rand((rows, 200), generator=gen, device=DEV) ** 2, "amax")
    s["logits"] = x.to(torch.float32 if case["dtype"] == "fp32" else torch.bfloat16)
    s["u"] = torch.rand(rows, generator=gen, device=DEV, dtype=torch.float64)
    s["how"] = dict(temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
    if case["mixed"]:
        pick = lambda values, dt: torch.tensor(values, dtype=dt, device=DEV)[torch.randint(0, len(values), (rows,), generator=gen, device=DEV)]  # noqa: E731
        s["how"] = dict(temperature=pick([0.0, 0.6, 0.7, 1.0, 1.2], torch.float32), top_k=pick([0, 0, 20, 50, 1], torch.int32), top_p=pick([1.0, 0.8, 0.9, 0.95], torch.float32),
                        min_p=pick([0.0, 0.0, 0.05, 0.1], torch.float32))
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    return (_run_own if own else {"step": _step_plain, "attn": _attn_plain, "sample": _sample_plain}[c["kind"]])(s, c)


def _run_own(s, c):
    sa = _package()
    if c["kind"] == "step":
        t = s["seats"]
        slots, pos = t.step(s["new"], s["drop"])
        return slots, pos, t.first, t.lens, t.table, t.free, t.left
    if c["kind"] == "attn":
        return sa.seats_attn(s["q"], s["cache"], s["seats"], c["d"] ** -0.5, window=c["window"] or None, softcap=c["softcap"] or None)
    return sa.sample_tokens(s["logits"], s["u"], **s["how"], return_prob=True)


def _step_plain(s, c):
    """first the last ``drop`` keys of every seat go, and their pages with them; then the new tokens come, seat by seat, to seats that have room: keys, rows and pages"""
    b, page, rows, keys = s["book"], c["page"], s["rows"], s["keys"]
    lens, table, free = b["lens"].long(), b["table"], b["free"]
    R, width = table.shape
    pages = lambda n: (n + page - 1) // page  # noqa: E731
    stay = lens - (torch.minimum(s["drop"].long().clamp(min=0), lens) if s["drop"] is not None else 0)
    j = torch.arange(width, device=DEV)
    gone = (j >= pages(stay)[:, None]) & (j < pages(lens)[:, None])
    at = gone.flatten().cumsum(0).view(R, width)          # the how-many-eth page to go back: seat by seat, page by page
    have = b["left"].long() + at[-1, -1]
    returned = torch.where(gone, have - at, len(free)).flatten()
    wide = torch.cat([free, free.new_zeros(1)]).scatter(0, returned, table.flatten())   # (what does not go back: one place behind the stack)
    free.copy_(wide[:-1])
    new = s["new"].long().clamp(min=0)
    new = torch.where(stay + new <= keys, new, 0)
    need = pages(stay + new) - pages(stay)
    fits = (new.cumsum(0) <= rows) & ((need == 0) | (need.cumsum(0) <= have))
    took = torch.where(fits, new, 0)
    need = torch.where(fits, need, 0)
    before = need.cumsum(0) - need
    come = (j >= pages(stay)[:, None]) & (j < (pages(stay) + need)[:, None])
    src = (have - 1 - before[:, None] - (j - pages(stay)[:, None])).clamp(0, max(len(free) - 1, 0))
    table.copy_(torch.where(come, free[src], table))
    b["left"].copy_(have - need.sum())
    b["lens"].copy_(stay + took)
    first = b["first"]
    first[1:] = took.cumsum(0)
    row = torch.arange(rows, device=DEV)
    seat = torch.searchsorted(first[1:].contiguous(), row.int(), right=True).clamp(max=R - 1)
    on = row < first[-1]
    place = stay[seat] + row - first[seat]
    slot = table[seat, (place // page).clamp(0, width - 1)].long() * page + place % page
    b["slots"].copy_(torch.where(on, slot, -1))
    text = b["text"][b["content"][seat].long()]           # (no content: the last entry, 0)
    b["pos"].copy_(torch.where(on, text + place, 0))
    return b["slots"], b["pos"], first, b["lens"], table, free, b["left"]


def _attn_plain(s, c):
    hq, hkv, d, W = c["hq"], c["hkv"], c["d"], c["window"]
    group = hq // hkv
    out = torch.zeros((s["rows"], hq, d), dtype=torch.bfloat16, device=DEV)
    row = np.concatenate([[0], np.cumsum(s["news"])])

    def scores(q, k, place, at):
        """[hkv, rows x group, keys]: capped, -inf behind a row's own place (``at``, of the rows) and outside its window"""
        t = (q @ k.transpose(1, 2)) * d**-0.5
        if c["softcap"]:
            t = c["softcap"] * torch.tanh(t / c["softcap"])
        see = place <= at[:, None]
        if W:
            see &= at[:, None] - place < W
        return t.masked_fill_(~see[None], float("-inf"))

    def part(t, v):
        """(maximum, sum, weighted sum)"""
        top = t.amax(-1, keepdim=True)
        top = torch.where(top.isinf(), 0.0, top)
        p = (t - top).exp_()
        return top, p.sum(-1, keepdim=True), p @ v

    for a, b, content in _runs(s["content"]):
        shared = None
        q = s["q"][row[a] : row[b]].float().view(-1, hkv, group, d).transpose(0, 1)   # [hkv, rows, group, d]
        P = int(s["stored"][content]) if content >= 0 else 0
        at = torch.cat([torch.arange(P + n - m, P + n, device=DEV) for n, m in zip(s["lens"][a:b], s["news"][a:b])]).repeat_interleave(group)
        q = q.reshape(hkv, -1, d)
        if P:
            k, v = (x[s["shared"][content]].flatten(0, 1)[:P].float().transpose(0, 1).contiguous() for x in (s["k"], s["v"]))
            place = torch.arange(P, device=DEV)
            some = max(1, (1 << 28) // (hkv * P))
            shared = [part(scores(q[:, i : i + some], k, place, at[i : i + some]), v) for i in range(0, q.shape[1], some)]
            shared = [torch.cat(x, 1) for x in zip(*shared)]
        for r in range(a, b):
            rows = slice((row[r] - row[a]) * group, (row[r + 1] - row[a]) * group)
            n = int(s["lens"][r])
            k, v = (x[s["places"][r]].flatten(0, 1)[:n].float().transpose(0, 1).contiguous() for x in (s["k"], s["v"]))
            top, total, o = part(scores(q[:, rows], k, P + torch.arange(n, device=DEV), at[rows]), v)
            if shared is not None:
                top2, total2, o2 = (x[:, rows] for x in shared)
                most = torch.maximum(torch.where(total > 0, top, -1e30), torch.where(total2 > 0, top2, -1e30))
                f, f2 = (top - most).exp() * (total > 0), (top2 - most).exp() * (total2 > 0)
                total, o = f * total + f2 * total2, f * o + f2 * o2
            out[row[r] : row[r + 1]] = (o / total).view(hkv, -1, group, d).transpose(0, 1).reshape(-1, hq, d).bfloat16()
    return out


def _runs(content):
    """seats that follow each other below one content: (first, end, content)"""
    cuts = np.flatnonzero(np.diff(content)) + 1
    return [(int(a), int(b), int(content[a])) for a, b in zip([0, *cuts], [*cuts, len(content)])]


def _settings(s, c):
    """temperature, top_k, top_p, min_p of every row, [rows, 1]: numbers as 32 bits hold them"""
    dev = dict(device=DEV)
    h = s["how"]
    full = lambda x, dt: (x if torch.is_tensor(x) else torch.full((c["rows"],), x, dtype=dt, **dev)).to(dt)[:, None]  # noqa: E731
    return full(h["temperature"], torch.float32).double(), full(h["top_k"], torch.int32).long(), full(h["top_p"], torch.float32).double(), full(h["min_p"], torch.float32).double()


def _sample_plain(s, c):
    T, k, p, least = _settings(s, c)
    x = s["logits"].float()
    vocab = x.shape[1]
    order, index = x.sort(dim=1, descending=True, stable=True)
    z = (order.double() - order[:, :1].double()) / torch.where(T > 0, T, 1.0)
    z = torch.where((T > 0) | (torch.arange(vocab, device=DEV) == 0), z, float("-inf"))   # no temperature: the first of the largest
    k = torch.where((k > 0) & (k < vocab), k, vocab)
    w = torch.where(torch.arange(vocab, device=DEV) < k, z.exp(), 0.0)
    run_sum = w.cumsum(1)
    keep = (w > 0) & ((p >= 1) | (run_sum - w < p * run_sum[:, -1:])) & (z >= least.log())
    keep[:, 0] = True
    w = torch.where(keep, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, index, w)   # back in the vocabulary's order
    run_sum = w.cumsum(1)
    token = torch.searchsorted(run_sum, s["u"][:, None] * run_sum[:, -1:], right=True)
    return token[:, 0], (w.gather(1, token) / run_sum[:, -1:])[:, 0].float()


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + case["rows"] * 20, "flops": 4 * n}
    if case["kind"] == "step":
        new = case["seats"] * (case["new"] or case["own"])
        return {"bytes": case["seats"] * 24 + 12 * new + 8 * (new // case["page"] + 1), "flops": 4 * new}
    stored, content, lens, new = _shape(case)
    d, hq, hkv, W = case["d"], case["hq"], case["hkv"], case["window"] or 1 << 40
    pairs = keys = 0
    seen = np.zeros(len(stored), np.int64)
    for c, n, m in zip(content, lens, new):
        at = np.arange(n - m, n)
        mine = np.minimum(at + 1, W)
        pairs += int(mine.sum())
        keys += int(min(n, m + W - 1))
        if c >= 0:
            theirs = np.clip(W - 1 - at, 0, stored[c])
            pairs += int(theirs.sum())
            seen[c] = max(seen[c], theirs.max())
    rows = int(new.sum())
    return {"bytes": (keys + int(seen.sum())) * hkv * d * 4 + rows * hq * d * 4, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------ from the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"step": _exact_step, "attn": _exact_attn, "sample": _exact_sample}[case["kind"]](s, case)


def _exact_step(s, case):
    """seat by seat, page by page, on the host"""
    b = {k: v.cpu().numpy().astype(np.int64) for k, v in s["book"].items()}
    if own:
        t = s["seats"]
        b.update({k: getattr(t, k).cpu().numpy().astype(np.int64) for k in ("lens", "table", "free", "left")})
    lens, table, free, page = b["lens"], b["table"], b["free"], case["page"]
    stack, top = free.copy(), int(b["left"][0])
    back = []
    for r in range(len(lens)):
        left = lens[r] - min(int(s["drop"][r]), lens[r])
        back += table[r, _pages_of(left, page) : _pages_of(lens[r], page)].tolist()
        lens[r] = left
    for x in reversed(back):
        stack[top] = x
        top += 1
    slots, pos, first = [], [], [0]
    room = s["rows"]
    for r, m in enumerate(s["new"].tolist()):
        assert lens[r] + m <= s["keys"] and len(slots) + m <= room
        for i in range(m):
            if lens[r] % page == 0:
                top -= 1
                table[r, lens[r] // page] = stack[top]
            slots.append(table[r, lens[r] // page] * page + lens[r] % page)
            pos.append(lens[r] + b["text"][b["content"][r]])
            lens[r] += 1
        first.append(len(slots))
    pad = room - len(slots)
    out = np.array(slots + [-1] * pad), np.array(pos + [0] * pad), np.array(first), lens, table, stack, np.array([top])
    return tuple(torch.from_numpy(x) for x in out)


def _exact_attn(s, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    group = hq // hkv
    out = torch.zeros((s["rows"], hq, d), dtype=torch.float64, device=DEV)
    base = 0
    for r, c in enumerate(s["content"]):
        n, m = int(s["lens"][r]), int(s["news"][r])
        P = int(s["stored"][c]) if c >= 0 else 0
        last = torch.arange(P + n - m, P + n, device=DEV)[:, None]
        first = int(max(0, P + n - m - case["window"] + 1)) if case["window"] else 0   # (no row sees a key before)
        key = torch.arange(first, P + n, device=DEV)[None]
        hidden = (key > last) | ((last - key >= case["window"]) if case["window"] else torch.zeros_like(key > last))
        for h in range(hkv):
            k, v = (torch.cat([x[s["shared"][c], :, h].reshape(-1, d)[:P] if P else x[:0, 0, h], x[s["places"][r], :, h].reshape(-1, d)[:n]])[first:].double() for x in (s["k"], s["v"]))
            for head in range(h * group, (h + 1) * group):
                logit = s["q"][base : base + m, head].double().matmul(k.t()).mul(d**-0.5)
                if case["softcap"]:
                    logit = (logit / case["softcap"]).tanh() * case["softcap"]
                logit[hidden] = -torch.inf
                out[base : base + m, head] = torch.softmax(logit, 1).matmul(v)
        base += m
    return out


def _exact_sample(s, case):
    T, k, p, least = (x[:, 0].cpu().numpy() for x in _settings(s, case))
    u = s["u"].cpu().numpy()
    tokens, probs = np.zeros(case["rows"], np.int64), np.zeros(case["rows"])
    for r in range(case["rows"]):
        x = s["logits"][r].float().cpu().numpy().astype(np.float64)
        if T[r] == 0:
            tokens[r], probs[r] = x.argmax(), 1.0
            continue
        weight = np.exp((x - x.max()) / T[r])
        stays = np.ones(len(x), bool)
        if 0 < k[r] < len(x) or p[r] < 1:
            order = np.lexsort((np.arange(len(x)), -x))
            if 0 < k[r] < len(x):
                order = order[: k[r]]
            if p[r] < 1:
                mass = np.cumsum(weight[order])
                order = order[: 1 + np.searchsorted(mass, p[r] * mass[-1], side="left")]
            stays[:] = False
            stays[order] = True
        stays &= weight >= least[r]
        mass = np.cumsum(np.where(stays, weight, 0.0))
        tokens[r] = np.flatnonzero(mass > u[r] * mass[-1])[0]
        probs[r] = weight[tokens[r]] / mass[-1]
    return torch.from_numpy(tokens), torch.from_numpy(probs)
