"""Answers token by token, with nothing on the host between two tokens: documents read once into a paged cache, requests below them that take seats, and one recorded
graph that is replayed for every token: the seats' step, one attention layer, the head, the draw of the next tokens.

    python examples/seats_session.py        (needs an MI355X and the built library)

Every answer is checked: against the same calls without a graph (token by token the same), and the last tokens' attention against tree_attn over documents and answers read anew.
"""

from __future__ import annotations

import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spinf-serve_amd"))

import spinf_serve_amd as sa  # noqa: E402

HQ, HKV, D, HIDDEN, VOCAB, PAGE = 16, 8, 128, 512, 5000, 32
END = 500   # tokens below it end an answer


class Model:
    """an embedding, one attention layer, a head"""

    def __init__(self, device, seed=0):
        g = torch.Generator().manual_seed(seed)
        w = lambda a, b, scale: (torch.randn((a, b), generator=g) * scale).to(torch.bfloat16).to(device)  # noqa: E731
        self.emb, self.head = w(VOCAB, HIDDEN, 1.0), w(VOCAB, HIDDEN, 2 * HIDDEN**-0.5)
        self.qkv, self.back = w(HIDDEN, (HQ + 2 * HKV) * D, HIDDEN**-0.5), w(HQ * D, HIDDEN, (HQ * D) ** -0.5)
        self.wq, self.wk = (torch.rand(D, generator=g).add_(0.5).to(device) for _ in range(2))
        ang = torch.arange(8192)[:, None] * 10000.0 ** (-torch.arange(D // 2) / (D // 2))[None]
        self.cos, self.sin = ang.cos().to(device), ang.sin().to(device)

    def project(self, tokens):
        return (t.unflatten(1, (-1, D)) for t in (self.emb[tokens] @ self.qkv).split([HQ * D, HKV * D, HKV * D], 1))

    def put(self, tokens, cache, slots, pos):
        q, k, v = self.project(tokens)
        return sa.qk_norm_rope_put(q, k, v, self.wq, self.wk, self.cos, self.sin, 1e-6, cache, slots, pos=pos)

    def draw(self, tokens, out, u):
        h = self.emb[tokens] + out.flatten(1) @ self.back
        return sa.sample_tokens(sa.lm_head_logprobs(h, None, self.head), u, temperature=0.9, top_k=200, top_p=0.95)


class Session:
    def __init__(self, model, documents, seats, rows, steps, device):
        self.model, self.documents = model, documents
        lens = [len(t) for t in documents]
        need = [-(-n // PAGE) for n in lens]
        ids = np.random.default_rng(0).permutation(sum(need) + 8 * seats)
        tables = np.split(ids[: sum(need)], np.cumsum(need)[:-1])
        self.cache = sa.PagedCache.empty(len(ids), PAGE, HKV, D, device)
        batch = sa.PagedBatch.build(lens, lens, tables, PAGE, device)          # the documents, once
        model.put(torch.cat(documents), self.cache, *batch.rows())
        self.seats = sa.PagedSeats.build(seats, rows, PAGE, 8 * PAGE, ids[sum(need) :], contents=(lens, tables), heads=[(HQ, HKV, D)], device=device)
        self.last = torch.zeros(seats, dtype=torch.int64, device=device)       # each seat's last token, and whether it goes on
        self.new = torch.zeros(seats, dtype=torch.int32, device=device)
        self.u = torch.rand((steps, seats), generator=torch.Generator().manual_seed(3)).to(device)
        self.now = torch.zeros(1, dtype=torch.int64, device=device)
        self.text = torch.full((steps, seats), -1, dtype=torch.int64, device=device)
        self.row = torch.arange(seats, dtype=torch.int32, device=device)

    def arrive(self, requests):
        """requests {seat: (content, prompt)}: they take the seats, whoever sat there; a whole prompt comes at once.  The others wait"""
        n = len(self.last)
        new, drop, content = np.zeros(n, np.int32), np.zeros(n, np.int32), self.seats.content.tolist()
        for r, (c, prompt) in requests.items():
            new[r], drop[r], content[r] = len(prompt), 1 << 30, c
        self.seats.content.copy_(torch.tensor(content, dtype=torch.int32))
        prompts = torch.cat([requests[r][1] for r in sorted(requests)])
        slots, pos = self.seats.step(*(torch.from_numpy(x).to(self.last.device) for x in (new, drop)), rows=len(prompts))
        out = sa.seats_attn(self.model.put(prompts, self.cache, slots, pos), self.cache, self.seats)
        ends = torch.from_numpy(np.cumsum(new)[sorted(requests)] - 1).to(self.last.device)
        at = torch.tensor(sorted(requests), device=self.last.device)
        self.last[at] = self.model.draw(prompts[ends], out[ends], self.u[0, at])
        self.new[at] = 1

    def token(self):
        """one token for every seat that goes on; no size, length or address changes from one call to the next"""
        s = self.seats
        slots, pos = s.step(self.new, rows=len(self.row))
        seat = (torch.searchsorted(s.first, self.row, right=True) - 1).clamp(max=len(self.row) - 1)
        tokens = self.last[seat]
        out = sa.seats_attn(self.model.put(tokens, self.cache, slots, pos), self.cache, s)
        drawn = self.model.draw(tokens, out, self.u[self.now].flatten()[seat])
        came = s.took > 0
        self.text.index_copy_(0, self.now, torch.where(came, self.last, -1)[None])
        self.last.copy_(torch.where(came, drawn[s.first[:-1].clamp(max=len(self.row) - 1).long()], self.last))
        self.new.copy_(came & (self.last >= END))
        self.now += 1
        return out

    def anew(self, answers):
        """the attention of the answers' last tokens, everything read again as one packed stream of trees; answers {seat: (content, tokens)}"""
        below = [[r for r, (c, _) in answers.items() if c == i] for i in range(len(self.documents))]
        stream = sa.pack_stream([sa.TokenTree([1] * len(t), [[2] * len(answers[r][1]) for r in b], [-1] * len(b)) for t, b in zip(self.documents, below)])
        real = np.flatnonzero(stream.art >= 0)
        tokens = torch.zeros(stream.length, dtype=torch.int64, device=self.last.device)
        tokens[torch.from_numpy(real).to(tokens.device)] = torch.cat([x for t, b in zip(self.documents, below) for x in (t, *(answers[r][1] for r in b))])
        q, k, v = self.model.project(tokens)
        q, k = sa.qk_norm_rope(q, k, self.model.wq, self.model.wk, self.model.cos, self.model.sin, 1e-6, torch.from_numpy(stream.pos.astype(np.int64)).to(tokens.device))
        out = sa.tree_attn(q, k, v, sa.block_masks(stream, None, device=tokens.device)["full_attention"], D**-0.5)
        ends, at = {}, 0
        for t, b in zip(self.documents, below):
            at += len(t)
            for r in b:
                at += len(answers[r][1])
                ends[r] = int(real[at - 1])
        return {r: out[i] for r, i in ends.items()}


def run(device, record, steps, seats=9):
    """-> the answers' tokens [steps, seats], the largest deviation of an answer's last attention from reading anew"""
    g = torch.Generator().manual_seed(1)
    text = lambda n: torch.randint(VOCAB, (n,), generator=g).to(device)  # noqa: E731
    x = Session(Model(device), [text(n) for n in (700, 333, 45)], seats, 320, steps, device)
    asked = {r: (r * 3 // seats, text(4 + 7 * r)) for r in range(seats)}
    x.arrive(asked)
    graph, out, worst, began = None, None, 0.0, {}
    for i in range(steps):
        if i == steps // 2:                                                    # two others take seats, below other documents
            for r, c in ((1, 2), (seats - 1, 0)):
                asked[r] = (c, text(11))
            x.arrive({r: asked[r] for r in (1, seats - 1)})
            began = {1: i, seats - 1: i}
        if record and i == 2:                                                  # (recorded once, between two tokens: recording runs nothing)
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                out = x.token()
        if graph is not None:
            graph.replay()
        else:
            out = x.token()
    torch.cuda.synchronize()
    said, took = x.text.tolist(), x.seats.took.tolist()
    answers = {}
    for r, (c, prompt) in asked.items():
        tokens = [line[r] for line in said[began.get(r, 0) :] if line[r] >= 0]
        answers[r] = (c, torch.cat([prompt, torch.tensor(tokens, dtype=torch.int64, device=device)]))
    assert x.seats.lens.tolist() == [len(answers[r][1]) for r in range(seats)]
    first = x.seats.first.tolist()
    for r, want in x.anew(answers).items():
        if took[r]:
            worst = max(worst, float((out[first[r]].float() - want.float()).abs().max()))
    return x.text, worst


def main(device="cuda", steps=8):
    plain, off = run(device, False, steps)
    replayed, off_too = run(device, True, steps)
    return {"same tokens": bool(torch.equal(plain, replayed)), "tokens": int((plain >= 0).sum()), "deviation": max(off, off_too)}


if __name__ == "__main__":
    for what, value in main().items():
        print(f"{what}: {value}")
