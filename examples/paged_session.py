"""Contents that stay: one attention layer that reads two documents once, keeps their keys and values in a paged cache, answers questions about them that
come later, goes on token by token, and trims what it keeps.

    python examples/paged_session.py        (needs an MI355X and the built library)

Every step is checked: against tree_attn over the same tokens packed into one stream, i.e. against reading the documents anew, and what follows the trimming
against plain attention over the keys that stayed.
"""

from __future__ import annotations

import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spinf-serve_amd"))

import spinf_serve_amd as sa  # noqa: E402

HQ, HKV, D, HIDDEN, PAGE = 16, 8, 128, 512, 64


class Layer:
    """a projection to queries, keys and values, norms per head, rotation by position"""

    def __init__(self, device, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.w = (torch.randn((HIDDEN, (HQ + 2 * HKV) * D), generator=g) * HIDDEN**-0.5).to(torch.bfloat16).to(device)
        self.wq, self.wk = (torch.rand(D, generator=g).add_(0.5).to(device) for _ in range(2))
        ang = torch.arange(8192)[:, None] * 10000.0 ** (-torch.arange(D // 2) / (D // 2))[None]
        self.cos, self.sin = ang.cos().to(device), ang.sin().to(device)

    def project(self, x):
        return (t.unflatten(1, (-1, D)) for t in (x @ self.w).split([HQ * D, HKV * D, HKV * D], 1))

    def paged(self, x, cache, batch, **how):
        """the new tokens' keys and values into the cache, their attention over all that is stored"""
        slots, pos = batch.rows()
        q, k, v = self.project(x)
        q = sa.qk_norm_rope_put(q, k, v, self.wq, self.wk, self.cos, self.sin, 1e-6, cache, slots, pos=pos)
        return q, sa.paged_attn(q, cache, batch, **how)

    def anew(self, x, stream):
        """the same tokens as one packed stream, nothing kept"""
        q, k, v = self.project(x)
        pos = torch.from_numpy(stream.pos.astype(np.int64)).to(x.device)
        q, k = sa.qk_norm_rope(q, k, self.wq, self.wk, self.cos, self.sin, 1e-6, pos)
        return sa.tree_attn(q, k, v, sa.block_masks(stream, None, device=x.device)["full_attention"], D**-0.5)

    def trimmed(self, text, asks, question, stay):
        """one text's questions (branches of question[i] tokens) over the keys that stayed [kv heads, keys], rotated by the positions they were read at"""
        q, k, v = self.project(torch.cat([text, asks]))
        at = [*range(len(text)), *(len(text) + i for b in question for i in range(b))]
        q, k = sa.qk_norm_rope(q, k, self.wq, self.wk, self.cos, self.sin, 1e-6, torch.tensor(at, device=text.device))
        out, first = [], len(text)
        for b in question:
            new = slice(first, first + b)
            for h in range(HQ):
                kk, vv = (torch.cat([t[stay[h // (HQ // HKV)], h // (HQ // HKV)], t[new, h // (HQ // HKV)]]).float() for t in (k, v))
                s = (q[new, h].float() @ kk.T) * D**-0.5
                s += torch.full_like(s, float("-inf")).triu(1 + kk.shape[0] - b)
                out.append(s.softmax(1) @ vv)
            first += b
        return torch.cat([torch.stack(out[i : i + HQ], 1) for i in range(0, len(out), HQ)])


def main(device="cuda", documents=(700, 333), questions=((7, 12, 9), (5, 16)), steps=3, keep=256):
    """-> the largest deviation from reading anew, by step"""
    g = torch.Generator().manual_seed(1)
    rand = lambda n: torch.randn((n, HIDDEN), generator=g).to(torch.bfloat16).to(device)  # noqa: E731
    layer = Layer(device)
    # pages of a simple allocator: a document's own, then scratch for its questions
    need = [-(-(n + sum(q) + steps) // PAGE) for n, q in zip(documents, questions)]
    free = list(np.random.default_rng(0).permutation(2 * sum(need)))
    tables = [[free.pop() for _ in range(n)] for n in need]
    cache = sa.PagedCache.empty(2 * sum(need), PAGE, HKV, D, device)
    off = {}

    # 1. the documents are read once
    docs = [rand(n) for n in documents]
    batch = sa.PagedBatch.build(documents, documents, tables, PAGE, device)
    _, out = layer.paged(torch.cat(docs), cache, batch)
    stream = sa.pack_stream([sa.TokenTree([1] * n, [], []) for n in documents])
    real = torch.from_numpy(np.flatnonzero(stream.art >= 0)).to(device)
    padded = torch.zeros((stream.length, HIDDEN), dtype=torch.bfloat16, device=device)
    padded[real] = torch.cat(docs)
    off["documents"] = float((layer.anew(padded, stream)[real] - out).abs().max())

    # 2. questions come later: trees of branches below the stored documents; their keys are scratch, the next call forgets them
    asks = [rand(sum(q)) for q in questions]
    end, pos, base = [], [], 0
    for n, q in zip(documents, questions):
        for b in q:
            end += [base + b] * b
            pos += range(n, n + b)
            base += b
    batch = sa.PagedBatch.build([sum(q) for q in questions], [n + sum(q) for n, q in zip(documents, questions)], tables, PAGE, device, end=end, pos=pos)
    _, out = layer.paged(torch.cat(asks), cache, batch)
    stream = sa.pack_stream([sa.TokenTree([1] * n, [[2] * b for b in q], [-1] * len(q)) for n, q in zip(documents, questions)])
    real = torch.from_numpy(np.flatnonzero(stream.art >= 0)).to(device)
    padded = torch.zeros((stream.length, HIDDEN), dtype=torch.bfloat16, device=device)
    padded[real] = torch.cat([t for d, a in zip(docs, asks) for t in (d, a)])
    want = layer.anew(padded, stream)[real].split([t for n, q in zip(documents, questions) for t in (n, sum(q))])[1::2]
    off["questions"] = float((torch.cat(want) - out).abs().max())

    # 3. token by token, and what the tokens look at
    weight, texts, lens = None, list(docs), list(documents)
    for _ in range(steps):
        new = rand(len(lens))
        texts = [torch.cat([t, new[i : i + 1]]) for i, t in enumerate(texts)]
        lens = [n + 1 for n in lens]
        batch = sa.PagedBatch.build([1] * len(lens), lens, tables, PAGE, device)
        q, (out, lse) = layer.paged(new, cache, batch, return_lse=True)
        if weight is not None:
            weight = torch.nn.functional.pad(weight, (0, max(lens) - weight.shape[2]))
        weight = sa.paged_weights(q, cache, batch, lse, acc=weight)
        stream = sa.pack_stream([sa.TokenTree([1] * n, [], []) for n in lens])
        ends = [int(np.flatnonzero(stream.art == a)[-1]) for a in sorted(set(stream.art[stream.art >= 0].tolist()))]
        real = torch.from_numpy(np.flatnonzero(stream.art >= 0)).to(device)
        padded = torch.zeros((stream.length, HIDDEN), dtype=torch.bfloat16, device=device)
        padded[real] = torch.cat(texts)
        off["steps"] = max(off.get("steps", 0.0), float((layer.anew(padded, stream)[ends] - out).abs().max()))
    off["weights"] = float((weight.sum(2) - steps * HQ / HKV).abs().max())   # each token gave every head's weight away, one in all

    # 4. the documents are trimmed to the keys that were looked at, and the old pages are free again; questions go on from where the texts are, below what is left of them
    fresh = [[free.pop() for _ in range(-(-(min(n, keep) + sum(q)) // PAGE))] for n, q in zip(lens, questions)]
    left = [min(n, keep) for n in lens]
    into = sa.PagedBatch.build([0] * len(lens), left, fresh, PAGE, device)
    kept, weight = sa.cache_evict(cache, batch, into, weight, keep, sink=4, recent=32)
    asks = [rand(sum(q)) for q in questions]
    end, pos, base = [], [], 0
    for n, q in zip(lens, questions):
        for b in q:
            end += [base + b] * b
            pos += range(n, n + b)                                             # (positions in the text, of which n - left tokens are gone)
            base += b
    batch = sa.PagedBatch.build([sum(q) for q in questions], [n + sum(q) for n, q in zip(left, questions)], fresh, PAGE, device, end=end, pos=pos,
                                dropped=[n - m for n, m in zip(lens, left)])
    _, out = layer.paged(torch.cat(asks), cache, batch)
    want = [layer.trimmed(t, a, q, stay[:, :m]) for t, a, q, stay, m in zip(texts, asks, questions, kept.long(), left)]
    off["trimmed"] = float((torch.cat(want) - out).abs().max())
    return off


if __name__ == "__main__":
    for step, worst in main().items():
        print(f"{step}: largest deviation {worst:.2e}")
