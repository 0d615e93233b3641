"""The paged cache's operators in float64, from their definitions (test infrastructure; csrc/paged_*.hip are checked against it)."""

from __future__ import annotations

import numpy as np


def stored(pages, table, n):
    """[n, heads, d]: a request's stored rows, key by key from the page list"""
    page = pages.shape[1]
    return np.stack([pages[table[s // page], s % page] for s in range(n)]).astype(np.float64) if n else np.zeros((0, *pages.shape[2:]))


def visible(T, L, end=None, pos=None, base=0, window=0):
    """[T, L] bool: which stored keys the new tokens of a request see; end, pos: of its rows, end in rows of the call (its first row is ``base``)"""
    c = L - T
    i, s = np.arange(T)[:, None], np.arange(L)[None, :]
    see = s <= c + i
    if end is not None:
        see[:, c:] &= i < (np.asarray(end) - base)[None, :]
    if window:
        at = np.arange(L)
        if pos is not None:
            at[c:] = pos
        see &= (at[c:] if c >= 0 else np.arange(c, L))[:, None] - at[None, :] < window
    return see


def attention(q, k, v, see, scale, softcap=0.0):
    """q [T, hq, d], k, v [L, hkv, d], see [T, L] -> out [T, hq, d], lse [T, hq], sum p |v| / sum p, sum |q| |k| scale (largest over the keys): the last
    two for error bounds"""
    T, hq, d = q.shape
    L, hkv, _ = k.shape
    out, mag = np.zeros((T, hq, d)), np.zeros((T, hq, d))
    lse, size = np.full((T, hq), -np.inf), np.zeros((T, hq))
    for h in range(hq):
        kk, vv = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        for i in range(T):
            on = np.flatnonzero(see[i])
            if len(on) == 0:
                continue
            t = kk[on] @ q[i, h] * scale
            if softcap:
                t = softcap * np.tanh(t / softcap)
            size[i, h] = (np.abs(kk[on]) @ np.abs(q[i, h])).max() * scale
            top = t.max()
            p = np.exp(t - top)
            out[i, h] = p @ vv[on] / p.sum()
            mag[i, h] = p @ np.abs(vv[on]) / p.sum()
            lse[i, h] = top + np.log(p.sum())
    return out, lse, mag, size
