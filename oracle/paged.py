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


def weights(q, k, see, lse, scale, softcap=0.0):
    """[hkv, L]: the weight each key got, exp(score - lse) over the rows that see it and the heads of its key / value head"""
    T, hq, d = q.shape
    L, hkv, _ = k.shape
    out = np.zeros((hkv, L))
    for h in range(hq):
        t = q[:, h] @ k[:, h // (hq // hkv)].T * scale
        if softcap:
            t = softcap * np.tanh(t / softcap)
        with np.errstate(invalid="ignore", over="ignore"):
            p = np.where(see, np.exp(t - lse[:, h : h + 1]), 0)
        out[h // (hq // hkv)] += p.sum(0)
    return out


def keep_places(acc, n, keep, sink, recent):
    """ascending places that stay of n, by acc [n]"""
    if n <= keep:
        return np.arange(n)
    mid = np.arange(sink, n - recent)
    a = np.where(np.isnan(acc[mid]), np.inf, acc[mid]).astype(np.float64)
    nan = np.isnan(acc[mid])
    order = np.lexsort((mid, -a, ~nan))   # NaN first, then by weight, then by place
    return np.sort(np.concatenate([np.arange(sink), mid[order[: keep - sink - recent]], np.arange(n - recent, n)]))


def norm_rope(x, w, cos, sin, eps, neighbours=False, plus_one=False):
    """x [T, H, d], w [d] or None, cos, sin [T, half] -> float64"""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if w is not None:
        y = y * (w.astype(np.float64) + (1 if plus_one else 0))
    half = cos.shape[1]
    c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
    i, j = (np.arange(0, 2 * half, 2), np.arange(1, 2 * half, 2)) if neighbours else (np.arange(half), np.arange(half, 2 * half))
    out = y.copy()
    out[..., i] = y[..., i] * c - y[..., j] * s
    out[..., j] = y[..., j] * c + y[..., i] * s
    return out
