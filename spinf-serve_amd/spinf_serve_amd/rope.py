"""What lies between a layer's projection and its attention: norms of queries and keys for each head, with the rotation by position in the same pass,
and the keys' and values' way into a paged cache; one HIP kernel of libspinf_tree.so.

    q, k = qk_norm_rope(q, k, wq, wk, cos, sin, eps, pos)                              # then tree_attn(q, k, v, mask, scale)
    slots, pos = batch.rows()
    q = qk_norm_rope_put(q, k, v, wq, wk, cos, sin, eps, cache, slots, pos=pos)        # then paged_attn(q, cache, batch, scale)

q, k, v may be views of one projection's output.  There is no CPU path.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

_TABLE = (torch.float32, torch.bfloat16)
_DENSE = torch.contiguous_format   # (an output made like its input costs the host half of what one of a given shape does)


def _rope_args(q, k, v, wq, wk, cos, sin, eps, pos, neighbours, plus_one, what):
    if not q.is_cuda:
        raise RuntimeError(f"spinf::{what} runs on ROCm device tensors only (no CPU path)")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t is None:
            continue
        if t.dtype != torch.bfloat16 or t.dim() != 3 or t.stride(2) != 1:
            raise ValueError(f"{name} must be bf16 [tokens, heads, head dim] with contiguous head dims")
        if t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
            raise ValueError(f"{name} must be 16-byte aligned with strides that are multiples of 8 elements")
    T, hq, d = q.shape
    hkv = k.shape[1]
    if k.shape != (T, hkv, d) or (v is not None and v.shape != (T, hkv, d)):
        raise ValueError(f"k {tuple(k.shape)}, v {None if v is None else tuple(v.shape)} do not match q {tuple(q.shape)}")
    if d not in (64, 128, 256, 512):
        raise ValueError(f"head dim {d} not supported (64, 128, 256, 512)")
    a = _lib.RopeArgs()
    for name, w in (("wq", wq), ("wk", wk)):
        if w is not None:
            if w.shape != (d,) or not w.is_contiguous() or w.dtype not in _TABLE or w.data_ptr() % 16:
                raise ValueError(f"{name} must hold {d} contiguous, 16-byte aligned fp32 or bf16 values")
            setattr(a, name, w.data_ptr())
    if wq is not None and wk is not None and wq.dtype != wk.dtype:
        raise ValueError("wq and wk must have one type")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype not in _TABLE or cos.dtype != sin.dtype:
        raise ValueError("cos and sin must be [positions, rotated dims / 2], fp32 or bf16, alike")
    rot = 2 * cos.shape[1]
    if rot > d or rot % 16:
        raise ValueError(f"{rot} of {d} dims rotated: a multiple of 16 is needed")
    per16 = 16 // cos.element_size()
    if rot and (cos.stride(1) != 1 or sin.stride(1) != 1 or (cos.shape[0] > 1 and (cos.stride(0) % per16 or sin.stride(0) % per16)) or cos.data_ptr() % 16 or sin.data_ptr() % 16):
        raise ValueError("rows of cos and sin must be contiguous and 16-byte aligned")
    if pos is not None and (pos.shape != (T,) or pos.dtype not in (torch.int32, torch.int64) or not pos.is_contiguous()):
        raise ValueError(f"pos must hold {T} contiguous int32 or int64 values")
    if rot and (cos.shape[0] < T if pos is None else T and not cos.shape[0]):
        raise ValueError(f"tables of {cos.shape[0]} positions for {T} tokens")
    if not 0 <= eps < float("inf"):
        raise ValueError(f"eps {eps}")
    _lib.same_device(q.device, k, v, wq, wk, cos, sin, pos)
    a.q, a.q_tok, a.q_head, a.k, a.k_tok, a.k_head = q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1)
    if v is not None:
        a.v, a.v_tok, a.v_head = v.data_ptr(), v.stride(0), v.stride(1)
    a.cos, a.sin, a.cos_ld, a.sin_ld, a.n_pos = cos.data_ptr(), sin.data_ptr(), cos.stride(0), sin.stride(0), cos.shape[0]
    if cos.shape[0] == 1:   # (one row: its stride is anything)
        a.cos_ld = a.sin_ld = 0
    a.pos = pos.data_ptr() if pos is not None else None
    a.T, a.hq, a.hkv, a.d, a.rot = T, hq, hkv, d, rot
    a.neighbours, a.plus_one = int(neighbours), int(plus_one)
    w = wq if wq is not None else wk
    a.w_f32, a.cs_f32, a.pos_i64 = int(w is not None and w.dtype == torch.float32), int(cos.dtype == torch.float32), int(pos is not None and pos.dtype == torch.int64)
    a.eps = eps
    return a


# Argument blocks without their tensors' addresses, by everything the checks above look at (shapes, strides, types, numbers): a layer's later calls
# check the devices and the alignment alone.
_SEEN: dict = {}


def _known(key, index, tensors):
    """the block kept for this key with the tensors' addresses, if they lie on GPU `index` and are aligned as the kernel wants them"""
    got = _SEEN.get(key)
    if got is None or index < 0:
        return None
    at, bits = [], 0
    for t in tensors:
        if t is None:
            at.append(None)
            continue
        if t.get_device() != index:
            return None   # (the checks say what is wrong)
        x = t.data_ptr()
        bits |= x
        at.append(x)
    if bits % 16:
        return None
    a = _lib.RopeArgs.from_buffer_copy(got)
    a.q, a.k, a.v, a.wq, a.wk, a.cos, a.sin = at[:7]
    return a


def _table(wq, wk, cos, sin, pos):
    """what the checks look at of the weights, the tables and the positions"""
    return (None if wq is None else (wq.shape, wq.stride(), wq.dtype), None if wk is None else (wk.shape, wk.stride(), wk.dtype), cos.shape, cos.stride(), cos.dtype,
            sin.shape, sin.stride(), sin.dtype, None if pos is None else (pos.shape, pos.stride(), pos.dtype))


def _note(key, a):
    if len(_SEEN) > 1024:
        _SEEN.clear()
    _SEEN[key] = bytes(a)


def _rope(q: torch.Tensor, k: torch.Tensor, wq: Optional[torch.Tensor], wk: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, eps: float,
          pos: Optional[torch.Tensor], neighbours: bool, plus_one: bool) -> tuple[torch.Tensor, torch.Tensor]:
    device, index = q.device, q.get_device()
    key = (q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, _table(wq, wk, cos, sin, pos), eps, neighbours, plus_one)
    a = _known(key, index, (q, k, None, wq, wk, cos, sin))
    if a is None or (pos is not None and pos.get_device() != index):
        a = _rope_args(q, k, None, wq, wk, cos, sin, eps, pos, neighbours, plus_one, "qk_norm_rope")
        _note(key, a)
    q_out, k_out = torch.empty_like(q, memory_format=_DENSE), torch.empty_like(k, memory_format=_DENSE)
    a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
    a.pos = pos.data_ptr() if pos is not None else None
    if q.shape[0]:
        _lib.launch(_lib.load_library().spinf_qk_norm_rope, a, device, "spinf_qk_norm_rope")
    return q_out, k_out


_rope_op = torch.library.custom_op("spinf::qk_norm_rope", _rope, mutates_args=())


@_rope_op.register_fake
def _(q, k, wq, wk, cos, sin, eps, pos, neighbours, plus_one):
    return tuple(torch.empty(t.shape, dtype=torch.bfloat16, device=q.device) for t in (q, k))


def qk_norm_rope(q, k, wq, wk, cos, sin, eps, pos=None, neighbours=False, plus_one=False):
    """q [tokens, hq, d], k [tokens, hkv, d] bf16 -> the same, dense: x / sqrt(mean x^2 + eps) * w per head (w [d] fp32 or bf16; None: no weight;
    ``plus_one``: 1 + w), then the first 2 cos.shape[1] dims rotated in pairs (i, i + half), or (2 i, 2 i + 1) with ``neighbours``, by the rows ``pos`` of cos
    and sin [positions, half] (pos None: row t for token t).  fp32 throughout, rounded once.  A position outside the tables gives NaN."""
    run = _rope if _lib.eager(q, k, wq, wk, cos, sin) else _rope_op
    return run(q, k, wq, wk, cos, sin, float(eps), pos, bool(neighbours), bool(plus_one))


def _put(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, wq: Optional[torch.Tensor], wk: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, eps: float,
         ck: torch.Tensor, cv: torch.Tensor, slots: torch.Tensor, pos: Optional[torch.Tensor], neighbours: bool, plus_one: bool, v_norm: bool) -> torch.Tensor:
    device, index = q.device, q.get_device()
    key = (q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, v.shape, v.stride(), v.dtype, ck.shape, ck.stride(), cv.stride(), slots.shape, slots.stride(), slots.dtype,
           _table(wq, wk, cos, sin, pos), eps, neighbours, plus_one, v_norm)
    a = _known(key, index, (q, k, v, wq, wk, cos, sin, ck, cv))
    if a is None or (pos is not None and pos.get_device() != index) or slots.get_device() != index:
        a = _rope_args(q, k, v, wq, wk, cos, sin, eps, pos, neighbours, plus_one, "qk_norm_rope_put")
        if ck.shape[2:] != k.shape[1:]:
            raise ValueError(f"the cache holds {tuple(ck.shape[2:])} a key, the layer makes {tuple(k.shape[1:])}")
        if slots.dtype != torch.int64 or slots.shape != (q.shape[0],) or not slots.is_contiguous():
            raise ValueError(f"slots must hold {q.shape[0]} contiguous int64 values")
        if q.shape[0] and (ck.shape[0] == 0 or ck.shape[0] * ck.shape[1] >= 1 << 31):
            raise ValueError(f"a cache of {ck.shape[0]} pages of {ck.shape[1]} keys")
        _lib.same_device(device, ck, cv, slots)
        a.k_page, a.k_row, a.kh_out = ck.stride()[:3]
        a.v_page, a.v_row, a.vh_out = cv.stride()[:3]
        a.pages, a.page, a.v_norm = ck.shape[0], ck.shape[1], int(v_norm)
        _note(key, a)
    q_out = torch.empty_like(q, memory_format=_DENSE)
    a.q_out, a.k_out, a.v_out, a.slots = q_out.data_ptr(), ck.data_ptr(), cv.data_ptr(), slots.data_ptr()
    a.pos = pos.data_ptr() if pos is not None else None
    if q.shape[0]:
        _lib.launch(_lib.load_library().spinf_qk_norm_rope, a, device, "spinf_qk_norm_rope")
    return q_out


_put_op = torch.library.custom_op("spinf::qk_norm_rope_put", _put, mutates_args=("ck", "cv"))


@_put_op.register_fake
def _(q, k, v, wq, wk, cos, sin, eps, ck, cv, slots, pos, neighbours, plus_one, v_norm):
    return torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)


def qk_norm_rope_put(q, k, v, wq, wk, cos, sin, eps, cache, slots, pos=None, neighbours=False, plus_one=False, v_norm=False):
    """as qk_norm_rope, but the keys and the values (``v_norm``: normed too, without weight) go into ``cache`` (a PagedCache): token t's become entry
    slots[t] % page of page slots[t] // page (slots int64; PagedBatch.rows() has them).  -> the queries.  A negative slot stores nothing (a pad); a slot
    behind the cache stores nothing either, and that token's query comes out as NaN.  Slots should differ: of two tokens with one, every 16 bytes are either's."""
    run = _put if _lib.eager(q, k, v, wq, wk, cos, sin, cache.k, cache.v) else _put_op
    return run(q, k, v, wq, wk, cos, sin, float(eps), cache.k, cache.v, slots, pos, bool(neighbours), bool(plus_one), bool(v_norm))
