"""Tokens drawn from logits by given random numbers: temperature, top-k, top-p and min-p of every row, by the HIP kernels of libspinf_tree.so.  There is no CPU path.

    lp = lm_head_logprobs(Hf, sel, W, None, softcap)               # or logits of any other head
    token = sample_tokens(lp, torch.rand(len(sel), device=dev), temperature=0.8, top_k=40)

The reference draws no tokens: it reads log-probs of given options and takes the best ones of its extraction decoder (spinf_serve/decode.py:246-300).
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib
from .paged import _whole

_SETTINGS = (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32))


def _sample(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor], top_k: Optional[torch.Tensor], top_p: Optional[torch.Tensor], min_p: Optional[torch.Tensor],
            numbers: list[float], want_prob: bool) -> tuple[torch.Tensor, torch.Tensor]:
    if not logits.is_cuda:
        raise RuntimeError("spinf::sample_tokens runs on ROCm device tensors only (no CPU path)")
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16) or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("sample_tokens: logits must be a fp32 or bf16 matrix with contiguous rows")
    rows, vocab = logits.shape
    if u.dtype not in (torch.float32, torch.float64) or u.shape != (rows,) or not u.is_contiguous():
        raise ValueError(f"sample_tokens: u must hold {rows} contiguous fp32 or fp64 values")
    given = (temperature, top_k, top_p, min_p)
    for (name, dt), t in zip(_SETTINGS, given):
        if t is not None and (t.dtype != dt or t.shape != (rows,) or not t.is_contiguous()):
            raise ValueError(f"sample_tokens: {name} must be a number or hold {rows} contiguous {dt} values")
    device = logits.device
    _lib.same_device(device, u, *given)
    a = _lib.SampleArgs()
    a.logits, a.ld, a.rows, a.vocab = logits.data_ptr(), logits.stride(0) if rows > 1 else max(logits.stride(0), vocab), rows, vocab
    a.dtype, a.u_f64 = int(logits.dtype == torch.bfloat16), int(u.dtype == torch.float64)
    a.u = u.data_ptr()
    a.temperature, a.top_k, a.top_p, a.min_p = (t.data_ptr() if t is not None else None for t in given)
    a.all_temperature, a.all_top_k, a.all_top_p, a.all_min_p = numbers[0], int(numbers[1]), numbers[2], numbers[3]
    token = torch.empty(rows, dtype=torch.int64, device=device)
    prob = torch.empty(rows if want_prob else 0, dtype=torch.float32, device=device)
    lib = _lib.load_library()
    need = C.c_int64()
    _lib.check(lib.spinf_sample_workspace(C.byref(a), C.byref(need)), "sample_tokens")
    if rows:
        work = torch.empty(max(need.value, 16), dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes, a.token = work.data_ptr(), work.numel(), token.data_ptr()
        if want_prob:
            a.prob = prob.data_ptr()
        _lib.launch(lib.spinf_sample, a, device, "sample_tokens")
    return token, prob


_sample_op = torch.library.custom_op("spinf::sample_tokens", _sample, mutates_args=())


@_sample_op.register_fake
def _(logits, u, temperature, top_k, top_p, min_p, numbers, want_prob):
    rows = logits.shape[0]
    return torch.empty(rows, dtype=torch.int64, device=logits.device), torch.empty(rows if want_prob else 0, dtype=torch.float32, device=logits.device)


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_prob=False):
    """logits [rows, vocab] fp32 / bf16 (log-probs will do), u [rows] fp32 / fp64 in 0 .. 1 -> tokens [rows] int64, drawn from softmax(logits / temperature) among what is kept: the
    ``top_k`` largest logits (0: all; of equal ones the lower index first), of these the fewest that hold ``top_p`` of their probability, of these the ones at least ``min_p`` times as
    likely as the likeliest.  The token drawn is the first, in the vocabulary's order, up to which the kept probabilities add up to more than u of their sum.  return_prob: also its
    probability among the kept ones, [rows] fp32.
    temperature, top_k, top_p, min_p: numbers (taken as 32 bits hold them), or [rows] device tensors (fp32; top_k int32).  Temperature 0: the largest logit.  Logits of -inf and NaN are never
    drawn; a row without any other, or with a setting that is negative or NaN, gives -1 (probability 0).  Probabilities and their sums are 64-bit, in steps of 2^-47 of the largest
    of 8,192 neighbours (one of less than half a step is none): the same call gives the same tokens whatever rows share it."""
    given, numbers = [], []
    for (name, _), x in zip(_SETTINGS, (temperature, top_k, top_p, min_p)):
        given.append(x if isinstance(x, torch.Tensor) else None)
        n = 0.0 if isinstance(x, torch.Tensor) else _whole(x, "sample_tokens: top_k") if name == "top_k" else float(x)
        if not n >= 0:
            raise ValueError(f"sample_tokens: {name} {x}")
        numbers.append(float(min(n, 1 << 30)) if name == "top_k" else n)
    run = _sample if _lib.eager(logits, u, *given) else _sample_op
    token, prob = run(logits, u, *given, numbers, bool(return_prob))
    return (token, prob) if return_prob else token
