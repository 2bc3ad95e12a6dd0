"""Choice of the next token from a model's logits (``gq_sample``).

The counterpart of ``eval.masked_nll_from_logits``, which scores given tokens
on the same logits: ``sample_tokens`` draws one per row from uniform numbers
that the caller provides, so a run can be repeated exactly.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _arrays as A
from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_KINDS = {torch.float32: 1, torch.float64: 2, torch.int32: 3, torch.int64: 4}


class Sampled(NamedTuple):
    tokens: torch.Tensor    # [rows] int64; -1 where no token was left
    logprobs: torch.Tensor  # [rows] float32: log of the token's share of what was kept


def _setting(name: str, v, rows: int, logits: torch.Tensor, lo: float, hi: float | None):
    """(pointer, kind, value, tensor kept alive) of a setting."""
    if not isinstance(v, torch.Tensor):
        if not v >= lo or (hi is not None and v > hi):
            raise ValueError(f"{name} must be at least {lo}"
                             + (f" and at most {hi}" if hi else "") + f", got {v}")
        return None, 0, v, None
    kind = _KINDS.get(v.dtype)
    if kind is None:
        raise ValueError(f"{name} must be float32, float64, int32 or int64, got {v.dtype}")
    if v.dim() != 1 or v.shape[0] != rows or v.get_device() != logits.get_device():
        raise ValueError(f"{name} must have one value per row ([{rows}] on {logits.device}), got "
                         f"{tuple(v.shape)} on {v.device}")
    t = v if v.is_contiguous() else v.contiguous()
    return t.data_ptr(), kind, 0.0, t


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0) -> Sampled:
    """One token per row of ``logits`` [rows, vocab] (or [vocab]: one row),
    float32, bf16 or fp16 on the device, at most 2^20 tokens.

    ``u``: float32 or float64 [rows] in [0, 1).  Each setting is a number or a
    tensor with one value per row.  With e = exp((logit - max) / temperature)
    and the tokens ordered by logit, equal ones by index, ``top_k`` keeps the
    first k (0: all); ``top_p`` keeps of those the ones before which less than
    that share of their mass lies; ``min_p`` keeps of those the ones with
    e >= min_p.  The most likely token always stays.  The result is the
    smallest index at which the running sum of the kept e exceeds u times their
    total.  ``temperature`` 0 takes the first largest logit; others count as at
    least 1e-37 and at most 1e36.  NaN and -inf logits are never taken; a row with
    nothing else gives -1 and -inf.  Terms are whole numbers of 2^-45 of the
    largest (2^-42 for the largest vocabularies): a token below half of that is
    never drawn.  The results carry no gradients."""
    dt = _DTYPES.get(logits.dtype)
    if dt is None:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() not in (1, 2) or not 1 <= logits.shape[-1] <= 1 << 20:
        raise ValueError(f"logits must be [rows, vocab] with 1 .. 2^20 tokens, got "
                         f"{tuple(logits.shape)}")
    if not logits.is_cuda:
        raise ValueError(f"logits must be on a CUDA device, got {logits.device}")
    lg = logits if logits.dim() == 2 else logits[None]
    rows, vocab = lg.shape
    if lg.stride(1) != 1 or (rows > 1 and lg.stride(0) < vocab):
        lg = lg.contiguous()
    ld = lg.stride(0) if rows > 1 else vocab  # (one row's stride may be any number)
    if u.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"u must be float32 or float64, got {u.dtype}")
    dev = lg.get_device()
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return sample_tokens(logits, u, temperature, top_k, top_p, min_p)
    uk = _KINDS[u.dtype]
    if u.dim() != 1 or u.shape[0] != rows or u.get_device() != dev or u.stride(0) != 1:
        up, uk, _, u = _setting("u", u.reshape(1) if u.dim() == 0 else u, rows, lg, 0.0, None)
    up = u.data_ptr()
    tp, tk, tv, t0 = _setting("temperature", temperature, rows, lg, 0.0, None)
    kp, kk, kv, t1 = _setting("top_k", top_k, rows, lg, 0, None)
    pp, pk, pv, t2 = _setting("top_p", top_p, rows, lg, 0.0, 1.0)
    mp, mk, mv, t3 = _setting("min_p", min_p, rows, lg, 0.0, 1.0)
    tokens = torch.empty_like(u, dtype=torch.int64)
    logprobs = torch.empty_like(u, dtype=torch.float32)
    if rows:
        status = _lib.lib().gq_sample(lg.data_ptr(), dt, rows, vocab, ld, up, uk, tp, tk,
                                      tv, kp, kk, kv, pp, pk, pv, mp, mk, mv, tokens.data_ptr(),
                                      logprobs.data_ptr(), A.raw_stream(dev))
        if status:
            _lib.raise_status(status)
    return Sampled(tokens, logprobs)


__all__ = ["Sampled", "sample_tokens"]
