"""Rotary positions of queries and keys (``gq_rotary``).

A :class:`RotaryPlan` holds the frequencies of one head layout, as 64-bit
fractions of a turn, so that far positions keep every digit of their angle;
``apply_rotary`` turns queries and keys by it.  Long-context scalings change
the frequencies only (and for :class:`YarnScaling` a factor on the result).
"""

from __future__ import annotations

import math
import struct
from dataclasses import dataclass
from fractions import Fraction

import torch

from . import _arrays as A
from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_POSITIONS = (torch.int64, torch.int32)
_STRIDES = struct.Struct("12q").pack  # the strides argument of gq_rotary
_PI = Fraction("3.14159265358979323846264338327950288419716939937510")


@dataclass(frozen=True)
class LinearScaling:
    """Positions divided by ``factor``."""
    factor: float


@dataclass(frozen=True)
class NtkScaling:
    """The base raised so that the slowest pair is slowed down by ``factor``
    and the fastest is kept: theta' = theta * factor^(d / (d - 2))."""
    factor: float


@dataclass(frozen=True)
class YarnScaling:
    """By parts: pairs that turn more than ``beta_fast`` times over
    ``original_positions`` keep their frequency, pairs that turn less than
    ``beta_slow`` times are slowed down by ``factor``, a linear ramp between;
    results are multiplied by ``attention_factor`` (None: 0.1 ln factor + 1)."""
    factor: float
    original_positions: int
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None


@dataclass(frozen=True)
class Llama3Scaling:
    """By wavelength: pairs longer than ``original_positions / low_freq_factor``
    are slowed down by ``factor``, shorter than ``original_positions /
    high_freq_factor`` kept, between them both are blended."""
    factor: float
    original_positions: int
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0


Scaling = LinearScaling | NtkScaling | YarnScaling | Llama3Scaling


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0,
                       scaling: Scaling | None = None) -> tuple[list[float], float]:
    """Radians per position of each pair, and the factor on the result."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not theta > 0 or not math.isfinite(theta):
        raise ValueError(f"theta must be positive, got {theta}")
    d = rotary_dim
    if scaling is not None and not (scaling.factor > 0 and math.isfinite(scaling.factor)):
        raise ValueError(f"scaling factor must be positive, got {scaling.factor}")
    if isinstance(scaling, NtkScaling) and d > 2:
        theta = theta * scaling.factor ** (d / (d - 2))
    inv = [theta ** (-2.0 * i / d) for i in range(d // 2)]
    if scaling is None or isinstance(scaling, NtkScaling):
        return inv, 1.0
    if isinstance(scaling, LinearScaling):
        return [w / scaling.factor for w in inv], 1.0
    n = scaling.original_positions
    if n < 1:
        raise ValueError(f"original_positions must be positive, got {n}")
    if isinstance(scaling, YarnScaling):
        if not scaling.beta_fast > 0 or not scaling.beta_slow > 0 or theta == 1.0:
            raise ValueError("beta_fast and beta_slow must be positive, theta not 1")

        def pair(turns):  # the pair that turns this often over n positions
            return d * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo = max(math.floor(pair(scaling.beta_fast)), 0)
        hi = min(math.ceil(pair(scaling.beta_slow)), d - 1)
        out = []
        for i, w in enumerate(inv):
            keep = 1.0 - min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
            out.append(w * keep + w / scaling.factor * (1.0 - keep))
        f = scaling.attention_factor
        if f is None:
            f = 0.1 * math.log(scaling.factor) + 1.0 if scaling.factor > 1 else 1.0
        return out, f
    if not 0 < scaling.low_freq_factor < scaling.high_freq_factor:
        raise ValueError("low_freq_factor must be positive and below high_freq_factor")
    out = []
    for w in inv:
        turns = n * w / (2 * math.pi)
        keep = (turns - scaling.low_freq_factor) / (scaling.high_freq_factor
                                                    - scaling.low_freq_factor)
        keep = min(max(keep, 0.0), 1.0)
        out.append(w * keep + w / scaling.factor * (1.0 - keep))
    return out, 1.0


@dataclass(frozen=True)
class RotaryPlan:
    """Frequencies of one head layout on the device (``rotary_plan``)."""
    turns: torch.Tensor     # [rotary_dim / 2] int64: 2^-64ths of a turn per position
    head_dim: int
    rotary_dim: int
    interleaved: bool
    factor: float


def rotary_plan(head_dim: int, theta: float = 10000.0, rotary_dim: int | None = None,
                interleaved: bool = False, scaling: Scaling | None = None) -> RotaryPlan:
    """Plan for heads of ``head_dim`` whose first ``rotary_dim`` components
    (default: all) are turned, paired (i, i + rotary_dim / 2) or, with
    ``interleaved``, (2 i, 2 i + 1); on the current device."""
    rd = head_dim if rotary_dim is None else rotary_dim
    if not 2 <= rd <= head_dim <= 4096 or rd % 2:
        raise ValueError(f"rotary_dim must be even and in 2 .. head_dim <= 4096, got {rd} of "
                         f"{head_dim}")
    inv, factor = rotary_frequencies(rd, theta, scaling)
    words = []
    for w in inv:
        t = round(Fraction(w) * (1 << 64) / (2 * _PI)) % (1 << 64)
        words.append(t - (1 << 64) if t >= 1 << 63 else t)
    A.require_cuda()
    return RotaryPlan(torch.tensor(words, dtype=torch.int64, device="cuda"), head_dim, rd,
                      bool(interleaved), float(factor))


def _heads(name: str, x: torch.Tensor, plan: RotaryPlan) -> torch.Tensor:
    if x.dim() != 4 or x.shape[3] != plan.head_dim:
        raise ValueError(f"{name} must be [batch, heads, seq, {plan.head_dim}], got "
                         f"{tuple(x.shape)}")
    return x if x.stride(3) == 1 else x.contiguous()


def _like(x: torch.Tensor) -> torch.Tensor:
    """A new tensor of x's layout; contiguous where that of an overlapping x would
    not leave the components so."""
    o = torch.empty_like(x)
    return o if o.stride(3) == 1 else x.new_empty(x.shape)


def _results(q, k, out):
    oq, ok = out
    if oq is None or (ok is None) != (k is None):
        raise ValueError("out must be a pair like (q, k)")
    if torch.is_grad_enabled() and (oq.requires_grad or (ok is not None and ok.requires_grad)):
        raise ValueError("out takes no gradients: call it under torch.no_grad()")
    pairs = [("q", q, oq)] + ([] if k is None else [("k", k, ok)])
    for name, x, o in pairs:
        if o.shape != x.shape or o.dtype != x.dtype or o.device != x.device or \
                (o.numel() and o.stride(3) != 1):
            raise ValueError(f"out of {name} must be like it, with contiguous components")
        if not A.distinct_elements(o):
            raise ValueError(f"out of {name} has elements that share memory")
        same = o is x or (o.data_ptr() == x.data_ptr() and o.stride() == x.stride())
        if not same and A.overlap(o, x):
            raise ValueError(f"out of {name} partly shares memory with it")
    if k is not None and (A.overlap(oq, ok) or A.overlap(oq, k) or A.overlap(ok, q)):
        raise ValueError("out of q and k share memory with each other or the other input")
    return oq, ok


class _Turned(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, plan, transpose):
        ctx.save_for_backward(positions, plan.turns)
        ctx.plan, ctx.transpose = plan, transpose
        return apply_rotary(q, k, positions, plan, transpose=transpose)

    @staticmethod
    def backward(ctx, gq, gk):
        positions, _ = ctx.saved_tensors
        dq, dk = apply_rotary(gq, gk, positions, ctx.plan, transpose=not ctx.transpose)
        return dq, dk, None, None, None


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                 plan: RotaryPlan, out=None, transpose: bool = False):
    """Queries [B, heads, S, head_dim] and keys [B, kv_heads, S, head_dim]
    (float32, bf16 or fp16, any strides with contiguous components) turned by
    their positions; returns new tensors ``(q, k)`` with the inputs' layout.

    ``positions``: int64 or int32, [S] or [B, S], any values.  ``k`` may be
    None.  ``out``: a pair of tensors to write, which may be ``(q, k)``
    themselves (then without gradients).  ``transpose`` turns back, which is
    the gradient's map: gradients flow to q and k through a second call."""
    dt = _DTYPES.get(q.dtype)
    if dt is None:
        raise ValueError(f"q must be float32, bfloat16 or float16, got {q.dtype}")
    if q.dim() != 4 or q.stride(3) != 1 or q.shape[3] != plan.head_dim:
        q = _heads("q", q, plan)
    b, h, s, d = q.shape
    hk = 0
    if k is not None:
        if k.dtype != q.dtype or k.get_device() != q.get_device():
            raise ValueError("q and k must have one type and device")
        if k.dim() != 4 or k.stride(3) != 1 or k.shape[3] != d:
            k = _heads("k", k, plan)
        kb, hk, ks, _ = k.shape
        if kb != b or ks != s:
            raise ValueError(f"q and k must have one batch and length, got {tuple(q.shape)} and "
                             f"{tuple(k.shape)}")
    if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("out takes no gradients: call it under torch.no_grad()")
        return _Turned.apply(q, k, positions, plan, transpose)
    pdim = positions.dim()
    if positions.dtype not in _POSITIONS or not 1 <= pdim <= 2 or positions.shape[-1] != s or \
            (pdim == 2 and positions.shape[0] != b):
        raise ValueError(f"positions must be int64 or int32 [{s}] or [{b}, {s}], got "
                         f"{positions.dtype} {tuple(positions.shape)}")
    dev = q.get_device()
    if dev < 0 or positions.get_device() != dev or plan.turns.get_device() != dev:
        raise ValueError(f"q, positions and the plan must be on one CUDA device, got {q.device}, "
                         f"{positions.device} and {plan.turns.device}")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return apply_rotary(q, k, positions, plan, out, transpose)
    if not positions.is_contiguous() and positions.stride(-1) != 1:
        positions = positions.contiguous()
    if out is None:
        oq, ok = _like(q), None if k is None else _like(k)
    else:
        oq, ok = _results(q, k, out)
        A.written(oq, ok)
    if b == 0 or s == 0 or h + hk == 0:
        return oq, ok
    q0, q1, q2, _ = q.stride()
    o0, o1, o2, _ = oq.stride()
    if hk:
        k0, k1, k2, _ = k.stride()
        p0, p1, p2, _ = ok.stride()
        strides = _STRIDES(q0, q1, q2, o0, o1, o2, k0, k1, k2, p0, p1, p2)
        kp, kop = k.data_ptr(), ok.data_ptr()
    else:
        strides = _STRIDES(q0, q1, q2, o0, o1, o2, 0, 0, 0, 0, 0, 0)
        kp = kop = None
    status = _lib.lib().gq_rotary(
        q.data_ptr(), oq.data_ptr(), h, kp, kop, hk, strides, positions.data_ptr(),
        positions.stride(0) if pdim == 2 else 0, positions.dtype is torch.int32,
        plan.turns.data_ptr(), b, s, d, plan.rotary_dim, plan.interleaved, plan.factor, transpose,
        dt, A.raw_stream(dev))
    if status:
        _lib.raise_status(status)
    return oq, ok


__all__ = ["LinearScaling", "Llama3Scaling", "NtkScaling", "RotaryPlan", "YarnScaling",
           "apply_rotary", "rotary_frequencies", "rotary_plan"]
