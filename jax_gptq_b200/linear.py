"""Linears that run on packed weights.

The reference stops at dequantized floats (``quant.py:37``), and
``packing.dequantize`` turns a packed layer back into them.  This module
multiplies with the packed form: ``prepare_linear`` lays a
:class:`packing.PackedLinear` out once for the tensor cores
(``gq_linear_layout``), ``packed_matmul`` computes ``x @ W.T`` from it
(``gq_linear``) for one token or thousands, and :class:`QuantLinear` is the
module form.  Weights are not rounded on the way: whole-number codes are
multiplied with x on the tensor cores, and each group's float32 sum is scaled
once.  Codes of 1 to 4 bits take 4 bits of memory each there, of 5 to 8 bits 8.
For thousands of tokens this saves memory rather than time: float weights
multiplied by the library are faster once they are decoded.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _arrays as A
from . import _lib
from .packing import PackedLinear

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@dataclass(frozen=True, eq=False)
class PreparedLinear:
    """Packed weights laid out for ``packed_matmul`` (see ``gq_linear_layout``)."""
    qweight: torch.Tensor   # laid-out codes, int32 words
    params: torch.Tensor    # [row blocks, granules, 16, 2] float32: scale, offset
    kmap: torch.Tensor      # [k] int32: original column of each position, -1 for padding
    m: int                  # out_features
    n: int                  # in_features
    k: int                  # positions
    bits: int
    granule: int            # columns that share one scale in the layout
    direct: bool            # positions are the columns in their own order

    def __post_init__(self):
        # the leading arguments of gq_linear, ready for every call
        object.__setattr__(self, "_head", (
            self.qweight.data_ptr(), self.params.data_ptr(), self.kmap.data_ptr(), self.m, self.n,
            self.k, self.bits, self.granule, self.direct))
        object.__setattr__(self, "_index", self.qweight.get_device())

    def __reduce__(self):  # a copy has tensors, and so addresses, of its own
        return PreparedLinear, (self.qweight, self.params, self.kmap, self.m, self.n, self.k,
                                self.bits, self.granule, self.direct)

    @property
    def device(self) -> torch.device:
        return self.qweight.device

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.qweight, self.params, self.kmap))


def _positions(g_idx: torch.Tensor, n_groups: int):
    """(granule, k, kmap, granule_group) of the column groups ``g_idx``: columns
    in group order, every group padded to whole granules, k a multiple of 128."""
    n = g_idx.numel()
    g = g_idx.long()
    counts = torch.bincount(g, minlength=n_groups)
    need = {}
    for gr in (128, 64, 32):
        need[gr] = int(((counts + gr - 1) // gr).sum()) * gr
    # the widest granule that pads no more than the narrowest: fewer scales to
    # read and fewer sums to scale
    granule = next(gr for gr in (128, 64, 32) if need[gr] <= need[32])
    k = -(-max(need[granule], 1) // 128) * 128
    grans = (counts + granule - 1) // granule
    order = torch.argsort(g, stable=True)
    first = torch.cumsum(counts, 0) - counts          # of the group, among sorted columns
    base = (torch.cumsum(grans, 0) - grans) * granule  # of the group, among positions
    pos = base[g[order]] + torch.arange(n, device=g.device) - first[g[order]]
    kmap = torch.full((k,), -1, dtype=torch.int32, device=g.device)
    kmap[pos] = order.to(torch.int32)
    gg = torch.full((k // granule,), -1, dtype=torch.int32, device=g.device)
    filled = torch.repeat_interleave(torch.arange(n_groups, device=g.device), grans)
    gg[:filled.numel()] = filled.to(torch.int32)
    return granule, k, kmap, gg


def _on_current(p: PackedLinear):
    """(qweight, g_idx, scales, zeros) on the current device, wherever they are."""
    s, z = (A.to_device(t.cuda()) for t in (p.scales, p.zeros))
    return p.qweight.cuda().contiguous(), p.g_idx.cuda(), s, z


def prepare_linear(p: PackedLinear) -> PreparedLinear:
    """Lay ``p`` out for ``packed_matmul`` on the current device (once per weight).

    Raises ``ValueError`` for shapes that do not fit together, groups outside
    the scales, zeros that are not whole numbers of the code range (the
    quantizers here only write those) and scales that are not finite."""
    A.require_cuda()
    bits, n = int(p.bits), int(p.n)
    words = _lib.lib().gq_packed_words(n, bits)
    if words < 0 or (p.sym and bits < 2):
        raise ValueError(f"bits must be 1..8 (2..8 symmetric), got {bits}")
    if n < 1:
        raise ValueError(f"in_features must be positive, got {n}")
    if p.qweight.dim() != 2 or p.qweight.dtype != torch.int32 or p.qweight.shape[1] < words:
        raise ValueError(f"qweight must be int32 [m, {words}], got {p.qweight.dtype} "
                         f"{tuple(p.qweight.shape)}")
    m = p.qweight.shape[0]
    if p.scales.dim() != 2 or p.scales.shape != p.zeros.shape or p.scales.shape[0] != m:
        raise ValueError(f"scales and zeros must be [m, groups] with m = {m}, got "
                         f"{tuple(p.scales.shape)} and {tuple(p.zeros.shape)}")
    if tuple(p.g_idx.shape) != (n,):
        raise ValueError(f"g_idx must be [{n}], got {tuple(p.g_idx.shape)}")
    q, g_idx, s, z = _on_current(p)
    lo, hi = (int(v) for v in torch.aminmax(g_idx))
    if lo < 0 or hi >= s.shape[1]:
        raise ValueError(f"g_idx must lie in [0, {s.shape[1]}), got {lo} .. {hi}")
    granule, k, kmap, gg = _positions(g_idx, s.shape[1])
    blocks = -(-m // 16)
    qw = torch.empty((blocks * 16 * k * (4 if bits <= 4 else 8) // 32,), dtype=torch.int32,
                     device="cuda")
    params = torch.empty((blocks, k // granule, 16, 2), dtype=torch.float32, device="cuda")
    bad = torch.empty((1,), dtype=torch.int32, device="cuda")
    _lib.call("gq_linear_layout", A.ptr(q), m, n, q.shape[1], bits, int(p.sym), A.ptr(s), A.ptr(z),
              s.shape[1], A.ptr(kmap), k, A.ptr(gg), granule, A.ptr(qw), A.ptr(params), A.ptr(bad),
              A.stream())
    fault = int(bad.item())
    if fault & 1:
        raise ValueError(f"zeros must be whole numbers inside the {bits}-bit code range")
    if fault & 2:
        raise ValueError("scales must be finite")
    direct = k == n and bool((kmap == torch.arange(k, device="cuda", dtype=torch.int32)).all())
    return PreparedLinear(qw, params, kmap, m, n, k, bits, granule, direct)


def packed_matmul(x, w: PreparedLinear, out: torch.Tensor | None = None):
    """``x @ W.T`` for ``x`` [..., n] (float32, bf16 or fp16) -> [..., m] of x's type.

    Products are summed in float32 (float32 x runs as three exact bf16 terms:
    it loses no bits above 2^-126) and rounded once; a granule is summed before
    its scale, so |x| has to stay below 2^112.  numpy in -> numpy out.
    ``out``, if given, is a contiguous tensor of the result's shape and type
    that does not share memory with ``x`` (under ``torch.no_grad()`` where it asks
    for gradients).  There is no gradient: an ``x`` that asks for one is refused.

    Waits inside the kernel are bounded.  One that expired leaves the result
    incomplete and a status word behind, which this call does not read (it
    would have to wait for the device): ``_lib.check_device()`` raises on it,
    and ``TinyLM.generate`` and ``evaluate_perplexity`` call that at their end."""
    dt = _DTYPES.get(getattr(x, "dtype", None))
    if dt is None:
        if A.is_host(x):
            if out is not None:
                raise ValueError("out goes with a tensor x, not with a host array")
            return A.like_input(packed_matmul(A.to_device(x), w), x)
        raise ValueError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("packed_matmul has no gradient: call it under torch.no_grad()")
    n, m, dev = w.n, w.m, x.get_device()
    if x.dim() < 1 or x.shape[-1] != n:
        raise ValueError(f"x must be [..., {n}], got {tuple(x.shape)}")
    if dev < 0 or dev != w._index:
        raise ValueError(f"x is on {x.device}, the weights on {w.qweight.device}")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return packed_matmul(x, w, out)
    x2 = x
    if x.dim() != 2 or x.stride(1) != 1 or x.stride(0) < n:
        x2 = x.reshape(-1, n).contiguous()
    tokens, ldx = x2.shape[0], x2.stride(0)
    given = out is not None
    if not given:
        out = x.new_empty(tokens, m) if x2 is x else x.new_empty(*x.shape[:-1], m)
    elif tuple(out.shape) != (*x.shape[:-1], m) or out.dtype != x.dtype or \
            out.device != x.device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {x.dtype} tensor {(*x.shape[:-1], m)} on "
                         f"{x.device}")
    elif A.overlap(out, x2):
        raise ValueError("out shares memory with x")
    elif out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out takes no gradients: call it under torch.no_grad()")
    if tokens == 0 or m == 0:
        return out
    if given:
        A.written(out)
    lib = _lib.lib()
    xp, wp, nbytes = x2.data_ptr(), None, 0
    if not (w.direct and dt and xp % 16 == 0 and ldx % 8 == 0):  # x is first put in order
        nbytes = lib.gq_linear_workspace_size(tokens, w.k, dt)
        ws = x2.new_empty(nbytes // x2.element_size())  # (a multiple of 256)
        wp = ws.data_ptr()
    status = lib.gq_linear(*w._head, xp, dt, tokens, ldx, out.data_ptr(), m, wp, nbytes,
                           A.raw_stream(dev))
    if status:
        _lib.raise_status(status)
    return out


class QuantLinear(torch.nn.Module):
    """A bias-free linear on packed weights (inference only).  They stay on the
    device they were laid out on and are not part of ``state_dict``: a packed
    checkpoint keeps them."""

    def __init__(self, p: PackedLinear | PreparedLinear):
        super().__init__()
        self.weights = p if isinstance(p, PreparedLinear) else prepare_linear(p)

    @property
    def in_features(self) -> int:
        return self.weights.n

    @property
    def out_features(self) -> int:
        return self.weights.m

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return packed_matmul(x, self.weights)

    def extra_repr(self) -> str:
        w = self.weights
        return f"in_features={w.n}, out_features={w.m}, bits={w.bits}"


__all__ = ["PreparedLinear", "QuantLinear", "packed_matmul", "prepare_linear"]
