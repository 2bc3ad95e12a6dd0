"""Array plumbing between the drop-in API and the C ABI.

Inputs may be numpy arrays (host) or torch tensors; they are moved to the
current CUDA device as contiguous tensors.  Results are returned in the
caller's container: numpy in -> numpy out, torch in -> torch (on the device).
"""

from __future__ import annotations

import ctypes

import numpy as np
import torch


def require_cuda() -> None:
    if not torch.cuda.is_available():
        raise RuntimeError("jax_gptq_b200 needs a CUDA device (sm_100a); none is available")


def is_host(x) -> bool:
    return not isinstance(x, torch.Tensor)


def to_device(x, dtype=torch.float32) -> torch.Tensor:
    """Contiguous CUDA tensor of ``dtype`` holding ``x`` (no copy if already so)."""
    require_cuda()
    if isinstance(x, torch.Tensor):
        t = x
    else:
        arr = np.asarray(x)
        if arr.dtype == np.float64 and dtype == torch.float32:
            arr = arr.astype(np.float32)
        t = torch.from_numpy(np.ascontiguousarray(arr))
    if dtype is not None and t.dtype != dtype:
        t = t.to(dtype)
    if not t.is_cuda:
        t = t.to("cuda", non_blocking=False)
    return t.contiguous()


def like_input(t: torch.Tensor, ref):
    """Return ``t`` in the container type of ``ref``."""
    if is_host(ref):
        return t.detach().cpu().numpy()
    return t


def ptr(t) -> ctypes.c_void_p:
    if t is None:
        return ctypes.c_void_p(0)
    return ctypes.c_void_p(t.data_ptr())


# torch's current stream as a number, without building a Stream object (where
# this torch has that call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def raw_stream(index: int) -> int:
    """torch's current stream on device ``index``, as the C ABI takes it."""
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def stream() -> ctypes.c_void_p:
    return ctypes.c_void_p(raw_stream(torch.cuda.current_device()))


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors may share memory.  Views side by side in one buffer
    (heads of a joint projection, columns of one matrix) are told apart by the
    outer dimensions they have in common; what is not decided counts as shared."""
    sa, sb = a.untyped_storage(), b.untyped_storage()
    pa, pb = sa.data_ptr(), sb.data_ptr()
    if pa + sa.nbytes() <= pb or pb + sb.nbytes() <= pa:  # nearly always, and quickly told
        return False
    if a.numel() == 0 or b.numel() == 0 or a.device != b.device:
        return False
    da = sorted((s * a.element_size(), n) for n, s in zip(a.shape, a.stride()) if n > 1)
    db = sorted((s * b.element_size(), n) for n, s in zip(b.shape, b.stride()) if n > 1)
    common = []  # outer dimensions, outermost first
    while True:
        if _apart(a, b, da, db, common):
            return False
        if not (da and db and da[-1] == db[-1]):
            return True
        common.append(da.pop())
        db.pop()


def _apart(a, b, da, db, common) -> bool:
    """Whether the inner blocks ``da`` and ``db`` of two tensors lie apart, in
    windows that the ``common`` outer strides never bring over each other."""
    a0, b0 = a.data_ptr(), b.data_ptr()
    a1 = a0 + sum(s * (n - 1) for s, n in da) + a.element_size()
    b1 = b0 + sum(s * (n - 1) for s, n in db) + b.element_size()
    whole = sum(s * (n - 1) for s, n in common)
    if a1 + whole <= b0 or b1 + whole <= a0:
        return True
    if a0 < b1 and b0 < a1:
        return False
    width = max(a1, b1) - min(a0, b0)
    for s, n in reversed(common):
        if s < width:
            return False
        width += s * (n - 1)
    return True


def written(*tensors) -> None:
    """Tells autograd that a kernel writes the caller's tensors: a graph that kept
    one of them for its backward pass then raises, as after torch's own in-place
    operations."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None])


def distinct_elements(t: torch.Tensor) -> bool:
    """Whether no two elements of ``t`` share memory, judged by its strides:
    each is at least the span of the ones below it."""
    if t.is_contiguous():
        return True
    span = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s < span:
            return False
        span = s * (n - 1) + span
    return True


def empty(shape, dtype=torch.float32) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device="cuda")


def workspace(nbytes: int) -> torch.Tensor:
    """Byte buffer, 256-byte aligned (the caching allocator guarantees 512)."""
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device="cuda")
