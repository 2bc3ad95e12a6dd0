"""Memory checks of output arguments: ``overlap`` and ``distinct_elements``
against the sets of elements themselves."""

import random

import torch

from jax_gptq_b200 import _arrays as A


def _elements(t):
    at = torch.zeros((), dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return (at.reshape(-1) + t.storage_offset()).tolist()


def _view(rng, buf):
    dims = rng.randint(1, 4)
    shape = [rng.randint(1, 4) for _ in range(dims)]
    stride = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 24, 48]) for _ in range(dims)]
    span = sum((n - 1) * s for n, s in zip(shape, stride))
    return torch.as_strided(buf, shape, stride, rng.randrange(0, buf.numel() - span))


def test_overlap_never_misses_a_shared_element():
    rng = random.Random(0)
    buf = torch.empty(1000)
    told = 0
    for _ in range(20000):
        a, b = _view(rng, buf), _view(rng, buf)
        if set(_elements(a)) & set(_elements(b)):
            assert A.overlap(a, b)
        told += not A.overlap(a, b)
        e = _elements(a)
        if len(set(e)) < len(e):
            assert not A.distinct_elements(a)
    assert told > 5000


def test_heads_of_a_joint_projection_are_apart():
    qkv = torch.empty(2, 7, 12 * 16)
    q = qkv[..., :8 * 16].view(2, 7, 8, 16).transpose(1, 2)
    k = qkv[..., 8 * 16:10 * 16].view(2, 7, 2, 16).transpose(1, 2)
    assert not A.overlap(q, k) and not A.overlap(k, q)
    assert A.overlap(q, qkv) and A.overlap(q, q) and A.overlap(q[:, :, 1:], q[:, :, :-1])
    assert A.distinct_elements(q) and A.distinct_elements(k)
    assert not A.distinct_elements(qkv[:, :1].expand(2, 7, 192))


def test_columns_of_one_matrix_are_apart():
    m = torch.empty(10, 64)
    assert not A.overlap(m[:, :32], m[:, 32:])
    assert A.overlap(m[:, :33], m[:, 32:])
