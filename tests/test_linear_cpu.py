"""Products with packed weights, what needs no GPU: the order of the positions
and the refusals of the C entry points (nothing is launched)."""

import ctypes

import numpy as np
import pytest
import torch

from jax_gptq_b200 import _lib, linear


@pytest.mark.parametrize("counts,granule,k", [([128, 128], 128, 256), ([64, 64, 64], 64, 256),
                                              ([96, 96], 32, 256), ([8, 8, 8], 32, 128),
                                              ([100, 0, 28], 128, 256), ([1], 128, 128),
                                              ([32] * 5, 32, 256), ([200, 56], 128, 384)])
def test_positions_cover_every_column_once(counts, granule, k):
    rng = np.random.default_rng(sum(counts))
    g_idx = rng.permutation(np.repeat(np.arange(len(counts)), counts)).astype(np.int32)
    gr, kk, kmap, gg = linear._positions(torch.from_numpy(g_idx), len(counts))
    need = {g: sum(-(-c // g) * g for c in counts) for g in (128, 64, 32)}
    assert need[gr] == need[32] and all(need[g] > need[32] for g in (128, 64) if g > gr)
    assert kk == -(-need[gr] // 128) * 128
    kmap, gg = kmap.numpy(), gg.numpy()
    assert sorted(kmap[kmap >= 0]) == list(range(len(g_idx)))
    for i, col in enumerate(kmap):
        if col >= 0:
            assert g_idx[col] == gg[i // gr]
    inside = [kmap[i:i + gr][kmap[i:i + gr] >= 0] for i in range(0, kk, gr)]
    assert all((np.diff(c) > 0).all() for c in inside)  # columns in order inside a granule


def test_identity_needs_no_gather():
    gr, k, kmap, _ = linear._positions(torch.arange(1024, dtype=torch.int32) // 128, 8)
    assert (gr, k) == (128, 1024) and torch.equal(kmap, torch.arange(1024, dtype=torch.int32))


def _call(**kw):
    p = ctypes.c_void_p(256)
    a = dict(qw=p, params=p, kmap=p, m=16, n=128, k=128, bits=4, granule=128, direct=0, x=p,
             dtype=1, tokens=1, ldx=128, y=p, ldy=16, ws=p, nbytes=1 << 20, stream=None)
    a.update(kw)
    return _lib.lib().gq_linear(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), b"dtype"), (dict(bits=0), b"bits"), (dict(bits=9), b"bits"),
    (dict(granule=16), b"granule"), (dict(m=-1), b"shape"), (dict(tokens=-1), b"shape"),
    (dict(tokens=1 << 29), b"shape"), (dict(n=0), b"shape"), (dict(k=192), b"bad k"),
    (dict(n=200, ldx=200), b"bad k"), (dict(ldx=127), b"leading"), (dict(ldy=15), b"leading"),
    (dict(qw=None), b"NULL"), (dict(x=None), b"NULL"), (dict(y=None), b"NULL"),
    (dict(kmap=None), b"NULL"), (dict(qw=ctypes.c_void_p(264)), b"aligned"),
    (dict(ws=None), b"workspace"), (dict(nbytes=8), b"workspace"),
    (dict(ws=ctypes.c_void_p(272)), b"workspace"), (dict(kmap=ctypes.c_void_p(260)), b"kmap")])
def test_product_refuses_before_launching(kw, text):
    before = _lib.lib().gq_launch_count()
    assert _call(**kw) == _lib.GQ_EINVAL
    assert text in _lib.lib().gq_last_error()
    assert _lib.lib().gq_launch_count() == before


def test_product_of_nothing_is_fine():
    assert _call(tokens=0, x=None, y=None) == _lib.GQ_OK
    assert _call(m=0, ldy=0, qw=None) == _lib.GQ_OK


def test_workspace_sizes():
    size = _lib.lib().gq_linear_workspace_size
    assert size(3, 256, 1) >= 3 * 256 * 2 and size(3, 256, 0) >= 3 * 3 * 256 * 2
    assert size(0, 256, 1) > 0 and size(7, 128, 2) % 256 == 0


@pytest.mark.parametrize("kw,text", [
    (dict(bits=0), b"bits"), (dict(bits=1, sym=1), b"bits"), (dict(granule=96), b"granule"),
    (dict(ldp=15), b"shape"), (dict(k=100), b"multiple of 128"), (dict(bad=None), b"bad")])
def test_layout_refuses_before_launching(kw, text):
    p = ctypes.c_void_p(256)
    a = dict(packed=p, m=16, n=128, ldp=16, bits=4, sym=0, scales=p, zeros=p, n_groups=1, kmap=p,
             k=128, gg=p, granule=128, qw=p, params=p, bad=p, stream=None)
    a.update(kw)
    assert _lib.lib().gq_linear_layout(*a.values()) == _lib.GQ_EINVAL
    assert text in _lib.lib().gq_last_error()
