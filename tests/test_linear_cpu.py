"""Products with packed weights, what needs no GPU: the order of the positions
and the refusals of the C entry points (nothing is launched)."""

import ctypes
import random

import numpy as np
import pytest
import torch

import linear_forms as F

from jax_gptq_b200 import _lib, linear, packing


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


def _forms():
    """Every form that some size reaches, by (bits, granule, dtype, columns, parts)."""
    found = {}
    for bits in (4, 8):
        for granule in (32, 64, 128):
            for dtype in (0, 1, 2):
                for m in (16, 4096, 65536):
                    for tokens in (1, 40, 100, 300, 5000):
                        f = F.form(m, 4096, bits, granule, dtype, tokens)
                        if f[0]:
                            found.setdefault((bits, granule, dtype, *f[:2]), f)
    return found


def test_every_form_can_be_chosen():
    got = {(b, dt, n, parts) for b, _, dt, n, parts in _forms()}
    want = {(b, 0, 96, parts) for b in (4, 8) for parts in (1, 2)}
    want |= {(b, dt, n, 1) for b in (4, 8) for dt in (1, 2) for n in (64, 128)}
    want |= {(4, dt, 128, 2) for dt in (1, 2)} | {(8, dt, 96, 2) for dt in (1, 2)}
    assert got == want
    assert F.form(4096, 4096, 4, 128, 1, 32) == (0,) * 10 == F.form(4096, 4096, 4, 128, 0, 8)


def test_the_sizes_of_the_gpu_tests_reach_every_form():
    """A change of the rule that moves them off a form fails here."""
    forms = {(bits, group, dtype, *F.form(m, n, bits, group, dtype, t)[:4])
             for t, m, n in F.SIZES for group in F.GROUPS for bits in F.BITS for dtype in (0, 1, 2)}
    width = lambda bits: 4 if bits <= 4 else 8
    reached = {(width(b), g, dt, n, parts) for b, g, dt, n, parts, *_ in forms if n}
    assert reached == {(width(b), g, dt, n, parts) for b, g, dt, n, parts in _forms()}
    again = {(width(b), g, dt, n, parts) for b, g, dt, n, parts, split, tiles in forms
             if split == 1 and tiles > F.SMS}
    assert again == reached  # a CTA that goes on to another tile
    split = {f[:5] for f in forms if f[4] == 2 and f[5] > 1}
    assert split == {f[:5] for f in forms if f[4] == 2}


def _early_passes(slots, barriers, runs=300, blocks=40):
    """Two groups take the blocks of a ring in turn.  Block n is copied into slot
    n % slots once that is free, its landing completes a phase of barrier
    n % barriers, and a group waits for the phase's parity, so it passes where the
    number of completed phases has another one.  Copies land, and groups look, in
    any order.  How often a group passed before its block had landed."""
    rng, early = random.Random(slots * 100 + barriers), 0
    for _ in range(runs):
        issued, landed, freed, phases = 0, set(), set(), [0] * barriers
        at, slow = [0, 1], rng.randrange(blocks)  # the groups' blocks; one copy that takes long
        while min(at) < blocks:
            what = rng.randrange(4)
            if what == 0 and issued < blocks and (issued < slots or issued - slots in freed):
                issued += 1
            elif what == 1:
                flying = [n for n in range(issued) if n not in landed]
                if flying:
                    n = rng.choice(flying)
                    if n != slow or len(flying) == 1 or rng.random() < 0.02:
                        landed.add(n)
                        phases[n % barriers] += 1
            elif what >= 2 and at[what - 2] < blocks:
                n = at[what - 2]
                if phases[n % barriers] % 2 != n // barriers % 2:
                    if n not in landed:
                        early += 1
                        break
                    freed.add(n)
                    at[what - 2] += 2
    return early


def test_no_group_takes_a_slot_before_its_block_has_landed():
    assert _early_passes(3, 3) > 0  # the model sees it: a group misses every second phase
    for key, f in _forms().items():
        rings = [(f[4], f[5]), (f[6], f[7])] + ([(f[8], f[9])] if f[1] == 2 else [])
        for slots, barriers in rings:
            assert barriers % slots == 0 and _early_passes(slots, barriers, runs=30) == 0, key


@pytest.mark.parametrize("kw", [dict(m=0), dict(k=100), dict(bits=9), dict(granule=48),
                                dict(dtype=3), dict(tokens=0), dict(sms=0)])
def test_form_refuses(kw):
    a = dict(m=16, k=128, bits=4, granule=32, dtype=1, tokens=40, sms=148)
    a.update(kw)
    with pytest.raises(ValueError, match="gq_test_linear_form"):
        F.form(**a)


def test_weights_of_another_device_are_moved(monkeypatch):
    """prepare_linear hands addresses of the current device alone to its launch."""
    class Here(torch.Tensor):
        is_cuda = True

    class There(torch.Tensor):  # of another device: cuda() copies it to the current one
        is_cuda = True

        def cuda(self):
            return self.clone().as_subclass(Here)

    monkeypatch.setattr(linear.A, "require_cuda", lambda: None)
    there = lambda *shape, dtype=torch.float32: torch.ones(shape, dtype=dtype).as_subclass(There)
    p = packing.PackedLinear(there(4, 8, dtype=torch.int32), there(4, 2), there(4, 2),
                             there(64, dtype=torch.int32), there(64, dtype=torch.int32), 4, 32,
                             False, 64)
    moved = linear._on_current(p)
    assert all(type(t) is Here for t in moved)
    assert [tuple(t.shape) for t in moved] == [(4, 8), (64,), (4, 2), (4, 2)]


def test_out_with_a_host_array_is_refused():
    with pytest.raises(ValueError, match="host array"):
        linear.packed_matmul(np.zeros((2, 64), np.float32), None, out=torch.zeros(2, 4))


def test_forms_follow_the_number_of_sms():
    few = (0,) * 10
    for sms in (100, 132, 148):
        assert F.form(sms * 128, 512, 4, 128, 1, 25, sms)[0] == 64
        assert F.form(sms * 128 - 1, 512, 4, 128, 1, 25, sms) == few
        assert F.form(sms * 128, 512, 4, 128, 1, 24, sms) == few
    split = lambda m, sms: F.form(m, 8192, 4, 128, 1, 128, sms)[1:4]
    assert split(14 * 128, 148) == (1, 8, 14) and split(15 * 128, 148) == (1, 4, 15)
    assert split(12 * 128, 132) == (1, 8, 12) and split(13 * 128, 132) == (1, 4, 13)
