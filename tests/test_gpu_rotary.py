"""Rotary positions (gq_rotary) against the formula in float64.

Tolerance.  The angle is a 64-bit product: the frequency is rounded to 2^-65
of a turn, so at |position| < 2^31 the angle is off by less than 2^-33 of a
turn.  As a float32 in half turns it is rounded by 2^-25 relative to at most
1 (pi * 2^-25 in the angle); sincospif is within 2 ulp (2^-23 of at most 1),
the factor and the two products and the sum round once each (3 * 2^-24, with
factor up to 2 in these tests: f).  Together an output is off by less than
f * (|a| + |b|) * (2 pi * 2^-33 + pi * 2^-25 + 2^-23 + 4 * 2^-24), below
f * (|a| + |b|) * 2^-21, plus eps / 2 of its value for the last rounding.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from jax_gptq_b200 import rotary

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _reference(x, positions, plan, inv, transpose=False):
    """(result, tolerance without the last rounding) in float64."""
    r = plan.rotary_dim
    pos = positions if positions.dim() == 2 else positions[None].expand(x.shape[0], -1)
    ang = pos.double()[:, None, :, None] * torch.tensor(inv, dtype=torch.float64, device="cuda")
    c, s = ang.cos() * plan.factor, ang.sin() * plan.factor * (-1 if transpose else 1)
    xd = x.double()
    out, tol = xd.clone(), torch.zeros_like(xd)
    if plan.interleaved:
        i, j = slice(0, r, 2), slice(1, r, 2)
    else:
        i, j = slice(0, r // 2), slice(r // 2, r)
    a, b = xd[..., i], xd[..., j]
    out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    tol[..., i] = tol[..., j] = abs(plan.factor) * (a.abs() + b.abs()) * 2.0 ** -21
    return out, tol


def _check(y, x, positions, plan, inv, transpose=False):
    assert y.shape == x.shape and y.dtype == x.dtype
    ref, tol = _reference(x, positions, plan, inv, transpose)
    fi = torch.finfo(x.dtype)
    tol = tol * (1 + fi.eps) + fi.eps / 2 * ref.abs() + fi.smallest_normal * fi.eps
    r = plan.rotary_dim
    assert torch.equal(y[..., r:], x[..., r:])
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def _heads(b, h, s, d, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((b, s, h, d), generator=gen, device="cuda").to(dtype).transpose(1, 2)


SHAPES = [  # batch, heads, kv_heads, seq, head_dim, rotary_dim
    (1, 1, 1, 1, 2, 2), (1, 32, 32, 1, 128, 128), (2, 8, 2, 17, 64, 64), (3, 20, 5, 33, 96, 48),
    (1, 4, 1, 130, 80, 80), (2, 3, 3, 65, 10, 6), (1, 5, 1, 7, 81, 18), (4, 1, 1, 3, 256, 130),
    (1, 64, 8, 129, 128, 128), (5, 2, 0, 9, 32, 16), (1, 2, 1, 2049, 64, 32),
    (70, 1, 1, 1, 1024, 1024),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_float64(shape, interleaved, dtype):
    b, h, hk, s, d, r = shape
    plan = rotary.rotary_plan(d, rotary_dim=r, interleaved=interleaved)
    inv, _ = rotary.rotary_frequencies(r)
    q = _heads(b, h, s, d, dtype, 1)
    k = _heads(b, hk, s, d, dtype, 2) if hk else None
    pos = torch.randint(0, 5000, (b, s), device="cuda")
    oq, ok = rotary.apply_rotary(q, k, pos, plan)
    _check(oq, q, pos, plan, inv)
    assert oq.stride() == q.stride() or q.numel() == d
    if hk:
        _check(ok, k, pos, plan, inv)
    else:
        assert ok is None
    # turned back: the transposed map of the same positions
    bq, _ = rotary.apply_rotary(oq, None, pos, plan, transpose=True)
    _check(bq, oq, pos, plan, inv, transpose=True)


@pytest.mark.parametrize("scaling", [rotary.LinearScaling(8.0), rotary.NtkScaling(4.0),
                                     rotary.YarnScaling(16.0, 4096),
                                     rotary.Llama3Scaling(8.0, 8192)])
@pytest.mark.parametrize("start", [0, -1000, 1 << 20, (1 << 31) - 64])
def test_far_positions_and_scalings(start, scaling):
    plan = rotary.rotary_plan(64, theta=500000.0, scaling=scaling)
    inv, f = rotary.rotary_frequencies(64, 500000.0, scaling)
    assert plan.factor == f
    q = _heads(2, 4, 40, 64, torch.float32, 3)
    for dt in (torch.int64, torch.int32):
        pos = (start + torch.arange(40, device="cuda")).to(dt)
        _check(rotary.apply_rotary(q, None, pos, plan)[0], q, pos, plan, inv)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts_alignment_and_in_place(interleaved, dtype):
    plan = rotary.rotary_plan(64, rotary_dim=32, interleaved=interleaved)
    inv, _ = rotary.rotary_frequencies(32)
    pos = torch.randint(0, 3000, (3, 20), device="cuda")
    qkv = torch.randn((3, 20, 12 * 64 + 5), device="cuda").to(dtype)
    for off in (0, 1, 5):  # views of one joint projection, 16-byte aligned and not
        q = qkv[..., off:off + 8 * 64].view(3, 20, 8, 64).transpose(1, 2)
        k = qkv[..., off + 8 * 64:off + 10 * 64].view(3, 20, 2, 64).transpose(1, 2)
        q0, k0, rest = q.clone(), k.clone(), qkv[..., off + 10 * 64:].clone()
        oq, ok = rotary.apply_rotary(q, k, pos, plan)
        _check(oq, q, pos, plan, inv)
        _check(ok, k, pos, plan, inv)
        rotary.apply_rotary(q, k, pos, plan, out=(q, k))
        assert torch.equal(q, oq) and torch.equal(k, ok)
        assert torch.equal(qkv[..., off + 10 * 64:], rest)
        q.copy_(q0)
        k.copy_(k0)
    for x in (torch.randn((3, 8, 20, 64), device="cuda").to(dtype),       # heads first
              torch.randn((3, 8, 64, 20), device="cuda").to(dtype).transpose(2, 3),
              torch.randn((3, 1, 20, 64), device="cuda").to(dtype).expand(3, 8, 20, 64)):
        _check(rotary.apply_rotary(x, None, pos, plan)[0], x, pos, plan, inv)
    x = _heads(3, 8, 20, 64, dtype, 5)
    wide = torch.zeros((3, 8, 40, 64), dtype=dtype, device="cuda")  # into every other position
    rotary.apply_rotary(x, None, pos, plan, out=(wide[:, :, ::2], None))
    _check(wide[:, :, ::2], x, pos, plan, inv)
    assert not wide[:, :, 1::2].any()
    _check(rotary.apply_rotary(x, None, pos[:, ::1].t().contiguous().t(), plan)[0], x, pos, plan, inv)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_overlapping_inputs(interleaved, dtype):
    """Views whose elements share memory: the result has memory of its own, with
    contiguous components, whatever the order of the view's strides."""
    plan = rotary.rotary_plan(8, rotary_dim=6, interleaved=interleaved)
    inv, _ = rotary.rotary_frequencies(6)
    x = torch.randn((2, 3, 12), device="cuda").to(dtype)
    pos = torch.randint(0, 3000, (2, 5), device="cuda")
    for v in (x.unfold(2, 8, 1), x.unfold(2, 8, 1)[:, :2, :2],
              x.as_strided((2, 3, 5, 8), (1, 1, 1, 1)), x.as_strided((2, 3, 5, 8), (0, 0, 0, 1))):
        p = pos[:, :v.shape[2]]
        oq, ok = rotary.apply_rotary(v, v, p, plan)
        assert oq.stride(3) == 1 and ok.stride(3) == 1
        _check(oq, v, p, plan, inv)
        assert torch.equal(oq, ok)
        g = v.clone().requires_grad_()
        gx, = torch.autograd.grad(rotary.apply_rotary(g, None, p, plan)[0], g, v)
        _check(gx, v, p, plan, inv, transpose=True)


@pytest.mark.parametrize("start", [0, -3000, 1 << 20, (1 << 40) + 7])
def test_angles_keep_their_digits(start):
    """Cosine and sine themselves, of pairs (1, 0) in float32, against whole-number
    turns.  The rest to the nearest quarter turn is rounded to float32 (2^-24 of it,
    and as much of its sine at most), sincospif is within 2 ulp (2^-22), the factor 1
    and the products with 1 and 0 add nothing: 5/4 of 2^-22 of the value, next to 0
    as well."""
    plan = rotary.rotary_plan(64, theta=500.0)
    pos = start + torch.arange(2000, device="cuda")
    x = torch.zeros((1, 1, 2000, 64), device="cuda")
    x[..., :32] = 1
    y = rotary.apply_rotary(x, None, pos, plan)[0][0, 0].double().cpu()
    near = 1.0
    for i, w in enumerate(plan.turns.tolist()):
        turn = [(p * w) % (1 << 64) for p in pos.tolist()]
        quarters = [((t + (1 << 61)) >> 62) & 3 for t in turn]
        rest = torch.tensor([(t - (q << 62) + (1 << 63)) % (1 << 64) - (1 << 63)
                             for t, q in zip(turn, quarters)], dtype=torch.float64)
        ang = rest * (math.pi * 2.0 ** -63)
        c, s, q = ang.cos(), ang.sin(), torch.tensor(quarters)
        cos = torch.where(q == 0, c, torch.where(q == 1, -s, torch.where(q == 2, -c, s)))
        sin = torch.where(q == 0, s, torch.where(q == 1, c, torch.where(q == 2, -s, -c)))
        for got, want in ((y[:, i], cos), (y[:, 32 + i], sin)):
            assert bool(((got - want).abs() <= 1.25 * 2.0 ** -22 * want.abs() + 2.0 ** -149).all())
            near = min(near, float(want[want != 0].abs().min()))
    assert near < 1e-3  # some of them do lie next to 0


def test_gradient_is_the_transposed_map():
    plan = rotary.rotary_plan(16, rotary_dim=12, scaling=rotary.YarnScaling(4.0, 64))
    inv, _ = rotary.rotary_frequencies(12, scaling=rotary.YarnScaling(4.0, 64))
    pos = torch.arange(5, device="cuda") + 9
    x = torch.randn((1, 2, 5, 16), device="cuda", dtype=torch.float64, requires_grad=True)
    gy = torch.randn((1, 2, 5, 16), device="cuda")
    ref, _ = _reference(x, pos, plan, inv)
    gx, = torch.autograd.grad((ref * gy.double()).sum(), x)
    got = rotary.apply_rotary(gy, None, pos, plan, transpose=True)[0]
    _check(got, gy, pos, plan, inv, transpose=True)
    # the transposed map is the gradient: equal up to _check's tolerance
    assert float((got.double() - gx).abs().max()) <= float(gy.abs().max()) * 2 * plan.factor * 2.0 ** -20


def test_empty_streams_and_graphs():
    plan = rotary.rotary_plan(64)
    q = _heads(2, 4, 9, 64, torch.bfloat16, 1)
    pos = torch.arange(9, device="cuda")
    e = rotary.apply_rotary(q[:0], q[:0], pos, plan)
    assert e[0].shape == (0, 4, 9, 64)
    assert rotary.apply_rotary(q[:, :, :0], None, pos[:0], plan)[0].shape == (2, 4, 0, 64)
    assert rotary.apply_rotary(q, q[:, :0], pos, plan)[1].shape == (2, 0, 9, 64)
    ref = rotary.apply_rotary(q, q, pos, plan)[1]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rotary.apply_rotary(q, None, pos, plan)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rotary.apply_rotary(q, None, pos, plan)[0]
    pos += 100
    want = rotary.apply_rotary(q, None, pos, plan)[0]
    g.replay()
    assert torch.equal(out, want) and not torch.equal(out, ref)


def test_refusals():
    plan = rotary.rotary_plan(64)
    q = _heads(2, 4, 9, 64, torch.float32, 1)
    pos = torch.arange(9, device="cuda")
    for args, text in (((q.double(), None, pos, plan), "float32, bfloat16"),
                       ((q[..., :32], None, pos, plan), "must be \\[batch"),
                       ((q[0], None, pos, plan), "must be \\[batch"),
                       ((q, q.half(), pos, plan), "one type"),
                       ((q, q[:1], pos, plan), "one batch"),
                       ((q, None, pos.float(), plan), "positions"),
                       ((q, None, pos[:8], plan), "positions"),
                       ((q.cpu(), None, pos.cpu(), plan), "one CUDA device"),
                       ((q, None, pos.cpu(), plan), "one CUDA device")):
        with pytest.raises(ValueError, match=text):
            rotary.apply_rotary(*args)
    wide = torch.zeros((2, 4, 10, 64), device="cuda")
    for out, text in (((q, q.clone()), "pair"), ((None, None), "pair"),
                      ((q.half(), None), "like it"), ((wide, None), "like it"),
                      ((torch.zeros((2, 1, 9, 64), device="cuda").expand(2, 4, 9, 64), None),
                       "share memory")):
        with pytest.raises(ValueError, match=text):
            rotary.apply_rotary(q, None, pos, plan, out=out)
    with pytest.raises(ValueError, match="partly"):
        rotary.apply_rotary(wide[:, :, :9], None, pos, plan, out=(wide[:, :, 1:], None))
    with pytest.raises(ValueError, match="share memory"):
        rotary.apply_rotary(q, q.clone(), pos, plan, out=(wide[:, :, :9], wide[:, :, 1:]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kv_heads", [0, 2])
def test_gradients(kv_heads, interleaved, dtype):
    """Against the formula's, and against differences: the map is linear, so
    f(q + v) - f(q) = f(v), and <w, f(v)> = <gradient, v> up to the tolerances
    of f(v) and of the gradient."""
    plan = rotary.rotary_plan(24, rotary_dim=12, interleaved=interleaved)
    inv, _ = rotary.rotary_frequencies(12)
    pos = torch.randint(0, 4000, (2, 19), device="cuda", dtype=torch.int32)
    q = _heads(2, 6, 19, 24, dtype, 5).requires_grad_()
    k = _heads(2, kv_heads, 19, 24, dtype, 6).requires_grad_() if kv_heads else None
    oq, ok = rotary.apply_rotary(q, k, pos, plan)
    leaves, outs = ([q, k], [oq, ok]) if kv_heads else ([q], [oq])
    ws = [torch.randn_like(o) for o in outs]
    grads = torch.autograd.grad(outs, leaves, ws)
    fi = torch.finfo(dtype)
    for x, w, g in zip(leaves, ws, grads):
        _check(g, w, pos, plan, inv, transpose=True)
        v = torch.randn_like(x)
        with torch.no_grad():
            fv = rotary.apply_rotary(v, None, pos, plan)[0]
        room = 0.0
        for a, b, back in ((v, w, False), (w, v, True)):
            ref, tol = _reference(a, pos, plan, inv, back)
            tol = tol * (1 + fi.eps) + fi.eps / 2 * ref.abs() + fi.smallest_normal * fi.eps
            room += float((b.double().abs() * tol).sum())
        assert abs(float((w.double() * fv.double()).sum() - (g.double() * v.double()).sum())) <= room
    # one output alone, an expanded gradient
    gq, = torch.autograd.grad(rotary.apply_rotary(q, k, pos, plan)[0].sum(), q)
    _check(gq, torch.ones_like(q), pos, plan, inv, transpose=True)
    with pytest.raises(ValueError, match="out takes no gradients"):
        rotary.apply_rotary(q, None, pos, plan, out=(torch.empty_like(q), None))


def test_autograd_sees_what_is_turned_in_place():
    """Tensors that a graph keeps for its backward pass, turned in between."""
    plan = rotary.rotary_plan(64)
    pos = torch.arange(9, device="cuda")
    for pair in ((True, False), (True, True)):
        leaf = _heads(2, 4, 9, 64, torch.float32, 1).requires_grad_()
        q, k = leaf.exp(), leaf.exp() if pair[1] else None  # kept: their gradient is themselves
        with torch.no_grad():
            rotary.apply_rotary(q, k, pos, plan, out=(q, k))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            (k if pair[1] else q).sum().backward()
    with torch.inference_mode():  # (tensors without a version)
        q = _heads(2, 4, 9, 64, torch.float32, 1)
        assert rotary.apply_rotary(q, None, pos, plan, out=(q, None))[0] is q


def test_out_that_asks_for_gradients_is_refused():
    plan = rotary.rotary_plan(64)
    pos = torch.arange(9, device="cuda")
    q = _heads(2, 4, 9, 64, torch.float32, 1)
    leaf = torch.zeros_like(q, requires_grad=True)
    plain = torch.zeros_like(q)
    for k, out in ((None, (leaf, None)), (q, (plain, leaf)), (q, (plain, leaf * 2))):
        with pytest.raises(ValueError, match="out takes no gradients"):
            rotary.apply_rotary(q, k, pos, plan, out=out)
        with torch.no_grad():
            got = rotary.apply_rotary(q, k, pos, plan, out=out)
        assert torch.equal(got[0], rotary.apply_rotary(q, None, pos, plan)[0])
