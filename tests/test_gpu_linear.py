"""Products with packed weights (gq_linear_layout, gq_linear) against the same
product in float64.

Tolerance.  x and code - offset enter the tensor cores exactly (float32 x as
three bf16 terms whose sum is x), so an error can only come from additions in
float32 and from the last rounding.  A granule's sum is at most 128 products
in steps of 16: 8 steps, each at most 17 additions of relative error 2^-23
(the tensor core may truncate) of the terms' absolute sum; then one fused
multiply-add per granule of a warp's or tile's share and at most 32 additions
across shares and terms.  With A = sum |x w| the error of an element is below
(8 * 17 + granules + 32) * 2^-23 * A, plus eps / 2 of the value for the last
rounding.  float32 terms below 2^-126 (the lowest bits of numbers under
2^-110) are not among the inputs.
"""

import copy
import functools
import pickle

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import linear_forms as F

from jax_gptq_b200 import _arrays as A
from jax_gptq_b200 import _lib, linear, packing
from jax_gptq_b200.config import QuantConfig
from jax_gptq_b200.gptq_ref import gptq_quantize
from oracle import inputs
from oracle import pack as P

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _packed(m, n, group, bits, sym, seed, act_order, uneven=False):
    """A PackedLinear of random codes, its weights in float64."""
    rng = np.random.default_rng(seed)
    levels = (1 << bits) - 1 if sym else 1 << bits
    codes = rng.integers(0, levels, (m, n)).astype(np.uint8)
    groups = max(1, n // group)
    scales = rng.uniform(0.5e-2, 2e-2, (m, groups)).astype(np.float32)
    zeros = np.zeros((m, groups), np.float32) if sym else \
        rng.integers(0, 1 << bits, (m, groups)).astype(np.float32)
    g_idx = (np.arange(n) // group).clip(0, groups - 1).astype(np.int32)
    if uneven:
        g_idx = rng.integers(0, groups, n).astype(np.int32)
    perm = rng.permutation(n).astype(np.int32) if act_order else np.arange(n, dtype=np.int32)
    back = np.empty(n, np.int32)
    back[perm] = g_idx
    q = torch.from_numpy(P.pack(codes, bits).view(np.int32)).cuda()
    p = packing.PackedLinear(q, torch.from_numpy(scales).cuda(), torch.from_numpy(zeros).cuda(),
                             torch.from_numpy(back).cuda(), torch.from_numpy(perm).cuda(), bits,
                             group, sym, n)
    qmin = 1 - (1 << (bits - 1)) if sym else 0
    w = (codes.astype(np.float64) + qmin - zeros[:, back]) * scales[:, back].astype(np.float64)
    return p, torch.from_numpy(w).cuda()


def _x(shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    scale = torch.exp(torch.randn(shape[-1:], generator=gen, device="cuda"))
    return (torch.randn(shape, generator=gen, device="cuda") * scale + 0.25).to(dtype)


def _check(y, x, w, p):
    assert y.dtype == x.dtype and tuple(y.shape) == (*x.shape[:-1], w.shape[0])
    ref = x.double() @ w.T
    amount = x.double().abs() @ w.abs().T
    granules = p.k // p.granule
    tol = (8 * 17 + granules + 32) * 2.0 ** -23 * amount \
        + torch.finfo(x.dtype).eps / 2 * ref.abs() * (1 + 1e-3) \
        + torch.finfo(x.dtype).smallest_normal
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


SHAPES = [  # tokens, m, n, group
    (1, 1, 32, 32), (1, 16, 128, 128), (2, 17, 96, 32), (3, 48, 1000, 125), (5, 33, 384, 96),
    (8, 130, 512, 64), (9, 64, 2048, 2048), (16, 20, 11008, 128), (17, 100, 1152, 48),
    (31, 65, 640, 128), (33, 31, 256, 8), (64, 257, 1024, 128), (65, 128, 896, 64),
    (130, 300, 1536, 128), (257, 513, 2048, 128), (300, 129, 288, 96),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_float64(shape, dtype):
    t, m, n, group = shape
    p, w = _packed(m, n, group, 4, False, sum(shape), act_order=(m % 2 == 1))
    pl = linear.prepare_linear(p)
    x = _x((t, n), dtype, m)
    y = linear.packed_matmul(x, pl)
    _check(y, x, w, pl)
    assert torch.equal(y, linear.packed_matmul(x, pl))  # fixed order of additions


@pytest.mark.parametrize("sym", [False, True])
@pytest.mark.parametrize("bits", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_width(bits, sym, dtype):
    if sym and bits < 2:
        pytest.skip("no symmetric 1-bit codes")
    p, w = _packed(70, 512, 64, bits, sym, bits, act_order=True)
    pl = linear.prepare_linear(p)
    for t in (1, 7, 150):
        x = _x((t, 512), dtype, t)
        _check(linear.packed_matmul(x, pl), x, w, pl)


@pytest.mark.parametrize("t", [1, 5, 8, 27])
@pytest.mark.parametrize("n", [2048, 4000, 16384])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_and_long_sums(dtype, n, t):
    """Clusters of 2 to 8 CTAs share a sum, with x in place and gathered."""
    for act_order in (False, True):
        p, w = _packed(37, n, 128, 4, False, n + t, act_order=act_order)
        pl = linear.prepare_linear(p)
        x = _x((t, n), dtype, t)
        y = linear.packed_matmul(x, pl)
        _check(y, x, w, pl)
        assert torch.equal(y, linear.packed_matmul(x, pl))


@pytest.mark.parametrize("t", [8, 24, 25, 32])
def test_many_rows(t):
    p, w = _packed(18950, 256, 128, 4, False, t, act_order=False)
    pl = linear.prepare_linear(p)
    x = _x((t, 256), torch.bfloat16, t)
    _check(linear.packed_matmul(x, pl), x, w, pl)


@functools.lru_cache(maxsize=1)
def _weights(m, n, group, bits):
    """Random prepared weights with columns in order, and their float64 values."""
    gen = torch.Generator(device="cuda").manual_seed(m + n + bits + group)
    rand = lambda hi, *shape: torch.randint(0, hi, shape, generator=gen, device="cuda")
    codes = rand(1 << bits, m, n).to(torch.uint8)
    scales = (5 + 15 * torch.rand((m, n // group), generator=gen, device="cuda")) * 1e-3
    zeros = rand(1 << bits, m, n // group).float()
    words = _lib.lib().gq_packed_words(n, bits)
    q = torch.empty((m, words), dtype=torch.int32, device="cuda")
    _lib.call("gq_pack_codes", A.ptr(codes), m, n, n, bits, A.ptr(q), words, A.stream())
    order = torch.arange(n, dtype=torch.int32, device="cuda")
    pl = linear.prepare_linear(packing.PackedLinear(q, scales, zeros, order // group, order, bits,
                                                    group, False, n))
    w = (codes.double().view(m, -1, group) - zeros.double()[..., None]) * scales.double()[..., None]
    return pl, w.view(m, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", F.SIZES)
@pytest.mark.parametrize("group", F.GROUPS)
@pytest.mark.parametrize("bits", F.BITS)
def test_every_form_of_many_tokens(bits, group, size, dtype):
    t, m, n = size
    pl, w = _weights(m, n, group, bits)
    assert pl.granule == group
    x = _x((t, n), dtype, t)
    y = linear.packed_matmul(x, pl)
    _check(y, x, w, pl)
    assert torch.equal(y, linear.packed_matmul(x, pl))


@pytest.mark.parametrize("t", [1, 12, 140])
def test_groups_of_uneven_sizes(t):
    p, w = _packed(40, 700, 50, 4, False, 3, act_order=False, uneven=True)
    pl = linear.prepare_linear(p)
    x = _x((t, 700), torch.bfloat16, 4)
    _check(linear.packed_matmul(x, pl), x, w, pl)


@pytest.mark.parametrize("t", [1, 4, 40, 200])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_alignment_and_extra_dimensions(t, dtype):
    p, w = _packed(50, 256, 128, 4, False, 5, act_order=False)
    pl = linear.prepare_linear(p)
    assert pl.direct
    wide = _x((t, 256 + 40), dtype, 6)
    for x in (wide[:, 8:264], wide[:, 3:259], wide[:, :256], _x((256, t), dtype, 7).t(),
              _x((1, 256), dtype, 8).expand(t, 256), _x((2, t, 256), dtype, 9),
              _x((t, 2, 256), dtype, 10).transpose(0, 1), _x((256,), dtype, 11)):
        _check(linear.packed_matmul(x, pl), x, w, pl)
    out = torch.full((t + 2, 50), 7.0, dtype=dtype, device="cuda")
    x = wide[:, :256]
    got = linear.packed_matmul(x, pl, out=out[1:t + 1])
    assert got.data_ptr() == out[1:].data_ptr()
    _check(got, x, w, pl)
    assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all())  # rows around it untouched


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_and_numpy(dtype):
    p, w = _packed(24, 128, 128, 4, False, 1, act_order=True)
    pl = linear.prepare_linear(p)
    assert linear.packed_matmul(torch.zeros((0, 128), dtype=dtype, device="cuda"), pl).shape == (0, 24)
    assert linear.packed_matmul(torch.zeros((2, 0, 128), dtype=dtype, device="cuda"), pl).shape \
        == (2, 0, 24)
    x = _x((3, 128), torch.float32, 2)
    y = linear.packed_matmul(x.cpu().numpy(), pl)
    assert isinstance(y, np.ndarray) and np.array_equal(y, linear.packed_matmul(x, pl).cpu().numpy())


@pytest.mark.parametrize("t", [4, 150])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_stay_in_their_row(t, dtype):
    p, w = _packed(40, 200, 40, 4, False, 2, act_order=True)  # padded positions
    pl = linear.prepare_linear(p)
    x = _x((t, 200), dtype, 3)
    x[1, 5], x[2, 7] = float("inf"), float("nan")
    y = linear.packed_matmul(x, pl)
    good = torch.tensor([i for i in range(t) if i not in (1, 2)], device="cuda")
    _check(y[good], x[good], w, pl)
    ref = x[1:3].double() @ w.T
    assert torch.equal(torch.isnan(y[1:3]), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(y[1:3].double()[inf], ref[inf])


@pytest.mark.parametrize("t", [1, 6, 200])
def test_float32_terms_are_exact(t):
    """Values that need all 24 bits, over the exponents of float32."""
    p, w = _packed(32, 128, 128, 8, False, 9, act_order=False)
    pl = linear.prepare_linear(p)
    gen = torch.Generator(device="cuda").manual_seed(t)
    x = (1 + torch.rand((t, 128), generator=gen, device="cuda"))
    x *= torch.exp2(torch.randint(-60, 60, (t, 1), generator=gen, device="cuda").float())
    _check(linear.packed_matmul(x, pl), x, w, pl)


def test_of_a_gptq_result_and_module():
    w, x = inputs.single_linear(0, m=96, n=512, tokens=2048)
    h = (x.astype(np.float64).T @ x / x.shape[0]).astype(np.float32)
    for bits, sym in ((4, False), (3, False), (4, True)):
        cfg = QuantConfig(w_bits=bits, group_size=128, sym=sym, ordering_mode="diag_h",
                          semantics="intended")
        p = packing.pack_result(gptq_quantize(w, h, cfg), bits, 128, sym)
        lin = linear.QuantLinear(p)
        assert (lin.in_features, lin.out_features) == (512, 96)
        xt = torch.from_numpy(x[:50]).cuda()
        # dequantize() rounds each weight to float32: half a step of A more
        ref = xt.double() @ packing.dequantize(p).double().T
        amount = xt.double().abs() @ packing.dequantize(p).double().abs().T
        tol = (8 * 17 + 4 + 32 + 1) * 2.0 ** -23 * amount + 2.0 ** -24 * ref.abs()
        assert bool(((lin(xt).double() - ref).abs() <= tol).all())


def test_copies_have_their_own_weights():
    p, w = _packed(40, 256, 64, 4, False, 8, act_order=True)
    lin = linear.QuantLinear(p)
    x = _x((5, 256), torch.bfloat16, 1)
    want = lin(x)
    for other in (copy.deepcopy(lin), pickle.loads(pickle.dumps(lin))):
        assert other.weights.qweight.data_ptr() != lin.weights.qweight.data_ptr()
        lin.weights.qweight.zero_()
        assert torch.equal(other(x), want)
        lin = linear.QuantLinear(p)


@pytest.mark.parametrize("t", [1, 8, 100, 260])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_streams_and_graphs(t, dtype):
    """The same bits on a side stream and from two captured graphs replayed in
    turn, with new inputs each time."""
    p, w = _packed(200, 1024, 128, 4, False, 6, act_order=True)
    pl = linear.prepare_linear(p)
    x = [_x((t, 1024), dtype, s) for s in (1, 2, 3, 4)]
    ref = [linear.packed_matmul(v, pl) for v in x]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = linear.packed_matmul(x[0], pl)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, ref[0])
    bufs = [x[0].clone(), x[1].clone()]
    graphs, outs = [], []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(linear.packed_matmul(b, pl))
        graphs.append(g)
    for a, c in ((0, 1), (2, 3), (3, 0)):
        bufs[0].copy_(x[a])
        bufs[1].copy_(x[c])
        graphs[0].replay()
        graphs[1].replay()
        assert torch.equal(outs[0], ref[a]) and torch.equal(outs[1], ref[c])


def test_refusals():
    p, _ = _packed(24, 128, 32, 4, False, 1, act_order=True)
    pl = linear.prepare_linear(p)
    x = torch.zeros((2, 128), device="cuda")
    with pytest.raises(ValueError, match="must be float32"):
        linear.packed_matmul(x.double(), pl)
    with pytest.raises(ValueError, match="must be \\[..., 128\\]"):
        linear.packed_matmul(x[:, :127], pl)
    with pytest.raises(ValueError, match="weights on"):
        linear.packed_matmul(x.cpu(), pl)
    with pytest.raises(ValueError, match="out must be"):
        linear.packed_matmul(x, pl, out=torch.zeros((2, 25), device="cuda"))
    buf = torch.zeros((2, 256), device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        linear.packed_matmul(buf[:, :128], pl, out=buf.view(-1)[100:148].view(2, 24))

    def broken(**kw):
        return packing.PackedLinear(**{**p.__dict__, **kw})

    for kw, text in ((dict(zeros=p.zeros + 0.5), "whole numbers"),
                     (dict(zeros=p.zeros - 16), "whole numbers"),
                     (dict(zeros=p.zeros * float("nan")), "whole numbers"),
                     (dict(scales=p.scales * float("inf")), "finite"),
                     (dict(g_idx=p.g_idx + 1), "g_idx must lie"),
                     (dict(g_idx=p.g_idx - 1), "g_idx must lie"),
                     (dict(g_idx=p.g_idx[:-1]), "g_idx must be"),
                     (dict(bits=9), "bits must be"),
                     (dict(n=0), "in_features"),
                     (dict(qweight=p.qweight[:, :-1]), "qweight must be"),
                     (dict(scales=p.scales[:-1]), "scales and zeros")):
        with pytest.raises(ValueError, match=text):
            linear.prepare_linear(broken(**kw))


def test_gradients_are_refused():
    p, w = _packed(40, 256, 64, 4, False, 8, act_order=False)
    x = _x((5, 256), torch.bfloat16, 1).requires_grad_()
    lin = linear.QuantLinear(p)
    with pytest.raises(ValueError, match="no gradient"):
        lin(x)
    with torch.no_grad():
        want = lin(x)
    assert torch.equal(lin(x.detach()), want)


def test_autograd_sees_that_out_is_written():
    """A tensor that a graph keeps for its backward pass, written in between."""
    p, _ = _packed(64, 64, 32, 4, False, 8, act_order=False)
    pl = linear.prepare_linear(p)
    leaf = _x((5, 64), torch.float32, 1).requires_grad_()
    y = leaf.exp()  # kept: its gradient is itself
    with torch.no_grad():
        linear.packed_matmul(_x((5, 64), torch.float32, 2), pl, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():  # (tensors without a version)
        out = torch.empty((5, 64), device="cuda")
        assert linear.packed_matmul(_x((5, 64), torch.float32, 2), pl, out=out) is out


def test_out_that_asks_for_gradients_is_refused():
    p, _ = _packed(64, 64, 32, 4, False, 8, act_order=False)
    pl = linear.prepare_linear(p)
    x = _x((5, 64), torch.float32, 1)
    leaf = torch.zeros((5, 64), device="cuda", requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="out takes no gradients"):
            linear.packed_matmul(x, pl, out=out)
        with torch.no_grad():
            assert torch.equal(linear.packed_matmul(x, pl, out=out), linear.packed_matmul(x, pl))
