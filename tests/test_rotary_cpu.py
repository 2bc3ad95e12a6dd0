"""Rotary positions, what needs no GPU: frequencies and scalings, the 64-bit
turns, and the refusals of the C entry point."""

import ctypes
import math

import pytest

from jax_gptq_b200 import _lib, rotary


def test_plain_frequencies():
    inv, f = rotary.rotary_frequencies(8, 10000.0)
    assert f == 1.0 and inv == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)


def test_scalings():
    d, theta, n = 64, 10000.0, 4096
    base, _ = rotary.rotary_frequencies(d, theta)
    lin, f = rotary.rotary_frequencies(d, theta, rotary.LinearScaling(4.0))
    assert f == 1.0 and lin == pytest.approx([w / 4 for w in base], rel=1e-15)
    ntk, f = rotary.rotary_frequencies(d, theta, rotary.NtkScaling(4.0))
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(base[-1] / 4, rel=1e-12)
    yarn, f = rotary.rotary_frequencies(d, theta, rotary.YarnScaling(4.0, n))
    assert f == pytest.approx(0.1 * math.log(4.0) + 1)
    for w, y in zip(base, yarn):
        turns = n * w / (2 * math.pi)
        assert w / 4 * (1 - 1e-12) <= y <= w * (1 + 1e-12)
        if turns > 45:  # past the ramp and its rounding to whole pairs
            assert y == w
        if turns < 0.7:
            assert y == pytest.approx(w / 4, rel=1e-12)
    assert rotary.rotary_frequencies(d, theta, rotary.YarnScaling(4.0, n, attention_factor=2.0))[1] == 2.0
    l3, f = rotary.rotary_frequencies(d, theta, rotary.Llama3Scaling(8.0, n))
    assert f == 1.0
    for w, y in zip(base, l3):
        length = 2 * math.pi / w
        if length > n:
            assert y == pytest.approx(w / 8, rel=1e-12)
        elif length < n / 4:
            assert y == w
        else:
            s = (n / length - 1) / 3
            assert y == pytest.approx((1 - s) * w / 8 + s * w, rel=1e-12)


@pytest.mark.parametrize("args", [(0,), (7,), (8, -1.0), (8, float("inf")),
                                  (8, 1e4, rotary.LinearScaling(0.0)),
                                  (8, 1e4, rotary.YarnScaling(2.0, 0)),
                                  (8, 1e4, rotary.YarnScaling(2.0, 64, beta_fast=0.0)),
                                  (8, 1e4, rotary.Llama3Scaling(2.0, 64, 4.0, 4.0))])
def test_bad_frequencies_are_refused(args):
    with pytest.raises(ValueError):
        rotary.rotary_frequencies(*args)


@pytest.mark.parametrize("args", [(8, 1e4, 10), (8, 1e4, 3), (8, 1e4, 0), (8192,)])
def test_bad_plans_are_refused(args):
    with pytest.raises(ValueError, match="rotary_dim"):
        rotary.rotary_plan(*args)


def _call(**kw):
    p = ctypes.c_void_p(256)
    a = dict(q=p, qo=p, heads=4, k=p, ko=p, kv=2, strides=(ctypes.c_int64 * 12)(*[64] * 12), pos=p,
             ps=0, p32=0, turns=p, batch=1, seq=3, d=64, r=64, inter=0, factor=1.0, tr=0, dtype=1,
             stream=None)
    a.update(kw)
    return _lib.lib().gq_rotary(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), b"dtype"), (dict(r=63), b"rotary_dim"), (dict(r=66), b"rotary_dim"),
    (dict(r=0), b"rotary_dim"), (dict(d=5000, r=64), b"head_dim"), (dict(batch=-1), b"shape"),
    (dict(heads=-1), b"shape"), (dict(heads=1 << 21), b"shape"), (dict(k=None), b"NULL"),
    (dict(q=None), b"NULL"), (dict(qo=None), b"NULL"), (dict(strides=None), b"NULL"),
    (dict(pos=None), b"NULL"), (dict(turns=None), b"NULL")])
def test_refuses_before_launching(kw, text):
    before = _lib.lib().gq_launch_count()
    assert _call(**kw) == _lib.GQ_EINVAL
    assert text in _lib.lib().gq_last_error()
    assert _lib.lib().gq_launch_count() == before


def test_nothing_to_turn_is_fine():
    assert _call(batch=0) == _lib.GQ_OK and _call(seq=0) == _lib.GQ_OK
    assert _call(heads=0, kv=0) == _lib.GQ_OK
