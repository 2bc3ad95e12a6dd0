"""The choice of the next token, what needs no GPU: the refusals of the C
entry point."""

import ctypes

import pytest

from jax_gptq_b200 import _lib


def _call(**kw):
    p = ctypes.c_void_p(256)
    a = dict(logits=p, dtype=0, rows=2, vocab=100, ld=100, u=p, uk=1, t=None, tk=0, tv=1.0, k=None,
             kk=0, kv=0.0, p=None, pk=0, pv=1.0, m=None, mk=0, mv=0.0, tokens=p, logprobs=p,
             stream=None)
    a.update(kw)
    return _lib.lib().gq_sample(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), b"dtype"), (dict(rows=-1), b"shape"), (dict(vocab=0), b"shape"),
    (dict(ld=99), b"shape"), (dict(vocab=(1 << 20) + 1, ld=1 << 21), b"2^20"),
    (dict(rows=1 << 27), b"rows"), (dict(uk=0), b"u must"), (dict(uk=3), b"u must"),
    (dict(tk=5), b"kind"), (dict(kk=-1), b"kind"), (dict(pk=1), b"NULL setting"),
    (dict(mk=4), b"NULL setting"), (dict(logits=None), b"NULL"), (dict(u=None), b"NULL"),
    (dict(tokens=None), b"NULL")])
def test_refuses_before_launching(kw, text):
    before = _lib.lib().gq_launch_count()
    assert _call(**kw) == _lib.GQ_EINVAL
    assert text in _lib.lib().gq_last_error()
    assert _lib.lib().gq_launch_count() == before


def test_no_rows_is_fine():
    assert _call(rows=0, logits=None, u=None, tokens=None) == _lib.GQ_OK
