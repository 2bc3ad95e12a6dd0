"""Sizes that reach every form of the many-token product (``gq_linear_tc.cu``):
both code widths, every granule and type, tiles of one and of two parts, K split
over a cluster, and more tiles than SMs, so that a CTA goes on to another tile.
Which sizes reach which form is checked without a GPU (``test_linear_cpu.py``)."""

import ctypes

from jax_gptq_b200 import _lib

SMS = 148  # of a B200

# tokens, out_features, in_features: ragged in tokens and rows
SIZES = [(50, 1300, 1024), (100, 5000, 1024), (300, 5000, 1024), (290, 1250, 2048),
         (300, 20000, 384), (100, 20000, 640), (60, 20000, 640), (30, 20000, 640)]
GROUPS = (32, 64, 128)  # each the granule of its own weights
BITS = (4, 7)           # stored in 4 and in 8 bits


def form(m, k, bits, granule, dtype, tokens, sms=SMS):
    """gq_test_linear_form as a tuple."""
    f = (ctypes.c_int64 * 10)()
    _lib.call("gq_test_linear_form", m, k, bits, granule, dtype, tokens, sms, f)
    return tuple(f)
