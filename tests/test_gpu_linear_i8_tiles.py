"""The 8-bit linear layer in every tile, dense and by expert, with outputs of 16 and of 32 bits (a layout each), ragged in rows
and channels; against the plain statement in 64 bits and with the tolerances of test_gpu_linear_i8.py."""
import numpy as np
import pytest

import experts_ref as R
from linear_i8_tiles import TILES
from test_gpu_experts import tb  # noqa: F401
from test_gpu_linear_i8 import _case, _check, _np, _run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DENSE, BY_EXPERT = [t for t in TILES if not t[4]], [t for t in TILES if t[4]]


@pytest.mark.parametrize("y_dtype", [0, 1, 2], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("tile,m,k,n,e", DENSE, ids=[t[0] for t in DENSE])
def test_dense(tb, tile, m, k, n, e, y_dtype):
    x, w, ws, b = _case(np.random.default_rng([m, k, n]), m, k, n, 1, y_dtype, "edge")
    q, s = R.quantize(_np(x))
    _check(_run(tb, x, y_dtype, w, ws, b, True), *R.linear(q, s, w[0], ws[0], b[0], True), y_dtype)


@pytest.mark.parametrize("kind", ["even", "one", "gaps"])
@pytest.mark.parametrize("y_dtype", [0, 1, 2], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("tile,m,k,n,e", BY_EXPERT, ids=[t[0] for t in BY_EXPERT])
def test_by_expert(tb, tile, m, k, n, e, y_dtype, kind):
    """even: all alike; one: every row to one expert in the middle; gaps: the first and last empty, and rows of none in
    front and behind"""
    x, w, ws, b = _case(np.random.default_rng([m, k, n, e]), m, k, n, e, y_dtype)
    if kind == "even":
        offsets = np.linspace(0, m, e + 1)
    elif kind == "one":
        offsets = np.where(np.arange(e + 1) <= e // 2, 0, m)
    else:
        offsets = np.linspace(m // 9, m - m // 9, e + 1)
        offsets[1], offsets[-2] = offsets[0], offsets[-1]
    offsets = offsets.astype(np.int32)
    q, s = R.quantize(_np(x))
    got = _run(tb, x, y_dtype, w, ws, b, False, offsets=offsets)
    for i in range(e):
        r = slice(offsets[i], offsets[i + 1])
        if offsets[i] < offsets[i + 1]:
            _check(got[r], *R.linear(q[r], s[r], w[i], ws[i], b[i], False), y_dtype)
    assert (got[:offsets[0]] == 77).all() and (got[offsets[-1]:] == 77).all()
