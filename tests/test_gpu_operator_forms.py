"""Sizes for the forms of the operators' kernels that the other tests do not reach: short rows on many rows with several blocks
of channels, few rows with long sums and many channels, every length of a memory access with every number of choices.
Against the same plain statements in 64 bits and with the same tolerances as test_gpu_experts.py and
test_gpu_linear_i8.py."""
import numpy as np
import pytest

import experts_ref as R
from test_gpu_experts import Guarded, _ids, _np, _rows, tb  # noqa: F401
from test_gpu_linear_i8 import _case, _check, _run, _x

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = ["f16", "bf16", "f32", "i8"]


def _layer(tb, m, k, n, x_dtype, y_dtype, relu=False, offsets=None):
    """One call, dense or by expert, against the statement; x_dtype 3: 8-bit rows given"""
    e = 1 if offsets is None else len(offsets) - 1
    rng = np.random.default_rng([m, k, n, x_dtype, y_dtype, e])
    x, w, ws, b = _case(rng, m, k, n, e, 2 if x_dtype == 3 else x_dtype, "edge" if offsets is None and x_dtype != 3 else "normal")
    given = None
    if x_dtype == 3:
        given = q, s = rng.integers(-128, 128, (m, k)), np.exp(rng.normal(size=m)).astype(np.float32) / 100
    else:
        q, s = R.quantize(_np(x))
    got = _run(tb, x, x_dtype, w, ws, b, relu, y_dtype=y_dtype, q=given, offsets=offsets)
    bounds = [0, m] if offsets is None else offsets
    for i in range(e):
        r = slice(bounds[i], bounds[i + 1])
        if bounds[i] < bounds[i + 1]:
            _check(got[r], *R.linear(q[r], s[r], w[i], ws[i], b[i], relu), y_dtype)
    assert (got[:bounds[0]] == 77).all() and (got[bounds[-1]:] == 77).all()


@pytest.mark.parametrize("n", [100, 300], ids=["2 blocks", "4 blocks and a part"])
@pytest.mark.parametrize("k", [40, 100, 200])
@pytest.mark.parametrize("x_dtype", range(4), ids=TYPES)
def test_short_rows_many_channels(tb, x_dtype, k, n):
    """256 tiles of rows and more, where a workgroup takes 128 or 256 channels, and fewer, where it takes 64"""
    for y_dtype in range(3) if x_dtype == 3 else [x_dtype, (x_dtype + 1) % 3]:
        for m in (16401, 301):
            _layer(tb, m, k, n, x_dtype, y_dtype, relu=True)


@pytest.mark.parametrize("x_dtype", range(4), ids=TYPES)
def test_tiny_rows_many_channels(tb, x_dtype):
    """fewer than 16 values a row"""
    for k in (1, 9):
        _layer(tb, 16401, k, 131, x_dtype, 0 if x_dtype == 3 else x_dtype)


@pytest.mark.parametrize("m,k,n,x_dtype", [(140001, 20, 70, 0), (140001, 70, 40, 2)])
def test_short_rows_on_very_many_rows(tb, m, k, n, x_dtype):
    """tiles of 128 rows"""
    _layer(tb, m, k, n, x_dtype, x_dtype)


@pytest.mark.parametrize("x_dtype", range(4), ids=TYPES)
@pytest.mark.parametrize("m,k,n,e", [(16500, 40, 100, 37), (17000, 150, 300, 3), (140001, 32, 64, 300)])
def test_short_rows_many_channels_by_expert(tb, m, k, n, e, x_dtype):
    """experts of very different numbers of rows, rows of none in front and behind"""
    rng = np.random.default_rng([m, e])
    offsets = np.sort(rng.integers(100, m - 100, e + 1)).astype(np.int32)
    offsets[e // 2] = offsets[e // 2 - 1]   # an empty one
    _layer(tb, m, k, n, x_dtype, 1 if x_dtype == 3 else x_dtype, offsets=offsets)


@pytest.mark.parametrize("x_dtype", range(4), ids=TYPES)
@pytest.mark.parametrize("k", [300, 301, 1100, 1101], ids=lambda k: "n_in %d" % k)
def test_few_rows(tb, k, x_dtype):
    """sums of up to 1024 values and longer ones, words and odd bytes of weights; one round of workgroups, several, and two
    blocks of channels each"""
    for m, n in ((7, 600), (16, 5003), (3, 17003)):
        _layer(tb, m, k, n, x_dtype, (m + k) % 3)


@pytest.mark.parametrize("x_dtype", range(4), ids=TYPES)
@pytest.mark.parametrize("k", [300, 1101], ids=lambda k: "n_in %d" % k)
def test_few_rows_by_expert(tb, k, x_dtype):
    """the same by expert: 9 experts of no row to 30"""
    offsets = np.array([2, 2, 3, 33, 50, 50, 62, 63, 79, 90], np.int32)
    for n in (50, 2100):
        _layer(tb, 95, k, n, x_dtype, (n + k) % 3, offsets=offsets)


@pytest.mark.parametrize("dtype", range(3), ids=TYPES[:3])
def test_quantize_single_elements_of_many_rows(tb, dtype):
    """q at odd places: one element an access, 64 threads a row"""
    rows, cols = 2050, 300
    x = _x(np.random.default_rng(dtype), rows, cols, dtype, "edge")
    gx = Guarded((rows, cols), x.dtype, fill=x)
    q, scale = Guarded((rows, cols), torch.int8, ld=cols + 1, skew=1), Guarded((rows,), torch.float32)
    tb.quantize_rows_i8(gx.ptr, dtype, rows, cols, cols, q.ptr, cols + 1, scale.ptr)
    want_q, want_s = R.quantize(_np(x))
    assert np.array_equal(q.get().astype(np.int64), want_q) and np.array_equal(scale.get(), want_s, equal_nan=True)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("dtype", range(4), ids=TYPES)
def test_choices_and_lengths(tb, dtype, k):
    """rows of one element, of 2, 4, 8 and 16 bytes and their pieces, for every way that a sample's choices are read"""
    n, e = 41, 6
    ids = _ids(n, k, e, "outside", seed=12)
    _, order, slot = R.plan(ids, e)
    kept = np.flatnonzero(order >= 0)
    go, gs = Guarded((n * k,), torch.int32, fill=order), Guarded((n * k,), torch.int32, fill=slot)
    for d in (1, 2, 3, 4, 6, 8, 12, 16, 40, 150, 1100):
        rng = np.random.default_rng([d, dtype, k])
        x = torch.from_numpy(rng.integers(-128, 128, (n, d)).astype(np.int8)) if dtype == 3 else _rows(rng, n, d, dtype)
        gx, out = Guarded((n, d), x.dtype, fill=x), Guarded((n * k, d), x.dtype)
        tb.expert_dispatch(gx.ptr, dtype, d, d, go.ptr, gs.ptr, n, k, out.ptr, d)
        want = np.full((n * k, d), 77, np.float32)
        want[kept] = _np(x)[order[kept] // k]
        assert np.array_equal(out.get().astype(np.float32), want), d
        if dtype == 3:
            continue
        rows, dy, w = _rows(rng, n * k, d, dtype), _rows(rng, n, d, dtype), rng.normal(size=(n, k)).astype(np.float32)
        gr, gdy, gw, y = Guarded((n * k, d), rows.dtype, fill=rows), Guarded((n, d), rows.dtype, fill=dy), Guarded((n * k,), torch.float32, fill=w), Guarded((n, d), rows.dtype)
        tb.expert_combine(gr.ptr, dtype, d, d, gw.ptr, gs.ptr, n, k, y.ptr, d)
        want, size = R.combine(_np(rows), w, slot)
        sums = k * 2.0 ** -24 * size * 1.01
        assert (np.abs(y.get() - want) <= sums + R.half_step(dtype) * (np.abs(want) + sums) + R.TINY[dtype]).all(), d
        drows, dw = Guarded((n * k, d), rows.dtype), Guarded((n * k,), torch.float32)
        tb.expert_combine_backward(gdy.ptr, d, gr.ptr, d, dtype, d, gw.ptr, gs.ptr, n, k, drows.ptr, d, dw.ptr)
        want_r, want_w, size = R.combine_grad(_np(dy), _np(rows), w, slot, np.full((n * k, d), 77.0))
        live = np.zeros(n * k, bool)
        live[slot[slot >= 0]] = True
        got, err = drows.get().astype(np.float64), 2.0 ** -24 * np.abs(want_r)
        assert (got[~live] == 77).all(), d
        assert (np.abs(got - want_r) <= err + R.half_step(dtype) * (np.abs(want_r) + err) + R.TINY[dtype])[live].all(), d
        assert (np.abs(dw.get().reshape(n, k) - want_w) <= d * 2.0 ** -24 * size * 1.01).all(), d
