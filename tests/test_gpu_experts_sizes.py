"""Samples sorted by expert at the sizes where the sort's steps change (one workgroup, counts added up by each workgroup,
counts summed by a step of their own), and rows of every length around a memory access."""
import numpy as np
import pytest

import experts_ref as R
from test_gpu_experts import Guarded, _ids, _np, _rows, _sort, tb  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("kind", ["random", "outside", "none", "one", "runs"])
@pytest.mark.parametrize("n,k,e", [(1024, 1, 5), (2049, 2, 1000), (1366, 3, 513), (4096, 1, 1024), (4097, 1, 1),                 # one workgroup
                                   (20000, 1, 1), (16385, 1, 1000), (30000, 1, 513), (8192, 2, 1024), (500000, 1, 66),           # counts added up
                                   (500000, 1, 67), (33000, 1, 1000), (2100000, 1, 3),                                          # summed before
                                   (1, 1, 1025), (4096, 1, 2000), (50000, 2, 3001)])                                            # many experts
def test_sort_sizes(tb, n, k, e, kind):
    ids = _ids(n, k, e, kind, seed=9)
    for got, want in zip(_sort(tb, ids, e), R.plan(ids, e)):
        assert np.array_equal(got, want)


LENGTHS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 23, 33, 63, 65, 127, 130, 257, 1030]


@pytest.mark.parametrize("skew", [0, 1, 3])
@pytest.mark.parametrize("dtype", [0, 1, 2, 3], ids=["f16", "bf16", "f32", "i8"])
def test_row_lengths(tb, dtype, skew):
    """There, back, and back's gradient, for lengths around 2, 4, 8 and 16 bytes; rows at any element"""
    n, k, e = 50, 3, 4
    ids = _ids(n, k, e, "outside", seed=4)
    _, order, slot = R.plan(ids, e)
    kept = np.flatnonzero(order >= 0)
    live = np.zeros(n * k, bool)
    live[slot[slot >= 0]] = True
    for d in LENGTHS:
        rng = np.random.default_rng([d, dtype, skew])
        x = torch.from_numpy(rng.integers(-128, 128, (n, d)).astype(np.int8)) if dtype == 3 else _rows(rng, n, d, dtype)
        gx = Guarded((n, d), x.dtype, ld=d + skew, skew=skew, fill=x)
        go, gs = Guarded((n * k,), torch.int32, fill=order), Guarded((n * k,), torch.int32, fill=slot)
        out = Guarded((n * k, d), x.dtype, ld=d + skew, skew=skew)
        tb.expert_dispatch(gx.ptr, dtype, d, d + skew, go.ptr, gs.ptr, n, k, out.ptr, d + skew)
        want = np.full((n * k, d), 77, np.float32)
        want[kept] = _np(x)[order[kept] // k]
        assert np.array_equal(out.get().astype(np.float32), want), d
        if dtype == 3:
            continue
        rows, dy, w = _rows(rng, n * k, d, dtype), _rows(rng, n, d, dtype), rng.normal(size=(n, k)).astype(np.float32)
        gr, gw = Guarded((n * k, d), rows.dtype, ld=d + skew, skew=skew, fill=rows), Guarded((n * k,), torch.float32, fill=w)
        y = Guarded((n, d), rows.dtype, ld=d + skew, skew=skew)
        tb.expert_combine(gr.ptr, dtype, d, d + skew, gw.ptr, gs.ptr, n, k, y.ptr, d + skew)
        want, size = R.combine(_np(rows), w, slot)
        sums = k * 2.0 ** -24 * size * 1.01   # (1.01: second order)
        assert (np.abs(y.get() - want) <= sums + R.half_step(dtype) * (np.abs(want) + sums) + R.TINY[dtype]).all(), d
        gdy = Guarded((n, d), rows.dtype, ld=d + skew, skew=skew, fill=dy)
        drows, dw = Guarded((n * k, d), rows.dtype, ld=d + skew, skew=skew), Guarded((n * k,), torch.float32)
        tb.expert_combine_backward(gdy.ptr, d + skew, gr.ptr, d + skew, dtype, d, gw.ptr, gs.ptr, n, k, drows.ptr, d + skew, dw.ptr)
        want_r, want_w, size = R.combine_grad(_np(dy), _np(rows), w, slot, np.full((n * k, d), 77.0))
        got_r, got_w = drows.get().astype(np.float64), dw.get().reshape(n, k).astype(np.float64)
        assert (got_r[~live] == 77).all(), d
        err = 2.0 ** -24 * np.abs(want_r)
        assert (np.abs(got_r - want_r) <= err + R.half_step(dtype) * (np.abs(want_r) + err) + R.TINY[dtype])[live].all(), d
        assert (np.abs(got_w - want_w) <= d * 2.0 ** -24 * size * 1.01).all(), d


@pytest.mark.parametrize("n,k,d,dtype", [(600001, 2, 4, 0), (600001, 1, 3, 2), (110001, 2, 33, 1), (262147, 1, 15, 0)])
def test_combine_many_samples(tb, n, k, d, dtype):
    """More samples than workgroups at a time: several pieces a thread"""
    rng = np.random.default_rng([n, k, d])
    ids = rng.integers(-1, 8, (n, k)).astype(np.int32)
    _, _, slot = R.plan(ids, 8)
    rows = torch.from_numpy(rng.normal(size=(n * k, d)).astype(np.float32)).to(R.TORCH[dtype])
    w = rng.normal(size=(n, k)).astype(np.float32)
    g, gw, gs = Guarded((n * k, d), rows.dtype, fill=rows), Guarded((n * k,), torch.float32, fill=w), Guarded((n * k,), torch.int32, fill=slot)
    for weights in (w, None):
        y = Guarded((n, d), rows.dtype)
        tb.expert_combine(g.ptr, dtype, d, d, 0 if weights is None else gw.ptr, gs.ptr, n, k, y.ptr, d)
        want, size = R.combine(_np(rows), weights, slot)
        sums = k * 2.0 ** -24 * size * 1.01
        assert (np.abs(y.get() - want) <= sums + R.half_step(dtype) * (np.abs(want) + sums) + R.TINY[dtype]).all()


@pytest.mark.parametrize("n,k,d,dtype", [(300007, 2, 7, 2), (300007, 3, 5, 0), (300007, 1, 40, 3), (200001, 2, 33, 1)])
def test_dispatch_many_samples(tb, n, k, d, dtype):
    """More samples than one step of every workgroup takes, in short rows and in longer ones"""
    rng = np.random.default_rng([n, k, d])
    ids = rng.integers(-1, 70, (n, k)).astype(np.int32)
    _, order, slot = R.plan(ids, 70)
    x = torch.from_numpy(rng.integers(-128, 128, (n, d)).astype(np.int8)) if dtype == 3 else _rows(rng, n, d, dtype)
    gx, go, gs = Guarded((n, d), x.dtype, fill=x), Guarded((n * k,), torch.int32, fill=order), Guarded((n * k,), torch.int32, fill=slot)
    out = Guarded((n * k, d), x.dtype)
    tb.expert_dispatch(gx.ptr, dtype, d, d, go.ptr, gs.ptr, n, k, out.ptr, d)
    want = np.full((n * k, d), 77, np.float32)
    kept = np.flatnonzero(order >= 0)
    want[kept] = _np(x)[order[kept] // k]
    assert np.array_equal(out.get().astype(np.float32), want)
