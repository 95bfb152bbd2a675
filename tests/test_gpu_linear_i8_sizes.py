"""The linear layer in 8-bit integers at the sizes where its kernels change: few rows, short rows, tiles of each size, sums
split over workgroups; inner sizes that no piece of a row divides; weights at any byte.  Against the same plain statement in
64 bits and with the same tolerances as test_gpu_linear_i8.py: the sums are exact however they are split."""
import numpy as np
import pytest

import experts_ref as R
from test_gpu_experts import tb  # noqa: F401
from test_gpu_linear_i8 import _case, _check, _np, _run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DENSE = [(1, 15, 70), (200, 2, 33), (70000, 9, 5),                     # below one piece
         (2, 129, 40), (3, 1025, 48), (16, 2047, 33), (9, 8209, 40), (5, 40001, 20),      # few rows, one and several passes
         (6, 300, 20000),                                                      # few rows, two fragments of channels a workgroup
         (17, 257, 65), (40, 2048, 200), (33, 4099, 70), (65, 2049, 129), (900, 8192, 65),   # small tiles, split from 16 steps on
         (500, 400, 1000), (1030, 641, 1100), (2305, 260, 4100),                 # larger tiles
         (4200, 129, 1030), (1100, 255, 4100), (4097, 256, 1025)]                # short rows with many channels


@pytest.mark.parametrize("given", [False, True], ids=["x", "8 bits"])
@pytest.mark.parametrize("m,k,n", DENSE)
def test_sizes(tb, m, k, n, given):
    rng = np.random.default_rng([m, k, n])
    dtype = (0, 1, 2)[(m + k + n) % 3]
    x, w, ws, b = _case(rng, m, k, n, 1, dtype, "edge")
    if given:
        q, s = rng.integers(-128, 128, (m, k)), np.exp(rng.normal(size=m)).astype(np.float32) / 100
    else:
        q, s = R.quantize(_np(x))
    got = _run(tb, x, dtype, w, ws, b, True, q=(q, s) if given else None)
    _check(got, *R.linear(q, s, w[0], ws[0], b[0], True), dtype)


@pytest.mark.parametrize("skew", [1, 2, 3, 4, 16])
@pytest.mark.parametrize("extra", [0, 1, 2])
@pytest.mark.parametrize("m,k,n", [(3, 1000, 77), (1, 272, 64), (20, 272, 64), (50, 2100, 100), (9, 64, 70), (200, 200, 130)])
def test_weights_at_any_byte(tb, m, k, n, extra, skew):
    rng = np.random.default_rng([m, k, n, extra, skew])
    x, w, ws, b = _case(rng, m, k, n, 1, 0)
    q, s = R.quantize(_np(x))
    want = R.linear(q, s, w[0], ws[0], b[0], False)
    for given in (None, (q, s)):
        _check(_run(tb, x, 0, w, ws, b, False, ld=(extra, extra, extra), skew=(skew, skew, skew), q=given), *want, 0)


@pytest.mark.parametrize("dtype,y_dtype", [(0, 1), (0, 2), (1, 0), (1, 2), (2, 0), (2, 1)])
@pytest.mark.parametrize("m,k,n", [(300, 31, 70), (300, 64, 256), (300, 250, 257), (20000, 100, 70), (5, 500, 33), (30, 700, 90)])
def test_types_there_and_back(tb, m, k, n, dtype, y_dtype):
    """y's type is not x's"""
    rng = np.random.default_rng([m, k, n, dtype, y_dtype])
    x, w, ws, b = _case(rng, m, k, n, 1, dtype)
    q, s = R.quantize(_np(x))
    _check(_run(tb, x, dtype, w, ws, b, True, y_dtype=y_dtype), *R.linear(q, s, w[0], ws[0], b[0], True), y_dtype)


BY_EXPERT = [(30, 2100, 50, 3), (100, 2048, 96, 2), (300, 4100, 130, 2), (250, 300, 400, 20), (2500, 300, 700, 20), (9000, 500, 520, 8), (1600, 1029, 140, 100),
             (3000, 200, 1500, 6), (500, 7, 40, 9), (40, 1000, 30, 1000)]


@pytest.mark.parametrize("kind", ["even", "one", "gaps"])
@pytest.mark.parametrize("m,k,n,e", BY_EXPERT)
def test_sizes_by_expert(tb, m, k, n, e, kind):
    """even: all alike; one: every row to one expert in the middle; gaps: half of the experts empty, rows before the first
    expert's and behind the last's"""
    rng = np.random.default_rng([m, k, n, e, len(kind)])
    dtype = (0, 1, 2)[(m + k + e) % 3]
    x, w, ws, b = _case(rng, m, k, n, e, dtype)
    if kind == "even":
        offsets = np.linspace(0, m, e + 1)
    elif kind == "one":
        offsets = np.where(np.arange(e + 1) <= e // 2, 0, m)
    else:
        offsets = np.linspace(m // 9, m - m // 9, e + 1)
        offsets[1::2] = offsets[0:-1:2][: offsets[1::2].size]
    offsets = offsets.astype(np.int32)
    q, s = R.quantize(_np(x))
    got = _run(tb, x, dtype, w, ws, b, False, offsets=offsets)
    for i in range(e):
        r = slice(offsets[i], offsets[i + 1])
        if offsets[i] < offsets[i + 1]:
            _check(got[r], *R.linear(q[r], s[r], w[i], ws[i], b[i], False), dtype)
    assert (got[:offsets[0]] == 77).all() and (got[offsets[-1]:] == 77).all()


def test_offsets_that_are_none_in_tiles(tb):
    """Offsets that fall or lie outside the rows, in the split and the unsplit tiles: nothing outside the arrays is touched."""
    rng = np.random.default_rng(3)
    for m, k, n in ((200, 2100, 48), (200, 500, 48)):
        x, w, ws, b = _case(rng, m, k, n, 6, 0)
        for off in ([0, 500, 20, -7, 2 ** 31 - 1, -2 ** 31, 3], [-5, -4, -3, -2, -1, 0, 10], [300] * 7, [2 ** 31 - 1] * 7):
            _run(tb, x, 0, w, ws, b, False, offsets=np.array(off, np.int32))


@pytest.mark.parametrize("m,k,n,e", [(40, 2050, 200, 1), (1000, 700, 512, 1), (60, 2048, 100, 2), (3, 4097, 512, 1)])
def test_two_streams_and_graphs(tb, m, k, n, e):
    """Two calls at once with workspaces of their own, eager and captured, each many times: the results of each alone."""
    rng = np.random.default_rng([m, k, n])
    size = tb.linear_i8_workspace(m, k, n, 0, e)
    calls = []
    for i in range(2):
        x, w, ws, b = _case(rng, m, k, n, e, 0)
        t = [x.cuda(), torch.from_numpy(w).cuda(), torch.from_numpy(ws).cuda(), torch.from_numpy(b).cuda(), torch.from_numpy(np.linspace(0, m, e + 1).astype(np.int32)).cuda(),
             torch.zeros(m, n, dtype=torch.float16, device="cuda"), torch.zeros(max(16, size), dtype=torch.uint8, device="cuda")]
        calls.append(t)

    def run(t, stream):
        x, w, ws, b, off, y, buf = t
        tb.linear_i8(x.data_ptr(), 0, m, k, k, w.data_ptr(), k, ws.data_ptr(), n, y.data_ptr(), 0, n, d_bias=b.data_ptr(), d_offsets=off.data_ptr() if e > 1 else 0,
                     n_experts=e, d_workspace=buf.data_ptr(), workspace_bytes=size, stream=stream.cuda_stream)

    want = []
    for t in calls:
        run(t, torch.cuda.current_stream())
        torch.cuda.synchronize()
        want.append(t[5].clone())
        assert t[5].abs().max() > 0
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for t, s in zip(calls, streams):
            run(t, s)
    torch.cuda.synchronize()
    for t, y in zip(calls, want):
        assert torch.equal(t[5], y)
        t[5].zero_()
    graphs = []
    for t, s in zip(calls, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            run(t, s)
        graphs.append(g)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for t, y in zip(calls, want):
            assert torch.equal(t[5], y)
            t[5].zero_()
        torch.cuda.synchronize()
