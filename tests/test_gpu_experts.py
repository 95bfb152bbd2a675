"""Samples sorted by expert and back with weights (sng_expert_*): against plain statements in 64 bits.

Tolerances, from the arithmetic the operators document:
  plan, dispatch      whole numbers and copies: equal;
  combine             k f32 fused multiply-adds, each off by at most 2^-24 of a partial sum (bounded by the sum of
                      magnitudes), then one rounding to the type;
  rows' gradient      one f32 product (2^-24), then one rounding to the type;
  weights' gradient   d f32 fused multiply-adds and additions in some order: d * 2^-24 of the sum of magnitudes.
Every output lies between guard values that have to survive."""
import ctypes

import numpy as np
import pytest

import experts_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def tb():
    from synerfgine_amd import Testbed
    t = Testbed(0)
    yield t
    t.close()


class Guarded:
    """A device array of `shape` with row stride `ld`, `skew` elements into an allocation full of guard values."""

    def __init__(self, shape, dtype, ld=None, skew=0, fill=None):
        self.rows, self.cols = shape if len(shape) == 2 else (1, shape[0])
        self.ld, self.skew = ld or self.cols, skew
        self.guard = 77 if not dtype.is_floating_point else 77.0
        self.all = torch.full((skew + max(0, self.rows - 1) * self.ld + self.cols + 64,), self.guard, dtype=dtype, device="cuda")
        if self.rows == 0:
            self.view = self.all[:0].reshape(0, self.cols)
        else:
            self.view = torch.as_strided(self.all, (self.rows, self.cols), (self.ld, 1), skew)
        if fill is not None:
            self.view.copy_(fill.reshape(self.rows, self.cols) if torch.is_tensor(fill) else torch.as_tensor(fill).reshape(self.rows, self.cols))
        self.shape = shape

    @property
    def ptr(self):
        return self.all.data_ptr() + self.skew * self.all.element_size()

    def get(self):
        torch.cuda.synchronize()
        inside = torch.zeros(self.all.shape, dtype=torch.bool, device="cuda")
        if self.rows:
            torch.as_strided(inside, (self.rows, self.cols), (self.ld, 1), self.skew).fill_(True)
        assert (self.all[~inside] == self.guard).all(), "written outside the rows"
        v = self.view.reshape(self.shape).cpu()
        return (v.float() if v.dtype == torch.bfloat16 else v).numpy()


def _ids(n, k, e, kind, seed=0):
    rng = np.random.default_rng([seed, n, k, e])
    if kind == "random":
        ids = rng.integers(0, e, (n, k))
    elif kind == "outside":
        ids = rng.integers(-2, e + 3, (n, k))
        far = rng.random((n, k)) < 0.05
        ids[far] = rng.choice([-2 ** 31, 2 ** 31 - 1, e, -1], far.sum())
    elif kind == "none":
        ids = np.full((n, k), -1)
    elif kind == "one":
        ids = np.full((n, k), e - 1)
    else:   # few experts, long runs, most experts empty
        ids = np.sort(rng.integers(0, max(1, e // 7 + 1), (n, k)), axis=0)
    return ids.astype(np.int32)


def _sort(tb, ids, e, stream=0):
    n, k = ids.shape
    d_ids = Guarded((n * k,), torch.int32, fill=ids) if n else Guarded((1,), torch.int32)
    off, order, slot = Guarded((e + 1,), torch.int32), Guarded((n * k,), torch.int32), Guarded((n * k,), torch.int32)
    size = tb.expert_sort_workspace(n, k, e)
    ws = Guarded((max(1, size),), torch.uint8)
    tb.expert_sort(d_ids.ptr, n, k, e, off.ptr, order.ptr, slot.ptr, ws.ptr if size else 0, size, stream)
    out = off.get(), order.get(), slot.get().reshape(n, k)
    ws.get()
    return out


@pytest.mark.parametrize("kind", ["random", "outside", "none", "one", "runs"])
@pytest.mark.parametrize("n,k,e", [(0, 1, 1), (0, 3, 4096), (1, 1, 1), (5, 2, 8), (64, 1, 1), (65, 1, 2), (1023, 1, 3), (512, 2, 1024), (1025, 1, 2), (100, 7, 1025),
                                   (16384, 1, 1000), (5461, 3, 1024), (16385, 1, 64), (4096, 5, 4096), (33333, 3, 17), (300001, 1, 511), (262144, 8, 64)])
def test_sort(tb, n, k, e, kind):
    ids = _ids(n, k, e, kind)
    for got, want in zip(_sort(tb, ids, e), R.plan(ids, e)):
        assert np.array_equal(got, want)


ROWS = [  # n, k, d, extra stride, skew: one element, 28-byte rows, odd lengths, wide rows, wider than a workgroup
    (1, 1, 1, 0, 0), (3, 2, 7, 0, 0), (257, 1, 4, 0, 0), (65, 3, 31, 2, 1), (33, 2, 64, 0, 0), (17, 4, 64, 8, 4), (40, 5, 333, 0, 0), (9, 8, 1024, 0, 0),
    (5, 9, 2049, 0, 3), (6, 2, 4096, 0, 0), (3, 1, 10000, 16, 8), (2000, 2, 4, 4, 0), (1, 300, 24, 0, 0)]


def _rows(rng, n, d, dtype):
    x = torch.from_numpy(rng.normal(size=(n, d)).astype(np.float32) * np.exp(rng.normal(size=(n, 1))).astype(np.float32))
    return x.to(R.TORCH[dtype])


def _np(t):
    return t.float().numpy()


@pytest.mark.parametrize("dtype", [0, 1, 2, 3], ids=["f16", "bf16", "f32", "i8"])
@pytest.mark.parametrize("n,k,d,extra,skew", ROWS)
def test_dispatch(tb, n, k, d, extra, skew, dtype):
    e = 5
    ids = _ids(n, k, e, "outside", seed=1)
    _, order, slot = R.plan(ids, e)
    rng = np.random.default_rng([n, k, d])
    x = torch.from_numpy(rng.integers(-128, 128, (n, d)).astype(np.int8)) if dtype == 3 else _rows(rng, n, d, dtype)
    gx = Guarded((n, d), x.dtype, ld=d + extra, skew=skew, fill=x)
    go, gs = Guarded((n * k,), torch.int32, fill=order), Guarded((n * k,), torch.int32, fill=slot)
    out = Guarded((n * k, d), x.dtype, ld=d + extra, skew=skew)   # rows of no choice keep the guard values
    tb.expert_dispatch(gx.ptr, dtype, d, d + extra, go.ptr, gs.ptr, n, k, out.ptr, d + extra)
    want = np.full((n * k, d), 77, np.float32)
    kept = np.flatnonzero(order >= 0)
    want[kept] = _np(x)[order[kept] // k]
    assert np.array_equal(out.get().astype(np.float32), want)


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("n,k,d,extra,skew", ROWS)
def test_combine(tb, n, k, d, extra, skew, dtype, weighted):
    ids = _ids(n, k, 6, "outside", seed=2)
    ids[n // 2] = -1   # a sample that nobody holds
    _, _, slot = R.plan(ids, 6)
    rng = np.random.default_rng([n, k, d, 5])
    rows = _rows(rng, n * k, d, dtype)
    w = rng.normal(size=(n, k)).astype(np.float32)
    w[slot < 0] = np.nan   # not read
    live = np.zeros(n * k, bool)
    live[slot[slot >= 0]] = True
    rows[torch.from_numpy(~live)] = float("nan")   # rows of no choice neither
    g = Guarded((n * k, d), rows.dtype, ld=d + extra, skew=skew, fill=rows)
    gw, gs = Guarded((n * k,), torch.float32, fill=w), Guarded((n * k,), torch.int32, fill=slot)
    y = Guarded((n, d), rows.dtype, ld=d + extra, skew=skew)
    tb.expert_combine(g.ptr, dtype, d, d + extra, gw.ptr if weighted else 0, gs.ptr, n, k, y.ptr, d + extra)
    got = y.get().astype(np.float64)
    want, size = R.combine(_np(rows), w if weighted else None, slot)
    tol = (k + 1) * 2.0 ** -24 * size * 1.01 + R.half_step(dtype) * (np.abs(want) + (k + 1) * 2.0 ** -24 * size) + R.TINY[dtype]
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    assert (got[(slot < 0).all(1)] == 0).all()


@pytest.mark.parametrize("wanted", ["both", "rows", "weights", "unweighted"])
@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("n,k,d,extra,skew", ROWS)
def test_combine_backward(tb, n, k, d, extra, skew, dtype, wanted):
    ids = _ids(n, k, 6, "outside", seed=3)
    _, _, slot = R.plan(ids, 6)
    rng = np.random.default_rng([n, k, d, 6])
    rows, dy = _rows(rng, n * k, d, dtype), _rows(rng, n, d, dtype)
    w = rng.normal(size=(n, k)).astype(np.float32)
    g, gdy = Guarded((n * k, d), rows.dtype, ld=d + extra, skew=skew, fill=rows), Guarded((n, d), rows.dtype, ld=d + extra, skew=skew, fill=dy)
    gw, gs = Guarded((n * k,), torch.float32, fill=w), Guarded((n * k,), torch.int32, fill=slot)
    drows, dw = Guarded((n * k, d), rows.dtype, ld=d + extra, skew=skew), Guarded((n * k,), torch.float32)
    ask_rows, ask_w = wanted != "weights", wanted != "rows"
    tb.expert_combine_backward(gdy.ptr, d + extra, g.ptr if ask_w else 0, d + extra, dtype, d, 0 if wanted == "unweighted" else gw.ptr, gs.ptr, n, k,
                               drows.ptr if ask_rows else 0, d + extra, dw.ptr if ask_w else 0)
    want, want_w, size = R.combine_grad(_np(dy), _np(rows), None if wanted == "unweighted" else w, slot, np.full((n * k, d), 77.0))
    got = drows.get().astype(np.float64)
    if ask_rows:
        assert (np.abs(got - want) <= (R.half_step(dtype) + 2.0 ** -23) * np.abs(want) + R.TINY[dtype]).all()
    else:
        assert (got == 77).all()
    got_w = dw.get().reshape(n, k).astype(np.float64)
    if ask_w:
        assert (np.abs(got_w - want_w) <= (d + 8) * 2.0 ** -24 * 1.01 * size).all()
        assert (got_w[slot < 0] == 0).all()
    else:
        assert (got_w == 77).all()


def test_backward_is_the_forwards_derivative(tb):
    """The gradients of sum(G * combine(dispatch(x), w)) against the formula's chain and against differences.  The function
    is linear in x and in w, so a central difference has only the f32 forward's rounding error: each output is off by at
    most (k + 1) 2^-24 of its magnitudes, twice, over 2h."""
    n, k, d, e, h = 23, 3, 12, 4, 0.5
    ids = _ids(n, k, e, "outside", seed=9)
    _, order, slot = R.plan(ids, e)
    rng = np.random.default_rng(4)
    x, G, w = (rng.normal(size=s).astype(np.float32) for s in ((n, d), (n, d), (n, k)))
    go, gs = Guarded((n * k,), torch.int32, fill=order), Guarded((n * k,), torch.int32, fill=slot)

    def forward(x, w):
        gx, gw = Guarded((n, d), torch.float32, fill=x), Guarded((n * k,), torch.float32, fill=w)
        rows, y = Guarded((n * k, d), torch.float32), Guarded((n, d), torch.float32)
        tb.expert_dispatch(gx.ptr, 2, d, d, go.ptr, gs.ptr, n, k, rows.ptr, d)
        tb.expert_combine(rows.ptr, 2, d, d, gw.ptr, gs.ptr, n, k, y.ptr, d)
        return rows, y.get().astype(np.float64)

    rows, _ = forward(x, w)
    gG, gw = Guarded((n, d), torch.float32, fill=G), Guarded((n * k,), torch.float32, fill=w)
    drows, dw, dx = Guarded((n * k, d), torch.float32), Guarded((n * k,), torch.float32), Guarded((n, d), torch.float32)
    tb.expert_combine_backward(gG.ptr, d, rows.ptr, d, 2, d, gw.ptr, gs.ptr, n, k, drows.ptr, d, dw.ptr)
    tb.expert_dispatch_backward(drows.ptr, 2, d, d, gs.ptr, n, k, dx.ptr, d)
    dx, dw = dx.get().astype(np.float64), dw.get().reshape(n, k).astype(np.float64)
    kept = (slot >= 0)
    assert np.abs(dx - G * (w * kept).sum(1, keepdims=True)).max() <= (2 * k + 2) * 2.0 ** -24 * np.abs(G * (np.abs(w) * kept).sum(1, keepdims=True)).max()
    size = (np.abs(w) * kept).sum(1) * (np.abs(x).max() + h) * np.abs(G).max() * d
    for t, c in [(0, 0), (5, 11), (22, 6), (13, 3)]:
        step = np.zeros_like(x)
        step[t, c] = h
        diff = ((forward(x + step, w)[1] - forward(x - step, w)[1]) * G).sum() / (2 * h)
        assert abs(diff - dx[t, c]) <= (4 * k + 8) * 2.0 ** -24 * (size[t] + np.abs(dx[t, c])) / h
    for t, j in [(0, 0), (5, 2), (22, 1), (13, 0)]:
        step = np.zeros_like(w)
        step[t, j] = h
        diff = ((forward(x, w + step)[1] - forward(x, w - step)[1]) * G).sum() / (2 * h)
        assert abs(diff - dw[t, j]) <= (4 * k + d + 8) * 2.0 ** -24 * (size[t] + h * np.abs(x).max() * np.abs(G).max() * d) / h


def test_plan_that_is_no_plan(tb):
    """Slots and orders outside [0, n * k) are taken as dropped ones: nothing outside the arrays is touched."""
    n, k, d = 50, 2, 24
    rng = np.random.default_rng(0)
    bad = rng.choice(np.array([-1, -2 ** 31, n * k, 2 ** 31 - 1, 3, 7], np.int64), (n, k)).astype(np.int32)
    gs = Guarded((n * k,), torch.int32, fill=bad)
    x, rows, w = Guarded((n, d), torch.float16, fill=torch.ones(n, d)), Guarded((n * k, d), torch.float16, fill=torch.ones(n * k, d)), Guarded((n * k,), torch.float32, fill=np.ones((n, k), np.float32))
    y, drows, dw = Guarded((n, d), torch.float16), Guarded((n * k, d), torch.float16), Guarded((n * k,), torch.float32)
    out = Guarded((n * k, d), torch.float16)
    tb.expert_dispatch(x.ptr, 0, d, d, gs.ptr, gs.ptr, n, k, out.ptr, d)
    tb.expert_combine(rows.ptr, 0, d, d, w.ptr, gs.ptr, n, k, y.ptr, d)
    tb.expert_combine_backward(x.ptr, d, rows.ptr, d, 0, d, w.ptr, gs.ptr, n, k, drows.ptr, d, dw.ptr)
    good = (bad == 3) | (bad == 7)
    assert np.array_equal(y.get(), np.repeat(good.sum(1), d).reshape(n, d).astype(np.float16))
    assert np.array_equal(dw.get().reshape(n, k), good * float(d))
    drows.get(), out.get()


@pytest.mark.parametrize("n", [300, 40000], ids=["one launch", "three launches"])
def test_captured_and_replayed(tb, n):
    """Sort, dispatch, combine and its gradient in one graph: each replay takes the ids and rows that are there then."""
    k, e, d = 2, 12, 16
    ids, x = torch.zeros(n, k, dtype=torch.int32, device="cuda"), torch.zeros(n, d, device="cuda", dtype=torch.float16)
    w, dy = torch.rand(n, k, device="cuda"), torch.randn(n, d, device="cuda").half()
    off, order, slot = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in (e + 1, n * k, n * k))
    rows, drows, y, dw = (torch.zeros(s, device="cuda", dtype=t) for s, t in (((n * k, d), torch.float16), ((n * k, d), torch.float16), ((n, d), torch.float16), ((n, k), torch.float32)))
    size = tb.expert_sort_workspace(n, k, e)
    ws = torch.zeros(max(16, size), dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream().cuda_stream
        tb.expert_sort(ids.data_ptr(), n, k, e, off.data_ptr(), order.data_ptr(), slot.data_ptr(), ws.data_ptr(), size, s)
        tb.expert_dispatch(x.data_ptr(), 0, d, d, order.data_ptr(), slot.data_ptr(), n, k, rows.data_ptr(), d, s)
        tb.expert_combine(rows.data_ptr(), 0, d, d, w.data_ptr(), slot.data_ptr(), n, k, y.data_ptr(), d, s)
        tb.expert_combine_backward(dy.data_ptr(), d, rows.data_ptr(), d, 0, d, w.data_ptr(), slot.data_ptr(), n, k, drows.data_ptr(), d, dw.data_ptr(), s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for it in range(4):
        host = _ids(n, k, e, ["random", "outside", "runs", "one"][it], seed=it)
        ids.copy_(torch.from_numpy(host))
        x.copy_(torch.randn(n, d, device="cuda"))
        outs = (off, order, slot, rows, y, drows, dw)
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [o.clone() for o in outs]
        for o in outs:
            o.zero_()
        step()
        torch.cuda.synchronize()
        for a, b in zip(replayed, outs):
            assert torch.equal(a, b)
        for got, want in zip((off, order, slot.view(n, k)), R.plan(host, e)):
            assert np.array_equal(got.cpu().numpy(), want)


def test_two_calls_at_once(tb):
    """Two streams, each with arrays and a workspace of its own."""
    n, k, e = 60000, 2, 33
    streams, held = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i, s in enumerate(streams):
        host = _ids(n, k, e, "outside", seed=50 + i)
        ids = torch.from_numpy(host).cuda()
        off, order, slot = (torch.zeros(m, dtype=torch.int32, device="cuda") for m in (e + 1, n * k, n * k))
        size = tb.expert_sort_workspace(n, k, e)
        held.append((host, ids, off, order, slot, torch.zeros(size, dtype=torch.uint8, device="cuda"), size))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (host, ids, off, order, slot, ws, size) in zip(streams, held):
            tb.expert_sort(ids.data_ptr(), n, k, e, off.data_ptr(), order.data_ptr(), slot.data_ptr(), ws.data_ptr(), size, s.cuda_stream)
    torch.cuda.synchronize()
    for host, _, off, order, slot, _, _ in held:
        for got, want in zip((off, order, slot.view(n, k)), R.plan(host, e)):
            assert np.array_equal(got.cpu().numpy(), want)


def test_long_rows_past_32_bits(tb):
    """Row offsets that pass 32 bits: 2.2e9 elements lie between the first and the last row's starts."""
    n, k, d, ld = 3, 1, 40, 1 << 30
    rows = torch.zeros(2 * ld + d, dtype=torch.float16, device="cuda")
    x = torch.arange(n * d, device="cuda", dtype=torch.float32).reshape(n, d).half()
    _, order, slot = R.plan(np.array([[2], [0], [1]], np.int32), 3)
    go, gs = torch.from_numpy(order).cuda(), torch.from_numpy(slot).cuda()
    tb.expert_dispatch(x.data_ptr(), 0, d, d, go.data_ptr(), gs.data_ptr(), n, k, rows.data_ptr(), ld)
    y = torch.zeros(n, d, dtype=torch.float16, device="cuda")
    tb.expert_combine(rows.data_ptr(), 0, d, ld, 0, gs.data_ptr(), n, k, y.data_ptr(), d)
    torch.cuda.synchronize()
    assert torch.equal(y, x)
    assert torch.equal(torch.as_strided(rows, (3, d), (ld, 1)).cpu(), x.cpu()[[1, 2, 0]])
