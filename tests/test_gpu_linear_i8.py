"""The linear layer in 8-bit integers (sng_linear_i8, sng_quantize_rows_i8): against a plain statement in 64 bits.

Tolerances: q and the int32 sums are exact, so y is off by the roundings that follow them: the sum to f32, two products and
the bias's addition (2^-24 each of the magnitudes), then one rounding to y's type."""
import ctypes

import numpy as np
import pytest

import experts_ref as R
from test_gpu_experts import Guarded, _ids, _np, tb  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _x(rng, m, k, dtype, kind="normal"):
    x = rng.normal(size=(m, k)).astype(np.float32) * np.exp(rng.normal(size=(m, 1))).astype(np.float32)
    if kind == "edge" and m >= 8:
        x[0] = 0.0
        x[1, k // 2] = np.nan
        x[2, k - 1] = np.inf
        x[3, 0] = -np.inf
        x[4] = 1e-30 if dtype else 6e-8      # the smallest rows: below 2^-100 nothing is left, f16's smallest step is kept
        x[5] = 65504.0 if dtype == 0 else 3e38
        x[6] = np.where(np.arange(k) % 2, 1.0, -0.5)   # 127 * 0.5 = 63.5: ties
        x[7] = np.arange(k) * (2.0 / 254)   # many values at and next to a half
        if k:
            x[7, 0] = 1.0
    return torch.from_numpy(x).to(R.TORCH[dtype])


QUANT = [(1, 1), (3, 7), (8, 16), (9, 64), (8, 100), (16, 128), (8, 513), (20, 2048), (8, 8192), (9, 8200), (4, 20001)]


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("extra,skew", [(0, 0), (3, 1)])
@pytest.mark.parametrize("rows,cols", QUANT)
def test_quantize(tb, rows, cols, extra, skew, dtype):
    x = _x(np.random.default_rng([rows, cols]), rows, cols, dtype, "edge")
    gx = Guarded((rows, cols), x.dtype, ld=cols + extra, skew=skew, fill=x)
    q, scale = Guarded((rows, cols), torch.int8, ld=cols + extra, skew=skew), Guarded((rows,), torch.float32)
    tb.quantize_rows_i8(gx.ptr, dtype, rows, cols, cols + extra, q.ptr, cols + extra, scale.ptr)
    want_q, want_s = R.quantize(_np(x))
    assert np.array_equal(q.get().astype(np.int64), want_q)
    assert np.array_equal(scale.get(), want_s, equal_nan=True)


def test_quantize_halves(tb):
    """Every f16 value below 2 against 1.0 and against 1.7: the roundings at each half, exactly."""
    v = np.arange(0x4000, dtype=np.uint16).view(np.float16).astype(np.float32)
    for top in (1.0, 1.7002):
        t = np.float32(np.float16(top))
        row = np.where(v <= t, v, np.float32(0))
        x = torch.from_numpy(np.stack([row, -row])).half()
        x[:, 0] = float(t)
        gx, q, scale = Guarded((2, x.shape[1]), x.dtype, fill=x), Guarded((2, x.shape[1]), torch.int8), Guarded((2,), torch.float32)
        tb.quantize_rows_i8(gx.ptr, 0, 2, x.shape[1], x.shape[1], q.ptr, x.shape[1], scale.ptr)
        want_q, want_s = R.quantize(_np(x))
        assert np.array_equal(q.get().astype(np.int64), want_q) and np.array_equal(scale.get(), want_s)


def _case(rng, m, k, n, e, dtype, kind="normal"):
    x = _x(rng, m, k, dtype, kind)
    w = rng.integers(-127, 128, (e, n, k)).astype(np.int8)
    ws = (np.exp(rng.normal(size=(e, n))) / (40 * 73 * np.sqrt(k))).astype(np.float32)
    return x, w, ws, rng.normal(size=(e, n)).astype(np.float32)


def _check(got, want, size, dtype):
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    tol = 5 * 2.0 ** -24 * size + R.half_step(dtype) * (np.abs(want) + 5 * 2.0 ** -24 * size) + R.TINY[dtype]
    top = float(torch.finfo(R.TORCH[dtype]).max)
    far = np.abs(want) > top * (1 - 2.0 ** -12)   # may round to an infinity
    ok = np.abs(np.where(far, 0, got - want)) <= tol
    assert (ok | nan).all(), np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300))


def _run(tb, x, dtype, w, ws, bias, relu, y_dtype=None, offsets=None, ld=(0, 0, 0), skew=(0, 0, 0), q=None, stream=0):
    """ld / skew: extra strides and offsets of x, w, y; q: (q, scale) given instead of x"""
    m, k = x.shape
    e, n, _ = w.shape
    y_dtype = dtype if y_dtype is None else y_dtype
    src = x if q is None else torch.from_numpy(q[0].astype(np.int8))
    t = dtype if q is None else 3
    gx = Guarded((m, k), src.dtype, ld=k + ld[0], skew=skew[0], fill=src)
    gw = Guarded((e * n, k), torch.int8, ld=k + ld[1], skew=skew[1], fill=w)
    gws, gb = Guarded((e * n,), torch.float32, fill=ws), Guarded((e * n,), torch.float32, fill=bias) if bias is not None else None
    gs = Guarded((m,), torch.float32, fill=q[1]) if q is not None else None
    go = Guarded((e + 1,), torch.int32, fill=offsets) if offsets is not None else None
    y = Guarded((m, n), R.TORCH[y_dtype], ld=n + ld[2], skew=skew[2])
    size = tb.linear_i8_workspace(m, k, n, t, e)
    ws_buf = Guarded((max(1, size),), torch.uint8)
    tb.linear_i8(gx.ptr, t, m, k, k + ld[0], gw.ptr, k + ld[1], gws.ptr, n, y.ptr, y_dtype, n + ld[2], d_bias=gb.ptr if gb else 0, relu=relu,
                 d_x_scale=gs.ptr if gs else 0, d_offsets=go.ptr if go else 0, n_experts=e, d_workspace=ws_buf.ptr if size else 0, workspace_bytes=size,
                 stream=stream)
    got = y.get().astype(np.float64)
    ws_buf.get()
    return got


SHAPES = [(1, 1, 1), (1, 16, 16), (2, 17, 5), (1, 4096, 512), (3, 1000, 77), (4, 256, 4096), (7, 640, 48), (16, 64, 64), (17, 96, 33), (31, 2048, 160), (33, 130, 130),
          (64, 32, 64), (100, 64, 64), (129, 128, 257), (200, 48, 16), (255, 333, 255), (300, 512, 640), (513, 1024, 272), (1000, 64, 3), (2050, 20, 40), (700, 200, 700)]


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear(tb, m, k, n, dtype):
    rng = np.random.default_rng([m, k, n, dtype])
    x, w, ws, b = _case(rng, m, k, n, 1, dtype, "edge")
    q, s = R.quantize(_np(x))
    for bias, relu in ((None, False), (b, True)):
        got = _run(tb, x, dtype, w, ws, bias, relu)
        _check(got, *R.linear(q, s, w[0], ws[0], None if bias is None else b[0], relu), dtype)


@pytest.mark.parametrize("ld,skew", [((1, 3, 5), (0, 0, 0)), ((0, 0, 0), (1, 5, 1)), ((8, 16, 8), (8, 16, 8)), ((7, 1, 3), (3, 7, 5))])
@pytest.mark.parametrize("m,k,n", [(1, 96, 64), (5, 64, 64), (40, 64, 80), (130, 256, 130), (260, 384, 512)])
def test_linear_strides_and_alignment(tb, m, k, n, ld, skew):
    rng = np.random.default_rng([m, k, n, 7])
    for dtype in (0, 2):
        x, w, ws, b = _case(rng, m, k, n, 1, dtype)
        q, s = R.quantize(_np(x))
        want = R.linear(q, s, w[0], ws[0], b[0], False)
        _check(_run(tb, x, dtype, w, ws, b, False, ld=ld, skew=skew), *want, dtype)
        _check(_run(tb, x, dtype, w, ws, b, False, ld=ld, skew=skew, q=(q, s)), *want, dtype)


@pytest.mark.parametrize("y_dtype", [0, 1, 2], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [(1, 128, 64), (6, 1000, 96), (50, 64, 64), (150, 144, 200), (512, 512, 512)])
def test_linear_of_8_bit_rows(tb, m, k, n, y_dtype):
    """x in 8 bits already, the full range -128 .. 127 on both sides, one quantisation for several products"""
    rng = np.random.default_rng([m, k, n, 8])
    q, s = rng.integers(-128, 128, (m, k)), np.exp(rng.normal(size=m)).astype(np.float32) / 100
    w, ws = rng.integers(-128, 128, (1, n, k)).astype(np.int8), (np.exp(rng.normal(size=(1, n))) / 4000).astype(np.float32)
    q[0], w[0, 0] = -128, -128   # the largest sum
    got = _run(tb, torch.zeros(m, k), y_dtype, w, ws, None, False, q=(q, s))
    _check(got, *R.linear(q, s, w[0], ws[0], None, False), y_dtype)


def test_linear_longest_rows(tb):
    """n_in = 131071: the largest sum, 131071 * 128 * 128 = 2^31 - 2^14, still fits"""
    m, k, n = 3, 131071, 20
    rng = np.random.default_rng(1)
    q, w = rng.integers(-128, 128, (m, k)), rng.integers(-128, 128, (1, n, k)).astype(np.int8)
    q[0], w[0, 0], w[0, 1] = -128, -128, 127
    s, ws = np.ones(m, np.float32), np.full((1, n), 2.0 ** -12, np.float32)
    got = _run(tb, torch.zeros(m, k), 2, w, ws, None, False, q=(q, s))
    _check(got, *R.linear(q, s, w[0], ws[0], None, False), 2)
    assert got[0, 0] == float(np.float32(131071 * 16384)) * 2.0 ** -12


EXPERTS = [(1, 16, 16, 1), (10, 64, 64, 4), (48, 256, 128, 16), (40, 32, 64, 64), (300, 32, 64, 100), (2000, 64, 64, 7), (700, 100, 33, 65), (900, 512, 320, 5),
           (64, 96, 40, 4096), (5000, 16, 16, 513), (1500, 128, 256, 3)]


@pytest.mark.parametrize("kind", ["random", "outside", "one", "runs", "none"])
@pytest.mark.parametrize("m,k,n,e", EXPERTS)
def test_linear_by_expert(tb, m, k, n, e, kind):
    rng = np.random.default_rng([m, k, n, e])
    dtype = (0, 1, 2)[(m + e) % 3]
    offsets, _, _ = R.plan(_ids(m, 1, e, kind), e)
    x, w, ws, b = _case(rng, m, k, n, e, dtype)
    q, s = R.quantize(_np(x))
    got = _run(tb, x, dtype, w, ws, b, True, offsets=offsets)
    for i in range(e):
        r = slice(offsets[i], offsets[i + 1])
        if offsets[i] < offsets[i + 1]:
            _check(got[r], *R.linear(q[r], s[r], w[i], ws[i], b[i], True), dtype)
    assert (got[offsets[-1]:] == 77).all(), "rows behind the last expert's"


def test_offsets_that_are_none(tb):
    """Offsets that fall, lie outside the rows or start late: nothing outside the arrays is touched."""
    m, k, n, e = 200, 64, 48, 6
    rng = np.random.default_rng(3)
    x, w, ws, b = _case(rng, m, k, n, e, 0)
    for off in ([0, 500, 20, -7, 2 ** 31 - 1, -2 ** 31, 3], [-5, -4, -3, -2, -1, 0, 10], [300, 300, 300, 300, 300, 300, 300], [2 ** 31 - 1] * 7):
        _run(tb, x, 0, w, ws, b, False, offsets=np.array(off, np.int32))
    q, s = R.quantize(_np(x))
    got = _run(tb, x, 0, w, ws, b, False, offsets=np.array([30, 30, 60, 61, 61, 61, 150], np.int32))   # rows before the first expert's too
    assert (got[:30] == 77).all() and (got[150:] == 77).all()
    for i, (lo, hi) in {1: (30, 60), 2: (60, 61), 5: (61, 150)}.items():
        _check(got[lo:hi], *R.linear(q[lo:hi], s[lo:hi], w[i], ws[i], b[i], False), 0)


def test_no_rows(tb):
    x, w, ws, b = _case(np.random.default_rng(0), 0, 64, 64, 1, 0)
    assert _run(tb, x, 0, w, ws, b, False).shape == (0, 64)
    tb.quantize_rows_i8(0, 0, 0, 64, 64, 0, 64, 0)


def test_field_of_experts(tb, synthetic_model):
    """A run as a user makes it: the framework's own encoding of the samples, two block fields a sample, the density MLP's
    two layers by expert in 8 bits, the results blended; against the same steps in 64 bits.

    The hidden rows are rounded to f16 and to 8 bits in between, where a value next to a border may round either way: each
    such change is one step of its row, so hidden rows are compared first and the second layer is stated from the ones the
    framework made."""
    cfg, params, grid = synthetic_model
    tb.set_nerf_model(cfg, params)
    n, k, e = 3000, 2, 6
    rng = np.random.default_rng(11)
    pos = np.zeros((n, 7), np.float32)
    pos[:, :3] = rng.uniform(0, 1, (n, 3))
    ids = np.stack([(pos[:, 0] * 3).astype(int), 3 + (pos[:, 1] * 3).astype(int)], 1).astype(np.int32)   # blocks along x, along y
    ids[pos[:, 2] > 0.9] = -1                                                                         # outside
    dev = dict(device="cuda")
    coords = torch.from_numpy(pos).cuda()
    feat = torch.zeros(n, 32, dtype=torch.float16, **dev)
    tb.encode(coords.data_ptr(), 7, n, feat.data_ptr())
    layers = []
    for n_in, n_out in ((32, 64), (64, 16)):
        wf = torch.from_numpy((rng.normal(size=(e * n_out, n_in)) / np.sqrt(n_in)).astype(np.float32)).cuda()
        wq, ws = torch.zeros(e * n_out, n_in, dtype=torch.int8, **dev), torch.zeros(e * n_out, **dev)
        tb.quantize_rows_i8(wf.data_ptr(), 2, e * n_out, n_in, n_in, wq.data_ptr(), n_in, ws.data_ptr())
        layers.append((n_in, n_out, wq, ws))
    off, order, slot = (torch.zeros(m, dtype=torch.int32, **dev) for m in (e + 1, n * k, n * k))
    d_ids, weights = torch.from_numpy(ids).cuda(), torch.softmax(torch.randn(n, k, generator=torch.Generator().manual_seed(3)), 1).cuda()
    tb.expert_sort(d_ids.data_ptr(), n, k, e, off.data_ptr(), order.data_ptr(), slot.data_ptr())
    rows = torch.zeros(n * k, 32, dtype=torch.float16, **dev)
    tb.expert_dispatch(feat.data_ptr(), 0, 32, 32, order.data_ptr(), slot.data_ptr(), n, k, rows.data_ptr(), 32)
    outs = []
    for i, (n_in, n_out, wq, ws) in enumerate(layers):
        y = torch.zeros(n * k, n_out, dtype=torch.float16, **dev)
        size = tb.linear_i8_workspace(n * k, n_in, n_out, 0, e)
        buf = torch.zeros(max(16, size), dtype=torch.uint8, **dev)
        tb.linear_i8(rows.data_ptr() if i == 0 else outs[0].data_ptr(), 0, n * k, n_in, n_in, wq.data_ptr(), n_in, ws.data_ptr(), n_out, y.data_ptr(), 0, n_out,
                     relu=i == 0, d_offsets=off.data_ptr(), n_experts=e, d_workspace=buf.data_ptr(), workspace_bytes=size)
        outs.append(y)
    blend = torch.zeros(n, 16, dtype=torch.float16, **dev)
    tb.expert_combine(outs[1].data_ptr(), 0, 16, 16, weights.data_ptr(), slot.data_ptr(), n, k, blend.data_ptr(), 16)
    torch.cuda.synchronize()
    o, _, sl = R.plan(ids, e)
    assert np.array_equal(off.cpu().numpy(), o) and np.array_equal(slot.cpu().numpy().reshape(n, k), sl)
    src = rows.cpu().float().numpy()
    t = np.flatnonzero(sl[:, 1] >= 0)
    assert np.array_equal(src[sl[t, 1]], feat.cpu().float().numpy()[t]) and np.abs(src).max() > 0
    for (n_in, n_out, wq, ws), y, relu in zip(layers, outs, (True, False)):
        q, s = R.quantize(src)
        for i in range(e):
            r, c = slice(o[i], o[i + 1]), slice(i * n_out, (i + 1) * n_out)
            _check(y.cpu().double().numpy()[r], *R.linear(q[r], s[r], wq.cpu().numpy()[c], ws.cpu().numpy()[c], None, relu), 0)
        src = y.cpu().float().numpy()
    want, size = R.combine(src, weights.cpu().numpy(), sl)
    got = blend.cpu().double().numpy()
    assert (np.abs(got - want) <= 3 * 2.0 ** -24 * size * 1.01 + R.half_step(0) * (np.abs(want) + 2.0 ** -22 * size) + R.TINY[0]).all()
    assert (got[pos[:, 2] > 0.9] == 0).all()


@pytest.mark.parametrize("m,k,n,e", [(4, 1024, 256, 1), (3000, 64, 64, 5), (600, 512, 512, 2)])
def test_captured_and_replayed(tb, m, k, n, e):
    rng = np.random.default_rng(6)
    x, w, ws, b = _case(rng, m, k, n, e, 1)
    x, w, ws, b = x.cuda(), torch.from_numpy(w).cuda(), torch.from_numpy(ws).cuda(), torch.from_numpy(b).cuda()
    off = torch.from_numpy(np.linspace(0, m, e + 1).astype(np.int32)).cuda()
    y = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    size = tb.linear_i8_workspace(m, k, n, 1, e)
    buf = torch.zeros(max(16, size), dtype=torch.uint8, device="cuda")

    def step():
        tb.linear_i8(x.data_ptr(), 1, m, k, k, w.data_ptr(), k, ws.data_ptr(), n, y.data_ptr(), 1, n, d_bias=b.data_ptr(), d_offsets=off.data_ptr() if e > 1 else 0,
                     n_experts=e, d_workspace=buf.data_ptr(), workspace_bytes=size, stream=torch.cuda.current_stream().cuda_stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for it in range(4):
        x.copy_(torch.randn(m, k, device="cuda"))
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        y.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, y) and got.abs().max() > 0
