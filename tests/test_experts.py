"""The operators for a field of several experts, without a GPU: workspace sizes, and every call that has to be refused.

Arguments are checked before the context, so a call with good arguments and no context fails with "null context", and a
refused one names its own fault."""
import ctypes

import pytest

OK_PTR = 0x10000   # never followed: the call is refused on the host


@pytest.fixture(scope="module")
def lib():
    from synerfgine_amd import _lib
    return _lib.load()


def _refused(lib, rc, text):
    assert rc == -1
    message = lib.sng_last_error().decode()
    assert text in message, message


def test_sort_workspace(lib):
    size = ctypes.c_uint64(7)
    for n, k, e, want in [(0, 1, 1, 0), (1, 1, 4096, (1 + 1) * 4096 * 4), (16384, 1, 1024, 0), (8192, 2, 1024, 0), (16385, 1, 1024, (5 + 1) * 1024 * 4),
                          (16384, 1, 1025, (4 + 1) * 1025 * 4), (1 << 28, 1, 4096, (65536 + 1) * 4096 * 4)]:
        assert lib.sng_expert_sort_workspace(n, k, e, ctypes.byref(size)) == 0
        assert size.value == want, (n, k, e)


@pytest.mark.parametrize("n,k,e,text", [(1, 0, 4, "k must be at least 1"), (1, 1, 0, "n_experts"), (1, 1, 4097, "n_experts"), ((1 << 28) + 1, 1, 4, "2^28"),
                                        (1 << 31, 1 << 31, 4, "2^28")])
def test_sort_sizes_refused(lib, n, k, e, text):
    size = ctypes.c_uint64()
    _refused(lib, lib.sng_expert_sort_workspace(n, k, e, ctypes.byref(size)), text)
    _refused(lib, lib.sng_expert_sort(None, OK_PTR, n, k, e, OK_PTR, OK_PTR, OK_PTR, None, 0, None), text)


def test_sort_refusals(lib):
    call = lambda ids=OK_PTR, off=OK_PTR, order=OK_PTR, slot=OK_PTR, ws=None, size=0, n=100: lib.sng_expert_sort(None, ids, n, 2, 8, off, order, slot, ws, size, None)
    _refused(lib, call(), "null context")
    for name in ("ids", "off", "order", "slot"):
        _refused(lib, call(**{name: None}), "null argument")
        _refused(lib, call(**{name: OK_PTR + 2}), "aligned to 4")
    big = 100000   # needs a workspace
    need = ctypes.c_uint64()
    assert lib.sng_expert_sort_workspace(big, 2, 8, ctypes.byref(need)) == 0 and need.value > 0
    _refused(lib, call(n=big), "workspace")
    _refused(lib, call(n=big, ws=OK_PTR, size=need.value - 1), "workspace")
    _refused(lib, call(n=big, ws=OK_PTR + 1, size=need.value), "aligned to 4")
    _refused(lib, call(n=big, ws=OK_PTR, size=need.value), "null context")
    _refused(lib, lib.sng_expert_sort_workspace(1, 1, 1, None), "null argument")


def test_dispatch_refusals(lib):
    def call(x=OK_PTR, dtype=0, d=16, ld=16, order=OK_PTR, slot=OK_PTR, n=4, k=2, rows=OK_PTR, ld_rows=16):
        return lib.sng_expert_dispatch(None, x, dtype, d, ld, order, slot, n, k, rows, ld_rows, None)
    _refused(lib, call(), "null context")
    _refused(lib, call(dtype=3), "null context")   # 8-bit rows too
    for bad in (-1, 4):
        _refused(lib, call(dtype=bad), "dtype")
    _refused(lib, call(d=0), "row length")
    _refused(lib, call(d=(1 << 20) + 1, ld=1 << 21, ld_rows=1 << 21), "row length")
    _refused(lib, call(ld=15), "ld_x")
    _refused(lib, call(ld_rows=15), "ld_rows")
    _refused(lib, call(ld=(1 << 31) + 1), "ld_x")
    _refused(lib, call(k=0), "k must")
    _refused(lib, call(n=1 << 28, k=2), "2^28")
    for name in ("x", "order", "slot", "rows"):
        _refused(lib, call(**{name: None}), "null argument")
    _refused(lib, call(x=OK_PTR + 1), "aligned")
    _refused(lib, call(dtype=2, rows=OK_PTR + 2), "aligned")
    _refused(lib, call(order=OK_PTR + 2), "aligned")


def test_combine_refusals(lib):
    def call(rows=OK_PTR, dtype=0, d=16, ld=16, w=OK_PTR, slot=OK_PTR, n=4, k=2, y=OK_PTR, ld_y=16):
        return lib.sng_expert_combine(None, rows, dtype, d, ld, w, slot, n, k, y, ld_y, None)
    _refused(lib, call(), "null context")
    _refused(lib, call(w=None), "null context")   # ones
    _refused(lib, call(dtype=3), "dtype")
    _refused(lib, call(ld=15), "ld_rows")
    _refused(lib, call(ld_y=15), "ld_y")
    for name in ("rows", "slot", "y"):
        _refused(lib, call(**{name: None}), "null argument")
    _refused(lib, call(w=OK_PTR + 2), "aligned")
    _refused(lib, call(y=OK_PTR + 1), "aligned")


def test_combine_backward_refusals(lib):
    def call(dy=OK_PTR, ld_dy=16, rows=OK_PTR, ld=16, dtype=0, d=16, w=OK_PTR, slot=OK_PTR, n=4, k=2, drows=OK_PTR, ld_drows=16, dw=OK_PTR):
        return lib.sng_expert_combine_backward(None, dy, ld_dy, rows, ld, dtype, d, w, slot, n, k, drows, ld_drows, dw, None)
    _refused(lib, call(), "null context")
    _refused(lib, call(drows=None, ld_drows=0), "null context")
    _refused(lib, call(dw=None, rows=None, ld=0), "null context")
    _refused(lib, call(drows=None, dw=None), "neither gradient")
    _refused(lib, call(rows=None), "null argument")
    _refused(lib, call(dy=None), "null argument")
    _refused(lib, call(slot=None), "null argument")
    _refused(lib, call(ld_dy=15), "ld_dy")
    _refused(lib, call(ld=15), "ld_rows")
    _refused(lib, call(ld_drows=15), "ld_drows")
    _refused(lib, call(dw=OK_PTR + 1), "aligned")
    _refused(lib, call(dtype=3), "dtype")


def test_quantize_refusals(lib):
    def call(x=OK_PTR, dtype=0, rows=4, cols=16, ld=16, q=OK_PTR, ld_q=16, scale=OK_PTR):
        return lib.sng_quantize_rows_i8(None, x, dtype, rows, cols, ld, q, ld_q, scale, None)
    _refused(lib, call(), "null context")
    _refused(lib, call(q=OK_PTR + 1), "null context")
    _refused(lib, call(dtype=3), "dtype")
    _refused(lib, call(cols=0), "row length")
    _refused(lib, call(ld=15), "ld_x")
    _refused(lib, call(ld_q=15), "ld_q")
    _refused(lib, call(rows=(1 << 30) + 1), "rows")
    for name in ("x", "q", "scale"):
        _refused(lib, call(**{name: None}), "null argument")
    _refused(lib, call(scale=OK_PTR + 2), "aligned")


def _linear_args(**kw):
    from synerfgine_amd import _lib
    a = _lib.sng_linear_i8_args(d_x=OK_PTR, d_w=OK_PTR, d_w_scale=OK_PTR, d_y=OK_PTR, d_workspace=OK_PTR, workspace_bytes=1 << 40, ld_x=16, ld_w=16, ld_y=8, rows=4,
                                n_in=16, n_out=8, n_experts=1, x_dtype=0, y_dtype=0, relu=0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(), "null context"), (dict(d_bias=OK_PTR, relu=1), "null context"), (dict(x_dtype=3, d_x_scale=OK_PTR), "null context"),
    (dict(d_offsets=OK_PTR, n_experts=4096), "null context"), (dict(d_w=OK_PTR + 1, ld_w=17), "null context"),
    (dict(n_in=0), "n_in"), (dict(n_in=131072, ld_x=131072, ld_w=131072), "n_in"), (dict(n_out=0), "n_out"), (dict(n_out=(1 << 20) + 1, ld_y=1 << 21), "n_out"),
    (dict(rows=(1 << 30) + 1), "rows"), (dict(n_experts=0), "n_experts"), (dict(n_experts=4097, d_offsets=OK_PTR), "n_experts"),
    (dict(n_experts=2), "offsets"), (dict(x_dtype=4), "dtype"), (dict(x_dtype=-1), "dtype"), (dict(y_dtype=3), "dtype"), (dict(ld_x=15), "ld_x"),
    (dict(ld_w=15), "ld_w"), (dict(ld_y=7), "ld_y"), (dict(relu=2), "relu"), (dict(d_x=None), "null argument"), (dict(d_w=None), "null argument"),
    (dict(d_w_scale=None), "null argument"), (dict(d_y=None), "null argument"), (dict(x_dtype=3), "null argument"), (dict(d_y=OK_PTR + 1), "aligned"),
    (dict(d_x=OK_PTR + 1), "aligned"), (dict(d_bias=OK_PTR + 2), "aligned"), (dict(d_workspace=OK_PTR + 8), "aligned to 16"),
])
def test_linear_refusals(lib, change, text):
    _refused(lib, lib.sng_linear_i8(None, ctypes.byref(_linear_args(**change)), None), text)


def test_linear_workspace(lib):
    size = ctypes.c_uint64(9)
    assert lib.sng_linear_i8_workspace(1000, 500, 64, 3, 1, ctypes.byref(size)) == 0 and size.value == 0   # 8-bit rows need none
    assert lib.sng_linear_i8_workspace(0, 500, 64, 0, 1, ctypes.byref(size)) == 0 and size.value == 0
    assert lib.sng_linear_i8_workspace(4096, 4096, 4096, 0, 1, ctypes.byref(size)) == 0 and size.value >= 4096 * 4096
    need = size.value
    a = dict(rows=4096, n_in=4096, n_out=4096, ld_x=4096, ld_w=4096, ld_y=4096)
    _refused(lib, lib.sng_linear_i8(None, ctypes.byref(_linear_args(workspace_bytes=need, **a)), None), "null context")
    _refused(lib, lib.sng_linear_i8(None, ctypes.byref(_linear_args(workspace_bytes=need - 1, **a)), None), "workspace")
    _refused(lib, lib.sng_linear_i8(None, ctypes.byref(_linear_args(d_workspace=None, workspace_bytes=need, **a)), None), "workspace")
    _refused(lib, lib.sng_linear_i8_workspace(1, 16, 16, 0, 1, None), "null argument")
    _refused(lib, lib.sng_linear_i8(None, None, None), "null argument")
