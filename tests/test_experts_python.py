"""The Python calls of the operators for a field of several experts, without a GPU: sizes that do not fit their C arguments are
refused.  ctypes keeps the low bits of such a number, so 2^32 rows would be none, and a negative workspace a large one."""
import pytest

PTR = 0x10000   # never followed: every call is refused on the host, a good one for its missing context


@pytest.fixture(scope="module")
def tb():
    from synerfgine_amd import Testbed, _lib
    t = object.__new__(Testbed)
    t._lib, t.ctx = _lib.load(), None
    return t


CALLS = {   # the arguments that are pointers lead where nothing is
    "expert_sort_workspace": dict(n=5, k=2, n_experts=8),
    "expert_sort": dict(d_experts=PTR, n=5, k=2, n_experts=8, d_offsets=PTR, d_order=PTR, d_slot=PTR, workspace_bytes=0),
    "expert_dispatch": dict(d_x=PTR, dtype=0, d=16, ld_x=16, d_order=PTR, d_slot=PTR, n=5, k=2, d_rows=PTR, ld_rows=16),
    "expert_dispatch_backward": dict(d_drows=PTR, dtype=0, d=16, ld_drows=16, d_slot=PTR, n=5, k=2, d_dx=PTR, ld_dx=16),
    "expert_combine": dict(d_rows=PTR, dtype=0, d=16, ld_rows=16, d_weights=0, d_slot=PTR, n=5, k=2, d_y=PTR, ld_y=16),
    "expert_combine_backward": dict(d_dy=PTR, ld_dy=16, d_rows=PTR, ld_rows=16, dtype=0, d=16, d_weights=0, d_slot=PTR, n=5, k=2, d_drows=PTR, ld_drows=16, d_dweights=PTR),
    "quantize_rows_i8": dict(d_x=PTR, dtype=0, rows=4, cols=16, ld_x=16, d_q=PTR, ld_q=16, d_scale=PTR),
    "linear_i8_workspace": dict(rows=4, n_in=16, n_out=8, x_dtype=0, n_experts=1),
    "linear_i8": dict(d_x=PTR, x_dtype=0, rows=4, n_in=16, ld_x=16, d_w=PTR, ld_w=16, d_w_scale=PTR, n_out=8, d_y=PTR, y_dtype=0, ld_y=8, n_experts=1, workspace_bytes=0),
}


@pytest.mark.parametrize("name", CALLS)
def test_sizes_that_do_not_fit(tb, name):
    from synerfgine_amd import SngError
    call, good = getattr(tb, name), CALLS[name]
    if name.endswith("workspace"):
        assert call(**good) == 0
    else:
        with pytest.raises(SngError, match="null context"):
            call(**good)
    for arg in good:
        if arg.startswith("d_"):
            continue
        past = 1 << (64 if arg == "workspace_bytes" else 32)
        for bad in (-1, past, past + good[arg]):
            with pytest.raises(SngError, match="whole number"):
                call(**dict(good, **{arg: bad}))


def test_sizes_of_numpys_types(tb):
    """Sizes that come from arrays, of types that do not mix"""
    import numpy as np
    assert tb.expert_sort_workspace(np.uint64(50000), np.int8(2), np.int64(8)) == tb.expert_sort_workspace(50000, 2, 8) > 0
    assert tb.linear_i8_workspace(np.int32(4096), np.uint64(4096), np.int64(4096), 0, np.uint8(1)) == tb.linear_i8_workspace(4096, 4096, 4096, 0, 1) > 0
