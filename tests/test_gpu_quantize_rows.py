"""Rows to 8 bits (sng_quantize_rows_i8) where x and q lie differently: each has a stride and a place of its own, which
decides between the kernel for aligned rows, the one for rows read at any place and the one for single elements.  q and the
scale are exact: compared for equality."""
import numpy as np
import pytest

import experts_ref as R
from test_gpu_experts import Guarded, _np, tb  # noqa: F401
from test_gpu_linear_i8 import _x

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# rows at any place, q aligned: 16, 256 (few rows and many) and 64 threads a row, and rows longer than a thread holds
SIZES = [(1, 16), (9, 48), (33, 64), (8, 1024), (9, 1040), (2050, 1040), (2050, 2048), (8, 4112), (9, 16400)]
PLACES = [(1, 0, 0, 0), (0, 1, 0, 0), (5, 3, 16, 0), (0, 0, 0, 16),           # q aligned, x not; both
          (0, 0, 1, 0), (8, 8, 0, 3), (0, 0, 4, 4), (3, 1, 2, 1)]            # q at any byte


@pytest.mark.parametrize("dtype", [0, 1, 2], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("ld_x,skew_x,ld_q,skew_q", PLACES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_x_and_q_at_places_of_their_own(tb, rows, cols, ld_x, skew_x, ld_q, skew_q, dtype):
    x = _x(np.random.default_rng([rows, cols, dtype]), rows, cols, dtype, "edge")   # rows with an infinity or NaN among them
    gx = Guarded((rows, cols), x.dtype, ld=cols + ld_x, skew=skew_x, fill=x)
    q, scale = Guarded((rows, cols), torch.int8, ld=cols + ld_q, skew=skew_q), Guarded((rows,), torch.float32)
    tb.quantize_rows_i8(gx.ptr, dtype, rows, cols, cols + ld_x, q.ptr, cols + ld_q, scale.ptr)
    want_q, want_s = R.quantize(_np(x))
    assert np.array_equal(scale.get(), want_s, equal_nan=True)
    assert np.array_equal(q.get().astype(np.int64), want_q)
