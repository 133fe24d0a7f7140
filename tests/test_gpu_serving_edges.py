"""Operators of a serving step at the edges of what their calls allow, against plain 64-bit forms."""
import numpy as np
import pytest

import serving_ref as ref
from serving_ref import Batch, f64

pytestmark = pytest.mark.gpu

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TYPES = [("bf16", "bf16"), ("f16", "f16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "f32")]


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 60])
def test_a_window_wider_than_every_sequence_is_none(q_type, kv_type, window):
    """More rows than entries among them: the first row's window begins 2^31 entries ahead of the sequence."""
    from rustane_b200 import ops
    batch = Batch([1, 0, 300, 2, 70], [4, 2, 3, 64, 1], 2, 64, 16, kv_type, seed=2, book=True)
    q = batch.normal(batch.rows, 4, 64, dtype=q_type)
    cache = batch.cache()
    want, want_lse = ops.paged_attention(cache, q, batch.row_start, 64, lse=True)
    out, lse = ops.paged_attention(cache, q, batch.row_start, 64, window=window, lse=True, collect=True)
    np.testing.assert_array_equal(f64(out), f64(want))
    np.testing.assert_array_equal(f64(lse), f64(want_lse))
    assert np.isneginf(f64(lse[:3])).all() and (f64(out[:3]) == 0).all() and np.isfinite(f64(lse[3])).all()  # three of four rows ahead of the one entry
    assert int(cache.status) == 0
