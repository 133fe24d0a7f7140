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


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("pairs", [1, 40])
def test_probabilities_of_terms_that_cancel(q_type, kv_type, pairs):
    """V is +1 and -1 in turn, and the scores (exact: one product each) differ by i / 1024 a sequence: what is left of the sum is small, so that a probability
    rounded to 11 bits would show.  Allowed: the result's rounding, and of the terms' sum 2^-20 (fp32 sums of up to 80 terms and their
    exponentials: 2^-22 each for 2^x and the score's scaling, 2^-24 a sum), with bf16 rows over bf16 2^-16 for P in two parts."""
    from rustane_b200 import ops
    n = 64
    batch = Batch([2 * pairs] * n, [1] * n, 1, 64, 16, kv_type, seed=1, values=False)
    for b in range(n):
        for t in range(2 * pairs):
            at = batch.pool[int(batch.table[b, t // 16]), :, 0, t % 16]
            at[0, 0] = (t % 2) * (b + 1) / 1024.0
            at[1] = 1.0 - 2.0 * (t % 2)
    q = batch.normal(n, 1, 64, dtype=q_type).zero_()
    q[:, :, 0] = 1.0
    out = ops.paged_attention(batch.cache(), q, batch.row_start, 1, scale=1.0)
    want, _, mass, _, _ = ref.attention(batch, q, 1.0)
    part = 2.0 ** -16 if q_type == "bf16" else 2.0 ** -20
    assert (np.abs(f64(out) - want) <= HALF_STEP[q_type] * np.abs(want) + part * mass).all(), np.abs(f64(out) - want).max()


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_past_the_digits_of_fp32(q_type, kv_type, hd):
    """Finite scores of some 2^32 (one product each, a scale of 2^7), where a unit of the last place is hundreds: the largest takes all, two equal ones half each.
    The result is an entry of V or the mean of two, off by its rounding and that of P's parts (2^-16 and less)."""
    import torch

    from rustane_b200 import ops
    lens = [300, 64, 33, 5000]
    batch = Batch(lens, [1, 2, 1, 1], 2, hd, 16, kv_type, seed=3)
    heads, rng = 8, np.random.default_rng(hd)
    for b, n in enumerate(lens):
        pages = batch.table[b, :-(-n // 16)].long()
        k = torch.zeros(len(pages), 16, hd, device="cuda").flatten(0, 1)
        k[:n, 0] = torch.from_numpy(rng.uniform(1000, 2000, n).round().astype(np.float32)).cuda()  # (bf16 keeps fewer of them apart)
        at = int(k[:n - 3, 0].argmax())
        k[(at + n // 2) % (n - 3), 0] = k[at, 0]
        batch.pool[pages, 0] = k.view(len(pages), 1, 16, hd).to(batch.pool.dtype).expand(-1, 2, -1, -1)
    q = batch.normal(batch.rows, heads, hd, dtype=q_type).zero_()
    q[:, :, 0] = 2.0 ** 14 * (1.0 + torch.arange(heads, device="cuda") / 64.0)  # exact in every type
    out, lse = ops.paged_attention(batch.cache(), q, batch.row_start, 2, scale=128.0, lse=True)
    want, want_lse, mass, _, _ = ref.attention(batch, q, 128.0)
    assert want_lse.min() > 2.0 ** 30
    assert (np.abs(f64(out) - want) <= HALF_STEP[q_type] * np.abs(want) + (2.0 ** -16 + 2.0 ** -20) * mass).all(), np.abs(f64(out) - want).max()
    np.testing.assert_allclose(f64(lse), want_lse, rtol=2.0 ** -21)
