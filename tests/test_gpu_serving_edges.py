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


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("down", [8, 16, 20])
def test_small_elements_of_q_that_meet_large_ones_of_k(q_type, kv_type, hd, down):
    """One element of q is 2^down times the others, and K holds zeros there and up to 2^14 elsewhere: the scores are sums of the small elements' products.
    A score's terms are off by 2^-21 of themselves for q's parts and hd 2^-24 for their sum."""
    from rustane_b200 import ops
    batch = Batch([300, 64, 1], [1, 2, 1], 2, hd, 16, kv_type, seed=9)
    batch.pool[:, 0] *= 2.0 ** 12
    batch.pool[:, 0, :, :, 5] = 0.0
    q = batch.normal(batch.rows, 6, hd, dtype=q_type) * 2.0 ** -down
    q[:, :, 5] = 1.0
    scale = 2.0 ** (down - 12) / 8
    out, lse = ops.paged_attention(batch.cache(), q, batch.row_start, 2, scale=scale, lse=True)
    want, want_lse, mass, _, worst = ref.attention(batch, q, scale)
    part = 2.0 ** -16 if q_type == kv_type == "bf16" else 2.0 ** -20
    moved = 2 * (hd * 2.0 ** -24 + 2.0 ** -21) * worst
    assert (np.abs(f64(out) - want) <= HALF_STEP[q_type] * np.abs(want) + (part + moved + 2.0 ** -20) * mass).all()
    np.testing.assert_allclose(f64(lse), want_lse, atol=(hd + 8) * 2.0 ** -24 * max(worst, 1) + 2.0 ** -20, rtol=2.0 ** -21)


def at_entry(batch, b, t):
    return int(batch.table[b, t // batch.page]), t % batch.page


def attend(batch, q, **more):
    from rustane_b200 import ops
    cache = batch.cache()
    out, lse = ops.paged_attention(cache, q, batch.row_start, max(batch.counts), lse=True, **more)
    assert int(cache.status) == 0
    return f64(out), f64(lse)


def near(out, want, mass, q_type, kv_type, hd, worst):
    """The result's rounding, and what scores (hd fp32 terms of at most `worst` together, 2^-21 for q's parts) and P's parts are off by."""
    part = 2.0 ** -16 if q_type == kv_type == "bf16" else 2.0 ** -20
    return np.abs(out - want) <= HALF_STEP[q_type] * np.abs(want) + (part + 2 * (hd * 2.0 ** -24 + 2.0 ** -21) * worst + 2.0 ** -20) * mass


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("heads", [2, 8, 24])
def test_infinities_and_nan_of_v_reach_the_rows_that_see_them(q_type, kv_type, hd, window, heads):
    """In single columns of V, with K finite: such a column of a row that sees the entry is +inf, -inf or NaN (both signs, NaN) exactly, in tiles that all rows see and
    in ones that only some do; its other columns are as ever, and rows that do not see the entry keep every bit."""
    lens, counts, inf, nan = [75, 200, 1000, 9000, 1], [3, 1, 2, 4, 1], float("inf"), float("nan")
    batch = Batch(lens, counts, 2, hd, 32, kv_type, seed=2)
    q = batch.normal(batch.rows, heads, hd, dtype=q_type)
    clean, clean_lse = attend(batch, q, window=window)
    want, _, mass, _, worst = ref.attention(batch, q, window=window)
    spoil = [(0, 74, 3, inf), (0, 10, 4, inf), (0, 33, 5, -inf), (0, 73, 5, inf), (0, 74, 6, nan), (1, 50, 1, -inf), (1, 170, 2, inf), (1, 199, 8, -inf), (1, 198, 8, -inf),
             (2, 500, 7, inf), (2, 999, 9, -inf), (2, 961, 10, inf), (2, 960, 11, -inf), (2, 990, 11, inf), (3, 4000, 12, inf), (3, 8999, 13, inf), (3, 8965, 14, -inf), (4, 0, 0, inf)]
    touched = np.zeros(batch.rows, dtype=bool)
    for b, t, col, value in spoil:
        page, off = at_entry(batch, b, t)
        batch.pool[page, 1, :, off, col] = value
        for j in range(counts[b]):
            row, last = batch.starts[b] + j, lens[b] - counts[b] + j
            if t <= last and (window == 0 or last - t < window):
                touched[row] = True
                was = want[row, :, col]
                want[row, :, col] = np.where(np.isfinite(was) | (was == value), value, nan)
    out, lse = attend(batch, q, window=window)
    np.testing.assert_array_equal(out[~touched], clean[~touched])
    odd = ~np.isfinite(want)
    np.testing.assert_array_equal(out[odd], want[odd])
    assert near(out[~odd], want[~odd], mass[~odd], q_type, kv_type, hd, worst).all()
    np.testing.assert_allclose(lse, clean_lse, rtol=2.0 ** -20, atol=2 * (hd + 8) * 2.0 ** -24 * max(worst, 1) + 2.0 ** -19)


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,counts", [(2, [1, 1, 1]), (8, [1, 1, 1]), (8, [3, 4, 2])])
def test_infinities_of_k(q_type, kv_type, hd, heads, counts):
    """An infinity of K that makes every score of its entry -inf leaves the rows, their log-sum-exp and the weights they hand on as if the entry had no
    part in them; one that makes a score +inf makes the rows that see it NaN, as inf - inf is."""
    lens = [75, 400, 9000]
    batch = Batch(lens, counts, 2, hd, 32, kv_type, seed=4, book=True)
    q = batch.normal(batch.rows, heads, hd, dtype=q_type)
    q[:, :, 11] = q[:, :, 11].abs() + 0.01  # (parts of either sign)
    _, _, _, _, worst = ref.attention(batch, q)
    for b, t in ((0, 5), (0, 74), (1, 200), (1, 396), (2, 0), (2, 5000)):
        page, off = at_entry(batch, b, t)
        batch.pool[page, 0, :, off, 11] = -float("inf")
    before = f64(batch.weight)
    out, lse = attend(batch, q, collect=True)
    want, want_lse, mass, got, _ = ref.attention(batch, q)
    assert np.isfinite(want).all() and np.isfinite(out).all() and near(out, want, mass, q_type, kv_type, hd, worst).all()
    np.testing.assert_allclose(lse, want_lse, atol=(hd + 8) * 2.0 ** -24 * max(worst, 1) + 2.0 ** -20, rtol=2.0 ** -21)
    moved = 2 * ((hd + 8) * 2.0 ** -24 + 2.0 ** -21) * max(worst, 1) + max(counts) * heads * 2.0 ** -24 + 2.0 ** -20
    for b, n in enumerate(lens):
        np.testing.assert_allclose(f64(batch.weight[b])[:, :n], before[b][:, :n] + got[b], rtol=moved, atol=1e-7)
    page, off = at_entry(batch, 1, 399)  # the newest entry: the last row alone sees it
    batch.pool[page, 0, :, off, 11] = float("inf")
    again, again_lse = attend(batch, q)
    last = batch.starts[2] - 1
    assert np.isnan(again[last]).all() and np.isnan(again_lse[last]).all()
    others = np.arange(batch.rows) != last
    np.testing.assert_array_equal(again[others], out[others])
    np.testing.assert_array_equal(again_lse[others], lse[others])


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_rows_of_q_that_are_not_finite(q_type, kv_type, value):
    """One element of one head's row: its scores are NaN (or of both infinities), and so is the row and its log-sum-exp; no other row changes a bit."""
    batch = Batch([70, 3000, 20], [3, 1, 20], 2, 64, 16, kv_type, seed=6)
    q = batch.normal(batch.rows, 8, 64, dtype=q_type)
    clean, clean_lse = attend(batch, q)
    hit = [(1, 3), (3, 0), (3, 7), (23, 5)]
    for row, head in hit:
        q[row, head, 17] = value
    out, lse = attend(batch, q)
    mask = np.zeros(lse.shape, dtype=bool)
    mask[tuple(zip(*hit))] = True
    assert np.isnan(out[mask]).all() and np.isnan(lse[mask]).all()
    np.testing.assert_array_equal(out[~mask], clean[~mask])
    np.testing.assert_array_equal(lse[~mask], clean_lse[~mask])


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("page", [7, 16])
def test_rows_of_nothing_but_infinite_scores(q_type, kv_type, page):
    """Every score of a row -inf: no entry has weight, the row is zeros and -inf, its neighbours are not touched."""
    batch = Batch([40, 40], [2, 2], 1, 64, page, kv_type, seed=5)
    q = batch.normal(4, 3, 64, dtype=q_type)
    clean, clean_lse = attend(batch, q)
    for t in range(40):
        p, off = at_entry(batch, 0, t)
        batch.pool[p, 0, :, off, 0] = -float("inf")
    q[:2, :, 0] = q[:2, :, 0].abs() + 0.01
    out, lse = attend(batch, q)
    assert (out[:2] == 0).all() and np.isneginf(lse[:2]).all()
    np.testing.assert_array_equal(out[2:], clean[2:])
    np.testing.assert_array_equal(lse[2:], clean_lse[2:])


# ------------------------------------------------------------------------------------------------ verification
def verify_inputs(counts, vocab, dtype, seed, near=0.7):
    import torch
    g = torch.Generator("cpu").manual_seed(seed)
    rows = sum(counts)
    target = torch.randn(rows, vocab, generator=g) * 2
    draft = target + near * torch.randn(rows, vocab, generator=g)
    tokens = torch.zeros(rows, dtype=torch.int32)
    tokens[1:] = draft[:-1].argmax(1).int()
    starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32)
    kind = ref.torch_dtype(dtype)
    return dict(target=target.to(kind), draft=draft.to(kind), tokens=tokens, starts=starts, u=torch.rand(rows, generator=g), d=torch.rand(len(counts), generator=g), most=max(counts + [1]))


def verify(x, temperature, with_draft=True, **more):
    """(accepted, out, status) as lists and a number."""
    import torch

    from rustane_b200 import ops
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    accepted, out = ops.verify_drafts(x["target"].cuda(), x["tokens"].cuda(), x["starts"].cuda(), x["most"], x["u"].cuda(), x["d"].cuda(),
                                      draft=x["draft"].cuda() if with_draft else None, temperature=temperature, status=status, **more)
    return accepted.tolist(), out.tolist(), int(status)


def verify64(x, temperature, with_draft=True):
    accepted, out = ref.verify(f64(x["target"]), f64(x["draft"]) if with_draft else None, x["tokens"].numpy(), f64(x["u"]), f64(x["d"]), x["starts"].numpy(), temperature)
    return accepted.tolist(), out.tolist()


@pytest.mark.parametrize("dtype,level", [("f32", -3.4028234663852886e38), ("f32", -1e30), ("f32", 1e30), ("f32", -65536.0), ("bf16", -3.3895313892515355e38), ("bf16", 1e25), ("f16", -65504.0)])
@pytest.mark.parametrize("temperature", [0.7, 0.9, 1.0, 1e-6, 1e6])
@pytest.mark.parametrize("with_draft", [True, False])
def test_rows_of_one_large_logit(dtype, level, temperature, with_draft):
    """Rows masked altogether with their type's lowest value, or shifted far off: every token as likely as the next, whatever the
    size of what they share.  Draws are 1/2 of a token's share off every border, 2^-15 of the whole, where 64-bit sums are off by 2^-45."""
    import torch
    vocab, counts = 8192, [3, 1, 4, 1]
    x = verify_inputs(counts, vocab, dtype, 5)
    x["target"][:] = level
    x["target"][7] = verify_inputs(counts, vocab, dtype, 5)["target"][7]
    x["draft"][:] = level / 2
    g = torch.Generator("cpu").manual_seed(1)
    x["d"] = ((torch.randint(0, vocab, (4,), generator=g) + 0.5) / vocab).float()
    x["u"][:] = torch.tensor([0.5, 0.5, 0, 0, 0.5, 0.999, 0.5, 0, 0])
    got, out, status = verify(x, temperature, with_draft)
    want = verify64(x, temperature, with_draft)
    assert (got, out) == want and status == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_draft_rows_with_no_draft_behind_them_are_not_read(dtype):
    """A sequence's last row of draft logits holds NaN, infinities or the largest values: nothing changes.  (That the last one of a batch may not even be
    memory cannot be tested here; the kernel asks for a draft row only once it knows that a draft is behind it.)"""
    counts = [4, 1, 3, 1, 6]
    x = verify_inputs(counts, 5003, dtype, 3)
    want = verify(x, 0.9)
    assert want[:2] == verify64(x, 0.9)
    for value in (float("nan"), float("inf"), -float("inf"), 6e4):
        for end in x["starts"][1:].tolist():
            x["draft"][end - 1] = value
        assert verify(x, 0.9) == want


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_sequences_that_are_left_out_say_so(temperature):
    """accepted -1 and tokens -1, without a look at the status; rows behind the batch keep what they held."""
    import torch

    from rustane_b200 import _ffi, ops
    x = verify_inputs([3, 2, 4, 3], 700, "bf16", 12)
    draft = temperature > 0
    want_n, want = verify64(x, temperature, draft)
    target, drafts, tokens, u, d = (x[k].cuda() for k in ("target", "draft", "tokens", "u", "d"))
    # row_start, the most rows, which sequences fit, the rows of the batch that none of them has
    for starts, most, fits, free in (([0, 3, -1, 9, 12], 4, [0, 3], range(3, 9)), ([0, 3, 5, 13, 13], 4, [0, 1], range(5, 12)), ([0, 3, 5, 9, 12], 3, [0, 1, 3], range(5, 9)),
                                     ([2 ** 31 - 1, 3, 5, 9, 9], 4, [1, 2, 3], range(0, 3)), ([-2 ** 31, 3, 5, 2 ** 31 - 1, 12], 4, [1], list(range(0, 3)) + list(range(5, 12)))):
        row_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        got_n, got = ops.verify_drafts(target, tokens, row_start, most, u, d, draft=drafts if draft else None, temperature=temperature)
        end = min(starts[-1], 12)
        for b in range(4):
            if b in fits and starts[b] < starts[b + 1]:
                r0, r1 = starts[b], starts[b + 1]
                assert int(got_n[b]) == want_n[b] and got[r0:r1].tolist() == want[r0:r1], (starts, b)
            else:
                assert int(got_n[b]) == (0 if b in fits else -1), (starts, b)
        assert all(int(got[r]) == -1 for r in free if r < end), starts
        # the same through the library, into memory that holds something
        out, accepted, status = torch.full_like(tokens, 77), torch.full_like(got_n, 77), torch.zeros(1, dtype=torch.int32, device="cuda")
        ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
        assert _ffi.lib.cd_verify_drafts(0, 2, 4, 12, most, 700, target.data_ptr(), 0, drafts.data_ptr(), 0, tokens.data_ptr(), row_start.data_ptr(), u.data_ptr(), d.data_ptr(),
                                         temperature, accepted.data_ptr(), out.data_ptr(), status.data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
        assert int(status) == 1 and torch.equal(accepted, got_n) and torch.equal(out[:end], got[:end]) and bool((out[end:] == 77).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,temperature", [(40, 1.0), (5003, 0.7), (32000, 1.0), (128000, 1.3)])
@pytest.mark.parametrize("with_draft", [True, False])
def test_drafts_on_the_border_of_acceptance(dtype, vocab, temperature, with_draft):
    """Uniform numbers that are the fp32 neighbours of p(x) / q(x): one below stays, one not below does not.  They lie up to 2^-24 of themselves off the border,
    which row sums in fp32 cannot tell.  (Those nearer than 2^-38, where the 64-bit forms themselves may differ, are moved a step away.)"""
    import torch
    counts = [1, 9, 25, 5, 2, 40]
    x = verify_inputs(counts, vocab, dtype, 7, near=0.4)
    p, q = (torch.log_softmax(x[k].double() / temperature, 1) for k in ("target", "draft"))
    g = torch.Generator("cpu").manual_seed(2)
    starts = x["starts"].tolist()
    for b, n in enumerate(counts):
        stop = int(torch.randint(0, n, (1,), generator=g))  # the draft of this sequence that does not stay (its last row has none)
        for j in range(n - 1):
            r = starts[b] + j
            # a token that q gives more than p, so that the border is below 1 (any token will do without q)
            x["tokens"][r + 1] = int((q[r] - p[r]).topk(3).indices[int(torch.randint(0, 3, (1,), generator=g))]) if with_draft else int(torch.randint(0, vocab, (1,), generator=g))
            t = int(x["tokens"][r + 1])
            border = float(torch.exp(p[r, t] - (q[r, t] if with_draft else 0.0)))
            u = np.float32(border)
            below = u if float(u) < border * (1 - 2.0 ** -38) else np.nextafter(u, np.float32(0))
            above = u if float(u) > border * (1 + 2.0 ** -38) else np.nextafter(u, np.float32(2))
            x["u"][r] = float(above if j == stop else below)
    got, out, status = verify(x, temperature, with_draft)
    want_n, want = verify64(x, temperature, with_draft)
    assert got == want_n and out == want and status == 0
    assert max(want_n) > 3  # (several borders in one sequence)


# ------------------------------------------------------------------------------------------------ eviction
@pytest.mark.parametrize("length,resident", [(300, True), (9001, True), (360000, False)])
@pytest.mark.parametrize("sinks,recent", [(0, 0), (3, 0), (0, 2), (3, 2)])
def test_entries_at_positions_below_zero_are_below_any_sinks(length, resident, sinks, recent):
    """A position below `sinks` stays, and a negative one is below 0: with no sinks and none recent too, however the keys are held."""
    import torch

    from rustane_b200 import ops
    batch = Batch([length, length - 7], [0, 0], 1, 64, 64, "bf16", seed=length, book=True, values=length < 10 ** 5)
    keep = length // 2
    far = torch.randperm(length - 20, generator=batch.g)[:9]
    batch.position[:, :, far.cuda()] = -1 - torch.arange(9, dtype=torch.int32, device="cuda")
    batch.weight[:, :, far.cuda()] = 0.0  # the lightest: only their position keeps them
    weight, position = f64(batch.weight), batch.position.cpu().numpy()
    lens, _, new = ops.cache_evict(batch.cache(), keep, sinks=sinks, recent=recent)
    assert lens.tolist() == [keep, keep]
    for b, n in enumerate(batch.lens):
        w, p, got = weight[b, 0, :n], position[b, 0, :n], new[b, 0, :keep].cpu().numpy()
        safe = (p < sinks) | (p > int(p.max()) - recent)
        order = np.lexsort((np.arange(n), np.where(safe, -np.inf, -w)))
        np.testing.assert_array_equal(np.sort(got), np.sort(p[order[:keep]]))


# ------------------------------------------------------------------------------------------------ a step as the documents show it
def test_the_step_in_the_readme():
    """Its lines as they stand: they run, and the cache it leaves is the one that was brought down (lengths, and what the next step attends over)."""
    import os
    import re

    import torch

    from rustane_b200 import ops
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")).read()
    block = next(b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "PagedCache(" in b)
    lens0, counts, kv, heads, vocab = [3000, 5, 2049], [2, 1, 3], 2, 4, 900
    batch = Batch(lens0, counts, kv, 128, 64, "bf16", seed=7, book=True)
    x = verify_inputs(counts, vocab, "bf16", 7)
    fused = batch.normal(batch.rows, heads + 2 * kv, 128, dtype="bf16")
    at = torch.cat([torch.arange(n - c, n) for n, c in zip(lens0, counts)]).to(torch.int32).cuda()
    names = dict(pool=batch.pool, page_table=batch.table, lens=batch.tlens, weight=batch.weight, position=batch.position, q=fused[:, :heads], k=fused[:, heads:heads + kv],
                 v=fused[:, heads + kv:], positions=at, row_start=batch.row_start, max_rows=3, target_logits=x["target"].cuda(), draft_logits=x["draft"].cuda(), tokens=x["tokens"].cuda(),
                 uniforms=x["u"].cuda(), draws=x["d"].cuda())
    exec(block, names)
    cache = names["cache"]
    kept = [min(n, 2048) for n in lens0]
    assert cache.lens.tolist() == kept and names["accepted"].tolist() == verify64(x, 1.0)[0]
    q = batch.normal(3, heads, 128, dtype="bf16")
    one = torch.arange(4, dtype=torch.int32, device="cuda")
    batch.lens, batch.counts, batch.starts, batch.row_start, batch.rows = kept, [1, 1, 1], np.arange(4), one, 3
    want, _, mass, _, worst = ref.attention(batch, q)  # (the pool as it is now)
    assert near(f64(ops.paged_attention(cache, q, one, 1)), want, mass, "bf16", "bf16", 128, worst).all()


# ------------------------------------------------------------------------------------------------ the most that calls take, and calls beside others
@pytest.mark.parametrize("q_type,kv_type", TYPES)
def test_as_many_sequences_as_there_may_be(q_type, kv_type):
    """4096 sequences of 0 to 9 entries and 0 to 4 rows: attention, append and eviction."""
    import torch

    from rustane_b200 import ops
    rng = np.random.default_rng(4)
    lens, counts = [int(n) for n in rng.integers(0, 10, 4096)], [int(n) for n in rng.integers(0, 5, 4096)]
    batch = Batch(lens, counts, 1, 64, 4, kv_type, seed=6, book=True)
    q = batch.normal(batch.rows, 5, 64, dtype=q_type)
    out, lse = attend(batch, q, collect=False)
    want, want_lse, mass, _, worst = ref.attention(batch, q)
    seen = np.isfinite(want_lse)
    assert (np.isneginf(lse) == ~seen).all() and near(out, want, mass, q_type, kv_type, 64, worst).all()
    k = batch.normal(batch.rows, 1, 64, dtype=q_type)
    at, cache = torch.arange(batch.rows, dtype=torch.int32, device="cuda"), batch.cache()
    before = batch.pool.clone()
    turned = ops.rope_append(cache, ops.Rope(64), q, k, k, at, batch.row_start)
    freq, magnitude = ref.frequencies(64, 10000.0, None, 1.0, 1)
    angle = np.abs(f64(turned) - ref.rotate(f64(q), np.arange(batch.rows), freq, magnitude, "half"))
    size = np.abs(f64(q)) + np.abs(np.roll(f64(q), 32, -1))
    assert (angle <= HALF_STEP[q_type] * size * 1.5 + 10 * 2.0 ** -24 * size + 2.0 ** -25).all()
    short = any(c > n for n, c in zip(lens, counts))
    assert int(cache.status) == (1 if short else 0)  # rows that have no entry
    for b in rng.integers(0, 4096, 200):
        n, m = lens[b], counts[b]
        r0, fit = int(batch.starts[b]), min(m, n)
        assert np.array_equal(batch.entries(b, 1)[0, n - fit:], f64(k.to(batch.pool.dtype))[r0 + m - fit:r0 + m, 0])
        assert np.array_equal(batch.entries(b, 1)[0, :n - fit], batch.entries(b, 1, before)[0, :n - fit])
    weight, position = f64(batch.weight), batch.position.cpu().numpy()
    lens1, _, new = ops.cache_evict(batch.cache(), 6, sinks=1, recent=2)
    assert lens1.tolist() == [min(n, 6) for n in lens]
    new = new.cpu().numpy()
    for b in rng.integers(0, 4096, 300):
        moved = position[b, 0].copy()
        for to, of in ref.evict(weight[b, 0], position[b, 0], lens[b], 6, 1, 2):
            moved[to] = position[b, 0, of]
        assert np.array_equal(new[b, 0], moved)


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("page", [1000, 4096, 65536])
def test_pages_longer_than_the_sequences(q_type, kv_type, page):
    batch = Batch([page + 3, 70, page], [1, 3, 2], 2, 64, page, kv_type, seed=1)
    q = batch.normal(batch.rows, 4, 64, dtype=q_type)
    out, _ = attend(batch, q)
    want, _, mass, _, worst = ref.attention(batch, q)
    assert near(out, want, mass, q_type, kv_type, 64, worst).all()


@pytest.mark.parametrize("q_type,kv_type", TYPES)
def test_the_same_bits_beside_other_work_and_in_place(q_type, kv_type):
    """Units of one, two and four row warps, cut over several CTAs: call after call while another stream keeps the GPU busy, and into q itself."""
    import torch

    from rustane_b200 import ops
    lens, counts = [9000, 5011, 64, 12000, 700, 1], [6, 2, 1, 8, 4, 1]
    batch = Batch(lens, counts, 2, 64, 16, kv_type, seed=8, book=True)
    q, cache = batch.normal(batch.rows, 16, 64, dtype=q_type), batch.cache()
    first, lse = ops.paged_attention(cache, q, batch.row_start, 8, lse=True)
    weight = batch.weight.clone()
    collected, _ = ops.paged_attention(cache, q, batch.row_start, 8, lse=True, collect=True)
    got = batch.weight.clone()
    noise, side = torch.randn(1 << 26, device="cuda"), torch.cuda.Stream()
    for i in range(40):
        with torch.cuda.stream(side):
            noise.mul_(1.0001)
        batch.weight.copy_(weight)
        again, again_lse = ops.paged_attention(cache, q, batch.row_start, 8, lse=True, collect=i % 2 == 1)
        assert torch.equal(again, first) and torch.equal(again_lse, lse)
        assert torch.equal(batch.weight, got if i % 2 else weight)
    assert torch.equal(collected, first)
    assert torch.equal(ops.paged_attention(cache, q, batch.row_start, 8), first)
    mine = q.clone()
    assert ops.paged_attention(cache, mine, batch.row_start, 8, out=mine) is mine and torch.equal(mine, first)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("temperature,with_draft", [(0.0, False), (0.8, True), (0.8, False)])
def test_as_large_a_vocabulary_as_there_may_be(dtype, temperature, with_draft):
    x = verify_inputs([2, 1], 1 << 22, dtype, 3)
    got, out, status = verify(x, temperature, with_draft)
    assert (got, out) == verify64(x, temperature, with_draft) and status == 0
