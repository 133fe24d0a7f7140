"""Operators of a serving step (rope_append, paged_attention, cache_evict, verify_drafts) against plain 64-bit forms."""
import numpy as np
import pytest

import serving_ref as ref
from serving_ref import Batch, f64

pytestmark = pytest.mark.gpu

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


# ------------------------------------------------------------------------------------------------ attention
def attention_tolerance(out, mass, q_type, kv_type, hd, worst):
    """The result's rounding, plus what reaches it of the scores and probabilities.  A score is a sum of hd fp32 terms (each within 2^-24 of
    its size `worst`, q's parts exact to 2^-22 of it), and moves p by that much either way; p is 16 bits with an fp16 pool and q
    (2^-11), two or more parts otherwise (2^-16)."""
    part = 2.0 ** -11 if q_type == kv_type == "f16" else 2.0 ** -16 if q_type == kv_type == "bf16" else 2.0 ** -21
    moved = 2 * (hd * 2.0 ** -24 + 2.0 ** -21) * worst
    return HALF_STEP[q_type] * np.abs(out) + (part + moved + 2.0 ** -20) * mass + 1e-30


def check_attention(batch, heads, q_type, window=0, scale=None, collect=False, q=None):
    from rustane_b200 import ops
    q = batch.normal(batch.rows, heads, batch.hd, dtype=q_type) if q is None else q
    before = None if batch.weight is None else f64(batch.weight)
    cache = batch.cache()
    out, lse = ops.paged_attention(cache, q, batch.row_start, max(batch.counts + [1]), scale=scale, window=window, collect=collect, lse=True)
    want, want_lse, mass, got, worst = ref.attention(batch, q, scale, window)
    off = np.abs(f64(out) - want)
    tol = attention_tolerance(want, mass, q_type, batch.kv, batch.hd, worst)
    assert np.isfinite(f64(out)).all()
    assert (off <= tol).all(), "off by %g where %g is allowed" % (off.max(), tol.flat[(off - tol).argmax()])
    seen = np.isfinite(want_lse)
    assert (np.isneginf(f64(lse)) == ~seen).all()
    np.testing.assert_allclose(f64(lse)[seen], want_lse[seen], atol=(batch.hd + 8) * 2.0 ** -24 * max(worst, 1) + 2.0 ** -20, rtol=2.0 ** -21)
    if collect:
        moved = 2 * ((batch.hd + 8) * 2.0 ** -24 + 2.0 ** -21) * max(worst, 1) + max(batch.counts) * heads * 2.0 ** -24 + 2.0 ** -20
        for b, n in enumerate(batch.lens):
            now = f64(batch.weight[b])
            np.testing.assert_allclose(now[:, :n], before[b][:, :n] + got[b], rtol=moved, atol=1e-7)
            np.testing.assert_array_equal(now[:, n:], before[b][:, n:])
    assert int(cache.status) == 0
    return out


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("f32", "f16"), ("f32", "bf16"), ("f32", "f32")]


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (6, 2), (8, 1), (40, 2)])
def test_attention_types_and_heads(q_type, kv_type, hd, heads, kv_heads):
    check_attention(Batch([1, 70, 333], [1, 1, 1], kv_heads, hd, 64, kv_type, seed=heads + hd), heads, q_type)


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 100])
def test_attention_pages(q_type, kv_type, page):
    check_attention(Batch([page, page + 1, 2 * page - 1, 5 * page + 3, 130], [1, 1, 1, 1, 1], 2, 128, page, kv_type, seed=page), 8, q_type)


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("heads,kv_heads,counts", [(4, 4, [3, 1, 0, 2]), (8, 2, [5, 1, 7, 2]), (8, 1, [8, 8, 3, 9]), (3, 1, [33, 1, 2, 20]), (16, 2, [1, 4, 6, 17])])
def test_attention_several_rows(q_type, kv_type, heads, kv_heads, counts):
    check_attention(Batch([40, 65, 129, 200], counts, kv_heads, 64, 16, kv_type, seed=7), heads, q_type)


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
def test_attention_window(q_type, kv_type, window):
    check_attention(Batch([1, 64, 300, 257], [1, 4, 3, 1], 2, 128, 24, kv_type, seed=window), 4, q_type, window=window)


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [0, 50])
def test_attention_collects_weights(q_type, kv_type, hd, window):
    check_attention(Batch([1, 64, 700, 90], [1, 2, 1, 5], 2, hd, 16, kv_type, seed=3, book=True), 6, q_type, window=window, collect=True)


@pytest.mark.parametrize("q_type,kv_type", TYPES)
def test_attention_long_sequences_are_cut_and_joined(q_type, kv_type):
    check_attention(Batch([20011, 3, 9000], [1, 1, 2], 1, 128, 64, kv_type, seed=5), 4, q_type)


@pytest.mark.parametrize("q_type,kv_type", TYPES)
def test_attention_rows_that_see_nothing(q_type, kv_type):
    """No entries, fewer entries than rows, no rows; rows behind the last sequence stay as they were."""
    import torch

    from rustane_b200 import ops
    batch = Batch([0, 2, 50, 0], [1, 4, 0, 2], 2, 64, 16, kv_type, seed=1)
    q = batch.normal(batch.rows + 3, 4, 64, dtype=q_type)
    out = torch.full_like(q, 7.0)
    got, lse = ops.paged_attention(batch.cache(), q, batch.row_start, 4, lse=True, out=out)
    assert got is out
    want, want_lse, mass, _, worst = ref.attention(batch, q[:batch.rows])
    n = batch.rows
    assert (np.abs(f64(out[:n]) - want) <= attention_tolerance(want, mass, q_type, kv_type, 64, max(worst, 1))).all()
    assert (f64(out[:3]) == 0).all() and np.isneginf(f64(lse[:3])).all()  # row 0; the first two of the four rows over two entries
    assert (f64(out[n - 2:n]) == 0).all()
    assert (f64(out[n:]) == 7.0).all()


@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_masked_places_do_not_reach_a_row(q_type, kv_type, value):
    """NaN and infinities behind the last entry, left of the window, and in entries that only later rows see."""
    batch = Batch([75, 200], [3, 1], 2, 128, 32, kv_type, seed=2)
    q = batch.normal(batch.rows, 4, 128, dtype=q_type)
    from rustane_b200 import ops

    def run(window):
        return f64(ops.paged_attention(batch.cache(), q, batch.row_start, 3, window=window))

    clean, clean_w = run(0), run(40)
    spoiled = batch.pool.clone()
    for b, n in enumerate(batch.lens):  # behind the last entry
        page = int(batch.table[b, (n - 1) // 32])
        spoiled[page, :, :, (n - 1) % 32 + 1:] = value
    used = set(batch.table[0, :3].tolist()) | set(batch.table[1, :7].tolist())
    for page in set(range(batch.pool.shape[0])) - used:
        spoiled[page] = value
    keep, batch.pool = batch.pool, spoiled
    np.testing.assert_array_equal(run(0), clean)
    last = spoiled.clone()  # the newest entry of sequence 0: rows 0 and 1 do not see it
    last[int(batch.table[0, 2]), :, :, 74 % 32] = value
    batch.pool = last
    got = run(0)
    np.testing.assert_array_equal(got[:2], clean[:2])
    np.testing.assert_array_equal(got[3:], clean[3:])
    assert not np.isfinite(got[2]).any() or (kv_type and np.isinf(value))
    old = spoiled.clone()  # entry 150 of sequence 1 is left of a window of 40 at 199; entry 33 of sequence 0 left of row 0's (72 - 40)
    old[int(batch.table[1, 150 // 32]), :, :, 150 % 32] = value
    old[int(batch.table[0, 1]), :, :, 32 % 32] = value
    batch.pool = old
    np.testing.assert_array_equal(run(40), clean_w)
    batch.pool = keep


@pytest.mark.parametrize("q_type,kv_type", [("bf16", "bf16"), ("f32", "f32")])
def test_attention_strides(q_type, kv_type):
    """q as a slice of a fused projection, a page table with longer rows."""
    import torch
    batch = Batch([33, 90], [2, 1], 2, 64, 16, kv_type, seed=4)
    fused = batch.normal(batch.rows, 12 * 64, dtype=q_type)
    q = fused[:, 128:128 + 8 * 64].unflatten(1, (8, 64))
    wide = torch.full((2, batch.table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :batch.table.shape[1]] = batch.table
    batch.table = wide[:, :batch.table.shape[1]]
    a = check_attention(batch, 8, q_type, q=q)
    b = check_attention(batch, 8, q_type, q=q.contiguous())
    assert torch.equal(a, b)


def test_attention_extreme_scores():
    """Scores hundreds apart, a scale of its own, one entry that takes all."""
    batch = Batch([300], [1], 1, 128, 64, "bf16", seed=6)
    check_attention(batch, 2, "bf16", scale=3.0)
    check_attention(batch, 2, "f32", scale=0.001)


def test_attention_same_result_every_time_and_in_graphs():
    import torch

    from rustane_b200 import ops
    batch = Batch([5000, 64, 1], [1, 3, 1], 2, 128, 64, "bf16", seed=8, book=True)
    q, cache = batch.normal(batch.rows, 8, 128, dtype="bf16"), batch.cache()
    first = ops.paged_attention(cache, q, batch.row_start, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = ops.paged_attention(cache, q, batch.row_start, 3)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attention(cache, q, batch.row_start, 3))
        graphs.append(g)
    batch.tlens.copy_(torch.tensor([4000, 60, 1], dtype=torch.int32))  # a replay follows the lengths
    for g in graphs:
        g.replay()
    want = ops.paged_attention(cache, q, batch.row_start, 3)
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and not torch.equal(want, first)


def test_attention_reports_what_it_leaves_out():
    import torch

    from rustane_b200 import ops
    batch = Batch([100, 90, 80], [1, 1, 1], 1, 64, 16, "f16", seed=9)
    q = batch.normal(batch.rows, 2, 64, dtype="f16")
    clean = ops.paged_attention(batch.cache(), q, batch.row_start, 1)
    broken = batch.table.clone()
    broken[0, 2] = batch.pool.shape[0]
    batch.table, keep = broken, batch.table
    cache = batch.cache()
    got = ops.paged_attention(cache, q, batch.row_start, 1)
    assert int(cache.status) == 2 and torch.equal(got[1:], clean[1:])
    batch.table = keep  # the third page's entries count as masked: the same as a cache without them
    gone = Batch([84], [1], 1, 64, 16, "f16", seed=9)
    gone.pool, gone.table = batch.pool, torch.cat([keep[:1, :2], keep[:1, 3:]], 1).contiguous()
    want, _, mass, _, worst = ref.attention(gone, q[:1])
    assert (np.abs(f64(got[:1]) - want) <= attention_tolerance(want, mass, "f16", "f16", 64, worst)).all()
    batch.tlens = torch.tensor([100, 10 ** 6, -3], dtype=torch.int32, device="cuda")
    cache = batch.cache()
    out = torch.full_like(q, 5.0)
    ops.paged_attention(cache, q, batch.row_start, 1, out=out)
    assert int(cache.status) == 1 and torch.equal(out[0], clean[0]) and bool((out[1:] == 5).all())
    batch.tlens = torch.tensor([100, 90, 80], dtype=torch.int32, device="cuda")
    for starts in ([0, 1, 0, 1], [0, 1, 2, 9], [-1, 1, 2, 3], [0, 3, 3, 3]):
        cache = batch.cache()
        ops.paged_attention(cache, q, torch.tensor(starts, dtype=torch.int32, device="cuda"), 1)
        assert int(cache.status) == 1


# ------------------------------------------------------------------------------------------------ rotary positions and append
@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rot", [(64, 64), (64, 32), (128, 128), (128, 96), (128, 6), (128, 2), (64, 50)])
def test_append_types_and_layouts(q_type, kv_type, layout, hd, rot):
    check_append(Batch([1, 40, 17, 0], [1, 5, 17, 0], 2, hd, 16, kv_type, seed=rot, book=True, values=False), 6, q_type, layout, rot)


@pytest.mark.parametrize("scaling,factor", [(None, 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 32.0)])
@pytest.mark.parametrize("first", [0, 1000, 10 ** 6, 2 ** 31 - 100])
def test_append_far_positions(scaling, factor, first):
    check_append(Batch([40, 8], [33, 1], 4, 128, 64, "f32", seed=1, values=False), 4, "f32", "half", 128, scaling, factor, first)


@pytest.mark.parametrize("page", [1, 7, 24, 64])
@pytest.mark.parametrize("rows", [1, 300, 1100])
def test_append_pages_and_lengths(page, rows):
    check_append(Batch([rows, rows + 5], [rows, rows], 1, 64, page, "bf16", seed=page, book=True, values=False), 2, "bf16", "interleaved", 64)


def check_append(batch, heads, q_type, layout, rot, scaling=None, factor=1.0, first=0):
    import torch

    from rustane_b200 import ops
    kv, hd, rows = batch.kv_heads, batch.hd, batch.rows
    fused = batch.normal(rows, (heads + 2 * kv) * hd, dtype=q_type)
    q, k, v = (fused[:, a * hd:z * hd].unflatten(1, (-1, hd)) for a, z in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    positions = np.random.default_rng(rows).integers(0, 99, rows).astype(np.int64) + first
    tpos = torch.from_numpy(positions.astype(np.int32)).cuda()
    rope = ops.Rope(rot, layout=layout, scaling=scaling, factor=factor, original=2048)
    before = batch.pool.clone()
    weight, position = (None, None) if batch.weight is None else (batch.weight.clone(), batch.position.clone())
    cache = batch.cache()
    got = ops.rope_append(cache, rope, q, k, v, tpos, batch.row_start)
    freq, magnitude = ref.frequencies(rot, 10000.0, scaling, factor, 2048)
    # cos and sin: the reduced angle rounds once (2^-24 of at most pi/4), sincospi is within 2 units, their products and sum within
    # three half steps more; |a| + |b| <= 1.5 |pair|
    def near(x, want, source, t):
        size = np.abs(source)
        pair = np.zeros_like(size)
        pair[..., :rot] = 0
        u = size[..., :rot]
        other = np.concatenate([u[..., rot // 2:], u[..., :rot // 2]], -1) if layout == "half" else u.reshape(*u.shape[:-1], -1, 2)[..., ::-1].reshape(u.shape)
        pair[..., :rot] = u + other
        tol = HALF_STEP[t] * np.abs(want) + 10 * 2.0 ** -24 * magnitude * pair + (2.0 ** -25 if t == "f16" else 0)
        assert (np.abs(x - want) <= tol).all(), float((np.abs(x - want) - tol).max())

    near(f64(got), ref.rotate(f64(q), positions, freq, magnitude, layout), f64(q), q_type)
    wk = ref.rotate(f64(k), positions, freq, magnitude, layout)
    for b, n in enumerate(batch.lens):
        r0, m = int(batch.starts[b]), batch.counts[b]
        if not m:
            continue
        near(batch.entries(b, 0)[:, n - m:].transpose(1, 0, 2), wk[r0:r0 + m], f64(k)[r0:r0 + m], batch.kv)
        assert np.array_equal(batch.entries(b, 1)[:, n - m:].transpose(1, 0, 2), f64(v.to(batch.pool.dtype))[r0:r0 + m])
        assert np.array_equal(batch.entries(b, 0)[:, :n - m], batch.entries(b, 0, before)[:, :n - m])
        if weight is not None:
            weight[b, :, n - m:n] = 0
            position[b, :, n - m:n] = tpos[r0:r0 + m]
            assert torch.equal(batch.weight[b], weight[b]) and torch.equal(batch.position[b], position[b])
    written = sum(batch.counts) * kv * 2 * hd
    assert int((batch.pool != before).sum()) <= written
    assert int(cache.status) == 0


def test_append_in_place_and_left_out_rows():
    import torch

    from rustane_b200 import ops
    batch = Batch([20, 30], [2, 3], 2, 64, 16, "bf16", seed=2, values=False)
    rope = ops.Rope(64)
    q, k, v = (batch.normal(7, n, 64, dtype="bf16") for n in (4, 2, 2))
    pos = torch.arange(7, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 9.0)
    ops.rope_append(batch.cache(), rope, q, k, v, pos, batch.row_start, out=out)
    assert bool((out[5:] == 9).all())
    inside = q.clone()
    assert ops.rope_append(batch.cache(), rope, inside, k, v, pos, batch.row_start, out=inside) is inside
    assert torch.equal(inside[:5], out[:5]) and torch.equal(inside[5:], q[5:])
    pool = batch.pool.clone()
    batch.table = torch.full_like(batch.table, -1)
    cache = batch.cache()
    ops.rope_append(cache, rope, q, k, v, pos, batch.row_start)
    assert int(cache.status) == 2 and torch.equal(batch.pool, pool)
    batch.tlens = torch.tensor([1, 10 ** 7], dtype=torch.int32, device="cuda")
    cache = batch.cache()
    ops.rope_append(cache, rope, q, k, v, pos, batch.row_start)
    assert int(cache.status) & 1 and torch.equal(batch.pool, pool)


# ------------------------------------------------------------------------------------------------ eviction
def check_evict(batch, keep, sinks=0, recent=0, in_place=False):
    import torch

    from rustane_b200 import ops
    weight, position, pool = f64(batch.weight), batch.position.cpu().numpy(), batch.pool.clone()
    kept_w, kept_p = batch.weight.clone(), batch.position.clone()
    cache = batch.cache()
    out = (torch.empty_like(batch.tlens), batch.weight, batch.position) if in_place else None
    lens, new_w, new_p = ops.cache_evict(cache, keep, sinks=sinks, recent=recent, out=out)
    assert lens.tolist() == [min(n, keep) for n in batch.lens]
    want_w, want_p, want = kept_w.cpu().numpy().copy(), position.copy(), pool.clone()
    for b, n in enumerate(batch.lens):
        for h in range(batch.kv_heads):
            for to, at in ref.evict(weight[b, h], position[b, h], n, keep, sinks, recent):
                want_w[b, h, to], want_p[b, h, to] = want_w[b, h, at], position[b, h, at]
                t = batch.table[b]
                want[t[to // batch.page], :, h, to % batch.page] = pool[t[at // batch.page], :, h, at % batch.page]
    np.testing.assert_array_equal(new_w.cpu().numpy(), want_w)
    np.testing.assert_array_equal(new_p.cpu().numpy(), want_p)
    assert torch.equal(batch.pool, want)
    if not in_place:
        np.testing.assert_array_equal(f64(batch.weight), f64(kept_w))
        assert torch.equal(batch.position, kept_p)
    assert int(cache.status) == 0


@pytest.mark.parametrize("kv_type", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_evict_types_and_pages(kv_type, hd, page):
    check_evict(Batch([100, 31, 64, 0], [0] * 4, 2, hd, page, kv_type, seed=page, book=True), 40, sinks=6, recent=12)


@pytest.mark.parametrize("keep", [0, 1, 2, 63, 64, 199, 200, 1000])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_how_many_stay(keep, in_place):
    check_evict(Batch([200, 1, 65], [0] * 3, 3, 64, 16, "bf16", seed=keep, book=True), keep, in_place=in_place)


@pytest.mark.parametrize("length,keep", [(9001, 4000), (20000, 19999), (30001, 100)])
def test_evict_over_a_cluster(length, keep):
    batch = Batch([length, length // 3], [0, 0], 1, 64, 64, "f16", seed=1, book=True)
    batch.weight.mul_(50).round_()  # many ties, across CTAs
    check_evict(batch, keep, sinks=5, recent=60)


@pytest.mark.parametrize("kind", ["equal", "zeros", "few values", "nan", "infinite", "negative"])
def test_evict_order_of_weights(kind):
    import torch
    batch = Batch([700, 90], [0, 0], 2, 64, 32, "bf16", seed=3, book=True)
    w = batch.weight
    if kind == "equal":
        w.fill_(0.25)
    elif kind == "zeros":
        w[:, :, ::2], w[:, :, 1::2] = 0.0, -0.0
    elif kind == "few values":
        w.mul_(2).round_()
    elif kind == "nan":
        w[:, :, ::3] = float("nan")
    elif kind == "infinite":
        w[:, :, ::5], w[:, :, 1::5] = float("inf"), -float("inf")
    else:
        w.sub_(2.0)
    for keep in (80, 350, 650):
        batch.position = torch.randperm(batch.cap, generator=batch.g).to(torch.int32).expand(2, 2, batch.cap).contiguous().cuda()
        check_evict(batch, keep, sinks=10, recent=keep // 3)


def test_evict_leaves_bad_lengths_and_pages():
    import torch

    from rustane_b200 import ops
    batch = Batch([100, 90], [0, 0], 1, 64, 16, "f16", seed=4, book=True)
    batch.tlens = torch.tensor([100, 10 ** 8], dtype=torch.int32, device="cuda")
    cache = batch.cache()
    lens, w, _ = ops.cache_evict(cache, 50)
    assert int(cache.status) == 1 and lens.tolist() == [50, 10 ** 8] and torch.equal(w[1], batch.weight[1])
    batch.tlens = torch.tensor([100, 90], dtype=torch.int32, device="cuda")
    batch.table = torch.full_like(batch.table, batch.pool.shape[0])
    pool, cache = batch.pool.clone(), batch.cache()
    _, w, _ = ops.cache_evict(cache, 50)
    assert int(cache.status) == 2 and torch.equal(batch.pool, pool) and torch.equal(w, batch.weight)


# ------------------------------------------------------------------------------------------------ verification
def verify_inputs(counts, vocab, dtype, seed, near=0.7, heat=1.0):
    import torch
    g = torch.Generator("cpu").manual_seed(seed)
    rows = sum(counts)
    target = torch.randn(rows, vocab, generator=g) * 2
    draft = (target + near * torch.randn(rows, vocab, generator=g)).to(ref.torch_dtype(dtype))
    target = target.to(ref.torch_dtype(dtype))
    noise = -torch.log(-torch.log(torch.rand(rows, vocab, generator=g).clamp(1e-20, 1 - 1e-7)))
    guess = (draft.float() / max(heat, 0.2) + noise).argmax(1).int()
    tokens = torch.zeros(rows, dtype=torch.int32)
    tokens[1:] = guess[:-1]
    starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32)
    return dict(target=target, draft=draft, tokens=tokens, starts=starts, u=torch.rand(rows, generator=g), d=torch.rand(len(counts), generator=g), most=max(counts + [1]))


def check_verify(x, temperature, with_draft=True):
    import torch

    from rustane_b200 import ops
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    draft = x["draft"].cuda() if with_draft else None
    accepted, out = ops.verify_drafts(x["target"].cuda(), x["tokens"].cuda(), x["starts"].cuda(), x["most"], x["u"].cuda(), x["d"].cuda(), draft=draft,
                                      temperature=temperature, status=status)
    want_n, want = ref.verify(f64(x["target"]), f64(x["draft"]) if with_draft else None, x["tokens"].numpy(), f64(x["u"]), f64(x["d"]), x["starts"].numpy(), temperature)
    np.testing.assert_array_equal(accepted.cpu().numpy(), want_n)
    np.testing.assert_array_equal(out.cpu().numpy()[:len(want)], want)
    return int(status), accepted, out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 7, 1000, 5003, 32000])
@pytest.mark.parametrize("temperature,with_draft", [(0.0, False), (1.0, True), (1.0, False), (0.6, True)])
def test_verify_types_and_vocabularies(dtype, vocab, temperature, with_draft):
    for seed in range(3):
        status, _, _ = check_verify(verify_inputs([5, 1, 3, 8], vocab, dtype, seed, heat=temperature), temperature, with_draft)
        assert status == 0


@pytest.mark.parametrize("near", [0.0, 0.1, 3.0])
@pytest.mark.parametrize("counts", [[1], [2], [9], [0, 3, 0, 1, 2, 0], [4] * 40, [40, 1]])
def test_verify_batches(near, counts):
    for temperature, with_draft in ((1.0, True), (0.8, False), (0.0, False)):
        check_verify(verify_inputs(counts, 3001, "bf16", 11, near=near, heat=temperature), temperature, with_draft)


def test_verify_uniforms_at_the_ends():
    import torch
    for value in (0.0, 1.0 - 2.0 ** -24):
        for with_draft in (True, False):
            x = verify_inputs([4, 4, 1], 2000, "f32", 5)
            x["u"], x["d"] = torch.full_like(x["u"], value), torch.full_like(x["d"], value)
            check_verify(x, 1.0, with_draft)


def test_verify_masked_logits_are_never_drawn():
    import torch
    for dtype, lowest in (("f32", -float("inf")), ("bf16", torch.finfo(torch.bfloat16).min), ("f16", -float("inf"))):
        x = verify_inputs([3, 1, 2], 4001, dtype, 6)
        x["target"][:, ::2] = lowest
        x["target"][3, 5:] = lowest
        x["d"] = torch.tensor([0.999999, 0.0, 0.5])
        _, _, out = check_verify(x, 1.0)
        drawn = [int(v) for v in out.cpu() if v >= 0]
        assert all(v % 2 for v in drawn)


def test_verify_ties_go_to_the_lowest_token():
    import torch
    x = verify_inputs([3, 2], 9001, "bf16", 7)
    x["target"] = torch.zeros_like(x["target"])
    x["target"][:, [77, 4000, 8999]] = 3.0
    x["tokens"] = torch.tensor([0, 77, 4000, 0, 77], dtype=torch.int32)
    _, accepted, out = check_verify(x, 0.0, False)
    assert accepted.tolist() == [1, 1] and out.tolist() == [77, 77, -1, 77, 77]


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_verify_rows_without_a_distribution(value, temperature):
    x = verify_inputs([3, 1, 2, 1], 1500, "f32", 8)
    x["u"][:] = 0.0  # every draft with some probability stays
    x["target"][1, 700] = value
    x["target"][3] = -float("inf")
    x["target"][6, 1499] = value
    if temperature == 0:
        x["tokens"][1] = int(x["target"][0].argmax())
        x["tokens"][5] = int(x["target"][4].argmax())
    status, accepted, out = check_verify(x, temperature, temperature > 0)
    assert status == 4 and out.tolist()[1] == -1 and out.tolist()[3] == -1 and out.tolist()[6] == -1 and int(accepted[0]) == 1


def test_verify_token_ids_outside_the_vocabulary_are_turned_down():
    x = verify_inputs([3, 3, 2], 800, "f32", 9)
    x["u"][:] = 0.0
    x["tokens"][1], x["tokens"][5], x["tokens"][7] = -5, 800, 2 ** 31 - 1
    for temperature, with_draft in ((1.0, True), (1.0, False), (0.0, False)):
        check_verify(x, temperature, with_draft)


def test_verify_strided_rows_unaligned_and_rows_behind_the_batch():
    import torch

    from rustane_b200 import ops
    x = verify_inputs([4, 2], 1001, "f16", 10)
    wide = torch.full((9, 1301), float("nan"), dtype=torch.float16, device="cuda")
    wide2 = wide.clone()
    wide[:6, 3:1004], wide2[:6, 5:1006] = x["target"].cuda(), x["draft"].cuda()
    pad = torch.nn.functional.pad
    accepted, out = ops.verify_drafts(wide[:, 3:1004], pad(x["tokens"], (0, 3)).cuda(), x["starts"].cuda(), 4, pad(x["u"], (0, 3)).cuda(), x["d"].cuda(),
                                      draft=wide2[:, 5:1006])
    want_n, want = ref.verify(f64(x["target"]), f64(x["draft"]), x["tokens"].numpy(), f64(x["u"]), f64(x["d"]), x["starts"].numpy(), 1.0)
    assert accepted.tolist() == want_n.tolist() and out.tolist()[:6] == want.tolist()


def test_verify_refuses_broadcast_logits():
    import torch

    from rustane_b200 import ops
    x = verify_inputs([4, 2], 1001, "f16", 10)
    tokens, starts, u, d = (x[k].cuda() for k in ("tokens", "starts", "u", "d"))
    target, draft = x["target"].cuda(), x["draft"].cuda()
    with pytest.raises(ValueError, match="target: broadcast"):
        ops.verify_drafts(target[:1].expand(6, 1001), tokens, starts, 4, u, d)
    with pytest.raises(ValueError, match="draft: broadcast"):
        ops.verify_drafts(target, tokens, starts, 4, u, d, draft=draft[:1].expand(6, 1001))


def test_verify_leaves_out_sequences_whose_rows_do_not_fit():
    import torch

    from rustane_b200 import ops
    x = verify_inputs([3, 2, 4], 700, "bf16", 12)
    want_n, want = ref.verify(f64(x["target"]), f64(x["draft"]), x["tokens"].numpy(), f64(x["u"]), f64(x["d"]), x["starts"].numpy(), 1.0)
    for starts, fits in (([0, 3, -1, 9], [0]), ([0, 3, 5, 10], [0, 1]), ([0, 3, 2, 9], [0]), ([-2 ** 31, 3, 5, 9], [1, 2]), ([2 ** 31 - 1, 3, 5, 9], [1, 2])):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        accepted, out = ops.verify_drafts(x["target"].cuda(), x["tokens"].cuda(), torch.tensor(starts, dtype=torch.int32, device="cuda"), 4, x["u"].cuda(), x["d"].cuda(),
                                          draft=x["draft"].cuda(), status=status)
        assert int(status) & 1
        for b in fits:
            assert int(accepted[b]) == want_n[b]
            r0, r1 = x["starts"][b], x["starts"][b + 1]
            assert out[r0:r1].tolist() == want[r0:r1].tolist()


# ------------------------------------------------------------------------------------------------ where calls meet
@pytest.mark.parametrize("q_type,kv_type", TYPES)
@pytest.mark.parametrize("page", [16, 24, 48])
def test_attention_many_units_a_cta_with_rows_of_every_size(q_type, kv_type, page):
    """More units than CTAs, one to four row warps in turn: every unit's stages follow another's, of another width."""
    rng = np.random.default_rng(page)
    lens, counts = [int(n) for n in rng.integers(1, 400, 96)], [int(n) for n in rng.integers(0, 7, 96)]
    check_attention(Batch(lens, counts, 2, 64, page, kv_type, seed=page), 16, q_type)
    check_attention(Batch(lens[:40], counts[:40], 4, 128, page, kv_type, seed=page), 16, q_type)


def test_offsets_past_32_bits():
    """A pool of 2^31 elements and more, its last pages in use: attention, append and eviction."""
    import torch

    from rustane_b200 import ops
    kv, hd, page = 8, 128, 64
    per = 2 * kv * page * hd
    pages = 2 ** 31 // per + 40
    pool = torch.zeros(pages, 2, kv, page, hd, dtype=torch.bfloat16, device="cuda")
    small = Batch([300, 130], [1, 1], kv, hd, page, "bf16", seed=3, book=True, spare_pages=0)
    used = small.pool.shape[0]
    pool[-used:] = small.pool
    table = torch.where(small.table >= 0, small.table + (pages - used), small.table)
    q = small.normal(2, 16, hd, dtype="bf16")
    want = ops.paged_attention(small.cache(), q, small.row_start, 1)
    cache = ops.PagedCache(pool, table, small.tlens, small.weight, small.position)
    assert torch.equal(ops.paged_attention(cache, q, small.row_start, 1), want)
    k, v, at = small.normal(2, kv, hd, dtype="bf16"), small.normal(2, kv, hd, dtype="bf16"), torch.tensor([299, 129], dtype=torch.int32, device="cuda")
    rope = ops.Rope(hd)
    for c in (small.cache(), cache):
        ops.rope_append(c, rope, q, k, v, at, small.row_start)
        ops.cache_evict(c, 100)
    assert torch.equal(pool[-used:], small.pool) and not bool(pool[:-used].any())


def test_long_score_rows_are_collected_past_32_bits():
    """scores of rows times entries pass 2^31 elements in the workspace."""
    batch = Batch([64] * 3, [1] * 3, 1, 64, 64, "bf16", seed=4, book=False)
    import torch
    rows, heads, entries = 3, 64, 12 * 2 ** 20
    table = torch.zeros(3, entries // 64, dtype=torch.int32, device="cuda")
    table[:, 0] = batch.table[:, 0]
    batch.table = table
    batch.cap = entries
    batch.weight = torch.zeros(3, 1, entries, device="cuda")
    batch.position = torch.zeros(3, 1, entries, dtype=torch.int32, device="cuda")
    assert rows * heads * entries > 2 ** 31
    check_attention(batch, heads, "bf16", collect=True)


@pytest.mark.parametrize("kv_type", ["bf16", "f32"])
def test_a_bounded_cache_over_many_steps(kv_type):
    """append, attend with weights, evict, step after step, each against a plain cache that is carried along; then the same
    steps from a captured graph."""
    import torch

    from rustane_b200 import ops
    nseq, heads, kv, hd, page, keep, steps = 3, 4, 2, 64, 16, 40, 60
    lens0 = [30, 5, 38]
    batch = Batch([48] * nseq, [1] * nseq, kv, hd, page, kv_type, seed=21, book=True)
    batch.lens = lens0
    batch.tlens = torch.tensor(lens0, dtype=torch.int32, device="cuda")
    g = torch.Generator("cpu").manual_seed(5)
    inputs = [torch.randn(nseq, heads + 2 * kv, hd, generator=g).to(batch.pool.dtype).cuda() for _ in range(steps)]
    rope = ops.Rope(hd, layout="half")
    start = (batch.pool.clone(), batch.weight.clone(), batch.position.clone())

    def reset():
        for mine, was in zip((batch.pool, batch.weight, batch.position), start):
            mine.copy_(was)

    def one_step(cache, x, at, lens, spare):
        lens.add_(1)
        q = ops.rope_append(cache, rope, x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], at, batch.row_start)
        out = ops.paged_attention(cache, q, batch.row_start, 1, collect=True)
        ops.cache_evict(cache, keep, sinks=2, recent=8, out=(spare, batch.weight, batch.position))
        lens.copy_(spare)
        return out

    # step by step, each against the plain form of what the cache holds at that moment
    lens, spare = batch.tlens, torch.empty_like(batch.tlens)
    cache, outs = batch.cache(), []
    at = torch.tensor([500, 9, 38], dtype=torch.int32, device="cuda")
    for x in inputs:
        lens.add_(1)
        q = ops.rope_append(cache, rope, x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], at, batch.row_start)
        batch.lens = lens.tolist()
        before = f64(batch.weight)
        out = ops.paged_attention(cache, q, batch.row_start, 1, collect=True)
        want, _, mass, got, worst = ref.attention(batch, q)
        assert (np.abs(f64(out) - want) <= attention_tolerance(want, mass, kv_type, kv_type, hd, worst)).all()
        weight, position, pool = f64(batch.weight), batch.position.cpu().numpy(), batch.pool.clone()
        for b, n in enumerate(batch.lens):
            np.testing.assert_allclose(weight[b][:, :n], before[b][:, :n] + got[b], rtol=1e-4, atol=1e-6)
        ops.cache_evict(cache, keep, sinks=2, recent=8, out=(spare, batch.weight, batch.position))
        for b, n in enumerate(batch.lens):
            for h in range(kv):
                for to, of in ref.evict(weight[b, h], position[b, h], n, keep, 2, 8):
                    t = batch.table[b]
                    pool[t[to // page], :, h, to % page] = pool[t[of // page], :, h, of % page]
        assert torch.equal(batch.pool, pool)
        lens.copy_(spare)
        assert lens.tolist() == [min(n, keep) for n in batch.lens]
        outs.append(out)
        at.add_(1)
    end = (batch.pool.clone(), batch.weight.clone(), batch.position.clone(), lens.clone())
    assert lens.tolist() == [keep] * nseq and int(cache.status) == 0

    # the same from one captured step
    reset()
    lens.copy_(torch.tensor(lens0, dtype=torch.int32))
    at.copy_(torch.tensor([500, 9, 38], dtype=torch.int32))
    x = inputs[0].clone()
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        one_step(cache, x, at, lens, spare)
    torch.cuda.synchronize()
    reset()
    lens.copy_(torch.tensor(lens0, dtype=torch.int32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one_step(cache, x, at, lens, spare)
        at.add_(1)
    at.copy_(torch.tensor([500, 9, 38], dtype=torch.int32))
    for i, more in enumerate(inputs):
        x.copy_(more)
        graph.replay()
        assert torch.equal(out, outs[i])
    for mine, was in zip((batch.pool, batch.weight, batch.position, lens), end):
        assert torch.equal(mine, was)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_a_drafting_step(temperature):
    """Pending token and drafts appended and attended together, verified, the cache cut back to what stays: the next step's rows see what a
    cache that never held the refused drafts gives."""
    import torch

    from rustane_b200 import ops
    kv, heads, hd, page, vocab = 2, 4, 64, 16, 900
    lens, counts = [40, 17, 90], [4, 1, 6]
    batch = Batch([n + c for n, c in zip(lens, counts)], counts, kv, hd, page, "f16", seed=31)
    x = verify_inputs(counts, vocab, "f32", 7, near=0.3, heat=max(temperature, 0.5))
    rope, cache = ops.Rope(hd), batch.cache()
    fresh = batch.normal(batch.rows, heads + 2 * kv, hd, dtype="f16")
    at = torch.cat([torch.arange(n, n + c) for n, c in zip(lens, counts)]).to(torch.int32).cuda()
    q = ops.rope_append(cache, rope, fresh[:, :heads], fresh[:, heads:heads + kv], fresh[:, heads + kv:], at, batch.row_start)
    ops.paged_attention(cache, q, batch.row_start, max(counts))
    accepted, out = ops.verify_drafts(x["target"].cuda(), x["tokens"].cuda(), batch.row_start, max(counts), x["u"].cuda(), x["d"].cuda(), draft=x["draft"].cuda() if temperature else None,
                                      temperature=temperature)
    want_n, want = ref.verify(f64(x["target"]), f64(x["draft"]) if temperature else None, x["tokens"].numpy(), f64(x["u"]), f64(x["d"]), batch.starts, temperature)
    assert accepted.tolist() == want_n.tolist() and out.tolist() == want.tolist()
    # one more token each on what stays: pending token and accepted drafts
    kept = [n + 1 + a for n, a in zip(lens, want_n)]
    batch.tlens.copy_(torch.tensor([n + 1 for n in kept], dtype=torch.int32))
    one = torch.arange(4, dtype=torch.int32, device="cuda")
    more = batch.normal(3, heads + 2 * kv, hd, dtype="f16")
    q = ops.rope_append(cache, rope, more[:, :heads], more[:, heads:heads + kv], more[:, heads + kv:], torch.tensor(kept, dtype=torch.int32, device="cuda"), one)
    batch.lens, batch.counts, batch.starts, batch.row_start, batch.rows = [n + 1 for n in kept], [1, 1, 1], np.arange(4), one, 3
    check_attention(batch, heads, "f16", q=q)


def test_two_streams_at_once():
    import torch

    from rustane_b200 import ops
    jobs = []
    for i in range(2):
        batch = Batch([4000 + i, 900], [1, 2], 2, 128, 64, "bf16", seed=40 + i, book=True)
        jobs.append((batch.cache(), batch.normal(3, 8, 128, dtype="bf16"), batch.row_start, verify_inputs([4, 3], 20000, "bf16", i)))
    moved = [{k: v.cuda() if hasattr(v, "cuda") else v for k, v in x.items()} for *_, x in jobs]

    def work(i):
        cache, q, starts, _ = jobs[i]
        x = moved[i]
        return (ops.paged_attention(cache, q, starts, 2), *ops.cache_evict(cache, 700, recent=50),
                *ops.verify_drafts(x["target"], x["tokens"], x["starts"], x["most"], x["u"], x["d"], draft=x["draft"]))

    pools = [j[0].pool.clone() for j in jobs]
    alone = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for j, was in zip(jobs, pools):
            j[0].pool.copy_(was)
        torch.cuda.synchronize()
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(work(i))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_python_refusals():
    import torch

    from rustane_b200 import ops
    batch = Batch([20, 30], [1, 1], 2, 64, 16, "f16", seed=1, book=True)
    cache, q = batch.cache(), batch.normal(2, 4, 64, dtype="f16")
    k = batch.normal(2, 2, 64, dtype="f16")
    pos, rope = torch.zeros(2, dtype=torch.int32, device="cuda"), ops.Rope(64)
    bad = [
        lambda: ops.PagedCache(batch.pool.cpu(), batch.table, batch.tlens), lambda: ops.PagedCache(batch.pool[:, :1], batch.table, batch.tlens),
        lambda: ops.PagedCache(batch.pool.double(), batch.table, batch.tlens), lambda: ops.PagedCache(batch.pool, batch.table.long(), batch.tlens),
        lambda: ops.PagedCache(batch.pool, batch.table, batch.tlens[:1]), lambda: ops.PagedCache(batch.pool, batch.table, batch.tlens.cpu()),
        lambda: ops.PagedCache(batch.pool, batch.table, batch.tlens, batch.weight), lambda: ops.PagedCache(batch.pool, batch.table, batch.tlens, batch.weight[:, :, 1:], batch.position),
        lambda: ops.Rope(64, layout="other"), lambda: ops.Rope(64, scaling="other"),
        lambda: ops.paged_attention(cache, q[0], batch.row_start, 1), lambda: ops.paged_attention(cache, q[:, :, :32], batch.row_start, 1),
        lambda: ops.paged_attention(cache, q.transpose(0, 1), batch.row_start, 1), lambda: ops.paged_attention(cache, q.cpu(), batch.row_start, 1),
        lambda: ops.paged_attention(cache, q, batch.row_start[:2], 1), lambda: ops.paged_attention(cache, q, batch.row_start.long(), 1),
        lambda: ops.paged_attention(cache, q, batch.row_start, 1, out=torch.empty(2, 4, 64, device="cuda")), lambda: ops.paged_attention(cache, q.double(), batch.row_start, 1),
        lambda: ops.paged_attention(cache, q, batch.row_start, 1, workspace=torch.empty(4, device="cuda")),
        lambda: ops.rope_append(cache, rope, q, q, k, pos, batch.row_start), lambda: ops.rope_append(cache, rope, q, k, k.float(), pos, batch.row_start),
        lambda: ops.rope_append(cache, rope, q, k, k, pos[:1], batch.row_start), lambda: ops.rope_append(cache, rope, q, k[:1], k, pos, batch.row_start),
        lambda: ops.cache_evict(ops.PagedCache(batch.pool, batch.table, batch.tlens), 5), lambda: ops.cache_evict(cache, 5, out=(batch.tlens, batch.weight[:1], batch.position)),
        lambda: ops.verify_drafts(q, pos, batch.row_start, 1, None, None), lambda: ops.verify_drafts(q[0], pos, batch.row_start, 1, None, None, temperature=0.0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was taken" % i)
    worse = [
        lambda: ops.paged_attention(cache, batch.normal(2, 3, 64, dtype="f16"), batch.row_start, 1), lambda: ops.paged_attention(cache, batch.normal(2, 4, 64, dtype="bf16"), batch.row_start, 1),
        lambda: ops.paged_attention(cache, q, batch.row_start, 0), lambda: ops.paged_attention(cache, q, batch.row_start, 1, window=-1),
        lambda: ops.paged_attention(cache, q, batch.row_start, 1, workspace=torch.empty(4, dtype=torch.uint8, device="cuda")),
        lambda: ops.rope_append(cache, ops.Rope(66), q, k, k, pos, batch.row_start), lambda: ops.cache_evict(cache, 5, sinks=3, recent=3),
        lambda: ops.cache_evict(cache, 5, out=(cache.lens, torch.empty_like(batch.weight), torch.empty_like(batch.position))),
    ]
    from rustane_b200 import CudaDecodeError
    for i, call in enumerate(worse):
        with pytest.raises(CudaDecodeError):
            call()
            pytest.fail("call %d was taken" % i)
