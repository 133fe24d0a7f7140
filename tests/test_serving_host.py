"""Host side of the serving-step operators: what they refuse, workspace sizes and rotary tables (no GPU)."""
import ctypes as C

import numpy as np
import pytest

import serving_ref as ref

A = 1 << 20  # stands for device memory: the calls below are refused before anything is launched


def cache(**over):
    from rustane_b200 import _ffi
    c = _ffi.CdPagedCache(2, 8, 128, 64, 10, 3, 4, -1)
    c.table_stride, c.pool, c.page_table, c.lens, c.weight, c.position = 4, A, A, A, A, A
    for k, v in over.items():
        setattr(c, k, v)
    return c


def refused(rc, code, text):
    from rustane_b200 import _ffi
    assert rc == code, (rc, _ffi.lib.cd_last_error(None))
    assert text in _ffi.lib.cd_last_error(None).decode()


INVALID, CAPACITY, UNSUPPORTED = -1, -4, -8
BAD_CACHES = [
    (dict(dtype=3), INVALID, "f32, f16 or bf16"), (dict(dtype=-1), INVALID, "f32, f16 or bf16"), (dict(kv_heads=0), INVALID, "kv_heads"), (dict(hd=96), UNSUPPORTED, "64 or 128"),
    (dict(page_tokens=0), INVALID, "page_tokens"), (dict(page_tokens=65537), INVALID, "page_tokens"), (dict(npages=0), INVALID, "at least one page"), (dict(max_pages=0), INVALID, "at least one page"),
    (dict(nseq=-1), UNSUPPORTED, "4096"), (dict(nseq=4097), UNSUPPORTED, "4096"), (dict(max_pages=1 << 25), UNSUPPORTED, "2^31"), (dict(table_stride=3), INVALID, "table_stride"),
    (dict(pool=None), INVALID, "null"), (dict(page_table=None), INVALID, "null"), (dict(lens=None), INVALID, "null"), (dict(position=None), INVALID, "come together"),
    (dict(pool=A + 8), INVALID, "16-byte"), (dict(lens=A + 2), INVALID, "4-byte"), (dict(status=A + 1), INVALID, "4-byte"),
]


def attention(c, dtype=2, heads=16, nrows=3, max_rows=1, q=A, stride=0, starts=A, scale=0.0, window=0, collect=0, out=A, lse=None, ws=A, room=1 << 40):
    from rustane_b200._ffi import lib
    return lib.cd_paged_attention(C.byref(c) if c else None, dtype, heads, nrows, max_rows, q, stride, starts, scale, window, collect, out, lse, ws, room, None)


def append(c, dtype=2, heads=16, nrows=3, q=A, qs=0, k=A, ks=0, v=A, vs=0, pos=A, starts=A, out=2 * A, rot=128, layout=1, magnitude=1.0, turns=A):
    from rustane_b200 import _ffi
    r = _ffi.CdRope(rot, layout, magnitude, 0, turns)
    return _ffi.lib.cd_rope_append(C.byref(c), C.byref(r), dtype, heads, nrows, q, qs, k, ks, v, vs, pos, starts, out, None)


def evict(c, keep=50, sinks=4, recent=10, lens=2 * A, weight=A, position=A, ws=A, room=1 << 40):
    from rustane_b200._ffi import lib
    return lib.cd_cache_evict(C.byref(c), keep, sinks, recent, lens, weight, position, ws, room, None)


def verify(dtype=0, nseq=2, nrows=4, max_rows=2, vocab=100, target=A, ts=0, draft=A, ds=0, tokens=A, starts=A, u=A, d=A, temperature=1.0, accepted=A, out=A, status=None, ws=A, room=1 << 40):
    from rustane_b200._ffi import lib
    return lib.cd_verify_drafts(-1, dtype, nseq, nrows, max_rows, vocab, target, ts, draft, ds, tokens, starts, u, d, temperature, accepted, out, status, ws, room, None)


@pytest.mark.parametrize("over,code,text", BAD_CACHES)
def test_bad_caches_are_refused_by_every_call(R, over, code, text):
    for call in (attention, append, evict):
        refused(call(cache(**over)), code, text)
    refused(attention(None), INVALID, "null cache")


@pytest.mark.parametrize("over,code,text", [
    (dict(heads=0), INVALID, "multiple"), (dict(heads=12), INVALID, "multiple"), (dict(heads=80000), UNSUPPORTED, "65536"), (dict(nrows=-1), INVALID, "nrows"), (dict(max_rows=0), INVALID, "max_rows"),
    (dict(dtype=1), INVALID, "pool's type"), (dict(dtype=3), INVALID, "pool's type"), (dict(window=-1), INVALID, "window"), (dict(scale=float("nan")), INVALID, "scale"),
    (dict(scale=float("inf")), INVALID, "scale"), (dict(q=None), INVALID, "null"), (dict(out=None), INVALID, "null"), (dict(starts=None), INVALID, "null"), (dict(ws=None), INVALID, "null"),
    (dict(q=A + 8), INVALID, "16-byte"), (dict(out=A + 4), INVALID, "16-byte"), (dict(stride=2047), INVALID, "shorter"), (dict(stride=2049), INVALID, "16-byte"),
    (dict(starts=A + 1), INVALID, "4-byte"), (dict(lse=A + 2), INVALID, "4-byte"), (dict(ws=A + 16), INVALID, "256-byte"), (dict(room=1000), CAPACITY, "workspace"),
    (dict(max_rows=70000), INVALID, "max_rows"),
])
def test_attention_refuses(R, over, code, text):
    refused(attention(cache(), **over), code, text)
    refused(attention(cache(weight=None, position=None), collect=1), INVALID, "weight")


@pytest.mark.parametrize("over,code,text", [
    (dict(dtype=1), INVALID, "pool's type"), (dict(heads=0), INVALID, "heads"), (dict(nrows=-1), INVALID, "nrows"), (dict(rot=0), INVALID, "rot_dim"), (dict(rot=5), INVALID, "rot_dim"),
    (dict(rot=130), INVALID, "rot_dim"), (dict(layout=2), INVALID, "layout"), (dict(magnitude=float("inf")), INVALID, "magnitude"), (dict(turns=None), INVALID, "null"), (dict(turns=A + 4), INVALID, "8-byte"),
    (dict(q=None), INVALID, "null"), (dict(k=None), INVALID, "null"), (dict(v=None), INVALID, "null"), (dict(out=None), INVALID, "null"), (dict(pos=None), INVALID, "null"), (dict(starts=None), INVALID, "null"),
    (dict(qs=2000), INVALID, "shorter"), (dict(ks=1000), INVALID, "shorter"), (dict(vs=1025), INVALID, "16-byte"), (dict(k=A + 2), INVALID, "16-byte"), (dict(out=A, qs=4096), INVALID, "packed"),
])
def test_append_refuses(R, over, code, text):
    refused(append(cache(), **over), code, text)


@pytest.mark.parametrize("over,code,text", [
    (dict(keep=-1), INVALID, "keep"), (dict(sinks=-1), INVALID, "sinks"), (dict(recent=-1), INVALID, "sinks"), (dict(sinks=41), INVALID, "more than keep"), (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), INVALID, "more than keep"),
    (dict(lens=None), INVALID, "null"), (dict(weight=None), INVALID, "null"), (dict(position=None), INVALID, "null"), (dict(ws=None), INVALID, "null"), (dict(lens=A), INVALID, "lens"),
    (dict(weight=A + 2), INVALID, "4-byte"), (dict(ws=A + 4), INVALID, "256-byte"), (dict(room=100), CAPACITY, "workspace"),
])
def test_evict_refuses(R, over, code, text):
    refused(evict(cache(), **over), code, text)
    refused(evict(cache(weight=None, position=None)), INVALID, "bookkeeping")
    refused(evict(cache(nseq=4096, kv_heads=32)), UNSUPPORTED, "65535")


@pytest.mark.parametrize("over,code,text", [
    (dict(dtype=3), INVALID, "f32, f16 or bf16"), (dict(nseq=-1), INVALID, "nseq"), (dict(nrows=-1), INVALID, "nrows"), (dict(vocab=0), INVALID, "vocab"), (dict(vocab=1 << 23), UNSUPPORTED, "4194304"),
    (dict(max_rows=0), INVALID, "max_rows"), (dict(temperature=-1.0), INVALID, "temperature"), (dict(temperature=float("nan")), INVALID, "temperature"), (dict(temperature=1e-9), INVALID, "temperature"),
    (dict(target=None), INVALID, "null"), (dict(tokens=None), INVALID, "null"), (dict(starts=None), INVALID, "null"), (dict(accepted=None), INVALID, "null"), (dict(out=None), INVALID, "null"),
    (dict(ws=None), INVALID, "null"), (dict(u=None), INVALID, "uniforms"), (dict(d=None), INVALID, "uniforms"), (dict(ts=99), INVALID, "shorter"), (dict(ds=99), INVALID, "shorter"),
    (dict(target=A + 2), INVALID, "aligned"), (dict(tokens=A + 2), INVALID, "4-byte"), (dict(ws=A + 8), INVALID, "256-byte"), (dict(room=0), CAPACITY, "workspace"),
])
def test_verify_refuses(R, over, code, text):
    refused(verify(**over), code, text)


def test_empty_batches_are_nothing_to_do(R):
    assert attention(cache(), nrows=0, q=None, out=None) == 0 and attention(cache(nseq=0)) == 0
    assert append(cache(), nrows=0, q=None) == 0 and evict(cache(nseq=0)) == 0 and verify(nseq=0) == 0


def test_workspaces_have_a_size(R):
    from rustane_b200 import _ffi
    lib, n, big = _ffi.lib, C.c_size_t(), C.c_size_t()
    assert lib.cd_paged_attention_workspace(C.byref(cache()), 16, 3, 1, 0, C.byref(n)) == 0
    assert lib.cd_paged_attention_workspace(C.byref(cache()), 16, 3, 1, 1, C.byref(big)) == 0
    assert big.value >= n.value + 3 * 16 * 4 * 64 * 4  # every row's and head's scores
    assert lib.cd_cache_evict_workspace(C.byref(cache()), 50, C.byref(n)) == 0 and n.value >= 2 * 3 * 8 * 50 * 4
    assert lib.cd_verify_drafts_workspace(4, 2, 100, C.byref(n)) == 0 and n.value > 0
    refused(lib.cd_paged_attention_workspace(C.byref(cache()), 16, 3, 1, 0, None), INVALID, "null")
    refused(lib.cd_cache_evict_workspace(C.byref(cache()), -1, C.byref(n)), INVALID, "keep")


@pytest.mark.parametrize("rot", [2, 6, 64, 96, 128])
@pytest.mark.parametrize("scaling,factor", [(None, 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 32.0)])
@pytest.mark.parametrize("base", [100.0, 10000.0, 500000.0])
def test_rope_frequencies(R, rot, scaling, factor, base):
    from rustane_b200 import ops
    turns, magnitude = ops.rope_frequencies(rot, base, scaling, factor, 4096)
    freq, want = ref.frequencies(rot, base, scaling, factor, 4096)
    # the frequency over 2 pi in 64-bit arithmetic (some units of 2^-52 of it), rounded to the table's steps of 2^-63 of a turn: half a
    # step is 2^-64 turns, 2^-64 * 2 pi radians
    np.testing.assert_allclose(turns.astype(np.float64) / 2.0 ** 64 * 2 * np.pi, freq, rtol=2.0 ** -48, atol=2.0 ** -64 * 2 * np.pi)
    assert magnitude == pytest.approx(want, rel=2.0 ** -23)


@pytest.mark.parametrize("args", [(0, 1e4, None, 1.0, 1), (3, 1e4, None, 1.0, 1), (64, 0.5, None, 1.0, 1), (64, float("nan"), None, 1.0, 1), (64, 1e4, "ntk", 0.5, 1), (64, 1e4, "yarn", 2.0, 0)])
def test_rope_frequencies_refuses(R, args):
    from rustane_b200 import ops
    with pytest.raises(R.CudaDecodeError):
        ops.rope_frequencies(*args)


def test_broadcast_rows_are_refused():
    # the library reads a stride of 0 as packed rows, which a tensor broadcast from one row does not have
    import torch

    from rustane_b200 import ops
    one = torch.zeros(1, 2, 64)
    with pytest.raises(ValueError, match="q: broadcast"):
        ops._row_stride(one.expand(3, 2, 64), "q", 3, 64, -1)
    with pytest.raises(ValueError, match="next to each other"):
        ops._row_stride(torch.zeros(3, 1, 64).expand(3, 2, 64), "q", 3, 64, -1)
    assert ops._row_stride(one, "q", 1, 64, -1) == 0
    assert ops._row_stride(one.expand(1, 2, 64), "q", 1, 64, -1) == 0
    assert ops._row_stride(torch.zeros(3, 6, 64)[:, 2:4], "q", 3, 64, -1) == 384


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1])
def test_counts_past_32_bits_are_refused(R, n):
    # (ahead of everything else: no cache is looked at)
    import torch

    from rustane_b200 import ops
    for call in (lambda: ops.paged_attention(None, None, None, 1, window=n), lambda: ops.paged_attention(None, None, None, n),
                 lambda: ops.cache_evict(None, n), lambda: ops.cache_evict(None, 5, sinks=n), lambda: ops.cache_evict(None, 5, recent=n),
                 lambda: ops.verify_drafts(torch.zeros(1, 2), None, None, n, None, None)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
