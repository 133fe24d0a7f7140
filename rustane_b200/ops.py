"""Single operators of the token loop on caller-supplied data.

flash_decode takes host arrays.  The operators of a serving step (PagedCache, Rope, rope_append, paged_attention, cache_evict,
verify_drafts) take CUDA tensors, enqueue on torch's current stream of their device and return without waiting, so they can be captured
into a CUDA graph; their workspaces come from torch's allocator, one per call.  A batch is described by `row_start`
(int32 [nseq + 1]: sequence b has the new rows row_start[b] .. row_start[b + 1]) and the cache's `lens` (entries of each
sequence, those of its new rows the last).
"""
import ctypes as C

import numpy as np

from . import _ffi
from ._ffi import CudaDecodeError, lib

_DT = {"f32": 0, "f16": 1, "bf16": 2}


def to_storage(a, dtype):
    """fp32 array -> the raw storage words of `dtype` (round to nearest even): float32 for
    f32, float16 for f16, uint16 bit patterns for bf16."""
    a = np.ascontiguousarray(a, dtype=np.float32)
    if dtype == "f32":
        return a
    if dtype == "f16":
        return a.astype(np.float16)
    u = a.view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_storage(s, dtype):
    if dtype == "bf16":
        return (s.astype(np.uint32) << 16).view(np.float32)
    return s.astype(np.float32)


def flash_decode(q, k, v, heads, kv_heads, hd, dtype="bf16", nsplit=0):
    """One query token against attn_len cached positions: q [heads*hd] fp32, k and v
    [attn_len, kv_heads*hd] already in storage form (see to_storage).  Returns [heads*hd] fp32."""
    q = np.ascontiguousarray(q, dtype=np.float32)
    k, v = np.ascontiguousarray(k), np.ascontiguousarray(v)
    attn_len = k.shape[0]
    out = np.empty(heads * hd, dtype=np.float32)
    f32p = C.POINTER(C.c_float)
    rc = lib.cd_flash_decode(_DT[dtype], heads, kv_heads, hd, attn_len, nsplit, q.ctypes.data_as(f32p),
                             k.ctypes.data_as(C.c_void_p), v.ctypes.data_as(C.c_void_p), out.ctypes.data_as(f32p))
    if rc:
        raise CudaDecodeError(rc, lib.cd_last_error(None).decode())
    return out


# ------------------------------------------------------------------------------------------------ operators of a serving step
torch = None   # loaded by the first cache, rope or verification: flash_decode does without
_CODES = {}    # torch dtype -> CD_DTYPE_*
_current = None  # a device's current stream as an address


def _load_torch():
    global torch, _current
    if torch is None:
        import torch as loaded
        _CODES.update({loaded.float32: 0, loaded.float16: 1, loaded.bfloat16: 2})
        _current = getattr(loaded._C, "_cuda_getCurrentRawStream", None) or (lambda i: loaded.cuda.current_stream(i).cuda_stream)
        torch = loaded


def _code(t, what):
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValueError("%s must be float32, float16 or bfloat16" % what)
    return code


def _tensor(t, what, dtype, shape, index):
    """The address of a packed tensor of the given type and shape on CUDA device `index`."""
    if t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():
        raise ValueError("%s must be a contiguous %s tensor on cuda:%d" % (what, str(dtype).replace("torch.", ""), index))
    if t.shape != shape:
        raise ValueError("%s must have shape %s, got %s" % (what, list(shape), list(t.shape)))
    return t.data_ptr()


def _row_stride(t, what, rows, hd, index):
    """[rows][heads][hd] with packed heads; the distance of its rows."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != rows or shape[2] != hd:
        raise ValueError("%s must have shape [%d, heads, %d], got %s" % (what, rows, hd, list(shape)))
    if t.get_device() != index:
        raise ValueError("%s must be on cuda:%d" % (what, index))
    row, head, one = t.stride()
    if one != 1 or (head != hd and shape[1] != 1):
        raise ValueError("%s: the heads of a row must lie next to each other" % what)
    return _distance(row, what, rows)


def _distance(stride, what, rows):
    """A stride of rows for the library, where 0 is packed: rows broadcast from one are refused."""
    if rows <= 1:
        return 0
    if stride == 0:
        raise ValueError("%s: broadcast rows have to be made contiguous first" % what)
    return stride


def _counts(*counts):
    """Counts for the library's 32-bit integers, which would keep the low bits of larger ones."""
    for n in counts:
        if not -0x80000000 <= n <= 0x7fffffff:
            raise ValueError("a count must fit 32 bits, got %d" % n)


def _check(rc):
    if rc:
        raise CudaDecodeError(rc, lib.cd_last_error(None).decode())


class PagedCache:
    """The paged K and V of a batch of sequences, on the caller's tensors: pool [npages, 2, kv_heads, page_tokens, hd] (f32, f16 or
    bf16), page_table [nseq, max_pages] int32 (a row's ids in order; rows may be strided), lens [nseq] int32.  weight (f32) and
    position (int32) [nseq, kv_heads, max_pages * page_tokens] are the bookkeeping that eviction needs.  status: an int32 tensor
    of one element that collects CD_STATUS_* bits of what a call had to leave out; made here if not given."""

    def __init__(self, pool, page_table, lens, weight=None, position=None, status=None):
        _load_torch()
        if not pool.is_cuda:
            raise ValueError("the pool must be a CUDA tensor")
        if pool.dim() != 5 or pool.shape[1] != 2 or not pool.is_contiguous():
            raise ValueError("the pool must be contiguous, [npages, 2, kv_heads, page_tokens, hd]")
        self.device, self._index = pool.device, pool.device.index
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != self.device or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table must be int32 [nseq, max_pages] on the pool's device, its rows packed")
        npages, _, kv_heads, page_tokens, hd = pool.shape
        nseq, max_pages = page_table.shape
        self.nseq, self.kv_heads, self.hd, self.capacity, self.dtype = nseq, kv_heads, hd, max_pages * page_tokens, pool.dtype
        if (weight is None) != (position is None):
            raise ValueError("weight and position come together")
        self.pool, self.page_table = pool, page_table
        c = self._c = _ffi.CdPagedCache(_code(pool, "the pool"), kv_heads, hd, page_tokens, npages, nseq, max_pages, self.device.index)
        c.pool, c.page_table = pool.data_ptr(), page_table.data_ptr()
        c.table_stride = page_table.stride(0) if nseq > 1 else max_pages
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device) if status is None else status
        c.status = _tensor(self.status, "status", torch.int32, (1,), self._index)
        self._ref, self._workspaces, self._starts = C.byref(c), {}, (nseq + 1,)
        self.lens = self.weight = self.position = None
        self.replace(lens, weight, position)

    def replace(self, lens=None, weight=None, position=None):
        """Take other tensors for the lengths or the bookkeeping, as cache_evict returned them (all of those given, or none where one does not fit)."""
        shape = (self.nseq, self.kv_heads, self.capacity)
        given = [(name, t, _tensor(t, name, dtype, of, self._index)) for name, t, dtype, of in (
            ("lens", lens, torch.int32, (self.nseq,)), ("weight", weight, torch.float32, shape), ("position", position, torch.int32, shape)) if t is not None]
        for name, t, address in given:
            setattr(self, name, t)
            setattr(self._c, name, address)

    def _workspace(self, given, size, *key):
        """A workspace as `size` (one of the library's *_workspace calls) asks for it."""
        need = self._workspaces.get((size.__name__, key))
        if need is None:
            n = C.c_size_t()
            _check(size(self._ref, *key, C.byref(n)))
            if len(self._workspaces) > 256:
                self._workspaces.clear()
            need = self._workspaces[(size.__name__, key)] = n.value
        return _workspace(given, need, self.device)


def _workspace(given, need, device):
    if given is None:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if given.dtype != torch.uint8 or given.device != device or not given.is_contiguous():
        raise ValueError("the workspace must be a contiguous uint8 tensor on %s" % device)
    return given


class Rope:
    """Rotary positions: the first rot_dim elements of a head turn in pairs, "interleaved" (2i, 2i + 1) or "half" (i, i + rot_dim / 2), pair i by
    base^(-2i / rot_dim) radians a position.  scaling "linear", "ntk" or "yarn" stretches them for contexts `factor` times the
    `original` number of positions."""

    LAYOUTS = {"interleaved": 0, "half": 1}
    SCALINGS = {None: 0, "none": 0, "linear": 1, "ntk": 2, "yarn": 3}

    def __init__(self, rot_dim, base=10000.0, layout="half", scaling=None, factor=1.0, original=4096, device="cuda"):
        if layout not in self.LAYOUTS or scaling not in self.SCALINGS:
            raise ValueError("layout is one of %s, scaling one of %s" % (sorted(self.LAYOUTS), sorted(k for k in self.SCALINGS if k)))
        _load_torch()
        turns, magnitude = rope_frequencies(rot_dim, base, scaling, factor, original)
        self.turns = torch.from_numpy(turns.view(np.int64)).to(device)
        self.rot_dim, self.layout, self.magnitude = rot_dim, layout, magnitude
        self._c = _ffi.CdRope(rot_dim, self.LAYOUTS[layout], magnitude, 0, self.turns.data_ptr())
        self._ref = C.byref(self._c)


def rope_frequencies(rot_dim, base=10000.0, scaling=None, factor=1.0, original=4096):
    """(turns, magnitude): pair i turns by turns[i] / 2^64 of a circle a position (uint64 [rot_dim / 2]); on the host."""
    turns, magnitude = np.zeros(max(rot_dim // 2, 1), dtype=np.uint64), C.c_float()
    _check(lib.cd_rope_frequencies(rot_dim, base, Rope.SCALINGS[scaling], factor, original, turns.ctypes.data_as(C.POINTER(C.c_uint64)), C.byref(magnitude)))
    return turns, magnitude.value


def rope_append(cache, rope, q, k, v, positions, row_start, out=None):
    """Rotate q [rows, heads, hd] and k [rows, kv_heads, hd] at `positions` [rows] int32, write k and v to their entries in the cache (with
    bookkeeping: weight 0, the position noted), return the rotated q.  q, k and v are f32 or of the pool's type; they may be
    slices of one fused projection.  out: a packed tensor for the result; q itself where q is packed.  Rows of a sequence that does not
    fit (cache.status says so) and rows from row_start[nseq] on are not written."""
    index, hd = cache._index, cache.hd
    rows, dtype = q.shape[0], q.dtype
    sq, sk, sv = _row_stride(q, "q", rows, hd, index), _row_stride(k, "k", rows, hd, index), _row_stride(v, "v", rows, hd, index)
    if k.shape[1] != cache.kv_heads or v.shape[1] != cache.kv_heads:
        raise ValueError("k and v must have the cache's %d heads" % cache.kv_heads)
    if k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("q, k and v must have one type")
    if rope.turns.get_device() != index:
        raise ValueError("rope must be on cuda:%d" % index)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _check(lib.cd_rope_append(cache._ref, rope._ref, _code(q, "q"), q.shape[1], rows, q.data_ptr(), sq, k.data_ptr(), sk, v.data_ptr(), sv,
                              _tensor(positions, "positions", torch.int32, (rows,), index), _tensor(row_start, "row_start", torch.int32, cache._starts, index),
                              _tensor(out, "out", dtype, q.shape, index), _current(index)))
    return out


def paged_attention(cache, q, row_start, max_rows, scale=None, window=0, collect=False, lse=False, out=None, workspace=None):
    """Attention of the new rows q [rows, heads, hd] (f32 or of the pool's type) over the cache, each row up to its own entry, or over its last
    `window` entries.  scale: above 0; None: 1 / sqrt(hd).  max_rows: the most rows a sequence has.  collect: add the probabilities to cache.weight.  Returns out, or
    (out, lse [rows, heads] f32) with lse.  out: a packed tensor for the result; q itself where q is packed.  Rows of a sequence that does not fit
    (cache.status says so) and rows from row_start[nseq] on are not written.  `window` counts entries: after an eviction the places are not in order of
    position, and the last `window` of them are not the newest ones."""
    _counts(max_rows, window)
    if scale is not None and not scale > 0:
        raise ValueError("scale must be above 0, got %r" % scale)
    index = cache._index
    shape = q.shape
    rows, heads, collect = shape[0], shape[1], 1 if collect else 0
    stride = _row_stride(q, "q", rows, cache.hd, index)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    norm = torch.empty((rows, heads), dtype=torch.float32, device=cache.device) if lse else None
    ws = cache._workspace(workspace, lib.cd_paged_attention_workspace, heads, rows, max_rows, collect)
    _check(lib.cd_paged_attention(cache._ref, _code(q, "q"), heads, rows, max_rows, q.data_ptr(), stride,
                                  _tensor(row_start, "row_start", torch.int32, cache._starts, index), 0.0 if scale is None else scale, window, collect,
                                  _tensor(out, "out", q.dtype, shape, index), norm.data_ptr() if lse else None, ws.data_ptr(), ws.numel(), _current(index)))
    return (out, norm) if lse else out


def cache_evict(cache, keep, sinks=0, recent=0, out=None, workspace=None):
    """Bring every sequence with more than `keep` entries down to `keep`, each kv head by its own weights; positions below `sinks` and the
    newest `recent` ones stay.  K and V move within the cache's pages, which no two sequences may share (a common prefix has to be copied
    first), and the entries that stay are not in order of position afterwards.  Returns new (lens, weight, position), which the caller
    hands to cache.replace(); out: tensors for them (weight and position may be the cache's own, lens may not)."""
    _counts(keep, sinks, recent)
    index = cache._index
    if cache.weight is None:
        raise ValueError("the cache has no weight and position")
    lens, weight, position = out if out is not None else (torch.empty_like(cache.lens), torch.empty_like(cache.weight), torch.empty_like(cache.position))
    ws = cache._workspace(workspace, lib.cd_cache_evict_workspace, keep)
    shape = cache.weight.shape
    _check(lib.cd_cache_evict(cache._ref, keep, sinks, recent, _tensor(lens, "lens", torch.int32, cache.lens.shape, index),
                              _tensor(weight, "weight", torch.float32, shape, index), _tensor(position, "position", torch.int32, shape, index),
                              ws.data_ptr(), ws.numel(), _current(index)))
    return lens, weight, position


def verify_drafts(target, tokens, row_start, max_rows, uniforms, draws, draft=None, temperature=1.0, status=None, workspace=None):
    """Which drafted tokens stay, by given random numbers.  target [rows, vocab]: logits behind each row; tokens [rows] int32: the pending token
    of each sequence, then its drafts; uniforms [rows] and draws [nseq] f32 in [0, 1) (not used at temperature 0, and None is fine there);
    draft [rows, vocab]: the logits the token behind each row was drawn from, None: drafts without a distribution.  Returns
    (accepted [nseq] int32, out_tokens [rows] int32: the drafts that stay, the drawn token, then -1).  A sequence whose rows do not fit (row_start not
    ascending, past the rows or max_rows) is left out: accepted -1, its rows -1.  A row of logits that is needed and holds NaN or has no finite maximum:
    the drawn token is -1.  status: an int32 tensor of one element, into which such things are OR-ed as CD_STATUS_* bits.  Rows from
    row_start[nseq] on are not written."""
    _load_torch()
    _counts(max_rows)
    device, shape = target.device, target.shape
    index = device.index
    if not target.is_cuda or len(shape) != 2 or (shape[1] > 1 and target.stride(1) != 1):
        raise ValueError("target must be a CUDA tensor [rows, vocab] with packed rows")
    if draft is not None and (draft.shape != shape or draft.dtype is not target.dtype or draft.get_device() != index or (shape[1] > 1 and draft.stride(1) != 1)):
        raise ValueError("draft must be as target is")
    rows, vocab = shape
    nseq = row_start.shape[0] - 1
    starts = _tensor(row_start, "row_start", torch.int32, (nseq + 1,), index)
    accepted, out = torch.empty(nseq, dtype=torch.int32, device=device), torch.empty(rows, dtype=torch.int32, device=device)
    need = _VERIFY.get((rows, nseq, vocab))
    if need is None:
        n = C.c_size_t()
        _check(lib.cd_verify_drafts_workspace(rows, nseq, vocab, C.byref(n)))
        if len(_VERIFY) > 256:
            _VERIFY.clear()
        need = _VERIFY[(rows, nseq, vocab)] = n.value
    ws = _workspace(workspace, need, device)
    random = temperature != 0
    _check(lib.cd_verify_drafts(index, _code(target, "target"), nseq, rows, max_rows, vocab, target.data_ptr(), _distance(target.stride(0), "target", rows),
                                None if draft is None else draft.data_ptr(), 0 if draft is None else _distance(draft.stride(0), "draft", rows),
                                _tensor(tokens, "tokens", torch.int32, (rows,), index), starts,
                                _tensor(uniforms, "uniforms", torch.float32, (rows,), index) if random else None,
                                _tensor(draws, "draws", torch.float32, (nseq,), index) if random else None, temperature, accepted.data_ptr(),
                                out.data_ptr(), None if status is None else _tensor(status, "status", torch.int32, (1,), index), ws.data_ptr(), ws.numel(),
                                _current(index)))
    return accepted, out


_VERIFY = {}  # (rows, nseq, vocab) -> bytes of the workspace
