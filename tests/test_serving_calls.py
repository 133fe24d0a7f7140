"""What the Python calls of the serving-step operators check by themselves (no GPU)."""
import pytest


def test_a_cache_takes_all_that_replace_gives_or_nothing():
    # (on host tensors, whose device index is -1: only what replace() itself does)
    import torch

    from rustane_b200 import _ffi, ops
    ops._load_torch()
    cache = object.__new__(ops.PagedCache)
    cache.nseq, cache.kv_heads, cache.capacity, cache._index, cache._c = 2, 1, 8, -1, _ffi.CdPagedCache()
    lens, weight, position = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, 8), torch.zeros(2, 1, 8, dtype=torch.int32)
    cache.replace(lens, weight, position)
    assert (cache._c.lens, cache._c.weight, cache._c.position) == (lens.data_ptr(), weight.data_ptr(), position.data_ptr())
    with pytest.raises(ValueError, match="position"):
        cache.replace(lens.clone(), weight.clone(), position.float())
    assert cache.lens is lens and cache.weight is weight and cache.position is position
    assert (cache._c.lens, cache._c.weight, cache._c.position) == (lens.data_ptr(), weight.data_ptr(), position.data_ptr())
    more = lens.clone()
    cache.replace(more)
    assert cache.lens is more and cache._c.lens == more.data_ptr() and cache.weight is weight


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan"), 0])
def test_a_scale_that_is_not_positive_is_refused(R, scale):
    # (the library takes it for its default, which is not what was asked for; ahead of everything else: no cache is looked at)
    from rustane_b200 import ops
    with pytest.raises(ValueError, match="scale"):
        ops.paged_attention(None, None, None, 1, scale=scale)
