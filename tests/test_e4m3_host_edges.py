"""Calls of the 8-bit cache's host side with numbers that no cache has."""
import numpy as np
import pytest
import torch

from e4m3_batches import ALL, BATCHES, plan
from lfm25_inference_b200 import _abi, ops
from lfm25_inference_b200.cache import KvAllocationError, KvPageAllocator

FREE = 0xFFFFFFFF


def table(length=8):
    return np.full(length, FREE, dtype=np.uint32)


@pytest.mark.parametrize("tokens", [2 ** 64 - 1, 2 ** 64 - 15, 2 ** 64 - 16, 2 ** 63])
def test_more_tokens_than_pages_can_be_counted_for(tokens):
    """Rounded up to whole pages, these wrapped to none: a fork then wrote behind its table."""
    allocator = KvPageAllocator(8)
    first, second = table(), table()
    allocator.grow_sequence(0, 64, first)
    library, pair = _abi.library(), np.zeros(2, dtype=np.uint32)

    def pointer(array):
        return array.ctypes.data_as(_abi._P(_abi.ctypes.c_uint32))

    code = library.lfm25_kv_allocator_fork_sequence(allocator._handle, tokens, pointer(first), pointer(second), 8, pointer(pair))
    assert code == _abi.KV_SEQUENCE_CAPACITY_EXCEEDED and (second == FREE).all()
    with pytest.raises(KvAllocationError, match="capacity"):
        allocator.grow_sequence(64, tokens, first)
    assert allocator.snapshot()["allocated_pages"] == 4


def test_negative_numbers_are_refused():
    """... and change nothing: as size_t they are huge, and a compaction would have written that many moves."""
    allocator = KvPageAllocator(8)
    first, second = table(), table()
    allocator.grow_sequence(0, 32, first)
    allocator.grow_sequence(0, 32, second)
    allocator.release_sequence(32, first)
    before = second.copy()
    for call in (lambda: allocator.compact(second, maximum_moves=-1), lambda: allocator.fork_sequence(-1, second, first),
                 lambda: allocator.release_window(-1, 4, 0, second), lambda: allocator.release_window(32, -1, 0, second),
                 lambda: allocator.release_window(32, 4, -1, second)):
        with pytest.raises(_abi.Lfm25Error, match="negative"):
            call()
    assert np.array_equal(second, before) and allocator.snapshot()["allocated_pages"] == 2
    assert len(allocator.compact(second, maximum_moves=0)[0]) == 0
    assert len(allocator.compact(second, maximum_moves=2 ** 40)[0]) == 2      # more than there are pages


@pytest.mark.parametrize("change,message", [
    (dict(value=torch.zeros((4, 3, 16, 64), dtype=torch.uint8)), "value codes"),
    (dict(value=torch.zeros((3, 4, 16 * 64), dtype=torch.uint8)), "value codes"),
    (dict(key_scales=torch.zeros((4, 3))), "scales must have shape"),
    (dict(value_scales=torch.zeros((4, 3))), "scales must have shape"),
    (dict(value_scales=torch.zeros((12,))), "scales must have shape"),
    (dict(key=torch.zeros((3, 4, 8, 128), dtype=torch.uint8)), "codes must have shape")])
def test_arenas_whose_buffers_disagree_are_refused(change, message):
    """Buffers of the right number of elements in another order, as a transposed table of scales has, are no cache."""
    whole = ops.E4m3KvArena.new(3, 4, 64, device="cpu")
    fields = {name: getattr(whole, name) for name in ("key", "value", "key_scales", "value_scales")}
    arena = ops.E4m3KvArena(**{**fields, **change})
    rows = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(_abi.Lfm25Error, match=message):
        arena.write(rows, rows, torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("layout,form,tokens,longest", ALL)
def test_batches_take_the_form_that_they_are_tested_for(layout, form, tokens, longest):
    assert plan(tokens, *layout, longest) == form
    warps, splits = plan(tokens, *layout, longest, clusters_of_16=False)
    assert splits <= 8 and warps in (4, 8) and (splits == form[1] or form[1] == 16)


def test_every_form_has_its_batch():
    forms = {(warps, splits) for warps in (4, 8) for splits in (1, 2, 4, 8, 16)}
    assert all(set(batches) == forms for batches in BATCHES.values())
