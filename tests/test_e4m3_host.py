"""Refusals of the 8-bit cache's entry points, before anything reaches a device, and the allocator's forks, windows and
compaction."""
import ctypes

import numpy as np
import pytest
import torch

from lfm25_inference_b200 import _abi, ops
from lfm25_inference_b200._abi import Slice
from lfm25_inference_b200.cache import KvAllocationError, KvPageAllocator

FREE = 0xFFFFFFFF


def fake(elements, address=0x1000):
    """A 'device pointer' that is never read: the checks fail before any launch."""
    return Slice(address, elements)


def cache(**changes):
    fields = dict(page_size=16, num_pages=3, kv_heads=2, head_dim=64, key_codes=fake(6144), value_codes=fake(6144), key_scales=fake(6),
                  value_scales=fake(6))
    return _abi.E4m3Cache(*{**fields, **changes}.values())


def call(name, launch):
    code = getattr(_abi.library(), name)(None, ctypes.byref(launch) if launch is not None else None)
    return code, _abi.library().lfm25_last_error().decode()


def write(**changes):
    fields = dict(cache=cache(), key=fake(256), value=fake(256), slot_mapping=fake(2), num_tokens=2, kv_token_stride=0)
    return call("lfm25_kv_cache_write_e4m3", _abi.KvCacheWriteE4m3Launch(*{**fields, **changes}.values()))[0]


def norm_write(**changes):
    fields = dict(cache=cache(), query=fake(512), query_out=fake(512, 0x2000), key=fake(256), value=fake(256), query_norm=fake(64),
                  key_norm=fake(64), inv_freq=fake(32), position_ids=fake(2), slot_mapping=fake(2), num_tokens=2, query_heads=4,
                  query_token_stride=0, kv_token_stride=0, eps=1e-5)
    return call("lfm25_qk_norm_rope_kv_write_e4m3", _abi.QkNormRopeKvWriteE4m3Launch(*{**fields, **changes}.values()))[0]


def attention(name="lfm25_paged_prompt_attention_e4m3", **changes):
    fields = dict(cache=cache(), query=fake(512), block_tables=fake(8), request_slots=fake(2), position_ids=fake(2), output=fake(512),
                  num_tokens=2, query_heads=4, query_token_stride=0, block_table_stride=4, window=0, sinks=0, maximum_context_tokens=0,
                  scale=0.125, token_order=Slice(None, 0), segment_offsets=fake(2), num_segments=1)
    return call(name, _abi.PagedAttentionE4m3Launch(*{**fields, **changes}.values()))[0]


CACHE_REFUSALS = [
    (dict(page_size=8), _abi.ERR_INVALID_ARGUMENT), (dict(page_size=32), _abi.ERR_UNSUPPORTED), (dict(head_dim=96), _abi.ERR_UNSUPPORTED),
    (dict(num_pages=0), _abi.ERR_INVALID_ARGUMENT), (dict(num_pages=2 ** 33), _abi.ERR_INVALID_ARGUMENT),
    (dict(kv_heads=0), _abi.ERR_INVALID_ARGUMENT), (dict(kv_heads=1025), _abi.ERR_INVALID_ARGUMENT),
    (dict(key_codes=fake(6143)), _abi.ERR_BUFFER_TOO_SMALL), (dict(value_codes=Slice(None, 6144)), _abi.ERR_NULL_POINTER),
    (dict(value_codes=fake(6144, 0x1008)), _abi.ERR_INVALID_ARGUMENT), (dict(value_scales=fake(5)), _abi.ERR_BUFFER_TOO_SMALL),
    (dict(key_scales=fake(6, 0x1002)), _abi.ERR_INVALID_ARGUMENT)]


@pytest.mark.parametrize("changes,code", CACHE_REFUSALS)
def test_caches_that_are_refused(changes, code):
    for entry in (write, norm_write, attention, lambda **c: attention("lfm25_paged_attention_e4m3", **c)):
        assert entry(cache=cache(**changes)) == code


def test_appends_that_are_refused():
    for entry in (write, norm_write):
        assert entry(num_tokens=0) == _abi.ERR_INVALID_ARGUMENT
        assert entry(num_tokens=2 ** 31) == _abi.ERR_INVALID_ARGUMENT
        assert entry(key=fake(255)) == _abi.ERR_BUFFER_TOO_SMALL
        assert entry(value=Slice(None, 256)) == _abi.ERR_NULL_POINTER
        assert entry(value=fake(256, 0x1002)) == _abi.ERR_INVALID_ARGUMENT
        assert entry(slot_mapping=fake(1)) == _abi.ERR_BUFFER_TOO_SMALL
        assert entry(kv_token_stride=120) == entry(kv_token_stride=132) == _abi.ERR_INVALID_ARGUMENT
        assert entry(kv_token_stride=136) == _abi.ERR_BUFFER_TOO_SMALL
        assert entry(kv_token_stride=2 ** 63) == _abi.ERR_OVERFLOW or entry(kv_token_stride=2 ** 63) == _abi.ERR_BUFFER_TOO_SMALL
    assert norm_write(query_heads=0) == _abi.ERR_INVALID_ARGUMENT
    assert norm_write(query=fake(511)) == norm_write(query_out=fake(511)) == _abi.ERR_BUFFER_TOO_SMALL
    assert norm_write(query_norm=fake(63)) == norm_write(inv_freq=fake(31)) == norm_write(position_ids=fake(1)) == _abi.ERR_BUFFER_TOO_SMALL
    assert norm_write(key_norm=fake(64, 0x1004)) == _abi.ERR_INVALID_ARGUMENT
    assert norm_write(eps=float("nan")) == norm_write(eps=-1.0) == _abi.ERR_INVALID_ARGUMENT
    assert norm_write(query=fake(2048), query_out=fake(2048), query_token_stride=264) == _abi.ERR_INVALID_ARGUMENT   # in place, not dense
    for name in ("lfm25_kv_cache_write_e4m3", "lfm25_qk_norm_rope_kv_write_e4m3", "lfm25_paged_attention_e4m3", "lfm25_paged_prompt_attention_e4m3"):
        assert call(name, None)[0] == _abi.ERR_NULL_POINTER


def test_attentions_that_are_refused():
    for name in ("lfm25_paged_attention_e4m3", "lfm25_paged_prompt_attention_e4m3"):
        def entry(**changes):
            return attention(name, **changes)
        assert entry(num_tokens=0) == entry(num_tokens=2 ** 25) == _abi.ERR_INVALID_ARGUMENT
        assert entry(query_heads=0) == entry(query_heads=3) == entry(query_heads=8192) == _abi.ERR_INVALID_ARGUMENT
        assert entry(scale=0.0) == entry(scale=-1.0) == entry(scale=float("inf")) == entry(scale=float("nan")) == _abi.ERR_INVALID_ARGUMENT
        assert entry(block_table_stride=0) == entry(block_table_stride=3) == entry(block_table_stride=2 ** 29) == _abi.ERR_INVALID_ARGUMENT
        assert entry(block_tables=fake(0)) == entry(request_slots=fake(1)) == entry(position_ids=fake(1)) == _abi.ERR_BUFFER_TOO_SMALL
        assert entry(query=fake(511)) == entry(output=fake(511)) == entry(query_token_stride=264) == _abi.ERR_BUFFER_TOO_SMALL
        assert entry(query=fake(512, 0x1008)) == entry(output=fake(512, 0x1008)) == entry(query_token_stride=260) == _abi.ERR_INVALID_ARGUMENT
        assert entry(output=Slice(None, 512)) == entry(request_slots=Slice(None, 2)) == _abi.ERR_NULL_POINTER
    assert attention(num_segments=0) == _abi.ERR_INVALID_ARGUMENT
    assert attention(num_segments=2) == _abi.ERR_BUFFER_TOO_SMALL
    assert attention(segment_offsets=Slice(None, 2)) == _abi.ERR_NULL_POINTER


def test_page_copies_that_are_refused():
    library = _abi.library()

    def copy(arenas=((0x1000, 64, 4),), source=fake(1), destination=fake(1), pairs=1, count=None):
        table = (_abi.PageArena * max(1, len(arenas)))(*[_abi.PageArena(*a) for a in arenas])
        return library.lfm25_kv_pages_copy(None, table, len(arenas) if count is None else count, source, destination, pairs)

    assert copy(count=0) == copy(count=65537) == copy(pairs=0) == copy(pairs=2 ** 31) == _abi.ERR_INVALID_ARGUMENT
    assert copy(((0x1000, 0, 4),)) == copy(((0x1000, 6, 4),)) == copy(((0x1002, 8, 4),)) == copy(((0x1000, 2 ** 31, 4),)) == _abi.ERR_INVALID_ARGUMENT
    assert copy(((0x1000, 64, 0),)) == _abi.ERR_INVALID_ARGUMENT
    assert copy(((None, 64, 4),)) == copy(source=Slice(None, 1)) == _abi.ERR_NULL_POINTER
    assert copy(((0x1000, 64, 4), (0x1000, 64, 2 ** 60))) == _abi.ERR_OVERFLOW
    assert copy(destination=fake(0)) == _abi.ERR_BUFFER_TOO_SMALL


def test_python_refuses_what_it_sees():
    arena = ops.E4m3KvArena.new(2, 2, 64, device="cpu")
    rows = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(_abi.Lfm25Error, match="bfloat16"):
        ops.kv_cache_write_e4m3(rows.float(), rows.float(), arena, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(_abi.Lfm25Error, match="shape"):
        ops.kv_cache_write_e4m3(rows[:, :1], rows[:, :1], arena, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(_abi.Lfm25Error, match="requires pages"):
        ops.E4m3KvArena.new(0, device="cpu")
    with pytest.raises(_abi.Lfm25Error, match="arenas"):
        ops.kv_pages_copy([], torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(_abi.Lfm25Error, match="segments"):
        ops.paged_prompt_attention_e4m3_into(rows, arena, None, None, None, torch.zeros(1, dtype=torch.int32), rows)


# ------------------------------------------------------------------------------------------------ allocator


def table(length=8):
    return np.full(length, FREE, dtype=np.uint32)


def pages_in_use(allocator):
    return allocator.snapshot()["allocated_pages"]


@pytest.mark.parametrize("tokens,copies", [(0, 0), (1, 1), (16, 0), (17, 1), (32, 0), (47, 1)])
def test_fork(tokens, copies):
    allocator = KvPageAllocator(8)
    first, second = table(), table()
    allocator.grow_sequence(0, tokens, first)
    used = pages_in_use(allocator)
    source, destination = allocator.fork_sequence(tokens, first, second)
    assert len(source) == len(destination) == copies and pages_in_use(allocator) == used + copies
    full = tokens // 16
    assert np.array_equal(first[:full], second[:full])
    if copies:
        assert source[0] == first[full] and destination[0] == second[full] != first[full]
    allocator.release_sequence(tokens, first)
    assert pages_in_use(allocator) == full + copies          # the other branch still has them
    allocator.release_sequence(tokens, second)
    assert pages_in_use(allocator) == 0 and (second == FREE).all()


def test_forks_that_are_refused_change_nothing():
    allocator = KvPageAllocator(3)
    first, second = table(), table()
    allocator.grow_sequence(0, 40, first)
    with pytest.raises(KvAllocationError, match="exhausted"):
        allocator.fork_sequence(40, first, second)             # no page left for the last one
    assert (second == FREE).all() and pages_in_use(allocator) == 3
    with pytest.raises(KvAllocationError, match="capacity"):
        allocator.fork_sequence(32, first, table(1))
    with pytest.raises(KvAllocationError, match="capacity"):
        allocator.fork_sequence(200, first, table(20))
    with pytest.raises(_abi.Lfm25Error, match="holds pages"):
        allocator.fork_sequence(32, first, first)
    with pytest.raises(KvAllocationError, match="exhausted"):
        allocator.fork_sequence(16, np.full(8, 2 ** 31, dtype=np.uint32), second)
    allocator.release_sequence(40, first)
    assert pages_in_use(allocator) == 0


@pytest.mark.parametrize("tokens,window,sinks,kept", [
    (100, 0, 0, [0, 1, 2, 3, 4, 5, 6]), (100, 100, 0, [0, 1, 2, 3, 4, 5, 6]), (100, 53, 0, [3, 4, 5, 6]), (100, 54, 0, [2, 3, 4, 5, 6]),
    (100, 53, 1, [0, 3, 4, 5, 6]), (100, 53, 17, [0, 1, 3, 4, 5, 6]), (100, 1, 0, [6]), (112, 1, 0, []), (100, 5, 10 ** 6, [0, 1, 2, 3, 4, 5, 6])])
def test_release_behind_a_window(tokens, window, sinks, kept):
    """Exactly the pages without a key that the next token (or a later one) sees go; its own page stays where it is begun."""
    allocator = KvPageAllocator(8)
    pages = table()
    allocator.grow_sequence(0, tokens, pages)
    before = pages.copy()
    released = allocator.release_window(tokens, window, sinks, pages)
    visible = {key // 16 for key in range(tokens + 1) if window == 0 or key > tokens - window or key < sinks}
    assert kept == sorted(visible & set(range(7)))
    assert [i for i in range(7) if pages[i] != FREE] == kept and released == 7 - len(kept)
    assert all(pages[i] == before[i] for i in kept)
    assert allocator.release_window(tokens, window, sinks, pages) == 0
    allocator.release_sequence(tokens, pages)
    assert pages_in_use(allocator) == 0


def test_fork_of_pages_of_32_tokens():
    allocator = KvPageAllocator(5, 32)
    first, second = table(2), table(2)
    allocator.grow_sequence(0, 50, first)
    source, destination = allocator.fork_sequence(50, first, second)
    assert source.tolist() == [first[1]] and destination.tolist() == [second[1]] and second[0] == first[0]
    with pytest.raises(KvAllocationError):
        allocator.fork_sequence(65, first, table(4))           # more than the source's table holds


def test_fork_of_a_sequence_behind_a_window():
    allocator = KvPageAllocator(12)
    first, second = table(), table()
    allocator.grow_sequence(0, 100, first)
    allocator.release_window(100, 40, 3, first)
    source, _ = allocator.fork_sequence(100, first, second)
    assert len(source) == 1 and np.array_equal(first[:6], second[:6]) and (second[1:3] == FREE).all()
    allocator.release_sequence(100, first)
    allocator.release_sequence(100, second)
    assert pages_in_use(allocator) == 0


def test_compaction():
    allocator = KvPageAllocator(16)
    tables = np.full((4, 4), FREE, dtype=np.uint32)
    for row in range(4):
        allocator.grow_sequence(0, 64, tables[row])
    allocator.release_sequence(64, tables[0])
    allocator.release_sequence(64, tables[2])
    allocator.pin_cached_pages([15])                         # a prefix cache holds the last page: it stays
    contents = {page: page for page in range(16)}            # page -> what it holds
    before = tables.copy()
    source, destination = allocator.compact(tables, maximum_moves=2)
    more = allocator.compact(tables)
    source, destination = np.concatenate((source, more[0])), np.concatenate((destination, more[1]))
    assert set(source) == {14, 13, 12, 7} and sorted(destination) == [0, 1, 2, 3]
    for s, d in zip(source, destination):
        contents[d] = contents[s]
    held = before != FREE
    assert np.array_equal(held, tables != FREE)
    assert [contents[p] for p in tables[held]] == list(before[held])
    assert len(allocator.compact(tables)[0]) == 0
    fresh = table()
    allocator.grow_sequence(0, 48, fresh)
    assert list(fresh[:3]) == [7, 8, 9]                      # the lowest free pages first
    for row in (1, 3):
        allocator.release_sequence(64, tables[row])
    allocator.release_sequence(48, fresh)
    assert pages_in_use(allocator) == 1                      # the pinned one


def test_compaction_keeps_shared_pages_together():
    allocator = KvPageAllocator(10)
    tables = np.full((3, 4), FREE, dtype=np.uint32)
    allocator.grow_sequence(0, 64, tables[0])
    allocator.grow_sequence(0, 32, tables[1])
    allocator.fork_sequence(32, tables[1], tables[2])
    allocator.release_sequence(64, tables[0])
    # only one branch's table is given: its pages have a reference that is not in it, and stay
    assert len(allocator.compact(tables[1])[0]) == 0
    source, destination = allocator.compact(tables)
    assert sorted(source) == [4, 5] and sorted(destination) == [0, 1]
    assert np.array_equal(tables[1], tables[2]) and sorted(tables[1][:2]) == [0, 1]
    for row in (1, 2):
        allocator.release_sequence(32, tables[row])
    assert pages_in_use(allocator) == 0
