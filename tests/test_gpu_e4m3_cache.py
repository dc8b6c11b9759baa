"""The 8-bit paged key/value cache: append, attention of tokens and of prompts, page copies, against definitions in 64 bits."""
import numpy as np
import pytest
import torch

import e4m3_cases as plain
from conftest import to_i64, to_u32
from lfm25_inference_b200 import ops
from lfm25_inference_b200.cache import FixedBlockTables, KvPageAllocator

pytestmark = pytest.mark.gpu

F16_WEIGHTS, BF16_WEIGHTS = 2.0 ** -11, 2.0 ** -8
PAGE = plain.PAGE


def bf16(array, device):
    return torch.from_numpy(np.ascontiguousarray(array, dtype=np.float32)).to(device).to(torch.bfloat16)


def host(tensor):
    return tensor.detach().float().cpu().numpy().astype(np.float64)


def arena_of(codes, scales, device):
    key, value = (torch.from_numpy(c).to(device) for c in codes)
    return ops.E4m3KvArena(key, value, *(torch.from_numpy(s.astype(np.float32)).to(device) for s in scales))


def random_cache(rng, pages, heads, dim, device, low=-9, high=-4, nan=False):
    codes = [rng.integers(0, 256, (pages, heads, PAGE, dim), dtype=np.uint8) for _ in range(2)]
    if not nan:
        for c in codes:
            c[(c & 0x7F) == 0x7F] = 0
    scales = [np.exp2(rng.integers(low, high, (pages, heads)).astype(np.float64)) for _ in range(2)]
    return arena_of(codes, scales, device), plain.Cache(codes[0], scales[0]), plain.Cache(codes[1], scales[1])


def assert_codes(tensor, scales, want):
    got = plain.CODE_VALUES[tensor.cpu().numpy()]
    assert np.array_equal(scales.cpu().numpy().astype(np.float64), want.scales)
    assert np.array_equal(got, want.values, equal_nan=True)


# ------------------------------------------------------------------------------------------------ append


def segments_of(rng, lengths, starts, pages):
    """Slots of segments at given positions, each in pages of its own, and the pool they need."""
    order, at, slots = rng.permutation(pages), 0, []
    for length, start in zip(lengths, starts):
        need = -(-(start + length) // PAGE)
        table = order[at:at + need]
        at += need
        slots += [table[p // PAGE] * PAGE + p % PAGE for p in range(start, start + length)]
    return np.array(slots, dtype=np.int64)


@pytest.mark.parametrize("heads,dim", [(8, 64), (2, 128), (1, 64), (3, 128), (40, 64)])
@pytest.mark.parametrize("lengths,starts", [
    ((1,), (0,)), ((1,), (15,)), ((1, 1, 1), (4, 16, 31)), ((3, 40, 17), (13, 0, 15)), ((16,), (16,)), ((1,) * 130, tuple(range(130))),
    ((700, 333), (5, 0)), ((15, 1, 31), (1, 15, 17))])
def test_append_is_exact(device, heads, dim, lengths, starts):
    rng = np.random.default_rng(sum(lengths) + dim + heads)
    pages = sum(-(-(a + b) // PAGE) for a, b in zip(lengths, starts)) + 2
    arena, key, value = random_cache(rng, pages, heads, dim, device)
    slots = segments_of(rng, lengths, starts, pages)
    # magnitudes over many powers of two, so that scales stay, grow a little and grow a lot
    rows = [rng.standard_normal((len(slots), heads, dim)) * np.exp2(rng.integers(-14, 9, (len(slots), heads, 1))) for _ in range(2)]
    tensors = [bf16(r, device) for r in rows]
    ops.kv_cache_write_e4m3(*tensors, arena, to_i64(slots, device))
    key.append(host(tensors[0]), slots)
    value.append(host(tensors[1]), slots)
    assert_codes(arena.key, arena.key_scales, key)
    assert_codes(arena.value, arena.value_scales, value)


def test_append_of_strided_rows_skipped_tokens_and_odd_values(device):
    rng = np.random.default_rng(5)
    arena, key, value = random_cache(rng, 5, 2, 64, device)
    slots = np.array([-1, 18, 19, 5 * PAGE, 36, -7, 48, 49, 50, 2 ** 40, 0, 1, 79], dtype=np.int64)
    packed = rng.standard_normal((len(slots), 40 + 4 * 64))
    packed[7, 40:40 + 64] = 0
    packed[8, 45], packed[8, 46], packed[8, 200] = np.inf, np.nan, -np.inf
    packed[10:12, 40:104] = 0                     # a page of zeros only
    packed[12] *= 1e30
    packed = bf16(packed, device)
    parts = packed[:, 40:168].view(-1, 2, 64), packed[:, 168:].view(-1, 2, 64)
    arena.write(*parts, to_i64(slots, device))
    key.append(host(parts[0]), slots)
    value.append(host(parts[1]), slots)
    assert_codes(arena.key, arena.key_scales, key)
    assert_codes(arena.value, arena.value_scales, value)


def test_scales_at_their_borders(device):
    """448 * 2^e keeps 2^e, the next bf16 value takes 2^(e + 1); the least and the largest magnitudes there are."""
    rows = []
    for value in (448.0, 450.0, 1.75 * 2.0 ** -30, 2.0 ** -133, 2.0 ** -118, 3.38e38, 0.0, 1.0):
        row = np.zeros((1, 1, 64))
        row[0, 0, 7] = -value
        rows.append(row)
    key = bf16(np.concatenate(rows), device)
    arena = ops.E4m3KvArena.new(8, 1, 64, device=device)
    slots = np.arange(8, dtype=np.int64) * PAGE + np.array([0, 3] * 4)          # fresh pages and, on the zeros of a new arena, continued ones
    ops.kv_cache_write_e4m3(key, key, arena, to_i64(slots, device))
    want = plain.Cache(np.zeros((8, 1, PAGE, 64), dtype=np.uint8), np.zeros((8, 1)))
    want.append(host(key), slots)
    assert_codes(arena.key, arena.key_scales, want)
    assert_codes(arena.value, arena.value_scales, want)


@pytest.mark.parametrize("heads,kv_heads,dim,tokens,first", [(32, 8, 64, 1, 0), (8, 2, 128, 40, 9), (12, 4, 64, 700, 100000), (5, 1, 128, 3, 2 ** 31)])
def test_norm_and_rotation_in_front_of_the_append(device, heads, kv_heads, dim, tokens, first):
    rng = np.random.default_rng(dim + tokens)
    eps = 1e-5
    pages = -(-tokens // PAGE) + 1
    arena, key_cache, value_cache = random_cache(rng, pages, kv_heads, dim, device)
    slots = np.arange(tokens, dtype=np.int64) + 3
    if tokens > 1:
        slots[min(12, tokens - 1)] = -1                  # the last of its page; its query is written all the same
    positions = np.arange(first, first + tokens, dtype=np.uint32)
    packed = bf16(rng.standard_normal((tokens, (heads + 2 * kv_heads) * dim)) * np.exp2(rng.integers(-6, 6, (tokens, 1))), device)
    query, key, value = (part.view(tokens, -1, dim) for part in packed.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    weights = [bf16(1 + 0.3 * rng.standard_normal(dim), device) for _ in range(2)]
    inv_freq = torch.from_numpy((1e6 ** (-np.arange(0, dim, 2) / dim)).astype(np.float32)).to(device)
    out = torch.empty((tokens, heads, dim), dtype=torch.bfloat16, device=device)
    ops.qk_norm_rope_kv_write_e4m3(query, key, value, *weights, inv_freq, to_u32(positions, device), to_i64(slots, device), arena, eps,
                                   query_out=out)
    want_query = plain.norm_rope(host(query), host(weights[0]), inv_freq.cpu().numpy(), positions, eps)
    want_key = plain.norm_rope(host(key), host(weights[1]), inv_freq.cpu().numpy(), positions, eps)
    # f32 in front of the rounding: dim squares and a handful of products, an angle of 2^-22 at most off
    def slack(x):
        half = dim // 2
        other = np.concatenate((x[:, :, half:], x[:, :, :half]), axis=2)
        return (dim / 2 + 16) * 2.0 ** -24 * (np.abs(x) + np.abs(other)) * 2
    assert np.all(np.abs(host(out) - want_query) <= 2.0 ** -8 * np.abs(want_query) + slack(want_query) * (1 + 2.0 ** -8))
    # a value that is rounded to E4M3: half a step, and what f32 is off may cross to the next one
    scales = arena.key_scales.cpu().numpy().astype(np.float64)
    got = plain.CODE_VALUES[arena.key.cpu().numpy()] * scales[:, :, None, None]
    for token, slot in enumerate(slots):
        if slot >= 0:
            page, offset = slot // PAGE, slot % PAGE
            error = np.abs(got[page, :, offset] - want_key[token])
            # values of pages that grew later were rounded twice
            bound = 2 * (2.0 ** -4 * np.abs(want_key[token]) + 2.0 ** -10 * scales[page][:, None]) + 2 * slack(want_key)[token]
            assert np.all(error <= bound)
    value_cache.append(host(value), slots)
    assert_codes(arena.value, arena.value_scales, value_cache)
    # scales from the exact keys, where those are not within f32's error of a border
    for shift in (1 - 2.0 ** -16, 1 + 2.0 ** -16):
        shifted = plain.Cache(np.zeros(arena.key.shape, dtype=np.uint8), key_cache.scales)
        shifted.append(want_key * shift, slots)
        if shift < 1:
            least = shifted.scales
    touched = (least != key_cache.scales) | (least == scales)
    assert np.all((scales == least) | (scales == shifted.scales)) and touched.any()


def test_norm_and_rotation_in_place(device):
    rng = np.random.default_rng(2)
    query = bf16(rng.standard_normal((17, 4, 64)), device)
    key = bf16(rng.standard_normal((17, 2, 64)), device)
    weight = bf16(np.ones(64), device)
    inv_freq = torch.ones(32, device=device)
    positions, slots = to_u32(np.arange(17), device), to_i64(np.arange(17), device)
    arenas = [ops.E4m3KvArena.new(2, 2, 64, device=device) for _ in range(2)]
    out = torch.empty_like(query)
    ops.qk_norm_rope_kv_write_e4m3(query, key, key, weight, weight, inv_freq, positions, slots, arenas[0], 1e-6, query_out=out)
    ops.qk_norm_rope_kv_write_e4m3(query, key, key, weight, weight, inv_freq, positions, slots, arenas[1], 1e-6)
    assert torch.equal(query, out)
    assert all(torch.equal(a, b) for a, b in zip(arenas[0].tensors(), arenas[1].tensors()))


# ------------------------------------------------------------------------------------------------ attention


def tables_of(rng, contexts, pool, spare_columns=0):
    stride = max(-(-c // PAGE) for c in contexts) + spare_columns
    order, at = rng.permutation(pool), 0
    tables = np.full((len(contexts), stride), plain.UNASSIGNED, dtype=np.int64)
    for row, context in enumerate(contexts):
        need = -(-context // PAGE)
        tables[row, :need] = order[at:at + need]
        at += need
    return tables


def pool_of(contexts):
    return sum(-(-c // PAGE) for c in contexts) + 2


def check_attention(got, query, cache, tables, rows, positions, rounding, before, **rule):
    exact, magnitude, score = plain.attend(host(query), cache[0].full(), cache[1].full(), tables, rows, positions, **rule)
    error = np.abs(host(got) - exact)
    bound = plain.tolerance(exact, magnitude, score, query.shape[2], rounding)
    without = np.isnan(exact).all(axis=(1, 2))
    assert torch.equal(got[torch.from_numpy(without)], before[torch.from_numpy(without)])
    worst = np.nanmax(np.where(without[:, None, None], 0, error / bound))
    assert not np.isnan(host(got)[~without]).any() and worst <= 1, f"error over its bound: {worst}"


LAYOUTS = [(32, 8, 64), (8, 2, 128), (3, 3, 64), (9, 1, 64), (16, 1, 128), (40, 2, 64), (35, 1, 128), (10, 2, 128)]


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("contexts,window,sinks", [
    ((1,), 0, 0), ((1, 15, 16, 17, 300), 0, 0), ((2049, 5, 777), 0, 0), ((1, 40, 500, 333), 1, 0), ((40, 500, 97), 33, 4),
    ((600, 31, 16), 100, 40), ((700,), 17, 500), ((64, 65, 80), 64, 16)])
def test_decode_attention(device, heads, kv_heads, dim, contexts, window, sinks):
    rng = np.random.default_rng(heads * dim + sum(contexts))
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, kv_heads, dim, device)
    tables = tables_of(rng, contexts, pool, spare_columns=1)
    order = rng.permutation(len(contexts))
    rows = np.concatenate((order, [len(contexts) + 3, plain.UNASSIGNED]))       # two tokens that belong to nobody
    positions = np.concatenate((np.array(contexts)[order] - 1, [0, 0]))
    query = bf16(rng.standard_normal((len(rows), heads, dim)) * 0.5, device)
    for longest in (0, max(contexts)):
        out = bf16(rng.standard_normal(query.shape), device)
        before = out.clone()
        ops.paged_attention_e4m3_into(query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device), out,
                                      window=window, sinks=sinks, maximum_context_tokens=longest)
        check_attention(out, query, cache, tables, rows, positions, F16_WEIGHTS, before, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("segments,window,sinks", [
    (((0, 1),), 0, 0), (((0, 17), (33, 1), (5, 40)), 0, 0), (((100, 65), (0, 130)), 0, 0), (((0, 70), (300, 33)), 20, 3),
    (((250, 40),), 100, 90), (((1000, 3),), 0, 0), (((0, 64), (64, 64)), 64, 0), (((500, 9), (0, 2)), 1, 1)])
def test_prompt_attention(device, heads, kv_heads, dim, segments, window, sinks):
    rng = np.random.default_rng(heads * dim + segments[0][1])
    contexts = [prefix + count for prefix, count in segments]
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, kv_heads, dim, device)
    tables = tables_of(rng, contexts, pool)
    lead = 3                                                    # tokens in front of the first segment and behind the last: nobody's
    rows = np.concatenate([np.zeros(lead, dtype=np.int64)] + [np.full(count, row) for row, (_, count) in enumerate(segments)] + [[0]])
    positions = np.concatenate([np.zeros(lead, dtype=np.int64)] + [np.arange(prefix, prefix + count) for prefix, count in segments] + [[0]])
    offsets = lead + np.concatenate(([0], np.cumsum([count for _, count in segments])))
    query = bf16(rng.standard_normal((len(rows), heads, dim)) * 0.5, device)
    out = bf16(rng.standard_normal(query.shape), device)
    before = out.clone()
    ops.paged_prompt_attention_e4m3_into(query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device),
                                         to_u32(offsets, device), out, window=window, sinks=sinks)
    nobody = np.concatenate((np.full(lead, len(tables)), rows[lead:-1], [len(tables)]))
    check_attention(out, query, cache, tables, nobody, positions, BF16_WEIGHTS, before, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 64), (32, 8, 128)])
def test_prompt_attention_of_more_tiles_than_run_at_once(device, heads, kv_heads, dim):
    """Six portions, 240 CTAs; every 41st token is compared, twice: behind other kernels and behind the call itself."""
    rng = np.random.default_rng(dim)
    segments = ((0, 300), (17, 301), (400, 290), (800, 257), (64, 320), (1200, 300))
    contexts = [prefix + count for prefix, count in segments]
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, kv_heads, dim, device)
    tables = tables_of(rng, contexts, pool)
    rows = np.concatenate([np.full(count, row) for row, (_, count) in enumerate(segments)])
    positions = np.concatenate([np.arange(prefix, prefix + count) for prefix, count in segments])
    query = bf16(rng.standard_normal((len(rows), heads, dim)) * 0.5, device)
    arguments = [to_u32(values, device) for values in (tables, rows, positions, np.concatenate(([0], np.cumsum([c for _, c in segments]))))]
    some = np.arange(5, len(rows), 41)
    outs = [torch.zeros_like(query) for _ in range(3)]
    for out in outs:
        ops.paged_prompt_attention_e4m3_into(query, arena, *arguments, out)
    check_attention(outs[0][some], query[some], cache, tables, rows[some], positions[some], BF16_WEIGHTS, outs[0][some])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("contexts", [(60001,), (9000, 16500, 12345, 8191)])
def test_decode_attention_of_few_long_contexts(device, contexts):
    rng = np.random.default_rng(len(contexts))
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, 8, 64, device)
    tables = tables_of(rng, contexts, pool)
    rows, positions = np.arange(len(contexts)), np.array(contexts) - 1
    query = bf16(rng.standard_normal((len(rows), 32, 64)) * 0.5, device)
    out = torch.zeros_like(query)
    ops.paged_attention_e4m3_into(query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device), out)
    check_attention(out, query, cache, tables, rows, positions, F16_WEIGHTS, out)


def attention_call(kind, query, arena, tables, rows, positions, out, **rule):
    if kind == "decode":
        ops.paged_attention_e4m3_into(query, arena, tables, rows, positions, out, **rule)
    else:
        offsets = torch.arange(query.shape[0] + 1, dtype=torch.int32, device=query.device)
        ops.paged_prompt_attention_e4m3_into(query, arena, tables, rows, positions, offsets, out, **rule)


@pytest.mark.parametrize("kind", ["decode", "prompts"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (21, 5)])
def test_what_is_not_seen_may_hold_anything(device, kind, window, sinks):
    """NaN codes behind the position, in front of the window and in pages between first tokens and window, of which some are
    unassigned, change nothing."""
    rng = np.random.default_rng(8)
    contexts = (70, 131, 9)
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, 2, 64, device)
    tables = tables_of(rng, contexts, pool)
    rows, positions = np.arange(3), np.array(contexts) - 1
    query = bf16(rng.standard_normal((3, 8, 64)), device)
    outs = []
    for stray in (False, True):
        if stray:
            for row, context in enumerate(contexts):
                for key in range(-(-context // PAGE) * PAGE):
                    if key >= context or (window and key <= context - 1 - window and key >= sinks):
                        for codes in (arena.key, arena.value):
                            codes[tables[row, key // PAGE], :, key % PAGE] = 0x7F
            if window:
                tables[1, 2:5] = plain.UNASSIGNED
                tables[0, 1] = pool + 7
        out = torch.zeros_like(query)
        attention_call(kind, query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device), out, window=window, sinks=sinks)
        outs.append(out)
    assert torch.equal(*outs) and not outs[0].isnan().any() and outs[0].any()


@pytest.mark.parametrize("kind", ["decode", "prompts"])
@pytest.mark.parametrize("stray", [float("nan"), float("inf"), -1.0])
def test_pages_of_nobody_may_hold_anything(device, kind, stray):
    """A sequence of an odd number of pages next to pages with NaN codes and stray scales, the first page of the pool among them."""
    rng = np.random.default_rng(17)
    arena, *cache = random_cache(rng, 8, 2, 64, device)
    for tensor in (arena.key, arena.value):
        tensor[[0, 7]] = 0x7F
    for tensor in (arena.key_scales, arena.value_scales):
        tensor[[0, 7]] = stray
    tables = np.array([[1, 2, 3, 4, 5, plain.UNASSIGNED], [6, plain.UNASSIGNED] + [7] * 4])
    rows, positions = np.arange(2), np.array([70, 3])
    query = bf16(rng.standard_normal((2, 8, 64)), device)
    out = torch.zeros_like(query)
    attention_call(kind, query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device), out)
    for part in cache:
        part.values[[0, 7]] = 0
    check_attention(out, query, cache, tables, rows, positions, F16_WEIGHTS if kind == "decode" else BF16_WEIGHTS, out)


@pytest.mark.parametrize("kind", ["decode", "prompts"])
def test_unassigned_pages_leave_the_row(device, kind):
    """... of the tokens that see them, and of no others."""
    rng = np.random.default_rng(9)
    contexts = (70, 2131, 9, 40)
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, 2, 128, device)
    tables = tables_of(rng, contexts, pool)
    tables[1, 77], tables[3, 0] = plain.UNASSIGNED, pool
    rows, positions = np.arange(4), np.array(contexts) - 1
    positions[2] = tables.shape[1] * PAGE                       # beyond the tables
    query = bf16(rng.standard_normal((4, 8, 128)), device)
    out = torch.full_like(query, 3.0)
    attention_call(kind, query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device), out)
    assert (out[1:] == 3.0).all() and (out[0] != 3.0).any()


@pytest.mark.parametrize("window", [0, 12])
def test_prompt_rows_see_their_own_nan_and_missing_pages_only(device, window):
    rng = np.random.default_rng(16)
    contexts = (200,)
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, 2, 64, device)
    tables = tables_of(rng, contexts, pool)
    first, count = 100, 100
    arena.value[tables[0, 150 // PAGE], 1, 150 % PAGE, 17] = 0xFF            # one NaN of KV head 1
    arena.key[tables[0, 170 // PAGE], 0, 170 % PAGE, 3] = 0x7F
    tables[0, 12] = plain.UNASSIGNED                                        # keys 192 ..
    rows, positions = np.zeros(count, dtype=np.int64), np.arange(first, first + count)
    query = bf16(rng.standard_normal((count, 4, 64)), device)
    out = torch.full_like(query, 3.0)
    ops.paged_prompt_attention_e4m3_into(query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device),
                                         to_u32([0, count], device), out, window=window)
    got = host(out)
    last = 191                                                # positions behind it see the page that is missing
    sees = lambda key: (positions >= key) & ((positions < key + window) if window else True)    # noqa: E731
    assert (got[positions > last] == 3.0).all()
    rest = positions <= last
    assert np.array_equal(np.isnan(got[rest, 2:]).all(2).all(1), sees(150)[rest])
    assert np.array_equal(np.isnan(got[rest, :2]).all(2).all(1), sees(170)[rest])
    for heads, key in ((slice(0, 2), 170), (slice(2, 4), 150)):
        keep = rest & ~sees(key)
        exact, magnitude, score = plain.attend(host(query)[keep], np.nan_to_num(cache[0].full()), np.nan_to_num(cache[1].full()), tables,
                                               rows[keep], positions[keep], window=window)
        bound = plain.tolerance(exact, magnitude, score, 64, BF16_WEIGHTS)
        assert np.all(np.abs(got[keep] - exact)[:, heads] <= bound[:, heads])


@pytest.mark.parametrize("kind,rounding", [("decode", F16_WEIGHTS), ("prompts", BF16_WEIGHTS)])
def test_scales_and_queries_of_any_size(device, kind, rounding):
    """Scales over hundreds of powers of two within one context, queries near both ends of what f16 holds and beyond."""
    rng = np.random.default_rng(10)
    contexts = (333, 64)
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, 2, 64, device, low=-60, high=40)
    arena.key_scales.fill_(2.0 ** -8)
    cache[0].scales[:] = 2.0 ** -8
    tables = tables_of(rng, contexts, pool)
    rows, positions = np.arange(2), np.array(contexts) - 1
    for size, scale in ((2.0 ** -100, 2.0 ** 99), (2.0 ** 60, 2.0 ** -62), (1.0, None)):
        query = bf16(rng.standard_normal((2, 8, 64)) * size, device)
        out = torch.zeros_like(query)
        attention_call(kind, query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device), out, scale=scale)
        check_attention(out, query, cache, tables, rows, positions, rounding, out, scale=scale)


@pytest.mark.parametrize("kind,rounding", [("decode", F16_WEIGHTS), ("prompts", BF16_WEIGHTS)])
def test_growing_maxima(device, kind, rounding):
    """Scores that rise by a few from page to page move the reference of the weights again and again, peaks take nearly all."""
    rng = np.random.default_rng(11)
    context = 900
    pool = pool_of((context,))
    arena, *cache = random_cache(rng, pool, 1, 64, device, low=-9, high=-8)
    tables = tables_of(rng, (context,), pool)
    for logical in range(tables.shape[1]):
        scale = 2.0 ** (-12 + logical // 6)
        arena.key_scales[tables[0, logical]] = scale
        cache[0].scales[tables[0, logical]] = scale
    query = bf16(rng.standard_normal((1, 4, 64)) * 0.3, device)
    out = torch.zeros_like(query)
    attention_call(kind, query, arena, to_u32(tables, device), to_u32([0], device), to_u32([context - 1], device), out)
    check_attention(out, query, cache, tables, [0], [context - 1], rounding, out)


def test_strided_queries_and_token_order(device):
    rng = np.random.default_rng(12)
    contexts = (100, 7, 1500)
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, 4, 64, device)
    tables = tables_of(rng, contexts, pool)
    rows, positions = np.arange(3), np.array(contexts) - 1
    packed = bf16(rng.standard_normal((3, 12 * 64 + 72)), device)
    query = packed[:, 8:8 + 12 * 64].view(3, 12, 64)
    outs = []
    for given, order in ((query, None), (query.contiguous(), [2, 0, 1])):
        out = torch.zeros((3, 12, 64), dtype=torch.bfloat16, device=device)
        ops.paged_attention_e4m3_into(given, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device), out,
                                      token_order=None if order is None else to_u32(order, device))
        outs.append(out)
    assert torch.equal(*outs)
    check_attention(outs[0], query, cache, tables, rows, positions, F16_WEIGHTS, outs[0])
    out = torch.zeros_like(outs[0])
    attention_call("prompts", query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device), out)
    check_attention(out, query, cache, tables, rows, positions, BF16_WEIGHTS, out)


def test_offsets_beyond_32_bits(device):
    """Pages in the upper half of a cache of more than 4 GiB a side."""
    pages = 2 ** 32 // (8 * PAGE * 128) + 9
    arena = ops.E4m3KvArena(*(torch.empty((pages, 8, PAGE, 128), dtype=torch.uint8, device=device) for _ in range(2)),
                            *(torch.empty((pages, 8), dtype=torch.float32, device=device) for _ in range(2)))
    rng = np.random.default_rng(13)
    small = ops.E4m3KvArena.new(9, 8, 128, device=device)
    first = pages - 9
    rows = [bf16(rng.standard_normal((9 * PAGE, 8, 128)), device) for _ in range(2)]
    arena.write(*rows, to_i64(np.arange(9 * PAGE) + first * PAGE, device))
    small.write(*rows, to_i64(np.arange(9 * PAGE), device))
    for big, little in zip(arena.tensors(), small.tensors()):
        assert torch.equal(big[first:], little)
    query = bf16(rng.standard_normal((5, 8, 128)), device)
    slots, positions = to_u32(np.zeros(5), device), to_u32(np.arange(5) + 130, device)
    for kind in ("decode", "prompts"):
        outs = []
        for where, base in ((arena, first), (small, 0)):
            out = torch.zeros_like(query)
            attention_call(kind, query, where, to_u32(base + np.arange(9)[None], device), slots, positions, out)
            outs.append(out)
        assert torch.equal(*outs) and outs[0].any()
    ops.kv_pages_copy(arena.tensors(), to_u32([first + 1, first + 2], device), to_u32([first + 8, 0], device))
    assert torch.equal(arena.key[0], small.key[2]) and torch.equal(arena.value[pages - 1], small.value[1])


@pytest.mark.parametrize("kind", ["decode", "prompts"])
def test_two_graphs_at_once_on_streams_of_their_own(device, kind):
    """Captured calls share nothing: two of them replayed side by side give what each gives by itself."""
    rng = np.random.default_rng(14)
    contexts = (3000, 50)
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, 2, 64, device)
    tables = to_u32(tables_of(rng, contexts, pool), device)
    rows, positions = to_u32([0, 1], device), to_u32(np.array(contexts) - 1, device)
    graphs, outs, wants, streams = [], [], [], [torch.cuda.Stream(device) for _ in range(2)]
    offsets = torch.arange(3, dtype=torch.int32, device=device)
    for stream in streams:
        query = bf16(rng.standard_normal((2, 8, 64)), device)
        out, want = torch.zeros_like(query), torch.zeros_like(query)

        def call(target):
            if kind == "decode":
                ops.paged_attention_e4m3_into(query, arena, tables, rows, positions, target)
            else:
                ops.paged_prompt_attention_e4m3_into(query, arena, tables, rows, positions, offsets, target)
        call(want)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(out)
        graphs.append((graph, query))
        outs.append(out)
        wants.append(want)
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and a.any() for a, b in zip(outs, wants))


def test_a_wait_that_runs_out_leaves_the_rows(device, library_option):
    """One warp that brings pages never reports its first stage: the waits end after their limit, the status words say so, no row
    is written, and the next call is as ever."""
    rng = np.random.default_rng(15)
    arena, *cache = random_cache(rng, 9, 2, 64, device)
    tables = np.arange(9)[None]
    query = bf16(rng.standard_normal((20, 8, 64)), device)
    given = to_u32(tables, device), to_u32(np.zeros(20), device), to_u32(np.arange(20) + 70, device), to_u32([0, 20], device)
    out = torch.full_like(query, 3.0)
    ops.device_status()
    library_option("wait_limit_ns", 2_000_000)
    library_option("wait_selftest_drop", 1)
    ops.paged_prompt_attention_e4m3_into(query, arena, *given, out)
    torch.cuda.synchronize()
    waits, tag, *_ = ops.device_status()
    assert waits > 0 and tag == 10 and (out == 3.0).all()
    library_option("wait_selftest_drop", 0)
    library_option("wait_limit_ns", 1_000_000_000)
    ops.paged_prompt_attention_e4m3_into(query, arena, *given, out)
    check_attention(out, query, cache, tables, np.zeros(20, dtype=int), np.arange(20) + 70, BF16_WEIGHTS, out)
    assert ops.device_status()[0] == 0


# ------------------------------------------------------------------------------------------------ pages


@pytest.mark.parametrize("shape,dtype,layers", [((8, 16, 64), torch.bfloat16, 3), ((8, 16, 64), torch.uint8, 1), ((3,), torch.float32, 70),
                                                ((1,), torch.float32, 1), ((5, 16, 128), torch.uint8, 2), ((33,), torch.int32, 2)])
def test_pages_copy(device, shape, dtype, layers):
    generator = torch.Generator(device=device).manual_seed(3)
    pool = 50
    store = torch.randint(0, 100, (layers, pool, *shape), generator=generator, device=device).to(dtype)
    want = store.clone()
    order = torch.randperm(pool, generator=generator, device=device)
    source, destination = order[:17], order[17:34].clone()
    want[:, destination] = want[:, source]
    given = torch.cat((source, torch.tensor([pool, 1, 2 ** 31 - 1], device=device))).int()      # pairs that no arena has
    target = torch.cat((destination, torch.tensor([0, pool + 1, 2], device=device))).int()
    ops.kv_pages_copy(store.unbind(0), given, target)
    assert torch.equal(store, want)


def test_pages_copy_of_unaligned_and_unequal_arenas(device):
    generator = torch.Generator(device=device).manual_seed(4)
    buffers = [torch.randint(0, 1000, (1 + pages * words,), generator=generator, device=device, dtype=torch.int32)
               for pages, words in ((9, 4), (6, 5000), (9, 4096))]
    arenas = [b[1:].view(pages, words) for b, (pages, words) in zip(buffers, ((9, 4), (6, 5000), (9, 4096)))]
    wants = [a.clone() for a in arenas]
    source, destination = [0, 7, 3], [5, 2, 8]
    for want in wants:
        for s, d in zip(source, destination):
            if max(s, d) < len(want):
                want[d] = want[s]
    ops.kv_pages_copy(arenas, to_u32(source, device), to_u32(destination, device))
    assert all(torch.equal(a, w) for a, w in zip(arenas, wants)) and all(int(b[0]) >= 0 for b in buffers)


# ------------------------------------------------------------------------------------------------ together


def test_a_conversation_forks_slides_and_is_compacted(device):
    """Two layers of cache: a prompt, decode steps, a fork with a copy of its last page, steps of both branches through a window
    whose pages are given back, and a compaction of the pool in between, each step against the definition."""
    rng = np.random.default_rng(21)
    layers, heads, kv_heads, dim, pool, window, sinks = 2, 8, 2, 64, 24, 48, 5
    allocator, tables = KvPageAllocator(pool), FixedBlockTables(3, 12)
    arenas = [ops.E4m3KvArena.new(pool, kv_heads, dim, device=device) for _ in range(layers)]
    caches = [[plain.Cache(np.zeros((pool, kv_heads, PAGE, dim), dtype=np.uint8), np.zeros((pool, kv_heads))) for _ in range(2)]
              for _ in range(layers)]
    lengths = {}

    def step(portions):
        """portions: (table row, tokens to add), as one batch."""
        rows, positions, slots, offsets = [], [], [], [0]
        for row, count in portions:
            table, before = tables.slot(row), lengths.get(row, 0)
            allocator.grow_sequence(before, before + count, table)
            for position in range(before, before + count):
                rows.append(row)
                positions.append(position)
                slots.append(int(table[position // PAGE]) * PAGE + position % PAGE)
            offsets.append(len(rows))
            lengths[row] = before + count
        index = tables.as_array().astype(np.int64)
        given = [to_u32(tables.as_array(), device), to_u32(rows, device), to_u32(positions, device)]
        decode = all(count == 1 for _, count in portions)
        for arena, cache in zip(arenas, caches):
            key, value = (bf16(rng.standard_normal((len(rows), kv_heads, dim)) * np.exp2(rng.integers(-3, 3)), device) for _ in range(2))
            query = bf16(rng.standard_normal((len(rows), heads, dim)), device)
            arena.write(key, value, to_i64(np.array(slots), device))
            for part, array in zip(cache, (key, value)):
                part.append(host(array), np.array(slots))
            out = torch.zeros_like(query)
            if decode:
                ops.paged_attention_e4m3_into(query, arena, *given, out, window=window, sinks=sinks)
            else:
                ops.paged_prompt_attention_e4m3_into(query, arena, *given, to_u32(offsets, device), out, window=window, sinks=sinks)
            check_attention(out, query, cache, index, rows, positions, F16_WEIGHTS if decode else BF16_WEIGHTS, out, window=window, sinks=sinks)

    def copy(pairs):
        source, destination = pairs
        if len(source):
            ops.kv_pages_copy([t for arena in arenas for t in arena.tensors()], to_u32(source, device), to_u32(destination, device))
            for part in (p for cache in caches for p in cache):
                part.values[destination], part.scales[destination] = part.values[source].copy(), part.scales[source].copy()

    step([(0, 75), (2, 21)])
    step([(0, 1)])
    assert allocator.release_window(lengths[0], window, sinks, tables.slot(0)) == 0
    copy(allocator.fork_sequence(lengths[0], tables.slot(0), tables.slot(1)))
    lengths[1] = lengths[0]
    for count in (1, 1, 9, 1, 30, 1):
        step([(0, 1), (1, count)] if count > 1 else [(0, 1), (1, 1)])
        for row in (0, 1):
            allocator.release_window(lengths[row], window, sinks, tables.slot(row))
    assert (tables.slot(1)[1:3] == plain.UNASSIGNED).all() and tables.slot(1)[0] != plain.UNASSIGNED
    allocator.release_sequence(lengths.pop(2), tables.slot(2))
    live = allocator.snapshot()["allocated_pages"]
    moves = allocator.compact(tables.as_array())
    assert len(moves[0]) > 0
    copy(moves)
    used = tables.as_array()[tables.as_array() != plain.UNASSIGNED]
    assert used.max() < live
    step([(0, 1), (1, 1)])
    step([(1, 40), (2, 33)])
