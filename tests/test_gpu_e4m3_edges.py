"""The 8-bit paged cache at the ends of its number formats, single tokens in every form of the kernel, many segments, and
page copies between other words."""
import numpy as np
import pytest
import torch

import e4m3_cases as plain
from e4m3_batches import ALL, plan
from conftest import to_i64, to_u32
from lfm25_inference_b200 import ops
from test_gpu_e4m3_cache import (BF16_WEIGHTS, F16_WEIGHTS, PAGE, arena_of, attention_call, bf16, check_attention, host, pool_of,
                                 random_cache, tables_of)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ number formats


@pytest.mark.parametrize("kind", ["decode", "prompts"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 64), (2, 1, 128), (16, 1, 64), (16, 1, 128)])
@pytest.mark.parametrize("above", [14.3, 20.6, 24.6, 27.3])
def test_a_first_token_that_takes_nearly_all(device, kind, heads, kv_heads, dim, above):
    """One key lies `above` (log2) over all others, and its value is zero: the result is what the others have, each with a weight of
    2^-above.  A weight is rounded by 2^-11 (f16) or 2^-8 (bf16) of itself or, in f16, by half of the smallest step: weights are at
    most 2^11 where they refer to the largest score, so that step is 2^-24 / 2^11 of the largest weight, which is 1 here."""
    context = 5000
    pool = pool_of((context,))
    rng = np.random.default_rng(int(above))
    tables = tables_of(rng, (context,), pool)
    # codes of 1.0 (0x38); all keys are zero but the first, whose score is above * ln 2
    codes = [np.zeros((pool, kv_heads, PAGE, dim), dtype=np.uint8) for _ in range(2)]
    codes[1][:] = 0x38
    codes[0][tables[0, 0], :, 0] = 0x38
    codes[1][tables[0, 0], :, 0] = 0
    scales = [np.ones((pool, kv_heads)) for _ in range(2)]
    arena = arena_of(codes, scales, device)
    cache = plain.Cache(codes[0], scales[0]), plain.Cache(codes[1], scales[1])
    query = bf16(np.ones((1, heads, dim)), device)
    rule = dict(scale=above * np.log(2.0) / dim)
    out = torch.zeros_like(query)
    given = to_u32(tables, device), to_u32([0], device), to_u32([context - 1], device)
    attention_call(kind, query, arena, *given, out, **rule)
    exact, magnitude, score = plain.attend(host(query), cache[0].full(), cache[1].full(), tables, [0], [context - 1], **rule)
    bound = plain.tolerance(exact, magnitude, score, dim, F16_WEIGHTS if kind == "decode" else BF16_WEIGHTS)
    if kind == "decode":
        bound = bound + context * 2.0 ** -36
    worst = np.abs((host(out) - exact) / bound).max()
    assert worst <= 1, f"error over its bound: {worst}, {host(out).max()} for {exact.max()}"


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("stray", [float("nan"), float("inf"), -float("inf"), -1.0])
def test_prompt_tiles_with_pages_that_none_of_their_rows_sees(device, heads, kv_heads, dim, stray):
    """A segment ends in tokens of nobody (a padded portion), whose pages are assigned and were never written: whatever lies there,
    the tokens in front of them have their results, and those behind keep their rows."""
    rng = np.random.default_rng(31)
    arena, *cache = random_cache(rng, 9, kv_heads, dim, device)
    tables = np.arange(9)[None]
    count, real = 50, 20                        # positions 60 .. 79, then up to 109: pages 5 and 6 belong to nobody
    for tensor in (arena.key_scales, arena.value_scales):
        tensor[5:7] = stray
    for part in cache:
        part.values[5:7] = 0
    rows = np.where(np.arange(count) < real, 0, plain.UNASSIGNED)
    positions = np.where(np.arange(count) < real, 60 + np.arange(count), 0)
    query = bf16(rng.standard_normal((count, heads, dim)), device)
    out = torch.full_like(query, 3.0)
    ops.paged_prompt_attention_e4m3_into(query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device),
                                         to_u32([0, count], device), out)
    assert (out[real:] == 3.0).all()
    check_attention(out[:real], query[:real], cache, tables, rows[:real], positions[:real], BF16_WEIGHTS, out[:real])


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_rows_that_see_a_page_whose_scale_is_no_number(device, dim):
    """... are no numbers either, and only they."""
    rng = np.random.default_rng(32)
    arena, *cache = random_cache(rng, 9, 2, dim, device)
    tables = np.arange(9)[None]
    arena.value_scales[5, 1] = float("nan")
    cache[1].scales[5, 1] = 0
    positions = 60 + np.arange(50)
    query = bf16(rng.standard_normal((50, 4, dim)), device)
    out = torch.full_like(query, 3.0)
    ops.paged_prompt_attention_e4m3_into(query, arena, to_u32(tables, device), to_u32(np.zeros(50), device), to_u32(positions, device),
                                         to_u32([0, 50], device), out)
    sees = positions >= 80
    got = host(out)
    assert np.isnan(got[sees, 2:]).all() and not np.isnan(got[:, :2]).any() and not np.isnan(got[~sees]).any()
    check_attention(out[:20], query[:20], cache, tables, np.zeros(20, dtype=int), positions[:20], BF16_WEIGHTS, out[:20])


@pytest.mark.parametrize("kind", ["decode", "prompts"])
@pytest.mark.parametrize("dim", [64, 128])
def test_large_values(device, kind, dim):
    """Values of 1e37 times a weight of 1 are what f32 holds; the factor that keeps small weights must not show."""
    rng = np.random.default_rng(35)
    arena = ops.E4m3KvArena.new(8, 1, dim, device=device)
    cache = [plain.Cache(np.zeros((8, 1, PAGE, dim), dtype=np.uint8), np.zeros((8, 1))) for _ in range(2)]
    key, value = bf16(rng.standard_normal((128, 1, dim)) * 0.1, device), bf16(rng.uniform(-1e37, 1e37, (128, 1, dim)) / 8, device)
    arena.write(key, value, to_i64(np.arange(128), device))
    for part, array in zip(cache, (key, value)):
        part.append(host(array), np.arange(128))
    positions = np.arange(30, 128)
    query = bf16(rng.standard_normal((98, 4, dim)), device)
    out = torch.zeros_like(query)
    given = to_u32(np.arange(8)[None], device), to_u32(np.zeros(98), device), to_u32(positions, device)
    attention_call(kind, query, arena, *given, out)
    check_attention(out, query, cache, np.arange(8)[None], np.zeros(98, dtype=int), positions,
                    F16_WEIGHTS if kind == "decode" else BF16_WEIGHTS, out)


@pytest.mark.parametrize("kind", ["decode", "prompts"])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_at_the_end_of_f32_reach_nobody_who_does_not_see_them(device, kind, dim):
    """A value of 3.35e38 is the code of 256 at 2^120, which f32 does not hold.  Tokens in front of it are as ever."""
    rng = np.random.default_rng(33)
    arena = ops.E4m3KvArena.new(8, 1, dim, device=device)
    cache = [plain.Cache(np.zeros((8, 1, PAGE, dim), dtype=np.uint8), np.zeros((8, 1))) for _ in range(2)]
    key, value = (rng.standard_normal((128, 1, dim)) for _ in range(2))
    value[64:] *= 1e37
    value[100, 0, 3] = 3.35e38
    key, value = bf16(key, device), bf16(value, device)
    arena.write(key, value, to_i64(np.arange(128), device))
    cache[0].append(host(key), np.arange(128))
    cache[1].append(host(value), np.arange(128))
    positions = np.arange(50, 128)
    query = bf16(rng.standard_normal((78, 4, dim)), device)
    out = torch.zeros_like(query)
    given = to_u32(np.arange(8)[None], device), to_u32(np.zeros(78), device), to_u32(positions, device)
    if kind == "decode":
        ops.paged_attention_e4m3_into(query, arena, *given, out)
    else:
        ops.paged_prompt_attention_e4m3_into(query, arena, *given, to_u32([0, 78], device), out)
    rows = np.zeros(50, dtype=int)
    check_attention(out[:50], query[:50], cache, np.arange(8)[None], rows, positions[:50], F16_WEIGHTS if kind == "decode" else BF16_WEIGHTS,
                    out[:50])
    assert not out[50:].isnan().any()


# ------------------------------------------------------------------------------------------------ append


@pytest.mark.parametrize("dim", [64, 128])
def test_append_to_pages_whose_scale_is_no_power_of_two(device, dim):
    """The scale becomes the next power of two at least, and what the page holds keeps its values up to one more rounding."""
    rng = np.random.default_rng(34)
    given = np.array([1.5, 0.75, 2.0, 1.0 + 2.0 ** -23, 3e-3, 1.99, 1.25 * 2.0 ** 100, 1.75 * 2.0 ** -126])
    heads, pages = 2, len(given)
    codes = [rng.integers(0, 256, (pages, heads, PAGE, dim), dtype=np.uint8) for _ in range(2)]
    scales = [np.repeat(given[:, None], heads, axis=1) for _ in range(2)]
    arena = arena_of(codes, scales, device)
    # the tokens bring nothing large to head 0 and 2^12 times the scale to head 1
    rows = np.ones((pages, heads, dim)) * 2.0 ** -133
    rows[:, 1] = (given * 2.0 ** 12)[:, None]
    offset = 9
    rows = bf16(rows, device)
    ops.kv_cache_write_e4m3(rows, rows, arena, to_i64(np.arange(pages) * PAGE + offset, device))
    for tensor, stored, before in ((arena.key, arena.key_scales, codes[0]), (arena.value, arena.value_scales, codes[1])):
        stored = stored.cpu().numpy().astype(np.float64)
        brought = host(rows)[:, :, 0]
        for page in range(pages):
            for head in range(heads):
                scale = 2.0 ** np.ceil(np.log2(np.float32(given[page]).astype(np.float64)))
                scale = max(scale, plain.scale_of(brought[page, head]))
                assert stored[page, head] == scale
                kept = plain.CODE_VALUES[before[page, head, :offset]] * np.float64(np.float32(given[page]))
                got = plain.CODE_VALUES[tensor[page, head].cpu().numpy()]
                assert np.array_equal(got[:offset], plain.round_e4m3(kept / scale), equal_nan=True)
                assert np.array_equal(got[offset], plain.round_e4m3(host(rows)[page, head] / scale))


@pytest.mark.parametrize("heads,kv_heads,dim,tokens,first", [
    (32, 8, 64, 1, 0), (32, 8, 64, 128, 77), (8, 2, 128, 40, 9), (12, 4, 64, 700, 100000), (5, 1, 128, 3, 2 ** 31), (8, 2, 128, 2400, 5),
    (12, 4, 64, 2401, 16384)])
def test_keys_are_rounded_once_behind_norm_and_rotation(device, heads, kv_heads, dim, tokens, first):
    """A key is off by half a step of E4M3 and by what f32 is off in front of it (dim squares and a handful of products, an angle of
    2^-22): nothing that a call brings is rounded a second time, since a page takes one run a call.  Few tokens and so many that CTAs
    of four warps take them."""
    rng = np.random.default_rng(tokens + dim)
    pages = -(-tokens // PAGE) + 1
    arena, *_ = random_cache(rng, pages, kv_heads, dim, device, low=-14, high=-12)
    slots = np.arange(tokens, dtype=np.int64) + 3
    positions = np.arange(first, first + tokens, dtype=np.uint32)
    query, key, value = (bf16(rng.standard_normal((tokens, n, dim)), device) for n in (heads, kv_heads, kv_heads))
    weights = [bf16(1 + 0.3 * rng.standard_normal(dim), device) for _ in range(2)]
    inv_freq = torch.from_numpy((1e6 ** (-np.arange(0, dim, 2) / dim)).astype(np.float32)).to(device)
    out = torch.empty_like(query)
    ops.qk_norm_rope_kv_write_e4m3(query, key, value, *weights, inv_freq, to_u32(positions, device), to_i64(slots, device), arena, 1e-5,
                                   query_out=out)
    half = dim // 2
    slack = lambda x: (dim / 2 + 16) * 2.0 ** -23 * (np.abs(x) + np.abs(np.concatenate((x[:, :, half:], x[:, :, :half]), axis=2)))  # noqa: E731
    want = plain.norm_rope(host(query), host(weights[0]), inv_freq.cpu().numpy(), positions, 1e-5)
    assert np.all(np.abs(host(out) - want) <= 2.0 ** -8 * np.abs(want) + (1 + 2.0 ** -8) * slack(want))
    want = plain.norm_rope(host(key), host(weights[1]), inv_freq.cpu().numpy(), positions, 1e-5)
    scales = arena.key_scales.cpu().numpy().astype(np.float64)[slots // PAGE]
    got = plain.CODE_VALUES[arena.key.cpu().numpy()][slots // PAGE, :, slots % PAGE] * scales[:, :, None]
    bound = np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * scales[:, :, None]) + 2 * slack(want)
    assert np.all(np.abs(got - want) <= bound)


# ------------------------------------------------------------------------------------------------ forms of the kernel


@pytest.mark.parametrize("windowed", [False, True])
@pytest.mark.parametrize("layout,form,tokens,longest", ALL)
def test_decode_attention_in_every_form(device, layout, form, tokens, longest, windowed):
    """4 or 8 warps a CTA, clusters of 1 to 16, few and many heads to a KV head, in batches that take them (that is looked at, too);
    some tokens are compared, the one of the longest context among them.  With a window that leaves as much to see."""
    heads, kv_heads, dim = layout
    window, sinks = (longest - 21, 5) if windowed else (0, 0)
    most = longest + (longest // 3 if windowed else 0)
    assert plan(tokens, *layout, most, window, sinks) == form
    rng = np.random.default_rng(tokens * dim + longest)
    contexts = tuple(int(c) for c in rng.integers(1, min(most, 6000) + 1, tokens - 1)) + (most,)
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, kv_heads, dim, device)
    tables = tables_of(rng, contexts, pool)
    order = rng.permutation(tokens)
    positions = np.array(contexts)[order] - 1
    query = bf16(rng.standard_normal((tokens, heads, dim)) * 0.5, device)
    out = torch.full_like(query, float("nan"))
    ops.paged_attention_e4m3_into(query, arena, to_u32(tables, device), to_u32(order, device), to_u32(positions, device), out,
                                  window=window, sinks=sinks, maximum_context_tokens=most)
    assert not out.isnan().any()
    some = np.unique(np.concatenate(([np.argmax(positions)], rng.integers(0, tokens, 6))))
    check_attention(out[some], query[some], cache, tables, order[some], positions[some], F16_WEIGHTS, out[some], window=window, sinks=sinks)


# ------------------------------------------------------------------------------------------------ segments


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 64), (8, 2, 128), (35, 1, 64)])
@pytest.mark.parametrize("count,window", [(33, 0), (64, 20), (101, 0)])
def test_prompt_attention_of_many_segments(device, heads, kv_heads, dim, count, window):
    """Tiles are found in blocks of 32 segments: short ones of unequal lengths, empty ones between them and at the ends of the blocks,
    some of two tiles or more, one that takes the place of a whole block's tiles, and tokens of nobody around all."""
    rng = np.random.default_rng(count + dim)
    lengths = rng.integers(1, 12, count)
    lengths[[5, 31, 32]] = 0
    lengths[rng.integers(0, count, count // 8)] = 0
    lengths[[0, 17, count - 1]] = 97, 140, 70
    if count > 64:
        lengths[[33, 63, 64, 90]] = 130, 0, 0, 66
    prefixes = rng.integers(0, 60, count)
    contexts = tuple(int(c) for c in np.maximum(prefixes + lengths, 1))
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, kv_heads, dim, device)
    tables = tables_of(rng, contexts, pool)
    lead, tail = 4, 5
    rows = np.concatenate((np.zeros(lead, dtype=np.int64), np.repeat(np.arange(count), lengths), np.zeros(tail, dtype=np.int64)))
    positions = np.concatenate([np.zeros(lead, dtype=np.int64)] + [np.arange(p, p + n) for p, n in zip(prefixes, lengths)] +
                               [np.zeros(tail, dtype=np.int64)])
    offsets = lead + np.concatenate(([0], np.cumsum(lengths)))
    query = bf16(rng.standard_normal((len(rows), heads, dim)) * 0.5, device)
    out = bf16(rng.standard_normal(query.shape), device)
    before = out.clone()
    ops.paged_prompt_attention_e4m3_into(query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device),
                                         to_u32(offsets, device), out, window=window)
    assert torch.equal(out[:lead], before[:lead]) and torch.equal(out[-tail:], before[-tail:])
    inside = slice(lead, len(rows) - tail)
    check_attention(out[inside], query[inside], cache, tables, rows[inside], positions[inside], BF16_WEIGHTS, before[inside], window=window)


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 64), (8, 2, 128)])
def test_prompt_attention_whose_shares_are_empty(device, heads, kv_heads, dim):
    """Block tables far wider than the contexts, and nothing said about these: eight CTAs share the keys of a tile that has one stage or
    a few, and most have none."""
    rng = np.random.default_rng(dim)
    contexts = (70, 9)
    pool = pool_of(contexts)
    arena, *cache = random_cache(rng, pool, kv_heads, dim, device)
    tables = tables_of(rng, contexts, pool, spare_columns=300)
    rows, positions = np.repeat([0, 1], 9), np.concatenate((np.arange(61, 70), np.arange(9)))
    query = bf16(rng.standard_normal((18, heads, dim)), device)
    for longest in (0, 70):
        out = torch.full_like(query, float("nan"))
        ops.paged_prompt_attention_e4m3_into(query, arena, to_u32(tables, device), to_u32(rows, device), to_u32(positions, device),
                                             to_u32([0, 9, 18], device), out, maximum_context_tokens=longest)
        check_attention(out, query, cache, tables, rows, positions, BF16_WEIGHTS, out)


# ------------------------------------------------------------------------------------------------ pages


@pytest.mark.parametrize("words", [1, 3, 4, 8, 33, 512, 2048, 5000])
@pytest.mark.parametrize("front", [1, 4])
def test_page_copies_stay_within_their_arena(device, words, front):
    """Words in front of each arena and behind it, on a 16-byte boundary and off one, and all pages that are no destination stay as they
    were; the first page and the last one are among those copied."""
    pages, source, destination = 40, [38, 20, 5, 39], [1, 21, 0, 7]
    buffers = [torch.arange(front + pages * words + 5, device=device, dtype=torch.int32) * 7 + index for index in range(3)]
    arenas = [buffer[front:front + pages * words].view(pages, words) for buffer in buffers]
    wants = [buffer.clone() for buffer in buffers]
    for want in wants:
        inner = want[front:front + pages * words].view(pages, words)
        inner[destination] = inner[source]
    ops.kv_pages_copy(arenas, to_u32(source, device), to_u32(destination, device))
    assert all(torch.equal(buffer, want) for buffer, want in zip(buffers, wants))
