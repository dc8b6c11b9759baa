"""Operators of the 8-bit paged key/value cache, each as a case of its own.

The cache holds E4M3 codes in pages of 16 tokens, `key` and `value` [pages, kv_heads, 16, dim], with one scale for each
page and head, [pages, kv_heads]: an element stands for code * scale.  A scale is the smallest power of two, 2^-126 at
least, under which the largest magnitude that the page's tokens of this head brought is at most 448.

  write        appends the keys and values of a step at their physical slots.  A run of tokens that starts a page sets its
               scale; one that continues a page raises the scale where it has to, and the codes that are there already are
               rounded again to the larger one.  With norms given, queries and keys are RMS-normed and rotated first
               (dimensions d and d + dim / 2 by position * inv_freq[d]), all in 32 bits with one rounding at the end.
  decode       attention of single tokens over the cache: softmax(scale * q k) v over the keys j <= position of the token's
               sequence with j > position - window (window 0: all) or j < sinks.
  prompts      the same for portions of prompts, whose own keys are in the cache already.
  pages        copies pages of all layers' caches at once: forked sequences, compaction of the pool.

Sizes inside a case are spread evenly over its ranges; caches, queries and the order of the pages come from the seed.
"""
from __future__ import annotations

import importlib
import math

import torch

own = False

PAGE = 16
UNASSIGNED = 0xFFFFFFFF
LARGEST = 448.0
EPS = 1e-5


def _write(name, *, heads=32, kv_heads=8, dim=64, norm, decode=0, prompts=0, prompt=(0, 0), context=(0, 0)) -> dict:
    case = {"op": "write", "heads": heads, "kv_heads": kv_heads, "dim": dim, "norm": norm, "decode": decode,
            "prompts": prompts, "prompt_low": prompt[0], "prompt_high": prompt[1], "context_low": context[0],
            "context_high": context[1]}
    return case if name is None else {"name": name, **case}


def _decode(name, *, heads=32, kv_heads=8, dim=64, tokens, padded=0, context, window=0, sinks=0) -> dict:
    case = {"op": "decode", "heads": heads, "kv_heads": kv_heads, "dim": dim, "tokens": tokens, "padded": padded,
            "context_low": context[0], "context_high": context[1], "window": window, "sinks": sinks}
    return case if name is None else {"name": name, **case}


def _prompts(name, *, heads=32, kv_heads=8, dim=64, prompts, prompt, prefix=(0, 0), window=0, sinks=0) -> dict:
    case = {"op": "prompts", "heads": heads, "kv_heads": kv_heads, "dim": dim, "prompts": prompts, "prompt_low": prompt[0],
            "prompt_high": prompt[1], "prefix_low": prefix[0], "prefix_high": prefix[1], "window": window, "sinks": sinks}
    return case if name is None else {"name": name, **case}


def _pages(name, *, kv_heads=8, dim=64, layers=6, pool, pairs, codes=True) -> dict:
    case = {"op": "pages", "kv_heads": kv_heads, "dim": dim, "layers": layers, "pool": pool, "pairs": pairs, "codes": codes}
    return case if name is None else {"name": name, **case}


def listed() -> list[dict]:
    return [
        # one interactive user: the new token of a step, projections already normed and rotated; a launch and little else
        _write("write 1", norm=False, decode=1, context=(1021, 1021)),
        # a full decode batch of the serving engine straight from its projections, pages at every fill
        _write("norm rope write 128", norm=True, decode=128, context=(128, 4096)),
        # a prefill step: eight chunks of about 512 tokens of unequal length behind cached prefixes
        _write("norm rope write 8 prompts", norm=True, prompts=8, prompt=(437, 512), context=(0, 3584)),
        # one interactive user at a moderate context
        _decode("decode 1 at 1024", tokens=1, context=(1024, 1024)),
        # the headline serving step: a full batch of mixed contexts
        _decode("decode 128", tokens=128, context=(128, 4096)),
        # a batch padded to its bucket, streaming through a window with a few first tokens kept; heads of 128
        _decode("decode 23 window", heads=8, kv_heads=2, dim=128, tokens=23, padded=9, context=(300, 20011), window=4096,
                sinks=4),
        # three users of very long contexts: little to do side by side, long ranges to split
        _decode("decode 3 long", tokens=3, context=(20480, 65536)),
        # a full prefill step: eight chunks of 512 tokens at every depth of long prompts
        _prompts("prompts 8x512", prompts=8, prompt=(512, 512), prefix=(0, 3584)),
        # fresh prompts of unequal lengths, heads of 128, a window shorter than the longest of them
        _prompts("prompts 7 window", heads=8, kv_heads=2, dim=128, prompts=7, prompt=(61, 1201), window=512, sinks=4),
        # the last, short portion of a long conversation: few rows, many keys
        _prompts("prompt 37 behind 8000", prompts=1, prompt=(37, 37), prefix=(8000, 8000)),
        # five candidates continue one sequence: each gets a copy of its last, partly filled page
        _pages("fork 5", pool=512, pairs=5),
        # the pool is compacted before it shrinks: a third of its pages move
        _pages("compact 2048", pool=6144, pairs=2048),
    ]


LAYOUTS = ((32, 8, 64), (32, 8, 64), (8, 2, 128), (12, 4, 64), (16, 1, 128), (8, 8, 64))


def _log_uniform(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    op = rng.choice(("write", "decode", "decode", "prompts", "prompts", "pages"))
    heads, kv_heads, dim = rng.choice(LAYOUTS)
    layout = {"heads": heads, "kv_heads": kv_heads, "dim": dim}
    window, sinks = rng.choice(((0, 0), (0, 0), (_log_uniform(rng, 1, 5000), rng.choice((0, 1, 4, 37)))))
    if op == "write":
        low = rng.randint(0, 3000)
        if rng.random() < 0.5:
            return _write(None, **layout, norm=rng.random() < 0.5, decode=_log_uniform(rng, 1, 200), context=(low, low + rng.randint(0, 2000)))
        prompts = rng.randint(1, 8)
        high = _log_uniform(rng, 2, 4000 // prompts)
        return _write(None, **layout, norm=rng.random() < 0.5, prompts=prompts, prompt=(rng.randint(1, high), high),
                      context=(low, low + rng.randint(0, 500)))
    if op == "decode":
        tokens = _log_uniform(rng, 1, 128)
        high = _log_uniform(rng, 16, min(65536, 250000 * 512 // (kv_heads * dim) // tokens))
        return _decode(None, **layout, tokens=tokens, padded=rng.choice((0, 0, rng.randint(1, 8))),
                       context=(rng.randint(1, high), high), window=window, sinks=sinks)
    if op == "prompts":
        prompts = rng.randint(1, 8)
        high = _log_uniform(rng, 1, 4000 // prompts)
        prefix = rng.choice((0, rng.randint(1, 2000)))
        return _prompts(None, **layout, prompts=prompts, prompt=(rng.randint(1, high), high), prefix=(prefix, prefix + rng.randint(0, 500)),
                        window=window, sinks=sinks)
    pool = _log_uniform(rng, 64, 6000)
    return _pages(None, kv_heads=kv_heads, dim=dim, layers=rng.randint(1, 6), pool=pool, pairs=_log_uniform(rng, 1, pool // 3),
                  codes=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ sizes of a case


def _spread(low: int, high: int, count: int) -> list[int]:
    return [low + (high - low) * i // max(1, count - 1) for i in range(count)]


def _sequences(case) -> list[tuple[int, int]]:
    """(cached tokens before the step, tokens of the step) of every sequence."""
    if case["op"] == "decode":
        return [(context - 1, 1) for context in _spread(case["context_low"], case["context_high"], case["tokens"])]
    if case["op"] == "prompts":
        return list(zip(_spread(case["prefix_low"], case["prefix_high"], case["prompts"]),
                        _spread(case["prompt_low"], case["prompt_high"], case["prompts"])))
    if case["decode"]:
        return [(context, 1) for context in _spread(case["context_low"], case["context_high"], case["decode"])]
    return list(zip(_spread(case["context_low"], case["context_high"], case["prompts"]),
                    _spread(case["prompt_low"], case["prompt_high"], case["prompts"])))


def _visible(position: int, window: int, sinks: int) -> int:
    """How many keys a token at `position` sees."""
    if window == 0 or position < window:
        return position + 1
    return window + min(sinks, position + 1 - window)


def work(case) -> dict:
    kv_heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "pages":
        element = kv_heads * PAGE * dim * 2
        page = element + kv_heads * 8 if case["codes"] else element * 2
        return {"bytes": 2 * page * case["layers"] * case["pairs"], "flops": 0}
    sequences = _sequences(case)
    tokens = sum(count for _, count in sequences)
    if case["op"] == "write":
        pages = sum((before + count - 1) // PAGE - before // PAGE + 1 for before, count in sequences)
        moved = tokens * kv_heads * dim * 2 * (2 + 1) + pages * kv_heads * 2 * 4 + tokens * 8
        flops = tokens * kv_heads * dim * 2 * 2
        if case["norm"]:
            moved += tokens * case["heads"] * dim * 4 + tokens * 4
            flops += tokens * (case["heads"] + kv_heads) * dim * 7
        return {"bytes": moved, "flops": flops}
    window, sinks = case["window"], case["sinks"]
    queries = tokens * case["heads"] * dim * 2 * 2
    keys = pairs = 0
    for before, count in sequences:
        last = before + count - 1
        # keys that any token of the sequence sees: from the first one's window on, and the first tokens of all
        first = max(0, before - window + 1) if window else 0
        keys += last + 1 - first + min(sinks, first)
        pairs += sum(_visible(position, window, sinks) for position in range(before, before + count))
    return {"bytes": keys * kv_heads * (2 * dim + 8 / PAGE) + queries + tokens * 8, "flops": 4 * pairs * case["heads"] * dim}


# ------------------------------------------------------------------------------------------------ inputs


def _tables(sequences, generator, spare: int):
    """Block tables of the sequences over a pool in random order, as u32 [rows, stride], and the size of the pool."""
    need = [-(-(before + count) // PAGE) for before, count in sequences]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=generator, device="cuda").tolist()
    stride = max(need)
    rows, at = [], 0
    for count in need:
        rows.append(order[at:at + count] + [UNASSIGNED] * (stride - count))
        at += count
    return torch.tensor(rows, dtype=torch.int64, device="cuda"), pool


def _u32(values) -> torch.Tensor:
    return torch.as_tensor(values, dtype=torch.int64, device="cuda").to(torch.uint32)


def _cache(shape, generator):
    """Codes and scales as a running server has them: normal values, every page and head at a scale of its own."""
    pages, kv_heads, _, dim = shape
    codes = (torch.randn(shape, generator=generator, device="cuda") * 110).clamp_(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
    scales = torch.exp2(torch.randint(-9, -5, (pages, kv_heads), generator=generator, device="cuda").float())
    return codes.view(torch.uint8), scales


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    kv_heads, dim = case["kv_heads"], case["dim"]
    state = {"case": case}

    def normal(*shape):
        return torch.randn(shape, generator=generator, device="cuda")

    if case["op"] == "pages":
        layers, pool, pairs = case["layers"], case["pool"], case["pairs"]
        order = torch.randperm(pool, generator=generator, device="cuda")
        state["source"], state["destination"] = order[:pairs].to(torch.uint32), order[pairs:2 * pairs].to(torch.uint32)
        shape = (layers * pool, kv_heads, PAGE, dim)
        if case["codes"]:
            for name in ("key", "value"):
                codes, scales = _cache(shape, generator)
                state[name] = codes.view(layers, pool, kv_heads, PAGE, dim)
                state[name + "_scales"] = scales.view(layers, pool, kv_heads)
        else:
            for name in ("key", "value"):
                state[name] = normal(*shape).to(torch.bfloat16).view(layers, pool, kv_heads, PAGE, dim)
        return state

    sequences = _sequences(case)
    tables, pool = _tables(sequences, generator, spare=3)
    state["key"], state["key_scales"] = _cache((pool, kv_heads, PAGE, dim), generator)
    state["value"], state["value_scales"] = _cache((pool, kv_heads, PAGE, dim), generator)
    rows = [row for row, (_, count) in enumerate(sequences) for _ in range(count)]
    positions = [before + i for before, count in sequences for i in range(count)]
    tokens = len(rows)
    if case["op"] == "write":
        position = torch.tensor(positions, device="cuda")
        page = tables[torch.tensor(rows, device="cuda"), position // PAGE]
        state["slots"] = page * PAGE + position % PAGE
        # channels of unequal size, as projections leave them
        state["raw_key"] = (normal(tokens, kv_heads, dim) * torch.exp(normal(kv_heads, dim) * 0.5)).to(torch.bfloat16)
        state["raw_value"] = (normal(tokens, kv_heads, dim) * torch.exp(normal(kv_heads, dim) * 0.5)).to(torch.bfloat16)
        if case["norm"]:
            state["raw_query"] = normal(tokens, case["heads"], dim).to(torch.bfloat16)
            state["query"] = torch.empty_like(state["raw_query"])
            state["query_norm"] = (1 + 0.2 * normal(dim)).to(torch.bfloat16)
            state["key_norm"] = (1 + 0.2 * normal(dim)).to(torch.bfloat16)
            state["inv_freq"] = (1e6 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)).float()
            state["positions"] = _u32(positions)
        return state

    padded = case.get("padded", 0)
    state["tables"] = tables.to(torch.uint32)
    state["rows"] = _u32(rows + [UNASSIGNED] * padded)
    state["positions"] = _u32(positions + [0] * padded)
    state["query"] = normal(tokens + padded, case["heads"], dim).to(torch.bfloat16)
    # rows of the batch behind the last sequence belong to nobody and stay as they are: values of the size of a result
    state["output"] = (normal(tokens + padded, case["heads"], dim) * 0.02).to(torch.bfloat16)
    state["longest"] = max(before + count for before, count in sequences)
    if case["op"] == "prompts":
        offsets = [0]
        for _, count in sequences:
            offsets.append(offsets[-1] + count)
        state["offsets"] = _u32(offsets)
        state["longest_prompt"] = max(count for _, count in sequences)
    return state


# ------------------------------------------------------------------------------------------------ plain forms


def _plain_scale(largest: torch.Tensor) -> torch.Tensor:
    """The smallest power of two, 2^-126 at least, that brings `largest` to at most 448 (f32, exact)."""
    mantissa, exponent = torch.frexp(largest)                  # largest = mantissa * 2^exponent, 0.5 <= mantissa < 1
    exponent = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    exponent = torch.where(largest > 0, exponent, torch.full_like(exponent, -126)).clamp(min=-126)
    return torch.ldexp(torch.ones_like(largest), exponent)


def _plain_append(codes, scales, values, slots):
    """Appends f32 `values` [tokens, kv_heads, dim] at `slots` [tokens]."""
    pages, inverse = torch.unique(slots // PAGE, return_inverse=True)
    offsets = slots % PAGE
    largest = torch.zeros((pages.numel(), values.shape[1]), device=values.device)
    largest.index_reduce_(0, inverse, values.abs().amax(2), "amax")
    first = torch.full((pages.numel(),), PAGE, device=slots.device).index_reduce_(0, inverse, offsets, "amin")
    continued = first > 0
    before = scales[pages]
    after = _plain_scale(largest)
    after = torch.where(continued[:, None], torch.maximum(before, after), after)
    # what is there already, rounded again where the scale has grown
    there = codes[pages].view(torch.float8_e4m3fn)
    again = (there.float() * (before / after)[:, :, None, None]).to(torch.float8_e4m3fn)
    row = torch.arange(PAGE, device=slots.device)
    keep = (row[None] < first[:, None])[:, None, :, None]
    codes[pages] = torch.where(keep, again.view(torch.uint8), there.view(torch.uint8))
    scales[pages] = after
    new = (values / after[inverse][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes[slots // PAGE, :, offsets] = new


def _plain_norm_rope(x, weight, inv_freq, positions):
    """RMS norm and rotation of [tokens, heads, dim] in f32, angles in f64."""
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS) * weight.float()
    angle = positions.to(torch.float64)[:, None] * inv_freq.double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    low, high = x.chunk(2, 2)
    return torch.cat((low * cos - high * sin, high * cos + low * sin), 2)


def _plain_gather(codes, scales, pages):
    """Values [rows, kv_heads, keys, dim] in f32 of pages [rows, count]."""
    values = codes[pages].view(torch.float8_e4m3fn).float() * scales[pages][:, :, :, None, None]
    rows, count, kv_heads, _, dim = values.shape
    return values.transpose(1, 2).reshape(rows, kv_heads, count * PAGE, dim)


def _plain_attention(query, key, value, position, valid, window, sinks):
    """query [rows, length, heads, dim], key / value [rows, kv_heads, keys, dim], position [rows, length] -> like query."""
    rows, length, heads, dim = query.shape
    kv_heads, keys = key.shape[1], key.shape[2]
    query = query.float().view(rows, length, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(query.reshape(rows, kv_heads, -1, dim), key.transpose(2, 3)) * dim ** -0.5
    index = torch.arange(keys, device=key.device)
    seen = index <= position[:, :, None]
    if window:
        seen &= (index > position[:, :, None] - window) | (index < sinks)
    seen = (seen & valid[:, :, None])[:, None, None].expand(rows, kv_heads, heads // kv_heads, length, keys)
    scores = scores.view(seen.shape).masked_fill(~seen, -math.inf)
    largest = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(largest.isinf(), torch.zeros_like(largest), largest))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.reshape(rows, kv_heads, -1, keys), value).view(*seen.shape[:4], dim) / total
    return out.permute(0, 3, 1, 2, 4).reshape(rows, length, heads, dim)


def _caches(state) -> dict:
    if state["case"].get("codes", True):
        return {name: state[name].view(torch.float8_e4m3fn) if state[name].dtype == torch.uint8 else state[name]
                for name in ("key", "value", "key_scales", "value_scales")}
    return {"key": state["key"], "value": state["value"]}


def _run_own(state):
    case = state["case"]
    ops = importlib.import_module("lfm25-inference_b200.ops")
    if case["op"] == "pages":
        arenas = [layer for name in ("key", "value", "key_scales", "value_scales") if name in state for layer in state[name].unbind(0)]
        ops.kv_pages_copy(arenas, state["source"], state["destination"])
        return _caches(state)
    arena = ops.E4m3KvArena(state["key"], state["value"], state["key_scales"], state["value_scales"])
    if case["op"] == "write":
        if not case["norm"]:
            ops.kv_cache_write_e4m3(state["raw_key"], state["raw_value"], arena, state["slots"])
            return _caches(state)
        ops.qk_norm_rope_kv_write_e4m3(state["raw_query"], state["raw_key"], state["raw_value"], state["query_norm"],
                                       state["key_norm"], state["inv_freq"], state["positions"], state["slots"], arena, EPS,
                                       query_out=state["query"])
        return {"query": state["query"], **_caches(state)}
    if case["op"] == "decode":
        ops.paged_attention_e4m3_into(state["query"], arena, state["tables"], state["rows"], state["positions"], state["output"],
                                      window=case["window"], sinks=case["sinks"], maximum_context_tokens=state["longest"])
    else:
        ops.paged_prompt_attention_e4m3_into(state["query"], arena, state["tables"], state["rows"], state["positions"],
                                             state["offsets"], state["output"], window=case["window"], sinks=case["sinks"])
    return state["output"]


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "pages":
        source, destination = state["source"].to(torch.int64), state["destination"].to(torch.int64)
        state["key"][:, destination] = state["key"][:, source]
        state["value"][:, destination] = state["value"][:, source]
        if case["codes"]:
            state["key_scales"][:, destination] = state["key_scales"][:, source]
            state["value_scales"][:, destination] = state["value_scales"][:, source]
        return _caches(state)
    if case["op"] == "write":
        key = state["raw_key"].float()
        if case["norm"]:
            key = _plain_norm_rope(state["raw_key"], state["key_norm"], state["inv_freq"], state["positions"])
            state["query"].copy_(_plain_norm_rope(state["raw_query"], state["query_norm"], state["inv_freq"], state["positions"]))
        _plain_append(state["key"], state["key_scales"], key, state["slots"])
        _plain_append(state["value"], state["value_scales"], state["raw_value"].float(), state["slots"])
        return {"query": state["query"], **_caches(state)} if case["norm"] else _caches(state)
    window, sinks = case["window"], case["sinks"]
    tables, rows = state["tables"].to(torch.int64), state["rows"].to(torch.int64)
    last = tables.shape[0]
    positions = state["positions"].to(torch.int64)
    if case["op"] == "decode":
        pages = tables[rows.clamp(max=last - 1)].clamp(max=state["key"].shape[0] - 1)
        key, value = (_plain_gather(state[name], state[name + "_scales"], pages) for name in ("key", "value"))
        valid = rows < last
        out = _plain_attention(state["query"][:, None], key, value, positions[:, None], valid[:, None], window, sinks)[:, 0]
        state["output"].copy_(torch.where(valid[:, None, None], out.to(torch.bfloat16), state["output"]))
        return state["output"]
    # prompts, padded to the longest one
    offsets = state["offsets"].to(torch.int64)
    index = offsets[:-1, None] + torch.arange(state["longest_prompt"], device=offsets.device)
    valid = index < offsets[1:, None]
    index = index.clamp(max=rows.numel() - 1)
    pages = tables[rows[offsets[:-1]]].clamp(max=state["key"].shape[0] - 1)
    key, value = (_plain_gather(state[name], state[name + "_scales"], pages) for name in ("key", "value"))
    out = _plain_attention(state["query"][index], key, value, positions[index], valid, window, sinks)
    state["output"][index[valid]] = out[valid].to(torch.bfloat16)
    return state["output"]


# ------------------------------------------------------------------------------------------------ definitions in 64 bits


def _exact_round(values):
    """The nearest E4M3 value of each (ties to the even one), |values| <= 448, in f64."""
    exponent = torch.floor(torch.log2(values.abs().clamp(min=2.0 ** -20)))
    exponent = torch.where(torch.exp2(exponent) > values.abs(), exponent - 1, exponent)
    exponent = torch.where(torch.exp2(exponent + 1) <= values.abs(), exponent + 1, exponent)
    step = torch.exp2(exponent.clamp(min=-6) - 3)
    return torch.round(values / step) * step


def _exact_append(codes, scales, values, slots):
    codes = codes.view(torch.float8_e4m3fn).double()
    scales = scales.double()
    by_page = {}
    for token, slot in enumerate(slots.tolist()):
        by_page.setdefault(slot // PAGE, []).append((token, slot % PAGE))
    pages = list(by_page)
    largest = torch.stack([values[[token for token, _ in by_page[page]]].abs().amax((0, 2)) for page in pages])
    # candidates for the scale, all powers of two there are: the first that is large enough
    powers = torch.exp2(torch.arange(-126, 121, device=values.device, dtype=torch.float64))
    fresh = powers[torch.searchsorted(powers * LARGEST, largest)]
    first = torch.tensor([min(offset for _, offset in by_page[page]) for page in pages], device=values.device)
    index = torch.tensor(pages, device=values.device)
    after = torch.where(first[:, None] > 0, torch.maximum(scales[index], fresh), fresh)
    there = codes[index]
    kept = torch.arange(PAGE, device=values.device)[None, None, :, None] < first[:, None, None, None]
    codes[index] = torch.where(kept, _exact_round(there * (scales[index] / after)[:, :, None, None]), there)
    scales[index] = after
    codes[slots // PAGE, :, slots % PAGE] = _exact_round(values / scales[slots // PAGE][:, :, None])
    return codes.float().to(torch.float8_e4m3fn), scales.float()


def _exact_norm_rope(x, weight, inv_freq, positions):
    x = x.double()
    half = x.shape[2] // 2
    x = x / torch.sqrt((x * x).sum(2, keepdim=True) / x.shape[2] + EPS) * weight.double()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), positions.double()[:, None, None] * inv_freq.double())
    turned = torch.complex(x[:, :, :half], x[:, :, half:]) * turn
    return torch.cat((turned.real, turned.imag), 2)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "pages":
        names = ("key", "value", "key_scales", "value_scales") if case["codes"] else ("key", "value")
        origin = torch.arange(case["pool"], device="cuda")
        origin[state["destination"].long()] = state["source"].long()
        moved = {name: state[name][:, origin] for name in names}
        return {name: x.view(torch.float8_e4m3fn) if x.dtype == torch.uint8 else x for name, x in moved.items()}
    if case["op"] == "write":
        out, key = {}, state["raw_key"].double()
        if case["norm"]:
            key = _exact_norm_rope(state["raw_key"], state["key_norm"], state["inv_freq"], state["positions"])
            out["query"] = _exact_norm_rope(state["raw_query"], state["query_norm"], state["inv_freq"], state["positions"])
        out["key"], out["key_scales"] = _exact_append(state["key"], state["key_scales"], key, state["slots"])
        out["value"], out["value_scales"] = _exact_append(state["value"], state["value_scales"], state["raw_value"].double(), state["slots"])
        return out
    kv_heads, dim, window, sinks = case["kv_heads"], case["dim"], case["window"], case["sinks"]
    group = case["heads"] // kv_heads
    out = state["output"].double()
    token = 0
    for row, (before, count) in enumerate(_sequences(case)):
        pages = state["tables"][row].long()[:-(-(before + count) // PAGE)]
        index = torch.arange(before + count, device="cuda")
        at = torch.arange(before, before + count, device="cuda")[:, None]
        seen = (index <= at) & ((index > at - window) | (index < sinks) if window else index <= at)
        for head in range(kv_heads):
            key, value = ((state[name][pages, head].view(torch.float8_e4m3fn).double() * state[name + "_scales"][pages, head].double()[:, None, None])
                          .reshape(-1, dim)[:before + count] for name in ("key", "value"))
            for member in range(head * group, (head + 1) * group):
                scores = state["query"][token:token + count, member].double() @ key.T / math.sqrt(dim)
                weights = torch.softmax(scores.masked_fill(~seen, -math.inf), -1)
                out[token:token + count, member] = weights @ value
        token += count
    return out
