"""The 8-bit paged cache at the ends of its number formats."""
import numpy as np
import pytest
import torch

import e4m3_cases as plain
from conftest import to_u32
from test_gpu_e4m3_cache import BF16_WEIGHTS, F16_WEIGHTS, PAGE, arena_of, attention_call, bf16, host, pool_of, tables_of

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
