"""Batches of single tokens that take each form of the 8-bit cache's decode attention: warps of a CTA and CTAs of a cluster."""
import ctypes

from lfm25_inference_b200 import _abi
from lfm25_inference_b200._abi import Slice


def plan(tokens, heads, kv_heads, dim, longest, window=0, sinks=0, clusters_of_16=True):
    """(warps, CTAs of a cluster) of a call."""
    def fake(elements):
        return Slice(0x1000, elements)
    stride = -(-longest // 16)
    pages = 4
    cache = _abi.E4m3Cache(16, pages, kv_heads, dim, fake(pages * kv_heads * 16 * dim), fake(pages * kv_heads * 16 * dim),
                           fake(pages * kv_heads), fake(pages * kv_heads))
    launch = _abi.PagedAttentionE4m3Launch(cache, fake(tokens * heads * dim), fake(stride), fake(tokens), fake(tokens),
                                           fake(tokens * heads * dim), tokens, heads, 0, stride, window, sinks, longest, 0.125,
                                           Slice(None, 0), Slice(None, 0), 0)
    warps, splits = ctypes.c_uint32(), ctypes.c_uint32()
    _abi.check(_abi.library().lfm25_paged_attention_e4m3_plan(ctypes.byref(launch), int(clusters_of_16), ctypes.byref(warps),
                                                              ctypes.byref(splits)))
    return warps.value, splits.value


# (heads, KV heads, dimensions) -> (warps, CTAs of a cluster) -> (tokens, longest context)
BATCHES = {
    (32, 8, 64): {(4, 1): (48, 40), (4, 2): (20, 600), (4, 4): (12, 1100), (4, 8): (6, 2100), (4, 16): (3, 65536), (8, 1): (5, 300),
                  (8, 2): (3, 600), (8, 4): (3, 1100), (8, 8): (3, 4200), (8, 16): (1, 65536)},
    (16, 1, 64): {(4, 1): (300, 40), (4, 2): (128, 600), (4, 4): (64, 1100), (4, 8): (32, 2100), (4, 16): (20, 4200), (8, 1): (5, 300),
                  (8, 2): (3, 600), (8, 4): (3, 1100), (8, 8): (12, 4200), (8, 16): (3, 6000)},
    (8, 2, 128): {(4, 1): (128, 40), (4, 2): (64, 600), (4, 4): (32, 1100), (4, 8): (16, 2100), (4, 16): (10, 4200), (8, 1): (5, 300),
                  (8, 2): (3, 600), (8, 4): (3, 1100), (8, 8): (6, 4200), (8, 16): (2, 65536)},
    (16, 1, 128): {(4, 1): (160, 40), (4, 2): (80, 600), (4, 4): (40, 1100), (4, 8): (20, 2100), (4, 16): (12, 65536), (8, 1): (5, 300),
                   (8, 2): (3, 600), (8, 4): (3, 1100), (8, 8): (12, 4200), (8, 16): (2, 6000)},
}
ALL = [(layout, form, *batch) for layout, forms in BATCHES.items() for form, batch in forms.items()]
