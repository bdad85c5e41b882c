"""Kernel names of a decoding step over a paged key-value cache: which kernels an operator takes for a shape.

Shared by the schedules (``decoder.py``) and by the operators on device tensors (``reef_b200/decode.py``).
"""
from __future__ import annotations

from .graph import kname

CACHE_TYPES = {"float32": 0, "bfloat16": 1, "float16": 2}


def page_tables(rows: int, max_pages: int, page_size: int, pages: int, tokens: int, fork: bool) -> str:
    """args: table, lens, new, [parent], table', lens', start, tok, status, [fork]"""
    return kname("reef_page_tables", rows=rows, mp=max_pages, ps=page_size, pages=pages, tokens=tokens, **({"fork": 1} if fork else {}))


def paged_append(tokens: int, kv_heads: int, dim: int, page_size: int, pages: int, cache: str, forks: int = 0, **strides) -> str:
    """args: k, v, tok, [fork], k_cache, v_cache; ``strides``: ks, vs (floats from token to token), ko, vo (floats to the first)"""
    return kname("reef_paged_append", tokens=tokens, kvh=kv_heads, d=dim, ps=page_size, pages=pages, kt=CACHE_TYPES[cache],
                 **({"forks": forks} if forks else {}), **strides)


def paged_attention(tokens: int, rows: int, heads: int, kv_heads: int, dim: int, page_size: int, max_pages: int, pages: int, cache: str,
                    **strides) -> list:
    """One name (args: q, k_cache, v_cache, table, tok, out), or two where the keys of a row are divided among blocks: the second
    (args: parts, out) joins what the first (args: q, k_cache, v_cache, table, tok, out, parts) leaves in ``parts``.
    ``strides``: qs (floats from token to token), qo (floats to the first).

    One kernel leaves a row's keys to one block per key head: no join, and blocks that wait for a free SM even out what SMs and rows differ by;
    two divide all keys evenly.  Measured (us, one kernel / two, floor; rows of random length up to the longest, whose keys and values of
    a head are B bytes): 12 heads of all rows, B = 512 KB 14.5 / 13.4 for the longest and 6.3 / 12.5 for a short one; 64, 1 MB 22.7 / 20.8 (6);
    192, 512 KB 18.6 / 20 (11), 1 MB 30.8 / 33.7 (18), 2 MB 54 / 53 (38); 512, 1 MB 71 / 70 (46); 768, 1 MB 79 / 88 (69), 2 MB 153 / 155 (139); 2048,
    1 MB 185 / 207 (164); but 512 of very uneven rows, 4 MB, would wait for the longest.  One kernel, therefore, up to 512 KB and as much
    again for every 320 heads; and where the steps of all rows are more than the division among blocks counts (0x70000000)."""
    shape = dict(tokens=tokens, rows=rows, heads=heads, kvh=kv_heads, d=dim, ps=page_size, mp=max_pages, pages=pages, kt=CACHE_TYPES[cache])
    longest = 2 * max_pages * page_size * dim * (4 if cache == "float32" else 2)
    one = [kname("reef_paged_attention", **shape, **strides)]
    if longest <= (512 << 10) * (1 + tokens * kv_heads / 320):
        return one
    two = [kname("reef_paged_attention_parts", **shape, **strides), kname("reef_paged_attention_join", **shape)]
    if tokens * heads * max_pages * page_size >= 0x70000000:        # (a step takes a key at least)
        from .. import capi
        try:
            capi.kernel_plan(two[0])
        except capi.ReefError:
            return one
    return two


def beam_select(requests: int, beams: int, vocab: int, eos: int, tokens: int | None = None) -> list:
    """args: logits, live, [start], parts; then parts, score, live, [start], token, parent, score', live'"""
    packed = {} if tokens is None else {"tokens": tokens}
    return [kname("reef_beam_scan", requests=requests, beams=beams, vocab=vocab, **packed),
            kname("reef_beam_pick", requests=requests, beams=beams, vocab=vocab, eos=eos, **packed)]
