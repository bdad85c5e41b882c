"""Decoding step of a transformer with paged key-value caches and beam search, as a schedule.

One pass takes the tokens that every row adds (one each while decoding, a prompt's at its start), appends their keys and values to the
caches, and selects each request's next beams.  A row is a beam, the beams of a request stand side by side.

    page tables                       reef_page_tables           table, lens, new, parent -> table_out, lens_out, start, tok, status, fork
    embedding at the rows' positions  reef_embedding (npos)      + LayerNorm
    per layer
        q, k, v projection (+bias)    reef_matmul_nt_bias        one buffer, [tokens][heads + 2 kv_heads][64]
        keys and values, page copies  reef_paged_append          out of that buffer into this layer's caches
        attention over the pages      reef_paged_attention (_parts, _join)
        output projection, LayerNorm, FFN with GELU, LayerNorm   as in the encoder (``bert.py``)
    logits                            reef_matmul_nt_bias        ``output``, [tokens][vocab]
    selection                         reef_beam_scan, reef_beam_pick   score, live -> token_out, parent_out, score_out, live_out

Inputs: ``ids`` (int64, [tokens], the rows' new tokens one row after the other), ``table`` [rows][max_pages], ``lens`` [rows], ``new`` [rows],
``parent`` [rows] (int32), ``score`` [rows] (float32), ``live`` [rows] (int32).  The client gives back what the last pass put out:
table_out, lens_out, and for beams parent_out, score_out, live_out (which is also ``new``).  The caches stay on the device.  Every kernel
reads one set of buffers and writes another, or writes the same values again, so a preempted pass can be resumed anywhere.
(The reference serves networks without state between requests only; its nearest schedule is resource/bert/bert.json.)
"""
from __future__ import annotations

from . import decoding
from .bert import _B
from .graph import kname


def build_decoder(*, name: str = "decoder", layers: int = 12, hidden: int = 768, heads: int = 12, kv_heads: int = 12, ffn: int = 2048,
                  vocab: int = 30524, requests: int = 4, beams: int = 4, tokens: int | None = None, page_size: int = 16, max_pages: int = 64,
                  pages: int = 1024, cache: str = "bfloat16", eos: int = 2, seed: int = 7000, conv_impl: str = "auto") -> _B:
    assert hidden == heads * 64 and heads % kv_heads == 0 and vocab % 4 == 0
    b = _B(name, seed, conv_impl)
    g, rows, kv = b.g, requests * beams, kv_heads * 64
    tokens = tokens or rows
    size = 4 if cache == "float32" else 2
    i32 = lambda n, name: g.add_storage(name, n, "int32")      # noqa: E731
    ids = g.input("ids", tokens, "int64")
    state = [g.input("table", rows * max_pages, "int32"), g.input("lens", rows, "int32"), g.input("new", rows, "int32"), g.input("parent", rows, "int32")]
    score, live = g.input("score", rows), g.input("live", rows, "int32")
    table, lens, start, tok = i32(rows * max_pages, "table_out"), i32(rows, "lens_out"), i32(rows + 1, "start"), i32(4 * tokens, "tok")
    status, fork = i32(rows, "status"), i32(4 * rows, "fork")
    g.kernel(decoding.page_tables(rows, max_pages, page_size, pages, tokens, True), state + [table, lens, start, tok, status, fork])
    longest = max_pages * page_size
    word, pos = g.param(b.normal(vocab, hidden)), g.param(b.normal(longest, hidden))
    emb = g.temp(tokens * hidden)
    g.kernel(kname("reef_embedding", s=tokens, h=hidden, vocab=vocab, npos=longest), [emb, word, ids, pos, tok])
    x = b.layernorm(emb, tokens, hidden)
    step = hidden + 2 * kv
    for layer in range(layers):
        qkv = b.matmul(x, tokens, step, hidden)
        caches = [g.add_storage(f"{n}_cache{layer}", pages * kv * page_size * size, "byte") for n in "kv"]
        g.kernel(decoding.paged_append(tokens, kv_heads, 64, page_size, pages, cache, rows, ks=step, vs=step, ko=hidden, vo=hidden + kv),
                 [qkv, qkv, tok, fork] + caches)
        names = decoding.paged_attention(tokens, rows, heads, kv_heads, 64, page_size, max_pages, pages, cache, qs=step)
        ctx = g.temp(tokens * hidden)
        args = [qkv] + caches + [table, tok, ctx]
        if len(names) > 1:
            from .. import capi
            parts = g.add_storage("parts", capi.Kernel(names[0]).arg_bytes[6], "byte")
            g.kernel(names[0], args + [parts])
            g.kernel(names[1], [parts, ctx])
        else:
            g.kernel(names[0], args)
        att = b.matmul(ctx, tokens, hidden, hidden, residual=x)
        x1 = b.layernorm(att, tokens, hidden)
        h1 = b.matmul(x1, tokens, ffn, hidden, gelu=True)
        h2 = b.matmul(h1, tokens, hidden, ffn, residual=x1)
        x = b.layernorm(h2, tokens, hidden)
    logits = b.matmul(x, tokens, vocab, hidden, out=g.add_storage("output", tokens * vocab))
    scan, pick = decoding.beam_select(requests, beams, vocab, eos, tokens=tokens)
    from .. import capi
    held = g.add_storage("beams", capi.Kernel(scan).arg_bytes[-1], "byte")
    g.kernel(scan, [logits, live, start, held])
    g.kernel(pick, [held, score, live, start, i32(rows, "token_out"), i32(rows, "parent_out"), g.add_storage("score_out", rows), i32(rows, "live_out")])
    return b
