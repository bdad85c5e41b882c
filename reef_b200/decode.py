"""Operators of a decoding step on device tensors: what a program calls between the projections of a model that answers token by token.

    state = page_state(rows, max_pages, tokens)                           # two of them, filled in turn
    state = page_tables(old.table, old.lens, new, pages=..., page_size=..., tokens=..., parent=..., out=state)
    paged_append(k, v, state.tok, k_cache, v_cache, fork=state.fork)      # per layer
    ctx = paged_attention(q, k_cache, v_cache, state.table, state.tok)    # per layer
    token, parent, score, live = beam_select(logits, score, live, beams=..., eos=..., start=state.start)

The same kernels run in schedules (kernel names in ``resources/decoding.py``, a model in ``resources/decoder.py``); here they are launched
on torch tensors.  Every call works on the current stream of its tensors' device, asynchronously; inputs used on another stream than
their own are the caller's to order and to keep alive, as with any other kernel.  Workspaces come from torch's allocator in every call, so
calls on several streams, from several threads and in captured graphs share nothing.  The first call on a device has to be made outside a
stream capture (it sets up the kernels there); with other shapes later calls may be captured at once.

Arguments are refused with ``ReefError`` (OutOfRange) before anything is launched.  Values on the device (lengths, ids, slots) are
not looked at by the host: the kernels bound every one of them.  There is no backward pass: inputs that require gradients are refused
while gradients are recorded.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .capi import OUT_OF_RANGE, FAIL, Kernel, ReefError
from .resources import decoding

_TYPES = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.float16: "float16"}


class PageState(NamedTuple):
    """What ``page_tables`` works out for a step; all int32, on the device."""
    table: torch.Tensor             # [rows][max_pages] pages of every row, -1 behind its last one
    lens: torch.Tensor              # [rows] tokens of every row, the new ones included
    start: torch.Tensor             # [rows + 1] first token of every row in the batch of new tokens
    tok: torch.Tensor               # [tokens][4] of every new token: slot in the cache, row, position + 1, 0; -1, -1, 0, 0 behind the last
    status: torch.Tensor            # [rows] 0; refused rows: 1 no pages left, 2 lengths, parent or ids out of range, 3 too many tokens
    fork: Optional[torch.Tensor] = None   # [rows][4] page to copy, its copy, tokens, 0; -1, -1, 0, 0 where there is nothing to copy


def page_state(rows: int, max_pages: int, tokens: int, *, fork: bool = False, device="cuda") -> PageState:
    """A state without any request: rows of length 0."""
    full = lambda *shape, value=0: torch.full(shape, value, dtype=torch.int32, device=device)   # noqa: E731
    tok = full(tokens, 4)
    tok[:, :2] = -1
    copies = full(rows, 4) if fork else None
    if fork:
        copies[:, :2] = -1
    return PageState(full(rows, max_pages, value=-1), full(rows), full(rows + 1), tok, full(rows), copies)


# ---- checks and launches -------------------------------------------------------------------------------------------------
def _refuse(what: str, why: str):
    raise ReefError(OUT_OF_RANGE, what, why)


_ready = set()      # devices whose kernels are set up
_kernels = {}       # (operator, device, shapes, strides, types, options) -> kernels: a signature is checked once


def _signature(*tensors):
    return tuple((t.shape, t.stride(), t.dtype, t.device) if t is not None else None for t in tensors)


def _inference(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _refuse(what, "inputs require gradients and there is no backward pass (use torch.no_grad)")


def _want(what, name, t, shape, dtype=torch.int32, device=None, dense=True):
    if not isinstance(t, torch.Tensor):
        _refuse(what, f"{name} is not a tensor")
    if t.dtype != dtype:
        _refuse(what, f"{name} is {t.dtype}, not {dtype}")
    if tuple(t.shape) != tuple(shape):
        _refuse(what, f"{name} has the shape {tuple(t.shape)}, not {tuple(shape)}")
    if not t.is_cuda:
        _refuse(what, f"{name} is on {t.device}, not on a GPU")
    if device is not None and t.device != device:
        _refuse(what, f"{name} is on {t.device}, not on {device}")
    if dense and not t.is_contiguous():
        _refuse(what, f"{name} is not contiguous")


def _tensors(what, **named):
    """Ahead of the signature: what is looked up has to be tensors."""
    for name, t in named.items():
        if not isinstance(t, torch.Tensor):
            _refuse(what, f"{name} is not a tensor")


def _whole(what, name, v, lo, hi):
    if isinstance(v, bool) or not isinstance(v, int) or not lo <= v <= hi:
        _refuse(what, f"{name} = {v!r} is not a whole number from {lo} to {hi}")


def _token_stride(what, name, t, heads, dim):
    """[tokens][heads][dim] with any stride from token to token that keeps 16-byte loads aligned."""
    if t.dim() != 3 or t.stride(2) != 1 or t.stride(1) != dim and heads > 1:
        _refuse(what, f"{name} has strides {t.stride()}: the heads of a token lie side by side")
    step = t.stride(0) if t.shape[0] > 1 else heads * dim
    if step % 4 or step < heads * dim:
        _refuse(what, f"{name}: {step} values from token to token are not a multiple of 4 from {heads * dim} on")
    return step


def _resolve(what, device, names):
    try:
        kernels = [Kernel(n) for n in names]
    except ReefError as e:
        raise ReefError(OUT_OF_RANGE, what, str(e)) from None
    if device not in _ready:
        if torch.cuda.get_device_capability(device)[0] != 10:
            raise ReefError(FAIL, what, f"{device} is not an sm_100 GPU")
        with torch.cuda.device(device):
            if torch.cuda.is_current_stream_capturing():
                raise ReefError(FAIL, what, f"the first call on {device} has to be made outside a stream capture")
            kernels[0].prepare([0] * kernels[0].num_args)
        _ready.add(device)
    return kernels


def _aligned(what, pointers):
    for p in pointers:
        if p & 15:
            _refuse(what, "a tensor does not begin at a 16-byte boundary")


def _apart(what, ins, outs):
    """No output lies over an input or another output: a step reads one state and writes another, so that it can be run again."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in outs if t is not None]
    for i, (a, b) in enumerate(spans):
        for c, d in spans[:i]:
            if a < d and c < b:
                _refuse(what, "outputs lie over each other")
    for t in ins:
        if t is not None:
            c = t.data_ptr()
            d = c + t.numel() * t.element_size()
            for a, b in spans:
                if a < d and c < b:
                    _refuse(what, "an output lies over an input")


def _launch(device, launches):
    """launches: (kernel, pointers), in order, on the device's current stream"""
    if device.index == torch.cuda.current_device():
        stream = torch.cuda.current_stream(device).cuda_stream
        for kernel, pointers in launches:
            kernel.launch(pointers, stream)
    else:
        with torch.cuda.device(device):
            stream = torch.cuda.current_stream(device).cuda_stream
            for kernel, pointers in launches:
                kernel.launch(pointers, stream)


# ---- operators -------------------------------------------------------------------------------------------------------------
def page_tables(table, lens, new, *, pages: int, page_size: int, tokens: int, parent=None, out: Optional[PageState] = None) -> PageState:
    """Page tables, token slots and page copies of a step, from the lengths of the requests.

    ``table`` [rows][max_pages] and ``lens`` [rows]: the state before the step; ``new`` [rows]: tokens that every row adds; all int32.
    ``pages`` of ``page_size`` tokens make up the cache; ``tokens``: the most new tokens.  ``parent`` [rows]: the row that each row goes on
    from (its own, another's, or -1: from nothing, for a request that begins or a row that ends); without it every row goes on
    from itself.  A row of length 0 is free: pages that no row names are free pages, nothing else keeps track of them.

    A row gets free pages, lowest id first, where its tokens need them.  Rows that go on from the same parent share its full pages; a last
    page that is partly filled stays with the lowest of them, and ``fork`` names the copies that the others need (``paged_append`` makes
    them).  Rows may come in with shared pages as long as these are full.  An id of -1 stands for a page that has been given up
    (``paged_attention`` leaves its tokens out).  Rows that cannot be served are refused by ``status`` and come out empty; the old state is
    still there, as ``out`` may not lie over it.
    """
    what = "page_tables"
    _tensors(what, table=table, lens=lens, new=new)
    key = (what, _signature(table, lens, new, parent, *(out or ())), pages, page_size, tokens)
    _inference(what, table, lens, new, parent)
    kernels = _kernels.get(key)
    if kernels is None:
        if table.dim() != 2:
            _refuse(what, "table is not [rows][max_pages]")
        rows, device = table.shape[0], table.device
        for name, v, hi in (("pages", pages, 1 << 19), ("page_size", page_size, 1024), ("tokens", tokens, 1 << 20)):
            _whole(what, name, v, 1, hi)
        if not 1 <= rows <= 1024 or table.shape[1] < 1:
            _refuse(what, f"a table of {tuple(table.shape)}: 1 to 1024 rows of a page or more")
        _want(what, "table", table, table.shape)
        _want(what, "lens", lens, (rows,), device=device)
        _want(what, "new", new, (rows,), device=device)
        if parent is not None:
            _want(what, "parent", parent, (rows,), device=device)
        if out is not None:
            if len(out) != 6:
                _refuse(what, "out is not a PageState")
            for name, t, shape in zip(PageState._fields, out, (table.shape, (rows,), (rows + 1,), (tokens, 4), (rows,), (rows, 4))):
                if name != "fork" or parent is not None:
                    _want(what, "out." + name, t, shape, device=device)
        kernels = _resolve(what, device, [decoding.page_tables(rows, table.shape[1], page_size, pages, tokens, parent is not None)])
        _kernels[key] = kernels
    if out is None:
        empty = lambda *shape: torch.empty(shape, dtype=torch.int32, device=table.device)    # noqa: E731
        rows = table.shape[0]
        out = PageState(torch.empty_like(table), empty(rows), empty(rows + 1), empty(tokens, 4), empty(rows),
                        None if parent is None else empty(rows, 4))
    elif parent is None and out[5] is not None:
        out = PageState(*out[:5], None)
    ins = [table, lens, new] + ([parent] if parent is not None else [])
    outs = [t for t in out if t is not None]
    _apart(what, ins, outs)
    pointers = [t.data_ptr() for t in ins + outs]
    _aligned(what, pointers[len(ins) + 3:len(ins) + 4] + pointers[len(ins) + 5:])
    _launch(table.device, [(kernels[0], pointers)])
    return out if isinstance(out, PageState) else PageState(*out)


def _cache(what, k_cache, v_cache, device):
    if k_cache.dim() != 4 or k_cache.dtype not in _TYPES:
        _refuse(what, f"k_cache is {k_cache.dtype} {tuple(k_cache.shape)}, not fp32, bf16 or fp16 [pages][kv heads][page size][dim]")
    _want(what, "k_cache", k_cache, k_cache.shape, k_cache.dtype, device)
    _want(what, "v_cache", v_cache, k_cache.shape, k_cache.dtype, device)
    pages, kv, page, dim = k_cache.shape
    if dim not in (64, 128, 256):
        _refuse(what, f"heads of {dim} dimensions: 64, 128 or 256")
    return pages, kv, page, dim


def paged_append(k, v, tok, k_cache, v_cache, *, fork=None) -> None:
    """Writes the keys and values of new tokens into the cache, and copies forked pages.

    ``k``, ``v`` [tokens][kv heads][dim] fp32, the heads of a token side by side, any stride from token to token (parts of a fused
    projection); ``tok`` [tokens][4] and ``fork`` [rows][4] from ``page_tables``; ``k_cache``, ``v_cache`` [pages][kv heads][page size][dim]
    in fp32, bf16 or fp16, rounded to nearest.  Tokens whose slot lies outside the cache are passed over.  Slots are distinct, and no
    token goes among those that a fork copies, as ``page_tables`` gives them; of two tokens with one slot either may be written, value by value.
    """
    what = "paged_append"
    _tensors(what, k=k, v=v, tok=tok, k_cache=k_cache, v_cache=v_cache)
    key = (what, _signature(k, v, tok, k_cache, v_cache, fork))
    _inference(what, k, v, k_cache, v_cache)
    kernels = _kernels.get(key)
    if kernels is None:
        device = k.device
        pages, kv, page, dim = _cache(what, k_cache, v_cache, device)
        shape = (k.shape[0] if k.dim() else 0, kv, dim)
        _want(what, "k", k, shape, torch.float32, device, dense=False)
        _want(what, "v", v, shape, torch.float32, device, dense=False)
        _want(what, "tok", tok, (shape[0], 4), device=device)
        if not shape[0]:
            _refuse(what, "no tokens")
        if fork is not None:
            if not isinstance(fork, torch.Tensor) or fork.dim() != 2 or not fork.shape[0]:
                _refuse(what, "fork is not [rows][4]")
            _want(what, "fork", fork, (fork.shape[0], 4), device=device)
        strides = dict(ks=_token_stride(what, "k", k, kv, dim), vs=_token_stride(what, "v", v, kv, dim))
        kernels = _resolve(what, device, [decoding.paged_append(shape[0], kv, dim, page, pages, _TYPES[k_cache.dtype],
                                                                0 if fork is None else fork.shape[0], **strides)])
        _kernels[key] = kernels
    _apart(what, [tok, fork], [k_cache, v_cache])
    ins = [k, v, tok] + ([fork] if fork is not None else [])
    pointers = [t.data_ptr() for t in ins + [k_cache, v_cache]]
    _aligned(what, pointers)
    lo, hi = (min(pointers[-2:]), max(p + c.numel() * c.element_size() for p, c in zip(pointers[-2:], (k_cache, v_cache))))
    for p, t in zip(pointers, (k, v)):
        if lo < p + 4 * ((t.shape[0] - 1) * t.stride(0) + t.shape[1] * t.shape[2]) and p < hi:
            _refuse(what, "keys or values lie within the caches' memory")
    _launch(k.device, [(kernels[0], pointers)])


def paged_attention(q, k_cache, v_cache, table, tok, *, out=None):
    """Attention of every token of the batch to the keys of its row: ``tok[t]`` = (anything, row, length, anything) from ``page_tables``.

    ``q`` [tokens][heads][dim] fp32 (any stride from token to token), caches [pages][kv heads][page size][dim] in fp32, bf16 or fp16,
    ``table`` [rows][max_pages] int32; heads are a multiple of the kv heads, consecutive heads share one.  A token sees the first ``length`` tokens
    of its row, but for those on pages whose id is outside the cache; where it sees none (a token without a row, length 0) its
    output is zero.  Scores are scaled by 1 / sqrt(dim); sums and the softmax are fp32 whatever the cache's type.  Returns
    [tokens][heads][dim] fp32.
    """
    what = "paged_attention"
    _tensors(what, q=q, k_cache=k_cache, v_cache=v_cache, table=table, tok=tok)
    key = (what, _signature(q, k_cache, v_cache, table, tok, out))
    _inference(what, q, k_cache, v_cache)
    kernels = _kernels.get(key)
    if kernels is None:
        device = q.device
        pages, kv, page, dim = _cache(what, k_cache, v_cache, device)
        if q.dim() != 3 or not q.shape[0] or not q.shape[1] or q.shape[1] % kv:
            _refuse(what, f"q of {tuple(q.shape)}: [tokens][heads][dim], heads a multiple of {kv}")
        _want(what, "q", q, (q.shape[0], q.shape[1], dim), torch.float32, device, dense=False)
        if table.dim() != 2 or not table.shape[0] or not table.shape[1]:
            _refuse(what, "table is not [rows][max_pages]")
        _want(what, "table", table, table.shape, device=device)
        _want(what, "tok", tok, (q.shape[0], 4), device=device)
        if out is not None:
            _want(what, "out", out, q.shape, torch.float32, device)
        names = decoding.paged_attention(q.shape[0], table.shape[0], q.shape[1], kv, dim, page, table.shape[1], pages, _TYPES[k_cache.dtype],
                                         qs=_token_stride(what, "q", q, q.shape[1], dim))
        kernels = _resolve(what, device, names)
        _kernels[key] = kernels
    if out is None:
        out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    else:
        _apart(what, [k_cache, v_cache, table, tok], [out])
        a, b = q.data_ptr(), out.data_ptr()
        if a < b + 4 * out.numel() and b < a + 4 * ((q.shape[0] - 1) * q.stride(0) + q.shape[1] * q.shape[2]):
            _refuse(what, "an output lies over an input")
    pointers = [q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), tok.data_ptr(), out.data_ptr()]
    _aligned(what, pointers[:3] + pointers[4:])
    if len(kernels) == 1:
        _launch(q.device, [(kernels[0], pointers)])
    else:
        parts = torch.empty(kernels[0].arg_bytes[6], dtype=torch.uint8, device=q.device)
        at = parts.data_ptr()
        _launch(q.device, [(kernels[0], pointers + [at]), (kernels[1], [at, pointers[5]])])
    return out


def beam_select(logits, score, live, *, beams: int, eos: int, start=None, out=None):
    """The ``beams`` best continuations of every request, over its beams and the vocabulary.

    ``logits`` [rows][vocab] fp32, a row per beam, or with ``start`` [rows + 1] (``PageState.start``) a row per new token: a beam's last
    token counts.  ``score`` [rows] fp32: sums of log-probabilities; ``live`` [rows] int32: 0 for beams that have ended, which compete with their
    score and the word ``eos``.  rows = requests * beams, the beams of a request side by side.

    Returns (token, parent, score, live) of the new beams, best first, int32 but for the score; equal candidates by the lowest
    beam * vocab + word.  ``parent`` is a row, as ``page_tables`` wants it, and ``live`` (0 or 1) is what each row adds in the next step.  Where a
    request has fewer candidates above -infinity than beams, the rest are token -1, parent -1, score -infinity, live 0: a row of logits with a
    NaN, an infinity or nothing but -infinity has none, nor has a beam whose score is not finite.
    """
    what = "beam_select"
    _tensors(what, logits=logits, score=score, live=live)
    key = (what, _signature(logits, score, live, start, *(out or ())), beams, eos)
    _inference(what, logits, score)
    kernels = _kernels.get(key)
    if kernels is None:
        device = logits.device
        if logits.dim() != 2 or not logits.shape[0] or not logits.shape[1]:
            _refuse(what, "logits are not [rows][vocab]")
        _whole(what, "beams", beams, 1, 16)
        _whole(what, "eos", eos, 0, logits.shape[1] - 1)
        rows = score.shape[0] if score.dim() else 0
        if not rows or rows % beams or (start is None and logits.shape[0] != rows):
            _refuse(what, f"{rows} scores, {logits.shape[0]} rows of logits, {beams} beams to a request")
        _want(what, "logits", logits, logits.shape, torch.float32, device)
        _want(what, "score", score, (rows,), torch.float32, device)
        _want(what, "live", live, (rows,), device=device)
        if start is not None:
            _want(what, "start", start, (rows + 1,), device=device)
        if out is not None:
            if len(out) != 4:
                _refuse(what, "out is not (token, parent, score, live)")
            for name, t, dtype in zip(("token", "parent", "score", "live"), out, (torch.int32, torch.int32, torch.float32, torch.int32)):
                _want(what, "out " + name, t, (rows,), dtype, device)
        kernels = _resolve(what, device, decoding.beam_select(rows // beams, beams, logits.shape[1], eos,
                                                              None if start is None else logits.shape[0]))
        _kernels[key] = kernels
    if out is None:
        block = torch.empty(4, score.shape[0], dtype=torch.int32, device=logits.device)
        out = (block[0], block[1], block[2].view(torch.float32), block[3])
    else:
        _apart(what, [logits, score, live, start], out)
    first = [] if start is None else [start.data_ptr()]
    parts = torch.empty(kernels[0].arg_bytes[-1], dtype=torch.uint8, device=logits.device)
    at, rows_at, live_at = parts.data_ptr(), logits.data_ptr(), live.data_ptr()
    _aligned(what, [rows_at])
    _launch(logits.device, [(kernels[0], [rows_at, live_at] + first + [at]),
                            (kernels[1], [at, score.data_ptr(), live_at] + first + [t.data_ptr() for t in out])])
    return tuple(out)
