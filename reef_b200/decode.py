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
while gradients are recorded, and so are those that carry forward-mode tangents.
"""
from __future__ import annotations

import threading
from typing import NamedTuple, Optional

import torch

from .capi import FAIL, OUT_OF_RANGE, Kernel, ReefError, cuda_lib
from .resources import decoding


class _Unbuilt:
    """Stands for the native module until the first call: the libraries need not be built to import this one."""
    def __getattr__(self, name):
        global _decode
        cuda_lib()              # (raises where the libraries are not built)
        from . import _decode
        return getattr(_decode, name)


_decode = _Unbuilt()
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
# A signature (types, devices, sizes, strides, options) is checked and resolved here, once; from then on _decode.call does everything, for the
# last 4096 of them.
_TABLES, _APPEND, _ATTENTION, _BEAMS = range(4)
_ready = set()      # devices whose kernels are set up
_lock = threading.Lock()


def _refuse(what: str, why: str):
    raise ReefError(OUT_OF_RANGE, what, why)


def _again(what, op, inputs, outputs, options):
    """The call of a signature that has just been defined, or one that _decode.call has said no to."""
    got = _decode.call(op, inputs, outputs, options)
    if got.__class__ is not tuple:
        _refuse(what, got if isinstance(got, str) else "arguments changed during the call")
    return got


def _inference(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                _refuse(what, "inputs require gradients and there is no backward pass (use torch.no_grad)")
    if torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
                _refuse(what, "inputs carry tangents and there is no forward-mode derivative")


def _want(what, name, t, shape, dtype=torch.int32, device=None, dense=True):
    if not isinstance(t, torch.Tensor):
        _refuse(what, f"{name} is not a tensor")
    if t.dtype != dtype:
        _refuse(what, f"{name} is {t.dtype}, not {dtype}")
    if tuple(t.shape) != tuple(shape):
        _refuse(what, f"{name} has the shape {tuple(t.shape)}, not {tuple(shape)}")
    if t.is_neg():
        _refuse(what, f"{name} is a view that stands for its negative (resolve_neg makes it a tensor of its own)")
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


def _at_most(what, **limits):
    """What the kernels' whole numbers hold: name=(value, limit)."""
    for name, (v, most) in limits.items():
        if v > most:
            _refuse(what, f"{name.replace('_', ' ')}: {v}, at most {most}")


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
    with _lock:
        if device not in _ready:
            if torch.cuda.get_device_capability(device)[0] != 10:
                raise ReefError(FAIL, what, f"{device} is not an sm_100 GPU")
            with torch.cuda.device(device):
                if torch.cuda.is_current_stream_capturing():
                    raise ReefError(FAIL, what, f"the first call on {device} has to be made outside a stream capture")
                kernels[0].prepare([0] * kernels[0].num_args)
            _ready.add(device)
    return kernels


def _define(op, inputs, outputs, options, kernels, args, allocate, workspace, aligned, apart):
    """``args``: per kernel the tensors of its arguments, by position among inputs and outputs, -1 the workspace; ``allocate``: (input whose type
    it has or -1 for int32, shape) per output; ``apart``: (position, positions that it must not lie over)."""
    _decode.define(op, inputs, outputs, options, [(k.handle, k.dims, k.dyn_smem, a) for k, a in zip(kernels, args)], allocate, workspace, aligned,
                   [x for i, others in apart for j in others for x in (i, j)], kernels)


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
    (``paged_attention`` leaves its tokens out).

    Rows that cannot be served are refused by ``status`` and come out empty; the old tables are still there, as ``out`` may not lie over them.
    Where pages or tokens ran out (1, 3) the old pages are too: no row gets them in this step, and the row can be tried again from the old
    state.  A row whose lengths, parent or ids are out of range (2), one that is to grow beyond max_pages * page_size among them, keeps
    nothing: its pages are free for other rows at once, and ``paged_append`` will write there.  Whoever wants to keep such a row looks at
    its length first, or gives it no new tokens.

    Without ``parent`` there is nothing to copy: the state that comes back has no ``fork``, and one that ``out`` has is left as it was.
    """
    inputs, options = (table, lens, new, parent), (pages, page_size, tokens)
    outputs = None if out is None else tuple(out[:5] if parent is None else out)
    got = _decode.call(_TABLES, inputs, outputs, options)
    if got.__class__ is not tuple:
        got = _page_tables("page_tables", got, inputs, outputs, options)
    return PageState(*got)


def _page_tables(what, why, inputs, outputs, options):
    if why is not None:
        _refuse(what, why)
    table, lens, new, parent = inputs
    pages, page_size, tokens = options
    _tensors(what, table=table, lens=lens, new=new)
    _inference(what, *inputs)
    if table.dim() != 2:
        _refuse(what, "table is not [rows][max_pages]")
    (rows, max_pages), device = table.shape, table.device
    for name, v, hi in (("pages", pages, 1 << 19), ("page_size", page_size, 1024), ("tokens", tokens, 1 << 20)):
        _whole(what, name, v, 1, hi)
    if not 1 <= rows <= 1024 or max_pages < 1:
        _refuse(what, f"a table of {tuple(table.shape)}: 1 to 1024 rows of a page or more")
    _at_most(what, tokens_of_a_row=(max_pages * page_size, 1 << 30), ids_of_the_table=(rows * max_pages, 1 << 30))
    _want(what, "table", table, table.shape)
    _want(what, "lens", lens, (rows,), device=device)
    _want(what, "new", new, (rows,), device=device)
    if parent is not None:
        _want(what, "parent", parent, (rows,), device=device)
    shapes = [(rows, max_pages), (rows,), (rows + 1,), (tokens, 4), (rows,)] + ([(rows, 4)] if parent is not None else [])
    if outputs is not None:
        if len(outputs) != len(shapes):
            _refuse(what, "out is not a PageState")
        for name, t, shape in zip(PageState._fields, outputs, shapes):
            _want(what, "out." + name, t, shape, device=device)
    kernels = _resolve(what, device, [decoding.page_tables(rows, max_pages, page_size, pages, tokens, parent is not None)])
    ins = [0, 1, 2] + ([3] if parent is not None else [])
    outs = list(range(4, 4 + len(shapes)))
    _define(_TABLES, inputs, outputs, options, kernels, [ins + outs], [(-1, s) for s in shapes], 0, [7] + outs[5:],
            [(o, ins + outs[:n]) for n, o in enumerate(outs)])
    return _again(what, _TABLES, inputs, outputs, options)


def _cache(what, k_cache, v_cache, device):
    if k_cache.dim() != 4 or k_cache.dtype not in _TYPES:
        _refuse(what, f"k_cache is {k_cache.dtype} {tuple(k_cache.shape)}, not fp32, bf16 or fp16 [pages][kv heads][page size][dim]")
    pages, kv, page, dim = k_cache.shape
    _at_most(what, kv_heads=(kv, 1024), tokens_of_a_page=(page, 1024), tokens_of_the_cache=(pages * page, 0x7fffffff))
    _want(what, "k_cache", k_cache, k_cache.shape, k_cache.dtype, device)
    _want(what, "v_cache", v_cache, k_cache.shape, k_cache.dtype, device)
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
    inputs = (k, v, tok, k_cache, v_cache, fork)
    got = _decode.call(_APPEND, inputs, None, ())
    if got.__class__ is not tuple:
        _paged_append("paged_append", got, inputs)


def _paged_append(what, why, inputs):
    if why is not None:
        _refuse(what, why)
    k, v, tok, k_cache, v_cache, fork = inputs
    _tensors(what, k=k, v=v, tok=tok, k_cache=k_cache, v_cache=v_cache)
    _inference(what, *inputs)
    device = k.device
    if k.dim() == 3:
        _at_most(what, tokens=(k.shape[0], 1 << 20), values_of_all_tokens=(k.shape.numel(), 0x70000000))
    if fork is not None:
        if not isinstance(fork, torch.Tensor) or fork.dim() != 2 or not fork.shape[0]:
            _refuse(what, "fork is not [rows][4]")
        _at_most(what, forks=(fork.shape[0], 1 << 20))
    pages, kv, page, dim = _cache(what, k_cache, v_cache, device)
    shape = (k.shape[0] if k.dim() else 0, kv, dim)
    _want(what, "k", k, shape, torch.float32, device, dense=False)
    _want(what, "v", v, shape, torch.float32, device, dense=False)
    _want(what, "tok", tok, (shape[0], 4), device=device)
    if not shape[0]:
        _refuse(what, "no tokens")
    if fork is not None:
        _want(what, "fork", fork, (fork.shape[0], 4), device=device)
    strides = dict(ks=_token_stride(what, "k", k, kv, dim), vs=_token_stride(what, "v", v, kv, dim))
    kernels = _resolve(what, device, [decoding.paged_append(shape[0], kv, dim, page, pages, _TYPES[k_cache.dtype],
                                                            0 if fork is None else fork.shape[0], **strides)])
    copies = [] if fork is None else [5]
    _define(_APPEND, inputs, None, (), kernels, [[0, 1, 2] + copies + [3, 4]], [], 0, [0, 1, 2, 3, 4] + copies,
            [(3, [0, 1, 2, 4] + copies), (4, [0, 1, 2] + copies)])
    _again(what, _APPEND, inputs, None, ())


def paged_attention(q, k_cache, v_cache, table, tok, *, out=None):
    """Attention of every token of the batch to the keys of its row: ``tok[t]`` = (anything, row, length, anything) from ``page_tables``.

    ``q`` [tokens][heads][dim] fp32 (any stride from token to token), caches [pages][kv heads][page size][dim] in fp32, bf16 or fp16,
    ``table`` [rows][max_pages] int32; heads are a multiple of the kv heads, consecutive heads share one.  A token sees the first ``length`` tokens
    of its row, but for those on pages whose id is outside the cache; where it sees none (a token without a row, length 0) its
    output is zero.  Scores are scaled by 1 / sqrt(dim); sums and the softmax are fp32 whatever the cache's type.  Returns
    [tokens][heads][dim] fp32.

    Up to 65536 tokens and rows, 1024 heads, pages of 1024 tokens, rows of 2^30; pages * kv heads * page size of the cache are below 2^31.
    """
    inputs, outputs = (q, k_cache, v_cache, table, tok), None if out is None else (out,)
    got = _decode.call(_ATTENTION, inputs, outputs, ())
    if got.__class__ is not tuple:
        got = _paged_attention("paged_attention", got, inputs, outputs)
    return got[0]


def _paged_attention(what, why, inputs, outputs):
    if why is not None:
        _refuse(what, why)
    q, k_cache, v_cache, table, tok = inputs
    _tensors(what, q=q, k_cache=k_cache, v_cache=v_cache, table=table, tok=tok)
    _inference(what, *inputs)
    device = q.device
    if q.dim() == 3 and table.dim() == 2 and k_cache.dim() == 4:
        _at_most(what, tokens=(q.shape[0], 1 << 16), heads=(q.shape[1], 1024), rows=(table.shape[0], 1 << 16),
                 tokens_of_a_row=(table.shape[1] * k_cache.shape[2], 1 << 30), keys_of_the_cache=(k_cache.shape[:3].numel(), 0x7fffffff))
    pages, kv, page, dim = _cache(what, k_cache, v_cache, device)
    if q.dim() != 3 or not q.shape[0] or not q.shape[1] or q.shape[1] % kv:
        _refuse(what, f"q of {tuple(q.shape)}: [tokens][heads][dim], heads a multiple of {kv}")
    _want(what, "q", q, (q.shape[0], q.shape[1], dim), torch.float32, device, dense=False)
    if table.dim() != 2 or not table.shape[0] or not table.shape[1]:
        _refuse(what, "table is not [rows][max_pages]")
    _want(what, "table", table, table.shape, device=device)
    _want(what, "tok", tok, (q.shape[0], 4), device=device)
    if outputs is not None:
        _want(what, "out", outputs[0], q.shape, torch.float32, device)
    names = decoding.paged_attention(q.shape[0], table.shape[0], q.shape[1], kv, dim, page, table.shape[1], pages, _TYPES[k_cache.dtype],
                                     qs=_token_stride(what, "q", q, q.shape[1], dim))
    kernels = _resolve(what, device, names)
    whole = [0, 1, 2, 3, 4, 5]
    args, workspace = ([whole], 0) if len(kernels) == 1 else ([whole + [-1], [-1, 5]], kernels[0].arg_bytes[6])
    _define(_ATTENTION, inputs, outputs, (), kernels, args, [(0, q.shape)], workspace, [0, 1, 2, 4, 5], [(5, [0, 1, 2, 3, 4])])
    return _again(what, _ATTENTION, inputs, outputs, ())


def beam_select(logits, score, live, *, beams: int, eos: int, start=None, out=None):
    """The ``beams`` best continuations of every request, over its beams and the vocabulary.

    ``logits`` [rows][vocab] fp32, a row per beam, or with ``start`` [rows + 1] (``PageState.start``) a row per new token: a beam's last
    token counts.  ``score`` [rows] fp32: sums of log-probabilities; ``live`` [rows] int32: 0 for beams that have ended, which compete with their
    score and the word ``eos``.  rows = requests * beams, the beams of a request side by side.

    Returns (token, parent, score, live) of the new beams, best first, int32 but for the score.  Candidates are compared in 64 bits; of equal ones
    the lower beam's come first, and of one beam's those of the greater logits, then of the lower words.  ``parent`` is a row, as ``page_tables`` wants it, and ``live`` (0 or 1) is what each row adds in the next step.  Where a
    request has fewer candidates above -infinity than beams, the rest are token -1, parent -1, score -infinity, live 0: a row of logits with a
    NaN, an infinity or nothing but -infinity has none, nor has a beam whose score is not finite.
    """
    inputs, outputs, options = (logits, score, live, start), None if out is None else tuple(out), (beams, eos)
    got = _decode.call(_BEAMS, inputs, outputs, options)
    if got.__class__ is not tuple:
        got = _beam_select("beam_select", got, inputs, outputs, options)
    return got


def _beam_select(what, why, inputs, outputs, options):
    if why is not None:
        _refuse(what, why)
    logits, score, live, start = inputs
    beams, eos = options
    _tensors(what, logits=logits, score=score, live=live)
    _inference(what, *inputs)
    device = logits.device
    if logits.dim() != 2 or not logits.shape[0] or not logits.shape[1]:
        _refuse(what, "logits are not [rows][vocab]")
    _whole(what, "beams", beams, 1, 16)
    _whole(what, "eos", eos, 0, logits.shape[1] - 1)
    rows = score.shape[0] if score.dim() else 0
    _at_most(what, words=(logits.shape[1], 0x7fffffff // 16), rows=(rows, 1 << 20), rows_of_logits=(logits.shape[0], 1 << 20))
    if not rows or rows % beams or (start is None and logits.shape[0] != rows):
        _refuse(what, f"{rows} scores, {logits.shape[0]} rows of logits, {beams} beams to a request")
    _want(what, "logits", logits, logits.shape, torch.float32, device)
    _want(what, "score", score, (rows,), torch.float32, device)
    _want(what, "live", live, (rows,), device=device)
    if start is not None:
        _want(what, "start", start, (rows + 1,), device=device)
    if outputs is not None:
        if len(outputs) != 4:
            _refuse(what, "out is not (token, parent, score, live)")
        for name, t, dtype in zip(("token", "parent", "score", "live"), outputs, (torch.int32, torch.int32, torch.float32, torch.int32)):
            _want(what, "out " + name, t, (rows,), dtype, device)
    kernels = _resolve(what, device, decoding.beam_select(rows // beams, beams, logits.shape[1], eos, None if start is None else logits.shape[0]))
    first = [] if start is None else [3]
    ins, outs = [0, 1, 2] + first, [4, 5, 6, 7]
    _define(_BEAMS, inputs, outputs, options, kernels, [[0, 2] + first + [-1], [-1, 1, 2] + first + outs],
            [(-1, (rows,)), (-1, (rows,)), (1, (rows,)), (-1, (rows,))], kernels[0].arg_bytes[-1], [0],
            [(o, ins + outs[:n]) for n, o in enumerate(outs)])
    return _again(what, _BEAMS, inputs, outputs, options)
