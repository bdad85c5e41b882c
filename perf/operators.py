"""The operators of a decoding step: what a server that answers token by token calls between its projections.

``tables``   page tables, token slots and page forks from the lengths of the requests (``decode.page_tables``)
``append``   new keys and values into the paged cache, forked pages copied first (``decode.paged_append``)
``attend``   attention of one new token per row over the paged cache (``decode.paged_attention``)
``beam``     the best continuations of every request's beams over the vocabulary (``decode.beam_select``)

The ranges: 1 to 256 rows, caches of one token to 131072 tokens a row in pages of 1 to 128, 1 to 64 heads over 1 to 16 key-value heads
of 64, 128 or 256 dimensions, fp32, bf16 and fp16 caches, 1 to 16 beams over vocabularies of 1000 to 131072 words.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- cases -------------------------------------------------------------------------------------------------------------
def _tables(name, rows, page, max_pages, pages, cached, new, tokens, beams=0):
    """``cached``: tokens in the caches of all rows together; ``new``: tokens they add together; ``tokens``: room for new ones;
    ``beams`` > 0: rows are beams of requests and continue from a parent each."""
    return dict(name=name, op="tables", rows=rows, page=page, max_pages=max_pages, pages=pages, cached=cached, new=new, tokens=tokens,
                beams=beams)


def _append(name, tokens, kv, dim, page, pages, type, idle=0, forks=0):
    """``idle``: tokens of the batch that belong to no row; ``forks``: rows whose last page is copied first."""
    return dict(name=name, op="append", tokens=tokens, kv=kv, dim=dim, page=page, pages=pages, type=type, idle=idle, forks=forks)


def _attend(name, rows, heads, kv, dim, page, longest, cached, type, idle=0, gone=0):
    """``longest``: the most tokens a row can hold; ``cached``: tokens of all rows; ``idle``: rows without a request; ``gone``: rows
    whose first page has been given up."""
    return dict(name=name, op="attend", rows=rows, heads=heads, kv=kv, dim=dim, page=page, longest=longest, cached=cached, type=type,
                idle=idle, gone=gone)


def _beam(name, requests, beams, vocab, finished=0):
    """``finished``: beams that have ended already and compete with their score."""
    return dict(name=name, op="beam", requests=requests, beams=beams, vocab=vocab, finished=finished)


def listed():
    return [
        # a small chat server's step: sixteen rows, one token each
        _tables("tables_decode_16", 16, 16, 64, 1024, 8000, 16, 16),
        # thirty-two requests of four beams that were just selected: every row continues from some beam of its request
        _tables("tables_beams_128", 128, 16, 129, 20001, 100000, 128, 128, beams=4),
        # a full server: 256 rows, most decoding, some with a prompt to come, two million tokens cached
        _tables("tables_mixed_256", 256, 32, 1024, 100000, 2000000, 8000, 8192),
        # the keys and values of a step of 128 beams, a third of which have to take a copy of their parent's last page
        _append("append_beams_128", 128, 12, 64, 16, 2048, "fp32", idle=3, forks=40),
        # prompts of 8192 tokens in all
        _append("append_prompt_8192", 8192, 8, 128, 32, 1024, "bf16"),
        # one user, a short question: the whole call is latency
        _attend("attend_1x77", 1, 12, 12, 64, 16, 1024, 77, "fp32"),
        # sixteen rows of a model with as many key heads as query heads
        _attend("attend_16_mha", 16, 12, 12, 64, 16, 1024, 9001, "bf16", idle=1),
        # grouped heads, ragged lengths: the ordinary full server
        _attend("attend_64_gqa", 64, 32, 8, 128, 32, 8192, 210000, "bf16"),
        # a single long document, few key-value heads: all parallelism is along the length
        _attend("attend_1x131072", 1, 16, 2, 128, 64, 131072, 131072, "fp16"),
        # nothing divides anything: pages of 24, groups of 5, rows that have given up their first page
        _attend("attend_37_odd", 37, 15, 3, 128, 24, 4008, 61003, "fp32", idle=2, gone=5),
        # one request, four beams
        _beam("beam_1x4", 1, 4, 30522),
        # thirty-two requests of eight beams over a wide vocabulary, some beams finished
        _beam("beam_32x8", 32, 8, 100003, finished=20),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend", "beam"])
    if op == "tables":
        page, rows = rng.choice([1, 8, 16, 24, 32, 64, 128]), _log(rng, 1, 256)
        max_pages = _log(rng, 4, 1024)
        cached = int(rows * page * max_pages * rng.uniform(0.05, 0.5))
        beams = rng.choice([0, 0, 2, 3, 4, 8])
        rows = max(beams, rows // beams * beams) if beams else rows
        cached = min(cached, rows * page * max_pages // 2)
        new = rows if beams else _log(rng, rows, max(rows, min(8192, rows * page * max_pages // 4)))
        # now and then more is asked for than there is room: tokens, or pages
        spare = rng.choice([2 * rows + new // page + 9, 2 * rows + new // page + rng.randint(1, 9999), rng.randint(0, 1 + rows // 2)])
        case = _tables("", rows, page, max_pages, cached // page + rows + spare, cached, new,
                       rng.choice([new + rng.randint(0, 9), new + rng.randint(0, 9), new - new // 4]), beams)
    elif op == "append":
        kv, dim, page, type = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([64, 128, 256]), rng.choice([1, 8, 16, 24, 32, 64, 128]), \
            rng.choice(["fp32", "bf16", "fp16"])
        tokens = _log(rng, 1, max(2, min(8192, 8192 * 8 * 128 // (kv * dim))))
        pages = tokens // page + 3 * rng.randint(1, 64) + 64
        case = _append("", tokens, kv, dim, page, pages, type, idle=rng.choice([0, 0, tokens // 7]),
                       forks=rng.choice([0, 0, min(tokens, 20)]) if page > 1 else 0)
    elif op == "attend":
        kv, group, dim = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16]), rng.choice([64, 64, 128, 128, 256])
        group = min(group, 64 // kv)
        type, page = rng.choice(["fp32", "bf16", "bf16", "fp16"]), rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
        rows = _log(rng, 1, 256)
        most = int(1.5e8 / (rows * kv * dim))                # so that no case reads more than the largest listed one
        longest = max(page, _log(rng, 16, max(17, min(131072, most))) // page * page)
        cached = max(rows, int(rows * longest * rng.uniform(0.1, 0.9)))
        case = _attend("", rows, kv * group, kv, dim, page, longest, cached, type, idle=rng.choice([0, 0, rows // 5]),
                       gone=rng.choice([0, 0, 0, rows // 6]))
    else:
        beams, vocab = rng.choice([1, 2, 3, 4, 5, 8, 8, 16]), _log(rng, 1000, 131072)
        requests = _log(rng, 1, max(1, min(64, int(2.5e7 / (beams * vocab)))))
        case = _beam("", requests, beams, vocab, finished=rng.choice([0, 0, requests * beams // 8]))
    del case["name"]
    return case


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _parts(rng, n, total, least, most):
    """n whole numbers from least to most that add up to total, ragged as lengths of requests are."""
    total = min(max(total, n * least), n * most)
    w = rng.lognormal(0.0, 0.8, n)
    x = np.minimum(least + np.floor((total - n * least) * w / w.sum()).astype(np.int64), most)
    while x.sum() < total:
        room = np.flatnonzero(x < most)
        step = max(1, (total - int(x.sum())) // len(room))
        x[room] = np.minimum(x[room] + step, most)
        over = int(x.sum()) - total
        for i in room[::-1]:
            if over <= 0:
                break
            back = min(over, int(x[i]) - least, step)
            x[i] -= back
            over -= back
    return x


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _normal(gen, *shape, type=torch.float32):
    out = torch.empty(*shape, dtype=type, device="cuda")
    return out.normal_(generator=gen)


def _paged(rng, lens, page, max_pages, pages):
    """A table of pages in no order for rows of these lengths, -1 behind each row's last page."""
    table = np.full((len(lens), max_pages), -1, np.int32)
    ids, at = rng.permutation(pages).astype(np.int32), 0
    for r, l in enumerate(lens):
        n = -(-int(l) // page)
        table[r, :n] = ids[at:at + n]
        at += n
    return table


def prepare(case, seed):
    rng = np.random.default_rng([seed, 77])
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "tables":
        rows, page, beams = case["rows"], case["page"], case["beams"]
        if beams:
            # beams of a request are of one length; they share the pages of the request's prompt (two thirds, whole pages)
            each = _parts(rng, rows // beams, case["cached"] // beams, 1, page * case["max_pages"] - 1)
            lens = np.repeat(each, beams)
            table = _paged(rng, lens, page, case["max_pages"], case["pages"] + rows * case["max_pages"])
            for r in range(rows):
                n = int(lens[r]) * 2 // (3 * page)
                table[r, :n] = table[r // beams * beams, :n]
            ids = np.unique(table[table >= 0])
            names = rng.permutation(case["pages"])[:len(ids)].astype(np.int32)
            assert len(names) == len(ids), "a pool that holds the rows"
            table[table >= 0] = names[np.searchsorted(ids, table[table >= 0])]
            s["parent"] = _dev((np.arange(rows) // beams * beams + rng.integers(0, beams, rows)).astype(np.int32))
            new = np.ones(rows, np.int64)
        else:
            lens = _parts(rng, rows, case["cached"], 0, page * case["max_pages"] * 3 // 4)
            table = _paged(rng, lens, page, case["max_pages"], case["pages"])
            new = np.ones(rows, np.int64)
            some = rng.permutation(rows)[:max(1, rows // 16)]
            new[some] += _parts(rng, len(some), case["new"] - rows, 0, page * case["max_pages"] // 4 - 1)
            s["parent"] = None
        s["table"], s["lens"], s["new"] = _dev(table), _dev(lens.astype(np.int32)), _dev(new.astype(np.int32))
        # the program's other set of tables, which this step fills
        shapes = [(rows, case["max_pages"]), (rows,), (rows + 1,), (case["tokens"], 4), (rows,)] + ([(rows, 4)] if beams else [])
        s["out"] = [torch.zeros(shape, dtype=torch.int32, device="cuda") for shape in shapes]
    elif case["op"] == "append":
        T, kv, dim, page, pages = (case[k] for k in ("tokens", "kv", "dim", "page", "pages"))
        kind = _TYPES[case["type"]]
        s["k"], s["v"] = _normal(gen, T, kv, dim), _normal(gen, T, kv, dim)
        s["k_cache"], s["v_cache"] = (_normal(gen, pages, kv, page, dim, type=kind) for _ in range(2))
        # forked rows write behind the tokens that they copy; the others into pages of their own
        ids = rng.permutation(pages)
        f = case["forks"]
        src, dst, rest = ids[:f], ids[f:2 * f], ids[2 * f:]
        slots = np.full(T, -1, np.int64)
        live = T - case["idle"]
        free = (rest[:, None] * page + np.arange(page)).reshape(-1)
        keep = rng.integers(1, page, f) if f else np.zeros(0, np.int64)
        slots[:live] = free[:live]
        slots[:min(f, live)] = (dst * page + keep)[:min(f, live)]
        tok = np.zeros((T, 4), np.int32)
        tok[:, 0], tok[:, 1], tok[:, 2] = slots, np.where(slots < 0, -1, np.arange(T)), np.where(slots < 0, 0, 1)
        s["tok"] = _dev(tok)
        s["fork"] = None
        if f:
            fork = np.full((T, 4), -1, np.int32)
            fork[:, 2:] = 0
            fork[:f] = np.stack([src, dst, keep, np.zeros(f, np.int64)], 1)
            s["fork"] = _dev(fork)
    elif case["op"] == "attend":
        rows, heads, kv, dim, page = (case[k] for k in ("rows", "heads", "kv", "dim", "page"))
        live = rows - case["idle"]
        lens = np.zeros(rows, np.int64)
        lens[:live] = _parts(rng, live, case["cached"], 1, case["longest"])
        pages = int(sum(-(-int(l) // page) for l in lens)) + 7
        table = _paged(rng, lens, page, -(-case["longest"] // page), pages)
        table[:case["gone"], 0] = -1
        tok = np.zeros((rows, 4), np.int32)
        tok[:, 0], tok[:, 1], tok[:, 2] = np.where(lens > 0, 0, -1), np.where(lens > 0, np.arange(rows), -1), lens
        s["table"], s["tok"] = _dev(table), _dev(tok)
        s["q"] = _normal(gen, rows, heads, dim)
        s["k_cache"], s["v_cache"] = (_normal(gen, pages, kv, page, dim, type=_TYPES[case["type"]]) for _ in range(2))
    else:
        n = case["requests"] * case["beams"]
        # logits as a bf16 projection gives them: equal ones among the highest are not rare
        s["logits"] = (3.0 * _normal(gen, n, case["vocab"])).bfloat16().float()
        s["score"] = _dev(np.sort(rng.normal(-12.0, 1.0, n).astype(np.float32)))
        live = np.ones(n, np.int32)
        live[rng.permutation(n)[:case["finished"]]] = 0
        s["live"] = _dev(live)
    return s


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _run_own(s):
    from reef_b200 import decode
    case = s["case"]
    if case["op"] == "tables":
        out = decode.page_tables(s["table"], s["lens"], s["new"], pages=case["pages"], page_size=case["page"], tokens=case["tokens"],
                                 parent=s["parent"], out=decode.PageState(*s["out"]))
        return [x for x in out if x is not None]
    if case["op"] == "append":
        decode.paged_append(s["k"], s["v"], s["tok"], s["k_cache"], s["v_cache"], fork=s["fork"])
        return [s["k_cache"], s["v_cache"]]
    if case["op"] == "attend":
        return [decode.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["tok"])]
    return list(decode.beam_select(s["logits"], s["score"], s["live"], beams=case["beams"], eos=2))


# ---- plain forms -------------------------------------------------------------------------------------------------------
def _plain_tables(case, table, lens, new, parent):
    R, M, S, N, T = case["rows"], case["max_pages"], case["page"], case["pages"], case["tokens"]
    dev, dump = table.device, torch.iinfo(torch.int64).max
    rows, cols = torch.arange(R, device=dev), torch.arange(M, device=dev)
    p = rows if parent is None else parent.long()
    named = (p >= -1) & (p < R)
    q = p.clamp(0, R - 1)
    l, n = torch.where(p < 0, 0, lens[q].long()), new.long()
    kept = torch.div(l + S - 1, S, rounding_mode="floor")
    have = cols < kept[:, None]
    entry = table[q].long()
    last = entry.gather(1, (kept - 1).clamp(0, M - 1)[:, None])[:, 0]
    valid = named & (l >= 0) & (n >= 0) & (l + n <= M * S)
    valid &= ~(have & ((entry < -1) | (entry >= N))).any(1) & ~((l % S > 0) & (last < 0))
    # room for tokens, then for pages: sums over the rows that are still in
    status = torch.where(valid, 0, 2)
    over = valid & (torch.cumsum(torch.where(valid, n, 0), 0) > T)
    status = torch.where(over, 3, status)
    slot_of = torch.where(valid & (p >= 0), q, R)
    first = torch.full((R + 1,), dump, device=dev).scatter_reduce(0, slot_of, rows, "amin")
    forked = valid & (p >= 0) & (l % S > 0) & (first[q] != rows)
    live = have & valid[:, None] & (entry >= 0)
    used = torch.zeros(N + 1, dtype=torch.int64, device=dev).scatter(0, torch.where(live, entry, N).reshape(-1), 1)[:N]
    rank = torch.cumsum(1 - used, 0)
    free = torch.zeros(N + 1, dtype=torch.int64, device=dev).scatter(0, torch.where(used > 0, N, rank - 1), torch.arange(N, device=dev))
    need = torch.div(l + n + S - 1, S, rounding_mode="floor") - kept + forked
    need = torch.where(status == 0, need, 0)
    upto = torch.cumsum(need, 0)
    status = torch.where((status == 0) & (need > 0) & (upto > N - used.sum()), 1, status)
    ok = status == 0
    l2, n2 = torch.where(ok, l, 0), torch.where(ok, n, 0)
    total = torch.div(l2 + n2 + S - 1, S, rounding_mode="floor")
    at = (upto - need)[:, None] + cols - kept[:, None] + forked[:, None]
    fresh = free[at.clamp(0, N)]
    mine = torch.where(have & ~(forked[:, None] & (cols == kept[:, None] - 1)), entry, fresh)
    mine = torch.where(cols < total[:, None], mine, -1)
    start = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), torch.cumsum(n2, 0)])
    t = torch.arange(T, device=dev)
    row = torch.searchsorted(start[1:], t, right=True)
    there = row < R
    r = row.clamp(max=R - 1)
    pos = torch.where(there, l2[r] + t - start[r], 0)
    slot = mine[r, torch.div(pos, S, rounding_mode="floor").clamp(max=M - 1)] * S + pos % S
    tok = torch.stack([torch.where(there, slot, -1), torch.where(there, r, -1), torch.where(there, pos + 1, 0), torch.zeros_like(pos)], 1)
    out = [mine, l2 + n2, start, tok, status]
    if parent is not None:
        copies = forked & ok
        dst = mine.gather(1, (kept - 1).clamp(0, M - 1)[:, None])[:, 0]
        out.append(torch.stack([torch.where(copies, last, -1), torch.where(copies, dst, -1), torch.where(copies, l % S, 0),
                                torch.zeros_like(l)], 1))
    return [x.to(torch.int32) for x in out]


def _plain_append(s):
    page = s["case"]["page"]
    slot = s["tok"][:, 0].long()
    first = (slot >= 0).int().argmax()
    t = torch.where(slot >= 0, torch.arange(len(slot), device=slot.device), first)      # idle tokens repeat one that is there
    at, off = torch.div(slot[t], page, rounding_mode="floor"), slot[t] % page
    for new, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        if s["fork"] is not None:
            src, dst, n = s["fork"][:, 0].long(), s["fork"][:, 1].long(), s["fork"][:, 2]
            lead = (src >= 0).int().argmax()
            f = torch.where(src >= 0, torch.arange(len(src), device=src.device), lead)
            keep = torch.arange(page, device=src.device)[None, None, :, None] < n[f][:, None, None, None]
            cache[dst[f]] = torch.where(keep, cache[src[f]], cache[dst[f]])
        cache[at, :, off] = new[t].to(cache.dtype)
    return [s["k_cache"], s["v_cache"]]


def _plain_attend(s):
    case, table, tok = s["case"], s["table"].long(), s["tok"].long()
    kv, dim, page = case["kv"], case["dim"], case["page"]
    rows, L = len(tok), table.shape[1] * page
    q = s["q"].view(rows, kv, -1, dim)
    ids = table[tok[:, 1].clamp(min=0)]
    there = (torch.arange(L, device=q.device) < tok[:, 2:3]) & (ids >= 0).repeat_interleave(page, 1)
    there = there[:, None, :, None]
    k, v = (c[ids.clamp(min=0)].transpose(1, 2).reshape(rows, kv, L, dim).float() for c in (s["k_cache"], s["v_cache"]))
    scores = torch.where(there.transpose(2, 3), q @ k.transpose(2, 3) / math.sqrt(dim), -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.where(scores == -math.inf, 0.0, torch.exp(scores - top))
    total = p.sum(-1, keepdim=True)
    o = p @ torch.where(there, v, 0.0)
    return [torch.where(total == 0, 0.0, o / total).view(rows, -1, dim)]


def _plain_beam(s):
    K, eos = s["case"]["beams"], 2
    logits = s["logits"].double()
    n, V = logits.shape
    norm = _log_sum(logits)
    score, live = s["score"].double()[:, None], s["live"][:, None] != 0
    cand = torch.where(torch.isfinite(norm), score + (logits - norm), -math.inf)
    ended = torch.where(torch.arange(V, device=logits.device) == eos, score, -math.inf)
    cand = torch.nan_to_num(torch.where(live, cand, ended), nan=-math.inf, posinf=math.inf, neginf=-math.inf).view(-1, K * V)
    best, at = torch.sort(cand, dim=1, descending=True, stable=True)
    best, at = best[:, :K].reshape(-1), at[:, :K].reshape(-1)
    there = best > -math.inf
    parent = torch.arange(n, device=at.device) // K * K + torch.div(at, V, rounding_mode="floor")
    token = torch.where(there, at % V, -1)
    alive = there & (live[parent, 0]) & (token != eos)
    return [token.int(), torch.where(there, parent, -1).int(), best.float(), alive.int()]


def _log_sum(x):
    top = x.amax(1, keepdim=True)
    return top + torch.log(torch.exp(x - top).sum(1, keepdim=True))


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "tables":
        return _plain_tables(state["case"], state["table"], state["lens"], state["new"], state["parent"])
    return {"append": _plain_append, "attend": _plain_attend, "beam": _plain_beam}[op](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "tables":
        R, M, T = case["rows"], case["max_pages"], case["tokens"]
        return {"bytes": 4.0 * (case["cached"] / case["page"] + R * M + 4 * T + 5 * R + (5 * R if case["beams"] else 0)), "flops": 0.0}
    if case["op"] == "append":
        e, row = _SIZE[case["type"]], case["kv"] * case["dim"]
        live = case["tokens"] - case["idle"]
        return {"bytes": 2.0 * live * row * (4 + e) + 16.0 * case["tokens"] + 2.0 * case["forks"] * row * e * case["page"], "flops": 0.0}
    if case["op"] == "attend":
        row = case["kv"] * case["dim"]
        seen = case["cached"] - case["gone"] * min(case["page"], case["cached"] / max(1, case["rows"] - case["idle"]))
        return {"bytes": 2.0 * seen * row * _SIZE[case["type"]] + 8.0 * case["rows"] * case["heads"] * case["dim"] + 16.0 * case["rows"] +
                4.0 * case["cached"] / case["page"], "flops": 4.0 * seen * case["heads"] * case["dim"]}
    n = case["requests"] * case["beams"]
    return {"bytes": 4.0 * (n - case["finished"]) * case["vocab"] + 24.0 * n, "flops": 4.0 * (n - case["finished"]) * case["vocab"]}


# ---- the definitions, in 64 bits ---------------------------------------------------------------------------------------
def _exact_tables(case, s):
    R, M, S, N, T = case["rows"], case["max_pages"], case["page"], case["pages"], case["tokens"]
    table, lens, new = (s[k].cpu().numpy().astype(np.int64) for k in ("table", "lens", "new"))
    parent = np.arange(R) if s["parent"] is None else s["parent"].cpu().numpy().astype(np.int64)
    out, length, status = np.full((R, M), -1, np.int64), np.zeros(R, np.int64), np.zeros(R, np.int64)
    fork = np.tile(np.array([-1, -1, 0, 0], np.int64), (R, 1))
    old, used, owner, room = [], set(), {}, 0
    for r in range(R):
        p = int(parent[r])
        l = int(lens[p]) if 0 <= p < R else 0
        ids = [int(x) for x in table[p, :-(-l // S)]] if 0 <= p < R and 0 <= l <= M * S else []
        bad = not -1 <= p < R or l < 0 or new[r] < 0 or l + new[r] > M * S or any(not -1 <= i < N for i in ids) or \
            (l % S > 0 and ids[-1] < 0)
        old.append((p, l, ids))
        if bad:
            status[r] = 2
            continue
        used.update(i for i in ids if i >= 0)
        owner.setdefault(p, r)
        room += int(new[r])
        if room > T:
            status[r] = 3
    free = [i for i in range(N) if i not in used]
    taken, refused = 0, 0
    start, tok = [0], []
    for r in range(R):
        p, l, ids = old[r]
        if status[r] == 0:
            copy = p >= 0 and l % S > 0 and owner[p] != r
            n = -(-(l + int(new[r])) // S) - len(ids) + copy
            if n > 0 and taken + refused + n > len(free):
                status[r] = 1
                refused += n
            else:
                mine = ids + free[taken:taken + n] if not copy else ids[:-1] + free[taken:taken + n]
                if copy:
                    fork[r] = (ids[-1], mine[len(ids) - 1], l % S, 0)
                taken += n
                out[r, :len(mine)] = mine
                length[r] = l + int(new[r])
                tok += [(mine[x // S] * S + x % S, r, x + 1, 0) for x in range(l, int(length[r]))]
        start.append(len(tok))
    tok += [(-1, -1, 0, 0)] * (T - len(tok))
    got = [out, length, np.array(start), np.array(tok, np.int64).reshape(T, 4), status] + ([fork] if s["parent"] is not None else [])
    return [torch.from_numpy(x.astype(np.int32)) for x in got]


def _exact_attend(s):
    tok, table, page = s["tok"].tolist(), s["table"].tolist(), s["case"]["page"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    kv = s["k_cache"].shape[1]
    for t, (_, row, n, _) in enumerate(tok):
        if n == 0:
            continue
        at = [i for i in range(-(-n // page)) if table[row][i] >= 0]
        pos = torch.tensor(at, device=q.device)[:, None] * page + torch.arange(page, device=q.device)
        ids, there = [table[row][i] for i in at], (pos < n).reshape(-1)
        k, v = (c[ids].double().transpose(0, 1).reshape(kv, -1, q.shape[2])[:, there] for c in (s["k_cache"], s["v_cache"]))
        if k.shape[1]:
            w = torch.softmax(torch.einsum("ghd,gnd->ghn", q[t].view(kv, -1, q.shape[2]), k) / math.sqrt(q.shape[2]), -1)
            out[t] = torch.einsum("ghn,gnd->ghd", w, v).reshape(q.shape[1:])
    return [out]


def _exact_append(s):
    caches = []
    for new, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        c = cache.double()
        if s["fork"] is not None:
            for src, dst, n, _ in s["fork"].tolist():
                if src >= 0:
                    c[dst, :, :n] = c[src, :, :n]
        slot = s["tok"][:, 0].long()
        live = torch.nonzero(slot >= 0)[:, 0]
        flat = c.transpose(1, 2).contiguous().view(-1, c.shape[1], c.shape[3])
        flat[slot[live]] = new[live].double()
        caches.append(flat.view(c.shape[0], c.shape[2], c.shape[1], c.shape[3]).transpose(1, 2).contiguous())
    return caches


def _exact_beam(case, s):
    K, V, eos = case["beams"], case["vocab"], 2
    score, live = s["score"].double().tolist(), s["live"].tolist()
    logp = torch.log_softmax(s["logits"].double(), 1)
    token, parent, best, alive = [], [], [], []
    for a in range(0, len(score), K):
        found = []
        for b in range(a, a + K):
            if live[b]:
                x = logp[b] + score[b]
                edge = torch.topk(x, min(K, V)).values[-1]
                at = torch.nonzero(x >= edge)[:, 0]
                found += [(-c, b, i) for c, i in zip(x[at].tolist(), at.tolist()) if c > -math.inf]
            elif score[b] > -math.inf:
                found.append((-score[b], b, eos))
        found = sorted(found)[:K]
        found += [(math.inf, -1, -1)] * (K - len(found))
        token += [i for _, _, i in found]
        parent += [b for _, b, _ in found]
        best += [-c for c, _, _ in found]
        alive += [int(b >= 0 and live[b] and i != eos) for _, b, i in found]
    return [torch.tensor(token, dtype=torch.int32), torch.tensor(parent, dtype=torch.int32), torch.tensor(best, dtype=torch.float64),
            torch.tensor(alive, dtype=torch.int32)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        return _exact_tables(case, s)
    if case["op"] == "append":
        return _exact_append(s)
    return _exact_attend(s) if case["op"] == "attend" else _exact_beam(case, s)
