"""The decoding operators against their definitions in 64 bits (or in whole numbers), at the sizes and masks where they can go wrong.

Tolerances.  A score is a sum of D products in fp32, scaled: its error is at most (D / lanes + log2 lanes + 3) 2^-24 sum |q k| / sqrt(D), and the
probability's relative error is that error plus what 2^x is off by (2^-22) plus the roundings of the argument; the sum over the values adds
its own roundings, which a sum in groups keeps near (log2 n + few) 2^-24.  With |score terms| below 8 sqrt(D) / sqrt(D) this is below
24 * 2^-24 * 8 + 8 * 2^-24 = 200 * 2^-24 of sum p |v|.  Outputs are held to ATTEND_TOL = 2^-16 of sum p |v| + 2^-24 of the largest.
A cache of type t rounds a value by at most eps(t) / 2 of it; both sides of the attention read the rounded values.
"""
import numpy as np
import pytest
import torch

from reef_b200 import capi, decode

pytestmark = pytest.mark.gpu

ATTEND_TOL = 2.0 ** -16
F, I = torch.float32, torch.int32


def dev(a, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(a)) if not isinstance(a, torch.Tensor) else a
    return t.to("cuda", dtype)


# ---- page tables -----------------------------------------------------------------------------------------------------------
def tables_by_hand(table, lens, new, parent, pages, S, tokens):
    R, M = table.shape
    out, length, status, fork = np.full((R, M), -1), np.zeros(R, int), np.zeros(R, int), np.tile([-1, -1, 0, 0], (R, 1))
    rows, used, owner, room = [], set(), {}, 0
    for r in range(R):
        q = r if parent is None else int(parent[r])
        named = -1 <= q < R
        l = int(lens[q]) if named and q >= 0 else 0
        good = named and 0 <= l and 0 <= new[r] and l + int(new[r]) <= M * S
        ids = [int(x) for x in table[q, :-(-l // S)]] if good and q >= 0 else []
        good = good and all(-1 <= i < pages for i in ids) and not (l % S and ids[-1] < 0)
        rows.append((q, l, ids))
        if not good:
            status[r] = 2
            continue
        used.update(i for i in ids if i >= 0)
        owner.setdefault(q, r)
        room += int(new[r])
        status[r] = 3 if room > tokens else 0
    free = [i for i in range(pages) if i not in used]
    taken = asked = 0
    start, tok = [0], []
    for r in range(R):
        q, l, ids = rows[r]
        if status[r] == 0:
            copy = q >= 0 and l % S != 0 and owner[q] != r
            n = -(-(l + int(new[r])) // S) - len(ids) + copy
            asked += n
            if n and asked > len(free):
                status[r] = 1
            else:
                mine = (ids[:-1] if copy else ids) + free[taken:taken + n]
                taken += n
                if copy:
                    fork[r] = ids[-1], mine[len(ids) - 1], l % S, 0
                out[r, :len(mine)] = mine
                length[r] = l + int(new[r])
                tok += [(mine[x // S] * S + x % S, r, x + 1, 0) for x in range(l, length[r])]
        start.append(len(tok))
    tok += [(-1, -1, 0, 0)] * (tokens - len(tok))
    return [out, length, np.array(start), np.array(tok).reshape(tokens, 4), status] + ([] if parent is None else [fork])


def check_tables(table, lens, new, parent, pages, S, tokens):
    want = tables_by_hand(table, lens, new, parent, pages, S, tokens)
    args = [dev(table, I), dev(lens, I), dev(new, I)]
    got = decode.page_tables(*args, pages=pages, page_size=S, tokens=tokens, parent=None if parent is None else dev(parent, I))
    for name, a, b in zip(decode.PageState._fields, got, want):
        assert np.array_equal(a.cpu().numpy(), b), name
    assert np.array_equal(args[0].cpu().numpy(), table)
    return got


def random_rows(rng, R, M, S, pages, most):
    lens = rng.integers(0, most + 1, R)
    lens[rng.random(R) < 0.2] = 0
    table, ids, at = rng.integers(-5, pages + 5, (R, M)), rng.permutation(pages), 0     # (anything behind the last page)
    for r in range(R):
        n = -(-int(lens[r]) // S)
        table[r, :n] = ids[at:at + n]
        at += n
    return table, lens


@pytest.mark.parametrize("R,M,S,pages,tokens", [(1, 1, 1, 1, 1), (1, 4, 16, 5, 1), (16, 64, 16, 1024, 16), (37, 9, 24, 500, 100), (256, 33, 8, 9000, 3000),
                                                (1024, 5, 3, 5200, 1500), (3, 1000, 128, 4000, 70000), (65, 130, 1, 8192, 300), (33, 7, 1024, 300, 2000)])
@pytest.mark.parametrize("forks", [False, True])
def test_page_tables(R, M, S, pages, tokens, forks):
    rng = np.random.default_rng([R, M, S, forks])
    most = min(M * S, pages * S // R)
    for kind in range(3):
        table, lens = random_rows(rng, R, M, S, pages, most * 3 // 4)
        new = rng.integers(0, 3, R) if kind < 2 else rng.integers(0, max(2, M * S // 3), R)
        parent = None
        if forks:
            parent = np.arange(R) // 4 * 4 + rng.integers(0, 4, R)
            parent = np.where(rng.random(R) < 0.15, -1, np.minimum(parent, R - 1))
            if kind == 1:
                parent[:] = R // 2                       # one row takes all
        check_tables(table, lens, new, parent, pages, S, tokens)


@pytest.mark.parametrize("pages", [230000, 1 << 19])
def test_page_tables_of_more_pages_than_a_window_marks(pages):
    rng = np.random.default_rng(pages)
    R, M, S = 40, 8200, 2
    table, lens = random_rows(rng, R, M, S, pages, 10000)
    for parent in (None, np.arange(R) // 2 * 2):
        check_tables(table, lens, rng.integers(0, 40, R), parent, pages, S, 900)


@pytest.mark.parametrize("bad", ["len", "len_long", "new", "new_long", "id", "id_low", "parent", "parent_low", "last_gone"])
def test_page_tables_refuse_single_rows(bad):
    rng = np.random.default_rng(3)
    table, lens = random_rows(rng, 8, 6, 16, 100, 60)
    lens[:] = np.maximum(lens, 17)
    for r in range(8):
        table[r, :4] = np.arange(4) + 10 * r
    new, parent = np.ones(8, int), np.arange(8)
    big = 2 ** 31 - 1
    if bad == "len": lens[3] = -1
    if bad == "len_long": lens[3] = big
    if bad == "new": new[3] = -1
    if bad == "new_long": new[3] = big
    if bad == "id": table[3, 0] = 100
    if bad == "id_low": table[3, 1] = -2
    if bad == "parent": parent[3] = 8
    if bad == "parent_low": parent[3] = -2
    if bad == "last_gone": lens[3], table[3, 1] = 20, -1
    got = check_tables(table, lens, new, parent, 100, 16, 64)
    assert got.status[3] == 2 and got.lens[3] == 0 and int((got.status != 0).sum()) == 1


def test_page_tables_that_run_out():
    table, lens, new = np.full((6, 4), -1), np.zeros(6, int), np.array([16, 33, 0, 16, 1, 0])
    got = check_tables(table, lens, new, None, 3, 16, 100)          # the second row wants three of the two that are left
    assert got.status.tolist() == [0, 1, 0, 1, 1, 0]
    got = check_tables(table, lens, np.array([5, 6, 0, 1, 1, 0]), None, 30, 16, 10)
    assert got.status.tolist() == [0, 3, 3, 3, 3, 3]                # from there on, whatever they add
    check_tables(table, lens, np.full(6, 64), None, 30, 16, 10)
    check_tables(np.zeros((6, 1 << 20), int) - 1, lens, np.full(6, 1 << 29), None, 30, 1024 // 2, 100)


def test_page_tables_keep_pages_that_were_given_up():
    table = np.array([[-1, -1, 7, 3, 9], [5, -1, 2, 0, 0]])
    got = check_tables(table, np.array([60, 40]), np.array([5, 8]), None, 20, 16, 32)
    assert got.table[0].tolist() == [-1, -1, 7, 3, 0] and got.status.tolist() == [0, 0]


def test_page_tables_over_many_steps():
    """A pool under beams that end and begin: no page belongs to two rows unless it is full, and every row's tokens stay its own."""
    rng = np.random.default_rng(11)
    R, M, S, pages = 24, 6, 4, 90
    state = decode.page_state(R, M, 3 * R, fork=True)
    other = decode.page_state(R, M, 3 * R, fork=True)
    book, cache = [[] for _ in range(R)], np.full(pages * S, -1)
    for step in range(60):
        new, parent = rng.integers(0, 4, R), np.arange(R) // 4 * 4 + rng.integers(0, 4, R)
        parent[rng.random(R) < 0.2] = -1
        state, other = decode.page_tables(state.table, state.lens, dev(new, I), pages=pages, page_size=S, tokens=3 * R, parent=dev(parent, I), out=other), state
        table, lens, tok, status, fork = (x.cpu().numpy() for x in (state.table, state.lens, state.tok, state.status, state.fork))
        for src, dst, n, _ in fork:
            if src >= 0:
                cache[dst * S:dst * S + n] = cache[src * S:src * S + n]
        book = [([] if status[r] or parent[r] < 0 else list(book[parent[r]])) for r in range(R)]
        for i, (slot, r, length, _) in enumerate(tok):
            if r >= 0:
                assert len(book[r]) == length - 1
                book[r].append(1000 * step + i)
                cache[slot] = 1000 * step + i
        owners = {}
        for r in range(R):
            assert lens[r] == len(book[r])
            assert [cache[table[r, x // S] * S + x % S] for x in range(lens[r])] == book[r]
            if lens[r] % S:
                page = table[r, lens[r] // S]
                assert page not in owners
                owners[page] = r


# ---- append ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", [F, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,kv,D,S,pages,forks,stride", [(1, 1, 64, 1, 1, 0, 0), (1, 12, 64, 16, 40, 3, 0), (77, 3, 128, 24, 40, 9, 4), (1000, 2, 256, 16, 200, 0, 12),
                                                         (5, 1, 64, 1024, 4, 1, 0), (130, 16, 64, 8, 60, 20, 1024)])
def test_append(type, T, kv, D, S, pages, forks, stride):
    rng = np.random.default_rng([T, kv, D])
    ids = rng.permutation(pages)
    src, dst, rest = ids[:forks], ids[forks:2 * forks], ids[2 * forks:]
    slots = rng.permutation((rest[:, None] * S + np.arange(S)).ravel())[:T]
    keep = rng.integers(0, S + 1, forks)
    tok = np.full((T, 4), 9)
    tok[:, 0] = slots
    if T > 4:
        tok[[1, 3], 0] = -1, pages * S               # outside the cache: passed over
    fork = np.concatenate([np.stack([src, dst, keep, 0 * src], 1), [[-1, -1, 0, 0], [pages, 0, S, 0], [0, -7, S, 0], [0, 0, -3, 0]]])
    wide = [torch.randn(T, kv * D + stride, device="cuda") for _ in range(2)]
    k, v = (x[:, :kv * D].unflatten(1, (kv, D)) for x in wide)
    caches = [torch.randn(pages, kv, S, D, device="cuda").to(type) for _ in range(2)]
    want = [c.clone() for c in caches]
    for c, x in zip(want, (k, v)):
        for a, b, n, _ in fork:
            if 0 <= a < pages and 0 <= b < pages and a != b:
                c[b, :, :n] = c[a, :, :n]
        for t in range(T):
            if 0 <= tok[t, 0] < pages * S:
                c[tok[t, 0] // S, :, tok[t, 0] % S] = x[t].to(type)
    for _ in range(2):                               # a second run gives the same
        decode.paged_append(k, v, dev(tok, I), *caches, fork=dev(fork, I))
        assert all(torch.equal(a, b) for a, b in zip(caches, want))


@pytest.mark.parametrize("type", [F, torch.bfloat16])
def test_append_copies_pages_of_several_pieces(type):
    test_append(type, 20, 3, 256, 100, 40, 7, 0)
    test_append(type, 2, 1, 128, 128, 9, 4, 0)


# ---- attention ---------------------------------------------------------------------------------------------------------------
def attend_by_hand(q, kc, vc, table, tok):
    """(result, sum p |v|) in 64 bits"""
    T, H, D = q.shape
    pages, kv, S, _ = kc.shape
    out, size = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    q, kc, vc = q.double().cpu(), kc.cpu(), vc.cpu()
    for t, (_, row, n, _) in enumerate(tok.tolist()):
        if not 0 <= row < len(table) or n <= 0:
            continue
        n = min(n, table.shape[1] * S)
        pos = [x for x in range(n) if 0 <= table[row, x // S] < pages]
        if not pos:
            continue
        at, off = torch.tensor([int(table[row, x // S]) for x in pos]), torch.tensor([x % S for x in pos])
        k, v = (c[at, :, off].double().transpose(0, 1) for c in (kc, vc))          # [kv][n][D]
        s = torch.einsum("ghd,gnd->ghn", q[t].view(kv, -1, D), k) / D ** 0.5
        top = s.amax(-1, keepdim=True)
        p = torch.where(s == -torch.inf, 0.0, torch.exp(s - top))
        total = p.sum(-1, keepdim=True)
        p = torch.where(total == 0, 0.0, p / total)
        out[t], size[t] = (torch.einsum("ghn,gnd->ghd", p, x).reshape(H, D) for x in (v, v.abs()))
    return out, size


def attend_inputs(rng, lens, H, kv, D, S, M, type, spread=1.0):
    """Rows of these lengths, pages in no order, more pages than rows need; NaN in every slot that no row has."""
    R = len(lens)
    need = [-(-max(0, min(int(l), M * S)) // S) for l in lens]
    pages = sum(need) + 3
    ids, at = rng.permutation(pages), 0
    table = np.full((R, M), -1)
    q = dev(rng.standard_normal((R, H, D)) * spread, F)
    kc, vc = (torch.full((pages, kv, S, D), torch.nan, device="cuda", dtype=type) for _ in range(2))
    for r in range(R):
        table[r, :need[r]] = ids[at:at + need[r]]
        at += need[r]
        n = max(0, min(int(lens[r]), M * S))
        for c in (kc, vc):
            full = torch.randn(need[r] * S, kv, D, device="cuda")
            full[n:] = torch.nan
            if need[r]:
                c[torch.as_tensor(table[r, :need[r]]).cuda()] = full.view(need[r], S, kv, D).transpose(1, 2).to(type)
    tok = np.zeros((R, 4), int)
    tok[:, 0], tok[:, 1], tok[:, 2] = 12345, np.arange(R), lens
    return q, kc, vc, table, tok


def check_attention(q, kc, vc, table, tok, out=None):
    want, size = attend_by_hand(q, kc, vc, table, tok)
    size = size.nan_to_num(0.0, posinf=0.0)            # (where the result is not finite either)
    got = decode.paged_attention(q, kc, vc, dev(table, I), dev(tok, I), out=out).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine].nan_to_num(5), want[~fine].nan_to_num(5))
    over = ((got - want).abs() - ATTEND_TOL * size - 2.0 ** -24 * size.amax())[fine]
    assert over.numel() == 0 or over.max() <= 0, float(over.max())
    return got


TYPES = [F, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,kv", [(1, 1), (4, 2), (6, 2), (12, 12), (5, 1), (14, 2), (8, 1), (16, 1), (24, 1), (40, 2), (4, 1), (12, 2), (9, 1)])
@pytest.mark.parametrize("M,S,lens", [(4, 16, [1, 0, 64, 17, 33]), (60, 16, [959, 1, 960, 0, 300]), (700, 3, [2100, 5, 1999])])
def test_attention(type, D, H, kv, M, S, lens):
    check_attention(*attend_inputs(np.random.default_rng([D, H, M]), lens, H, kv, D, S, M, type))


@pytest.mark.parametrize("S", [1, 2, 7, 16, 100, 1024])
@pytest.mark.parametrize("type", TYPES)
def test_attention_page_sizes(S, type):
    M = -(-1300 // S)
    check_attention(*attend_inputs(np.random.default_rng(S), [1300 // S * S, 1, S, min(S + 1, M * S), 777], 6, 3, 64, S, M, type))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("D,H,kv", [(64, 16, 16), (128, 24, 8), (256, 16, 8), (64, 40, 8)])
def test_attention_of_many_short_rows(type, D, H, kv):
    """Passes enough for all warps: one, two or four warps to a pass, rows without keys and of one key among them."""
    for R, M in ((90, 2), (200, 3), (130, 9)):
        rng = np.random.default_rng([R, D, H])
        lens = rng.integers(-1, M * 16 + 3, R)
        lens[rng.random(R) < 0.2] = 1
        check_attention(*attend_inputs(rng, lens, H, kv, D, 16, M, type))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,kv", [(2, 2), (8, 1)])
def test_attention_of_one_long_row(type, H, kv):
    """A row that many blocks share, alone and between short ones."""
    rng = np.random.default_rng(4)
    check_attention(*attend_inputs(rng, [40000], H, kv, 64, 64, 700, type))
    check_attention(*attend_inputs(rng, [3, 0, 30001, 1, 0, 17], H, kv, 128, 64, 700, type))


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,kv", [(3, 3), (16, 2)])
@pytest.mark.parametrize("M", [8, 200])
def test_attention_of_bad_pages_and_rows(type, H, kv, M):
    """Ids outside the cache hold no keys; rows, lengths out of range have none, or as many as a table can name."""
    rng = np.random.default_rng(5)
    q, kc, vc, table, tok = attend_inputs(rng, [100, 128, 16, 70, 128, 128, 5, 128], H, kv, 64, 16, M, type)
    table[0, 0], table[0, 3], table[1, :], table[2, 0], table[3, 4] = -1, len(kc), -1, 2 ** 31 - 1, -2 ** 31
    tok[4, 1], tok[5, 1], tok[6, 2], tok[7, 2] = 8, -1, -5, 2 ** 31 - 1
    got = check_attention(q, kc, vc, table, tok)
    assert not got[[1, 2, 4, 5, 6]].any() and got[[0, 3, 7]].any()


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,kv", [(2, 2), (8, 1)])
@pytest.mark.parametrize("M", [8, 100])
@pytest.mark.parametrize("where,value", [("k", np.inf), ("k", -np.inf), ("k", np.nan), ("v", np.inf), ("v", np.nan), ("k_all", -np.inf), ("q", np.inf), ("q", np.nan),
                                         ("q", 1e30), ("k", 6e4), ("v", 6e4), ("q", 3e38), ("q", 1e-30)])
def test_attention_of_extreme_values(type, H, kv, M, where, value):
    """One dimension of one key, value or query; fp32 gives the same: -infinity is a probability of zero, a row of them none."""
    q, kc, vc, table, tok = attend_inputs(np.random.default_rng(6), [100, 120, 1], H, kv, 64, 16, M, type)
    if where[0] in "kv":
        page, slot = int(table[0, 2]), 5
        (kc if where[0] == "k" else vc)[page, :, slot, 9] = value
        q[0, :, 9] = q[0, :, 9].abs() + 0.5
        if where == "k_all":
            for i in range(7):
                kc[int(table[0, i]), :, :, 9] = value
    else:
        q[0, 0, 9] = value
    if value == 3e38:
        return          # sums of products beyond fp32: no result to compare with
    check_attention(q, kc, vc, table, tok)


def test_attention_of_large_scores():
    """Differences of scores of a few hundred: one key has all the weight."""
    for type in TYPES:
        q, kc, vc, table, tok = attend_inputs(np.random.default_rng(8), [500, 64, 33], 4, 2, 64, 16, 40, type, spread=100.0)
        want, size = attend_by_hand(q, kc, vc, table, tok)
        got = decode.paged_attention(q, kc, vc, dev(table, I), dev(tok, I)).double().cpu()
        # terms of a score go up to 100 * 4 * 4 / 8: the error of a score, 24 * 2^-24 * 64 * 100 / 8, is the relative error of its weight
        assert ((got - want).abs() <= 24 * 2.0 ** -24 * 800 * 2 * size + 1e-7).all()


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,kv", [(6, 2), (16, 2)])
def test_attention_of_several_tokens_of_a_row(type, H, kv):
    """A chunk of a prompt: every token sees those up to itself; queries are a slice of a fused projection; idle tokens behind it."""
    rng = np.random.default_rng(9)
    q, kc, vc, table, _ = attend_inputs(rng, [300, 120], H, kv, 64, 16, 20, type)
    T = 40
    wide = torch.randn(T, (H + 2 * kv) * 64, device="cuda")
    tok = np.zeros((T, 4), int)
    tok[:25, 1], tok[:25, 2] = 0, np.arange(276, 301)
    tok[25:35, 1], tok[25:35, 2] = 1, np.arange(1, 11)
    tok[35:, :2] = -1
    out = torch.full((T, H, 64), 7.0, device="cuda")
    got = check_attention(wide[:, :H * 64].unflatten(1, (H, 64)), kc, vc, table, tok, out=out)
    assert not got[35:].any()


@pytest.mark.parametrize("type,pages", [(torch.bfloat16, 2200), (F, 1100)])
def test_offsets_beyond_32_bits(type, pages):
    """Caches of more than 2^32 values and 2^33 bytes: the last page is written, copied and read."""
    kv, S, D = 16, 1024, 128
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB of device memory")
    kc, vc = (torch.zeros(pages, kv, S, D, device="cuda", dtype=type) for _ in range(2))
    assert kc.numel() * kc.element_size() > 1 << 33
    k, v = torch.randn(2, kv, D, device="cuda"), torch.randn(2, kv, D, device="cuda")
    last = pages - 1
    tok = np.array([[last * S + 1023, 0, 1024, 0], [last * S, 0, 1, 0]])
    decode.paged_append(k, v, dev(tok, I), kc, vc)
    assert torch.equal(kc[last, :, 1023], k[0].to(type)) and torch.equal(vc[last, :, 0], v[1].to(type))
    decode.paged_append(k, v, dev(np.full((2, 4), -1), I), kc, vc, fork=dev([[last, last - 1, 1024, 0]], I))
    assert torch.equal(kc[last], kc[last - 1]) and torch.equal(vc[last], vc[last - 1])
    for H in (16, 64):
        q = torch.randn(1, H, D, device="cuda")
        got = decode.paged_attention(q, kc, vc, dev([[last]], I), dev([[0, 0, 1024, 0]], I))
        ks, vs = kc[last].double(), vc[last].double()
        p = torch.softmax(torch.einsum("ghd,gnd->ghn", q[0].double().view(kv, -1, D), ks) / D ** 0.5, -1)
        want = torch.einsum("ghn,gnd->ghd", p, vs).reshape(1, H, D)
        assert (got - want).abs().max() <= ATTEND_TOL * torch.einsum("ghn,gnd->ghd", p, vs.abs()).max()


# ---- beam selection ------------------------------------------------------------------------------------------------------------
def select_by_hand(logits, score, live, K, eos, start=None):
    logits, score, live = logits.double().cpu(), score.double().cpu(), live.cpu()
    out = []
    for a in range(0, len(score), K):
        found = []
        for b in range(a, a + K):
            s = float(score[b])
            if live[b] == 0:
                if np.isfinite(s):
                    found.append((-s, b, eos, 0))
                continue
            row = b
            if start is not None:
                if start[b + 1] <= start[b]:
                    continue
                row = int(start[b + 1]) - 1
            top = logits[row].max()
            norm = torch.log(torch.exp(logits[row] - top).sum())
            if not np.isfinite(float(norm + top) + s):
                continue
            c = s + (logits[row] - top - norm)          # (top + norm would lose norm at the type's lowest value)
            order = torch.sort(logits[row], descending=True, stable=True).indices[:K]
            found += [(-float(c[i]), b, int(i), int(i != eos)) for i in order if float(c[i]) > -np.inf]
        found = sorted(found)[:K]
        out += [(i, b, -c, l) for c, b, i, l in found] + [(-1, -1, -np.inf, 0)] * (K - len(found))
    return [np.array(x) for x in zip(*out)]


def check_beams(logits, score, live, K, eos, start=None, out=None):
    want = select_by_hand(logits, score, live, K, eos, start)
    got = [x.cpu().numpy() for x in decode.beam_select(logits, score, live, beams=K, eos=eos, start=None if start is None else dev(start, I), out=out)]
    for name, i in (("token", 0), ("parent", 1), ("live", 3)):
        assert np.array_equal(got[i], want[i]), name
    there = np.isfinite(want[2])
    assert np.array_equal(got[2][~there], want[2][~there])
    # the sum of exponentials is off by 2^-21 at most (exponents up to 16 in units of 2^-24, 2^-22 for 2^x), its logarithm by as much; one rounding
    assert np.all(np.abs(got[2][there] - want[2][there]) <= 2.0 ** -21 + 2.0 ** -24 * np.abs(want[2][there]))


@pytest.mark.parametrize("Q,K,V", [(1, 1, 1), (1, 4, 3), (1, 4, 30522), (3, 16, 4097), (7, 5, 4093), (40, 2, 1001), (2, 8, 100003), (5, 3, 8), (1, 16, 70001), (300, 1, 50)])
def test_beam_select(Q, K, V):
    g = torch.Generator("cuda").manual_seed(Q * V)
    for kind in range(3):
        logits = 3 * torch.randn(Q * K, V, device="cuda", generator=g)
        if kind:
            logits = logits.bfloat16().float()          # many equal ones
        score = -10 + torch.randn(Q * K, device="cuda", generator=g)
        live = torch.ones(Q * K, device="cuda", dtype=I)
        if kind == 2:
            live = (torch.rand(Q * K, device="cuda", generator=g) < 0.7).int()
            score[torch.rand(Q * K, device="cuda", generator=g) < 0.2] = -torch.inf
        check_beams(logits, score, live, K, V // 2)


@pytest.mark.parametrize("V", [600, 30000])
@pytest.mark.parametrize("K", [1, 4, 16])
def test_beam_select_of_equal_values(K, V):
    """More equal candidates than there is room to rank them side by side: the lowest come first."""
    for logits in (torch.zeros(2 * K, V, device="cuda"), (torch.arange(2 * K * V, device="cuda") % 2).float().view(2 * K, V)):
        live = torch.ones(2 * K, device="cuda", dtype=I)
        check_beams(logits, torch.full((2 * K,), -1.0, device="cuda"), live, K, 0)
        score = torch.full((2 * K,), -torch.inf, device="cuda")
        score[::K] = 0                                  # a request's first step: one beam
        check_beams(logits, score, live, K, 1)


@pytest.mark.parametrize("Q,K", [(75, 8), (40, 16)])
def test_beam_select_of_words_in_few_places(Q, K):
    """Words that stand where few threads look, more than are ranked side by side; words in order."""
    V, R = 20000, Q * K
    w = torch.arange(V, device="cuda")
    logits = torch.where(w // 4 % 16 == 3, torch.randn(R, V, device="cuda"), -torch.inf)
    logits[K:2 * K, w // 4 % 16 == 3] = 5.0             # all of them equal
    logits[2 * K:3 * K] = torch.where(w // 4 % 16 == 3, 5.0, torch.finfo(F).min)
    logits[3 * K:4 * K] = torch.where(w // 4 % 16 < 7, w % 5000 / 1000, -torch.inf)
    logits[4 * K:5 * K] = w / 1000
    logits[5 * K:6 * K] = -w / 1000
    logits[6 * K:7 * K] = torch.where(w > V - 30, 1.0, torch.where(w % 128 < 64, 2.0, 0.0))
    logits[7 * K:8 * K] = torch.where((w // 4 % 32 == 9) | (w % 1999 == 0), 2.0 + w % 3, -1.0)
    check_beams(logits, -torch.rand(R, device="cuda"), torch.ones(R, device="cuda", dtype=I), K, 2)


@pytest.mark.parametrize("V", [5, 10001])
def test_beam_select_of_masked_words_and_rows(V):
    K = 4
    logits = torch.randn(6 * K, V, device="cuda")
    low = torch.finfo(F).min
    logits[0] = -torch.inf
    logits[1, 3] = torch.nan
    logits[2, 1] = torch.inf
    logits[4:8] = -torch.inf
    logits[4, 2] = 0.0                                  # a single word, in one row
    logits[8:12] = low                                  # a row of the type's lowest value, another of it but for one word
    logits[9, 4] = 1.0
    logits[12:16, : V - 2] = -torch.inf
    logits[16:20] = torch.nan
    score = -torch.rand(6 * K, device="cuda")
    score[20] = torch.nan
    score[21] = torch.inf
    check_beams(logits, score, torch.ones(6 * K, device="cuda", dtype=I), K, 2)
    check_beams(logits, score, torch.zeros(6 * K, device="cuda", dtype=I), K, 2)


def test_beam_select_of_the_last_token_of_each_row():
    K, V = 3, 777
    start = np.array([0, 1, 1, 5, 9, 9, 9, 10, 11, 14, 14, 14, 14])
    logits = torch.randn(16, V, device="cuda")
    live = torch.ones(12, device="cuda", dtype=I)
    live[4] = 0
    check_beams(logits, -torch.rand(12, device="cuda"), live, K, 5, start)
    start[5:] = 2 ** 31 - 1                             # rows out of range have no candidates
    got = decode.beam_select(logits, torch.zeros(12, device="cuda"), torch.ones(12, device="cuda", dtype=I), beams=K, eos=5, start=dev(start, I))
    assert got[0][6:].tolist() == [-1] * 6 and got[0][:3].min() >= 0


def test_scores_that_32_bits_cannot_tell_apart():
    """A beam far down: sums of 32 bits would make equal what the logits order."""
    K, V = 4, 2000
    logits = torch.zeros(K, V, device="cuda")
    logits += torch.randperm(K * V, device="cuda").view(K, V) * 2.0 ** -22
    score = torch.full((K,), -torch.inf, device="cuda")
    score[2] = -5000.0
    check_beams(logits, score, torch.ones(K, device="cuda", dtype=I), K, 0)


# ---- refusals, streams, graphs, threads ------------------------------------------------------------------------------------------
def small(T=4, H=4, kv=2, D=64, S=16, M=40, type=torch.bfloat16):
    q, kc, vc, table, tok = attend_inputs(np.random.default_rng(1), [500] * T, H, kv, D, S, M, type)
    return q, kc, vc, dev(table, I), dev(tok, I)


def test_refusals():
    q, kc, vc, table, tok = small()
    no = lambda *a, **k: pytest.raises(capi.ReefError, decode.paged_attention, *a, **k)     # noqa: E731
    no(q.half(), kc, vc, table, tok)
    no(q, kc.float(), vc, table, tok)
    no(q, kc, vc[:-1], table, tok)
    no(q, kc, vc, table.long(), tok)
    no(q, kc, vc, table[:, ::2], tok)
    no(q, kc, vc, table, tok[:-1])
    no(q[:, :3], kc, vc, table, tok)
    no(q[:0], kc, vc, table, tok[:0])
    no(q.transpose(1, 2).contiguous().transpose(1, 2), kc, vc, table, tok)
    no(q, kc, vc, table, tok, out=q)
    no(q, kc, vc, table, tok, out=torch.empty(4, 4, 128, device="cuda")[..., :64])
    no(q, kc[..., :32].contiguous(), vc[..., :32].contiguous(), table, tok)
    no(torch.empty(4 * 4 * 64 + 1, device="cuda")[1:].view(4, 4, 64), kc, vc, table, tok)
    k = torch.zeros(4, 2, 64, device="cuda")
    no = lambda *a, **k: pytest.raises(capi.ReefError, decode.paged_append, *a, **k)        # noqa: E731
    no(k, k, tok, kc, kc)
    no(k.half(), k, tok, kc, vc)
    no(k[:3], k, tok, kc, vc)
    no(k, k, tok, kc.transpose(1, 2), vc.transpose(1, 2))
    no(k, k, tok, kc, vc, fork=tok[:, :3])
    f = kc.float().contiguous()
    no(f.view(-1)[:512].view(4, 2, 64), k, tok, f, vc.float())
    lens = torch.zeros(4, dtype=I, device="cuda")
    state = decode.page_state(4, 40, 8)
    no = lambda *a, **k: pytest.raises(capi.ReefError, decode.page_tables, *a, pages=100, page_size=16, tokens=8, **k)      # noqa: E731
    no(table, lens[:3], lens)
    no(table, lens, lens.long())
    no(table, lens, lens, parent=lens[:2])
    no(state.table, state.lens, lens, out=state)
    no(table, lens, lens, out=decode.page_state(4, 40, 9))
    no(table, lens, lens, parent=lens, out=state)
    logits, score = torch.zeros(4, 100, device="cuda"), torch.zeros(4, device="cuda")
    no = lambda *a, **k: pytest.raises(capi.ReefError, decode.beam_select, *a, beams=2, eos=1, **k)     # noqa: E731
    no(logits.half(), score, lens)
    no(logits[:, ::2], score, lens)
    no(logits[:3], score, lens)
    no(logits, score, lens, start=lens)
    no(logits, score, lens, out=(lens, torch.empty_like(lens), torch.empty_like(score), torch.empty_like(lens)))
    no(logits, score, lens.cpu())
    assert capi.device_error() == 0


def test_streams_graphs_and_threads():
    """The same calls on another stream, captured and replayed with new inputs, two graphs side by side, from several threads."""
    import threading
    q, kc, vc, table, tok = small(T=6, M=300)
    want = decode.paged_attention(q, kc, vc, table, tok)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = decode.paged_attention(q, kc, vc, table, tok)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs, qs = [], [], [q.clone(), q.clone()]
    for x in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(decode.paged_attention(x, kc, vc, table, tok))
        graphs.append(g)
    wants = []
    for i, x in enumerate(qs):
        x.copy_(torch.randn_like(x))
        wants.append(decode.paged_attention(x, kc, vc, table, tok))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, wants))
    logits, score, live = torch.randn(8, 5000, device="cuda"), torch.zeros(8, device="cuda"), torch.ones(8, device="cuda", dtype=I)
    first = decode.beam_select(logits, score, live, beams=4, eos=0)
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for n in range(30):
                a = decode.paged_attention(q, kc, vc, table, tok)
                b = decode.beam_select(logits, score, live, beams=4, eos=0)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(a, want) or not all(torch.equal(x, y) for x, y in zip(b, first)):
                    bad.append(n)
    threads = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad and capi.device_error() == 0


def test_nothing_depends_on_the_run():
    """Bit for bit the same, whatever ran before."""
    for T, M in ((1, 1000), (37, 90), (3, 8)):
        q, kc, vc, table, tok = attend_inputs(np.random.default_rng(2), [M * 16 - 5] * T, 16, 2, 128, 16, M, torch.bfloat16)
        table, tok = dev(table, I), dev(tok, I)
        first = decode.paged_attention(q, kc, vc, table, tok)
        for _ in range(10):
            assert torch.equal(decode.paged_attention(q, kc, vc, table, tok), first)
