"""The decoding operators at sizes and values where one form of a kernel ends and another begins, against their definitions."""
import numpy as np
import pytest
import torch

from reef_b200 import capi, decode
from reef_b200.resources import decoding
from test_gpu_decode import ATTEND_TOL, F, I, attend_by_hand, attend_inputs, check_attention, dev

pytestmark = pytest.mark.gpu
TYPES = [F, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("T", [3583, 8192])
def test_many_tokens_over_a_long_table(T):
    """Steps of all rows' whole tables below and beyond 0x70000000, in the form that takes a row's keys to one block."""
    R, H, D, S, M = 4, 32, 128, 64, 2048
    assert len(decoding.paged_attention(T, R, H, H, D, S, M, 20, "bfloat16")) == 1
    q, kc, vc, table, _ = attend_inputs(np.random.default_rng(T), [150, 64, 1, 0], H, H, D, S, M, torch.bfloat16)
    q = torch.randn(T, H, D, device="cuda")
    tok = np.zeros((T, 4), int)
    tok[:, 1] = np.arange(T) % R
    tok[:, 2] = np.array([150, 64, 1, 0])[tok[:, 1]]
    got = decode.paged_attention(q, kc, vc, dev(table, I), dev(tok, I)).double().cpu()
    some = np.r_[0:8, T // 2:T // 2 + 8, T - 8:T]
    want, size = attend_by_hand(q[some], kc, vc, table, tok[some])
    assert ((got[some] - want).abs() <= ATTEND_TOL * size + 2.0 ** -24 * size.amax()).all()
    assert not got[tok[:, 2] == 0].any() and capi.device_error() == 0


# ---- beam selection: candidates that are equal in 64 bits ------------------------------------------------------------------------
def check_order(logits, score, live, K, eos):
    """Sorted by the value in 64 bits, then the beam, the logit as it is, the word."""
    x, token, parent = logits.double().cpu().numpy(), [], []
    for a in range(0, len(x), K):
        found = []
        for b in range(a, a + K):
            if live[b] == 0:
                found.append((-float(score[b]), b, 0.0, eos))
                continue
            top = x[b].max()
            c = float(score[b]) + (x[b] - top - np.log(np.exp(x[b] - top).sum()))
            best = np.lexsort((np.arange(len(c)), -x[b], -c))[:K]
            found += [(-c[w], b, -x[b][w], w) for w in best]
        for _, b, _, w in sorted(found)[:K]:
            token.append(w)
            parent.append(b)
    got = decode.beam_select(logits, score, live, beams=K, eos=eos)
    assert got[0].tolist() == token and got[1].tolist() == parent


@pytest.mark.parametrize("V", [300, 30000, 100003])
@pytest.mark.parametrize("K", [3, 8, 16])
def test_equal_candidates_go_by_their_logits(K, V):
    g = torch.Generator("cuda").manual_seed(V + K)
    live = torch.ones(2 * K, device="cuda", dtype=I)
    # logits far below 64 bits of the highest one
    logits = 1e-20 * torch.randn(2 * K, V, device="cuda", generator=g)
    logits[:, V // 2] = 100.0
    check_order(logits, torch.zeros(2 * K, device="cuda"), live, K, 2)
    # scores beside which the logits do not count, of live beams and of one that has ended
    logits = torch.randn(2 * K, V, device="cuda", generator=g)
    score = torch.full((2 * K,), -3e38, device="cuda")
    check_order(logits, score, live, K, 2)
    live[K + 1] = 0
    score[:K - 1] = -3.1e38
    check_order(logits, score, live, K, 2)
    # zeros of either sign are equal, and so are more than are ranked side by side
    logits = torch.where(torch.rand(2 * K, V, device="cuda", generator=g) < 0.5, 0.0, -0.0)
    check_order(logits, score, live, K, 2)


# ---- attention: queries of very different sizes ------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("D,H,kv", [(64, 8, 1), (128, 6, 2), (256, 16, 2), (64, 4, 4)])
@pytest.mark.parametrize("M", [8, 400])
@pytest.mark.parametrize("size", [1000.0, 1e5, 1e8, 1e12, 1e30])
def test_a_large_query_beside_a_key_of_zero(type, D, H, kv, M, size):
    """One dimension in which the keys are zero: the score is what the others say, whatever the query holds there."""
    q, kc, vc, table, tok = attend_inputs(np.random.default_rng([D, H]), [100, 120, 1, 128], H, kv, D, 16, M, type)
    kc[..., 9] = torch.where(kc[..., 9].isnan(), kc[..., 9], 0.0)
    q[:3, :, 9] = size
    check_attention(q, kc, vc, table, tok)


# ---- signatures that have been given up ------------------------------------------------------------------------------------------
def test_more_signatures_than_are_kept():
    """A call whose signature has been given up is defined again; a graph that it was captured in goes on."""
    q, kc, vc, table, tok = attend_inputs(np.random.default_rng(3), [500, 3000, 1], 8, 2, 64, 16, 400, torch.bfloat16)
    table, tok = dev(table, I), dev(tok, I)
    want = decode.paged_attention(q, kc, vc, table, tok)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = decode.paged_attention(q, kc, vc, table, tok)
    logits, score, live = torch.randn(2, 5000, device="cuda"), torch.zeros(2, device="cuda"), torch.tensor([0, 1], device="cuda", dtype=I)
    first = decode.beam_select(logits, score, live, beams=2, eos=0)
    for eos in range(1, 4300):
        last = decode.beam_select(logits, score, live, beams=2, eos=eos)
        if eos == 2000:
            torch.cuda.synchronize()
    assert decode._decode.count() == 4096
    assert last[0][0].item() == 4299 and first[0][0].item() == 0
    again = decode.beam_select(logits, score, live, beams=2, eos=0)
    assert all(torch.equal(a, b) for a, b in zip(again, first))
    got.zero_()
    graph.replay()
    assert torch.equal(got, want) and torch.equal(decode.paged_attention(q, kc, vc, table, tok), want)
    assert capi.device_error() == 0


def test_tangents_are_refused_by_a_known_signature_too():
    import torch.autograd.forward_ad as fw
    q, kc, vc, table, tok = attend_inputs(np.random.default_rng(3), [50, 3], 4, 2, 64, 16, 4, F)
    table, tok = dev(table, I), dev(tok, I)
    want = decode.paged_attention(q, kc, vc, table, tok)
    for _ in range(2):
        with fw.dual_level():
            with pytest.raises(capi.ReefError, match="tangents"):
                decode.paged_attention(fw.make_dual(q, torch.ones_like(q)), kc, vc, table, tok)
            assert torch.equal(decode.paged_attention(q, kc, vc, table, tok), want)


def test_views_that_stand_for_their_negative_are_refused():
    logits, live = torch.randn(1, 50, device="cuda"), torch.ones(1, device="cuda", dtype=I)
    score = torch.full((1,), 3 - 7j, device="cuda").conj().imag            # 7, in memory -7
    assert score.is_neg() and score.is_contiguous()
    decode.beam_select(logits, score.resolve_neg(), live, beams=1, eos=0)
    for _ in range(2):
        with pytest.raises(capi.ReefError, match="negative"):
            decode.beam_select(logits, score, live, beams=1, eos=0)


# ---- attention: the keys of all rows divided among blocks, more tokens than a warp has lanes, and than a block has threads ---------------
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,kv,D", [(2, 2, 64), (8, 1, 64), (6, 2, 128), (10, 1, 128), (3, 1, 256)])
@pytest.mark.parametrize("T", [32, 33, 256, 257, 600])
def test_division_of_many_tokens(type, H, kv, D, T):
    R, S, M = 7, 16, 4096
    assert len(decoding.paged_attention(T, R, H, kv, D, S, M, 100, {F: "float32", torch.bfloat16: "bfloat16", torch.float16: "float16"}[type])) == 2
    rng = np.random.default_rng([T, H, D])
    lens = np.array([700, 0, 1, 16, 333, 17, 512])
    _, kc, vc, table, _ = attend_inputs(rng, lens, H, kv, D, S, M, type)
    q = torch.randn(T, H, D, device="cuda")
    for kind in range(3):
        tok = np.zeros((T, 4), int)
        tok[:, 1] = rng.integers(0, R, T) if kind else np.arange(T) * R // T
        tok[:, 2] = lens[tok[:, 1]]
        if kind == 1:                                       # any length up to the row's; tokens without a row
            tok[:, 2] = rng.integers(0, tok[:, 2] + 1)
            tok[rng.random(T) < 0.1, 1] = -1
            tok[T // 3, 1] = R
        if kind == 2:                                       # runs of tokens without keys, at both ends and between
            tok[: T // 4, 2] = 0
            tok[T // 2:T // 2 + T // 5, 2] = -3
            tok[-T // 8:, 2] = 0
        out = torch.full((T, H, D), 7.0, device="cuda")
        got = check_attention(q, kc, vc, table, tok, out=out)
        assert not got[(tok[:, 2] <= 0) | (tok[:, 1] < 0) | (tok[:, 1] >= R)].any()


@pytest.mark.parametrize("type", TYPES)
def test_division_of_a_single_row_among_many_tokens(type):
    """One token with keys among hundreds without, wherever it stands."""
    T, H, kv, D, S, M = 300, 8, 2, 64, 16, 4096
    q, kc, vc, table, _ = attend_inputs(np.random.default_rng(1), [30000], H, kv, D, S, M, type)
    q = torch.randn(T, H, D, device="cuda")
    for at in (0, 1, 255, 256, 299):
        tok = np.zeros((T, 4), int)
        tok[:, 1] = -1
        tok[at] = 0, 0, 30000, 0
        got = check_attention(q, kc, vc, table, tok, out=torch.full((T, H, D), 7.0, device="cuda"))
        assert got[at].any() and not got[np.arange(T) != at].any()


# ---- attention: the largest queries ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("H,kv", [(2, 2), (8, 1), (6, 2)])
@pytest.mark.parametrize("M", [8, 400])
@pytest.mark.parametrize("size", [3e38, -3e38])
def test_the_largest_queries(type, H, kv, M, size):
    """3e38 times a key of 4 is within fp32 once it is scaled by log2 e / 8, and a single key, or equal ones, have all the weight: scores of keys
    that differ there are 1e29 apart or more, and what the other dimensions say is lost in 32 and in 64 bits alike.  Beside keys of zero it counts."""
    q, kc, vc, table, tok = attend_inputs(np.random.default_rng(6), [100, 120, 1], H, kv, 64, 16, M, type)
    kc[..., 9] = torch.where(kc[..., 9].isnan(), kc[..., 9], kc[..., 9].clamp(-4, 4))
    q[0, 0, 9] = size
    check_attention(q, kc, vc, table, tok)
    kc[..., 9] = torch.where(kc[..., 9].isnan(), kc[..., 9], 0.0)
    check_attention(q, kc, vc, table, tok)


# ---- page tables: what becomes of a refused row's pages --------------------------------------------------------------------------------
def _refuse_one(lens, new, tokens=100, pages=8, parent=None):
    """Two rows of the pages 0, 1 and 2, 3 in a pool of eight, four tokens to a page, four pages to a row."""
    table = dev([[0, 1, -1, -1], [2, 3, -1, -1]], I)
    return table, decode.page_tables(table, dev(lens, I), dev(new, I), pages=pages, page_size=4, tokens=tokens, parent=parent)


def test_pages_of_refused_rows():
    # no pages left, or no tokens: the old ones are nobody else's
    _, s = _refuse_one([8, 8], [4, 5], pages=5)
    assert s.status.tolist() == [0, 1] and s.table.tolist() == [[0, 1, 4, -1], [-1] * 4] and s.lens.tolist() == [12, 0]
    _, s = _refuse_one([8, 8], [4, 8], tokens=11)
    assert s.status.tolist() == [0, 3] and s.table[0].tolist() == [0, 1, 4, -1]
    # and the row can be tried again from the old state
    old, s = _refuse_one([8, 8], [0, 4], pages=5)
    assert s.status.tolist() == [0, 0] and s.table.tolist() == [[0, 1, -1, -1], [2, 3, 4, -1]]
    # beyond the longest row it keeps nothing: its pages are the first free ones
    old, s = _refuse_one([8, 8], [9, 8])
    assert s.status.tolist() == [2, 0] and s.table[1].tolist() == [2, 3, 0, 1] and old[0].tolist() == [0, 1, -1, -1]
    # but for those that another row goes on from
    _, s = _refuse_one([8, 8], [9, 8], parent=dev([0, 0], I))
    assert s.status.tolist() == [2, 0] and s.table[1].tolist() == [0, 1, 2, 3]
    # given no new tokens it stays
    _, s = _refuse_one([8, 16], [8, 0])
    assert s.status.tolist() == [0, 0] and s.lens.tolist() == [16, 16]


def test_a_state_without_parents_has_no_copies():
    out = decode.page_state(2, 4, 100, fork=True)
    out.fork.fill_(5)
    table, lens, new = dev([[0, 1, -1, -1], [2, 3, -1, -1]], I), dev([8, 7], I), dev([1, 1], I)
    s = decode.page_tables(table, lens, new, pages=8, page_size=4, tokens=100, out=out)
    assert s.fork is None and (out.fork == 5).all() and s.lens.tolist() == [9, 8]
    s = decode.page_tables(table, lens, new, pages=8, page_size=4, tokens=100, out=out, parent=dev([0, 1], I))
    assert s.fork is out.fork and s.fork.tolist() == [[-1, -1, 0, 0]] * 2
