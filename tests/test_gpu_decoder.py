"""A run of the decoding operators as they are used: the decoding schedule over several steps, in every flavour, preempted, beside real-time
requests, and the same step on torch tensors.

Every kernel's output is held against its definition on the inputs that the GPU's own buffers hold (no buffer is used twice), so that a
difference in a projection's last bits cannot move a beam in one of the two.  Matmuls multiply TF32 operands (10 bits: two roundings of
2^-11, and truncation of activations 2^-10): 2^-9 of the sum of magnitudes.  LayerNorm: 1e-5 of the row's scale.
"""
import json

import numpy as np
import pytest
import torch

from gpu_util import all_storage, load_executor
from reef_b200 import capi, decode
from reef_b200.resources.graph import parse_kname
from test_gpu_decode import attend_by_hand, select_by_hand, tables_by_hand

pytestmark = pytest.mark.gpu
R, K, M, S, PAGES, T, EOS = 6, 3, 12, 8, 80, 40, 2


def check_pass(model, data, caches_before):
    """Every kernel of a pass from the buffers it read."""
    for k in model["kernels"]:
        op, a = parse_kname(k["name"])
        buf = [data[i] for i in k["args"]]
        if op == "reef_page_tables":
            want = tables_by_hand(buf[0].reshape(R, M), buf[1], buf[2], buf[3], PAGES, S, T)
            for x, y in zip(buf[4:], want):
                assert np.array_equal(x, y.ravel())
        elif op == "reef_embedding":
            pos = np.clip(buf[4].reshape(T, 4)[:, 2] - 1, 0, a["npos"] - 1)
            assert np.array_equal(buf[0].reshape(T, -1), buf[1].reshape(a["vocab"], -1)[buf[2]] + buf[3].reshape(a["npos"], -1)[pos])
        elif op == "reef_layernorm":
            x = buf[1].reshape(T, -1).astype(np.float64)
            y = (x - x.mean(1, keepdims=True)) / np.sqrt(x.var(1, keepdims=True) + 1e-12) * buf[2] + buf[3]
            assert np.abs(buf[0].reshape(T, -1) - y).max() <= 1e-5 * np.abs(y).max()
        elif op.startswith("reef_matmul_nt"):
            x, w = buf[0].reshape(T, -1).astype(np.float64), buf[1].reshape(a["n"], -1).astype(np.float64)
            y, size = x @ w.T + buf[3], np.abs(x) @ np.abs(w).T
            if "gelu" in op:
                from math import erf
                y = y * 0.5 * (1 + np.vectorize(erf)(y / np.sqrt(2)))
            if "residual" in op:
                y = y + buf[4].reshape(y.shape)
            assert (np.abs(buf[2].reshape(y.shape) - y) <= 2.0 ** -9 * size * 1.2 + 1e-5).all(), k["name"]
        elif op == "reef_paged_append":
            tok, fork = buf[2].reshape(T, 4), buf[3].reshape(R, 4)
            for which, off in ((4, a["ko"]), (5, a["vo"])):
                want = caches_before[k["args"][which]].clone()
                for src, dst, n, _ in fork:
                    if src >= 0:
                        want[dst, :, :n] = want[src, :, :n]
                new = torch.from_numpy(buf[0].reshape(T, -1)[:, off:off + 128].copy()).view(T, 2, 64).bfloat16()
                for i, (slot, r, _, _) in enumerate(tok):
                    if r >= 0:
                        want[slot // S, :, slot % S] = new[i]
                assert torch.equal(torch.from_numpy(buf[which].view(np.int16)).view(torch.bfloat16).view(PAGES, 2, S, 64).view(torch.int16), want.view(torch.int16))
        elif op == "reef_paged_attention":
            kc, vc = (torch.from_numpy(x.view(np.int16)).view(torch.bfloat16).view(PAGES, 2, S, 64) for x in buf[1:3])
            q = torch.from_numpy(buf[0].reshape(T, -1)[:, :256].copy()).view(T, 4, 64)
            want, size = attend_by_hand(q, kc, vc, buf[3].reshape(R, M), buf[4].reshape(T, 4))
            got = torch.from_numpy(buf[5]).view(T, 4, 64)
            assert ((got - want).abs() <= 2.0 ** -16 * size + 2.0 ** -24 * size.amax()).all()
        elif op == "reef_beam_pick":
            logits = data[[i for i, s in enumerate(model["storage"]) if s["name"] == "output"][0]].reshape(T, -1)
            want = select_by_hand(torch.from_numpy(logits), torch.from_numpy(buf[1]), torch.from_numpy(buf[2]), K, EOS, buf[3])
            assert np.array_equal(buf[4], want[0]) and np.array_equal(buf[5], want[1]) and np.array_equal(buf[7], want[3])
            there = np.isfinite(want[2])
            assert np.allclose(buf[6][there], want[2][there], atol=2e-6, rtol=1e-6) and np.array_equal(buf[6][~there], want[2][~there])
        else:
            assert op == "reef_beam_scan", op


def inputs_of(step, state):
    """Prompts of two requests in the first step, then a token for every live beam; a request ends and another begins on the way."""
    rng = np.random.default_rng(step)
    ids = rng.integers(3, 1000, T).astype(np.int64)
    if step == 0:
        new, parent = np.array([9, 0, 0, 17, 0, 0]), np.array([-1] * 6)
        score, live = np.array([0, -np.inf, -np.inf] * 2, np.float32), np.ones(R, int)
        return dict(ids=ids, table=np.full(R * M, -1), lens=np.zeros(R, int), new=new, parent=parent, score=score, live=live)
    d = dict(ids=ids, table=state["table_out"], lens=state["lens_out"], new=state["live_out"], parent=state["parent_out"], score=state["score_out"],
             live=state["live_out"])
    if step == 4:                                           # the first request is done: a new prompt takes its place
        for name, v in (("parent", -1), ("new", [13, 0, 0]), ("live", 1), ("score", [0, -np.inf, -np.inf])):
            d[name] = d[name].copy()
            d[name][:K] = v
    ids[:R] = np.where(state["token_out"] >= 0, state["token_out"], 0)[:R]
    return d


def feed(set_input, d):
    for name, v in d.items():
        set_input(name, v.astype({"ids": np.int64, "score": np.float32}.get(name, np.int32)))


NAMES = ("table_out", "lens_out", "status", "fork", "token_out", "parent_out", "score_out", "live_out", "output")


def outputs(model, data):
    return {s["name"]: data[i] for i, s in enumerate(model["storage"]) if s["name"] in NAMES}


@pytest.fixture(scope="module")
def decoder(gen):
    base = gen("decoder_tiny")
    return base, json.load(open(base + ".json"))


def test_steps_of_the_schedule(decoder):
    base, model = decoder
    e = load_executor(base)
    state = None
    for step in range(7):
        before = {i: torch.from_numpy(e.get_data(i, s["size"], np.int16)).view(torch.bfloat16).view(PAGES, 2, S, 64)
                  for i, s in enumerate(model["storage"]) if "_cache" in s["name"]}
        feed(e.set_input, inputs_of(step, state))
        e.execute()
        data = all_storage(e, model)
        check_pass(model, data, before)
        state = outputs(model, data)
        assert not state["status"].any()
        for run in (e.execute_graph, e.execute_preemptable, e.execute_dispatch, lambda: e.execute_preempt_resume(30), lambda: e.execute_preempt_resume(90)):
            run()                                           # the same inputs again: the same bits
            again = outputs(model, all_storage(e, model))
            assert all(np.array_equal(again[n], state[n], equal_nan=True) for n in NAMES), step
    assert capi.device_error() == 0
    e.close()


def test_best_effort_decoder_beside_real_time_requests(decoder, gen):
    """The steps of the schedule as a best-effort client, preempted and padded by a real-time one, give what they give alone."""
    base, model = decoder
    alone, state, e = [], None, load_executor(base)
    for step in range(6):
        feed(e.set_input, inputs_of(step, state))
        e.execute_graph()
        state = outputs(model, all_storage(e, model))
        alone.append(state)
    e.close()
    other = gen("resnet18_64")
    s = capi.REEFScheduler(capi.REEFScheduler.REEF, 0)
    be = s.load_model_files(base + ".json", base + ".profile.json", base + ".param")
    rt = s.load_model_files(other + ".json", other + ".profile.json", other + ".param")
    s.bind_model_queue(s.create_queue(capi.REEFScheduler.BestEffortQueue), be)
    s.bind_model_queue(s.create_queue(capi.REEFScheduler.RealTimeQueue), rt)
    s.run()
    x = np.random.default_rng(1).standard_normal(3 * 64 * 64).astype(np.float32)
    try:
        state = None
        for step in range(6):
            feed(lambda n, v: s.set_input(be, v, n), inputs_of(step, state))
            task = s.new_task(be)
            for _ in range(4):
                s.set_input(rt, x)
                s.wait_task(s.new_task(rt))
            s.wait_task(task)
            state = {n: s.get_output(be, n, np.float32 if n in ("score_out", "output") else np.int32) for n in NAMES}
            assert all(np.array_equal(state[n], alone[step][n], equal_nan=True) for n in NAMES), step
    finally:
        s.close()
    assert capi.device_error() == 0


def test_real_time_decoder(decoder):
    base, model = decoder
    s = capi.REEFScheduler(capi.REEFScheduler.REEF, 0)
    rt = s.load_model_files(base + ".json", base + ".profile.json", base + ".param")
    be = s.load_model_files(base + ".json", base + ".profile.json", base + ".param")
    s.bind_model_queue(s.create_queue(capi.REEFScheduler.RealTimeQueue), rt)
    s.bind_model_queue(s.create_queue(capi.REEFScheduler.BestEffortQueue), be)
    s.run()
    try:
        states = {rt: None, be: None}
        for step in range(6):
            for mid in (be, rt):
                feed(lambda n, v: s.set_input(mid, v, n), inputs_of(step, states[mid]))
            tasks = [s.new_task(be), s.new_task(rt)]
            for t in tasks:
                s.wait_task(t)
            for mid in (rt, be):
                states[mid] = {n: s.get_output(mid, n, np.float32 if n in ("score_out", "output") else np.int32) for n in NAMES}
            assert all(np.array_equal(states[rt][n], states[be][n], equal_nan=True) for n in NAMES), step
            assert not states[rt]["status"].any()
    finally:
        s.close()


def test_attention_with_parts_is_preempted_and_resumed(tmp_path):
    """The form with parts and its join as best-effort kernels: left in the middle, launched again, the same bits."""
    from reef_b200.resources import decoding
    from reef_b200.resources.graph import Graph
    T, H, kv, D, S, M, pages = 8, 8, 2, 64, 16, 3000, 12000
    names = decoding.paged_attention(T, T, H, kv, D, S, M, pages, "bfloat16")
    assert len(names) == 2
    g = Graph("parts")
    rng = np.random.default_rng(0)
    q, k, v = g.input("q", T * H * D), g.input("k", pages * kv * S * D * 2, "byte"), g.input("v", pages * kv * S * D * 2, "byte")
    table, tok = g.input("table", T * M, "int32"), g.input("tok", 4 * T, "int32")
    out = g.add_storage("output", T * H * D)
    parts = g.add_storage("parts", capi.Kernel(names[0]).arg_bytes[6], "byte")
    g.kernel(names[0], [q, k, v, table, tok, out, parts])
    g.kernel(names[1], [parts, out])
    base = g.write(str(tmp_path), capi.plan_fn)
    e = load_executor(base, params=False)
    cache = [torch.randn(pages, kv, S, D).bfloat16() for _ in range(2)]
    ids = np.stack([rng.permutation(pages)[:M] for _ in range(T)]).astype(np.int32)
    lens = np.array([48000, 1, 0, 20011, 777, 47999, 16, 30000])
    toks = np.zeros((T, 4), np.int32)
    toks[:, 1], toks[:, 2] = np.arange(T), lens
    qs = rng.standard_normal((T, H, D)).astype(np.float32)
    e.set_input("q", qs)
    e.set_input("k", cache[0].view(torch.int16).numpy())
    e.set_input("v", cache[1].view(torch.int16).numpy())
    e.set_input("table", ids)
    e.set_input("tok", toks)
    e.execute()
    first = e.get_output()
    want, size = attend_by_hand(torch.from_numpy(qs), *cache, ids, toks[:5])
    assert (np.abs(first.reshape(T, H, D)[:5] - want[:5].numpy()) <= 2.0 ** -16 * size[:5].numpy() + 1e-7).all()
    for run in [e.execute_graph, e.execute_preemptable, e.execute_dispatch] + [lambda d=d: e.execute_preempt_resume(d) for d in (5, 15, 25, 40, 60)]:
        run()
        assert np.array_equal(e.get_output(), first)
    assert capi.device_error() == 0
    e.close()


@pytest.mark.parametrize("rows,most", [(16, 64), (70, 130)])
def test_tables_in_every_flavour(tmp_path, rows, most):
    """The blocks of a launch of its own and those of a dispatcher give the same tables, whatever their threads."""
    from reef_b200.resources import decoding
    from reef_b200.resources.graph import Graph
    size, pages, tokens = 4, 12000, 200
    g = Graph("tables")
    rng = np.random.default_rng(rows)
    lens, new, parent = rng.integers(0, most * size - 4, rows), rng.integers(0, 4, rows), np.arange(rows) // 2 * 2
    table, ids, at = np.full((rows, most), -1), rng.permutation(pages), 0
    for r in range(rows):
        n = -(-int(lens[r]) // size)
        table[r, :n] = ids[at:at + n]
        at += n
    names = ("table", "lens", "new", "parent", "table_out", "lens_out", "start", "tok", "status", "fork")
    name = decoding.page_tables(rows, most, size, pages, tokens, fork=True)
    k = capi.Kernel(name)
    sizes = [k.arg_bytes[i] // 4 for i in range(10)]
    bufs = [g.input(n, sizes[i], "int32") if i < 4 else g.add_storage("output" if n == "table_out" else n, sizes[i], "int32") for i, n in enumerate(names)]
    g.kernel(name, bufs)
    e = load_executor(g.write(str(tmp_path), capi.plan_fn), params=False)
    for n, v in zip(names, (table, lens, new, parent)):
        e.set_input(n, v.astype(np.int32))
    want = tables_by_hand(table, lens, new, parent, pages, size, tokens)
    for run in (e.execute, e.execute_graph, e.execute_preemptable, e.execute_dispatch):
        run()
        for b, n, y in zip(bufs[4:], sizes[4:], want):
            assert np.array_equal(e.get_data(b, 4 * n, np.int32), y.ravel())
    e.close()


def test_a_step_on_tensors():
    """The operators one after the other on torch tensors, captured as one graph and replayed, against an uncached computation."""
    torch.manual_seed(0)
    R, K, H, kv, D, S, M, pages, V, layers = 4, 2, 6, 2, 64, 4, 8, 60, 500, 2
    I = torch.int32     # noqa: E741
    caches = [[torch.zeros(pages, kv, S, D, device="cuda", dtype=torch.float32) for _ in range(2)] for _ in range(layers)]
    emb, pos = torch.randn(V, H * D, device="cuda"), torch.randn(M * S, H * D, device="cuda")
    proj = [torch.randn(H * D, (H + 2 * kv) * D, device="cuda") / 20 for _ in range(layers)]
    back = torch.randn(H * D, V, device="cuda") / 10
    states = [decode.page_state(R, M, R, fork=True) for _ in range(2)]
    new, parent = torch.ones(R, device="cuda", dtype=I), torch.full((R,), -1, device="cuda", dtype=I)
    ids = torch.tensor([3, 4, 5, 6], device="cuda")
    score, live = torch.tensor([0.0, -torch.inf, 0.0, -torch.inf], device="cuda"), torch.ones(R, device="cuda", dtype=I)
    names = ("token", "parent", "score", "live")

    def step(old, out):
        decode.page_tables(old.table, old.lens, new, pages=pages, page_size=S, tokens=R, parent=parent, out=out)
        x = emb[ids] + pos[(out.tok[:, 2] - 1).clamp(min=0).long()]
        for w, (kc, vc) in zip(proj, caches):
            qkv = x @ w
            q, k, v = (y.unflatten(1, (-1, D)) for y in qkv.split([H * D, kv * D, kv * D], 1))
            decode.paged_append(k, v, out.tok, kc, vc, fork=out.fork)
            x = x + decode.paged_attention(q, kc, vc, out.table, out.tok).flatten(1)
        return decode.beam_select(x @ back, score, live, beams=K, eos=1, start=out.start)

    def uncached(words):
        x = (emb[words] + pos[:len(words)]).double()
        for w in proj:
            q, k, v = (y.unflatten(1, (-1, D)) for y in (x @ w.double()).split([H * D, kv * D, kv * D], 1))
            k, v = (y.repeat_interleave(H // kv, 1) for y in (k, v))
            s = torch.einsum("ihd,jhd->hij", q, k) / D ** 0.5
            s = torch.where(torch.ones_like(s[0]).tril().bool(), s, -torch.inf)
            x = x + torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).flatten(1)
        return torch.log_softmax(x[-1] @ back.double(), 0)

    graphs = []
    step(states[0], states[1])                              # set up outside of a capture; nothing is kept of it
    for old, out in (states, states[::-1]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step(old, out)))
    for c in caches:
        for x in c:
            x.zero_()
    for old in states:
        old.lens.zero_()
    words, total = [[3], [4], [5], [6]], [0.0, -np.inf, 0.0, -np.inf]
    for n in range(M * S - 1):
        g, got = graphs[n % 2]
        g.replay()
        found = {k: v.clone() for k, v in zip(names, got)}
        assert not states[1 - n % 2].status.any()
        # every chosen beam's score is the sum of its words' log-probabilities, and the best ones were chosen
        for a in range(0, R, K):
            cand = torch.stack([uncached(torch.tensor(words[r], device="cuda")) + total[r] if live[r] and np.isfinite(total[r]) else
                                torch.full((V,), -torch.inf, device="cuda", dtype=torch.float64).index_fill(
                                    0, torch.tensor([1], device="cuda"), total[r] if not live[r] else -np.inf) for r in range(a, a + K)]).flatten()
            best = cand.sort(descending=True).values[:K]
            mine = found["score"][a:a + K].double()
            assert torch.allclose(mine, best, atol=2e-4), n
        words = [words[int(p)] + [int(t)] if lv else words[int(p)] for p, t, lv in zip(found["parent"], found["token"], found["live"])]
        total = found["score"].double().tolist()
        ids.copy_(found["token"].clamp(min=0))
        parent.copy_(found["parent"])
        score.copy_(found["score"])
        live.copy_(found["live"])
        new.copy_(found["live"])
        if not live.any():
            break
    assert n > 5 and capi.device_error() == 0
