"""The decoding schedule over tables made for long rows, where a row's keys are divided among blocks: every attention against its definition, in
every flavour and preempted, the same bits."""
import json

import numpy as np
import pytest
import torch

import test_gpu_decoder as short
from gpu_util import all_storage, load_executor
from reef_b200 import capi
from reef_b200.resources.graph import parse_kname
from test_gpu_decode import ATTEND_TOL, attend_by_hand

pytestmark = pytest.mark.gpu
M = 2000


def test_steps_of_a_schedule_for_long_rows(gen, monkeypatch):
    base = gen("decoder_tiny", variant="_long", max_pages=M)
    model = json.load(open(base + ".json"))
    ops = [parse_kname(k["name"])[0] for k in model["kernels"]]
    assert ops.count("reef_paged_attention_parts") == ops.count("reef_paged_attention_join") == 2 and "reef_paged_attention" not in ops
    monkeypatch.setattr(short, "M", M)
    e, state = load_executor(base), None
    for step in range(6):
        short.feed(e.set_input, short.inputs_of(step, state))
        e.execute()
        data = all_storage(e, model)
        for k, op in zip(model["kernels"], ops):
            if op != "reef_paged_attention_parts":
                continue
            buf = [data[i] for i in k["args"]]
            kc, vc = (torch.from_numpy(x.view(np.int16)).view(torch.bfloat16).view(short.PAGES, 2, short.S, 64) for x in buf[1:3])
            q = torch.from_numpy(buf[0].reshape(short.T, -1)[:, :256].copy()).view(short.T, 4, 64)
            want, size = attend_by_hand(q, kc, vc, buf[3].reshape(short.R, M), buf[4].reshape(short.T, 4))
            got = torch.from_numpy(buf[5]).view(short.T, 4, 64)
            assert ((got - want).abs() <= ATTEND_TOL * size + 2.0 ** -24 * size.amax()).all()
        state = short.outputs(model, data)
        assert not state["status"].any() and state["lens_out"].max() > step
        for run in (e.execute_graph, e.execute_preemptable, e.execute_dispatch, lambda: e.execute_preempt_resume(30), lambda: e.execute_preempt_resume(90)):
            run()
            again = short.outputs(model, all_storage(e, model))
            assert all(np.array_equal(again[n], state[n], equal_nan=True) for n in short.NAMES), step
    assert capi.device_error() == 0
    e.close()
