"""The decoding operators at sizes and values where one form of a kernel ends and another begins, against their definitions."""
import numpy as np
import pytest
import torch

from reef_b200 import capi, decode
from reef_b200.resources import decoding
from test_gpu_decode import ATTEND_TOL, F, I, attend_by_hand, attend_inputs, dev

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
