"""Calls of the serving-step operators at the edges of what their documentation allows."""
import numpy as np
import pytest
import torch

from test_serving_step_gpu import BF, F32, FP, _check_logprobs, _logits

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ log probabilities
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("v", [1501, 5003, 32003, 70003])
def test_logprobs_of_many_infinite_logits(dtype, v):
    """+inf counts as the largest float32, which is no value of the 16-bit types and lies above all of theirs: rows of it alone, more of it
    than a workgroup ranks at a time, a few beside as many of the type's own largest value, one row a workgroup and in pieces."""
    inf, most = float("inf"), torch.finfo(dtype).max
    gen = torch.Generator().manual_seed(v)
    x = torch.randn(13, v, generator=gen)
    some = torch.randperm(v, generator=gen)
    x[0] = inf
    x[1, some[:513]] = inf
    x[2, some[:min(3000, v - 1)]] = inf
    x[3, ::2] = inf
    x[4, some[:512]] = inf
    x[5, some[:1000]] = most
    x[5, some[1000:1007]] = inf
    x[6, :1000] = most                                        # the infinite ones behind all of them
    x[6, -3:] = inf
    x[7] = most
    x[7, 1::2] = inf
    x[8] = most
    x[9] = -inf
    x[9, 1:v - 1] = inf
    x[10, some[:700]] = inf
    x[10, some[700:1400]] = float("nan")
    x[11, :600] = -inf
    x[11, 600:601] = inf
    x[12, -600:] = inf
    x = x.to(dtype).cuda()
    for n in (1, 20, 64):
        for tokens in (np.arange(13) * (v // 13), np.r_[v - 1, some[:12].numpy()], np.r_[1, some[990:1002].numpy()]):
            _check_logprobs(x, tokens, n)
    wide = torch.full((3, v + 3), inf, dtype=dtype, device="cuda")
    wide[1, 2::2] = most
    wide[2, :700] = most
    for first in (1, 3):
        _check_logprobs(wide[:, first:first + v - 1], np.array([0, 5, v - 2]), 20)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("v", [65536, 98304, 131072])
def test_logprobs_of_rows_that_end_where_a_piece_begins(dtype, v):
    """The last workgroup of an aligned row has no column then, of others a few."""
    wide = _logits(3, v + 8, dtype, v)
    for first in (0, 1, 8):
        x = wide[:, first:first + v]
        for n in (0, 5, 64):
            _check_logprobs(x, np.array([0, v - 1, v // 2]), n)
    x[0] = float("-inf")
    x[1, :-3] = float("nan")
    x[2, -1] = float("inf")
    _check_logprobs(x, np.array([0, v - 2, v - 1]), 5)
