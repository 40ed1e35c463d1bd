"""Scores of given tokens at the ends of their ranges: temperatures, vocabularies, rows that hold NaN."""
import math

import pytest
import torch

import drakes_amd
from drakes_amd import ops
from test_token_scores import ULP, close, oracle


@pytest.mark.gpu
@pytest.mark.parametrize('V', [5, 300, 9001])
def test_a_large_gradient_of_the_entropy_leaves_far_columns_alone(dev, V):
    """Where a probability is 0 nothing is passed on, however large the factor and however far the logit."""
    lg = torch.zeros(2, V)
    lg[:, 1] = torch.finfo(torch.float32).min
    lg[1, 2] = -1e30
    tok = torch.zeros(2, dtype=torch.int64)
    s = ops.token_scores(lg.to(dev), tok.to(dev))
    d = ops.token_scores_bwd(lg.to(dev), tok.to(dev), s, g_entropy=torch.full((2,), 1e25, device=dev)).cpu()
    assert torch.isfinite(d).all() and bool((d[:, 1] == 0).all()) and float(d[1, 2]) == 0
