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


def test_temperatures_out_of_range_are_refused():
    """1 / temp times log2 e has to be a number, and a difference of two logits that still counts has to be told from -inf."""
    lib = drakes_amd._lib.load()
    rc = lambda t: (lib.drk_token_scores(None, 0, 5, None, None, 0, t, 0, None, None, None, None, None, 2, 5, None, 0, None), lib.drk_last_error())
    for t in (2.95e-39, 4.2e-39, 9.9e-39, 1.1e26, 1e30, 3e38):
        code, text = rc(t)
        assert code < 0 and b'temp' in text, (t, text)
    for t in (1e-38, 0.1, 1e26):
        code, text = rc(t)
        assert code < 0 and b'temp' not in text, (t, text)               # the null pointers are what is wrong


@pytest.mark.gpu
@pytest.mark.parametrize('V', [3, 40, 700, 9001, 70001])
@pytest.mark.parametrize('temp', [1e-38, 1e-30, 1e-3, 1e19, 1e22, 1e26])
def test_logits_of_a_temperatures_own_size(dev, V, temp):
    """Differences from far below to far above the temperature.  The exponential's argument, up to ~20, and the entropy's sum are
    rounded as at temperature 1."""
    g = torch.Generator().manual_seed(V)
    lg = (torch.randn(4, V, generator=g).double() * 3 * temp).float()
    lg[1, 0] = torch.finfo(torch.float32).min
    lg[2] = 0.0
    lg[3, V // 2] = -math.inf
    tok = torch.full((4,), V - 1)
    exact = torch.tensor(temp, dtype=torch.float32).double().item()
    s = ops.token_scores(lg.to(dev), tok.to(dev), temp=temp, topk=2)
    logp, H, ids, top, lp, p = oracle(lg, tok, None, exact, 2)
    # at 1e-38 logits and differences are subnormal: the inputs are what they are, and the oracle takes the same ones
    close(s.logp, logp, 'logp', 256)
    close(s.entropy, H, 'entropy', 256)
    assert torch.equal(s.top_ids.cpu(), ids)
    gh = torch.full((4,), min(max(temp, 1e-30), 1.0))
    d = ops.token_scores_bwd(lg.to(dev), tok.to(dev), s, g_entropy=gh.to(dev), temp=temp).cpu().double()
    lp0, gh = torch.where(p > 0, lp, torch.zeros_like(lp)), gh.double().unsqueeze(-1)
    want = -p * (lp0 + H.unsqueeze(-1)) * gh / exact
    # with half a step of a product below the normal range, before and after it is divided by the temperature
    bar = p * (lp0.abs() + H.unsqueeze(-1)) * gh / exact * (256 + 4 * lp0.abs()) * ULP + 2.0 ** -148 / exact + 2.0 ** -148
    assert bool(((d - want).abs() <= bar).all())


@pytest.mark.gpu
def test_temperatures_out_of_range_are_refused_from_python(dev):
    lg, tok = torch.zeros(2, 5, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    s = ops.token_scores(lg, tok)
    for t in (4.2e-39, 1e-40, 1e27, 1e39, math.inf):
        with pytest.raises(ValueError, match='temp'):
            ops.token_scores(lg, tok, temp=t)
        with pytest.raises(ValueError, match='temp'):
            ops.token_scores_bwd(lg, tok, s, temp=t)


@pytest.mark.gpu
@pytest.mark.parametrize('V', [2 ** 30 + 1, 2 ** 31 + 7, 2 ** 32 + 7])
def test_a_vocabulary_beyond_the_limit_is_refused(dev, V):
    """Not scored over its first V mod 2^32 columns.  (No row, so nothing is allocated or launched.)"""
    lg, tok = torch.empty(0, V, dtype=torch.float16, device=dev), torch.empty(0, dtype=torch.int64, device=dev)
    with pytest.raises(ValueError, match='2\\^30'):
        ops.token_scores(lg, tok)
    e = torch.empty(0, device=dev)
    with pytest.raises(ValueError, match='2\\^30'):
        ops.token_scores_bwd(lg, tok, ops.TokenScores(e, e, None, None, torch.empty(0, 2, device=dev)), g_logp=e)


@pytest.mark.gpu
@pytest.mark.parametrize('V', [7, 64, 65, 1001, 9001, 140001])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shared', [True, False])
def test_columns_that_do_not_count_get_no_gradient_in_a_row_with_nan(dev, V, dtype, shared):
    """The given token is one of them, and its log-probability is the row's NaN."""
    for t in (0, V // 3, V - 1):
        lg = torch.randn(2, V, generator=torch.Generator().manual_seed(V)).to(dtype)
        lg[:, (t + 2) % V] = math.nan
        allowed = torch.ones(V, dtype=torch.bool)
        allowed[t] = False
        al = (allowed if shared else allowed.expand(2, V).contiguous()).to(dev)
        tok = torch.full((2,), t, device=dev)
        s = ops.token_scores(lg.to(dev), tok, allowed=al, topk=2)
        assert torch.isnan(s.logp).all()
        one = torch.ones(2, device=dev)
        d = ops.token_scores_bwd(lg.to(dev), tok, s, g_logp=one, g_entropy=one, g_top=torch.ones(2, 2, device=dev), allowed=al).cpu()
        assert bool((d[:, t] == 0).all()), d[:, t]
        assert torch.isnan(d[:, allowed]).all()


@pytest.mark.gpu
@pytest.mark.parametrize('V', [5, 22, 64, 65, 1001, 9001, 140001])
@pytest.mark.parametrize('bad', [math.nan, math.inf])
def test_rows_that_are_not_scored_pass_no_gradient_whatever_they_hold(dev, V, bad):
    """The padding of a batch: negative tokens, and logits that came from nothing."""
    x = torch.randn(6, V, generator=torch.Generator().manual_seed(V))
    x[2:4] = bad
    x[4, V // 2] = bad
    tok = torch.tensor([1, 0, -1, -1, -1, V - 1], device=dev)
    ref = x.clone()
    ref[2:5] = 0.0
    out = []
    for lg in (x, ref):
        s = ops.token_scores(lg.to(dev), tok)
        out.append(ops.token_scores_bwd(lg.to(dev), tok, s, g_logp=torch.full((6,), 0.5, device=dev),
                                        g_entropy=torch.tensor([1.0, 1, 0, 0, 0, 1], device=dev)).cpu())
    got, want = out
    assert bool((got[2:5] == 0).all())
    assert torch.equal(got, want)
    live = x.to(dev).requires_grad_()
    drakes_amd.autograd.token_scores_with_grad(live, tok)[0].sum().backward()
    assert torch.isfinite(live.grad).all() and bool((live.grad[2:5] == 0).all())
