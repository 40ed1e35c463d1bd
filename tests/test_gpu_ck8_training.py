"""The bf16 differentiable path with its activations kept in 8 bits (model.hip_checkpoint = 'int8').

Two bars.  (1) The backward against the same formulas in torch, fed the checkpoints' own values, gates and statistics and
rounding the gated gradient to bf16 where the kernels do.  fp32 summation order (~1e-6) turns a rounding of 1e-6 / 2^-9 = 5e-4
of the first layer's elements; what those move turns more in the next layer, and below a few layers the two sides' roundings
are independent: each is uniform within 2^-9 of a value (half a step is at most 2^-8 of it, 2^-9 to 2^-8: taken at 2^-8 / sqrt 3
rms, 2^-8 * sqrt(2 / 3) = 3.2e-3 for the difference of two), at each of 21 layers, in quadrature 1.5e-2 at most of a tensor's
norm when every layer's input gradient is as large as the stream it joins, and the mean of a random mantissa halves it: 7.5e-3.
(2) Against the path without checkpoints:
a kept value is off by at most half a step, and a step is at most 1 / 63.5 of the block's largest magnitude; LayerNorm bounds
that by sqrt(127), so the error's rms is at most 11.3 / 63.5 / sqrt(12) = 0.051 of a value's; the LayerNorm backward adds the
same relative error to the one direction of 128 that it projects out, below 0.051 / sqrt(128) a layer, 20 layers in
quadrature 0.02; bf16 roundings of two forwards that differ in a last place, 0.02: 0.1 in all."""
import math

import pytest
import torch

import drakes_amd
from drakes_amd import autograd, ops

pytestmark = pytest.mark.gpu
C = 128


def _model(dev, det_sd, **kw):
    m = drakes_amd.Diffusion(drakes_amd.default_config(**kw)).to(dev)
    m.load_state_dict(det_sd, strict=True)
    m.hip_dtype = 'bf16'
    return m


def _grads(m):
    g = {k: p.grad.detach().clone() for k, p in m.backbone.named_parameters() if p.grad is not None}
    m.zero_grad(set_to_none=True)
    return g


def _open(gates):
    return ((gates.unsqueeze(-1).to(torch.int64) >> torch.arange(8, device=gates.device)) & 1).flatten(-2).float()


def _backward_in_torch(fn, m, dlogits, seq):
    """Parameter gradients from the node's checkpoints, in fp32 torch with the kernels' bf16 rounding points."""
    bb = m.backbone
    P = dict(bb.named_parameters())
    n = bb.num_layers
    conv = lambda dc, w, d: torch.nn.functional.conv_transpose1d(dc.transpose(1, 2).double(), w.detach().bfloat16().double(), padding=(w.shape[2] // 2) * d, dilation=d).transpose(1, 2).float()

    def wgrad(h, dc, taps, d):
        out = torch.zeros(taps, C, C, device=dc.device, dtype=torch.float64)
        L = h.shape[1]
        for t in range(taps):
            off = (t - taps // 2) * d
            lo, hi = max(0, -off), min(L, L - off)
            if hi > lo:
                out[t] = h[:, lo + off:hi + off].reshape(-1, C).double().t().contiguous() @ dc[:, lo:hi].reshape(-1, C).double()
        return out.permute(2, 1, 0)

    g = {}
    y, flat = fn.y.clone(), lambda t: t.reshape(-1, t.shape[-1]).double()
    g['final_conv.2.weight'] = (flat(dlogits).t() @ flat(y)).unsqueeze(-1)
    g['final_conv.2.bias'] = flat(dlogits).sum(0)
    dpre = (dlogits @ P['final_conv.2.weight'].detach().squeeze(-1)) * (y > 0)
    g['final_conv.0.bias'] = flat(dpre).sum(0)
    dc = dpre.bfloat16().float()
    g['final_conv.0.weight'] = wgrad(ops.ck8_unpack(fn.kept[n]), dc, 1, 0)
    gr = conv(dc, P['final_conv.0.weight'], 1)
    up = gr * _open(fn.kept[n].gates)
    for i in reversed(range(n)):
        g[f'convs.{i}.bias'] = flat(up).sum(0)
        dc = up.bfloat16().float()
        xq = ops.ck8_unpack(fn.kept[i])
        gam, bet = P[f'norms.{i}.weight'].detach(), P[f'norms.{i}.bias'].detach()
        g[f'convs.{i}.weight'] = wgrad(xq.double() * gam.double() + bet.double(), dc, 9, bb.dilation(i))
        dh = conv(dc, P[f'convs.{i}.weight'], bb.dilation(i))
        g[f'norms.{i}.weight'], g[f'norms.{i}.bias'] = flat(dh * xq).sum(0), flat(dh).sum(0)
        a = dh * gam
        mean = lambda t: t.mean(-1, keepdim=True)
        dx = fn.kept[i].rstd.unsqueeze(-1) * (a - mean(a) - xq * mean(a * xq))
        g[f'time_layers.{i}.dense.bias'] = flat(dx).sum(0)
        gr = gr + dx
        up = gr * _open(fn.kept[i].gates)
    g['linear.bias'] = flat(up).sum(0)
    x = torch.nn.functional.one_hot(seq, 5).double() if seq.dtype == torch.int64 else seq.double()
    L = seq.shape[1]
    dw = torch.zeros(9, 5, C, device=dlogits.device, dtype=torch.float64)
    for t in range(9):
        lo, hi = max(0, 4 - t), min(L, L + 4 - t)
        if hi > lo:
            dw[t] = x[:, lo + t - 4:hi + t - 4].reshape(-1, 5).t() @ up[:, lo:hi].reshape(-1, C).double()
    g['linear.weight'] = dw.permute(2, 1, 0)
    return g


@pytest.mark.parametrize('B,L,soft', [(5, 200, False), (3, 77, True), (2, 1024, False), (1, 3, True), (33, 200, True)])
def test_backward_equals_the_formulas_on_the_checkpoints(dev, det_sd, B, L, soft):
    m = _model(dev, det_sd, length=L)
    g = torch.Generator().manual_seed(B)
    seq = torch.softmax(torch.randn(B, L, 5, generator=g), -1).to(dev) if soft else torch.randint(0, 5, (B, L), generator=g).to(dev)
    seq.requires_grad_(soft)
    logits = autograd.backbone_with_grad(m.backbone, seq, torch.zeros(1, device=dev), 'bf16', keep='int8')
    dlogits = torch.randn(B, L, 5, generator=g).to(dev)
    want = _backward_in_torch(logits.grad_fn, m, dlogits, seq.detach())
    logits.backward(dlogits)
    got = _grads(m)
    for k, w in want.items():
        err = float((got[k].double() - w).norm())
        assert err <= 7.5e-3 * float(w.norm()) + 1e-6, (k, err, float(w.norm()))
    if soft:
        assert seq.grad.shape == seq.shape and torch.isfinite(seq.grad).all() and float(seq.grad.norm()) > 0


@pytest.mark.parametrize('B,L', [(32, 200), (4, 500)])
def test_against_the_path_without_checkpoints(dev, det_sd, B, L):
    m = _model(dev, det_sd, length=L)
    x = torch.randint(0, 5, (B, L), generator=torch.Generator().manual_seed(1)).to(dev)
    tgt = torch.randint(0, 4, (B, L), generator=torch.Generator().manual_seed(2)).to(dev)
    only = torch.where(x == 4, tgt, torch.full_like(tgt, -1))
    out = {}
    for keep in (None, 'int8'):
        m.hip_checkpoint = keep
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        logp = m.score_tokens(x, torch.zeros(B, device=dev), only)[0]
        held = torch.cuda.memory_allocated() - before
        (-logp.sum() / (x == 4).sum()).backward()
        out[keep] = (logp.detach(), held, _grads(m))
    (a, held_a, ga), (b, held_b, gb) = out[None], out['int8']
    # the forwards differ where a LayerNorm output's bf16 rounding does; the logits' own bar of the bf16 path is 0.05
    assert float((a - b).abs().max()) < 0.05
    assert held_b * 3.5 < held_a, (held_a, held_b)
    for k in ga:
        rel = float((ga[k] - gb[k]).norm()) / float(ga[k].norm())
        assert rel < 0.1, (k, rel)


def test_chain_and_frozen_model(dev, det_sd):
    """Two forwards of one chain collect the same gradients as two single ones; a frozen model passes on the input's only."""
    m = _model(dev, det_sd, length=64)
    g = torch.Generator().manual_seed(3)
    s = [torch.softmax(torch.randn(4, 64, 5, generator=g), -1).to(dev) for _ in range(2)]
    dl = [torch.randn(4, 64, 5, generator=g).to(dev) for _ in range(2)]
    z = torch.zeros(1, device=dev)
    for x, d in zip(s, dl):
        autograd.backbone_with_grad(m.backbone, x, z, 'bf16', keep='int8').backward(d)
    want = _grads(m)
    sink, anchor = autograd.grad_chain(m.backbone)
    outs = [autograd.backbone_with_grad(m.backbone, x, z, 'bf16', flat=anchor, sink=sink, sigma_key=0.0, keep='int8') for x in s]
    torch.autograd.backward(outs, dl)
    got = _grads(m)
    assert set(got) == set(want)
    for k in want:                                          # the same sums in another order
        assert float((got[k] - want[k]).norm()) <= 1e-5 * float(want[k].norm()) + 1e-7, k
    x = s[0].clone().requires_grad_()
    autograd.backbone_with_grad(m.backbone, x, z, 'bf16', keep='int8').backward(dl[0])
    dx = x.grad.clone()
    for p in m.backbone.parameters():
        p.requires_grad_(False)
    y = s[0].clone().requires_grad_()
    autograd.backbone_with_grad(m.backbone, y, z, 'bf16', keep='int8').backward(dl[0])
    assert torch.equal(y.grad, dx)


def test_time_conditioned_rows(dev, det_sd):
    """A sigma per batch row: gradients equal those of the rows run one by one."""
    m = _model(dev, det_sd, length=50, time_conditioning=True)
    g = torch.Generator().manual_seed(5)
    x = torch.randint(0, 5, (3, 50), generator=g).to(dev)
    sig = torch.tensor([0.1, 1.0, 3.0], device=dev)
    dl = torch.randn(3, 50, 5, generator=g).to(dev)
    autograd.backbone_with_grad(m.backbone, x, sig, 'bf16', keep='int8').backward(dl)
    got = _grads(m)
    for i in range(3):
        autograd.backbone_with_grad(m.backbone, x[i:i + 1], sig[i:i + 1], 'bf16', keep='int8').backward(dl[i:i + 1])
    want = _grads(m)
    for k in want:
        assert float((got[k] - want[k]).norm()) <= 1e-5 * float(want[k].norm()) + 1e-6, k


def test_fine_tune_sampler_and_refusals(dev, det_sd):
    m = _model(dev, det_sd, length=200, steps=8, truncate_steps=3)
    out = {}
    for keep in (None, 'int8'):
        m.hip_checkpoint = keep
        sample, *_ = m._sample_finetune_gradient(eval_sp_size=8, copy_flag_temp=1.0, seed=11)
        (sample * torch.linspace(-1, 1, 4, device=dev)).sum().backward()
        out[keep] = _grads(m)
    assert set(out[None]) == set(out['int8'])
    for k, v in out['int8'].items():
        assert torch.isfinite(v).all(), k
    dot = sum(float((out[None][k] * out['int8'][k]).sum()) for k in out[None])
    na, nb = (math.sqrt(sum(float((v ** 2).sum()) for v in out[k].values())) for k in (None, 'int8'))
    # the whole gradient as one vector: within 0.1 of each other (above) is a cosine of 0.995; the two chains' bf16 forwards
    # also part by a few flipped ReLU gates per step (the bf16 path's own bar for those: 0.97)
    assert dot / (na * nb) > 0.97
    m.hip_dtype = 'fp32'
    with pytest.raises(NotImplementedError):
        m.score_tokens(torch.zeros(1, 200, dtype=torch.int64, device=dev), torch.zeros(1, device=dev), torch.zeros(1, 200, dtype=torch.int64, device=dev))
    m.hip_dtype, m.hip_checkpoint = 'bf16', 'int4'
    with pytest.raises(ValueError):
        m.score_tokens(torch.zeros(1, 200, dtype=torch.int64, device=dev), torch.zeros(1, device=dev), torch.zeros(1, 200, dtype=torch.int64, device=dev))
    m.hip_checkpoint = 'int8'
    lp = m.score_tokens(torch.full((1, 200), 4, device=dev), torch.zeros(1, device=dev), torch.zeros(1, 200, dtype=torch.int64, device=dev))[0].sum()
    lp.backward(retain_graph=True)
    with pytest.raises(RuntimeError):
        lp.backward()


def _input_gradient_in_torch(fn, m, dlogits):
    """dL/dseq from the node's checkpoints, gates and statistics, with the kernels' bf16 rounding points."""
    bb = m.backbone
    P = {k: p.detach() for k, p in bb.named_parameters()}
    n = bb.num_layers
    conv = lambda dc, w, d: torch.nn.functional.conv_transpose1d(dc.transpose(1, 2).double(), w.bfloat16().double(), padding=(w.shape[2] // 2) * d, dilation=d).transpose(1, 2).float()
    mean = lambda t: t.mean(-1, keepdim=True)
    dpre = (dlogits @ P['final_conv.2.weight'].squeeze(-1)) * (fn.y > 0)
    gr = conv(dpre.bfloat16().float(), P['final_conv.0.weight'], 1)
    up = gr * _open(fn.kept[n].gates)
    for i in reversed(range(n)):
        dh = conv(up.bfloat16().float(), P[f'convs.{i}.weight'], bb.dilation(i))
        a, xq = dh * P[f'norms.{i}.weight'], ops.ck8_unpack(fn.kept[i])
        gr = gr + fn.kept[i].rstd.unsqueeze(-1) * (a - mean(a) - xq * mean(a * xq))
        up = gr * _open(fn.kept[i].gates)
    w = P['linear.weight'].double()
    return torch.nn.functional.conv_transpose1d(up.transpose(1, 2).double(), w, padding=w.shape[2] // 2).transpose(1, 2)


@pytest.mark.parametrize('B,L', [(3, 77), (33, 200), (1, 3), (70, 200), (2, 1024)])
@pytest.mark.parametrize('frozen', [False, True])
def test_input_gradient_equals_the_formulas_on_the_checkpoints(dev, det_sd, B, L, frozen):
    """Bar (1) of the head: the input gradient is the last of the tensors that the same chain of roundings reaches."""
    m = _model(dev, det_sd, length=L)
    if frozen:
        m.requires_grad_(False)
    g = torch.Generator().manual_seed(B)
    seq = torch.softmax(torch.randn(B, L, 5, generator=g), -1).to(dev).requires_grad_()
    logits = autograd.backbone_with_grad(m.backbone, seq, torch.zeros(1, device=dev), 'bf16', keep='int8')
    dlogits = torch.randn(B, L, 5, generator=g).to(dev)
    want = _input_gradient_in_torch(logits.grad_fn, m, dlogits)
    logits.backward(dlogits)
    err = float((seq.grad.double() - want).norm())
    assert err <= 7.5e-3 * float(want.norm()), (err, float(want.norm()))


@pytest.mark.parametrize('B,L', [(32, 200), (70, 200), (4, 1024)])
def test_gradients_stay_within_a_few_percent_of_the_path_without_checkpoints(dev, det_sd, B, L):
    """Bar (2) of the head taken per block of 32 channels: a block's largest magnitude is at most sqrt(32) of its rms, so a kept
    value's error has an rms of at most 5.7 / 63.5 / sqrt(12) = 0.026 of the block's; both a weight gradient and its error are
    sums over the same rows.  With a LayerNorm backward of 0.026 / sqrt(128) at each of 20 layers (0.010) and two forwards' bf16
    roundings (0.02), in quadrature 0.034: 0.04.  Over all parameters, whose blocks are not all at that extreme: half of it."""
    m = _model(dev, det_sd, length=L)
    x = torch.randint(0, 5, (B, L), generator=torch.Generator().manual_seed(1)).to(dev)
    tgt = torch.randint(0, 4, (B, L), generator=torch.Generator().manual_seed(2)).to(dev)
    only = torch.where(x == 4, tgt, torch.full_like(tgt, -1))
    out = {}
    for keep in (None, 'int8'):
        m.hip_checkpoint = keep
        (-m.score_tokens(x, torch.zeros(B, device=dev), only)[0].sum() / (x == 4).sum()).backward()
        out[keep] = _grads(m)
    a, b = out[None], out['int8']
    rel = {k: float((a[k] - b[k]).norm()) / float(a[k].norm()) for k in a}
    worst = max(rel, key=rel.get)
    print(f'worst {worst} {rel[worst]:.4f}, median {sorted(rel.values())[len(rel) // 2]:.4f}')
    assert rel[worst] < 0.04, (worst, rel[worst])
    assert sorted(rel.values())[len(rel) // 2] < 0.02


@pytest.mark.gpu
def test_a_model_from_before_the_setting_runs_without_it(dev, det_sd):
    """A module that was stored whole brings its own attributes along, and hip_checkpoint may not be among them."""
    m = drakes_amd.Diffusion(drakes_amd.default_config(length=16)).to(dev)
    m.load_state_dict(det_sd)
    m.hip_dtype = 'bf16'
    x = torch.full((2, 16), 4, dtype=torch.int64, device=dev)
    want = m.score_tokens(x, torch.zeros(1, device=dev), x.clamp(max=3))[0].detach()
    m.__dict__.pop('hip_checkpoint', None)
    assert torch.equal(m.score_tokens(x, torch.zeros(1, device=dev), x.clamp(max=3))[0].detach(), want)
    m.forward(x, torch.zeros(2, device=dev)).sum().backward()


@pytest.mark.parametrize('soft', [False, True])
def test_an_empty_batch(dev, det_sd, soft):
    """No rows: empty logits, gradients of zero, as the path without checkpoints gives; alone and as one of a chain."""
    m = _model(dev, det_sd, length=16, time_conditioning=True)
    x = torch.empty(0, 16, 5, device=dev, requires_grad=True) if soft else torch.empty(0, 16, dtype=torch.int64, device=dev)
    out = {}
    for keep in (None, 'int8'):
        lg = autograd.backbone_with_grad(m.backbone, x, torch.zeros(1, device=dev), 'bf16', keep=keep)
        assert lg.shape == (0, 16, 5)
        lg.sum().backward()
        out[keep] = _grads(m)
    assert set(out[None]) == set(out['int8'])
    assert all(bool((g == 0).all()) for g in out['int8'].values())
    if soft:
        assert x.grad.shape == x.shape
    sink, anchor = autograd.grad_chain(m.backbone)
    one = torch.randint(0, 5, (2, 16), generator=torch.Generator().manual_seed(1)).to(dev)
    z = torch.zeros(1, device=dev)
    both = [autograd.backbone_with_grad(m.backbone, s, z, 'bf16', flat=anchor, sink=sink, sigma_key=0.0, keep='int8') for s in (x, one)]
    torch.autograd.backward(both, [torch.ones_like(b) for b in both])
    got = _grads(m)
    autograd.backbone_with_grad(m.backbone, one, z, 'bf16', keep='int8').sum().backward()
    for k, g in _grads(m).items():
        assert float((g - got[k]).norm()) <= 1e-5 * float(g.norm()) + 1e-7, k
