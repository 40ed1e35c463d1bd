"""Activation checkpoints in 8 bits (drk_ln_fwd_ck8, drk_ck8_unpack, drk_ln_bwd_ck8, drk_conv_wgrad_ck8) against their
definitions in 64 bits on the CPU.

Tolerances.  Codes are the definition's own: statistics and codes are computed in fp64 on both sides, so a code could only
differ within ~1e-13 of a border, which the inputs here do not reach: equality.  fp32 results: 64 * 2^-24 of the sum of the
magnitudes of their terms (8 elements per lane and a 4-step tree, at most ~20 roundings).  Sums over rows: a lane's chain of
at most rows / 16384 + 1 rows (rows / 16 per workgroup below 16384 rows: 1), 16 in order, then 32 slab chains and a tree: 128
roundings at the sizes here.  Weight gradients: exact products, a chain of one addition per 32 rows of a chunk and per chunk."""
import math

import pytest
import torch

from drakes_amd import _lib, ops
from drakes_amd._lib import DrakesHipError

C, BLK = 128, 32
ULP = 2.0 ** -24


def quantise(x):
    """(values, scale bytes) of x [..., 128] in 64 bits; one block at a time, from the definition."""
    b = x.double().reshape(-1, BLK)
    a = b.abs().max(-1).values
    e = torch.full_like(a, -126.0)
    for _ in range(260):                                  # the smallest e >= -126 with a <= 127 * 2^e
        e = torch.where(a > 127 * torch.exp2(e), e + 1, e)
    step = torch.exp2(e).unsqueeze(-1)
    val = torch.round(b / step) * step                    # torch.round: ties to even
    bad = ~(a <= 127 * 2.0 ** 120)                        # infinities and NaN among them
    val[bad] = math.nan
    byte = torch.where(bad, torch.full_like(e, 255.0), torch.where(a == 0, torch.zeros_like(e), e + 127))
    return val.reshape(x.shape), byte.reshape(*x.shape[:-1], C // BLK)


def bits(on):
    w = 2 ** torch.arange(8)
    return (on.reshape(*on.shape[:-1], C // 8, 8).to(torch.int64) * w).sum(-1).to(torch.uint8)


def unbits(g):
    return ((g.to(torch.int64).unsqueeze(-1) >> torch.arange(8)) & 1).flatten(-2).double()


def rnd(seed, *s):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed))


def checkpoint(seed, B, L, dev, gates=True):
    """A checkpoint and its values in 64 bits."""
    x = rnd(seed, B, L, C)
    val, byte = quantise(x)
    codes = (val.reshape(B, L, C // BLK, BLK) / torch.exp2(byte - 127).unsqueeze(-1)).reshape(B, L, C).to(torch.int8)
    g = torch.randint(0, 256, (B, L, C // 8), generator=torch.Generator().manual_seed(seed + 1), dtype=torch.uint8)
    rstd = 0.5 + torch.rand(B, L, generator=torch.Generator().manual_seed(seed + 2))
    return ops.Checkpoint8(codes.to(dev), byte.to(torch.uint8).to(dev), rstd.to(dev), g.to(dev) if gates else None), val


SIZES = [(1, 1), (2, 3), (1, 17), (3, 200), (5, 333), (40, 1), (2, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize('B,L', SIZES + [(700, 200)])
@pytest.mark.parametrize('tb', ['none', 'shared', 'rows'])
@pytest.mark.parametrize('gate', ['none', 'mask', 'self'])
def test_forward(dev, B, L, tb, gate):
    feat = rnd(B * L, B, L, C) * 1.5 + 0.3
    gamma, beta = 1 + 0.2 * rnd(1, C), 0.2 * rnd(2, C)
    tbias = None if tb == 'none' else rnd(3, 1 if tb == 'shared' else B, C)
    mask = (torch.rand(B, L, C, generator=torch.Generator().manual_seed(4)) < 0.5).to(torch.uint8) if gate == 'mask' else None
    up = lambda t: None if t is None else t.to(dev)
    h, ck = ops.ln_fwd_ck8(up(feat), up(tbias), C if tb == 'rows' else 0, up(gamma), up(beta), relu_mask=up(mask), gate_self=gate == 'self')
    x = feat.double()
    if tbias is not None:
        x = x + tbias.double().unsqueeze(1)
    d = x - x.mean(-1, keepdim=True)
    r = 1 / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    x = d * r
    val, byte = quantise(x)
    assert torch.equal(ck.exps.cpu().double(), byte)
    assert torch.equal(ops.ck8_unpack(ck).cpu().double(), val)
    assert torch.equal(ops.ck8_unpack(ck, torch.bfloat16).cpu().double(), val)
    assert bool(((val - x).abs() <= torch.exp2(byte - 128).repeat_interleave(BLK, -1)).all())       # half a step
    assert float((ck.rstd.cpu().double() / r.squeeze(-1) - 1).abs().max()) <= ULP * 1.01
    want = x * gamma.double() + beta.double()
    assert bool(((h.cpu().double() - want).abs() <= want.abs() * (2.0 ** -8) * 1.0001 + 1e-30).all())
    if gate == 'none':
        assert ck.gates is None
    else:
        assert torch.equal(ck.gates.cpu(), bits(mask != 0 if gate == 'mask' else feat > 0))


@pytest.mark.gpu
@pytest.mark.parametrize('B,L', SIZES)
def test_forward_without_layernorm(dev, B, L):
    feat = rnd(B + L, B, L, C) * torch.exp2(torch.randint(-30, 30, (B, L, 1), generator=torch.Generator().manual_seed(1)).float())
    h, ck = ops.ln_fwd_ck8(feat.to(dev), None, 0, None, None, gate_self=True)
    val, byte = quantise(feat)
    assert ck.rstd is None and torch.equal(ck.exps.cpu().double(), byte)
    assert torch.equal(ops.ck8_unpack(ck).cpu().double(), val)
    assert torch.equal(h.cpu(), feat.to(torch.bfloat16)) and torch.equal(ck.gates.cpu(), bits(feat > 0))


@pytest.mark.gpu
def test_borders_and_extremes(dev):
    """Ties go to even; 127 steps still fit; zeros, subnormal, huge, infinite and NaN blocks; a constant row."""
    x = torch.zeros(1, 12, C)
    s = 2.0 ** -4
    x[0, 0, 0], x[0, 0, 1:9] = 127 * s, torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5, 3.25]) * s
    x[0, 1, 0], x[0, 1, 1:4] = 127 * s * (1 + 2.0 ** -20), torch.tensor([1.0, 3.0, 5.0]) * s       # just over: the next scale, ties in it
    x[0, 2, 32:64] = 2.0 ** -140                                                                # below half of the smallest step: zero codes
    x[0, 3, 5], x[0, 3, 6] = torch.finfo(torch.float32).max, 1e-3
    x[0, 4, 7], x[0, 5, 40], x[0, 6, 127] = math.inf, math.nan, -math.inf
    x[0, 7, :] = 5.0
    x[0, 8, 0] = 127 * 2.0 ** -126
    x[0, 9, 0] = -128 * s
    x[0, 10, ::2] = -0.0
    x[0, 11, 0] = 127 * 2.0 ** 120
    h, ck = ops.ln_fwd_ck8(x.to(dev), None, 0, None, None)
    got, (val, byte) = ops.ck8_unpack(ck).cpu().double(), quantise(x)
    assert torch.equal(ck.exps.cpu().double(), byte)
    assert torch.equal(torch.isnan(got), torch.isnan(val)) and torch.equal(got.nan_to_num(), val.nan_to_num())
    assert int(torch.isnan(got).sum()) == 4 * BLK                            # the other blocks of those rows are unharmed
    one = torch.ones(C, device=dev)
    h, ck = ops.ln_fwd_ck8(x.to(dev), None, 0, one, one)                     # with a LayerNorm: whole rows are lost, and only those
    got = ops.ck8_unpack(ck).cpu()
    assert torch.isnan(got[0, 4:7]).all() and torch.isfinite(got[0, [0, 1, 2, 3, 7, 8, 9, 10, 11]]).all()
    assert bool((got[0, 7] == 0).all()) and bool((ck.exps[0, 7] == 0).all()) and bool((h[0, 7] == 1).all())


def _ln_bwd_oracle(dh, val, rstd, gamma, gr, on):
    a = dh.double() * gamma.double()
    mean = lambda t: t.mean(-1, keepdim=True)
    r = rstd.double().unsqueeze(-1)
    dx = r * (a - mean(a) - val * mean(a * val))
    mag = r * (a.abs() + mean(a.abs()) + val.abs() * mean((a * val).abs()))
    df = dx + (0 if gr is None else gr.double())
    return dx, df, df * on, mag, mag + (0 if gr is None else gr.double().abs())


@pytest.mark.gpu
@pytest.mark.parametrize('B,L', SIZES + [(160, 200)])
@pytest.mark.parametrize('mode', ['hand_over', 'gated', 'plain', 'alias'])
def test_ln_bwd(dev, B, L, mode):
    ck, val = checkpoint(B * L + 7, B, L, dev, gates=mode != 'plain')
    dh, gr = rnd(1, B, L, C), None if mode == 'plain' else rnd(2, B, L, C)
    gamma = 1 + 0.2 * rnd(3, C)
    on = unbits(ck.gates.cpu()) if ck.gates is not None else torch.ones(B, L, C, dtype=torch.float64)
    dx, df, gated, m1, m2 = _ln_bwd_oracle(dh, val, ck.rstd.cpu(), gamma, gr, on)
    sums = torch.full((4, C), 0.5, device=dev)
    dxin = torch.empty(B, L, C, device=dev)
    dh_d, gr_d = dh.to(dev), None if gr is None else gr.to(dev)
    dfeat, dc = ops.ln_bwd_ck8(dh_d, ck, gamma.to(dev), gr_d, sums=sums, dxin=dxin, hand_over=mode in ('hand_over', 'alias'),
                               dfeat=gr_d if mode == 'alias' else None)
    near = lambda g, w, m, k=64: bool(((g.cpu().double() - w).abs() <= k * ULP * m + 1e-35).all())
    assert near(dxin, dx, m1)
    if mode in ('hand_over', 'alias'):
        assert near(dfeat, df, m2)
        assert bool(((dc.cpu().double() - gated).abs() <= gated.abs() * 2.0 ** -8 + 66 * ULP * m2).all())
        assert (mode == 'alias') == (dfeat.data_ptr() == gr_d.data_ptr())
    else:
        assert dc is None and near(dfeat, gated, m2)
    flat = lambda t: t.reshape(-1, C).sum(0)
    want = torch.stack([flat(dh.double() * val), flat(dh.double()), flat(dx), flat(gated)]) + 0.5
    size = torch.stack([flat((dh.double() * val).abs()), flat(dh.double().abs()), flat(m1), flat(m2)]) + 0.5
    assert near(sums, want, size, 256)
    again = torch.full((4, C), 0.5, device=dev)
    ops.ln_bwd_ck8(dh_d, ck, gamma.to(dev), None if gr is None else gr.to(dev), sums=again, hand_over=mode in ('hand_over', 'alias'))
    assert torch.equal(again, sums)                      # reproducible bit for bit


@pytest.mark.gpu
def test_ln_bwd_against_differences(dev):
    """The gradient of a loss through the LayerNorm, by central differences in 64 bits: what the 8 bits cost is at most the
    formula's own response to half a step of every kept value."""
    B, L = 2, 9
    feat, w, gamma = rnd(1, B, L, C), rnd(2, B, L, C), 1 + 0.2 * rnd(3, C)
    h, ck = ops.ln_fwd_ck8(feat.to(dev), None, 0, gamma.to(dev), torch.zeros(C, device=dev), gate_self=True)
    dfeat, _ = ops.ln_bwd_ck8(w.to(dev), ck, gamma.to(dev), None, hand_over=False)
    on = (feat > 0).double()
    f = lambda x: (torch.nn.functional.layer_norm(x, (C,), gamma.double(), None, 1e-5) * w.double()).sum()
    x = feat.double()
    half = torch.exp2(ck.exps.cpu().double() - 128).repeat_interleave(BLK, -1)
    a = w.double() * gamma.double()
    xh = torch.nn.functional.layer_norm(x, (C,), None, None, 1e-5)
    r = ck.rstd.cpu().double().unsqueeze(-1)
    mean = lambda t: t.mean(-1, keepdim=True)
    # d = r (a - mean a - xq mean(a xq)), xq = x^ + t, |t| <= half
    bar = r * (half * mean(a * xh).abs() + (xh.abs() + half) * mean(a.abs() * half)) + 1e-5
    for c in (0, 5, 31, 32, 77, 127):
        eps = 1e-4
        up, dn = x.clone(), x.clone()
        up[..., c] += eps
        dn[..., c] -= eps
        fu = (torch.nn.functional.layer_norm(up, (C,), gamma.double(), None, 1e-5) * w.double()).sum(-1)
        fd = (torch.nn.functional.layer_norm(dn, (C,), gamma.double(), None, 1e-5) * w.double()).sum(-1)
        slope = (fu - fd) / (2 * eps) * on[..., c]
        assert bool(((dfeat.cpu().double()[..., c] - slope).abs() <= bar[..., c]).all())


@pytest.mark.gpu
@pytest.mark.parametrize('B,L', SIZES)
def test_gate(dev, B, L):
    g = rnd(1, B, L, C)
    ck, _ = checkpoint(3, B, L, dev)
    colsum = torch.ones(C, device=dev)
    dc = ops.gate_ck8(g.to(dev), ck.gates, colsum=colsum)
    want = g * unbits(ck.gates.cpu()).float()
    assert torch.equal(dc.cpu(), want.to(torch.bfloat16))
    w = want.double().reshape(-1, C)
    assert bool(((colsum.cpu().double() - 1 - w.sum(0)).abs() <= 256 * ULP * (w.abs().sum(0) + 1)).all())


def _wgrad_oracle(h, dc, taps, dil):
    B, L, _ = h.shape
    out = torch.zeros(taps, C, C, dtype=torch.float64)
    for t in range(taps):
        off = (t - taps // 2) * dil
        lo, hi = max(0, -off), min(L, L - off)
        if hi > lo:
            out[t] = h[:, lo + off:hi + off].reshape(-1, C).t() @ dc[:, lo:hi].reshape(-1, C)
    return out


WGRAD = [(1, 1, 9, 1), (3, 7, 9, 1), (5, 33, 9, 4), (2, 200, 9, 16), (3, 200, 9, 64), (4, 77, 9, 64), (300, 5, 9, 1), (7, 64, 9, 2),
         (2, 1024, 9, 64), (1, 4097, 9, 16), (30, 200, 9, 1), (2, 40, 9, 100), (3, 500, 9, 200), (1, 1500, 9, 131), (5, 200, 1, 0), (200, 200, 1, 0), (3, 111, 3, 7),
         (2, 129, 5, 3), (4, 65, 7, 11), (2, 50, 9, 0), (150, 200, 9, 4), (2, 3, 9, 2 ** 30)]


@pytest.mark.gpu
@pytest.mark.parametrize('B,L,taps,dil', WGRAD)
@pytest.mark.parametrize('affine', [True, False])
def test_wgrad(dev, B, L, taps, dil, affine):
    ck, val = checkpoint(B + L, B, L, dev)
    gamma, beta = (1 + 0.2 * rnd(1, C), 0.5 * rnd(2, C)) if affine else (None, None)
    dc = (rnd(3, B, L, C) * (rnd(4, B, L, C) > 0)).to(torch.bfloat16)
    up = lambda t: None if t is None else t.to(dev)
    dwt = torch.full((taps, C, C), 0.25, device=dev)
    ops.conv_wgrad_ck8(ck, up(gamma), up(beta), dc.to(dev), dwt, dil)
    h = val * gamma.double() + beta.double() if affine else val
    size = (val * gamma.double()).abs() + beta.double().abs() if affine else val.abs()
    want = _wgrad_oracle(h, dc.double(), taps, dil) + 0.25
    mag = _wgrad_oracle(size, dc.double().abs(), taps, dil) + 0.25
    bar = (2 * (B * L / 32) + 256) * ULP * mag
    err = (dwt.cpu().double() - want).abs()
    assert bool((err <= bar).all()), float((err / bar).max())
    again = torch.full((taps, C, C), 0.25, device=dev)
    ops.conv_wgrad_ck8(ck, up(gamma), up(beta), dc.to(dev), again, dil)
    assert torch.equal(again, dwt)


@pytest.mark.gpu
def test_nan_in_a_checkpoint_reaches_the_gradients(dev):
    x = rnd(0, 1, 40, C)
    x[0, 7, 3] = math.nan
    _, ck = ops.ln_fwd_ck8(x.to(dev), None, 0, None, None, gate_self=True)
    dwt = torch.zeros(1, C, C, device=dev)
    ops.conv_wgrad_ck8(ck, None, None, torch.ones(1, 40, C, dtype=torch.bfloat16, device=dev), dwt, 0)
    assert torch.isnan(dwt[0, :BLK]).all() and torch.isfinite(dwt[0, BLK:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize('B,L', [(3, 77), (64, 200)])
def test_a_layer_kept_and_differentiated_in_graphs_and_streams(dev, B, L):
    """Forward, LayerNorm backward and weight gradient together, eager, on another stream and replayed from two graphs."""
    feat, gr = rnd(1, B, L, C).to(dev), rnd(2, B, L, C).to(dev)
    gamma, beta = (1 + 0.2 * rnd(3, C)).to(dev), rnd(4, C).to(dev)
    dcv = rnd(5, B, L, C).to(torch.bfloat16).to(dev)

    def layer():
        h, ck = ops.ln_fwd_ck8(feat, None, 0, gamma, beta, gate_self=True)
        dwt, sums = torch.zeros(9, C, C, device=dev), torch.zeros(4, C, device=dev)
        ops.conv_wgrad_ck8(ck, gamma, beta, dcv, dwt, 4)
        dfeat, dc = ops.ln_bwd_ck8(gr, ck, gamma, gr, sums=sums)
        return [h, *ck, dwt, sums, dfeat, dc]

    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = layer()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(layer())
    for it in range(3):
        feat.add_(0.25)
        want = layer()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.gpu
def test_rows_beyond_32_bit_offsets(dev):
    """2^24 + 5 rows: the last rows of feat lie behind 2^31 elements and 2^33 bytes."""
    L = (1 << 24) + 5
    feat = torch.zeros(1, L, C, device=dev)
    tail = rnd(1, 1, 8, C)
    feat[:, -8:] = tail.to(dev)
    h, ck = ops.ln_fwd_ck8(feat, None, 0, None, None)
    assert torch.equal(ops.ck8_unpack(ck)[:, -8:].cpu().double(), quantise(tail)[0])
    assert bool((h[:, -8:].cpu() == tail.to(torch.bfloat16)).all())
    dwt = torch.zeros(1, C, C, device=dev)
    ops.conv_wgrad_ck8(ck, None, None, h, dwt, 0)
    want = quantise(tail)[0][0].t() @ tail[0].to(torch.bfloat16).double()
    assert float((dwt[0].cpu().double() - want).abs().max()) <= 64 * ULP * 8 * 16


def test_refusals_cpu():
    z = torch.zeros(1, 4, C)
    ck = ops.Checkpoint8(torch.zeros(1, 4, C, dtype=torch.int8), torch.zeros(1, 4, 4, dtype=torch.uint8), torch.ones(1, 4), None)
    for call in (lambda: ops.ln_fwd_ck8(z, None, 0, None, None), lambda: ops.ck8_unpack(ck),
                 lambda: ops.ln_bwd_ck8(z, ck, torch.ones(C), None, hand_over=False),
                 lambda: ops.gate_ck8(z, torch.zeros(1, 4, 16, dtype=torch.uint8)),
                 lambda: ops.conv_wgrad_ck8(ck, None, None, z.to(torch.bfloat16), torch.zeros(9, C, C), 1)):
        with pytest.raises(DrakesHipError):
            call()
    lib = _lib.load()
    P = 4096                                             # never read: every call below is turned away on the host
    assert lib.drk_ln_fwd_ck8(*[None] * 2, 0, *[None] * 3, 0, *[None] * 5, 0, 5, 1, None) == 0      # an empty batch
    assert lib.drk_ln_fwd_ck8(P, None, 0, P, P, None, 0, P, P, P, None, None, 1, 5, 1, None) < 0    # LayerNorm without rstd
    assert lib.drk_ln_fwd_ck8(P, None, 0, P, P, None, 0, P, P, P, P, P, 1, 5, 1, None) < 0          # gates from nothing
    assert lib.drk_ln_fwd_ck8(P + 4, None, 0, P, P, None, 0, P, P, P, P, None, 1, 5, 1, None) < 0   # alignment
    assert lib.drk_ln_fwd_ck8(P, None, 0, P, P, None, 0, P, P, P, P, None, 1, 0, 1, None) < 0       # L = 0
    assert lib.drk_ck8_unpack(P, P, P, 2, 1, 5, None) < 0                                           # fp16
    assert lib.drk_ln_bwd_ck8(P, P, P, P, P, None, None, P, P, None, None, 1, 5, None, 0, None) < 0  # dc without gates
    assert lib.drk_ln_bwd_ck8(P, P, P, P, P, None, P, P, P, None, P, 1, 5, P, 16, None) < 0          # workspace too small
    for taps, dil in ((0, 1), (2, 1), (11, 1), (9, -1)):
        assert lib.drk_conv_wgrad_ck8(P, P, None, None, P, P, 1, 5, taps, dil, P, 1 << 40, None) < 0
    assert lib.drk_conv_wgrad_ck8(P, P, P, None, P, P, 1, 5, 9, 1, P, 1 << 40, None) < 0             # gamma without beta
    assert lib.drk_conv_wgrad_ck8(P, P, None, None, P, P, 1, 5, 9, 1, P, 1024, None) < 0             # workspace too small
    assert b'workspace' in lib.drk_last_error()


@pytest.mark.gpu
def test_refusals(dev):
    z = torch.zeros(2, 4, C, device=dev)
    one = torch.ones(C, device=dev)
    h, ck = ops.ln_fwd_ck8(z, None, 0, one, one)
    _, raw = ops.ln_fwd_ck8(z, None, 0, None, None)
    dc = z.to(torch.bfloat16)
    dwt = torch.zeros(9, C, C, device=dev)
    for err, call in [
            (ValueError, lambda: ops.ln_fwd_ck8(z[..., :64], None, 0, one, one)),
            (ValueError, lambda: ops.ln_fwd_ck8(z.transpose(0, 1), None, 0, one, one)),
            (TypeError, lambda: ops.ln_fwd_ck8(dc, None, 0, one, one)),
            (ValueError, lambda: ops.ln_fwd_ck8(z, None, 0, one, None)),
            (ValueError, lambda: ops.ln_fwd_ck8(z, one, 0, None, None)),
            (ValueError, lambda: ops.ln_fwd_ck8(z, one.view(1, C), C, one, one)),          # one row, read as one per sequence
            (ValueError, lambda: ops.ln_fwd_ck8(z, None, 0, one, one, relu_mask=torch.zeros(2, 4, C, dtype=torch.uint8, device=dev), gate_self=True)),
            (ValueError, lambda: ops.ln_fwd_ck8(z, None, 0, one[:64], one[:64])),
            (TypeError, lambda: ops.ck8_unpack(ck, torch.float16)),
            (ValueError, lambda: ops.ln_bwd_ck8(z, ck, one, None)),                        # no gates to hand over
            (ValueError, lambda: ops.ln_bwd_ck8(z, raw, one, None, hand_over=False)),      # kept without a LayerNorm
            (ValueError, lambda: ops.ln_bwd_ck8(z[:1], ck, one, None, hand_over=False)),
            (ValueError, lambda: ops.ln_bwd_ck8(z, ck, one, None, sums=torch.zeros(3, C, device=dev), hand_over=False)),
            (ValueError, lambda: ops.conv_wgrad_ck8(ck, one, None, dc, dwt, 1)),
            (ValueError, lambda: ops.conv_wgrad_ck8(ck, one, one, dc, dwt[:8], 1)),
            (ValueError, lambda: ops.conv_wgrad_ck8(ck, one, one, dc, dwt, -1)),
            (ValueError, lambda: ops.conv_wgrad_ck8(ck, one, one, dc[:1], dwt, 1)),
            (TypeError, lambda: ops.conv_wgrad_ck8(ck, one, one, z, dwt, 1)),
            (DrakesHipError, lambda: ops.ln_fwd_ck8(z.view(-1)[:0].view(0, 4, C), None, 0, one.cpu(), one.cpu()))]:
        with pytest.raises(err):
            call()
    e, eck = ops.ln_fwd_ck8(z[:0], None, 0, one, one, gate_self=True)
    assert e.shape == (0, 4, C) and ops.ck8_unpack(eck).shape == (0, 4, C)
    d, dce = ops.ln_bwd_ck8(z[:0], eck, one, None, sums=torch.zeros(4, C, device=dev))
    assert dce.shape == (0, 4, C)
    ops.conv_wgrad_ck8(eck, one, one, dc[:0], dwt, 1)
    assert float(dwt.abs().sum()) == 0


@pytest.mark.gpu
def test_a_dilation_beyond_an_int_is_refused(dev):
    _, ck = ops.ln_fwd_ck8(torch.zeros(1, 4, C, device=dev), None, 0, None, None)
    dc, dwt = torch.zeros(1, 4, C, dtype=torch.bfloat16, device=dev), torch.zeros(9, C, C, device=dev)
    for dil in (2 ** 31, 2 ** 32 + 1):
        with pytest.raises(ValueError):
            ops.conv_wgrad_ck8(ck, None, None, dc, dwt, dil)
