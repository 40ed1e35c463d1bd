"""The convolution weight gradient from 8-bit checkpoints at the sizes where all taps run in one workgroup, and on both sides of
the rule that chooses between its two kernels, against the definition in 64 bits (tolerance: as for the smaller sizes in
test_ck8.py, exact products and one addition per 32 rows of a chunk and per chunk).

Which kernel a call takes shows in the workspace that it asks for: one slab of 129 x 128 floats per tap and chunk of rows, with
at most 64 chunks where all taps share a workgroup and 512 / (2 taps) where they do not."""
import math

import pytest
import torch

from drakes_amd import _lib, ops
from test_ck8 import C, ULP, _wgrad_oracle, checkpoint, rnd


def kernel_of(B, L, taps, dil):
    slab = 4 * taps * (C + 1) * C
    chunks = _lib.load().drk_conv_wgrad_ck8_workspace_bytes(B, L, taps, dil) / slab
    tiles = -(-B * L // 64)
    cut = lambda most: -(-tiles // -(-tiles // most))
    ring, tap = cut(64), cut(512 // (2 * taps))
    assert ring != tap and chunks in (ring, tap)
    return 'ring' if chunks == ring else 'tap'


# lengths and shifts that are multiples of 32 (a step is all in or all out), the model's other dilations at its two lengths, the
# widest shift that a ring holds, sequences shorter than a step, odd lengths, fewer taps, no shift, and every ring size
RING = [(13, 1024, 9, 64), (13, 1024, 9, 16), (26, 512, 9, 32), (65, 200, 9, 16), (70, 200, 9, 64), (65, 200, 9, 1), (2600, 5, 9, 1),
        (13, 1001, 9, 104), (13001, 1, 3, 7), (130, 101, 5, 3), (130, 101, 7, 11), (65, 200, 9, 0), (410, 32, 9, 32), (1, 12800, 3, 416),
        (7, 1999, 5, 208), (430, 31, 9, 8)]


def test_the_ring_shapes_take_the_ring():
    for s in RING:
        assert kernel_of(*s) == 'ring', s
    for s in ((32, 200, 9, 64), (63, 200, 9, 4), (13, 1024, 9, 105), (7, 1999, 5, 209), (70, 200, 1, 0)):
        assert kernel_of(*s) == 'tap', s


@pytest.mark.gpu
@pytest.mark.parametrize('B,L,taps,dil', RING)
@pytest.mark.parametrize('affine', [True, False])
def test_ring(dev, B, L, taps, dil, affine):
    assert kernel_of(B, L, taps, dil) == 'ring'
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
@pytest.mark.parametrize('B,L,taps,dil', [(32, 200, 9, 64), (70, 200, 9, 64), (63, 200, 9, 16), (65, 200, 9, 16), (3, 33, 9, 4), (2, 7, 9, 9),
                                          (1, 1, 3, 1), (2, 1024, 9, 64), (13, 1024, 9, 105), (5, 40, 1, 0)])
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
def test_a_nan_or_an_infinity_in_dc_reaches_every_tap(dev, B, L, taps, dil, bad):
    """As where h is padded with zeros: the row meets a zero in a tap that leaves its sequence.  Whichever kernel runs."""
    ck, _ = checkpoint(B + L, B, L, dev)
    gamma, beta = (1 + 0.2 * rnd(1, C)).to(dev), (0.5 * rnd(2, C)).to(dev)
    dc = (rnd(3, B, L, C) * (rnd(4, B, L, C) > 0)).to(torch.bfloat16)
    at = [(0, 0, 0), (B // 2, L // 2, 77), (B - 1, L - 1, 127), (B - 1, 0, 6)]
    cols = [c for _, _, c in at]
    out = []
    for v in (0.0, bad):
        for b, l, c in at:
            dc[b, l, c] = v
        dwt = torch.zeros(taps, C, C, device=dev)
        ops.conv_wgrad_ck8(ck, gamma, beta, dc.to(dev), dwt, dil)
        out.append(dwt.cpu())
    clean, got = out
    assert torch.isfinite(clean).all()
    assert not torch.isfinite(got[:, :, cols]).any(), [(t, c) for t in range(taps) for c in cols if torch.isfinite(got[t, :, c]).any()]
    rest = [c for c in range(C) if c not in cols]
    assert torch.equal(got[:, :, rest], clean[:, :, rest])
