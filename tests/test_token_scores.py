"""Scores of given tokens (drk_token_scores / _bwd) against their definition in 64 bits.

Tolerances.  logp = (x - m) / T - log s: the difference, its product and log s are each rounded a few times in fp32, and s
is a sum of V terms of relative error a few 2^-24 joined pairwise over at most ~20 levels plus a thread's own chain, so an
error of 64 * 2^-24 * max(1, |value|) covers it; the exponential's argument, scaled by log2 e, adds |logp| * 2^-22 to a
single probability.  Gradients of a 16-bit type are rounded once more, by at most eps / 2 of the value."""
import math

import pytest
import torch

import drakes_amd
from drakes_amd import autograd, ops
from drakes_amd._lib import DrakesHipError

ULP = 2.0 ** -24


def oracle(lg, tok, allowed, temp, k):
    """(logp, entropy, ids, top, p) in 64 bits on the CPU, row by row as the header defines them."""
    z = lg.detach().cpu().double()
    V = z.shape[-1]
    al = torch.ones(V, dtype=torch.bool) if allowed is None else allowed.cpu().bool()
    on = al.expand(z.shape) & (z != -math.inf)
    zz = torch.where(on, z, torch.full_like(z, -math.inf)) / temp
    lse = torch.logsumexp(zz, -1, keepdim=True)
    lp = torch.where(on, zz - lse, torch.full_like(z, -math.inf))
    p = torch.where(on, lp.exp(), torch.zeros_like(z))
    H = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    t = tok.cpu()
    got = lp.gather(-1, t.clamp(0, V - 1).unsqueeze(-1)).squeeze(-1)
    logp = torch.where(t < 0, torch.zeros_like(got), torch.where(t >= V, torch.full_like(got, math.nan), got))
    ids = top = None
    if k:
        order = sorted
        flat, fon = zz.reshape(-1, V), on.reshape(-1, V)
        ids = torch.full((flat.shape[0], k), -1)
        top = torch.full((flat.shape[0], k), -math.inf, dtype=torch.float64)
        for r in range(flat.shape[0]):
            cand = torch.nonzero(fon[r]).flatten().tolist()
            best = order(cand, key=lambda j: (-float(flat[r, j]), j))[:k]
            for i, j in enumerate(best):
                ids[r, i] = j
                top[r, i] = lp.reshape(-1, V)[r, j]
        ids, top = ids.reshape(*t.shape, k), top.reshape(*t.shape, k)
    return logp, H, ids, top, lp, p


def close(got, want, what, scale=64):
    got, want = got.cpu().double(), want.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), what
    err = (got - want)[fin].abs()
    bar = scale * ULP * want[fin].abs().clamp(min=1.0)
    assert bool((err <= bar).all()), (what, float((err / bar).max()))


def case(V, rows, dtype, seed, allow, dev, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    lg = (torch.randn(*rows, V, generator=g) * spread).to(dtype)
    tok = torch.randint(0, V, rows, generator=g)
    tok[torch.rand(*rows, generator=g) < 0.15] = -1
    allowed = None
    if allow == 'vocab':
        allowed = torch.rand(V, generator=g) < 0.8
        allowed[0] = True
        lg[..., ~allowed] = math.nan                    # what stands in other columns is never looked at
    elif allow == 'rows':
        allowed = torch.rand(*rows, V, generator=g) < 0.6
        allowed.reshape(-1, V)[0] = False                # a row in which nothing counts
        lg[~allowed] = math.inf
    return lg.to(dev), tok.to(dev), None if allowed is None else allowed.to(dev)


SIZES = [(1, (3,)), (2, (1, 5)), (5, (7, 29)), (22, (3, 101)), (33, (70,)), (64, (5, 13)), (65, (9,)), (127, (4, 3)), (513, (11,)),
         (1001, (2, 6)), (2048, (5,)), (4097, (4,)), (8192, (3,)), (50021, (3,)), (131072, (2,))]


@pytest.mark.gpu
@pytest.mark.parametrize('V,rows', SIZES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('allow', ['none', 'vocab', 'rows'])
def test_scores_and_gradient(dev, V, rows, dtype, allow):
    k = min(V, (0, 1, 5, 8, 32)[(V + len(rows)) % 5])
    temp = (1.0, 0.25, 3.0)[V % 3]
    lg, tok, allowed = case(V, rows, dtype, V, allow, dev)
    s = ops.token_scores(lg, tok, allowed=allowed, temp=temp, topk=k)
    logp, H, ids, top, lp, p = oracle(lg, tok, allowed, temp, k)
    close(s.logp, logp, 'logp')
    close(s.entropy, H, 'entropy')
    if k:
        assert torch.equal(s.top_ids.cpu(), ids)
        close(s.top_logp, top, 'top')
    else:
        assert s.top_ids is None and s.top_logp is None
    g = torch.Generator().manual_seed(1)
    g1, gh = torch.randn(*rows, generator=g), torch.randn(*rows, generator=g)
    gt = torch.randn(*rows, k, generator=g) if k else None
    got = ops.token_scores_bwd(lg, tok, s, g_logp=g1.to(dev), g_entropy=gh.to(dev), g_top=gt.to(dev) if k else None,
                               allowed=allowed, temp=temp)
    assert got.dtype == dtype and got.shape == lg.shape
    t = tok.cpu()
    live = ((t >= 0) & torch.isfinite(logp)).double()
    hot = torch.zeros_like(p).scatter_add_(-1, t.clamp(min=0).unsqueeze(-1), (g1.double() * live).unsqueeze(-1))
    size = g1.abs().double()
    whole = g1.double() * live
    if k:
        gl = gt.double() * (ids >= 0)
        hot.scatter_add_(-1, ids.clamp(min=0), gl)
        whole = whole + gl.sum(-1)
        size = size + gt.abs().double().sum(-1)
    lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
    want = (hot - p * (whole.unsqueeze(-1) + gh.double().unsqueeze(-1) * (lp0 + H.unsqueeze(-1)))) / temp
    # every term: p has a relative error of (64 + 4 |logp|) ulp, the bracket that of its largest summand
    mag = (hot.abs() + p * (size.unsqueeze(-1) + gh.abs().double().unsqueeze(-1) * (lp0.abs() + H.unsqueeze(-1)))) / temp
    bar = mag * (128 + 4 * lp0.abs()) * ULP + 1e-30
    if dtype != torch.float32:
        bar = bar + want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + (2.0 ** -25 if dtype == torch.float16 else 0)  # + half a step below fp16's normal range
    err = (got.cpu().double() - want).abs()
    assert bool((err <= bar).all()), float((err / bar).max())


@pytest.mark.gpu
@pytest.mark.parametrize('V', [3, 22, 300, 5000, 70001])
def test_degenerate_rows(dev, V):
    low = torch.finfo(torch.float32).min
    lg = torch.zeros(8, V)
    lg[1] = -math.inf                                    # nothing counts
    lg[2] = low                                          # a mask of the type's lowest value everywhere: uniform
    lg[3] = low
    lg[3, V - 1] = 80.0                                  # all but one column at the lowest value
    lg[4, V // 2] = math.nan
    lg[5, V // 2] = math.inf
    lg[6, ::2] = -0.0                                    # -0 and 0 are equal: the lower index first
    lg[7] = -math.inf
    lg[7, V - 1] = 3e38
    tok = torch.full((8,), V - 1)
    k = min(V, 4)
    s = ops.token_scores(lg.to(dev), tok.to(dev), topk=k, temp=0.5)
    U = -math.log(V)
    want_lp = [U, -math.inf, U, 0.0, math.nan, math.nan, U, 0.0]
    close(s.logp, torch.tensor(want_lp, dtype=torch.float64), 'logp')
    close(s.entropy, torch.tensor([-U, 0.0, -U, 0.0, math.nan, math.nan, -U, 0.0], dtype=torch.float64), 'entropy')
    ids = s.top_ids.cpu()
    first = list(range(k))
    assert ids[0].tolist() == first and ids[2].tolist() == first and ids[6].tolist() == first
    assert ids[1].tolist() == [-1] * k and ids[7].tolist() == [V - 1] + [-1] * (k - 1)
    assert ids[3].tolist() == [V - 1] + first[:k - 1] and ids[5, 0] == V // 2
    assert V // 2 not in ids[4].tolist()
    ones = torch.ones(8, device=dev)
    d = ops.token_scores_bwd(lg.to(dev), tok.to(dev), s, g_logp=ones, g_entropy=ones, g_top=torch.ones(8, k, device=dev), temp=0.5).cpu()
    assert torch.isfinite(d[[0, 1, 2, 3, 6, 7]]).all()
    assert bool((d[1] == 0).all()) and bool((d[7] == 0).all())
    assert abs(float(d[3].sum())) < 1e-5                 # a softmax's gradient sums to nothing


@pytest.mark.gpu
@pytest.mark.parametrize('V', [70, 301, 9001])
def test_nan_and_infinity_at_the_edges_of_odd_rows(dev, V):
    """Rows that start off a 16-byte boundary: their first and last elements take a path of their own."""
    lg = torch.randn(8, V, generator=torch.Generator().manual_seed(V)).to(torch.bfloat16)
    for r in range(4):
        lg[r, 0], lg[r + 4, V - 1] = (math.nan, math.inf, -math.inf, 40.0)[r], (math.nan, math.inf, -math.inf, 40.0)[r]
    tok = torch.full((8,), V // 3)
    s = ops.token_scores(lg.to(dev), tok.to(dev), topk=3)
    logp, H, ids, top, _, _ = oracle(lg, tok, None, 1.0, 3)
    good = [2, 3, 6, 7]
    close(s.logp[good], logp[good], 'logp')
    close(s.entropy[good], H[good], 'entropy')
    assert torch.equal(s.top_ids.cpu()[good], ids[good])
    assert torch.isnan(s.logp.cpu()[[0, 1, 4, 5]]).all() and torch.isnan(s.entropy.cpu()[[0, 1, 4, 5]]).all()
    clean = torch.where(torch.isnan(lg), torch.full_like(lg, -math.inf), lg)          # NaN is no alternative, an infinity is the first
    assert torch.equal(s.top_ids.cpu(), oracle(torch.where(clean == math.inf, torch.full_like(clean, 1e30), clean), tok, None, 1.0, 3)[2])


@pytest.mark.gpu
def test_tokens_outside_and_unscored(dev):
    lg = torch.randn(4, 9, generator=torch.Generator().manual_seed(0)).to(dev)
    allowed = torch.ones(9, dtype=torch.bool, device=dev)
    allowed[3] = False
    tok = torch.tensor([-5, 9, 3, 2 ** 40], device=dev)
    s = ops.token_scores(lg, tok, allowed=allowed)
    lp = s.logp.cpu()
    assert lp[0] == 0 and torch.isnan(lp[1]) and lp[2] == -math.inf and torch.isnan(lp[3])
    d = ops.token_scores_bwd(lg, tok, s, g_logp=torch.ones(4, device=dev), allowed=allowed)
    assert bool((d == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize('V,wide,off', [(5, 8, 0), (21, 22, 1), (50, 64, 7), (1000, 1024, 3), (30000, 30011, 5)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_slices_of_wider_rows(dev, V, wide, off, dtype):
    """A padded vocabulary: the columns outside hold NaN; rows of one batch repeated by expand()."""
    big = torch.full((6, wide), math.nan)
    big[:, off:off + V] = torch.randn(6, V, generator=torch.Generator().manual_seed(V))
    big = big.to(dtype).to(dev)
    lg = big[:, off:off + V]
    tok = torch.arange(6, device=dev) % V
    a, b = ops.token_scores(lg, tok, topk=min(V, 5)), ops.token_scores(lg.contiguous(), tok, topk=min(V, 5))
    close(a.logp, b.logp.cpu(), 'logp', 128)
    close(a.entropy, b.entropy.cpu(), 'entropy', 128)
    assert torch.equal(a.top_ids, b.top_ids)
    g = torch.ones(6, device=dev)
    da, db = (ops.token_scores_bwd(x, tok, s, g_logp=g) for x, s in ((lg, a), (lg.contiguous(), b)))
    assert da.is_contiguous() and torch.isfinite(da.float()).all()
    # two orders of one sum: each side rounds to the type once, so a step of it may lie between them
    assert float((da.float() - db.float()).abs().max()) <= 256 * ULP + 2 * torch.finfo(dtype).eps
    e = lg[:1].expand(6, V)
    s = ops.token_scores(e, tok)
    close(s.entropy, a.entropy[:1].expand(6).cpu(), 'expanded', 128)


@pytest.mark.gpu
@pytest.mark.parametrize('rows,V', [(3, 131072), (513, 300), (40000, 5)])
def test_same_bits_twice_and_in_a_graph(dev, rows, V):
    lg, tok, _ = case(V, (rows,), torch.bfloat16, 3, 'none', dev)
    k = min(V, 6)
    ref = ops.token_scores(lg, tok, topk=k)
    g1 = torch.randn(rows, generator=torch.Generator().manual_seed(5)).to(dev)
    dref = ops.token_scores_bwd(lg, tok, ref, g_logp=g1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                       # another stream than the inputs' own
        s2 = ops.token_scores(lg, tok, topk=k)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, s2))
    x = lg.clone()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for gr in graphs:                                   # two captured graphs, replayed in turn
        with torch.cuda.graph(gr):
            s = ops.token_scores(x, tok, topk=k)
            outs.append((s, ops.token_scores_bwd(x, tok, s, g_logp=g1)))
    for it in range(3):
        x.copy_(lg if it != 1 else lg.roll(1, 0))
        want = ops.token_scores(x, tok, topk=k)
        dwant = ops.token_scores_bwd(x, tok, want, g_logp=g1)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for s, d in outs:
            assert all(torch.equal(a, b) for a, b in zip(s, want)) and torch.equal(d, dwant)
    assert torch.equal(dref, ops.token_scores_bwd(lg, tok, ref, g_logp=g1))


@pytest.mark.gpu
def test_rows_beyond_32_bit_offsets(dev):
    """3000 rows of 2^20 logits: the last rows lie behind 2^32 bytes and 2^31 elements."""
    V = 1 << 20
    lg = torch.zeros(3000, V, dtype=torch.bfloat16, device=dev)
    lg[-1] = torch.arange(V, device=dev, dtype=torch.float32).to(torch.bfloat16) / V
    tok = torch.zeros(3000, dtype=torch.int64, device=dev)
    tok[-1] = V - 1
    s = ops.token_scores(lg, tok, topk=1)
    logp, H, ids, top, _, _ = oracle(lg[-1:], tok[-1:], None, 1.0, 0)
    close(s.logp[-1:], logp, 'logp')
    close(s.entropy[-1:], H, 'entropy')
    assert float(s.logp[0]) == pytest.approx(-math.log(V), abs=1e-4)
    assert int(s.top_ids[0]) == 0 and int(s.top_ids[-1]) == int((lg[-1] == lg[-1].max()).int().argmax())
    d = ops.token_scores_bwd(lg, tok, s, g_logp=torch.ones(3000, device=dev), out=lg)      # in place
    assert float(d[-1, V - 1]) == pytest.approx(1.0, abs=1e-2) and float(d[5, 0]) == pytest.approx(1.0, abs=1e-2)


@pytest.mark.gpu
def test_wider_lists_through_the_c_abi(dev):
    """A per-row list whose rows are longer than V."""
    import ctypes
    from drakes_amd import _lib
    for V, wide in ((7, 12), (50, 64), (200, 333)):
        lg = torch.randn(70, V, generator=torch.Generator().manual_seed(V)).to(dev)
        tok = torch.zeros(70, dtype=torch.int64, device=dev)
        big = torch.zeros(70, wide, dtype=torch.uint8)
        big[:, :V] = torch.rand(70, V, generator=torch.Generator().manual_seed(1)) < 0.5
        ref = ops.token_scores(lg, tok, allowed=big[:, :V].contiguous().to(dev))
        wide_list = big.to(dev)
        logp, stats = torch.empty(70, device=dev), torch.empty(70, 2, device=dev)
        P = lambda t: ctypes.c_void_p(t.data_ptr())
        _lib.call('drk_token_scores', P(lg), 0, V, P(tok), P(wide_list), wide, 1.0, 0, P(logp), None, None, None, P(stats), 70, V, None, 0,
                  ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert torch.equal(logp, ref.logp) and torch.equal(stats, ref.stats)


@pytest.mark.gpu
def test_one_row_without_batch_dimensions(dev):
    lg = torch.randn(30, generator=torch.Generator().manual_seed(1)).to(dev)
    allowed = torch.arange(30, device=dev) != 4
    s = ops.token_scores(lg, torch.tensor(7, device=dev), allowed=allowed, topk=2)
    logp, H, ids, top, _, _ = oracle(lg.unsqueeze(0), torch.tensor([7]), allowed, 1.0, 2)
    assert s.logp.shape == () and s.top_ids.shape == (2,)
    close(s.logp.unsqueeze(0), logp, 'logp')
    assert torch.equal(s.top_ids.cpu(), ids[0])


@pytest.mark.gpu
def test_calls_at_once_on_two_streams(dev):
    """Split rows and whole ones, forward and backward, on two streams without an order between them."""
    a, ta, _ = case(70000, (4,), torch.float32, 1, 'none', dev)
    b, tb, _ = case(70000, (4,), torch.float32, 2, 'none', dev)
    g = torch.ones(4, device=dev)
    run = lambda x, t: (lambda s: [*s, ops.token_scores_bwd(x, t, s, g_logp=g)])(ops.token_scores(x, t, topk=7))
    wa, wb = run(a, ta), run(b, tb)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for s in (s1, s2):
            s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s1):
            ra = run(a, ta)
        with torch.cuda.stream(s2):
            rb = run(b, tb)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(ra, wa)) and all(torch.equal(x, y) for x, y in zip(rb, wb))


@pytest.mark.gpu
def test_another_device_is_refused(dev, monkeypatch):
    lg, tok = torch.zeros(2, 5, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    z = torch.zeros(1, 4, 128, device=dev)
    monkeypatch.setattr(ops, '_current', lambda: (1, 0))          # as if another GPU were the current one; nothing is launched
    with pytest.raises(ValueError, match='current device'):
        ops.token_scores(lg, tok)
    with pytest.raises(ValueError, match='current device'):
        ops.ln_fwd_ck8(z, None, 0, None, None)


def test_refusals_cpu():
    lg, tok = torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(DrakesHipError):
        ops.token_scores(lg, tok)
    with pytest.raises(DrakesHipError):
        ops.token_scores_bwd(lg, tok, ops.TokenScores(None, None, None, None, torch.zeros(2, 2)))
    lib = drakes_amd._lib.load()
    ok = dict(dtype=0, stride=5, ast=0, temp=1.0, k=0, rows=2, V=5)
    def rc(**kw):
        a = {**ok, **kw}
        return lib.drk_token_scores(None, a['dtype'], a['stride'], None, None, a['ast'], a['temp'], a['k'], None, None, None, None,
                                    None, a['rows'], a['V'], None, 0, None)
    assert rc(rows=0) == 0                              # an empty batch is a no-op, whatever its pointers
    for bad in (dict(), dict(V=0), dict(rows=-1), dict(temp=0.0), dict(temp=-1.0), dict(temp=math.inf), dict(temp=math.nan),
                dict(temp=1e-45), dict(k=6), dict(k=-1), dict(k=33, V=100), dict(ast=3), dict(stride=-1)):
        assert rc(**bad) < 0, bad
        assert b'drk_token_scores' in lib.drk_last_error()


@pytest.mark.gpu
def test_refusals(dev):
    lg, tok = torch.zeros(2, 3, 5, device=dev), torch.zeros(2, 3, dtype=torch.int64, device=dev)
    s = ops.token_scores(lg, tok)
    for err, call in [
            (TypeError, lambda: ops.token_scores(lg.double(), tok)),
            (TypeError, lambda: ops.token_scores(lg, tok.int())),
            (TypeError, lambda: ops.token_scores(lg, tok, allowed=torch.ones(5, device=dev))),
            (ValueError, lambda: ops.token_scores(lg, tok[:1])),
            (ValueError, lambda: ops.token_scores(lg.transpose(1, 2), torch.zeros(2, 5, dtype=torch.int64, device=dev))),
            (ValueError, lambda: ops.token_scores(lg, tok, allowed=torch.ones(4, dtype=torch.bool, device=dev))),
            (ValueError, lambda: ops.token_scores(lg, tok, topk=6)),
            (ValueError, lambda: ops.token_scores(lg, tok, temp=0.0)),
            (ValueError, lambda: ops.token_scores(lg, tok, temp=math.nan)),
            (DrakesHipError, lambda: ops.token_scores(lg, tok.cpu())),
            (ValueError, lambda: ops.token_scores_bwd(lg, tok, s, g_logp=torch.zeros(2, device=dev))),
            (ValueError, lambda: ops.token_scores_bwd(lg, tok, s, g_top=torch.zeros(2, 3, 1, device=dev))),
            (ValueError, lambda: ops.token_scores_bwd(lg, tok, ops.token_scores(lg, tok, entropy=False), g_entropy=torch.zeros(2, 3, device=dev))),
            (ValueError, lambda: ops.token_scores(torch.zeros(4, 3, 8, device=dev)[::2, :, :5].transpose(0, 1), torch.zeros(3, 2, dtype=torch.int64, device=dev)))]:
        with pytest.raises(err):
            call()
    e = ops.token_scores(lg[:0], tok[:0], topk=2)
    assert e.logp.shape == (0, 3) and e.top_ids.shape == (0, 3, 2)
    assert ops.token_scores_bwd(lg[:0], tok[:0], e).shape == (0, 3, 5)


# ---------------------------------------------------------------------------------------- the framework's own callers
def _loss(logp, H, top):
    return (1.3 * logp).sum() + (0.7 * H).sum() + (top * torch.arange(1, top.shape[-1] + 1, device=top.device)).sum()


@pytest.mark.gpu
def test_autograd_formula_and_differences(dev):
    """One loss through all outputs: its gradient against the formula's in 64 bits and against central differences."""
    g = torch.Generator().manual_seed(2)
    lg = torch.randn(2, 7, 22, generator=g)
    tok = torch.randint(0, 21, (2, 7), generator=g)
    allowed = torch.arange(22) != 21
    x = lg.to(dev).requires_grad_()
    logp, H, ids, top = autograd.token_scores_with_grad(x, tok.to(dev), allowed=allowed.to(dev), temp=0.8, topk=3)
    assert not ids.requires_grad
    _loss(logp, H, top).backward()
    z = lg.double().requires_grad_()
    lp = torch.log_softmax((z / 0.8)[..., :21], -1)
    Hd = -(lp.exp() * lp).sum(-1)
    want_loss = _loss(lp.gather(-1, tok.unsqueeze(-1)).squeeze(-1), Hd, lp.gather(-1, ids.cpu()))
    want, = torch.autograd.grad(want_loss, z)
    # |terms| below 10 per element, each within 200 * 2^-24 of itself
    assert float((x.grad.cpu().double() - want).abs().max()) < 2000 * ULP * 10
    v = torch.randn(2, 7, 22, generator=g)
    h = 2.0 ** -6
    def f(s):                                            # the alternatives stay those of the centre: where two of them change
        y = (lg + s * h * v).to(dev)                     # places the sorted outputs have a kink, and no derivative
        kw = dict(allowed=allowed.to(dev), temp=0.8)
        lp_t, Ht = autograd.token_scores_with_grad(y, tok.to(dev), **kw)[:2]
        top_t = torch.stack([autograd.token_scores_with_grad(y, ids[..., i].contiguous(), **kw)[0] for i in range(3)], -1)
        return _loss(lp_t.double(), Ht.double(), top_t.double())
    slope = float((f(1) - f(-1)) / (2 * h))
    # the difference's error: h^2 / 6 of a third derivative (14 rows, cubes of v / temp) and rounding over 2 h
    assert abs(slope - float((x.grad.cpu() * v).sum())) < 0.02 * max(1.0, abs(slope)) + 0.05


@pytest.mark.gpu
def test_autograd_broadcast_and_partial_gradients(dev):
    """expand()ed logits sum their gradients; an output that no loss reads passes none."""
    x = torch.randn(1, 300, device=dev, requires_grad=True)
    tok = torch.arange(6, device=dev)
    logp, H, ids, top = autograd.token_scores_with_grad(x.expand(6, 300), tok)
    assert ids is None and top is None
    logp.sum().backward()
    lp = torch.log_softmax(x.detach().double(), -1)
    want = -6 * lp.exp()
    want[0, :6] += 1
    assert float((x.grad.double() - want).abs().max()) < 6 * 300 * ULP
    x.grad = None
    autograd.token_scores_with_grad(x.expand(6, 300), tok)[1].sum().backward()
    Hd = -(lp.exp() * lp).sum()
    assert float((x.grad.double() + 6 * lp.exp() * (lp + Hd)).abs().max()) < 6 * 1000 * ULP


@pytest.mark.gpu
def test_diffusion_score_tokens(dev, gpu_model):
    """Scores equal the SUBS log-probabilities at masked positions, and train the denoiser."""
    m = gpu_model
    g = torch.Generator().manual_seed(4)
    x = torch.randint(0, 5, (3, 200), generator=g).to(dev)
    tgt = torch.randint(0, 4, (3, 200), generator=g).to(dev)
    sig = torch.zeros(3, device=dev)
    with torch.no_grad():
        logp, H, ids, top = m.score_tokens(x, sig, tgt, topk=4)
        subs = m.forward(torch.full_like(x, 4), sig)                     # all masked: the raw distribution everywhere
        lp2, _, _, _ = m.score_tokens(torch.full_like(x, 4), sig, tgt)
    assert float((lp2 - subs.gather(-1, tgt.unsqueeze(-1)).squeeze(-1)).abs().max()) < 256 * ULP * 16
    assert torch.equal(ids.sort(-1).values, torch.arange(4, device=dev).expand(3, 200, 4))
    assert float((top.double().exp().sum(-1) - 1).abs().max()) < 1e-5
    m.zero_grad()
    only = torch.where(x == 4, tgt, torch.full_like(tgt, -1))
    logp = m.score_tokens(x, sig, only)[0]
    assert bool((logp[x != 4] == 0).all())
    (-logp.sum()).backward()
    gw = {k: p.grad.clone() for k, p in m.backbone.named_parameters() if p.grad is not None}
    m.zero_grad()
    lg = m.backbone(x, sig[:1])
    sub = autograd.subs_with_grad(lg, x)
    (-(sub.gather(-1, tgt.unsqueeze(-1)).squeeze(-1) * (x == 4)).sum()).backward()     # the same loss through SUBS
    for k, p in m.backbone.named_parameters():
        if p.grad is not None:
            assert float((gw[k] - p.grad).norm()) <= 2e-4 * float(p.grad.norm()) + 1e-6, k
    m.zero_grad(set_to_none=True)


@pytest.mark.gpu
def test_interpolant_score_tokens(dev):
    from types import SimpleNamespace as NS
    from drakes_amd.protein import Interpolant
    W = torch.randn(22, 22, generator=torch.Generator().manual_seed(3)).to(dev).to(torch.bfloat16).requires_grad_()
    it = Interpolant(NS(num_timesteps=10, min_t=0.01, temp=0.1, interpolant_type='masking'))
    aa = torch.randint(0, 22, (2, 31), generator=torch.Generator().manual_seed(1)).to(dev)
    tgt = torch.randint(0, 21, (2, 31), generator=torch.Generator().manual_seed(2)).to(dev)
    mask = torch.ones(2, 31, device=dev)
    mask[1, 20:] = 0                                                     # a padded batch
    model = lambda X, S, *a: W[S]
    no_c = torch.arange(22, device=dev) != 1
    logp, H, ids, top = it.score_tokens(model, None, aa, tgt, mask, mask, None, None, topk=5, allowed=no_c)
    assert bool((logp[1, 20:] == 0).all()) and not bool(((ids == 21) | (ids == 1)).any())
    logp[torch.isfinite(logp)].sum().backward()
    assert torch.isfinite(W.grad.float()).all() and float(W.grad[:, [1, 21]].abs().sum()) == 0


@pytest.mark.gpu
def test_more_rows_than_one_launch_holds(dev):
    """2^26 + 3 rows of one wave each: more than 2^32 threads."""
    rows, V = (1 << 26) + 3, 65
    lg = torch.zeros(rows, V, dtype=torch.bfloat16, device=dev)
    at = torch.tensor([0, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, rows - 2, rows - 1])       # (a launch takes 2^24 - 1 rows)
    lg[at.to(dev)] = torch.randn(6, V, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    part = lg[at.to(dev)]
    tok = torch.full((rows,), 7, dtype=torch.int64, device=dev)
    s = ops.token_scores(lg, tok, topk=1)
    logp, H, ids, top, _, p = oracle(part, tok[:6], None, 1.0, 1)
    close(s.logp[at.to(dev)], logp, 'logp')
    close(s.entropy[at.to(dev)], H, 'entropy')
    assert torch.equal(s.top_ids[at.to(dev)].cpu(), ids)
    assert bool((s.stats[:, 1] > 0).all())                                                  # no row left out
    d = ops.token_scores_bwd(lg, tok, s, g_logp=torch.ones(rows, device=dev), out=lg)
    want = -p
    want[:, 7] += 1
    bar = torch.finfo(torch.bfloat16).eps / 2 * want.abs() + 256 * ULP
    assert bool(((d[at.to(dev)].cpu().double() - want).abs() <= bar).all())
    assert bool((d[:, 7] > 0).all())


@pytest.mark.gpu
def test_diffusion_score_tokens_keeps_no_tensor(dev, gpu_model):
    """A tensor made by one call (on its stream, or inside its capture) is not another call's input."""
    x = torch.full((1, 200), 4, dtype=torch.int64, device=dev)
    held = set(vars(gpu_model))
    with torch.no_grad():
        gpu_model.score_tokens(x, torch.zeros(1, device=dev), x.clamp(max=3))
    assert not [k for k in set(vars(gpu_model)) - held if isinstance(vars(gpu_model)[k], torch.Tensor)]


@pytest.mark.gpu
def test_interpolant_score_tokens_of_transposed_inputs(dev):
    from types import SimpleNamespace as NS
    from drakes_amd.protein import Interpolant
    lg = torch.randn(31, 2, 22, generator=torch.Generator().manual_seed(3)).to(dev)
    it = Interpolant(NS(num_timesteps=10, min_t=0.01, temp=0.5, interpolant_type='masking'))
    tgt = torch.randint(0, 21, (31, 2), generator=torch.Generator().manual_seed(2)).to(dev)
    mask = torch.ones(31, 2, device=dev)
    mask[20:, 1] = 0
    allowed = torch.full((22,), 2, dtype=torch.uint8, device=dev)
    allowed[1] = 0
    model = lambda X, S, *a: lg.transpose(0, 1)
    logp, H, ids, _ = it.score_tokens(model, None, None, tgt.t(), mask.t(), None, None, None, topk=2, allowed=allowed)
    on = allowed.cpu() != 0
    on[21] = False
    want = oracle(lg.transpose(0, 1), torch.where(mask != 0, tgt, torch.full_like(tgt, -1)).t(), on, 0.5, 2)
    close(logp, want[0], 'logp')
    close(H, want[1], 'entropy')
    assert torch.equal(ids.cpu(), want[2])
