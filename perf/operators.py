"""Work of the operators that score given tokens and that keep activations in 8 bits for the backward pass.

  scores       drakes_amd.ops.token_scores: log-probability of a given token, entropy and the k most likely tokens of
               every row of logits, over the allowed columns and at a temperature
  scores_grad  that, and drakes_amd.ops.token_scores_bwd: the loss end of a training step
  keep         drakes_amd.ops.ln_fwd_ck8: LayerNorm in front of a convolution, its normalised input kept in 8 bits (32
               channels share a power-of-two scale) and the ReLU gates in single bits, and ck8_unpack, which reads it back
  ln_bwd       drakes_amd.ops.ln_bwd_ck8: the LayerNorm's backward from that checkpoint
  wgrad        drakes_amd.ops.conv_wgrad_ck8: the convolution's weight gradient from that checkpoint

`own` False computes them in elementary torch operations, True calls the package.
"""
import math

import torch

own = False

C = 128          # channels of a residual-stream row
BLK = 32         # channels that share one scale
EPS = 1e-5       # LayerNorm
TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def listed():
    return [
        # one 200-bp sequence, as a user scores a single design: nothing but latency
        dict(name='scores: one DNA sequence', op='scores', B=1, L=200, V=5, dtype='float32', k=0, temp=1.0, allow='vocab'),
        # a batch of protein designs, per-residue alternatives at the sampler's low temperature, mask token excluded
        dict(name='scores: protein batch', op='scores', B=64, L=257, V=22, dtype='float32', k=5, temp=0.1, allow='vocab'),
        # the last position of three running sequences over a large vocabulary
        dict(name='scores: single tokens, large V', op='scores', B=3, L=1, V=131072, dtype='bfloat16', k=8, temp=1.0, allow='none'),
        # likelihood training of the DNA denoiser at the sampling batch
        dict(name='scores_grad: DNA batch', op='scores_grad', B=1024, L=200, V=5, dtype='float32', k=0, temp=1.0, allow='vocab'),
        # a codon- or k-mer-sized vocabulary with a per-position list of allowed tokens; all outputs are trained on
        dict(name='scores_grad: mid V, masked', op='scores_grad', B=16, L=255, V=1001, dtype='float16', k=4, temp=0.7, allow='rows'),
        # a language-model head: odd vocabulary, so that most rows start off a 16-byte boundary
        dict(name='scores_grad: large odd V', op='scores_grad', B=3, L=683, V=50021, dtype='bfloat16', k=0, temp=1.0, allow='none'),
        # one sequence's layer
        dict(name='keep: one sequence', op='keep', B=1, L=200, norm=True, gate='mask', tb='shared'),
        # a layer of the long-sequence configuration at the sampling batch
        dict(name='keep: long batch', op='keep', B=512, L=1024, norm=True, gate='mask', tb='shared'),
        # fine-tune batch
        dict(name='ln_bwd: fine-tune batch', op='ln_bwd', B=32, L=200),
        dict(name='ln_bwd: long batch', op='ln_bwd', B=512, L=1024),
        dict(name='wgrad: fine-tune batch', op='wgrad', B=128, L=200, taps=9, dilation=4, affine=True),
        # the widest dilation of the model over long sequences
        dict(name='wgrad: long batch', op='wgrad', B=256, L=1024, taps=9, dilation=64, affine=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['scores', 'scores_grad', 'keep', 'ln_bwd', 'wgrad'])
    if op in ('scores', 'scores_grad'):
        V = rng.choice([5, 22, rng.randint(2, 64), _log(rng, 65, 150000), _log(rng, 65, 150000)])
        rows = _log(rng, 1, max(4, min(262144, 100_000_000 // V)))
        B = min(rows, rng.randint(1, 64))
        return dict(op=op, B=B, L=max(1, rows // B), V=V, dtype=rng.choice(sorted(TYPES)), k=min(V, rng.choice([0, 1, 4, 5, 8, 20])),
                    temp=rng.choice([1.0, 0.1, 0.8, 2.0]), allow=rng.choice(['none', 'vocab', 'rows'] if rows * V < 30_000_000 else ['none', 'vocab']))
    rows = _log(rng, 1, 524288 if op != 'wgrad' else 262144)
    L = min(rows, _log(rng, 1, 4096))
    c = dict(op=op, B=max(1, rows // L), L=L)
    if op == 'keep':
        norm = rng.random() < 0.8
        c.update(norm=norm, gate=rng.choice(['mask', 'self', 'none']), tb=rng.choice(['shared', 'rows', 'none']) if norm else 'none')
    if op == 'wgrad':
        taps = rng.choice([9, 9, 9, 1, 3])
        c.update(taps=taps, dilation=rng.choice([1, 4, 16, 64, rng.randint(1, 200)]) if taps > 1 else 0, affine=rng.random() < 0.8)
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _codes(g, B, L, dev):
    """A checkpoint as it lies in memory: normalised rows quantised block by block."""
    x = torch.randn(B, L, C, generator=g, device=dev)
    e = torch.randint(121, 123, (B, L, C // BLK), generator=g, device=dev)                 # 2^-6, 2^-5
    q = (x * torch.exp2(127.0 - e.float()).repeat_interleave(BLK, dim=-1)).round().clamp(-127, 127)
    return q.to(torch.int8), e.to(torch.uint8)


def prepare(case, seed):
    dev = torch.device('cuda', torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)
    rand = lambda *s: torch.rand(*s, generator=g, device=dev)
    B, L, op = case['B'], case['L'], case['op']
    st = dict(case=case)
    if op in ('scores', 'scores_grad'):
        V = case['V']
        # trained logits: a wide background and one column that the model is confident of
        lg = randn(B, L, V) * 2.5
        lg.scatter_add_(-1, torch.randint(0, V, (B, L, 1), generator=g, device=dev), 8 * rand(B, L, 1))
        tok = torch.randint(0, V, (B, L), generator=g, device=dev)
        st['allowed'] = None
        if case['allow'] == 'vocab':           # the mask token (last column) is no answer; its column is not looked at
            st['allowed'] = torch.arange(V, device=dev) < max(1, V - 1)
            tok = tok.clamp(max=max(0, V - 2))
        elif case['allow'] == 'rows':          # a list of allowed tokens per position, the given one among them
            st['allowed'] = (rand(B, L, V) < 0.7).scatter_(-1, tok.unsqueeze(-1), True)
            lg = torch.where(st['allowed'], lg, torch.full_like(lg, float('nan')))
        tok = torch.where(rand(B, L) < 0.1, torch.full_like(tok, -1), tok)                 # positions that are not scored
        st['logits'], st['tokens'] = lg.to(TYPES[case['dtype']]), tok
        if op == 'scores_grad':
            st['g_logp'], st['g_entropy'] = randn(B, L), 0.1 * randn(B, L)
            st['g_top'] = 0.1 * randn(B, L, case['k']) if case['k'] else None
        return st
    affine = lambda: (1 + 0.2 * randn(C), 0.2 * randn(C))
    if op == 'keep':
        st['feat'] = (randn(B, L, C) * (0.5 + rand(B, L, 1)) + 0.3 * randn(C)).clamp_(min=0.0 if case['gate'] == 'self' else -1e30)
        st['gamma'], st['beta'] = affine() if case['norm'] else (None, None)
        st['tbias'] = None if case['tb'] == 'none' else randn(1 if case['tb'] == 'shared' else B, C)
        st['mask'] = (rand(B, L, C) < 0.5).to(torch.uint8) if case['gate'] == 'mask' else None
        return st
    codes, exps = _codes(g, B, L, dev)
    st['codes'], st['exps'] = codes, exps
    if op == 'ln_bwd':
        st['gamma'] = affine()[0]
        st['rstd'] = 0.5 + rand(B, L)
        st['gates'] = torch.randint(0, 256, (B, L, C // 8), generator=g, device=dev, dtype=torch.uint8)
        st['dh'], st['g_resid'] = randn(B, L, C), randn(B, L, C)
        return st
    st['gamma'], st['beta'] = affine() if case['affine'] else (None, None)
    # output gradients behind a ReLU: half of them are zero
    st['dc'] = (randn(B, L, C) * (rand(B, L, C) < 0.5)).to(torch.bfloat16)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _scores(lg, tok, allowed, temp, k):
    """logp, entropy, top ids, top logp, and what the gradient needs."""
    V = lg.shape[-1]
    ok = torch.isneginf(lg).logical_not()
    if allowed is not None:
        ok = ok & allowed
    x = torch.where(ok, lg, torch.full_like(lg, -math.inf))
    m = x.max(-1, keepdim=True).values
    d = (x - torch.where(torch.isinf(m), torch.zeros_like(m), m)) / temp
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    lp = d - torch.log(s)
    p = torch.where(s > 0, e / s, torch.zeros_like(e))
    H = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    got = (tok >= 0) & (tok < V)
    at = tok.clamp(0, V - 1).unsqueeze(-1)
    valid = got & ok.expand_as(x).gather(-1, at).squeeze(-1)
    logp = torch.where(tok < 0, torch.zeros_like(H), torch.where(valid, lp.gather(-1, at).squeeze(-1), torch.full_like(H, -math.inf)))
    top_ids = top_lp = None
    if k:
        order = torch.sort(x, dim=-1, descending=True, stable=True)
        none = torch.isneginf(order.values[..., :k])
        top_ids = torch.where(none, torch.full_like(order.indices[..., :k], -1), order.indices[..., :k])
        top_lp = torch.where(none, torch.full_like(order.values[..., :k], -math.inf), lp.gather(-1, order.indices[..., :k]))
    return logp, H, top_ids, top_lp, lp, p, valid


def _scores_grad(lp, p, H, valid, tok, top_ids, g_logp, g_entropy, g_top, temp):
    g1 = torch.where(valid, g_logp.to(p.dtype), torch.zeros_like(H))
    hot = torch.zeros_like(p).scatter_add_(-1, tok.clamp(0, p.shape[-1] - 1).unsqueeze(-1), g1.unsqueeze(-1))
    whole = g1
    if top_ids is not None:
        gt = torch.where(top_ids >= 0, g_top.to(p.dtype), torch.zeros_like(g_top, dtype=p.dtype))
        hot.scatter_add_(-1, top_ids.clamp(min=0), gt)
        whole = whole + gt.sum(-1)
    ent = g_entropy.to(p.dtype).unsqueeze(-1) * (torch.where(p > 0, lp, torch.zeros_like(lp)) + H.unsqueeze(-1))
    return (hot - p * (whole.unsqueeze(-1) + ent)) / temp


def _decode(codes, exps, dtype):
    scale = torch.where(exps == 0, torch.zeros((), dtype=dtype, device=codes.device), torch.exp2(exps.to(dtype) - 127))
    return codes.to(dtype) * scale.repeat_interleave(BLK, dim=-1)


def _quantise(x):
    """Decoded values of x in 8 bits: the smallest power of two that keeps a block within +-127 steps, ties to even."""
    b = x.unflatten(-1, (-1, BLK))
    a = b.abs().amax(-1, keepdim=True)
    man, ex = torch.frexp(a)
    e = torch.where(man <= 127 / 128, ex - 7, ex - 6).clamp(min=-126)
    step = torch.exp2(e.to(x.dtype))
    return torch.where(a > 0, (b / step).round() * step, torch.zeros_like(b)).flatten(-2)


def _bits(on):
    w = 2 ** torch.arange(8, device=on.device)
    return (on.to(torch.int64).unflatten(-1, (-1, 8)) * w).sum(-1).to(torch.uint8)


def _on(bits):
    return ((bits.unsqueeze(-1).to(torch.int64) >> torch.arange(8, device=bits.device)) & 1).flatten(-2) != 0


def _plain(st):
    c, op = st['case'], st['case']['op']
    if op in ('scores', 'scores_grad'):
        lg = st['logits'].float()
        logp, H, ids, top, lp, p, valid = _scores(lg, st['tokens'], st['allowed'], c['temp'], c['k'])
        out = dict(logp=logp, entropy=H, ids=ids, top=top)
        if op == 'scores_grad':
            out['dlogits'] = _scores_grad(lp, p, H, valid, st['tokens'], ids, st['g_logp'], st['g_entropy'], st['g_top'],
                                          c['temp']).to(st['logits'].dtype)
        return out
    if op == 'keep':                 # in 64 bits: a value next to the border of two codes
        x = st['feat'].double()
        out = {}
        if c['norm']:
            if st['tbias'] is not None:
                x = x + st['tbias'].double().unsqueeze(1)
            mean = x.mean(-1, keepdim=True)
            rstd = torch.rsqrt((x - mean).square().mean(-1, keepdim=True) + EPS)
            x = (x - mean) * rstd
            out['h'] = (x * st['gamma'].double() + st['beta'].double()).to(torch.bfloat16)
            out['rstd'] = rstd.squeeze(-1).float()
        else:
            out['h'] = x.to(torch.bfloat16)
        out['kept'] = _quantise(x).float()
        if c['gate'] != 'none':
            out['gates'] = _bits(st['mask'] != 0 if c['gate'] == 'mask' else st['feat'] > 0)
        return out
    xq = _decode(st['codes'], st['exps'], torch.float32)
    if op == 'ln_bwd':
        a = st['dh'] * st['gamma']
        dx = st['rstd'].unsqueeze(-1) * (a - a.mean(-1, keepdim=True) - xq * (a * xq).mean(-1, keepdim=True))
        df = dx + st['g_resid']
        gated = torch.where(_on(st['gates']), df, torch.zeros_like(df))
        sums = torch.stack([(st['dh'] * xq).sum((0, 1)), st['dh'].sum((0, 1)), dx.sum((0, 1)), gated.sum((0, 1))])
        return dict(dfeat=df, dc=gated.to(torch.bfloat16), sums=sums)
    # wgrad: dw[t][ci][co] = sum over rows of h[row + off_t][ci] * dc[row][co], h = gamma * xq + beta, zero outside the sequence
    h = xq * st['gamma'] + st['beta'] if c['affine'] else xq
    L, T = c['L'], c['taps']
    at = torch.arange(L, device=h.device) + ((torch.arange(T, device=h.device) - T // 2) * c['dilation']).unsqueeze(-1)   # [T, L]
    inside = ((at >= 0) & (at < L)).unsqueeze(-1)
    win = torch.where(inside, h[:, at.clamp(0, L - 1)], torch.zeros((), device=h.device))                               # [B, T, L, C]
    G = max(1, min(c['B'], 4096 // L))         # one product over the rows of G sequences, so that no sum of 32 bits gets long
    n = -(-c['B'] // G)
    group = lambda t: torch.cat([t, t.new_zeros(n * G - c['B'], *t.shape[1:])]).unflatten(0, (n, G))
    win = group(win).permute(0, 2, 4, 1, 3).flatten(3)                                                                   # [n, T, C, G L]
    dc = group(st['dc'].float()).flatten(1, 2)                                                                           # [n, G L, C]
    return dict(dwt=torch.matmul(win, dc.unsqueeze(1)).sum(0))


def run(state):
    if not own:
        return _plain(state)
    from drakes_amd import ops
    c, op = state['case'], state['case']['op']
    if op in ('scores', 'scores_grad'):
        s = ops.token_scores(state['logits'], state['tokens'], allowed=state['allowed'], temp=c['temp'], topk=c['k'])
        out = dict(logp=s.logp, entropy=s.entropy, ids=s.top_ids, top=s.top_logp)
        if op == 'scores_grad':
            out['dlogits'] = ops.token_scores_bwd(state['logits'], state['tokens'], s, g_logp=state['g_logp'],
                                                  g_entropy=state['g_entropy'], g_top=state['g_top'],
                                                  allowed=state['allowed'], temp=c['temp'])
        return out
    if op == 'keep':
        tb = state['tbias']
        h, ck = ops.ln_fwd_ck8(state['feat'], tb, 0 if tb is None or tb.shape[0] == 1 else C, state['gamma'], state['beta'],
                               relu_mask=state['mask'], gate_self=c['gate'] == 'self')
        out = dict(h=h, kept=ops.ck8_unpack(ck))
        if c['norm']:
            out['rstd'] = ck.rstd
        if c['gate'] != 'none':
            out['gates'] = ck.gates
        return out
    if op == 'ln_bwd':
        ck = ops.Checkpoint8(state['codes'], state['exps'], state['rstd'], state['gates'])
        sums = torch.zeros(4, C, device=state['dh'].device)
        dfeat, dc = ops.ln_bwd_ck8(state['dh'], ck, state['gamma'], state['g_resid'], sums=sums)
        return dict(dfeat=dfeat, dc=dc, sums=sums)
    dwt = torch.zeros(c['taps'], C, C, device=state['dc'].device)
    ck = ops.Checkpoint8(state['codes'], state['exps'], None, None)
    ops.conv_wgrad_ck8(ck, state['gamma'], state['beta'], state['dc'], dwt, c['dilation'])
    return dict(dwt=dwt)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    c, op = case, case['op']
    if op in ('scores', 'scores_grad'):
        V, k, T = c['V'], c['k'], c['temp']
        z = st['logits'].double().flatten(0, 1)
        out_of = torch.isneginf(z)
        if st['allowed'] is not None:
            out_of = out_of | ~(st['allowed'] if st['allowed'].ndim == 1 else st['allowed'].flatten(0, 1))
        z = (z / T).masked_fill(out_of, -math.inf)
        lse = torch.logsumexp(z, -1)
        lp = (z - lse.unsqueeze(-1)).masked_fill(out_of, -math.inf)
        p = torch.exp(lp)
        H = -torch.nan_to_num(p * lp, nan=0.0).sum(-1)
        tok = st['tokens'].flatten()
        row = torch.arange(tok.numel(), device=tok.device)
        logp = torch.where(tok >= 0, lp[row, tok.clamp(min=0)], torch.zeros_like(H))
        ids = top = None
        if k:
            key = z.clone()
            ids = torch.empty(tok.numel(), k, dtype=torch.int64, device=tok.device)
            for j in range(k):                       # the first of the largest, k times
                best = key.max(-1).values
                ids[:, j] = (key == best.unsqueeze(-1)).int().argmax(-1)
                ids[:, j] = torch.where(torch.isneginf(best), torch.full_like(ids[:, j], -1), ids[:, j])
                key[row, ids[:, j].clamp(min=0)] = -math.inf
            top = lp.gather(-1, ids.clamp(min=0)).masked_fill(ids < 0, -math.inf)
        shape = lambda t: None if t is None else t.unflatten(0, (c['B'], c['L']))
        out = dict(logp=shape(logp), entropy=shape(H), ids=shape(ids), top=shape(top))
        if op == 'scores_grad':
            # d logp_t / d z_j = [j = t] - p_j, d H / d z_j = -p_j (log p_j + H)
            g1 = (st['g_logp'].double().flatten() * ((tok >= 0) & torch.isfinite(logp)))
            dz = -p * g1.unsqueeze(-1) - p * torch.nan_to_num(lp, neginf=0.0).add_(H.unsqueeze(-1)) * st['g_entropy'].double().flatten().unsqueeze(-1)
            dz[row, tok.clamp(min=0)] += g1
            for j in range(k):
                gj = st['g_top'][..., j].double().flatten() * (ids[:, j] >= 0)
                dz -= p * gj.unsqueeze(-1)
                dz[row, ids[:, j].clamp(min=0)] += gj
            out['dlogits'] = shape(dz / T)
        return out
    if op == 'keep':
        x = st['feat'].double()
        out = {}
        if c['norm']:
            if st['tbias'] is not None:
                x = x + st['tbias'].double()[:, None, :]
            mu = x.sum(-1, keepdim=True) / C
            r = 1.0 / torch.sqrt(((x - mu) ** 2).sum(-1, keepdim=True) / C + EPS)
            x = (x - mu) * r
            out['rstd'] = r[..., 0]
            out['h'] = x * st['gamma'].double() + st['beta'].double()
        else:
            out['h'] = x
        kept = torch.empty_like(x)
        for b in range(C // BLK):
            v = x[..., b * BLK:(b + 1) * BLK]
            a = v.abs().amax(-1)
            e = torch.floor(torch.log2(a.clamp(min=1e-300))) - 7            # start low, raise while the block does not fit
            for _ in range(3):
                e = torch.where(a > 127 * torch.exp2(e), e + 1, e)
            step = torch.exp2(e.clamp(min=-126)).unsqueeze(-1)
            kept[..., b * BLK:(b + 1) * BLK] = torch.round(v / step) * step
        out['kept'] = kept
        if c['gate'] != 'none':
            out['gates'] = None
        return out
    step = torch.where(st['exps'] == 0, 0.0, torch.pow(2.0, st['exps'].double() - 127))
    xq = (st['codes'].double().reshape(c['B'], c['L'], C // BLK, BLK) * step.unsqueeze(-1)).reshape(c['B'], c['L'], C)
    if op == 'ln_bwd':
        dh, gam = st['dh'].double(), st['gamma'].double()
        u = dh * gam
        dx = (u - u.sum(-1, keepdim=True) / C - xq * ((u * xq).sum(-1, keepdim=True) / C)) * st['rstd'].double()[..., None]
        df = dx + st['g_resid'].double()
        on = torch.stack([(st['gates'] >> i) & 1 for i in range(8)], -1).reshape(c['B'], c['L'], C).double()
        flat = lambda t: t.reshape(-1, C).sum(0)
        return dict(dfeat=df, dc=df * on, sums=torch.stack([flat(dh * xq), flat(dh), flat(dx), flat(df * on)]))
    h = xq * st['gamma'].double() + st['beta'].double() if c['affine'] else xq
    dc = st['dc'].double()
    out = torch.zeros(c['taps'], C, C, dtype=torch.float64, device=h.device)
    for t in range(c['taps']):
        off = (t - c['taps'] // 2) * c['dilation']
        lo, hi = max(0, -off), min(c['L'], c['L'] - off)
        if hi > lo:
            out[t] = h[:, lo + off:hi + off].reshape(-1, C).t().contiguous() @ dc[:, lo:hi].reshape(-1, C)
    return dict(dwt=out)


def work(case):
    rows, op = case['B'] * case['L'], case['op']
    if op in ('scores', 'scores_grad'):
        n, w = rows * case['V'], 4 if case['dtype'] == 'float32' else 2
        mask = {'none': 0, 'vocab': case['V'], 'rows': n}[case['allow']]
        b = n * w + mask + rows * (8 + 4 + 4 + 12 * case['k'])
        if op == 'scores_grad':                    # the gradient needs the sum over the whole row before its first element
            b += n * w + rows * (8 + 4 * case['k'])
        return dict(bytes=b, flops=(6 if op == 'scores' else 12) * n)
    if op == 'keep':
        read = 4 * C + (C if case['gate'] == 'mask' else 0)
        write = 2 * C + 4 * C + (4 if case['norm'] else 0) + (C // 8 if case['gate'] != 'none' else 0)
        return dict(bytes=rows * (read + write), flops=12 * rows * C)
    kept = C + C // BLK
    if op == 'ln_bwd':
        return dict(bytes=rows * (kept + 4 + C // 8 + 8 * C + 4 * C + 2 * C), flops=16 * rows * C)
    off = [abs(t - case['taps'] // 2) * case['dilation'] for t in range(case['taps'])]
    live = sum(max(0, case['L'] - o) for o in off)           # rows of one sequence that each tap multiplies
    return dict(bytes=rows * (kept + 2 * C) + 4 * case['taps'] * C * C, flops=2 * case['B'] * live * C * C)
