"""Timing cases of the differential-attention block's operators (mep_amd.diff_block): rotary positions, the norms
before and after a block with its gate and residual scale, and differential attention, in both directions.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, angles in 64, one rounding at the
end), or, with ``own`` set, through mep_amd.diff_block.  ``exact`` computes it in 64 bits with torch's own autograd.

What the cases stand for:
  rotary_train_cmu      rotating the queries and keys of the B = 64, T = 50 encoder (12 half heads of 8) each step
  rotary_decode         one new token per sequence at far positions of a scaled context: latency
  rotary_prefill        a long batch, half of each head rotated
  norm_heads            the norm of each head's output row (short rows, many of them)
  residual_train_cmu    post-norm + gate + residual + next pre-norm at D = 96, B = 64, T = 50, fp32
  residual_train_large  the same joint of a wide bf16 model with a gate per sequence, both directions
  residual_odd          rows of an odd width, no vector access possible
  attn_train_cmu        the B = 64, T = 50, D = 96 encoder's attention step under the loader's key mask, fp32
  attn_train_ren        the 32-row, T = 300, D = 128 encoder's attention step, bf16
  attn_train_long       a causal training step over 4096 tokens, bf16
  attn_prefill          a causal prompt of 8192 tokens with shared key heads, bf16
  attn_decode           single tokens against ragged caches of up to 8192 keys, shared key heads, fp16
"""
import math

import torch

own = False

TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
EPS = 1e-5


# ------------------------------------------------------------------ cases
def _rotary(**k):
    return dict(dict(op='rotary', B=1, T=1, H=1, G=1, D=64, rot=64, layout='half', dtype='bfloat16', bwd=False,
                     base=10000.0, scaling='none', factor=1.0, first=0), **k)


def _norm(**k):
    return dict(dict(op='norm', B=1, T=1, D=64, kind='rms', bias=False, dtype='bfloat16', wtype='float32', bwd=False), **k)


def _residual(**k):
    return dict(dict(op='residual', B=1, T=1, D=64, kind='rms', next_kind='rms', bias=False, gate='channel', learned=False,
                     scale=1.0, dtype='bfloat16', wtype='float32', bwd=False), **k)


def _attn(**k):
    return dict(dict(op='attn', B=1, Tq=1, Tk=1, H=1, G=1, d=64, dv=128, dtype='bfloat16', causal=False, mask='none',
                     ragged=False, lam='head', bwd=False), **k)


def listed():
    return [
        _rotary(name='rotary_train_cmu', B=64, T=50, H=12, G=12, D=8, rot=8, dtype='float32', bwd=True),
        _rotary(name='rotary_decode', B=32, T=1, H=32, G=8, D=128, rot=128, layout='interleaved', scaling='parts',
                factor=8.0, first=40000),
        _rotary(name='rotary_prefill', B=4, T=8192, H=16, G=4, D=128, rot=64, scaling='ntk', factor=4.0, bwd=True),
        _norm(name='norm_heads', B=2, T=4096 * 8, D=128, bwd=True),
        _residual(name='residual_train_cmu', B=64, T=50, D=96, kind='layer', next_kind='layer', bias=True, learned=True,
                  dtype='float32', bwd=True),
        _residual(name='residual_train_large', B=8, T=2048, D=4096, gate='sequence', scale=0.7, bwd=True),
        _residual(name='residual_odd', B=3, T=1111, D=1537, kind='layer', gate='full', dtype='float16', wtype='float16',
                  bwd=True),
        _attn(name='attn_train_cmu', B=64, Tq=50, Tk=50, H=3, G=3, d=16, dv=32, dtype='float32', mask='keys', bwd=True),
        _attn(name='attn_train_ren', B=32, Tq=300, Tk=300, H=4, G=4, d=16, dv=32, mask='keys', bwd=True),
        _attn(name='attn_train_long', B=2, Tq=4096, Tk=4096, H=8, G=8, d=64, dv=128, causal=True, bwd=True),
        _attn(name='attn_prefill', B=1, Tq=8192, Tk=8192, H=16, G=4, d=64, dv=128, causal=True),
        _attn(name='attn_decode', B=32, Tq=1, Tk=8192, H=16, G=4, d=64, dv=128, dtype='float16', ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(['float32', 'bfloat16', 'bfloat16', 'float16'])
    op = rng.choice(['rotary', 'norm', 'residual', 'attn', 'attn', 'attn'])
    bwd = rng.random() < 0.6
    wtype = rng.choice(['float32', dtype])
    if op == 'rotary':
        D = rng.choice([8, 16, 32, 64, 80, 96, 128, 256])
        H = _log(rng, 1, 32)
        G = rng.choice([g for g in range(1, H + 1) if H % g == 0])
        T = 1 if rng.random() < 0.25 else _log(rng, 1, 8192)
        B = max(1, min(_log(rng, 1, 64), 32 * 1024 * 1024 // (T * (H + G) * D)))
        return _rotary(B=B, T=T, H=H, G=G, D=D, rot=D if rng.random() < 0.5 else 2 * rng.randint(2, D // 2),
                       layout=rng.choice(['half', 'interleaved']), dtype=dtype, bwd=bwd, base=rng.choice([1e4, 5e5]),
                       scaling=rng.choice(['none', 'linear', 'ntk', 'parts']), factor=rng.choice([2.0, 4.0, 8.0]),
                       first=rng.choice([0, 17, 30000]))
    if op == 'norm':
        D = _log(rng, 8, 8192)
        T = _log(rng, 1, 65536)
        B = _log(rng, 1, 64)
        T = max(1, min(T, 32 * 1024 * 1024 // (B * D)))
        return _norm(B=B, T=T, D=D, kind=rng.choice(['rms', 'layer']), bias=rng.random() < 0.5, dtype=dtype, wtype=wtype, bwd=bwd)
    if op == 'residual':
        D = _log(rng, 8, 8192)
        B = _log(rng, 1, 64)
        T = max(1, min(_log(rng, 1, 16384), 32 * 1024 * 1024 // (B * D)))
        return _residual(B=B, T=T, D=D, kind=rng.choice(['rms', 'layer', 'none']), next_kind=rng.choice(['rms', 'layer', 'none']),
                         bias=rng.random() < 0.5, gate=rng.choice(['none', 'channel', 'sequence', 'full']),
                         learned=rng.random() < 0.3, scale=round(rng.uniform(0.5, 1.5), 3), dtype=dtype, wtype=wtype, bwd=bwd)
    d = rng.choice([8, 16, 20, 32, 40, 64, 64, 96, 128])
    dv = rng.choice([d, 2 * d])
    G = _log(rng, 1, 8)
    H = G * rng.choice([1, 1, 2, 4])
    form = rng.choice(['decode', 'self', 'self', 'cross'])
    if form == 'decode':
        bwd = False
        Tk = _log(rng, 16, 16384)
        Tq = rng.choice([1, 1, 1, 2, 4])
        c = _attn(B=max(1, min(_log(rng, 1, 64), (1 << 28) // (Tk * G * (2 * d + dv) * 2))), Tq=Tq, Tk=Tk, causal=Tq > 1,
                  ragged=rng.random() < 0.7)
    else:
        Tq = _log(rng, 8, 4096)
        Tk = Tq if form == 'self' else _log(rng, 8, 4096)
        c = _attn(Tq=Tq, Tk=Tk, causal=form == 'self' and rng.random() < 0.5, mask=rng.choice(['none', 'keys', 'full']),
                  ragged=rng.random() < 0.3)
        most = 0.5 * 2 * 8 * 4096 * 4096 * 256   # half the long training case's products
        c['B'] = max(1, min(_log(rng, 1, 64), int(most / (H * Tq * Tk * (2 * d + dv)))))
    c.update(H=H, G=G, d=d, dv=dv, dtype=dtype, lam=rng.choice(['head', 'row']), bwd=bwd)
    return c


# ------------------------------------------------------------------ inputs
def _frequencies(c):
    """(freqs float64 [rot / 2], amplitude): plain, positions divided, base raised, or interpolated by parts."""
    r, base, f = c['rot'], c['base'], c['factor']
    if c['scaling'] == 'ntk':
        base = base * f ** (r / max(r - 2, 1))
    w = torch.pow(torch.tensor(base, dtype=torch.float64), -torch.arange(0, r, 2, dtype=torch.float64) / r)
    if c['scaling'] == 'linear':
        return w / f, 1.0
    if c['scaling'] == 'parts':   # under 1 turn of the 4096-token context: divided; over 32: kept; between: a ramp
        turns = 4096 * w / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return w * keep + (w / f) * (1 - keep), 0.1 * math.log(f) + 1.0
    return w, 1.0


def prepare(case, seed):
    c, dev = case, 'cuda'
    t, g = TYPES[c['dtype']], torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, dtype=t, grad=True, mean=0.0, std=1.0):
        x = (torch.randn(*shape, generator=g, device=dev) * std + mean).to(dtype)
        return x.requires_grad_(bool(c['bwd'] and grad))

    s = {'case': c}
    if c['op'] == 'rotary':
        f, s['amplitude'] = _frequencies(c)
        s['freqs'] = f.to(dev)
        s['positions'] = c['first'] + torch.arange(c['T'], device=dev) + torch.randint(0, 100, (c['B'], 1), generator=g, device=dev)
        for n, heads in (('q', c['H']), ('k', c['G'])):
            s[n] = normal(c['B'], c['T'], heads, c['D'])
            s['d' + n] = normal(c['B'], c['T'], heads, c['D'], grad=False) if c['bwd'] else None
    elif c['op'] in ('norm', 'residual'):
        wt, B, T, D = TYPES[c['wtype']], c['B'], c['T'], c['D']
        shift = 0.5 if c['kind'] == 'layer' else 0.0
        weight = lambda on: normal(D, dtype=wt, mean=1.0, std=0.2) if on else None  # noqa: E731
        bias = lambda on: normal(D, dtype=wt, std=0.2) if on else None  # noqa: E731
        s['y'] = normal(B, T, D, mean=shift)
        s['weight'], s['bias'] = weight(c['kind'] != 'none'), bias(c['kind'] != 'none' and c['bias'])
        s['dnormed'] = normal(B, T, D, grad=False) if c['bwd'] else None
        if c['op'] == 'residual':
            s['residual'] = normal(B, T, D)
            nk = c['next_kind'] != 'none'
            s['next_weight'], s['next_bias'] = weight(nk), bias(nk and c['bias'])
            shape = {'none': None, 'channel': (D,), 'sequence': (B, D), 'full': (B, T, D)}[c['gate']]
            s['gate'] = None if shape is None else normal(*shape, dtype=t if c['gate'] == 'full' else wt, mean=0.5, std=0.3)
            s['scale'] = torch.full((1,), c['scale'], device=dev).requires_grad_(bool(c['bwd'])) if c['learned'] else c['scale']
            s['dstream'] = normal(B, T, D, grad=False) if c['bwd'] else None
            s['dnormed'] = s['dnormed'] if nk else None
    else:
        B, Tq, Tk, H, G = c['B'], c['Tq'], c['Tk'], c['H'], c['G']
        s['q'] = normal(B, Tq, H, 2, c['d'])
        s['k'] = normal(B, Tk, G, 2, c['d'])
        s['v'] = normal(B, Tk, G, c['dv'])
        shape = (H,) if c['lam'] == 'head' else (B, Tq, H)
        s['lam'] = (torch.rand(*shape, generator=g, device=dev) * 0.6 + 0.2).requires_grad_(bool(c['bwd']))
        s['dout'] = normal(B, Tq, H, c['dv'], grad=False) if c['bwd'] else None
        s['mask'] = s['lengths'] = s['q_start'] = None
        if c['mask'] == 'keys':       # the loader's float mask: ones, then zeros behind each row's last step
            n = torch.randint(max(1, Tk // 2), Tk + 1, (B, 1), generator=g, device=dev)
            s['mask'] = (torch.arange(Tk, device=dev) < n).float()
        elif c['mask'] == 'full':     # any pair of a query and a key; some queries see no key
            s['mask'] = torch.rand(B, Tq, Tk, generator=g, device=dev) < 0.7
            s['mask'] &= (torch.rand(B, Tq, 1, generator=g, device=dev) < 0.95)
        if c['ragged']:
            s['lengths'] = torch.randint(max(1, Tk // 4), Tk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        if c['causal']:
            s['q_start'] = (s['lengths'] - Tq).clamp(min=0) if c['ragged'] and Tq < Tk else None
    return s


# ------------------------------------------------------------------ plain forms
def _turn(x, cos, sin, c):
    """The pairs of the first rot channels turned by (cos, sin), the rest as it is; x in 32 bits."""
    r = c['rot']
    if c['layout'] == 'half':
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _plain_rotary(s):
    c = s['case']
    angle = s['positions'].double()[:, :, None, None] * s['freqs']
    cos, sin = (torch.cos(angle) * s['amplitude']).float(), (torch.sin(angle) * s['amplitude']).float()
    out = [_turn(s[n].float(), cos, sin, c).to(s[n].dtype) for n in 'qk']
    if c['bwd']:
        out += [_turn(s['d' + n].float(), cos, -sin, c).to(s[n].dtype) for n in 'qk']
    return out


def _stat(x, kind):
    """(normalised x, 1 / deviation) of the last dimension"""
    if kind == 'layer':
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * r, r


def _affine(x, w, b):
    x = x if w is None else x * w.float()
    return x if b is None else x + b.float()


def _norm_back(g, xh, r, w, kind):
    """the gradient through a norm of upstream gradient g"""
    u = g if w is None else g * w.float()
    u = u - xh * (u * xh).mean(-1, keepdim=True) - (u.mean(-1, keepdim=True) if kind == 'layer' else 0.0)
    return u * r


def _columns(g, like):
    return None if like is None else g.sum((0, 1)).to(like.dtype)


def _plain_norm(s):
    c = s['case']
    y = s['y'].float()
    yh, r = _stat(y, c['kind'])
    out = [_affine(yh, s['weight'], s['bias']).to(s['y'].dtype)]
    if c['bwd']:
        g = s['dnormed'].float()
        out += [_norm_back(g, yh, r, s['weight'], c['kind']).to(s['y'].dtype), _columns(g * yh, s['weight']), _columns(g, s['bias'])]
    return out


def _plain_residual(s):
    c, t = s['case'], s['y'].dtype
    y, x = s['y'].float(), s['residual'].float()
    yh, r = _stat(y, c['kind']) if c['kind'] != 'none' else (y, None)
    n = _affine(yh, s['weight'], s['bias'])
    gate = s['gate']
    gf = None if gate is None else gate.float()[:, None] if c['gate'] == 'sequence' else gate.float()
    stream = s['scale'] * x + (n if gf is None else gf * n)
    out = [stream.to(t)]
    if c['next_kind'] != 'none':
        h, hr = _stat(stream, c['next_kind'])
        out.append(_affine(h, s['next_weight'], s['next_bias']).to(t))
    if c['bwd']:
        dx = s['dstream'].float()
        dnw = dnb = None
        if c['next_kind'] != 'none':
            g = s['dnormed'].float()
            dx = dx + _norm_back(g, h, hr, s['next_weight'], c['next_kind'])
            dnw, dnb = _columns(g * h, s['next_weight']), _columns(g, s['next_bias'])
        dg = None
        if gate is not None:
            dg = dx * n
            dg = (dg.sum((0, 1)) if c['gate'] == 'channel' else dg.sum(1) if c['gate'] == 'sequence' else dg).to(gate.dtype)
        dn = dx if gf is None else dx * gf
        dy = dn if c['kind'] == 'none' else _norm_back(dn, yh, r, s['weight'], c['kind'])
        out += [dy.to(t), (s['scale'] * dx).to(t), _columns(dn * yh, s['weight']), _columns(dn, s['bias']), dg,
                (dx * x).sum().reshape(1) if c['learned'] else None, dnw, dnb]
    return out


def _allowed(s):
    """[B or 1, 1, 1, 1, Tq or 1, Tk] truth values, or None"""
    c = s['case']
    dev = s['q'].device
    key, ok = torch.arange(c['Tk'], device=dev), None
    if s['mask'] is not None:
        m = s['mask'] != 0
        ok = m[:, None] if c['mask'] == 'keys' else m
    if s['lengths'] is not None:
        m = (key < s['lengths'][:, None])[:, None]
        ok = m if ok is None else ok & m
    if c['causal']:
        first = torch.full((1,), c['Tk'] - c['Tq'], device=dev) if s['q_start'] is None else s['q_start']
        m = key <= (first[:, None] + torch.arange(c['Tq'], device=dev))[:, :, None]
        ok = m if ok is None else ok & m
    return None if ok is None else ok[:, None, None, None]


def _plain_attn(s):
    c, t = s['case'], s['q'].dtype
    B, Tq, Tk, H, G, d, dv = (c[n] for n in ('B', 'Tq', 'Tk', 'H', 'G', 'd', 'dv'))
    n = H // G
    q = s['q'].float().reshape(B, Tq, G, n, 2, d).permute(0, 2, 3, 4, 1, 5)          # B G n 2 Tq d
    k = s['k'].float().permute(0, 2, 3, 1, 4)[:, :, None]                            # B G 1 2 Tk d
    v = s['v'].float().permute(0, 2, 1, 3)[:, :, None]                               # B G 1 Tk dv
    lam = s['lam'] if c['lam'] == 'row' else s['lam'].expand(B, Tq, H)
    lam = lam.reshape(B, Tq, G, n).permute(0, 2, 3, 1)[..., None]                     # B G n Tq 1
    a = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5)
    ok = _allowed(s)
    if ok is not None:
        a.masked_fill_(~ok, -math.inf)
    a.sub_(a.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    a.div_(a.sum(-1, keepdim=True).clamp_(min=1e-38))                                 # B G n 2 Tq Tk
    p = a[:, :, :, 0] - lam * a[:, :, :, 1]
    out = [torch.matmul(p, v).permute(0, 3, 1, 2, 4).reshape(B, Tq, H, dv).to(t)]
    if c['bwd']:
        do = s['dout'].float().reshape(B, Tq, G, n, dv).permute(0, 2, 3, 1, 4)        # B G n Tq dv
        dval = torch.matmul(p.transpose(-1, -2), do).sum(2).permute(0, 2, 1, 3).to(t)
        del p
        dp = torch.matmul(do, v.transpose(-1, -2))
        row = (a * dp[:, :, :, None]).sum(-1, keepdim=True)                           # B G n 2 Tq 1
        sign = torch.stack([torch.ones_like(lam), -lam], 3)
        ds = a.mul_(dp[:, :, :, None] - row).mul_(sign * d ** -0.5)
        dq = torch.matmul(ds, k).permute(0, 4, 1, 2, 3, 5).reshape(B, Tq, H, 2, d).to(t)
        dk = torch.matmul(ds.transpose(-1, -2), q).sum(2).permute(0, 3, 1, 2, 4).to(t)
        dl = -row[:, :, :, 1, :, 0].permute(0, 3, 1, 2).reshape(B, Tq, H)
        out += [dq, dk, dval, dl if c['lam'] == 'row' else dl.sum((0, 1))]
    return out


# ------------------------------------------------------------------ the framework's calls
def _grads(outs, gouts, leaves):
    on = [x for x in leaves if torch.is_tensor(x)]
    got = iter(torch.autograd.grad(outs, on, gouts))
    return [next(got) if torch.is_tensor(x) else None for x in leaves]


def _own(s):
    import mep_import
    mep_import.load()
    from mep_amd import diff_block as db
    c = s['case']
    if c['op'] == 'rotary':
        out = db.rotary(s['q'], s['k'], positions=s['positions'], freqs=s['freqs'], layout=c['layout'], amplitude=s['amplitude'])
        return list(out) + (_grads(out, [s['dq'], s['dk']], [s['q'], s['k']]) if c['bwd'] else [])
    if c['op'] == 'norm':
        out = db.norm(s['y'], s['weight'], s['bias'], kind=c['kind'], eps=EPS)
        return [out] + (_grads([out], [s['dnormed']], [s['y'], s['weight'], s['bias']]) if c['bwd'] else [])
    if c['op'] == 'residual':
        out = db.norm_residual(s['y'], s['residual'], s['weight'], s['bias'], kind=c['kind'], gate=s['gate'], scale=s['scale'],
                               next_kind=c['next_kind'], next_weight=s['next_weight'], next_bias=s['next_bias'], eps=EPS)
        out = list(out) if c['next_kind'] != 'none' else [out]
        if not c['bwd']:
            return out
        up = [s['dstream']] + ([s['dnormed']] if c['next_kind'] != 'none' else [])
        return out + _grads(out, up, [s['y'], s['residual'], s['weight'], s['bias'], s['gate'], s['scale'],
                                      s['next_weight'], s['next_bias']])
    out = db.diff_attention(s['q'], s['k'], s['v'], s['lam'], mask=s['mask'], lengths=s['lengths'], causal=c['causal'],
                            q_start=s['q_start'])
    return [out] + (_grads([out], [s['dout']], [s['q'], s['k'], s['v'], s['lam']]) if c['bwd'] else [])


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {'rotary': _plain_rotary, 'norm': _plain_norm, 'residual': _plain_residual, 'attn': _plain_attn}[state['case']['op']](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    e = 4 if c['dtype'] == 'float32' else 2
    both = 2 if c['bwd'] else 1
    if c['op'] == 'rotary':
        n = c['B'] * c['T'] * (c['H'] + c['G'])
        return {'bytes': both * (2 * n * c['D'] * e + 8 * c['B'] * c['T']), 'flops': both * n * 3 * c['rot']}
    if c['op'] == 'norm':
        n = c['B'] * c['T'] * c['D']
        return {'bytes': (5 if c['bwd'] else 2) * n * e, 'flops': (14 if c['bwd'] else 5) * n}
    if c['op'] == 'residual':
        n = c['B'] * c['T'] * c['D']
        full, nxt = int(c['gate'] == 'full'), int(c['next_kind'] != 'none')
        fwd = 2 + full + 1 + nxt
        return {'bytes': n * e * (fwd + (3 + full + nxt + 2 + full if c['bwd'] else 0)), 'flops': (40 if c['bwd'] else 12) * n}
    rows = c['B'] * c['H'] * c['Tq']
    keys = c['Tk'] * (0.625 if c['ragged'] else 1.0)
    pairs = rows * (keys - c['Tq'] / 2 if c['causal'] and c['Tq'] > 1 else keys)
    io = (rows * (2 * c['d'] + c['dv']) + c['B'] * keys * c['G'] * (2 * c['d'] + c['dv'])) * e
    flops = 2 * pairs * (2 * c['d'] + c['dv'])
    if c['bwd']:
        io = 3 * io
        flops += 2 * pairs * (6 * c['d'] + 2 * c['dv'])
    return {'bytes': io, 'flops': max(flops, 1)}


# ------------------------------------------------------------------ 64 bits
def _wide(s, *names):
    return [None if s[n] is None else s[n].detach().double().requires_grad_(True) if torch.is_tensor(s[n]) else s[n] for n in names]


def _back(outs, ups, leaves):
    on = [x for x in leaves if torch.is_tensor(x)]
    got = iter(torch.autograd.grad(outs, on, ups))
    return [next(got) if torch.is_tensor(x) else None for x in leaves]


def _exact_rotary(s):
    c = s['case']
    r = c['rot']
    z = torch.polar(torch.full_like(s['freqs'], s['amplitude']), torch.zeros_like(s['freqs']))
    z = z * torch.exp(1j * (s['positions'].double()[..., None] * s['freqs']))          # B T r/2
    leaves = _wide(s, 'q', 'k')
    outs = []
    for x in leaves:
        head = x[..., :r]
        pairs = head.unflatten(-1, (2, r // 2)).transpose(-1, -2) if c['layout'] == 'half' else head.unflatten(-1, (r // 2, 2))
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z[:, :, None])
        y = y.transpose(-1, -2).flatten(-2) if c['layout'] == 'half' else y.flatten(-2)
        outs.append(torch.cat([y, x[..., r:]], -1))
    grads = _back(outs, [s['dq'].double(), s['dk'].double()], leaves) if c['bwd'] else []
    return outs + grads


def _exact_norm_of(x, kind, w, b):
    if kind == 'none':
        return x
    if kind == 'layer':
        return torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, EPS)
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w
    return y if b is None else y + b


def _exact_norm(s):
    c = s['case']
    leaves = _wide(s, 'y', 'weight', 'bias')
    out = _exact_norm_of(leaves[0], c['kind'], leaves[1], leaves[2])
    return [out] + (_back([out], [s['dnormed'].double()], leaves) if c['bwd'] else [])


def _exact_residual(s):
    c = s['case']
    leaves = _wide(s, 'y', 'residual', 'weight', 'bias', 'gate', 'scale', 'next_weight', 'next_bias')
    y, x, w, b, gate, scale, nw, nb = leaves
    n = _exact_norm_of(y, c['kind'], w, b)
    if gate is not None:
        n = n * (gate.unsqueeze(1) if c['gate'] == 'sequence' else gate)
    stream = x * scale + n
    outs = [stream]
    if c['next_kind'] != 'none':
        outs.append(_exact_norm_of(stream, c['next_kind'], nw, nb))
    if not c['bwd']:
        return outs
    ups = [s['dstream'].double()] + ([s['dnormed'].double()] if c['next_kind'] != 'none' else [])
    return outs + _back(outs, ups, leaves)


def _exact_attn(s):
    c = s['case']
    B, Tq, Tk, H, G, d = (c[n] for n in ('B', 'Tq', 'Tk', 'H', 'G', 'd'))
    if B * H > 1024:
        return None
    dev = s['q'].device
    n = H // G
    out = torch.empty(B, Tq, H, c['dv'], dtype=torch.float64, device=dev)
    keep = {x: torch.zeros(s[x].shape, dtype=torch.float64, device=dev) for x in ('q', 'k', 'v', 'lam')}
    rowno, keyno = torch.arange(Tq, device=dev)[:, None], torch.arange(Tk, device=dev)[None]
    for b in range(B):
        ok = torch.ones(Tq, Tk, dtype=torch.bool, device=dev)
        if s['mask'] is not None:
            ok &= s['mask'][b].bool()
        if s['lengths'] is not None:
            ok &= keyno < s['lengths'][b]
        if c['causal']:
            ok &= keyno - rowno <= (Tk - Tq if s['q_start'] is None else s['q_start'][b])
        some = ok.any(1, keepdim=True).double()
        hide = torch.zeros(Tq, Tk, dtype=torch.float64, device=dev).masked_fill_(~ok, -1e300)
        for h in range(H):
            q = s['q'][b, :, h].detach().double().requires_grad_(True)
            k = s['k'][b, :, h // n].detach().double().requires_grad_(True)
            v = s['v'][b, :, h // n].detach().double().requires_grad_(True)
            lam = s['lam'][b, :, h] if c['lam'] == 'row' else s['lam'][h]
            lam = lam.detach().double().requires_grad_(True)
            one, two = (torch.softmax(q[:, m] @ k[:, m].T / math.sqrt(d) + hide, -1) for m in (0, 1))
            o = some * (one @ v - lam.reshape(-1, 1) * (two @ v))
            out[b, :, h] = o.detach()
            if c['bwd']:
                gq, gk, gv, gl = torch.autograd.grad(o, (q, k, v, lam), s['dout'][b, :, h].double())
                keep['q'][b, :, h] = gq
                keep['k'][b, :, h // n] += gk
                keep['v'][b, :, h // n] += gv
                if c['lam'] == 'row':
                    keep['lam'][b, :, h] = gl
                else:
                    keep['lam'][h] += gl
    return [out] + ([keep[x] for x in ('q', 'k', 'v', 'lam')] if c['bwd'] else [])


def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        got = {'rotary': _exact_rotary, 'norm': _exact_norm, 'residual': _exact_residual, 'attn': _exact_attn}[case['op']](s)
    return got if got is None else [x.detach() if torch.is_tensor(x) else x for x in got]
