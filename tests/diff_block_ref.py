"""Plain 64-bit forms of mep_amd.diff_block for its tests, on the CPU, with torch's autograd for the gradients, and the
tolerance that the tests share."""
import math

import torch

U = 2.0 ** -24          # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def wide(t):
    return None if t is None else t.detach().cpu().double().requires_grad_(True)


def close(got, want, mag, terms, what=''):
    """|got - want| <= half a step of got's type at want, and `terms` roundings of fp32 at the magnitude `mag` of what was
    summed (a tensor that broadcasts, or a number); half a step more where the sum's own error moves the last rounding."""
    g, w = got.detach().cpu().double(), want.detach().double()
    assert g.shape == w.shape, (what, g.shape, w.shape)
    tiny = torch.finfo(got.dtype).smallest_normal * half_step(got.dtype) * 2   # a subnormal's half step
    inner = terms * U * mag
    tol = half_step(got.dtype) * (w.abs() + inner) + inner + tiny
    err = (g - w).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), '%s: %d of %d off, worst %.3g over %.3g' % (
        what, int(bad.sum()), bad.numel(), float(err[bad].max()), float((tol + torch.zeros_like(err))[bad].min()))


# ------------------------------------------------------------------ rotary
def rotary(x, positions, freqs, layout, amplitude):
    r = 2 * freqs.numel()
    B, T = x.shape[:2]
    a = positions.double().expand(B, T)[..., None] * freqs
    shape = (B, T) + (1,) * (x.dim() - 3) + (r // 2,)
    c, s = (torch.cos(a) * amplitude).reshape(shape), (torch.sin(a) * amplitude).reshape(shape)
    i, j = (slice(0, r // 2), slice(r // 2, r)) if layout == 'half' else (slice(0, r, 2), slice(1, r, 2))
    y = x.clone()
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    return y


# ------------------------------------------------------------------ norms
def norm(x, w, b, kind, eps):
    if kind == 'none':
        return x
    if kind == 'layer':
        x = x - x.mean(-1, keepdim=True)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    y = y if w is None else y * w
    return y if b is None else y + b


def norm_residual(y, x, w, b, kind, gate, scale, next_kind, nw, nb, eps):
    n = norm(y, w, b, kind, eps)
    if gate is not None:
        n = n * (gate[:, None] if gate.dim() == 2 and y.dim() == 3 else gate)
    s = n if x is None else scale * x + n
    return (s, norm(s, nw, nb, next_kind, eps)) if next_kind != 'none' else (s,)


# ------------------------------------------------------------------ differential attention
def allowed(B, Tq, Tk, mask, lengths, causal, q_start):
    ok = torch.ones(B, Tq, Tk, dtype=torch.bool)
    key = torch.arange(Tk)
    if mask is not None:
        m = mask.cpu() != 0
        ok &= m[:, None] if m.dim() == 2 else m
    if lengths is not None:
        ok &= (key < lengths.cpu()[:, None].long())[:, None]
    if causal:
        first = torch.full((B,), Tk - Tq) if q_start is None else q_start.cpu().long()
        ok &= key <= (first[:, None] + torch.arange(Tq))[:, :, None]
    return ok


def diff_attention(q, k, v, lam, ok, scale=None):
    B, Tq, H, _, d = q.shape
    G = k.shape[2]
    n = H // G
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    kk, vv = k.repeat_interleave(n, 2), v.repeat_interleave(n, 2)
    some = ok.any(-1)[:, None, None, :, None].double()
    s = torch.einsum('bthmd,bshmd->bhmts', q, kk) * scale
    a = torch.softmax(s.masked_fill(~ok[:, None, None], -1e300), -1) * some
    lam = lam.expand(B, Tq, H).permute(0, 2, 1)[..., None]
    return torch.einsum('bhts,bshe->bthe', a[:, :, 0] - lam * a[:, :, 1], vv)
