"""Operators of a differential-attention block on libmep_hip, with their gradients:

    h  = norm(x, w)                                       the norm before the block
    q, k = rotary(q, k, positions=..., freqs=...)         rotary positions (rotary_frequencies makes freqs)
    a  = diff_attention(q, k, v, lam, ...)                the difference of two softmax maps
    x, h = norm_residual(y, x, ...)                       norm behind the block, gate, residual scale, next norm

They stand beside the residual-attention blocks of the reference (its Attention_Block takes position tables, one
softmax map and a LayerNorm behind the block, cmu-mosei/run.py:206-262) and have no counterpart there.  Each call launches
its kernels (one; more where column sums or splits are joined, an unaligned input is copied, dq, dk and lam's gradient
follow each other, or float16 gradients are scaled into range) on the current stream of its tensors' device, allocates nothing
but its results and workspace, never synchronises, and may be captured into a graph.  float32, bfloat16 and float16
activations; sums, statistics and angles in 32 bits or more; results do not depend on the order of atomics.

Gradients come through torch.autograd.  To capture a backward pass into a graph, make the leaves it differentiates inside
the capture (``x.detach().requires_grad_()``) and use ``torch.autograd.grad``: torch ends the process when a captured
backward meets accumulators that an eager graph of the same leaves still holds.
"""
import ctypes
import math

import torch

from . import _lib
from ._autograd import require_cuda

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # MEP_F32 / MEP_BF16 / MEP_F16
KINDS = {'none': 0, 'rms': 1, 'layer': 2}


def _on_device(first, *others):
    """The last check of a call's arguments: all on one GPU."""
    for t in others:
        if torch.is_tensor(t) and t.device != first.device:
            raise ValueError('all tensors of a call live on one device; got %s and %s' % (first.device, t.device))
    require_cuda(first)


def _type_of(t, what):
    if t.dtype not in TYPES:
        raise ValueError('%s must be float32, bfloat16 or float16; got %s' % (what, t.dtype))
    return TYPES[t.dtype]


def _launch(name, desc, device):
    """An entry point that takes its descriptor from the host, on the current stream of `device`."""
    i = device.index
    if torch._C._cuda_getDevice() != i or _lib.TIMER is not None:
        with torch.cuda.device(i):
            return _lib.call(name, ctypes.byref(desc))
    # the raw stream: this call is most of a short operator's time, and torch.cuda.current_stream() most of this call
    rc = getattr(_lib.lib(), name)(ctypes.byref(desc), torch._C._cuda_getCurrentRawStream(i))
    if rc:
        _lib.check(rc, name)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _places(saved):
    """Where saved tensors lie.  Hooks on them (a checkpoint that computes them again, offloading) give the backward others."""
    return [None if t is None else (t.data_ptr(), t.stride()) for t in saved]


def _moved(desc, names, tensors):
    """A copy of the descriptor with the addresses of `tensors`."""
    d = type(desc).from_buffer_copy(desc)
    for n, t in zip(names, tensors):
        setattr(d, n, _ptr(t))
    return d


# ------------------------------------------------------------------ rotary positions
def rotary_frequencies(rot_dim, base=10000.0, *, scaling=None, factor=1.0, original_len=None, low_turns=1.0,
                       high_turns=32.0, device='cuda'):
    """(freqs float64 [rot_dim / 2] in radians per position, amplitude) for rotary().

    Pair i turns by base ** (-2 i / rot_dim) per position.  Contexts `factor` times as long as the trained one:
      'linear'  every position divided by factor
      'ntk'     the base raised to base * factor ** (rot_dim / (rot_dim - 2)): the fastest pair stays, the slowest is divided
      'parts'   interpolated by parts: pairs that make fewer than `low_turns` turns over `original_len` positions are divided
                by factor, pairs with more than `high_turns` stay, a linear ramp in between; amplitude 0.1 ln(factor) + 1
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError('rot_dim must be a positive even number; got %r' % (rot_dim,))
    if not base > 0 or not factor > 0:
        raise ValueError('base and factor must be positive')
    if scaling not in (None, 'linear', 'ntk', 'parts'):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'parts'; got %r" % (scaling,))
    if scaling == 'ntk':
        if rot_dim < 4:
            raise ValueError("scaling 'ntk' needs rot_dim >= 4")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    f = torch.tensor([base ** (-i / rot_dim) for i in range(0, rot_dim, 2)], dtype=torch.float64)
    amplitude = 1.0
    if scaling == 'linear':
        f = f / factor
    elif scaling == 'parts':
        if original_len is None or original_len < 1 or not high_turns > low_turns:
            raise ValueError("scaling 'parts' needs original_len and high_turns > low_turns")
        keep = ((original_len * f / (2 * math.pi) - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return f.to(device), amplitude


def _rotary_launch(xs, positions, freqs, interleaved, amplitude, inverse):
    d = _lib.RotaryDesc()
    xs = [x if x.stride(-1) == 1 else x.contiguous() for x in xs]
    ys = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs]
    on = [(x, y) for x, y in zip(xs, ys) if x.numel()]
    if not on:
        return ys
    for i, (x, y) in enumerate(on):
        d.x[i], d.y[i] = x.data_ptr(), y.data_ptr()
        d.sB[i], d.sT[i], d.sH[i] = x.stride(0), x.stride(1), x.stride(2)
        d.H[i], d.M[i], d.sM[i] = (x.shape[2], x.shape[3], x.stride(3)) if x.dim() == 5 else (x.shape[2], 1, 0)
    x = on[0][0]
    d.B, d.T, d.D, d.rot = x.shape[0], x.shape[1], x.shape[-1], 2 * freqs.numel()
    d.freqs, d.pos, d.pos64 = freqs.data_ptr(), positions.data_ptr(), int(positions.dtype == torch.int64)
    d.pos_sB, d.pos_sT = (0, positions.stride(0)) if positions.dim() == 1 else positions.stride()
    d.interleaved, d.inverse, d.type, d.amplitude = int(interleaved), int(inverse), TYPES[x.dtype], amplitude
    _launch('mep_rotary', d, x.device)
    return ys


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, freqs, interleaved, amplitude, *xs):
        ctx.save_for_backward(positions, freqs)
        ctx.meta = (interleaved, amplitude)
        ctx.set_materialize_grads(False)
        return tuple(_rotary_launch(list(xs), positions, freqs, interleaved, amplitude, False))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *gs):
        positions, freqs = ctx.saved_tensors
        interleaved, amplitude = ctx.meta
        on = [i for i, g in enumerate(gs) if g is not None and ctx.needs_input_grad[4 + i]]
        out = [None] * len(gs)
        if on:
            for i, y in zip(on, _rotary_launch([gs[i] for i in on], positions, freqs, interleaved, amplitude, True)):
                out[i] = y
        return (None, None, None, None, *out)


def rotary(q, k=None, *, positions, freqs, layout='half', amplitude=1.0):
    """Rotary positions of q, or of q and k in one launch; returns what it was given, contiguous.

    q, k [B, T, heads, D] or [B, T, heads, maps, D] (any strides), of one type; positions int32 / int64 [T] or [B, T];
    freqs float64 [r / 2] (rotary_frequencies): the first r channels of each head are turned, the rest copied.
    layout 'half' pairs channels (i, i + r / 2), 'interleaved' pairs (2i, 2i + 1).  The angles are formed in 64 bits.
    """
    xs = [q] if k is None else [q, k]
    _type_of(q, 'q')
    for x in xs:
        if x.dim() not in (4, 5) or x.shape[:2] != q.shape[:2] or x.shape[-1] != q.shape[-1] or x.dtype != q.dtype:
            raise ValueError('q and k must be [batch, time, heads, (maps,) channels] of one type, batch, time and channels; got %s'
                             % ', '.join('%s %s' % (tuple(x.shape), x.dtype) for x in xs))
    B, T, D = q.shape[0], q.shape[1], q.shape[-1]
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous() or not 1 <= freqs.numel() <= D // 2:
        raise ValueError('freqs must be contiguous float64 [r / 2] with 2 <= r <= channels; got %s %s' % (tuple(freqs.shape), freqs.dtype))
    if freqs.requires_grad:
        raise ValueError('freqs have no gradient')
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ((T,), (B, T)):
        raise ValueError('positions must be int32 or int64 [time] or [batch, time]; got %s %s' % (tuple(positions.shape), positions.dtype))
    if layout not in ('half', 'interleaved'):
        raise ValueError("layout must be 'half' or 'interleaved'; got %r" % (layout,))
    _on_device(q, k, positions, freqs)
    out = _RotaryFn.apply(positions, freqs, layout == 'interleaved', float(amplitude), *xs)
    return out[0] if k is None else out


# ------------------------------------------------------------------ the norms around a block
def _rows(t, D):
    """(rows, row stride) of [..., D]: as it is, or a 2-D view; a copy only where the rows have no common stride"""
    if t.is_contiguous():
        return t, D
    t = t.reshape(-1, D)
    if D > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, y, x, w, b, gate, scale, nw, nb):
        kind, next_kind, gate_form, T, eps, scale_value, grad = cfg
        D = y.shape[-1]
        dev = y.device
        y2, y_ld = _rows(y, D)
        x2, x_ld = _rows(x, D) if x is not None else (None, 0)
        g2, g_ld = _rows(gate, D) if gate_form == 3 else (gate.contiguous() if gate is not None else None, 0)
        w, b, nw, nb = (None if t is None else t.contiguous() for t in (w, b, nw, nb))
        n = y.numel() // D
        stream = torch.empty(y.shape, dtype=y.dtype, device=dev)
        normed = torch.empty_like(stream) if next_kind else None
        keep = grad and any(ctx.needs_input_grad)
        stats = torch.empty(n, 4, dtype=torch.float32, device=dev) if keep else None
        params = [t for t in (w, b, nw, nb) if t is not None]
        d = _lib.BlockNormDesc(y=_ptr(y2), x=_ptr(x2), gate=_ptr(g2), w=_ptr(w), b=_ptr(b), nw=_ptr(nw), nb=_ptr(nb),
                               scale=_ptr(scale), stream=_ptr(stream), normed=_ptr(normed), stats=_ptr(stats), y_ld=y_ld, x_ld=x_ld,
                               g_ld=g_ld, rows=n, D=D, T=T, kind=kind, next_kind=next_kind, gate_form=gate_form,
                               type=TYPES[y.dtype], wtype=TYPES[params[0].dtype] if params else 0,
                               gtype=TYPES[gate.dtype] if gate is not None else 0, eps=eps, scale_value=scale_value)
        if n:
            _launch('mep_block_norm_fwd', d, dev)
        if keep:
            ctx.set_materialize_grads(False)
            saved = (y2, x2, g2, w, b, scale, nw, nb, stats)
            ctx.save_for_backward(*saved)
            ctx.shapes = (y.shape, None if gate is None else gate.shape, None if scale is None else scale.shape)
            # the backward reads the forward's inputs by address, and asks of its results only which there were
            ctx.desc, ctx.places = d, _places(saved)
        return (stream, normed) if next_kind else stream

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dstream, dnormed=None):
        saved = ctx.saved_tensors
        none = (None,) * 9
        if dstream is None and dnormed is None:
            return none
        need = ctx.needs_input_grad
        shape, gate_shape, scale_shape = ctx.shapes
        d = ctx.desc
        if _places(saved) != ctx.places:
            D = d.D
            y2, x2, g2 = saved[:3]
            (y2, y_ld), (x2, x_ld) = _rows(y2, D), _rows(x2, D) if x2 is not None else (None, 0)
            g2, g_ld = _rows(g2, D) if d.gate_form == 3 else (g2, 0)
            saved = (y2, x2, g2, *(None if t is None else t.contiguous() for t in saved[3:]))
            d = _moved(d, ('y', 'x', 'gate', 'w', 'b', 'scale', 'nw', 'nb', 'stats'), saved)
            d.y_ld, d.x_ld, d.g_ld = y_ld, x_ld, g_ld
        y2, x2, g2, w, b, scale, nw, nb, _ = saved
        n, D, dev = d.rows, d.D, y2.device
        rows = lambda on: torch.empty(shape, dtype=y2.dtype, device=dev) if on else None  # noqa: E731
        like = lambda t, on: torch.empty_like(t) if t is not None and on else None  # noqa: E731
        dy, dx = rows(True), rows(x2 is not None and need[2])
        dw, db, dgate, dscale, dnw, dnb = (like(t, need[i]) for t, i in ((w, 3), (b, 4), (None if d.gate_form == 3 else g2, 5),
                                                                         (scale, 6), (nw, 7), (nb, 8)))
        if d.gate_form == 3:
            dgate = rows(need[5])
        if dnormed is None:    # the second norm took no part
            for t in (dnw, dnb):
                if t is not None:
                    t.zero_()
        if n == 0:
            for t in (dw, db, dnw, dnb, dscale, dgate):
                if t is not None:
                    t.zero_()
        else:
            ds2, ds_ld = _rows(dstream, D) if dstream is not None else (None, 0)
            dn2, dn_ld = _rows(dnormed, D) if dnormed is not None else (None, 0)
            sums = [t for t in (dw, db, dnw if dn2 is not None else None, dnb if dn2 is not None else None,
                                dgate if d.gate_form != 3 else None) if t is not None]
            partial = None
            if sums or dscale is not None:
                p = _lib.lib().mep_block_norm_partial(ctypes.byref(d))
                if p < 0:
                    _lib.check(p, 'mep_block_norm_partial')
                partial = torch.empty(p * (len(sums) * D + 1), dtype=torch.float32, device=dev)
            bd = _lib.BlockNormBwdDesc(f=d, dstream=_ptr(ds2), dnormed=_ptr(dn2), dy=_ptr(dy), dx=_ptr(dx),
                                       dgate_rows=_ptr(dgate) if d.gate_form == 3 else 0, dw=_ptr(dw), db=_ptr(db),
                                       dnw=_ptr(dnw) if dn2 is not None else 0, dnb=_ptr(dnb) if dn2 is not None else 0,
                                       dgate=_ptr(dgate) if d.gate_form != 3 else 0, dscale=_ptr(dscale),
                                       partial=_ptr(partial), ds_ld=ds_ld, dn_ld=dn_ld, n_sums=len(sums))
            _launch('mep_block_norm_bwd', bd, dev)
        if dgate is not None and dgate.shape != gate_shape:
            dgate = dgate.reshape(gate_shape)
        if dscale is not None and dscale.shape != scale_shape:
            dscale = dscale.reshape(scale_shape)
        return (None, dy if need[1] else None, dx, dw, db, dgate, dscale, dnw, dnb)


def _affine_ok(w, b, D, what):
    for t, n in ((w, 'weight'), (b, 'bias')):
        if t is not None and (tuple(t.shape) != (D,) or t.dtype not in TYPES):
            raise ValueError('%s%s must be a [%d] tensor of a floating type; got %s %s' % (what, n, D, tuple(t.shape), t.dtype))


def norm_residual(y, residual, weight=None, bias=None, *, kind='rms', gate=None, scale=1.0, next_kind='none',
                  next_weight=None, next_bias=None, eps=1e-6):
    """stream = scale * residual + gate * N(y) and, with a next_kind, normed = N'(stream), in one pass over the rows.

    y, residual [..., D] of one type, D <= 8192.  kind / next_kind: 'rms', 'layer' (biased variance) or 'none'.  weight, bias,
    next_weight, next_bias [D] in float32 or y's type (all the same).  gate: None, [D] (learned per channel),
    [B, D] or [B, 1, D] for y [B, T, D] (one row per sequence), or y's shape; float32 or y's type, y's type for the last.
    scale: a number, or a one-element float32 tensor that is learned.  Returns stream, or (stream, normed).
    Under torch.autocast, where products are of 16 bits, all are widened to float32 if y or the residual is.
    With both kinds 'none', small rows are slower than the torch operations they stand for.
    """
    _type_of(y, 'y')
    if torch.is_autocast_enabled('cuda') and (y.dtype == torch.float32 or (residual is not None and residual.dtype == torch.float32)):
        y, residual, weight, bias, gate, next_weight, next_bias = (
            t.float() if t is not None and t.dtype in TYPES else t for t in (y, residual, weight, bias, gate, next_weight, next_bias))
    if y.dim() < 1 or not 1 <= y.shape[-1] <= _lib.BLOCK_NORM_MAX_D:
        raise ValueError('rows must have 1 to %d channels; got %s' % (_lib.BLOCK_NORM_MAX_D, tuple(y.shape)))
    D = y.shape[-1]
    if residual is not None and (residual.shape != y.shape or residual.dtype != y.dtype):
        raise ValueError('residual must have the shape and type of y; got %s %s' % (tuple(residual.shape), residual.dtype))
    for k in (kind, next_kind):
        if k not in KINDS:
            raise ValueError("kinds are 'rms', 'layer' and 'none'; got %r" % (k,))
    if (kind == 'none' and (weight is not None or bias is not None)) or \
            (next_kind == 'none' and (next_weight is not None or next_bias is not None)):
        raise ValueError("a norm of kind 'none' has no weight and no bias")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError('eps must be finite and not negative; got %r' % (eps,))
    _affine_ok(weight, bias, D, '')
    _affine_ok(next_weight, next_bias, D, 'next_')
    types = {t.dtype for t in (weight, bias, next_weight, next_bias) if t is not None}
    if len(types) > 1 or not types <= {torch.float32, y.dtype}:
        raise ValueError('weights and biases must all be float32 or all of the type of y')
    form, T = 0, 1
    if gate is not None:
        if gate.dtype not in (torch.float32, y.dtype):
            raise ValueError('gate must be float32 or of the type of y; got %s' % gate.dtype)
        per_seq = y.dim() == 3 and tuple(gate.shape) in ((y.shape[0], D), (y.shape[0], 1, D))
        if gate.shape == y.shape and gate.dtype == y.dtype:
            form = 3
        elif tuple(gate.shape) == (D,):
            form = 1
        elif per_seq and y.shape[0] <= 65000:
            form, T = 2, max(1, y.shape[1])
        else:
            raise ValueError('gate must be [D], [B, D] or [B, 1, D] for y [B, T, D] with B <= 65000, or of the shape and type of y; '
                             'got %s %s for %s' % (tuple(gate.shape), gate.dtype, tuple(y.shape)))
    st, sv = None, 1.0
    if torch.is_tensor(scale):
        if scale.numel() != 1 or scale.dtype != torch.float32:
            raise ValueError('a learned scale is a one-element float32 tensor; got %s %s' % (tuple(scale.shape), scale.dtype))
        st = scale
    else:
        sv = float(scale)
    _on_device(y, residual, weight, bias, gate, next_weight, next_bias, st)
    cfg = (KINDS[kind], KINDS[next_kind], form, T, float(eps), sv, torch.is_grad_enabled())
    return _NormFn.apply(cfg, y, residual, weight, bias, gate, st, next_weight, next_bias)


def norm(x, weight=None, bias=None, *, kind='rms', eps=1e-6):
    """N(x) over the last dimension: the norm before a block, or of each head's row.  As norm_residual without its residual."""
    if kind not in ('rms', 'layer'):
        raise ValueError("kind must be 'rms' or 'layer'; got %r" % (kind,))
    return norm_residual(x, None, weight, bias, kind=kind, eps=eps)


# ------------------------------------------------------------------ differential attention
def _packed(t, heads=0):
    """t [B, T, H, (2,) n] as the attention kernels read it: 16 bytes at a time, 64 time steps with their heads within 2 GiB; a copy with
    rows padded by zeros (mep_pack_rows) where it does not lie so."""
    V = 16 // t.element_size()
    st = t.stride()
    sM = st[3] if t.dim() == 5 else 0
    if st[-1] == 1 and t.shape[-1] % V == 0 and t.data_ptr() % 16 == 0 and not any(s % V for s in st[:-1]) and \
            st[1] < 1 << 23 and sM < 1 << 28 and st[2] * heads < 1 << 28 and 64 * st[1] + sM + st[2] * heads < (V << 27) - 512:
        return t
    n = t.shape[-1]
    y = torch.empty(*t.shape[:-1], -(-n // V) * V, dtype=t.dtype, device=t.device)
    if t.numel():
        _launch('mep_pack_rows', _lib.PackRowsDesc(x=_ptr(t), y=_ptr(y), sB=st[0], sT=st[1], sH=st[2], sM=sM, sN=st[-1], B=t.shape[0], T=t.shape[1],
                                                   H=t.shape[2], M=t.shape[3] if t.dim() == 5 else 1, n=n, type=TYPES[t.dtype]), t.device)
    return y


def _workspace(name, desc, device):
    n = getattr(_lib.lib(), name)(ctypes.byref(desc))
    if n < 0:
        _lib.check(n, name)
    return torch.empty(n // 4, dtype=torch.float32, device=device) if n else None


def _strides(d, q, k, v, lam, mask):
    d.q_sB, d.q_sT, d.q_sH, d.q_sM, _ = q.stride()
    d.k_sB, d.k_sT, d.k_sH, d.k_sM, _ = k.stride()
    d.v_sB, d.v_sT, d.v_sH, _ = v.stride()
    d.lam_sB, d.lam_sT, d.lam_sH = (0, 0, lam.stride(0)) if lam.dim() == 1 else lam.stride()
    if mask is not None:
        d.m_sB, d.m_sQ, d.m_sK = (mask.stride(0), 0, mask.stride(1)) if mask.dim() == 2 else mask.stride()


class _DiffAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, mask, lengths, q_start, q, k, v, lam):
        causal, scale, grad = cfg
        B, Tq, H, _, hd = q.shape
        Tk, G, dv = k.shape[1], k.shape[2], v.shape[3]
        dev = q.device
        qp, kp, vp = _packed(q, H // G), _packed(k), _packed(v)
        out = torch.empty(B, Tq, H, dv, dtype=q.dtype, device=dev)
        keep = grad and any(ctx.needs_input_grad)
        stats = torch.empty(B, H, Tq, 4, dtype=torch.float32, device=dev) if keep else None
        second = torch.empty_like(out) if keep else None
        d = _lib.DiffAttnDesc(q=_ptr(qp), k=_ptr(kp), v=_ptr(vp), lam=_ptr(lam), out=_ptr(out), stats=_ptr(stats), second=_ptr(second),
                              mask=_ptr(mask), lengths=_ptr(lengths), q_start=_ptr(q_start), B=B, Tq=Tq, Tk=Tk, H=H, G=G, d=hd, dv=dv, type=TYPES[q.dtype], causal=int(causal),
                              mask_form=0 if mask is None else mask.dim() - 1,
                              mask_float=int(mask is not None and mask.dtype == torch.float32), scale=scale)
        _strides(d, qp, kp, vp, lam, mask)
        ws = _workspace('mep_diff_attn_workspace', d, dev)
        d.workspace = _ptr(ws)
        _launch('mep_diff_attn_fwd', d, dev)
        if keep:
            ctx.set_materialize_grads(False)
            saved = (mask, lengths, q_start, qp, kp, vp, lam, out, stats, second)
            ctx.save_for_backward(*saved)
            ctx.desc, ctx.places = d, _places(saved)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        if dout is None:
            return (None,) * 8
        saved, d = ctx.saved_tensors, ctx.desc
        if _places(saved) != ctx.places:
            mask, lengths, q_start, q, k, v, lam, out, stats, second = saved
            q, k, v = _packed(q, d.H // d.G), _packed(k), _packed(v)
            saved = (mask, lengths, q_start, q, k, v, lam, *(t.contiguous() for t in (out, stats, second)))
            d = _moved(d, ('mask', 'lengths', 'q_start', 'q', 'k', 'v', 'lam', 'out', 'stats', 'second'), saved)
            _strides(d, q, k, v, lam, mask)
        lam = saved[6]
        need = ctx.needs_input_grad
        B, Tq, Tk, H, G = d.B, d.Tq, d.Tk, d.H, d.G
        dev = lam.device
        dout = _packed(dout, H // G)
        new = lambda *shape: torch.empty(shape, dtype=dout.dtype, device=dev)  # noqa: E731
        dq = new(B, Tq, H, 2, d.d) if need[4] else None
        dk, dv = (new(B, Tk, G, 2, d.d), new(B, Tk, G, d.dv)) if need[5] or need[6] else (None, None)
        dlam = torch.empty(lam.shape, dtype=torch.float32, device=dev) if need[7] else None
        delta = torch.empty(B, H, Tq, 4, dtype=torch.float32, device=dev)
        shared = lam.dim() == 1
        ws = _workspace('mep_diff_attn_bwd_workspace', d, dev) if dk is not None or dout.dtype == torch.float16 else None
        bd = _lib.DiffAttnBwdDesc(f=d, dout=_ptr(dout), o_sB=dout.stride(0), o_sT=dout.stride(1), o_sH=dout.stride(2),
                                  dq=_ptr(dq), dk=_ptr(dk), dv=_ptr(dv), dlam=_ptr(dlam) if shared else 0,
                                  dlam_rows=0 if shared else _ptr(dlam), delta=_ptr(delta), workspace=_ptr(ws))
        _launch('mep_diff_attn_bwd', bd, dev)
        return (None, None, None, None, dq, dk if need[5] else None, dv if need[6] else None, dlam)


def diff_attention(q, k, v, lam, *, mask=None, lengths=None, causal=False, q_start=None, scale=None):
    """The difference of two softmax maps, applied to the values: out = (A_1 - lam A_2) v [B, Tq, H, dv], with
    A_m = softmax(scale q_m k_m^T) over the keys that a query may see; a query that sees none gives zeros.

    q [B, Tq, H, 2, d], k [B, Tk, G, 2, d], v [B, Tk, G, dv] (any strides) of one type, d <= 128, dv <= 256; H a multiple of G:
    head h reads key head h // (H // G).  lam float32 [H] (learned per head) or [B, Tq, H] (per query).  scale: 1 / sqrt(d).
    What a query sees:
      mask      [B, Tk] or [B, Tq, Tk], bool, uint8 or float32: nonzero keeps a key (the loaders' masks of ones and zeros)
      lengths   int32 [B]: the keys at and behind it are not there (a padded batch, a cache)
      causal    query t of row b sees the keys up to q_start[b] + t; q_start int32 [B], Tk - Tq without it
    Keys past the lengths, past every query's causal reach or of a zero in a [B, Tk] mask never enter a result, whatever they
    hold; the keys that only some queries may see must be finite.  Scores, scale q_m k_m^T, must lie within 2^22: they are formed in
    float32, and past that the rounding of an exponent alone can pass a type's range.
    q, k, v and upstream gradients whose rows are not whole and aligned 16 bytes are copied first, a cache whole at every call.
    float32 with gradients is slower than elementary torch operations where heads are wider than 64.
    """
    _type_of(q, 'q')
    if q.dim() != 5 or k.dim() != 5 or v.dim() != 4 or q.shape[3] != 2 or k.shape[3] != 2 or q.shape[4] != k.shape[4] or \
            not q.shape[0] == k.shape[0] == v.shape[0] or k.shape[1:3] != v.shape[1:3]:
        raise ValueError('q, k, v must be [B, Tq, H, 2, d], [B, Tk, G, 2, d], [B, Tk, G, dv]; got %s, %s, %s'
                         % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    B, Tq, H, _, hd = q.shape
    Tk, G, dv = k.shape[1], k.shape[2], v.shape[3]
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError('q, k and v must be of one type; got %s, %s, %s' % (q.dtype, k.dtype, v.dtype))
    if not 1 <= hd <= _lib.DIFF_ATTN_MAX_D or not 1 <= dv <= _lib.DIFF_ATTN_MAX_DV:
        raise ValueError('head widths up to %d (q, k) and %d (v); got %d and %d'
                         % (_lib.DIFF_ATTN_MAX_D, _lib.DIFF_ATTN_MAX_DV, hd, dv))
    if G < 1 or H < 1 or H % G:
        raise ValueError('the query heads must be a multiple of the key heads; got %d and %d' % (H, G))
    if lam.dtype != torch.float32 or tuple(lam.shape) not in ((H,), (B, Tq, H)):
        raise ValueError('lam must be float32 [H] or [B, Tq, H]; got %s %s' % (tuple(lam.shape), lam.dtype))
    if mask is not None and (mask.dtype not in (torch.bool, torch.uint8, torch.float32) or
                             tuple(mask.shape) not in ((B, Tk), (B, Tq, Tk))):
        raise ValueError('mask must be bool, uint8 or float32 [B, Tk] or [B, Tq, Tk]; got %s %s' % (tuple(mask.shape), mask.dtype))
    for t, n in ((lengths, 'lengths'), (q_start, 'q_start')):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (B,) or not t.is_contiguous()):
            raise ValueError('%s must be contiguous int32 [B]; got %s %s' % (n, tuple(t.shape), t.dtype))
    if mask is not None and mask.requires_grad:
        raise ValueError('a mask has no gradient')
    if q_start is not None and not causal:
        raise ValueError('q_start places the queries of a causal call; causal is False')
    scale = hd ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale <= 1e6:
        raise ValueError('scale must be positive and at most 1e6; got %r' % (scale,))
    _on_device(q, k, v, lam, mask, lengths, q_start)
    return _DiffAttnFn.apply((bool(causal), scale, torch.is_grad_enabled()), mask, lengths, q_start, q, k, v, lam)
