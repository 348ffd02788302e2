"""What mep_amd.diff_block refuses, on the CPU: arguments of another shape, type or range, tensors that are not on a GPU, and
descriptors that the library turns down before any launch."""
import ctypes

import pytest
import torch

from mep_amd import _lib
from mep_amd import diff_block as db


def t(*s, dtype=torch.float32):
    return torch.zeros(*s, dtype=dtype)


FREQS = torch.ones(4, dtype=torch.float64)
POS = torch.arange(3)


@pytest.mark.parametrize('kw', [
    dict(q=t(2, 3, 8)), dict(q=t(2, 3, 1, 8, dtype=torch.float64)), dict(q=t(2, 3, 1, 6)), dict(k=t(2, 4, 1, 8)), dict(k=t(1, 3, 1, 8)),
    dict(k=t(2, 3, 1, 10)), dict(k=t(2, 3, 1, 8, dtype=torch.bfloat16)), dict(freqs=FREQS.float()), dict(freqs=FREQS[::2]),
    dict(freqs=FREQS[:0]), dict(freqs=FREQS[None]), dict(positions=POS.float()), dict(positions=torch.arange(4)),
    dict(positions=torch.zeros(1, 3, dtype=torch.int64)), dict(layout='pairs')])
def test_rotary_refuses(kw):
    a = dict(q=t(2, 3, 1, 8), k=None, positions=POS, freqs=FREQS, layout='half')
    a.update(kw)
    with pytest.raises(ValueError):
        db.rotary(a.pop('q'), a.pop('k'), **a)


@pytest.mark.parametrize('kw', [dict(rot_dim=3), dict(rot_dim=0), dict(base=0.0), dict(factor=-1.0), dict(scaling='other'),
                                dict(rot_dim=2, scaling='ntk'), dict(scaling='parts'),
                                dict(scaling='parts', original_len=10, low_turns=2.0, high_turns=2.0)])
def test_rotary_frequencies_refuses(kw):
    with pytest.raises(ValueError):
        db.rotary_frequencies(**dict(dict(rot_dim=8, device='cpu'), **kw))


def test_rotary_frequencies():
    f, a = db.rotary_frequencies(8, 10000.0, device='cpu')
    torch.testing.assert_close(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    assert a == 1.0
    g, _ = db.rotary_frequencies(8, scaling='linear', factor=4.0, device='cpu')
    torch.testing.assert_close(g, f / 4)
    g, _ = db.rotary_frequencies(8, scaling='ntk', factor=4.0, device='cpu')      # the fastest pair stays, the slowest is divided
    torch.testing.assert_close(g[[0, 3]], torch.stack([f[0], f[3] / 4]))
    g, a = db.rotary_frequencies(8, scaling='parts', factor=4.0, original_len=1000, device='cpu')
    assert g[0] == f[0] and g[3] == f[3] / 4 and f[2] / 4 < g[2] < f[2] and abs(a - 1.1386294361119891) < 1e-15


@pytest.mark.parametrize('kw', [
    dict(y=t(2, 3, 8, dtype=torch.float64)), dict(y=t(2, 8193)), dict(y=t(2, 3, 0)), dict(residual=t(2, 3, 4)),
    dict(residual=t(2, 3, 8, dtype=torch.bfloat16)), dict(kind='batch'), dict(next_kind=None), dict(weight=t(7)), dict(weight=t(2, 8)),
    dict(weight=t(8, dtype=torch.bfloat16)), dict(bias=t(8, dtype=torch.float64)), dict(kind='none', weight=t(8)),
    dict(next_weight=t(8)), dict(weight=t(8), next_kind='rms', next_weight=t(8, dtype=torch.bfloat16)), dict(gate=t(3, 8)),
    dict(gate=t(8, dtype=torch.float16)), dict(gate=t(2, 3, 1)), dict(scale=t(2)), dict(scale=t(1, dtype=torch.bfloat16)),
    dict(eps=-1e-6), dict(eps=float('inf')), dict(eps=float('nan'))])
def test_norm_residual_refuses(kw):
    a = dict(y=t(2, 3, 8), residual=t(2, 3, 8))
    a.update(kw)
    if 'y' in kw and 'residual' not in kw:
        a['residual'] = a['y'].clone()
    with pytest.raises(ValueError):
        db.norm_residual(a.pop('y'), a.pop('residual'), **a)


def test_norm_refuses():
    with pytest.raises(ValueError):
        db.norm(t(2, 8), kind='none')


@pytest.mark.parametrize('kw', [
    dict(q=t(2, 5, 4, 8)), dict(q=t(2, 5, 4, 3, 8)), dict(q=t(3, 5, 4, 2, 8)), dict(q=t(2, 5, 3, 2, 8)), dict(q=t(2, 5, 4, 2, 7)),
    dict(q=t(2, 5, 4, 2, 8, dtype=torch.float64)), dict(k=t(2, 6, 2, 2, 8, dtype=torch.bfloat16)), dict(k=t(2, 7, 2, 2, 8)),
    dict(v=t(2, 6, 1, 8)), dict(v=t(2, 6, 2, 257)), dict(v=t(2, 6, 2, 0)), dict(q=t(2, 5, 4, 2, 129), k=t(2, 6, 2, 2, 129)),
    dict(lam=t(5)), dict(lam=t(4, dtype=torch.bfloat16)), dict(lam=t(2, 4, 5)), dict(mask=t(2, 5)), dict(mask=t(2, 6, 5)),
    dict(mask=t(2, 6, dtype=torch.bfloat16)), dict(mask=t(2, 6, dtype=torch.int64)), dict(lengths=t(2, dtype=torch.int64)),
    dict(lengths=t(1, dtype=torch.int32)), dict(q_start=t(2, dtype=torch.int32)), dict(causal=True, q_start=t(3, dtype=torch.int32)),
    dict(lengths=t(4, dtype=torch.int32)[::2]), dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')), dict(scale=2e6)])
def test_diff_attention_refuses(kw):
    a = dict(q=t(2, 5, 4, 2, 8), k=t(2, 6, 2, 2, 8), v=t(2, 6, 2, 8), lam=t(4))
    a.update(kw)
    with pytest.raises(ValueError):
        db.diff_attention(a.pop('q'), a.pop('k'), a.pop('v'), a.pop('lam'), **a)


def test_cpu_tensors_are_refused():
    for call in (lambda: db.rotary(t(2, 3, 1, 8), positions=POS, freqs=FREQS), lambda: db.norm(t(2, 8)),
                 lambda: db.norm_residual(t(2, 8), t(2, 8)),
                 lambda: db.diff_attention(t(2, 5, 4, 2, 8), t(2, 6, 2, 2, 8), t(2, 6, 2, 8), t(4))):
        with pytest.raises(RuntimeError, match='no CPU fallback'):
            call()


def _refused(name, desc):
    rc = getattr(_lib.lib(), name)(ctypes.byref(desc) if desc is not None else None, None)
    return rc == -1000 and name in _lib.last_error()


def test_descriptors_refused_before_any_launch():
    """pointers below are never read: every descriptor is turned down on the host"""
    for n in ('mep_rotary', 'mep_block_norm_fwd', 'mep_block_norm_bwd', 'mep_diff_attn_fwd', 'mep_diff_attn_bwd'):
        assert _refused(n, None), n

    def rot(**kw):
        d = _lib.RotaryDesc(freqs=16, pos=16, B=1, T=1, D=8, rot=8)
        d.x[0], d.y[0], d.H[0], d.M[0] = 16, 16, 1, 1
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    for kw in (dict(rot=10), dict(rot=3), dict(rot=0), dict(D=0), dict(type=3), dict(freqs=0), dict(pos=0), dict(B=-1), dict(B=1 << 30, T=1 << 20)):
        assert _refused('mep_rotary', rot(**kw)), kw

    def norm(**kw):
        return _lib.BlockNormDesc(**dict(dict(y=16, stream=16, rows=1, D=8, T=1, kind=1), **kw))

    for kw in (dict(D=0), dict(D=8193), dict(y=0), dict(stream=0), dict(type=-1), dict(wtype=1), dict(kind=3), dict(next_kind=-1),
               dict(gate_form=1), dict(gate=16), dict(gate=16, gate_form=4), dict(gate=16, gate_form=2, rows=3, T=2),
               dict(gate=16, gate_form=2, rows=65001, T=1), dict(gate=16, gate_form=3, type=1), dict(eps=-1.0), dict(rows=-1)):
        assert _refused('mep_block_norm_fwd', norm(**kw)), kw
        assert _refused('mep_block_norm_bwd', _lib.BlockNormBwdDesc(f=norm(**kw))), kw
    ok = norm(stats=16)
    for kw in (dict(), dict(dy=16, dnormed=16), dict(dy=16, dw=16), dict(dy=16, dw=16, n_sums=1), dict(dy=16, dgate_rows=16),
               dict(dy=16, dscale=16)):
        assert _refused('mep_block_norm_bwd', _lib.BlockNormBwdDesc(f=ok, **kw)), kw

    def attn(**kw):
        return _lib.DiffAttnDesc(**dict(dict(q=16, k=16, v=16, lam=16, out=16, B=1, Tq=1, Tk=1, H=1, G=1, d=8, dv=8, scale=1.0), **kw))

    for kw in (dict(B=-1), dict(Tq=-1), dict(Tk=-1), dict(H=0), dict(G=0), dict(H=3, G=2), dict(d=0), dict(d=129), dict(dv=0), dict(dv=257),
               dict(type=3), dict(scale=0.0), dict(scale=float('nan')), dict(mask=16), dict(mask_form=1), dict(mask_form=3, mask=16), dict(q=0),
               dict(k=0), dict(lam=0), dict(out=0), dict(Tk=1 << 30), dict(Tq=1 << 30), dict(B=1 << 20, Tq=1 << 20)):
        assert _refused('mep_diff_attn_fwd', attn(**kw)), kw
        assert _refused('mep_diff_attn_bwd', _lib.DiffAttnBwdDesc(f=attn(**kw), dout=16, delta=16)), kw
    for kw in (dict(q=8), dict(k=2), dict(v=4), dict(q_sT=4), dict(k_sM=2), dict(v_sH=1), dict(q_sT=1 << 23), dict(k_sM=1 << 28),
               dict(k_sT=-8), dict(q_sH=1 << 28), dict(stats=16), dict(second=16)):
        assert _refused('mep_diff_attn_fwd', attn(type=1, **kw)), kw
    for kw in (dict(), dict(x=16), dict(x=16, y=8), dict(x=16, y=16, n=0), dict(x=16, y=16, type=3), dict(x=16, y=16, B=-1), dict(x=16, y=16, M=0)):
        assert _refused('mep_pack_rows', _lib.PackRowsDesc(**dict(dict(B=1, T=1, H=1, M=1, n=8), **kw))), kw
    for kw in (dict(), dict(dout=16), dict(dout=16, delta=16, dk=16), dict(dout=8, delta=16)):
        assert _refused('mep_diff_attn_bwd', _lib.DiffAttnBwdDesc(f=attn(stats=16, second=16), **kw)), kw


def test_what_has_no_gradient_is_refused():
    with pytest.raises(ValueError, match='freqs'):
        db.rotary(t(1, 3, 2, 8), positions=POS, freqs=FREQS.clone().requires_grad_())
    with pytest.raises(ValueError, match='mask'):
        db.diff_attention(t(1, 3, 2, 2, 8), t(1, 3, 2, 2, 8), t(1, 3, 2, 8), t(2), mask=t(1, 3).requires_grad_())


def test_strides_whose_sum_passes_2_gib():
    """each stride is within its limit, but a tile's farthest element of fp32 is not"""
    strides = dict(q_sT=64, q_sH=(1 << 28) // 64 - 64, q_sM=(1 << 28) - 64)
    assert (64 * 64 + 64 * strides['q_sH'] + strides['q_sM']) * 4 >= (1 << 31) - 2048
    assert _refused('mep_diff_attn_fwd', _lib.DiffAttnDesc(q=16, k=16, v=16, lam=16, out=16, B=1, Tq=1, Tk=1, H=64, G=1, d=8, dv=8,
                                                           scale=1.0, **strides))
