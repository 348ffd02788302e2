"""The differential-attention block under torch.autocast: products in 16 bits on a float32 stream."""
import math

import pytest
import torch

from tests import diff_block_ref as ref
from tests.test_gpu_diff_attention import rand

pytestmark = pytest.mark.gpu


def parameters(E, H, G, d, dv):
    g = torch.Generator().manual_seed(3)
    lin = lambda i, o: (torch.randn(i, o, generator=g) / math.sqrt(i)).cuda().requires_grad_()  # noqa: E731
    one = lambda n: (1 + 0.1 * torch.randn(n, generator=g)).cuda().requires_grad_()  # noqa: E731
    return dict(w1=one(E), wq=lin(E, H * 2 * d), wk=lin(E, G * 2 * d), wv=lin(E, G * dv), lam=(0.2 + 0.6 * torch.rand(H, generator=g)).cuda().requires_grad_(),
                wh=one(dv), wo=lin(H * dv, E), w2=one(E), gate=one(E), scale=torch.tensor([0.9], device='cuda', requires_grad=True), w3=one(E))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('gated', ['channel', 'rows'])
def test_block(cuda, dtype, gated):
    """The block of the documentation.  Relative errors in the Frobenius norm: under autocast 9 tensors are rounded to 16 bits on the way
    (the norm's output and four weights at their products, projections, rotary, attention, its norm, the output projection), a
    gate of rows one more, independently, by half a step at most, and each changes what follows by at most 4 of its own relative size (a
    score's |s| <= 4 at unit variance); on the way back as many again.  A parameter's gradient sums rows of both signs, its errors as
    well: 2, and 4 where it is one sum or four (scale, lam), which may come out smaller than most."""
    from mep_amd import diff_block as db
    B, T, E, H, G, d, dv = 2, 70, 96, 4, 2, 32, 64
    p = parameters(E, H, G, d, dv)
    x = rand((B, T, E), torch.float32, 1)
    pos = torch.arange(T, device='cuda')
    freqs, amplitude = db.rotary_frequencies(d)
    lengths = torch.tensor([T, 40], dtype=torch.int32, device='cuda')
    up = [rand((B, T, E), torch.float32, 5 + i, grad=False) for i in range(2)]
    with torch.autocast('cuda', dtype=dtype):
        h = db.norm(x, p['w1'])
        q, k, v = (h @ p['wq']).view(B, T, H, 2, d), (h @ p['wk']).view(B, T, G, 2, d), (h @ p['wv']).view(B, T, G, dv)
        q, k = db.rotary(q, k, positions=pos, freqs=freqs, amplitude=amplitude)
        a = db.norm(db.diff_attention(q, k, v, p['lam'], lengths=lengths, causal=True), p['wh'])
        y = a.reshape(B, T, -1) @ p['wo']
        gate = p['gate'] if gated == 'channel' else torch.sigmoid(h @ p['wo'][:E])      # of 16 bits, as the product is
        out = db.norm_residual(y, x, p['w2'], gate=gate, scale=p['scale'], next_kind='rms', next_weight=p['w3'])
    assert q.dtype == a.dtype == y.dtype == dtype and out[0].dtype == out[1].dtype == torch.float32
    names = [n for n in p if gated == 'channel' or n != 'gate']
    got = torch.autograd.grad(out, [x] + [p[n] for n in names], up)
    w = {n: ref.wide(t) for n, t in p.items()}
    xw = ref.wide(x)
    h = ref.norm(xw, w['w1'], None, 'rms', 1e-6)
    q, k, v = (h @ w['wq']).view(B, T, H, 2, d), (h @ w['wk']).view(B, T, G, 2, d), (h @ w['wv']).view(B, T, G, dv)
    q, k = (ref.rotary(t, pos.cpu(), freqs.cpu(), 'half', amplitude) for t in (q, k))
    a = ref.norm(ref.diff_attention(q, k, v, w['lam'], ref.allowed(B, T, T, None, lengths, True, None)), w['wh'], None, 'rms', 1e-6)
    gate = w['gate'] if gated == 'channel' else torch.sigmoid(h @ w['wo'][:E])
    want = ref.norm_residual(a.reshape(B, T, -1) @ w['wo'], xw, w['w2'], None, 'rms', gate, w['scale'], 'rms', w['w3'], None, 1e-6)
    exact = torch.autograd.grad(want, [xw] + [w[n] for n in names], [t.cpu().double() for t in up])
    half = ref.half_step(dtype)
    for name, a, b, n, more in [('stream', out[0], want[0], 10, 1), ('normed', out[1], want[1], 10, 1)] + \
            [(m, a, b, 20, 4 if m in ('lam', 'scale') else 2) for m, a, b in zip(['x'] + names, got, exact)]:
        err, tol = float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm()), 4 * math.sqrt(n) * more * half
        print(name, '%.1e of %.1e' % (err, tol), flush=True)
        assert err <= tol, (name, err, tol)


def test_other_types_are_still_refused(cuda):
    """outside autocast, and of types that are not an activation's"""
    from mep_amd import diff_block as db
    y, x = rand((4, 8), torch.bfloat16, 1), rand((4, 8), torch.float32, 2)
    with pytest.raises(ValueError, match='residual'):
        db.norm_residual(y, x)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        assert db.norm_residual(y, x).dtype == torch.float32
        with pytest.raises(ValueError, match='residual'):
            db.norm_residual(y, x.double())
        with pytest.raises(ValueError, match='gate'):
            db.norm_residual(y, x, gate=torch.ones(8, dtype=torch.int32, device='cuda'))


def test_gate_of_a_product_on_a_float32_block(cuda):
    """y and the stream are float32, the gate comes out of a product; and all of 16 bits with a float32 gate stay in 16"""
    from mep_amd import diff_block as db
    y, x, g = (rand((3, 5, 16), torch.float32, i) for i in range(3))
    with pytest.raises(ValueError, match='gate'):
        db.norm_residual(y, x, gate=g.bfloat16())
    with torch.autocast('cuda', dtype=torch.bfloat16):
        for gate in (g.bfloat16(), g.bfloat16()[0, 0], g.bfloat16()[:, 0]):
            assert torch.equal(db.norm_residual(y, x, gate=gate), db.norm_residual(y, x, gate=gate.float()))
        assert torch.equal(db.norm_residual(y, None, gate=g.bfloat16()), db.norm_residual(y, None, gate=g.bfloat16().float()))
        assert db.norm_residual(y.bfloat16(), x.bfloat16(), gate=g[0, 0]).dtype == torch.bfloat16
