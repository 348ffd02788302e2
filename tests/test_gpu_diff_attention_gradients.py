"""Gradients of mep_amd.diff_block.diff_attention by their whole error (the Frobenius norm), against the 64-bit form: keys and values
that have a mean, and float16 upstream gradients of any size."""
import math

import pytest
import torch

from tests import diff_block_ref as ref
from tests.test_gpu_diff_attention import rand

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]


def case(B, Tq, Tk, H, G, d, dv, dtype, k_mean, v_mean, v_std=1.0, seed=1):
    """keys and values with a mean of either sign in each channel"""
    g = torch.Generator().manual_seed(seed + 7)
    sign = lambda *s: (torch.randint(0, 2, s, generator=g) * 2 - 1).float()  # noqa: E731
    make = lambda shape, mean, std, at, tail: (  # noqa: E731
        (torch.randn(shape, generator=torch.Generator().manual_seed(at)) + mean * sign(*tail)) * std).to(dtype).cuda().requires_grad_()
    q = rand((B, Tq, H, 2, d), dtype, seed)
    k = make((B, Tk, G, 2, d), k_mean, 1.0, seed + 1, (2, d))
    v = make((B, Tk, G, dv), v_mean, v_std, seed + 2, (dv,))
    lam = (torch.rand(H, generator=g) * 0.6 + 0.2).cuda().requires_grad_()
    return q, k, v, lam


def check(q, k, v, lam, dout, by=None, **masks):
    """The error of a whole gradient.  With half = half a step of the type, dS = A (dP - D):

    dq   rounding dS adds at most half sqrt(sum dS^2 |k|^2) / sqrt(3) on average, independent from key to key.  A row's D may be off
         from what the row's sums say, by up to 3 times half / 2 sqrt(sum dS^2) in the root mean square over 32 rows before that is
         put right: 1.5 half sqrt(sum dS^2), which meets |sum A k| <= sqrt(sum A |k|^2).  Both together are under 2 half of
         S = sqrt(sum over rows of (sum dS^2) (sum A |k|^2)) plus sqrt(sum dS^2 |k|^2).
    dk   sums dS^T q of rows with their D as summed: 2 half sqrt(sum dS^2 |q|^2) for its 0.6.
    dv   sums P^T dO: likewise.
    Each is rounded once more (half, and half a subnormal step of every element).  float32's own sums are far below.
    by: dk and dv by that many keys at a time."""
    from mep_amd import diff_block as db
    B, Tq, H, _, d = q.shape
    Tk, G = k.shape[1], k.shape[2]
    n, sc = H // G, d ** -0.5
    half = ref.half_step(q.dtype)
    tiny = torch.finfo(q.dtype).smallest_normal * half
    got = torch.autograd.grad(db.diff_attention(q, k, v, lam, **masks), (q, k, v, lam), dout)
    w = [ref.wide(t) for t in (q, k, v, lam)]
    ok = ref.allowed(B, Tq, Tk, masks.get('mask'), masks.get('lengths'), masks.get('causal', False), masks.get('q_start'))
    exact = torch.autograd.grad(ref.diff_attention(*w, ok), w, dout.cpu().double())
    with torch.no_grad():
        kk, vv, do = w[1].repeat_interleave(n, 2), w[2].repeat_interleave(n, 2), dout.cpu().double()
        s = torch.einsum('bthmd,bshmd->bhmts', w[0], kk) * sc
        a = torch.softmax(s.masked_fill(~ok[:, None, None], -1e300), -1) * ok.any(-1)[:, None, None, :, None]
        l = w[3].reshape(1, H, 1, 1)
        dp = torch.einsum('bthe,bshe->bhts', do, vv)
        ds = a * (dp[:, :, None] - (a * dp[:, :, None]).sum(-1, keepdim=True)) * torch.stack([torch.ones_like(l), l], 2) * sc
        k2 = (kk * kk).sum(-1).permute(0, 2, 3, 1)[:, :, :, None]          # [B, H, 2, 1, Tk]
        q2 = (w[0] * w[0]).sum(-1).permute(0, 2, 3, 1)[..., None]
        ds2 = ds * ds
        tq = math.sqrt(float((ds2 * k2).sum())) + math.sqrt(float((ds2.sum(-1) * (a * k2).sum(-1)).sum()))
        tk = (ds2 * q2).sum((0, 1, 2, 3))                                 # by key
        p = a[:, :, 0] - l * a[:, :, 1]
        tv = (p * p * (do * do).sum(-1).permute(0, 2, 1)[..., None]).sum((0, 1, 2))
    report = []
    parts = [('dq', got[0], exact[0], tq)]
    for i in range(0, Tk, by or Tk):
        at = slice(i, i + (by or Tk))
        parts += [('dk', got[1][:, at], exact[1][:, at], math.sqrt(float(tk[at].sum()))), ('dv', got[2][:, at], exact[2][:, at], math.sqrt(float(tv[at].sum())))]
    for name, x, e, t in parts:
        x = x.cpu().double()
        norm = float(e.norm())
        tol = half * (norm + 2 * t) + tiny * math.sqrt(e.numel())
        err = float((x - e).norm())
        report.append('%s %.2e of %.2e' % (name, err / (norm or 1.0), tol / (norm or 1.0)))
        if not (bool(x.isfinite().all()) and err <= tol):
            report[-1] += ' OFF'
    report = '; '.join(report)
    print(report, flush=True)
    assert 'OFF' not in report, report


MEANS = [(0.0, 0.0), (1.0, 1.0), (1.0, 3.0), (3.0, 3.0), (0.0, 3.0)]
MEAN_SIZES = [(1, 128, 4096, 1, 1, 64, 128), (1, 1024, 1024, 2, 1, 64, 64), (1, 200, 1500, 2, 1, 128, 128), (1, 130, 1000, 1, 1, 128, 256),
              (1, 200, 1500, 2, 1, 32, 64)]


@pytest.mark.parametrize('dtype', HALVES)
@pytest.mark.parametrize('size,k_mean,v_mean', [(s, *m) for s in MEAN_SIZES for m in MEANS] +
                         [((16, 160, 1024, 8, 8, 64, 128), *m) for m in (MEANS[1], MEANS[3])])
def test_means(cuda, size, k_mean, v_mean, dtype):
    """whole rows, shared heads, a row's keys shared by two waves (few workgroups) and not (the last: 256)"""
    a = case(*size, dtype, k_mean, v_mean)
    check(*a, rand((*size[:2], size[3], size[6]), dtype, 77, grad=False))


@pytest.mark.parametrize('dtype', HALVES)
def test_means_causal(cuda, dtype):
    check(*case(2, 700, 700, 4, 2, 64, 128, dtype, 2.0, 2.0), rand((2, 700, 4, 128), dtype, 77, grad=False), causal=True)


SIZES = [(1, 64, 4096, 1, 1, 64, 128), (1, 300, 700, 2, 1, 32, 64), (1, 70, 2, 2, 2, 64, 64), (1, 40, 1000, 2, 1, 128, 256),
         (1, 600, 100, 1, 1, 16, 32)]


@pytest.mark.parametrize('size', SIZES)
@pytest.mark.parametrize('std,v_std', [(1e-6, 1.0), (1e-4, 1.0), (1.0, 1.0), (700.0, 1.0), (1500.0, 4.0), (4000.0, 1.0), (4000.0, 0.01)])
def test_float16_upstream_gradients_of_any_size(cuda, size, std, v_std):
    """dP past float16's largest number and below its smallest, where the gradients are inside (what a loss scale does)"""
    a = case(*size, torch.float16, 0.0, 0.0, v_std)
    if size[2] < 10:      # two keys share a row's weight: their scores are made small, or dq would pass 65504 with dP
        with torch.no_grad():
            a[1].mul_(0.05)
    dout = rand((*size[:2], size[3], size[6]), torch.float16, 77, std, grad=False)
    check(*a, dout.clamp(-30000, 30000))


def test_float16_upstream_gradients_that_differ_by_rows(cuda):
    """rows' sizes 2^-16 to 2^10 in one block, growing along the queries and falling"""
    a = case(1, 256, 600, 2, 1, 64, 128, torch.float16, 0.0, 0.0)
    size = 2.0 ** torch.linspace(-16, 10, 256, device='cuda')[:, None, None]
    up = rand((1, 256, 2, 128), torch.float32, 77, grad=False)
    for way in (size, size.flip(0)):
        check(*a, (up * way).half())


@pytest.mark.parametrize('dtype', [torch.float32] + HALVES)
@pytest.mark.parametrize('size', [(1, 70, 200, 2, 1, 64, 128), (1, 200, 200, 2, 2, 16, 32), (1, 2, 1500, 4, 1, 64, 64), (1, 40, 100, 1, 1, 128, 256)])
def test_scores_up_to_their_limit(cuda, size, dtype):
    """Scores of up to 2^22: finite, and rows whose largest scores are alone by 64 or more (their roundings are 1 at most) give those keys'
    values, by the whole error.  Four operands and the result are rounded (2 half of |v_1| + |v_2|, independent), and each time that
    a larger score of the second map came up the one before it left half a step of at most 1.25 lam of its own value: H_47 = 4.4
    times in 47 tiles of keys, independent: sqrt(4.4) 1.25 0.8 = 2.1 half.  Together under 4."""
    from mep_amd import diff_block as db
    q, k, v, lam = case(*size, dtype, 0.0, 0.0)
    B, Tq, H, _, d = q.shape
    n = H // k.shape[2]
    score = lambda: torch.einsum('bthmd,bshmd->bhmts', q.detach().cpu().double(), k.detach().cpu().double().repeat_interleave(n, 2)) * d ** -0.5  # noqa: E731
    with torch.no_grad():
        f = math.sqrt(2.0 ** 22 / float(score().abs().max())) * 0.99
        q.mul_(f)
        k.mul_(f)
    s = score()
    assert 2.0 ** 21 < float(s.abs().max()) < 2.0 ** 22
    out = db.diff_attention(q, k, v, lam)
    got = torch.autograd.grad(out, (q, k, v, lam), rand(out.shape, dtype, 77, grad=False))
    assert all(bool(x.isfinite().all()) for x in (out, *got))
    top = s.topk(2, -1)
    alone = (top.values[..., 0] - top.values[..., 1] > 64).all(2)                  # [B, H, Tq], in both maps
    assert float(alone.double().mean()) > 0.9
    vv = v.detach().cpu().double().repeat_interleave(n, 2)
    pick = [torch.gather(vv.transpose(1, 2), 2, top.indices[:, :, m, :, :1].expand(-1, -1, -1, v.shape[-1])) for m in (0, 1)]
    want = pick[0] - lam.detach().cpu().double()[:, None, None] * pick[1]
    err = (out.detach().cpu().double().transpose(1, 2) - want)[alone]
    tol = 4 * (ref.half_step(dtype) + 16 * ref.U) * float((pick[0].abs() + pick[1].abs())[alone].norm())
    print('%.2e of %.2e' % (float(err.norm()), tol), flush=True)
    assert float(err.norm()) <= tol


def test_float16_captured_and_replayed(cuda):
    """a float16 training pass in a graph, on upstream gradients and values of other sizes at each replay, against the eager pass"""
    from mep_amd import diff_block as db
    a = [t.detach() for t in case(2, 150, 300, 4, 2, 64, 128, torch.float16, 0.0, 0.0)]
    up = rand((2, 150, 4, 128), torch.float16, 9, grad=False)

    def train():
        leaves = [t.detach().requires_grad_() for t in a]
        out = db.diff_attention(*leaves)
        return (out,) + torch.autograd.grad(out, leaves, up)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        train()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = train()
    for std, v_std in ((1.0, 1.0), (3000.0, 0.01), (1e-4, 4.0), (1000.0, 1.0)):
        up.copy_(rand(up.shape, torch.float16, 11, std, grad=False))
        a[2].copy_(rand(a[2].shape, torch.float16, 12, v_std, grad=False))
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, train()):
            assert torch.equal(x, y) and bool(x.isfinite().all())


@pytest.mark.parametrize('values', [[1e-3, 0.5], [-30.0, 0.2], [900.0, -900.0]])
def test_float16_lam_of_any_size(cuda, values):
    q, k, v, _ = case(1, 150, 500, 2, 1, 64, 64, torch.float16, 0.0, 0.0)
    check(q, k, v, torch.tensor(values, device='cuda', requires_grad=True), rand((1, 150, 2, 64), torch.float16, 77, grad=False))


@pytest.mark.parametrize('size', [(1, 600, 600, 2, 1, 64, 128), (1, 600, 600, 1, 1, 16, 32), (2, 300, 900, 2, 2, 128, 128)])
def test_float16_upstream_gradients_that_fall_along_a_causal_row(cuda, size):
    """the last keys' gradients come from rows that are 2^-24 of the first's"""
    a = case(*size, torch.float16, 0.0, 0.0)
    fall = 2.0 ** torch.linspace(9, -15, size[1], device='cuda')[:, None, None]
    up = rand((*size[:2], size[3], size[6]), torch.float32, 77, grad=False)
    check(*a, (up * fall).half(), by=100, causal=True)


def test_float16_rows_that_see_nothing(cuda):
    """whatever upstream gradients they have"""
    a = case(2, 200, 300, 2, 1, 64, 64, torch.float16, 0.0, 0.0)
    up = rand((2, 200, 2, 64), torch.float16, 77, 1e-3, grad=False)
    up[:, :50] = 60000.0
    check(*a, up, by=100, causal=True, q_start=torch.full((2,), -50, dtype=torch.int32, device='cuda'))
    mask = torch.ones(2, 200, 300, dtype=torch.bool, device='cuda')
    mask[:, :50] = False
    check(*a, up, by=100, mask=mask)
