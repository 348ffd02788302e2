"""mep_amd.diff_block.diff_attention against its 64-bit form: types, widths, shared heads, masks, empty rows, lengths,
causal offsets, strides, gradients by formula and by differences, graphs and streams."""
import pytest
import torch

from tests import diff_block_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rand(shape, dtype, seed, std=1.0, grad=True):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda().requires_grad_(grad)


def case(B, Tq, Tk, H, G, d, dv, dtype, lam='head', seed=1, std=1.0):
    q, k, v = rand((B, Tq, H, 2, d), dtype, seed, std), rand((B, Tk, G, 2, d), dtype, seed + 1, std), rand((B, Tk, G, dv), dtype, seed + 2)
    g = torch.Generator().manual_seed(seed + 3)
    l = (torch.rand((H,) if lam == 'head' else (B, Tq, H), generator=g) * 0.6 + 0.2).cuda().requires_grad_()
    return q, k, v, l


def check(q, k, v, lam, grads=True, dout=None, scale=None, same_maps=False, **masks):
    """Errors counted where they arise.  A score's 2^(s c - m) is off by its rounding and by |s| roundings of fp32 (both of the sum
    over d and of the exponent): `terms` of them at the products' magnitudes.  P and dS are rounded once to the type (half a step each);
    the output or gradient once more (ref.close counts that one).  An operand of P or dS below the type's smallest normal number lies
    on the grid of its subnormals, smallest_normal * eps apart (2^-24 in float16): it is off by half of that whatever its size, which
    counts against the other operand, `low` per allowed pair."""
    from mep_amd import diff_block as db
    out = db.diff_attention(q, k, v, lam, scale=scale, **masks)
    B, Tq, H, _, d = q.shape
    Tk, G, dv = k.shape[1], k.shape[2], v.shape[3]
    n = H // G
    ok = ref.allowed(B, Tq, Tk, masks.get('mask'), masks.get('lengths'), masks.get('causal', False), masks.get('q_start'))
    used = ok.any(1) if masks.get('mask') is None or masks['mask'].dim() == 2 else torch.ones(B, Tk, dtype=torch.bool)
    w = [ref.wide(t) for t in (q, k, v, lam)]
    with torch.no_grad():   # what is never read takes no part in the 64-bit form either
        w[1][~used] = 0.0
        w[2][~used] = 0.0
    want = ref.diff_attention(*w, ok, scale)
    sc = d ** -0.5 if scale is None else scale
    # magnitudes, in 64 bits, of the sums of absolute terms
    with torch.no_grad():
        kk, vv = w[1].repeat_interleave(n, 2), w[2].repeat_interleave(n, 2)
        s = torch.einsum('bthmd,bshmd->bhmts', w[0], kk) * sc
        some = ok.any(-1)[:, None, None, :, None].double()
        a = torch.softmax(s.masked_fill(~ok[:, None, None], -1e300), -1) * some
        big = float((torch.einsum('bthmd,bshmd->bhmts', w[0].abs(), kk.abs()) * sc).max()) if Tk else 0.0
        lamb = w[3].expand(B, Tq, H).permute(0, 2, 1)[..., None].abs()
        both = a[:, :, 0] + lamb * a[:, :, 1]
        diff = (a[:, :, 0] - lamb * a[:, :, 1]).abs()
        upto = lambda x: x.cumsum(-1)[..., [min(32 * (i // 32) + 31, Tk - 1) for i in range(Tk)]] if Tk else x  # noqa: E731
        # rho, the estimate that f1 e_1 - f2 e_2 is formed with, comes from the keys that the wave has seen: the rounded operand is at most
        # A_1 + rho A_2 with rho <= lam (1.25 late + 0.25), late the ratio of the maps' sums over those keys.  Where two waves share a row,
        # one sees the even 32 of the keys and the other the odd,
        # and its own sums up to there stand in the same bound
        late = upto(a[:, :, 0]) / upto(a[:, :, 1]).clamp_min(1e-300)
        odd = (torch.arange(Tk) // 32 % 2).bool()
        for side in (odd, ~odd):
            own = upto(a[:, :, 0] * side) / upto(a[:, :, 1] * side).clamp_min(1e-300)
            late = torch.where(side, torch.maximum(late, own), late)
        fwd = diff if same_maps else a[:, :, 0] + lamb * a[:, :, 1] * (1.25 * late + 0.25)
    half = ref.half_step(q.dtype) if q.dtype != torch.float32 else 0.0
    terms = 64 + 16 * big + Tk / 8      # the exponents, and the sums over keys
    low = torch.finfo(q.dtype).smallest_normal * half
    pairs = ok.double()[:, None].expand(B, H, Tq, Tk)

    def tol(sum_abs, rounded, other):
        """fp32 roundings at the sum of absolute terms, half a step of the type per rounded operand, and its subnormals'"""
        return terms * ref.U * sum_abs + half * rounded + low * other

    tout = tol(torch.einsum('bhts,bshe->bthe', both, vv.abs()), torch.einsum('bhts,bshe->bthe', fwd, vv.abs()),
               torch.einsum('bhts,bshe->bthe', pairs, vv.abs()))
    ref.close(out, want, tout / ref.U, 1, 'out')
    assert torch.equal(out[~ok.any(-1).cuda()], torch.zeros_like(out[~ok.any(-1).cuda()])), 'empty rows'
    if not grads:
        return out
    dout = rand(out.shape, out.dtype, 77, grad=False) if dout is None else dout
    got = torch.autograd.grad(out, (q, k, v, lam), dout)
    exact = torch.autograd.grad(want, w, dout.cpu().double())
    with torch.no_grad():
        do = dout.cpu().double()
        dp = torch.einsum('bthe,bshe->bhts', do, vv)
        dpa = torch.einsum('bthe,bshe->bhts', do.abs(), vv.abs())
        D = (a * dp[:, :, None]).sum(-1, keepdim=True)
        Da = (a * dpa[:, :, None]).sum(-1, keepdim=True)
        sgn = torch.stack([torch.ones_like(lamb), lamb], 2)
        dsr = a * (dp[:, :, None] - D).abs() * sgn * sc          # what is rounded
        dsa = a * (dpa[:, :, None] + Da) * sgn * sc              # what fp32 sums of absolute terms may be off at
        tq = tol(torch.einsum('bhmts,bshmd->bthmd', dsa, kk.abs()), torch.einsum('bhmts,bshmd->bthmd', dsr, kk.abs()),
                 sc * torch.einsum('bhts,bshmd->bthmd', pairs, kk.abs()))
        group = lambda x: x.unflatten(2, (G, n)).sum(3)  # noqa: E731
        rows = Tq * n / 8
        tk = tol(group(torch.einsum('bhmts,bthmd->bshmd', dsa, w[0].abs())), group(torch.einsum('bhmts,bthmd->bshmd', dsr, w[0].abs())),
                 sc * group(torch.einsum('bhts,bthmd->bshmd', pairs, w[0].abs())))
        tv = tol(group(torch.einsum('bhts,bthe->bshe', both, do.abs())), group(torch.einsum('bhts,bthe->bshe', diff, do.abs())),
                 group(torch.einsum('bhts,bthe->bshe', pairs, do.abs())))
        tl = terms * ref.U * Da[:, :, 1, :, 0].permute(0, 2, 1)
        if lam.dim() == 1:
            tl = tl.sum((0, 1)) * (1 + B * Tq / 256)
    more = 1 + rows / terms
    for name, x, e, t in zip(('dq', 'dk', 'dv', 'dlam'), got, exact, (tq, tk * more, tv * more, tl)):
        ref.close(x, e, t / ref.U, 1, name)
    for x in got[1:3]:
        assert not bool(x[~used.cuda()].any()), 'a key that no query sees has no gradient'
    return out


SIZES = [  # B, Tq, Tk, H, G, d, dv
    (1, 1, 1, 1, 1, 1, 1), (2, 3, 5, 2, 1, 7, 9), (1, 32, 32, 1, 1, 16, 32), (2, 33, 65, 3, 3, 16, 32), (2, 50, 50, 3, 3, 16, 32),
    (1, 129, 100, 4, 2, 32, 64), (1, 70, 130, 2, 2, 40, 40), (1, 64, 96, 4, 1, 64, 64), (1, 130, 200, 2, 1, 64, 128),
    (1, 40, 70, 2, 2, 72, 72), (1, 37, 67, 2, 1, 128, 128), (1, 45, 90, 2, 1, 128, 256), (1, 35, 66, 1, 1, 100, 133)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', SIZES)
def test_sizes(cuda, size, dtype):
    check(*case(*size, dtype))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('lam', ['head', 'row'])
def test_causal(cuda, dtype, lam):
    check(*case(2, 150, 150, 4, 2, 32, 64, dtype, lam), causal=True)
    check(*case(1, 40, 170, 2, 1, 16, 32, dtype, lam), causal=True)      # the queries are the last ones
    check(*case(1, 170, 40, 2, 2, 16, 32, dtype, lam), causal=True)      # the first 130 queries see nothing
    q_start = torch.tensor([-5, 0, 60], dtype=torch.int32, device='cuda')
    check(*case(3, 40, 100, 2, 1, 16, 32, dtype, lam), causal=True, q_start=q_start)


def some_mask(shape, seed, p=0.6):
    return (torch.rand(shape, generator=torch.Generator().manual_seed(seed)) < p).cuda()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('as_type', [torch.bool, torch.uint8, torch.float32])
def test_masks(cuda, dtype, as_type):
    a = case(3, 50, 70, 4, 2, 16, 32, dtype)
    m = some_mask((3, 70), 1)
    m[1] = False                                   # a row without keys
    check(*a, mask=m.to(as_type))
    m = some_mask((3, 50, 70), 2)
    m[0, 3] = m[2, 49] = False
    check(*a, mask=m.to(as_type))
    check(*a, mask=m.to(as_type), causal=True, lengths=torch.tensor([0, 1, 69], dtype=torch.int32, device='cuda'))
    check(*a, mask=m.to(as_type).transpose(1, 2).contiguous().transpose(1, 2))     # keys not contiguous
    check(*a, mask=(m[:1, :, :].to(as_type)).expand(3, 50, 70))


def test_lengths(cuda):
    lengths = torch.tensor([0, 1, 64, 130, 200, -3], dtype=torch.int32, device='cuda')      # clamped to [0, Tk]
    for dtype in TYPES:
        a = case(6, 20, 130, 2, 1, 16, 32, dtype)
        got = check(*a, lengths=lengths.clamp(0, 130))
        from mep_amd import diff_block as db
        assert torch.equal(db.diff_attention(*a, lengths=lengths), got)


@pytest.mark.parametrize('dtype', TYPES)
def test_what_is_masked_may_hold_anything(cuda, dtype):
    """NaN and infinities in keys and values past the lengths, past the causal reach and under a key mask"""
    q, k, v, lam = case(2, 40, 100, 2, 1, 16, 32, dtype)
    lengths = torch.tensor([70, 33], dtype=torch.int32, device='cuda')
    q_start = torch.tensor([20, 3], dtype=torch.int32, device='cuda')
    mask = some_mask((2, 100), 5)
    for masks, hidden in ((dict(lengths=lengths), torch.arange(100, device='cuda') >= lengths[:, None]),
                          (dict(mask=mask), ~mask),
                          (dict(causal=True, q_start=q_start), torch.arange(100, device='cuda') >= q_start[:, None] + 40)):
        with torch.no_grad():
            k2, v2 = k.detach().clone(), v.detach().clone()
            for x in (k2, v2):
                y = x[hidden]
                y[:] = float('nan')
                y[..., ::3] = float('inf')
                x[hidden] = y
        check(q, k2.requires_grad_(), v2.requires_grad_(), lam, **masks)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('Tq', [1, 2, 5])
def test_single_tokens(cuda, dtype, Tq):
    """a cache longer than its contents, shared heads, a few queries"""
    a = case(3, Tq, 700, 8, 2, 64, 128, dtype)
    lengths = torch.tensor([700, Tq, 333], dtype=torch.int32, device='cuda')
    with torch.no_grad():
        check(*a, grads=False, causal=True, lengths=lengths, q_start=lengths - Tq)
        check(*a, grads=False, lengths=lengths)
        check(*a, grads=False)


def test_large_scores_and_equal_maps(cuda):
    """scores in the hundreds (the maximum is not folded into a logarithm of the sum), and two maps that are the same"""
    for dtype in TYPES:
        check(*case(1, 40, 80, 2, 1, 32, 64, dtype, std=8.0))
        q, k, v, lam = case(1, 40, 80, 2, 1, 32, 64, dtype)
        with torch.no_grad():
            q[..., 1, :] = q[..., 0, :]
            k[..., 1, :] = k[..., 0, :]
            lam.fill_(0.96875)
        check(q, k, v, lam, same_maps=True)


def test_scale(cuda):
    check(*case(1, 33, 40, 2, 1, 16, 32, torch.float32), scale=0.03)
    check(*case(1, 33, 40, 2, 1, 16, 32, torch.bfloat16), scale=1.7)


@pytest.mark.parametrize('dtype', TYPES)
def test_strides(cuda, dtype):
    """slices of one projection (aligned and not), head-major tensors, expanded keys, an expanded upstream gradient"""
    g = rand((2, 30, 2 * 2 * 16 * 3 + 3), dtype, 4, grad=False)
    _, k, v, lam = case(2, 40, 50, 2, 1, 16, 32, dtype)
    for off in (0, 1, 8):
        q = g[..., off:off + 64].unflatten(-1, (2, 2, 16)).requires_grad_()
        check(q, k, v, lam)
    q = rand((2, 2, 2, 30, 16), dtype, 5, grad=False).permute(0, 3, 1, 2, 4).requires_grad_()
    k2 = rand((2, 1, 2, 50, 16), dtype, 6, grad=False).permute(0, 3, 1, 2, 4).requires_grad_()
    v2 = rand((2, 1, 32, 50), dtype, 7, grad=False).permute(0, 3, 1, 2).requires_grad_()
    check(q, k2, v2, lam, dout=torch.ones(1, dtype=dtype, device='cuda').expand(2, 30, 2, 32))
    check(q, k2, v2, lam, dout=rand((2, 2, 30, 32), dtype, 8, grad=False).transpose(1, 2))
    one = rand((1, 50, 1, 2, 16), dtype, 9)
    check(q, one.expand(2, 50, 1, 2, 16).detach().requires_grad_(), v2, lam)


def test_partial_gradients(cuda):
    from mep_amd import diff_block as db
    q, k, v, lam = case(2, 30, 40, 2, 1, 16, 32, torch.float32)
    full = torch.autograd.grad(db.diff_attention(q, k, v, lam).sum(), (q, k, v, lam))
    for i in range(4):
        a = [t.detach().requires_grad_(i == n) for n, t in enumerate((q, k, v, lam))]
        (g,) = torch.autograd.grad(db.diff_attention(*a).sum(), (a[i],))
        assert torch.equal(g, full[i])


def test_empty(cuda):
    from mep_amd import diff_block as db
    lam = torch.ones(2, device='cuda', requires_grad=True)
    z = lambda *s: torch.zeros(*s, device='cuda', requires_grad=True)  # noqa: E731
    for B, Tq, Tk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = z(B, Tq, 2, 2, 8), z(B, Tk, 1, 2, 8), z(B, Tk, 1, 8)
        out = db.diff_attention(q, k, v, lam)
        g = torch.autograd.grad(out.sum(), (q, k, v, lam))
        assert out.shape == (B, Tq, 2, 8) and not out.any()
        assert all(a.shape == b.shape and not a.any() for a, b in zip(g, (q, k, v, lam)))


def test_differences(cuda):
    """the gradient against central differences of the forward, along one direction"""
    from mep_amd import diff_block as db
    a = case(1, 20, 30, 2, 1, 16, 32, torch.float32)
    u = rand((1, 20, 2, 32), torch.float64, 50, grad=False)
    v = [rand(t.shape, torch.float32, 60 + i, grad=False) for i, t in enumerate(a)]
    f = lambda h: (db.diff_attention(*[t.detach() + h * e for t, e in zip(a, v)], causal=True).double() * u).sum()  # noqa: E731
    g = torch.autograd.grad((db.diff_attention(*a, causal=True).double() * u).sum(), a)
    slope = sum(float((x.double() * e.double()).sum()) for x, e in zip(g, v))
    h = 2.0 ** -8
    num = float((f(h) - f(-h)) / (2 * h))
    # 1280 outputs off by ~2^-22 each, random: 2^-17 over 2 h = 2^-7; and the third derivative's h^2 term
    assert abs(num - slope) < 2.0 ** -8 + 256 * h * h * (1 + abs(slope)), (num, slope)


def test_same_results_again(cuda):
    from mep_amd import diff_block as db
    a = case(2, 200, 300, 8, 2, 64, 128, torch.bfloat16)
    run = lambda: torch.autograd.grad(db.diff_attention(*a), a, torch.ones(2, 200, 8, 128, dtype=torch.bfloat16, device='cuda'))  # noqa: E731
    first = run()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, run()))


def test_on_another_stream(cuda):
    from mep_amd import diff_block as db
    a = [t.detach() for t in case(2, 64, 600, 4, 2, 64, 128, torch.bfloat16)]
    want = db.diff_attention(*a)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = db.diff_attention(*a)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)


def test_captured_and_replayed(cuda):
    """a training pass and a single-token pass in two graphs, replayed in turn on new inputs, each replay against the eager result"""
    from mep_amd import diff_block as db
    a = [t.detach() for t in case(2, 60, 60, 4, 2, 16, 32, torch.bfloat16)]
    b = [t.detach() for t in case(2, 1, 900, 4, 2, 64, 128, torch.float16)]
    lengths = torch.tensor([900, 20], dtype=torch.int32, device='cuda')
    up = rand((2, 60, 4, 32), torch.bfloat16, 9, grad=False)

    def train():
        leaves = [t.detach().requires_grad_() for t in a]
        out = db.diff_attention(*leaves, causal=True)
        return (out,) + torch.autograd.grad(out, leaves, up)

    def token():
        return (db.diff_attention(*b, lengths=lengths),)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        train(), token()
    torch.cuda.current_stream().wait_stream(st)
    graphs = []
    for f in (train, token):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, f, out))
    for seed in (1, 2, 3):
        with torch.no_grad():
            for i, t in enumerate(a + b):
                t.copy_(rand(t.shape, t.dtype, 100 * seed + i, 0.5, grad=False))
            lengths.copy_(torch.tensor([300 * seed, 900 - seed], dtype=torch.int32))
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, f, out in graphs:
            for x, y in zip(out, f()):
                assert torch.equal(x, y)
