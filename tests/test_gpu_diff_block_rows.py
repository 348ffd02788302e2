"""Rotary positions and the norms around a block (mep_amd.diff_block) against 64-bit forms: types, layouts, odd
widths, strides, far positions, gradients by formula and by differences, graphs, streams."""
import pytest
import torch

from tests import diff_block_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rand(shape, dtype, seed, std=1.0, mean=0.0, grad=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * std + mean).to(dtype).cuda()
    return x.requires_grad_(grad)


# ------------------------------------------------------------------ rotary
# |y| error: cosine and sine are off by under 4 roundings (the angle's, the series' and the amplitude's), the two products
# and their sum by 3 more, each at A (|x1| + |x2|); 16 covers both
ROTARY = [(1, 1, 1, 2, 2, 'half'), (2, 5, 3, 8, 8, 'half'), (2, 5, 3, 8, 8, 'interleaved'), (1, 7, 2, 64, 32, 'half'),
          (1, 7, 2, 64, 48, 'interleaved'), (3, 4, 5, 20, 6, 'half'), (3, 4, 5, 21, 6, 'interleaved'),
          (2, 3, 4, 128, 128, 'half'), (2, 130, 9, 128, 64, 'interleaved'), (1, 2, 1, 256, 254, 'half')]


def rotary_mag(x, r, layout, amplitude):
    a = x.detach().cpu().double().abs()
    i, j = (slice(0, r // 2), slice(r // 2, r)) if layout == 'half' else (slice(0, r, 2), slice(1, r, 2))
    m = torch.zeros_like(a)
    m[..., i] = m[..., j] = amplitude * (a[..., i] + a[..., j])
    return m


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,T,H,D,r,layout', ROTARY)
def test_rotary(cuda, B, T, H, D, r, layout, dtype):
    from mep_amd import diff_block as db
    q, k = rand((B, T, H, D), dtype, 1), rand((B, T, 2, 2, D), dtype, 2)
    freqs, amp = db.rotary_frequencies(r, scaling='parts', factor=4.0, original_len=4096)
    pos = torch.randint(0, 1000000, (B, T), generator=torch.Generator().manual_seed(3)).cuda()
    dq, dk = rand(q.shape, dtype, 4, grad=False), rand(k.shape, dtype, 5, grad=False)
    out = db.rotary(q, k, positions=pos, freqs=freqs, layout=layout, amplitude=amp)
    grads = torch.autograd.grad(out, (q, k), (dq, dk))
    for x, y, g, dx, n in zip((q, k), out, (dq, dk), grads, 'qk'):
        w = ref.wide(x)
        want = ref.rotary(w, pos.cpu(), freqs.cpu(), layout, amp)
        assert y.is_contiguous()
        ref.close(y, want, rotary_mag(x, r, layout, amp), 16, n)
        (dw,) = torch.autograd.grad(want, w, g.cpu().double())
        ref.close(dx, dw, rotary_mag(g, r, layout, amp), 16, 'd' + n)
        assert torch.equal(y[..., r:], x[..., r:])


@pytest.mark.parametrize('scaling', [None, 'linear', 'ntk', 'parts'])
def test_rotary_far_positions_and_scalings(cuda, scaling):
    """positions up to 2^30 and behind zero; [T] positions of both integer types"""
    from mep_amd import diff_block as db
    freqs, amp = db.rotary_frequencies(32, base=500000.0, scaling=scaling, factor=8.0, original_len=8192)
    for p in (torch.tensor([0, 1, 12345, 2 ** 30, -77], dtype=torch.int32), torch.tensor([2 ** 31 + 5, 2 ** 40, -1, 3, 9])):
        x = rand((2, 5, 3, 32), torch.float32, 7)
        y = db.rotary(x, positions=p.cuda(), freqs=freqs, amplitude=amp)
        ref.close(y, ref.rotary(ref.wide(x), p, freqs.cpu(), 'half', amp), rotary_mag(x, 32, 'half', amp),
                  16 + (float(p.abs().max()) * 2.0 ** -52 * 8) / ref.U, scaling)   # + the angle's own 64-bit roundings


def test_rotary_strides(cuda):
    """slices of one fused projection, a transposed [B, H, T, D] tensor, expanded batches and gradients"""
    from mep_amd import diff_block as db
    freqs, amp = db.rotary_frequencies(16)
    pos = torch.arange(6).cuda()
    fused = rand((2, 6, 3 * 4 * 16 + 1), torch.bfloat16, 1, grad=False)
    for x in (fused[..., :64].unflatten(-1, (4, 16)), fused[..., 65:129].unflatten(-1, (4, 16)), fused[..., 1:].unflatten(-1, (12, 16)),
              rand((2, 4, 6, 16), torch.bfloat16, 2, grad=False).transpose(1, 2),
              rand((1, 6, 4, 16), torch.bfloat16, 3, grad=False).expand(2, 6, 4, 16),
              rand((2, 6, 16, 4), torch.bfloat16, 4, grad=False).transpose(2, 3)):
        y = db.rotary(x, positions=pos, freqs=freqs)
        ref.close(y, ref.rotary(ref.wide(x), pos.cpu(), freqs.cpu(), 'half', 1.0), rotary_mag(x, 16, 'half', 1.0), 16)
    x = rand((2, 6, 4, 16), torch.float32, 5)
    db.rotary(x, positions=pos, freqs=freqs).sum().backward()      # an expanded upstream gradient
    w = ref.wide(x)
    ref.rotary(w, pos.cpu(), freqs.cpu(), 'half', 1.0).sum().backward()
    ref.close(x.grad, w.grad, 2.0, 16)


def test_rotary_empty(cuda):
    from mep_amd import diff_block as db
    freqs, _ = db.rotary_frequencies(8)
    q, k = db.rotary(torch.zeros(2, 0, 3, 8, device='cuda'), torch.zeros(2, 0, 1, 8, device='cuda'),
                     positions=torch.zeros(2, 0, dtype=torch.int64, device='cuda'), freqs=freqs)
    assert q.shape == (2, 0, 3, 8) and k.shape == (2, 0, 1, 8)
    k = rand((2, 3, 2, 8), torch.float32, 1)
    pos = torch.arange(3).cuda()
    _, y = db.rotary(torch.zeros(2, 3, 0, 8, device='cuda'), k, positions=pos, freqs=freqs)
    ref.close(y, ref.rotary(ref.wide(k), pos.cpu(), freqs.cpu(), 'half', 1.0), rotary_mag(k, 8, 'half', 1.0), 16)


# ------------------------------------------------------------------ norms
# A row's statistics sum at most 16 values in a lane and 9 levels over lanes and waves: under 32 roundings of the mean
# magnitude; a gradient meets four such sums.  256 covers a chain of them at the magnitudes below.
ROWS = 256


def norm_case(shape, dtype, wtype, kind, next_kind, gate, bias, learned, seed=11, eps=1e-5):
    D = shape[-1]
    t = {'y': rand(shape, dtype, seed, mean=0.3), 'x': rand(shape, dtype, seed + 1)}
    t['w'] = rand((D,), wtype, seed + 2, 0.2, 1.0) if kind != 'none' else None
    t['b'] = rand((D,), wtype, seed + 3, 0.2) if kind != 'none' and bias else None
    t['nw'] = rand((D,), wtype, seed + 4, 0.2, 1.0) if next_kind != 'none' else None
    t['nb'] = rand((D,), wtype, seed + 5, 0.2) if next_kind != 'none' and bias else None
    gshape = {'none': None, 'channel': (D,), 'sequence': (shape[0], D), 'full': shape}[gate]
    t['gate'] = None if gshape is None else rand(gshape, dtype if gate == 'full' else wtype, seed + 6, 0.5, 0.5)
    t['scale'] = torch.tensor([0.7], device='cuda', requires_grad=True) if learned else 1.3
    return t


def check_norm(t, kind, next_kind, eps=1e-5, upstream=(True, True)):
    from mep_amd import diff_block as db
    out = db.norm_residual(t['y'], t['x'], t['w'], t['b'], kind=kind, gate=t['gate'], scale=t['scale'], next_kind=next_kind,
                           next_weight=t['nw'], next_bias=t['nb'], eps=eps)
    out = out if isinstance(out, tuple) else (out,)
    names = [n for n in ('y', 'x', 'w', 'b', 'gate', 'scale', 'nw', 'nb') if torch.is_tensor(t[n])]
    w = {n: ref.wide(t[n]) if torch.is_tensor(t[n]) else t[n] for n in t}
    want = ref.norm_residual(w['y'], w['x'], w['w'], w['b'], kind, w['gate'], w['scale'], next_kind, w['nw'], w['nb'], eps)
    ups = [rand(o.shape, o.dtype, 31 + i, grad=False) for i, o in enumerate(out)]
    on = [i for i in range(len(out)) if upstream[i]]
    got = torch.autograd.grad([out[i] for i in on], [t[n] for n in names], [ups[i] for i in on], allow_unused=True)
    exact = torch.autograd.grad([want[i] for i in on], [w[n] for n in names], [ups[i].cpu().double() for i in on], allow_unused=True)
    # magnitudes: of a row's largest value, and of the sums that a column gathers
    row = lambda z: z.detach().abs().amax(-1, keepdim=True) + 1.0  # noqa: E731
    for i, o in enumerate(out):
        ref.close(o, want[i], row(want[i]) + row(want[0]), ROWS, 'out %d' % i)
    D = t['y'].shape[-1]
    r = lambda z: 1.0 / torch.sqrt((z.detach() - z.detach().mean(-1, keepdim=True)).square().mean(-1, keepdim=True) + eps)  # noqa: E731
    g = sum(row(ups[i].cpu().double()) for i in on) * (1.0 + (r(want[0]) if next_kind != 'none' else 0.0)) * 4.0
    n = t['y'].numel() // D
    for name, a, e in zip(names, got, exact):
        if e is None:
            assert a is None or float(a.abs().max()) == 0.0, name
            continue
        if name in ('y', 'x') or (name == 'gate' and e.shape == w['y'].shape):
            mag = g * (2.0 + (r(w['y']) if name == 'y' and kind != 'none' else 0.0)) * 4.0
        else:   # sums of n rows (or all elements) of terms of about the magnitude g
            mag = float(g.mean()) * 4.0 * (n if name != 'scale' else n * D) ** 0.5 * 4.0
        ref.close(a, e, mag, ROWS, 'd' + name)
    return out


NORM_SHAPES = [(1, 1, 1), (2, 3, 8), (3, 5, 7), (2, 17, 96), (1, 9, 128), (2, 7, 130), (3, 4, 512), (2, 5, 1000), (2, 3, 1537),
               (2, 5, 2048), (3, 2, 4096), (1, 3, 4100), (1, 2, 8192), (1, 2, 8191)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', NORM_SHAPES)
def test_norm_residual_widths(cuda, shape, dtype):
    check_norm(norm_case(shape, dtype, torch.float32, 'layer', 'rms', 'channel', True, True), 'layer', 'rms')


@pytest.mark.parametrize('dtype,wtype', [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize('gate', ['none', 'channel', 'sequence', 'full'])
@pytest.mark.parametrize('kind,next_kind', [('rms', 'layer'), ('layer', 'none'), ('none', 'rms'), ('none', 'none'), ('rms', 'rms')])
def test_norm_residual_forms(cuda, kind, next_kind, gate, dtype, wtype):
    check_norm(norm_case((3, 50, 96), dtype, wtype, kind, next_kind, gate, kind == 'rms', gate == 'full'), kind, next_kind)
    check_norm(norm_case((2, 3, 600), dtype, wtype, kind, next_kind, gate, kind == 'rms', gate == 'full'), kind, next_kind)


@pytest.mark.parametrize('upstream', [(True, False), (False, True)])
def test_norm_residual_one_output_used(cuda, upstream):
    check_norm(norm_case((2, 9, 300), torch.float32, torch.float32, 'rms', 'layer', 'channel', True, True), 'rms', 'layer',
               upstream=upstream)


def test_norm_residual_many_rows(cuda):
    """more rows than workgroups walk at once, sequences of an odd length"""
    check_norm(norm_case((7, 1237, 64), torch.bfloat16, torch.float32, 'rms', 'rms', 'sequence', False, True), 'rms', 'rms')
    check_norm(norm_case((1, 9001, 40), torch.float32, torch.float32, 'layer', 'rms', 'channel', True, True), 'layer', 'rms')


@pytest.mark.parametrize('kind', ['rms', 'layer'])
def test_norm_alone(cuda, kind):
    from mep_amd import diff_block as db
    x, w = rand((4, 6, 3, 24), torch.bfloat16, 1), rand((24,), torch.float32, 2, 0.2, 1.0)
    g = rand(x.shape, torch.bfloat16, 3, grad=False)
    y = db.norm(x, w, kind=kind, eps=1e-5)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    a, b = ref.wide(x), ref.wide(w)
    want = ref.norm(a, b, None, kind, 1e-5)
    ex, ew = torch.autograd.grad(want, (a, b), g.cpu().double())
    ref.close(y, want, 8.0, ROWS)
    ref.close(dx, ex, 32.0, ROWS)
    ref.close(dw, ew, 32.0 * 72 ** 0.5, ROWS)
    assert db.norm(torch.zeros(0, 24, device='cuda'), w).shape == (0, 24)


def test_norm_strided_rows_and_expanded_gradients(cuda):
    from mep_amd import diff_block as db
    big = rand((6, 10, 50), torch.float32, 1, grad=False)
    w = rand((16,), torch.float32, 2, 0.2, 1.0)
    for x in (big[:, :, 3:19], big[:, ::2, 8:24], big.transpose(0, 1)[:, :, :16], big[:1, :, :16].expand(6, 10, 16), big[:, :16, 0:10].transpose(1, 2)[:, :, :10]):
        ww = w if x.shape[-1] == 16 else None
        ref.close(db.norm(x, ww), ref.norm(ref.wide(x), None if ww is None else ref.wide(ww), None, 'rms', 1e-6), 8.0, ROWS)
    x = rand((5, 16), torch.float32, 3)
    a, b = ref.wide(x), ref.wide(w)
    gx, gw = torch.autograd.grad(db.norm(x, w).sum(), (x, w))
    ex, ew = torch.autograd.grad(ref.norm(a, b, None, 'rms', 1e-6).sum(), (a, b))
    ref.close(gx, ex, 16.0, ROWS)
    ref.close(gw, ew, 16.0, ROWS)


def test_norm_empty_rows_give_zero_parameter_gradients(cuda):
    from mep_amd import diff_block as db
    y, w = torch.zeros(2, 0, 8, device='cuda', requires_grad=True), rand((8,), torch.float32, 2)
    gate = rand((2, 8), torch.float32, 3)
    s, h = db.norm_residual(y, y, w, gate=gate, next_kind='rms')
    dw, dg, dy = torch.autograd.grad((s, h), (w, gate, y), (torch.zeros_like(s), torch.zeros_like(h)))
    assert dy.shape == y.shape and not dw.any() and not dg.any()


def test_norm_differences(cuda):
    """the gradient against central differences of the forward, along one direction"""
    from mep_amd import diff_block as db
    t = norm_case((2, 6, 40), torch.float32, torch.float32, 'layer', 'rms', 'sequence', True, True)
    names = ['y', 'x', 'w', 'b', 'gate', 'scale', 'nw', 'nb']

    def f(move):
        u = {n: t[n].detach() + move * v[n] if move else t[n] for n in names}
        s, h = db.norm_residual(u['y'], u['x'], u['w'], u['b'], kind='layer', gate=u['gate'], scale=u['scale'], next_kind='rms',
                                next_weight=u['nw'], next_bias=u['nb'])
        return (s.double() * us).sum() + (h.double() * uh).sum()

    v = {n: rand(t[n].shape, torch.float32, 50 + i, grad=False) for i, n in enumerate(names)}
    us, uh = (rand((2, 6, 40), torch.float64, 70 + i, grad=False) for i in range(2))
    g = torch.autograd.grad(f(0.0), [t[n] for n in names])
    slope = sum(float((a.double() * v[n].double()).sum()) for a, n in zip(g, names))
    h = 2.0 ** -8
    num = float((f(h) - f(-h)) / (2 * h))
    # 960 outputs of rounding 2^-24 * ~4 each, random: under 2^-15 over 2 h = 2^-7; the third derivative's h^2 term
    assert abs(num - slope) < 2.0 ** -8 + 64 * h * h * (1 + abs(slope)), (num, slope)


# ------------------------------------------------------------------ streams, graphs
def test_rows_on_another_stream(cuda):
    from mep_amd import diff_block as db
    x, w = rand((64, 50, 96), torch.float32, 1), rand((96,), torch.float32, 2)
    want = db.norm(x, w)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = db.norm(x, w)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(y, want)


def test_rows_captured_and_replayed(cuda):
    """both directions in one graph, replayed on new inputs; every replay equals the eager result bit for bit"""
    from mep_amd import diff_block as db
    freqs, _ = db.rotary_frequencies(8)
    pos = torch.arange(50).cuda()
    sy, sx, w, gate = (rand(s, torch.float32, i, grad=False) for i, s in enumerate([(4, 50, 96), (4, 50, 96), (96,), (4, 96)]))
    up = rand((4, 50, 12, 8), torch.float32, 9, grad=False)

    def step():
        leaves = [t.detach().requires_grad_() for t in (sy, sx, w, gate)]
        s, h = db.norm_residual(leaves[0], leaves[1], leaves[2], gate=leaves[3], next_kind='layer')
        q = db.rotary((s + h).unflatten(-1, (12, 8)), positions=pos, freqs=freqs)
        return (s, h, q) + torch.autograd.grad(q, leaves, up)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        with torch.no_grad():
            sy.copy_(rand(sy.shape, torch.float32, 100 + seed, grad=False))
            gate.copy_(rand(gate.shape, torch.float32, 200 + seed, grad=False))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
