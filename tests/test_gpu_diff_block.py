"""mep_amd.diff_block's operators as a block uses them, together, and the calls between operators: saved tensors that come
back elsewhere (checkpoints, offloading), calls without gradients, rows and keys split over workgroups, two streams at once."""
import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from tests import diff_block_ref as ref
from tests.test_gpu_diff_attention import case, check, rand

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


# ------------------------------------------------------------------ the block
def parameters(E, H, G, d, dv, seed=5):
    g = torch.Generator().manual_seed(seed)
    lin = lambda o, i: torch.randn(o, i, generator=g) / math.sqrt(i)  # noqa: E731
    return dict(n1=1 + 0.1 * torch.randn(E, generator=g), wq=lin(H * 2 * d, E), wk=lin(G * 2 * d, E), wv=lin(G * dv, E),
                nh=1 + 0.1 * torch.randn(dv, generator=g), lam=0.2 + 0.6 * torch.rand(H, generator=g), wo=lin(E, H * dv),
                n2=1 + 0.1 * torch.randn(E, generator=g), gate=0.5 + 0.1 * torch.randn(E, generator=g),
                scale=torch.tensor([0.9]), n3=1 + 0.1 * torch.randn(E, generator=g))


def block(x, p, H, G, d, dv, pos, freqs, lengths, ops):
    """norm, projections, rotary positions, differential attention, a norm of each head, projection, gate, residual and next norm"""
    B, T, _ = x.shape
    lin = lambda h, w: (h.reshape(B * T, -1) @ w.to(h.dtype).t().contiguous()).reshape(B, T, -1)  # noqa: E731
    h = ops.norm(x, p['n1'])
    q, k, v = (lin(h, p['w' + n]) for n in 'qkv')
    q, k = ops.rotary(q.reshape(B, T, H, 2, d), k.reshape(B, T, G, 2, d), pos, freqs)
    a = ops.attention(q, k, v.reshape(B, T, G, dv), p['lam'], lengths)
    a = ops.norm(a, p['nh'])
    return ops.residual(lin(a.reshape(B, T, H * dv), p['wo']), x, p)


class Own:
    @staticmethod
    def norm(x, w):
        from mep_amd import diff_block as db
        return db.norm(x, w)

    @staticmethod
    def rotary(q, k, pos, freqs):
        from mep_amd import diff_block as db
        return db.rotary(q, k, positions=pos, freqs=freqs)

    @staticmethod
    def attention(q, k, v, lam, lengths):
        from mep_amd import diff_block as db
        return db.diff_attention(q, k, v, lam, lengths=lengths, causal=True)

    @staticmethod
    def residual(y, x, p):
        from mep_amd import diff_block as db
        return db.norm_residual(y, x, p['n2'], gate=p['gate'], scale=p['scale'], next_kind='layer', next_weight=p['n3'])


class Wide:
    @staticmethod
    def norm(x, w):
        return ref.norm(x, w, None, 'rms', 1e-6)

    @staticmethod
    def rotary(q, k, pos, freqs):
        return ref.rotary(q, pos, freqs, 'half', 1.0), ref.rotary(k, pos, freqs, 'half', 1.0)

    @staticmethod
    def attention(q, k, v, lam, lengths):
        return ref.diff_attention(q, k, v, lam, ref.allowed(q.shape[0], q.shape[1], k.shape[1], None, lengths, True, None))

    @staticmethod
    def residual(y, x, p):
        return ref.norm_residual(y, x, p['n2'], None, 'rms', p['gate'], p['scale'], 'layer', p['n3'], None, 1e-6)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,T,E,H,G,d,dv', [(2, 50, 48, 3, 3, 16, 32), (2, 150, 96, 4, 2, 32, 64), (1, 7, 40, 2, 1, 20, 40)])
def test_block(cuda, B, T, E, H, G, d, dv, dtype):
    """Relative errors in the Frobenius norm.  The block rounds 9 tensors one after another (norm, three projections at once, rotary,
    attention, norm, projection, stream, norm), the way back as many: by half a step of the type at most, independently, so that n of them
    add up to sqrt(n).  In fp32 a product of up to 96 terms counts as sqrt(96) < 10 roundings more.  Each changes what follows by at
    most A times its own relative size; the largest A is a score's: |s| <= 4 at unit variance of q and k, and an error of s
    is one of its exponential, so A = 4.  A parameter's gradient sums rows of both signs, its errors as well: 2, and where
    it has few elements (lam, scale: 1 to 4 sums, any of which may happen to cancel) 16."""
    from mep_amd import diff_block as db
    p = parameters(E, H, G, d, dv)
    x = rand((B, T, E), dtype, 3, grad=False)
    dl = [rand((B, T, E), dtype, 4 + i, grad=False) for i in range(2)]
    pos = torch.arange(T)
    freqs, _ = db.rotary_frequencies(d, device='cpu')
    lengths = torch.tensor([T, max(1, T // 2)][:B], dtype=torch.int32)
    mine = {n: t.cuda().requires_grad_() for n, t in p.items()}
    xo = x.detach().requires_grad_()
    got = block(xo, mine, H, G, d, dv, pos.cuda(), freqs.cuda(), lengths.cuda(), Own)
    gg = torch.autograd.grad(got, [xo] + list(mine.values()), dl)
    wide = {n: t.double().requires_grad_() for n, t in p.items()}
    for n in ('wq', 'wk', 'wv', 'wo'):       # the weights as the products see them
        wide[n] = p[n].to(dtype).double().requires_grad_()
    xw = ref.wide(x)
    want = block(xw, wide, H, G, d, dv, pos, freqs, lengths, Wide)
    wg = torch.autograd.grad(want, [xw] + list(wide.values()), [t.cpu().double() for t in dl])
    once = ref.half_step(dtype) + (10 * ref.U if dtype == torch.float32 else 0.0)
    few = {'lam': 16, 'scale': 16, 'x': 1}
    for name, a, b, n, more in [('stream', got[0], want[0], 9, 1), ('normed', got[1], want[1], 9, 1)] + \
            [(m, a, b, 18, few.get(m, 2)) for m, a, b in zip(['x'] + list(p), gg, wg)]:
        err, tol = float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm()), 4 * math.sqrt(n) * more * once
        assert err <= tol, (name, err, tol)


# ------------------------------------------------------------------ saved tensors that come back elsewhere
def _calls():
    from mep_amd import diff_block as db
    freqs, amp = db.rotary_frequencies(8)
    pos = torch.arange(40, device='cuda')
    lengths = torch.tensor([40, 11], dtype=torch.int32, device='cuda')
    mask = (torch.arange(80, device='cuda').reshape(2, 40) % 7 != 3).float()
    y, x, gate = (rand((2, 40, 24), torch.bfloat16, 20 + i) for i in range(3))
    w, nw = rand((24,), torch.float32, 30), rand((24,), torch.float32, 31)
    wide = rand((2, 40, 2, 2, 24), torch.bfloat16, 32)       # of which 20 channels are read: copied by the call
    a = case(2, 40, 40, 2, 1, 16, 32, torch.bfloat16)
    return {
        'rotary': (lambda q, k: db.rotary(q, k, positions=pos, freqs=freqs, amplitude=amp), (a[0], a[1])),
        'residual': (lambda *t: db.norm_residual(t[0] * 1.0, t[1], t[3], gate=t[2], next_kind='layer', next_weight=t[4]), (y, x, gate, w, nw)),
        'attention': (lambda *t: (db.diff_attention(t[0] * 1.0, t[1] * 1.0, t[2], t[3], mask=mask, lengths=lengths),), a),
        'unaligned': (lambda q, k, v, lam: (db.diff_attention(q[..., :20], k * 1.0, v, lam),),
                      (wide, rand((2, 40, 1, 2, 20), torch.bfloat16, 33), a[2], a[3])),
    }


@pytest.mark.parametrize('name', ['rotary', 'residual', 'attention', 'unaligned'])
@pytest.mark.parametrize('way', ['checkpoint', 'offloaded'])
def test_saved_tensors_elsewhere(cuda, name, way):
    f, leaves = _calls()[name]
    outs = f(*leaves)
    ups = [rand(o.shape, o.dtype, 50 + i, grad=False) for i, o in enumerate(outs)]
    want = torch.autograd.grad(outs, leaves, ups)
    if way == 'checkpoint':
        outs = checkpoint(f, *leaves, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu():
            outs = f(*leaves)
    fill = [torch.full((2, 40, 2, 2, 24), float('nan'), dtype=torch.bfloat16, device='cuda') for _ in range(20)]
    got = torch.autograd.grad(outs, leaves, ups)
    del fill
    for x, y in zip(want, got):
        assert torch.equal(x, y)


def test_second_backward(cuda):
    f, leaves = _calls()['attention']
    out = f(*leaves)
    up = torch.ones_like(out[0])
    first = torch.autograd.grad(out, leaves, up, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(out, leaves, up)))


# ------------------------------------------------------------------ splits
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size,masks', [
    ((1, 600, 70, 1, 1, 16, 32), {}), ((1, 400, 130, 4, 2, 32, 64), {'causal': True}), ((1, 300, 40, 4, 1, 64, 128), {}),
    ((2, 500, 60, 1, 1, 100, 40), {'causal': True}), ((1, 280, 50, 2, 1, 128, 256), {})])
def test_rows_split(cuda, size, masks, dtype):
    """few keys and many rows: the gradients of keys and values are summed by several workgroups"""
    masks = dict(masks)
    if masks:
        masks['q_start'] = torch.full((size[0],), -100, dtype=torch.int32, device='cuda')     # the first 100 queries see nothing
    check(*case(*size, dtype), **masks)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('size', [(1, 40, 1100, 2, 1, 16, 32), (1, 100, 1030, 1, 1, 40, 200), (2, 3, 300, 4, 1, 72, 256), (2, 3, 1100, 4, 1, 72, 256)])
def test_keys_split(cuda, size, dtype):
    """few rows and many keys, with gradients"""
    lengths = torch.full((size[0],), size[2] - 90, dtype=torch.int32, device='cuda')
    check(*case(*size, dtype, lam='row'), lengths=lengths)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,G,Tk', [(7, 2, 1500), (300, 1, 200), (300, 1, 1024)])
def test_ragged_cache(cuda, B, G, Tk, dtype):
    """single tokens against caches of very different lengths, empty ones among them: workgroups share out the tiles of all"""
    H = 2 * G
    lengths = torch.tensor([(0, Tk, 1, 64, 65, Tk - 1, 700, 129)[i % 8] % (Tk + 1) for i in range(B)], dtype=torch.int32, device='cuda')
    check(*case(B, 1, Tk, H, G, 32, 64, dtype), grads=B < 10, lengths=lengths)


@pytest.mark.parametrize('dtype', TYPES)
def test_new_tokens_of_long_caches(cuda, dtype):
    """three new tokens a row at places of their own (one row's first sees nothing), masked keys, and the same call in a graph whose
    lengths, places and masks change between the replays"""
    from mep_amd import diff_block as db
    q, k, v, lam = case(4, 3, 1300, 4, 2, 20, 40, dtype)
    start = torch.tensor([1297, 5, -1, 700], dtype=torch.int32, device='cuda')
    lengths = torch.tensor([1300, 8, 3, 650], dtype=torch.int32, device='cuda')
    mask = (torch.arange(4 * 1300, device='cuda').reshape(4, 1300) % 11 != 4).to(torch.uint8)
    kw = dict(mask=mask, lengths=lengths, causal=True, q_start=start)
    check(q, k, v, lam, **kw)
    a = [t.detach() for t in (q, k, v, lam)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        db.diff_attention(*a, **kw)
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = db.diff_attention(*a, **kw)
    for step in range(4):
        lengths.copy_(torch.tensor([1300 - 400 * step, 0 if step == 2 else 900, 1300, 64 * step], dtype=torch.int32))
        start.copy_(torch.tensor([1000, 400 * step, 1297, -2], dtype=torch.int32))
        mask[1].fill_(step % 2)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, db.diff_attention(*a, **kw))


@pytest.mark.parametrize('size', [(2, 140, 70, 4, 4, 40, 160), (1, 140, 70, 8, 4, 40, 160), (1, 300, 70, 1, 1, 40, 160)])
@pytest.mark.parametrize('causal', [False, True])
def test_values_in_two_halves(cuda, size, causal):
    """over 128 value channels, with (batch, key head) pairs that go evenly over the XCDs, over some of them, and not"""
    check(*case(*size, torch.bfloat16), causal=causal)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('values', [[-0.5, -0.1], [0.0, 0.0], [0.0, -0.7], [1.0, -2.0]])
def test_any_lam(cuda, values, dtype):
    q, k, v, _ = case(1, 70, 90, 2, 1, 64, 64, dtype)
    check(q, k, v, torch.tensor(values, device='cuda', requires_grad=True))


# ------------------------------------------------------------------ calls
def test_lam_of_one_parameter(cuda):
    """a lam that is expanded from one value: its gradient is summed by torch"""
    from mep_amd import diff_block as db
    q, k, v, _ = (t.detach() for t in case(2, 30, 30, 4, 2, 16, 32, torch.float32))
    one = torch.tensor(0.4, device='cuda', requires_grad=True)
    per = torch.full((2, 30, 4), 0.4, device='cuda', requires_grad=True)
    up = rand((2, 30, 4, 32), torch.float32, 8, grad=False)
    a, = torch.autograd.grad(db.diff_attention(q, k, v, one.expand(2, 30, 4)), one, up)
    b, = torch.autograd.grad(db.diff_attention(q, k, v, per), per, up)
    assert abs(float(a) - float(b.sum())) <= 240 * ref.U * float(b.abs().sum())       # two sums of 240 terms


def test_without_gradients(cuda, monkeypatch):
    """parameters that need gradients, under no_grad: nothing is kept for a backward pass, and the results are the same"""
    from mep_amd import diff_block as db
    a = case(2, 64, 64, 4, 2, 16, 32, torch.bfloat16)
    y, w = rand((6, 24), torch.bfloat16, 1), rand((24,), torch.float32, 2)
    want = db.diff_attention(*a), db.norm(y, w)
    kept, launch = [], db._launch

    def see(name, desc, device):
        kept.append(desc.stats)
        launch(name, desc, device)

    monkeypatch.setattr(db, '_launch', see)
    with torch.no_grad():
        got = db.diff_attention(*a), db.norm(y, w)
    assert kept == [0, 0]
    assert all(torch.equal(x, z) for x, z in zip(want, got))


def test_two_streams_at_once(cuda):
    from mep_amd import diff_block as db
    a, b = case(2, 300, 300, 4, 2, 32, 64, torch.bfloat16), case(1, 1, 4000, 8, 2, 64, 128, torch.bfloat16, seed=9)
    y, w = rand((2000, 512), torch.bfloat16, 1), rand((512,), torch.float32, 2)
    up, uy = rand((2, 300, 4, 64), torch.bfloat16, 4, grad=False), rand((2000, 512), torch.bfloat16, 5, grad=False)

    def one():
        return torch.autograd.grad(db.diff_attention(*a), a, up)

    def two():
        return (db.diff_attention(*b),) + torch.autograd.grad(db.norm(y, w), (y, w), uy)

    want = one(), two()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = ([], [])
    for _ in range(5):
        for i, f in enumerate((one, two)):
            with torch.cuda.stream(streams[i]):
                got[i].append(f())
    torch.cuda.synchronize()
    for w_, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(x, z) for x, z in zip(w_, r))


def test_block_captured_and_replayed(cuda):
    """forward and backward of the block in one graph, replayed on new inputs against the eager result"""
    from mep_amd import diff_block as db
    B, T, E, H, G, d, dv = 2, 50, 48, 3, 3, 16, 32
    p = {n: t.cuda() for n, t in parameters(E, H, G, d, dv).items()}
    x, up = rand((B, T, E), torch.float32, 1, grad=False), rand((B, T, E), torch.float32, 2, grad=False)
    freqs, _ = db.rotary_frequencies(d)
    pos, lengths = torch.arange(T, device='cuda'), torch.tensor([T, 9], dtype=torch.int32, device='cuda')

    def step():
        leaves = {n: t.detach().requires_grad_() for n, t in p.items()}
        out = block(x, leaves, H, G, d, dv, pos, freqs, lengths, Own)
        return out + torch.autograd.grad(out, [leaves[n] for n in ('n1', 'nh', 'lam', 'n2', 'gate', 'scale', 'n3')], [up, up])

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (1, 2, 3):
        x.copy_(rand((B, T, E), torch.float32, 60 + seed, grad=False))
        lengths.copy_(torch.tensor([seed, T - seed], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        want = step()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
