"""Launches of mep_amd.diff_block.diff_attention with more workgroups than run at once, in every order that they are dealt out in, long
rows, and maps that nearly cancel."""
import math

import pytest
import torch

from tests import diff_block_ref as ref
from tests.test_gpu_diff_attention import TYPES, case, check, rand

pytestmark = pytest.mark.gpu
# B, T, H, G: over 256 workgroups of 128 rows, whose second 256 go the other way.  (Batch row, key head) pairs that go evenly over
# the 8 XCDs, those of which several XCDs share one, and others
ORDERS = [(7, 520, 8, 8), (4, 528, 16, 1), (43, 200, 3, 3), (17, 200, 8, 8), (2, 1100, 16, 1)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', ORDERS)
def test_causal_orders(cuda, size, dtype):
    B, T, H, G = size
    assert B * G * -(-T * (H // G) // 128) > 256
    check(*case(B, T, T, H, G, 16, 32, dtype), causal=True)


def test_orders_without_a_mask(cuda):
    for B, T, H, G in ((7, 520, 8, 8), (43, 200, 3, 3)):
        check(*case(B, T, T, H, G, 16, 32, torch.bfloat16))
    check(*case(19, 256, 256, 7, 7, 40, 160, torch.float16, seed=3), causal=True)      # values in two halves


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('causal', [False, True])
def test_long_rows(cuda, causal, dtype):
    check(*case(1, 2048, 2048, 2, 1, 64, 128, dtype), causal=causal)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('size', [(1, 96, 2000, 2, 1, 64, 128), (1, 1, 2000, 2, 1, 64, 128), (6, 700, 700, 8, 8, 16, 32), (1, 70, 1500, 1, 1, 100, 200)])
def test_maps_that_nearly_cancel(cuda, size, dtype):
    """What is rounded is the difference of the maps.  With rho, the estimate of lam's ratio that the operand f1 e_1 - f2 e_2 is formed
    with, off by the part delta of itself, the operand is at most |A_1 - lam A_2| + lam delta A_2 and A_2's own rounding counts
    lam delta: both by at most half a step, independent from key to key, and the output once more.  rho comes from the sums over
    some of the row's tiles of 32 keys; a ratio of sums lies between the least and the largest of the tiles', and so delta is at most
    the largest deviation of a tile's ratio from the row's.  The exponents add 64 roundings of fp32 of either map."""
    from mep_amd import diff_block as db
    B, Tq, Tk, H, G, d, dv = size
    q, k, v, lam = (t.detach() for t in case(*size, dtype))
    near = lambda x: torch.stack([x[..., 0, :], (x[..., 0, :].float() + 0.01 * rand(x[..., 0, :].shape, torch.float32, 9, grad=False)).to(dtype)], -2)  # noqa: E731
    q, k = near(q), near(k)
    lam.fill_(0.97)
    out = db.diff_attention(q, k, v, lam).cpu().double()
    w = [ref.wide(t).detach() for t in (q, k, v, lam)]
    kk, vv = w[1].repeat_interleave(H // G, 2), w[2].repeat_interleave(H // G, 2)
    a = torch.softmax(torch.einsum('bthmd,bshmd->bhmts', w[0], kk) * d ** -0.5, -1)
    want = torch.einsum('bhts,bshe->bthe', a[:, :, 0] - 0.97 * a[:, :, 1], vv)
    tile = lambda x: torch.nn.functional.pad(x, (0, -Tk % 32)).unflatten(-1, (-1, 32)).sum(-1)  # noqa: E731
    delta = (tile(a[:, :, 0]) / tile(a[:, :, 1]) - 1).abs().amax(-1, keepdim=True)
    v2 = (vv * vv).sum(-1).permute(0, 2, 1)[:, :, None]
    size_of = lambda x: math.sqrt(float((x * x * v2).sum()))  # noqa: E731
    half = ref.half_step(dtype)
    tol = half * (size_of((a[:, :, 0] - 0.97 * a[:, :, 1]).abs() + 0.97 * delta * a[:, :, 1]) + size_of(0.97 * delta * a[:, :, 1]) + float(want.norm())) + \
        64 * ref.U * size_of(a.sum(2))
    err = float((out - want).norm())
    print('%.2e of %.2e, of rounded maps %.2e' % (err, tol, half * size_of(a.sum(2))), flush=True)
    assert err <= tol and tol < 0.2 * half * size_of(a.sum(2))
