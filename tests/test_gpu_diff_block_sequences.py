"""mep_amd.diff_block.norm_residual under a gate per sequence with more sequences than workgroups."""
import ctypes

import pytest
import torch

from mep_amd import _lib
from tests.test_gpu_diff_block_rows import TYPES, check_norm, norm_case


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape', [(700, 1, 40), (520, 3, 130), (1100, 2, 24), (600, 17, 16), (513, 1, 1000), (300, 2, 2500), (270, 1, 4200)])
def test_many_sequences(cuda, shape, dtype):
    for wtype, kind, next_kind, bias in ((torch.float32, 'rms', 'none', False), (dtype, 'layer', 'rms', True)):
        check_norm(norm_case(shape, dtype, wtype, kind, next_kind, 'sequence', bias, True), kind, next_kind)


@pytest.mark.gpu
def test_gate_alone_and_without(cuda):
    """the gate's gradient alone, and those of the others without it, are the whole backward's bits"""
    from mep_amd import diff_block as db
    t = norm_case((600, 2, 72), torch.bfloat16, torch.float32, 'rms', 'none', 'sequence', False, True)
    leaves = [t[n] for n in ('y', 'x', 'w', 'gate', 'scale')]
    run = lambda on: torch.autograd.grad(db.norm_residual(*(a if i in on else a.detach() for i, a in enumerate(leaves[:3])),  # noqa: E731
                                                          gate=leaves[3] if 3 in on else leaves[3].detach(),
                                                          scale=leaves[4] if 4 in on else leaves[4].detach()).sum(), [leaves[i] for i in on])
    whole = run(range(5))
    for on in ([3], [0, 1, 2, 4], [2], [0]):
        assert all(torch.equal(a, whole[i]) for a, i in zip(run(on), on))


@pytest.mark.parametrize('type', [0, 1, 2])
@pytest.mark.parametrize('D', [8, 128, 1000, 2048, 4096, 8192])
def test_partial_sums_do_not_grow_with_the_sequences(D, type):
    at = 1 << 20
    rows = []
    for nseq, T in ((1, 100000), (300, 7), (513, 1), (4096, 1), (65000, 1), (65000, 30)):
        d = _lib.BlockNormDesc(y=at, stream=at, gate=at, rows=nseq * T, D=D, T=T, kind=1, gate_form=2, type=type, wtype=type, gtype=type)
        rows.append(_lib.lib().mep_block_norm_partial(ctypes.byref(d)))
    assert 0 < min(rows) and max(rows) <= 1024, rows
