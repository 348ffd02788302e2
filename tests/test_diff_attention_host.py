"""What the differential-attention entry points work out on the host, on the CPU: workspaces, and what they turn down before any launch."""
import ctypes

import pytest

from mep_amd import _lib

F32, BF16, F16 = 0, 1, 2


def forward(type=F16, B=2, Tq=40, Tk=50, H=4, G=2, d=16, dv=32):
    """a descriptor of contiguous tensors (at an address that nothing reads here)"""
    at = 1 << 20
    return _lib.DiffAttnDesc(q=at, k=at, v=at, lam=at, out=at, stats=at, second=at, q_sB=Tq * H * 2 * d, q_sT=H * 2 * d, q_sH=2 * d, q_sM=d,
                             k_sB=Tk * G * 2 * d, k_sT=G * 2 * d, k_sH=2 * d, k_sM=d, v_sB=Tk * G * dv, v_sT=G * dv, v_sH=dv, lam_sH=1,
                             B=B, Tq=Tq, Tk=Tk, H=H, G=G, d=d, dv=dv, type=type, scale=0.25)


def backward(f, **k):
    at, H, dv = 1 << 20, f.H, f.dv
    return _lib.DiffAttnBwdDesc(**dict(dict(f=f, dout=at, o_sB=f.Tq * H * dv, o_sT=H * dv, o_sH=dv, dq=at, dk=at, dv=at, dlam=at, delta=at), **k))


@pytest.mark.parametrize('workspace', [0, (1 << 20) + 4])
def test_float16_backward_needs_its_workspace(workspace):
    rc = _lib.lib().mep_diff_attn_bwd(ctypes.byref(backward(forward(F16), workspace=workspace)), None)
    assert rc < 0
    buf = ctypes.create_string_buffer(256)
    _lib.lib().mep_last_error(buf, 256)
    assert b'workspace' in buf.value


@pytest.mark.parametrize('type', [F32, BF16, F16])
@pytest.mark.parametrize('wrong', [dict(k=0), dict(v=0), dict(k=(1 << 20) + 4), dict(v_sT=7), dict(k_sM=3)])
def test_backward_without_queries_still_reads_keys(type, wrong):
    """dk and dv of no queries are zeros, formed by the kernel that loads the keys: their addresses have to be there"""
    f = forward(type, Tq=0)
    for n, x in wrong.items():
        setattr(f, n, x)
    assert _lib.lib().mep_diff_attn_bwd(ctypes.byref(backward(f, workspace=1 << 20)), None) == -1000


@pytest.mark.parametrize('size', [dict(), dict(B=1, Tq=1, Tk=1, H=1, G=1), dict(B=1, Tq=4096, Tk=64, H=8, G=1), dict(B=3000, G=1, H=1), dict(Tq=0), dict(Tk=0)])
def test_workspace_bytes(size):
    """room for the float16 backward's sizes whatever is split, and none in the other types where nothing is"""
    n = _lib.lib().mep_diff_attn_bwd_workspace
    half, other = n(ctypes.byref(forward(F16, **size))), n(ctypes.byref(forward(BF16, **size)))
    f = forward(F16, **size)
    assert other >= 0 and half - other >= 16 * f.B * f.G and half % 16 == 0
    assert half - (other + 15) // 16 * 16 <= 16 * 64 * f.B * f.G
