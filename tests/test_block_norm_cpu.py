"""Refusals of the fused residual / norm entry points that need no GPU."""
import ctypes

import pytest
import torch

import mia_amd
from mia_amd.block_norm import gated_residual_norm

P = ctypes.c_void_p(4096)


def _fwd(dtype=0, x=P, f=P, images=2, rows=3, C=16, post=0, w1=None, b1=None, pre=1, w2=P, b2=None, eps=1e-6, y=P, z=P, gate=None):
    mia_amd.lib().mia_blocknorm_fwd(dtype, x, f, images, rows, C, None, gate, post, w1, b1, pre, w2, b2, eps, y, z, None, None)


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=2), "bad dtype"), (dict(images=0), "bad shape"), (dict(rows=-1), "bad shape"), (dict(C=8193), "C <= 8192"),
    (dict(rows=1 << 40), "too many"), (dict(images=1 << 22, rows=1, gate=P), "gates of"), (dict(post=3, w1=P), "bad norm kind"), (dict(eps=-1.0), "eps"), (dict(x=None), "null"), (dict(z=None), "null"),
    (dict(w2=None), "comes with its weight"), (dict(w1=P), "comes with its weight"), (dict(post=1), "comes with its weight"),
    (dict(b1=P), "only then with a bias"), (dict(pre=0, w2=None, b2=P), "only then with a bias")])
def test_forward_entry_refuses(kw, match):
    with pytest.raises(mia_amd.MiaError, match=match):
        _fwd(**kw)


def test_backward_entry_refuses():
    lib = mia_amd.lib()
    need = lib.mia_blocknorm_ws_floats(2, 3, 16, 1)
    assert need >= 2 * 4 * 16

    def bwd(dy=P, dz=P, stats=P, ws=P, n=need, gate=P, pre=1, w2=P):
        lib.mia_blocknorm_bwd(0, dy, dz, P, P, stats, 2, 3, 16, None, gate, 0, None, None, pre, w2, ws, n, P, P, None, None, None, None,
                              None, None, None)
    for kw, match in ((dict(dy=None, dz=None), "null"), (dict(stats=None), "null"), (dict(ws=None), "null"), (dict(n=need - 1), "too small"),
                      (dict(pre=0, w2=None), "only then with a gradient")):
        with pytest.raises(mia_amd.MiaError, match=match):
            bwd(**kw)


def test_wrapper_refuses():
    x, w = torch.zeros(2, 3, 16), torch.ones(16)
    for kw, err, match in (
            (dict(pre_weight=w), RuntimeError, "no CPU path"),
            (dict(pre_weight=w, post="batch"), ValueError, "norms are"),
            (dict(), ValueError, "pre_weight"),
            (dict(pre=None, pre_weight=w), ValueError, "no weight"),
            (dict(pre=None, pre_bias=w), ValueError, "no weight"),
            (dict(pre_weight=w, post="rms"), ValueError, "post_weight"),
            (dict(pre_weight=w, scale=torch.ones(15)), ValueError, "scale must be fp32"),
            (dict(pre_weight=w.bfloat16()), ValueError, "pre_weight must be fp32"),
            (dict(pre_weight=w, gate=torch.ones(3, 16)), ValueError, "gate must be fp32"),
            (dict(pre_weight=w, eps=-1e-6), ValueError, "eps"),
            (dict(pre_weight=w, eps=float("nan")), ValueError, "eps")):
        with pytest.raises(err, match=match):
            gated_residual_norm(x, x, **kw)
    with pytest.raises(TypeError, match="both"):
        gated_residual_norm(x, x.bfloat16(), pre_weight=w)
    with pytest.raises(TypeError, match="both"):
        gated_residual_norm(x.double(), x.double(), pre_weight=w)
    with pytest.raises(ValueError, match="one shape"):
        gated_residual_norm(x, x[:1], pre_weight=w)
    with pytest.raises(ValueError, match="8192"):
        gated_residual_norm(torch.zeros(1, 8200), torch.zeros(1, 8200), pre=None)
    with pytest.raises(ValueError, match="two dimensions"):
        gated_residual_norm(torch.zeros(16), torch.zeros(16), pre=None, gate=torch.ones(16, 16))


def test_scratch_alignment_is_checked():
    """Statistics are read and written 16 bytes at a time, the workspace holds doubles behind its rows."""
    lib, odd = mia_amd.lib(), ctypes.c_void_p(4104)
    need = lib.mia_blocknorm_ws_floats(2, 3, 16, 1)
    with pytest.raises(mia_amd.MiaError, match="16 bytes"):
        lib.mia_blocknorm_fwd(0, P, P, 2, 3, 16, None, None, 0, None, None, 1, P, None, 1e-6, P, P, odd, None)
    for ws, stats in ((odd, P), (P, odd)):
        with pytest.raises(mia_amd.MiaError, match="16 bytes"):
            lib.mia_blocknorm_bwd(0, P, P, P, P, stats, 2, 3, 16, None, None, 0, None, None, 1, P, ws, need, P, P, None, None, None, None, None, None, None)
