"""Norms before and after a residual branch fused with its gate and its residual scale, on the gfx950 kernels of
csrc/blocknorm.hip."""
import torch

from ._lib import nodes
from .ops import _DT

_KINDS = {None: 0, "rms": 1, "layer": 2}


def gated_residual_norm(x, f, scale=None, gate=None, post=None, post_weight=None, post_bias=None, pre="rms", pre_weight=None,
                        pre_bias=None, eps=1e-6):
    """The end of one residual branch and the norm in front of the next one, in one pass over the data:

        u = norm_post(f)                 (f itself for post=None)
        y = x + scale * gate * u
        z = norm_pre(y)                  (None for pre=None)

    x, f [..., C]: the residual stream and the branch's output, fp32 or bf16, the same shape and type. scale [C] and gate
    [x.shape[0], C] (one row per image, broadcast over its tokens) are optional; post and pre name the norms, "rms" or
    "layer", each with a weight [C] and optionally a bias [C] (population variance over C, eps added to it). Parameters and
    gate are fp32. All arithmetic is fp32: z is formed from y before y is rounded to the tensors' type. Returns (y, z);
    differentiable (once, backward) in every tensor. C <= 8192."""
    if post not in _KINDS or pre not in _KINDS:
        raise ValueError(f"norms are 'rms', 'layer' or None (got post={post!r}, pre={pre!r})")
    dtype, shape = x.dtype, x.shape
    if dtype not in _DT or f.dtype != dtype:
        raise TypeError(f"x and f are both fp32 or both bf16 (got {dtype}, {f.dtype})")
    if len(shape) < 1 or f.shape != shape:
        raise ValueError(f"x and f have one shape [..., C] (got {tuple(shape)}, {tuple(f.shape)})")
    C = shape[-1]
    if not 1 <= C <= 8192:
        raise ValueError(f"C must be 1..8192 (got {C})")
    for kind, w, b, which in ((post, post_weight, post_bias, "post"), (pre, pre_weight, pre_bias, "pre")):
        if (kind is None) != (w is None) or (kind is None and b is not None):
            raise ValueError(f"{which}={kind!r} needs {'no weight and no bias' if kind is None else which + '_weight'}")
    if gate is not None and len(shape) < 2:
        raise ValueError("a gate needs x of at least two dimensions")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative (got {eps})")
    device = x.get_device()
    for name, t, want in (("scale", scale, (C,)), ("gate", gate, (shape[0], C)), ("post_weight", post_weight, (C,)), ("post_bias", post_bias, (C,)),
                          ("pre_weight", pre_weight, (C,)), ("pre_bias", pre_bias, (C,))):
        if t is None:
            continue
        if t.shape != want or t.dtype != torch.float32:
            raise ValueError(f"{name} must be fp32 {want} (got {t.dtype} {tuple(t.shape)})")
        if t.get_device() != device:
            raise RuntimeError(f"gated_residual_norm needs its tensors on one MI355X device; there is no CPU path ({name} on {t.device}, x on {x.device})")
    if device < 0 or f.get_device() != device:
        raise RuntimeError(f"gated_residual_norm needs its tensors on one MI355X device; there is no CPU path (x on {x.device}, f on {f.device})")
    return nodes().residual(x, f, scale, gate, post_weight, post_bias, pre_weight, pre_bias, _KINDS[post], _KINDS[pre], eps)
